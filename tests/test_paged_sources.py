"""What the sources and the built kernels of the batched-cache operators must not hold; no GPU needed."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastvideo_amd", "csrc")
FILES = ("attn_ragged.h", "attn_ragged.hip", "attn_rows.hip", "paged.hip")


def asm_statements(text):
    """The argument text of every asm statement."""
    for m in re.finditer(r"\basm\s+volatile\s*\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        yield text[m.end():at - 1]


def loads_into_registers(statement):
    """An asm load that returns its register before the data is there: a load that is neither LDS-DMA nor waited for in the same statement."""
    code = " ".join(re.findall(r'"((?:[^"\\]|\\.)*)"', statement.split("\n:")[0].split(" : ")[0]))
    load = re.search(r"\b(global|buffer|flat|scratch|s)_load_|\bds_read", code)
    return bool(load) and not re.search(r"\blds\b", code) and "s_waitcnt" not in code


@pytest.mark.parametrize("name", FILES)
def test_no_load_in_assembly_leaves_its_register_behind(name):
    text = open(os.path.join(CSRC, name)).read()
    assert not [s for s in asm_statements(text) if loads_into_registers(s)]


def test_the_rule_knows_such_a_load():
    assert loads_into_registers('"global_load_dwordx4 %0, %1, off" : "=a"(x) : "v"(p) : "memory"')
    assert not loads_into_registers('"global_load_dwordx4 %0, %1, off\\n\\ts_waitcnt vmcnt(0)" : "=a"(x) : "v"(p) : "memory"')
    assert not loads_into_registers('"buffer_load_dwordx4 %4, s[96:99], 0 offen lds" : : "v"(at) : "memory"')
    assert not loads_into_registers('"s_waitcnt vmcnt(0)" ::: "memory"')


def kernels(tmp_path, names):
    """name -> (registers of a wave, spilled vector registers, bytes of scratch) of the built library's kernels."""
    import subprocess
    import test_register_claims as claims
    objcopy, readelf = os.path.join(claims.LLVM, "llvm-objcopy"), os.path.join(claims.LLVM, "llvm-readelf")
    if not (os.path.exists(claims.LIB) and os.path.exists(objcopy) and os.path.exists(readelf)):
        pytest.skip("library not built or no llvm tools")
    fat, seen = str(tmp_path / "fat.bin"), {}
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", claims.LIB, str(tmp_path / "copy.so")], check=True)
    for i, elf in enumerate(claims._device_elfs(open(fat, "rb").read())):
        f = tmp_path / f"co{i}.elf"
        f.write_bytes(elf)
        for blk in subprocess.run([readelf, "--notes", str(f)], capture_output=True, text=True).stdout.split("- .agpr_count:")[1:]:
            name = re.search(r"\.name:\s+(\S+)", blk).group(1)
            if any(n in name for n in names):
                seen[name] = tuple(int(re.search(rf"\.{k}:\s+(\d+)", blk).group(1)) for k in ("vgpr_count", "vgpr_spill_count", "private_segment_fixed_size"))
    return seen


def test_rows_kernels_leave_no_room_beside_them(tmp_path):
    """One workgroup per compute unit (the two-stage ring, the 64-row tile): all 512 registers of a SIMD.  Two of them: half each."""
    ring = kernels(tmp_path, ["attn_rows_ring_kernel"])
    assert len(ring) == 6 and all(v == (512, 0, 0) for v in ring.values()), ring
    one = kernels(tmp_path, ["attn_rows_kernel"])
    assert len(one) == 6 and all(v == ((512 if "ILi4E" in n else 256), 0, 0) for n, v in one.items()), one


def test_the_block_kernel_keeps_its_state_in_registers(tmp_path):
    """All 512 of them, no spilled vector register and no scratch memory, paged and packed."""
    blocks = kernels(tmp_path, ["attn_ragged_kernel"])
    assert len(blocks) == 2 and all(v == (512, 0, 0) for v in blocks.values()), blocks
