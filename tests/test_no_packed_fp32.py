"""No kernel of the built library holds a packed-fp32 instruction (v_pk_add / mul / fma_f32): such results have been wrong beside a foreign MFMA stream, and
hipcc makes them by itself from ordinary float code unless the feature is off for every file.  Reads this build's own code objects."""
import os
import re
import subprocess

import pytest

import test_register_claims as claims


def packed_in(objdump, path):
    text = subprocess.run([objdump, "-d", "--mcpu=gfx950", path], capture_output=True, text=True, check=True).stdout
    return len(re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text)), text.count("v_mfma_")


def test_the_library_holds_no_packed_fp32(tmp_path):
    objcopy, objdump = os.path.join(claims.LLVM, "llvm-objcopy"), os.path.join(claims.LLVM, "llvm-objdump")
    if not (os.path.exists(claims.LIB) and os.path.exists(objcopy) and os.path.exists(objdump)):
        pytest.skip("library not built or no llvm tools")
    fat = str(tmp_path / "fat.bin")
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", claims.LIB, str(tmp_path / "copy.so")], check=True)
    packed = mfma = 0
    for i, elf in enumerate(claims._device_elfs(open(fat, "rb").read())):
        f = tmp_path / f"co{i}.elf"
        f.write_bytes(elf)
        p, m = packed_in(objdump, str(f))
        packed, mfma = packed + p, mfma + m
    assert mfma > 10_000, "the disassembly holds the kernels"
    assert packed == 0


def test_every_source_is_built_without_them():
    from fastvideo_amd import _build
    assert set(_build.SOURCES + _build.PROBE_SOURCES) <= set(_build.NO_PACKED_FP32)
