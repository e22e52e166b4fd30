"""The guard-page allocator (scripts/probes/guard_alloc.cpp) without an overrun: where it puts a tensor is arithmetic, checked here on the host, and a correct
program stays correct under it.  No program of this tree overruns a tensor to see what happens."""
import ctypes as C
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def layout():
    import torch  # noqa: F401  (one HIP runtime in the process: torch's)
    from fastvideo_amd import _build
    f = C.CDLL(_build.build_guard()).guard_layout
    f.argtypes, f.restype = [C.c_size_t, C.c_size_t, C.c_size_t, C.c_int] + [C.POINTER(C.c_size_t)] * 3, None

    def call(size, gran, align, front):
        out = [C.c_size_t() for _ in range(3)]
        f(size, gran, align, front, *(C.byref(x) for x in out))
        return tuple(x.value for x in out)
    return call


@pytest.mark.parametrize("gran", [4096, 2 << 20])
@pytest.mark.parametrize("align", [1, 16, 256])
def test_a_tensor_ends_where_its_mapping_ends(layout, gran, align):
    for size in (1, 2, 15, 16, 17, 8192, gran - align, gran - 1, gran, gran + 1, 3 * gran - 1, 5 * 2**30 + 7):
        mapped, reserved, offset = layout(size, gran, align, 0)
        assert mapped % gran == 0 and reserved == mapped + gran, "whole granules, one unmapped granule behind them"
        assert offset % align == 0 and offset + size <= mapped < offset + size + align, "the first aligned access behind the tensor is outside the mapping"
        assert mapped - gran < size + align
        assert layout(size, gran, align, 1) == (mapped, reserved, 0)


def test_no_program_overruns_on_purpose():
    """The self-test takes no arguments (the call below ends before anything touches a device)."""
    r = subprocess.run([sys.executable, "scripts/guard_selftest.py", "oob"], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert r.returncode != 0 and "takes no arguments" in r.stderr
    sweep = open(os.path.join(ROOT, "scripts", "guard_sweep.sh")).read()
    assert "guard_selftest.py oob" not in sweep and sweep.count("exit $rc") == 3
    assert not [f for f in ("sp_abort_hunt.py", "oob_probe.py", "uninit_probe.py") if os.path.exists(os.path.join(ROOT, "scripts", f))]


@pytest.mark.gpu
def test_a_correct_program_stays_correct():
    r = subprocess.run([sys.executable, "scripts/guard_selftest.py"], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and "mismatches 0" in r.stdout, r.stdout[-2000:]
