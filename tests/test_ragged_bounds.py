"""The attention kernels' row, table and key addresses on the CPU (tests/ragged_bounds.cpp over the kernels' own fastvideo_amd/csrc/ragged_walk.h), built with
the address and undefined-behaviour sanitizers of the host compiler."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("bounds") / "ragged_bounds")
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(HERE, "ragged_bounds.cpp"), "-o", exe], check=True)
    return exe


@pytest.mark.parametrize("seed", range(4))
def test_every_address_lies_in_its_tensor(program, seed):
    r = subprocess.run([program, str(seed), "2500"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "2500 cases hold" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
