"""The native front end (fastvideo_amd/_launch.so) belongs to one torch and one Python: a build for another is stale however new its file is, and is not
used where it is loaded all the same.  Host code, no GPU."""
import os

import pytest
import torch

from fastvideo_amd import _build, _lib


@pytest.fixture
def built(tmp_path, monkeypatch):
    lib = tmp_path / "_launch.so"
    lib.write_bytes(b"x")
    monkeypatch.setattr(_build, "LAUNCH_LIB", str(lib))
    later = os.path.getmtime(str(lib)) + 10_000
    os.utime(str(lib), (later, later))   # newer than every source
    (tmp_path / "_launch.so.flags").write_text(_build._launch_stamp())
    return lib


def test_a_fresh_build_is_kept(built, monkeypatch):
    assert _build.launch_needs_build() is False
    assert _build.HERE not in _build._launch_stamp(), "the stamp holds in a copy of the tree too"
    monkeypatch.setattr(_build.subprocess, "run", lambda *a, **k: pytest.fail("built again"))
    assert _build.build_launch() == str(built)


def test_another_torch_makes_it_stale(built, monkeypatch):
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    assert _build.launch_needs_build() is True


def test_no_stamp_an_older_file_or_none_is_stale(built, tmp_path):
    os.utime(str(built), (1, 1))
    assert _build.launch_needs_build() is True
    os.utime(str(built), None)
    os.remove(str(built) + ".flags")
    assert _build.launch_needs_build() is True
    (tmp_path / "_launch.so.flags").write_text(_build._launch_stamp())
    os.remove(str(built))
    assert _build.launch_needs_build() is True


def test_a_module_for_another_torch_is_refused(monkeypatch):
    module = _lib.launch()
    assert module.made_for == _build.launch_made_for()
    monkeypatch.setattr(_lib, "_native", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(RuntimeError, match="built for torch .*this is torch 9.9.9"):
        _lib.launch()
    monkeypatch.undo()
    assert _lib.launch() is module
