"""The build's torch front end on boxes that cannot have it or had another torch."""
import sysconfig

import pytest

from blackwell_b200 import build


@pytest.fixture
def no_compiler(monkeypatch):
    def run(cmd, **kw):
        raise AssertionError(f"compiles: {cmd}")

    monkeypatch.setattr(build.subprocess, "run", run)


def test_front_is_left_out_without_headers(monkeypatch, tmp_path, no_compiler, capsys):
    """Without Python's headers the library's build succeeds, as before there was a front end."""
    monkeypatch.setattr(build, "FRONT", tmp_path / "_front.so")
    monkeypatch.setattr(sysconfig, "get_paths", lambda *a, **k: {"include": str(tmp_path)})
    assert build.build_front() is None
    assert "Python.h" in capsys.readouterr().err
    for p in ("OUT", "HARNESS"):
        (tmp_path / p).touch()
        monkeypatch.setattr(build, p, tmp_path / p)
    assert build.up_to_date()
    assert build.build() == build.OUT           # nothing left to do


def test_up_to_date_wants_the_front_where_it_can_be_built(monkeypatch, tmp_path):
    for p in ("OUT", "HARNESS"):
        (tmp_path / p).touch()
        monkeypatch.setattr(build, p, tmp_path / p)
    monkeypatch.setattr(build, "FRONT", tmp_path / "_front.so")
    assert build.front_lacks() is None and not build.up_to_date()


def test_front_of_another_torch_is_noticed(monkeypatch):
    """By the build, which makes it again, and by the first call, which says so."""
    import torch

    import blackwell_b200 as bw
    from blackwell_b200 import cache
    assert build.front_fits()
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    assert not build.front_fits() and not build.up_to_date()
    monkeypatch.setattr(cache, "_front", None)
    with pytest.raises(RuntimeError, match="built with torch"):
        bw.rope(torch.zeros(3, 4, 64), None, torch.zeros(8, 64))
