"""The build's own steps, without compiling."""
import importlib.util
import os

import pytest

from text_guided_face_recognition_amd import build


@pytest.fixture
def recorded(monkeypatch, tmp_path):
    """A build into an empty folder whose commands only leave empty files."""
    for name in ("LIB", "FRONT", "STAMP"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(build, "OBJ_DIR", str(tmp_path / "obj"))
    ran = []

    def run(cmd, verbose):
        ran.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
    monkeypatch.setattr(build, "_run", run)
    return ran


@pytest.mark.parametrize("torch_there", [True, False], ids=["torch", "no torch"])
def test_build_with_and_without_torch(recorded, monkeypatch, torch_there):
    """The kernel library needs no torch; the front-end is built where it is."""
    find = importlib.util.find_spec
    if not torch_there:
        monkeypatch.setattr(importlib.util, "find_spec",
                            lambda name, *a: None if name == "torch" else find(name, *a))
    assert build.stale()
    build.build()
    outputs = [c[c.index("-o") + 1] for c in recorded]
    assert (build.FRONT + ".tmp" in outputs) == torch_there
    assert build.LIB + ".tmp" in outputs and len(outputs) == len(build.sources()) + 1 + torch_there
    assert os.path.exists(build.LIB) and os.path.exists(build.FRONT) == torch_there
    assert not build.stale()
