"""What the build compiles, without compiling: the C library needs nvcc alone, and torch's
face of the serving operators is built against the torch that is there."""
import subprocess

import pytest

from actune_b200 import build as B


@pytest.fixture
def fake(tmp_path, monkeypatch):
    """A package folder of its own, and a compiler that writes its output and is recorded."""
    csrc = tmp_path / "csrc"
    (csrc / "torch").mkdir(parents=True)
    (csrc / "a.cu").write_text("")
    (csrc / "torch" / "serving.cpp").write_text("")
    for name, path in dict(PKG=tmp_path, CSRC=csrc, INCLUDE=tmp_path / "include", BUILD=tmp_path / "_build",
                           LIB=tmp_path / "lib.so", TORCH_SOURCE=csrc / "torch" / "serving.cpp",
                           TORCH_MODULE=tmp_path / "_serving.so").items():
        monkeypatch.setattr(B, name, path)
    monkeypatch.setattr(B, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    ran = []

    def run(cmd, **kw):
        out = cmd[cmd.index("-o") + 1]
        ran.append(out.rsplit("/", 1)[1])
        open(out, "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(B.subprocess, "run", run)

    def built(**kw):
        ran.clear()
        B.build(**kw)
        return sorted(ran)

    return built


def test_everything_once(fake):
    assert fake() == ["_serving.so", "a.o", "lib.so"]
    assert fake() == []


def test_the_library_builds_without_torch(fake, monkeypatch, capsys):
    monkeypatch.setattr(B, "torch_installed", lambda: None)
    assert fake() == ["a.o", "lib.so"]
    assert "_serving.so" in capsys.readouterr().err


def test_the_library_alone(fake):
    assert fake(library_only=True) == ["a.o", "lib.so"]
    assert fake() == ["_serving.so"]


def test_another_torch_gets_another_module(fake, monkeypatch):
    fake()
    monkeypatch.setattr(B, "torch_installed", lambda: "9.9 at another place")
    assert fake() == ["_serving.so"]
    assert fake() == []
