"""What quartz_b200.build builds, keeps and refuses of the _fastcall extension."""

import subprocess

import pytest

import quartz_b200.device as qd
from quartz_b200 import build

pytest.importorskip("torch")


@pytest.mark.parametrize("error", [
    subprocess.CalledProcessError(1, ["g++"]), FileNotFoundError("g++"), ImportError("no torch"),
    RuntimeError("nvcc not found")])
def test_the_library_is_built_without_the_extension(monkeypatch, error):
    made = []

    def no_extension(force=False):
        assert made == ["library"]            # the library comes first
        raise error

    monkeypatch.setattr(build, "build_library", lambda *a: made.append("library"))
    monkeypatch.setattr(build, "build_fastcall", no_extension)
    with pytest.warns(RuntimeWarning, match="_fastcall.so is not built"):
        assert build.build() == build.OUT


def test_a_failed_library_build_is_an_error(monkeypatch):
    def fails(*a):
        raise subprocess.CalledProcessError(1, ["nvcc"])

    monkeypatch.setattr(build, "build_library", fails)
    with pytest.raises(subprocess.CalledProcessError):
        build.build()


def test_an_extension_of_another_torch_is_built_anew(monkeypatch, tmp_path):
    build.build_fastcall()
    assert build.fast_up_to_date() and build.fast_stamp() == build.fast_tag()
    import torch
    assert f"torch={torch.__version__};" in build.fast_tag()
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    build.build_fastcall()
    assert not ran
    monkeypatch.setattr(torch, "__version__", "9.9")
    assert not build.fast_up_to_date()
    build.build_fastcall()
    assert len(ran) == 1 and any("torch=9.9;" in x for x in ran[0])
    # nothing that can be read, nothing there
    other = tmp_path / "other.so"
    assert build.fast_stamp(other) == ""
    other.write_bytes(b"no library")
    assert build.fast_stamp(other) == ""


def test_an_extension_of_another_torch_is_not_loaded(monkeypatch):
    import builtins
    real = builtins.__import__

    def loads(name, globals=None, locals=None, fromlist=(), level=0):
        assert "_fastcall" not in (fromlist or ()), "loaded"
        return real(name, globals, locals, fromlist, level)

    monkeypatch.setattr(qd, "_fast", None)
    monkeypatch.setattr(build, "fast_tag", lambda: "torch=9.9;python=x;cxx11=1")
    monkeypatch.setattr(builtins, "__import__", loads)
    with pytest.warns(RuntimeWarning, match="built for torch=.*this is torch=9.9"):
        qd._bind_fast(0)
    assert qd._fast is None
