"""The paged-cache calls without the _fastcall extension: a warning, not an error."""

import builtins

import pytest

import quartz_b200.device as qd


def test_missing_extension_warns(monkeypatch):
    real = builtins.__import__

    def without(name, globals=None, locals=None, fromlist=(), level=0):
        if "_fastcall" in (fromlist or ()):
            raise ImportError("not built")
        return real(name, globals, locals, fromlist, level)

    monkeypatch.setattr(qd, "_fast", None)
    monkeypatch.setattr(builtins, "__import__", without)
    with pytest.warns(RuntimeWarning, match="_fastcall"):
        qd._bind_fast(0)
    assert qd._fast is None
