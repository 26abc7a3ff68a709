"""Which context the native calls are given, and what is done where their extension cannot be used: nothing here reaches a GPU."""
import ctypes
import os
import types
import warnings

import pytest
import torch

from frisk_b200 import calls, capi


@pytest.fixture
def native():
    if not calls.path(torch.__version__).exists():
        pytest.skip("built without native calls")
    if not calls._loaded:
        calls._load()
    return calls


def test_a_call_takes_the_context_that_is_there(native, monkeypatch):
    """Not one that has been closed, or has given place to another: its memory is free."""
    def made(address):  # (a context has its handle there, and None once it is closed)
        return types.SimpleNamespace(_h=ctypes.c_void_p(address))

    held = native.execute._contexts
    assert native.address(7) is None
    first, second = made(0x1000), made(0x2000)
    monkeypatch.setitem(held, 7, first)
    assert native.address(7) == 0x1000 and native.address(8) is None
    first._h = None
    assert native.address(7) is None
    held[7] = second
    assert native.address(7) == 0x2000
    del held[7]
    assert native.address(7) is None
    held[7] = object()
    assert native.address(7) is None
    for bad in (None, "7", 7.0, 1 << 70, -1):
        assert native.address(bad) is None
    closed = capi.Context.__new__(capi.Context)
    closed._h = ctypes.c_void_p(None)
    held[7] = closed
    assert native.address(7) is None
    closed._h = None


FUNCTIONS = ("verify", "change", "keep", "copy", "adapters", "write", "address")


@pytest.fixture
def unloaded(monkeypatch):
    """As before the first call."""
    monkeypatch.setattr(calls, "_loaded", False)
    for name in FUNCTIONS:
        monkeypatch.setattr(calls, name, calls._unknown)


@pytest.mark.parametrize("content", [b"", b"no library", b"\x7fELF" + bytes(60)], ids=["empty", "text", "header"])
def test_an_extension_that_cannot_be_loaded(unloaded, monkeypatch, tmp_path, content):
    """Calls are then made in Python, from the first one on; it is said once."""
    file = tmp_path / "_calls_cut_short.so"
    file.write_bytes(content)
    context = object()
    monkeypatch.setattr(calls, "path", lambda version: file)
    monkeypatch.setitem(calls.execute._contexts, 5, context)
    with pytest.warns(RuntimeWarning, match="cannot be loaded"):
        assert calls.context_for(5) is context
    assert all(getattr(calls, name) is calls._unknown for name in FUNCTIONS)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert calls.context_for(5) is context


def test_an_extension_of_another_source_does_not_stay(monkeypatch, tmp_path):
    """Where it cannot be built again (no compiler, no headers), an older one goes; one that is up to date stays."""
    from frisk_b200 import build
    file = tmp_path / "_calls.so"
    monkeypatch.setattr(calls, "path", lambda version: file)
    monkeypatch.setattr(build.shutil, "which", lambda name: None if name == "g++" else "/bin/" + name)
    monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    file.write_bytes(b"x")
    os.utime(file, (1, 1))
    assert build.build_calls() is None and not file.exists()
    file.write_bytes(b"x")
    later = max(p.stat().st_mtime for p in (build.CSRC / "calls.cpp", build.INCLUDE / "frisk_b200.h")) + 5
    os.utime(file, (later, later))
    assert build.build_calls() == file and file.exists()
    assert build.build_calls(force=True) is None and not file.exists()


def test_an_extension_of_another_source(unloaded, monkeypatch):
    """One that takes other functions than this package has."""
    if not calls.path(torch.__version__).exists():
        pytest.skip("built without native calls")
    context = object()
    monkeypatch.setattr(calls, "_FUNCTIONS", calls._FUNCTIONS[:-1])
    monkeypatch.setitem(calls.execute._contexts, 5, context)
    with pytest.warns(RuntimeWarning, match="cannot be loaded"):
        assert calls.context_for(5) is context
    assert all(getattr(calls, name) is calls._unknown for name in FUNCTIONS)
