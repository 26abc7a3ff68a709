"""Which context the native calls are given, and what is done where their extension cannot be used: nothing here reaches a GPU."""
import ctypes
import types

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
