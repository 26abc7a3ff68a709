"""Loads ``_calls`` (``csrc/calls.cpp``): the usual calls of the serving operators, made natively.

``verify``, ``change``, ``keep``, ``copy``, ``adapters`` and ``write`` give an operator's results, an error number of the C ABI, or None where the Python functions
have to look for themselves (and report what is wrong, if anything is): always where the extension is not built for this interpreter
and this torch, which costs time and nothing else.
"""
import ctypes
import importlib.machinery
import importlib.util
import os
import pathlib

from . import capi, execute

_FUNCTIONS = ("draft_verify", "cache_fork", "cache_grow", "cache_compact", "cache_pages_workspace_bytes", "cache_copy", "cache_keep", "adapter_gemm",
              "adapter_workspace_bytes", "cache_write")


def path(torch_version):
    """Where the extension for that torch is: the suffix names the interpreter's ABI, the name torch's."""
    name = "_calls_" + "".join(c if c.isalnum() else "_" for c in torch_version)
    return pathlib.Path(__file__).resolve().parent / "lib" / (name + importlib.machinery.EXTENSION_SUFFIXES[0])


def _unknown(*_):
    return None


verify = change = keep = copy = adapters = write = _unknown
_register, _known = None, set()


def context_for(device):
    """The device's context; once it has been made, calls there may be made natively."""
    context = execute.context_for(device)
    if device not in _known:
        _known.add(device)
        _know(device, context)
    return context


def _know(device, context):
    global verify, change, keep, copy, adapters, write, _register
    if _register is None:
        import torch
        file = path(torch.__version__)
        if not file.exists():
            _register = _unknown
            return
        loader = importlib.machinery.ExtensionFileLoader("_calls", os.fspath(file))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_calls", loader))
        loader.exec_module(module)
        lib = capi.load()
        module.library(*(ctypes.cast(getattr(lib, "frisk_b200_" + name), ctypes.c_void_p).value for name in _FUNCTIONS))
        verify, change, keep, copy, adapters, write, _register = module.verify, module.change, module.keep, module.copy, module.adapters, module.write, module.context
    _register(device, context.handle.value)


def result(r, device):
    """What a native call gave, unless it is an error."""
    if type(r) is int:
        capi.raise_for(r, execute.context_for(device).handle)
    return r
