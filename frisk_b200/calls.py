"""Loads ``_calls`` (``csrc/calls.cpp``): the usual calls of the serving operators, made natively.

``verify``, ``change``, ``keep``, ``copy``, ``adapters`` and ``write`` give an operator's results, an error number of the C ABI, or None where the Python functions
have to look for themselves (and report what is wrong, if anything is): always where the extension is not built for this interpreter
and this torch or cannot be loaded, which costs time and nothing else, and where the device has no open context.  ``address`` gives the one that calls would take.
"""
import ctypes
import importlib.machinery
import importlib.util
import os
import pathlib
import warnings

from . import capi, execute

_FUNCTIONS = ("draft_verify", "cache_fork", "cache_grow", "cache_compact", "cache_pages_workspace_bytes", "cache_copy", "cache_keep", "adapter_gemm",
              "adapter_workspace_bytes", "cache_write")


def path(torch_version):
    """Where the extension for that torch is: the suffix names the interpreter's ABI, the name torch's."""
    name = "_calls_" + "".join(c if c.isalnum() else "_" for c in torch_version)
    return pathlib.Path(__file__).resolve().parent / "lib" / (name + importlib.machinery.EXTENSION_SUFFIXES[0])


def _unknown(*_):
    return None


verify = change = keep = copy = adapters = write = address = _unknown
_loaded = False


def context_for(device):
    """The device's context; once one has been made, calls may be made natively, each with the context that is there then."""
    if not _loaded:
        _load()
    return execute.context_for(device)


def _load():
    global verify, change, keep, copy, adapters, write, address, _loaded
    import torch
    _loaded = True
    file = path(torch.__version__)
    if not file.exists():
        return
    lib = capi.load()
    loader = importlib.machinery.ExtensionFileLoader("_calls", os.fspath(file))
    try:
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_calls", loader))
        loader.exec_module(module)
        made = module.verify, module.change, module.keep, module.copy, module.adapters, module.write, module.context
        module.library(execute._contexts, *(ctypes.cast(getattr(lib, "frisk_b200_" + name), ctypes.c_void_p).value for name in _FUNCTIONS))
    except (ImportError, OSError, AttributeError, TypeError, ValueError) as e:  # (built against another torch of that version, from another source, or cut short)
        warnings.warn(f"frisk_b200: {file.name} cannot be loaded, calls are made in Python: {e}", RuntimeWarning, stacklevel=3)
        return
    verify, change, keep, copy, adapters, write, address = made


def result(r, device):
    """What a native call gave, unless it is an error."""
    if type(r) is int:
        capi.raise_for(r, execute.context_for(device).handle)
    return r
