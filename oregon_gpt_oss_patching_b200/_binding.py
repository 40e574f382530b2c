"""Loads the extension module of the training-step operators (``csrc/train_binding.cpp``) and gives it the library.

There is deliberately no fallback: if the module or the library cannot be loaded, a ``RuntimeError`` is raised.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import threading

import torch  # noqa: F401  (the module links against torch's libraries, which this import loads)

from . import _cabi
from . import build as _build

_NAMES = ("b200attn_strerror", "b200moe_router_topk", "b200moe_router_topk_bwd", *_cabi.TRAIN_EXPORTS)
_lock = threading.Lock()
_module = None


def load():
    """Load (once) and return the extension module, calling the library that ``_cabi.load`` returns."""
    global _module
    if _module is not None:
        return _module
    lib = _cabi.load()
    with _lock:
        if _module is not None:
            return _module
        path = _build.binding_path()
        if not os.path.exists(path):
            raise RuntimeError(f"{path} not found: the extension module has not been built "
                               "(run `python -m oregon_gpt_oss_patching_b200.build`); there is no fallback path")
        loader = importlib.machinery.ExtensionFileLoader("_train_binding", path)
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_train_binding", loader))
        loader.exec_module(module)
        module.set_library({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _NAMES})
        _module = module
    return _module
