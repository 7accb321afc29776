"""The torch operators of csrc/_bindings.so: group norm, embedding and expert rows over the C ABI, with their gradients.

Like the library itself the module is built ahead of time and has no fallback.  It is loaded with ``nn``; where that
fails, the operators raise the error when they are asked for, and a program of convolutions alone runs without them."""
from __future__ import annotations

import importlib.util
import os

from . import _lib  # the library first: the module links to it

PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "_bindings.so")
_OPERATORS = ("group_rows", "group_norm", "embedding", "expert_sort", "expert_dispatch", "expert_combine")


def _load():
    if not os.path.exists(PATH):
        raise ImportError(f"{PATH} is missing: build it with `python torchsparse_b200/csrc/build.py`. There is no PyTorch "
                          "fallback for these operators.")
    import torch  # noqa: F401  (its libraries have to be loaded before the module's)

    spec = importlib.util.spec_from_file_location("_bindings", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


try:
    _error, _module = None, _load()
    globals().update({name: getattr(_module, name) for name in _OPERATORS})
except ImportError as error:
    _error = error


def __getattr__(name: str):      # of what was not loaded
    if name in _OPERATORS:
        raise ImportError(f"the torch operators of torchsparse_b200 could not be loaded: {_error}") from _error
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
