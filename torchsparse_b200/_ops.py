"""The torch operators of csrc/_bindings.so: group norm, embedding and expert rows over the C ABI, with their gradients.

Like the library itself the module is built ahead of time and has no fallback: without it the import fails."""
from __future__ import annotations

import importlib.util
import os

from . import _lib  # the library first: the module links to it

PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "_bindings.so")


def _load():
    if not os.path.exists(PATH):
        raise ImportError(f"{PATH} is missing: build it with `python torchsparse_b200/csrc/build.py`. There is no PyTorch "
                          "fallback for these operators.")
    import torch  # noqa: F401  (its libraries have to be loaded before the module's)

    spec = importlib.util.spec_from_file_location("_bindings", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


_module = _load()
group_rows = _module.group_rows
group_norm = _module.group_norm
embedding = _module.embedding
expert_sort = _module.expert_sort
expert_dispatch = _module.expert_dispatch
expert_combine = _module.expert_combine
