"""The compiled Python binding of the stateless operators (``csrc/bind.cpp``), loaded at its first use."""
from __future__ import annotations

import importlib.machinery
import importlib.util
import os

from . import _lib

PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "_wisp_bind.so")


def _load():
    _lib.lib()                          # the library it is linked with; raises where that is missing
    if not os.path.exists(PATH):
        raise ImportError(f"wisp_b200 Python binding missing at {PATH}; build it with `python -m wisp_b200.build`")
    import torch  # noqa: F401  (its libraries)
    loader = importlib.machinery.ExtensionFileLoader("_wisp_bind", PATH)
    spec = importlib.util.spec_from_file_location("_wisp_bind", PATH, loader=loader)
    module = importlib.util.module_from_spec(spec)
    loader.exec_module(module)
    return module


class _Native:
    def __getattr__(self, name):
        module = _load()
        self.__dict__.update({k: getattr(module, k) for k in dir(module) if not k.startswith("_")})
        return self.__dict__[name]


native = _Native()
