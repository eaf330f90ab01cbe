"""Loads the binding of the C ABI's dense side (``csrc/dense_ops.cpp``): q/k norm with rotary positions, attention over
key intervals, and the 8-bit key/value cache.  The public functions are in ``models``."""

from __future__ import annotations

import importlib.util
import os

import torch  # noqa: F401  (the binding's symbols come from its libraries)

from . import _native

OPS_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_lib", "_dense_ops.so")

CACHE_BLOCK = 64  # tokens of a head that share a scale

_ops = None


def ops():
    """The binding; raises where it has not been built (there is no fallback)."""
    global _ops
    if _ops is None:
        if not os.path.exists(OPS_PATH):
            raise _native.BSAError(f"BSA binding not found at {OPS_PATH}; build it with "
                                   "`python longcat-video-mlx_b200/build.py` (there is no CPU fallback)")
        _native.lib()
        spec = importlib.util.spec_from_file_location("_dense_ops", OPS_PATH)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.load(_native.LIB_PATH, _native.BSAError)
        _ops = module
    return _ops
