"""lazyweights_amd: MI355X-native decode-on-demand weight path of LazyWeights.

Coded K-quant matrices (lane-interleaved Huffman bundles) are decoded on gfx950 and fused into the batch-1 GEMV and
the skinny verify GEMM, behind the reference runtime's C-ABI (include/lazyweights_amd.h).
"""
from ._lib import LIB_PATH, last_error, load_library  # noqa: F401
from .runtime import Runtime  # noqa: F401

_TORCH = {"Batch": "attention", "KvCache": "attention", "KvCache8": "attention", "Pages": "pages"}


def __getattr__(name):
    """Batch, KvCache, KvCache8 and Pages when they are first asked for: they need torch, which takes longer to import than all
    else here."""
    if name in _TORCH:
        from importlib import import_module
        return getattr(import_module("." + _TORCH[name], __name__), name)
    raise AttributeError("module %r has no attribute %r" % (__name__, name))


def __dir__():
    return sorted(set(globals()) | set(_TORCH))
