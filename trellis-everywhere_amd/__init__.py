"""trellis-everywhere_amd: MI355X (gfx950) trellis packed-linear decode-matmul.

A drop-in for the reference's packed linear (web/packed.js PackedOps.linear, Python
mirror scripts/run_packed_headless.py:87-99): y = restore(decode(bits)) @ x over the
reference's packed K-bit trellis format (scripts/export_packed.py).

The directory name contains a hyphen, so import it with importlib:
    te = importlib.import_module("trellis-everywhere_amd")
"""
from . import _capi
from ._capi import TrellisError, TrellisLibraryMissing
from .format import PackedRecord, fit_block, read_packed, write_packed

__all__ = ["PackedRecord", "read_packed", "write_packed", "fit_block", "TrellisError",
           "TrellisLibraryMissing", "PackedLinear", "PackedGroup", "PackedOps", "load_packed",
           "encode_tiles", "library", "TrellisLinear", "TrellisGroupLinear", "swap_linears",
           "rms_norm", "residual_norm", "append_kv", "paged_attention", "evict_kv", "PagedKVCache"]


def library():
    """The loaded libtrellis_amd.so (raises TrellisLibraryMissing when not built)."""
    return _capi.load()


# torch-dependent pieces load lazily so the format tools import without torch
_LAZY = {"packed_linear": ("PackedLinear", "PackedGroup", "PackedOps", "load_packed", "encode_tiles"),
         "modules": ("TrellisLinear", "TrellisGroupLinear", "swap_linears"),
         "norms": ("rms_norm", "residual_norm"),
         "kv_cache": ("append_kv", "paged_attention", "evict_kv", "PagedKVCache")}


def __getattr__(name):
    for module, names in _LAZY.items():
        if name in names:
            import importlib
            value = getattr(importlib.import_module("." + module, __name__), name)
            globals()[name] = value   # the next access is a plain one
            return value
    raise AttributeError(name)
