"""warpforth_b200 -- B200 (sm_100a) replacement for WarpForth's attention hot path.

The kernels and the C ABI live in libwfattn (``csrc/``, ``include/wfattn.h``);
this package holds the Python side of the drop-in boundary:

* ``warpforth.AttentionKernel`` -- the reference's demo/warpforth.py interface;
* ``warpforth.attention`` / ``warpforth.decode`` -- batched prefill and decode;
* ``cache`` -- a key/value cache in f32, bf16, e4m3 or 4 bits: writing and reading its rows,
  attention of a tree of drafted tokens over it, keeping the accepted ones;
* ``gpt2`` -- the GPT-2 attention patch of demo/gpt2_generate.py, batched;
* ``sharded`` -- head-sharded multi-GPU prefill; the kernel stores O into every rank's
  buffer (``peer``: CUDA IPC mappings over NVLink), or NCCL all-gathers it.
"""

from __future__ import annotations

__all__ = ["AttentionKernel", "attention", "attention_gather",
           "attention_gather_ptrs", "decode", "DecodeWorkspace", "KVCache", "cache_write",
           "cache_read", "cache_keep", "tree_decode", "tree_words"]
_CACHE = ("KVCache", "cache_write", "cache_read", "cache_keep", "tree_decode", "tree_words")


def __getattr__(name):  # lazy: importing the package does not import torch
    if name not in __all__:
        raise AttributeError(name)
    from . import cache, warpforth

    value = getattr(cache if name in _CACHE else warpforth, name)
    globals()[name] = value  # the next look-up finds it
    return value
