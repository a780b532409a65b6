"""Key/value caches: writing and reading rows, attention of drafted trees, keeping accepted rows.

A ``KVCache`` holds the keys and values of a batch of sequences in one of four row formats
(``fmt``): ``"f32"``, ``"bf16"``, ``"e4m3"`` (8 bits a value and a power-of-two f32 scale a row) or
``"int4"`` (4 bits a value and a bf16 scale and minimum a row); include/wfattn.h defines them.
The reference has no cache (demo/README.md:45); GPT-2's generation with drafted tokens
(``gpt2.generate_drafted``) runs on these calls:

* ``cache_write`` puts new rows at given positions, quantising them;
* ``tree_decode`` attends from a tree of up to 64 drafted tokens (one token: a decode step) to the
  rows before it and to the nodes each one follows;
* ``cache_keep`` moves the accepted nodes' rows to the end of the sequence;
* ``cache_read`` returns rows as f32 or bf16, e.g. as keys and values of ``attention``.

Lengths and positions are int32 CUDA tensors, read on the device; an entry that points outside the
cache reads and writes nothing there, and ``device_status`` raises.  Every call runs on the current
stream of the cache's device.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from . import _lib
from .warpforth import _DTYPES, DecodeWorkspace, _ptr, _raw_stream, _require_cuda

_FORMATS = {"f32": (_lib.CACHE_F32, torch.float32), "bf16": (_lib.CACHE_BF16, torch.bfloat16),
            "e4m3": (_lib.CACHE_E4M3, torch.float8_e4m3fn), "int4": (_lib.CACHE_INT4, torch.uint8)}
_BY_DTYPE = {dtype: fmt for fmt, (_, dtype) in _FORMATS.items()}

MAX_NODES = 64  # of a drafted tree


class KVCache:
    """Keys and values of ``batch`` sequences, ``heads`` heads and up to ``max_len`` tokens.

    ``k`` and ``v`` are ``[batch, heads, max_len, head_dim]`` (``"int4"``: uint8, head_dim / 2, two
    values a byte, the even one low); ``k_scale`` and ``v_scale`` are None (``"f32"``, ``"bf16"``),
    f32 ``[batch, heads, max_len]`` (``"e4m3"``) or bf16 ``[batch, heads, max_len, 2]`` (``"int4"``:
    scale, minimum).  head_dim is 64 or 128.  The tensors start at zero; they belong to the object
    and are not to be replaced.
    """

    def __init__(self, batch: int, heads: int, max_len: int, head_dim: int = 64, *,
                 fmt: str = "bf16", device: torch.device | str = "cuda") -> None:
        if fmt not in _FORMATS:
            raise ValueError(f"fmt must be one of {sorted(_FORMATS)}, got {fmt!r}")
        if min(batch, heads, max_len) < 1 or head_dim not in (64, 128):
            raise ValueError("sizes must be >= 1 and head_dim 64 or 128")
        rows = (batch, heads, max_len)
        width = head_dim // 2 if fmt == "int4" else head_dim

        def scale():
            if fmt == "e4m3":
                return torch.zeros(rows, dtype=torch.float32, device=device)
            if fmt == "int4":
                return torch.zeros((*rows, 2), dtype=torch.bfloat16, device=device)
            return None

        k, v = (torch.zeros((*rows, width), dtype=_FORMATS[fmt][1], device=device)
                for _ in range(2))
        self._set(k, v, scale(), scale())

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
             v_scale: torch.Tensor | None = None) -> KVCache:
        """A cache over existing tensors, without a copy (e.g. some of a larger cache's sequences).

        Their format is told by ``k``'s dtype.  A head's rows are contiguous, and all the tensors
        have the same batch and head strides, counted in rows.
        """
        cache = cls.__new__(cls)
        cache._set(k, v, k_scale, v_scale)
        return cache

    def _set(self, k, v, k_scale, v_scale) -> None:
        for name, t in (("k", k), ("v", v)):
            _require_cuda(name, t)
            if t.dim() != 4 or t.dtype not in _BY_DTYPE:
                raise ValueError(f"{name} must be [batch, heads, max_len, row] of float32, bfloat16, "
                                 "float8_e4m3fn or uint8")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must have one shape and dtype")
        fmt = _BY_DTYPE[k.dtype]
        batch, heads, max_len, width = k.shape
        rows = (batch, heads, max_len)
        scaled = fmt in ("e4m3", "int4")
        parts = [("k", k, width), ("v", v, width)]
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if not scaled:
                if t is not None:
                    raise ValueError(f"an {fmt} cache has no {name}")
                continue
            _require_cuda(name, t)
            shape = rows if fmt == "e4m3" else (*rows, 2)
            dtype = torch.float32 if fmt == "e4m3" else torch.bfloat16
            if t.shape != shape or t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype} of shape {shape}")
            parts.append((name, t, 1 if fmt == "e4m3" else 2))
        strides = set()
        for name, t, unit in parts:
            if t.device != k.device:
                raise ValueError("the cache's tensors must be on one device")
            st = t.stride()
            if (t.dim() == 4 and st[3] != 1 and t.shape[3] > 1) or \
                    (max_len > 1 and st[2] != unit):
                raise ValueError(f"{name}: the rows of a head must be contiguous")
            if (batch > 1 and st[0] % unit) or (heads > 1 and st[1] % unit):
                raise ValueError(f"{name}: batch and head strides must be whole rows")
            strides.add((st[0] // unit if batch > 1 else 0, st[1] // unit if heads > 1 else 0))
        if len(strides) != 1:
            raise ValueError("the cache's tensors must have the same strides, counted in rows")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.fmt, self.device = fmt, k.device
        self.batch, self.heads, self.max_len = rows
        self.head_dim = 2 * width if fmt == "int4" else width
        if self.head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {self.head_dim}")
        sb, sh = strides.pop()
        self._c = _lib.Cache(_FORMATS[fmt][0], self.head_dim, batch, heads, max_len, sb, sh,
                             _ptr(k), _ptr(v), _ptr(k_scale) if scaled else None,
                             _ptr(v_scale) if scaled else None)
        # what every call needs, looked up once
        self._lib = _lib.load()
        self._at = ctypes.addressof(self._c)
        self._index = k.get_device()
        self._batch_shape = (batch,)
        self._new = {t: torch.empty(0, dtype=t, device=k.device).new_empty for t in _DTYPES}
        self._tree_bytes: dict[tuple, int] = {}  # workspace sizes by call shape


_strides = struct.Struct("3q").pack  # of a 4-d tensor, as the library takes them
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _run(cache: KVCache, fn, *args) -> None:
    """fn(cache, *args, stream) with the cache's device current."""
    index = cache._index
    if index == _current_device():
        status = fn(cache._at, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(cache._at, *args, _raw_stream(index))
    if status:
        _lib.check(status)


def _ints(name: str, t: torch.Tensor, shape, cache: KVCache,
          dtype: torch.dtype = torch.int32) -> int:
    """The address of integers with a unit last stride on the cache's device."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or \
            t.get_device() != cache._index or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} of shape {tuple(shape)} on {cache.device}")
    if t.stride(-1) != 1 and shape[-1] > 1:
        raise ValueError(f"{name} must have a unit last stride")
    return t.data_ptr()


def _rows(name: str, t: torch.Tensor, shape, dtype, cache: KVCache) -> bytes:
    """The strides of f32 or bf16 rows of this shape on the cache's device."""
    if not isinstance(t, torch.Tensor) or t.shape != shape or t.get_device() != cache._index:
        raise ValueError(f"{name} must be of shape {tuple(shape)} on {cache.device}")
    if t.dtype is not dtype or dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32 or bfloat16, as its companions (got {t.dtype})")
    a, b, c, d = t.stride()
    if d != 1:
        raise ValueError(f"{name} must have a unit head_dim stride")
    return _strides(a, b, c)


def cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                counts: torch.Tensor | None = None) -> None:
    """Writes rows ``starts[b] .. starts[b] + counts[b] - 1`` of every sequence and head.

    k, v: [batch, heads, n, head_dim] f32 or bf16, any batch/head/row strides; the first
    ``counts[b]`` rows of sequence b are taken (all n without ``counts``).  The other rows of the
    cache stay as they are.  k and v share no memory with the rows that are written.
    """
    if not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("k must be a [batch, heads, n, head_dim] tensor")
    dtype, n = k.dtype, k.shape[2]
    shape = (cache.batch, cache.heads, n, cache.head_dim)
    ks, vs = _rows("k", k, shape, dtype, cache), _rows("v", v, shape, dtype, cache)
    _run(cache, cache._lib.wfattn_cache_write, _DTYPES[dtype], n, k.data_ptr(), ks, v.data_ptr(),
         vs, _ints("starts", starts, cache._batch_shape, cache),
         None if counts is None else _ints("counts", counts, cache._batch_shape, cache))


def cache_read(cache: KVCache, starts: torch.Tensor, rows: int, *,
               counts: torch.Tensor | None = None, dtype: torch.dtype | None = None,
               out: tuple[torch.Tensor, torch.Tensor] | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``starts[b] .. starts[b] + counts[b] - 1`` of every sequence and head, as values.

    Returns (k, v), each [batch, heads, rows, head_dim] of ``dtype`` (float32 for an f32 cache,
    else bfloat16, by default).  Rows from ``counts[b]`` on are zero in new tensors, and left as
    they are in ``out``, whose strides may be any with a unit last one, and whose memory is neither
    shared between the two nor with the rows that are read.
    """
    shape = (cache.batch, cache.heads, int(rows), cache.head_dim)
    if out is None:
        dtype = dtype or (torch.float32 if cache.fmt == "f32" else torch.bfloat16)
        if dtype not in _DTYPES:
            raise ValueError(f"dtype must be float32 or bfloat16, got {dtype}")
        k = cache._new[dtype](shape)
        v = torch.empty_like(k)
        ks = vs = None  # contiguous
    else:
        k, v = out
        dtype = dtype or k.dtype
        ks, vs = (_rows(name, t, shape, dtype, cache) for name, t in (("out[0]", k), ("out[1]", v)))
    _run(cache, cache._lib.wfattn_cache_read, _DTYPES[dtype], shape[2], k.data_ptr(), ks,
         v.data_ptr(), vs, _ints("starts", starts, cache._batch_shape, cache),
         None if counts is None else _ints("counts", counts, cache._batch_shape, cache),
         out is None)
    return k, v


def cache_keep(cache: KVCache, lens: torch.Tensor, path: torch.Tensor, *,
               counts: torch.Tensor | None = None, out: torch.Tensor | None = None
               ) -> torch.Tensor:
    """Keeps the accepted nodes of a drafted tree and returns the new lengths.

    Row ``lens[b] + i`` becomes what row ``lens[b] + path[b, i]`` was, for i < ``counts[b]`` (the
    whole path without ``counts``); path is int32 [batch, depth], depth <= 64, in any order.
    Returns ``out`` (a new int32 [batch] tensor when not given, never ``lens`` itself):
    ``lens + counts``.
    """
    at = _ints("lens", lens, cache._batch_shape, cache)
    if not isinstance(path, torch.Tensor) or path.dim() != 2:
        raise ValueError("path must be int32 [batch, depth]")
    depth = path.shape[1]
    steps = _ints("path", path, (cache.batch, depth), cache)
    if out is None:
        out = torch.empty_like(lens)
    _run(cache, cache._lib.wfattn_cache_keep, at, depth, steps, path.stride(0),
         None if counts is None else _ints("counts", counts, cache._batch_shape, cache),
         _ints("out", out, cache._batch_shape, cache))
    return out


def tree_decode(q: torch.Tensor, cache: KVCache, kv_lens: torch.Tensor, *,
                tree: torch.Tensor | None = None, nodes: torch.Tensor | None = None,
                scale: float | None = None, out: torch.Tensor | None = None,
                workspace: DecodeWorkspace | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens over the cache; one token is a decode step.

    q: [batch, heads_q, n, head_dim], n <= 64, heads_q a multiple of the cache's heads (query head
    h reads cache head h // (heads_q // heads)); bf16 over a bf16, e4m3 or int4 cache, f32 over an
    f32, e4m3 or int4 one.  Node j of sequence b is row ``kv_lens[b] + j`` of the cache.  Every node
    sees the ``kv_lens[b]`` rows before the tree, and node i sees node j when bit j of
    ``tree[b, i]`` is set (``tree_words``; int64 [batch, n], or [n] for one tree of all; without
    it, nodes 0..i).  ``nodes`` (int32 [batch]) is how many of the n nodes each sequence has; the
    rest is padding, and gives zeros like a node that sees nothing.  What a node does not see does
    not reach its output, whatever it holds.  Over e4m3 and int4 rows errors are relative to the
    largest value that a node sees.

    Returns [batch, heads_q, n, head_dim] of q's dtype (``out`` where given).
    """
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be a [batch, heads_q, nodes, head_dim] tensor")
    dtype, shape = q.dtype, q.shape
    _, hq, n, _ = shape
    qs = _rows("q", q, (cache.batch, hq, n, cache.head_dim), dtype, cache)
    if out is None:
        out, os = cache._new[dtype](shape), None  # contiguous
    else:
        os = _rows("out", out, shape, dtype, cache)
    at = _ints("kv_lens", kv_lens, cache._batch_shape, cache)
    words, words_stride = None, 0
    if tree is not None:
        one = isinstance(tree, torch.Tensor) and tree.dim() == 1
        words = _ints("tree", tree, (n,) if one else (cache.batch, n), cache, torch.int64)
        words_stride = 0 if one else tree.stride(0)
    count = None if nodes is None else _ints("nodes", nodes, cache._batch_shape, cache)
    lib = cache._lib
    nbytes = cache._tree_bytes.get((dtype, hq, n))
    if nbytes is None:
        nbytes = lib.wfattn_tree_decode_workspace_size(cache._at, _DTYPES[dtype], hq, n)
        if nbytes == 0:
            _lib.check_last(lib)
        cache._tree_bytes[dtype, hq, n] = nbytes
    ws = (workspace or DecodeWorkspace()).get_tree(nbytes, cache.device)
    _run(cache, lib.wfattn_tree_decode, _DTYPES[dtype], hq, n, q.data_ptr(), qs, at, words,
         words_stride, count, out.data_ptr(), os, scale or 0.0, ws.data_ptr(), ws.numel())
    return out


def tree_words(parents) -> torch.Tensor:
    """The words of ``tree_decode`` for a tree given by each node's parent.

    parents: [..., n] integers (a list or a tensor), n <= 64, the parent of node i an earlier node
    or -1 where it follows the rows before the tree alone.  Every node sees itself and its
    ancestors.  Returns int64 [..., n] on the CPU or the tensor's device.
    """
    parents = torch.as_tensor(parents, dtype=torch.int64)
    n = parents.shape[-1] if parents.dim() else 0
    if not 1 <= n <= MAX_NODES:
        raise ValueError(f"a tree has 1 to {MAX_NODES} nodes, got {n}")
    index = torch.arange(n, device=parents.device)
    if bool(((parents >= index) | (parents < -1)).any()):
        raise ValueError("a node's parent is an earlier node, or -1")
    bit = torch.ones((), dtype=torch.int64, device=parents.device) << index
    words = torch.zeros_like(parents)
    for i in range(n):
        up = parents[..., i:i + 1]
        above = words.gather(-1, up.clamp_min(0)).masked_fill(up < 0, 0)
        words[..., i:i + 1] = above | bit[i]
    return words
