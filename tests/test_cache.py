"""Key/value caches without a GPU: refusals on the host and the words of drafted trees."""

from __future__ import annotations

import ctypes

import pytest

from warpforth_b200 import _lib

torch = pytest.importorskip("torch")


def _cache(**kw):
    c = dict(format=_lib.CACHE_E4M3, head_dim=64, batch=2, heads=3, max_len=10, batch_stride=30,
             head_stride=10, k=16, v=16, k_scale=16, v_scale=16)
    c.update(kw)
    return ctypes.byref(_lib.Cache(**c))


def _write(cache, dtype=_lib.DTYPE_BF16, n=4, k=16, v=16, starts=16, strides=None):
    st = (ctypes.c_int64 * 3)(*strides) if strides else None
    return _lib.load().wfattn_cache_write(cache, dtype, n, k, st, v, st, starts, None, None)


def _read(cache, dtype=_lib.DTYPE_BF16, n=4, k=16, v=16, starts=16, strides=None):
    st = (ctypes.c_int64 * 3)(*strides) if strides else None
    return _lib.load().wfattn_cache_read(cache, dtype, n, k, st, v, st, starts, None, 0, None)


def _keep(cache, lens=1024, depth=4, path=16, path_stride=4, new_lens=4096, counts=None):
    return _lib.load().wfattn_cache_keep(cache, lens, depth, path, path_stride, counts, new_lens,
                                         None)


def _tree(cache, dtype=_lib.DTYPE_BF16, hq=6, n=4, q=16, lens=16, tree=16, stride=4, o=16,
          o_strides=None, scale=0.0, ws=16, nbytes=1 << 40):
    st = (ctypes.c_int64 * 3)(*o_strides) if o_strides else None
    return _lib.load().wfattn_tree_decode(cache, dtype, hq, n, q, None, lens, tree, stride, None,
                                          o, st, scale, ws, nbytes, None)


@pytest.mark.parametrize("call", [_write, _read, _keep, _tree])
@pytest.mark.parametrize("bad", [
    {"format": 4}, {"format": -1}, {"batch": 0}, {"heads": 0}, {"max_len": 0}, {"k": None},
    {"v": None}, {"k_scale": None}, {"v_scale": None}, {"k": 24}, {"v": 8}, {"k_scale": 18},
    {"head_stride": 9}, {"batch_stride": 29}, {"batch_stride": -30}, {"head_stride": 1 << 50},
    {"batch": 1 << 31}, {"batch": 1 << 40, "heads": 1 << 40, "batch_stride": 1 << 40},
    {"max_len": 1 << 31, "head_stride": 1 << 31, "batch_stride": 1 << 33},
])
def test_bad_caches_are_refused(call, bad):
    assert call(_cache(**bad)) == _lib.INVALID_ARG
    assert _lib.load().wfattn_last_error()


@pytest.mark.parametrize("call", [_write, _read, _keep, _tree])
@pytest.mark.parametrize("d", [0, 32, 80, 256])
def test_other_head_sizes_are_refused(call, d):
    assert call(_cache(head_dim=d)) == _lib.UNSUPPORTED


@pytest.mark.parametrize("call", [_write, _read, _keep, _tree])
def test_a_null_cache_is_refused(call):
    assert call(None) == _lib.INVALID_ARG


def test_strides_of_single_entries_are_not_looked_at():
    # refused for its dtype, after the cache has passed
    c = _cache(batch=1, heads=1, batch_stride=0, head_stride=0)
    assert _write(c, dtype=9) == _lib.INVALID_ARG
    assert b"dtype" in _lib.load().wfattn_last_error()
    # sequences inside, heads outside
    c = _cache(batch_stride=10, head_stride=20)
    assert _write(c, dtype=9) == _lib.INVALID_ARG
    assert b"dtype" in _lib.load().wfattn_last_error()


@pytest.mark.parametrize("call", [_write, _read])
@pytest.mark.parametrize("bad", [{"dtype": 2}, {"n": -1}, {"n": 11}, {"k": None}, {"v": None},
                                 {"starts": None}, {"k": 17}, {"strides": (64, -1, 64)}])
def test_bad_rows_are_refused(call, bad):
    assert call(_cache(), **bad) == _lib.INVALID_ARG


@pytest.mark.parametrize("call", ["write", "read"])
@pytest.mark.parametrize("starts,counts", [(18, 16), (16, 18), (17, None), (16, 19)])
def test_positions_off_their_alignment_are_refused(call, starts, counts):
    lib, rows = _lib.load(), (_cache(), _lib.DTYPE_BF16, 4, 16, None, 16, None, starts, counts)
    status = lib.wfattn_cache_write(*rows, None) if call == "write" else \
        lib.wfattn_cache_read(*rows, 0, None)
    assert status == _lib.INVALID_ARG and b"aligned" in lib.wfattn_last_error()


@pytest.mark.parametrize("bad", [{"lens": 1026}, {"path": 18}, {"counts": 2049},
                                 {"new_lens": 8193}])
def test_paths_off_their_alignment_are_refused(bad):
    assert _keep(_cache(), **bad) == _lib.INVALID_ARG
    assert b"aligned" in _lib.load().wfattn_last_error()


def test_reading_into_broadcast_rows_is_refused():
    assert _read(_cache(), strides=(1000, 300, 0)) == _lib.INVALID_ARG
    assert b"broadcast" in _lib.load().wfattn_last_error()


def test_no_rows_is_no_work():
    assert _write(_cache(), n=0, k=None, v=None, starts=None) == _lib.OK
    assert _read(_cache(), n=0, k=None, v=None, starts=None) == _lib.OK


@pytest.mark.parametrize("bad", [{"lens": None}, {"path": None}, {"new_lens": None}, {"depth": 0},
                                 {"depth": 65}, {"path_stride": -4}, {"new_lens": 1024},
                                 {"new_lens": 1028}, {"new_lens": 1020}, {"path": 4092},
                                 {"path": 4100}, {"path": 4096 - 7 * 4, "path_stride": 5},
                                 {"counts": 4096}, {"counts": 4100}, {"counts": 4092}])
def test_bad_paths_are_refused(bad):
    assert _keep(_cache(), **bad) == _lib.INVALID_ARG


@pytest.mark.parametrize("bad", [
    {"dtype": 2}, {"hq": 0}, {"hq": 4}, {"hq": 3 << 40}, {"n": 0}, {"n": 65}, {"q": None},
    {"o": None}, {"lens": None}, {"q": 17}, {"o": 17}, {"tree": 20}, {"lens": 18}, {"stride": -4},
    {"scale": float("nan")}, {"ws": None}, {"ws": 24}, {"nbytes": 4},
    {"o_strides": (0, 64, 384)}, {"o_strides": (4096, 0, 64)}, {"o_strides": (4096, 64, 0)},
])
def test_bad_trees_are_refused(bad):
    assert _tree(_cache(), **bad) == _lib.INVALID_ARG


@pytest.mark.parametrize("fmt,dtype", [(_lib.CACHE_F32, _lib.DTYPE_BF16),
                                       (_lib.CACHE_BF16, _lib.DTYPE_F32)])
def test_a_plain_cache_takes_queries_of_its_type(fmt, dtype):
    c = _cache(format=fmt, k_scale=None, v_scale=None)
    assert _tree(c, dtype=dtype) == _lib.UNSUPPORTED
    assert _lib.load().wfattn_tree_decode_workspace_size(c, dtype, 6, 4) == 0


def test_workspace_size_of_refused_shapes_is_zero():
    lib = _lib.load()
    assert lib.wfattn_tree_decode_workspace_size(_cache(), _lib.DTYPE_BF16, 6, 4) >= 16
    assert lib.wfattn_tree_decode_workspace_size(_cache(), _lib.DTYPE_BF16, 7, 4) == 0
    assert lib.wfattn_tree_decode_workspace_size(_cache(), _lib.DTYPE_BF16, 6, 65) == 0
    assert lib.wfattn_tree_decode_workspace_size(None, _lib.DTYPE_BF16, 6, 4) == 0


def test_outgrown_workspaces_stay():
    """A captured graph goes on using the buffer that it was captured with."""
    from warpforth_b200 import DecodeWorkspace

    ws, cpu = DecodeWorkspace(), torch.device("cpu")
    small = ws.get_tree(5000, cpu)
    assert small.numel() == 5000 and not small[:_lib.TREE_DECODE_ZEROED].any()
    assert ws.get_tree(4096, cpu) is small
    small[0] = 7
    big = ws.get_tree(9000, cpu)
    assert big.numel() == 9000 and not big[:_lib.TREE_DECODE_ZEROED].any()
    assert ws.get_tree(5000, cpu) is big
    assert any(b is small for b in ws.tree_buffers[cpu])


def test_a_buffer_made_in_a_capture_is_not_kept(monkeypatch):
    """Its counters are zero only when the graph has run."""
    from warpforth_b200 import DecodeWorkspace, warpforth

    ws, cpu, capturing = DecodeWorkspace(), torch.device("cpu"), [True]
    monkeypatch.setattr(warpforth, "_capturing", lambda device: capturing[0], raising=False)
    first = ws.get_tree(5000, cpu)
    assert first.numel() == 5000 and ws.get_tree(5000, cpu) is not first
    capturing[0] = False
    kept = ws.get_tree(5000, cpu)
    assert kept is not first and ws.get_tree(5000, cpu) is kept
    capturing[0] = True
    assert ws.get_tree(4500, cpu) is kept  # zeroed before the capture
    assert ws.get_tree(5001, cpu).numel() == 5001
    capturing[0] = False
    assert ws.get_tree(5000, cpu) is kept


def test_caches_need_cuda_tensors():
    from warpforth_b200 import KVCache

    t = torch.zeros(1, 2, 8, 64)
    with pytest.raises(ValueError, match="CUDA"):
        KVCache.wrap(t, t)
    with pytest.raises(ValueError, match="fmt"):
        KVCache(1, 2, 8, fmt="e5m2")
    with pytest.raises(ValueError, match="head_dim"):
        KVCache(1, 2, 8, 80, device="cpu")


def test_tree_words():
    from warpforth_b200 import tree_words

    # 0 -> 1 -> 3, 0 -> 2, and a second root 4
    assert tree_words([-1, 0, 0, 1, -1]).tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10000]
    chain = tree_words(list(range(-1, 63)))
    assert chain.tolist() == [(2 << i) - 1 if i < 63 else -1 for i in range(64)]
    both = tree_words(torch.tensor([[-1, 0, 1], [-1, -1, 0]]))
    assert both.tolist() == [[1, 3, 7], [1, 2, 5]]
    for bad in ([0], [-1, 1], [-2], [], list(range(-1, 64)), -1):
        with pytest.raises(ValueError):
            tree_words(bad)
