"""GPU parity of the cache operators against plain implementations in 64 bits.

Writing and reading are defined value by value, so codes, scales and values are equal.  Attention is
held to the formula on the stored values within what its arithmetic can be off.  With A = sum of
p |v| over the keys, S = scale * max over the keys of sum |q k|, n keys:

* a score is a sum of D products in f32, by tensor cores that may cut instead of round: off by at
  most (D + 3) 2^-23 S, which moves a weight by that much relatively, in the sum and in its total;
* weights are exp2 of at most a few units of 2^-22, kept in f32 for the total and, for the products
  with bf16 queries, in 16 bits: 2^-11 (f16 beside quantised rows; bf16 rows take two bf16 terms),
  with f32 queries in two terms: 2^-21;
* f16 weights (beside quantised rows) are p s / s_top 2^7 or more, s_top being the largest row scale,
  and below 2^-14 they are held in steps of 2^-24: off by 2^-25 each, with a total of weights >= 1
  and codes c (e4m3 codes; u - 8) of |c| s_top <= 2.2 max |v| (e4m3: 448 s < 2 * 2 * 224 s / 2 and
  max |x| > 224 s; int4: 8 s <= 8/15 (1 + 2^-7) times a span of at most 2 max |v|).  The sum is off
  by at most n 2^-25 2^-7 2.2 max |v| < n 2^-30 max |v|;
* the sum over n keys adds n / 16 matrix products in f32: 2^-23 each;
* the output is rounded once: 2^-8 |o| in bf16, 2^-24 |o| in f32.

A 4-bit value is (m + 8 s) + s (u - 8), so |v| counts both parts there.
"""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

KINDS = [("f32", "f32"), ("bf16", "bf16"), ("e4m3", "bf16"), ("int4", "bf16"), ("e4m3", "f32"),
         ("int4", "f32")]
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def wf():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import warpforth_b200

    return warpforth_b200


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        from warpforth_b200 import warpforth

        warpforth.device_status(clear=True)


# ------------------------------------------------------------------ plain implementations


def bf16_directed(x, down):
    """f32 array -> the nearest bf16 below (down) or above."""
    cut = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
    away = (cut.view(np.uint32) + np.uint32(0x10000)).view(np.float32)
    return np.where(cut > x if down else cut < x, away, cut)


def e4m3_table():
    i = np.arange(256)
    field, frac = i % 128 // 8, i % 8 / 8
    t = np.where(field == 0, frac * 2.0 ** -6, (1 + frac) * 2.0 ** (field - 7.0))
    t[i % 128 == 127] = np.nan
    return np.where(i >= 128, -t, t)


def encode(fmt, x):
    """Rows x [..., D] (f32 array) -> codes (values for f32/bf16), scales."""
    if fmt in TYPES:
        return torch.from_numpy(x).to(TYPES[fmt]), None
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    x = np.where(bad, np.float32(0), x)
    if fmt == "e4m3":
        f, e = np.frexp(np.abs(x).max(-1, keepdims=True).astype(np.float64))
        e = np.where(f == 0, -126, np.maximum(e - 9 + (f > 0.875), -126))
        table = np.unique(np.abs(e4m3_table()[np.arange(127)]))
        y = np.abs(np.ldexp(x.astype(np.float64), -e))
        at = np.clip(np.searchsorted(table, y), 1, 126)
        low, high = table[at - 1], table[at]
        odd = (at - 1) % 2  # codes count up with the table
        up = (y - low > high - y) | ((y - low == high - y) & (odd == 1))
        code = np.where(up, at, at - 1) | np.where(np.signbit(x), 128, 0)
        scale = np.where(bad, np.nan, np.ldexp(1.0, e))[..., 0]
        return torch.from_numpy(np.where(bad, 0, code).astype(np.uint8)), \
            torch.from_numpy(scale.astype(np.float32))
    with np.errstate(all="ignore"):
        m = bf16_directed(x.min(-1, keepdims=True), True)
        s = bf16_directed((x.max(-1, keepdims=True) - m) / np.float32(15), False)
        bad = bad | ~np.isfinite(s)
        u = np.clip(np.rint((x - m) / s), 0, 15)
    u = np.where(bad | (s == 0), 0, u).astype(np.uint8)
    scale = np.where(bad, np.float32(np.nan), np.concatenate([s, m], -1))
    return torch.from_numpy(u[..., 0::2] | u[..., 1::2] << 4), \
        torch.from_numpy(scale.astype(np.float32)).bfloat16()


def values(fmt, codes, scale):
    """Stored rows -> f64 values."""
    if fmt in TYPES:
        return codes.double().numpy()
    if fmt == "e4m3":
        with np.errstate(invalid="ignore"):
            return e4m3_table()[codes.view(torch.uint8).numpy()] * scale.double().numpy()[..., None]
    c, sc = codes.numpy(), scale.double().numpy()
    u = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    return sc[..., 1:] + sc[..., :1] * u


def parts(fmt, codes, scale):
    """What |v| counts for: the value, or the two parts of a 4-bit one."""
    v = values(fmt, codes, scale)
    if fmt != "int4":
        return np.abs(v)
    sc = scale.double().numpy()
    return np.abs(sc[..., 1:] + 8 * sc[..., :1]) + np.abs(v - sc[..., 1:] - 8 * sc[..., :1])


def attend(fmt, cache, q, lens, words, nodes, scale=None):
    """The formula in 64 bits: outputs, and how far off they may be (relative to q's type)."""
    b, hq, n, d = q.shape
    sc = scale or d ** -0.5
    kc, vc = ((cache.k, cache.k_scale), (cache.v, cache.v_scale))
    dev = [(x.cpu(), None if y is None else y.cpu()) for x, y in (kc, vc)]
    k, v, size = values(fmt, *dev[0]), values(fmt, *dev[1]), parts(fmt, *dev[1])
    f32 = q.dtype == torch.float32
    qd = q.double().numpy()
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    g = hq // cache.heads
    for i in range(b):
        for t in range(min(n, nodes[i])):
            sees = list(range(lens[i])) + [lens[i] + j for j in range(nodes[i])
                                           if words[i][t] >> j & 1]
            if not sees:
                continue
            for h in range(hq):
                kk, vv = k[i, h // g, sees], v[i, h // g, sees]
                s = kk @ qd[i, h, t] * sc
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h, t] = p @ vv
                big = (np.abs(kk) @ np.abs(qd[i, h, t])).max() * abs(sc)
                e = 2 * (d + 3) * 2.0 ** -23 * big + (len(sees) / 16 + 64) * 2.0 ** -23
                e += 2.0 ** -21 if f32 else 2.0 ** -11
                tol[i, h, t] = e * (p @ size[i, h // g, sees])
                if fmt not in TYPES:
                    tol[i, h, t] += len(sees) * 2.0 ** -30 * np.abs(vv).max()
    return out, tol + np.abs(out) * (2.0 ** -24 if f32 else 2.0 ** -8)


def make_cache(wf, fmt, b, h, lmax, d, seed):
    """A filled cache (rows of very different sizes) and its rows as they were written."""
    rng = np.random.default_rng(seed)
    cache = wf.KVCache(b, h, lmax, d, fmt=fmt)
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        rows = rng.standard_normal((b, h, lmax, d)) * np.exp(rng.standard_normal((b, h, lmax, 1)))
        codes, scale = encode(fmt, rows.astype(np.float32))
        if fmt == "e4m3":
            x.view(torch.uint8).copy_(codes)
        else:
            x.copy_(codes)
        if scale is not None:
            s.copy_(scale)
    return cache


def random_trees(b, n, seed):
    rng = np.random.default_rng(seed)
    return [[int(rng.integers(-1, i)) for i in range(n)] for _ in range(b)]


def check(out, ref, tol):
    o = out.double().cpu().numpy()
    assert np.isfinite(o).all()
    worst = (np.abs(o - ref) / np.maximum(tol, 1e-30)).max()
    assert worst <= 1, f"off by {worst:.2f} times what the arithmetic allows"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ----------------------------------------------------------------------- write and read


@pytest.mark.parametrize("fmt", ["f32", "bf16", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,n", [(64, 1), (64, 37), (128, 5), (128, 64)])
def test_write_stores_what_the_format_says(wf, fmt, dtype, d, n):
    b, h, lmax = 3, 2, 67
    rng = np.random.default_rng(n)
    cache = make_cache(wf, fmt, b, h, lmax, d, 1)
    before = [None if t is None else t.clone() for t in
              (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    new = [torch.from_numpy((rng.standard_normal((b, n, h, d)) *
                             np.exp(3 * rng.standard_normal((b, n, h, 1)))).astype(np.float32))
           .to(TYPES[dtype]).transpose(1, 2) for _ in range(2)]
    starts, counts = [0, lmax - n, 2], [n, n // 2, max(0, n - 3)]
    wf.cache_write(cache, new[0].cuda(), new[1].cuda(), ints(starts), counts=ints(counts))
    read = wf.cache_read(cache, ints(starts), n, counts=ints(counts), dtype=torch.float32)
    for x, codes, scale, codes0, scale0, got in zip(
            new, (cache.k, cache.v), (cache.k_scale, cache.v_scale), before[:2], before[2:], read):
        want, want_scale = encode(fmt, x.float().contiguous().numpy())
        raw = (lambda t: t.cpu().view(torch.uint8)) if fmt == "e4m3" else (lambda t: t.cpu())
        expect, expect_scale = raw(codes0), None if scale0 is None else scale0.cpu()
        for i in range(b):
            at = slice(starts[i], starts[i] + counts[i])
            expect[i, :, at] = want[i, :, :counts[i]]
            if scale is not None:
                expect_scale[i, :, at] = want_scale[i, :, :counts[i]]
        assert torch.equal(raw(codes), expect)
        if scale is not None:
            assert torch.equal(scale.cpu(), expect_scale)
        back = values(fmt, want if fmt != "e4m3" else want.view(torch.float8_e4m3fn), want_scale)
        for i in range(b):
            assert np.array_equal(got[i, :, :counts[i]].cpu().numpy(),
                                  back[i, :, :counts[i]].astype(np.float32))
            assert not got[i, :, counts[i]:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
def test_write_rows_at_the_edges_of_the_types(wf, fmt):
    """Zeros, one value, the smallest and largest numbers, ties, NaN and infinities."""
    d = 64
    top, tiny, low = 3.4028235e38, 1e-45, 2.0 ** -126
    rows = np.zeros((1, 1, 14, d), np.float32)
    rows[0, 0, 1] = -0.0
    rows[0, 0, 2] = 7.25
    rows[0, 0, 3, 5] = top
    rows[0, 0, 4] = np.linspace(-top, top, d)
    rows[0, 0, 5, ::2] = tiny
    rows[0, 0, 6] = low * np.linspace(-3, 3, d)
    rows[0, 0, 7] = np.arange(d) / 2 - 16  # halves of a step
    rows[0, 0, 8] = 448 * 2.0 ** np.arange(-d // 2, d // 2)
    rows[0, 0, 9] = np.nextafter(np.float32(448), np.float32(1e9))
    rows[0, 0, 10, 3] = np.nan
    rows[0, 0, 11, 63] = np.inf
    rows[0, 0, 12, 0] = -np.inf
    rows[0, 0, 13] = np.linspace(1, 2, d)
    cache = wf.KVCache(1, 1, 14, d, fmt=fmt)
    x = torch.from_numpy(rows).cuda()
    wf.cache_write(cache, x, -x, ints([0]))
    k, v = wf.cache_read(cache, ints([0]), 14, dtype=torch.float32)
    for x, codes, scale, got in ((rows, cache.k, cache.k_scale, k), (-rows, cache.v, cache.v_scale, v)):
        want, want_scale = encode(fmt, x)
        assert torch.equal(codes.cpu().view(torch.uint8), want)
        assert torch.equal(scale.cpu().nan_to_num(-1.0), want_scale.nan_to_num(-1.0))
        got = got.cpu().numpy()
        assert np.isnan(got[0, 0, 10:13]).all()
        with np.errstate(over="ignore"):
            back = values(fmt, want.view(torch.float8_e4m3fn) if fmt == "e4m3" else want, want_scale)
            assert np.array_equal(got, back.astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("fmt", ["f32", "bf16", "e4m3", "int4"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_read_into_strided_rows_leaves_the_rest(wf, fmt, dtype):
    b, h, lmax, d, n = 2, 3, 50, 64, 9
    cache = make_cache(wf, fmt, b, h, lmax, d, 2)
    # rows at odd offsets: 3 elements before each, and a gap between them
    store = torch.full((2, b, n, h, d + 5), 7.0, dtype=TYPES[dtype], device="cuda")
    out = tuple(store[i, :, :, :, 3:3 + d].transpose(1, 2) for i in range(2))
    starts, counts = [41, 7], [9, 4]
    wf.cache_read(cache, ints(starts), n, counts=ints(counts), out=out)
    for got, codes, scale in zip(out, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        full = values(fmt, codes.cpu(), None if scale is None else scale.cpu())
        for i in range(b):
            want = torch.from_numpy(full[i, :, starts[i]:starts[i] + counts[i]].astype(np.float32))
            assert torch.equal(got[i, :, :counts[i]].cpu(), want.to(TYPES[dtype]))
            assert (got[i, :, counts[i]:] == 7).all()
    assert (store[..., :3] == 7).all() and (store[..., 3 + d:] == 7).all()


def test_write_takes_any_strides_and_alignment(wf):
    b, h, d, n = 2, 3, 128, 6
    rng = np.random.default_rng(4)
    x = torch.from_numpy(rng.standard_normal((b, n, h, d + 7)).astype(np.float32)).cuda()
    for dtype in (torch.float32, torch.bfloat16):
        odd = x.to(dtype)[..., 5:5 + d].transpose(1, 2)
        one = odd[:, :, :1].expand(b, h, n, d)  # one row for all
        got = []
        for k, v in ((odd, one), (odd.contiguous(), one.contiguous())):
            cache = wf.KVCache(b, h, 11, d, fmt="int4")
            wf.cache_write(cache, k, v, ints([5, 0]))
            got.append((cache.k, cache.v, cache.k_scale, cache.v_scale))
        for s, t in zip(*got):
            assert torch.equal(s, t)


def test_positions_outside_the_cache_touch_nothing_and_are_reported(wf):
    from warpforth_b200 import _lib, warpforth

    b, h, lmax, d, n = 4, 2, 20, 64, 6
    cache = make_cache(wf, "e4m3", b, h, lmax, d, 5)
    before = cache.k.view(torch.uint8).clone(), cache.k_scale.clone()
    x = torch.ones(b, h, n, d, device="cuda")
    starts, counts = ints([-3, 17, 2 ** 31 - 2, 4]), ints([6, 6, 6, -1])
    wf.cache_write(cache, x, x, starts, counts=counts)
    with pytest.raises(_lib.WfattnError, match="row position"):
        warpforth.device_status()
    warpforth.device_status()  # cleared
    changed = (cache.k.view(torch.uint8) != before[0]).any(-1)[:, 0].cpu()
    assert changed[0].nonzero().flatten().tolist() == [0, 1, 2]
    assert changed[1].nonzero().flatten().tolist() == [17, 18, 19]
    assert not changed[2:].any()
    k, _ = wf.cache_read(cache, starts, n, counts=ints([6, 6, 6, 99]), dtype=torch.float32)
    with pytest.raises(_lib.WfattnError, match="row position"):
        warpforth.device_status()
    assert not k[0, :, :3].any() and (k[0, :, 3:] == 1).all()
    assert (k[1, :, :3] == 1).all() and not k[1, :, 3:].any() and not k[2].any()


# ------------------------------------------------------------------------------- keep


@pytest.mark.parametrize("fmt", ["f32", "bf16", "e4m3", "int4"])
@pytest.mark.parametrize("d", [64, 128])
def test_keep_moves_rows(wf, fmt, d):
    b, h, lmax, n = 6, 2, 90, 64
    rng = np.random.default_rng(6)
    path = np.stack([np.sort(rng.permutation(n)), rng.permutation(n), np.arange(n)[::-1],
                     np.full(n, 5), np.arange(1, n + 1), rng.integers(0, n, n)]).astype(np.int32)
    lens, counts = [0, 3, 26, 10, 7, 1], [9, 64, 64, 12, 63, 0]
    cache = make_cache(wf, fmt, b, h, lmax, d, 7)
    tensors = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    raw = [t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in tensors]
    want = [t.cpu().clone() for t in raw]
    for t in want:
        src = t.clone()
        for i in range(b):
            for j in range(counts[i]):
                t[i, :, lens[i] + j] = src[i, :, lens[i] + path[i, j]]
    new = wf.cache_keep(cache, ints(lens), torch.from_numpy(path).cuda(), counts=ints(counts))
    assert new.tolist() == [x + y for x, y in zip(lens, counts)]
    for t, w in zip(raw, want):
        assert torch.equal(t.cpu(), w)


def test_keep_refuses_sequences_that_leave_the_cache(wf):
    from warpforth_b200 import _lib, warpforth

    cache = make_cache(wf, "bf16", 6, 2, 20, 64, 8)
    before = cache.k.clone()
    path = ints([[0, 1, 2]] * 3 + [[0, 9, 2], [0, -1, 2], [2, 2, 0]])
    lens = [-1, 18, 5, 11, 5, 17]
    new = wf.cache_keep(cache, ints(lens), path, counts=ints([3, 3, 4, 3, 3, 3]))
    with pytest.raises(_lib.WfattnError, match="row position"):
        warpforth.device_status()
    assert new.tolist() == [-1, 18, 5, 11, 5, 20]
    before[5, :, 17:20] = before[5, :, [19, 19, 17]]
    assert torch.equal(cache.k, before)


# -------------------------------------------------------------------------- attention


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("d,g,n", [(64, 1, 1), (64, 5, 1), (64, 1, 7), (128, 8, 1), (128, 3, 16),
                                   (64, 2, 33), (128, 1, 64), (128, 5, 61)])
def test_tree_decode_over_ragged_lengths(wf, fmt, dtype, d, g, n):
    lens = [0, 1, 15, 64, 63, 130, 257]
    b, h = len(lens), 2
    cache = make_cache(wf, fmt, b, h, 257 + n, d, n)
    q = torch.randn(b, n, h * g, d, generator=torch.Generator().manual_seed(n))
    q = q.to(TYPES[dtype]).transpose(1, 2)
    trees = random_trees(b, n, n)
    words = wf.tree_words(trees)
    nodes = [n, n, max(1, n - 2), n, 0, n // 2, n]
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda(), nodes=ints(nodes))
    ref, tol = attend(fmt, cache, q, lens, words.tolist(), nodes)
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_tree_decode_over_long_rows(wf, fmt, dtype):
    # one sequence split over the whole GPU, one of a single key, one token each
    lens, d, n = [6001, 0, 2999], 64, 1
    cache = make_cache(wf, fmt, 3, 1, 6002, d, 3)
    q = torch.randn(3, 4, n, d, generator=torch.Generator().manual_seed(3)).to(TYPES[dtype])
    out = wf.tree_decode(q.cuda(), cache, ints(lens))
    ref, tol = attend(fmt, cache, q, lens, [[1]] * 3, [1] * 3)
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("b,longest", [(33, 1100), (129, 600), (300, 300)])
@pytest.mark.parametrize("g,n", [(2, 1), (3, 4), (8, 5)])
def test_tree_decode_of_many_sequences(wf, fmt, dtype, b, longest, g, n):
    """More sequences than a warp, and than a block, has threads to share them out; the longest are
    dealt in units (4-bit rows of few queries: with 33 sequences only) and many are empty."""
    d, gen = 64, torch.Generator().manual_seed(b)
    rng = np.random.default_rng(b)
    lens = [int(x) for x in rng.integers(0, 40, b)]
    for i in range(0, b, 7):
        lens[i] = 0
    lens[3] = lens[b - 2] = longest
    cache = wf.KVCache(b, 1, longest + n, d, fmt=fmt)
    x = torch.randn(2, b, 1, longest + n, d, generator=gen).cuda()
    wf.cache_write(cache, x[0], x[1], ints([0] * b))
    q = torch.randn(b, g, n, d, generator=gen).to(TYPES[dtype])
    words = wf.tree_words(random_trees(b, n, b))
    nodes = [int(x) for x in rng.integers(0, n + 1, b)]
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda(), nodes=ints(nodes))
    ref, tol = attend(fmt, cache, q, lens, words.tolist(), nodes)
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_masked_and_missing_rows_never_reach_an_output(wf, fmt, dtype):
    """Rows past the end hold NaN; node 2 holds NaN and infinities, and nodes 2 and 4 see it."""
    b, h, d, n, lmax = 2, 2, 64, 6, 80
    lens, nodes = [50, 3], [6, 5]
    cache = make_cache(wf, fmt, b, h, lmax, d, 9)
    for t in (cache.k, cache.v):
        for i in range(b):
            if fmt in TYPES:
                t[i, :, lens[i] + nodes[i]:] = math.nan
                t[i, 0, lens[i] + 2] = math.nan
                t[i, 1, lens[i] + 2, 1::2] = -math.inf
            elif fmt == "e4m3":
                t.view(torch.uint8)[i, :, lens[i] + nodes[i]:] = 0x7F
                t.view(torch.uint8)[i, 1, lens[i] + 2] = 0xFF
    for t in (cache.k_scale, cache.v_scale):
        for i in range(b):
            if t is not None:
                t[i, :, lens[i] + nodes[i]:] = math.nan
                t[i, :, lens[i] + 2] = math.nan
    q = torch.randn(b, 4, n, d, generator=torch.Generator().manual_seed(9)).to(TYPES[dtype])
    words = wf.tree_words([-1, 0, 0, 1, 2, 0])
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda(), nodes=ints(nodes))
    sees = torch.tensor([w >> 2 & 1 == 1 for w in words.tolist()])
    assert not torch.isfinite(out[:, :, sees].float()).all(-1).any()
    clean = wf.KVCache.wrap(*(None if t is None else t.clone() for t in
                              (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    for t in (clean.k, clean.v):
        raw = t.view(torch.uint8) if fmt == "e4m3" else t
        for i in range(b):
            raw[i, :, lens[i] + 2] = 0
            raw[i, :, lens[i] + nodes[i]:] = 0
    for t in (clean.k_scale, clean.v_scale):
        if t is not None:
            t.nan_to_num_(0.0)
    ref, tol = attend(fmt, clean, q, lens, [words.tolist()] * b, nodes)
    keep = ~sees
    check(out[:, :, keep], ref[:, :, keep], tol[:, :, keep])


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_nodes_that_see_nothing_give_zeros(wf, fmt, dtype):
    cache = make_cache(wf, fmt, 2, 1, 70, 64, 10)
    q = torch.randn(2, 2, 3, 64, generator=torch.Generator().manual_seed(10)).to(TYPES[dtype])
    words = torch.tensor([[0, 2, 0], [0, 0, 7]])
    out = wf.tree_decode(q.cuda(), cache, ints([0, 67]), tree=words.cuda(), nodes=ints([2, 3]))
    ref, tol = attend(fmt, cache, q, [0, 67], words.tolist(), [2, 3])
    assert not out[0, :, 0].any() and not out[0, :, 2].any()
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_large_scores_and_a_scale(wf, fmt, dtype):
    # scores of several hundred, rising along the sequence: the maximum moves in every block
    b, h, d, n, length = 1, 1, 64, 2, 500
    cache = wf.KVCache(b, h, 512, d, fmt=fmt)
    ramp = torch.linspace(-1, 1, length)[:, None] + 0.02 * torch.randn(
        length, d, generator=torch.Generator().manual_seed(11))
    x = ramp.expand(b, h, length, d).contiguous().cuda()
    wf.cache_write(cache, x, x.flip(-1), ints([0]))
    q = (8 * torch.ones(b, h, n, d)).to(TYPES[dtype])
    q[..., 1, :] *= -1
    for scale in (None, 0.5):
        out = wf.tree_decode(q.cuda(), cache, ints([length - n]), scale=scale)
        ref, tol = attend(fmt, cache, q, [length - n], [[1, 3]], [n], scale)
        check(out, ref, tol)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int4"])
def test_values_of_very_different_sizes(wf, fmt):
    # the largest rows of V have almost no weight: the small ones must keep their precision
    d, length = 64, 300
    rng = np.random.default_rng(12)
    cache = wf.KVCache(1, 1, 320, d, fmt=fmt)
    k = rng.standard_normal((1, 1, length, d)).astype(np.float32)
    v = rng.standard_normal((1, 1, length, d)).astype(np.float32)
    k[..., ::50, :] = -3.0
    v[..., ::50, :] *= 4096
    wf.cache_write(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints([0]))
    q = torch.ones(1, 1, 1, d).bfloat16()
    out = wf.tree_decode(q.cuda(), cache, ints([length - 1]))
    ref, tol = attend(fmt, cache, q, [length - 1], [[1]], [1])
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", [k for k in KINDS if k[0] not in TYPES])
@pytest.mark.parametrize("g,n", [(1, 2), (2, 4), (4, 4), (4, 8), (5, 8), (3, 64)])
@pytest.mark.parametrize("power", [30, 90])
def test_values_of_unseen_nodes_may_be_huge(wf, fmt, dtype, g, n, power):
    """Node 1's values are 2^power times the others'; those who do not see it keep their bits."""
    lens, d, h = [0, 3, 50, 300], 64, 2
    b = len(lens)
    cache = wf.KVCache(b, h, 300 + n, d, fmt=fmt)
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(2, b, h, 300 + n, d, generator=gen)
    for i in range(b):
        x[1, i, :, lens[i] + 1] *= 2.0 ** power
    wf.cache_write(cache, x[0].cuda(), x[1].cuda(), ints([0] * b))
    q = torch.randn(b, g * h, n, d, generator=gen).to(TYPES[dtype])
    words = wf.tree_words([-1, 0, 0, 1, 2, 0, 3, 4][:n] + [i // 2 for i in range(8, n)])
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda())
    ref, tol = attend(fmt, cache, q, lens, [words.tolist()] * b, [n] * b)
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("g,n", [(1, 4), (3, 4), (5, 8)])
@pytest.mark.parametrize("scale", [None, 1e-3, 1e-12, 1e-38])
def test_zero_queries_and_small_scales(wf, fmt, dtype, g, n, scale):
    """Scores next to 0: a node's output is the mean of what it sees, and of nothing else."""
    lens, d, h = [0, 5, 130], 64, 1
    cache = make_cache(wf, fmt, 3, h, 130 + n, d, 28)
    q = torch.randn(3, g * h, n, d, generator=torch.Generator().manual_seed(28)).to(TYPES[dtype])
    q[:, :, ::2] = 0
    words = wf.tree_words([i - 2 if i > 1 else -1 for i in range(n)])
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda(), scale=scale)
    ref, tol = attend(fmt, cache, q, lens, [words.tolist()] * 3, [n] * 3, scale)
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", [k for k in KINDS if k[0] not in TYPES])
@pytest.mark.parametrize("g,n", [(1, 1), (2, 4), (4, 4), (4, 8), (5, 8)])
def test_scales_of_either_sign(wf, fmt, dtype, g, n):
    """A program's own cache may hold them: a value is code * scale, or minimum + scale * code."""
    lens, d, h = [0, 7, 300], 64, 2
    cache = make_cache(wf, fmt, 3, h, 300 + n, d, 29)
    gen = torch.Generator().manual_seed(29)
    for s in (cache.k_scale, cache.v_scale):
        sign = (1 - 2 * torch.randint(0, 2, s.shape[:3], generator=gen)).cuda()
        sign[1] = -1
        (s if fmt == "e4m3" else s[..., 0]).mul_(sign)
    q = torch.randn(3, g * h, n, d, generator=gen).to(TYPES[dtype])
    words = wf.tree_words(random_trees(1, n, 29)[0])
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda())
    ref, tol = attend(fmt, cache, q, lens, [words.tolist()] * 3, [n] * 3)
    check(out, ref, tol)
    for t, codes, scale in zip(wf.cache_read(cache, ints([0] * 3), 300, dtype=torch.float32),
                               (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        want = values(fmt, codes.cpu(), scale.cpu())[:, :, :300].astype(np.float32)
        assert np.array_equal(t.cpu().numpy(), want)


@pytest.mark.parametrize("fmt,dtype", [k for k in KINDS if k[0] not in TYPES])
@pytest.mark.parametrize("g,n", [(1, 2), (3, 4), (5, 8)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_keys_that_are_not_finite_are_not_passed_over(wf, fmt, dtype, g, n, bad):
    """A scale of K that is not finite, in a row before the tree (head 0) and in node 0 (head 1)."""
    lens, d, h = [4, 130], 64, 2
    cache = make_cache(wf, fmt, 2, h, 130 + n, d, 38)
    scale = cache.k_scale if fmt == "e4m3" else cache.k_scale[..., 0]
    for i in range(2):
        scale[i, 0, 2] = scale[i, 1, lens[i]] = bad
    q = torch.randn(2, g * h, n, d, generator=torch.Generator().manual_seed(38)).to(TYPES[dtype])
    out = wf.tree_decode(q.cuda(), cache, ints(lens))
    assert torch.isnan(out).all()


def test_strided_queries_outputs_and_caches(wf):
    b, h, d, n = 3, 4, 128, 5
    big = make_cache(wf, "int4", 2 * b, h, 99, d, 13)
    part = wf.KVCache.wrap(*(t[1::2, 1:3] for t in (big.k, big.v, big.k_scale, big.v_scale)))
    q = torch.randn(b, n, 6, d + 3, generator=torch.Generator().manual_seed(13)).bfloat16()
    q = q[..., 1:1 + d].transpose(1, 2)
    store = torch.full((b, 6, n, d + 9), 5.0, dtype=torch.bfloat16, device="cuda")
    out = store[..., 7:7 + d]
    words = wf.tree_words(random_trees(1, n, 13)[0])
    qc = torch.empty(b, n, 6, d + 3, dtype=torch.bfloat16, device="cuda")[..., 1:1 + d]
    qc = qc.transpose(1, 2)
    qc.copy_(q)
    got = wf.tree_decode(qc, part, ints([0, 94, 33]), tree=words.cuda(), out=out)
    assert got is out
    ref, tol = attend("int4", part, q, [0, 94, 33], [words.tolist()] * b, [n] * b)
    check(out, ref, tol)
    assert (store[..., :7] == 5).all() and (store[..., 7 + d:] == 5).all()


def test_offsets_past_32_bits(wf):
    # the second sequence begins 4.3 GB into each array
    d, lmax = 64, (1 << 25) + 64
    k, v = (torch.empty(2, 1, lmax, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = wf.KVCache.wrap(k, v)
    x = torch.randn(2, 1, 200, d, generator=torch.Generator().manual_seed(14)).bfloat16()
    starts = ints([0, 0])
    wf.cache_write(cache, x.cuda(), x.flip(-1).cuda(), starts)
    q = torch.randn(2, 3, 2, d, generator=torch.Generator().manual_seed(15)).bfloat16()
    out = wf.tree_decode(q.cuda(), cache, ints([150, 198]))
    small = wf.KVCache.wrap(k[:, :, :200].contiguous(), v[:, :, :200].contiguous())
    ref, tol = attend("bf16", small, q, [150, 198], [[1, 3]] * 2, [2, 2])
    check(out, ref, tol)
    # and the far end of one sequence
    far = ints([lmax - 200, lmax - 200])
    wf.cache_write(cache, x.cuda(), x.cuda(), far)
    new = wf.cache_keep(cache, far, ints([[3, 199], [7, 2]]))
    assert new.tolist() == [lmax - 198] * 2
    got, _ = wf.cache_read(cache, far, 2)
    assert torch.equal(got[0, 0].cpu(), x[0, 0, [3, 199]])
    assert torch.equal(got[1, 0].cpu(), x[1, 0, [7, 2]])


def test_lengths_outside_the_cache_are_clamped_and_reported(wf):
    from warpforth_b200 import _lib, warpforth

    cache = make_cache(wf, "e4m3", 4, 1, 40, 64, 16)
    q = torch.randn(4, 1, 4, 64, generator=torch.Generator().manual_seed(16)).bfloat16()
    out = wf.tree_decode(q.cuda(), cache, ints([-5, 38, 1000, 10]), nodes=ints([4, 4, 4, 9]))
    with pytest.raises(_lib.WfattnError, match="length"):
        warpforth.device_status()
    words = [[1, 3, 7, 15]] * 4
    ref, tol = attend("e4m3", cache, q, [0, 38, 40, 10], words, [4, 2, 0, 4])
    check(out, ref, tol)


def test_bad_tensors_are_refused(wf):
    cache = wf.KVCache(2, 2, 16, 64, fmt="e4m3")
    lens, x = ints([0, 0]), torch.zeros(2, 2, 3, 64, device="cuda")
    for k, v, at in ((x[:1], x, lens), (x, x[..., :32], lens), (x, x.bfloat16(), lens),
                     (x.half(), x.half(), lens), (x.cpu(), x, lens), (x, x, lens[:1]),
                     (x, x, lens.long()), (x, x, lens.cpu()), (x.expand(2, 2, 3, 64)[..., ::2], x, lens),
                     (None, x, lens)):
        with pytest.raises(ValueError):
            wf.cache_write(cache, k, v, at)
    for kw in (dict(dtype=torch.float16), dict(out=(x, x[:1])), dict(counts=lens[:1])):
        with pytest.raises(ValueError):
            wf.cache_read(cache, lens, 3, **kw)
    from warpforth_b200 import _lib

    with pytest.raises(_lib.WfattnError):
        wf.cache_read(cache, lens, 17)
    path = ints([[0, 1], [0, 1]])
    for p, kw in ((path[0], {}), (path.long(), {}), (path, dict(counts=lens.long())),
                  (path, dict(out=lens[:1])), (path.t(), {})):
        with pytest.raises(ValueError):
            wf.cache_keep(cache, lens, p, **kw)
    with pytest.raises(_lib.WfattnError, match="new_lens"):
        wf.cache_keep(cache, lens, path, out=lens)
    q = torch.zeros(2, 4, 3, 64, device="cuda")
    words = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for args, kw in (((q[0], cache, lens), {}), ((q.half(), cache, lens), {}),
                     ((q[..., :32], cache, lens), {}), ((q, cache, lens[:1]), {}),
                     ((q, cache, lens), dict(tree=words[:1])), ((q, cache, lens), dict(tree=words.int())),
                     ((q, cache, lens), dict(out=q.bfloat16())), ((q, cache, lens), dict(nodes=words))):
        with pytest.raises(ValueError):
            wf.tree_decode(*args, **kw)
    for bad in (q[:, :3], torch.zeros(2, 4, 65, 64, device="cuda")):
        with pytest.raises(_lib.WfattnError):
            wf.tree_decode(bad, cache, lens)
    k = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    s = torch.zeros(2, 2, 16, device="cuda")
    f8 = k.to(torch.float8_e4m3fn)
    for bad in ((k, k.float()), (k, k[:1]), (k, k, s, s), (f8, f8), (f8, f8, s, s[:1]),
                (f8, f8, s, s.double()), (k[..., ::2], k[..., ::2]), (k.transpose(1, 2),) * 2,
                (k[..., :32], k[..., :32]), (k, k.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            wf.KVCache.wrap(*bad)


# ------------------------------------- many query rows a cache head (products on tcgen05)

WIDE = [k for k in KINDS if k[1] == "bf16"]


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("d", [64, 128])
def test_unseen_rows_of_large_trees(wf, fmt, dtype, d):
    """60 and 132 query rows a head; rows past the end hold NaN, node 2 NaN and infinities, its
    unit being the first, the middle of one and the last of one."""
    lens, nodes, n, h = [0, 61, 126, 190], [6, 5, 6, 3], 6, 2
    b, lmax = len(lens), 200
    words = wf.tree_words([-1, 0, 0, 1, 2, 0])
    sees = torch.tensor([w >> 2 & 1 == 1 for w in words.tolist()])
    for g in (10, 22):
        cache = make_cache(wf, fmt, b, h, lmax, d, 30)
        clean = wf.KVCache.wrap(*(None if t is None else t.clone() for t in
                                  (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        for t in (cache.k, cache.v):
            for i in range(b):
                end, node = lens[i] + nodes[i], lens[i] + 2
                if fmt in TYPES:
                    t[i, :, end:] = math.nan
                    t[i, 0, node, ::7] = math.nan
                    t[i, 1, node, 1::2] = math.inf
                elif fmt == "e4m3":
                    t.view(torch.uint8)[i, :, end:] = 0x7F
                    t.view(torch.uint8)[i, 1, node, 1::2] = 0xFF
        for t in (cache.k_scale, cache.v_scale):
            for i in range(b):
                if t is not None:
                    t[i, :, lens[i] + nodes[i]:] = math.nan
                    t[i, 0, lens[i] + 2] = math.nan
                    if fmt == "int4":
                        t[i, 1, lens[i] + 2, 0] = math.inf
        q = torch.randn(b, g * h, n, d, generator=torch.Generator().manual_seed(30))
        q = q.to(TYPES[dtype])
        out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda(), nodes=ints(nodes))
        for i in range(b):
            live = sees & (torch.arange(n) < nodes[i])
            assert not torch.isfinite(out[i][:, live].float()).all(-1).any()
        ref, tol = attend(fmt, clean, q, lens, [words.tolist()] * b, nodes)
        check(out[:, :, ~sees], ref[:, :, ~sees], tol[:, :, ~sees])


@pytest.mark.parametrize("fmt,dtype", WIDE[:2])
def test_what_is_not_finite_stays_in_its_column(wf, fmt, dtype):
    """Only V's values at one place of a seen node are not finite: the others are as ever."""
    d, n, lens = 64, 34, [0, 64, 100]
    cache = make_cache(wf, fmt, 3, 1, 140, d, 31)
    clean = wf.KVCache.wrap(*(None if t is None else t.clone() for t in
                              (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    for i in range(3):
        if fmt == "e4m3":
            cache.v.view(torch.uint8)[i, 0, lens[i] + 3, 5] = 0x7F
        else:
            cache.v[i, 0, lens[i] + 3, 5] = math.inf
    q = torch.randn(3, 1, n, d, generator=torch.Generator().manual_seed(31)).to(TYPES[dtype])
    words = wf.tree_words(random_trees(1, n, 31)[0])
    out = wf.tree_decode(q.cuda(), cache, ints(lens), tree=words.cuda())
    ref, tol = attend(fmt, clean, q, lens, [words.tolist()] * 3, [n] * 3)
    odd = torch.zeros(n, d, dtype=torch.bool)
    odd[[i for i, w in enumerate(words.tolist()) if w >> 3 & 1], 5] = True
    got = out[:, 0].cpu()
    assert (torch.isnan if fmt == "e4m3" else torch.isposinf)(got[:, odd]).all()
    check(out[:, 0][:, ~odd], ref[:, 0][:, ~odd], tol[:, 0][:, ~odd])


@pytest.mark.parametrize("fmt,dtype", WIDE)
def test_many_nodes_that_see_nothing_give_zeros(wf, fmt, dtype):
    cache = make_cache(wf, fmt, 2, 1, 70, 64, 32)
    q = torch.randn(2, 20, 3, 64, generator=torch.Generator().manual_seed(32)).to(TYPES[dtype])
    words = torch.tensor([[0, 2, 0], [0, 0, 7]])
    out = wf.tree_decode(q.cuda(), cache, ints([0, 67]), tree=words.cuda(), nodes=ints([2, 3]))
    ref, tol = attend(fmt, cache, q, [0, 67], words.tolist(), [2, 3])
    assert not out[0, :, 0].any() and not out[0, :, 2].any()
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", WIDE)
@pytest.mark.parametrize("d", [64, 128])
def test_large_rising_scores_of_many_rows(wf, fmt, dtype, d):
    h, g, n, length = 2, 20, 2, 1500
    cache = wf.KVCache(1, h, length, d, fmt=fmt)
    ramp = torch.linspace(-1, 1, length)[:, None] + 0.02 * torch.randn(
        length, d, generator=torch.Generator().manual_seed(33))
    x = ramp.expand(1, h, length, d).contiguous().cuda()
    wf.cache_write(cache, x, x.flip(-1), ints([0]))
    q = (8 * torch.ones(1, h * g, n, d)).to(TYPES[dtype])
    q[..., 1, :] *= -1
    q[:, ::3] *= 0.01
    for scale in (None, 0.5):
        out = wf.tree_decode(q.cuda(), cache, ints([length - n]), scale=scale)
        ref, tol = attend(fmt, cache, q, [length - n], [[1, 3]], [n], scale)
        check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", WIDE)
def test_many_rows_over_values_of_very_different_sizes(wf, fmt, dtype):
    # the largest rows of V have almost no weight, and come last
    d, length, g = 64, 600, 40
    rng = np.random.default_rng(34)
    cache = wf.KVCache(1, 1, length, d, fmt=fmt)
    k = rng.standard_normal((1, 1, length, d)).astype(np.float32)
    v = rng.standard_normal((1, 1, length, d)).astype(np.float32)
    k[..., 300::50, :] = -3.0
    v[..., 300::50, :] *= 4096
    wf.cache_write(cache, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints([0]))
    q = torch.linspace(0.5, 1, g).reshape(1, g, 1, 1).expand(1, g, 1, d).to(TYPES[dtype])
    out = wf.tree_decode(q.cuda(), cache, ints([length - 1]))
    ref, tol = attend(fmt, cache, q, [length - 1], [[1]], [1])
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", WIDE)
@pytest.mark.parametrize("d", [64, 128])
def test_many_rows_of_strided_queries_outputs_and_caches(wf, fmt, dtype, d):
    b, n, hq, lens = 3, 7, 12, [0, 90, 33]
    big = make_cache(wf, fmt, 2 * b, 4, 99, d, 35)
    part = wf.KVCache.wrap(*(None if t is None else t[1::2, 1:3] for t in
                             (big.k, big.v, big.k_scale, big.v_scale)))
    q = torch.randn(b, n, hq, d + 3, generator=torch.Generator().manual_seed(35))
    q = q.to(TYPES[dtype])[..., 1:1 + d].transpose(1, 2)
    qc = torch.empty(b, n, hq, d + 3, dtype=q.dtype, device="cuda")[..., 1:1 + d].transpose(1, 2)
    qc.copy_(q)
    store = torch.full((b, hq, n, d + 9), 5.0, dtype=q.dtype, device="cuda")
    out = store[..., 7:7 + d]
    words = wf.tree_words(random_trees(b, n, 35))
    assert wf.tree_decode(qc, part, ints(lens), tree=words.cuda(), out=out) is out
    ref, tol = attend(fmt, part, q, lens, words.tolist(), [n] * b)
    check(out, ref, tol)
    assert (store[..., :7] == 5).all() and (store[..., 7 + d:] == 5).all()
    # the output in the place of the queries, one query head for all of a group
    wf.tree_decode(qc, part, ints(lens), tree=words.cuda(), out=qc)
    assert torch.equal(qc, out)


@pytest.mark.parametrize("fmt,dtype", WIDE)
def test_lengths_of_many_rows_are_clamped_and_reported(wf, fmt, dtype):
    from warpforth_b200 import _lib, warpforth

    cache = make_cache(wf, fmt, 4, 1, 40, 64, 36)
    q = torch.randn(4, 10, 4, 64, generator=torch.Generator().manual_seed(36)).to(TYPES[dtype])
    out = wf.tree_decode(q.cuda(), cache, ints([-5, 38, 1000, 10]), nodes=ints([4, 4, 4, 9]))
    with pytest.raises(_lib.WfattnError, match="length"):
        warpforth.device_status()
    ref, tol = attend(fmt, cache, q, [0, 38, 40, 10], [[1, 3, 7, 15]] * 4, [4, 2, 0, 4])
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("d,g,n", [(64, 1, 2), (128, 4, 12), (64, 8, 61)])
def test_trees_over_one_long_sequence(wf, fmt, dtype, d, g, n):
    # one cache head dealt to the whole GPU: 8,000 keys, up to 488 query rows
    length = 8000
    cache = make_cache(wf, fmt, 1, 1, length + n, d, 37)
    q = torch.randn(1, g, n, d, generator=torch.Generator().manual_seed(37)).to(TYPES[dtype])
    words = wf.tree_words(random_trees(1, n, 37)[0])
    out = wf.tree_decode(q.cuda(), cache, ints([length]), tree=words.cuda())
    ref, tol = attend(fmt, cache, q, [length], [words.tolist()], [n])
    check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_the_smallest_cache(wf, fmt, dtype):
    for d in (64, 128):
        cache = make_cache(wf, fmt, 1, 1, 1, d, 39)
        q = torch.randn(1, 70, 1, d, generator=torch.Generator().manual_seed(39)).to(TYPES[dtype])
        for g in (1, 12, 70):
            for length, nodes in ((0, 1), (1, 0), (0, 0)):
                out = wf.tree_decode(q[:, :g].cuda(), cache, ints([length]), nodes=ints([nodes]))
                ref, tol = attend(fmt, cache, q[:, :g], [length], [[1]], [nodes])
                check(out, ref, tol)


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_the_most_query_rows(wf, fmt, dtype):
    """2^20 of one cache head: 16,384 query heads that are one in memory, of 64 nodes."""
    d, g, n, length = 64, 1 << 14, 64, 70
    cache = make_cache(wf, fmt, 1, 1, length + n, d, 40)
    q = torch.randn(1, 1, n, d, generator=torch.Generator().manual_seed(40)).to(TYPES[dtype])
    words = wf.tree_words(random_trees(1, n, 40)[0])
    out = wf.tree_decode(q.cuda().expand(1, g, n, d), cache, ints([length]), tree=words.cuda())
    ref, tol = attend(fmt, cache, q, [length], [words.tolist()], [n])
    check(out[:, :1], ref, tol)
    check(out[:, -1:], ref, tol)
    low, high = out.amin(1, keepdim=True), out.amax(1, keepdim=True)
    check(low, ref, tol)
    check(high, ref, tol)


# ---------------------------------------------------------------------- used together


@pytest.mark.parametrize("fmt,dtype", KINDS)
def test_drafting_steps_as_they_are_used(wf, fmt, dtype):
    """Prompt, drafted trees, kept nodes and single tokens: every attention equals the formula
    over the tokens that were kept."""
    b, h, g, d, n = 2, 2, 2, 64, 6
    gen = torch.Generator().manual_seed(17)
    cache = wf.KVCache(b, h, 96, d, fmt=fmt)
    ws = wf.DecodeWorkspace()
    lens = [37, 5]

    def rows(count):
        return torch.randn(b, h, count, d, generator=gen).to(TYPES[dtype]).cuda()

    device_lens = ints([0, 0])
    wf.cache_write(cache, rows(40), rows(40), device_lens, counts=ints(lens))
    device_lens = ints(lens)
    for step in range(4):
        trees = random_trees(b, n, step)
        words = wf.tree_words(trees)
        wf.cache_write(cache, rows(n), rows(n), device_lens)
        q = torch.randn(b, h * g, n, d, generator=gen).to(TYPES[dtype])
        out = wf.tree_decode(q.cuda(), cache, device_lens, tree=words.cuda(), workspace=ws)
        ref, tol = attend(fmt, cache, q, lens, words.tolist(), [n] * b)
        check(out, ref, tol)
        # keep the way from the root to the last node
        paths = []
        for tree in trees:
            path = [n - 1]
            while tree[path[0]] >= 0:
                path.insert(0, tree[path[0]])
            paths.append(path)
        counts = [len(p) for p in paths]
        path = ints([p + [0] * (n - len(p)) for p in paths])
        stored = values(fmt, cache.k.cpu(), None if cache.k_scale is None else cache.k_scale.cpu())
        device_lens = wf.cache_keep(cache, device_lens, path, counts=ints(counts))
        after, _ = wf.cache_read(cache, ints([0, 0]), 96, counts=device_lens, dtype=torch.float32)
        for i in range(b):
            want = np.concatenate([stored[i, :, :lens[i]],
                                   stored[i][:, [lens[i] + p for p in paths[i]]]], 1)
            lens[i] += counts[i]
            assert np.array_equal(after[i, :, :lens[i]].cpu().numpy(), want.astype(np.float32))
        assert device_lens.tolist() == lens
        # the last kept token again, as a single step, sees what the last node saw
        q1 = q[:, :, n - 1:]
        single = wf.tree_decode(q1.cuda(), cache, device_lens - 1, workspace=ws)
        ref1, tol1 = attend(fmt, cache, q1, [x - 1 for x in lens], [[1]] * b, [1] * b)
        check(single, ref1, tol1)


@pytest.mark.parametrize("fmt,dtype", [("e4m3", "bf16"), ("f32", "f32")])
def test_captured_steps_replay_with_new_lengths(wf, fmt, dtype):
    b, h, d, n = 2, 3, 64, 3
    cache = wf.KVCache(b, h, 400, d, fmt=fmt)
    ws = wf.DecodeWorkspace()
    gen = torch.Generator().manual_seed(18)
    x = torch.randn(2, b, h, n, d, generator=gen).to(TYPES[dtype]).cuda()
    q = torch.randn(b, 2 * h, n, d, generator=gen).to(TYPES[dtype])
    prompt = torch.randn(b, h, 390, d, generator=gen).to(TYPES[dtype]).cuda()
    wf.cache_write(cache, prompt, prompt, ints([0, 0]))
    qc, lens, path = q.cuda(), ints([300, 2]), ints([[0, 2], [1, 2]])
    out, new = torch.empty_like(qc), torch.empty_like(lens)

    def step():
        wf.cache_write(cache, x[0], x[1], lens)
        wf.tree_decode(qc, cache, lens, out=out, workspace=ws)
        wf.cache_keep(cache, lens, path, out=new)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for at in ([300, 2], [17, 397], [0, 250]):
        lens.copy_(ints(at))
        graph.replay()
        got = out.clone()
        assert new.tolist() == [i + 2 for i in at]
        wf.cache_write(cache, x[0], x[1], lens)
        ref, tol = attend(fmt, cache, q, at, [[1, 3, 7]] * b, [n] * b)
        check(got, ref, tol)


@pytest.mark.parametrize("n", [1, 16])
def test_a_captured_step_outlives_its_workspace(wf, n):
    """A larger call through the same workspace gets a larger buffer; a graph
    captured before replays with the one that it has."""
    d, ws = 64, wf.DecodeWorkspace()
    small = make_cache(wf, "e4m3", 1, 1, 200 + n, d, 24)
    large = make_cache(wf, "e4m3", 10, 8, 516, 128, 25)
    gen = torch.Generator().manual_seed(26)
    q = torch.randn(1, 4, n, d, generator=gen).bfloat16().cuda()
    lens, out = ints([200]), torch.zeros_like(q)
    want = wf.tree_decode(q, small, lens, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        wf.tree_decode(q, small, lens, out=out, workspace=ws)
    before = ws.get_tree(1, q.device)
    big = torch.randn(10, 32, 16, 128, generator=gen).bfloat16().cuda()
    all_lens = ints([500 - 7 * i for i in range(10)])
    want_big = wf.tree_decode(big, large, all_lens)
    for _ in range(2):
        got_big = wf.tree_decode(big, large, all_lens, workspace=ws)
        graph.replay()
        assert torch.equal(got_big, want_big)
        assert torch.equal(out, want)
        out.zero_()
    assert ws.get_tree(1, q.device).numel() > before.numel()


@pytest.mark.parametrize("n", [1, 16, 40])
def test_a_workspace_first_used_in_a_capture(wf, n):
    """Calls outside it, before the graph's first replay and between two, join their parts by
    counters of their own; so does a second graph that is replayed first."""
    d, ws, length = 64, wf.DecodeWorkspace(), 6000
    cache = make_cache(wf, "e4m3", 1, 1, length + n, d, 27)
    q = torch.randn(1, 1, n, d, generator=torch.Generator().manual_seed(27)).bfloat16().cuda()
    lens = ints([length])
    want = wf.tree_decode(q, cache, lens)
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    torch.cuda.synchronize()
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            wf.tree_decode(q, cache, lens, out=out, workspace=ws)
            wf.tree_decode(q, cache, lens, out=out, workspace=ws)
    for _ in range(2):
        for graph, out in reversed(list(zip(graphs, outs))):
            got = torch.zeros_like(q)
            wf.tree_decode(q, cache, lens, out=got, workspace=ws)
            graph.replay()
            assert torch.equal(got, want) and torch.equal(out, want)
            out.zero_()


def test_calls_on_two_streams_at_once(wf):
    d, n, length = 128, 8, 3000
    caches = [make_cache(wf, "e4m3", 1, 2, length + n, d, 19 + i) for i in range(2)]
    q = torch.randn(1, 8, n, d, generator=torch.Generator().manual_seed(19)).bfloat16()
    qc, lens = q.cuda(), ints([length])
    want = [wf.tree_decode(qc, c, lens) for c in caches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [wf.DecodeWorkspace() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(wf.tree_decode(qc, caches[i], lens, workspace=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])  # no atomics: the same bits
