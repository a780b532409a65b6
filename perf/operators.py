"""Cases of the cache operators: writing a key/value cache (f32, bf16, e4m3 or 4-bit rows), reading
rows of it back, keeping the accepted rows of a drafted tree, and attention of a tree of drafted
tokens (one token included) over the cache.

Formats of a cache row (one token of one head, D values):

* ``f32`` / ``bf16``: the values, rounded to the type;
* ``e4m3``: one e4m3 code a value and one f32 scale a row, the smallest power of two s >= 2^-126
  with max|x| <= 448 s; the code is x / s rounded to nearest even, the value it stands for code * s;
* ``int4``: one 4-bit code u a value (value 2i in the low half of byte i) and two bf16 numbers a
  row, (s, m): m is the largest bf16 <= min(x), s the smallest bf16 >= (max(x) - m) / 15, and u is
  (x - m) / s in f32, rounded to nearest even, in 0..15; it stands for m + s u.

Attention: node i of sequence b sees the kv_lens[b] rows before the tree and those nodes j < nodes[b]
of the tree, at rows kv_lens[b] + j, whose bit j is set in word i; a node that sees nothing, and a
padding node i >= nodes[b], gives zeros.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_ROW_BYTES = {"f32": 4.0, "bf16": 2.0, "e4m3": 1.0, "int4": 0.5}  # bytes a value
_LOW = -126


# ------------------------------------------------------------------------------------ cases


def listed():
    return [
        # one decode step's new K/V rows of a served batch go into an 8-bit cache (latency)
        dict(name="write step e4m3", op="write", fmt="e4m3", dtype="bf16", B=64, H=8, D=128, T=1,
             lo=1, hi=1, L=1031),
        # GPT-2 in f32: a step's rows of its 12 heads into a 4-bit cache (the smallest call)
        dict(name="write gpt2 int4", op="write", fmt="int4", dtype="f32", B=1, H=12, D=64, T=7,
             lo=7, hi=7, L=1024),
        # a batch of ragged prompts written after prefill, read back for the next chunk
        dict(name="write prompts int4", op="write", fmt="int4", dtype="bf16", B=8, H=16, D=128,
             T=4999, lo=1250, hi=4999, L=5003),
        # a cached prefix of several sequences read back as bf16 for a chunked prefill
        dict(name="read prefix e4m3", op="read", fmt="e4m3", dtype="bf16", B=16, H=12, D=64,
             T=8192, lo=2048, hi=8192, L=8192),
        # a short prefix of an f32 model read back from a 4-bit cache
        dict(name="read short int4", op="read", fmt="int4", dtype="f32", B=3, H=12, D=64, T=129,
             lo=1, hi=129, L=1024),
        # the accepted nodes of one drafted tree, GPT-2 in f32
        dict(name="keep gpt2 f32", op="keep", fmt="f32", dtype="f32", B=1, H=12, D=64, T=16,
             lo=2, hi=5, L=1024),
        # the accepted nodes of a served batch's trees
        dict(name="keep batch e4m3", op="keep", fmt="e4m3", dtype="bf16", B=256, H=8, D=128, T=63,
             lo=0, hi=9, L=515),
        # one token of GPT-2 over its f32 cache (latency)
        dict(name="step gpt2 f32", op="tree", fmt="f32", dtype="f32", B=1, H=12, G=1, D=64, T=1,
             lo=159, hi=159, L=1024),
        # one token of a batch of ragged sequences, every head with its own K/V
        dict(name="step ragged e4m3", op="tree", fmt="e4m3", dtype="bf16", B=64, H=25, G=1, D=64,
             T=1, lo=512, hi=4038, L=4096),
        # one token with shared K/V heads over a 4-bit cache
        dict(name="step shared int4", op="tree", fmt="int4", dtype="bf16", B=32, H=8, G=8, D=128,
             T=1, lo=5000, hi=16383, L=16384),
        # small drafted trees over a bf16 cache with shared heads
        dict(name="tree bf16", op="tree", fmt="bf16", dtype="bf16", B=16, H=8, G=4, D=128, T=15,
             lo=700, hi=4000, L=4096),
        # a large drafted tree over one long 8-bit cache
        dict(name="tree long e4m3", op="tree", fmt="e4m3", dtype="bf16", B=2, H=8, G=4, D=128,
             T=61, lo=65000, hi=131000, L=131072),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("write", "read", "keep", "tree", "tree", "tree"))
    fmt = rng.choice(("f32", "bf16", "e4m3", "e4m3", "int4", "int4"))
    c = dict(op=op, fmt=fmt, D=rng.choice((64, 128)), B=_log_int(rng, 1, 128),
             H=rng.choice((1, 2, 5, 8, 12, 16, 25)))
    # attention takes a plain cache with a query of its type, a quantised one with either
    c["dtype"] = fmt if fmt in _TYPES and op == "tree" else rng.choice(("f32", "bf16"))
    if op == "tree":
        c["G"] = rng.choice((1, 1, 2, 4, 5, 8))
        c["T"] = rng.choice((1, 1, _log_int(rng, 2, 64)))
        c["hi"] = _log_int(rng, 1, 65536)
        c["lo"] = rng.randint(0, c["hi"])
        c["L"] = c["hi"] + c["T"] + rng.randint(0, 9)
    elif op == "keep":
        c["T"] = rng.randint(1, 64)
        c["hi"] = rng.randint(0, min(12, c["T"]))
        c["lo"] = rng.randint(0, c["hi"])
        c["L"] = c["T"] + _log_int(rng, 1, 1000)
    else:
        c["T"] = c["hi"] = rng.choice((1, _log_int(rng, 1, 8192)))
        c["lo"] = rng.randint(0, c["hi"])
        c["L"] = c["T"] + rng.randint(0, 40)
    top = {k: max(work(x)[k] for x in listed()) for k in ("bytes", "flops")}
    rows = 80e6 * 2  # values of K and V in the cache: what the plain form has to hold
    while c["B"] > 1 and (work(c)["bytes"] > top["bytes"] / 2 or work(c)["flops"] > top["flops"] / 2
                          or 2 * c["B"] * c["H"] * c["L"] * c["D"] > rows):
        c["B"] -= max(1, c["B"] // 4)
    while 2 * c["B"] * c["H"] * c["L"] * c["D"] > rows:
        c["H"] = max(1, c["H"] // 2)
    return c


def _spread(case):
    """B lengths evenly spread over lo..hi, the longest first."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, B - 1) for i in range(B)]


def work(case):
    B, H, D, T = case["B"], case["H"], case["D"], case["T"]
    total = sum(_spread(case))
    row = D * _ROW_BYTES[case["fmt"]] + (0 if case["fmt"] in _TYPES else 4)
    vec = D * (4 if case["dtype"] == "f32" else 2)
    if case["op"] == "write":  # new rows in, stored rows out and in again, values out
        return {"bytes": 2 * H * total * (2 * vec + 2 * row) + 8 * B, "flops": 8 * H * total * D}
    if case["op"] == "read":
        return {"bytes": 2 * H * total * (vec + row) + 8 * B, "flops": 4 * H * total * D}
    if case["op"] == "keep":  # stored rows in and out, the paths, the lengths
        return {"bytes": 4 * H * total * row + 4 * total + 12 * B, "flops": 0}
    G = case["G"]
    keys = total + B * T
    return {"bytes": 2 * H * keys * row + 2 * B * H * G * T * vec + 8 * B * T + 8 * B,
            "flops": 4 * H * G * T * keys * D}


# ----------------------------------------------------------------------------------- inputs


def _bits(x):
    return x.view(torch.int32)


def _values(shape, gen):
    """Keys or values of a model: every token and head with a size of its own."""
    size = torch.exp(0.5 * torch.randn(*shape[:-1], 1, generator=gen, device="cuda"))
    return torch.randn(*shape, generator=gen, device="cuda") * size


def _cache_of(case, gen):
    """A cache whose rows hold earlier tokens: codes and scales."""
    B, H, L, D = case["B"], case["H"], case["L"], case["D"]
    got = {}
    for n in ("k", "v"):
        codes, scale = _pack(case["fmt"], _values((B, H, L, D), gen))
        got[n], got[n + "_scale"] = codes, scale
    return got


def _tree(B, T, gen):
    """Trees of T nodes: every node's parent is an earlier one, near it more often than not."""
    i = torch.arange(T, device="cuda")
    back = 1 + (torch.rand(B, T, generator=gen, device="cuda") ** 2 * i).long()
    parent = (i - back).clamp_min(0)
    sees = torch.eye(T, dtype=torch.bool, device="cuda").expand(B, T, T).clone()
    for t in range(1, T):
        sees[:, t] |= sees.gather(1, parent[:, t].view(B, 1, 1).expand(B, 1, T))[:, 0]
    return (sees.long() << i).sum(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, D, T, L = case["B"], case["H"], case["D"], case["T"], case["L"]
    dtype = _TYPES[case["dtype"]]
    order = torch.randperm(B, generator=gen, device="cuda")
    spread = torch.tensor(_spread(case), dtype=torch.int32, device="cuda")[order]
    s = dict(case=case, **_cache_of(case, gen))
    if case["op"] == "write":
        # as a model's projection leaves them: [B, T, H, D], seen as [B, H, T, D]
        s["new_k"], s["new_v"] = (_values((B, T, H, D), gen).to(dtype).transpose(1, 2)
                                  for _ in range(2))
        s["starts"] = torch.randint(0, L - T + 1, (B,), generator=gen, device="cuda",
                                    dtype=torch.int32)
        s["counts"] = spread
    elif case["op"] == "read":
        s["starts"] = torch.zeros(B, dtype=torch.int32, device="cuda")
        s["counts"] = spread
    elif case["op"] == "keep":
        deep = max(1, case["hi"])
        s["lens"] = torch.randint(0, L - T + 1, (B,), generator=gen, device="cuda",
                                  dtype=torch.int32)
        # a path from the root: nodes in rising order
        pick = torch.rand(B, T, generator=gen, device="cuda").topk(deep, dim=1).indices
        s["path"] = pick.sort(dim=1).values.to(torch.int32)
        s["counts"] = spread
    else:
        q = torch.randn(B, T, H * case["G"], D, generator=gen, device="cuda")
        s["q"] = q.to(dtype).transpose(1, 2)
        s["lens"] = spread
        s["tree"] = _tree(B, T, gen)
        fewer = torch.randint(0, 2, (B,), generator=gen, device="cuda") * (T // 3)
        s["nodes"] = (T - fewer).to(torch.int32)
    if own:
        import warpforth_b200 as wf

        # the cache's handle and the scratch that a program keeps from call to call
        s["cache"] = wf.KVCache.wrap(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["workspace"] = wf.DecodeWorkspace()
    return s


# --------------------------------------------------------------------------------- operators


def run(s):
    case = s["case"]
    if own:
        import warpforth_b200 as wf

        cache = s["cache"]
        if case["op"] == "write":
            wf.cache_write(cache, s["new_k"], s["new_v"], s["starts"], counts=s["counts"])
        if case["op"] in ("write", "read"):
            return wf.cache_read(cache, s["starts"], case["T"], counts=s["counts"],
                                 dtype=_TYPES[case["dtype"]])
        if case["op"] == "keep":
            lens = wf.cache_keep(cache, s["lens"], s["path"], counts=s["counts"])
            return _stored(s) + [lens]
        return wf.tree_decode(s["q"], cache, s["lens"], tree=s["tree"], nodes=s["nodes"],
                              workspace=s["workspace"])
    if case["op"] == "write":
        _write(s)
    if case["op"] in ("write", "read"):
        return _read(s)
    if case["op"] == "keep":
        return _stored(s) + [_keep(s)]
    return _attend(s)


def _stored(s):
    """The cache's own buffers: rows are moved as they are stored."""
    return [s[n].view(torch.uint8) if s["case"]["fmt"] == "e4m3" and n in "kv" else s[n]
            for n in ("k", "v", "k_scale", "v_scale") if s[n] is not None]


def _pack(fmt, x):
    """Codes and scales of rows x [..., D]."""
    if fmt in _TYPES:
        return x.to(_TYPES[fmt]), None
    x = x.float()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    if fmt == "e4m3":
        top = torch.where(bad, 0, x.abs().amax(-1, keepdim=True))
        e, frac = _bits(top) >> 23, _bits(top) & 0x7FFFFF
        e = (e - 127 - 8 + (frac > 0x600000)).clamp_min(_LOW)  # 448 = 1.75 * 2^8
        codes = torch.where(bad, 0, x * _power(-e)).to(torch.float8_e4m3fn)
        return codes, torch.where(bad, math.nan, _power(e)).squeeze(-1)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = _to_bf16(torch.where(bad, 0, low), down=True)
    s = _to_bf16((torch.where(bad, 0, high) - m) / torch.full_like(m, 15), down=False)
    bad = bad | ~torch.isfinite(s)
    u = torch.where(bad | (s == 0), 0, ((x - m) / s).round()).clamp(0, 15).to(torch.uint8)
    scale = torch.where(bad, math.nan, torch.cat((s, m), -1)).to(torch.bfloat16)
    return u[..., 0::2] | u[..., 1::2] << 4, scale


def _power(e):
    """2^e in f32, exactly, for -126 <= e <= 127."""
    return ((e + 127) << 23).view(torch.float32)


def _to_bf16(x, down):
    """x as the nearest bf16 not above it (down) or not below it, in f32."""
    cut = (_bits(x) & -65536).view(torch.float32)  # towards zero
    step = (_bits(cut) + 65536).view(torch.float32)  # away from it
    return torch.where((cut > x) if down else (cut < x), step, cut)


def _unpack(fmt, codes, scale):
    """The values of rows, in f32."""
    if fmt in _TYPES:
        return codes.float()
    if fmt == "e4m3":
        return codes.float() * scale[..., None]
    u = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return scale[..., 1:].float() + scale[..., :1].float() * u


def _rows(s, starts, n):
    """Indices [B, H, n] of the rows starts[b] + 0..n-1, as far as the cache goes."""
    B, H = s["case"]["B"], s["case"]["H"]
    at = starts.long()[:, None] + torch.arange(n, device="cuda")
    return (torch.arange(B, device="cuda")[:, None, None],
            torch.arange(H, device="cuda")[None, :, None],
            at.clamp_max(s["case"]["L"] - 1)[:, None, :])


def _write(s):
    fmt, T = s["case"]["fmt"], s["case"]["T"]
    at = _rows(s, s["starts"], T)
    live = (torch.arange(T, device="cuda") < s["counts"][:, None])[:, None, :]
    live = live.expand(s["case"]["B"], s["case"]["H"], T)
    to = tuple(i.expand_as(live)[live] for i in at)
    for n in ("k", "v"):
        codes, scale = _pack(fmt, s["new_" + n][live])
        codes8 = s[n].view(torch.uint8) if fmt == "e4m3" else s[n]
        codes8[to] = codes.view(torch.uint8) if fmt == "e4m3" else codes
        if scale is not None:
            s[n + "_scale"][to] = scale


def _read(s):
    T, dtype = s["case"]["T"], _TYPES[s["case"]["dtype"]]
    at = _rows(s, s["starts"], T)
    live = (torch.arange(T, device="cuda") < s["counts"][:, None])[:, None, :, None]
    got = []
    for n in ("k", "v"):
        codes = s[n].view(torch.uint8)[at].view(s[n].dtype)
        scale = None if s[n + "_scale"] is None else s[n + "_scale"][at]
        got.append(torch.where(live, _unpack(s["case"]["fmt"], codes, scale), 0).to(dtype))
    return tuple(got)


def _keep(s):
    deep = s["path"].shape[1]
    lens, counts = s["lens"], s["counts"]
    b, h, to = _rows(s, lens, deep)
    come = (lens[:, None] + s["path"]).long()[:, None, :]
    live = (torch.arange(deep, device="cuda") < counts[:, None])[:, None, :]
    live = live.expand(s["case"]["B"], s["case"]["H"], deep)
    b, h, to, come = (i.expand_as(live)[live] for i in (b, h, to, come))
    for n in ("k", "v", "k_scale", "v_scale"):
        if s[n] is not None:
            x = s[n].view(torch.uint8) if s[n].dtype == torch.float8_e4m3fn else s[n]
            x[b, h, to] = x[b, h, come]
    return lens + counts


def _attend(s):
    c = s["case"]
    B, H, G, D, T, L = (c[n] for n in ("B", "H", "G", "D", "T", "L"))
    k, v = (_unpack(c["fmt"], s[n], s[n + "_scale"]) for n in ("k", "v"))
    q = s["q"].float().reshape(B, H, G * T, D)
    x = (q @ k.transpose(-1, -2)).view(B, H, G, T, L) / math.sqrt(D)
    lens, nodes = s["lens"].long(), s["nodes"].long()
    j = torch.arange(L, device="cuda") - lens[:, None]  # [B, L]: which node a row holds
    bit = s["tree"][:, :, None] >> j.clamp(0, 63)[:, None, :] & 1
    sees = (j < 0)[:, None, :] | ((bit == 1) & (j < nodes[:, None])[:, None, :])
    sees = sees & (torch.arange(T, device="cuda") < nodes[:, None])[:, :, None]
    x = torch.where(sees[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0, top))
    o = (p.view(B, H, G * T, L) @ v).view(B, H * G, T, D)
    total = p.sum(-1, keepdim=True).view(B, H * G, T, 1)
    return (o / torch.where(total == 0, 1, total)).to(s["q"].dtype)


# --------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The operators' definitions in 64 bits, sequence by sequence."""
    if case["op"] == "keep":
        return None  # rows are moved, nothing is computed
    s = prepare(case, seed)
    B, T, fmt = case["B"], case["T"], case["fmt"]
    starts, counts = (s[n].tolist() if n in s else [0] * B for n in ("starts", "counts"))
    if case["op"] == "tree":
        return torch.stack([_exact_attention(s, b) for b in range(B)])
    if case["op"] == "write" and fmt == "int4" and case["dtype"] == "f32":
        return None  # the codes are defined by f32 arithmetic; f32 values show every one of them
    got = {}
    for n in ("k", "v"):
        got[n] = torch.zeros(B, case["H"], T, case["D"], dtype=torch.float64, device="cuda")
        for b in range(B):
            if case["op"] == "write":
                rows = _exact_rounding(fmt, s["new_" + n][b, :, :counts[b]].double())
            else:
                rows = _exact_values(s, n, b, starts[b], starts[b] + counts[b])
            got[n][b, :, :counts[b]] = rows
    return got["k"], got["v"]


def _exact_values(s, n, b, lo, hi):
    fmt, codes = s["case"]["fmt"], s[n][b, :, lo:hi]
    if fmt in _TYPES:
        return codes.double()
    scale = s[n + "_scale"][b, :, lo:hi].double()
    if fmt == "int4":
        u = torch.empty(*codes.shape[:-1], s["case"]["D"], dtype=torch.float64, device="cuda")
        u[..., 0::2], u[..., 1::2] = (codes % 16).double(), (codes // 16).double()
        return u * scale[..., 0:1] + scale[..., 1:2]
    i = torch.arange(256, dtype=torch.float64, device="cuda")
    field, frac = i % 128 // 8, i % 8 / 8
    table = torch.where(field == 0, frac * 2.0 ** -6, (1 + frac) * _exact_power(field - 7))
    table = torch.where(i >= 128, -table, table)
    return table[codes.view(torch.uint8).long()] * scale[..., None]


def _exact_rounding(fmt, x):
    if fmt == "f32":
        return x  # what is written is at most 32 bits wide
    if fmt == "bf16":
        return _nearest(x, 7, -126)
    if fmt == "e4m3":
        f, e = torch.frexp(x.abs().amax(-1, keepdim=True))  # f in [1/2, 1); 448 = 7/8 * 2^9
        e = (e - 9 + (f > 7 / 8)).clamp_min(_LOW)
        return _nearest(x / _exact_power(e), 3, -6) * _exact_power(e)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)

    def grid(y, to):
        unit = _exact_power(torch.frexp(y).exponent - 8)
        return to(y / unit) * unit

    m = grid(low, torch.floor)
    s = grid((high - m) / 15, torch.ceil)
    return m + s * torch.where(s == 0, 0, torch.round((x - m) / s)).clamp(0, 15)


def _exact_power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _nearest(x, bits, lowest):
    """x rounded to `bits` bits of fraction, exponents from `lowest` on."""
    unit = _exact_power((torch.frexp(x).exponent - 1).clamp_min(lowest) - bits)
    return torch.round(x / unit) * unit


def _exact_attention(s, b):
    c = s["case"]
    H, G, D, T = c["H"], c["G"], c["D"], c["T"]
    n, nodes = int(s["lens"][b]), int(s["nodes"][b])
    o = torch.zeros(H * G, T, D, dtype=torch.float64, device="cuda")
    words = s["tree"][b].tolist()
    masks = torch.ones(nodes, n + nodes, dtype=torch.bool)
    for i in range(nodes):
        masks[i, n:] = torch.tensor([words[i] >> j & 1 == 1 for j in range(nodes)])
    masks = masks.to("cuda")
    k, v = (_exact_values(s, x, b, 0, n + nodes) for x in ("k", "v"))
    for head in range(H * G):
        x = s["q"][b, head, :nodes].double() @ k[head // G].T * D ** -0.5
        x = x.masked_fill(~masks, -math.inf)
        o[head, :nodes] = torch.softmax(x, -1) @ v[head // G]
    return o
