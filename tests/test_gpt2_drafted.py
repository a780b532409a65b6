"""Generation with drafted trees over a key/value cache: drafting and acceptance on the CPU, GPT-2 on
the GPU.  Over an f32 cache the tokens are those of plain greedy generation; a difference is only
accepted where the stock model's top two logits are within 1e-4 (a tie that f32 rounding may break
either way)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytest.importorskip("transformers")


def test_drafts_follow_the_longest_earlier_match_first():
    from warpforth_b200.gpt2 import draft_tree

    tokens = [1, 2, 3, 9, 4, 5, 2, 3, 7, 8, 1, 2, 3]
    drafted, parents = draft_tree(tokens, 64, depth=2)
    # after 1 2 3 came 9 4; after 2 3 came 7 8 too
    assert drafted == [3, 9, 4, 7, 8] and parents == [-1, 0, 1, 0, 3]
    assert draft_tree(tokens, 1) == ([3], [-1])
    drafted, parents = draft_tree(tokens, 4, depth=8)
    assert drafted == [3, 9, 4, 5] and parents == [-1, 0, 1, 2]
    assert draft_tree([5], 8) == ([5], [-1])
    assert draft_tree([5, 6], 8) == ([6], [-1])
    drafted, parents = draft_tree([4, 4, 4, 4], 8)
    assert drafted[:2] == [4, 4] and all(p < i for i, p in enumerate(parents))


def test_acceptance_walks_the_chosen_tokens():
    from warpforth_b200.gpt2 import accepted_path

    drafted, parents = [3, 9, 4, 7, 8], [-1, 0, 1, 0, 3]
    assert accepted_path(drafted, parents, [7, 0, 0, 8, 1]) == [0, 3, 4]
    assert accepted_path(drafted, parents, [9, 5, 0, 0, 0]) == [0, 1]
    assert accepted_path(drafted, parents, [1, 4, 0, 8, 0]) == [0]
    assert accepted_path([3], [-1], [3]) == [0]


class PlainCache:
    """A KVCache's rows in plain tensors."""

    def __init__(self, batch, heads, max_len, head_dim, *, fmt, device):
        self.k, self.v = (torch.zeros(batch, heads, max_len, head_dim) for _ in range(2))


@pytest.fixture
def on_cpu(monkeypatch):
    """warpforth_b200.gpt2 with the cache calls in plain operations, for one f32 sequence."""
    from warpforth_b200 import gpt2

    def write(cache, k, v, starts):
        at = slice(int(starts), int(starts) + k.shape[2])
        cache.k[:, :, at], cache.v[:, :, at] = k, v

    def read(cache, starts, rows, dtype):
        return cache.k[:, :, :rows], cache.v[:, :, :rows]

    def keep(cache, lens, path):
        for t in (cache.k, cache.v):
            t[:, :, int(lens):int(lens) + path.shape[1]] = t[:, :, int(lens) + path[0].long()]
        return lens + path.shape[1]

    def attend(q, k, v, mask, scale):
        return (q @ k.mT * scale).masked_fill(~mask, -torch.inf).softmax(-1) @ v

    def tree(q, cache, lens, tree, scale, workspace):
        rows, n = int(lens), q.shape[2]
        sees = (tree[:, None] >> torch.arange(n) & 1).bool()
        mask = torch.cat([torch.ones(n, rows, dtype=torch.bool), sees], 1)
        return attend(q, cache.k[:, :, :rows + n], cache.v[:, :, :rows + n], mask, scale)

    def causal(q, k, v, causal, scale):
        n, rows = q.shape[2], k.shape[2]
        return attend(q, k, v, torch.ones(n, rows, dtype=torch.bool).tril(rows - n), scale)

    for name, f in (("KVCache", PlainCache), ("cache_write", write), ("cache_read", read),
                    ("cache_keep", keep), ("tree_decode", tree), ("attention", causal)):
        monkeypatch.setattr(gpt2, name, f)
    return gpt2


def _small_gpt2(seed=0, attention="eager", **kw):
    from transformers import GPT2Config, GPT2LMHeadModel

    torch.manual_seed(seed)
    model = GPT2LMHeadModel(GPT2Config(n_layer=3, n_embd=128, n_head=2, vocab_size=50,
                                       n_positions=64, initializer_range=0.2, **kw)).eval()
    if attention:
        model.set_attn_implementation(attention)
    return model


def _greedy(model, prompt, count):
    ids = prompt
    with torch.no_grad():
        for _ in range(count):
            ids = torch.cat([ids, model(ids, use_cache=False).logits[:, -1:].argmax(-1)], 1)
    return ids


@pytest.mark.parametrize("nodes,chunk", [(1, 512), (9, 512), (64, 3)])
def test_small_models_generate_the_greedy_tokens(on_cpu, nodes, chunk):
    model, prompt = _small_gpt2(), torch.arange(10).remainder(4)[None]
    want = _greedy(model, prompt, 20)
    got, _ = on_cpu.generate_drafted(model, prompt, 20, nodes=nodes, prompt_chunk=chunk)
    assert got.tolist() == want.tolist()


@pytest.mark.parametrize("kw", [dict(attention=None), dict(attention="sdpa"),
                                dict(reorder_and_upcast_attn=True)])
def test_models_that_pass_the_cache_by_are_refused(on_cpu, kw):
    model = _small_gpt2(**kw)
    with pytest.raises(RuntimeError, match="eager"):
        on_cpu.generate_drafted(model, torch.arange(10)[None], 5)
    # and the model attends as it did before
    _greedy(model, torch.arange(10)[None], 1)


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, "f32"), (torch.float32, "bf16"),
                                         (torch.float16, "f32"), (torch.float32, "e5m2")])
def test_caches_that_the_queries_do_not_take_are_refused_first(on_cpu, monkeypatch, dtype, cache):
    model = _small_gpt2().to(dtype)
    monkeypatch.setattr(model, "forward", None)  # never called
    with pytest.raises(ValueError, match="bfloat16 models .*'bf16'"):
        on_cpu.generate_drafted(model, torch.arange(10)[None], 5, cache=cache)


def test_other_models_and_threads_attend_as_ever_meanwhile(on_cpu, monkeypatch):
    """While one model generates: another one runs in the same thread, the same one in another, and
    a second generation begins and ends in a third."""
    from concurrent.futures import ThreadPoolExecutor

    import transformers.models.gpt2.modeling_gpt2 as gpt2_module

    stock = gpt2_module.eager_attention_forward
    model, other = _small_gpt2(0), _small_gpt2(1)
    prompt = torch.arange(10).remainder(4)[None]
    want, want_other = _greedy(model, prompt, 12), _greedy(other, prompt, 12)
    tree, seen = on_cpu.tree_decode, []

    def meddled(*args, **kwargs):
        monkeypatch.setattr(on_cpu, "tree_decode", tree)  # once
        seen.append(_greedy(other, prompt, 12))
        with ThreadPoolExecutor(1) as pool:
            seen.append(pool.submit(_greedy, model, prompt, 12).result())
            seen.append(pool.submit(on_cpu.generate_drafted, other, prompt, 12).result()[0])
        return tree(*args, **kwargs)

    monkeypatch.setattr(on_cpu, "tree_decode", meddled)
    got, _ = on_cpu.generate_drafted(model, prompt, 12)
    assert got.tolist() == want.tolist()
    assert [x.tolist() for x in seen] == [x.tolist() for x in (want_other, want, want_other)]
    assert gpt2_module.eager_attention_forward is stock


@pytest.fixture(scope="module")
def gpt2():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from warpforth_b200 import gpt2

    return gpt2


def _assert_same_or_tie(model, want, got, prompt_len):
    a, b = want[0].tolist(), got[0].tolist()
    assert len(a) == len(b)
    if a == b:
        return
    p = next(i for i in range(len(a)) if a[i] != b[i])
    assert p >= prompt_len
    with torch.no_grad():
        logits = model(want[:, :p]).logits[0, -1].float()
    top2 = torch.topk(logits, 2).values
    assert float(top2[0] - top2[1]) < 1e-4, f"tokens diverge at {p} without a tie"


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,chunk", [(1, 512), (12, 512), (64, 7)])
def test_drafted_tokens_are_the_greedy_ones(gpt2, nodes, chunk):
    model = gpt2.random_gpt2(seed=1)
    prompt = gpt2.synthetic_prompt(32, seed=1)
    want = gpt2.generate(model, prompt, 64, use_cache=True)
    got, runs = gpt2.generate_drafted(model, prompt, 64, nodes=nodes, prompt_chunk=chunk)
    assert got.shape == (1, 96) and 1 <= runs <= 63
    if nodes == 1:
        assert runs == 63
    _assert_same_or_tie(model, want, got, 32)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["e4m3", "int4"])
def test_quantised_caches_generate(gpt2, fmt):
    model = gpt2.random_gpt2(seed=2)
    prompt = gpt2.synthetic_prompt(40, seed=2)
    want = gpt2.generate(model, prompt, 1, use_cache=False)
    got, _ = gpt2.generate_drafted(model, prompt, 20, nodes=8, cache=fmt)
    assert got.shape == (1, 60)
    assert got[0, :40].tolist() == prompt[0].tolist()
    _assert_same_or_tie(model, want, got[:, :41], 40)  # the prompt is attended to unrounded


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int4"])
@pytest.mark.parametrize("nodes", [1, 64])
def test_bf16_models_generate(gpt2, fmt, nodes):
    model = gpt2.random_gpt2(seed=4).bfloat16()
    prompt = gpt2.synthetic_prompt(40, seed=4)
    got, runs = gpt2.generate_drafted(model, prompt, 12, nodes=nodes, cache=fmt, prompt_chunk=17)
    assert got.shape == (1, 52) and got[0, :40].tolist() == prompt[0].tolist()
    assert 1 <= runs <= 11 and (nodes > 1 or runs == 11)


@pytest.mark.gpu
def test_generation_to_the_last_position(gpt2):
    model = gpt2.random_gpt2(seed=3)
    prompt = torch.arange(990).remainder(5)[None]
    got, _ = gpt2.generate_drafted(model, prompt, 34, nodes=64, prompt_chunk=400)
    assert got.shape == (1, 1024)
    with pytest.raises(ValueError, match="positions"):
        gpt2.generate_drafted(model, prompt, 35)
    for bad in (dict(nodes=0), dict(nodes=65), dict(prompt_chunk=0)):
        with pytest.raises(ValueError):
            gpt2.generate_drafted(model, prompt[:, :4], 4, **bad)
    with pytest.raises(ValueError, match="prompt"):
        gpt2.generate_drafted(model, prompt[0], 4)
