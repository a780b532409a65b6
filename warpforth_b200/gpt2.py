"""GPT-2 generation with every attention routed through libwfattn.

Mirrors demo/gpt2_generate.py (tetsuo-cpp/warpforth): Hugging Face's
``modeling_gpt2.eager_attention_forward`` is replaced by a function that calls
the WarpForth attention kernel.  The reference loops over heads of batch entry
0 and launches one kernel per head (demo/gpt2_generate.py:35-52); here one
``attention`` call covers every batch entry and head, reads the strided
q/k/v views without copies, and runs on torch's current stream.

Semantics kept from the reference: causal masking only -- ``attention_mask``
(padding) and ``dropout`` are ignored, exactly as the reference ignores them;
``scaling`` is honoured (GPT-2 passes 1/sqrt(head_dim), the reference kernel's
fixed scale).  With a KV cache (``use_cache=True``, which the reference does
not support) the prompt goes through the prefill kernel and every later
single-token step through the split-KV decode kernel (``wfattn_decode_f32``
for the f32 model) over the cached keys and values.

``generate_drafted`` generates greedily over a ``KVCache`` of its own, f32, e4m3 or 4-bit: each step
drafts a small tree of tokens (what followed the last words where they stood before), attends from
all of them at once (``tree_decode``) and keeps those that the model would have chosen
(``cache_keep``).

    python -m warpforth_b200.gpt2 --max-tokens 128      # random-init GPT-2 small
    python -m warpforth_b200.gpt2 --draft-nodes 12 --cache e4m3
"""

from __future__ import annotations

import argparse
import contextlib
import threading
import time
from collections.abc import Callable

import torch

from .cache import KVCache, cache_keep, cache_read, cache_write, tree_decode, tree_words
from .warpforth import DecodeWorkspace, attention, decode


# library calls made by the patched attention, by kind (read by count_calls)
_calls = {"prefill": 0, "decode": 0}


def make_warpforth_eager_attn() -> Callable:
    """Replacement for transformers' eager_attention_forward (see the module docstring)."""

    workspace = DecodeWorkspace()
    lens_cache: dict = {}

    def warpforth_eager_attn(module, query, key, value, attention_mask=None, scaling=None,
                             dropout=0.0, **kwargs):
        b, _, sq, d = query.shape
        sk = key.shape[2]
        if (sq == 1 and sk > 1 and query.dtype in (torch.float32, torch.bfloat16)
                and d == 64 and key.stride(2) == d and value.stride(2) == d
                and key.stride(3) == 1 and value.stride(3) == 1):
            # one new token against the cached keys: the decode kernel
            _calls["decode"] += 1
            lens = lens_cache.get((b, sk, query.device))
            if lens is None:
                lens = torch.full((b,), sk, dtype=torch.int32, device=query.device)
                lens_cache[(b, sk, query.device)] = lens
            out = decode(query, key, value, lens, scale=scaling, workspace=workspace)
            return out.to(query.dtype).unsqueeze(1), None
        _calls["prefill"] += 1
        out = attention(query, key, value, causal=True, scale=scaling)
        return out.transpose(1, 2), None

    return warpforth_eager_attn


def count_calls(fn: Callable[[], object]) -> dict:
    """Runs fn() and returns how many prefill and decode calls the patched attention made."""
    before = dict(_calls)
    fn()
    return {k: _calls[k] - before[k] for k in _calls}


def patch_gpt2() -> Callable[[], None]:
    """Route GPT-2 attention through libwfattn; returns a function that undoes it."""
    import transformers.models.gpt2.modeling_gpt2 as gpt2_module

    original = gpt2_module.eager_attention_forward
    gpt2_module.eager_attention_forward = make_warpforth_eager_attn()

    def restore() -> None:
        gpt2_module.eager_attention_forward = original

    return restore


def random_gpt2(seed: int = 1, device: str | torch.device = "cuda"):
    """GPT-2 small (12 layers, d_model 768, 12 heads, vocab 50257, ctx 1024), N(0, 0.02) init."""
    from transformers import GPT2Config, GPT2LMHeadModel

    cfg = GPT2Config(n_layer=12, n_embd=768, n_head=12, vocab_size=50257, n_positions=1024,
                     initializer_range=0.02)
    cfg._attn_implementation = "eager"
    torch.manual_seed(seed)
    model = GPT2LMHeadModel(cfg).to(device).float().eval()
    return model


def synthetic_prompt(length: int = 32, seed: int = 1) -> torch.Tensor:
    return torch.randint(0, 50257, (1, length), generator=torch.Generator().manual_seed(seed))


@torch.no_grad()
def generate(model, prompt: torch.Tensor, max_new_tokens: int, use_cache: bool = False):
    ids = prompt.to(next(model.parameters()).device)
    return model.generate(ids, attention_mask=torch.ones_like(ids),
                          max_new_tokens=max_new_tokens, min_new_tokens=max_new_tokens,
                          do_sample=False, use_cache=use_cache, pad_token_id=50256)


class _CachedAttention:
    """GPT-2's attention over one ``KVCache`` a layer, for ``generate_drafted``."""

    def __init__(self, model, max_len: int, fmt: str) -> None:
        cfg, device = model.config, next(model.parameters()).device
        self.caches = [KVCache(1, cfg.n_head, max_len, cfg.n_embd // cfg.n_head, fmt=fmt,
                               device=device) for _ in range(cfg.n_layer)]
        self.lens = torch.zeros(1, dtype=torch.int32, device=device)  # rows in the caches
        self.start = torch.zeros_like(self.lens)
        self.length = 0  # the same on the host
        self.words: torch.Tensor | None = None  # of the drafted tree; None in the prompt
        self.workspace = DecodeWorkspace()
        self.modules = set(model.modules())
        self.reached: list[int] = []  # layers whose attention ran here in this forward

    def forward(self, model, ids: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """The model's logits, every layer having attended over its cache."""
        self.reached.clear()
        logits = model(ids, position_ids=positions, use_cache=False).logits
        if self.reached != list(range(len(self.caches))):
            raise RuntimeError(
                "the model's attention does not run over the cache (layers reached: "
                f"{self.reached}): generate_drafted needs eager attention "
                '(model.set_attn_implementation("eager")) without reorder_and_upcast_attn')
        return logits

    def __call__(self, module, query, key, value, attention_mask=None, scaling=None, dropout=0.0,
                 **kwargs):
        self.reached.append(module.layer_idx)
        cache = self.caches[module.layer_idx]
        cache_write(cache, key, value, self.lens)
        if self.words is not None:
            out = tree_decode(query, cache, self.lens, tree=self.words, scale=scaling,
                              workspace=self.workspace)
        else:
            if self.length:  # a later part of the prompt: the rows before it come from the cache
                key, value = cache_read(cache, self.start, self.length + query.shape[2],
                                        dtype=query.dtype)
            out = attention(query, key, value, causal=True, scale=scaling)
        return out.transpose(1, 2), None

    def keep(self, path: list[int]) -> None:
        """The nodes of the path follow the rows that are there; the others are dropped."""
        rows = torch.tensor([path], dtype=torch.int32, device=self.lens.device)
        lens = self.lens
        for cache in self.caches:
            self.lens = cache_keep(cache, lens, rows)
        self.length += len(path)


def draft_tree(tokens: list[int], nodes: int, depth: int = 8) -> tuple[list[int], list[int]]:
    """A tree of at most ``nodes`` drafted tokens: (tokens, parents), the last token as its root.

    Its branches are what followed earlier places of the last three, two or one tokens, the longest
    match and the latest place first; common beginnings share their nodes.
    """
    drafted, parents = [tokens[-1]], [-1]
    children: dict[tuple[int, int], int] = {}
    for n in (3, 2, 1):
        last = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if len(drafted) >= nodes:
                return drafted, parents
            if len(last) < n or tokens[at:at + n] != last:
                continue
            node = 0
            for token in tokens[at + n:at + n + depth]:
                if (node, token) not in children:
                    if len(drafted) >= nodes:
                        break
                    children[node, token] = len(drafted)
                    drafted.append(token)
                    parents.append(node)
                node = children[node, token]
    return drafted, parents


def accepted_path(drafted: list[int], parents: list[int], chosen: list[int]) -> list[int]:
    """The nodes from the root on whose tokens the model chose (``chosen[i]`` after node i)."""
    path = [0]
    while True:
        following = [i for i, parent in enumerate(parents)
                     if parent == path[-1] and drafted[i] == chosen[path[-1]]]
        if not following:
            return path
        path.append(following[0])


# Generations that run now, one a thread: transformers looks its eager attention up in the module
# that all models share, so what stands there sends a layer to the generation of its own thread and
# model, and every other to the function that stood there before.
_generating = threading.local()
_routing = threading.Lock()
_routed = 0


def _route(otherwise: Callable) -> Callable:
    def routed_attention(module, *args, **kwargs):
        state = getattr(_generating, "state", None)
        if state is not None and module in state.modules:
            return state(module, *args, **kwargs)
        return otherwise(module, *args, **kwargs)

    routed_attention.otherwise = otherwise
    return routed_attention


@contextlib.contextmanager
def _attention_of(state: _CachedAttention):
    """This thread's calls of the model's layers go to `state`."""
    global _routed
    import transformers.models.gpt2.modeling_gpt2 as gpt2_module

    with _routing:
        _routed += 1
        if not hasattr(gpt2_module.eager_attention_forward, "otherwise"):
            gpt2_module.eager_attention_forward = _route(gpt2_module.eager_attention_forward)
    before, _generating.state = getattr(_generating, "state", None), state
    try:
        yield
    finally:
        _generating.state = before
        with _routing:
            _routed -= 1
            now = gpt2_module.eager_attention_forward
            if _routed == 0 and hasattr(now, "otherwise"):
                gpt2_module.eager_attention_forward = now.otherwise


# caches that tree_decode takes with a model's queries
_CACHES = {torch.float32: ("f32", "e4m3", "int4"), torch.bfloat16: ("bf16", "e4m3", "int4")}


@torch.no_grad()
def generate_drafted(model, prompt: torch.Tensor, max_new_tokens: int, *, nodes: int = 12,
                     cache: str = "f32", prompt_chunk: int = 512) -> tuple[torch.Tensor, int]:
    """Greedy generation with drafted trees of up to ``nodes`` tokens over a ``cache`` of that format.

    model: a GPT2LMHeadModel in eager mode (RuntimeError where its attention does not run over the
    cache), in f32 (caches "f32", "e4m3", "int4") or bf16 ("bf16", "e4m3", "int4").  prompt: [1, n];
    one longer than ``prompt_chunk`` is read in parts.  Over an f32 cache the tokens are those of
    ``generate`` (but for ties); the other formats round what is attended to.
    Returns the tokens [1, n + max_new_tokens] and how many times the model ran after the prompt.
    """
    if prompt.dim() != 2 or prompt.shape[0] != 1 or prompt.shape[1] < 1:
        raise ValueError(f"prompt must be [1, n], got {tuple(prompt.shape)}")
    if max_new_tokens < 1 or not 1 <= nodes <= 64 or prompt_chunk < 1:
        raise ValueError("max_new_tokens and prompt_chunk must be >= 1, nodes in 1..64")
    weight = next(model.parameters())
    device = weight.device
    takes = _CACHES.get(weight.dtype)
    if takes is None or cache not in takes:
        raise ValueError(f"cache={cache!r} for a model of {weight.dtype}: float32 models take "
                         f"{_CACHES[torch.float32]}, bfloat16 models {_CACHES[torch.bfloat16]}")
    ids = prompt.to(device)
    tokens, end = prompt[0].tolist(), prompt.shape[1] + max_new_tokens
    limit = model.config.n_positions
    if end > limit:
        raise ValueError(f"the model has {limit} positions, {end} are asked for")
    state = _CachedAttention(model, end + nodes, cache)
    runs = 0
    with _attention_of(state):
        for at in range(0, ids.shape[1], prompt_chunk):
            part = ids[:, at:at + prompt_chunk]
            positions = torch.arange(at, at + part.shape[1], device=device)[None]
            logits = state.forward(model, part, positions)
            state.lens = state.lens + part.shape[1]
            state.length += part.shape[1]
        tokens.append(int(logits[0, -1].argmax()))
        while len(tokens) < end:
            drafted, parents = draft_tree(tokens, nodes)
            # a node past the model's last position is not drafted
            depths = [0]
            for parent in parents[1:]:
                depths.append(depths[parent] + 1)
            while state.length + max(depths) >= limit:
                longest = max(depths)
                keep = [i for i, depth in enumerate(depths) if depth < longest]
                drafted, parents, depths = ([x[i] for i in keep] for x in (drafted, parents, depths))
                renamed = {old: new for new, old in enumerate(keep)}
                parents = [renamed.get(parent, -1) for parent in parents]
            state.words = tree_words(parents).to(device)
            positions = torch.tensor([[state.length + depth for depth in depths]], device=device)
            logits = state.forward(model, torch.tensor([drafted], device=device), positions)
            runs += 1
            chosen = logits[0].argmax(-1).tolist()
            path = accepted_path(drafted, parents, chosen)
            state.keep(path)
            tokens += [drafted[i] for i in path[1:]] + [chosen[path[-1]]]
    return torch.tensor([tokens[:end]], device=device), runs


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--max-tokens", type=int, default=128)
    ap.add_argument("--prompt-len", type=int, default=32)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--use-cache", action="store_true")
    ap.add_argument("--draft-nodes", type=int, default=0,
                    help="generate with drafted trees of up to this many tokens (1 to 64)")
    ap.add_argument("--cache", choices=("f32", "e4m3", "int4"), default="f32",
                    help="format of the key/value cache under --draft-nodes")
    args = ap.parse_args()
    model = random_gpt2(args.seed)
    prompt = synthetic_prompt(args.prompt_len, args.seed)
    restore = patch_gpt2()
    try:
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        if args.draft_nodes:
            out, runs = generate_drafted(model, prompt, args.max_tokens, nodes=args.draft_nodes,
                                         cache=args.cache)
        else:
            out = generate(model, prompt, args.max_tokens, use_cache=args.use_cache)
        torch.cuda.synchronize()
        dt = time.perf_counter() - t0
    finally:
        restore()
    print(out[0].tolist())
    print(f"{args.max_tokens / dt:.1f} tokens/s ({out.shape[1]} tokens total)")
    if args.draft_nodes:
        print(f"{runs} runs of the model after the prompt")


if __name__ == "__main__":
    main()
