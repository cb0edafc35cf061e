"""A small decoder with drafted token trees on one GPU: the paged-cache operators around the FP8 MoE layer.

    python examples/tree_decode.py [--requests 4] [--steps 16] [--cache fp8 | fp4] [--window 64 --sinks 4] [--repetition 1.2]

Each step takes every request's last token and a small tree of guesses for what follows it, runs them all in one pass
(cache_plan, then per layer: products, qk_norm_rope into the cache, tree_attention, residual_norm, the MoE layer; adjust_logits where there is a
penalty, token_logprobs on the logits), and keeps the guesses that the model itself would have chosen.  The guesses are what the model answered the last time it saw a
token, at first what its output layer makes of the token's embedding alone.  Weights are random, so the text means nothing; what is shown is how many tokens come out of a step.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from __graft_entry__ import load_package  # noqa: E402

pkg = load_package()


class Decoder:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=256, vocab=2048, device="cuda:0", seed=0,
                 window=None, sinks=0):
        """window: every other layer, from the first on, sees the last `window` tokens and the first `sinks`."""
        self.views = [dict(window=window, sinks=sinks) if window and i % 2 == 0 else {} for i in range(layers)]
        self.heads, self.kv_heads, self.head_dim, self.hidden, self.vocab = heads, kv_heads, head_dim, hidden, vocab
        g = torch.Generator().manual_seed(seed)

        def rand(*shape, std):
            return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16).to(device)

        def dense(n, k):
            return pkg.pack_weights(rand(n, k, std=k ** -0.5))

        self.embedding = rand(vocab, hidden, std=1.0)
        self.output = dense(vocab, hidden)
        self.layers = []
        for i in range(layers):
            w13, s13 = pkg.synthetic_weights(experts, 2 * inter, hidden, device, seed * 100 + 2 * i, std=hidden ** -0.5)
            w2, s2 = pkg.synthetic_weights(experts, hidden, inter, device, seed * 100 + 2 * i + 1, std=inter ** -0.5)
            self.layers.append(dict(
                qkv=dense((heads + 2 * kv_heads) * head_dim, hidden), o=dense(hidden, heads * head_dim),
                q_norm=1 + rand(head_dim, std=0.1), k_norm=1 + rand(head_dim, std=0.1),
                moe=pkg.FusedMoE(rand(experts, hidden, std=hidden ** -0.5), w13, s13, w2, s2, top_k)))
        angles = torch.arange(4096)[:, None] / 10000 ** (torch.arange(head_dim // 2) / (head_dim // 2))
        self.cos_sin = torch.cat([angles.cos(), angles.sin()], 1).to(device)

    def guesses(self):
        """-> the four likeliest tokens after each token of the vocabulary, as far as its embedding says."""
        logits = pkg.mm_bf16(pkg.residual_norm(self.embedding)[0], self.output)
        return pkg.token_logprobs(logits, torch.arange(self.vocab, device=logits.device), top_k=4).top_ids.tolist()

    def forward(self, tokens, plan, cache):
        """tokens [T] of the plan's rows -> logits [T, vocab] bf16."""
        y, x = pkg.residual_norm(self.embedding[tokens.clamp(min=0)])
        for layer, view, (k_cache, v_cache), (k_scale, v_scale) in zip(self.layers, self.views, cache.layers, cache.scales):
            qkv = pkg.mm_bf16(y, layer["qkv"])
            q = pkg.qk_norm_rope(qkv, plan.positions, self.cos_sin, self.heads, self.kv_heads, layer["q_norm"], layer["k_norm"],
                                 k_cache=k_cache, v_cache=v_cache, slots=plan.slots, k_scale=k_scale, v_scale=v_scale)
            o = pkg.tree_attention(q, k_cache, v_cache, cache.tables, plan.kv_lens, plan.cu_tokens, plan.masks, k_scale=k_scale, v_scale=v_scale, **view)
            y, x = pkg.residual_norm(pkg.mm_bf16(o.flatten(1), layer["o"]), x)
            y, x = pkg.residual_norm(layer["moe"](y), x)
        return pkg.mm_bf16(y, self.output)


class Cache:
    """Pages of all layers, one table for all of them, and the stack of free pages."""

    def __init__(self, model, requests, pages_each=8, page=16, dtype=torch.bfloat16):
        device = model.embedding.device
        blocks = requests * pages_each
        shape = (blocks, page, model.kv_heads, model.head_dim)
        def zeros(dtype, per):                           # `per` elements to one of dtype
            if dtype not in (torch.float4_e2m1fn_x2, torch.float8_e8m0fnu):
                return torch.zeros(shape, device=device).to(dtype)
            return torch.zeros(*shape[:3], shape[3] // per, dtype=torch.uint8, device=device).view(dtype)

        four = dtype == torch.float4_e2m1fn_x2             # a cache in 4 bits has powers of two beside it
        self.page, self.layers = page, [(zeros(dtype, 2), zeros(dtype, 2)) for _ in model.layers]
        self.scales = [(zeros(torch.float8_e8m0fnu, 32), zeros(torch.float8_e8m0fnu, 32)) if four else (None, None) for _ in model.layers]
        self.tables = torch.zeros(requests, pages_each, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks, dtype=torch.int32, device=device)
        self.n_free = torch.full((1,), blocks, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.text = torch.zeros(requests, pages_each * page, dtype=torch.int32, device=device)        # the tokens whose keys are cached

    def plan(self, counts, max_tokens, parents=None):
        p = pkg.cache_plan(self.tables, self.lens, counts, self.free, self.n_free, self.page, max_tokens, parents)
        if bool(((counts > 0) & (p.kv_lens == 0)).any()):
            raise RuntimeError("no room in the cache")
        self.n_free = p.n_free
        return p

    def keep(self, plan, kept, tokens=None):
        """kept[b]: the rows of the step that stay, in text order.  Their keys and values move up behind the cached text (their angles
        are already those of their depth), and pages that nothing needs any more go back on the stack."""
        rows = [(b, self.lens[b].item() + i, row) for b, some in enumerate(kept) for i, row in enumerate(some)]
        if rows:
            b, place, row = (torch.tensor(x, device=self.lens.device) for x in zip(*rows))
            to = self.tables[b, place // self.page].long() * self.page + place % self.page
            for cache in [c for pair in self.layers + self.scales for c in pair if c is not None]:
                flat = cache.view(torch.uint8).flatten(0, 1)
                flat[to] = flat[plan.slots[row]]
            if tokens is not None:
                self.text[b, place] = tokens[row].int()
        had = (plan.kv_lens + self.page - 1) // self.page
        self.lens = self.lens + torch.tensor([len(k) for k in kept], dtype=torch.int32, device=self.lens.device)
        column = torch.arange(self.tables.shape[1], device=self.lens.device)
        back = self.tables[(column >= ((self.lens + self.page - 1) // self.page)[:, None]) & (column < had[:, None])]
        n = self.n_free.item()
        self.free[n:n + back.numel()] = back
        self.n_free = self.n_free + back.numel()


def prefill(model, cache, prompts, repetition=None):
    """prompts: a list of token lists -> each request's most likely next token."""
    device = model.embedding.device
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    plan = cache.plan(counts, tokens.numel())
    logits = model.forward(tokens, plan, cache)
    cache.lens = plan.kv_lens
    for b, p in enumerate(prompts):
        cache.text[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    last = (plan.cu_tokens[1:] - 1).long()
    logits = logits[last]
    if repetition is not None:
        logits = pkg.adjust_logits(logits, history=cache.text, history_lens=cache.lens, repetition=repetition)
    return pkg.token_logprobs(logits, tokens[last], top_k=1).top_ids[:, 0].tolist()


def step(model, cache, trees, repetition=None):
    """trees[b]: (tokens, parents) of request b, the first token the last one chosen, the others guesses.  -> per request the
    tokens chosen after it and their log probabilities; the best continuations of every token that was run."""
    device = model.embedding.device
    counts = torch.tensor([len(t) for t, _ in trees], dtype=torch.int32, device=device)
    flat = [t for tree, _ in trees for t in tree]
    tokens = torch.tensor(flat, device=device)
    parents = torch.tensor([p for _, above in trees for p in above], dtype=torch.int32, device=device)
    plan = cache.plan(counts, tokens.numel(), parents)
    logits = model.forward(tokens, plan, cache)
    if repetition is not None:                             # each token under what its request has said and its own path through the tree
        logits = pkg.adjust_logits(logits, plan.cu_tokens, history=cache.text, history_lens=cache.lens, tokens=tokens, masks=plan.masks,
                                   repetition=repetition)
    # each guess under the logits of the token before it, and the best continuations of every token
    best = pkg.token_logprobs(logits, tokens, top_k=4)
    start = plan.cu_tokens[:-1].repeat_interleave(counts)
    guessed = pkg.token_logprobs(logits[(start + parents.clamp(min=0)).long()], tokens)
    top, top_lp, lp = best.top_ids.tolist(), best.top_logprobs.tolist(), guessed.logprobs.tolist()
    chosen, kept, first = [], [], 0
    for tree, above in trees:
        at, path, said = 0, [first], []
        while True:
            nxt = next((i for i in range(at + 1, len(tree)) if above[i] == at and tree[i] == top[first + at][0]), None)
            if nxt is None:
                said.append((top[first + at][0], top_lp[first + at][0]))
                break
            said.append((tree[nxt], lp[first + nxt]))
            at = nxt
            path.append(first + at)
        chosen.append(said)
        kept.append(path)
        first += len(tree)
    cache.keep(plan, kept, tokens)
    return chosen, dict(zip(flat, top))


def draft(token, answers, width=2, depth=3):
    """A tree of what followed these tokens before: the likeliest `width` of each, `depth` deep."""
    tokens, parents, level = [token], [-1], [0]
    for _ in range(depth):
        nxt = []
        for at in level:
            for guess in answers[tokens[at]][:width]:
                nxt.append(len(tokens))
                tokens.append(guess)
                parents.append(at)
        level = nxt
    return tokens, parents


def generate(model, cache, prompts, steps, repetition=None):
    """-> per request the first token (prefill's), and the (token, log probability) list of what followed it in `steps` steps.
    repetition: a penalty for tokens that a request has had before, of all requests alike."""
    if repetition is not None:
        repetition = torch.full((len(prompts),), float(repetition), device=cache.lens.device)
    first = last = prefill(model, cache, prompts, repetition)
    last, text, answers = list(last), [[] for _ in prompts], model.guesses()
    for _ in range(steps):
        trees = [draft(t, answers) for t in last]
        chosen, seen = step(model, cache, trees, repetition)
        for token, top in seen.items():
            answers[token] = top
        for b, said in enumerate(chosen):
            text[b] += said
            last[b] = said[-1][0]
    return first, text


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--cache", choices=["bf16", "fp8", "fp4"], default="bf16")
    ap.add_argument("--window", type=int, help="every other layer sees the last so many tokens")
    ap.add_argument("--sinks", type=int, default=0, help="and the first so many")
    ap.add_argument("--repetition", type=float, help="a penalty above 1 for tokens that a request has had")
    args = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    dtype = dict(bf16=torch.bfloat16, fp8=torch.float8_e4m3fn, fp4=torch.float4_e2m1fn_x2)[args.cache]
    model = Decoder(window=args.window, sinks=args.sinks)
    prompts = [torch.randint(model.vocab, (5 + 3 * b,), generator=g).tolist() for b in range(args.requests)]
    _, text = generate(model, Cache(model, args.requests, dtype=dtype), prompts, args.steps, args.repetition)
    for b, said in enumerate(text):
        print(f"request {b}: {len(said)} tokens in {args.steps} steps, mean log probability {sum(lp for _, lp in said) / len(said):.3f}")


if __name__ == "__main__":
    main()
