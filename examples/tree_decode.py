"""A small decoder with drafted token trees on one GPU: the paged-cache operators around the FP8 MoE layer.

    python examples/tree_decode.py [--requests 4] [--steps 16] [--cache fp8]

Each step takes every request's last token and a small tree of guesses for what follows it, runs them all in one pass
(cache_plan, then per layer: products, qk_norm_rope into the cache, tree_attention, the MoE layer; token_logprobs on the logits),
and keeps the guesses that the model itself would have chosen.  The guesses are what the model answered the last time it saw a
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
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, experts=8, top_k=2, inter=256, vocab=2048, device="cuda:0", seed=0):
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
        logits = pkg.mm_bf16(self.norm(self.embedding), self.output)
        return pkg.token_logprobs(logits, torch.arange(self.vocab, device=logits.device), top_k=4).top_ids.tolist()

    @staticmethod
    def norm(x):
        x = x.float()
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)

    def forward(self, tokens, plan, cache):
        """tokens [T] of the plan's rows -> logits [T, vocab] bf16."""
        x = self.embedding[tokens.clamp(min=0)]
        for layer, (k_cache, v_cache) in zip(self.layers, cache.layers):
            qkv = pkg.mm_bf16(self.norm(x), layer["qkv"])
            q = pkg.qk_norm_rope(qkv, plan.positions, self.cos_sin, self.heads, self.kv_heads, layer["q_norm"], layer["k_norm"],
                                 k_cache=k_cache, v_cache=v_cache, slots=plan.slots)
            o = pkg.tree_attention(q, k_cache, v_cache, cache.tables, plan.kv_lens, plan.cu_tokens, plan.masks)
            x = x + pkg.mm_bf16(o.flatten(1), layer["o"])
            x = x + layer["moe"](self.norm(x))
        return pkg.mm_bf16(self.norm(x), self.output)


class Cache:
    """Pages of all layers, one table for all of them, and the stack of free pages."""

    def __init__(self, model, requests, pages_each=8, page=16, dtype=torch.bfloat16):
        device = model.embedding.device
        blocks = requests * pages_each
        shape = (blocks, page, model.kv_heads, model.head_dim)
        self.page, self.layers = page, [(torch.zeros(shape, device=device).to(dtype), torch.zeros(shape, device=device).to(dtype)) for _ in model.layers]
        self.tables = torch.zeros(requests, pages_each, dtype=torch.int32, device=device)
        self.free = torch.arange(blocks, dtype=torch.int32, device=device)
        self.n_free = torch.full((1,), blocks, dtype=torch.int32, device=device)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)

    def plan(self, counts, max_tokens, parents=None):
        p = pkg.cache_plan(self.tables, self.lens, counts, self.free, self.n_free, self.page, max_tokens, parents)
        if bool(((counts > 0) & (p.kv_lens == 0)).any()):
            raise RuntimeError("no room in the cache")
        self.n_free = p.n_free
        return p

    def keep(self, plan, kept):
        """kept[b]: the rows of the step that stay, in text order.  Their keys and values move up behind the cached text (their angles
        are already those of their depth), and pages that nothing needs any more go back on the stack."""
        rows = [(b, self.lens[b].item() + i, row) for b, some in enumerate(kept) for i, row in enumerate(some)]
        if rows:
            b, place, row = (torch.tensor(x, device=self.lens.device) for x in zip(*rows))
            to = self.tables[b, place // self.page].long() * self.page + place % self.page
            for pair in self.layers:
                for cache in pair:
                    flat = cache.view(torch.uint8).flatten(0, 1)
                    flat[to] = flat[plan.slots[row]]
        had = (plan.kv_lens + self.page - 1) // self.page
        self.lens = self.lens + torch.tensor([len(k) for k in kept], dtype=torch.int32, device=self.lens.device)
        column = torch.arange(self.tables.shape[1], device=self.lens.device)
        back = self.tables[(column >= ((self.lens + self.page - 1) // self.page)[:, None]) & (column < had[:, None])]
        n = self.n_free.item()
        self.free[n:n + back.numel()] = back
        self.n_free = self.n_free + back.numel()


def prefill(model, cache, prompts):
    """prompts: a list of token lists -> each request's most likely next token."""
    device = model.embedding.device
    counts = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=device)
    tokens = torch.tensor([t for p in prompts for t in p], device=device)
    plan = cache.plan(counts, tokens.numel())
    logits = model.forward(tokens, plan, cache)
    cache.lens = plan.kv_lens
    last = (plan.cu_tokens[1:] - 1).long()
    return pkg.token_logprobs(logits[last], tokens[last], top_k=1).top_ids[:, 0].tolist()


def step(model, cache, trees):
    """trees[b]: (tokens, parents) of request b, the first token the last one chosen, the others guesses.  -> per request the
    tokens chosen after it and their log probabilities; the best continuations of every token that was run."""
    device = model.embedding.device
    counts = torch.tensor([len(t) for t, _ in trees], dtype=torch.int32, device=device)
    flat = [t for tree, _ in trees for t in tree]
    tokens = torch.tensor(flat, device=device)
    parents = torch.tensor([p for _, above in trees for p in above], dtype=torch.int32, device=device)
    plan = cache.plan(counts, tokens.numel(), parents)
    logits = model.forward(tokens, plan, cache)
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
    cache.keep(plan, kept)
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


def generate(model, cache, prompts, steps):
    """-> per request the first token (prefill's), and the (token, log probability) list of what followed it in `steps` steps."""
    first = last = prefill(model, cache, prompts)
    last, text, answers = list(last), [[] for _ in prompts], model.guesses()
    for _ in range(steps):
        trees = [draft(t, answers) for t in last]
        chosen, seen = step(model, cache, trees)
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
    ap.add_argument("--cache", choices=["bf16", "fp8"], default="bf16")
    args = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    dtype = torch.bfloat16 if args.cache == "bf16" else torch.float8_e4m3fn
    model = Decoder()
    prompts = [torch.randint(model.vocab, (5 + 3 * b,), generator=g).tolist() for b in range(args.requests)]
    _, text = generate(model, Cache(model, args.requests, dtype=dtype), prompts, args.steps)
    for b, said in enumerate(text):
        print(f"request {b}: {len(said)} tokens in {args.steps} steps, mean log probability {sum(lp for _, lp in said) / len(said):.3f}")


if __name__ == "__main__":
    main()
