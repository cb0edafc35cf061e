"""The operators of a serving step with drafted tokens around the MoE layer, their cases, inputs and plain forms.

A step of a server that lets a small model draft a tree of tokens for every request and has the large one look at all of them
at once: the cache's bookkeeping, the norms and rotation of queries and keys on their way into the cache, attention over the
paged cache, and what the logits say about the drafted tokens.  "kind" names the operator of a case:

  plan      `cache_plan`: block tables, slots, positions and tree masks from the requests' lengths
  rope      `qk_norm_rope`: norms per head, rotation, keys and values into the cache
  attention `tree_attention`: one token, a tree of drafted tokens or a causal chunk of each request over the paged cache
  logprobs  `token_logprobs`: log probability of given tokens, entropy, top alternatives
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"


def _package():
    """The package directory `torch-tpu_amd/` of the working folder, under its importable name."""
    name = "torch_tpu_amd"
    if name not in sys.modules:
        folder = os.path.join(os.getcwd(), "torch-tpu_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules[name] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules[name])
    return sys.modules[name]


# ---------------------------------------------------------------------------------------------- cases
def _plan(B, most, L, page, tree):
    return dict(kind="plan", B=B, most=most, L=L, page=page, tree=tree)


def _rope(T, Hq, Hkv, D, R, pairs, fp8, page=64):
    return dict(kind="rope", T=T, Hq=Hq, Hkv=Hkv, D=D, R=R, pairs=pairs, fp8=fp8, page=page)


def _attention(B, L, most, tree, Hq, Hkv, D, page, fp8, even=False):
    """most: new tokens of the request that has most; even: all requests alike, else from a fifth of L (most) up to it."""
    return dict(kind="attention", B=B, L=L, most=most, tree=tree, Hq=Hq, Hkv=Hkv, D=D, page=page, fp8=fp8, even=even)


def _logprobs(T, V, k, bf16, masked, temp):
    return dict(kind="logprobs", T=T, V=V, k=k, bf16=bf16, masked=masked, temp=temp)


def listed():
    return [
        # one conversation's tree of drafted tokens: launch latency is all there is
        dict(name="plan_b1_tree", **_plan(1, 8, 1000, 64, True)),
        # a thousand requests with the largest trees, small pages: tables and slots of tens of thousands of tokens
        dict(name="plan_b1024_tree64", **_plan(1024, 64, 4000, 16, True)),
        # one user's next token: a latency between two products
        dict(name="rope_t1", **_rope(1, 32, 4, 128, 128, False, False)),
        # a decode batch of trees, narrow heads, half of each rotated in neighbouring pairs, ragged
        dict(name="rope_t613_d64", **_rope(613, 24, 8, 64, 32, True, False, 16)),
        # a long prompt into an 8-bit cache: bytes count
        dict(name="rope_t16384_fp8", **_rope(16384, 32, 4, 128, 128, False, True)),
        # one user's next token over a long document: the cache's one pass has to be cut over the whole chip
        dict(name="attention_b1_l32767", **_attention(1, 32767, 1, False, 32, 4, 128, 64, False, True)),
        # a decode batch of ragged lengths: the cache streams at full rate or it does not
        dict(name="attention_b64_decode", **_attention(64, 8192, 1, False, 32, 4, 128, 16, False)),
        # trees of up to 16 drafted tokens over an 8-bit cache, ragged in both
        dict(name="attention_b32_tree16_fp8", **_attention(32, 8001, 16, True, 32, 4, 128, 64, True)),
        # the largest trees, many rows to each cached key: the matrix cores count
        dict(name="attention_b16_tree64", **_attention(16, 12288, 64, True, 32, 4, 128, 64, False)),
        # two prompts' next chunks beside their cached beginnings, causal
        dict(name="attention_b2_chunk1021", **_attention(2, 8190, 1021, False, 32, 8, 128, 64, False)),
        # one row of logits at decode: the row has to be cut over the chip, then joined
        dict(name="logprobs_t1", **_logprobs(1, 131072, 20, True, False, 1.0)),
        # all drafted tokens of a large batch under a grammar's mask, an odd vocabulary
        dict(name="logprobs_t2048_masked", **_logprobs(2048, 100003, 8, True, True, 0.7)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "attention", "attention", "attention", "attention", "logprobs", "logprobs"])
    if kind == "plan":
        return _plan(_log_int(rng, 1, 1024), _log_int(rng, 1, 64), _log_int(rng, 1, 8000), rng.choice([16, 32, 64, 128]), rng.random() < 0.7)
    if kind == "rope":
        D = rng.choice([64, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8])
        return _rope(_log_int(rng, 1, 16384), Hkv * rng.choice([1, 2, 3, 4, 5, 8]), Hkv, D, rng.choice([D, D, D // 2]),
                     rng.random() < 0.4, rng.random() < 0.4, rng.choice([16, 64]))
    if kind == "attention":
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = min(64, Hkv * rng.choice([1, 2, 3, 4, 5, 8, 8, 16]))
        tree = rng.random() < 0.5
        most = _log_int(rng, 1, 64) if tree else rng.choice([1, 1, 1, _log_int(rng, 2, 600)])
        B, L = _log_int(rng, 1, 64), _log_int(rng, 16, 32768)
        # no more cached keys, and no more products, than the largest listed cases have; a plain form's scores fit too
        while B > 1 and (B * L * Hkv > 16 * 12288 * 4 or B * L * Hq * most > 16 * 12288 * 32 * 64):
            B = B // 2
        while L * Hq * most > 2 * 8190 * 32 * 1021:
            L = L // 2
        return _attention(B, max(L, most), most, tree, Hq, Hkv, rng.choice([64, 128, 128, 128]), rng.choice([16, 32, 64, 128]),
                          rng.random() < 0.4, rng.random() < 0.3)
    V = _log_int(rng, 1000, 131072)
    return _logprobs(min(_log_int(rng, 1, 2048), 2048 * 100003 // V), V, rng.choice([0, 1, 5, 8, 20, 32]), rng.random() < 0.7,
                     rng.random() < 0.3, rng.choice([1.0, 1.0, 0.6, 1.3]))


def _spread(case):
    """(cached length, new tokens) of each request: the same for every seed, ragged by the golden section."""
    B, L, most = case["B"], case["L"], case["most"]
    got = []
    for b in range(B):
        f = 1.0 if case.get("even") or b == 0 else (b * 0.6180339887) % 1.0
        n = max(1, round(most * (1.0 if f == 1.0 else 0.25 + 0.75 * ((b * 0.7548776662) % 1.0))))
        got.append((max(0, round(L * (0.2 + 0.8 * f)) - n), n))
    return got


def work(case):
    c = dict(case)
    if c["kind"] == "plan":
        n = sum(x for _, x in _spread(c))
        new = sum(-(-(l + x) // c["page"]) - -(-l // c["page"]) for l, x in _spread(c))
        used = sum(-(-(l + x) // c["page"]) - l // c["page"] for l, x in _spread(c))
        # lens, counts, cu, kv_lens; parents, positions, slots, masks; free blocks and table entries
        return {"bytes": 16 * c["B"] + n * (4 + 8 + (12 if c["tree"] else 0)) + 8 * new + 4 * used, "flops": 0}
    if c["kind"] == "rope":
        rows = c["T"] * c["D"]
        out = 1 if c["fp8"] else 2
        return {"bytes": rows * (2 * (2 * c["Hq"] + 2 * c["Hkv"]) + 2 * out * c["Hkv"]) + c["T"] * (4 * c["R"] + 12),
                "flops": rows * (8 * c["Hq"] + 8 * c["Hkv"])}
    if c["kind"] == "attention":
        reqs = _spread(c)
        keys, new = sum(l + n for l, n in reqs), sum(n for _, n in reqs)
        seen = sum(n * l + (n if c["tree"] else n * (n + 1) // 2) for l, n in reqs)
        return {"bytes": 2 * keys * c["Hkv"] * c["D"] * (1 if c["fp8"] else 2) + 2 * 2 * new * c["Hq"] * c["D"],
                "flops": 4 * seen * c["Hq"] * c["D"]}
    e = 2 if c["bf16"] else 4
    return {"bytes": c["T"] * (c["V"] * e + 4 + 8 + 8 * c["k"]), "flops": 6 * c["T"] * c["V"]}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(1000003 * (int(seed) % (1 << 40)) + part)


def _randn(seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device=DEV)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _trees(rng, counts):
    """Parents of every request's drafted tokens: -1 at the root's level, mostly one of the last few tokens."""
    return [-1 if j == 0 or rng.random() < 0.08 else max(0, j - 1 - int(rng.expovariate(0.5))) for n in counts for j in range(n)]


def _masks(parents, counts):
    out, at = [], 0
    for n in counts:
        own_masks = []
        for j in range(n):
            p = parents[at + j]
            own_masks.append((1 << j) | (own_masks[p] if p >= 0 else 0))
        out += own_masks
        at += n
    return [m - (1 << 64) if m >= 1 << 63 else m for m in out]


def prepare(case, seed):
    c, seed = dict(case), int(seed)
    rng = random.Random(seed * 7919 + 17)
    if c["kind"] == "plan":
        reqs = _spread(c)
        rng.shuffle(reqs)
        W = -(-(c["L"] + c["most"]) // c["page"]) + 1
        blocks = torch.randperm(c["B"] * W, generator=_gen(seed, 1), device=DEV).to(torch.int32)
        have = _ints([-(-l // c["page"]) for l, _ in reqs])
        tables = blocks.view(c["B"], W)
        held = torch.arange(W, device=DEV)[None, :] < have[:, None]
        free = torch.zeros_like(blocks)                    # a stack with room for every block
        free[:int((~held).sum())] = tables[~held]
        return dict(c, tables=torch.where(held, tables, torch.full_like(tables, -1)), lens=_ints([l for l, _ in reqs]),
                    counts=_ints([n for _, n in reqs]), free=free, n_free=_ints([int((~held).sum())]),
                    tokens=sum(n for _, n in reqs), parents=_ints(_trees(rng, [n for _, n in reqs])) if c["tree"] else None)
    if c["kind"] == "rope":
        T, Hq, Hkv, D, R = c["T"], c["Hq"], c["Hkv"], c["D"], c["R"]
        heads = Hq + 2 * Hkv
        qkv = (_randn(seed, 1, T, heads * D) * (0.5 + _randn(seed, 2, 1, heads, 1).abs()).expand(1, heads, D).reshape(1, -1)).to(torch.bfloat16)
        angle = torch.arange(32768, device=DEV, dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R))[None, :]
        n_blocks = -(-T // c["page"]) + 3
        slots = torch.randperm(n_blocks * c["page"], generator=_gen(seed, 3), device=DEV)[:T]
        kind = torch.float8_e4m3fn if c["fp8"] else torch.bfloat16
        scale = (lambda part: 0.03 * (0.5 + torch.rand(Hkv, generator=_gen(seed, part), device=DEV))) if c["fp8"] else (lambda part: None)
        start = int(torch.randint(0, 32768 - T, (1,), generator=_gen(seed, 4), device=DEV)) if T < 32768 else 0
        return dict(c, qkv=qkv, positions=torch.arange(start, start + T, device=DEV, dtype=torch.int32),
                    cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float(),
                    q_weight=(1 + 0.2 * _randn(seed, 5, D)).to(torch.bfloat16), k_weight=(1 + 0.2 * _randn(seed, 6, D)).to(torch.bfloat16),
                    k_cache=_randn(seed, 7, n_blocks, c["page"], Hkv, D).to(kind), v_cache=_randn(seed, 8, n_blocks, c["page"], Hkv, D).to(kind),
                    slots=slots, k_scale=scale(9), v_scale=scale(10))
    if c["kind"] == "attention":
        reqs = _spread(c)
        rng.shuffle(reqs)
        counts, lens = [n for _, n in reqs], [l + n for l, n in reqs]
        page, Hkv, D = c["page"], c["Hkv"], c["D"]
        pages = [-(-l // page) for l in lens]
        n_blocks = sum(pages) + 2
        ids = torch.randperm(n_blocks, generator=_gen(seed, 1), device=DEV).to(torch.int32)
        tables = torch.full((c["B"], max(pages) + 1), -1, dtype=torch.int32, device=DEV)
        row = torch.repeat_interleave(torch.arange(c["B"], device=DEV), _ints(pages, torch.int64))
        first = _ints([sum(pages[:b]) for b in range(c["B"])], torch.int64)
        col = torch.arange(sum(pages), device=DEV) - first[row]
        tables[row, col] = ids[:sum(pages)]
        kind = torch.float8_e4m3fn if c["fp8"] else torch.bfloat16
        up = 40.0 if c["fp8"] else 1.0                     # codes use the type's range, the scales bring them back
        T = sum(counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        k = (_randn(seed, 2, n_blocks, page, Hkv, D) * up).to(kind)
        v = ((_randn(seed, 3, n_blocks, page, Hkv, D) + _randn(seed, 4, 1, 1, Hkv, D)) * up).to(kind)
        scale = (lambda part: (0.9 + 0.2 * torch.rand(Hkv, generator=_gen(seed, part), device=DEV)) / up) if c["fp8"] else (lambda part: None)
        return dict(c, q=(_randn(seed, 5, T, c["Hq"], D) * 1.5).to(torch.bfloat16), k_cache=k, v_cache=v, tables=tables,
                    kv_lens=_ints(lens), cu=_ints(cu), longest=max(lens), widest=max(counts),
                    masks=_ints(_masks(_trees(rng, counts), counts), torch.int64) if c["tree"] else None,
                    k_scale=scale(6), v_scale=scale(7))
    T, V = c["T"], c["V"]
    logits = _randn(seed, 1, T, V) * 2.0
    if c["masked"]:                                        # a grammar lets a tenth of the vocabulary through
        logits.masked_fill_(torch.rand(T, V, generator=_gen(seed, 2), device=DEV) < 0.9, float("-inf"))
    tokens = torch.randint(0, V, (T,), generator=_gen(seed, 3), device=DEV)
    logits.scatter_add_(1, tokens[:, None], torch.full((T, 1), 6.0, device=DEV))
    return dict(c, logits=logits.to(torch.bfloat16 if c["bf16"] else torch.float32), tokens=tokens)


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["kind"] == "plan":
        return _run_plan(s) if own else _plain_plan(s)
    if s["kind"] == "rope":
        return _run_rope(s) if own else _plain_rope(s)
    if s["kind"] == "attention":
        return _run_attention(s) if own else _plain_attention(s)
    return _run_logprobs(s) if own else _plain_logprobs(s)


def _run_plan(s):
    p = _package().cache_plan(s["tables"], s["lens"], s["counts"], s["free"], s["n_free"], s["page"], s["tokens"], parents=s["parents"])
    return dict(tables=s["tables"], cu=p.cu_tokens, positions=p.positions, slots=p.slots, masks=p.masks, kv_lens=p.kv_lens, n_free=p.n_free)


def _run_rope(s):
    q = _package().qk_norm_rope(s["qkv"], s["positions"], s["cos_sin"], s["Hq"], s["Hkv"], s["q_weight"], s["k_weight"], eps=1e-6,
                                interleaved=s["pairs"], k_cache=s["k_cache"], v_cache=s["v_cache"], slots=s["slots"],
                                k_scale=s["k_scale"], v_scale=s["v_scale"])
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])


def _run_attention(s):
    return dict(out=_package().tree_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu"], masks=s["masks"],
                                              k_scale=s["k_scale"], v_scale=s["v_scale"]))


def _run_logprobs(s):
    r = _package().token_logprobs(s["logits"], s["tokens"], top_k=s["k"], temperature=s["temp"])
    return dict(logprobs=r.logprobs, entropy=r.entropy, top_logprobs=r.top_logprobs, top_ids=r.top_ids)


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_plan(s):
    tables, page, T = s["tables"], s["page"], s["tokens"]
    B, W = tables.shape
    lens, n = s["lens"].long(), s["counts"].long().clamp_min(0)
    have, want = (lens + page - 1) // page, (lens + n + page - 1) // page
    fits = (lens >= 0) & (lens + n <= W * page)
    if s["parents"] is not None:
        fits &= n <= 64
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= s["n_free"]))
    taken = torch.where(granted & (need > 0), upto, 0).amax()
    col = torch.arange(W, device=tables.device)
    new = granted[:, None] & (col >= have[:, None]) & (col < want[:, None])
    pick = s["n_free"].long() - 1 - ((upto - need)[:, None] + col - have[:, None])
    tables.copy_(torch.where(new, s["free"][pick.clamp(0, s["free"].numel() - 1)], tables))
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=tables.device), n.cumsum(0)])
    t = torch.arange(T, device=tables.device)
    b = torch.searchsorted(cu[1:], t, right=True).clamp_max(B - 1)
    j = t - cu[b]
    live = (t < cu[B]) & granted[b]
    depth, masks = j, None
    if s["parents"] is not None:
        up = s["parents"].long()
        root = (up < 0) | (up >= j)
        up = torch.where(root, T, cu[b] + up)              # row T: the end of every path
        up = torch.cat([up, up.new_full((1,), T)])
        masks = torch.cat([torch.bitwise_left_shift(torch.ones_like(j), j.clamp(0, 63)), j.new_zeros(1)])
        depth = torch.cat([torch.ones_like(j), j.new_zeros(1)])
        for _ in range(6):                                 # paths of up to 64 by doubling
            masks, depth, up = masks | masks[up], depth + depth[up], up[up]
        masks = torch.where(live, masks[:T], 0)
        depth = depth[:T] - 1
    at = lens[b] + j
    slot = tables[b, (at // page).clamp(0, W - 1)].long() * page + at % page
    return dict(tables=tables, cu=cu.int(), positions=torch.where(live, lens[b] + depth, -1).int(), slots=torch.where(live, slot, -1),
                masks=masks, kv_lens=torch.where(granted, lens + n, 0).int(), n_free=(s["n_free"] - taken).int())


def _turn(x, cos, sin, R, pairs):
    """Rotates the first R of the last dimension; cos, sin [T, 1, R/2]."""
    turned = x[..., :R]
    a, b = (turned[..., 0::2], turned[..., 1::2]) if pairs else (turned[..., :R // 2], turned[..., R // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _store(cache, rows, slots, scale):
    """Rows [T, Hkv, D] into the cache's slots, in its type."""
    if scale is not None:
        rows = (rows / scale[None, :, None]).clamp(-448.0, 448.0)
    rows = rows.to(cache.dtype)
    flat = cache.view(-1, *cache.shape[2:])
    if scale is not None:
        flat, rows = flat.view(torch.uint8), rows.view(torch.uint8)
    flat[slots] = rows


def _plain_rope(s):
    T, Hq, Hkv, D, R = s["T"], s["Hq"], s["Hkv"], s["D"], s["R"]
    x = s["qkv"].view(T, Hq + 2 * Hkv, D).float()
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    angle = s["cos_sin"][s["positions"].long()][:, None, :]
    cos, sin = angle[..., :R // 2], angle[..., R // 2:]
    q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_weight"].float()
    k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_weight"].float()
    _store(s["k_cache"], _turn(k, cos, sin, R, s["pairs"]), s["slots"], s["k_scale"])
    _store(s["v_cache"], v, s["slots"], s["v_scale"])
    return dict(q=_turn(q, cos, sin, R, s["pairs"]).to(torch.bfloat16), k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attention(s):
    B, Hq, Hkv, D, page = s["B"], s["Hq"], s["Hkv"], s["D"], s["page"]
    G, n, S = Hq // Hkv, s["widest"], s["longest"]
    cu, lens = s["cu"].long(), s["kv_lens"].long()
    counts = cu[1:] - cu[:-1]
    j = torch.arange(n, device=DEV)
    there = j < counts[:, None]                                            # [B, n]
    row = (cu[:-1, None] + j).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(B, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D)
    key = torch.arange(S, device=DEV)
    at = (s["tables"].long()[:, key // page].clamp_min(0) * page + key % page)  # [B, S]
    k = s["k_cache"].view(-1, Hkv, D)[at].float().transpose(1, 2)          # [B, Hkv, S, D]
    v = s["v_cache"].view(-1, Hkv, D)[at].float().transpose(1, 2)
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    new = key[None, :] - (lens - counts)[:, None]                          # [B, S]: which of the new tokens a key is
    if s["masks"] is not None:
        sees = torch.bitwise_right_shift(s["masks"][row][:, :, None], new.clamp(0, 63)[:, None, :]).bitwise_and(1).bool()
    else:
        sees = new[:, None, :] <= j[None, :, None]
    sees = ((new < 0)[:, None, :] | sees) & (key < lens[:, None])[:, None, :] & there[:, :, None]
    hide = torch.zeros(sees.shape, device=DEV).masked_fill_(~sees, float("-inf"))  # [B, n, S]
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, Hkv, n, G, S).add_(hide[:, None, :, None, :])
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-3.0e38)).exp_()
    out = torch.matmul(x.view(B, Hkv, n * G, S), v) / x.sum(-1).view(B, Hkv, n * G, 1).clamp_min(1e-38)
    out = out.view(B, Hkv, n, G, D).transpose(1, 2).reshape(B, n, Hq, D).to(torch.bfloat16)
    return dict(out=out.view(B * n, Hq, D)[(torch.arange(B, device=DEV) * n).repeat_interleave(counts, output_size=s["q"].shape[0])
                                           + torch.arange(s["q"].shape[0], device=DEV) - cu[:-1].repeat_interleave(counts, output_size=s["q"].shape[0])])


def _plain_logprobs(s):
    x = s["logits"].float()
    T, V, k = s["T"], s["V"], s["k"]
    y = x / s["temp"]
    m = y.amax(-1, keepdim=True)
    e = (y - m).exp()
    total = e.sum(-1, keepdim=True)
    lse = m + total.log()
    entropy = lse[:, 0] - (e * torch.where(e > 0, y, 0.0)).sum(-1) / total[:, 0]
    out = dict(logprobs=y.gather(1, s["tokens"][:, None])[:, 0] - lse[:, 0], entropy=entropy, top_logprobs=y.new_empty(T, 0),
               top_ids=torch.empty(T, 0, dtype=torch.int32, device=DEV))
    if k:
        # equal values: the lower index first.  The value's bits in order, then the index, in one whole number
        bits = (x + 0.0).view(torch.int32)
        order = (bits ^ (bits >> 31).bitwise_and(0x7fffffff)).long()
        ids = 0xffffffff - (torch.topk((order << 32) | (0xffffffff - torch.arange(V, device=DEV)), k, dim=1).values & 0xffffffff)
        out.update(top_logprobs=y.gather(1, ids) - lse, top_ids=ids.int())
    return out


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "plan":
        return _exact_plan(s)
    if kind == "rope":
        return _exact_rope(s)
    if kind == "attention":
        return _exact_attention(s)
    return _exact_logprobs(s)


def _exact_plan(s):
    tables, free = s["tables"].tolist(), s["free"].tolist()
    lens, counts, page, T = s["lens"].tolist(), s["counts"].tolist(), s["page"], s["tokens"]
    parents = s["parents"].tolist() if s["parents"] is not None else None
    top = int(s["n_free"])
    left, cu, pos, slots, masks, kv = top, [0], [], [], [], []
    missed = False
    for b, (l, n) in enumerate(zip(lens, counts)):
        have, want = -(-l // page), -(-(l + n) // page)
        ok = l + n <= len(tables[b]) * page and (parents is None or n <= 64)
        if ok and want > have:
            missed = missed or want - have > left
            ok = not missed
            if ok:
                for c in range(have, want):
                    left -= 1
                    tables[b][c] = free[left]
        own_masks = []
        for j in range(n):
            p = parents[cu[-1] + j] if parents is not None else j - 1
            own_masks.append((1 << j) | (own_masks[p] if 0 <= p < j else 0))
            pos.append(l + bin(own_masks[-1]).count("1") - 1 if ok else -1)
            slots.append(tables[b][(l + j) // page] * page + (l + j) % page if ok else -1)
            masks.append((own_masks[-1] - (1 << 64) if own_masks[-1] >= 1 << 63 else own_masks[-1]) if ok else 0)
        cu.append(cu[-1] + n)
        kv.append(l + n if ok else 0)
    return dict(tables=_ints(tables), cu=_ints(cu), positions=_ints(pos), slots=_ints(slots, torch.int64),
                masks=_ints(masks, torch.int64) if parents is not None else None, kv_lens=_ints(kv), n_free=_ints([left]))


def _exact_rope(s):
    T, Hq, Hkv, D, R = s["T"], s["Hq"], s["Hkv"], s["D"], s["R"]
    x = s["qkv"].double().reshape(T, Hq + 2 * Hkv, D)
    table = s["cos_sin"].double().index_select(0, s["positions"].long())
    i = torch.arange(R // 2, device=DEV)
    first, second = (2 * i, 2 * i + 1) if s["pairs"] else (i, i + R // 2)

    def normed(part, weight):
        y = part / (part.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * weight.double()
        z, c, sn = y.clone(), table[:, None, :R // 2], table[:, None, R // 2:]
        z[..., first] = y[..., first] * c - y[..., second] * sn
        z[..., second] = y[..., second] * c + y[..., first] * sn
        return z

    # what the caches hold in 64 bits: the rows stored, everything else as it was (in units of the scale where there is one)
    def cache(held, rows, scale):
        flat = held.double().reshape(-1, Hkv, D)
        flat[s["slots"]] = rows if scale is None else (rows / scale.double()[None, :, None]).clamp(-448.0, 448.0)
        return flat.view(held.shape)

    return dict(q=normed(x[:, :Hq], s["q_weight"]), k_cache=cache(s["k_cache"], normed(x[:, Hq:Hq + Hkv], s["k_weight"]), s["k_scale"]),
                v_cache=cache(s["v_cache"], x[:, Hq + Hkv:], s["v_scale"]))


def _exact_attention(s):
    Hq, Hkv, D, page = s["Hq"], s["Hkv"], s["D"], s["page"]
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, S in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        n = hi - lo
        blocks = s["tables"][b, :-(-S // page)].long()
        sees = torch.ones(n, S, dtype=torch.bool, device=DEV)
        if s["masks"] is None:
            sees[:, S - n:] = torch.ones(n, n, dtype=torch.bool, device=DEV).tril()
        else:
            sees[:, S - n:] = (s["masks"][lo:hi, None] >> torch.arange(n, device=DEV)) & 1 == 1
        for h in range(Hkv):
            K = s["k_cache"][blocks, :, h].double().reshape(-1, D)[:S]
            V = s["v_cache"][blocks, :, h].double().reshape(-1, D)[:S]
            if s["k_scale"] is not None:
                K, V = K * s["k_scale"][h].double(), V * s["v_scale"][h].double()
            g = Hq // Hkv
            x = torch.einsum("tgd,sd->gts", s["q"][lo:hi, h * g:(h + 1) * g].double(), K) / math.sqrt(D)
            p = torch.softmax(x.masked_fill(~sees, float("-inf")), -1)
            out[lo:hi, h * g:(h + 1) * g] = torch.einsum("gts,sd->tgd", p, V)
    return dict(out=out)


def _exact_logprobs(s):
    x, k = s["logits"].double(), s["k"]
    lp = torch.log_softmax(x / s["temp"], -1)
    p = lp.exp()
    entropy = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    ids = torch.stack([r.sort(descending=True, stable=True).indices[:k] for r in x]) if k else torch.empty(s["T"], 0, dtype=torch.int64, device=DEV)
    return dict(logprobs=lp.gather(1, s["tokens"][:, None])[:, 0], entropy=entropy, top_logprobs=lp.gather(1, ids), top_ids=ids.int())
