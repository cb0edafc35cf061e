"""More operators of a serving step around the MoE layer, their cases, inputs and plain forms.

What stands between the paged cache and the next token beside the operators of operators.py: a cache held in 4 bits, layers
that see a window of the text and its first tokens, the norms and the residual stream between blocks, and what a request
asks of its logits before a token is drawn.  "kind" names the operator of a case:

  attention  `tree_attention` over a cache in 4 bits, or with a window and first tokens that stay visible, or both
  norm       `residual_norm`: a block's output normalised, gated, scaled and added to the residual, and normalised for the next block
  logits     `adjust_logits`: penalties for repeated tokens, biases of single tokens, grammar masks
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
FP4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)           # magnitudes of the 4-bit codes 0 .. 7; bit 3 is the sign


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
def _attention(B, L, most, tree, Hq, Hkv, D, page, cache, window=0, sinks=0, even=False):
    """most: new tokens of the request that has most; window 0: none; even: all requests alike, else from a fifth of L (most) up to it."""
    return dict(kind="attention", B=B, L=L, most=most, tree=tree, Hq=Hq, Hkv=Hkv, D=D, page=page, cache=cache, window=window,
                sinks=sinks, even=even)


def _norm(T, H, after, gate, wide, scale):
    """after: a norm of the block's output too; gate: "", "column", "token" or "full"; wide: the residual in float32."""
    return dict(kind="norm", T=T, H=H, after=after, gate=gate, wide=wide, scale=scale)


def _logits(B, most, V, L, tree, bf16, masked, biases):
    """most: drafted tokens of each request; L: tokens of the longest history; masked: every other row has a grammar."""
    return dict(kind="logits", B=B, most=most, V=V, L=L, tree=tree, bf16=bf16, masked=masked, biases=biases)


def listed():
    return [
        # one user's next token over a long document in a 4-bit cache: latency, and one pass cut over the whole chip
        dict(name="attention4_b1_l32767", **_attention(1, 32767, 1, False, 32, 4, 128, 64, "fp4", even=True)),
        # a decode batch of ragged lengths: a quarter of the 16-bit cache's bytes, if decoding them does not take longer
        dict(name="attention4_b64_decode", **_attention(64, 8192, 1, False, 32, 4, 128, 16, "fp4")),
        # trees of up to 16 drafted tokens, ragged in both
        dict(name="attention4_b32_tree16", **_attention(32, 8001, 16, True, 32, 4, 128, 64, "fp4")),
        # a local layer at decode: long texts of which a window and the first tokens are read
        dict(name="window_b64_decode", **_attention(64, 16384, 1, False, 32, 4, 128, 16, "bf16", 1024, 4)),
        # two prompts' next chunks through a local layer, causal
        dict(name="window_b2_chunk1021", **_attention(2, 8190, 1021, False, 32, 8, 128, 64, "bf16", 1024, 4)),
        # the largest trees over a window of a 4-bit cache
        dict(name="window4_b16_tree64", **_attention(16, 12288, 64, True, 32, 4, 128, 64, "fp4", 4095, 64)),
        # one user's next token: a latency between two products
        dict(name="norm_t1", **_norm(1, 7168, False, "", False, 1.0)),
        # a decode batch of trees, a width that no vector divides, gated per token, the stream in 32 bits
        dict(name="norm_t613_h1999", **_norm(613, 1999, True, "token", True, 0.7)),
        # a long prompt, norms on both sides of the block and a gate per column: bytes count
        dict(name="norm_t16384", **_norm(16384, 7168, True, "column", False, 1.0)),
        # one request's logits: its history read by the whole chip
        dict(name="logits_b1", **_logits(1, 1, 131072, 4000, False, True, True, 20)),
        # a decode batch with long histories
        dict(name="logits_b64", **_logits(64, 1, 131072, 8192, False, False, False, 8)),
        # all drafted tokens of a large batch, each under its own path and grammar, an odd vocabulary
        dict(name="logits_b128_tree16", **_logits(128, 16, 100003, 2048, True, True, True, 0)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "norm", "norm", "logits", "logits"])
    if kind == "attention":
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = min(64, Hkv * rng.choice([1, 2, 3, 4, 5, 8, 8, 16]))
        tree = rng.random() < 0.5
        most = _log_int(rng, 1, 64) if tree else rng.choice([1, 1, 1, _log_int(rng, 2, 600)])
        B, L = _log_int(rng, 1, 64), _log_int(rng, 16, 32768)
        cache = rng.choice(["fp4", "fp4", "fp4", "bf16", "fp8"])
        window = _log_int(rng, 1, 8192) if cache != "fp4" or rng.random() < 0.4 else 0
        sinks = rng.choice([0, 1, 4, 4, 64, 130]) if window else 0
        # no more cached keys, and no more products, than the largest listed cases have; a plain form's scores fit too
        while B > 1 and (B * L * Hkv > 16 * 12288 * 4 or B * min(L, window + sinks + most if window else L) * Hq * most > 16 * 4223 * 32 * 64):
            B = B // 2
        while min(L, window + sinks + most if window else L) * Hq * most > 2 * 2049 * 32 * 1021:
            L = L // 2
        return _attention(B, max(L, most), most, tree, Hq, Hkv, rng.choice([64, 128, 128, 128]), rng.choice([16, 32, 64, 128]),
                          cache, window, sinks, rng.random() < 0.3)
    if kind == "norm":
        H = rng.choice([_log_int(rng, 16, 8192), _log_int(rng, 16, 1024) * 8, 64 * _log_int(rng, 1, 128)])
        return _norm(min(_log_int(rng, 1, 16384), 16384 * 7168 // H), H, rng.random() < 0.5, rng.choice(["", "", "column", "token", "full"]),
                     rng.random() < 0.4, rng.choice([1.0, 1.0, 0.25, 1.4]))
    V, tree = _log_int(rng, 1000, 131072), rng.random() < 0.4
    B, most = _log_int(rng, 1, 256), _log_int(rng, 1, 64) if tree else rng.choice([1, 1, 1, 5])
    while B > 1 and B * most * V > 2048 * 100003:
        B = B // 2
    return _logits(B, most, V, _log_int(rng, 1, 8192), tree, rng.random() < 0.6, rng.random() < 0.5, rng.choice([0, 1, 20, 300]))


def _spread(case, most="most"):
    """(cached length, new tokens) of each request: the same for every seed, ragged by the golden section."""
    B, L, most = case["B"], case["L"], case[most]
    got = []
    for b in range(B):
        f = 1.0 if case.get("even") or b == 0 else (b * 0.6180339887) % 1.0
        n = max(1, round(most * (1.0 if f == 1.0 else 0.25 + 0.75 * ((b * 0.7548776662) % 1.0))))
        got.append((max(0, round(L * (0.2 + 0.8 * f)) - n), n))
    return got


def work(case):
    c = dict(case)
    if c["kind"] == "attention":
        reqs, per = _spread(c), {"bf16": 2.0, "fp8": 1.0, "fp4": 0.5 + 1 / 32}[c["cache"]]
        new = sum(n for _, n in reqs)
        W, S = c["window"] or 1 << 40, c["sinks"]
        keys = sum(min(l + n, W + S + n - 1) for l, n in reqs)
        if c["tree"]:
            seen = sum(n * min(l + n, W + S) for l, n in reqs)
        else:
            seen = sum(min(l + j + 1, W + min(S, max(0, l + j + 1 - W))) for l, n in reqs for j in range(n))
        return {"bytes": 2 * keys * c["Hkv"] * c["D"] * per + 2 * 2 * new * c["Hq"] * c["D"], "flops": 4 * seen * c["Hq"] * c["D"]}
    if c["kind"] == "norm":
        T, H = c["T"], c["H"]
        gate = {"": 0, "column": 2 * H, "token": 2 * T, "full": 2 * T * H}[c["gate"]]
        return {"bytes": T * H * (4 + (8 if c["wide"] else 4)) + 2 * H * (2 if c["after"] else 1) + gate,
                "flops": T * H * (14 if c["after"] else 8)}
    reqs = _spread(c)
    T, e = sum(n for _, n in reqs), 2 if c["bf16"] else 4
    grammar = (T + 1) // 2 * -(-c["V"] // 32) * 4 if c["masked"] else 0
    return {"bytes": 2 * T * c["V"] * e + grammar + sum(4 * l for l, _ in reqs) + 8 * T + c["B"] * (28 + 8 * c["biases"]), "flops": T * c["V"]}


# ---------------------------------------------------------------------------------------------- inputs
def _gen(seed, part):
    return torch.Generator(device=DEV).manual_seed(1000003 * (int(seed) % (1 << 40)) + part)


def _randn(seed, part, *shape):
    return torch.randn(*shape, generator=_gen(seed, part), device=DEV)


def _rand(seed, part, *shape):
    return torch.rand(*shape, generator=_gen(seed, part), device=DEV)


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


def _in_4_bits(x):
    """x [..., D] -> codes [..., D/2], two to a byte, and a power of two for each 32 elements, [..., D/32]: the least that brings them to 7 or less."""
    blocks = x.unflatten(-1, (-1, 32))
    up = torch.ceil(torch.log2(blocks.abs().amax(-1) / 7)).clamp(-120, 120)
    y = blocks * torch.exp2(-up)[..., None]
    codes = torch.bucketize(y.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV), out_int32=True)
    codes = (codes + 8 * (y < 0)).to(torch.uint8).flatten(-2)
    return (codes[..., 0::2] | codes[..., 1::2] << 4).view(torch.float4_e2m1fn_x2), (up + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    c, seed = dict(case), int(seed)
    rng = random.Random(seed * 7919 + 17)
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
        tables[row, torch.arange(sum(pages), device=DEV) - first[row]] = ids[:sum(pages)]
        T = sum(counts)
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        k = _randn(seed, 2, n_blocks, page, Hkv, D)
        v = _randn(seed, 3, n_blocks, page, Hkv, D) + _randn(seed, 4, 1, 1, Hkv, D)
        k_scale = v_scale = None
        if c["cache"] == "fp4":
            # some channels of keys are much larger than the others
            k, k_scale = _in_4_bits(k * (1 + 4 * (_rand(seed, 8, 1, 1, Hkv, D) < 0.03)))
            v, v_scale = _in_4_bits(v)
        elif c["cache"] == "fp8":
            up = 40.0                                      # codes use the type's range, the scales bring them back
            k, v = (k * up).to(torch.float8_e4m3fn), (v * up).to(torch.float8_e4m3fn)
            k_scale, v_scale = ((0.9 + 0.2 * _rand(seed, part, Hkv)) / up for part in (6, 7))
        else:
            k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        return dict(c, q=(_randn(seed, 5, T, c["Hq"], D) * 1.5).to(torch.bfloat16), k_cache=k, v_cache=v, tables=tables,
                    kv_lens=_ints(lens), cu=_ints(cu), longest=max(lens), widest=max(counts),
                    masks=_ints(_masks(_trees(rng, counts), counts), torch.int64) if c["tree"] else None, k_scale=k_scale, v_scale=v_scale)
    if c["kind"] == "norm":
        T, H = c["T"], c["H"]
        gate = {"": None, "column": (1, H), "token": (T, 1), "full": (T, H)}[c["gate"]]
        residual = _randn(seed, 2, T, H) * (1 + 20 * (_rand(seed, 3, 1, H) < 0.004))     # a few columns of a stream are very large
        return dict(c, x=(_randn(seed, 1, T, H) * (0.2 + 3 * _rand(seed, 4, T, 1))).to(torch.bfloat16),
                    residual=residual if c["wide"] else residual.to(torch.bfloat16),
                    weight=(1 + 0.2 * _randn(seed, 5, H)).to(torch.bfloat16),
                    post_weight=(1 + 0.2 * _randn(seed, 6, H)).to(torch.bfloat16) if c["after"] else None,
                    gate=None if gate is None else torch.sigmoid(_randn(seed, 7, *gate)).to(torch.bfloat16))
    B, V, L = c["B"], c["V"], c["L"]
    reqs = _spread(c)
    rng.shuffle(reqs)
    counts = [n for _, n in reqs]
    T, cu = sum(counts), [0]
    for n in counts:
        cu.append(cu[-1] + n)
    # words are used again: low ids much more often than high ones
    words = lambda part, *shape: (V * _rand(seed, part, *shape) ** 3).long().clamp(max=V - 1)  # noqa: E731
    logits = _randn(seed, 1, T, V) * 2.5
    s = dict(c, logits=logits.to(torch.bfloat16) if c["bf16"] else logits, cu=_ints(cu), widest=max(counts),
             history=words(2, B, L).to(torch.int32), history_lens=_ints([l for l, _ in reqs]), prompt_lens=_ints([l // 3 for l, _ in reqs]),
             repetition=1 + 0.3 * _rand(seed, 3, B), frequency=0.5 * _rand(seed, 4, B), presence=0.5 * _rand(seed, 5, B),
             tokens=words(6, T) if c["most"] > 1 else None,
             masks=_ints(_masks(_trees(rng, counts), counts), torch.int64) if c["tree"] else None,
             bias_ids=None, bias=None, allowed=None, allowed_rows=None)
    if c["biases"]:
        s.update(bias_ids=words(7, B, c["biases"]).to(torch.int32), bias=3 * _randn(seed, 8, B, c["biases"]))
    if c["masked"]:                                        # a grammar lets a tenth of the vocabulary through
        bits = (_rand(seed, 9, (T + 1) // 2, -(-V // 32), 32) < 0.1).long() << torch.arange(32, device=DEV)
        bits = bits.sum(-1)
        turn = torch.arange(T, device=DEV)
        s.update(allowed=torch.where(bits < 1 << 31, bits, bits - (1 << 32)).to(torch.int32),
                 allowed_rows=torch.where(turn % 2 == 0, turn // 2, -1).to(torch.int32))
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if s["kind"] == "attention":
        return _run_attention(s) if own else _plain_attention(s)
    if s["kind"] == "norm":
        return _run_norm(s) if own else _plain_norm(s)
    return _run_logits(s) if own else _plain_logits(s)


def _run_attention(s):
    return dict(out=_package().tree_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["cu"], masks=s["masks"],
                                              k_scale=s["k_scale"], v_scale=s["v_scale"], window=s["window"] or None, sinks=s["sinks"]))


def _run_norm(s):
    y, residual = _package().residual_norm(s["x"], s["residual"], s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                                           scale=s["scale"], eps=1e-6)
    return dict(y=y, residual=residual)


def _run_logits(s):
    return dict(logits=_package().adjust_logits(s["logits"], s["cu"], history=s["history"], history_lens=s["history_lens"],
                                                prompt_lens=s["prompt_lens"], tokens=s["tokens"],
                                                masks=s["masks"] if s["tokens"] is not None else None,    # (of no drafted tokens there are none)
                                                repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                                                bias_ids=s["bias_ids"], bias=s["bias"], allowed=s["allowed"], allowed_rows=s["allowed_rows"]))


# ---------------------------------------------------------------------------------------------- plain forms
def _widened(cache, scale, at):
    """The cache's rows `at` in float32."""
    Hkv = cache.shape[2]
    if cache.dtype == torch.float4_e2m1fn_x2:
        codes = cache.view(torch.uint8).flatten(0, 1)[at]
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
        values = torch.tensor([*FP4, *(-x for x in FP4)], device=DEV)[codes]
        up = (scale.view(torch.uint8).flatten(0, 1)[at].int() << 23).view(torch.float32)
        return (values.unflatten(-1, (-1, 32)) * up[..., None]).flatten(-2)
    rows = cache.flatten(0, 1).view(-1, Hkv, cache.shape[3])[at].float()
    return rows if scale is None else rows * scale[:, None]


def _plain_attention(s):
    B, Hq, Hkv, D, page = s["B"], s["Hq"], s["Hkv"], s["D"], s["page"]
    W, sinks = s["window"] or 1 << 40, s["sinks"]
    G, n = Hq // Hkv, s["widest"]
    cu, lens = s["cu"].long(), s["kv_lens"].long()
    counts = cu[1:] - cu[:-1]
    prefix = lens - counts
    j = torch.arange(n, device=DEV)
    there = j < counts[:, None]                                            # [B, n]
    row = (cu[:-1, None] + j).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[row].view(B, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, D)
    # the first tokens, then those from the first one that a request's first row sees on
    S = min(s["longest"], W + sinks + n)
    col = torch.arange(S, device=DEV)
    skip = (prefix - W + 1 - sinks).clamp_min(0)
    key = torch.where(col < sinks, col, col + skip[:, None])               # [B, S]
    at = torch.gather(s["tables"].long(), 1, (key // page).clamp_max(s["tables"].shape[1] - 1)).clamp_min(0) * page + key % page
    k = _widened(s["k_cache"], s["k_scale"], at).transpose(1, 2)           # [B, Hkv, S, D]
    v = _widened(s["v_cache"], s["v_scale"], at).transpose(1, 2)
    new = key - prefix[:, None]                                            # [B, S]: which of the new tokens a key is
    if s["masks"] is not None:
        bits = torch.bitwise_right_shift(s["masks"][row][:, :, None], j).bitwise_and(1)   # [B, n, n]
        rank = prefix[:, None, None] + bits.cumsum(-1) - bits              # of a new token among what a row may see
        own_rank = prefix[:, None] + bits.sum(-1) - 1
        pick = new.clamp(0, n - 1)[:, None, :].expand(B, n, S)
        may = torch.where((new >= 0)[:, None, :], bits.gather(2, pick).bool(), True)
        rank = torch.where((new >= 0)[:, None, :], rank.gather(2, pick), key[:, None, :])
    else:
        own_rank = prefix[:, None] + j
        rank = key[:, None, :].expand(B, n, S)
        may = rank <= own_rank[:, :, None]
    sees = may & ((rank > own_rank[:, :, None] - W) | (rank < sinks)) & (key < lens[:, None])[:, None, :] & there[:, :, None]
    hide = torch.zeros(sees.shape, device=DEV).masked_fill_(~sees, float("-inf"))
    x = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D)).view(B, Hkv, n, G, S).add_(hide[:, None, :, None, :])
    x = x.sub_(x.amax(-1, keepdim=True).clamp_min(-3.0e38)).exp_()
    out = torch.matmul(x.view(B, Hkv, n * G, S), v) / x.sum(-1).view(B, Hkv, n * G, 1).clamp_min(1e-38)
    out = out.view(B, Hkv, n, G, D).transpose(1, 2).reshape(B * n, Hq, D).to(torch.bfloat16)
    T = s["q"].shape[0]
    each = lambda t: t.repeat_interleave(counts, output_size=T)            # noqa: E731
    return dict(out=out[each(torch.arange(B, device=DEV) * n) + torch.arange(T, device=DEV) - each(cu[:-1])])


def _rms(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()


def _plain_norm(s):
    x = s["x"].float()
    if s["post_weight"] is not None:
        x = _rms(x, s["post_weight"])
    if s["gate"] is not None:
        x = x * s["gate"].float()
    h = s["residual"].float() + s["scale"] * x
    return dict(y=_rms(h, s["weight"]).to(torch.bfloat16), residual=h.to(s["residual"].dtype))


def _plain_logits(s):
    T, V, B = s["logits"].shape[0], s["V"], s["B"]
    cu = s["cu"].long()
    b = torch.repeat_interleave(torch.arange(B, device=DEV), cu[1:] - cu[:-1], output_size=T)
    at = torch.arange(s["history"].shape[1], device=DEV)
    held, asked = at < s["history_lens"][:, None], at < s["prompt_lens"][:, None]
    ids = s["history"].long()
    said = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, (held & ~asked).float())[b]      # how often, of what was generated
    seen = torch.zeros(B, V, device=DEV).scatter_add_(1, ids, (held & asked).float())[b]
    if s["tokens"] is not None:                                            # and the row's own path
        j = torch.arange(s["widest"], device=DEV)
        i = torch.arange(T, device=DEV) - cu[:-1][b]
        path = torch.bitwise_right_shift(s["masks"][:, None], j).bitwise_and(1).float() if s["masks"] is not None else (j <= i[:, None]).float()
        said.scatter_add_(1, s["tokens"][(cu[:-1][b][:, None] + j).clamp_max(T - 1)], path)
    x = s["logits"].float()
    rep = s["repetition"][b][:, None]
    x = torch.where(said + seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][b][:, None] * said - s["presence"][b][:, None] * (said > 0).float()
    if s["bias_ids"] is not None:                                          # of a token named twice the last bias counts
        last = torch.zeros(B, V, dtype=torch.int64, device=DEV).scatter_reduce_(
            1, s["bias_ids"].long(), torch.arange(1, s["biases"] + 1, device=DEV).expand(B, -1), "amax")
        x = x + torch.cat([torch.zeros(B, 1, device=DEV), s["bias"]], 1).gather(1, last)[b]
    if s["allowed"] is not None:
        word = s["allowed"][s["allowed_rows"].long().clamp_min(0)].repeat_interleave(32, 1)[:, :V]
        let = torch.bitwise_right_shift(word, torch.arange(V, device=DEV, dtype=torch.int32) % 32).bitwise_and(1).bool()
        x = torch.where(let | (s["allowed_rows"] < 0)[:, None], x, float("-inf"))
    return dict(logits=x.to(s["logits"].dtype))


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "attention":
        return _exact_attention(s)
    if s["kind"] == "norm":
        return _exact_norm(s)
    return _exact_logits(s)


def _exact_rows(cache, scale, blocks, h, n):
    """The first n keys of head h in a request's blocks, in 64 bits."""
    if cache.dtype == torch.float4_e2m1fn_x2:
        byte = cache.view(torch.uint8)[blocks, :, h].reshape(-1, cache.shape[3])[:n]
        nibble = torch.stack([byte % 16, byte // 16], 2).reshape(n, -1)
        size = torch.tensor(FP4, dtype=torch.float64, device=DEV).index_select(0, (nibble % 8).long().flatten()).view(nibble.shape)
        power = scale.view(torch.uint8)[blocks, :, h].reshape(-1, scale.shape[3])[:n].double() - 127
        return torch.where(nibble >= 8, -size, size) * torch.pow(torch.full_like(power, 2.0), power).repeat_interleave(32, 1)
    rows = cache[blocks, :, h].double().reshape(-1, cache.shape[3])[:n]
    return rows if scale is None else rows * scale[h].double()


def _exact_attention(s):
    Hq, Hkv, D, page = s["Hq"], s["Hkv"], s["D"], s["page"]
    cu, lens = s["cu"].tolist(), s["kv_lens"].tolist()
    masks = s["masks"].tolist() if s["masks"] is not None else None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, S in enumerate(lens):
        lo, hi = cu[b], cu[b + 1]
        n, p = hi - lo, S - (hi - lo)
        blocks = s["tables"][b, :-(-S // page)].long()
        may = torch.zeros(n, S, dtype=torch.bool)
        may[:, :p] = True
        for j in range(n):
            may[j, p:] = torch.tensor([masks[lo + j] >> i & 1 == 1 if masks is not None else i <= j for i in range(n)])
        if s["window"]:
            number = may.long().cumsum(1) - 1                              # of what a row may see: the last ones, and the first
            may &= (number >= may.sum(1, keepdim=True) - s["window"]) | (number < s["sinks"])
        sees = may.to(DEV)
        for h in range(Hkv):
            K = _exact_rows(s["k_cache"], s["k_scale"], blocks, h, S)
            V = _exact_rows(s["v_cache"], s["v_scale"], blocks, h, S)
            g = Hq // Hkv
            x = torch.einsum("tgd,sd->gts", s["q"][lo:hi, h * g:(h + 1) * g].double(), K) / math.sqrt(D)
            out[lo:hi, h * g:(h + 1) * g] = torch.einsum("gts,sd->tgd", torch.softmax(x.masked_fill(~sees, float("-inf")), -1), V)
    return dict(out=out)


def _exact_norm(s):
    unit = lambda t: t / (t.pow(2).sum(-1, keepdim=True) / s["H"] + 1e-6).sqrt()  # noqa: E731
    u = s["x"].double()
    if s["after"]:
        u = unit(u) * s["post_weight"].double()
    if s["gate"] is not None:
        u = u * s["gate"].double()
    h = s["residual"].double() + u * s["scale"]
    return dict(y=unit(h) * s["weight"].double(), residual=h)


def _exact_logits(s):
    cu, V = s["cu"].tolist(), s["V"]
    out = s["logits"].double()
    lens, asked = s["history_lens"].tolist(), s["prompt_lens"].tolist()
    masks = s["masks"].tolist() if s["masks"] is not None else None
    rows = s["allowed_rows"].tolist() if s["allowed"] is not None else None
    for b in range(s["B"]):
        told = torch.bincount(s["history"][b, asked[b]:lens[b]].long(), minlength=V).double()
        heard = torch.bincount(s["history"][b, :asked[b]].long(), minlength=V) > 0
        add = torch.zeros(V, dtype=torch.float64, device=DEV)
        if s["bias_ids"] is not None:
            named = dict(zip(s["bias_ids"][b].tolist(), s["bias"][b].tolist()))
            add[_ints(list(named), torch.int64)] = torch.tensor(list(named.values()), dtype=torch.float64, device=DEV)
        for t in range(cu[b], cu[b + 1]):
            count = told.clone()
            if s["tokens"] is not None:
                near = [i for i in range(cu[b + 1] - cu[b]) if (masks[t] >> i & 1 if masks is not None else i <= t - cu[b])]
                count += torch.bincount(s["tokens"][_ints(near, torch.int64) + cu[b]], minlength=V).double()
            x, rep = out[t], s["repetition"][b].double()
            x = torch.where(heard | (count > 0), torch.where(x > 0, x / rep, x * rep), x)
            x = x - count * s["frequency"][b].double() - torch.where(count > 0, s["presence"][b].double(), 0.0) + add
            if rows is not None and rows[t] >= 0:
                bit = torch.arange(V, device=DEV)
                x = torch.where((s["allowed"][rows[t]].long()[bit // 32] >> (bit % 32)) & 1 == 1, x, -math.inf)
            out[t] = x
    return dict(logits=out)
