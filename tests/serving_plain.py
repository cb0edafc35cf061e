"""Plain 64-bit forms of the serving step's operators (on the CPU, loops over requests and rows), and how far a kernel that
holds its sums in 32 bits and rounds where it says may be from them."""
import math

import torch

U16 = 2.0 ** -8          # a bf16 rounding, relative: half a unit of the last of 8 digits
U32 = 2.0 ** -24         # an fp32 rounding


def plan(tables, lens, counts, free, n_free, page, T, parents=None):
    """-> (tables, cu, positions, slots, masks, kv_lens, n_free) as lists; -> masks None without parents."""
    tables = [list(r) for r in tables]
    B, W = len(lens), len(tables[0]) if tables else 0
    n_free = max(0, min(n_free, len(free)))
    cu, kv, taken, wanted, total = [0], [], 0, 0, 0
    pos, slots, masks = [-1] * T, [-1] * T, [0] * T
    for b in range(B):
        l, n = lens[b], max(counts[b], 0)
        have, want = -(-l // page), -(-(l + n) // page)
        fits = l >= 0 and l + n <= W * page and total + n <= T and (parents is None or n <= 64)
        need = want - have if fits else 0
        ok = fits and (need == 0 or wanted + need <= n_free)
        if ok:
            for i in range(need):
                tables[b][have + i] = free[n_free - 1 - (wanted + i)]
            if need:
                taken = wanted + need
            seen = []
            for j in range(n):
                t = total + j
                up = parents[t] if parents is not None else j - 1
                seen.append((1 << j) | (seen[up] if 0 <= up < j else 0))
                depth = bin(seen[j]).count("1") - 1 if parents is not None else j
                pos[t] = l + depth
                slots[t] = tables[b][(l + j) // page] * page + (l + j) % page
                masks[t] = (seen[j] - (1 << 64) if seen[j] >> 63 else seen[j]) if parents is not None else 0
        wanted += need
        total += n
        cu.append(min(total, T))
        kv.append(l + n if ok else 0)
    return tables, cu, pos, slots, masks if parents is not None else None, kv, n_free - taken


def norm_rope(x, weight, eps, positions, cos_sin, interleaved):
    """x [T, heads, D] -> float64 [T, heads, D]; rows at positions outside the table are zero."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    P, R = cos_sin.shape
    placed = (positions >= 0) & (positions < P)
    row = cos_sin.double()[positions.clamp(0, max(P - 1, 0)).long()][:, None, :] if P else torch.zeros(x.shape[0], 1, 0, dtype=torch.float64)
    half = R // 2
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    out = x.clone()
    if R:
        out[..., a] = x[..., a] * row[..., :half] - x[..., b] * row[..., half:]
        out[..., b] = x[..., b] * row[..., :half] + x[..., a] * row[..., half:]
    return out * placed[:, None, None]


def attention(q, k_cache, v_cache, tables, kv_lens, cu, masks, scale, k_scale=None, v_scale=None):
    """-> (out, lse, reach) in float64; reach [T, Hq, D] = sum of p |v|, what an error of p is relative to.  A key that a row does
    not see is left out of it, whatever the cache holds there."""
    T, Hq, D = q.shape
    Hkv, page = k_cache.shape[2], k_cache.shape[1]
    out = torch.zeros(T, Hq, D, dtype=torch.float64)
    reach = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    for b in range(len(kv_lens)):
        t0, t1, S = cu[b], min(cu[b + 1], T), kv_lens[b]
        n = t1 - t0
        if S < n:
            continue
        K = torch.stack([k_cache[tables[b][s // page], s % page] for s in range(S)]).double() if S else None
        V = torch.stack([v_cache[tables[b][s // page], s % page] for s in range(S)]).double() if S else None
        for j in range(n):
            seen = list(range(S - n)) + [S - n + i for i in range(n) if (masks[t0 + j] >> i & 1 if masks is not None else i <= j)]
            if not seen:
                continue
            for h in range(Hq):
                kh = h // (Hq // Hkv)
                ks = 1.0 if k_scale is None else float(k_scale[kh])
                vs = 1.0 if v_scale is None else float(v_scale[kh])
                s = K[seen, kh] @ q[t0 + j, h].double() * (scale * ks)
                p = torch.softmax(s, 0)
                out[t0 + j, h] = p @ V[seen, kh] * vs
                reach[t0 + j, h] = p @ V[seen, kh].abs() * abs(vs)
                lse[t0 + j, h] = torch.logsumexp(s, 0)
    return out, lse, reach


def attention_bound(out, reach):
    """The probabilities may be rounded to bf16 before they meet the values, the result is; 32-bit scores of rows up to a few
    hundred apart move a probability by less than 2e-4 of itself."""
    return (U16 + 2e-4) * reach + U16 * out.abs() + 1e-30


def logprobs(logits, tokens, k, temperature):
    """-> (logprobs, entropy, top_logprobs, top_ids) in float64."""
    T, V = logits.shape
    x = logits.double()
    y = x / temperature
    lp = torch.full((T,), -math.inf, dtype=torch.float64)
    ent = torch.zeros(T, dtype=torch.float64)
    tops = torch.full((T, k), -math.inf, dtype=torch.float64)
    ids = torch.zeros(T, k, dtype=torch.int64)
    for t in range(T):
        order = sorted(range(V), key=lambda i: (-float(x[t, i]), i))[:k]
        ids[t] = torch.tensor(order, dtype=torch.int64)
        if bool((x[t] == -math.inf).all()):
            continue
        lse = torch.logsumexp(y[t], 0)
        p = torch.exp(y[t] - lse)
        ent[t] = -(p * torch.where(p > 0, y[t] - lse, torch.zeros(()).double())).sum()
        if 0 <= int(tokens[t]) < V:
            lp[t] = y[t, int(tokens[t])] - lse
        tops[t] = y[t, order] - lse
    return lp, ent, tops, ids


def logprobs_bound(V, temperature, logits):
    """A thread adds up to V / 256 + 16 exponentials one after the other, each sum a rounding; exponents of size y are
    off by two roundings of y; the entropy weighs such errors with distances from the maximum of up to y again."""
    y = float(logits.double()[torch.isfinite(logits)].abs().max()) / temperature if bool(torch.isfinite(logits).any()) else 1.0
    sums = (V / 256 + 32) * U32
    return sums + 8 * U32 * (1 + y), (sums + 8 * U32 * (1 + y)) * (2 + 2 * y)
