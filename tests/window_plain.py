"""Plain 64-bit forms of what 4-bit caches hold and of attention with a window and first tokens (on the CPU)."""
import math

import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
TIES = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)      # halfway between neighbours


def decode(codes, powers):
    """codes uint8 [..., D/2], powers uint8 [..., D/32] -> float64 [..., D]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    values = torch.where(c >= 8, -1.0, 1.0) * MAGNITUDES[c & 7]
    up = torch.where(powers == 255, math.nan, torch.exp2(powers.double() - 127))
    return (values.unflatten(-1, (-1, 32)) * up[..., None]).flatten(-2)


def power_bytes(x):
    """x float64 [..., D] -> the bytes of the least powers of two that bring each 32 elements to 7 or below, from 2^-126 to 2^125."""
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1)
    mantissa, exponent = torch.frexp(top)                                # in [0.5, 1): 8 mantissa is in [4, 8)
    byte = exponent - 3 + (mantissa > 0.875).int() + 127
    byte = torch.where(top == 0, 1, byte).clamp(1, 252)
    return torch.where(top.isfinite(), byte, 255).to(torch.uint8)


def nearest(x, powers):
    """The magnitude codes 0 .. 7 nearest to |x| under given powers, ties to the even one; and the signs."""
    y = x.abs() * torch.exp2(127 - powers.double()).repeat_interleave(32, -1)
    up, down = torch.bucketize(y, TIES, right=True), torch.bucketize(y, TIES, right=False)
    return torch.where(up % 2 == 0, up, down)            # (alike but at a tie, where one of them is even)


def encode(x):
    """-> (codes uint8 [..., D/2], powers uint8 [..., D/32]) of float64 x."""
    powers = power_bytes(x)
    c = (nearest(x, powers) + 8 * torch.signbit(x).long()).to(torch.uint8)
    return c[..., 0::2] | c[..., 1::2] << 4, powers


def attention(q, k, v, tables, kv_lens, cu, masks, scale, window=None, sinks=0):
    """k, v float64 [blocks, page, heads, D] -> (out, lse, reach) in float64, reach = sum of p |v|.  A key that a row does not see is left
    out of it, whatever the cache holds there."""
    T, Hq, D = q.shape
    page, Hkv = k.shape[1], k.shape[2]
    G = Hq // Hkv
    out, reach = torch.zeros(T, Hq, D, dtype=torch.float64), torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    for b, S in enumerate(kv_lens):
        t0, t1 = cu[b], min(cu[b + 1], T)
        n = t1 - t0
        if S < n or n == 0:
            continue
        p = S - n
        may = torch.zeros(n, S, dtype=torch.bool)
        may[:, :p] = True
        if masks is None:
            may[:, p:] = torch.ones(n, n, dtype=torch.bool).tril()
        else:
            may[:, p:] = torch.tensor([[m >> i & 1 == 1 for i in range(n)] for m in masks[t0:t1]])
        if window is not None:
            number = may.long().cumsum(1) - 1
            may &= (number >= may.sum(1, keepdim=True) - window) | (number < sinks)
        used = may.any(0).nonzero()[:, 0]                                # (the table may hold nothing for the others)
        at = torch.tensor(tables[b], dtype=torch.long)[used // page] * page + used % page
        K, V, sees = k.flatten(0, 1)[at], v.flatten(0, 1)[at], may[:, used]
        for h in range(Hkv):
            x = torch.einsum("ngd,sd->ngs", q[t0:t1, h * G:(h + 1) * G].double(), K[:, h].nan_to_num(0.0, 0.0, 0.0)) * scale
            bad = ~K[:, h].isfinite().all(-1)
            x = torch.where(bad[None, None, :], math.nan, x).masked_fill(~sees[:, None, :], -math.inf)
            some = sees.any(1)
            w = torch.softmax(x, -1).masked_fill(~sees[:, None, :], 0.0)
            w[~some] = 0.0
            Vh = V[:, h]
            odd = ~Vh.isfinite()
            clean = Vh.masked_fill(odd, 0.0)
            o, r = torch.einsum("ngs,sd->ngd", w, clean), torch.einsum("ngs,sd->ngd", w, clean.abs())
            touched = (sees.double() @ odd.double() > 0)[:, None, :].expand_as(o)
            out[t0:t1, h * G:(h + 1) * G] = torch.where(touched, math.nan, o)
            reach[t0:t1, h * G:(h + 1) * G] = torch.where(touched, math.nan, r)
            lse[t0:t1, h * G:(h + 1) * G] = torch.where(some[:, None], torch.logsumexp(x, -1), -math.inf)
    return out, lse, reach
