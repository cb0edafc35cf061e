"""Plain 64-bit forms of residual_norm and adjust_logits (on the CPU), and how far a kernel that computes in 32 bits and rounds once may
be from them."""
import math

import torch

U16 = 2.0 ** -8          # a bf16 rounding, relative: half a unit of the last of 8 digits
U32 = 2.0 ** -24         # an fp32 rounding


def residual_norm(x, residual, weight, post_weight, gate, scale, eps):
    """-> (y, h, reach) in float64; reach = |residual| + |scale gate u|, what an error of h is relative to."""
    unit = lambda t, w: t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    u = x.double()
    if post_weight is not None:
        u = unit(u, post_weight)
    if gate is not None:
        u = u * gate.double()
    r = torch.zeros_like(u) if residual is None else residual.double()
    h = r + scale * u
    return unit(h, weight), h, r.abs() + (scale * u).abs()


def residual_norm_bounds(y, h, reach, weight, eps, out_unit):
    """A lane adds up to 32 squares one after the other, then 6 steps over lanes and 16 over wavefronts: a mean is off by less than
    64 roundings of itself, its root by half of that; x eight roundings on the way.  Twice (two norms), and h's error weighs in y with
    the second norm's factor."""
    off_h = 100 * U32 * reach
    factor = (1.0 if weight is None else weight.double().abs()) / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return U16 * y.abs() + 100 * U32 * y.abs() + factor * off_h + factor * h.abs() * off_h.norm(dim=-1, keepdim=True) / h.norm(dim=-1, keepdim=True).clamp_min(1e-30) + 1e-30, \
        out_unit * h.abs() + off_h + 1e-30


def adjust_logits(x, cu, history, lens, asked, tokens, masks, rep, freq, pres, bias_ids, bias, allowed, rows):
    """x [T, V] float64, everything else lists (or None) -> (out, reach): reach the sum of the magnitudes that were added."""
    T, V = x.shape
    out, reach = x.clone(), x.abs()
    B = len(cu) - 1 if cu is not None else T
    for b in range(B):
        t0, t1 = (cu[b], min(cu[b + 1], T)) if cu is not None else (b, b + 1)
        held = history[b][:lens[b] if lens is not None else None] if history is not None else []
        cut = asked[b] if asked is not None else 0
        named = dict(zip(bias_ids[b], bias[b])) if bias_ids is not None else {}
        for t in range(max(t0, 0), t1):
            path = []
            if tokens is not None:
                path = [tokens[t0 + i] for i in range(t1 - t0) if (masks[t] >> i & 1 if masks is not None else i <= t - t0)]
            n, heard = {}, set(held[:max(cut, 0)])
            for v in held[max(cut, 0):] + path:
                n[v] = n.get(v, 0) + 1
            r, f, p = (w[b] if w is not None else d for w, d in ((rep, 1.0), (freq, 0.0), (pres, 0.0)))
            for v in heard | set(n) | set(named):
                if not 0 <= v < V:
                    continue
                y, c = float(x[t, v]), n.get(v, 0)
                if v in heard or c:
                    y = y / r if y > 0 else y * r
                    reach[t, v] = abs(y) + abs(f) * c + abs(p)
                    y = y - f * c - (p if c else 0.0)
                if v in named:
                    y += named[v]
                    reach[t, v] += abs(named[v])
                out[t, v] = y
            row = -1 if allowed is None else rows[t] if rows is not None else t
            if allowed is not None and 0 <= row < len(allowed):
                bits = torch.tensor([(allowed[row][v // 32] >> (v % 32)) & 1 for v in range(V)], dtype=torch.bool)
                out[t] = torch.where(bits, out[t], -math.inf)
    return out, reach
