"""A serving step around the MoE layer: paged cache, attention over it, what lies between two blocks, and what is asked of logits and what they say.

    plan = cache_plan(block_tables, lens, counts, free_blocks, n_free, page_size, max_tokens, parents)
    q = qk_norm_rope(qkv, plan.positions, cos_sin, heads, kv_heads, q_weight, k_weight,
                     k_cache=k_cache, v_cache=v_cache, slots=plan.slots)                       # each layer
    o = tree_attention(q, k_cache, v_cache, block_tables, plan.kv_lens, plan.cu_tokens, plan.masks)
    x, residual = residual_norm(projection, residual, weight)
    logits = adjust_logits(logits, plan.cu_tokens, history, history_lens, prompt_lens, tokens, plan.masks, repetition=repetition)
    said = token_logprobs(logits, tokens, top_k=8)

The functions are thin: the operators of the same names in torch.ops.my_ops check, allocate and launch (csrc/serving_ops.cpp).
Everything stays on the device, so that a step can be captured into a graph.  Inference only: a backward pass through them warns and
gives no gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import my_ops as _my_ops  # noqa: F401  (loads the operators)

_ops = torch.ops.my_ops


class CachePlan(NamedTuple):
    cu_tokens: torch.Tensor              # [B + 1] int32: request b holds rows cu_tokens[b] .. cu_tokens[b + 1]
    positions: torch.Tensor              # [T] int32, -1: no token
    slots: torch.Tensor                  # [T] int64, -1: nothing to store
    masks: Optional[torch.Tensor]        # [T] int64 with parents, else None: causal
    kv_lens: torch.Tensor                # [B] int32, cached and new; 0: refused
    n_free: torch.Tensor                 # [1] int32: free pages left


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor               # [T] float32
    entropy: torch.Tensor                # [T] float32, nats
    top_logprobs: torch.Tensor           # [T, k] float32
    top_ids: torch.Tensor                # [T, k] int32


def cache_plan(block_tables, lens, counts, free_blocks, n_free, page_size: int, max_tokens: int, parents=None) -> CachePlan:
    """Block tables, slots, positions and tree masks of one step from request lengths, on the GPU.

    block_tables [B, pages] int32 (new pages are appended in place); lens [B] cached and counts [B] new tokens, int32;
    free_blocks [F] int32 with n_free [1] int32 of them free, taken from the top; page_size a power of two up to 1024;
    max_tokens rows of the batch; parents [max_tokens] int32: each drafted token's parent among its request's tokens,
    -1 for none (trees of at most 64 tokens), or None: every request's tokens follow one another.
    A request that finds no room - in its table row, the batch's rows, or the free pages - is refused: kv_lens 0, slots -1.
    It still counts against the rows and pages of those after it: once the rows are exceeded all later requests are
    refused, once the pages are all later ones that need any."""
    return CachePlan(*_ops.cache_plan.default(block_tables, lens, counts, free_blocks, n_free, page_size, max_tokens, parents))


def qk_norm_rope(qkv, positions, cos_sin, n_heads: int, n_kv_heads: int, q_weight=None, k_weight=None, eps: float = 1e-6,
                 interleaved: bool = False, k_cache=None, v_cache=None, slots=None, k_scale=None, v_scale=None, out=None):
    """Norms of queries and keys per head, rotation by position, and keys and values into the cache, in one pass.

    qkv [T, (n_heads + 2 n_kv_heads) D] bf16, the rows at any distance; positions [T] int32; cos_sin [P, R] float32: R/2
    cosines, then R/2 sines of each position's angles, R <= D a multiple of 16; weights [D] bf16 or float32, None: that
    side is not normalised.  Pairs (i, i + R/2), or neighbours with interleaved.
    With caches [blocks, page, n_kv_heads, D] (bf16, or e4m3 with optional scales [n_kv_heads] that values are divided by)
    and slots [T] int64: stores keys and values, returns q [T, n_heads, D].  Without: returns (q, k).
    Caches in 4 bits are float4_e2m1fn_x2 [blocks, page, n_kv_heads, D / 2] (two elements to a byte, the first in the low bits), their scales
    float8_e8m0fnu [blocks, page, n_kv_heads, D / 32], written beside them: the power of two of 32 neighbouring elements, the least that
    brings them to 7 or below (the largest code is 6).  D a multiple of 32.  Slots inside the cache must differ."""
    q, k = _ops.qk_norm_rope.default(qkv, positions, cos_sin, n_heads, n_kv_heads, q_weight, k_weight, eps, interleaved, k_cache, v_cache,
                                     slots, k_scale, v_scale, out)
    return q if k is None else (q, k)


def tree_attention(q, k_cache, v_cache, block_tables, kv_lens, cu_tokens, masks=None, scale=None, k_scale=None, v_scale=None, out=None,
                   return_lse: bool = False, window=None, sinks: int = 0):
    """Attention of the new tokens over the paged cache that holds them too: a tree of drafted tokens of each request (masks
    [T] int64 from cache_plan), or without masks one token or a causal chunk.

    q [T, Hq, D] bf16, D 64 or 128, Hq a multiple of the cache's heads; caches [blocks, page, heads, D] bf16 or e4m3 (with the
    scales of qk_norm_rope), or in 4 bits as qk_norm_rope writes them; kv_lens [B] and cu_tokens [B + 1] from the plan; scale, of any sign, defaults to
    D ** -0.5.  window: of the keys that a row may see by these rules, in the cache's order, it sees the last `window` and the first
    `sinks`; pages that none of a request's rows sees are not read (their table entries may be anything; of a tree a row that sees no new
    token counts too).
    Returns out [T, Hq, D] bf16, or (out, lse [T, Hq] float32).  A row that sees no key is 0, its lse -inf."""
    o, lse = _ops.tree_attention.default(q, k_cache, v_cache, block_tables, kv_lens, cu_tokens, masks, scale, k_scale, v_scale, out, return_lse,
                                       window, sinks)
    return (o, lse) if return_lse else o


def token_logprobs(logits, tokens, top_k: int = 0, temperature: float = 1.0) -> TokenLogprobs:
    """Log probability of tokens [T] int64 under logits [T, V] (float32 or bf16, rows at any distance) / temperature, the row's
    entropy, and its top_k <= 32 most likely tokens (equal logits: the lower index first).  -inf logits are masked tokens;
    a row of nothing else gives -inf and entropy 0; a token outside [0, V) gives -inf; NaN or +inf in a row give NaN."""
    return TokenLogprobs(*_ops.token_logprobs.default(logits, tokens, top_k, temperature))


def residual_norm(x, residual=None, weight=None, post_weight=None, gate=None, scale: float = 1.0, eps: float = 1e-6, out=None,
                  residual_out=None):
    """What stands between two blocks, in one pass: a norm of the block's output, its gate, the residual, a norm for the next block.

    u = x rsqrt(mean(x^2) + eps) post_weight (x itself without a post_weight);  h = residual + scale gate u;
    y = h rsqrt(mean(h^2) + eps) weight.  x [T, H] bf16; residual [T, H] bf16 or float32 (None: 0); weights [H] bf16 or float32 (both alike);
    gate bf16 or float32, [H] or [T or 1, H or 1].  Rows at any distance.  Returns (y [T, H] bf16, h in the residual's dtype).
    out and residual_out may each be x or the residual itself; other overlaps are refused.  H up to 32768."""
    return _ops.residual_norm.default(x, residual, weight, post_weight, gate, scale, eps, out, residual_out)


def adjust_logits(logits, cu_tokens=None, history=None, history_lens=None, prompt_lens=None, tokens=None, masks=None, repetition=None,
                  frequency=None, presence=None, bias_ids=None, bias=None, allowed=None, allowed_rows=None, out=None):
    """Penalties for repeated tokens, biases of single ones and grammar masks on logits [T, V] (float32 or bf16), in one pass.

    Rows belong to requests by cu_tokens [B + 1] from cache_plan (None: a row each).  history [B, L] int32 holds each request's
    history_lens [B] tokens (None: L), the first prompt_lens [B] of them its prompt (None: none); with tokens [T] int64 a row's history
    goes on with those that its mask names (masks [T] from cache_plan; None: those up to its own).  Of a token generated n times or
    heard in the prompt: x / repetition where x > 0, else x repetition; then - frequency n - presence (where n > 0); [B] float32
    each.  Then + bias [B, N] float32 of the tokens bias_ids [B, N] int32 (of equal ids the last counts; N <= 1023), and -inf where
    allowed [M, ceil(V / 32)] int32 has no bit for the token in the row's grammar, allowed_rows [T] int32 (None: its own; -1: none).
    Ids outside [0, V) are passed over.  Returns out, a new tensor unless given; logits itself may be given."""
    return _ops.adjust_logits.default(logits, cu_tokens, history, history_lens, prompt_lens, tokens, masks, repetition, frequency, presence,
                                      bias_ids, bias, allowed, allowed_rows, out)
