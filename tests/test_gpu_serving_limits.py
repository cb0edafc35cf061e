"""The serving step's operators at the limits of what they accept."""
import math

import pytest
import torch

import serving_plain as plain
from test_gpu_attention_tiles import ROOM, attend, tile_rows, with_room
from test_gpu_serving import STEPS, Step, check_rows, ints, say

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ token_logprobs
def log_probabilities(x, tokens, k, temperature):
    """float64, distances from the maximum first, so that nothing cancels -> (logprobs, entropy, top_logprobs, top_ids)."""
    x = x.double()
    d = (x - x.amax(-1, keepdim=True)) / temperature
    e = d.exp()
    s = e.sum(-1, keepdim=True)
    lp = d - s.log()
    entropy = s.log()[:, 0] - (e * d.clamp(min=-1000)).sum(-1) / s[:, 0]
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    return lp.gather(1, tokens[:, None])[:, 0], entropy, lp.gather(1, ids), ids


def check_sharp(pkg, dev, x, k, temperature, tokens):
    """A logarithm is off by roundings of its own size, and by those of the sum it comes from: V / 256 + 32 additions one after the other,
    and exponentials of up to -30 (smaller ones add nothing) whose exponents went through four roundings.  None of it grows with the logits."""
    say("token_logprobs", tuple(x.shape), x.dtype, "temperature", temperature)
    said = pkg.token_logprobs(x.to(dev), tokens.to(dev), top_k=k, temperature=temperature)
    lp, ent, tops, ids = log_probabilities(x, tokens, k, temperature)
    sums = (x.shape[1] / 256 + 32 + 30 * 4) * plain.U32

    def close(got, want, most):
        got = got.double().cpu()
        beyond = want.abs() > 3.3e38                     # more than float32 holds
        assert bool((got[beyond] < -3.3e38).all())
        worst = ((got - want).abs() / most)[~beyond]
        assert worst.numel() == 0 or float(worst.max()) <= 1, f"{float(worst.max())} of the bound"
    assert said.top_ids.cpu().tolist() == ids.tolist()
    close(said.logprobs, lp, sums + 8 * plain.U32 * lp.abs())
    close(said.top_logprobs, tops, sums + 8 * plain.U32 * tops.abs())
    close(said.entropy, ent, sums * (1 + 2 * ent))
    assert bool((said.logprobs <= sums).all()) and bool((said.top_logprobs <= sums).all())


SHAPES = [(3, 5000), (2, 131072), (1100, 517)]           # in segments, in one piece; short rows


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("temperature", [1e-3, 1e-5, 1e-6, 1e-8, 1e-20, 1e-29])
def test_logprobs_at_small_temperatures(pkg, dev, temperature, T, V, bf16):
    """One token dominates, or several equal ones do, in different threads and segments."""
    g = torch.Generator().manual_seed(V)
    x = (10 + 18 * torch.rand(T, V, generator=g)).to(torch.bfloat16 if bf16 else torch.float32)
    x[0, V // 3] = 29.7
    x[1, 0] = x[1, 300] = x[1, V // 2 + 1] = x[1, V - 1] = 29.3
    tokens = torch.randint(0, V, (T,), generator=g)
    tokens[0], tokens[1] = V // 3, V - 1
    check_sharp(pkg, dev, x, 5, temperature, tokens)


@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("far", [300.0, 1e4, -1e4, 1e6])
def test_logprobs_of_logits_far_from_zero(pkg, dev, far, T, V):
    g = torch.Generator().manual_seed(V)
    x = far + torch.randn(T, V, generator=g)
    check_sharp(pkg, dev, x, 5, 1.0, torch.randint(0, V, (T,), generator=g))


@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_logprobs_of_the_largest_logits(pkg, dev, temperature, T, V):
    """Tokens forced by the type's highest value."""
    x = torch.randn(T, V, generator=torch.Generator().manual_seed(V)).to(torch.bfloat16)
    top = torch.finfo(torch.bfloat16).max
    x[0, V // 3] = top
    x[1, 1] = x[1, 400] = x[1, V - 1] = top
    x[1, 2:100] = 1e38
    x[2 % T] = top
    check_sharp(pkg, dev, x, 5, temperature, torch.full((T,), V - 1))


# ------------------------------------------------------------------------------------------------ cache_plan
def test_plan_of_tensors_side_by_side_in_memory(pkg, dev):
    """One allocation for all, results right before and after what is read, lengths between the rows of the table: nothing overlaps."""
    say("cache_plan in one allocation")
    tables, lens, counts, free, T = [[4, -1, -1], [6, 1, -1]], [3, 7], [2, 4], [0, 2, 3, 5], 6
    want = plain.plan(tables, lens, counts, free, 4, 4, T, None)
    mem = torch.full((64,), -9, dtype=torch.int32, device=dev)
    rows = mem[:32].view(2, 16)
    rows[:, :3] = ints(tables, dev)
    mem[4:6], mem[6:8], mem[32:36], mem[36] = ints(lens, dev), ints(counts, dev), ints(free, dev), 4
    at = lambda i: mem.data_ptr() + 4 * i
    slots = torch.zeros(T, dtype=torch.int64, device=dev)
    kv, cu, left, pos = 8, 10, 37, 38                     # kv_lens right behind counts, the count left right behind the stack's
    rc = pkg._lib.lib.moe_cache_plan(torch.cuda.current_stream().cuda_stream, at(0), 16, 2, 3, at(4), at(6), at(32), 4, at(36), 4, None, T, at(cu), at(pos),
                                     slots.data_ptr(), None, at(kv), at(left))
    torch.cuda.synchronize()
    assert rc == 0
    assert (rows[:, :3].tolist(), mem[cu:cu + 3].tolist(), mem[pos:pos + T].tolist(), slots.tolist(), mem[kv:kv + 2].tolist(), int(mem[left])) == (
        want[0], want[1], want[2], want[3], want[5], want[6])
    assert mem[4:8].tolist() == lens + counts and mem[32:37].tolist() == free + [4]


# ------------------------------------------------------------------------------------------------ tree_attention
@pytest.mark.parametrize("step", [s for s in STEPS if len(s[1]) > 2], ids=lambda s: s[0])
def test_attention_of_a_part_of_a_batch(pkg, dev, step):
    """The last requests of a batch by slices of its tensors: the rows before theirs are rows of no request."""
    _, reqs, Hq, Hkv, D, page, fp8, as_tree = step
    say("tree_attention part of", step)
    s = Step(len(reqs) * 7 + Hq, reqs, Hq, Hkv, D, page, fp8, as_tree, spare_rows=3)
    a = s.args(dev)
    skip = len(reqs) - 2
    out = torch.full_like(a["q"], 7.0)
    out, lse = pkg.tree_attention(**{**a, "kv_lens": a["kv_lens"][skip:], "cu_tokens": a["cu_tokens"][skip:], "block_tables": a["block_tables"][skip:]},
                                  out=out, return_lse=True)
    s.tables, s.lens, first = s.tables[skip:], s.lens[skip:], s.cu[skip]
    s.cu = s.cu[skip:]
    s.check(out, lse)
    assert first > 0 and bool((out[:first] == 0).all()) and bool((lse[:first] == -math.inf).all())


def test_attention_of_no_request(pkg, dev):
    say("tree_attention of no request")
    for cached in (torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16, device=dev), torch.zeros(0, 16, 2, 64, dtype=torch.bfloat16, device=dev)):
        for first in (0, 2):
            out, lse = pkg.tree_attention(torch.ones(5, 4, 64, dtype=torch.bfloat16, device=dev), cached, cached, ints([], dev).view(0, 4), ints([], dev),
                                          ints([first], dev), out=torch.full((5, 4, 64), 7.0, dtype=torch.bfloat16, device=dev), return_lse=True)
            assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("rows,n,Hq,B", [(16, 64, 4, 70), (64, 64, 8, 8), (128, 64, 13, 8), (256, 64, 32, 8)])
@pytest.mark.parametrize("as_tree", [True, False])
def test_attention_ends_where_cu_tokens_descends(pkg, dev, as_tree, rows, n, Hq, B):
    """Every second request claims all rows: more work than the batch can have.  The results are undefined, but the call ends, writes inside
    its results only, and the next one is right."""
    say("tree_attention with descending cu_tokens", rows, n)
    s = with_room(Step(5, [(900, n)] + [(700, 0)] * (B - 1), Hq, 1, 64, 16, False, as_tree))
    a, T = s.args(dev), s.T
    mem = torch.full((T + 8, Hq, 64), 7.0, dtype=torch.bfloat16, device=dev)
    bad = ints([0, T] * B, dev)[:B + 1].contiguous()
    assert tile_rows(pkg, s) == rows
    pkg.tree_attention(**{**a, "cu_tokens": bad, "kv_lens": ints([ROOM] * B, dev)}, out=mem[4:4 + T])
    torch.cuda.synchronize()
    assert bool((mem[:4] == 7).all()) and bool((mem[4 + T:] == 7).all())
    s.check(*attend(pkg, dev, s, rows))


TILES = [(16, [(300, 1), (180, 2), (256, 1)], 8, 2), (64, [(300, 8)], 8, 1), (128, [(300, 16), (288, 16)], 8, 1), (256, [(300, 32)], 8, 1)]


def ramp(s, of_key):
    """Every value of request b's i-th key is of_key(i)."""
    page = s.k.shape[1]
    for b, l in enumerate(s.lens):
        for i in range(l):
            s.k[s.tables[b][i // page], i % page] = torch.tensor(float(of_key(i))).to(s.kind)


@pytest.mark.parametrize("rows,reqs,Hq,Hkv", TILES)
@pytest.mark.parametrize("slope", [0.3, -0.3])
@pytest.mark.parametrize("how", ["scale", "k_scale", "both"])
def test_attention_with_negative_scales(pkg, dev, how, slope, rows, reqs, Hq, Hkv):
    """Scores far apart, rising or falling along the keys."""
    say("tree_attention", how, "negative, slope", slope)
    s = Step(11, reqs, Hq, Hkv, 64, 16, how != "scale", True)
    s = with_room(s) if rows > 16 else s
    s.q[:] = 2
    ramp(s, lambda i: (i - 200) * slope)
    if how != "k_scale":
        s.scale = -s.scale
    if how != "scale":
        s.ks = -torch.linspace(0.7, 1.0, Hkv)
        s.vs = -s.vs
    s.check(*attend(pkg, dev, s, rows, scale=s.scale))


LONG = [(16, [(2600, 1), (2400, 2)], 8, 2), (64, [(2600, 8)], 8, 1), (128, [(2600, 16), (2300, 16)], 8, 1), (256, [(2600, 32)], 8, 1)]


@pytest.mark.parametrize("rows,reqs,Hq,Hkv", LONG)
@pytest.mark.parametrize("size,rise", [(1e25, 39.0), (1e30, 39.0), (1e30, 10.0), (2e34, 39.0), (2e34, 0.0)])
def test_attention_of_large_values(pkg, dev, size, rise, rows, reqs, Hq, Hkv):
    """Values near the type's largest, and keys here and there that outscore the ones before them by `rise`: the weighted mean is a
    number, and so is everything on the way to it while the values' size times the number of keys is one."""
    say("tree_attention of values around", size, "rise", rise)
    s = Step(12, reqs, Hq, Hkv, 64, 16, False, True)
    s = with_room(s) if rows > 16 else s
    s.v = (s.v.float() * size).to(torch.bfloat16)
    s.q[:] = 2
    ramp(s, lambda i: rise / 16 if i // 128 % 2 and i % 32 == 5 else 0)          # a score is 64 products, 2 k / 8 each
    out, lse = attend(pkg, dev, s, rows)
    assert bool(out.isfinite().all())
    s.check(out, lse)


# ------------------------------------------------------------------------------------------------ qk_norm_rope
@pytest.mark.parametrize("T,Hq,Hkv,D,R,pairs", [(5, 6, 2, 128, 64, True), (33, 8, 8, 96, 96, False), (613, 4, 3, 64, 64, False), (2049, 32, 4, 128, 128, False),
                                               (70, 3, 1, 256, 128, True)])
def test_norm_rope_of_many_tokens_without_a_cache(pkg, dev, T, Hq, Hkv, D, R, pairs):
    say("qk_norm_rope without a cache", T, Hq, Hkv, D)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16)
    pos = torch.randint(-1, 41, (T,), generator=g).to(torch.int32)               # -1 and 40: no such places
    cs, w = torch.randn(40, R, generator=g), [(1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16) for _ in range(2)]
    q, k = pkg.qk_norm_rope(x.to(dev), pos.to(dev), cs.to(dev), Hq, Hkv, w[0].to(dev), w[1].to(dev), 1e-5, pairs)
    heads = x.view(T, Hq + 2 * Hkv, D)
    check_rows(q, plain.norm_rope(heads[:, :Hq], w[0], 1e-5, pos, cs, pairs), "q")
    check_rows(k, plain.norm_rope(heads[:, Hq:Hq + Hkv], w[1], 1e-5, pos, cs, pairs), "k")


# ------------------------------------------------------------------------------------------------ the registered ops
def test_schemas_say_what_is_written_and_shared(pkg, dev):
    """torch's own check of a schema: which arguments are written, and which results share memory with them or each other."""
    from torch.library import opcheck
    ops = torch.ops.my_ops
    check = lambda op, args, kwargs=None: opcheck(op.default, args, kwargs or {}, test_utils="test_schema")
    s = Step(21, [(60, 9), (7, 3)], 8, 2, 128, 16, False, True)
    a = s.args(dev)
    del a["k_scale"], a["v_scale"]
    check(ops.tree_attention, (), a)
    check(ops.tree_attention, (), {**a, "out": torch.zeros_like(a["q"]), "return_lse": True})
    for parents in (None, ints([-1, 0, 0, -1, 0], dev)):
        check(ops.cache_plan, (ints([[3, -1], [1, -1]], dev), ints([5, 2], dev), ints([3, 2], dev), ints([0, 2], dev), ints([2], dev), 4, 5, parents))
    x = torch.randn(3, 8 * 64, device=dev).to(torch.bfloat16)
    rope = (x, ints([0, 1, 2], dev), torch.randn(8, 64, device=dev), 4, 2)
    check(ops.qk_norm_rope, rope)
    k, v = (torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device=dev) for _ in range(2))
    check(ops.qk_norm_rope, rope, dict(k_cache=k, v_cache=v, slots=ints([0, 1, 2], dev, torch.int64), out=torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=dev)))
    check(ops.token_logprobs, (torch.randn(3, 50, device=dev), ints([1, 2, 3], dev, torch.int64), 4, 1.0))


def test_results_of_inputs_with_gradients_warn_in_backward(pkg, dev):
    """The operators have no gradient: a backward pass through them says so instead of going past them silently."""
    s = Step(21, [(60, 9), (7, 3)], 8, 2, 128, 16, False, True)
    a = s.args(dev)
    a["q"].requires_grad_()
    w = torch.ones(64, device=dev, requires_grad=True)
    x = torch.randn(3, 8 * 64, device=dev).to(torch.bfloat16)
    results = [pkg.tree_attention(**a), pkg.tree_attention(**a, out=torch.zeros_like(a["q"])),
               *pkg.qk_norm_rope(x, ints([0, 1, 2], dev), torch.randn(8, 64, device=dev), 4, 2, w, w),
               pkg.token_logprobs(torch.randn(3, 50, device=dev, requires_grad=True), ints([1, 2, 3], dev, torch.int64)).logprobs]
    for r in results:
        assert r.requires_grad
        with pytest.warns(UserWarning, match="autograd kernel was not registered"):
            r.sum().backward()
