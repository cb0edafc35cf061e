"""The serving step's operators on the GPU against their plain 64-bit forms, at the sizes and masks where they can go wrong."""
import math
import random

import pytest
import torch

import serving_plain as plain

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def ints(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


def tree(rng, n, root=0.1):
    return [-1 if j == 0 or rng.random() < root else max(0, j - 1 - int(rng.expovariate(0.7))) for j in range(n)]


# ------------------------------------------------------------------------------------------------ cache_plan
def run_plan(pkg, dev, tables, lens, counts, free, n_free, page, T, parents):
    say("cache_plan", len(lens), "requests, page", page, "rows", T, "tree" if parents is not None else "chain")
    W = len(tables[0]) if tables else 4
    wide = torch.full((len(lens), W + 3), -7, dtype=torch.int32, device=dev)       # rows of a wider table
    view = wide[:, :W]
    if tables:
        view.copy_(ints(tables, dev))
    left = ints([n_free], dev)
    p = pkg.cache_plan(view, ints(lens, dev), ints(counts, dev), ints(free, dev), left, page, T,
                       None if parents is None else ints(parents, dev))
    torch.cuda.synchronize()
    want = plain.plan(tables, lens, counts, free, n_free, page, T, parents)
    assert view.tolist() == want[0]
    assert bool((wide[:, W:] == -7).all()) and left.item() == n_free
    for got, ref in zip((p.cu_tokens, p.positions, p.slots, p.masks, p.kv_lens), want[1:6]):
        assert (got is None and ref is None) or got.tolist() == ref
    assert p.n_free.tolist() == [want[6]]


def pool(rng, B, W, page, lens):
    ids = list(range(B * W))
    rng.shuffle(ids)
    tables = []
    for b in range(B):
        have = -(-max(lens[b], 0) // page)
        tables.append([ids.pop() for _ in range(min(have, W))] + [-1] * (W - min(have, W)))
    return tables, ids


@pytest.mark.parametrize("B,most,page,as_tree", [(1, 1, 1, False), (1, 64, 64, True), (3, 5, 4, True), (17, 64, 16, True), (64, 1, 128, False),
                                                (65, 3, 1024, True), (5, 300, 8, False), (257, 9, 2, True), (1025, 2, 32, True), (4096, 3, 16, False)])
def test_plan_equals_the_plain_form(pkg, dev, B, most, page, as_tree):
    rng = random.Random(B * 1000 + most)
    counts = [rng.randint(0, most) for _ in range(B)]
    counts[rng.randrange(B)] = most
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, 5 * page)]) for _ in range(B)]
    W = -(-(5 * page + page + most) // page) + 1
    tables, free = pool(rng, B, W, page, lens)
    T = sum(counts) + rng.choice([0, 0, 7, 700])
    parents = [p for n in counts for p in tree(rng, n)] + [5] * (T - sum(counts)) if as_tree else None
    run_plan(pkg, dev, tables, lens, counts, free, len(free), page, T, parents)


@pytest.mark.parametrize("as_tree", [False, True])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.9])
def test_plan_refuses_what_does_not_fit(pkg, dev, as_tree, share):
    rng = random.Random(int(share * 10) + as_tree)
    B, page, W = 80, 8, 12
    lens = [rng.choice([0, 5, 8, 40, 90, 96, 95, -3]) for _ in range(B)]
    counts = [rng.choice([0, 1, 3, 17, 64, -5]) for _ in range(B)]
    tables, free = pool(rng, B, W, page, lens)
    total = sum(max(n, 0) for n in counts)
    need = sum(-(-(l + max(n, 0)) // page) - -(-l // page) for l, n in zip(lens, counts) if 0 <= l and l + max(n, 0) <= W * page)
    for T in (total, max(total - 30, 0)):
        parents = ([p for n in counts for p in tree(rng, max(n, 0))])[:T] if as_tree else None
        run_plan(pkg, dev, tables, lens, counts, free, int(need * share), page, T, parents)
        run_plan(pkg, dev, tables, lens, counts, free, int(need * share) - 100000, page, T, parents)
        run_plan(pkg, dev, tables, lens, counts, free[:int(need * share)], 1 << 30, page, T, parents)


def test_plan_of_strange_trees_and_no_requests(pkg, dev):
    # parents that do not come before their children count as none; a tree of 65 is refused, its neighbours are not
    counts = [4, 65, 2]
    parents = [0, 1, 70, -9] + list(range(-1, 64)) + [1, 0]
    run_plan(pkg, dev, [[3, -1, -1, -1, -1]] * 3, [2, 3, 1], counts, [9, 8, 7, 6, 5, 4, 2, 1, 0], 9, 16, 71, parents)
    p = pkg.cache_plan(torch.empty(0, 4, dtype=torch.int32, device=dev), ints([], dev), ints([], dev), ints([1, 2], dev), ints([2], dev), 16, 5)
    assert p.cu_tokens.tolist() == [0] and p.positions.tolist() == [-1] * 5 and p.n_free.tolist() == [2]
    p = pkg.cache_plan(ints([[1]], dev), ints([1], dev), ints([0], dev), ints([], dev), ints([0], dev), 16, 0, parents=ints([], dev))
    assert p.cu_tokens.tolist() == [0, 0] and p.kv_lens.tolist() == [1]


# ------------------------------------------------------------------------------------------------ qk_norm_rope
def check_rows(got, want, what):
    """bf16 of what 64 bits give: one rounding, and fp32's on the way (relative to the head's largest, for the rotation's difference)."""
    bound = plain.U16 * want.abs() + 64 * plain.U32 * want.abs().amax(-1, keepdim=True) + 1e-30
    off = (got.double().cpu() - want).abs()
    assert bool((off <= bound).all()), f"{what}: {float((off / bound).max())} of the bound"


@pytest.mark.parametrize("T,Hq,Hkv,D,R,pairs,cache,weights", [
    (1, 1, 1, 64, 64, False, None, "both"), (1, 32, 4, 128, 128, False, "bf16", "both"), (5, 6, 2, 128, 64, True, "fp8", "both"),
    (33, 8, 8, 96, 96, False, "bf16", "q"), (7, 10, 2, 256, 256, True, "fp8", "f32"), (64, 3, 1, 256, 128, False, "bf16", None),
    (19, 4, 2, 8, 0, False, "bf16", "both"), (300, 5, 1, 80, 32, False, "fp8", "k"), (3, 64, 8, 192, 176, False, "bf16", "f32"),
    (1030, 12, 4, 64, 64, False, "fp8", "both"), (2049, 4, 1, 128, 128, True, "bf16", "both"), (0, 4, 1, 128, 128, False, "bf16", "both")])
def test_norm_rope_equals_the_plain_form(pkg, dev, T, Hq, Hkv, D, R, pairs, cache, weights):
    say("qk_norm_rope", T, Hq, Hkv, D, R, pairs, cache, weights)
    g = torch.Generator().manual_seed(T * 31 + D)
    rng = random.Random(T + D)
    width, page, P = (Hq + 2 * Hkv) * D, rng.choice([1, 8, 64]), 700
    rows = torch.randn(T, width + 16, generator=g).to(torch.bfloat16)
    rows[:, ::7] *= 30
    big = rows.to(dev)
    qkv = big[:, 8:8 + width] if T > 1 else rows[:, :width].contiguous().to(dev)
    src = qkv.cpu().view(T, Hq + 2 * Hkv, D) if T else torch.zeros(0, Hq + 2 * Hkv, D)
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32)
    if T > 4:
        pos[1], pos[3] = -1, P                         # no such places
    cs = torch.randn(P, R, generator=g)
    wt = lambda: (1 + 0.3 * torch.randn(D, generator=g)).to(torch.float32 if weights == "f32" else torch.bfloat16)
    qw = wt() if weights in ("both", "q", "f32") else None
    kw = wt() if weights in ("both", "k", "f32") else None
    to = lambda t: None if t is None else t.to(dev)
    want_q = plain.norm_rope(src[:, :Hq], qw, 1e-5, pos, cs, pairs)
    want_k = plain.norm_rope(src[:, Hq:Hq + Hkv], kw, 1e-5, pos, cs, pairs)
    args = (qkv, pos.to(dev), cs.to(dev), Hq, Hkv, to(qw), to(kw), 1e-5, pairs)
    if cache is None:
        q, k = pkg.qk_norm_rope(*args)
        torch.cuda.synchronize()
        check_rows(q, want_q, "q")
        check_rows(k, want_k, "k")
        return
    n_blocks = -(-T // page) + 3
    kind = torch.float8_e4m3fn if cache == "fp8" else torch.bfloat16
    both = torch.randn(n_blocks, 2, page, Hkv, D, generator=g).to(kind)             # K and V of a block side by side
    both_dev = both.to(dev)
    slots = torch.randperm(n_blocks * page, generator=g)[:T]
    if T > 4:
        slots[0], slots[2] = -1, n_blocks * page
    scale = (lambda: 0.1 + torch.rand(Hkv, generator=g)) if cache == "fp8" else (lambda: None)
    ks, vs = scale(), scale()
    out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16, device=dev)
    q = pkg.qk_norm_rope(*args, k_cache=both_dev[:, 0], v_cache=both_dev[:, 1], slots=slots.to(dev), k_scale=to(ks), v_scale=to(vs), out=out)
    torch.cuda.synchronize()
    assert q.data_ptr() == out.data_ptr()
    check_rows(q, want_q, "q")
    got = both_dev.cpu()
    held = both.float().transpose(1, 2).reshape(n_blocks * page, 2, Hkv, D)
    new = got.float().transpose(1, 2).reshape(n_blocks * page, 2, Hkv, D)
    here = [t for t in range(T) if 0 <= int(slots[t]) < n_blocks * page and 0 <= int(pos[t]) < P]
    untouched = torch.ones(n_blocks * page, dtype=torch.bool)
    untouched[slots[here]] = False
    assert torch.equal(new[untouched].nan_to_num(9), held[untouched].nan_to_num(9)) if untouched.any() else True
    if not here:
        return
    k, v = new[slots[here], 0], new[slots[here], 1]
    if cache == "bf16":
        check_rows(k, want_k[here], "k")
        assert torch.equal(v, src[here, Hq + Hkv:].float())
        return
    for got8, want8, sc, what in ((k, want_k[here], ks, "k"), (v, src[here, Hq + Hkv:].double(), vs, "v")):
        w = (want8 / sc.double()[None, :, None]).clamp(-448, 448)
        # e4m3: half a unit of 4 digits, or of its smallest step 2^-9; and fp32's errors before it
        bound = 2.0 ** -4 * w.abs() + 2.0 ** -10 + 64 * plain.U32 * w.abs().amax(-1, keepdim=True)
        off = (got8.double() - w).abs()
        assert bool((off <= bound).all()), f"{what}: {float((off / bound).max())} of the bound"


def test_norm_rope_of_values_that_are_no_numbers(pkg, dev):
    """A NaN or infinity stays in its own head; e4m3 keeps a NaN and cuts an infinity to its largest value."""
    say("qk_norm_rope: NaN, inf")
    T, Hq, Hkv, D = 3, 2, 1, 64
    x = torch.randn(T, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    x[0, 5] = math.nan
    x[1, 3 * D + 7] = math.inf                           # a value
    x[1, 3 * D + 8] = math.nan
    cs = torch.randn(8, D, generator=torch.Generator().manual_seed(2))
    k = torch.zeros(1, 4, 1, D, dtype=torch.float8_e4m3fn, device=dev)
    v = torch.zeros_like(k)
    q = pkg.qk_norm_rope(x.to(dev), ints([0, 1, 2], dev), cs.to(dev), Hq, Hkv, torch.ones(D, device=dev, dtype=torch.bfloat16),
                         torch.ones(D, device=dev, dtype=torch.bfloat16), k_cache=k, v_cache=v, slots=ints([0, 1, 2], dev, torch.int64))
    q, v = q.float().cpu(), v.float().cpu()[0, :, 0]
    assert bool(q[0, 0].isnan().all()) and bool(q[0, 1].isfinite().all()) and bool(q[1:].isfinite().all())
    assert v[1, 7] == 448 and v[1, 8].isnan() and int(v.isfinite().sum()) == 4 * D - 1


# ------------------------------------------------------------------------------------------------ tree_attention
class Step:
    """One step's tensors: random caches, tables with unused entries -1, trees or chains."""

    def __init__(self, seed, reqs, Hq, Hkv, D, page, fp8, as_tree, spare_rows=0, q_scale=1.0):
        g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        self.counts, self.lens = [n for _, n in reqs], [l + n if l >= 0 else 0 for l, n in reqs]
        pages = [-(-l // page) for l in self.lens]
        n_blocks = sum(pages) + 2
        ids = list(range(n_blocks))
        rng.shuffle(ids)
        W = max(pages + [0]) + 2
        self.tables = [[ids.pop() for _ in range(p)] + [-1] * (W - p) for p in pages]
        self.kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
        up = 30.0 if fp8 else 1.0
        self.k = (torch.randn(n_blocks, page, Hkv, D, generator=g) * up).to(self.kind)
        self.v = ((torch.randn(n_blocks, page, Hkv, D, generator=g) + 0.5) * up).to(self.kind)
        self.ks = (0.8 + 0.4 * torch.rand(Hkv, generator=g)) / up if fp8 else None
        self.vs = (0.8 + 0.4 * torch.rand(Hkv, generator=g)) / up if fp8 else None
        self.cu = [0]
        for n in self.counts:
            self.cu.append(self.cu[-1] + n)
        self.T = self.cu[-1] + spare_rows
        self.q = (torch.randn(self.T, Hq, D, generator=g) * q_scale).to(torch.bfloat16)
        self.masks = None
        if as_tree:
            self.masks = []
            for n in self.counts:
                seen = []
                for j, p in enumerate(tree(rng, n)):
                    seen.append((1 << j) | (seen[p] if p >= 0 else 0))
                self.masks += seen
            self.masks = [m - (1 << 64) if m >> 63 else m for m in self.masks] + [-1] * spare_rows
        self.scale = D ** -0.5

    def args(self, dev, **other):
        to = lambda t: None if t is None else t.to(dev)
        v = dict(q=to(self.q), k_cache=to(self.k), v_cache=to(self.v), block_tables=ints(self.tables, dev), kv_lens=ints(self.lens, dev),
                 cu_tokens=ints(self.cu, dev), masks=None if self.masks is None else ints(self.masks, dev, torch.int64),
                 k_scale=to(self.ks), v_scale=to(self.vs))
        return {**v, **other}

    def check(self, out, lse):
        ref, ref_lse, reach = plain.attention(self.q, self.k.float(), self.v.float(), self.tables, self.lens, self.cu, self.masks, self.scale,
                                              self.ks, self.vs)
        got, bound = out.double().cpu(), plain.attention_bound(ref, reach)
        # where a visible value is no number the result is none either
        there = reach.isfinite()
        off = (got - ref).abs()
        assert bool((off <= bound)[there].all()), f"out: {float((off / bound)[there].max())} of the bound"
        assert bool((~got.isfinite() == ~there).all())
        if lse is not None:
            lse, none = lse.double().cpu(), ref_lse == -math.inf
            assert bool((lse[none] == -math.inf).all()) and bool((got[none] == 0).all())
            fin = ref_lse.isfinite()
            assert bool(((lse - ref_lse).abs()[fin] <= 2e-4 + 1e-5 * ref_lse.abs()[fin]).all())


STEPS = [
    # reqs (cached, new), Hq, Hkv, D, page, fp8, tree
    ("one token, one key", [(0, 1)], 1, 1, 64, 16, False, False),
    ("one token over a few pages", [(100, 1)], 8, 1, 128, 16, False, False),
    ("lengths around the tiles", [(n, 1) for n in (0, 1, 15, 16, 17, 30, 31, 32, 33, 62, 63, 64, 65, 126, 127, 128, 129, 255, 256)], 4, 2, 128, 16, False, False),
    ("the same, 8 bits, narrow heads", [(n, 1) for n in (0, 1, 15, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257)], 5, 1, 64, 8, True, False),
    ("pages of one key", [(37, 3), (5, 2)], 4, 4, 64, 1, False, True),
    ("a page larger than all", [(200, 5), (3, 1)], 16, 1, 128, 1024, False, True),
    ("trees", [(50, 16), (0, 7), (129, 64), (64, 1), (10, 0), (31, 33)], 8, 2, 128, 32, False, True),
    ("trees, 8 bits", [(50, 16), (0, 7), (129, 64), (64, 1), (10, 0), (31, 33)], 6, 2, 128, 32, True, True),
    ("trees of many heads a key", [(70, 64), (33, 20)], 16, 1, 64, 16, False, True),
    ("chains", [(0, 70), (33, 1), (100, 65), (5, 0)], 3, 3, 128, 16, False, False),
    ("a prompt from its start", [(0, 300)], 8, 2, 64, 64, False, False),
    ("a chunk, 8 bits", [(90, 150), (0, 20)], 8, 1, 128, 64, True, False),
    ("refused and empty requests", [(-1, 5), (40, 3), (-1, 1), (0, 0), (7, 2)], 4, 2, 128, 16, False, True),
]


@pytest.mark.parametrize("step", STEPS, ids=[s[0] for s in STEPS])
def test_attention_equals_the_plain_form(pkg, dev, step):
    say("tree_attention", step)
    _, reqs, Hq, Hkv, D, page, fp8, as_tree = step
    s = Step(len(reqs) * 7 + Hq, reqs, Hq, Hkv, D, page, fp8, as_tree, spare_rows=3)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)
    again = pkg.tree_attention(**s.args(dev))
    assert torch.equal(out, again)                       # the same inputs, the same bits


@pytest.mark.parametrize("B,L,n,Hq,Hkv,D,fp8", [(1, 5000, 1, 4, 1, 128, False), (2, 3000, 9, 4, 1, 128, True), (1, 2100, 40, 8, 1, 64, False),
                                               (3, 1500, 64, 4, 1, 128, False)])
def test_attention_over_long_caches(pkg, dev, B, L, n, Hq, Hkv, D, fp8):
    """Caches long enough to be cut over the chip and joined."""
    say("tree_attention long", B, L, n)
    s = Step(L, [(L - 111 * b, max(1, n - 3 * b)) for b in range(B)], Hq, Hkv, D, 64, fp8, True)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_attention_of_flat_and_of_sharp_rows(pkg, dev, size):
    say("tree_attention scores of size", size)
    s = Step(5, [(200, 20), (700, 3)], 4, 2, 128, 16, False, True, q_scale=size)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    ref, ref_lse, reach = plain.attention(s.q, s.k.float(), s.v.float(), s.tables, s.lens, s.cu, s.masks, s.scale)
    # scores of up to a few hundred: fp32 sums of 128 products leave them 128 roundings of their terms' size off
    slack = 128 * plain.U32 * 128 * float(s.q.abs().max()) * float(s.k.abs().max()) * s.scale
    off = (out.double().cpu() - ref).abs()
    assert bool((off <= plain.attention_bound(ref, reach) + slack * reach * 2).all())


def test_attention_growing_scores(pkg, dev):
    """Every key outscores the ones before it by far: the running maximum moves all the time."""
    say("tree_attention growing scores")
    s = Step(11, [(300, 4)], 4, 1, 64, 16, False, True)
    q, at = torch.ones(64) * 2, torch.zeros(304, 64)
    for i in range(304):
        at[i] = (i - 200) * 0.05
    for i in range(304):
        s.k[s.tables[0][i // 16], i % 16, 0] = at[i].to(torch.bfloat16)
    s.q[:] = q.to(torch.bfloat16)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)


UNSEEN = [([(40, 12), (0, 3), (130, 1)], 4, 2, False), ([(70, 64)], 16, 2, False), ([(61, 33), (7, 5)], 8, 1, True)]


@pytest.mark.parametrize("reqs,Hq,Hkv,fp8,what", [(*u, w) for u in UNSEEN for w in (math.nan, math.inf, -math.inf)
                                                  if not (u[3] and math.isinf(w))])      # (e4m3 has no infinity)
def test_attention_ignores_what_a_row_does_not_see(pkg, dev, what, reqs, Hq, Hkv, fp8):
    """NaN and infinities behind the end of a request, in pages of no request, and in drafted tokens that other branches see."""
    say("tree_attention", what, reqs)
    s = Step(3, reqs, Hq, Hkv, 128, 16, fp8, True)
    held = set()
    for b, l in enumerate(s.lens):
        for i in range(l):
            held.add((s.tables[b][i // 16], i % 16))
    for blk in range(s.k.shape[0]):
        for i in range(16):
            if (blk, i) not in held:
                s.k[blk, i] = torch.tensor(what).to(s.kind)
                s.v[blk, i] = torch.tensor(what).to(s.kind)
    # the second drafted token of the first request: the rows that do not see it stay numbers
    at = s.lens[0] - s.counts[0] + 1
    s.v[s.tables[0][at // 16], at % 16, 0, 5:9] = torch.tensor(what).to(s.kind)
    if what != what:
        s.k[s.tables[0][at // 16], at % 16, Hkv - 1, 3] = torch.tensor(what).to(s.kind)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    got = out.double().cpu()
    ref, _, reach = plain.attention(s.q, s.k.float(), s.v.float(), s.tables, s.lens, s.cu, s.masks, s.scale, s.ks, s.vs)
    there = reach.isfinite()
    off = (got - ref).abs()
    assert bool((off <= plain.attention_bound(ref, reach))[there].all())
    assert int((~there).sum()) > 0 and bool((~got.isfinite())[~there].all())


def test_attention_masks_that_leave_nothing(pkg, dev):
    say("tree_attention empty rows")
    s = Step(9, [(0, 6), (0, 64), (20, 3)], 4, 2, 64, 16, False, True)
    for j in (0, 3, 6 + 63, 6 + 10):
        s.masks[j] = 0
    s.masks[70] = 0                                      # sees the cached keys all the same
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)
    assert bool((lse[[0, 3, 69, 16]] == -math.inf).all()) and bool((out[[0, 3, 69, 16]] == 0).all()) and bool(lse[70].isfinite().all())


def test_attention_strides_streams_and_graphs(pkg, dev):
    say("tree_attention strides, streams, graphs")
    s = Step(21, [(300, 9), (77, 16), (0, 1)], 8, 2, 128, 16, False, True)
    want = pkg.tree_attention(**s.args(dev))
    # queries inside a projection's rows, K and V of a block side by side, tables of a wider matrix
    wide = torch.randn(s.T, 8 * 128 + 64, device=dev).to(torch.bfloat16)
    wide[:, 32:32 + 1024] = s.q.view(s.T, -1).to(dev)
    both = torch.stack([s.k, s.v], 1).to(dev)
    tables = torch.full((3, 90), 3, dtype=torch.int32, device=dev)
    tables[:, :len(s.tables[0])] = ints(s.tables, dev)
    a = s.args(dev, q=wide[:, 32:32 + 1024].view(s.T, 8, 128), k_cache=both[:, 0], v_cache=both[:, 1], block_tables=tables[:, :80])
    assert torch.equal(pkg.tree_attention(**a), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.tree_attention(**a)
    side.synchronize()
    assert torch.equal(got, want)
    # a captured step follows the lengths and tables that the buffers hold at replay
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.tree_attention(**a, out=out)
    for lens in ([309, 93, 1], [200, 16, 1], [309, 40, 0], [309, 93, 1]):
        a["kv_lens"].copy_(ints(lens, dev))
        eager = pkg.tree_attention(**a)
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens


def test_attention_offsets_beyond_32_bits(pkg, dev):
    """A cache of more than 2^32 bytes, the request's pages at its end."""
    say("tree_attention large cache")
    s = Step(4, [(130, 5)], 4, 2, 128, 64, False, True)
    n_blocks = (1 << 32) // (64 * 2 * 128 * 2) + 40
    k = torch.empty(n_blocks, 64, 2, 128, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    old = [t for t in s.tables[0] if t >= 0]
    new = [n_blocks - 1 - 3 * i for i in range(len(old))]
    for o, n in zip(old, new):
        k[n], v[n] = s.k[o].to(dev), s.v[o].to(dev)
    table = new + [-1] * (len(s.tables[0]) - len(new))
    out, lse = pkg.tree_attention(**s.args(dev, k_cache=k, v_cache=v, block_tables=ints([table], dev)), return_lse=True)
    s.check(out, lse)
    # and what goes into it
    x = torch.randn(2, 8 * 128, device=dev).to(torch.bfloat16)
    slots = ints([n_blocks * 64 - 1, n_blocks * 64 - 64 * 7], dev, torch.int64)
    cs = torch.randn(4, 128, device=dev)
    pkg.qk_norm_rope(x, ints([1, 2], dev), cs, 4, 2, k_cache=k, v_cache=v, slots=slots)
    assert torch.equal(v[n_blocks - 1, 63], x[0].view(8, 128)[6:]) and torch.equal(v[n_blocks - 7, 0], x[1].view(8, 128)[6:])


# ------------------------------------------------------------------------------------------------ token_logprobs
def check_logprobs(pkg, dev, logits, tokens, k, temp, on_dev=None):
    said = pkg.token_logprobs(logits.to(dev) if on_dev is None else on_dev, tokens.to(dev), top_k=k, temperature=temp)
    torch.cuda.synchronize()
    lp, ent, tops, ids = plain.logprobs(logits.float(), tokens, k, temp)
    off, off_ent = plain.logprobs_bound(logits.shape[1], temp, logits.float())
    close = lambda a, b, most: bool(torch.where(b.isfinite(), (a.double().cpu() - b).abs() <= most * (1 + b.abs().nan_to_num(0, 0, 0)), a.double().cpu() == b).all())
    assert said.top_ids.cpu().tolist() == ids.tolist()
    assert close(said.logprobs, lp, off) and close(said.top_logprobs, tops, off) and close(said.entropy, ent, off_ent)


@pytest.mark.parametrize("T,V,k,bf16,temp", [(1, 1, 1, True, 1.0), (1, 7, 7, False, 0.5), (3, 33, 32, True, 1.0), (2, 2047, 5, True, 2.0), (1, 2048, 0, False, 1.0),
                                             (5, 2049, 20, True, 0.7), (1, 50001, 32, True, 1.0), (4, 16383, 8, False, 1.0), (1, 131072, 20, True, 1.0),
                                             (1, 131071, 3, False, 1.3), (1100, 517, 4, True, 1.0), (1030, 3001, 1, False, 0.9), (0, 100, 3, True, 1.0)])
def test_logprobs_equal_the_plain_form(pkg, dev, T, V, k, bf16, temp):
    say("token_logprobs", T, V, k, bf16, temp)
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(T, V, generator=g) * 3).to(torch.bfloat16 if bf16 else torch.float32)
    tokens = torch.randint(0, V, (T,), generator=g)
    if T > 2:
        tokens[1], tokens[2] = -1, V
    check_logprobs(pkg, dev, logits, tokens, k, temp)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("make", ["same", "up", "down", "two values", "signed zeros", "blocks", "masked", "almost all masked"])
@pytest.mark.parametrize("T,V", [(2, 20011), (1025, 9001)])
def test_logprobs_of_ties_order_and_masks(pkg, dev, make, bf16, T, V):
    say("token_logprobs", make, bf16, T, V)
    g = torch.Generator().manual_seed(5)
    row = {"same": lambda: torch.full((V,), 1.5), "up": lambda: torch.arange(V) * 0.001, "down": lambda: -torch.arange(V) * 0.001,
           "two values": lambda: (torch.rand(V, generator=g) < 0.5).float(), "signed zeros": lambda: torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0),
           "blocks": lambda: (torch.arange(V) // 256 % 3).float(), "masked": lambda: torch.where(torch.rand(V, generator=g) < 0.95, -math.inf, torch.randn(V, generator=g)),
           "almost all masked": lambda: torch.full((V,), -math.inf)}[make]()
    if make == "almost all masked":
        row[V // 2], row[V - 1] = 0.5, 0.5
    rows = row.to(torch.bfloat16 if bf16 else torch.float32)
    few = 2 if T < 10 else T
    logits = rows[None].expand(few, V).contiguous()
    tokens = torch.full((few,), V - 1)
    said = pkg.token_logprobs(logits.to(dev), tokens.to(dev), top_k=20)
    for t in sorted({0, few - 1}):
        lp, ent, tops, ids = plain.logprobs(logits[t:t + 1].float(), tokens[t:t + 1], 20, 1.0)
        off, off_ent = plain.logprobs_bound(V, 1.0, logits[t:t + 1].float())
        assert said.top_ids[t].tolist() == ids[0].tolist()
        fin = tops[0].isfinite()
        got = said.top_logprobs[t].double().cpu()
        assert bool(((got - tops[0]).abs()[fin] <= off * (1 + tops[0].abs()[fin])).all()) and bool((got[~fin] == -math.inf).all())
        assert abs(float(said.entropy[t]) - float(ent)) <= off_ent * (1 + float(ent))
        assert float(said.logprobs[t]) == float(lp) or abs(float(said.logprobs[t]) - float(lp)) <= off * (1 + abs(float(lp)))
    assert bool((said.top_ids == said.top_ids[:1]).all())


def test_logprobs_of_rows_that_are_no_distribution(pkg, dev):
    say("token_logprobs NaN, inf, nothing")
    for T, V in ((6, 40000), (1500, 1001)):
        logits = torch.randn(T, V, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        logits[0] = -math.inf
        logits[1, V - 3] = math.nan
        logits[2, 5] = math.inf
        logits[3] = math.nan
        logits[4] = -3.38e38                             # the type's lowest, as a mask
        logits[4, 9] = 1.0
        said = pkg.token_logprobs(logits.to(dev), torch.full((T,), 9, device=dev), top_k=4)
        assert said.logprobs[0] == -math.inf and said.entropy[0] == 0 and said.top_ids[0].tolist() == [0, 1, 2, 3]
        assert bool((said.top_logprobs[0] == -math.inf).all())
        for t in (1, 2, 3):
            assert bool(said.logprobs[t].isnan()) and bool(said.entropy[t].isnan()) and bool(said.top_logprobs[t].isnan().all())
        assert bool(((said.top_ids[:4] >= -1) & (said.top_ids[:4] < V)).all()) and said.top_ids[3].tolist() == [-1] * 4 and said.top_ids[2, 0] == 5
        assert said.logprobs[4] == 0 and said.entropy[4] == 0 and said.top_ids[4].tolist() == [9, 0, 1, 2]
        assert bool(said.logprobs[5:].isfinite().all())


def test_logprobs_strides_and_graphs(pkg, dev):
    say("token_logprobs strides, graphs")
    g = torch.Generator().manual_seed(8)
    wide = torch.randn(5, 70003, generator=g)
    for kind in (torch.bfloat16, torch.float32):
        big = wide.to(kind).to(dev)
        for lo, hi in ((0, 70003), (1, 70000), (3, 50000), (8, 1000), (5, 12)):
            check_logprobs(pkg, dev, wide.to(kind)[:, lo:hi].contiguous(), torch.arange(5), min(6, hi - lo), 1.0, on_dev=big[:, lo:hi])
    x = torch.randn(3, 60000, device=dev)
    tokens = torch.tensor([1, 2, 3], device=dev)
    pkg.token_logprobs(x, tokens, 5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = pkg.token_logprobs(x, tokens, 5)
    for i in range(4):
        x.normal_()
        eager = pkg.token_logprobs(x, tokens, 5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), i
