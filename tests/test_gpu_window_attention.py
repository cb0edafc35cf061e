"""tree_attention with a window and first tokens, and over caches in 4 bits, and qk_norm_rope's way into such caches, on the GPU against
their plain 64-bit forms."""
import math

import pytest
import torch

import serving_plain as plain
import window_plain as window
from test_gpu_serving import Step as Bf16OrFp8Step, ints, say

pytestmark = pytest.mark.gpu
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


class Step(Bf16OrFp8Step):
    """Like its base, with a cache type "bf16", "fp8" or "fp4", and a window."""

    def __init__(self, seed, reqs, Hq, Hkv, D, page, cache, as_tree, W=None, sinks=0, spare_rows=0, q_scale=1.0):
        super().__init__(seed, reqs, Hq, Hkv, D, page, cache == "fp8", as_tree, spare_rows, q_scale)
        self.cache, self.window = cache, dict(window=W, sinks=sinks)
        if cache == "fp4":
            g = torch.Generator().manual_seed(seed + 1)
            for name in ("k", "v"):
                x = getattr(self, name).double() * torch.exp2(torch.randint(-2, 3, (*self.k.shape[:3], 1), generator=g))
                codes, powers = window.encode(x)
                setattr(self, name, codes)
                setattr(self, name + "s", powers)

    def held(self):
        """Keys and values that the caches stand for, float64."""
        if self.cache == "fp4":
            return window.decode(self.k, self.ks), window.decode(self.v, self.vs)
        one = lambda t, s: t.double() * (1.0 if s is None else s.double()[:, None])
        return one(self.k, self.ks), one(self.v, self.vs)

    def args(self, dev, **other):
        v = super().args(dev, **self.window)
        if self.cache == "fp4":
            v.update(k_cache=v["k_cache"].view(FP4), v_cache=v["v_cache"].view(FP4), k_scale=v["k_scale"].view(E8M0), v_scale=v["v_scale"].view(E8M0))
        return {**v, **other}

    def want(self):
        masks = None if self.masks is None else [m & ((1 << 64) - 1) for m in self.masks]
        return window.attention(self.q, *self.held(), self.tables, self.lens, self.cu, masks, self.scale, self.window["window"], self.window["sinks"])

    def check(self, out, lse):
        ref, ref_lse, reach = self.want()
        got, bound = out.double().cpu(), plain.attention_bound(ref, reach)
        there = reach.isfinite()
        off = (got - ref).abs()
        assert bool((off <= bound)[there].all()), f"out: {float((off / bound)[there].max())} of the bound"
        assert bool((~got.isfinite() == ~there).all())
        if lse is not None:
            lse, none = lse.double().cpu(), ref_lse == -math.inf
            assert bool((lse[none] == -math.inf).all()) and bool((got[none] == 0).all())
            fin = ref_lse.isfinite()
            assert bool(((lse - ref_lse).abs()[fin] <= 2e-4 + 1e-5 * ref_lse.abs()[fin]).all())

    def rows(self, pkg):
        (T, Hq, _), (_, page, Hkv, _) = self.q.shape, self.k.shape
        return pkg._lib.lib.moe_window_attention_tile_rows(T, Hq, Hkv, len(self.lens), {"bf16": 1, "fp8": 2, "fp4": 3}[self.cache], self.masks is not None,
                                                           len(self.tables[0]), page, min(self.window["window"] or 0, 2 ** 31 - 1), self.window["sinks"])


AROUND = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 641]
TREES = [(50, 16), (0, 7), (129, 64), (64, 1), (10, 0), (31, 33), (300, 9)]
FOUR = [
    # reqs (cached, new), Hq, Hkv, D, page, tree
    ("one token, one key", [(0, 1)], 1, 1, 64, 16, False),
    ("lengths around the tiles", [(n, 1) for n in AROUND], 4, 2, 128, 16, False),
    ("the same, narrow heads", [(n, 1) for n in AROUND], 5, 1, 64, 8, False),
    ("pages of one key", [(37, 3), (5, 2)], 4, 4, 64, 1, True),
    ("a page larger than all", [(200, 5), (3, 1)], 16, 1, 128, 1024, True),
    ("trees", TREES, 8, 2, 128, 32, True),
    ("trees, narrow heads", TREES, 16, 1, 64, 16, True),
    ("chains", [(0, 70), (33, 1), (100, 65), (5, 0)], 3, 3, 128, 16, False),
    ("a prompt from its start", [(0, 300)], 8, 2, 64, 64, False),
    ("refused and empty requests", [(-1, 5), (40, 3), (-1, 1), (0, 0), (7, 2)], 4, 2, 128, 16, True),
    ("a long cache", [(5000, 1), (3000, 2)], 4, 1, 128, 64, False),
    ("many heads", [(260, 1), (70, 1)], 64, 2, 128, 16, False),
]


@pytest.mark.parametrize("step", FOUR, ids=[s[0] for s in FOUR])
def test_four_bits_equal_the_plain_form(pkg, dev, step):
    say("tree_attention, 4 bits", step)
    _, reqs, Hq, Hkv, D, page, as_tree = step
    s = Step(len(reqs) * 7 + Hq, reqs, Hq, Hkv, D, page, "fp4", as_tree, spare_rows=3)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)
    assert torch.equal(out, pkg.tree_attention(**s.args(dev)))


def one_request_in_room(s, room):
    s.tables = [row + [-1] * (room // s.k.shape[1] - len(row)) for row in s.tables]
    return s


LARGE = [
    (64, [(50, 4), (0, 3), (129, 2), (64, 1), (10, 0), (31, 5)], 16, 2, True), (64, [(0, 4), (90, 5), (5, 1), (300, 4)], 8, 1, False),
    (128, [(50, 8), (0, 7), (129, 5), (64, 1), (10, 0), (31, 9)], 16, 2, True), (128, [(0, 10), (90, 5), (5, 1), (300, 9)], 8, 1, False),
    (128, [(50, 16), (0, 7), (129, 13), (64, 1), (200, 16), (33, 30)], 16, 2, True), (128, [(0, 150), (63, 65), (64, 64)], 3, 3, False),
    (256, [(50, 64), (0, 33), (129, 20), (10, 0), (64, 64), (7, 13)], 16, 2, True), (256, [(0, 150), (90, 65), (33, 1), (100, 129)], 8, 2, False),
    (256, [(1500, 64), (1391, 61), (1280, 33)], 8, 2, True),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,reqs,Hq,Hkv,as_tree", LARGE)
def test_four_bits_in_larger_tiles(pkg, dev, rows, reqs, Hq, Hkv, as_tree, D):
    say("tree_attention, 4 bits, tiles of", rows, reqs, D)
    s = one_request_in_room(Step(rows + D, reqs, Hq, Hkv, D, 16, "fp4", as_tree, spare_rows=2), 131072)
    assert s.rows(pkg) == rows
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)


@pytest.mark.parametrize("W,sinks", [(1, 0), (1, 1), (2, 4), (31, 0), (32, 4), (33, 130), (127, 0), (128, 1), (129, 64), (300, 4), (1000, 0), (2 ** 31 - 1, 5), (10 ** 12, 0)])
@pytest.mark.parametrize("cache,D", [("bf16", 128), ("fp8", 64), ("fp4", 128), ("fp4", 64)])
def test_windows_of_single_tokens(pkg, dev, cache, D, W, sinks):
    say("tree_attention, window", W, sinks, cache, D)
    s = Step(W % 1000 + sinks, [(n, 1) for n in [*AROUND, 1500]], 6, 2, D, 16, cache, False, W, sinks, spare_rows=1)
    assert s.rows(pkg) == 16
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)


@pytest.mark.parametrize("W,sinks", [(1, 0), (2, 3), (7, 52), (20, 1), (64, 0), (65, 4), (100, 130), (1000, 4)])
@pytest.mark.parametrize("cache,Hq,Hkv,D,as_tree", [("bf16", 4, 4, 128, True), ("bf16", 16, 2, 64, True), ("fp8", 16, 2, 128, True), ("fp4", 16, 2, 128, True),
                                                    ("fp4", 3, 3, 64, True), ("bf16", 16, 2, 128, False), ("fp4", 12, 2, 64, False)])
def test_windows_of_trees_and_chains(pkg, dev, cache, Hq, Hkv, D, as_tree, W, sinks):
    say("tree_attention, window", W, sinks, cache, Hq, D, "tree" if as_tree else "chain")
    s = Step(W + sinks + D, TREES + [(700, 40)], Hq, Hkv, D, 32, cache, as_tree, W, sinks, spare_rows=2)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)


@pytest.mark.parametrize("rows,cache,reqs,Hq,Hkv,D,as_tree,W,sinks", [
    (64, "fp8", [(400, 30), (90, 17)], 8, 2, 128, False, 100, 4), (64, "bf16", [(700, 300)], 4, 1, 128, False, 200, 70),
    (128, "bf16", [(1100 + 13 * b, 8) for b in range(16)], 64, 4, 128, False, 1000, 4), (128, "fp4", [(1300 + 13 * b, 7) for b in range(16)], 64, 4, 64, False, 1201, 64),
    (128, "fp8", [(2600 + 13 * b, 8) for b in range(16)], 64, 4, 64, True, 2500, 4),
    (256, "bf16", [(900, 300), (300, 300)], 16, 2, 128, False, 850, 4), (256, "fp8", [(900, 300), (0, 900)], 16, 2, 64, False, 850, 0),
    (256, "fp4", [(900, 300), (300, 300)], 16, 2, 128, False, 850, 65), (256, "fp4", [(2600, 64), (2900, 60), (2500, 63), (1000, 64)], 32, 2, 128, True, 2500, 4),
    (256, "bf16", [(2600, 64), (2900, 60), (2500, 63), (1000, 64)], 32, 2, 64, True, 2530, 4)])
def test_windows_in_larger_tiles(pkg, dev, rows, cache, reqs, Hq, Hkv, D, as_tree, W, sinks):
    say("tree_attention, window, tiles of", rows, cache, W, sinks)
    s = one_request_in_room(Step(rows + W, reqs, Hq, Hkv, D, 64, cache, as_tree, W, sinks), 131072)
    assert s.rows(pkg) == rows
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)


@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 4), (64, 6, 2), (64, 16, 8)])
@pytest.mark.parametrize("W,sinks", [(None, 0), (70, 3)])
def test_two_heads_to_a_workgroup(pkg, dev, D, Hq, Hkv, W, sinks):
    """Single tokens of many requests over a 4-bit cache: neighbouring heads' keys are read together."""
    say("tree_attention, 4 bits, two heads", D, Hq, Hkv, W)
    g = torch.Generator().manual_seed(D + Hkv)
    reqs = [(int(n), 1) for n in torch.randint(0, 700, (130 // Hkv + 30,), generator=g)] + [(-1, 1), (0, 0), (1500, 1), (5, 1)]
    s = Step(D, reqs, Hq, Hkv, D, 16, "fp4", False, W, sinks, spare_rows=2)
    assert len(reqs) * Hkv >= 128 and s.rows(pkg) == 16
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)
    assert torch.equal(out, pkg.tree_attention(**s.args(dev)))


@pytest.mark.parametrize("cache,D,Hq,Hkv", [("bf16", 128, 8, 4), ("bf16", 64, 12, 6), ("fp8", 128, 4, 4), ("fp8", 64, 16, 8), ("fp4", 128, 6, 2), ("fp4", 64, 8, 4)])
@pytest.mark.parametrize("W,sinks", [(7000, 300), (7000, 0)])
def test_two_heads_to_a_workgroup_in_a_wide_window(pkg, dev, cache, D, Hq, Hkv, W, sinks):
    """The same over every cache, in windows wide enough for it: some texts end inside theirs, some begin before it."""
    say("tree_attention, two heads", cache, D, Hq, Hkv, W, sinks)
    g = torch.Generator().manual_seed(D + Hkv)
    reqs = [(int(n), 1) for n in torch.randint(0, 900, (120 // Hkv,), generator=g)] + [(-1, 1), (0, 0), (7400, 1), (5, 1), (7003, 1), (8191, 1)]
    s = one_request_in_room(Step(D + W, reqs, Hq, Hkv, D, 64, cache, False, W, sinks, spare_rows=1), 131072)
    assert len(reqs) * Hkv >= 64 and len(reqs) * Hkv * W >= 3 << 18 and s.rows(pkg) == 16
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)
    assert torch.equal(out, pkg.tree_attention(**s.args(dev)))


@pytest.mark.parametrize("cache", ["bf16", "fp8", "fp4"])
def test_keys_outside_the_window_are_not_read_into_it(pkg, dev, cache):
    """Units that hold the ends of first tokens and windows, whose other keys and values are no numbers, for tiles of every size."""
    for n, Hq, Hkv, as_tree, W, sinks in ((1, 4, 2, False, 200, 5), (1, 4, 2, False, 130, 0), (5, 16, 2, True, 77, 3), (30, 16, 2, True, 100, 1), (300, 8, 2, False, 150, 70)):
        say("tree_attention, no numbers outside", cache, n, W, sinks)
        s = one_request_in_room(Step(n + W, [(701, n), (333, n)], Hq, Hkv, 128, 16, cache, as_tree, W, sinks), 131072)
        for b, (l, new) in enumerate(zip(s.lens, s.counts)):
            for i in range(sinks, l - new - W):            # cached keys that no row sees
                where = s.tables[b][i // 16], i % 16
                if cache == "fp4":
                    s.ks[where] = s.vs[where] = 255
                else:
                    s.k[where] = s.v[where] = torch.tensor(math.nan).to(s.k.dtype)
        out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
        torch.cuda.synchronize()
        assert bool(out.isfinite().all())
        s.check(out, lse)


@pytest.mark.parametrize("cache,reqs,Hq,Hkv,D,W,sinks", [
    # a tile to each workgroup or several, parts of one, and lengths too different for either
    ("bf16", [(400 + b, 1) for b in range(100)], 8, 4, 64, 200, 4), ("bf16", [(300, 1)] * 260, 4, 2, 128, 100, 0), ("fp8", [(900, 1)] * 3, 4, 2, 64, 500, 1),
    ("fp4", [(90 * b, 1) for b in range(70)], 2, 1, 64, 600, 0), ("bf16", [(2000, 1), (100, 1)], 2, 1, 64, 1900, 7),
    # prompts: more tiles than lanes, and many requests with tiles of their own
    ("bf16", [(0, 1500), (700, 900)], 8, 2, 64, 300, 4), ("fp4", [(100, 2500)], 2, 2, 64, None, 0), ("fp4", [(13 * b, 40 + b) for b in range(70)], 4, 1, 64, 64, 2),
    ("fp8", [(500, 200), (0, 3), (40, 700)], 16, 1, 128, 90, 0), ("fp4", [(0, 1100), (3, 1), (-1, 4), (90, 600)], 3, 1, 64, None, 0)])
def test_ways_along_the_line(pkg, dev, cache, reqs, Hq, Hkv, D, W, sinks):
    say("tree_attention, lines of", len(reqs), "requests", cache, W)
    for room in (None, 131072):                          # (another room, another tile)
        s = Step(len(reqs) + D, reqs, Hq, Hkv, D, 64, cache, False, W, sinks)
        if room:
            one_request_in_room(s, room)
        out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
        torch.cuda.synchronize()
        s.check(out, lse)
        assert torch.equal(out, pkg.tree_attention(**s.args(dev)))


@pytest.mark.parametrize("cu", [[0, 5, 3, 9], [9, 0, 9, 2], [0, 9, 0, 9], [-4, 20, 1, 3]])
def test_every_walk_ends(pkg, dev, cu):
    """cu_tokens that do not ascend: results are undefined, but the launch ends."""
    say("tree_attention in a window, cu_tokens", cu)
    for W, cache in ((20, "bf16"), (None, "fp4")):
        s = Step(2, [(300, 3), (200, 3), (64, 3)], 8, 2, 64, 16, cache, False, W)
        pkg.tree_attention(**s.args(dev, cu_tokens=ints(cu, dev)))
        pkg.tree_attention(**s.args(dev, kv_lens=ints([2 ** 31 - 1, -5, 7], dev)))
    torch.cuda.synchronize()


@pytest.mark.parametrize("cache", ["bf16", "fp8", "fp4"])
@pytest.mark.parametrize("as_tree", [False, True])
def test_scores_that_grow_along_a_window(pkg, dev, cache, as_tree):
    """The first visible keys lie far below the later ones, and what is not seen far above all of them."""
    say("tree_attention growing scores in a window", cache, as_tree)
    s = Step(31, [(600, 20), (200, 3)], 4, 1, 64, 16, cache, as_tree, 150, 3, q_scale=3.0)
    for b, l in enumerate(s.lens):
        for i in range(l):
            at = (s.tables[b][i // 16], i % 16, 0)
            up = 3 - i // 100
            if cache == "fp4":
                s.ks[at] = 127 + up
            else:
                s.k[at] = (s.k[at].float().clamp(-100, 100) * 2.0 ** up).to(s.kind)
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)
    for b, l in enumerate(s.lens):                       # and the other way round
        for i in range(l):
            if cache == "fp4":
                s.ks[s.tables[b][i // 16], i % 16, 0] = 124 + i // 100
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("cache", ["bf16", "fp4"])
@pytest.mark.parametrize("reqs,Hq,Hkv,as_tree,W,sinks", [([(400, 1), (90, 1)], 4, 2, False, 100, 4), ([(300, 30), (130, 9)], 16, 2, True, 40, 70),
                                                        ([(500, 40), (10, 5)], 16, 2, False, 64, 0)])
def test_what_is_not_seen_may_be_anything(pkg, dev, cache, reqs, Hq, Hkv, as_tree, W, sinks):
    """NaN behind the window, beyond the end and in pages of no request; pages behind the window given back (their entries -1)."""
    say("tree_attention, NaN behind the window", cache, reqs, W, sinks)
    s = Step(17, reqs, Hq, Hkv, 128, 16, cache, as_tree, W, sinks)
    clean = pkg.tree_attention(**s.args(dev))
    seen = set()
    for b, l in enumerate(s.lens):
        n = s.counts[b]
        lowest = max(0, l - n + 1 - W - (n if as_tree else 0))
        seen |= {(s.tables[b][i // 16], i % 16) for i in range(l) if i >= lowest or i < sinks}
        for p in range(-(-sinks // 16), lowest // 16):
            s.tables[b][p] = -1
    for blk in range(s.k.shape[0]):
        for i in range(16):
            if (blk, i) not in seen:
                if cache == "fp4":
                    s.ks[blk, i], s.vs[blk, i] = 255, 255
                else:
                    s.k[blk, i], s.v[blk, i] = math.nan, math.inf
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    assert torch.equal(out, clean)
    s.check(out, lse)


@pytest.mark.parametrize("cache", ["bf16", "fp4"])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(pkg, dev, cache):
    say("tree_attention, NaN in the window", cache)
    for hit in (330, 260, 2):                            # among the new tokens, in some rows' window, a first token
        s = Step(23, [(300, 40), (50, 2)], 8, 2, 64, 16, cache, False, 50, 4)
        at = (s.tables[0][hit // 16], hit % 16, 1)
        if cache == "fp4":
            s.vs[at] = 255
        else:
            s.v[(*at, slice(3, 9))] = math.nan
        out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
        ref, _, reach = s.want()
        there, got = reach.isfinite(), out.double().cpu()
        assert bool(((got - ref).abs() <= plain.attention_bound(ref, reach))[there].all())
        assert int((~there).sum()) > 0 and bool((~got.isfinite())[~there].all())


def test_every_code_under_every_power(pkg, dev):
    """One key: the output is its value, exactly where bf16 holds it (codes of up to 3 digits times a power of two)."""
    say("tree_attention, every code")
    page, D = 256, 128
    powers = torch.arange(256, dtype=torch.uint8).view(1, page, 1, 1).expand(1, page, 1, 4).contiguous()
    codes = (torch.arange(D // 2) * 37 % 256).to(torch.uint8).view(1, 1, 1, -1).expand(1, page, 1, D // 2).contiguous()
    k = torch.zeros(1, page, 1, D // 2, dtype=torch.uint8)
    one = torch.full((1, page, 1, 4), 127, dtype=torch.uint8)
    q = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=dev)
    tables, cu = ints([[0]], dev), ints([0, 1], dev)
    want = window.decode(codes, powers)[0, :, 0]
    for place in range(0, 256, 5):
        # the key at `place` alone: the last of place + 1 keys in a window of 1
        out = pkg.tree_attention(q, k.to(dev).view(FP4), codes.to(dev).view(FP4), tables, ints([place + 1], dev), cu, k_scale=one.to(dev).view(E8M0),
                                 v_scale=powers.to(dev).view(E8M0), window=1)
        got, ref = out.double().cpu()[0, 0], want[place]
        if place == 255:
            assert bool(got.isnan().all())
        elif place >= 253:
            assert bool((got[ref.abs() < 3e38] == ref[ref.abs() < 3e38]).all())
        elif place > 1:                                  # (below, results are subnormal)
            assert torch.equal(got, ref)


@pytest.mark.parametrize("cache", ["bf16", "fp4"])
def test_masks_that_leave_nothing(pkg, dev, cache):
    say("tree_attention, empty rows in a window", cache)
    s = Step(9, [(0, 6), (0, 64), (20, 3)], 4, 2, 64, 16, cache, True, 2, 1)
    for j in (0, 3, 69, 16, 70):
        s.masks[j] = 0
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)
    assert bool((lse[[0, 3, 69, 16]] == -math.inf).all()) and bool((out[[0, 3, 69, 16]] == 0).all()) and bool(lse[70].isfinite().all())


def test_masks_that_are_no_trees(pkg, dev):
    """Of any mask the last and the first of what it names count, whatever lies between."""
    s = Step(10, [(0, 64), (3, 50), (90, 64)], 4, 2, 128, 16, "bf16", True, 9, 5)
    g = torch.Generator().manual_seed(1)
    s.masks = torch.randint(-2 ** 63, 2 ** 63 - 1, (s.T,), generator=g).tolist()
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    s.check(out, lse)


@pytest.mark.parametrize("cache", ["bf16", "fp4"])
def test_strides_streams_and_graphs(pkg, dev, cache):
    say("windows: strides, streams, graphs", cache)
    s = Step(21, [(300, 9), (77, 16), (0, 1)], 8, 2, 128, 16, cache, True, 90, 4)
    want = pkg.tree_attention(**s.args(dev))
    a = s.args(dev)
    n = s.k.shape[0]
    if cache == "fp4":                                   # a block's keys, values and their powers in one piece of memory
        each = 16 * 2 * 64
        whole = torch.zeros(n, 2 * each + 2 * 16 * 2 * 4 + 64, dtype=torch.uint8, device=dev)
        cut = lambda at, t: whole[:, at:at + t[0].numel()].unflatten(1, t.shape[1:])
        parts = [cut(0, s.k), cut(each, s.v), cut(2 * each, s.ks), cut(2 * each + 128, s.vs)]
        for p, t in zip(parts, (s.k, s.v, s.ks, s.vs)):
            p.copy_(t)
        a.update(k_cache=parts[0].view(FP4), v_cache=parts[1].view(FP4), k_scale=parts[2].view(E8M0), v_scale=parts[3].view(E8M0))
    else:
        both = torch.stack([s.k, s.v], 1).to(dev)
        a.update(k_cache=both[:, 0], v_cache=both[:, 1])
    wide = torch.randn(s.T, 8 * 128 + 64, device=dev).to(torch.bfloat16)
    wide[:, 32:32 + 1024] = s.q.view(s.T, -1).to(dev)
    a["q"] = wide[:, 32:32 + 1024].view(s.T, 8, 128)
    assert torch.equal(pkg.tree_attention(**a), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.tree_attention(**a)
    side.synchronize()
    assert torch.equal(got, want)
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


def test_a_cache_of_more_than_32_bits(pkg, dev):
    """Codes of more than 2^32 bytes, the request's pages at their end; and what is stored there."""
    say("4 bits, large cache")
    s = Step(4, [(130, 5)], 4, 2, 128, 64, "fp4", True, 100, 4)
    n_blocks = (1 << 32) // (64 * 2 * 64) + 40
    big = [torch.empty(n_blocks, 64, 2, w, dtype=torch.uint8, device=dev) for w in (64, 64, 4, 4)]
    old = [t for t in s.tables[0] if t >= 0]
    new = [n_blocks - 1 - 3 * i for i in range(len(old))]
    for to, src in zip(big, (s.k, s.v, s.ks, s.vs)):
        for o, n in zip(old, new):
            to[n] = src[o].to(dev)
    k, v, ks, vs = big[0].view(FP4), big[1].view(FP4), big[2].view(E8M0), big[3].view(E8M0)
    table = new + [-1] * (len(s.tables[0]) - len(new))
    out, lse = pkg.tree_attention(**s.args(dev, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, block_tables=ints([table], dev)), return_lse=True)
    s.check(out, lse)
    x = torch.randn(2, 8 * 128, device=dev).to(torch.bfloat16)
    slots = ints([n_blocks * 64 - 1, n_blocks * 64 - 64 * 7], dev, torch.int64)
    pkg.qk_norm_rope(x, ints([1, 2], dev), torch.randn(4, 128, device=dev), 4, 2, k_cache=k, v_cache=v, slots=slots, k_scale=ks, v_scale=vs)
    codes, powers = window.encode(x.cpu().double().view(2, 8, 128)[:, 6:])
    for i, (blk, place) in enumerate(((n_blocks - 1, 63), (n_blocks - 7, 0))):
        assert torch.equal(big[1][blk, place].cpu(), codes[i]) and torch.equal(big[3][blk, place].cpu(), powers[i])


# ------------------------------------------------------------------------------------------------ into the cache
@pytest.mark.parametrize("T,Hq,Hkv,D,R,pairs,weights", [
    (1, 32, 4, 128, 128, False, True), (5, 6, 2, 128, 64, True, True), (33, 8, 8, 96, 96, False, False), (7, 10, 2, 256, 256, True, True),
    (19, 4, 2, 32, 32, False, True), (300, 5, 1, 160, 32, False, True), (1030, 12, 4, 64, 64, False, False), (2049, 4, 1, 128, 128, True, True),
    (0, 4, 1, 128, 128, False, True)])
def test_the_way_into_a_cache_in_four_bits(pkg, dev, T, Hq, Hkv, D, R, pairs, weights):
    say("qk_norm_rope, 4 bits", T, Hq, Hkv, D, R, pairs)
    g = torch.Generator().manual_seed(T * 31 + D)
    page, P = 16, 700
    x = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * torch.exp2(torch.randint(-9, 9, (T, Hq + 2 * Hkv, 1), generator=g))
    x[:, :, ::13] *= 20
    qkv = x.to(torch.bfloat16).flatten(1)
    src = qkv.view(T, Hq + 2 * Hkv, D)
    if T > 4:
        src[2, -1, :32] = 0                              # a block of zeros; values that are no numbers
        src[3, -1, 5] = math.nan
        src[4, -1, 7] = -math.inf
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32)
    cs = torch.randn(P, R, generator=g).clamp(-1, 1)
    wt = (1 + 0.3 * torch.randn(D, generator=g)).to(torch.bfloat16) if weights else None
    n_blocks = T // page + 3
    slots = torch.randperm(n_blocks * page, generator=g)[:T]
    if T > 6:
        slots[0], slots[1], pos[5] = -1, n_blocks * page, -1                     # nothing to store
    held = {n: torch.randint(0, 256, (n_blocks, page, Hkv, w), generator=g).to(torch.uint8) for n, w in (("k", D // 2), ("v", D // 2), ("ks", D // 32), ("vs", D // 32))}
    on = {n: t.to(dev) for n, t in held.items()}
    to = lambda t: None if t is None else t.to(dev)
    q = pkg.qk_norm_rope(qkv.to(dev), pos.to(dev), cs.to(dev), Hq, Hkv, to(wt), to(wt), 1e-5, pairs, on["k"].view(FP4), on["v"].view(FP4), slots.to(dev),
                         on["ks"].view(E8M0), on["vs"].view(E8M0))
    without = pkg.qk_norm_rope(qkv.to(dev), pos.to(dev), cs.to(dev), Hq, Hkv, to(wt), to(wt), 1e-5, pairs)[0] if T else q
    torch.cuda.synchronize()
    assert torch.equal(q.nan_to_num(), without.nan_to_num())
    stored = [t for t in range(T) if 0 <= slots[t] < n_blocks * page and 0 <= pos[t] < P]
    got = {n: t.cpu().flatten(0, 1) for n, t in on.items()}
    others = torch.ones(n_blocks * page, dtype=torch.bool)
    others[slots[stored]] = False
    for n in got:                                        # what no token is stored in stays
        assert torch.equal(got[n][others], held[n].flatten(0, 1)[others])
    if not stored:
        return
    # values are what 64 bits say, to the bit
    codes, powers = window.encode(src[stored, Hq + Hkv:].double())
    assert torch.equal(got["vs"][slots[stored]], powers)
    fine = (powers != 255).repeat_interleave(16, -1)
    assert torch.equal(got["v"][slots[stored]][fine], codes[fine])
    # keys: fp32 on the way may bring one past a border that is nearer than its error
    want = plain.norm_rope(src[:, Hq:Hq + Hkv], wt, 1e-5, pos, cs, pairs)[stored]
    off = 64 * plain.U32 * want.abs().amax(-1, keepdim=True)
    p = got["ks"][slots[stored]]
    top = want.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    least, most = (window.power_bytes((top + s * off[..., None]).clamp_min(0).expand(*top.shape[:-1], 32).flatten(-2)) for s in (-1, 1))
    assert bool(((p >= least) & (p <= most)).all())
    c = got["k"][slots[stored]]
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2).long()
    lo, hi = (window.nearest((want.abs() + s * off).clamp_min(0), p) for s in (-1, 1))
    assert bool(((c & 7 >= lo) & (c & 7 <= hi)).all())
    assert bool(((c >= 8) == torch.signbit(want))[want.abs() > off].all())


def test_into_a_captured_cache(pkg, dev):
    """Norms, rotation and store, then attention in a window, captured together and replayed as the text grows."""
    say("4 bits: captured store and attention")
    g = torch.Generator().manual_seed(2)
    Hq, Hkv, D, page = 8, 2, 128, 16
    caches = [torch.zeros(12, page, Hkv, w, dtype=torch.uint8, device=dev) for w in (64, 64, 4, 4)]
    k, v, ks, vs = caches[0].view(FP4), caches[1].view(FP4), caches[2].view(E8M0), caches[3].view(E8M0)
    qkv = torch.zeros(1, 12 * D, dtype=torch.bfloat16, device=dev)
    pos, slots, lens = ints([0], dev), ints([0], dev, torch.int64), ints([1], dev)
    tables, cu, cs = ints([[3, 7, 1, 0, 5]], dev), ints([0, 1], dev), torch.randn(100, D, generator=g).to(dev)
    out = torch.zeros(1, Hq, D, dtype=torch.bfloat16, device=dev)

    def step():
        q = pkg.qk_norm_rope(qkv, pos, cs, Hq, Hkv, k_cache=k, v_cache=v, slots=slots, k_scale=ks, v_scale=vs)
        return pkg.tree_attention(q, k, v, tables, lens, cu, k_scale=ks, v_scale=vs, window=20, sinks=2, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(40):
        qkv.copy_(torch.randn(1, 12 * D, generator=g))
        pos.fill_(t)
        lens.fill_(t + 1)
        slots.fill_(int(tables[0, t // page]) * page + t % page)
        graph.replay()
        got = out.clone()
        out.zero_()
        assert torch.equal(step(), got), t
    s = Step(0, [(39, 1)], Hq, Hkv, D, page, "fp4", False, 20, 2)
    s.k, s.v, s.ks, s.vs = (c.cpu() for c in caches)
    s.tables = tables.tolist()
    s.q = pkg.qk_norm_rope(qkv, pos, cs, Hq, Hkv)[0].cpu()
    s.check(got, None)


# ------------------------------------------------------------------------------------------------ workspaces
def in_c(pkg, s, dev, workspace, given, window=None, sinks=0):
    """tree_attention of Step s by its C entry, with `given` bytes of `workspace`: the entry with a window where there is one."""
    a = s.args(dev)
    q, k, ptr = a["q"].contiguous(), a["k_cache"], lambda t: None if t is None else t.data_ptr()
    (T, Hq, D), (n_blocks, page, Hkv, _) = q.shape, k.shape
    out, tables = torch.zeros_like(q), a["block_tables"].contiguous()
    stream, block = torch.cuda.current_stream().cuda_stream, page * Hkv * D
    kind = {"bf16": 1, "fp8": 2}[s.cache]
    head = (stream, ptr(q), Hq * D, T, Hq, Hkv, D, ptr(k), ptr(a["v_cache"]), kind, n_blocks, block, block, page, ptr(tables), tables.shape[1], tables.shape[1],
            ptr(a["kv_lens"]), ptr(a["cu_tokens"]), len(s.lens), ptr(a.get("masks")), s.scale, ptr(a.get("k_scale")), ptr(a.get("v_scale")))
    tail = (ptr(out), None, ptr(workspace), given)
    lib = pkg._lib.lib
    rc = lib.moe_window_attention(*head, 0, 0, window, sinks, *tail) if window else lib.moe_tree_attention(*head, *tail)
    torch.cuda.synchronize()
    return rc, out


@pytest.mark.parametrize("cache,B,Hkv", [("bf16", 70, 4), ("bf16", 260, 2), ("fp8", 70, 4)])
def test_calls_ask_for_what_they_use(pkg, dev, cache, B, Hkv):
    """Without a window one head's parts are room enough, with one too, and nothing behind the room is touched."""
    say("workspaces", cache, B, Hkv)
    D, W = 128, 8000
    one = 2 * (256 if cache == "bf16" else 512) * 16 * (D * 4 + 8) + (256 if cache == "bf16" else 512) * 32
    s = one_request_in_room(Step(B, [(17 * b % 900 + (7500 if b == 3 else 0), 1) for b in range(B)], 2 * Hkv, Hkv, D, 64, cache, False), 131072)
    lib = pkg._lib.lib
    more = lib.moe_window_attention_workspace_bytes(B, 2 * Hkv, Hkv, D, B, 1 if cache == "bf16" else 2)
    room = torch.full((more + 65536,), 7, dtype=torch.uint8, device=dev)
    for given, window in ((one, None), (one, W), (more, W)):
        s.window = dict(window=window, sinks=4 if window else 0)
        room.fill_(7)
        rc, out = in_c(pkg, s, dev, room, given, window, 4)
        assert rc == 0
        assert bool((room[given:] == 7).all())
        s.check(out, None)
        if given == more or not window:
            assert torch.equal(out, pkg.tree_attention(**s.args(dev)))


def heads_of(pkg, s):
    (T, Hq, _), (_, page, Hkv, _) = s.q.shape, s.k.shape
    return pkg._lib.lib.moe_window_attention_heads(T, Hq, Hkv, len(s.lens), {"bf16": 1, "fp8": 2, "fp4": 3}[s.cache], s.masks is not None, len(s.tables[0]), page,
                                                   min(s.window["window"] or 0, 2 ** 31 - 1), s.window["sinks"])


@pytest.mark.parametrize("cache,D,Hq,Hkv,W,sinks", [
    ("fp4", 128, 8, 4, None, 0), ("fp4", 64, 6, 2, None, 0), ("fp4", 64, 16, 8, None, 0), ("fp4", 128, 32, 4, 9000, 5), ("fp4", 64, 4, 4, 9000, 0),
    ("fp8", 128, 8, 2, 9000, 70), ("fp8", 64, 16, 8, 9000, 0), ("bf16", 128, 8, 4, 9000, 1), ("bf16", 64, 6, 6, 9000, 130)])
@pytest.mark.parametrize("lengths", ["ragged", "alike", "one long"])
def test_the_kernel_of_two_heads(pkg, dev, cache, D, Hq, Hkv, W, sinks, lengths):
    """Two heads to a workgroup: tiles cut across workgroups and joined, whole tiles, and one tile over many workgroups."""
    say("tree_attention, two heads", cache, D, Hq, Hkv, W, sinks, lengths)
    g = torch.Generator().manual_seed(D + Hkv)
    some = torch.randint(0, 700, (130 // Hkv + 30,), generator=g).tolist()
    cached = {"ragged": some, "alike": [410] * len(some), "one long": [3 + n % 40 for n in some]}[lengths]
    reqs = [(n, 1) for n in cached] + [(-1, 1), (0, 0), (9100 if lengths != "alike" else 411, 1), (5, 1)]
    s = one_request_in_room(Step(D, reqs, Hq, Hkv, D, 16, cache, False, W, sinks, spare_rows=2), 131072)
    assert heads_of(pkg, s) == 2 and s.rows(pkg) == 16
    out, lse = pkg.tree_attention(**s.args(dev), return_lse=True)
    torch.cuda.synchronize()
    s.check(out, lse)
    assert torch.equal(out, pkg.tree_attention(**s.args(dev)))
