"""tree_attention's kernels of large tiles against the plain form in 64 bits.  Which kernel runs goes by the rows of a request and by the
room of the block table, so the tables here have room for 131072 tokens, as a server's have, and every test says which tile it is for."""
import math

import pytest
import torch

import serving_plain as plain
from test_gpu_serving import Step, ints, say

pytestmark = pytest.mark.gpu

ROOM = 131072


def with_room(step):
    """The step's tables with unused entries up to ROOM tokens."""
    page = step.k.shape[1]
    step.tables = [row + [-1] * (ROOM // page - len(row)) for row in step.tables]
    return step


def tile_rows(pkg, step):
    (T, Hq, _), (_, page, Hkv, _) = step.q.shape, step.k.shape
    return pkg._lib.lib.moe_tree_attention_tile_rows(T, Hq, Hkv, len(step.lens), 2 if step.ks is not None else 1, step.masks is not None,
                                                     len(step.tables[0]), page)


def attend(pkg, dev, step, rows, **other):
    say("tree_attention in tiles of", rows)
    assert tile_rows(pkg, step) == rows
    out, lse = pkg.tree_attention(**step.args(dev, **other), return_lse=True)
    torch.cuda.synchronize()
    return out, lse


# tile rows, what, (cached, new) of the requests, query heads, cache heads, a tree
STEPS = [
    (64, "trees", [(50, 8), (0, 7), (129, 5), (64, 1), (10, 0), (31, 9)], 16, 2, True),
    (64, "chunks", [(0, 10), (90, 5), (5, 1), (300, 9)], 8, 1, False),
    (128, "trees", [(50, 16), (0, 7), (129, 13), (64, 1), (200, 16), (33, 30)], 16, 2, True),
    (128, "trees without room in the cache", [(-1, 20), (40, 13), (-1, 1), (0, 0), (7, 33)], 8, 1, True),
    (128, "chunks", [(0, 20), (90, 13), (5, 1), (300, 16)], 16, 2, False),
    (128, "chunks, no shared heads", [(0, 150), (63, 65), (64, 64)], 3, 3, False),
    (128, "long caches", [(1500, 16), (1391, 11)], 8, 1, True),
    (256, "trees", [(50, 64), (0, 33), (129, 20), (10, 0), (64, 64), (7, 13)], 16, 2, True),
    (256, "trees without room in the cache", [(-1, 40), (40, 30), (-1, 1), (0, 0), (7, 33)], 8, 1, True),
    (256, "chunks", [(0, 150), (90, 65), (33, 1), (100, 129)], 8, 2, False),
    (256, "chunks, no shared heads", [(0, 300), (20, 257)], 3, 3, False),
    (256, "long caches", [(1500, 64), (1391, 61), (1280, 33)], 8, 2, True),
    (256, "a prompt from its start", [(0, 515)], 4, 1, False),
]


@pytest.mark.parametrize("D,fp8", [(128, False), (128, True), (64, False), (64, True)])
@pytest.mark.parametrize("rows,what,reqs,Hq,Hkv,as_tree", STEPS, ids=[f"{s[0]} {s[1]}" for s in STEPS])
def test_tiles_equal_the_plain_form(pkg, dev, rows, what, reqs, Hq, Hkv, as_tree, D, fp8):
    say(what, reqs, D, fp8)
    s = with_room(Step(len(reqs) * 13 + rows + D, reqs, Hq, Hkv, D, 64 if fp8 else 16, fp8, as_tree, spare_rows=3))
    out, lse = attend(pkg, dev, s, rows)
    s.check(out, lse)
    assert torch.equal(out, pkg.tree_attention(**s.args(dev)))       # the same inputs, the same bits


SMALL = {64: ([(61, 8), (7, 5), (130, 1)], 16, 2), 128: ([(61, 16), (7, 13), (130, 11)], 16, 2), 256: ([(61, 64), (7, 33), (130, 13)], 16, 2)}


@pytest.mark.parametrize("rows", [64, 128, 256])
@pytest.mark.parametrize("fp8", [False, True])
def test_tiles_whose_masks_leave_rows_nothing(pkg, dev, rows, fp8):
    reqs, Hq, Hkv = SMALL[rows]
    s = with_room(Step(rows, [(0, n) for _, n in reqs] + [(70, 3)], Hq, Hkv, 128, 16, fp8, True, spare_rows=5))
    n = s.counts[0]
    empty = [0, 3, n - 1, n, n + 4]
    for j in empty:
        s.masks[j] = 0
    s.masks[s.cu[3]] = 0                                             # sees the cached keys all the same
    out, lse = attend(pkg, dev, s, rows)
    s.check(out, lse)
    assert bool((lse[empty] == -math.inf).all()) and bool((out[empty] == 0).all()) and bool(lse[s.cu[3]].isfinite().all())


@pytest.mark.parametrize("as_tree", [True, False])
@pytest.mark.parametrize("rows", [64, 128, 256])
@pytest.mark.parametrize("what,fp8", [(math.nan, False), (math.inf, False), (-math.inf, False), (math.nan, True)])
def test_tiles_ignore_what_a_row_does_not_see(pkg, dev, what, fp8, rows, as_tree):
    """NaN and infinities behind the end of a request, in pages of no request, and in new tokens that not every row sees."""
    reqs, Hq, Hkv = SMALL[rows]
    s = with_room(Step(3, reqs, Hq, Hkv, 128, 16, fp8, as_tree))
    held = {(s.tables[b][i // 16], i % 16) for b, l in enumerate(s.lens) for i in range(l)}
    for blk in range(s.k.shape[0]):
        for i in range(16):
            if (blk, i) not in held:
                s.k[blk, i] = torch.tensor(what).to(s.kind)
                s.v[blk, i] = torch.tensor(what).to(s.kind)
    at = s.lens[0] - s.counts[0] + 1                                 # the first request's second new token
    s.v[s.tables[0][at // 16], at % 16, 0, 5:9] = torch.tensor(what).to(s.kind)
    if what != what:
        s.k[s.tables[0][at // 16], at % 16, Hkv - 1, 3] = torch.tensor(what).to(s.kind)
    out, _ = attend(pkg, dev, s, rows)
    got = out.double().cpu()
    ref, _, reach = plain.attention(s.q, s.k.float(), s.v.float(), s.tables, s.lens, s.cu, s.masks, s.scale, s.ks, s.vs)
    there = reach.isfinite()
    off = (got - ref).abs()
    assert bool((off <= plain.attention_bound(ref, reach))[there].all())
    assert int((~there).sum()) > 0 and bool((~got.isfinite())[~there].all())


@pytest.mark.parametrize("rows,reqs,Hq", [(64, [(300, 16)], 4), (128, [(300, 16), (288, 16)], 8), (256, [(300, 32)], 8), (256, [(300, 14)], 16)])
def test_tiles_growing_scores(pkg, dev, rows, reqs, Hq):
    """Every key outscores the ones before it by far: the running offset moves all the time."""
    s = with_room(Step(11, reqs, Hq, 1, 64, 16, False, True))
    for b, l in enumerate(s.lens):
        for i in range(l):
            s.k[s.tables[b][i // 16], i % 16, 0] = torch.full((64,), (i - 200) * 0.05).to(torch.bfloat16)
    s.q[:] = 2
    s.check(*attend(pkg, dev, s, rows))


@pytest.mark.parametrize("rows", [128, 256])
def test_tiles_in_graphs(pkg, dev, rows):
    reqs, Hq, Hkv = SMALL[rows]
    s = with_room(Step(21, reqs, Hq, Hkv, 128, 16, False, True))
    a = s.args(dev)
    want, _ = attend(pkg, dev, s, rows)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.tree_attention(**a, out=out)
    for lens in (s.lens, [s.counts[0], s.lens[1], s.lens[2]], [s.lens[0], 0, s.lens[2] - 100], s.lens):
        a["kv_lens"].copy_(ints(lens, dev))
        eager = pkg.tree_attention(**a)
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens
    assert torch.equal(out, want)
