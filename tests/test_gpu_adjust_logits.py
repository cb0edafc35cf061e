"""adjust_logits on the GPU against its plain 64-bit form: histories, paths, repeated and foreign ids, odd vocabularies, in place."""
import math
import random

import pytest
import torch

import between_plain as plain

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


class Case:
    def __init__(self, seed, counts, V, L, bf16, tree=False, path=True, history=True, penalties="all", biases=0, masked=None, spare=0, gap=0):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        B = len(counts)
        self.cu = [gap]
        for n in counts:
            self.cu.append(self.cu[-1] + n)
        T = self.cu[-1] + spare
        self.T, self.V = T, V
        self.x = (torch.randn(T, V, generator=g) * 3).to(torch.bfloat16 if bf16 else torch.float32)
        word = lambda: rng.choice([rng.randrange(V), rng.randrange(min(V, 6)), V - 1, rng.randrange(-2, V + 3)])
        self.history = [[word() for _ in range(L)] for _ in range(B)] if history else None
        self.lens = [rng.choice([0, L, L, rng.randint(0, L), L + 5, -1]) for _ in range(B)] if history else None
        self.asked = [rng.randint(-1, L + 1) for _ in range(B)] if history else None
        self.tokens = [word() for _ in range(T)] if path else None
        self.masks = None
        if tree and path:
            self.masks = [0] * T
            for b, n in enumerate(counts):
                for j in range(n):
                    up = rng.choice([-1, j - 1, j - 1, j - 1, max(0, j - 3)])
                    self.masks[self.cu[b] + j] = 1 << j | (self.masks[self.cu[b] + up] if 0 <= up < j else 0)
        on = lambda name: penalties == "all" or penalties == name
        some = lambda lo, hi: [rng.choice([lo, rng.uniform(lo, hi)]) for _ in range(B)]
        f32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32).tolist()
        self.rep, self.freq, self.pres = (f32(v) if on(k) else None for k, v in
                                          (("repetition", some(1.0, 2.0)), ("frequency", some(0.0, 1.0)), ("presence", some(-0.5, 1.0))))
        self.bias_ids = [[word() for _ in range(biases)] for _ in range(B)] if biases else None
        self.bias = [f32([rng.uniform(-5, 5) for _ in range(biases)]) for _ in range(B)] if biases else None
        self.allowed = self.rows = None
        if masked is not None:
            n = T if masked == "own" else max(1, T // 2)
            few = lambda: rng.getrandbits(32) & rng.getrandbits(32)
            self.allowed = [[rng.choice([0, few(), 0xffffffff]) for _ in range(-(-V // 32))] for _ in range(n)]
            self.allowed[0] = [0] * (-(-V // 32))        # leaves nothing
            self.rows = None if masked == "own" else [rng.choice([-1, n, rng.randrange(n)]) for _ in range(T)]

    def args(self, dev, **other):
        t = lambda v, kind=torch.int32: None if v is None else torch.tensor(v, dtype=kind).to(dev)
        signed = lambda v, n: None if v is None else [x - (1 << n) if x >> (n - 1) & 1 else x for x in v]
        two = lambda v: None if v is None else t(v).view(len(v), len(v[0]) if v else 0)
        a = dict(logits=self.x.to(dev), cu_tokens=t(self.cu), history=two(self.history), history_lens=t(self.lens), prompt_lens=t(self.asked),
                 tokens=t(self.tokens, torch.int64), masks=t(signed(self.masks, 64), torch.int64), repetition=t(self.rep, torch.float32),
                 frequency=t(self.freq, torch.float32), presence=t(self.pres, torch.float32), bias_ids=two(self.bias_ids),
                 bias=t(self.bias, torch.float32), allowed=None if self.allowed is None else t([signed(r, 32) for r in self.allowed]), allowed_rows=t(self.rows))
        a.update(other)
        return a

    def check(self, got):
        lens = None if self.lens is None else [min(max(n, 0), len(h)) for n, h in zip(self.lens, self.history)]
        allowed = self.allowed
        x, reach = plain.adjust_logits(self.x.double(), self.cu, self.history, lens, self.asked, self.tokens, self.masks, self.rep, self.freq,
                                       self.pres, self.bias_ids, self.bias, allowed, self.rows)
        none = [t for t in range(self.T) if not self.cu[0] <= t < self.cu[-1]]
        x[none] = self.x[none].double()
        got = got.double().cpu()
        unit = plain.U16 if self.x.dtype == torch.bfloat16 else plain.U32
        fine = x.isfinite()
        assert bool((got[~fine] == x[~fine]).all())
        # five operations of fp32, of numbers up to the reach; then the output's rounding.  What nothing touches is the very value.
        most = unit * x.abs() + 8 * plain.U32 * reach
        off = (got - x).abs()
        assert bool((off[fine] <= most[fine]).all()), float((off / most)[fine].max())
        same = x == self.x.double()
        assert bool((got[same] == x[same]).all())


@pytest.mark.parametrize("counts,V,L,bf16,tree,how", [
    ([1], 1, 3, False, False, {}), ([1], 5, 0, True, False, dict(biases=3)), ([1, 1, 1], 37, 9, True, False, dict(masked="rows")),
    ([1], 50000, 700, True, False, dict(biases=20, masked="own")), ([3, 0, 5], 8192, 100, False, False, dict(masked="own")),
    ([16, 4, 9], 8191, 300, True, True, dict(biases=5)), ([64, 1, 33], 16390, 64, False, True, dict(masked="rows", spare=3)),
    ([7, 2], 100, 40, True, True, dict(history=False)), ([2, 3], 9001, 2000, True, False, dict(path=False, biases=40, gap=2)),
    ([40, 1], 333, 50, False, False, dict(biases=2, spare=2, gap=1)), ([1] * 33, 1001, 30, True, False, dict(masked="rows")),
    ([5, 6], 513, 20, True, True, dict(penalties="repetition")), ([5, 6], 514, 20, False, True, dict(penalties="frequency")),
    ([4], 515, 20, True, True, dict(penalties="presence", biases=1)), ([4, 4], 516, 20, True, True, dict(penalties=None, biases=7, masked="own")),
    ([2], 24600, 5, False, False, dict(biases=1023)), ([0, 0], 40, 4, True, False, dict(spare=5)), ([300], 60, 8, True, False, {})])
def test_equals_the_plain_form(pkg, dev, counts, V, L, bf16, tree, how):
    say("adjust_logits", len(counts), "requests", V, L, "bf16" if bf16 else "f32", tree, how)
    c = Case(V + L, counts, V, L, bf16, tree, **how)
    a = c.args(dev)
    got = pkg.adjust_logits(**a)
    torch.cuda.synchronize()
    c.check(got)
    assert torch.equal(a["logits"].cpu(), c.x)
    again = a["logits"].clone()
    a["logits"] = again
    assert pkg.adjust_logits(**a, out=again).data_ptr() == again.data_ptr()
    assert torch.equal(again, got)


@pytest.mark.parametrize("bf16,V,at,out_at", [(True, 1003, 3, 3), (True, 1003, 8, 5), (False, 9000, 1, 2), (True, 20001, 0, 1)])
def test_rows_at_any_distance(pkg, dev, bf16, V, at, out_at):
    say("adjust_logits strided", V, at, out_at)
    c = Case(V, [4, 1, 6], V, 50, bf16, True, biases=4, masked="rows")
    a = c.args(dev)
    want = pkg.adjust_logits(**a)
    wide = torch.full((c.T, V + 77), 9.0, dtype=c.x.dtype, device=dev)
    wide[:, at:at + V] = c.x.to(dev)
    out = torch.full((c.T, V + 61), 7.0, dtype=c.x.dtype, device=dev)
    history = torch.full((3, 90), 1, dtype=torch.int32, device=dev)
    history[:, 2:52] = a["history"]
    a.update(logits=wide[:, at:at + V], history=history[:, 2:52], out=out[:, out_at:out_at + V])
    pkg.adjust_logits(**a)
    torch.cuda.synchronize()
    assert torch.equal(out[:, out_at:out_at + V], want)
    assert bool((out[:, :out_at] == 7).all()) and bool((out[:, out_at + V:] == 7).all())
    a["out"] = a["logits"]
    pkg.adjust_logits(**a)
    assert torch.equal(wide[:, at:at + V], want) and bool((wide[:, :at] == 9).all()) and bool((wide[:, at + V:] == 9).all())


def test_the_last_of_equal_biases_counts(pkg, dev):
    x = torch.zeros(1, 100, device=dev)
    ids = torch.tensor([[7, 3, 7, 99, 3, 7]], dtype=torch.int32, device=dev)
    bias = torch.tensor([[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]], device=dev)
    for _ in range(3):
        y = pkg.adjust_logits(x, bias_ids=ids, bias=bias)
        assert y[0, 7] == 6 and y[0, 3] == 5 and y[0, 99] == 4 and y.count_nonzero() == 3


def test_a_row_each_without_cu_tokens(pkg, dev):
    c = Case(5, [1] * 9, 700, 30, True, biases=3, masked="own")
    a = c.args(dev)
    want = pkg.adjust_logits(**a)
    a["cu_tokens"] = None
    assert torch.equal(pkg.adjust_logits(**a), want)


def test_infinities_and_nan(pkg, dev):
    """A masked token is -inf whatever it held; penalties leave infinities and NaN what they are; neighbours are untouched."""
    x = torch.zeros(1, 64, device=dev)
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, math.inf, -math.inf, math.nan])
    history = torch.arange(6, dtype=torch.int32, device=dev)[None]
    allowed = torch.tensor([[~0b111000, ~0]], dtype=torch.int32, device=dev)
    two = torch.full((1,), 2.0, device=dev)
    y = pkg.adjust_logits(x, history=history, repetition=two, frequency=two, allowed=allowed).cpu()[0]
    assert y[0] == math.inf and y[1] == -math.inf and y[2].isnan() and bool((y[3:6] == -math.inf).all()) and bool((y[6:] == 0).all())
    low = torch.full((1, 64), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device=dev)     # a mask of the type's lowest value
    assert bool((pkg.adjust_logits(low, history=history, repetition=two)[0, :6] == -math.inf).all())


def test_streams_and_graphs(pkg, dev):
    say("adjust_logits streams, graphs")
    c = Case(12, [5, 1, 7], 9500, 80, True, True, biases=4, masked="rows")
    a = c.args(dev)
    want = pkg.adjust_logits(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.adjust_logits(**a)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.adjust_logits(**a, out=out)
    for lens in ([80, 3, 0], [0, 0, 0], [11, 80, 40]):
        a["history_lens"].copy_(torch.tensor(lens))
        eager = pkg.adjust_logits(**a)
        out.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), lens


def test_cu_tokens_out_of_order_end(pkg, dev):
    """Results are undefined there, but every launch ends and stays in bounds."""
    c = Case(13, [5, 1, 7], 300, 10, True, True)
    a = c.args(dev)
    for cu in ([9, 2, 5, 13], [0, 0, 99, 3], [-5, 200, 1, -7]):
        a["cu_tokens"].copy_(torch.tensor(cu))
        pkg.adjust_logits(**a)
    torch.cuda.synchronize()


@pytest.mark.parametrize("counts,V,L,bf16,tree,how", [
    # large enough for segments of 24 KB, and of 64 KB where rows have long histories
    ([1] * 40, 60001, 700, True, False, dict(masked="rows")), ([1] * 36, 131072, 4200, False, False, dict(biases=3)), ([3, 16, 5, 1], 100003, 500, True, True, dict(masked="own")),
    ([1] * 70, 130001, 4100, True, False, {}), ([7, 1], 262145, 60, False, True, {}),
    # of 24 KB again where there are more rows than that
    ([1] * 70, 131077, 300, False, False, dict(masked="rows", biases=3)), ([1] * 90, 200003, 4200, True, False, dict(masked="own")), ([1] * 72, 131072, 64, False, False, {})])
def test_large_vocabularies(pkg, dev, counts, V, L, bf16, tree, how):
    say("adjust_logits, large", len(counts), V, L, bf16)
    c = Case(V + L, counts, V, L, bf16, tree, **how)
    got = pkg.adjust_logits(**c.args(dev))
    torch.cuda.synchronize()
    c.check(got)


def test_texts_that_repeat_themselves(pkg, dev):
    """Thousands of equal tokens, of two in turn, of none; counted exactly."""
    x = torch.zeros(4, 9000, device=dev)
    history = torch.zeros(4, 5000, dtype=torch.int32, device=dev)
    history[0], history[1], history[2], history[3] = 7, 8191, -1, 8999
    history[1, ::2] = 3
    lens = torch.tensor([5000, 4999, 5000, 4097], dtype=torch.int32, device=dev)
    prompt = torch.tensor([0, 1030, 5, 4096], dtype=torch.int32, device=dev)
    one = torch.ones(4, device=dev)
    y = pkg.adjust_logits(x, history=history, history_lens=lens, prompt_lens=prompt, frequency=one)
    want = torch.zeros(4, 9000)
    want[0, 7], want[1, 3], want[1, 8191], want[3, 8999] = -5000, -1985, -1984, -1
    assert torch.equal(y.cpu(), want)


def test_tokens_beyond_32_bits_are_no_tokens(pkg, dev):
    x = torch.zeros(2, 50, device=dev)
    tokens = torch.tensor([(1 << 32) + 3, -(1 << 40)], device=dev)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=dev)
    for masks in (None, torch.tensor([1, 3], device=dev)):
        assert not pkg.adjust_logits(x, cu, tokens=tokens, masks=masks, presence=torch.ones(1, device=dev)).any()


@pytest.mark.parametrize("bf16,V", [(True, 1003), (False, 4096)])
def test_results_beside_what_they_come_from(pkg, dev, bf16, V):
    """Logits and results in the two halves of one buffer, where no row lies over another."""
    say("adjust_logits, two halves of a buffer", V)
    c = Case(V + 1, [3, 1, 4], V, 60, bf16, True, biases=3, masked="rows")
    a = c.args(dev)
    want = pkg.adjust_logits(**a)
    both = torch.full((c.T, 2 * V), 5.0, dtype=c.x.dtype, device=dev)
    for first in (0, V):
        both[:, first:first + V] = c.x.to(dev)
        a.update(logits=both[:, first:first + V], out=both[:, V - first:2 * V - first])
        assert torch.equal(pkg.adjust_logits(**a), want)
        assert torch.equal(both[:, first:first + V].cpu(), c.x)
    a.update(logits=both[:, :V], out=both[:, 1:V + 1])
    with pytest.raises(RuntimeError):
        pkg.adjust_logits(**a)


@pytest.mark.parametrize("counts,V,L,bf16,tree,how,most", [
    # every size of segment in both types: rows on 16 bytes and beside them, trees, grammars, biases
    ([1] * 41, 131072, 4200, True, False, dict(masked="rows", biases=3), 64), ([1] * 45, 130001, 4100, True, False, {}, 64), ([1] * 24, 131072, 4096, False, False, dict(masked="own"), 64),
    ([1] * 22, 130007, 5000, False, False, dict(biases=9), 64), ([16, 3, 22, 4], 131072, 4100, True, True, dict(masked="rows"), 64), ([1] * 128, 32000, 8192, False, False, {}, 64),
    ([1] * 130, 32000, 8192, False, False, {}, 24), ([1] * 250, 64001, 8192, True, False, {}, 64), ([1] * 66, 131072, 4096, True, False, {}, 24), ([1] * 33, 131072, 4200, False, False, dict(masked="rows"), 24),
    ([1] * 12, 131072, 8192, False, False, {}, 24), ([1] * 11, 131072, 8192, False, False, {}, 16), ([1] * 20, 131072, 5000, True, False, dict(biases=2), 16)])
def test_segments_of_every_size(pkg, dev, counts, V, L, bf16, tree, how, most):
    say("adjust_logits, segments of", most, "KB:", len(counts), V, L, bf16)
    c = Case(V + L, counts, V, L, bf16, tree, **how)
    assert pkg._lib.lib.moe_adjust_logits_segment_bytes(1 if bf16 else 0, c.T, V, L) == most << 10
    got = pkg.adjust_logits(**c.args(dev))
    torch.cuda.synchronize()
    c.check(got)
