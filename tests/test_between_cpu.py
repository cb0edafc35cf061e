"""residual_norm and adjust_logits without a GPU: refusals, and the plain forms on cases small enough to be seen."""
import ctypes
import math

import pytest
import torch

import between_plain as plain
from test_serving_cpu import E_ALIGN, E_MODE, E_NULL, E_SHAPE, fake, lib, odd, test_no_kernel_spills as no_kernel_spills

at = lambda n: ctypes.c_void_p(0x100000 * n)


def test_residual_norm_refusals(pkg):
    names = ["x", "xs", "T", "H", "res", "rt", "rs", "w", "pw", "wt", "gate", "gt", "gr", "gc", "scale", "eps", "y", "ys", "h", "hs"]
    good = dict(x=at(1), xs=256, T=4, H=256, res=at(2), rt=1, rs=256, w=at(3), pw=at(4), wt=1, gate=at(5), gt=1, gr=256, gc=1, scale=1.0, eps=1e-6,
                y=at(6), ys=256, h=at(7), hs=256)

    def call(**other):
        a = {**good, **other}
        return lib().moe_residual_norm(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(H=0), dict(H=32769, xs=40000, ys=40000, rs=40000, hs=40000, gr=40000), dict(xs=255), dict(ys=255), dict(rs=255), dict(hs=255),
                dict(eps=-1.0), dict(eps=math.nan), dict(gc=2), dict(gr=-1), dict(gr=255)):
        assert call(**bad) == E_SHAPE, bad
    for bad in (dict(rt=2), dict(wt=2), dict(gt=3)):
        assert call(**bad) == E_MODE, bad
    for bad in (dict(x=None), dict(y=None)):
        assert call(**bad) == E_NULL, bad
    for bad in (dict(x=ctypes.c_void_p(0x100001)), dict(res=ctypes.c_void_p(0x200002), rt=0), dict(gate=ctypes.c_void_p(0x500002), gt=0),
                dict(H=16385, xs=20000, ys=20000, rs=20000, hs=20000, gr=20000), dict(H=20000, xs=20001, ys=20000, rs=20000, hs=20000, gr=20000)):
        assert call(**bad) == E_ALIGN, bad
    row = lambda p, n: ctypes.c_void_p(p.value + 2 * n)
    # over what is read, but not row on row
    for bad in (dict(y=row(at(1), 8)), dict(y=row(at(1), -8)), dict(y=at(3)), dict(y=row(at(5), 1016)), dict(h=row(at(2), 1)),
                dict(h=at(6)), dict(h=at(4)), dict(y=row(at(1), -1016)), dict(y=at(1), ys=264)):
        assert call(**bad) == E_MODE, bad
    assert call(T=0, x=None, y=None) == 0


def test_adjust_logits_refusals(pkg):
    names = ["x", "dt", "xs", "T", "V", "cu", "B", "hist", "hs", "L", "lens", "asked", "tok", "masks", "rep", "freq", "pres", "bi", "bis", "bv", "bvs", "nb",
             "al", "als", "na", "rows", "out", "os"]
    good = dict(x=at(1), dt=1, xs=1000, T=4, V=1000, cu=at(3), B=2, hist=at(4), hs=50, L=50, lens=at(5), asked=at(5), tok=at(6), masks=at(7), rep=at(8),
                freq=at(8), pres=at(8), bi=at(9), bis=5, bv=at(10), bvs=5, nb=5, al=at(11), als=32, na=3, rows=at(12), out=at(2), os=1000)

    def call(**other):
        a = {**good, **other}
        return lib().moe_adjust_logits(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(V=0), dict(B=-1), dict(L=-1), dict(nb=-1), dict(nb=2048, bis=3000, bvs=3000), dict(xs=999), dict(os=999), dict(na=-1), dict(cu=None),
                dict(hs=49), dict(bis=4), dict(bvs=4), dict(als=31), dict(rows=None), dict(L=(1 << 20) - 4, hs=1 << 20)):
        assert call(**bad) == E_SHAPE, bad
    assert call(dt=2) == E_MODE
    for bad in (dict(x=None), dict(out=None), dict(bi=None), dict(bv=None), dict(tok=None)):
        assert call(**bad) == E_NULL, bad
    assert call(x=ctypes.c_void_p(0x100001)) == E_ALIGN and call(out=odd, dt=0) == E_ALIGN
    for bad in (dict(out=ctypes.c_void_p(0x100002)), dict(out=ctypes.c_void_p(0x100000 - 7998)), dict(out=at(1), os=1001)):
        assert call(**bad) == E_MODE, bad
    assert call(T=0, x=None, out=None) == 0


def test_ops_refuse_what_does_not_fit(pkg):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.residual_norm(bf(2, 8))
    with pytest.raises(RuntimeError, match="bfloat16"):
        pkg.residual_norm(torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.adjust_logits(bf(2, 8))
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        pkg.adjust_logits(torch.zeros(2, 8, dtype=torch.float16))


@pytest.mark.parametrize("source", ["residual_norm.hip", "adjust_logits.hip"])
def test_no_kernel_spills(source, tmp_path):
    no_kernel_spills(source, tmp_path)


def test_plain_residual_norm_by_hand():
    x, r = torch.tensor([[3.0, 4.0]]), torch.tensor([[1.0, 1.0]])
    y, h, reach = plain.residual_norm(x, r, torch.tensor([1.0, 2.0]), None, torch.tensor([2.0, 0.0]), 0.5, 0.0)
    assert h.tolist() == [[4.0, 1.0]] and reach.tolist() == [[4.0, 1.0]]
    assert torch.allclose(y, torch.tensor([[4.0, 2.0]]).double() / math.sqrt(8.5))
    y, h, _ = plain.residual_norm(x, None, None, torch.tensor([1.0, 1.0]), None, 1.0, 0.0)
    assert torch.allclose(h, x.double() / math.sqrt(12.5)) and torch.allclose(y, h)


def test_plain_adjust_logits_by_hand():
    x = torch.tensor([[2.0, -2.0, 2.0, 1.0, 1.0]], dtype=torch.float64)
    out, _ = plain.adjust_logits(x, None, [[0, 1, 2, 2, 7]], None, [1], None, None, [2.0], [0.25], [0.5], [[3, 4, 3]], [[9.0, 1.0, 2.0]], [[0b01111]], None)
    # 0 in the prompt only; 1 once; 2 twice; 3 biased by the last of its two; 4 not allowed
    assert out.tolist() == [[1.0, -4.75, 0.0, 3.0, -math.inf]]
    # the path of the second drafted token: itself and the first
    out, _ = plain.adjust_logits(x.repeat(3, 1), [0, 3], None, None, None, [0, 2, 3], [1, 3, 4], [2.0], None, None, None, None, None, None)
    assert out[:, [0, 2, 3]].tolist() == [[1.0, 2.0, 1.0], [1.0, 1.0, 1.0], [2.0, 2.0, 0.5]]
