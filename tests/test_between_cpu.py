"""residual_norm and adjust_logits without a GPU: refusals, and the plain forms on cases small enough to be seen."""
import ctypes
import math

import pytest
import torch

import between_plain as plain
from test_serving_cpu import E_ALIGN, E_MODE, E_NULL, E_SHAPE, E_WS, fake, lib, odd, test_no_kernel_spills as no_kernel_spills

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
    for bad in (dict(x=ctypes.c_void_p(0x100001)), dict(res=ctypes.c_void_p(0x200002), rt=0), dict(gate=ctypes.c_void_p(0x500002), gt=0)):
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
    for bad in (dict(T=-1), dict(V=0), dict(B=-1), dict(L=-1), dict(nb=-1), dict(nb=1024, bis=3000, bvs=3000), dict(xs=999), dict(os=999), dict(na=-1), dict(cu=None),
                dict(hs=49), dict(bis=4), dict(bvs=4), dict(als=31), dict(rows=None), dict(L=(1 << 20) - 4, hs=1 << 20)):
        assert call(**bad) == E_SHAPE, bad
    assert call(dt=2) == E_MODE
    for bad in (dict(x=None), dict(out=None), dict(bi=None), dict(bv=None), dict(tok=None)):
        assert call(**bad) == E_NULL, bad
    assert call(x=ctypes.c_void_p(0x100001)) == E_ALIGN and call(out=odd, dt=0) == E_ALIGN
    for bad in (dict(out=ctypes.c_void_p(0x100002)), dict(out=ctypes.c_void_p(0x100000 - 7998)), dict(out=at(1), os=1001)):
        assert call(**bad) == E_MODE, bad
    for name in ("cu", "hist", "lens", "asked", "tok", "masks", "rep", "freq", "pres", "bi", "bv", "al", "rows"):       # out over what is read
        for there in (0x200000, 0x200000 + 7992, 0x200000 - 4):
            assert call(**{name: ctypes.c_void_p(there)}) == E_MODE, (name, there)
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


def test_window_attention_refusals(pkg):
    names = ["q", "qs", "T", "Hq", "Hkv", "D", "kc", "vc", "ct", "blocks", "ks", "vs", "page", "bt", "bts", "W", "lens", "cu", "B", "masks", "scale",
             "kscale", "vscale", "kss", "vss", "window", "sinks", "out", "lse", "ws", "wsb"]
    ws = lib().moe_tree_attention_workspace_bytes(4, 8, 2, 128, 3, 3)
    assert ws > 0 and ws % 256 == 0
    good = dict(q=fake, qs=1024, T=4, Hq=8, Hkv=2, D=128, kc=fake, vc=fake, ct=3, blocks=5, ks=16 * 256, vs=16 * 256, page=16, bt=fake, bts=4, W=4,
                lens=fake, cu=fake, B=3, masks=None, scale=0.1, kscale=fake, vscale=fake, kss=128, vss=128, window=5, sinks=1, out=fake, lse=None, ws=fake, wsb=ws)

    def call(**other):
        a = {**good, **other}
        return lib().moe_window_attention(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(Hkv=3), dict(D=96), dict(B=5000), dict(page=12), dict(qs=1000), dict(bts=3), dict(ks=128), dict(kss=127), dict(vss=127),
                dict(kss=1 << 31), dict(window=-1), dict(sinks=-1), dict(blocks=-1)):
        assert call(**bad) == E_SHAPE, bad
    for bad in (dict(q=odd), dict(kc=odd), dict(out=odd), dict(ks=16 * 256 + 16), dict(ws=odd)):
        assert call(**bad) == E_ALIGN, bad
    assert call(ct=0) == E_MODE and call(ct=4) == E_MODE
    assert call(wsb=ws - 1) == E_WS
    for name in ("q", "kc", "vc", "bt", "lens", "cu", "out", "ws", "kscale", "vscale"):
        assert call(**{name: None}) == E_NULL, name
    assert call(T=0, q=None, out=None) == 0
    rows = lambda *a: lib().moe_window_attention_tile_rows(*a)
    assert rows(64, 32, 4, 64, 3, 0, 512, 16, 0, 0) == 16 and rows(2042, 32, 8, 2, 1, 0, 512, 16, 0, 0) == 256 and rows(200, 32, 8, 2, 1, 0, 8192, 16, 500, 4) == 64
    for bad in ((-1, 4, 2, 1, 1, 0, 4, 16, 1, 0), (1, 4, 2, 1, 4, 0, 4, 16, 1, 0), (1, 4, 2, 1, 1, 0, 4, 16, -1, 0), (1, 4, 2, 1, 1, 0, 4, 16, 1, -1)):
        assert rows(*bad) == 0


def test_store_in_four_bits_refusals(pkg):
    names = ["qkv", "stride", "T", "Hq", "Hkv", "D", "pos", "cs", "P", "R", "pairs", "qw", "kw", "wt", "eps", "q", "kc", "vc", "blocks",
             "ks", "vs", "page", "slots", "kscale", "vscale", "kss", "vss"]
    good = dict(qkv=fake, stride=8 * 128, T=2, Hq=4, Hkv=2, D=128, pos=fake, cs=fake, P=10, R=128, pairs=0, qw=fake, kw=fake, wt=1, eps=1e-6, q=fake,
                kc=fake, vc=fake, blocks=3, ks=16 * 256, vs=16 * 256, page=16, slots=fake, kscale=fake, vscale=fake, kss=128, vss=128)

    def call(**other):
        a = {**good, **other}
        return lib().moe_qk_norm_rope_fp4(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(D=0), dict(page=24), dict(ks=100), dict(kss=127), dict(vss=0)):
        assert call(**bad) == E_SHAPE, bad
    for bad in (dict(D=112, stride=1024, R=96), dict(ks=16 * 256 + 8), dict(kc=odd)):
        assert call(**bad) == E_ALIGN, bad
    for name in ("qkv", "pos", "q", "kc", "vc", "slots", "kscale", "vscale"):
        assert call(**{name: None}) == E_NULL, name
    assert call(T=0, qkv=None, pos=None, q=None) == 0


def test_ops_refuse_caches_that_do_not_fit(pkg):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.tree_attention(bf(2, 4, 64), bf(3, 16, 2, 64), bf(3, 16, 2, 64), i32(1, 3), i32(1), i32(2), window=4)


def test_no_window_kernel_spills(tmp_path):
    no_kernel_spills("window_attention.hip", tmp_path)


def test_four_bits_by_hand():
    import window_plain as window
    x = torch.zeros(32, dtype=torch.float64)
    x[:6] = torch.tensor([7.0, -6.9, 5.0, 0.25, 0.75, -0.24])
    codes, powers = window.encode(x)
    assert powers.tolist() == [127] and codes.tolist()[:3] == [0xf7, 0x06, 0x82]      # 5 and 0.25 are ties: to 4 and 0; -0.24 to -0
    assert window.decode(codes, powers).tolist()[:6] == [6.0, -6.0, 4.0, 0.0, 1.0, 0.0]
    x[0] = 7.5
    codes, powers = window.encode(x)
    assert powers.tolist() == [128] and window.decode(codes, powers).tolist()[:3] == [8.0, -6.0, 4.0]


def test_plain_window_by_hand():
    import window_plain as window
    q, k = torch.zeros(2, 1, 4), torch.zeros(2, 4, 1, 4).double()
    v = torch.arange(8.0)[:, None].expand(8, 4).reshape(2, 4, 1, 4).double()
    # rows see 0 .. 4 and 0 .. 5; of these the last two and the first one
    out, lse, _ = window.attention(q, k, v, [[0, 1]], [6], [0, 2], None, 1.0, 2, 1)
    assert torch.allclose(out[:, 0, 0], torch.tensor([(0 + 3 + 4) / 3, (0 + 4 + 5) / 3]).double()) and torch.allclose(lse, torch.tensor(3.0).double().log())
    # a tree whose second token does not see the first
    out, _, _ = window.attention(q, k, v, [[0, 1]], [6], [0, 2], [0b01, 0b10], 1.0, 2, 0)
    assert torch.allclose(out[:, 0, 0], torch.tensor([(3 + 4) / 2, (3 + 5) / 2]).double())


def test_attention_workspaces(pkg):
    """Calls without a window ask for one head's parts; with one for two heads' where two share a workgroup."""
    of = lambda groups, heads, D=128: 2 * groups * 16 * heads * (D * 4 + 8) + groups * 32
    tree, window = lib().moe_tree_attention_workspace_bytes, lib().moe_window_attention_workspace_bytes
    for B in (64, 256):
        assert tree(B, 32, 4, 128, B, 1) == of(256, 1) and tree(B, 32, 4, 128, B, 2) == of(512, 1)
        assert tree(B, 32, 4, 64, B, 1) == of(256, 1, 64)
        assert window(B, 32, 4, 128, B, 1) == of(256 if B == 64 else 512, 2) and window(B, 32, 4, 128, B, 2) == of(512, 2)
        assert tree(B, 32, 4, 128, B, 3) == window(B, 32, 4, 128, B, 3) == of(512, 2)
    for T in (1, 7, 64, 1000, 5000):                       # a window asks for no less, and over a 4-bit cache there is no other call
        for B in (1, 3, 40):
            for cache in (1, 2, 3):
                assert window(T, 8, 2, 128, B, cache) >= tree(T, 8, 2, 128, B, cache) > 0
    assert window(4, 8, 3, 128, 3, 1) == 0 and window(4, 8, 2, 128, 3, 0) == 0 and window(4, 8, 2, 128, 3, 4) == 0


def test_which_calls_take_two_heads_to_a_workgroup(pkg):
    heads = lambda *a: lib().moe_window_attention_heads(*a)
    # 64 single tokens over 4 heads: in 4 bits, in a wide window, in a narrow one; one token; an odd number of heads; trees of many rows
    assert heads(64, 32, 4, 64, 3, 0, 512, 16, 0, 0) == 2 and heads(64, 32, 4, 64, 1, 0, 1024, 16, 8000, 4) == 2 and heads(64, 32, 4, 64, 1, 0, 1024, 16, 500, 4) == 1
    assert heads(1, 32, 4, 1, 3, 0, 2048, 16, 0, 0) == 1 and heads(64, 24, 3, 64, 3, 0, 512, 16, 0, 0) == 1 and heads(512, 32, 4, 8, 3, 1, 512, 16, 0, 0) == 1
    for bad in ((-1, 4, 2, 1, 1, 0, 4, 16, 1, 0), (1, 4, 2, 1, 4, 0, 4, 16, 1, 0), (1, 4, 2, 1, 1, 0, 4, 16, -1, 0), (1, 4, 2, 1, 1, 0, 4, 16, 1, -1)):
        assert heads(*bad) == 0


def test_four_bits_are_off_by_a_fifth_at_most():
    """The power leaves the largest of 32 elements above 3.5 and at most 7.  Up to 4 a value is off by 1 / 2 at most, above by 1: a fifth of the
    largest at most, which the tie at 5 reaches."""
    import window_plain as window
    off = lambda x: ((window.decode(*window.encode(x)) - x).abs() / x.abs().amax(-1, keepdim=True)).amax(-1)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20000, 32, generator=g).double() * torch.exp2(torch.randint(-30, 30, (20000, 1), generator=g).double())
    assert off(x).max() <= 0.2 and (off(x) > 1 / 7).double().mean() > 0.2
    top = torch.linspace(3.5, 7, 7001, dtype=torch.float64)[1:]
    alone = torch.zeros(len(top), 32, dtype=torch.float64)
    alone[:, 5] = top
    assert off(alone).max() == 0.2 and top[off(alone).argmax()] == 5
    assert off(alone)[top <= 4].max() <= 1 / 7 and off(alone)[top >= 6].max() <= 1 / 7


def test_launches_of_too_many_threads_are_refused(pkg):
    """Of 2^32 threads and more: by the entry points, not by the launch (nor cut off by it)."""
    far = lambda n: ctypes.c_void_p(n << 44)
    norm = lambda T, H: lib().moe_residual_norm(None, far(1), H, T, H, far(2), 1, H, None, None, 1, None, 1, 0, 0, 1.0, 1e-6, far(3), H, far(4), H)
    for T, H in ((1 << 22, 8192), (1 << 22, 4104), (1 << 26, 512), (1 << 25, 1024), ((1 << 31) - 1, 1), (1 << 22, 32768)):
        assert norm(T, H) == E_SHAPE, (T, H)
    assert lib().moe_adjust_logits(None, far(1), 0, 1 << 20, (1 << 20) - 1, 1 << 20, None, (1 << 20) - 1, *[None, 0, 0], *[None] * 7, None, 0, None, 0, 0, None, 0, 0, None,
                                   far(3), 1 << 20) == E_SHAPE
    assert lib().moe_qk_norm_rope(None, far(1), 24, 1 << 30, 1, 1, 8, far(2), None, 0, 0, 0, None, None, 1, 1e-6, far(3), None, None, None, 1, 0, 0, 0, 1, None, None,
                                  None) == E_SHAPE


def host_check(tmp_path, name, said):
    """Builds tests/<name>.cpp with g++ and its sanitizers, and runs it."""
    import os
    import shutil
    import subprocess
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    exe, src = tmp_path / name, os.path.join(os.path.dirname(os.path.abspath(__file__)), name + ".cpp")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-static-libasan", src, "-o", str(exe)],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout[-3000:]
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert r.returncode == 0 and said in r.stdout, r.stdout[-3000:]


def test_keys_that_no_row_sees_are_not_read(tmp_path):
    """The arithmetic of a tile's way over the keys against what every row sees."""
    host_check(tmp_path, "host_reach_check", "reach checks passed")


def test_rows_between_rows(tmp_path):
    """What tells whether results lie over what is read, against a look at every byte."""
    host_check(tmp_path, "host_rows_check", "row checks passed")


def test_segments_of_logits(pkg):
    """64 KB to a workgroup where these fill the chip once or twice and histories are long; never for rows that leave them empty."""
    of = lambda *a: lib().moe_adjust_logits_segment_bytes(*a)
    for (T, V, L, bf16), kb in {(1, 131072, 4096, 1): 16, (32, 131072, 8192, 1): 24, (20, 131072, 8192, 1): 16, (40, 131072, 8192, 1): 64, (64, 131072, 8192, 1): 64,
                                (65, 131072, 8192, 1): 24, (80, 131072, 8192, 1): 24, (96, 131072, 8192, 1): 24, (128, 131072, 8192, 1): 64, (128, 131072, 8191, 1): 24,
                                (129, 131072, 8192, 1): 24, (160, 100003, 4096, 1): 24, (64, 131072, 8192, 0): 64, (64, 131072, 4096, 0): 24, (64, 131072, 4095, 1): 24,
                                (64, 131072, 0, 1): 24, (256, 1000, 8192, 1): 16, (512, 17000, 8192, 1): 24, (200, 33000, 8192, 1): 24}.items():
        assert of(bf16, T, V, L) == kb << 10, (T, V, L, bf16)
    for bad in ((2, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1 << 30, 1), (1, 1, 1, -1)):
        assert of(*bad) == 0
