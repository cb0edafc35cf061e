"""The serving step's operators without a GPU: what the C entry points and the registered ops refuse, and the plain forms that
the GPU tests compare with, on cases small enough to be seen."""
import ctypes
import math
import os
import subprocess

import pytest
import torch

import serving_plain as plain
from isa_hazards import scratch_bytes

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

E_NULL, E_SHAPE, E_ALIGN, E_WS, E_MODE = -1, -2, -3, -4, -5
fake = ctypes.c_void_p(0x10000)              # never dereferenced: validation fails first
odd = ctypes.c_void_p(0x10002)


def lib():
    from torch_tpu_amd._lib import lib as it
    return it


def test_cache_plan_refusals(pkg):
    names = ["tables", "stride", "B", "W", "lens", "counts", "free", "F", "n_free", "page", "parents", "T", "cu", "pos", "slots", "masks", "kv", "left"]
    good = dict(tables=fake, stride=8, B=2, W=8, lens=fake, counts=fake, free=fake, F=4, n_free=fake, page=16, parents=None, T=4, cu=fake,
                pos=fake, slots=fake, masks=None, kv=fake, left=odd)

    def call(**other):
        a = {**good, **other}
        return lib().moe_cache_plan(None, *[a[n] for n in names])
    for bad in (dict(B=-1), dict(B=4097), dict(W=-1), dict(F=-1), dict(T=-1), dict(page=0), dict(page=24), dict(page=2048), dict(stride=7),
                dict(W=1 << 28, stride=1 << 28)):
        assert call(**bad) == E_SHAPE, bad
    for name in ("tables", "lens", "counts", "free", "n_free", "cu", "pos", "slots", "kv", "left"):
        assert call(**{name: None}) == E_NULL, name
    assert call(parents=fake) == E_NULL       # masks are missing
    assert call(left=fake) == E_MODE          # the count read and the count written are one


def test_cache_plan_refuses_results_over_what_it_reads(pkg):
    """Every workgroup reads the lengths while another writes results already: lengths updated in place would be a race."""
    read = dict(lens=8, counts=8, free=16, n_free=4, parents=16)
    written = dict(cu=12, pos=16, slots=32, masks=32, kv=8, left=4, tables=4 * (8 + 6))
    names = ["tables", "stride", "B", "W", "lens", "counts", "free", "F", "n_free", "page", "parents", "T", "cu", "pos", "slots", "masks", "kv", "left"]
    at = {n: 0x10000 + 0x1000 * i for i, n in enumerate([*read, *written])}

    def call(**moved):
        a = {**dict(stride=8, B=2, W=6, F=4, page=16, T=4), **{n: ctypes.c_void_p(p) for n, p in {**at, **moved}.items()}}
        return lib().moe_cache_plan(None, *[a[n] for n in names])
    for r, size in read.items():
        for w, wide in written.items():
            for moved in (at[r], at[r] + size - 4, at[r] - wide + 4):             # at its start, on its last value, its first value under the last result
                assert call(**{w: moved}) == E_MODE, (r, w, moved - at[r])


def test_qk_norm_rope_refusals(pkg):
    names = ["qkv", "stride", "T", "Hq", "Hkv", "D", "pos", "cs", "P", "R", "pairs", "qw", "kw", "wt", "eps", "q", "k", "kc", "vc", "ct", "blocks",
             "ks", "vs", "page", "slots", "kscale", "vscale"]
    good = dict(qkv=fake, stride=8 * 128, T=2, Hq=4, Hkv=2, D=128, pos=fake, cs=fake, P=10, R=128, pairs=0, qw=fake, kw=fake, wt=1, eps=1e-6, q=fake,
                k=None, kc=fake, vc=fake, ct=1, blocks=3, ks=16 * 256, vs=16 * 256, page=16, slots=fake, kscale=None, vscale=None)

    def call(**other):
        a = {**good, **other}
        return lib().moe_qk_norm_rope(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(Hq=0), dict(Hkv=0), dict(D=0), dict(D=264, stride=8 * 264), dict(R=144), dict(stride=1000), dict(P=-1),
                dict(page=24), dict(page=0), dict(blocks=-1), dict(ks=100), dict(vs=100)):
        assert call(**bad) == E_SHAPE, bad
    for bad in (dict(D=100, stride=8 * 104, R=96, ks=1 << 16, vs=1 << 16), dict(R=24), dict(stride=8 * 128 + 4), dict(ks=16 * 256 + 4), dict(qkv=odd), dict(q=odd), dict(kc=odd), dict(qw=odd)):
        assert call(**bad) == E_ALIGN, bad
    assert call(wt=2) == E_MODE and call(ct=0) == E_MODE
    for bad in (dict(qkv=None), dict(pos=None), dict(cs=None), dict(q=None), dict(vc=None), dict(kc=None), dict(slots=None)):
        assert call(**bad) == E_NULL, bad
    assert call(T=0, qkv=None, pos=None, q=None) == 0


def test_tree_attention_refusals(pkg):
    names = ["q", "qs", "T", "Hq", "Hkv", "D", "kc", "vc", "ct", "blocks", "ks", "vs", "page", "bt", "bts", "W", "lens", "cu", "B", "masks", "scale",
             "kscale", "vscale", "out", "lse", "ws", "wsb"]
    ws = lib().moe_tree_attention_workspace_bytes(4, 8, 2, 128, 3, 1)
    assert ws > 0 and ws % 256 == 0
    good = dict(q=fake, qs=1024, T=4, Hq=8, Hkv=2, D=128, kc=fake, vc=fake, ct=1, blocks=5, ks=16 * 256, vs=16 * 256, page=16, bt=fake, bts=4, W=4,
                lens=fake, cu=fake, B=3, masks=None, scale=0.1, kscale=None, vscale=None, out=fake, lse=None, ws=fake, wsb=ws)

    def call(**other):
        a = {**good, **other}
        return lib().moe_tree_attention(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(Hq=0), dict(Hkv=3), dict(D=96), dict(B=-1), dict(B=5000), dict(page=12), dict(qs=1000), dict(bts=3), dict(ks=128),
                dict(W=1 << 28, bts=1 << 28), dict(blocks=-1)):
        assert call(**bad) == E_SHAPE, bad
    for bad in (dict(q=odd), dict(kc=odd), dict(out=odd), dict(qs=1028), dict(ks=16 * 256 + 8), dict(ws=odd)):
        assert call(**bad) == E_ALIGN, bad
    assert call(ct=0) == E_MODE
    assert call(wsb=ws - 1) == E_WS
    for name in ("q", "kc", "vc", "bt", "lens", "cu", "out", "ws"):
        assert call(**{name: None}) == E_NULL, name
    assert call(T=0, q=None, out=None) == 0
    assert lib().moe_tree_attention_workspace_bytes(4, 8, 3, 128, 3, 1) == 0
    assert lib().moe_tree_attention_workspace_bytes(4, 8, 2, 128, 3, 0) == 0


def test_token_logprobs_refusals(pkg):
    names = ["x", "dt", "stride", "T", "V", "tok", "k", "temp", "lp", "ent", "top", "ids", "ws", "wsb"]
    ws = lib().moe_token_logprobs_workspace_bytes(2, 100000, 5, 1)
    good = dict(x=fake, dt=1, stride=100000, T=2, V=100000, tok=fake, k=5, temp=1.0, lp=fake, ent=fake, top=fake, ids=fake, ws=fake, wsb=ws)

    def call(**other):
        a = {**good, **other}
        return lib().moe_token_logprobs(None, *[a[n] for n in names])
    for bad in (dict(T=-1), dict(V=0), dict(k=-1), dict(k=33), dict(V=3, k=4), dict(stride=99999), dict(temp=0.0), dict(temp=-1.0),
                dict(temp=math.nan), dict(temp=math.inf), dict(temp=1e-38)):
        assert call(**bad) == E_SHAPE, bad
    assert call(dt=2) == E_MODE
    assert call(wsb=ws - 1) == E_WS
    assert call(x=ctypes.c_void_p(0x10001)) == E_ALIGN
    for name in ("x", "tok", "lp", "ent", "top", "ids", "ws"):
        assert call(**{name: None}) == E_NULL, name
    assert call(T=0, x=None) == 0
    assert lib().moe_token_logprobs_workspace_bytes(2, 0, 5, 1) == 0


def test_ops_refuse_tensors_that_are_not_on_the_gpu(pkg):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.cache_plan(i32(2, 3), i32(2), i32(2), i32(4), i32(1), 16, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.qk_norm_rope(bf(2, 8 * 64), i32(2), torch.zeros(4, 64), 4, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.tree_attention(bf(2, 4, 64), bf(3, 16, 2, 64), bf(3, 16, 2, 64), i32(1, 3), i32(1), i32(2))
    with pytest.raises(RuntimeError, match="GPU"):
        pkg.token_logprobs(bf(2, 100), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="bfloat16"):
        pkg.tree_attention(torch.zeros(2, 4, 64), bf(3, 16, 2, 64), bf(3, 16, 2, 64), i32(1, 3), i32(1), i32(2))


def test_plain_plan_by_hand():
    # 3 of 4 places of block 7 are taken; two new tokens: one more there, one in the new block 5 (the stack's top)
    got = plain.plan([[7, -1]], [3], [2], [4, 5], 2, 4, 3)
    assert got == ([[7, 5]], [0, 2], [3, 4, -1], [31, 20, -1], None, [5], 1)
    # a tree: 0 and 1 follow the text, 2 follows 0
    got = plain.plan([[7]], [0], [3], [], 0, 4, 3, [-1, -1, 0])
    assert got[1:] == ([0, 3], [-1] * 3, [-1] * 3, [0] * 3, [0], 0)          # no page left
    got = plain.plan([[-1]], [0], [3], [9], 1, 4, 3, [-1, -1, 0])
    assert got == ([[9]], [0, 3], [0, 0, 1], [36, 37, 38], [1, 2, 5], [3], 0)


def test_plain_attention_is_the_softmax_of_what_is_seen():
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(2, 2, 8, generator=g), torch.randn(3, 2, 1, 8, generator=g), torch.randn(3, 2, 1, 8, generator=g)
    out, lse, _ = plain.attention(q, k, v, [[2, 0]], [4], [0, 2], [0b01, 0b10], 0.5)
    keys = torch.stack([k[2, 0, 0], k[2, 1, 0], k[0, 0, 0]]).double()
    vals = torch.stack([v[2, 0, 0], v[2, 1, 0], v[0, 0, 0]]).double()
    s = keys @ q[0, 1].double() * 0.5
    assert torch.allclose(out[0, 1], torch.softmax(s, 0) @ vals) and torch.allclose(lse[0, 1], torch.logsumexp(s, 0))


@pytest.mark.parametrize("source", ["cache_plan.hip", "qk_norm_rope.hip", "tree_attention.hip", "token_logprobs.hip"])
def test_no_kernel_spills(source, tmp_path):
    hipcc = "/opt/rocm/bin/hipcc" if os.path.exists("/opt/rocm/bin/hipcc") else "hipcc"
    out = tmp_path / (source + ".s")
    cmd = [hipcc, "--offload-arch=gfx950", "--cuda-device-only", "-O3", "-std=c++17", "-S", "-Wno-inline-asm",
           "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
           os.path.join(ROOT, "torch-tpu_amd", "csrc", source), "-o", str(out)]
    r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    if r.returncode != 0:
        pytest.fail("hipcc failed:\n" + r.stdout[-2000:])
    sizes = scratch_bytes(out.read_text())
    assert sizes, "no kernel found"
    spills = {n: b for n, b in sizes.items() if b}
    assert not spills, f"kernels spill to scratch: {spills}"


@pytest.mark.parametrize("T,Hq,Hkv,B,trees,room,rows", [
    (64, 32, 4, 64, False, 8192, 16), (128, 32, 4, 64, True, 8192, 16), (64, 32, 32, 1, True, 131072, 64), (384, 32, 4, 64, True, 8192, 64),
    (768, 32, 4, 64, True, 32768, 128), (512, 32, 4, 32, True, 32768, 128), (512, 32, 4, 32, True, 1024, 64), (1024, 32, 4, 16, True, 32768, 256),
    (2042, 32, 8, 2, False, 8192, 256), (200, 32, 8, 2, False, 1024, 64), (0, 4, 2, 0, False, 0, 16)])
def test_tile_rows_by_rows_and_room(pkg, T, Hq, Hkv, B, trees, room, rows):
    for dtype in (1, 2):
        assert lib().moe_tree_attention_tile_rows(T, Hq, Hkv, B, dtype, trees, room // 16, 16) == rows


def test_tile_rows_of_refused_shapes(pkg):
    for bad in ((-1, 4, 2, 1, 1, 0, 4, 16), (1, 4, 3, 1, 1, 0, 4, 16), (1, 0, 1, 1, 1, 0, 4, 16), (1, 4, 2, 4097, 1, 0, 4, 16), (1, 4, 2, 1, 0, 0, 4, 16),
                (1, 4, 2, 1, 1, 0, -1, 16), (1, 4, 2, 1, 1, 0, 4, 24), (1, 4, 2, 1, 1, 0, 4, 2048)):
        assert lib().moe_tree_attention_tile_rows(*bad) == 0, bad
