"""residual_norm on the GPU against its plain 64-bit form, at the widths, types and layouts where it can go wrong."""
import pytest
import torch

import between_plain as plain

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def make(T, H, seed, wide=False, gate=None, gate_f32=False, weights="both", weights_f32=False):
    g = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g)
    x = (randn(T, H) * (0.1 + 4 * torch.rand(T, 1, generator=g))).to(torch.bfloat16)
    residual = randn(T, H) * 2
    residual[:, ::37] *= 30
    wt = lambda: (1 + 0.3 * randn(H)).to(torch.float32 if weights_f32 else torch.bfloat16)
    shape = {None: None, "column": (H,), "row": (1, H), "token": (T, 1), "one": (1, 1), "full": (T, H)}[gate]
    return dict(x=x, residual=residual if wide else residual.to(torch.bfloat16), weight=wt() if weights in ("both", "weight") else None,
                post_weight=wt() if weights in ("both", "post") else None,
                gate=None if shape is None else randn(*shape).to(torch.float32 if gate_f32 else torch.bfloat16))


def check(a, got, scale, eps):
    y, h = got
    want_y, want_h, reach = plain.residual_norm(a["x"], a["residual"], a["weight"], a["post_weight"], a["gate"], scale, eps)
    wide = h.dtype == torch.float32
    off_y, off_h = plain.residual_norm_bounds(want_y, want_h, reach, a["weight"], eps, plain.U32 if wide else plain.U16)
    for what, g, w, most in (("y", y, want_y, off_y), ("h", h, want_h, off_h)):
        off = (g.double().cpu() - w).abs()
        assert bool((off <= most).all()), f"{what}: {float((off / most).max())} of the bound"


@pytest.mark.parametrize("T,H,wide,gate,gate_f32,weights,weights_f32,scale", [
    (1, 7168, False, None, False, "weight", False, 1.0), (1, 1, True, "token", True, "both", True, 0.5), (3, 8, False, "full", False, "both", False, 1.0),
    (5, 7, False, "column", False, "both", False, -1.5), (7, 64, True, "row", True, "post", False, 1.0), (9, 512, False, None, False, None, False, 0.3),
    (13, 520, False, "full", True, "both", True, 1.0), (4, 1024, True, "token", False, "weight", True, 2.0), (33, 1999, True, "token", False, "both", False, 0.7),
    (6, 2048, False, "one", False, "both", False, 1.0), (2, 4096, True, "column", True, "both", True, 1.0), (3, 4104, False, "full", False, "post", True, 1.0),
    (2, 8192, False, None, False, "both", False, 1.0), (2, 8200, True, "column", False, "both", False, 1.0), (3, 8193, False, "full", False, "both", False, 1.0),
    (1, 16384, False, "row", False, "both", False, 1.0), (2, 16383, True, "full", True, "both", False, 1.0), (2, 32768, True, "column", False, "both", True, 1.0), (2, 32761, False, "full", True, "both", False, 1.0),
    (1030, 255, False, "token", True, "both", False, 1.0), (613, 1000, False, None, False, "weight", False, 1.0), (0, 128, False, None, False, "both", False, 1.0)])
def test_equals_the_plain_form(pkg, dev, T, H, wide, gate, gate_f32, weights, weights_f32, scale):
    say("residual_norm", T, H, wide, gate, weights)
    a = make(T, H, T * 7 + H, wide, gate, gate_f32, weights, weights_f32)
    got = pkg.residual_norm(**{k: None if v is None else v.to(dev) for k, v in a.items()}, scale=scale, eps=1e-5)
    torch.cuda.synchronize()
    assert got[0].dtype == torch.bfloat16 and got[1].dtype == a["residual"].dtype
    check(a, got, scale, 1e-5)


@pytest.mark.parametrize("H", [96, 97, 2048])
def test_without_a_residual(pkg, dev, H):
    say("residual_norm without residual", H)
    a = make(4, H, 3)
    a["residual"] = None
    on = {k: None if v is None else v.to(dev) for k, v in a.items()}
    y, h = pkg.residual_norm(**on)
    check(a, (y, h), 1.0, 1e-6)
    assert h.dtype == torch.bfloat16
    wide = torch.empty(4, H, device=dev)
    y, h = pkg.residual_norm(**on, residual_out=wide)
    assert h.data_ptr() == wide.data_ptr()
    check(a, (y, h), 1.0, 1e-6)


@pytest.mark.parametrize("H,at", [(128, 8), (128, 3), (1999, 1), (4096, 16)])
def test_strided_rows_and_in_place(pkg, dev, H, at):
    """Rows inside wider ones, the stream updated in place, the result over x; what lies beside the rows stays."""
    say("residual_norm strided", H, at)
    a = make(21, H, H + at, gate="full")
    want = pkg.residual_norm(**{k: v.to(dev) for k, v in a.items()})
    big = {}
    for k in ("x", "residual", "gate"):
        big[k] = torch.full((21, H + 40), -3.0, dtype=torch.bfloat16, device=dev)
        big[k][:, at:at + H] = a[k].to(dev)
    view = {k: v[:, at:at + H] for k, v in big.items()}
    y, h = pkg.residual_norm(view["x"], view["residual"], a["weight"].to(dev), a["post_weight"].to(dev), view["gate"], out=view["x"], residual_out=view["residual"])
    torch.cuda.synchronize()
    assert y.data_ptr() == view["x"].data_ptr() and h.data_ptr() == view["residual"].data_ptr()
    if at % 8 == 0:                                      # (another split of the row: other roundings of the sums)
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
    check(a, (y, h), 1.0, 1e-6)
    for k in ("x", "residual"):
        assert bool((big[k][:, :at] == -3).all()) and bool((big[k][:, at + H:] == -3).all())


@pytest.mark.parametrize("H", [*range(1, 18), *range(505, 522), 1029, 2049, 4103, 8191, 8195, 16386])
def test_last_pieces(pkg, dev, H):
    """Rows of every length around a piece's and a wavefront's, in place, in types of their own, beside values that stay."""
    say("residual_norm, last piece", H)
    for wide, gate in ((False, "column"), (True, "full")):
        a = make(5, H, H, wide, gate, gate_f32=wide, weights_f32=not wide)
        big = {k: torch.full((5, H + 3), -3.0, dtype=a[k].dtype, device=dev) for k in ("x", "residual")}
        for k, t in big.items():
            t[:, 1:H + 1] = a[k].to(dev)
        view = {k: t[:, 1:H + 1] for k, t in big.items()}
        y, h = pkg.residual_norm(view["x"], view["residual"], a["weight"].to(dev), a["post_weight"].to(dev), a["gate"].to(dev), out=view["x"],
                                 residual_out=view["residual"])
        torch.cuda.synchronize()
        check(a, (y, h), 1.0, 1e-6)
        for t in big.values():
            assert bool((t[:, 0] == -3).all()) and bool((t[:, H + 1:] == -3).all())


def test_two_halves_of_one_buffer(pkg, dev):
    """Results in the columns beside what is read share no value with it."""
    a = make(6, 256, 5)
    big = torch.zeros(6, 1024, dtype=torch.bfloat16, device=dev)
    big[:, :256], big[:, 256:512] = a["x"].to(dev), a["residual"].to(dev)
    y, h = pkg.residual_norm(big[:, :256], big[:, 256:512], a["weight"].to(dev), a["post_weight"].to(dev), out=big[:, 512:768], residual_out=big[:, 768:])
    check(a, (y, h), 1.0, 1e-6)


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_no_numbers_stay_in_their_row(pkg, dev, what):
    a = make(5, 200, 8, gate="column")
    on = {k: v.to(dev) for k, v in a.items()}
    want = pkg.residual_norm(**on)
    on["x"][2, 7] = what
    y, h = pkg.residual_norm(**on)
    rows = [0, 1, 3, 4]
    assert torch.equal(y[rows], want[0][rows]) and torch.equal(h[rows], want[1][rows])
    assert bool(y[2].isnan().any())


def test_a_row_of_zeros(pkg, dev):
    x = torch.zeros(3, 64, dtype=torch.bfloat16, device=dev)
    y, h = pkg.residual_norm(x, x, torch.ones(64, device=dev), torch.ones(64, device=dev))
    assert bool((y == 0).all()) and bool((h == 0).all())


def test_streams_and_graphs(pkg, dev):
    say("residual_norm streams, graphs")
    a = {k: v.to(dev) for k, v in make(17, 1024, 2, gate="token").items()}
    want = pkg.residual_norm(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pkg.residual_norm(**a)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    y, stream = torch.zeros_like(want[0]), a["residual"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.residual_norm(a["x"], stream, a["weight"], a["post_weight"], a["gate"], out=y, residual_out=stream)
    stream.copy_(a["residual"])
    for _ in range(4):                                   # the stream grows with every replay
        eager = pkg.residual_norm(a["x"], stream, a["weight"], a["post_weight"], a["gate"])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager[0]) and torch.equal(stream, eager[1])


def test_offsets_beyond_32_bits(pkg, dev):
    say("residual_norm, rows 2^32 bytes apart")
    a = make(2, 64, 4)
    big = torch.empty((1 << 31) + 64, dtype=torch.bfloat16, device=dev)
    x = big.as_strided((2, 64), (1 << 31, 1))
    x.copy_(a["x"].to(dev))
    y, h = pkg.residual_norm(x, a["residual"].to(dev), a["weight"].to(dev), a["post_weight"].to(dev))
    check(a, (y, h), 1.0, 1e-6)


@pytest.mark.parametrize("gate", ["full", "token"])
def test_a_gate_beside_what_it_gates(pkg, dev, gate):
    """A projection's columns hold the block's output and its gate; the results take the output's and the residual's place."""
    say("residual_norm, gate beside x", gate)
    H, T = 256, 9
    a = make(T, H, 11, gate=gate)
    want = pkg.residual_norm(**{k: v.to(dev) for k, v in a.items()})
    wide = torch.zeros(T, 2 * H, dtype=torch.bfloat16, device=dev)
    cols = a["gate"].shape[1]
    wide[:, :H], wide[:, H:H + cols] = a["x"].to(dev), a["gate"].to(dev)
    x, g, r = wide[:, :H], wide[:, H:H + cols], a["residual"].to(dev)
    y, h = pkg.residual_norm(x, r, a["weight"].to(dev), a["post_weight"].to(dev), g, out=x, residual_out=r)
    assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and torch.equal(g.cpu(), a["gate"])
    for bad in (wide[:, H:], wide[:, 1:H + 1]):          # over the gate, over part of x
        with pytest.raises(RuntimeError):
            pkg.residual_norm(x, r, a["weight"].to(dev), a["post_weight"].to(dev), g, out=bad)
