"""GPU tests of the gated feed-forward projection (glint_htile_gated_stream, device.htile_gated)
against its formula in 64 bits, written here.

The weights that a kernel multiplies by are known: in fast mode FP16(cell) * absmax (up to 32 rows), or
cell * absmax rounded to FP16 at the row's power of two (more); the cell's two BF16 halves, 2^-17 of it off at
most (precise mode, and the shapes that only mma.sync takes); f32 (the kernel for any shape).  x is exact: its values
here are all within 2^29 of their row's largest.  The reference takes those weights, so that what is left is
the sums' own error, with S = sum |w x|:
  fast, more than 32 rows: K / 16 products added up in one f32 accumulator whose adder
      truncates: (K / 16 + 8) 2^-22 S.
  else blocks of 64 in accumulators of their own, and K / 64 (any shape: K / 32 + 5) f32 sums: (K / 32 + 24)
      2^-23 S, and 2^-17 S for the halves.
Through h = act(g) u, |act'| <= 1.13: 1.13 dg (|u| + du) + |act(g)| du, 2^-16 of it for the
activation's own arithmetic (2^-17 for the exponential), and half a BF16 step, 2^-8.
"""
import math
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HEADER = Path(__file__).resolve().parent.parent / "include" / "glint_cells.h"


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from glint_b200 import build
    build.build()
    torch.cuda.set_device(0)


def D():
    from glint_b200 import device
    return device


def kernel_error():
    return D().lib().glint_kernel_error(1)


def cells():
    text = HEADER.read_text()
    text = text[text.index("GLINT_CELLS_INIT"):]
    return torch.tensor([float.fromhex(v) for v in re.findall(r"-?0x[0-9a-f.]+p[-+]\d+", text)[:256]], device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def planes(rows, K, bs, g):
    n = rows * K
    b = [torch.randint(0, 256, ((n + 1) // 2,), device="cuda", generator=g, dtype=torch.uint8) for _ in range(2)]
    return b[0], b[1], 0.01 + 0.05 * torch.rand((n + bs - 1) // bs, device="cuda", generator=g)


def weights(hole, plug, absmax, rows, K, bs, kind):
    """[rows, K] f64: what the kernels of this kind multiply by."""
    n = rows * K
    h, p = (torch.stack([b & 15, b >> 4], 1).view(-1)[:n].long() for b in (hole, plug))
    c = cells()[h * 16 + p]
    am = absmax[torch.arange(n, device="cuda") // bs]
    if kind == "product":
        per = absmax.view(rows, K // bs)
        by = torch.exp2(-torch.floor(torch.log2(per.amax(1, keepdim=True).double())) - 1)
        by = by.repeat_interleave(K, 1).view(-1)
        w = (c * (am * by.float())).half().double() / by
    elif kind == "cell":
        w = c.half().double() * am.double()
    else:  # f32, or the two halves
        w = c.double() * am.double()
    return w.view(rows, K)


def act(g, name):
    z = g if name == "silu" else math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3)
    return g * torch.sigmoid(z)


def reference(x, pl, F, bs, kind, name):
    K = x.shape[1]
    w = weights(*pl, 2 * F, K, bs, kind)
    xd = x.double()
    y, s = xd @ w.T, xd.abs() @ w.abs().T
    per = (K / 16 + 8) * 2.0 ** -22 if kind == "product" else (K / 32 + 24) * 2.0 ** -23 + (2.0 ** -17 if kind == "halves" else 0)
    g, u, dg, du = y[:, 0::2], y[:, 1::2], per * s[:, 0::2], per * s[:, 1::2]
    a = act(g, name)
    h = a * u
    # the last term: what __fdividef gives up below z = -87
    return h, 1.13 * dg * (u.abs() + du) + a.abs() * du + (2.0 ** -8 + 2.0 ** -16) * h.abs() + 1e-36 * (1 + u.abs())


def kind_of(M, K, bs, mode):
    if bs % 64 or K % 64:
        return "f32"
    if mode == "precise" or bs != 64 or K % 256:
        return "halves"
    return "cell" if M <= 32 else "product"


def within(got, want, bound):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= bound)
    assert bool(same.all()), f"{int((~same).sum())} of {same.numel()} off, " \
        f"worst {float(((got - want).abs() / bound)[~same].max()):.3g} of its bound"


def check(M, K, F, bs=64, mode="fast", name="silu", seed=0, x=None, pl=None):
    g = gen(seed + M + K + F)
    pl = planes(2 * F, K, bs, g) if pl is None else pl
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16() if x is None else x
    wide = torch.full((M + 2, F), 7.0, dtype=torch.bfloat16, device="cuda")  # rows before and behind stay
    h = D().htile_gated(x, *pl, F, bs, mode=mode, act=name, out=wide[1:M + 1])
    torch.cuda.synchronize()
    assert kernel_error() == 0
    assert bool((wide[0] == 7).all()) and bool((wide[-1] == 7).all())
    want, bound = reference(x, pl, F, bs, kind_of(M, K, bs, mode), name)
    within(h, want, bound)
    again = D().htile_gated(x, *pl, F, bs, mode=mode, act=name)
    assert torch.equal(h.view(torch.int16), again.view(torch.int16)), "not the same bits twice"
    return pl, x, h


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 16, 17, 32, 33, 64, 127, 128, 200, 257])
@pytest.mark.parametrize("K,F", [(256, 1), (512, 2), (1024, 7), (256, 8), (768, 17), (512, 300), (256, 1001)])
def test_shapes(M, K, F, mode, name):
    check(M, K, F, mode=mode, name=name)


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("M,K,F", [(1, 4096, 14336), (5, 2048, 6911), (16, 1024, 28672), (31, 512, 18001), (32, 16384, 500),
                                   (511, 1024, 14336), (300, 512, 9473), (1030, 256, 10000), (16, 10240, 6000), (2, 8192, 4999),
                                   (9, 2560, 9728), (7, 5120, 3000), (8, 3584, 2222), (13, 33280, 50),
                                   (98, 6656, 174), (1771, 5888, 204), (33, 33280, 3), (640, 4096, 1535), (65, 1792, 129),
                                   (769, 256, 4700), (2311, 768, 1021), (2817, 2304, 1537), (1025, 512, 9345), (5000, 256, 650)])
def test_wide_layers(M, K, F, mode):
    """More rows than two blocks a CTA; tiles shared between CTA pairs (511 and 300 rows); weights expanded first, with
    whole tiles alone and with a cut rest (769 rows and more)."""
    check(M, K, F, mode=mode)


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("M,K,F,bs", [(1, 64, 5, 64), (4, 192, 33, 64), (12, 448, 700, 64), (16, 2880, 1111, 64), (20, 2880, 50, 64), (40, 320, 9, 64), (3, 512, 10, 128), (9, 96, 6, 32), (2, 34, 3, 17),
                                      (11, 33, 4, 16), (1, 1, 1, 1), (65, 640, 1000, 64)])
def test_any_shape(M, K, F, bs, mode):
    check(M, K, F, bs=bs, mode=mode, name="gelu_tanh")


def test_alignment():
    """Operands at odd addresses: the same formula by another kernel."""
    g = gen(1)
    M, K, F = 3, 512, 20
    hole, plug, am = planes(2 * F, K, 64, g)
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()

    def moved(t):
        b = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        b[1:] = t.reshape(-1)
        return b[1:].view(t.shape)
    for pl, xx in (((moved(hole), plug, am), x), ((hole, plug, moved(am)), x), ((hole, plug, am), moved(x))):
        h = D().htile_gated(xx, *pl, F, mode="fast", out=moved(torch.zeros(M, F, dtype=torch.bfloat16, device="cuda")))
        got, near = h.double(), torch.zeros(M, F, dtype=torch.bool, device="cuda")
        for kind in ("f32", "halves"):
            want, bound = reference(x, (hole, plug, am), F, 64, kind, "silu")
            near |= (got - want).abs() <= bound
        assert bool(near.all())


@pytest.mark.parametrize("M", [4, 40])
@pytest.mark.parametrize("mode", ["fast", "precise"])
def test_values_that_are_not_finite_stay_in_their_row(M, mode):
    g = gen(M)
    K, F = 512, 70
    pl = planes(2 * F, K, 64, g)
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    want = D().htile_gated(x, *pl, F, mode=mode)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[2, 77] = bad
        h = D().htile_gated(y, *pl, F, mode=mode)
        keep = torch.arange(M, device="cuda") != 2
        assert torch.equal(h[keep].view(torch.int16), want[keep].view(torch.int16))
        if math.isnan(bad):
            assert bool(h[2].isnan().all())
    zero = D().htile_gated(x, pl[0], pl[1], torch.zeros_like(pl[2]), F, mode=mode)
    assert bool((zero == 0).all())


@pytest.mark.parametrize("M", [2, 50])
@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
def test_large_gates(M, name):
    """Gates far into both tails of the activation, where the exponential is 0 or infinite."""
    x = torch.zeros(M, 256, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = torch.logspace(-3, 5, M, device="cuda").bfloat16()
    x[:, 1] = 1.0
    check(M, 256, 64, mode="precise", name=name, x=x)


@pytest.mark.parametrize("M", [1, 5, 12, 30, 40, 300])
def test_rows_of_other_sizes(M):
    """Rows of x far past FP16's range, far below it and of both at once, rows of W likewise: each by its own
    power of two."""
    g = gen(M)
    K, F = 512, 150
    pl = planes(2 * F, K, 64, g)
    by = torch.logspace(-6, 4, 2 * F, device="cuda")[torch.randperm(2 * F, device="cuda", generator=g)]
    pl = pl[0], pl[1], (pl[2].view(2 * F, -1) * by[:, None]).view(-1)
    x = torch.randn(M, K, device="cuda", generator=g)
    x *= torch.logspace(-12, 9, M, device="cuda")[:, None] if M > 1 else 1e9
    x[M // 2, 7] *= 2.0 ** 20  # the row's others lie far below it
    check(M, K, F, x=x.bfloat16(), pl=pl)
    x[0] = 0
    h = D().htile_gated(x.bfloat16(), *pl, F, mode="fast")
    assert bool((h[0] == 0).all())


def test_packed_planes():
    """pack_gated of separately encoded weights, and the call, against the two linears' products."""
    g = gen(9)
    F, K, M = 96, 1024, 5
    gate, up = (D().encode((torch.randn(F, K, device="cuda", generator=g) * 0.02).bfloat16()) for _ in range(2))
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    pl = D().pack_gated(gate, up, F, K)
    h = D().htile_gated(x, *pl, F, act="silu")
    want, bound = reference(x, pl, F, 64, "halves", "silu")
    within(h, want, bound)
    yg, yu = (D().htile(x, *p, F).double() for p in (gate, up))
    within(h, act(yg, "silu") * yu, 2 * bound)
    assert torch.equal(pl[2].view(F, 2, -1)[:, 1].reshape(-1), up[2])
    for bad in (dict(K=K + 1), dict(F=F + 1), dict(blocksize=48), dict(blocksize=0)):
        with pytest.raises(ValueError):
            D().pack_gated(**{**dict(gate=gate, up=up, F=F, K=K), **bad})


def test_streams_and_graphs():
    """Two captured calls replayed at once on two streams, each with a workspace of its own."""
    g = gen(10)
    M, K, F = 300, 512, 9473  # tiles shared between pairs: the largest workspace
    pl = [planes(2 * F, K, 64, g) for _ in range(2)]
    xs = [torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = [D().htile_gated(x, *p, F, mode="fast") for x, p in zip(xs, pl)]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [D().htile_gated(x, *p, F, mode="fast", stream=s) for x, p, s in zip(xs, pl, side)]
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want))
    graphs, outs = [], []
    for x, p in zip(xs, pl):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(D().htile_gated(x, *p, F, mode="fast"))
        graphs.append(graph)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want))
    assert kernel_error() == 0


def test_empty():
    g = gen(11)
    pl = planes(8, 256, 64, g)
    x = torch.randn(3, 256, device="cuda", generator=g).bfloat16()
    assert D().htile_gated(x[:0], *pl, 4).shape == (0, 4)
    assert D().htile_gated(x, *pl, 0).shape == (3, 0)
    h = D().htile_gated(x[:, :0].contiguous(), *pl, 4)
    assert bool((h == 0).all()) and h.shape == (3, 4)


def test_refusals():
    g = gen(12)
    pl = planes(8, 256, 64, g)
    x = torch.randn(3, 256, device="cuda", generator=g).bfloat16()
    ok = dict(x=x, hole=pl[0], plug=pl[1], absmax=pl[2], F=4)
    D().htile_gated(**ok)
    for kw, match in ((dict(x=x.float()), "bfloat16"), (dict(x=x.cpu()), "CUDA"), (dict(x=x[0]), "2-D"), (dict(x=x[:, ::2]), "contiguous"),
                      (dict(hole=pl[0][:-1]), "planes"), (dict(plug=pl[1].to(torch.int16)), "planes"), (dict(absmax=pl[2][:-1]), "planes"),
                      (dict(absmax=pl[2].double()), "planes"), (dict(F=5), "planes"), (dict(F=-1), "F must"), (dict(blocksize=0), "blocksize"),
                      (dict(mode="quick"), "mode"), (dict(act="relu"), "act"), (dict(out=torch.empty(3, 5, device="cuda").bfloat16()), "out"),
                      (dict(out=torch.empty(3, 4, device="cuda")), "out"), (dict(out=x.view(-1)[:12].view(3, 4)), "overlap")):
        with pytest.raises(ValueError, match=match):
            D().htile_gated(**{**ok, **kw})
