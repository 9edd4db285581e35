"""The gated product's activation where its gates lie far below 0, relative to its value.

With one x that is not 0 a row's g and u are one product each: off by `per` of themselves (as in test_gpu_gated), the
activation by |z'| dg of itself (z = g, or 2 sqrt(2 / pi) (g + 0.044715 g^3)), the exponential by (2 + 1.18 |z|) 2^-23
(its documented 2 + 1.173 |z| units in the last place), a division and four products by 2^-22 and 2^-24 each.  Below
f32's normal range act(g) is off by 2^-149 more and so is e, which g multiplies; h by half a BF16 step, 2^-8 of
it, or 2^-134 below BF16's normal range.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_gated import D, cells, gen, gpu, kernel_error, kind_of, planes, weights, within  # noqa: E402,F401


def multiplied(hole, plug, absmax, rows, K, bs, kind):
    """[rows, K] f64: what the kernels multiply by.  Products of FP16 weights: a row's power of two brings its largest
    absmax into [2^14, 2^15), so that weights far below it have all their bits too."""
    if kind != "product":
        return weights(hole, plug, absmax, rows, K, bs, kind)
    top = absmax.view(rows, -1).amax(1).double()
    by = torch.exp2(14 - torch.floor(torch.log2(top)))
    w = weights(hole, plug, torch.ones_like(absmax), rows, K, bs, "f32")  # cells, exact
    am = absmax.view(rows, -1).repeat_interleave(bs, 1)
    return (w.float() * (am * by[:, None].float())).half().double() / by[:, None]


def tail(g, name):
    """(act(g), z, |z'|) in 64 bits, exact in the tail too."""
    c = math.sqrt(8 / math.pi)
    z, dz = (g, torch.ones_like(g)) if name == "silu" else (c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2))
    e = torch.exp(-z.abs())
    return torch.where(z < 0, g * e, g) / (1 + e), z, dz


def gates(F, K, bs, lo, hi, g):
    """Planes whose row 2f gives a gate of lo to hi, of its cell's sign, for an x of 1 in column 3 alone."""
    hole, plug, am = planes(2 * F, K, bs, g)
    row = torch.arange(2 * F, device="cuda")
    at = (row * K + 3) // 2  # an odd element: the high nibble
    c = cells()[(hole[at] >> 4).long() * 16 + (plug[at] >> 4).long()].abs()
    size = torch.where(row % 2 == 0, lo + (hi - lo) * torch.rand(2 * F, device="cuda", generator=g), 20.0)
    am[(row * K + 3) // bs] = size / c
    return hole, plug, am


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("name,lo,hi", [("silu", 60.0, 105.0), ("gelu_tanh", 8.5, 10.3)])
@pytest.mark.parametrize("M,K,F,bs", [(2, 256, 500, 64), (14, 512, 300, 64), (30, 256, 300, 64), (50, 256, 200, 64), (200, 512, 9473, 64), (800, 256, 2400, 64),
                                      (6, 192, 200, 64), (40, 512, 100, 128), (9, 96, 100, 32)])
def test_tails(M, K, F, bs, name, lo, hi, mode):
    g = gen(M + F)
    pl = gates(F, K, bs, lo, hi, g)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = torch.linspace(0.9, 1, M, device="cuda").bfloat16()
    h = D().htile_gated(x, *pl, F, bs, mode=mode, act=name)
    torch.cuda.synchronize()
    assert kernel_error() == 0
    kind = kind_of(M, K, bs, mode)
    per = (K / 16 + 8) * 2.0 ** -22 if kind == "product" else (K / 32 + 24) * 2.0 ** -23 + (2.0 ** -17 if kind == "halves" else 0)
    y = x.double() @ multiplied(*pl, 2 * F, K, bs, kind).T
    gate, up = y[:, 0::2], y[:, 1::2]
    a, z, dz = tail(gate, name)
    off = torch.expm1(1.1 * dz * per * gate.abs()) + (4 + 1.18 * z.abs()) * 2.0 ** -23 + per + 2.0 ** -20
    want = a * up
    bound = (2.0 ** -8 + off) * want.abs() + 2.0 ** -149 * (2 + gate.abs()) * up.abs() + 2.0 ** -134
    far = (z < -85) & (want.abs() > 2.0 ** -126)
    assert int(far.sum()) > 10
    within(h, want, bound)


@pytest.mark.parametrize("name", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,F", [(2, 64), (50, 64), (800, 2400)])
def test_gates_of_any_size(M, F, name):
    """Gates up to 10^30 and down to 0 in fast mode: no infinity and no NaN where the formula has none."""
    g = gen(M)
    pl = planes(2 * F, 256, 64, g)
    x = torch.zeros(M, 256, dtype=torch.bfloat16, device="cuda")
    x[:, 70] = torch.logspace(-30, 15, M, device="cuda").bfloat16()
    h = D().htile_gated(x, *pl, F, mode="fast", act=name).double()
    y = x.double() @ multiplied(*pl, 2 * F, 256, 64, kind_of(M, 256, 64, "fast")).T
    want = tail(y[:, 0::2], name)[0] * y[:, 1::2]
    assert bool(h.isfinite().all()) and bool((h[want == 0] == 0).all())
    near = (y[:, 0::2] > -3) & (want.abs() > 2.0 ** -120)
    assert int(near.sum()) > 20
    assert bool(((h - want).abs() <= 0.006 * want.abs())[near].all())
