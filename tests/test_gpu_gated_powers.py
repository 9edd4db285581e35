"""The powers of two that bring x's rows and W's rows into FP16's range in the gated product's fast mode come out of
its results again wherever these are numbers in f32, whatever the two powers' own product is.

x has one value a row, so that g and u are one product each, off by `per` of themselves; silu(g) = g / 2 for the
small gates here, h by half a BF16 step, 2^-8 of it."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_gated import D, cells, gen, gpu, kernel_error, kind_of, planes, weights, within  # noqa: E402,F401
from test_gpu_gated_tails import multiplied  # noqa: E402

WAYS = [(3, 512, 300), (20, 256, 70), (40, 512, 100), (300, 512, 9473), (300, 256, 1000), (800, 256, 2400)]


@pytest.mark.parametrize("M,K,F", WAYS)
def test_small_gates_beside_large_ups(M, K, F):
    """x about 2^-92, gates' absmax 2^-30, ups' 2^93: g is below 2^-119 and the two powers' product below 2^-149."""
    g = gen(M)
    hole, plug, am = planes(2 * F, K, 64, g)
    am.view(F, 2, -1).mul_(torch.tensor([2.0 ** -25, 2.0 ** 98], device="cuda")[None, :, None])
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = (2.0 ** -92 * torch.linspace(1, 2, M, device="cuda")).bfloat16()
    h = D().htile_gated(x, hole, plug, am, F, mode="fast")
    torch.cuda.synchronize()
    assert kernel_error() == 0
    kind = kind_of(M, K, 64, "fast")
    per = (K / 16 + 8) * 2.0 ** -22 if kind == "product" else (K / 32 + 24) * 2.0 ** -23
    y = x.double() @ multiplied(hole, plug, am, 2 * F, K, 64, kind).T
    gate, up = y[:, 0::2], y[:, 1::2]
    want = gate / 2 * up
    assert float(gate.abs().max()) < 2.0 ** -119 and int((want.abs() > 2.0 ** -126).sum()) > M * F // 4
    # g is below f32's normal range, or its half is: 2^-149 of each, which up multiplies
    within(h, want, (2.0 ** -8 + 4 * per) * want.abs() + 2.0 ** -148 * up.abs() + 2.0 ** -134)


@pytest.mark.parametrize("M,K,F", WAYS)
def test_large_values_that_meet_no_weight(M, K, F):
    """x of 2^120 in a block of weights 0, beside blocks of 2^40: the sums are 0, and so is h."""
    g = gen(M + 1)
    hole, plug, am = planes(2 * F, K, 64, g)
    am.view(2 * F, -1).mul_(2.0 ** 45)
    am.view(2 * F, -1)[:, 0] = 0
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[:, 3] = 2.0 ** 120
    for name in ("silu", "gelu_tanh"):
        h = D().htile_gated(x, hole, plug, am, F, mode="fast", act=name)
        assert bool((h == 0).all())
    assert kernel_error() == 0


@pytest.mark.parametrize("e", [0, 9, 27])
@pytest.mark.parametrize("M,K,F", WAYS)
def test_weights_of_small_blocks_keep_their_bits(M, K, F, e):
    """The only x that is not 0 meets a block whose absmax is 2^-e of the row's largest, twice, so that the two products
    of each gate all but cancel: what FP16 made of the two weights, 2^-11 of each at most, stands beside a small g.  The
    sums' own error is (K / 16 + 8) 2^-22 of S = sum |w x| at most (see test_gpu_gated)."""
    g = gen(M + e)
    hole, plug, am = planes(2 * F, K, 64, g)
    am = am.view(2 * F, -1)
    am[:, 0] = 1.0
    am[:, 1] = 2.0 ** -e * torch.rand(2 * F, device="cuda", generator=g).add(1)
    c = cells()
    one, two = (int((c - v).abs().argmin()) for v in (0.9 + 0.01 * e / 9, 0.6))
    for col, code in ((64, one), (65, two)):  # a byte: the even column in the low nibble
        for plane, v in ((hole, code >> 4), (plug, code & 15)):
            byte = plane.view(2 * F, K // 2)[::2, col // 2]
            byte.copy_(byte & (0x0F if col % 2 else 0xF0) | (v << 4 if col % 2 else v))
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    by = 2.0 ** e * 2.0 ** (torch.arange(M, device="cuda") % 4)
    x[:, 64], x[:, 65] = by, -(c[one] / c[two] * by).bfloat16()
    h = D().htile_gated(x, hole, plug, am.reshape(-1), F, mode="fast")
    torch.cuda.synchronize()
    w = weights(hole, plug, am.reshape(-1), 2 * F, K, 64, "f32")
    y, s = x.double() @ w.T, x.double().abs() @ w.abs().T
    off = (2.0 ** -11 + (K / 16 + 8) * 2.0 ** -22) * s
    gate, up, dg, du = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
    assert bool((gate.abs() < 2.0 ** -7 * s[:, 0::2]).all())
    a = gate * torch.sigmoid(gate)
    within(h, a * up, 1.13 * dg * (up.abs() + du) + a.abs() * du + (2.0 ** -8 + 2.0 ** -16) * (a * up).abs())
