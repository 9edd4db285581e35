"""The gated product's ways for more rows (weights expanded first; K cut for all of few tiles) where it can go wrong
beside its sizes: values that are not finite, rows of other sizes, streams, captured calls on new values."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_gated import D, act, check, gen, gpu, kernel_error, planes, weights, within  # noqa: E402,F401

WAYS = [(800, 512, 2400), (1100, 256, 2000), (90, 1024, 130)]  # expanded: with a cut rest, without; few tiles


@pytest.mark.parametrize("M,K,F", WAYS)
def test_values_that_are_not_finite_stay_in_their_row(M, K, F):
    g = gen(M)
    pl = planes(2 * F, K, 64, g)
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    want = D().htile_gated(x, *pl, F, mode="fast")
    for bad in (float("nan"), float("-inf")):
        y = x.clone()
        y[M - 1, 77] = bad
        h = D().htile_gated(y, *pl, F, mode="fast")
        assert torch.equal(h[:-1].view(torch.int16), want[:-1].view(torch.int16))
        if math.isnan(bad):
            assert bool(h[-1].isnan().all())
    # a weight block that is not finite reaches its own column alone
    am = pl[2].clone()
    am.view(2 * F, -1)[2 * 5 + 1, 0] = float("nan")
    h = D().htile_gated(x, pl[0], pl[1], am, F, mode="fast")
    keep = torch.arange(F, device="cuda") != 5
    assert torch.equal(h[:, keep].view(torch.int16), want[:, keep].view(torch.int16)) and bool(h[:, 5].isnan().all())
    assert bool((D().htile_gated(x, pl[0], pl[1], torch.zeros_like(pl[2]), F, mode="fast") == 0).all())


@pytest.mark.parametrize("M,K,F", WAYS)
def test_rows_of_other_sizes(M, K, F):
    g = gen(M)
    pl = planes(2 * F, K, 64, g)
    by = torch.logspace(-6, 4, 2 * F, device="cuda")[torch.randperm(2 * F, device="cuda", generator=g)]
    pl = pl[0], pl[1], (pl[2].view(2 * F, -1) * by[:, None]).view(-1)
    x = torch.randn(M, K, device="cuda", generator=g) * torch.logspace(-12, 9, M, device="cuda")[:, None]
    check(M, K, F, x=x.bfloat16(), pl=pl)
    x[0] = 0
    assert bool((D().htile_gated(x.bfloat16(), *pl, F, mode="fast")[0] == 0).all())


@pytest.mark.parametrize("M,K,F", WAYS + [(5, 512, 700), (300, 512, 1000)])
def test_weights_made_just_before(M, K, F):
    """The call right behind the kernels that write its weights and x, many times over: the same bits each time."""
    g = gen(M)
    made = [planes(2 * F, K, 64, g) for _ in range(2)]
    xs = [torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = [D().htile_gated(x, *p, F, mode="fast") for x, p in zip(xs, made)]
    torch.cuda.synchronize()
    pl, x = [torch.empty_like(t) for t in made[0]], torch.empty_like(xs[0])
    got = []
    for i in range(12):
        for t, s in zip((*pl, x), (*made[i % 2], xs[i % 2])):
            torch.add(s, 0, out=t)
        got.append(D().htile_gated(x, *pl, F, mode="fast"))
    torch.cuda.synchronize()
    assert all(torch.equal(h.view(torch.int16), want[i % 2].view(torch.int16)) for i, h in enumerate(got))
    assert kernel_error() == 0


@pytest.mark.parametrize("M,K,F", WAYS)
def test_streams_and_graphs(M, K, F):
    g = gen(M)
    pl = [planes(2 * F, K, 64, g) for _ in range(2)]
    xs = [torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(2)]
    want = [D().htile_gated(x, *p, F, mode="fast") for x, p in zip(xs, pl)]
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        outs = [D().htile_gated(x, *p, F, mode="fast", stream=s) for x, p, s in zip(xs, pl, side)]
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want))
    graphs, outs = [], []
    for x, p in zip(xs, pl):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = D().htile_gated(x, *p, F, mode="fast")
            outs.append((first, D().htile_gated(x, *p, F, mode="fast")))  # its workspace may be the first call's
        graphs.append(graph)
    for r in range(4):
        if r == 2:  # other values in the same places
            for x, p in zip(xs, pl):
                x.copy_(torch.randn(M, K, device="cuda", generator=g))
                p[0].random_(0, 256, generator=g)
            want = [D().htile_gated(x, *p, F, mode="fast") for x, p in zip(xs, pl)]
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.view(torch.int16), b.view(torch.int16)) for two, b in zip(outs, want) for o in two)
    assert kernel_error() == 0


@pytest.mark.parametrize("M,K,F", WAYS + [(20, 512, 300), (300, 512, 1000)])
def test_blocks_of_other_sizes(M, K, F):
    """Blocks of a row whose absmax differ by up to 2^24: each weight keeps its FP16 rounding, 2^-11 of itself."""
    g = gen(M + 1)
    hole, plug, am = planes(2 * F, K, 64, g)
    am = torch.exp2(-24 * torch.rand(am.shape, device="cuda", generator=g))
    # activations that lift the small blocks to the others' height, so that their errors would show
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    am.view(2 * F, -1)[:, 1:] = am.view(2 * F, -1)[:, 1:] * 2.0 ** -10
    x[:, 64:] *= 2.0 ** 10
    h = D().htile_gated(x, hole, plug, am, F, mode="fast")
    w = weights(hole, plug, am, 2 * F, K, 64, "f32")
    y, s = x.double() @ w.T, x.double().abs() @ w.abs().T
    off = (2.0 ** -11 + (K / 16 + 8) * 2.0 ** -22) * s
    gate, up, dg, du = y[:, 0::2], y[:, 1::2], off[:, 0::2], off[:, 1::2]
    a = act(gate, "silu")
    bound = 1.13 * dg * (up.abs() + du) + a.abs() * du + (2.0 ** -8 + 2.0 ** -16) * (a * up).abs() + 1e-36 * (1 + up.abs())
    within(h, a * up, bound)
