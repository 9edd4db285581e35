"""The gated product where rows' and weights' offsets pass 2^31, and captured where the workspace holds counts and sums:
rows and columns at both ends against the formula (bounds of test_gpu_gated), the same bits from replays."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_gated import D, gen, gpu, kernel_error, kind_of, planes, reference, within  # noqa: E402,F401


def cut(pl, K, bs, f, n):
    """The planes of outputs f .. f + n - 1; f K is even and whole blocks."""
    a, b = 2 * f * K, 2 * (f + n) * K
    return pl[0][a // 2:b // 2], pl[1][a // 2:b // 2], pl[2][a // bs:b // bs]


def ends(n, k, step):
    return sorted({0, (n - k) // 2 // step * step, (n - k) // step * step})


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("M,K,F", [(2, 8192, 140000), (20, 8192, 140000), (40, 8192, 140000), (800, 8192, 140000), (3, 8128, 140000),
                                   (1, 8176, 140000), (80000, 256, 28672), (270000, 8192, 8)])
def test_offsets_past_32_bits(M, K, F, mode):
    g = gen(M + K)
    pl = planes(2 * F, K, 64, g)
    x = torch.randn(M, K, device="cuda", generator=g, dtype=torch.bfloat16)
    h = D().htile_gated(x, *pl, F, mode=mode)
    assert max(2 * F * K, M * F, M * K) > 2 ** 31 and kernel_error() == 0
    kind = kind_of(M, K, 64, mode)
    for f in ends(F, 8, 64):
        for m in ends(M, 40, 1):
            rows = slice(max(m, 0), max(m, 0) + 40)
            within(h[rows, f:f + 8], *reference(x[rows], cut(pl, K, 64, f, 8), 8, 64, kind, "silu"))


@pytest.mark.parametrize("mode", ["fast", "precise"])
@pytest.mark.parametrize("M,K,F", [(1, 512, 300), (16, 512, 18001), (31, 512, 18001), (20, 12544, 96), (40, 1024, 130), (300, 512, 9473),
                                   (900, 256, 4700), (40, 448, 50), (5, 96, 33)])
def test_captured_calls_of_two_streams(M, K, F, mode):
    g = gen(M + F)
    bs = 64 if K % 64 == 0 else 32
    pl = [planes(2 * F, K, bs, g) for _ in range(2)]
    xs = [torch.randn(M, K, device="cuda", generator=g).bfloat16() for _ in range(2)]
    side, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for x, p in zip(xs, pl):
        D().htile_gated(x, *p, F, bs, mode=mode)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            first = D().htile_gated(x, *p, F, bs, mode=mode)
            outs.append((first, D().htile_gated(x, *p, F, bs, mode=mode, act="gelu_tanh")))
        graphs.append(graph)
    for r in range(4):
        if r == 2:  # other values in the same places
            for x, p in zip(xs, pl):
                x.copy_(torch.randn(M, K, device="cuda", generator=g))
                p[0].random_(0, 256, generator=g)
        want = [[D().htile_gated(x, *p, F, bs, mode=mode, act=a) for a in ("silu", "gelu_tanh")] for x, p in zip(xs, pl)]
        for two in outs:
            for o in two:
                o.fill_(7)
        torch.cuda.synchronize()
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for two, wants in zip(outs, want):
            for o, w in zip(two, wants):
                assert torch.equal(o.view(torch.int16), w.view(torch.int16))
    assert kernel_error() == 0
