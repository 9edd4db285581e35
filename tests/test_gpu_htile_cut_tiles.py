"""H-TILE products whose last tiles are cut into fewer pieces than there are CTA pairs: few K groups (of 256), few
tiles over a round.  Against the expanded BF16 weights in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention_layer import gpu  # noqa: E402,F401


@pytest.mark.parametrize("K", [256, 512, 1024, 4096])
@pytest.mark.parametrize("over", [1, 2, 7])
def test_cut_tiles(K, over):
    from glint_b200 import device as D
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    M, N = 200, 256 * (pairs + over) - 3
    g = torch.Generator(device="cuda").manual_seed(K + over)
    pl = D.encode((torch.randn(N, K, device="cuda", generator=g) * 0.02).bfloat16())
    w = D.expand(*pl, N * K, 64, torch.bfloat16).view(N, K).double()
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    want, s = x.double() @ w.T, x.double().abs() @ w.abs().T
    for _ in range(2):
        y = torch.full((M, N), 7.0, device="cuda")
        D.htile(x, *pl, N, mode="fast", out=y)
        # K / 16 products added up in one f32 accumulator whose adder truncates, and f32 sums of the cut tiles' parts
        assert bool(((y.double() - want).abs() <= (K / 16 + 24) * 2.0 ** -22 * s).all())
