"""The attention layer example refuses what its pages cannot hold, before any device work."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention_layer import gpu  # noqa: E402,F401


def test_layer_refuses_more_than_its_slots():
    import attention_layer as example
    hidden, heads, kv, dim = 512, 4, 2, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    planes = (example.random_planes((heads + 2 * kv) * dim, hidden, g), example.random_planes(hidden, heads * dim, g))
    layer = example.AttentionLayer(*planes, hidden, heads, kv, dim, 2, 64, 64, 8)  # a page of 64 slots each; slack past it
    x = torch.randn(70, hidden, device="cuda", generator=g).bfloat16()
    for lens in ([65, 5], [70], [70, 0], [30, 30]):
        with pytest.raises(ValueError):
            layer.prompt(x, lens)
    layer.prompt(x, [62, 8])
    for _ in range(2):
        assert bool(layer.step(x[:2]).isfinite().all())
    with pytest.raises(ValueError):
        layer.step(x[:2])
    with pytest.raises(ValueError):
        layer.step(x[:1])
    torch.cuda.synchronize()
    assert layer.lens.tolist() == [64, 10]
