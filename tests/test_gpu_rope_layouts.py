"""rope and rope_append in place, in buffers whose heads lie in turn: the same bits as into new tensors."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_rope import A, bits, freqs, gen, gpu, randn  # noqa: E402,F401


@pytest.mark.parametrize("dim,half", [(64, 32), (128, 48), (128, 21)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,heads", [(1, 4), (37, 4), (700, 6), (300, 1)])
def test_heads_in_turn(dim, half, inter, tokens, heads):
    """Each head's query, key and value side by side."""
    g = gen(tokens + heads + half)
    y = randn(tokens, heads, 3, dim, g=g)
    at = torch.randint(0, 5000, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    w = 1 + torch.rand(dim, device="cuda", generator=g)
    q, k, v = (y[:, :, i].clone() for i in range(3))
    want_q, want_k = A().rope(q, k, at, freqs(half), interleaved=inter, q_norm=w)
    z = y.clone()
    A().rope(z[:, :, 0], z[:, :, 1], at, freqs(half), interleaved=inter, q_norm=w, q_out=z[:, :, 0], k_out=z[:, :, 1])
    for got, want in zip((z[:, :, i] for i in range(3)), (want_q, want_k, v)):
        assert torch.equal(bits(got), bits(want))
    slots = torch.randperm(1024, generator=g, device="cuda")[:tokens].to(torch.int32)
    caches = [A().KV4Cache.empty(16, heads, dim, 64) for _ in range(2)]
    A().kv4_append(caches[0], want_k, v, slots)
    z = y.clone()
    A().rope_append(caches[1], z[:, :, 0], z[:, :, 1], z[:, :, 2], at, freqs(half), slots, interleaved=inter, q_norm=w,
                    q_out=z[:, :, 0], k_out=z[:, :, 1])
    for got, want in zip((z[:, :, i] for i in range(3)), (want_q, want_k, v)):
        assert torch.equal(bits(got), bits(want))
    for a, b in zip(*(A().kv4_read(c, slots) for c in caches)):
        assert torch.equal(bits(a), bits(b))


def test_one_tensor_as_queries_and_keys():
    g = gen(3)
    t, at = randn(9, 4, 64, g=g), torch.arange(9, dtype=torch.int32, device="cuda")
    kept = t.clone()
    for kw in (dict(q_out=t), dict(k_out=t), dict(q_out=t, k_out=t)):
        with pytest.raises(ValueError, match="_out must be"):
            A().rope(t, t, at, freqs(32), **kw)
    assert torch.equal(bits(t), bits(kept))
    a, b = A().rope(t, t, at, freqs(32))
    assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize("dim", [64, 128])
def test_heads_of_zeros_with_the_least_eps(dim):
    x = torch.zeros(3, 4, dim, dtype=torch.bfloat16, device="cuda")
    at, w = torch.arange(3, dtype=torch.int32, device="cuda"), torch.ones(dim, device="cuda")
    for eps in (2.0 ** -250, 1e-30):
        q, k = A().rope(x, x, at, freqs(dim // 2), q_norm=w, k_norm=w, eps=eps)
        assert bool((q == 0).all()) and bool((k == 0).all())
    with pytest.raises(ValueError, match="eps"):
        A().rope(x, x, at, freqs(dim // 2), q_norm=w, eps=1e-80)
