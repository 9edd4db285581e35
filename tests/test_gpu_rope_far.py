"""rope and rope_append on rows whose offsets pass 2^31 elements, and on no rows at all."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_rope import A, bits, freqs, gen, gpu, randn  # noqa: E402,F401


@pytest.mark.parametrize("dim,half,inter", [(128, 64, False), (64, 21, False), (64, 32, True)])
def test_rows_past_32_bits(dim, half, inter):
    """Tokens 2^28 elements apart, and heads 2^28 apart."""
    g = gen(dim + half)
    buf = torch.empty(9 * 2 ** 28 + 64 * dim, dtype=torch.bfloat16, device="cuda")
    for strides, (T, H) in (((2 ** 28, dim), (10, 3)), ((dim, 2 ** 28), (3, 10))):
        span = T * H * dim

        def place(off):
            return buf.as_strided((T, H, dim), (*strides, 1), off)
        q, k, v = (randn(T, H, dim, g=g) for _ in range(3))
        at = torch.randint(0, 4000, (T,), generator=g, device="cuda", dtype=torch.int32)
        want_q, want_k = A().rope(q, k, at, freqs(half), interleaved=inter)
        slots = torch.randperm(128, generator=g, device="cuda")[:T].to(torch.int32)
        caches = [A().KV4Cache.empty(2, H, dim, 64) for _ in range(2)]
        A().kv4_append(caches[0], want_k, v, slots)
        qo, ko, vo = place(0), place(span), place(2 * span)  # a token's or head's neighbours, far from the next
        for far, t in ((qo, q), (ko, k), (vo, v)):
            far.copy_(t)
        got_q, got_k = A().rope(qo, ko, at, freqs(half), interleaved=inter)
        assert torch.equal(bits(got_q), bits(want_q)) and torch.equal(bits(got_k), bits(want_k))
        A().rope_append(caches[1], qo, ko, vo, at, freqs(half), slots, interleaved=inter, q_out=qo, k_out=ko)
        assert torch.equal(bits(qo), bits(want_q)) and torch.equal(bits(ko), bits(want_k)) and torch.equal(bits(vo), bits(v))
        for a, b in zip(*(A().kv4_read(c, slots) for c in caches)):
            assert torch.equal(bits(a), bits(b))


def test_no_tokens():
    x, at = torch.empty(0, 4, 128, dtype=torch.bfloat16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    q, k = A().rope(x, x, at, freqs(64))
    assert q.shape == x.shape and k.shape == x.shape
    q, k = A().rope(x, None, at, freqs(64), q_out=x)
    assert q is x and k is None
    cache = A().KV4Cache.empty(2, 4, 128, 64)
    held = [t.view(torch.uint8) for t in (cache.k_code, cache.k_meta, cache.v_code, cache.v_meta)]  # of any content
    before = [t.clone() for t in held]
    assert A().rope_append(cache, x, x, x, at, freqs(64), at).shape == x.shape
    assert all(torch.equal(a, b) for a, b in zip(before, held))


def test_keys_of_no_heads():
    g = gen(5)
    q, at = randn(7, 4, 64, g=g), torch.arange(7, dtype=torch.int32, device="cuda")
    got, k = A().rope(q, q[:, :0], at, freqs(32))
    want, _ = A().rope(q, None, at, freqs(32))
    assert torch.equal(bits(got), bits(want)) and k.shape == (7, 0, 64)
