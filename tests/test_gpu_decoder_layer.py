"""The operators of a decoder's layer in their order (examples/attention_layer.py): rotation into the cache,
attention, the gated product, the down linear; each against what it stands for, and the run of them captured."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attention_layer import gpu  # noqa: E402,F401
from test_gpu_gated import gen, kind_of, reference, weights  # noqa: E402


def layers(lens, **more):
    import attention_layer as example
    hidden, heads, kv, dim = 512, 4, 2, 128
    g = gen(3)
    planes = example.random_planes((heads + 2 * kv) * dim, hidden, g), example.random_planes(hidden, heads * dim, g)
    return [example.AttentionLayer(*planes, hidden, heads, kv, dim, len(lens), max(lens) + 40, 64, 16, slack=4, **m)
            for m in more.values()]


def test_rotation_on_the_way_into_the_cache_is_the_callers():
    """freqs, and a callback that rotates and leaves the append to the layer: the same bits everywhere."""
    from glint_b200 import attn
    freqs, scale = attn.rope_freqs(128, 10000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64))
    lens = [90, 1, 70]
    one, two = layers(lens, a=dict(freqs=(freqs, scale)),
                      b=dict(rope=lambda q, k, at: attn.rope(q, k, at.to(torch.int32), freqs, scale=scale)))
    g = gen(4)
    x = torch.randn(sum(lens), 512, device="cuda", generator=g).bfloat16()
    a, b = one.prompt(x, lens), two.prompt(x, lens)
    for _ in range(8):  # past the first eviction
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and bool(a.isfinite().all())
        x = torch.randn(len(lens), 512, device="cuda", generator=g).bfloat16()
        a, b = one.step(x), two.step(x)
    assert one.lens.tolist() == two.lens.tolist()
    slots = one._slots(torch.zeros(64, dtype=torch.int64, device="cuda"), torch.arange(64, device="cuda"))
    for m, n in zip(attn.kv4_read(one.cache, slots), attn.kv4_read(two.cache, slots)):
        assert torch.equal(m.view(torch.int16), n.view(torch.int16))


def test_rope_or_freqs():
    from glint_b200 import attn
    with pytest.raises(ValueError):
        layers([1], a=dict(freqs=attn.rope_freqs(128), rope=lambda q, k, at: (q, k)))


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M", [1, 5, 32, 33, 200])
def test_feed_forward(M, act):
    import attention_layer as example
    hidden, ff = 512, 1280
    g = gen(M)
    gate, up, down = (example.random_planes(*s, g) for s in ((ff, hidden), (ff, hidden), (hidden, ff)))
    layer = example.FeedForward(gate, up, down, hidden, ff, act)
    x = torch.randn(M, hidden, device="cuda", generator=g).bfloat16()
    y = layer(x)
    h, bound = reference(x, layer.gated, ff, 64, kind_of(M, hidden, 64, "fast"), act)
    w = weights(*down, hidden, ff, 64, "f32")
    want, s = h @ w.T, h.abs() @ w.abs().T
    # h's own bound; a weight rounded to BF16 once, 2^-8 of it; sums as in fast mode there; y rounded to BF16
    off = (bound @ w.abs().T) * (1 + 2.0 ** -7) + (2.0 ** -8 + (ff / 16 + 8) * 2.0 ** -22) * s
    off = off * (1 + 2.0 ** -7) + 2.0 ** -8 * want.abs()
    assert bool(((y.double() - want).abs() <= off).all())


def test_captured_token():
    """A token's operators in a graph, replayed on new rows, positions and slots: the bits of the same calls made
    one by one on another cache."""
    import attention_layer as example
    from glint_b200 import attn, device
    B, H, KV, Dh, hidden, ff, per = 3, 8, 2, 64, 512, 768, 4
    g = gen(6)
    wqkv, wo = example.random_planes((H + 2 * KV) * Dh, hidden, g), example.random_planes(hidden, H * Dh, g)
    feed = example.FeedForward(*(example.random_planes(*s, g) for s in ((ff, hidden), (ff, hidden), (hidden, ff))), hidden, ff)
    freqs, scale = attn.rope_freqs(Dh)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(B * per, **i32).view(B, per)
    norm = 1 + torch.randn(Dh, device="cuda", generator=g)

    def token(cache, x, lens, slots):
        y = device.htile(x, *wqkv, (H + 2 * KV) * Dh, mode="fast", out_dtype=torch.bfloat16).view(B, H + 2 * KV, Dh)
        q, k, v = y.split([H, KV, KV], 1)
        attn.rope_append(cache, q, k, v, lens - 1, freqs, slots, scale=scale, q_norm=norm, k_norm=norm, q_out=q)
        o, _ = attn.kv4_attn(q[:, None], cache, table, lens)
        x = x + device.htile(o.view(B, H * Dh), *wo, hidden, mode="fast", out_dtype=torch.bfloat16)
        return x + feed(x)

    caches = [attn.KV4Cache.empty(B * per, KV, Dh, 16) for _ in range(2)]
    x, lens, slots = torch.zeros(B, hidden, device="cuda", dtype=torch.bfloat16), torch.ones(B, **i32), table[:, 0] * 16
    slots = slots.contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(caches[0], x, lens, slots)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token(caches[0], x, lens, slots)
    for t in range(20):  # over a page's end
        x.copy_(torch.randn(B, hidden, device="cuda", generator=g))
        lens.fill_(t + 1)
        slots.copy_(table[:, t // 16] * 16 + t % 16)
        graph.replay()
        want = token(caches[1], x, lens, slots)
        assert torch.equal(out.view(torch.int16), want.view(torch.int16)) and bool(out.isfinite().all())
