"""GPU tests of rope and rope_append (include/glint_attn.h, glint_b200/attn.py) against the
formula in 64 bits, written here.

Bound, per element: y carries three roundings to f32 (r, and x r w's two), c or s one, a
product one, the sum one: six of 2^-24 of |y1 c| + |y2 s|, a seventh for their products; and
half a BF16 step, 2^-8 of the value.  What rope_append caches: equal, byte for byte, to rope
and then kv4_append.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from glint_b200 import build
    build.build()
    torch.cuda.set_device(0)


def A():
    from glint_b200 import attn
    return attn


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, g, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()


def bits(t):
    return t.contiguous().view(torch.int16)


def freqs(half, base=10000.0):
    return (base ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float().cuda()


def reference(x, positions, inv_freq, inter, scale, w, eps=EPS):
    """(o, bound) in 64 bits."""
    y, half = x.double(), inv_freq.shape[0]
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    a = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(a) * scale)[:, None], (torch.sin(a) * scale)[:, None]
    one = torch.arange(half, device="cuda") * (2 if inter else 1)
    two = one + (1 if inter else half)
    o, part = y.clone(), y.abs()
    y1, y2 = y[..., one], y[..., two]
    o[..., one], o[..., two] = y1 * c - y2 * s, y2 * c + y1 * s
    part[..., one], part[..., two] = (y1 * c).abs() + (y2 * s).abs(), (y2 * c).abs() + (y1 * s).abs()
    return o, 2.0 ** -8 * o.abs() + 7 * 2.0 ** -24 * part


def within(got, want, bound, what):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= bound) | (got.isnan() & want.isnan())
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} off, " \
        f"worst {float(((got - want).abs() / bound.clamp_min(1e-30))[~same].max()):.3g} of its bound"


def check(q, k, positions, inv_freq, inter=False, scale=1.0, qw=None, kw=None, **more):
    qo, ko = A().rope(q, k, positions, inv_freq, interleaved=inter, scale=scale, q_norm=qw, k_norm=kw, **more)
    within(qo, *reference(q, positions, inv_freq, inter, scale, qw), "q")
    if k is not None:
        within(ko, *reference(k, positions, inv_freq, inter, scale, kw), "k")
    return qo, ko


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norms", ["", "q", "k", "qk"])
@pytest.mark.parametrize("heads,kv", [(32, 8), (5, 1), (3, 3)])
@pytest.mark.parametrize("tokens", [1, 2, 77, 1300])
def test_rope(dim, inter, norms, heads, kv, tokens):
    g = gen(tokens + dim)
    y = randn(tokens, heads + 2 * kv, dim, g=g, scale=3)  # views of one fused output
    w = [1 + torch.randn(dim, device="cuda", generator=g) if n in norms else None for n in "qk"]
    positions = torch.randint(0, 200000, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    check(y[:, :heads], y[:, heads:heads + kv], positions, freqs(dim // 2), inter, 1.25, *w)


@pytest.mark.parametrize("dim,half", [(64, 32), (128, 64), (128, 48), (128, 21)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norms", [False, True])
def test_products_and_sums_are_rounded_one_by_one(dim, half, inter, norms):
    """The formula in f32, operation by operation, bit for bit: no product goes into its sum unrounded."""
    g = gen(dim + half)
    T = 1500
    q = randn(T, 8, dim, g=g)
    w = 1 + torch.rand(dim, device="cuda", generator=g) if norms else None
    positions = torch.randint(0, 1 << 20, (T,), device="cuda", generator=g, dtype=torch.int32)
    y, f = q.float(), freqs(half)
    if norms:
        y = y * torch.rsqrt(q.double().square().mean(-1, keepdim=True) + EPS).float() * w
    a = positions.double()[:, None, None] * f.double()
    c, s = (a.cos() * 1.25).float(), (a.sin() * 1.25).float()
    y1, y2 = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if inter else (y[..., :half], y[..., half:2 * half])
    one, two = y1 * c - y2 * s, y2 * c + y1 * s
    turned = torch.stack([one, two], -1).flatten(-2) if inter else torch.cat([one, two], -1)
    want = torch.cat([turned, y[..., 2 * half:]], -1).bfloat16()
    got, _ = A().rope(q, None, positions, f, interleaved=inter, scale=1.25, q_norm=w)
    # cos, sin and r of 64 bits come out of two libraries' last places: after f32 they differ once in 2^28
    assert int((bits(got) != bits(want)).sum()) <= 2


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("half", [0, 1, 5, 8, 15, 16, 24, 31, 32, 48, 63, 64])
def test_part_of_the_head(dim, inter, half):
    """The places behind the rotated ones stay as they are, whatever stands there."""
    if half > dim // 2:
        pytest.skip("more than the head has")
    g = gen(half + dim)
    q, k = randn(9, 4, dim, g=g), randn(9, 2, dim, g=g)
    q[0, 0, 2 * half:] = float("nan")
    q[1, 1, 2 * half:] = -0.0
    q[2, 2, 2 * half:] = float("inf")
    positions = torch.arange(9, dtype=torch.int32, device="cuda") * 1009
    qo, ko = A().rope(q, k, positions, freqs(half), interleaved=inter)
    within(qo, *reference(q, positions, freqs(half), inter, 1.0, None), "q")
    within(ko, *reference(k, positions, freqs(half), inter, 1.0, None), "k")
    rest, was = qo[..., 2 * half:], q[..., 2 * half:]
    assert torch.equal(rest.isnan(), was.isnan()) and torch.equal(bits(rest)[~was.isnan()], bits(was)[~was.isnan()])
    w = torch.linspace(0.5, 2, dim, device="cuda")
    check(q[3:], k[3:], positions[3:], freqs(half), inter, 0.75, w, w.flip(0).contiguous())


@pytest.mark.parametrize("inter", [False, True])
def test_far_positions(inter):
    """Angles of far positions, the farthest and negative ones among them."""
    g = gen(3)
    positions = torch.tensor([0, -1, 131071, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    q, k = randn(7, 6, 128, g=g), randn(7, 2, 128, g=g)
    check(q, k, positions, freqs(64, 500000.0), inter)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("norms", [False, True])
def test_layouts(dim, norms):
    """Heads before tokens, odd offsets and strides, in place, without keys, without tokens: one answer."""
    g = gen(dim)
    T, H, KV = 133, 6, 2
    q, k = randn(T, H, dim, g=g), randn(T, KV, dim, g=g)
    w = dict(q_norm=1 + torch.rand(dim, device="cuda", generator=g), k_norm=1 + torch.rand(dim, device="cuda", generator=g)) \
        if norms else {}
    positions = torch.arange(T, dtype=torch.int32, device="cuda")
    f = freqs(dim // 2)
    for inter in (False, True):
        qo, ko = A().rope(q, k, positions, f, interleaved=inter, **w)

        def same(a, b):
            assert torch.equal(bits(a), bits(qo)) and (b is None or torch.equal(bits(b), bits(ko)))
        ht = q.transpose(0, 1).contiguous().transpose(0, 1)  # [heads, tokens, dim] in memory
        out = torch.empty_like(ht)
        same(*A().rope(ht, k, positions, f, interleaved=inter, q_out=out, **w))
        wide = torch.zeros(T, H + KV + 1, dim + 3, dtype=torch.bfloat16, device="cuda")  # rows at odd addresses
        wide[:, :H, 1:dim + 1], wide[:, H:H + KV, 1:dim + 1] = q, k
        wq, wk = wide[:, :H, 1:dim + 1], wide[:, H:H + KV, 1:dim + 1]
        same(*A().rope(wq, wk, positions, f, interleaved=inter, **w))
        was = wide.clone()
        same(*A().rope(wq, wk, positions, f, interleaved=inter, q_out=wq, k_out=wk, **w))  # in place
        was[:, :H, 1:dim + 1], was[:, H:H + KV, 1:dim + 1] = qo, ko
        assert torch.equal(bits(wide), bits(was)), "something beside the heads was written"
        fused = torch.cat([q, k], 1)
        same(*A().rope(fused[:, :H], fused[:, H:], positions, f, interleaved=inter, q_out=fused[:, :H],
                       k_out=fused[:, H:], **w))
        alone, none = A().rope(q, None, positions, f, interleaved=inter, q_norm=w.get("q_norm"))
        same(alone, None)
        assert none is None
    e, z = A().rope(q[:0], k[:0], positions[:0], f)
    assert e.shape == (0, H, dim) and z.shape == (0, KV, dim)
    assert A().rope(q, k[:, :0], positions, f)[1].shape == (T, 0, dim)


def test_values_that_are_not_finite_stay_in_their_head():
    g = gen(5)
    T = 40
    q, k = randn(T, 4, 128, g=g), randn(T, 2, 128, g=g)
    positions = torch.arange(T, dtype=torch.int32, device="cuda")
    w = torch.ones(128, device="cuda")
    for kw in (dict(), dict(q_norm=w, k_norm=w)):
        want = A().rope(q, k, positions, freqs(64), **kw)
        for bad in (float("nan"), float("inf"), -float("inf"), 3e38):
            p = q.clone()
            p[7, 2, 9] = bad
            got = A().rope(p, k, positions, freqs(64), **kw)
            mask = torch.ones(T, 4, dtype=torch.bool, device="cuda")
            mask[7, 2] = False
            assert torch.equal(bits(got[0])[mask], bits(want[0])[mask]) and torch.equal(bits(got[1]), bits(want[1]))
            if not math.isfinite(bad):
                assert not bool(got[0][7, 2, [9, 73]].isfinite().any())
    tiny = torch.full((1, 1, 128), 1e-30, dtype=torch.bfloat16, device="cuda")  # squares far below eps
    check(tiny, None, positions[:1], freqs(64), qw=w)
    zero = A().rope(tiny * 0, None, positions[:1], freqs(64), q_norm=w)[0]
    assert bool((zero == 0).all())


@pytest.mark.parametrize("dim,page", [(64, 16), (64, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("heads,kv", [(10, 5), (8, 1)])
@pytest.mark.parametrize("tokens", [1, 6, 83, 1200])
def test_append_is_rope_and_then_append(dim, page, inter, norms, heads, kv, tokens):
    """The same queries and the same bytes; skipped tokens and other slots' bytes as they were."""
    g = gen(tokens + dim + page)
    y = randn(tokens, heads + 2 * kv, dim, g=g)
    q, k, v = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    w = dict(q_norm=1 + torch.rand(dim, device="cuda", generator=g), k_norm=1 + torch.rand(dim, device="cuda", generator=g)) \
        if norms else {}
    half = dim // 2 if page != 32 else 24  # at page 32: partners through shared memory
    if tokens > 5:
        y[3, heads, 5], y[4, heads + kv, 7] = float("nan"), float("inf")  # blocks of k and v that read as NaN
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].int()
    if tokens > 5:
        slots[1], slots[2], slots[5] = -1, pages * page, 2 ** 31 - 1  # outside: rotated, not cached
    positions = torch.randint(0, 70000, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    kw = dict(interleaved=inter, scale=1.1, **w)
    caches = []
    for _ in range(2):
        c = A().KV4Cache.empty(pages, kv, dim, page)
        for t in (c.k_code, c.v_code, c.k_meta.view(torch.uint8), c.v_meta.view(torch.uint8)):
            t.fill_(0x5A)
        caches.append(c)
    qo, ko = A().rope(q, k, positions, freqs(half), **kw)
    A().kv4_append(caches[0], ko, v, slots)

    def same():
        for n in ("k_code", "v_code", "k_meta", "v_meta"):
            a, b = (getattr(c, n).view(torch.uint8) for c in caches)
            assert torch.equal(a, b), n
    got = A().rope_append(caches[1], q, k, v, positions, freqs(half), slots, **kw)
    assert torch.equal(bits(got), bits(qo))
    same()
    out = torch.empty(tokens, kv, dim, dtype=torch.bfloat16, device="cuda")
    for t in (caches[1].k_code, caches[1].v_code):
        t.fill_(0x5A)
    got = A().rope_append(caches[1], q, k, v, positions, freqs(half), slots, q_out=q, k_out=out, **kw)  # q in place
    assert torch.equal(bits(got), bits(qo)) and torch.equal(bits(out), bits(ko)) and torch.equal(bits(q), bits(qo))
    same()


def test_run_of_a_layer():
    """A prompt rotated into the cache, its attention, then a token over the cache: the last prompt
    token again gives what attention over the read-back keys gives."""
    g = gen(11)
    T, H, KV, D = 150, 8, 2, 128
    y = randn(T, H + 2 * KV, D, g=g)
    q, k, v = y[:, :H], y[:, H:H + KV], y[:, H + KV:]
    i32 = dict(dtype=torch.int32, device="cuda")
    at, table, slots = torch.arange(T, **i32), torch.arange(3, **i32)[None], torch.arange(T, **i32)
    f, scale = A().rope_freqs(D, 10000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=64))
    cache = A().KV4Cache.empty(3, KV, D, 64)
    raw = y.clone()
    A().rope_append(cache, q, k, v, at, f, slots, scale=scale, q_out=q, k_out=k)  # in the linear's output
    assert torch.equal(bits(y[:, H + KV:]), bits(raw[:, H + KV:]))
    o, _ = A().attn_prompt(q, k, v, torch.tensor([0, T], **i32))
    for x, n, w in ((q, slice(0, H), "q"), (k, slice(H, H + KV), "k")):
        within(x, *reference(raw[:, n], at, f, False, scale, None), w)
    o1, _ = A().kv4_attn(q[-1:, None], cache, table, torch.tensor([T], **i32))
    kc, vc = A().kv4_read(cache, slots)
    for keys, vals, got in ((k, v, o[-1]), (kc, vc, o1[0, 0])):
        qd = q[-1].double().view(KV, H // KV, D)
        p = torch.softmax(torch.einsum("hgd,jhd->hgj", qd, keys.double()) * D ** -0.5, -1)
        want = torch.einsum("hgj,jhd->hgd", p, vals.double()).reshape(H, D)
        part = torch.einsum("hgj,jhd->hgd", p, vals.double().abs()).reshape(H, D)
        # o and every weight rounded to BF16, over the cache weight * step too: 2^-8 each, of sum p |v| and its range
        assert bool(((got.double() - want).abs() <= 2.0 ** -7 * (want.abs() + 2 * part + vals.double().abs().max())).all())


def test_streams_and_graphs():
    g = gen(12)
    T, H, KV, D = 7, 8, 2, 128
    y = randn(T, H + 2 * KV, D, g=g)
    q, k, v = y[:, :H], y[:, H:H + KV], y[:, H + KV:]
    i32 = dict(dtype=torch.int32, device="cuda")
    positions, slots = torch.arange(T, **i32), torch.arange(T, **i32)
    want = A().rope(q, k, positions, freqs(64))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = A().rope(q, k, positions, freqs(64), stream=side)
    side.synchronize()
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))
    cache = A().KV4Cache.empty(1, KV, D, 16)
    f = freqs(64)
    A().rope_append(cache, q, k, v, positions, f, slots)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo = A().rope_append(cache, q, k, v, positions, f, slots)
    y.copy_(randn(T, H + 2 * KV, D, g=g))
    positions += 1000
    graph.replay()
    wq, wk = A().rope(q, k, positions, f)
    other = A().KV4Cache.empty(1, KV, D, 16)
    A().kv4_append(other, wk, v, slots)
    assert torch.equal(bits(qo), bits(wq))
    assert all(torch.equal(a, b) for a, b in zip(A().kv4_read(cache, slots), A().kv4_read(other, slots)))


def test_refusals():
    i32 = dict(dtype=torch.int32, device="cuda")
    q, k = torch.zeros(4, 6, 128, device="cuda").bfloat16(), torch.zeros(4, 2, 128, device="cuda").bfloat16()
    p, f, w = torch.arange(4, **i32), freqs(64), torch.ones(128, device="cuda")
    A().rope(q, k, p, f, q_norm=w)
    cache = A().KV4Cache.empty(1, 2, 128, 16)
    bad = [(dict(q=q.float()), "bfloat16"), (dict(q=q.cpu()), "CUDA"), (dict(q=q[..., :96]), "head_dim"), (dict(q=q[:, :0]), "head"),
           (dict(k=k[:3]), "shape"), (dict(k=k[..., ::2].repeat(1, 1, 2)[..., ::2]), "shape|contiguous"),
           (dict(positions=p.long()), "int32"), (dict(positions=p[:3]), "shape"), (dict(inv_freq=f.double()), "float32"),
           (dict(inv_freq=freqs(65)), "frequencies"), (dict(inv_freq=f[::2]), "contiguous"), (dict(q_norm=w.bfloat16()), "float32"),
           (dict(q_norm=w[:64]), "shape"), (dict(q_norm=torch.ones(129, device="cuda")[1:]), "aligned"), (dict(eps=0.0), "eps"),
           (dict(eps=float("nan")), "eps"), (dict(scale=float("inf")), "scale"), (dict(k=None, k_norm=w), "need k"),
           (dict(k=None, k_out=k), "need k"), (dict(q_out=q[:3]), "shape"), (dict(k_out=q[:, :2]), "overlap"),
           (dict(q_out=q.flip(0)[:1].expand(4, 6, 128)), "overlap"), (dict(q_out=q[:, :1].expand(4, 6, 128)), "overlap")]
    for kw, match in bad:
        with pytest.raises(ValueError, match=match):
            A().rope(**{**dict(q=q, k=k, positions=p, inv_freq=f), **kw})
    big = torch.zeros(5, 6, 128, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="overlap"):
        A().rope(big[:4], None, p, f, q_out=big[1:])  # a row further
    both = torch.zeros(4, 8, 128, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="apart"):
        A().rope(q, k, p, f, q_out=both[:, :6], k_out=both[:, 5:7])
    slots = torch.arange(4, **i32)
    for kw, match in ((dict(k=k[:, :1]), "shape"), (dict(v=k[:, :, :64]), "shape"), (dict(slots=slots.long()), "int32"),
                      (dict(slots=slots[:2]), "shape"), (dict(v=q[:, :2], q_out=q), "overlap")):
        with pytest.raises(ValueError, match=match):
            A().rope_append(**{**dict(cache=cache, q=q, k=k, v=k.clone(), positions=p, inv_freq=f, slots=slots), **kw})
