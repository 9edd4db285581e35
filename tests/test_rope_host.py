"""What rope and rope_append decide on the host, without a GPU: arguments of the C entry points
(checked before any device work), which outputs may lie where, stretched frequencies."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from glint_b200 import attn, build
    build.build()
    return attn._lib()


def structs(**kw):
    from glint_b200 import attn
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    cache = attn._Cache(p, p, p, p, 4, 2, 64, 128)
    a = attn._Rope(p, p, p, p, p, p, None, None, *[8] * 8, 1.0, 1e-6, 4, 8, 2, 128, 64, 0)
    for n, v in kw.items():
        setattr(a, n, p + 4 if v == "odd" else v)
    return buf, p, cache, a


def test_arguments(lib):
    for kw, rc in ((dict(q=None), -1), (dict(k=None), -1), (dict(q_out=None), -1), (dict(k_out=None), -1), (dict(positions=None), -1),
                   (dict(inv_freq=None), -1), (dict(tokens=-1), -1), (dict(heads=0), -1), (dict(kv_heads=-1), -1),
                   (dict(half=65), -1), (dict(half=-1), -1), (dict(eps=0.0), -1), (dict(eps=math.nan), -1),
                   (dict(q_norm="odd"), -1), (dict(k_norm="odd"), -1), (dict(head_dim=96), -6), (dict(head_dim=256), -6),
                   (dict(heads=2 ** 31 - 1), -1), (dict(tokens=0), 0), (dict(tokens=0, q=None), 0)):
        _, p, cache, a = structs(**kw)
        assert lib.glint_rope_stream(a, None) == rc, kw
        if "k_out" not in kw:
            assert lib.glint_kv4_rope_append_stream(cache, a, p, 8, 8, p, None) == rc, kw
    _, p, cache, a = structs()
    assert lib.glint_rope_stream(None, None) == -1
    assert lib.glint_kv4_rope_append_stream(None, a, p, 8, 8, p, None) == -1
    assert lib.glint_kv4_rope_append_stream(cache, None, p, 8, 8, p, None) == -1
    assert lib.glint_kv4_rope_append_stream(cache, a, None, 8, 8, p, None) == -1
    assert lib.glint_kv4_rope_append_stream(cache, a, p, 8, 8, None, None) == -1
    for kw in (dict(kv_heads=3), dict(kv_heads=0), dict(head_dim=64, half=32)):  # other heads than the cache's
        _, p, cache, a = structs(**kw)
        assert lib.glint_kv4_rope_append_stream(cache, a, p, 8, 8, p, None) == -1, kw
    cache.page_size = 48
    assert lib.glint_kv4_rope_append_stream(cache, a, p, 8, 8, p, None) == -6


def test_python_refuses_cpu_tensors():
    from glint_b200 import attn
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attn.rope(q, q, torch.arange(4, dtype=torch.int32), torch.ones(64))


def places(t):
    base = t.storage_offset()
    T, H, D = t.shape
    return [base + i * t.stride(0) + h * t.stride(1) + d for i in range(T) for h in range(H) for d in range(D)]


def test_outputs_that_may_overlap_are_found():
    """Every answer "apart" is right, and the layouts that are used get it."""
    from glint_b200 import attn
    views = []
    for shape, strides in (((3, 2, 4), (16, 4, 1)), ((3, 1, 4), (16, 4, 1)), ((3, 2, 4), (8, 4, 1)), ((2, 2, 4), (4, 12, 1)),
                           ((3, 2, 4), (5, 4, 1)), ((3, 2, 4), (0, 4, 1)), ((3, 2, 4), (16, 0, 1)), ((1, 3, 4), (7, 4, 1)),
                           ((0, 2, 4), (8, 4, 1)), ((3, 2, 4), (16, 5, 1))):
        for off in (0, 4, 8, 9, 12, 24, 48):
            views.append(torch.arange(200, dtype=torch.int16).as_strided(shape, strides, off))
    store = torch.zeros(200, dtype=torch.int16)
    views = [store.as_strided(v.shape, v.stride(), v.storage_offset()) for v in views]
    for a in views:
        if attn._heads_apart(a):
            assert len(set(places(a))) == a.numel(), (a.shape, a.stride())
        for b in views:
            if attn._rows_apart(a, b):
                assert not set(places(a)) & set(places(b)), (a.shape, a.stride(), a.storage_offset(), b.stride(), b.storage_offset())
    y = torch.zeros(5, 8, 64, dtype=torch.bfloat16)
    assert attn._rows_apart(y[:, :4], y[:, 4:6]) and attn._rows_apart(y[:, 4:6], y[:, :4]) and attn._rows_apart(y, y.clone())
    assert not attn._rows_apart(y[:, :4], y[:, 3:6]) and not attn._rows_apart(y[:4], y[1:])
    for t in (y, y[:, :3], y.transpose(0, 1), y[:1].expand(1, 8, 64), y[:, :1]):
        assert attn._heads_apart(t)
    assert not attn._heads_apart(y[:1].expand(5, 8, 64)) and not attn._heads_apart(y[:, :1].expand(5, 8, 64))


def test_frequencies():
    from glint_b200 import attn

    def f(dim, base, scaling=None):
        inv, scale = attn.rope_freqs(dim, base, scaling, device="cpu")
        assert inv.dtype is torch.float32 and inv.shape == (dim // 2,)
        return inv.double().tolist(), scale
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]

    def near(got, want):
        assert all(abs(a - b) <= 2.0 ** -24 * b for a, b in zip(got, want)), (got, want)
    got, scale = f(64, 10000.0)
    near(got, plain)
    assert scale == 1.0
    got, scale = f(64, 10000.0, dict(type="linear", factor=4))
    near(got, [v / 4 for v in plain])
    got, scale = f(64, 10000.0, dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                     original_max_position_embeddings=8192))
    want = []
    for v in plain:
        wave = 2 * math.pi / v
        if wave < 8192 / 4:
            want.append(v)
        elif wave > 8192:
            want.append(v / 8)
        else:
            smooth = (8192 / wave - 1) / 3
            want.append((1 - smooth) * v / 8 + smooth * v)
    near(got, want)
    assert scale == 1.0 and got[0] == plain[0] and got[-1] < plain[-1] / 7
    got, scale = f(64, 10000.0, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096))

    def number(turns):
        return 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))
    low, high = math.floor(number(32)), math.ceil(number(1))
    ramp = [min(1, max(0, (i - low) / (high - low))) for i in range(32)]
    near(got, [v / 16 * r + v * (1 - r) for v, r in zip(plain, ramp)])
    assert abs(scale - (0.1 * math.log(16) + 1)) < 1e-15
    assert f(64, 1e4, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096, attention_factor=1.5))[1] == 1.5
    factors = [1 + i / 8 for i in range(24)]
    got, scale = f(48, 10000.0, dict(rope_type="longrope", factors=factors, factor=32.0, original_max_position_embeddings=4096))
    near(got, [10000.0 ** (-2 * i / 48) / by for i, by in enumerate(factors)])
    assert abs(scale - math.sqrt(1 + math.log(32) / math.log(4096))) < 1e-15
    assert f(0, 10000.0) == ([], 1.0)
    for dim, scaling in ((63, None), (64, dict(rope_type="other")), (64, dict(rope_type="linear")), (64, dict(type="linear", factor=0)),
                         (64, dict(rope_type="longrope", factors=[1.0] * 31)), (64, dict(rope_type="longrope", factors=[-1.0] * 32)),
                         (64, dict(rope_type="llama3", factor=8, low_freq_factor=4, high_freq_factor=4,
                                   original_max_position_embeddings=8192)),
                         (64, dict(rope_type="yarn", factor=2))):
        with pytest.raises(ValueError):
            attn.rope_freqs(dim, 10000.0, scaling, device="cpu")
    with pytest.raises(ValueError):
        attn.rope_freqs(64, 0.0, device="cpu")
