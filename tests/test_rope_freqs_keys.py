"""rope_freqs takes a model's rope_scaling: every key of it that changes the frequencies or the scale counts, and one
that it does not read is refused."""
import math

import pytest

torch = pytest.importorskip("torch")

LENGTH = dict(original_max_position_embeddings=4096)


def freqs(dim, base, scaling):
    from glint_b200 import attn
    inv, scale = attn.rope_freqs(dim, base, scaling, device="cpu")
    return inv.double().tolist(), scale


def yarn(dim, base, factor, length, fast=32.0, slow=1.0, truncate=True):
    """The published formula, a frequency at a time."""
    def number(turns):
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = number(fast), number(slow)
    if truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    out = []
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        ramp = min(1.0, max(0.0, (i - low) / (high - low)))
        out.append(f / factor * ramp + f * (1 - ramp))
    return out


@pytest.mark.parametrize("truncate", [True, False])
@pytest.mark.parametrize("dim,base,factor,length", [(64, 150000.0, 32.0, 4096), (128, 10000.0, 40.0, 4096), (96, 1e6, 4.0, 32768)])
def test_ends_of_the_ramp(dim, base, factor, length, truncate):
    got, _ = freqs(dim, base, dict(rope_type="yarn", factor=factor, original_max_position_embeddings=length, truncate=truncate))
    want = yarn(dim, base, factor, length, truncate=truncate)
    assert all(abs(a - b) <= 2.0 ** -23 * b for a, b in zip(got, want)), (got, want)


def test_whole_ends_are_the_default():
    plain = dict(rope_type="yarn", factor=32.0, **LENGTH)
    assert freqs(64, 150000.0, plain) == freqs(64, 150000.0, dict(plain, truncate=True))
    assert freqs(64, 150000.0, plain) == freqs(64, 150000.0, dict(plain, truncate=None))
    assert freqs(64, 150000.0, plain)[0] != freqs(64, 150000.0, dict(plain, truncate=False))[0]


def test_scale():
    def scale(factor=40.0, **kw):
        return freqs(64, 1e4, dict(type="yarn", factor=factor, **LENGTH, **kw))[1]

    def m(by, factor=40.0):
        return 0.1 * by * math.log(factor) + 1
    assert scale(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert abs(scale(mscale=0.707, mscale_all_dim=1.0) - m(0.707) / m(1.0)) < 1e-15
    assert abs(scale(mscale=2, mscale_all_dim=0.5) - m(2) / m(0.5)) < 1e-15
    assert abs(scale() - m(1)) < 1e-15 and abs(scale(mscale=None, mscale_all_dim=None) - m(1)) < 1e-15
    assert scale(mscale=2.0, mscale_all_dim=0.5, attention_factor=1.25) == 1.25
    assert scale(factor=1.0, mscale=2.0, mscale_all_dim=0.5) == 1.0
    for kw in (dict(mscale=1.0), dict(mscale_all_dim=1.0), dict(mscale=0.0, mscale_all_dim=1.0), dict(mscale=1.0, mscale_all_dim=-1.0)):
        with pytest.raises(ValueError, match="mscale"):
            scale(**kw)


GOOD = dict(
    default=dict(rope_type="default"),
    linear=dict(rope_type="linear", factor=2.0),
    llama3=dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, **LENGTH),
    yarn=dict(rope_type="yarn", factor=4.0, **LENGTH),
    longrope=dict(rope_type="longrope", factors=[1.5] * 32, factor=4.0, **LENGTH),
)


@pytest.mark.parametrize("kind", sorted(GOOD))
def test_keys_that_are_not_read(kind):
    for key, v in (("mrope_section", [16, 24, 24]), ("alpha", 1000.0), ("beta", 3.0), ("scale", 2.0)):
        with pytest.raises(ValueError, match=key):
            freqs(64, 1e4, {**GOOD[kind], key: v})
    if kind != "yarn":
        for key in ("beta_fast", "mscale", "truncate"):
            with pytest.raises(ValueError, match=key):
                freqs(64, 1e4, {**GOOD[kind], key: 1})
    if kind in ("default", "linear", "llama3"):
        with pytest.raises(ValueError, match="attention_factor"):
            freqs(64, 1e4, {**GOOD[kind], "attention_factor": 1.5})


@pytest.mark.parametrize("kind", sorted(GOOD))
def test_keys_that_change_nothing(kind):
    want = freqs(64, 1e4, GOOD[kind])
    more = dict(rope_theta=10000.0, finetuned=True, partial_rotary_factor=0.5, original_max_position_embeddings=4096, mrope_section=None)
    if kind == "longrope":
        more.update(short_factor=[1.0] * 32, long_factor=[1.5] * 32)
    assert freqs(64, 1e4, {**GOOD[kind], **more}) == want
    with pytest.raises(ValueError, match="rope_theta"):
        freqs(64, 1e4, {**GOOD[kind], "rope_theta": 500000.0})


def test_factors_in_a_tensor():
    factors = [1 + i / 8 for i in range(32)]
    want = freqs(64, 1e4, dict(rope_type="longrope", factors=factors, factor=4.0, **LENGTH))
    for f in (torch.tensor(factors), torch.tensor(factors, dtype=torch.float64), tuple(factors)):
        assert freqs(64, 1e4, dict(rope_type="longrope", factors=f, factor=4.0, **LENGTH)) == want
    assert freqs(64, 1e4, dict(rope_type="longrope", factors=factors))[1] == 1.0
    assert freqs(64, 1e4, dict(rope_type="longrope", factors=factors, factor=4.0, attention_factor=1.5))[1] == 1.5


def test_sizes_without_a_logarithm():
    for base, scaling in ((1.0, dict(rope_type="yarn", factor=4.0, **LENGTH)),
                          (1e4, dict(rope_type="longrope", factors=[1.0] * 32, factor=4.0, original_max_position_embeddings=1))):
        with pytest.raises(ValueError):
            freqs(64, base, scaling)
    for scaling in (dict(rope_type="longrope"), dict(rope_type="longrope", factors=torch.ones(31)), dict(rope_type="longrope", factors=[])):
        with pytest.raises(ValueError, match="factors"):
            freqs(64, 1e4, scaling)
