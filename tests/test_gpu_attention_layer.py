"""The attention layer example (examples/attention_layer.py): prompts, cache, tokens and
eviction together, against plain attention over what the cache reads as."""
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from glint_b200 import build
    build.build()
    torch.cuda.set_device(0)


def test_layer_prompts_tokens_and_eviction():
    import attention_layer as example
    from glint_b200 import attn, device
    hidden, heads, kv, dim, lens, budget, recent = 512, 4, 2, 128, [90, 1, 260], 64, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    wqkv, wo = (example.random_planes((heads + 2 * kv) * dim, hidden, g), example.random_planes(hidden, heads * dim, g))
    layer = example.AttentionLayer(wqkv, wo, hidden, heads, kv, dim, len(lens), max(lens) + 40, budget, recent, slack=4)
    x = torch.randn(sum(lens), hidden, device="cuda", generator=g).bfloat16()
    y = layer.prompt(x, lens)
    assert y.shape == (sum(lens), hidden) and bool(y.isfinite().all())
    assert layer.lens.tolist() == [min(n, budget) for n in lens]

    # a prompt of one token attends to itself: o is its v, through the o linear
    v = device.htile(x[90:91], *wqkv, (heads + 2 * kv) * dim, mode="fast", out_dtype=torch.bfloat16)
    v = v.view(heads + 2 * kv, dim)[heads + kv:].repeat_interleave(heads // kv, 0).reshape(1, -1).contiguous()
    want = device.htile(v, *wo, hidden, mode="fast", out_dtype=torch.bfloat16)
    # the same bits into a row of a larger product: BF16 roundings of sums of 512 terms, in any order
    bound = 2.0 ** -7 * want.double().abs() + 512 * 2.0 ** -22 * v.double().abs().sum()
    assert bool(((y[90:91].double() - want.double()).abs() <= bound).all())

    z = torch.randn(len(lens), hidden, device="cuda", generator=g).bfloat16()
    for i in range(12):
        before = layer.lens.clone()
        q = device.htile(z, *wqkv, (heads + 2 * kv) * dim, mode="fast", out_dtype=torch.bfloat16)
        q = q.view(len(lens), heads + 2 * kv, dim)[:, :heads]
        evicting = layer.longest + 1 > budget + layer.slack
        out = layer.step(z)
        assert bool(out.isfinite().all())
        if not evicting:  # the slots are still those that the step attended to
            for b in range(len(lens)):
                n = int(before[b]) + 1
                t = torch.arange(n, device="cuda")
                k, v = (a.double() for a in attn.kv4_read(layer.cache, layer._slots(torch.full_like(t, b), t)))
                for h in range(heads):
                    kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
                    p = torch.softmax(kh @ q[b, h].double() * dim ** -0.5, 0)
                    # keys and values as read carry one more BF16 rounding (2^-8) than the kernel's:
                    # of the scores, of the values and of the result, and the kernel's weights' own
                    ds = 2.0 ** -8 * dim ** -0.5 * (kh.abs() @ q[b, h].double().abs()).max()
                    bound = (2 * ds + 2.0 ** -6) * (p @ vh.abs())
                    diff = (layer.attended[b, 0, h].double() - p @ vh).abs()
                    assert bool((diff <= bound).all())
        assert int(layer.lens.max()) <= budget + layer.slack
    assert layer.seen.tolist() == [n + 12 for n in lens]
    # protected tokens are still there: the newest `recent` positions of the long sequence
    held = layer.pos[0][2, 0, :int(layer.lens[2])].tolist()
    assert set(range(272 - recent, 272)) <= set(held) and len(set(held)) == len(held)
