"""GPU tests of the serving attention operators past the lengths of test_gpu_attn.py: prompts
whose keys are cut over the SMs, values that are not finite at such lengths, eviction with more
slots than a CTA's shared memory holds keys.  References and bounds are that file's."""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_attn import (A, bits, check_prompt, cu, evict_reference, gen, gpu, kernel_error,  # noqa: E402,F401
                           prompt_reference, quantise, randn, values, within)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,lq,lk", [(8, 2, [1], [1000]), (4, 4, [130], [9000]), (16, 1, [17], [897]),
                                            (5, 1, [100, 30], [5000, 3001]), (2, 2, [5, 0, 64, 1], [1024, 2000, 4097, 7]),
                                            (1, 1, [300], [2049])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_keys_cut_over_sms(dim, heads, kv, lq, lk, causal):
    """Few queries with many keys: parts of the keys, joined by a second kernel."""
    g = gen(sum(lk) + dim)
    check_prompt(randn(sum(lq), heads, dim, g=g), randn(sum(lk), kv, dim, g=g), randn(sum(lk), kv, dim, g=g), lq, lk, causal)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_cut_large_scores(dim):
    """Parts whose maxima lie far apart."""
    g = gen(dim + 1)
    k = randn(6000, 2, dim, g=g) * torch.linspace(0.1, 20, 6000, device="cuda")[:, None, None].bfloat16()
    q, v = randn(90, 4, dim, g=g, scale=4), randn(6000, 2, dim, g=g)
    check_prompt(q, k, v, [90], [6000])
    check_prompt(q, k.flip(0).contiguous(), v, [90], [6000])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("heads,kv,lq,lk", [(4, 2, [200], [5000]), (4, 1, [40, 150], [3000, 1200]), (64, 32, [700], [700])])
def test_prompt_masked_values_stay_out_of_long_rows(dim, bad, heads, kv, lq, lk):
    """As for short sequences: with the keys cut, and with more blocks than are cut."""
    g = gen(dim + sum(lk))
    n, m = sum(lq), sum(lk)
    q, k, v = randn(n, heads, dim, g=g), randn(m + 50, kv, dim, g=g), randn(m + 50, kv, dim, g=g)
    want = prompt_reference(q, k[:m], v[:m], lq, lk, True, dim ** -0.5)
    for tail in (1, 30, 97):  # the last keys of every sequence
        k2, v2 = k.clone(), v.clone()
        rows = torch.ones(n, dtype=torch.bool, device="cuda")
        at = kat = 0
        for a, b in zip(lq, lk):
            at, kat = at + a, kat + b
            rows[max(at - a, at - tail):at] = False
            for x in (k2, v2):
                x[kat - tail:kat] = bad
        for x in (k2, v2):
            x[m:] = bad
        o, lse = A().attn_prompt(q, k2, v2, cu(lq), cu(lk))
        assert kernel_error() == 0
        within(o[rows], want[0][rows], want[1][rows], "o")
        within(lse[:, rows], want[2][:, rows], want[3][:, rows], "lse")


@pytest.mark.parametrize("length,page", [(330001, 128), (524288, 64), (5000, 128)])
def test_evict_past_the_keys_held(length, page):
    """A table of 524288 slots: weights are read again for every digit.  Ties run over every
    stretch of slots; rows, weights and positions move as `kept` says."""
    g = gen(length)
    kv, dim, pages, budget, recent = 1, 64, 524288 // page, 4001, 100
    cache = A().KV4Cache.empty(pages, kv, dim, page)
    for t in (cache.k_code, cache.v_code):
        t.copy_(torch.randint(0, 256, t.shape, device="cuda", generator=g, dtype=torch.uint8))
    for t in (cache.k_meta, cache.v_meta):
        t.copy_(torch.rand(t.shape, device="cuda", generator=g))
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)[None]
    w = torch.randint(0, 40, (1, kv, pages * page), device="cuda", generator=g).float()  # the 4001st is one of thousands
    pos = torch.rand(w.shape, device="cuda", generator=g).argsort(-1).to(torch.int32)
    seen = torch.tensor([pages * page], dtype=torch.int32, device="cuda")
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    t = torch.arange(length, device="cuda")
    slots = (table[0, t // page] * page + t % page).int()
    before = A().kv4_read(cache, slots)
    wo, po = torch.full_like(w, -1.0), torch.full_like(pos, -1)
    kept, new = A().kv4_evict(cache, table, lens, w, pos, seen, budget, recent, weight_out=wo, pos_out=po)
    after = A().kv4_read(cache, slots)
    n = min(length, budget)
    assert int(new) == n
    want = evict_reference(w[0, 0].tolist(), pos[0, 0].tolist(), pages * page, length, budget, recent)
    assert kept[0, 0].tolist() == want + [-1] * (budget - n)
    src = torch.tensor(want, dtype=torch.long, device="cuda")
    assert torch.equal(wo[0, 0, :n], w[0, 0][src]) and torch.equal(po[0, 0, :n], pos[0, 0][src])
    assert bool((wo[0, 0, n:] == -1).all()) and bool((po[0, 0, n:] == -1).all())
    for x, y in zip(before, after):
        assert torch.equal(bits(y[:n]), bits(x[src])) and torch.equal(bits(y[n:]), bits(x[n:]))


def gpu_ms(f, n=3):
    f()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    for _ in range(n):
        f()
    end.record()
    end.synchronize()
    return begin.elapsed_time(end) / n


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk", [(4096, 4096), (100, 20000)])
def test_prompt_masked_values_cost_little(dim, lq, lk):
    """Values that are not finite past the last sequence, and at its last key: a look at V (its
    bytes are a small part of the call) for the blocks that meet them, and no more."""
    g = gen(dim + lq)
    q, k, v = randn(lq, 8, dim, g=g), randn(lk + 64, 8, dim, g=g), randn(lk + 64, 8, dim, g=g)
    a = (cu([lq]), cu([lk]))
    clean = gpu_ms(lambda: A().attn_prompt(q, k, v, *a))
    want = A().attn_prompt(q, k, v, *a)[0]
    v[lk - 1:] = float("nan")
    bad = gpu_ms(lambda: A().attn_prompt(q, k, v, *a))
    got = A().attn_prompt(q, k, v, *a)[0]
    assert kernel_error() == 0
    assert bool(got[-1].isnan().all()) and torch.equal(got[:-1], want[:-1])
    assert bad <= 4 * clean + 0.2, f"{bad:.3f} ms against {clean:.3f}"


def test_prompt_masked_values_stay_out_of_very_long_rows():
    """300000 keys, more blocks than are cut: nothing a block does for odd values may outlast the
    bounded waits of its other warps."""
    g = gen(77)
    n, m, heads, dim = 600, 300000, 32, 64
    q = randn(n, heads, dim, g=g)
    k, v = (randn(m + 100, heads, dim, g=g) for _ in range(2))
    v[m - 1], v[m:] = float("nan"), float("inf")
    o, lse = A().attn_prompt(q, k, v, cu([n]), cu([m]))
    torch.cuda.synchronize()
    assert kernel_error() == 0
    assert bool(o[-1].isnan().all())
    for h in (0, heads - 1):
        rows = slice(0, n, 13)
        want, bound, z, bz = prompt_reference(q[:, h:h + 1], k[:m, h:h + 1], v[:m, h:h + 1].nan_to_num(), [n], [m], True,
                                              dim ** -0.5)
        within(o[:-1, h:h + 1][rows], want[:-1][rows], bound[:-1][rows], "o")
        within(lse[h:h + 1, :-1], z[:, :-1], bz[:, :-1], "lse")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv,lq,lk", [(64, 32, [700, 90], [700, 90]), (4, 2, [150], [2500]), (5, 1, [33], [33]),
                                            (16, 16, [1500], [1700])])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("plain", [False, True])
def test_prompt_infinities_that_rows_see(dim, heads, kv, lq, lk, causal, plain):
    """In tiles of keys without a masked place and with one, where a weight is large, small and 0 in
    f32; the other columns are as they are without."""
    g = gen(dim + sum(lk))
    n, m = sum(lq), sum(lk)
    q, k, v = randn(n, heads, dim, g=g, scale=6), randn(m, kv, dim, g=g), randn(m, kv, dim, g=g)
    if plain:
        v = torch.cat([v, v[..., :1]], -1)[..., :dim]  # rows that are not 16-byte aligned
    want = prompt_reference(q, k, v, lq, lk, causal, dim ** -0.5)
    marks = torch.zeros(3, m, dim, dtype=torch.bool, device="cuda")  # NaN, +inf, -inf by key and column
    for key, column, kind in ((3, 5, 1), (20, 5, 2), (7, 7, 2), (30, 9, 0), (m - 1, 0, 1), (m - 40 if m > 80 else 31, 33, 2),
                              (0, 63, 1), (m // 2, dim - 2, 1), (m // 2 + 1, dim - 2, 1)):
        marks[kind, key, column] = True
    for kind, value in enumerate((float("nan"), float("inf"), -float("inf"))):
        v[marks[kind][:, None].expand(-1, kv, -1)] = value
    o, lse = A().attn_prompt(q, k, v, cu(lq), cu(lk), causal=causal)
    assert kernel_error() == 0
    expect = want[0].clone()
    at = kat = 0
    for a, b in zip(lq, lk):
        seen = torch.arange(a, device="cuda") + 1 + b - a if causal else torch.full((a,), b, device="cuda")
        counts = torch.cat([torch.zeros(3, 1, dim, device="cuda"), marks[:, kat:kat + b].float().cumsum(1)], 1)
        some = counts[:, seen.clamp(0, b)] > 0
        x = torch.where(some[0] | (some[1] & some[2]), float("nan"),
                        torch.where(some[1], float("inf"), torch.where(some[2], -float("inf"), 0.0)))[:, None]
        expect[at:at + a] = torch.where(x == 0, expect[at:at + a], x.expand(-1, heads, -1).double())
        at, kat = at + a, kat + b
    odd = ~expect.isfinite()
    assert bool(odd.any()) and torch.equal(o.isfinite(), ~odd)
    assert bool(((o.double() == expect) | (o.isnan() & expect.isnan()))[odd].all())
    within(torch.where(odd, 0.0, o.double()), torch.where(odd, 0.0, expect), want[1], "o")
    within(lse, want[2], want[3], "lse")


@pytest.mark.parametrize("length", [2 ** 31 - 16, 2 ** 31 - 29])
def test_cache_attention_longest_sequence(length):
    """As many slots as a table of 16-slot pages can name, all of them in one page: the softmax of that
    page's 16 over again, lse the log of the pages more.  A warp of 2368 adds four weights a tile of
    32 to its sums, each addition 2^-23 of the sum off at most: 2^28 / 2368 * 2^-23 in all."""
    g = gen(31)
    pages, dim = 2 ** 27 - 1, 64
    cache = A().KV4Cache.empty(2, 1, dim, 16)
    k, v = randn(16, 1, dim, g=g), randn(16, 1, dim, g=g)
    slots = torch.arange(16, 32, dtype=torch.int32, device="cuda")
    A().kv4_append(cache, k, v, slots)
    table = torch.ones(1, pages, dtype=torch.int32, device="cuda")
    lens = torch.tensor([length], dtype=torch.int32, device="cuda")
    q = randn(1, 1, 2, dim, g=g)
    weight = torch.empty(1, 1, pages * 16, device="cuda")
    o, lse = A().kv4_attn(q, cache, table, lens, weight_out=weight)
    torch.cuda.synchronize()
    kd, vd = (values(*quantise(x), dtype=torch.float64)[:, 0] for x in (k, v))
    off = 2.0 ** 28 / 2368 * 2.0 ** -23
    total = torch.zeros(16, dtype=torch.float64, device="cuda")
    for h in range(2):
        s = kd @ q[0, 0, h].double() * dim ** -0.5
        p = torch.softmax(s, 0)
        total += p / pages
        assert bool(((o[0, 0, h].double() - p @ vd).abs() <= (2 * off + 2.0 ** -8) * (p @ vd.abs() + 1)).all())
        assert abs(float(lse[0, h, 0]) - float(torch.logsumexp(s, 0)) - math.log(pages)) <= 2 * off
    for at in (0, 2 ** 30, 2 ** 31 - 48):
        assert bool(((weight[0, 0, at:at + 16].double() / total - 1).abs() <= 4 * off).all())


def test_refusals_of_layouts_and_sizes():
    """What the C entry points answer with -1 is a ValueError here, and nothing has run."""
    attn = A()
    g = gen(40)
    cache = attn.KV4Cache.empty(4, 2, 128, 16)
    q = randn(3, 1, 4, 128, g=g)
    table = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    shifted = torch.empty(q.numel() + 4, dtype=torch.bfloat16, device="cuda")[4:].view(q.shape)
    flat = torch.zeros(3 * 2 * 32 + 8, device="cuda")
    near = (flat[:-8].view(3, 2, 32), flat[8:].view(3, 2, 32))
    for bad in (dict(out=shifted), dict(table=table[:, :0]), dict(weight=near[0], weight_out=near[1])):
        with pytest.raises(ValueError):
            attn.kv4_attn(**{**dict(q=q, cache=cache, table=table, lens=lens), **bad})
    many = 40000  # sequences times kv heads past a grid's second dimension
    with pytest.raises(ValueError):
        attn.kv4_attn(randn(many, 1, 2, 128, g=g), cache, table[:1].expand(many, -1).contiguous(), lens[:1].expand(many).contiguous())
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    rows = torch.empty(3 * 2 * 128 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(3, 2, 128)
    for bad in (dict(k_out=rows), dict(v_out=rows)):
        with pytest.raises(ValueError):
            attn.kv4_read(cache, slots, **bad)
    pos = torch.zeros(3, 2, 32, dtype=torch.int32, device="cuda")
    wo, po = torch.zeros(3, 2, 32, device="cuda"), torch.zeros_like(pos)
    for bad in (dict(budget=2 ** 31), dict(weight=near[0], weight_out=near[1])):
        with pytest.raises(ValueError):
            attn.kv4_evict(**{**dict(cache=cache, table=table, lens=lens, weight=near[0], pos=pos, seen=lens, budget=4,
                                     recent=0, weight_out=wo, pos_out=po), **bad})
    k = randn(3, 2, 128, g=g)
    with pytest.raises(ValueError):
        attn.attn_prompt(q[:, 0, :0], k, k, cu([3]))


def test_calls_without_a_sequence():
    attn = A()
    cache = attn.KV4Cache.empty(4, 2, 128, 16)
    none = dict(device="cuda")
    table = torch.zeros(0, 2, dtype=torch.int32, **none)
    lens = torch.zeros(0, dtype=torch.int32, **none)
    weight, pos = torch.zeros(0, 2, 32, **none), torch.zeros(0, 2, 32, dtype=torch.int32, **none)
    o, lse = attn.kv4_attn(torch.zeros(0, 1, 4, 128, dtype=torch.bfloat16, **none), cache, table, lens, weight_out=weight)
    assert o.shape == (0, 1, 4, 128) and lse.shape == (0, 4, 1)
    kept, new = attn.kv4_evict(cache, table, lens, weight, pos, lens, 7, weight_out=weight.clone(), pos_out=pos.clone())
    assert kept.shape == (0, 2, 7) and new.shape == (0,)
    rows = torch.zeros(0, 2, 128, dtype=torch.bfloat16, **none)
    attn.kv4_append(cache, rows, rows, lens)
    assert attn.kv4_read(cache, lens)[0].shape == (0, 2, 128)
