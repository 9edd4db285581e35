"""GPU tests of the serving attention operators (include/glint_attn.h, glint_b200/attn.py)
against plain implementations in 64 bits written here.

Bounds, per element, from the kernels' roundings:
  o (BF16): rounding of o and of each softmax weight to BF16, 2^-9 each, of sum p |v|
     (over the cache the rounded product is weight * step, |code - 8| <= 8, so its part is
     2^-9 * sum p * 8 step), an eighth more for the f32 arithmetic, and twice the score
     error as a relative error of every weight.
  scores: head_dim exact products summed in f32, any order, truncating adders:
     ds = head_dim * 2^-22 * scale * sum |q k|.
  lse: ds + 2^-20 (1 + |lse|).
  weights: (2 ds + 2^-18) of the added weight, and 2^-22 of the sum.
Codes, (step, lo), read values and everything of eviction: equal bit for bit.
"""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

NEG = -math.inf


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


def kernel_error():
    from glint_b200 import device
    return device.lib().glint_kernel_error(1)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, g, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).bfloat16()


def cu(lens):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")


# ---- attention over packed prompts -----------------------------------------------------

def prompt_reference(q, k, v, lq, lk, causal, scale, ol=None, zl=None):
    """o, lse and their bounds in f64; masked keys are left out, not multiplied by 0."""
    H, D, group = q.shape[1], q.shape[2], q.shape[1] // k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bo, z = torch.zeros_like(o), torch.full((H, q.shape[0]), NEG, dtype=torch.float64, device="cuda")
    bz = torch.zeros_like(z)
    at = kat = 0
    for n, m in zip(lq, lk):
        for h in range(H):
            qh = q[at:at + n, h].double()
            kh, vh = k[kat:kat + m, h // group].double(), v[kat:kat + m, h // group].double()
            hide = torch.zeros(n, m, dtype=torch.bool, device="cuda")
            if causal:
                hide = torch.arange(m, device="cuda")[None] > torch.arange(n, device="cuda")[:, None] + m - n
            s = (qh @ kh.T * scale).masked_fill(hide, NEG)
            some = ~hide.all(1) if m else torch.zeros(n, dtype=torch.bool, device="cuda")
            if not bool(some.any()):
                continue
            zz = torch.logsumexp(s, 1)
            p = torch.where(hide, 0.0, torch.exp(s - zz[:, None]))
            ds = D * 2.0 ** -22 * abs(scale) * torch.where(hide, 0.0, qh.abs() @ kh.abs().T)
            ds = ds.amax(1, keepdim=True)
            o[at:at + n, h] = torch.where(some[:, None], p @ vh, 0.0)
            bo[at:at + n, h] = torch.where(some[:, None], (2.0 ** -8 * 1.125 + 2 * ds) * (p @ vh.abs()), 0.0)
            z[h, at:at + n] = torch.where(some, zz, NEG)
            bz[h, at:at + n] = torch.where(some, ds[:, 0] + 2.0 ** -20 * (1 + zz.abs()), 0.0)
        at, kat = at + n, kat + m
    return o, bo, z, bz


def within(got, want, bound, what):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= bound)
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} off, " \
        f"worst {float(((got - want).abs() / bound.clamp_min(1e-30))[~same].max()):.3g} of its bound"


def check_prompt(q, k, v, lq, lk, causal=True, scale=None):
    o, lse = A().attn_prompt(q, k, v, cu(lq), None if lq == lk else cu(lk), causal=causal, scale=scale)
    torch.cuda.synchronize()
    assert kernel_error() == 0
    want = prompt_reference(q, k, v, lq, lk, causal, q.shape[2] ** -0.5 if scale is None else scale)
    n = sum(lq)
    within(o[:n], want[0][:n], want[1][:n], "o")
    within(lse[:, :n], want[2][:, :n], want[3][:, :n], "lse")
    again = A().attn_prompt(q, k, v, cu(lq), None if lq == lk else cu(lk), causal=causal, scale=scale)
    assert torch.equal(o[:n].view(torch.int16), again[0][:n].view(torch.int16)), "not the same bits twice"


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(8, 2), (4, 4), (5, 1)])
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [127, 128, 129], [17, 0, 300, 0, 255, 256, 257], [0], [641]])
def test_prompt_packed(dim, heads, kv, lens):
    g = gen(sum(lens) + dim)
    T = sum(lens)
    y = randn(T, heads + 2 * kv, dim, g=g)  # views of one fused output
    check_prompt(y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], lens, lens)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk", [([5, 130], [700, 131]), ([1, 1, 1], [1, 255, 513]), ([200], [333]),
                                   ([300, 20], [100, 0]), ([140], [139])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_other_keys(dim, lq, lk, causal):
    """Keys before the queries, fewer keys than queries (rows that see nothing), none."""
    g = gen(len(lq) + dim)
    check_prompt(randn(sum(lq), 4, dim, g=g), randn(sum(lk), 2, dim, g=g), randn(sum(lk), 2, dim, g=g), lq, lk, causal)


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_large_scores(dim):
    """Scores whose running maximum keeps growing, far past what f32 exponentials hold."""
    g = gen(dim)
    T = 700
    k = randn(T, 2, dim, g=g) * torch.linspace(0.1, 30, T, device="cuda")[:, None, None].bfloat16()
    check_prompt(randn(T, 4, dim, g=g, scale=4), k, randn(T, 2, dim, g=g), [T], [T])
    check_prompt(randn(T, 4, dim, g=g, scale=4), k.flip(0).contiguous(), randn(T, 2, dim, g=g), [300, 400], [300, 400],
                 scale=-0.25)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.3e38])
def test_prompt_masked_values_stay_out(dim, bad):
    """Keys and values that a row does not see (later tokens, the next sequence, rows past
    the last sequence) may hold anything; rows that see them are not compared."""
    g = gen(dim)
    lens = [70, 130, 300]
    T = sum(lens) + 40
    q, k, v = randn(T, 4, dim, g=g), randn(T, 2, dim, g=g), randn(T, 2, dim, g=g)
    n = sum(lens)
    want = prompt_reference(q[:n], k[:n], v[:n], lens, lens, True, dim ** -0.5)
    ends = cu(lens)
    for first in (69, 70 + 60, 70 + 130 + 211):  # poisoned from here to its sequence's end
        end = 70 if first < 70 else 200 if first < 200 else n
        k2, v2 = k.clone(), v.clone()
        for x in (k2, v2):
            x[first:end] = bad
            x[n:] = bad
        o, lse = A().attn_prompt(q, k2, v2, ends)
        rows = torch.ones(n, dtype=torch.bool, device="cuda")
        rows[first:end] = False
        within(o[:n][rows], want[0][rows], want[1][rows], "o")
        within(lse[:, :n][:, rows], want[2][:, rows], want[3][:, rows], "lse")
        if bad != bad:
            assert bool(o[first:end].isnan().all())


def test_prompt_unaligned_and_strided():
    g = gen(3)
    lens, heads, kv, dim = [90, 33], 4, 2, 64
    T = sum(lens)
    flat = randn(T * (heads + 2 * kv) * (dim + 3) + 1, g=g)[1:].view(T, heads + 2 * kv, dim + 3)[..., 2:2 + dim]
    check_prompt(flat[:, :heads], flat[:, heads:heads + kv], flat[:, heads + kv:], lens, lens)
    by_head = randn(heads + 2 * kv, T, dim, g=g).transpose(0, 1)  # [heads, tokens, dim] storage
    check_prompt(by_head[:, :heads], by_head[:, heads:heads + kv], by_head[:, heads + kv:], lens, lens)
    out = torch.full((T, heads, dim + 5), 7.0, dtype=torch.bfloat16, device="cuda")
    q, k, v = by_head[:, :heads], by_head[:, heads:heads + kv], by_head[:, heads + kv:]
    A().attn_prompt(q, k, v, cu(lens), out=out[..., 1:1 + dim])
    assert torch.equal(out[..., 1:1 + dim], A().attn_prompt(q, k, v, cu(lens))[0])
    assert bool((out[..., 0] == 7).all()) and bool((out[..., 1 + dim:] == 7).all())


def test_prompt_tokens_outside_sequences_are_not_written():
    g = gen(4)
    q, k, v = (randn(50, h, 128, g=g) for h in (4, 2, 2))
    out = torch.full_like(q, 7.0)
    lse = torch.full((4, 50), 7.0, device="cuda")
    ends = torch.tensor([5, 20, 33], dtype=torch.int32, device="cuda")
    A().attn_prompt(q, k, v, ends, out=out, lse=lse)
    want = prompt_reference(q[5:33], k[5:33], v[5:33], [15, 13], [15, 13], True, 128 ** -0.5)
    within(out[5:33], want[0], want[1], "o")
    assert bool((out[:5] == 7).all()) and bool((out[33:] == 7).all())
    assert bool((lse[:, :5] == 7).all()) and bool((lse[:, 33:] == 7).all())


def test_prompt_past_32_bits():
    """Rows of q, k, v and o more than 2^32 elements apart."""
    g = gen(17)
    step, T = 2 ** 26, 70
    flat = torch.empty(step * T, dtype=torch.bfloat16, device="cuda")
    y = flat.view(T, step)[:, :8 * 128].view(T, 8, 128)
    y.copy_(randn(T, 8, 128, g=g))
    out = flat.view(T, step)[:, 2048:2048 + 4 * 128].view(T, 4, 128)
    A().attn_prompt(y[:, :4], y[:, 4:6], y[:, 6:], cu([T]), out=out)
    want = prompt_reference(y[:, :4], y[:, 4:6], y[:, 6:], [T], [T], True, 128 ** -0.5)
    within(out, want[0], want[1], "o")


def test_prompt_many_sequences():
    """More sequences than a block keeps the sizes of."""
    g = gen(18)
    lens = [1 + i % 5 for i in range(1500)] + [70]
    T = sum(lens)
    check_prompt(randn(T, 2, 64, g=g), randn(T, 1, 64, g=g), randn(T, 1, 64, g=g), lens, lens)


def test_prompt_other_stream_and_graph():
    g = gen(5)
    q, k, v = randn(200, 8, 128, g=g), randn(200, 2, 128, g=g), randn(200, 2, 128, g=g)
    ends = cu([150, 50])
    want = A().attn_prompt(q, k, v, ends)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = A().attn_prompt(q, k, v, ends, stream=side)[0]
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A().attn_prompt(q, k, v, ends)[0]
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---- the 4-bit cache ---------------------------------------------------------------------

def quantise(x):
    """BF16 [..., dim] -> codes [..., dim], step and lo [..., dim / 64] f32, by the header's rule."""
    x = x.float().unflatten(-1, (-1, 64))
    bad = ~x.isfinite().all(-1)
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) / 15).bfloat16().float()
    bad |= ~step.isfinite()
    code = torch.where((step > 0)[..., None], torch.round((x - lo[..., None]) / step[..., None]).clamp(0, 15), 0.0)
    code = torch.where(bad[..., None], 0.0, code).flatten(-2)
    return code, torch.where(bad, 0.0, step), torch.where(bad, float("nan"), lo)


def values(code, step, lo, dtype=torch.float32):
    c = code.to(dtype).unflatten(-1, (-1, 64))
    return (lo.to(dtype)[..., None] + step.to(dtype)[..., None] * c).flatten(-2)


def pack(code, slot):
    c = code.to(torch.uint8)
    rows = c[..., 0::2] | (c[..., 1::2] << 4)
    if rows.shape[-1] == 64:
        rows = torch.where((slot & 2).bool()[..., None], rows.roll(32, -1), rows)
    return rows


def bits(t):
    return t.contiguous().view(torch.int16) if t.dtype == torch.bfloat16 else t


def same_values(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,tokens", [(1, 1), (8, 3), (3, 301)])
def test_append_and_read(dim, page, kv, tokens):
    g = gen(tokens + page)
    pages = -(-tokens // page) + 3
    y = randn(tokens, 2 * kv, dim, g=g, scale=3)
    y[::5, 0, 7] = 90.0
    y[::7, -1] = 0.625            # a constant block: step 0
    y[::11, kv, 3] = 0.0
    k, v = y[:, :kv], y[:, kv:]
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:tokens].to(torch.int32)
    cache = A().KV4Cache.empty(pages, kv, dim, page)
    for t in (cache.k_code, cache.v_code):
        t.fill_(0xA5)
    A().kv4_append(cache, k, v, slots)
    p, r = slots.long() // page, slots.long() % page
    got = A().kv4_read(cache, slots)
    for x, codes, metas, back in ((k, cache.k_code, cache.k_meta, got[0]), (v, cache.v_code, cache.v_meta, got[1])):
        code, step, lo = quantise(x)
        assert torch.equal(codes[p, :, r], pack(code, r[:, None]))
        assert torch.equal(bits(metas[p, :, r]), bits(torch.stack([step, lo], -1).bfloat16()))
        assert torch.equal(bits(back), bits(values(code, step, lo).bfloat16()))
        # half a step, and what the top code loses where the BF16 step is below a fifteenth of the range
        near = (x.double() - values(code, step, lo, torch.float64)).abs()
        assert bool((near <= (0.5 + 15 * 2.0 ** -8) * step.double().repeat_interleave(64, -1) + 1e-30).all())
    left = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    left[p, r] = False
    assert bool((cache.k_code.transpose(1, 2)[left] == 0xA5).all()), "other slots were written"


@pytest.mark.parametrize("dim", [64, 128])
def test_append_odd_values(dim):
    """NaN, infinities, an overflowing range, subnormals, signed zeros."""
    g = gen(dim)
    x = randn(12, 1, dim, g=g)
    x[0, 0, 5], x[1, 0, 63], x[2, 0, 0] = float("nan"), float("inf"), -float("inf")
    x[3, 0, :2] = torch.tensor([3e38, -3e38])
    x[4] *= 1e-39
    x[5] = torch.where(x[5] > 0, 0.0, -0.0)
    x[6, 0, 1:] = 0
    x[7] *= 2.0 ** 100
    x[8] *= 1e-36
    x[9, 0] = torch.arange(dim, device="cuda") % 16  # every code once, exact
    x[10, 0] = (torch.arange(dim, device="cuda") % 31) * 0.5  # ties between codes
    cache = A().KV4Cache.empty(1, 1, dim, 16)
    slots = torch.arange(12, dtype=torch.int32, device="cuda")
    A().kv4_append(cache, x, x, slots)
    code, step, lo = quantise(x)
    for got in A().kv4_read(cache, slots):
        assert same_values(got, values(code, step, lo).bfloat16())
    assert torch.equal(cache.k_code[0, :, :12].transpose(0, 1), pack(code, slots[:, None]))
    assert torch.equal(cache.v_code[0, :, :12], cache.k_code[0, :, :12])


def test_append_skips_slots_outside():
    g = gen(9)
    cache = A().KV4Cache.empty(2, 2, 128, 16)
    for t in (cache.k_code, cache.v_code, cache.k_meta, cache.v_meta):
        t.zero_()
    x = randn(5, 2, 128, g=g)
    slots = torch.tensor([-1, 32, 31, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    A().kv4_append(cache, x, x, slots)
    assert int((cache.k_code.sum(-1) != 0).sum()) == 2 and bool(cache.k_code[1, :, 15].any())
    k, v = A().kv4_read(cache, slots)
    assert not bool(k[[0, 1, 3, 4]].any()) and bool(k[2].any()) and torch.equal(k, v)


@pytest.mark.parametrize("shift", [1, 8])
def test_append_strides(shift):
    """Rows at any alignment, and by head."""
    g = gen(shift)
    flat = randn(40 * 4 * 136 + shift, g=g)[shift:].view(40, 4, 136)[..., :128]
    k, v = flat[:, :2], flat[:, 2:]
    caches = [A().KV4Cache.empty(3, 2, 128, 16) for _ in range(2)]
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    A().kv4_append(caches[0], k, v, slots)
    A().kv4_append(caches[1], k.contiguous(), v.transpose(0, 1).contiguous().transpose(0, 1), slots)
    for a, b in zip(A().kv4_read(caches[0], slots), A().kv4_read(caches[1], slots)):
        assert torch.equal(bits(a), bits(b))


# ---- attention over the cache ------------------------------------------------------------

def filled(lens, kv, dim, page, g, spare=2, outside=float("nan")):
    """A cache with a shuffled page table; every slot no sequence owns reads as `outside`."""
    used = [-(-n // page) for n in lens]
    pages = sum(used) + spare
    cache = A().KV4Cache.empty(pages, kv, dim, page)
    for t in (cache.k_code, cache.v_code):
        t.fill_(0x7B)
    for t in (cache.k_meta, cache.v_meta):
        t.fill_(outside)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(len(lens)))
    table = torch.full((len(lens), max(used + [1]) + 1), pages + 5, dtype=torch.int32)
    at = 0
    rows = []
    for b, (n, u) in enumerate(zip(lens, used)):
        table[b, :u] = order[at:at + u].to(torch.int32)
        at += u
        t = torch.arange(n)
        rows.append((order[at - u:at][t // page] * page + t % page) if n else t)
    slots = torch.cat(rows).to(torch.int32).cuda()
    k, v = randn(len(slots), kv, dim, g=g), randn(len(slots), kv, dim, g=g)
    k[..., 3::29] *= 4
    v[..., 1::7] += 1
    A().kv4_append(cache, k, v, slots)
    kd, vd = (values(*quantise(x), dtype=torch.float64) for x in (k, v))
    steps = quantise(v)[1].double().repeat_interleave(64, -1)
    return cache, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), kd, vd, steps


def attn_reference(q, lens, kd, vd, steps, scale, skip=None):
    """o, lse, added weights and their bounds; skip[b]: slots masked by a page outside the cache."""
    B, R, H, D = q.shape
    kv = kd.shape[1]
    group = H // kv
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    bo = torch.zeros_like(o)
    z = torch.full((B, H, R), NEG, dtype=torch.float64, device="cuda")
    bz = torch.zeros_like(z)
    ws = []
    at = 0
    for b, n in enumerate(lens):
        w, bw = torch.zeros(2, kv, n, dtype=torch.float64, device="cuda")
        for h in range(H):
            k, v, st = kd[at:at + n, h // group], vd[at:at + n, h // group], steps[at:at + n, h // group]
            for r in range(R):
                see = torch.arange(n, device="cuda") < n - R + r + 1
                if skip is not None:
                    see &= ~skip[b][:n]
                if not bool(see.any()):
                    continue
                s = k[see] @ q[b, r, h].double() * scale
                zz = torch.logsumexp(s, 0)
                p = torch.exp(s - zz)
                ds = D * 2.0 ** -22 * abs(scale) * (k[see].abs() @ q[b, r, h].double().abs()).max()
                o[b, r, h] = p @ v[see]
                bo[b, r, h] = 1.125 * 2.0 ** -9 * (o[b, r, h].abs() + p @ (8 * st[see])) + 2 * ds * (p @ v[see].abs())
                z[b, h, r], bz[b, h, r] = zz, ds + 2.0 ** -20 * (1 + zz.abs())
                w[h // group][see] += p
                bw[h // group][see] += (2 * ds + 2.0 ** -18) * p
        ws.append((w, bw))
        at += n
    return o, bo, z, bz, ws


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv,rows", [(4, 1, 1), (8, 2, 1), (3, 3, 1), (5, 1, 2), (16, 2, 4), (32, 1, 2)])
def test_cache_attention(dim, page, heads, kv, rows):
    g = gen(dim + page + rows)
    lens = [1, 0, 2, 63, 64, 65, 129, 700, 16, 33]
    cache, table, dl, kd, vd, steps = filled(lens, kv, dim, page, g)
    wide = table.shape[1] * page + 3
    q = randn(len(lens), rows, heads + 1, dim, g=g)[:, :, 1:]  # a strided view
    old = torch.rand(len(lens), kv, wide, device="cuda", generator=g)
    new = torch.full_like(old, 7.0)
    o, lse = A().kv4_attn(q, cache, table, dl, weight=old, weight_out=new)
    assert kernel_error() == 0
    want = attn_reference(q, lens, kd, vd, steps, dim ** -0.5)
    within(o, want[0], want[1], "o")
    within(lse, want[2], want[3], "lse")
    for b, n in enumerate(lens):
        base = old[b, :, :n].double()
        base[:, max(0, n - rows):] = 0
        w, bw = want[4][b]
        within(new[b, :, :n], base + w, bw + 2.0 ** -22 * (base + w), f"weights of sequence {b}")
        assert bool((new[b, :, n:] == 7).all())
    # without weights, and in place: the same bits; and twice the same bits
    o2, lse2 = A().kv4_attn(q, cache, table, dl)
    inplace = old.clone()
    A().kv4_attn(q, cache, table, dl, weight=inplace, weight_out=inplace)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for b, n in enumerate(lens):
        assert torch.equal(inplace[b, :, :n], new[b, :, :n])


@pytest.mark.parametrize("dim,lens,heads,kv,rows", [(128, [9001], 8, 1, 1), (128, [5000, 1, 2500], 4, 2, 3),
                                                    (64, [20000, 333], 2, 1, 1), (128, [3000] * 3, 40, 1, 1)])
def test_cache_attention_long(dim, lens, heads, kv, rows):
    """Long sequences: the slots of one are shared out and joined."""
    g = gen(dim + len(lens))
    cache, table, dl, kd, vd, steps = filled(lens, kv, dim, 64, g)
    q = randn(len(lens), rows, heads, dim, g=g, scale=2)
    o, lse = A().kv4_attn(q, cache, table, dl)
    want = attn_reference(q, lens, kd, vd, steps, dim ** -0.5)
    within(o, want[0], want[1], "o")
    within(lse, want[2], want[3], "lse")
    for _ in range(3):
        again = A().kv4_attn(q, cache, table, dl)
        assert torch.equal(o, again[0]) and torch.equal(lse, again[1]), "not the same bits twice"


@pytest.mark.parametrize("dim", [64, 128])
def test_cache_attention_scores_keep_f32(dim):
    """lse of one slot is its scaled score.  The products take codes with 16 added, so a 64-block's
    sum is about 24 * sqrt(64) = 192 for unit q; each of its four steps may drop 2^-23 of that,
    evenly spread: 2^-23 * 192 / sqrt(3) * 2 = 2^-23 * 222, times a step of 4.7 / 15 for 64 unit
    normals, over a score of sqrt(64): 8.7 * 2^-23 of the scores in the mean square (two
    blocks: sqrt(2) in both)."""
    g = gen(dim + 5)
    seqs, kv, heads = 256, 2, 8
    cache = A().KV4Cache.empty(seqs, kv, dim, 16)
    k, v = randn(seqs, kv, dim, g=g), randn(seqs, kv, dim, g=g)
    A().kv4_append(cache, k, v, torch.arange(seqs, dtype=torch.int32, device="cuda") * 16)
    table = torch.arange(seqs, dtype=torch.int32, device="cuda")[:, None]
    q = randn(seqs, 1, heads, dim, g=g)
    _, lse = A().kv4_attn(q, cache, table, torch.ones(seqs, dtype=torch.int32, device="cuda"))
    kd = values(*quantise(k), dtype=torch.float64).repeat_interleave(heads // kv, 1)
    want = (q[:, 0].double() * kd).sum(-1) * dim ** -0.5
    error = float((lse[..., 0].double() - want).norm() / want.norm())
    assert error <= 8.7 * 2.0 ** -23, f"scores are {error} off"


@pytest.mark.parametrize("dim", [64, 128])
def test_cache_attention_large_scores(dim):
    g = gen(dim)
    lens = [515, 130]
    cache, table, dl, kd, vd, steps = filled(lens, 2, dim, 32, g)
    q = randn(2, 2, 8, dim, g=g, scale=40)
    for scale in (None, 1.0, -1.0):
        o, lse = A().kv4_attn(q, cache, table, dl, scale=scale)
        want = attn_reference(q, lens, kd, vd, steps, dim ** -0.5 if scale is None else scale)
        within(o, want[0], want[1], "o")
        within(lse, want[2], want[3], "lse")


def test_cache_attention_pages_outside_are_masked():
    g = gen(12)
    lens = [200, 64]
    cache, table, dl, kd, vd, steps = filled(lens, 2, 128, 32, g)
    table[0, 2], table[0, 5], table[1, :] = -1, cache.pages, -7
    skip = torch.zeros(2, 256, dtype=torch.bool, device="cuda")
    skip[0, 64:96] = skip[0, 160:192] = True
    skip[1] = True
    q = randn(2, 1, 4, 128, g=g)
    old = torch.rand(2, 2, table.shape[1] * 32, device="cuda", generator=g)
    new = torch.empty_like(old)
    o, lse = A().kv4_attn(q, cache, table, dl, weight=old, weight_out=new)
    want = attn_reference(q, lens, kd, vd, steps, 128 ** -0.5, skip)
    within(o, want[0], want[1], "o")
    within(lse, want[2], want[3], "lse")
    assert not bool(o[1].any()) and bool((lse[1] == NEG).all())
    assert torch.equal(new[0, :, 64:96], old[0, :, 64:96])


def test_cache_attention_hidden_rows_stay_out():
    """A drafted token's row that holds NaN reaches its own and later rows, no earlier one."""
    g = gen(13)
    lens, rows = [100], 4
    cache, table, dl, kd, vd, steps = filled(lens, 1, 128, 16, g)
    q = randn(1, rows, 4, 128, g=g)
    want = attn_reference(q, lens, kd, vd, steps, 128 ** -0.5)
    bad = torch.full((1, 1, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    A().kv4_append(cache, bad, bad, table[0, 98 // 16:98 // 16 + 1] * 16 + 98 % 16)
    o, lse = A().kv4_attn(q, cache, table, dl)
    within(o[:, :2], want[0][:, :2], want[1][:, :2], "o")
    assert bool(o[:, 2:].isnan().all())
    within(lse[..., :2], want[2][..., :2], want[3][..., :2], "lse")


def test_cache_attention_lens_past_the_table_are_cut():
    g = gen(14)
    cache, table, dl, *_ = filled([64, 64], 2, 64, 32, g)
    table = table[:, :2].contiguous()
    q = randn(2, 1, 4, 64, g=g)
    want = A().kv4_attn(q, cache, table, dl)
    got = A().kv4_attn(q, cache, table, torch.tensor([2 ** 31 - 1, 65], dtype=torch.int32, device="cuda"))
    assert torch.equal(want[0], got[0])
    got = A().kv4_attn(q, cache, table, torch.tensor([-5, -2 ** 31], dtype=torch.int32, device="cuda"))
    assert not bool(got[0].any()) and bool((got[1] == NEG).all())


def test_cache_attention_other_stream_and_graph():
    g = gen(15)
    lens = [900, 31]
    cache, table, dl, *_ = filled(lens, 2, 128, 64, g)
    q = randn(2, 1, 8, 128, g=g)
    old = torch.rand(2, 2, table.shape[1] * 64, device="cuda", generator=g)
    w0, w1, w2 = (torch.zeros_like(old) for _ in range(3))
    want = A().kv4_attn(q, cache, table, dl, weight=old, weight_out=w0)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = A().kv4_attn(q, cache, table, dl, weight=old, weight_out=w1, stream=side)[0]
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(w0, w1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = A().kv4_attn(q, cache, table, dl, weight=old, weight_out=w2)[0]
    for _ in range(2):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(w0, w2)


def test_cache_past_32_bits():
    """Pages whose bytes lie past 4 GiB of a cache's codes: append, read, attention, eviction."""
    g = gen(16)
    kv, dim, page, n = 8, 128, 64, 150
    pages = (2 ** 32 + 2 ** 24) // (kv * page * dim // 2)
    cache = A().KV4Cache.empty(pages, kv, dim, page)
    table = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device="cuda")
    t = torch.arange(n, device="cuda")
    slots = (table[0, t // page] * page + t % page).int()
    k, v = randn(n, kv, dim, g=g), randn(n, kv, dim, g=g)
    A().kv4_append(cache, k, v, slots)
    for x, got in zip((k, v), A().kv4_read(cache, slots)):
        assert torch.equal(bits(got), bits(values(*quantise(x)).bfloat16()))
    kd, vd = (values(*quantise(x), dtype=torch.float64) for x in (k, v))
    q = randn(1, 1, 16, dim, g=g)
    o, lse = A().kv4_attn(q, cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    want = attn_reference(q, [n], kd, vd, quantise(v)[1].double().repeat_interleave(64, -1), dim ** -0.5)
    within(o, want[0], want[1], "o")
    within(lse, want[2], want[3], "lse")
    w = torch.arange(3 * page, device="cuda").float().expand(1, kv, -1).contiguous()
    pos = torch.zeros_like(w, dtype=torch.int32)
    one = torch.tensor([n], dtype=torch.int32, device="cuda")
    kept, _ = A().kv4_evict(cache, table, one, w, pos, one, 20, weight_out=torch.empty_like(w),
                            pos_out=torch.empty_like(pos))
    assert kept[0, 0].tolist() == list(range(130, 150))
    assert torch.equal(bits(A().kv4_read(cache, slots[:20])[0]), bits(values(*quantise(k[130:])).bfloat16()))


# ---- eviction ------------------------------------------------------------------------------

def evict_reference(w, pos, seen, L, budget, recent):
    """Source slot of each kept one, plain Python."""
    n = min(L, budget)
    def key(t):
        return (0, 0.0, t) if pos[t] >= seen - recent else (2, 0.0, t) if w[t] != w[t] else (1, -w[t], t)
    order = sorted(range(L), key=key)
    keep = set(order[:n])
    far = [t for t in range(n, L) if t in keep]
    return [t if t in keep else far.pop(0) for t in range(n)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (40, 8), (129, 129), (1000, 0), (5000, 100)])
def test_evict(dim, page, budget, recent):
    g = gen(budget + page)
    lens, kv = [0, 1, 39, 41, 130, 1001, 3000, 128], 2
    cache, table, dl, *_ = filled(lens, kv, dim, page, g)
    wide = table.shape[1] * page + 1
    w = torch.rand(len(lens), kv, wide, device="cuda", generator=g)
    w = torch.where(w < 0.5, 0.0, w.mul(64).round() / 64)  # many ties
    w[:, 0, 20:24] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0], device="cuda")
    pos = torch.rand(len(lens), kv, wide, device="cuda", generator=g).argsort(-1).to(torch.int32)
    seen = torch.full((len(lens),), wide, dtype=torch.int32, device="cuda")
    slots = [(table[b, torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page).int()
             for b, n in enumerate(lens)]
    before = [A().kv4_read(cache, s) for s in slots]
    wo, po = torch.full_like(w, 7.0), torch.full_like(pos, 7)
    kept, new = A().kv4_evict(cache, table, dl, w, pos, seen, budget, recent, weight_out=wo, pos_out=po)
    torch.cuda.synchronize()
    after = [A().kv4_read(cache, s) for s in slots]
    assert new.tolist() == [min(n, budget) for n in lens]
    for b, L in enumerate(lens):
        n = min(L, budget)
        for h in range(kv):
            # -0 and 0 tie, so the sign is dropped before sorting
            want = evict_reference((w[b, h] + 0.0).tolist(), pos[b, h].tolist(), wide, L, budget, recent)
            assert kept[b, h].tolist() == want + [-1] * (budget - n), (b, h)
            src = torch.tensor(want, dtype=torch.long, device="cuda")
            assert torch.equal(wo[b, h, :n].view(torch.int32), w[b, h][src].view(torch.int32))
            assert torch.equal(po[b, h, :n], pos[b, h][src])
            for x, y in zip(before[b], after[b]):
                assert same_values(y[:n, h], x[src, h]), "rows are not where `kept` says"
                assert same_values(y[n:, h], x[n:, h]), "rows past the budget were written"
        assert bool((wo[b, :, n:] == 7).all()) and bool((po[b, :, n:] == 7).all())


def test_evict_all_protected_and_equal():
    g = gen(21)
    cache, table, dl, *_ = filled([500], 1, 64, 16, g)
    w = torch.zeros(1, 1, table.shape[1] * 16, device="cuda")
    pos = torch.arange(w.shape[2], dtype=torch.int32, device="cuda").expand(1, 1, -1).contiguous()
    wo, po = torch.empty_like(w), torch.empty_like(pos)
    seen = torch.tensor([500], dtype=torch.int32, device="cuda")
    kept, _ = A().kv4_evict(cache, table, dl, w, pos, seen, 100, 30, weight_out=wo, pos_out=po)
    assert kept[0, 0].tolist() == list(range(70)) + list(range(470, 500))
    seen.fill_(-2 ** 31)  # everything protected: the lowest slots
    kept, _ = A().kv4_evict(cache, table, dl, w, pos, seen, 100, 30, weight_out=wo, pos_out=po)
    assert kept[0, 0].tolist() == list(range(100))


@pytest.mark.parametrize("length", [40000, 200001])
def test_evict_long(length):
    """More slots than a block's shared memory holds keys."""
    g = gen(length)
    cache, table, dl, *_ = filled([length], 1, 64, 128, g)
    w = torch.rand(1, 1, table.shape[1] * 128, device="cuda", generator=g)
    pos = torch.zeros_like(w, dtype=torch.int32)
    wo, po = torch.empty_like(w), torch.empty_like(pos)
    seen = torch.tensor([10], dtype=torch.int32, device="cuda")
    kept, _ = A().kv4_evict(cache, table, dl, w, pos, seen, 1777, 0, weight_out=wo, pos_out=po)
    keep = w[0, 0, :length].sort(descending=True, stable=True).indices[:1777].sort().values
    low, far = keep[keep < 1777], keep[keep >= 1777]
    want = torch.arange(1777, device="cuda")
    free = torch.ones(1777, dtype=torch.bool, device="cuda")
    free[low] = False
    want[free] = far
    assert torch.equal(kept[0, 0].long(), want)


# ---- refusals --------------------------------------------------------------------------------

def test_refusals():
    attn = A()
    g = gen(30)
    q, k = randn(4, 4, 128, g=g), randn(4, 2, 128, g=g)
    ends = cu([4])
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[0]), dict(k=k[:, :, :64]), dict(v=k[:3]),
                dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(q=randn(4, 3, 128, g=g)),
                dict(cu_q=ends.long()), dict(cu_q=ends[:0]), dict(cu_k=cu([2, 2])), dict(q=q[:3]),
                dict(out=q.float()), dict(lse=torch.empty(4, 5, device="cuda")), dict(q=randn(4, 4, 96, g=g))):
        with pytest.raises(ValueError):
            attn.attn_prompt(**{**dict(q=q, k=k, v=k, cu_q=ends), **bad})
    empty = attn.attn_prompt(q[:0], k[:0], k[:0], cu([]))
    assert empty[0].shape == (0, 4, 128) and empty[1].shape == (4, 0)
    with pytest.raises(ValueError):
        attn.KV4Cache.empty(2, 2, 96)
    with pytest.raises(ValueError):
        attn.KV4Cache.empty(2, 2, 128, page_size=48)
    cache = attn.KV4Cache.empty(4, 2, 128, 16)
    with pytest.raises(ValueError):
        attn.KV4Cache(cache.k_code, cache.k_meta[:2], cache.v_code, cache.v_meta)
    slots = torch.arange(4, dtype=torch.int32, device="cuda")
    for bad in (dict(k=k.half()), dict(slots=slots.long()), dict(slots=slots[:3]), dict(v=k[:2]), dict(k=q, v=q)):
        with pytest.raises(ValueError):
            attn.kv4_append(cache, **{**dict(k=k, v=k, slots=slots), **bad})
    q4 = q[:, None]
    table = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(4, dtype=torch.int32, device="cuda")
    w = torch.zeros(4, 2, 16, device="cuda")
    for bad in (dict(q=q), dict(q=randn(4, 1, 3, 128, g=g)), dict(table=table.long()), dict(lens=lens[:2]),
                dict(weight=w), dict(weight_out=w[:, :, :8].contiguous()), dict(weight_out=w, weight=w[:, :1]),
                dict(q=randn(4, 129, 4, 128, g=g)), dict(out=q)):
        with pytest.raises(ValueError):
            attn.kv4_attn(**{**dict(q=q4, cache=cache, table=table, lens=lens), **bad})
    pos = torch.zeros(4, 2, 16, dtype=torch.int32, device="cuda")
    wo, po = w.clone(), pos.clone()
    for bad in (dict(budget=0), dict(recent=5), dict(recent=-1), dict(weight_out=w), dict(pos_out=pos),
                dict(pos=pos.long()), dict(weight=w[:, :, :15].contiguous()), dict(seen=lens[:1])):
        with pytest.raises(ValueError):
            attn.kv4_evict(**{**dict(cache=cache, table=table, lens=lens, weight=w, pos=pos, seen=lens, budget=4,
                                     recent=0, weight_out=wo, pos_out=po), **bad})
