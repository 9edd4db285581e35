"""Cases of the serving attention operators: attention over packed prompts, the paged
4-bit key/value cache (append, read), attention over that cache, and eviction from it.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the
framework's kernels; both take what prepare() gives.  The plain form is also the
written definition of each operator:

prompt  query i of a sequence (Lq queries, Lk >= Lq keys) sees the keys
        j <= i + Lk - Lq; o = softmax(scale q k^T) v, lse = log sum exp.
cache   blocks of 64 values of one head vector: lo = min, step = BF16((max - min) / 15),
        code = rint((x - lo) / step) in 0..15, value lo + step * code.  Pages of
        `page` slots per head: codes [pages, kv, page, dim / 2] (element 2i in the low
        nibble; at dim 128 the two 32-byte halves of a row are swapped where slot & 2),
        (step, lo) [pages, kv, page, dim / 64, 2] BF16.
decode  the last `rows` tokens of each sequence attend to its cached slots, causally;
        optionally each slot's weight, summed over the query heads and rows of its
        key/value head, is added to a running sum (newest slots start from zero).
evict   per sequence and head keep n = min(len, budget) slots: those with
        pos >= seen - recent, then the largest weights, ties to the lowest slot; kept
        slots >= n move into the freed slots < n, in order.
"""
import math
import random

import torch

own = False

BLOCK = 64


# ---- cases ---------------------------------------------------------------------------

def listed():
    return [
        # one short question, alone: launch latency is all there is
        dict(name="prompt 17", op="prompt", seqs=1, longest=17, past=0, heads=32, kv=8, dim=128),
        # a serving step's prompts packed together, most short, a few long (8B-shaped heads)
        dict(name="prompt packed", op="prompt", seqs=12, longest=2011, past=0, heads=32, kv=8, dim=128),
        # the next chunk of a long document after the earlier ones, small heads
        dict(name="prompt chunk", op="prompt", seqs=1, longest=512, past=7777, heads=16, kv=4, dim=64),
        # one whole long document
        dict(name="prompt 16384", op="prompt", seqs=1, longest=16384, past=0, heads=32, kv=8, dim=128),
        # one decoded token for each of eight sequences
        dict(name="append 8", op="append", tokens=8, kv=8, dim=128, page=64),
        # a whole prompt into the cache
        dict(name="append 16383", op="append", tokens=16383, kv=8, dim=128, page=64),
        # one user, one token, about a thousand slots: latency
        dict(name="decode 1x1021", op="decode", seqs=1, longest=1021, even=True, rows=1, heads=32, kv=8, dim=128,
             page=16, weights=False),
        # a batch of conversations of very different lengths, weights kept for eviction
        dict(name="decode 32 ragged", op="decode", seqs=32, longest=8191, even=False, rows=1, heads=32, kv=8,
             dim=128, page=64, weights=True),
        # four drafted tokens at once, small heads, groups of eight
        dict(name="decode drafts", op="decode", seqs=16, longest=4097, even=False, rows=4, heads=16, kv=2, dim=64,
             page=32, weights=False),
        # a full long-context batch (70B-shaped heads): the cache's bytes are all there is
        dict(name="decode 64x32768", op="decode", seqs=64, longest=32768, even=True, rows=1, heads=64, kv=8,
             dim=128, page=64, weights=False),
        # a step of a cache held at its budget: one slot a head goes
        dict(name="evict 1 of 1025", op="evict", seqs=8, longest=1025, even=True, budget=1024, recent=64, kv=8,
             dim=128, page=64),
        # long prompts cut down to their budget
        dict(name="evict 32768", op="evict", seqs=16, longest=32768, even=False, budget=4096, recent=256, kv=8,
             dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "append", "decode", "decode", "evict"])
    most = max((work(c) for c in listed() if c["op"] == op), key=lambda w: w["bytes"] + w["flops"])
    while True:
        dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        group, page = rng.choice([1, 2, 4, 5, 8]), rng.choice([16, 32, 64, 128])
        if op == "prompt":
            c = dict(op=op, seqs=_log(rng, 1, 32), longest=_log(rng, 1, 16384),
                     past=rng.choice([0, 0, _log(rng, 1, 8000)]), heads=kv * group, kv=kv, dim=dim)
        elif op == "append":
            c = dict(op=op, tokens=_log(rng, 1, 16383), kv=kv, dim=dim, page=page)
        elif op == "decode":
            c = dict(op=op, seqs=_log(rng, 1, 64), longest=_log(rng, 1, 32768), even=rng.random() < 0.3,
                     rows=rng.choice([1, 1, 1, 2, 4]), heads=kv * group, kv=kv, dim=dim, page=page,
                     weights=rng.random() < 0.4)
            c["longest"] = max(c["longest"], c["rows"])
        else:
            longest = _log(rng, 64, 32768)
            budget = _log(rng, max(16, longest // 16), longest)
            c = dict(op=op, seqs=_log(rng, 1, 16), longest=longest, even=rng.random() < 0.5, budget=budget,
                     recent=rng.randint(0, budget // 2), kv=kv, dim=dim, page=page)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _lens(case):
    """Lengths of the case's sequences: the first the longest, the others spread over
    the logarithm below it (or all nearly as long as the first)."""
    n, top, low = case["seqs"], case["longest"], case.get("rows", 1)
    r = random.Random(n * 1000003 + top)
    rest = [max(low, top - r.randint(0, 15)) if case.get("even") else _log(r, low, top) for _ in range(n - 1)]
    return [top] + rest


def _row_bytes(dim):
    return dim // 2 + 4 * (dim // BLOCK)


def work(case):
    if case["op"] == "append":
        # K and V rows in as BF16, out as codes with their (step, lo); then back to BF16
        return {"bytes": case["tokens"] * case["kv"] * 2 * 2 * (2 * case["dim"] + _row_bytes(case["dim"])), "flops": 0}
    lens = _lens(case)
    total = sum(lens)
    if case["op"] == "prompt":
        keys = total + case["past"] * len(lens)
        pairs = sum(n * (n + 1) // 2 + n * case["past"] for n in lens)
        return {"bytes": 2 * case["dim"] * (2 * total * case["heads"] + 2 * keys * case["kv"]) + 4 * total * case["heads"],
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    if case["op"] == "decode":
        q = len(lens) * case["rows"] * case["heads"]
        return {"bytes": total * case["kv"] * (2 * _row_bytes(case["dim"]) + (8 if case["weights"] else 0))
                + q * (4 * case["dim"] + 4),
                "flops": 4 * case["dim"] * case["heads"] * case["rows"] * total}
    keep = [min(n, case["budget"]) for n in lens]
    # rows that move: of the kept slots those that lie past the budget, about a share keep / len of what is cut
    moved = sum((n - k) * (k / n) for n, k in zip(lens, keep))
    return {"bytes": int(case["kv"] * (8 * total + 12 * sum(keep) + 2 * moved * 2 * _row_bytes(case["dim"]))), "flops": 0}


# ---- inputs --------------------------------------------------------------------------

class State:
    pass


def _keys(shape, g):
    """Keys as a model makes them: a few channels large, some with an offset."""
    k = torch.randn(shape, device="cuda", generator=g)
    k[..., 3::29] *= 4
    k[..., 5::17] += 1.5
    return k


def _pages(case, lens, g):
    """A filled cache: pages of quantised rows, each page scaled by a factor of its own."""
    s, kv, dim, page = State(), case["kv"], case["dim"], case["page"]
    most = -(-max(lens) // page)
    used = [-(-n // page) for n in lens]
    pages, pool = sum(used) + 3, 32
    s.table = torch.zeros(len(lens), most, dtype=torch.int32)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(case["seqs"] * 7 + most))
    at = 0
    for b, u in enumerate(used):
        s.table[b, :u] = order[at:at + u]
        at += u
    s.table = s.table.cuda()
    made = []
    for rows in (_keys((pool, kv, page, dim), g), torch.randn((pool, kv, page, dim), device="cuda", generator=g)):
        code, meta = _quantise(rows.bfloat16())
        slot = torch.arange(page, device="cuda").expand(pool, kv, page)
        pick = torch.randint(0, pool, (pages,), device="cuda", generator=g)
        by = 0.75 + 0.5 * torch.rand((pages, 1, 1, 1, 1), device="cuda", generator=g)
        made += [_pack(code, slot)[pick], (meta[pick].float() * by).bfloat16()]
    s.k_code, s.k_meta, s.v_code, s.v_meta = made
    s.host_lens = lens
    s.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dim, kv = case["dim"], case["kv"]
    if case["op"] == "prompt":
        s = State()
        s.lens, s.past = _lens(case), case["past"]
        total = sum(s.lens)
        # q, k and v as views of one fused linear's output; with earlier tokens, k and v are gathered rows
        y = torch.randn(total, (case["heads"] + 2 * kv), dim, device="cuda", generator=g).bfloat16()
        s.q = y[:, :case["heads"]]
        s.k, s.v = y[:, case["heads"]:case["heads"] + kv], y[:, case["heads"] + kv:]
        if s.past:
            keys = total + s.past * len(s.lens)
            s.k = _keys((keys, kv, dim), g).bfloat16()
            s.v = torch.randn(keys, kv, dim, device="cuda", generator=g).bfloat16()
        ends = [0]
        kends = [0]
        for n in s.lens:
            ends.append(ends[-1] + n)
            kends.append(kends[-1] + n + s.past)
        s.cu_q = torch.tensor(ends, dtype=torch.int32, device="cuda")
        s.cu_k = torch.tensor(kends, dtype=torch.int32, device="cuda")
    elif case["op"] == "append":
        s = State()
        page, tokens = case["page"], case["tokens"]
        pages = -(-tokens // page) + 2
        y = torch.cat([_keys((tokens, kv, dim), g), torch.randn(tokens, kv, dim, device="cuda", generator=g)], 1)
        y = y.bfloat16()
        s.k, s.v = y[:, :kv], y[:, kv:]
        order = torch.randperm(pages, device="cuda", generator=g)
        t = torch.arange(tokens, device="cuda")
        s.slots = (order[t // page] * page + t % page).to(torch.int32)
        s.k_code = torch.zeros(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
        s.v_code = torch.zeros_like(s.k_code)
        s.k_meta = torch.zeros(pages, kv, page, dim // BLOCK, 2, dtype=torch.bfloat16, device="cuda")
        s.v_meta = torch.zeros_like(s.k_meta)
    else:
        lens = _lens(case)
        s = _pages(case, lens, g)
        b, wide = len(lens), s.table.shape[1] * case["page"]
        if case["op"] == "decode":
            s.q = torch.randn(b, case["rows"], case["heads"], dim, device="cuda", generator=g).bfloat16()
            s.weights = case["weights"]
            if s.weights:
                s.weight = torch.rand(b, kv, wide, device="cuda", generator=g)
                s.weight_out = torch.zeros_like(s.weight)
        else:
            s.budget, s.recent = case["budget"], case["recent"]
            # sums of attention weights: most tiny, a few large, some equal
            w = torch.rand(b, kv, wide, device="cuda", generator=g).pow(6) * 8
            s.weight = torch.where(w < 1e-3, 0.0, w)
            s.weight_out = torch.zeros_like(s.weight)
            # a cache at its budget has lost tokens before, and its order is no longer that of time
            s.seen = (s.lens + s.lens // 3).to(torch.int32)
            s.pos = torch.zeros(b, kv, wide, dtype=torch.int32, device="cuda")
            for i, n in enumerate(lens):
                pick = torch.rand(kv, n + n // 3, device="cuda", generator=g).argsort(1)[:, :n]
                s.pos[i, :, :n] = pick.to(torch.int32)
            s.pos_out = torch.zeros_like(s.pos)
    s.op = case["op"]
    if own and s.op != "prompt":
        from glint_b200 import attn
        s.cache = attn.KV4Cache(s.k_code, s.k_meta, s.v_code, s.v_meta)
    return s


# ---- the operators -------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from glint_b200 import attn
    if s.op == "prompt":
        return attn.attn_prompt(s.q, s.k, s.v, s.cu_q, s.cu_k)
    if s.op == "append":
        attn.kv4_append(s.cache, s.k, s.v, s.slots)
        return attn.kv4_read(s.cache, s.slots)
    if s.op == "decode":
        if s.weights:
            o, lse = attn.kv4_attn(s.q, s.cache, s.table, s.lens, weight=s.weight, weight_out=s.weight_out)
            return o, lse, s.weight_out
        return attn.kv4_attn(s.q, s.cache, s.table, s.lens)
    kept, lens = attn.kv4_evict(s.cache, s.table, s.lens, s.weight, s.pos, s.seen, s.budget, s.recent,
                                weight_out=s.weight_out, pos_out=s.pos_out)
    # rows are moved, never computed: their bytes and (step, lo) pairs come back as they lie in the cache
    return kept, lens, s.weight_out, s.pos_out, s.k_code, s.k_meta, s.v_code, s.v_meta


def _plain(s):
    return {"prompt": _plain_prompt, "append": _plain_append, "decode": _plain_decode, "evict": _plain_evict}[s.op](s)


def _softmax(x):
    """Rows of scores -> (weights, log of the sum of exponentials)."""
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True)
    return e / z, (top + torch.log(z)).squeeze(-1)


def _plain_prompt(s):
    heads, dim, kv = s.q.shape[1], s.q.shape[2], s.k.shape[1]
    o = torch.empty(s.q.shape, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(heads, s.q.shape[0], device="cuda")
    at = kat = 0
    for n in s.lens:
        keys = n + s.past
        q = s.q[at:at + n].float().transpose(0, 1).reshape(kv, heads // kv, n, dim)
        k = s.k[kat:kat + keys].float().permute(1, 2, 0)[:, None]
        v = s.v[kat:kat + keys].float().transpose(0, 1)[:, None]
        step = max(1, (1 << 28) // (heads * keys))
        for r in range(0, n, step):
            e = min(n, r + step)
            seen = e + s.past
            x = torch.matmul(q[:, :, r:e], k[..., :seen]) * dim ** -0.5
            i = torch.arange(r, e, device="cuda")[:, None] + s.past
            x = x.masked_fill(torch.arange(seen, device="cuda") > i, float("-inf"))
            p, z = _softmax(x)
            o[at + r:at + e] = torch.matmul(p, v[:, :, :seen]).reshape(heads, e - r, dim).transpose(0, 1)
            lse[:, at + r:at + e] = z.reshape(heads, e - r)
        at, kat = at + n, kat + keys
    return o, lse


def _quantise(x):
    """BF16 rows [..., dim] -> (codes [..., dim] uint8, (step, lo) [..., dim / 64, 2] BF16)."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((hi - lo) / 15).bfloat16().float()
    code = torch.where(step > 0, torch.round((x - lo) / step).clamp(0, 15), 0.0)
    return code.to(torch.uint8).flatten(-2), torch.cat([step, lo], -1).bfloat16()


def _swapped(rows, slot):
    """Rows of bytes [..., dim / 2] with their two 32-byte halves swapped where slot & 2."""
    if rows.shape[-1] != 64:
        return rows
    return torch.where((slot & 2).bool()[..., None], rows.roll(32, -1), rows)


def _pack(code, slot):
    return _swapped(code[..., 0::2] | (code[..., 1::2] << 4), slot)


def _values(rows, meta, slot, dtype=torch.float32):
    rows = _swapped(rows, slot)
    code = torch.stack([rows & 15, rows >> 4], -1).flatten(-2).unflatten(-1, (-1, BLOCK)).to(dtype)
    meta = meta.to(dtype)
    return (meta[..., 1:] + meta[..., :1] * code).flatten(-2)


def _plain_append(s):
    page = s.k_code.shape[2]
    p, r = s.slots.long() // page, s.slots.long() % page
    out = []
    for x, codes, metas in ((s.k, s.k_code, s.k_meta), (s.v, s.v_code, s.v_meta)):
        code, meta = _quantise(x)
        codes[p, :, r] = _pack(code, r[:, None])
        metas[p, :, r] = meta
        out.append(_values(codes[p, :, r], metas[p, :, r], r[:, None]).bfloat16())
    return tuple(out)


def _cached(s, b, dtype):
    """Keys and values of sequence b: [kv, len, dim] each."""
    page, n = s.k_code.shape[2], s.host_lens[b]
    pages = s.table[b, :-(-n // page)].long()
    slot = torch.arange(page, device="cuda")
    return [_values(codes[pages], metas[pages], slot, dtype).transpose(0, 1).flatten(1, 2)[:, :n]
            for codes, metas in ((s.k_code, s.k_meta), (s.v_code, s.v_meta))]


def _plain_decode(s):
    seqs, rows, heads, dim = s.q.shape
    kv = s.k_code.shape[1]
    group = heads // kv
    o = torch.empty(s.q.shape, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(seqs, heads, rows, device="cuda")
    for b, n in enumerate(s.host_lens):
        k, v = _cached(s, b, torch.float32)
        q = s.q[b].float().transpose(0, 1).reshape(kv, group * rows, dim)
        x = torch.matmul(q, k.transpose(1, 2)) * dim ** -0.5
        i = torch.arange(n - rows, n, device="cuda")
        hide = torch.arange(n, device="cuda") > i.repeat(group)[:, None]
        p, z = _softmax(x.masked_fill(hide, float("-inf")))
        o[b] = torch.matmul(p, v).reshape(heads, rows, dim).transpose(0, 1)
        lse[b] = z.reshape(heads, rows)
        if s.weights:
            old = s.weight[b, :, :n].clone()
            old[:, n - rows:] = 0
            s.weight_out[b, :, :n] = old + p.sum(1)
    return (o, lse, s.weight_out) if s.weights else (o, lse)


def _plain_evict(s):
    kv, page = s.k_code.shape[1], s.k_code.shape[2]
    kept = torch.full((len(s.host_lens), kv, s.budget), -1, dtype=torch.int32, device="cuda")
    lens = s.lens.clamp(max=s.budget)
    heads = torch.arange(kv, device="cuda")[:, None]
    for b, length in enumerate(s.host_lens):
        n = min(length, s.budget)
        key = torch.where(s.pos[b, :, :length] >= s.seen[b] - s.recent, float("inf"), s.weight[b, :, :length])
        order = key.sort(dim=1, descending=True, stable=True).indices
        keep = torch.zeros(kv, length, dtype=torch.bool, device="cuda").scatter_(1, order[:, :n], True)
        # kept slots below n stay; the k-th free slot below n takes the k-th kept slot from n on
        src = torch.arange(n, device="cuda").repeat(kv, 1)
        h, dst = (~keep[:, :n]).nonzero(as_tuple=True)
        h, far = keep[:, n:].nonzero(as_tuple=True)
        src[h, dst] = far + n
        kept[b, :, :n] = src.to(torch.int32)
        s.weight_out[b, :, :n] = s.weight[b].gather(1, src)
        s.pos_out[b, :, :n] = s.pos[b].gather(1, src)
        to, fr = s.table[b, dst // page].long(), s.table[b, (far + n) // page].long()
        rt, rf = dst % page, (far + n) % page
        for codes, metas in ((s.k_code, s.k_meta), (s.v_code, s.v_meta)):
            codes[to, h, rt] = _swapped(_swapped(codes[fr, h, rf], rf), rt)
            metas[to, h, rt] = metas[fr, h, rf]
    return kept, lens, s.weight_out, s.pos_out, s.k_code, s.k_meta, s.v_code, s.v_meta


# ---- the definitions in 64 bits -------------------------------------------------------

def exact(case, seed):
    if case["op"] == "evict":
        return None  # whole numbers and moved rows: nothing is computed
    s = prepare(case, seed)
    if case["op"] == "append":
        out = []
        for x in (s.k, s.v):
            x = x.double().reshape(case["tokens"], case["kv"], -1, BLOCK)
            lo = x.min(-1).values
            step = ((x.max(-1).values - lo) / 15).float().bfloat16().double()
            c = torch.nan_to_num(((x - lo[..., None]) / step[..., None])).round().clamp(0, 15)
            out.append((lo[..., None] + step[..., None] * c).reshape(case["tokens"], case["kv"], -1))
        return tuple(out)
    if case["op"] == "prompt":
        group = case["heads"] // case["kv"]
        o = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
        lse = torch.empty(case["heads"], s.q.shape[0], dtype=torch.float64, device="cuda")
        at = kat = 0
        for n in s.lens:
            keys = n + s.past
            for h in range(case["heads"]):
                k, v = s.k[kat:kat + keys, h // group].double(), s.v[kat:kat + keys, h // group].double()
                for r in range(0, n, 2048):
                    e = min(n, r + 2048)
                    m = e + s.past
                    x = s.q[at + r:at + e, h].double() @ k[:m].T / math.sqrt(case["dim"])
                    i = torch.arange(r, e, device="cuda") + s.past
                    x[torch.arange(m, device="cuda")[None] > i[:, None]] = -math.inf
                    z = torch.logsumexp(x, 1)
                    o[at + r:at + e, h] = torch.exp(x - z[:, None]) @ v[:m]
                    lse[h, at + r:at + e] = z
            at, kat = at + n, kat + keys
        return o, lse
    seqs, rows, heads, dim = s.q.shape
    group = heads // case["kv"]
    o = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(seqs, heads, rows, dtype=torch.float64, device="cuda")
    total = torch.zeros(s.weight.shape, dtype=torch.float64, device="cuda") if s.weights else None
    page = case["page"]
    for b, n in enumerate(s.host_lens):
        t = torch.arange(n, device="cuda")
        where, off = s.table[b].long()[t // page], t % page
        for h in range(case["kv"]):
            kv = []
            for codes, metas in ((s.k_code, s.k_meta), (s.v_code, s.v_meta)):
                e = torch.arange(dim, device="cuda")
                byte = (e // 2)[None].expand(n, dim)
                if dim == 128:
                    byte = byte ^ (((off >> 1) & 1) * 32)[:, None]
                c = (codes[where, h, off].gather(1, byte).long() >> (4 * (e % 2))[None]) & 15
                m = metas[where, h, off].double().repeat_interleave(BLOCK, 1)
                kv.append(m[..., 1] + m[..., 0] * c.double())
            for r in range(rows):
                m = n - rows + r + 1
                x = kv[0][:m] @ s.q[b, r, h * group:(h + 1) * group].double().T / math.sqrt(dim)
                z = torch.logsumexp(x, 0)
                p = torch.exp(x - z)
                o[b, r, h * group:(h + 1) * group] = p.T @ kv[1][:m]
                lse[b, h * group:(h + 1) * group, r] = z
                if total is not None:
                    total[b, h, :m] += p.sum(1)
        if total is not None:
            old = s.weight[b, :, :n].double()
            old[:, n - rows:] = 0
            total[b, :, :n] += old
    return (o, lse) if total is None else (o, lse, total)
