"""Cases of the operators beside a served decoder layer's attention: rotary positions with
norms of the heads, the same with keys and values written to the 4-bit cache, and the gated
feed-forward projection on GLINT planes.

`own` chooses between the plain form (elementary torch operations in 32 bits, angles and
norms in 64) and the framework's kernels; both take what prepare() gives.  The plain form
is also the written definition of each operator:

rope    a head x of dim values, rot <= dim of them rotated; with norms y = x r w, r = 1 /
        sqrt(mean(x^2) + eps), else y = x.  a_i = position * inv_freq[i], c = scale cos a,
        s = scale sin a; pairs (i, i + rot / 2), or (2i, 2i + 1) where interleaved:
        (y1 c - y2 s, y2 c + y1 s).  Values from rot on are y.
append  rope, and the rotated k (rounded to BF16) and v into the 4-bit cache: blocks of 64
        values of one head: lo = min, step = BF16((max - min) / 15), code = rint((x - lo) /
        step) in 0..15, value lo + step * code; what the slots then hold is read back.
gated   h[m, f] = act(g) u, g = W[2f] . x[m], u = W[2f + 1] . x[m]; W [2 ff, hidden] in
        GLINT planes: CELLS[hole][plug] * absmax of its 64 values, even elements of a plane in
        the low nibble.  act(g) = g / (1 + exp(-z)), z = g (silu) or 2 sqrt(2 / pi) (g +
        0.044715 g^3) (gelu).
"""
import math
import random
import re

import torch

own = False

BLOCK = 64
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------

def listed():
    return [
        # one user's next token: launch latency is all there is
        dict(name="rope 1", op="rope", tokens=1, heads=32, kv=8, dim=128, rot=128, inter=False, norms=False, far=8191,
             stretched=False),
        # a chunk of a long document, a part of each head rotated, frequencies stretched for the length
        dict(name="rope 513 part", op="rope", tokens=513, heads=24, kv=8, dim=128, rot=96, inter=False, norms=False,
             far=131071, stretched=True),
        # packed prompts, small heads, neighbouring values paired
        dict(name="rope 4099 pairs", op="rope", tokens=4099, heads=16, kv=4, dim=64, rot=64, inter=True, norms=False,
             far=4099, stretched=False),
        # a whole long document, queries and keys normed
        dict(name="rope 32768 norms", op="rope", tokens=32768, heads=32, kv=8, dim=128, rot=128, inter=False, norms=True,
             far=32768, stretched=False),
        # a decoded token for each of seven sequences
        dict(name="append 7", op="append", tokens=7, heads=32, kv=8, dim=128, rot=128, inter=False, norms=True, far=131071,
             stretched=True, page=64, keys=False),
        # a prompt, small heads, half of each rotated, its keys also wanted for the attention over the prompt
        dict(name="append 1999 pairs", op="append", tokens=1999, heads=16, kv=2, dim=64, rot=32, inter=True, norms=False,
             far=1999, stretched=False, page=32, keys=True),
        # a long document's queries, keys and values
        dict(name="append 16383", op="append", tokens=16383, heads=32, kv=8, dim=128, rot=128, inter=False, norms=True,
             far=16383, stretched=False, page=64, keys=True),
        # one token through an 8B-shaped layer: the planes' bytes
        dict(name="gated 1", op="gated", rows=1, hidden=4096, ff=14336, gelu=False),
        # a batch of tokens through a small layer of odd width
        dict(name="gated 29", op="gated", rows=29, hidden=2560, ff=6911, gelu=True),
        # sixteen tokens, 70B-shaped
        dict(name="gated 16 wide", op="gated", rows=16, hidden=8192, ff=28672, gelu=False),
        # a few hundred tokens of packed prompts
        dict(name="gated 511", op="gated", rows=511, hidden=4096, ff=14336, gelu=False),
        # a long prompt: the tensor cores' rate
        dict(name="gated 8191", op="gated", rows=8191, hidden=4096, ff=14336, gelu=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "gated"])
    most = {}
    for c in listed():
        if c["op"] == op:
            for k, v in work(c).items():
                most[k] = max(most.get(k, 0), v)
    while True:
        if op == "gated":
            c = dict(op=op, rows=_log(rng, 1, 8191), hidden=256 * rng.randint(2, 32), ff=_log(rng, 64, 28672),
                     gelu=rng.random() < 0.3)
        else:
            dim, kv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
            rot = rng.choice([dim, dim, dim // 2, 3 * dim // 4, 2 * rng.randint(1, dim // 2)])
            tokens = _log(rng, 1, 32768 if op == "rope" else 16383)
            c = dict(op=op, tokens=tokens, heads=kv * rng.choice([1, 2, 4, 5, 8]), kv=kv, dim=dim, rot=rot,
                     inter=rng.random() < 0.4, norms=rng.random() < 0.5, far=_log(rng, tokens, 1 << 20),
                     stretched=rng.random() < 0.4)
            if op == "append":
                c.update(page=rng.choice([16, 32, 64, 128]), keys=rng.random() < 0.5)
        w = work(c)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return c


def _row_bytes(dim):
    return dim // 2 + 4 * (dim // BLOCK)


def work(case):
    if case["op"] == "gated":
        m, k, f = case["rows"], case["hidden"], case["ff"]
        return {"bytes": 2 * f * k + 2 * f * k // 16 + 2 * m * k + 2 * m * f, "flops": 4 * m * f * k}
    t, dim, kv = case["tokens"], case["dim"], case["kv"]
    small = 4 * t + 2 * case["rot"] + (8 * dim if case["norms"] else 0)
    if case["op"] == "rope":
        return {"bytes": t * (case["heads"] + kv) * 4 * dim + small, "flops": 0}
    # q in and out, k and v in, codes out; the keys once more where they are wanted; the slots read back as BF16
    rows = case["heads"] * 4 * dim + kv * (4 * dim + (2 * dim if case["keys"] else 0))
    return {"bytes": t * (rows + kv * 2 * (2 * _row_bytes(dim) + 2 * dim)) + small + 4 * t, "flops": 0}


# ---- inputs --------------------------------------------------------------------------

class State:
    pass


def _cells():
    """GLINT_CELLS [256] f32, from the library's header."""
    text = open("include/glint_cells.h").read()
    text = text[text.index("GLINT_CELLS_INIT"):]
    return torch.tensor([float.fromhex(v) for v in re.findall(r"-?0x[0-9a-f.]+p[-+]\d+", text)[:256]])


def _planes(rows, hidden, g):
    """Codes and scales as an encoded weight has them: a pool of rows, each row scaled by a factor of its own."""
    cells = _cells().cuda()
    pool = torch.randn(512, hidden // BLOCK, BLOCK, device="cuda", generator=g) * 0.02
    pool = torch.where(torch.rand(pool.shape, device="cuda", generator=g) < 1e-3, 20 * pool, pool)
    absmax = pool.abs().amax(-1)
    code = torch.bucketize(pool / absmax[..., None], (cells[1:] + cells[:-1]) / 2).view(512, hidden)
    hole, plug = (code >> 4).to(torch.uint8), (code & 15).to(torch.uint8)
    pick = torch.randint(0, 512, (rows,), device="cuda", generator=g)
    by = 0.5 + torch.rand((rows, 1), device="cuda", generator=g)
    return [(p[:, 0::2] | (p[:, 1::2] << 4))[pick].view(-1) for p in (hole, plug)] + [(absmax[pick] * by).view(-1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = State()
    s.op = case["op"]
    if s.op == "gated":
        s.ff, s.hidden, s.gelu = case["ff"], case["hidden"], case["gelu"]
        s.hole, s.plug, s.absmax = _planes(2 * s.ff, s.hidden, g)
        s.x = torch.randn(case["rows"], s.hidden, device="cuda", generator=g).bfloat16()
        s.cells = _cells().cuda()
        return s
    t, heads, kv, dim, rot = case["tokens"], case["heads"], case["kv"], case["dim"], case["rot"]
    # q, k and v as views of one fused linear's rows; a few channels of k larger, some with an offset
    y = torch.randn(t, heads + 2 * kv, dim, device="cuda", generator=g)
    y[:, heads:heads + kv, 3::29] *= 2
    y[:, heads:heads + kv, 5::17] += 1
    y = y.bfloat16()
    s.q, s.k, s.v = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    # a prompt's tokens in a row up to the farthest, or (few tokens) each of a sequence of its own
    r = random.Random(seed)
    if t > 256:
        s.positions = torch.arange(case["far"] - t + 1, case["far"] + 1, dtype=torch.int32, device="cuda")
    else:
        s.positions = torch.tensor([r.randint(0, case["far"]) for _ in range(t)], dtype=torch.int32, device="cuda")
    i = torch.arange(rot // 2, dtype=torch.float64)
    freq = 500000.0 ** (-2 * i / rot)
    s.scale = 1.0
    if case["stretched"]:  # slow frequencies slowed eight times, fast ones kept, a ramp between
        turns = 8192 * freq / (2 * math.pi)
        keep = ((turns - 1) / 31).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / 8)
        s.scale = 0.1 * math.log(8) + 1
    s.inv_freq = freq.float().cuda()
    s.inter = case["inter"]
    s.q_norm = s.k_norm = None
    if case["norms"]:
        s.q_norm, s.k_norm = 1 + 0.2 * torch.randn(2, dim, device="cuda", generator=g)
    if s.op == "append":
        page = case["page"]
        pages = -(-t // page) + 2
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(t, device="cuda")
        s.slots = (order[at // page] * page + at % page).to(torch.int32)
        s.k_code = torch.zeros(pages, kv, page, dim // 2, dtype=torch.uint8, device="cuda")
        s.v_code = torch.zeros_like(s.k_code)
        s.k_meta = torch.zeros(pages, kv, page, dim // BLOCK, 2, dtype=torch.bfloat16, device="cuda")
        s.v_meta = torch.zeros_like(s.k_meta)
        s.k_out = torch.empty(t, kv, dim, dtype=torch.bfloat16, device="cuda") if case["keys"] else None
        if own:
            from glint_b200 import attn
            s.cache = attn.KV4Cache(s.k_code, s.k_meta, s.v_code, s.v_meta)
    return s


# ---- the operators -------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    if s.op == "gated":
        from glint_b200 import device
        return device.htile_gated(s.x, s.hole, s.plug, s.absmax, s.ff, mode="fast", act="gelu_tanh" if s.gelu else "silu")
    from glint_b200 import attn
    if s.op == "rope":
        return attn.rope(s.q, s.k, s.positions, s.inv_freq, interleaved=s.inter, scale=s.scale, q_norm=s.q_norm,
                         k_norm=s.k_norm, eps=EPS)
    q = attn.rope_append(s.cache, s.q, s.k, s.v, s.positions, s.inv_freq, s.slots, interleaved=s.inter, scale=s.scale,
                         q_norm=s.q_norm, k_norm=s.k_norm, eps=EPS, k_out=s.k_out)
    return (q, s.k_out) + attn.kv4_read(s.cache, s.slots)


def _plain(s):
    return {"rope": _plain_rope, "append": _plain_append, "gated": _plain_gated}[s.op](s)


def _turned(x, s, norm):
    """Rows [tokens, heads, dim], normed (where there is a weight) and rotated, as BF16."""
    x = x.float()
    if norm is not None:
        r = torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS).float()
        x = x * r * norm
    a = s.positions.double()[:, None, None] * s.inv_freq.double()
    c, n = (a.cos() * s.scale).float(), (a.sin() * s.scale).float()
    half = c.shape[-1]
    if s.inter:
        x1, x2 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([x1 * c - x2 * n, x2 * c + x1 * n], -1).flatten(-2)
    else:
        x1, x2 = x[..., :half], x[..., half:2 * half]
        y = torch.cat([x1 * c - x2 * n, x2 * c + x1 * n], -1)
    return torch.cat([y, x[..., 2 * half:]], -1).bfloat16()


def _plain_rope(s):
    return _turned(s.q, s, s.q_norm), _turned(s.k, s, s.k_norm)


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


def _plain_append(s):
    page = s.k_code.shape[2]
    p, r = s.slots.long() // page, s.slots.long() % page
    q, k = _plain_rope(s)

    def cached(x, codes, metas):
        code, meta = _quantise(x)
        codes[p, :, r] = _swapped(code[..., 0::2] | (code[..., 1::2] << 4), r[:, None])
        metas[p, :, r] = meta
        rows, meta = _swapped(codes[p, :, r], r[:, None]), metas[p, :, r].float()
        code = torch.stack([rows & 15, rows >> 4], -1).flatten(-2).unflatten(-1, (-1, BLOCK)).float()
        return (meta[..., 1:] + meta[..., :1] * code).flatten(-2).bfloat16()

    if s.k_out is not None:
        s.k_out.copy_(k)
    return q, s.k_out, cached(k, s.k_code, s.k_meta), cached(s.v, s.v_code, s.v_meta)


def _codes(plane, hidden):
    return torch.stack([plane & 15, plane >> 4], -1).view(-1, hidden)


def _plain_gated(s):
    code = (_codes(s.hole, s.hidden) << 4 | _codes(s.plug, s.hidden)).int()
    w = (s.cells[code].view(-1, BLOCK) * s.absmax[:, None]).view(-1, s.hidden)
    y = torch.matmul(s.x.float(), w.T)
    g, u = y[:, 0::2], y[:, 1::2]
    z = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g) if s.gelu else g
    return (g / (1 + torch.exp(-z)) * u).bfloat16()


# ---- the definitions in 64 bits -------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "gated":
        h = torch.empty(case["rows"], s.ff, dtype=torch.float64, device="cuda")
        cells, half = s.cells.double(), s.hidden // 2
        hole, plug = s.hole.view(s.ff, 2, half), s.plug.view(s.ff, 2, half)
        am = s.absmax.view(s.ff, 2, -1).double().repeat_interleave(BLOCK, -1)
        x = s.x.double()
        for f in range(0, s.ff, 2048):
            y = []
            for part in (0, 1):
                lo, hi = hole[f:f + 2048, part].long(), plug[f:f + 2048, part].long()
                w = torch.empty(lo.shape[0], s.hidden, dtype=torch.float64, device="cuda")
                w[:, 0::2], w[:, 1::2] = cells[(lo % 16) * 16 + hi % 16], cells[(lo // 16) * 16 + hi // 16]
                y.append(x @ (w * am[f:f + 2048, part]).T)
            z = y[0] if not s.gelu else math.sqrt(8 / math.pi) * (y[0] + 0.044715 * y[0] ** 3)
            h[:, f:f + 2048] = y[0] * torch.sigmoid(z) * y[1]
        return h

    def turned(x, w):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w.double()
        z = y.clone()
        half = case["rot"] // 2
        for i in range(half):
            a = s.positions.double() * s.inv_freq[i].double()
            c, n = s.scale * torch.cos(a)[:, None], s.scale * torch.sin(a)[:, None]
            p, o = (2 * i, 2 * i + 1) if s.inter else (i, i + half)
            z[..., p] = y[..., p] * c - y[..., o] * n
            z[..., o] = y[..., o] * c + y[..., p] * n
        return z

    def held(x):
        x = x.double().reshape(case["tokens"], case["kv"], -1, BLOCK)
        lo = x.min(-1).values
        step = ((x.max(-1).values - lo) / 15).float().bfloat16().double()
        c = torch.nan_to_num((x - lo[..., None]) / step[..., None]).round().clamp(0, 15)
        return (lo[..., None] + step[..., None] * c).reshape(case["tokens"], case["kv"], -1)

    q, k = turned(s.q, s.q_norm), turned(s.k, s.k_norm)
    if s.op == "rope":
        return q, k
    return q, (k if case["keys"] else None), held(k.bfloat16()), held(s.v)
