"""Serving attention on torch CUDA tensors, through the C ABI of include/glint_attn.h:
what runs between a decoder's q|k|v and o linears (device.htile).

  attn_prompt   causal attention over packed prompts, grouped heads
  KV4Cache      a paged key/value cache held in 4 bits (4.5 bits a value in all)
  kv4_append    new key/value rows into their slots;  kv4_read  slots back to BF16
  kv4_attn      the newest tokens of each sequence attend to its slots
  kv4_evict     sequences cut down to a budget of slots, by accumulated weight

As in device.py torch only owns the memory and the stream, there is no CPU fallback,
bad arguments raise ValueError and a failed call RuntimeError("... rc=N").  Calls are
stream ordered and may be captured in CUDA graphs.  Tensors live on the current device.
"""
from __future__ import annotations

import ctypes
import struct
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .device import _check, lib

BLOCK = 64
_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class _Prompt(ctypes.Structure):
    """struct GlintAttnPrompt"""
    _fields_ = [(n, _vp) for n in ("q", "k", "v", "o", "lse", "cu_q", "cu_k", "work")] + \
               [(n, _i64) for n in ("q_tok", "q_head", "k_tok", "k_head", "v_tok", "v_head", "o_tok", "o_head")] + \
               [(n, _i32) for n in ("seqs", "q_tokens", "k_tokens", "heads", "kv_heads", "head_dim", "causal")] + \
               [("scale", _f32)]


class _Cache(ctypes.Structure):
    """struct GlintKv4Cache"""
    _fields_ = [(n, _vp) for n in ("k_code", "k_meta", "v_code", "v_meta")] + \
               [(n, _i32) for n in ("pages", "kv_heads", "page_size", "head_dim")]


class _Attn(ctypes.Structure):
    """struct GlintKv4Attn"""
    _fields_ = [(n, _vp) for n in ("q", "o", "lse", "table", "lens", "weight", "weight_out", "work")] + \
               [(n, _i64) for n in ("q_seq", "q_row", "q_head", "weight_stride")] + \
               [(n, _i32) for n in ("seqs", "rows", "heads", "max_pages")] + [("scale", _f32)]


class _Evict(ctypes.Structure):
    """struct GlintKv4Evict"""
    _fields_ = [(n, _vp) for n in ("table", "lens", "weight", "pos", "seen", "kept", "new_lens", "weight_out",
                                   "pos_out")] + \
               [("stride", _i64)] + [(n, _i32) for n in ("seqs", "max_pages", "budget", "recent")]


def bind(L: ctypes.CDLL) -> ctypes.CDLL:
    P = ctypes.POINTER
    L.glint_attn_prompt_work_bytes.argtypes = [P(_Prompt)]
    L.glint_attn_prompt_stream.argtypes = [P(_Prompt), _vp]
    L.glint_kv4_append_stream.argtypes = [P(_Cache), _vp, _vp, _i64, _i64, _i64, _i64, _vp, _i32, _vp]
    L.glint_kv4_read_stream.argtypes = [P(_Cache), _vp, _i32, _vp, _vp, _vp]
    L.glint_kv4_attn_work_bytes.argtypes = [P(_Cache), P(_Attn)]
    L.glint_kv4_attn_stream.argtypes = [P(_Cache), P(_Attn), _vp]
    L.glint_kv4_evict_stream.argtypes = [P(_Cache), P(_Evict), _vp]
    for f in (L.glint_attn_prompt_stream, L.glint_kv4_append_stream, L.glint_kv4_read_stream,
              L.glint_kv4_attn_stream, L.glint_kv4_evict_stream):
        f.restype = _i32
    L.glint_attn_prompt_work_bytes.restype = L.glint_kv4_attn_work_bytes.restype = _i64
    return L


def _lib() -> ctypes.CDLL:
    L = lib()
    if not getattr(L, "_attn_bound", False):
        bind(L)
        L._attn_bound = True
    return L


class _Calls:
    """The entry points taking their structs as packed bytes (a third of the time that
    filling a ctypes.Structure takes), looked up once."""

    def __init__(self):
        L = _lib()
        cp = ctypes.c_char_p

        def get(name, *args, res=_i32):
            return ctypes.CFUNCTYPE(res, *args)((name, L))
        self.prompt = get("glint_attn_prompt_stream", cp, _vp)
        self.append = get("glint_kv4_append_stream", cp, _vp, _vp, _i64, _i64, _i64, _i64, _vp, _i32, _vp)
        self.read = get("glint_kv4_read_stream", cp, _vp, _i32, _vp, _vp, _vp)
        self.attn = get("glint_kv4_attn_stream", cp, cp, _vp)
        self.evict = get("glint_kv4_evict_stream", cp, cp, _vp)
        self.prompt_work = get("glint_attn_prompt_work_bytes", cp, res=_i64)
        self.attn_work = get("glint_kv4_attn_work_bytes", cp, cp, res=_i64)


_calls: Optional[_Calls] = None


def _c() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


# the layouts of the structs above, pointers and strides in 64 bits
_pack_prompt = struct.Struct("8P8q7if").pack
_pack_cache = struct.Struct("4P4i").pack
_pack_attn = struct.Struct("8P4q4if4x").pack
_pack_evict = struct.Struct("9Pq4i").pack


# sizes grow with the current device's SMs: `dev` is part of what they are kept by
@lru_cache(maxsize=256)
def _prompt_work(dev: int, q_tokens: int, k_tokens: int, heads: int, kv_heads: int, head_dim: int) -> int:
    return max(0, _c().prompt_work(_pack_prompt(*[0] * 16, 1, q_tokens, k_tokens, heads, kv_heads, head_dim, 1, 1.0)))


@lru_cache(maxsize=256)
def _attn_work(dev: int, kv_heads: int, page_size: int, head_dim: int, seqs: int, rows: int, heads: int,
               max_pages: int, weights: bool) -> int:
    cache = _pack_cache(16, 16, 16, 16, 1, kv_heads, page_size, head_dim)  # sizes are all that counts here
    return _c().attn_work(cache, _pack_attn(*[0] * 6, 1 if weights else 0, 0, *[0] * 4, seqs, rows, heads, max_pages, 1.0))


def _raw(like: torch.Tensor, stream: Optional[torch.cuda.Stream], *others) -> int:
    """The stream's handle (torch.cuda.current_stream() itself takes 5 us of a 15 us call),
    once all tensors are seen to live on the current device."""
    dev = like.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"all tensors must be on one device, not on cuda:{dev} and {t.device}")
    if dev != torch.cuda.current_device():
        raise ValueError(f"the tensors are on cuda:{dev}, which is not the current device")
    return torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream


def _empty(like: torch.Tensor, shape, dtype: torch.dtype, stream) -> torch.Tensor:
    """Memory for the stream that writes it."""
    if stream is None:
        return like.new_empty(*shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(*shape, dtype=dtype)


def _want(t: torch.Tensor, name: str, dtype: torch.dtype, shape: Tuple[Optional[int], ...], dense: bool = True):
    """A CUDA tensor of this type and shape (None: any size); dense: contiguous,
    otherwise its last dimension contiguous."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    got = t.shape
    if got != shape:
        bad = len(got) != len(shape)
        for w, n in zip(shape, got):  # a loop: a generator's start takes as long as the rest
            if n != w and w is not None:
                bad = True
        if bad:
            raise ValueError(f"{name} must have shape {shape}, not {tuple(got)}")
    if dense:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"the last dimension of {name} must be contiguous")


def _want16(t: torch.Tensor, name: str) -> None:
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two contiguous tensors of one size."""
    return abs(a.data_ptr() - b.data_ptr()) < a.numel() * a.element_size()


def _head_dim(d: int) -> None:
    if d not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, not {d}")


def attn_prompt(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor,
                cu_k: Optional[torch.Tensor] = None, causal: bool = True, scale: Optional[float] = None,
                out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, stream=None):
    """o [q_tokens, heads, head_dim] BF16 and lse [heads, q_tokens] f32 of packed sequences.

    q [q_tokens, heads, head_dim], k and v [k_tokens, kv_heads, head_dim] BF16, any strides with
    a contiguous last dimension (views of a fused q|k|v output, for example); cu_q and
    cu_k [seqs + 1] int32: where each sequence's tokens begin and end (cu_k = cu_q when
    left out).  Query i of Lq sees keys j <= i + Lk - Lq when causal (the last queries
    line up with the last keys, so earlier tokens' keys go first), every key otherwise.
    scale defaults to head_dim ** -0.5.  A row that sees no key gets 0 and -inf."""
    _want(q, "q", torch.bfloat16, (None, None, None), dense=False)
    T, H, D = q.shape
    _head_dim(D)
    _want(k, "k", torch.bfloat16, (None, None, D), dense=False)
    Tk, Hk = k.shape[0], k.shape[1]
    _want(v, "v", torch.bfloat16, (Tk, Hk, D), dense=False)
    if Hk < 1 or H < 1 or H % Hk:
        raise ValueError(f"heads ({H}) must be a multiple of kv_heads ({Hk})")
    _want(cu_q, "cu_q", torch.int32, (None,))
    if cu_k is None:
        if Tk != T:
            raise ValueError("cu_k may be left out only where k has q's tokens")
        cu_k = cu_q
    else:
        _want(cu_k, "cu_k", torch.int32, cu_q.shape)
    if cu_q.shape[0] < 1:
        raise ValueError("cu_q must have one entry more than there are sequences")
    if out is None:
        out = _empty(q, (T, H, D), torch.bfloat16, stream)
    else:
        _want(out, "out", torch.bfloat16, (T, H, D), dense=False)
    if lse is None:
        lse = _empty(q, (H, T), torch.float32, stream)
    else:
        _want(lse, "lse", torch.float32, (H, T))
    raw = _raw(q, stream, k, v, cu_q, cu_k, out, lse)
    n = _prompt_work(q.get_device(), T, Tk, H, Hk, D)
    work = _empty(q, (n,), torch.uint8, stream) if n else None
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    a = _pack_prompt(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), cu_q.data_ptr(),
                     cu_k.data_ptr(), work.data_ptr() if n else 0, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
                     cu_q.shape[0] - 1, T, Tk, H, Hk, D, 1 if causal else 0, D ** -0.5 if scale is None else scale)
    _check(_c().prompt(a, raw), "glint_attn_prompt_stream")
    return out, lse


class KV4Cache:
    """One layer's key/value cache in 4 bits, in pages of page_size slots.

    k_code, v_code [pages, kv_heads, page_size, head_dim / 2] uint8 and k_meta, v_meta
    [pages, kv_heads, page_size, head_dim / 64, 2] BF16 (step, lo): include/glint_attn.h
    has the layout.  The tensors are the caller's to keep; slots are filled by
    kv4_append and need no initial value."""

    def __init__(self, k_code: torch.Tensor, k_meta: torch.Tensor, v_code: torch.Tensor, v_meta: torch.Tensor):
        _want(k_code, "k_code", torch.uint8, (None, None, None, None))
        pages, kv_heads, page_size, half = k_code.shape
        _head_dim(2 * half)
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, not {page_size}")
        if pages < 1 or kv_heads < 1 or pages * page_size > 2 ** 31 - 1:
            raise ValueError(f"a cache has between 1 and 2**31 - 1 slots, not {pages} pages of {page_size}")
        _want(v_code, "v_code", torch.uint8, k_code.shape)
        for t, name in ((k_meta, "k_meta"), (v_meta, "v_meta")):
            _want(t, name, torch.bfloat16, (pages, kv_heads, page_size, half // 32, 2))
        if any(t.data_ptr() % 16 for t in (k_code, k_meta, v_code, v_meta)):
            raise ValueError("the cache's tensors must be 16-byte aligned")
        if any(t.device != k_code.device for t in (k_meta, v_code, v_meta)):
            raise ValueError("the cache's tensors must be on one device")
        self.k_code, self.k_meta, self.v_code, self.v_meta = k_code, k_meta, v_code, v_meta
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, kv_heads, page_size, 2 * half
        self._c = _pack_cache(k_code.data_ptr(), k_meta.data_ptr(), v_code.data_ptr(), v_meta.data_ptr(), pages,
                              kv_heads, page_size, 2 * half)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "KV4Cache":
        _head_dim(head_dim)

        def code():
            return torch.empty((pages, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)

        def meta():
            return torch.empty((pages, kv_heads, page_size, head_dim // BLOCK, 2), dtype=torch.bfloat16, device=device)
        return cls(code(), meta(), code(), meta())


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, stream=None) -> None:
    """k, v [tokens, kv_heads, head_dim] BF16 (any strides, last dimension contiguous), quantised
    into slots[t] = page * page_size + place in the page (int32; negative: skipped)."""
    _want(k, "k", torch.bfloat16, (None, cache.kv_heads, cache.head_dim), dense=False)
    _want(v, "v", torch.bfloat16, k.shape, dense=False)
    _want(slots, "slots", torch.int32, k.shape[:1])
    ks, vs = k.stride(), v.stride()
    _check(_c().append(cache._c, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), k.shape[0],
                       _raw(k, stream, v, slots, cache.k_code)), "glint_kv4_append_stream")


def kv4_read(cache: KV4Cache, slots: torch.Tensor, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [tokens, kv_heads, head_dim] BF16: the values of slots[t] (zeros for a slot outside
    the cache), for example as attn_prompt's keys of an earlier part of a prompt."""
    _want(slots, "slots", torch.int32, (None,))
    shape = (slots.shape[0], cache.kv_heads, cache.head_dim)
    if k_out is None:
        k_out = _empty(slots, shape, torch.bfloat16, stream)
    else:
        _want(k_out, "k_out", torch.bfloat16, shape)
        _want16(k_out, "k_out")
    if v_out is None:
        v_out = _empty(slots, shape, torch.bfloat16, stream)
    else:
        _want(v_out, "v_out", torch.bfloat16, shape)
        _want16(v_out, "v_out")
    _check(_c().read(cache._c, slots.data_ptr(), shape[0], k_out.data_ptr(), v_out.data_ptr(),
                     _raw(slots, stream, k_out, v_out, cache.k_code)), "glint_kv4_read_stream")
    return k_out, v_out


def kv4_attn(q: torch.Tensor, cache: KV4Cache, table: torch.Tensor, lens: torch.Tensor,
             scale: Optional[float] = None, weight: Optional[torch.Tensor] = None,
             weight_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             lse: Optional[torch.Tensor] = None, stream=None):
    """o (as q, contiguous) and lse [seqs, heads, rows] f32 of each sequence's newest `rows`
    tokens over its lens[b] cached slots, which end with those tokens' own.

    q [seqs, rows, heads, head_dim] BF16 (any strides, last dimension contiguous); table
    [seqs, max_pages] int32: the pages of a sequence in order; lens [seqs] int32.  With
    weight_out [seqs, kv_heads, >= max_pages * page_size] f32 each slot's softmax weights,
    summed over the head's query heads and rows, are added to weight (zero when left
    out, and in the newest `rows` slots) and written there; weight_out may be weight."""
    _want(q, "q", torch.bfloat16, (None, None, None, cache.head_dim), dense=False)
    B, R, H, D = q.shape
    if H < 1 or H % cache.kv_heads:
        raise ValueError(f"heads ({H}) must be a multiple of kv_heads ({cache.kv_heads})")
    if R < 1 or H // cache.kv_heads * R > 256:
        raise ValueError(f"rows ({R}) times query heads a kv head must be 1 to 256")
    _want(table, "table", torch.int32, (B, None))
    _want(lens, "lens", torch.int32, (B,))
    P = table.shape[1]
    if P < 1 or P * cache.page_size > 2 ** 31 - 1:
        raise ValueError(f"table must name between 1 and 2**31 - 1 slots a sequence, not {P} pages of {cache.page_size}")
    wide = 0
    if weight_out is not None:
        _want(weight_out, "weight_out", torch.float32, (B, cache.kv_heads, None))
        wide = weight_out.shape[2]
        if wide < P * cache.page_size:
            raise ValueError(f"weight_out must have {P * cache.page_size} slots or more, not {wide}")
        if weight is not None:
            _want(weight, "weight", torch.float32, (B, cache.kv_heads, wide))
            if weight.data_ptr() != weight_out.data_ptr() and _overlap(weight, weight_out):
                raise ValueError("weight_out must be weight or apart from it")
    elif weight is not None:
        raise ValueError("weight needs weight_out")
    if out is None:
        out = _empty(q, (B, R, H, D), torch.bfloat16, stream)
    else:
        _want(out, "out", torch.bfloat16, (B, R, H, D))
        _want16(out, "out")
    if lse is None:
        lse = _empty(q, (B, H, R), torch.float32, stream)
    else:
        _want(lse, "lse", torch.float32, (B, H, R))
    raw = _raw(q, stream, cache.k_code, table, lens, weight, weight_out, out, lse)
    n = _attn_work(q.get_device(), cache.kv_heads, cache.page_size, D, B, R, H, P, weight_out is not None)
    if n < 0:
        raise ValueError(f"{B} sequences of up to {P} pages, {cache.kv_heads} kv heads and {H // cache.kv_heads * R} rows a kv "
                         "head are more than one call takes")
    work = _empty(q, (n,), torch.uint8, stream)
    qs = q.stride()
    a = _pack_attn(q.data_ptr(), out.data_ptr(), lse.data_ptr(), table.data_ptr(), lens.data_ptr(),
                   0 if weight is None else weight.data_ptr(), 0 if weight_out is None else weight_out.data_ptr(),
                   work.data_ptr(), qs[0], qs[1], qs[2], wide, B, R, H, P,
                   D ** -0.5 if scale is None else scale)
    _check(_c().attn(cache._c, a, raw), "glint_kv4_attn_stream")
    return out, lse


def kv4_evict(cache: KV4Cache, table: torch.Tensor, lens: torch.Tensor, weight: torch.Tensor, pos: torch.Tensor,
              seen: torch.Tensor, budget: int, recent: int = 0, *, weight_out: torch.Tensor, pos_out: torch.Tensor,
              stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cut every sequence down to n = min(lens[b], budget) slots, each kv head on its own:
    kept are the slots with pos >= seen[b] - recent, then the largest weights, ties to
    the lowest slot; kept slots from n on move into the freed slots below n.

    weight f32 and pos int32 [seqs, kv_heads, >= max_pages * page_size] belong to the
    slots (pos: the token's position); seen [seqs] int32: tokens seen so far.  weight_out
    and pos_out get the kept slots' entries and may not be weight and pos themselves
    (two pairs of tensors that take turns).  Returns
    (kept [seqs, kv_heads, budget] int32: the slot each one came from, -1 from n on;
    new_lens [seqs] int32)."""
    B, P = table.shape if table.dim() == 2 else (None, 0)
    _want(table, "table", torch.int32, (None, None))
    _want(lens, "lens", torch.int32, (B,))
    _want(seen, "seen", torch.int32, (B,))
    _want(weight, "weight", torch.float32, (B, cache.kv_heads, None))
    wide = weight.shape[2]
    _want(pos, "pos", torch.int32, (B, cache.kv_heads, wide))
    if not 1 <= budget < 2 ** 31 or recent < 0 or recent > budget:
        raise ValueError("budget must be 1 or more (in 31 bits) and recent between 0 and budget")
    if P < 1 or P * cache.page_size > min(wide, 524288):
        raise ValueError(f"table has room for {P * cache.page_size} slots: weight must cover them, 524288 at most")
    kept = _empty(table, (B, cache.kv_heads, budget), torch.int32, stream)
    new_lens = _empty(table, (B,), torch.int32, stream)
    _want(weight_out, "weight_out", torch.float32, weight.shape)
    _want(pos_out, "pos_out", torch.int32, pos.shape)
    if _overlap(weight_out, weight) or _overlap(pos_out, pos):
        raise ValueError("weight_out and pos_out must not be weight and pos, nor overlap them")
    e = _pack_evict(table.data_ptr(), lens.data_ptr(), weight.data_ptr(), pos.data_ptr(), seen.data_ptr(), kept.data_ptr(),
               new_lens.data_ptr(), weight_out.data_ptr(), pos_out.data_ptr(), wide, B, P, budget, recent)
    _check(_c().evict(cache._c, e, _raw(table, stream, cache.k_code, lens, weight, pos, seen, weight_out, pos_out)),
           "glint_kv4_evict_stream")
    return kept, new_lens
