"""Serving attention on torch CUDA tensors, through the C ABI of include/glint_attn.h:
what runs between a decoder's q|k|v and o linears (device.htile).

  rope          rotary positions of q and k, norms of their heads before them
  rope_freqs    its frequencies, stretched for long contexts or not
  rope_append   rope, and keys and values into the cache, in one pass
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
import math
import struct
from functools import lru_cache
from typing import Optional, Tuple

import torch

from .device import _check, lib

BLOCK = 64
_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


class _Rope(ctypes.Structure):
    """struct GlintRope"""
    _fields_ = [(n, _vp) for n in ("q", "k", "q_out", "k_out", "positions", "inv_freq", "q_norm", "k_norm")] + \
               [(n, _i64) for n in ("q_tok", "q_head", "k_tok", "k_head", "qo_tok", "qo_head", "ko_tok", "ko_head")] + \
               [("scale", ctypes.c_double), ("eps", ctypes.c_double)] + \
               [(n, _i32) for n in ("tokens", "heads", "kv_heads", "head_dim", "half", "interleaved")]


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
    L.glint_rope_stream.argtypes = [P(_Rope), _vp]
    L.glint_kv4_rope_append_stream.argtypes = [P(_Cache), P(_Rope), _vp, _i64, _i64, _vp, _vp]
    L.glint_attn_prompt_work_bytes.argtypes = [P(_Prompt)]
    L.glint_attn_prompt_stream.argtypes = [P(_Prompt), _vp]
    L.glint_kv4_append_stream.argtypes = [P(_Cache), _vp, _vp, _i64, _i64, _i64, _i64, _vp, _i32, _vp]
    L.glint_kv4_read_stream.argtypes = [P(_Cache), _vp, _i32, _vp, _vp, _vp]
    L.glint_kv4_attn_work_bytes.argtypes = [P(_Cache), P(_Attn)]
    L.glint_kv4_attn_stream.argtypes = [P(_Cache), P(_Attn), _vp]
    L.glint_kv4_evict_stream.argtypes = [P(_Cache), P(_Evict), _vp]
    for f in (L.glint_rope_stream, L.glint_kv4_rope_append_stream, L.glint_attn_prompt_stream, L.glint_kv4_append_stream, L.glint_kv4_read_stream,
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
        self.rope = get("glint_rope_stream", cp, _vp)
        self.rope_append = get("glint_kv4_rope_append_stream", cp, cp, _vp, _i64, _i64, _vp, _vp)
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
_pack_rope = struct.Struct("8P8q2d6i").pack
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


# of a model's rope_scaling: what each rope_type reads, and what changes nothing (the original length alone only
# says when to stretch, short_factor and long_factor are what `factors` was taken from)
_ROPE_KEYS = {
    "default": {"original_max_position_embeddings"},
    "linear": {"factor", "original_max_position_embeddings"},
    "llama3": {"factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor", "mscale",
             "mscale_all_dim", "truncate"},
    "longrope": {"factors", "factor", "original_max_position_embeddings", "attention_factor", "short_factor", "long_factor"},
}
_ROPE_INERT = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "finetuned"}


def rope_freqs(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
               device="cuda") -> Tuple[torch.Tensor, float]:
    """(inv_freq [rotary_dim / 2] f32, scale) for rope: base ** (-2 i / rotary_dim), stretched for contexts
    longer than a model was trained on as `scaling` says, in the keys of a model's rope_scaling
    (rope_type, or type):

    default   not stretched
    linear    every frequency divided by `factor`
    llama3    wavelengths over original_max_position_embeddings / low_freq_factor divided by `factor`,
              those under .. / high_freq_factor kept, between them a ramp over their turns
    yarn      frequencies of fewer than beta_slow (1) turns in the original length divided by `factor`,
              those of more than beta_fast (32) kept, between them a ramp over their numbers, whose ends
              are whole numbers unless truncate is False; scale attention_factor, or with mscale
              and mscale_all_dim m(mscale) / m(mscale_all_dim), or m(1), m(s) = 0.1 s ln(factor) + 1
    longrope  each divided by its own of `factors` (a model's short_factor or long_factor); scale
              attention_factor, or with `factor` sqrt(1 + ln(factor) / ln(original length)), or 1

    rotary_dim is the part of a head that is rotated, partial_rotary_factor included; rope_theta, where
    `scaling` has it, must be `base`.  A key that the kind does not read and that could change the
    result raises ValueError; keys whose value is None count as absent."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, not {rotary_dim}")
    if not base > 0:
        raise ValueError(f"base must be above 0, not {base}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = base ** (-2 * i / max(rotary_dim, 1))
    scaling = {key: v for key, v in (scaling or {}).items() if v is not None}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in _ROPE_KEYS:
        raise ValueError(f"rope_type must be default, linear, llama3, yarn or longrope, not {kind!r}")
    unread = sorted(set(scaling) - _ROPE_KEYS[kind] - _ROPE_INERT)
    if unread:
        raise ValueError(f"rope_type {kind!r} does not read {', '.join(map(repr, unread))}")
    if scaling.get("rope_theta", base) != base:
        raise ValueError(f"base is {base}, but 'rope_theta' {scaling['rope_theta']}")

    def of(key, *default):
        v = scaling.get(key)
        if v is None:
            if not default:
                raise ValueError(f"rope_type {kind!r} needs {key!r}")
            return default[0]
        if key != "attention_factor" and not v > 0:
            raise ValueError(f"{key!r} must be above 0, not {v}")
        return float(v)
    scale = 1.0
    if kind == "linear":
        freq = freq / of("factor")
    elif kind == "llama3":
        low, high = of("low_freq_factor"), of("high_freq_factor")
        if not high > low:
            raise ValueError(f"'high_freq_factor' must be above 'low_freq_factor', not {high} and {low}")
        turns = of("original_max_position_embeddings") * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / of("factor"))
    elif kind == "yarn":
        factor, length = of("factor"), of("original_max_position_embeddings")
        if base == 1:
            raise ValueError("rope_type 'yarn' needs a base other than 1")

        def number(turns):  # of the frequency that makes so many turns
            return rotary_dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = number(of("beta_fast", 32.0)), number(of("beta_slow", 1.0))
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        keep = 1 - ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq * (keep + (1 - keep) / factor)

        def magnitude(by):
            return 0.1 * by * math.log(factor) + 1 if factor > 1 else 1.0
        if ("mscale" in scaling) != ("mscale_all_dim" in scaling):
            raise ValueError("'mscale' and 'mscale_all_dim' go together")
        scale = of("attention_factor", magnitude(of("mscale", 1.0)) / magnitude(of("mscale_all_dim"))
                   if "mscale_all_dim" in scaling else magnitude(1.0))
    elif kind == "longrope":
        factors = torch.as_tensor(scaling.get("factors", []), dtype=torch.float64, device="cpu")
        if factors.shape != freq.shape or not bool((factors > 0).all()):
            raise ValueError(f"'factors' must be {rotary_dim // 2} numbers above 0")
        freq = freq / factors
        by, scale = of("factor", 1.0), of("attention_factor", 1.0)
        if by > 1 and "attention_factor" not in scaling:
            length = of("original_max_position_embeddings")
            if length == 1:
                raise ValueError("'original_max_position_embeddings' must be above 1")
            scale = math.sqrt(1 + math.log(by) / math.log(length))
    return freq.float().to(device), scale


def _heads_apart(t: torch.Tensor) -> bool:
    """No two heads of [tokens, heads, head_dim] lie on one another."""
    (T, H, D), (st, sh, _) = t.shape, t.stride()
    return not T or not H or (sh >= D or H == 1) and (st >= (H - 1) * sh + D or T == 1) or \
        (st >= D or T == 1) and (sh >= (T - 1) * st + D or H == 1)


def _rows_apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Two [tokens, heads, head_dim] tensors of one type surely share no element: their spans do
    not meet, or they are different heads of one buffer, beside one another or in turn, with either axis the outer one."""
    (Ta, Ha, D), (sa, ha, _) = a.shape, a.stride()
    (Tb, Hb, _), (sb, hb, _) = b.shape, b.stride()
    if not (Ta and Ha and Tb and Hb):
        return True
    size, pa, pb = a.element_size(), a.data_ptr(), b.data_ptr()
    if pa + ((Ta - 1) * sa + (Ha - 1) * ha + D) * size <= pb or pb + ((Tb - 1) * sb + (Hb - 1) * hb + D) * size <= pa:
        return True
    if (pb - pa) % size:
        return False
    off = (pb - pa) // size
    # counts and strides of the outer and the inner axis of each
    for na, sa, ma, ra, nb, sb, mb, rb in ((Ta, sa, Ha, ha, Tb, sb, Hb, hb), (Ha, ha, Ta, sa, Hb, hb, Tb, sb)):
        # beside: of every s places a's inner axis takes the first, b's others
        s = sa if na > 1 else sb if nb > 1 else 0
        if s and (na == 1 or sa == s) and (nb == 1 or sb == s) and (ma - 1) * ra + D <= off % s <= s - (mb - 1) * rb - D:
            return True
        # in turn: of every r places a has the first D and b those from off % r on
        r = ra if ma > 1 else rb if mb > 1 else 0
        if r and (ma == 1 or ra == r) and (mb == 1 or rb == r) and (na == 1 or sa % r == 0) and (nb == 1 or sb % r == 0) and \
                D <= off % r <= r - D:
            return True
    return False


def _outputs_apart(q, k, q_out, k_out, more) -> None:
    """Outputs that the caller gave lie in their own input's place or touch no input, nor one another."""
    inputs = (q, k, *more)
    for own, (o, name) in enumerate(((q_out, "q_out"), (k_out, "k_out"))):
        if o is None:
            continue
        if not _heads_apart(o):
            raise ValueError(f"the heads of {name} overlap one another")
        for i, x in enumerate(inputs):  # by place: one tensor may be both q and k
            if x is not None and not (i == own and x.data_ptr() == o.data_ptr() and x.stride() == o.stride()) and \
                    not _rows_apart(o, x):
                raise ValueError(f"{name} must be {name[0]} itself or apart from q, k and v, which it may overlap")
    if k_out is not None and q_out is not None and not _rows_apart(q_out, k_out):
        raise ValueError("q_out and k_out must be apart")


_DENSE = torch.contiguous_format
_LEAST_EPS = 2.0 ** -250  # below, a head of zeros would have an infinite 1 / sqrt(eps) in f32


def _rope(q, k, positions, inv_freq, interleaved, scale, q_norm, k_norm, eps, q_out, k_out, stream, more, keys):
    """The checks that rope and rope_append share; (struct, stream, q_out, k_out).  more: further
    inputs of q's type; keys: k_out is wanted whether it was given or not."""
    # a check that holds costs half of _want's call: what does not pass here is named there
    if q.dtype is not torch.bfloat16 or not q.is_cuda or q.dim() != 3 or q.stride(2) != 1:
        _want(q, "q", torch.bfloat16, (None, None, None), dense=False)
    T, H, D = q.shape
    _head_dim(D)
    if H < 1:
        raise ValueError("q must have a head or more")
    Hk = 0
    if k is not None:
        shape = k.shape
        if k.dtype is not torch.bfloat16 or not k.is_cuda or len(shape) != 3 or shape[0] != T or shape[2] != D or \
                k.stride(2) != 1:
            _want(k, "k", torch.bfloat16, (T, None, D), dense=False)
        Hk = shape[1]
    elif k_norm is not None or k_out is not None:
        raise ValueError("k_norm and k_out need k")
    if positions.dtype is not torch.int32 or not positions.is_cuda or positions.shape != (T,) or \
            not positions.is_contiguous():
        _want(positions, "positions", torch.int32, (T,))
    if inv_freq.dtype is not torch.float32 or not inv_freq.is_cuda or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        _want(inv_freq, "inv_freq", torch.float32, (None,))
    half = inv_freq.shape[0]
    if half > D // 2:
        raise ValueError(f"inv_freq must have {D // 2} frequencies or fewer, not {half}")
    for w, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if w is not None:
            _want(w, name, torch.float32, (D,))
            _want16(w, name)
    if not (eps >= _LEAST_EPS and math.isfinite(eps) and math.isfinite(scale)):
        raise ValueError(f"eps must be 2^-250 or more and scale finite, not {eps} and {scale}")
    if q_out is not None or k_out is not None:
        for o, shape, name in ((q_out, (T, H, D), "q_out"), (k_out, (T, Hk, D), "k_out")):
            if o is not None:
                _want(o, name, torch.bfloat16, shape, dense=False)
        _outputs_apart(q, k, q_out, k_out, more)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=_DENSE) if stream is None else \
            _empty(q, (T, H, D), torch.bfloat16, stream)
    if k_out is None and keys and k is not None:
        k_out = torch.empty_like(k, memory_format=_DENSE) if stream is None else \
            _empty(q, (T, Hk, D), torch.bfloat16, stream)
    dev = q.get_device()
    if stream is None and q_norm is None and k_norm is None and (k is None or k.get_device() == dev) and \
            positions.get_device() == dev and inv_freq.get_device() == dev and q_out.get_device() == dev and \
            (k_out is None or k_out.get_device() == dev) and dev == torch.cuda.current_device():
        raw = torch._C._cuda_getCurrentRawStream(dev)
    else:
        raw = _raw(q, stream, k, positions, inv_freq, q_norm, k_norm, q_out, k_out)
    qs, os = q.stride(), q_out.stride()
    ks = (0, 0) if k is None else k.stride()
    kos = (0, 0) if k_out is None else k_out.stride()
    a = _pack_rope(q.data_ptr(), 0 if k is None else k.data_ptr(), q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
                   positions.data_ptr(), inv_freq.data_ptr(), 0 if q_norm is None else q_norm.data_ptr(),
                   0 if k_norm is None else k_norm.data_ptr(), qs[0], qs[1], ks[0], ks[1], os[0], os[1], kos[0], kos[1],
                   scale, eps, T, H, Hk, D, half, 1 if interleaved else 0)
    return a, raw, q_out, k_out


def rope(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
         interleaved: bool = False, scale: float = 1.0, q_norm: Optional[torch.Tensor] = None,
         k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None,
         k_out: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(q_out, k_out): q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] BF16 (any strides,
    last dimension contiguous; k may be None) rotated by positions [tokens] int32.

    inv_freq [half] f32 (rope_freqs): 2 * half <= head_dim values of a head are rotated, the pairs (i, i +
    half), or (2i, 2i + 1) with interleaved, by position * inv_freq[i]; the others stay.  scale multiplies cos
    and sin.  q_norm, k_norm [head_dim] f32: each head is divided by sqrt(mean of squares + eps) and
    multiplied by these first.  q_out may be q itself and k_out k (any other overlap
    with an input or one another is refused); left out, they are new and contiguous."""
    a, raw, q_out, k_out = _rope(q, k, positions, inv_freq, interleaved, scale, q_norm, k_norm, eps, q_out, k_out, stream,
                                 (), True)
    _check(_c().rope(a, raw), "glint_rope_stream")
    return q_out, k_out


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
        self.device = k_code.get_device()
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


def rope_append(cache: KV4Cache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                inv_freq: torch.Tensor, slots: torch.Tensor, *, interleaved: bool = False, scale: float = 1.0,
                q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """rope(q, k, ...), then kv4_append(cache, the rotated k, v, slots), in one pass: the same q_out (which is
    returned) and the same bytes in the cache.  The rotated keys go to the cache alone unless k_out is given (k
    itself, or a tensor of k's shape), as a prompt's attention wants them.  A token whose slot is
    negative is rotated and not cached; no slot twice in one call."""
    shape = k.shape
    if len(shape) != 3 or shape[1] != cache.kv_heads or shape[2] != cache.head_dim:
        _want(k, "k", torch.bfloat16, (None, cache.kv_heads, cache.head_dim), dense=False)
    if v.dtype is not torch.bfloat16 or not v.is_cuda or v.shape != shape or v.stride(2) != 1:
        _want(v, "v", torch.bfloat16, shape, dense=False)
    if slots.dtype is not torch.int32 or not slots.is_cuda or slots.shape != shape[:1] or not slots.is_contiguous():
        _want(slots, "slots", torch.int32, shape[:1])
    a, raw, q_out, _ = _rope(q, k, positions, inv_freq, interleaved, scale, q_norm, k_norm, eps, q_out, k_out, stream,
                             (v,), False)
    if slots.get_device() != cache.device or v.get_device() != cache.device or q.get_device() != cache.device:
        raise ValueError("q, k, v, slots and the cache must be on one device")
    vs = v.stride()
    _check(_c().rope_append(cache._c, a, v.data_ptr(), vs[0], vs[1], slots.data_ptr(), raw), "glint_kv4_rope_append_stream")
    return q_out


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
