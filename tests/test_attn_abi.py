"""The serving attention entry points (include/glint_attn.h) without a GPU: arguments are
checked before any device work."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from glint_b200 import attn, build
    build.build()
    return attn._lib()


def structs():
    from glint_b200 import attn
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    cache = attn._Cache(p, p, p, p, 4, 2, 64, 128)
    prompt = attn._Prompt(*[p] * 7, None, *[8] * 8, 1, 4, 4, 4, 2, 128, 1, 1.0)
    at = attn._Attn(p, p, p, p, p, None, None, p, 8, 8, 8, 256, 1, 1, 4, 4, 1.0)
    ev = attn._Evict(p, p, p, p, p, p, p, p + 16, p + 16, 256, 1, 4, 8, 2)
    return buf, p, cache, prompt, at, ev


def put(s, **kw):
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def test_prompt_arguments(lib):
    f = lib.glint_attn_prompt_stream
    for kw, rc in ((dict(q=None), -1), (dict(o=None), -1), (dict(cu_q=None), -1), (dict(k=None), -1),
                   (dict(seqs=-1), -1), (dict(q_tokens=-1), -1), (dict(heads=3), -1), (dict(heads=0), -1),
                   (dict(kv_heads=0), -1), (dict(head_dim=96), -6), (dict(seqs=0), 0), (dict(q_tokens=0), 0)):
        buf, p, _, prompt, _, _ = structs()
        assert f(put(prompt, **kw), None) == rc, kw
    assert f(None, None) == -1
    buf, p, _, prompt, _, _ = structs()
    assert f(put(prompt, work=p + 8), None) == -1
    assert lib.glint_attn_prompt_work_bytes(put(prompt, head_dim=96)) == -6
    assert lib.glint_attn_prompt_work_bytes(None) == -1
    assert lib.glint_attn_prompt_work_bytes(put(prompt, head_dim=128, q_tokens=10 ** 6)) == 0


def test_cache_arguments(lib):
    for kw, rc in ((dict(k_code=None), -1), (dict(pages=0), -1), (dict(kv_heads=0), -1), (dict(page_size=48), -6),
                   (dict(head_dim=80), -6), (dict(pages=2 ** 30), -1)):
        buf, p, cache, _, at, ev = structs()
        put(cache, **kw)
        assert lib.glint_kv4_append_stream(cache, p, p, 8, 8, 8, 8, p, 1, None) == rc, kw
        assert lib.glint_kv4_read_stream(cache, p, 1, p, p, None) == rc, kw
        assert lib.glint_kv4_attn_stream(cache, at, None) == rc, kw
        assert lib.glint_kv4_evict_stream(cache, ev, None) == rc, kw
    buf, p, cache, _, at, ev = structs()
    cache.k_code = p + 8
    assert lib.glint_kv4_append_stream(cache, p, p, 8, 8, 8, 8, p, 1, None) == -1
    buf, p, cache, _, at, ev = structs()
    assert lib.glint_kv4_append_stream(cache, p, p, 8, 8, 8, 8, p, -1, None) == -1
    assert lib.glint_kv4_append_stream(cache, None, p, 8, 8, 8, 8, p, 1, None) == -1
    assert lib.glint_kv4_append_stream(cache, None, None, 8, 8, 8, 8, None, 0, None) == 0
    assert lib.glint_kv4_read_stream(cache, p, 1, p + 2, p, None) == -1
    assert lib.glint_kv4_read_stream(cache, None, 0, None, None, None) == 0
    assert lib.glint_kv4_append_stream(None, p, p, 8, 8, 8, 8, p, 1, None) == -1


def test_attn_arguments(lib):
    f = lib.glint_kv4_attn_stream
    for kw, rc in ((dict(q=None), -1), (dict(o=None), -1), (dict(table=None), -1), (dict(lens=None), -1),
                   (dict(work=None), -1), (dict(rows=0), -1), (dict(rows=129), -1), (dict(heads=3), -1), (dict(max_pages=0), -1),
                   (dict(seqs=-1), -1), (dict(seqs=0), 0)):
        buf, p, cache, _, at, _ = structs()
        assert f(cache, put(at, **kw), None) == rc, kw
    buf, p, cache, _, at, _ = structs()
    assert f(cache, put(at, weight_out=p, weight_stride=255), None) == -1            # weights too short
    more = lib.glint_kv4_attn_work_bytes(cache, at)
    assert more > lib.glint_kv4_attn_work_bytes(cache, put(at, weight_out=None)) > 0
    assert f(cache, put(at, work=p + 8), None) == -1
    assert f(cache, put(at, work=p, o=p + 8), None) == -1
    assert f(cache, None, None) == -1


def test_evict_arguments(lib):
    f = lib.glint_kv4_evict_stream
    for kw, rc in ((dict(table=None), -1), (dict(seen=None), -1), (dict(kept=None), -1), (dict(budget=0), -1),
                   (dict(recent=9), -1), (dict(recent=-1), -1), (dict(stride=255), -1), (dict(max_pages=0), -1),
                   (dict(max_pages=8193, stride=2 ** 20), -1), (dict(seqs=0), 0)):
        buf, p, cache, _, _, ev = structs()
        assert f(cache, put(ev, **kw), None) == rc, kw
    buf, p, cache, _, _, ev = structs()
    assert f(cache, put(ev, weight_out=p), None) == -1
    assert f(cache, None, None) == -1


def test_python_refuses_cpu_tensors():
    from glint_b200 import attn
    q = torch.zeros(4, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attn.attn_prompt(q, q, q, torch.tensor([0, 4], dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        attn.KV4Cache.empty(2, 2, 128, 16, device="cpu")
