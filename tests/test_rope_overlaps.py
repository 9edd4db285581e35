"""Which outputs rope and rope_append take: what they decide by addresses and strides, without a GPU."""
import pytest

torch = pytest.importorskip("torch")


def apart(*a):
    from glint_b200 import attn
    attn._outputs_apart(*a)


def test_one_tensor_as_queries_and_keys():
    """In place for the one is not in place for the other: the keys would be read from rows that are rotated already."""
    t, other = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, 4, 64, dtype=torch.bfloat16)
    for q, k, q_out, k_out, more in ((t, t, t, None, ()), (t, t, None, t, ()), (t, t, t, other, ()), (t, t, other, t, ()), (t, t, t, t, ()),
                                     (t, other, None, other, (other,)), (t, other, t, None, (t,)), (t, None, t, None, (t,))):
        with pytest.raises(ValueError, match="_out must be"):
            apart(q, k, q_out, k_out, more)
    apart(t, t, other, None, ())
    apart(t, t, None, other, ())
    apart(t, other, t, other, ())
    apart(t, None, t, None, ())


def places(t):
    base = t.storage_offset()
    T, H, D = t.shape
    return {base + i * t.stride(0) + h * t.stride(1) + d for i in range(T) for h in range(H) for d in range(D)}


def test_heads_in_turn():
    """A fused buffer with each head's query, key and value side by side: they share nothing, and are taken in place."""
    from glint_b200 import attn
    for T, H in ((5, 4), (1, 4), (5, 1), (1, 1)):
        y = torch.zeros(T, H, 3, 64, dtype=torch.bfloat16)
        q, k, v = (y[:, :, i] for i in range(3))
        apart(q, k, q, k, (v,))
        apart(q, k, q, None, (v,))
        apart(q, k, v, None, ())
        with pytest.raises(ValueError):
            apart(q, k, k, None, (v,))
        with pytest.raises(ValueError):
            apart(q, k, q, v, (v,))
    # groups of two queries and a key: the first queries of the groups beside the keys
    y = torch.zeros(5, 4, 3, 64, dtype=torch.bfloat16)
    assert attn._rows_apart(y[:, :, 0], y[:, :, 2]) and attn._rows_apart(y[:, ::2, 0], y[:, 1::2, 0])
    assert not attn._rows_apart(y[:, :, 0], y[:, ::2, 0]) and not attn._rows_apart(y[:, 0], y[:, :, 0])


def test_every_answer_apart_is_right():
    from glint_b200 import attn
    store = torch.zeros(400, dtype=torch.int16)
    views = [store.as_strided((T, H, 4), (st, sh, 1), off) for T in (1, 2, 3) for H in (1, 2, 3)
             for st, sh in ((24, 8), (24, 12), (12, 24), (8, 8), (20, 8), (16, 8), (0, 8), (8, 0), (36, 12), (4, 12), (7, 12))
             for off in (0, 1, 4, 8, 12, 20, 33)]
    where = [places(v) for v in views]
    said = 0
    for a, pa in zip(views, where):
        for b, pb in zip(views, where):
            if attn._rows_apart(a, b):
                said += 1
                assert not pa & pb, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert said > 10000


def test_heads_outermost():
    """[heads, 3, tokens, head_dim] and [heads, tokens, 3, head_dim] buffers, seen as [tokens, heads, head_dim]."""
    for T, H in ((5, 4), (1, 4), (5, 1)):
        for y in (torch.zeros(H, 3, T, 64, dtype=torch.bfloat16).permute(2, 0, 1, 3),
                  torch.zeros(H, T, 3, 64, dtype=torch.bfloat16).permute(1, 0, 2, 3)):
            q, k, v = (y[:, :, i] for i in range(3))
            apart(q, k, q, k, (v,))
            for bad in (k, v):
                with pytest.raises(ValueError):
                    apart(q, k, bad, None, (v,))
        y = torch.zeros(2 * H, T, 64, dtype=torch.bfloat16).transpose(0, 1)
        apart(y[:, ::2], y[:, 1::2], y[:, ::2], y[:, 1::2], ())
        apart(y[:, :H], y[:, H:], y[:, :H], y[:, H:], ())
