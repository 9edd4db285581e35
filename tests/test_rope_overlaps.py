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
