"""An eps whose root has no inverse in f32 would make NaN of a head of zeros: the entry points refuse it."""
import pytest

torch = pytest.importorskip("torch")

from test_rope_host import lib, structs  # noqa: E402,F401


@pytest.mark.parametrize("eps,rc", [(2.0 ** -250, 0), (1e-30, 0), (2.0 ** -251, -1), (1e-80, -1), (1e-300, -1), (0.0, -1), (-1.0, -1)])
def test_least_eps(lib, eps, rc):  # noqa: F811
    _, p, cache, a = structs(eps=eps, tokens=0)
    assert lib.glint_rope_stream(a, None) == rc
    assert lib.glint_kv4_rope_append_stream(cache, a, p, 8, 8, p, None) == rc
