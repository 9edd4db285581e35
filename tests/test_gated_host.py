"""The gated feed-forward projection's entry point without a GPU: arguments are checked before
any device work, and pack_gated's layout, which is plain indexing."""
import ctypes

import pytest

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from glint_b200 import build, device
    build.build()
    L = device.lib()
    L.glint_htile_gated_work_bytes.argtypes = [ctypes.POINTER(device.GlintHtileGated)]
    L.glint_htile_gated_work_bytes.restype = ctypes.c_int64
    L.glint_htile_gated_stream.argtypes = [ctypes.POINTER(device.GlintHtileGated), ctypes.c_void_p]
    return L


def call(**kw):
    from glint_b200 import device
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    a = device.GlintHtileGated(p, p, p, p, p, p, 4, 8, 256, 64, 0, 0)
    for n, v in kw.items():
        setattr(a, n, v)
    return buf, a


def test_arguments(lib):
    f, work = lib.glint_htile_gated_stream, lib.glint_htile_gated_work_bytes
    for kw, rc in ((dict(hole=None), -1), (dict(plug=None), -1), (dict(absmax=None), -1), (dict(x=None), -1), (dict(h=None), -1),
                   (dict(M=-1), -1), (dict(F=-1), -1), (dict(K=-1), -1), (dict(F=2 ** 30), -1), (dict(blocksize=0), -2),
                   (dict(mode=2), -1), (dict(act=2), -1), (dict(act=-1), -1), (dict(M=0), 0), (dict(F=0), 0), (dict(M=0, h=None), 0)):
        _, a = call(**kw)
        assert f(a, None) == rc, kw
    for kw in (dict(M=-1), dict(F=2 ** 30), dict(mode=5), dict(act=9), dict(blocksize=0)):
        assert work(call(**kw)[1]) == -1, kw
    assert f(None, None) == -1 and work(None) == -1
    for kw in (dict(M=32), dict(M=500, mode=0), dict(M=500, mode=1, K=64), dict(M=500, mode=1, blocksize=32), dict(M=0), dict(M=500, F=0)):
        assert work(call(**kw)[1]) == 0, kw


def test_packed_rows():
    from glint_b200 import device
    F, K = 6, 64
    gate = [torch.arange(F * K // 2, dtype=torch.int64).to(torch.uint8), torch.zeros(F * K // 2, dtype=torch.uint8), torch.arange(F).float()]
    up = [255 - gate[0], torch.ones(F * K // 2, dtype=torch.uint8), -torch.arange(F).float()]
    hole, plug, am = device.pack_gated(gate, up, F, K)
    for r in range(2 * F):
        src = (gate, up)[r % 2]
        assert torch.equal(hole.view(2 * F, -1)[r], src[0].view(F, -1)[r // 2])
        assert torch.equal(plug.view(2 * F, -1)[r], src[1].view(F, -1)[r // 2])
        assert am[r] == src[2][r // 2]
    assert [t.is_contiguous() for t in (hole, plug, am)] == [True] * 3
    for bad in (dict(K=63), dict(K=96), dict(F=5), dict(F=-1), dict(blocksize=0), dict(up=[up[0].int(), *up[1:]])):
        with pytest.raises(ValueError):
            device.pack_gated(**{**dict(gate=gate, up=up, F=F, K=K), **bad})
