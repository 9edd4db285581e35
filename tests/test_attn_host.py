"""What the serving attention operators decide on the host: refusals before any device work,
workspace sizes, and the control flow that a kernel file shares with the CPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

NATIVE = Path(__file__).resolve().parent / "native"


@pytest.fixture(scope="module")
def lib():
    from glint_b200 import attn, build
    build.build()
    return attn._lib()


@pytest.mark.parametrize("field", ["lens", "seen"])
@pytest.mark.parametrize("by", [0, 1, -1, 2, -2])
def test_evict_refuses_new_lens_in_place(lib, field, by):
    """Other heads read a sequence's lens and seen after one of them has written new_lens."""
    from glint_b200 import attn
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 15) & ~15
    cache = attn._Cache(p, p, p, p, 4, 2, 64, 128)
    at = {n: p + 256 * i for i, n in enumerate(("table", "lens", "weight", "pos", "seen", "kept", "new_lens",
                                                "weight_out", "pos_out"))}
    at["new_lens"] = at[field] + 4 * by
    ev = attn._Evict(*at.values(), 256, 3, 4, 8, 2)
    assert lib.glint_kv4_evict_stream(cache, ev, None) == -1


def test_workspaces_are_sized_for_their_device(monkeypatch):
    """Devices of different SM counts in one process: no size kept for one is used for another."""
    from glint_b200 import attn
    device = 0

    class Calls:
        def prompt_work(self, a):
            return 1000 * (device + 1)

        def attn_work(self, c, a):
            return 2000 * (device + 1)
    monkeypatch.setattr(attn, "_c", lambda: Calls())
    for f in (attn._prompt_work, attn._attn_work):
        f.cache_clear()
    try:
        for device in (0, 1, 0, 1):
            assert attn._prompt_work(device, 4, 5000, 4, 2, 128) == 1000 * (device + 1)
            assert attn._attn_work(device, 2, 64, 128, 1, 1, 4, 8, False) == 2000 * (device + 1)
    finally:
        for f in (attn._prompt_work, attn._attn_work):
            f.cache_clear()


@pytest.mark.parametrize("mode", ["loop", "alone"])
def test_no_warp_is_left_at_a_barrier(tmp_path, mode):
    """The prompt kernel's item loop where bounded waits run out in some warps of a tile and not in
    others; and that the harness sees the hang of warps that leave by themselves."""
    exe = tmp_path / "check_item_loop"
    subprocess.run(["g++", "-O1", "-std=c++17", "-pthread", "-o", str(exe), str(NATIVE / "check_item_loop.cpp")], check=True)
    r = subprocess.run([str(exe), mode], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith(f"OK {mode}"), r.stdout + r.stderr
