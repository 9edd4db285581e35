"""The gated product's plan does not depend on which operator a process ran first."""
import subprocess
import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_gated import gpu  # noqa: E402,F401

CODE = """
import sys, torch
from glint_b200 import device as D
g = torch.Generator(device="cuda").manual_seed(0)
SHAPES = [(40, 512, 100), (300, 512, 9473), (900, 256, 4700), (2311, 256, 1021)]
def planes(n, k):
    b = [torch.randint(0, 256, (n * k // 2,), device="cuda", generator=g, dtype=torch.uint8) for _ in range(2)]
    return b[0], b[1], 0.01 + 0.05 * torch.rand(n * k // 64, device="cuda", generator=g)
cases = [(torch.randn(M, K, device="cuda", generator=g).bfloat16(), planes(2 * F, K), F) for M, K, F in SHAPES]
def gated():
    for x, pl, F in cases:
        h = D.htile_gated(x, *pl, F, mode="fast")
        print(D._gated_work.__wrapped__(0, 0, x.shape[0], F, x.shape[1], 64, 1), int(h.view(torch.int16).long().sum()))
def alone():
    for x, pl, F in cases:
        y = D.htile(x, *pl, 2 * F, mode="fast")
        print(int(y.view(torch.int32).long().sum()))
for part in sys.argv[1:]:
    print(part)
    {"gated": gated, "alone": alone}[part]()
torch.cuda.synchronize()
assert D.lib().glint_kernel_error(1) == 0
"""


def test_order_of_first_calls():
    got = {}
    for order in (("gated", "alone"), ("alone", "gated")):
        out = subprocess.run([sys.executable, "-c", CODE, *order], cwd=Path(__file__).resolve().parent.parent, text=True,
                             capture_output=True, timeout=300)
        assert out.returncode == 0, out.stderr[-2000:]
        lines = out.stdout.split("\n")
        at = {part: lines.index(part) for part in order}
        for part in order:
            end = min([i for i in at.values() if i > at[part]], default=len(lines))
            got.setdefault(part, []).append([line for line in lines[at[part] + 1:end] if line])
    for part, (a, b) in got.items():
        assert a == b and len(a) == 4, part


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("M,K,F", [(1, 4096, 14336), (32, 4096, 128256), (9, 8192, 28672), (32, 12544, 384), (32, 33280, 50), (16, 256, 18001),
                                   (33, 4096, 14336), (511, 4096, 14336), (98, 6656, 174), (900, 4096, 14336), (2311, 768, 1021)])
def test_workspace_is_as_large_as_documented(M, K, F, mode):
    from glint_b200 import device
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    need = device._gated_work.__wrapped__(0, 0, M, F, K, 64, mode)
    copies = 2 * M * K + 8 * F + 1024 if mode else 0  # x in FP16, scales of its rows
    if mode and M > 32:
        copies += 8 * F
    if mode and M > 768 and need > 4 * F * K:
        copies += 4 * F * K
    sums = 780 * F if 2 * F > 224 * sms else 10e6
    if M > 32:
        sums = 39e6 if mode else 0
    assert need <= copies + sums + 64 * 1024, (need, copies, sums)
