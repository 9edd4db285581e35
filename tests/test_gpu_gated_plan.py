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
