"""Rules of the gated product's kernels that no run shows, held in their sources."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "glint_b200" / "csrc"


def source(name):
    text = (CSRC / name).read_text()
    return re.sub(r"/\*.*?\*/|//[^\n]*", " ", text, flags=re.S)


def test_scales_are_not_read_as_constant():
    """x_scale and row_scale are written by gated_prep_kernel while the product's kernel is resident: the read-only
    path is for data that nobody writes during a kernel's life."""
    for path in sorted(CSRC.glob("*.cu")) + sorted(CSRC.glob("*.cuh")):
        text = source(path.name)
        for m in re.finditer(r"(__ldg|ld\.global\.nc)\s*\(", text):
            depth, at = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[at], 0)
                at += 1
            assert not re.search(r"x_scale|row_scale", text[m.end():at]), f"{path.name}: {text[m.start():at]}"
        assert not re.search(r"__restrict__\s+(x_scale|row_scale)", text), path.name
