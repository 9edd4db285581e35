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


def test_waits_for_tensor_memory_name_the_registers():
    """A wait for tcgen05.ld that names no register lets arithmetic on the loaded values move ahead of it."""
    text = source("htile_gemm.cu")
    calls = re.findall(r"(tmem_ld16|tmem_ld32|tmem_ld_wait)\s*\(([^;{]*)\)\s*;", text)
    assert len([c for c in calls if c[0] == "tmem_ld_wait"]) >= 6
    waiting = None
    for name, args in calls:
        last = args.split(",")[-1].strip()
        if name == "tmem_ld_wait":
            assert waiting and last == waiting, (name, args, waiting)
            waiting = None
        else:
            assert waiting is None, (name, args)
            waiting = last
    assert waiting is None
    for m in re.finditer(r"tcgen05\.wait::ld[^;]*;\"\s*:([^:]*):", text):
        assert '"+r"' in m.group(1), m.group(0)


def test_pairs_are_counted_behind_the_kernels_own_limit():
    """max_pairs(): a kernel's shared memory limit is raised before the device is asked how many fit, each kernel is
    asked about itself, and a guess is not kept for the calls that follow."""
    text = source("htile_gemm.cu")
    body = text[text.index("int max_pairs("):]
    body = body[:body.index("\n}\n")]
    assert body.index("ensure_smem(") < body.index("cudaOccupancyMaxActiveClusters(")
    kept = [line for line in body.splitlines() if re.search(r"cached\[dev\]\[kind\]\s*=[^=]", line)]
    assert len(kept) == 1 and body.index(kept[0]) > body.rindex("cudaGetLastError()")
    for kernel in ("htile_gemm_kernel<false>", "htile_gemm_kernel<true>", "gated_wide_kernel", "htile_gemm_precise_kernel<false>",
                   "int8_tc_kernel<false>"):
        assert kernel in body, kernel


def test_writers_of_planes_let_nobody_start_early():
    """htile (to 32 rows) and htile_gated read planes before the kernel ahead of them is done if that one lets its
    successors start early; what writes planes, scales or K-major copies of them does not."""
    early = {path.name for path in CSRC.glob("*.cu*") if "griddepcontrol.launch_dependents" in source(path.name)}
    assert early == {"attn_prompt.cu", "htile_decode.cu", "htile_gated.cu", "kv4_attn.cu"}  # none of which writes any
