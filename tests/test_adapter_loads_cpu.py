"""The adapter's and the clipping's kernels are resident before the launch that writes their inputs
has completed (programmatic dependent launch), so none of them may read global memory through a path
that assumes it unchanged for the kernel's lifetime."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xvec_b200", "csrc")
# Files with kernels that launch_pdl starts, and what they share.
FILES = sorted(f for f in os.listdir(CSRC) if f.startswith("adapter") or f == "clip.cu")


def code(name):
    """The file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def test_every_file_with_early_launches_is_looked_at():
    users = sorted(f for f in os.listdir(CSRC)
                   if f.endswith((".cu", ".cuh")) and "launch_pdl" in code(f))
    assert users and set(users) <= set(FILES)


@pytest.mark.parametrize("name", FILES)
def test_no_non_coherent_loads(name):
    """Neither by name nor by a qualifier that lets the compiler choose them."""
    assert not re.findall(r"__ldg|__ldcs|__ldlu|ld\.global\.nc|__restrict__|__restrict\b", code(name))


@pytest.mark.parametrize("name", [f for f in FILES if f.endswith((".cu", ".cuh"))])
def test_kernels_wait_before_they_touch_memory(name):
    """Every kernel's first statement is the wait; the product's kernel, whose set-up touches shared and
    tensor memory only, waits once that is done."""
    for kernel in re.findall(r"__global__.*?\n}\n", code(name), flags=re.S):
        body = kernel[kernel.index("{") + 1:]
        if "gemm_kernel" in kernel:
            before = body[:body.index("pdl_begin")]
            assert "p.partial" not in before and "load_box" not in before and "column_sums" not in before
        else:
            assert body.strip().startswith(("pdl_begin();", "constexpr")), kernel[:200]
            assert "pdl_begin();" in body[:120]
