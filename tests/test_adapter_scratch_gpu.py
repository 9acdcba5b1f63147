"""The adapter's scratch: it comes from a pool of the library's own, what stays of it between calls is
bounded, and it can be given back."""
import os
import subprocess
import sys

import pytest
import torch

from adapter_cases import ptr

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
GIB = 1 << 30

# In a process of its own, since creating an index sets the default pool up for its searches.
DEFAULT_POOL = """
import sys, torch
sys.path[:0] = [{root!r}]
import xvec_b200 as xb
from cuda.bindings import runtime as rt, driver as dr
torch.zeros(1, device="cuda")
err, pool = rt.cudaDeviceGetDefaultMemPool(0)
attr = rt.cudaMemPoolAttr.cudaMemPoolAttrReleaseThreshold
assert rt.cudaMemPoolSetAttribute(pool, attr, dr.cuuint64_t(12345))[0] == 0
n, k, m = 1000, 96, 128
x, w = torch.randn(n, k, device="cuda"), torch.randn(m, k, device="cuda")
y, dw, norm = torch.empty(n, m, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty((), device="cuda")
s = torch.cuda.current_stream().cuda_stream
xb.linear_device(0, 1, n, k, m, x.data_ptr(), w.data_ptr(), y.data_ptr(), stream=s)
xb.linear_backward_device(0, 1, n, k, m, y.data_ptr(), x.data_ptr(), w.data_ptr(), dw_ptr=dw.data_ptr(), stream=s)
xb.clip_gradients_device(0, [(1, dw.data_ptr(), dw.data_ptr(), dw.numel())], 1.0, norm.data_ptr(), stream=s)
torch.cuda.synchronize()
err, kept = rt.cudaMemPoolGetAttribute(pool, attr)
assert err == 0 and int(kept) == 12345, kept
print("kept")
"""


def test_default_pool_stays_as_the_caller_set_it_up():
    p = subprocess.run([sys.executable, "-c", DEFAULT_POOL.format(root=ROOT)], capture_output=True,
                       text=True, timeout=300)
    assert p.returncode == 0 and "kept" in p.stdout, p.stderr[-2000:]


def test_kept_scratch_is_bounded_and_can_be_given_back():
    import xvec_b200 as xb
    n, most, k, m = 200_000, 1_000_000, 1024, 2048
    x, dy = torch.zeros(most, k, device="cuda"), torch.zeros(most, m, device="cuda")
    w, dw = torch.zeros(m, k, device="cuda"), torch.empty(m, k, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def call(rows):  # 6 bytes for each element of x and dy: 3.4 and 17.2 GiB
        xb.linear_backward_device(0, 1, rows, k, m, ptr(dy), ptr(x), ptr(w), dw_ptr=ptr(dw),
                                  stream=stream)

    def missing():
        torch.cuda.synchronize()
        return before - torch.cuda.mem_get_info()[0]

    def trim():  # (what an enqueued call still uses stays)
        torch.cuda.synchronize()
        xb.trim_scratch(0)

    call(1000)
    trim()
    before = torch.cuda.mem_get_info()[0]
    call(n)
    assert 3 * GIB < missing() < 4.5 * GIB  # kept for the next call
    call(n)
    trim()
    assert missing() < GIB // 4
    # Two calls at once on two streams need more than 20 GiB; no more than 16 of it stay.
    other, dw2 = torch.cuda.Stream(), torch.empty_like(dw)
    other.wait_stream(torch.cuda.current_stream())
    call(most)
    xb.linear_backward_device(0, 1, n, k, m, ptr(dy), ptr(x), ptr(w), dw_ptr=ptr(dw2),
                              stream=other.cuda_stream)
    assert missing() < 16.5 * GIB
    trim()
    assert missing() < GIB // 4


def test_trimming_without_calls_and_between_calls_that_run():
    import xvec_b200 as xb
    xb.trim_scratch(0)
    n, k, m = 5000, 512, 512
    x, w = torch.randn(n, k, device="cuda"), torch.randn(m, k, device="cuda")
    want, y = torch.empty(n, m, device="cuda"), torch.empty(n, m, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    xb.linear_device(0, 1, n, k, m, ptr(x), ptr(w), ptr(want), stream=stream)
    for _ in range(5):
        xb.linear_device(0, 1, n, k, m, ptr(x), ptr(w), ptr(y), stream=stream)
        xb.trim_scratch(0)
    assert torch.equal(y, want)
    with pytest.raises(xb.XvecGPUError):
        xb.trim_scratch(1000)
