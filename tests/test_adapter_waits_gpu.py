"""Device-side waits that run out (a bound of 1 ns) in the kernels of long sums and in backward calls,
whose two products run side by side: the status is set, the device stays usable, and the same call is
right afterwards."""
import pytest
import torch

from adapter_cases import STORAGE, TYPES, Maker, ptr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def expire(xb, call, outs, status):
    """The call as it should be, then expired, then as it should be again."""
    call()
    want = [t.clone() for t in outs]
    torch.cuda.synchronize()
    assert status.item() == 0
    xb.set_wait_limit_ns(1)
    try:
        call()
        torch.cuda.synchronize()
        assert status.item() == 4  # XVEC_GPU_TIMEOUT
    finally:
        xb.set_wait_limit_ns(0)
    status.zero_()
    call()
    torch.cuda.synchronize()
    assert status.item() == 0 and all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [100, 9472])  # single CTAs or split depths, pairs
def test_long_sums(xb, kind, n):
    k, m = 8200, 1000
    mk = Maker(kind, 1)
    x, w = mk.matrix(n, k).contiguous(), mk.matrix(m, k, k ** -0.5).contiguous()
    y = torch.empty(n, m, device="cuda", dtype=x.dtype)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    expire(xb, lambda: xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y),
                                        status_ptr=ptr(status), stream=stream()), [y], status)


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients(xb, kind):
    n, k, m = 12_000, 512, 2304
    mk = Maker(kind, 2)
    x, wg, wu = (mk.matrix(*s).contiguous() for s in ((n, k), (m, k), (m, k)))
    dh, g, u = (mk.matrix(n, m).contiguous() for _ in range(3))
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    expire(xb, lambda: xb.gated_backward_device(
        0, STORAGE[kind], n, k, m, ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g), ptr(u), dx_ptr=ptr(dx),
        dgate_weight_ptr=ptr(dwg), dup_weight_ptr=ptr(dwu), status_ptr=ptr(status), stream=stream()),
        [dx, dwg, dwu], status)
