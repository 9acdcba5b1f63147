"""Binary16 backward passes whose pre-activation gradients lie outside binary16's range while the
results do not: the gradients are products of two or three stored values."""
import math

import pytest
import torch

from adapter_cases import ACTS, Maker, act, close, half_step, ptr, slope

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# Independent roundings of the pre-activation gradients and of the results to binary16, each of an rms
# below its half step 2^-11, and float32 sums that are far better: sqrt(2) 2^-11 < 2^-10.
BOUND = 2.0 ** -10

# sizes of dh, up (and gate), weights, x
SCALES = {"large": (300.0, 300.0, 2.0 ** -12, 2.0 ** -12), "ordinary": (1.0, 1.0, 1.0, 1.0),
          "small": (2.0 ** -13, 2.0 ** -10, 2.0 ** 10, 2.0 ** 10), "tiny": (2.0 ** -14, 2.0 ** -14, 2.0 ** 15, 2.0 ** 15)}


def make(mk, rows, cols, scale):
    return (mk.matrix(rows, cols).float().clamp(-3.5, 3.5) * scale).half().contiguous()


@pytest.mark.parametrize("scale", list(SCALES))
@pytest.mark.parametrize("shape", [(1021, 72, 130), (40_000, 64, 96), (5, 200, 40), (3000, 1000, 768)],
                         ids=str)
def test_gated(xb, shape, scale):
    n, k, m = shape
    sdh, sup, sw, sx = SCALES[scale]
    mk = Maker("fp16", 1)
    dh, u, g = make(mk, n, m, sdh), make(mk, n, m, sup), make(mk, n, m, min(sup, 4.0))
    wg, wu, x = make(mk, m, k, sw * m ** -0.5), make(mk, m, k, sw * m ** -0.5), make(mk, n, k, sx * n ** -0.5)
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu)
    dbg, dbu = (torch.empty(m, device="cuda", dtype=torch.float16) for _ in range(2))
    for parts in ("all", "dx", "weights", "up"):
        a, b, c = ({"all": (dx, dwg, dwu), "dx": (dx, None, None), "weights": (None, dwg, dwu),
                    "up": (None, None, dwu)}[parts])
        for t in (dx, dwg, dwu):
            t.fill_(math.nan)
        xb.gated_backward_device(0, 2, n, k, m, ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g), ptr(u),
                                 activation=xb.ACT_SILU, dx_ptr=ptr(a), dgate_weight_ptr=ptr(b),
                                 dup_weight_ptr=ptr(c), dgate_bias_ptr=ptr(dbg), dup_bias_ptr=ptr(dbu),
                                 stream=stream())
        d, z, v = dh.double(), g.double(), u.double()
        dg, du = d * v * slope("silu", z), d * act("silu", z)
        if a is not None:
            assert relative(dx, dg @ wg.double() + du @ wu.double()) < BOUND
        # (The two weights' gradients differ in size: with large values only the gate's leave the range.)
        if b is not None:
            assert relative(dwg, dg.t() @ x.double()) < BOUND
        if c is not None:
            # Values 2^-40 below the largest gradient are lost; here du is at most 300 times smaller.
            assert relative(dwu, du.t() @ x.double()) < BOUND


@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("scale", [18000.0, 1.0, 2.0 ** -12, 2.0 ** -20])
def test_linear(xb, activation, scale):
    """Incoming gradients up to 3.5 x 18000 = 63000, which a slope of up to 1.13 brings above 65504."""
    n, k, m = 1500, 136, 200
    mk = Maker("fp16", 2)
    dy, z = make(mk, n, m, scale), make(mk, n, m, 1.0)
    back = 1 / scale if scale >= 1 else min(2.0 ** 12, 1 / scale)
    w, x = make(mk, m, k, back * m ** -0.5), make(mk, n, k, back * n ** -0.5)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    xb.linear_backward_device(0, 2, n, k, m, ptr(dy), ptr(x), ptr(w), preact_ptr=ptr(z),
                              activation=ACTS[activation], dx_ptr=ptr(dx), dw_ptr=ptr(dw), stream=stream())
    d = dy.double() * slope(activation, z.double())
    # (dy itself may be subnormal: it is exact, whatever it holds.)  A result below the normal range
    # moves by 2^-25.
    for got, want in ((dx, d @ w.double()), (dw, d.t() @ x.double())):
        err = (got.double() - want).norm().item()
        assert err < BOUND * want.norm().item() + 2.0 ** -25 * math.sqrt(want.numel())


def test_values_that_are_not_finite_stay_in_their_rows(xb):
    """An infinity or a NaN among the incoming gradients does not decide how the others are held."""
    n, k, m = 300, 64, 72
    mk = Maker("fp16", 3)
    for scale in (1.0, 2.0 ** -12):
        dy, z = make(mk, n, m, scale), make(mk, n, m, 1.0)
        w = make(mk, m, k, 1.0)
        dy[7, 5], dy[11, 3] = math.inf, math.nan
        z[7, 5] = 1.0
        dx = torch.empty(n, k, device="cuda", dtype=torch.float16)
        xb.linear_backward_device(0, 2, n, k, m, ptr(dy), 0, ptr(w), preact_ptr=ptr(z),
                                  activation=xb.ACT_GELU, dx_ptr=ptr(dx), stream=stream())
        bad = torch.zeros(n, dtype=torch.bool, device="cuda")
        bad[7] = bad[11] = True
        assert bool((torch.isfinite(dx).all(1) == ~bad).all())
        d = dy.double() * slope("gelu", z.double())
        want = (d @ w.double())[~bad]
        err = (dx[~bad].double() - want).norm() / want.norm()
        assert err.item() < BOUND


def test_zero_gradients(xb):
    n, k, m = 100, 64, 72
    z = torch.randn(n, m, device="cuda").half()
    w, dy = torch.randn(m, k, device="cuda").half(), torch.zeros(n, m, device="cuda").half()
    dx = torch.full((n, k), math.nan, device="cuda").half()
    xb.linear_backward_device(0, 2, n, k, m, ptr(dy), 0, ptr(w), preact_ptr=ptr(z),
                              activation=xb.ACT_GELU, dx_ptr=ptr(dx), stream=stream())
    assert bool((dx == 0).all())


def test_captured_and_replayed_with_other_sizes_of_gradients(xb):
    """The decision is the device's: a captured call follows the values that it is replayed on."""
    n, k, m = 500, 64, 96
    mk = Maker("fp16", 4)
    z, w, x = make(mk, n, m, 1.0), make(mk, m, k, 0.1), make(mk, n, k, 0.1)
    dy = make(mk, n, m, 1.0)
    dx, dw = torch.empty_like(x), torch.empty_like(w)

    def call():
        xb.linear_backward_device(0, 2, n, k, m, ptr(dy), ptr(x), ptr(w), preact_ptr=ptr(z),
                                  activation=xb.ACT_SILU, dx_ptr=ptr(dx), dw_ptr=ptr(dw),
                                  stream=stream())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for scale in (1.0, 2.0 ** -14, 2.0 ** 12, 2.0 ** -18, 1.0):
        dy.copy_(make(mk, n, m, scale))
        graph.replay()
        torch.cuda.synchronize()
        got = dx.clone(), dw.clone()
        call()
        assert torch.equal(dx, got[0]) and torch.equal(dw, got[1])
        d = dy.double() * slope("silu", z.double())
        want = d @ w.double()
        err = (got[0].double() - want).norm().item()
        assert err < BOUND * want.norm().item() + 2.0 ** -25 * math.sqrt(want.numel())
    del graph
