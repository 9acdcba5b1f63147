"""float32 through every kind of the adapter's products: modes, tile shapes, split and long depths,
the few-row kernel, packed layouts.  The values' three bfloat16 parts all count (adapter_parts.py), so a
missing or misplaced part of any operand shows in the 2-norm."""
import pytest
import torch

from adapter_cases import Maker, ld, ptr
from adapter_parts import relative, values

pytestmark = pytest.mark.gpu

# A float32 product is exact to 2^-23 of itself; sums are truncated (2^-23 of the running sum, of either
# sign, at most 48 in a row before a float32 addition in registers): sqrt(48) 2^-23 = 8e-7, and below
# 2e-7 for the additions in registers.  See test_adapter_parts_cpu.py for what this limit sees.
LIMIT = 1e-6

SHAPES = [  # n, in_dim, out_dim
    (3, 960, 200), (40, 768, 100), (150, 136, 200), (700, 960, 500), (257, 640, 513), (1537, 72, 1027),
    (10_000, 192, 576), (5000, 1111, 192), (300, 20_000, 40), (20_000, 100, 2050), (40_001, 129, 258),
    (9472, 8320, 1000), (2300, 4096, 1024),
]
LAYOUTS = [(0, 0), (8, 0), (5, 1)]  # pad, skew


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def check(got, want, name):
    error = relative(got, want)
    assert error < LIMIT, f"{name}: {error:.3g}"


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_products(xb, shape, layout):
    n, k, m = shape
    mk = Maker("fp32", 1, *layout)

    def make(rows, cols):
        t = mk.matrix(rows, cols)
        t.copy_(values(mk.gen, rows, cols))
        return t

    def signs(rows, cols):  # powers of two: a product with them keeps the parts
        t = mk.matrix(rows, cols)
        t.copy_(torch.randint(0, 2, (rows, cols), generator=mk.gen, device="cuda") * 3.0 - 2.0)
        return t

    x, w, w2 = make(n, k), make(m, k), make(m, k)
    x64, w64, v64 = x.double(), w.double(), w2.double()
    z, z2 = x64 @ w64.t(), x64 @ v64.t()

    y, _ = mk.out(n, m)
    xb.linear_device(0, 1, n, k, m, ptr(x), ptr(w), ptr(y), ldx=ld(x), ldw=ld(w), ldy=ld(y), stream=stream())
    check(y, z, "y")

    (h, _), (g, _), (u, _) = mk.out(n, m), mk.out(n, m), mk.out(n, m)
    xb.gated_device(0, 1, n, k, m, ptr(x), ptr(w), ptr(w2), ptr(h), gate_ptr=ptr(g), up_ptr=ptr(u),
                    activation=xb.ACT_NONE, ldx=ld(x), ldw=ld(w), ldh=ld(h), ldg=ld(g), stream=stream())
    for got, want, name in ((g, z, "gate"), (u, z2, "up")):
        check(got, want, name)
    # (Its factors' errors add up, largest where a factor is small and the other is not.)
    assert relative(h, z * z2) < 2 * LIMIT
    del h, g, u, z, z2

    dy = make(n, m)
    d64 = dy.double()
    (dx, _), (dw, _), (dw2, _) = mk.out(n, k), mk.out(m, k), mk.out(m, k)
    xb.linear_backward_device(0, 1, n, k, m, ptr(dy), ptr(x), ptr(w), dx_ptr=ptr(dx), dw_ptr=ptr(dw),
                              lddy=ld(dy), ldx=ld(x), ldw=ld(w), lddx=ld(dx), lddw=ld(dw), stream=stream())
    check(dx, d64 @ w64, "dx")
    check(dw, d64.t() @ x64, "dw")

    gate, up = signs(n, m), signs(n, m)
    for t in (dx, dw):
        t.fill_(float("nan"))
    xb.gated_backward_device(0, 1, n, k, m, ptr(dy), ptr(x), ptr(w), ptr(w2), ptr(gate), ptr(up),
                             activation=xb.ACT_NONE, dx_ptr=ptr(dx), dgate_weight_ptr=ptr(dw),
                             dup_weight_ptr=ptr(dw2), lddh=ld(dy), ldx=ld(x), ldw=ld(w), ldg=ld(gate),
                             lddx=ld(dx), lddw=ld(dw), stream=stream())
    dg, du = d64 * up.double(), d64 * gate.double()
    check(dx, dg @ w64 + du @ v64, "dx of both")
    check(dw, dg.t() @ x64, "dwg")
    check(dw2, du.t() @ x64, "dwu")
    # The second weight's gradient alone, and dx alone.
    for t in (dx, dw2):
        t.fill_(float("nan"))
    for a, b in ((dx, None), (None, dw2)):
        xb.gated_backward_device(0, 1, n, k, m, ptr(dy), ptr(x), ptr(w), ptr(w2), ptr(gate), ptr(up),
                                 activation=xb.ACT_NONE, dx_ptr=ptr(a), dup_weight_ptr=ptr(b),
                                 lddh=ld(dy), ldx=ld(x), ldw=ld(w), ldg=ld(gate), lddx=ld(dx),
                                 lddw=ld(dw2), stream=stream())
    check(dx, dg @ w64 + du @ v64, "dx alone")
    check(dw2, du.t() @ x64, "dwu alone")


@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
def test_column_sums(xb, activation, layout):
    """dbias in float32: a thread adds at most 256 gradients in a row, their sums in four runs: below
    sqrt(256) 2^-24 = 1e-6 of the 2-norm with the activation's own 2^-21."""
    from adapter_cases import ACTS, slope
    n, m = 20_011, 301
    mk = Maker("fp32", 2, *layout)
    dy, z = mk.matrix(n, m), mk.matrix(n, m)
    db, untouched = mk.out(m)
    xb.linear_backward_device(0, 1, n, 8, m, ptr(dy), 0, 0, preact_ptr=ptr(z), activation=ACTS[activation],
                              db_ptr=ptr(db), lddy=ld(dy), ldz=ld(z), stream=stream())
    untouched()
    check(db, (dy.double() * slope(activation, z.double())).sum(0), "db")
