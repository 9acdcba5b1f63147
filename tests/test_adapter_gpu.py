"""The learned adapter's operators on the GPU against their formulas in 64 bits: every storage type,
one row to many, odd sizes, strides, offsets from alignment, saved pre-activations, values that
are not finite, streams, graphs, repeatability, and one adapter trained and then searched with."""
import math

import numpy as np
import pytest
import torch

from adapter_cases import (ACTS, SENTINEL, STORAGE, TYPES, Maker, act, close, half_step, ld, ptr,
                           rounded_terms_error, slope, sum_error)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


# Small arithmetic after the sums (bias, activation, product, residual), in float32: at most 16
# roundings or 2-ulp functions, 2^-20 of the values together.
SMALL = 2.0 ** -20
# The largest |act'| (gelu: 1.13).
STEEP = 1.13

SHAPES = [  # n, in_dim, out_dim
    (1, 1, 1), (1, 768, 768), (2, 33, 7), (3, 100, 129), (4, 1024, 2048), (5, 960, 64), (8, 64, 515),
    (9, 301, 96), (16, 128, 128), (17, 2048, 40), (31, 8, 1000), (64, 512, 256), (127, 65, 63),
    (128, 64, 128), (129, 257, 130), (300, 960, 960), (513, 31, 17), (1000, 127, 770), (2049, 768, 384),
]
LAYOUTS = [(0, 0), (8, 0), (5, 1)]  # pad, skew
# Sizes that reach every tile shape of the matrix kernel, whole and split depth, tiles whose last
# rows and columns are few, more tiles than SMs, and the borders of the few-row path.
LARGE = [
    (65, 4096, 72), (64, 1030, 4000), (66, 96, 9000), (200, 5000, 300), (257, 640, 513), (1537, 72, 1027),
    (3000, 640, 1210), (5000, 1111, 192), (10_000, 192, 576), (40_001, 129, 258), (20_000, 100, 2050),
    (300, 20_000, 40), (2300, 4096, 1024),
]


def run_linear(xb, kind, n, k, m, activation, bias, residual, save, pad=0, skew=0, seed=0):
    mk = Maker(kind, seed, pad, skew)
    x, w = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5)
    b = mk.vector(m) if bias else None
    r = mk.matrix(n, m) if residual else None
    y, y_ok = mk.out(n, m)
    z, z_ok = mk.out(n, m) if save else (None, None)
    xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y), bias_ptr=ptr(b),
                     residual_ptr=ptr(r), activation=ACTS[activation], preact_ptr=ptr(z), ldx=ld(x),
                     ldw=ld(w), ldr=ld(r), ldy=ld(y), ldz=ld(z), stream=stream())
    y_ok()
    if save:
        z_ok()
    return x, w, b, r, y, z


def check_linear(x, w, b, r, y, z, activation):
    x64, w64 = x.double(), w.double()
    want = x64 @ w64.t() + (0 if b is None else b.double())
    err = sum_error(x64, w64, want) + SMALL * want.abs()
    if z is not None:
        close(z, want, err, "preact")
    out = act(activation, want)
    err = STEEP * err + SMALL * (want.abs() + out.abs())
    if r is not None:
        out = out + r.double()
        err = err + SMALL * r.double().abs()
    close(y, out, err, "y")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(xb, kind, shape):
    i = SHAPES.index(shape)
    activation = list(ACTS)[i % 4]
    pad, skew = LAYOUTS[i % 3]
    out = run_linear(xb, kind, *shape, activation, bias=i % 2 == 0, residual=i % 3 != 1,
                     save=i % 4 != 0, pad=pad, skew=skew, seed=i)
    check_linear(*out, activation)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", LARGE, ids=str)
def test_large(xb, kind, shape):
    """Each operator at the sizes that choose other tiles."""
    i = LARGE.index(shape)
    pad, skew = LAYOUTS[i % 3]
    activation = list(ACTS)[i % 4]
    out = run_linear(xb, kind, *shape, activation, i % 2 == 0, i % 3 != 0, i % 2 == 1, pad, skew, seed=i)
    check_linear(*out, activation)
    out = run_gated(xb, kind, *shape, activation, i % 2 == 1, i % 2 == 0, pad, skew, seed=i)
    check_gated(*out, activation)
    out = run_linear_backward(xb, kind, *shape, activation, "xwb", pad, skew, seed=i)
    check_backward(kind, activation, *out)
    out = run_gated_backward(xb, kind, *shape, activation, "xgubc", pad, skew, seed=i)
    check_backward(kind, activation, *out)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 24, 33, 63, 64, 65])
def test_few_rows(xb, kind, n):
    for k, m in ((40, 3), (8, 130), (700, 257), (1500, 1000)):
        out = run_linear(xb, kind, n, k, m, "silu", True, n % 2 == 0, True, n % 3, n % 2, seed=n)
        check_linear(*out, "silu")
        out = run_gated(xb, kind, n, k, m, "gelu", n % 2 == 1, n % 2 == 0, n % 3, n % 2, seed=n)
        check_gated(*out, "gelu")


def test_leading_dimension_of_a_single_row_is_ignored(xb):
    x, w = torch.randn(1, 64, device="cuda"), torch.randn(32, 64, device="cuda")
    y, want = torch.empty(1, 32, device="cuda"), torch.empty(1, 32, device="cuda")
    xb.linear_device(0, 1, 1, 64, 32, ptr(x), ptr(w), ptr(want), stream=stream())
    xb.linear_device(0, 1, 1, 64, 32, ptr(x), ptr(w), ptr(y), ldx=1, ldy=5, stream=stream())
    assert torch.equal(y, want)


@pytest.mark.parametrize("pad,skew", LAYOUTS)
@pytest.mark.parametrize("activation", list(ACTS))
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_activations_and_layouts(xb, kind, activation, pad, skew):
    for n, k, m in ((6, 72, 40), (150, 136, 200)):
        out = run_linear(xb, kind, n, k, m, activation, True, True, True, pad, skew, seed=n)
        check_linear(*out, activation)


def run_gated(xb, kind, n, k, m, activation, bias, save, pad=0, skew=0, seed=0):
    mk = Maker(kind, seed, pad, skew)
    x, wg, wu = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5), mk.matrix(m, k, k ** -0.5)
    bg, bu = (mk.vector(m), mk.vector(m)) if bias else (None, None)
    h, h_ok = mk.out(n, m)
    g, g_ok = mk.out(n, m) if save else (None, None)
    u, u_ok = mk.out(n, m) if save else (None, None)
    xb.gated_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(wg), ptr(wu), ptr(h), gate_bias_ptr=ptr(bg),
                    up_bias_ptr=ptr(bu), activation=ACTS[activation], gate_ptr=ptr(g), up_ptr=ptr(u),
                    ldx=ld(x), ldw=ld(wg), ldh=ld(h), ldg=ld(g), stream=stream())
    h_ok()
    if save:
        g_ok()
        u_ok()
    return x, wg, wu, bg, bu, h, g, u


def check_gated(x, wg, wu, bg, bu, h, g, u, activation):
    x64 = x.double()
    pre, errs = [], []
    for w, b, saved, name in ((wg, bg, g, "gate"), (wu, bu, u, "up")):
        v = x64 @ w.double().t() + (0 if b is None else b.double())
        e = sum_error(x64, w.double(), v) + SMALL * v.abs()
        if saved is not None:
            close(saved, v, e, name)
        pre.append(v)
        errs.append(e)
    a = act(activation, pre[0])
    ea = STEEP * errs[0] + SMALL * (pre[0].abs() + a.abs())
    want = a * pre[1]
    err = ea * pre[1].abs() + a.abs() * errs[1] + ea * errs[1] + SMALL * want.abs()
    close(h, want, err, "h")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gated(xb, kind, shape):
    i = SHAPES.index(shape)
    activation = list(ACTS)[(i + 3) % 4]
    pad, skew = LAYOUTS[i % 3]
    out = run_gated(xb, kind, *shape, activation, bias=i % 2 == 0, save=i % 3 != 0, pad=pad, skew=skew,
                    seed=i)
    check_gated(*out, activation)


def slopes64(activation, dy, pre):
    if len(pre) == 1:
        return [dy * slope(activation, pre[0])]
    return [dy * pre[1] * slope(activation, pre[0]), dy * act(activation, pre[0])]


def check_backward(kind, activation, dy, x, ws, pre, dx, dws, dbs):
    """ws, pre, dws, dbs: one of each (linear) or two (gated)."""
    dtype = TYPES[kind]
    x64 = x.double()
    d64 = slopes64(activation, dy.double(), [p.double() for p in pre])
    # 16-bit storage multiplies pre-activation gradients rounded to it (linear without an
    # activation: dy itself, exact).
    rounded = kind != "fp32" and (activation != "none" or len(pre) == 2)

    # act' is a sum of terms of either sign up to STEEP (gelu' and silu' pass through zero near
    # z = -0.75 and -1.28), so float32 leaves an absolute error below 2^-20 of |dy| (times |up|) in the
    # pre-activation gradient, however small the gradient itself is; likewise 2^-20 |gate| in act.
    size = [dy.double().abs()]
    if len(pre) == 2:
        g, u = (p.double().abs() for p in pre)
        size = [size[0] * u, size[0] * g]

    def product_error(a, b, size):
        e = sum_error(a, b) + SMALL * (size @ b.abs().t())
        return e + rounded_terms_error(a, b, dtype) if rounded else e

    if dx is not None:
        want = sum(d @ w.double() for d, w in zip(d64, ws))
        err = sum(product_error(d, w.double().t(), q) for d, w, q in zip(d64, ws, size))
        close(dx, want, err, "dx")
    for i, (d, dw, db, q) in enumerate(zip(d64, dws, dbs, size)):
        if dw is not None:
            close(dw, d.t() @ x64, product_error(d.t(), x64.t(), q.t()), f"dw{i}")
        if db is not None:
            ones = torch.ones(1, d.shape[0], dtype=torch.float64, device=d.device)
            err = sum_error(d.t(), ones)[:, 0] + SMALL * q.sum(0)
            close(db, d.sum(0), err, f"db{i}")


def run_linear_backward(xb, kind, n, k, m, activation, want, pad=0, skew=0, seed=0):
    mk = Maker(kind, seed, pad, skew)
    x, w = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5)
    dy, z = mk.matrix(n, m), mk.matrix(n, m)
    dx, dx_ok = mk.out(n, k) if "x" in want else (None, lambda: 0)
    dw, dw_ok = mk.out(m, k) if "w" in want else (None, lambda: 0)
    db, db_ok = mk.out(m) if "b" in want else (None, lambda: 0)
    xb.linear_backward_device(0, STORAGE[kind], n, k, m, ptr(dy), ptr(x), ptr(w),
                              preact_ptr=0 if activation == "none" else ptr(z),
                              activation=ACTS[activation], dx_ptr=ptr(dx), dw_ptr=ptr(dw),
                              db_ptr=ptr(db), lddy=ld(dy), ldx=ld(x), ldw=ld(w), ldz=ld(z),
                              lddx=ld(dx), lddw=ld(dw), stream=stream())
    dx_ok(), dw_ok(), db_ok()
    return dy, x, [w], [z], dx, [dw], [db]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_backward(xb, kind, shape):
    i = SHAPES.index(shape)
    activation = list(ACTS)[(i + 1) % 4]
    pad, skew = LAYOUTS[i % 3]
    want = ("xwb", "xw", "xwb", "wb", "x", "xwb", "b")[i % 7]
    out = run_linear_backward(xb, kind, *shape, activation, want, pad, skew, seed=i)
    check_backward(kind, activation, *out)


@pytest.mark.parametrize("pad,skew", LAYOUTS)
@pytest.mark.parametrize("activation", list(ACTS))
@pytest.mark.parametrize("kind", list(TYPES))
def test_linear_backward_activations_and_layouts(xb, kind, activation, pad, skew):
    for n, k, m in ((6, 72, 40), (150, 136, 200)):
        out = run_linear_backward(xb, kind, n, k, m, activation, "xwb", pad, skew, seed=n)
        check_backward(kind, activation, *out)


def run_gated_backward(xb, kind, n, k, m, activation, want, pad=0, skew=0, seed=0):
    mk = Maker(kind, seed, pad, skew)
    x, wg, wu = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5), mk.matrix(m, k, k ** -0.5)
    dh, g, u = mk.matrix(n, m), mk.matrix(n, m), mk.matrix(n, m)
    none = (None, lambda: 0)
    dx, o0 = mk.out(n, k) if "x" in want else none
    dwg, o1 = mk.out(m, k) if "g" in want else none
    dwu, o2 = mk.out(m, k) if "u" in want else none
    dbg, o3 = mk.out(m) if "b" in want else none
    dbu, o4 = mk.out(m) if "c" in want else none
    xb.gated_backward_device(0, STORAGE[kind], n, k, m, ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g),
                             ptr(u), activation=ACTS[activation], dx_ptr=ptr(dx),
                             dgate_weight_ptr=ptr(dwg), dup_weight_ptr=ptr(dwu),
                             dgate_bias_ptr=ptr(dbg), dup_bias_ptr=ptr(dbu), lddh=ld(dh), ldx=ld(x),
                             ldw=ld(wg), ldg=ld(g), lddx=ld(dx),
                             lddw=ld(dwg if dwg is not None else dwu), stream=stream())
    for ok in (o0, o1, o2, o3, o4):
        ok()
    return dh, x, [wg, wu], [g, u], dx, [dwg, dwu], [dbg, dbu]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gated_backward(xb, kind, shape):
    i = SHAPES.index(shape)
    activation = list(ACTS)[(i + 2) % 4]
    pad, skew = LAYOUTS[i % 3]
    want = ("xgubc", "xgu", "xubc", "gub", "x", "xgubc", "u")[i % 7]
    out = run_gated_backward(xb, kind, *shape, activation, want, pad, skew, seed=i)
    check_backward(kind, activation, *out)


def test_float32_keeps_float32_accuracy(xb):
    """Relative 2-norm error of float32 products below 1e-6: a float32 product is exact to 2^-23
    (its three-part form or a float32 multiply), sums are rounded or truncated (2^-23 a step, of
    either sign of the running sum) over at most 48 matrix steps between float32 additions in
    registers: sqrt(48) 2^-23 = 8e-7."""
    x, w, _, _, y, _ = run_linear(xb, "fp32", 700, 960, 500, "none", False, False, False)
    want = x.double() @ w.double().t()
    assert ((y.double() - want).norm() / want.norm()).item() < 1e-6
    dy, x, ws, _, dx, dws, _ = run_linear_backward(xb, "fp32", 5000, 200, 300, "none", "xw")
    want = dy.double().t() @ x.double()
    assert ((dws[0].double() - want).norm() / want.norm()).item() < 1e-6
    want = dy.double() @ ws[0].double()
    assert ((dx.double() - want).norm() / want.norm()).item() < 1e-6


@pytest.mark.parametrize("kind", list(TYPES))
def test_float32_range(xb, kind):
    """Large and small magnitudes of the type's normal range give finite, correct products."""
    mk = Maker(kind, 3)
    n, k, m = 40, 96, 72
    big = 2.0 ** (10 if kind == "fp16" else 100)
    x, w = mk.matrix(n, k, big), mk.matrix(m, k, 1 / big)
    y, _ = mk.out(n, m)
    xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y), stream=stream())
    # fp16 weights near 2^-10 lie within the normal range but for a few subnormals, exact either way.
    want = x.double() @ w.double().t()
    close(y, want, sum_error(x.double(), w.double(), want), "y")


@pytest.mark.parametrize("n", [4, 300])
def test_float32_near_the_ends_of_its_range(xb, n):
    """Three bfloat16 parts hold a float32 exactly down to bfloat16's smallest step: each element is off
    by at most 2^-134.  Next to the largest float32 the first part must not round to an infinity."""
    k, m = 64, 48
    mk = Maker("fp32", 12)
    small, w = mk.matrix(n, k, 2.0 ** -126).contiguous(), mk.matrix(m, k, 2.0 ** 100).contiguous()
    y = torch.empty(n, m, device="cuda")
    xb.linear_device(0, 1, n, k, m, ptr(small), ptr(w), ptr(y), stream=stream())
    x64, w64 = small.double(), w.double()
    want = x64 @ w64.t()
    close(y, want, sum_error(x64, w64, want) + 2.0 ** -134 * w64.abs().sum(1), "y")
    big = torch.full((n, 1), torch.finfo(torch.float32).max, device="cuda")
    one = torch.ones(1, 1, device="cuda")
    y = torch.empty(n, 1, device="cuda")
    xb.linear_device(0, 1, n, 1, 1, ptr(big), ptr(one), ptr(y), stream=stream())
    assert bool((y == big).all())


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [5, 300])
def test_values_that_are_not_finite_stay_in_their_rows_and_columns(xb, kind, n):
    k, m = 130, 150
    mk = Maker(kind, 9)
    x, w, b = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5), mk.vector(m)
    x[1, 7], x[3, 100], w[11, 5] = math.inf, math.nan, math.nan
    y, _ = mk.out(n, m)
    xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y), bias_ptr=ptr(b), ldx=ld(x),
                     ldw=ld(w), stream=stream())
    bad = torch.zeros(n, m, dtype=torch.bool, device="cuda")
    bad[1], bad[3], bad[:, 11] = True, True, True
    assert bool((torch.isfinite(y) == ~bad).all())
    assert bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[:, 11]).all())
    keep = [i for i in range(n) if i not in (1, 3)]
    cols = [j for j in range(m) if j != 11]
    xs, wsub = x[keep].double(), w[cols].double()
    want = xs @ wsub.t() + b[cols].double()
    close(y[keep][:, cols], want, sum_error(xs, wsub, want) + SMALL * want.abs(), "y")


def test_relu_of_nan_and_zero(xb):
    x = torch.tensor([[math.nan], [0.0], [-1.0], [2.0]], device="cuda")
    w = torch.ones(1, 1, device="cuda")
    y = torch.empty(4, 1, device="cuda")
    xb.linear_device(0, 1, 4, 1, 1, ptr(x), ptr(w), ptr(y), activation=xb.ACT_RELU, stream=stream())
    assert math.isnan(y[0, 0].item()) and y[1:, 0].tolist() == [0.0, 0.0, 2.0]
    dx = torch.empty(4, 1, device="cuda")
    dy = torch.full((4, 1), 3.0, device="cuda")
    xb.linear_backward_device(0, 1, 4, 1, 1, ptr(dy), 0, ptr(w), preact_ptr=ptr(x),
                              activation=xb.ACT_RELU, dx_ptr=ptr(dx), stream=stream())
    assert dx[1:, 0].tolist() == [0.0, 0.0, 3.0]


@pytest.mark.parametrize("kind", list(TYPES))
def test_far_activation_arguments(xb, kind):
    """Pre-activations far from zero: no overflow inside the activations or their derivatives."""
    z = torch.tensor([-60000.0, -500.0, -100.0, -89.0, -20.0, 0.0, 20.0, 89.0, 100.0, 60000.0],
                     device="cuda").to(TYPES[kind])[:, None].contiguous()
    one = torch.ones(1, 1, device="cuda", dtype=z.dtype)
    n = z.shape[0]
    for name in ("gelu", "silu", "relu"):
        y, dx = torch.empty_like(z), torch.empty_like(z)
        xb.linear_device(0, STORAGE[kind], n, 1, 1, ptr(z), ptr(one), ptr(y), activation=ACTS[name],
                         stream=stream())
        z64 = z.double()
        close(y, act(name, z64), SMALL * z64.abs().clamp(max=1e3), name)
        dy = torch.ones_like(z)
        xb.linear_backward_device(0, STORAGE[kind], n, 1, 1, ptr(dy), 0, ptr(one), preact_ptr=ptr(z),
                                  activation=ACTS[name], dx_ptr=ptr(dx), stream=stream())
        want = slope(name, z64)
        # The pre-activation gradient is rounded to the type once before the product.
        close(dx, want, half_step(z.dtype) * want.abs() + 16 * SMALL, name + "'")


def test_residual_in_place(xb):
    for kind in TYPES:
        for n in (3, 200):
            mk = Maker(kind, 5)
            x, w, r = mk.matrix(n, 96), mk.matrix(80, 96, 0.1), mk.matrix(n, 80)
            y = r.clone()
            want, _ = mk.out(n, 80)
            args = dict(activation=xb.ACT_GELU, ldx=ld(x), ldw=ld(w), stream=stream())
            xb.linear_device(0, STORAGE[kind], n, 96, 80, ptr(x), ptr(w), ptr(want),
                             residual_ptr=ptr(r), ldr=ld(r), **args)
            xb.linear_device(0, STORAGE[kind], n, 96, 80, ptr(x), ptr(w), ptr(y), residual_ptr=ptr(y),
                             **args)
            assert torch.equal(y, want)


def test_no_rows(xb):
    w = torch.ones(8, 16, device="cuda")
    xb.linear_device(0, 1, 0, 16, 8, 0, ptr(w), 0)
    xb.gated_device(0, 1, 0, 16, 8, 0, ptr(w), ptr(w), 0)
    buf = torch.full((8, 20), SENTINEL, device="cuda")
    db = torch.full((8,), SENTINEL, device="cuda")
    xb.linear_backward_device(0, 1, 0, 16, 8, 0, 0, ptr(w), dw_ptr=ptr(buf), db_ptr=ptr(db), lddw=20,
                              stream=stream())
    assert bool((buf[:, :16] == 0).all()) and bool((buf[:, 16:] == SENTINEL).all())
    assert bool((db == 0).all())
    dg, du = torch.ones(8, 16, device="cuda"), torch.ones(8, 16, device="cuda")
    xb.gated_backward_device(0, 1, 0, 16, 8, 0, 0, ptr(w), ptr(w), 0, 0, dgate_weight_ptr=ptr(dg),
                             dup_weight_ptr=ptr(du), stream=stream())
    assert bool((dg == 0).all()) and bool((du == 0).all())


@pytest.mark.parametrize("kind", ["fp16", "fp32"])
def test_offsets_past_31_bits(xb, kind):
    """More than 2^31 elements in one operand and one output: the last rows are right."""
    n, k, m, wide = (1 << 20) + 3, 16, 8, 2304
    dtype = TYPES[kind]
    buf = torch.zeros(n, wide, device="cuda", dtype=dtype)
    out = torch.full((n, wide), SENTINEL, device="cuda", dtype=dtype)
    mk = Maker(kind, 2)
    w = mk.matrix(m, k)
    x, y = buf[:, 100:100 + k], out[:, 64:64 + m]
    x[-200:] = torch.randn(200, k, device="cuda").to(dtype)
    xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y), ldx=wide, ldw=ld(w), ldy=wide,
                     stream=stream())
    x64, w64 = x[-200:].double(), w.double()
    want = x64 @ w64.t()
    close(y[-200:], want, sum_error(x64, w64, want), "y")
    assert bool((y[:1000] == 0).all())
    assert bool((out[:, :64] == SENTINEL).all()) and bool((out[:, 64 + m:] == SENTINEL).all())
    dy, dw = out[:, 64:64 + m], torch.empty(m, k, device="cuda", dtype=dtype)
    xb.linear_backward_device(0, STORAGE[kind], n, k, m, ptr(dy), ptr(x), 0, dw_ptr=ptr(dw), lddy=wide,
                              ldx=wide, stream=stream())
    d64 = dy[-200:].double()
    close(dw, d64.t() @ x64, sum_error(d64.t(), x64.t()), "dw")


CALLS = {
    "linear": lambda xb, k: run_linear(xb, k, 200, 130, 90, "gelu", True, True, True)[4:6],
    "linear query": lambda xb, k: run_linear(xb, k, 2, 130, 90, "gelu", True, True, True)[4:6],
    "gated": lambda xb, k: run_gated(xb, k, 200, 130, 90, "silu", True, True)[5:],
    "gated query": lambda xb, k: run_gated(xb, k, 3, 130, 90, "silu", True, True)[5:],
    "linear backward": lambda xb, k: [t for v in run_linear_backward(
        xb, k, 2000, 130, 90, "gelu", "xwb")[4:] for t in (v if isinstance(v, list) else [v])],
    "gated backward": lambda xb, k: [t for v in run_gated_backward(
        xb, k, 2000, 130, 90, "silu", "xgubc")[4:] for t in (v if isinstance(v, list) else [v])],
}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("call", list(CALLS))
def test_results_repeat(xb, call, kind):
    a, b = CALLS[call](xb, kind), CALLS[call](xb, kind)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("call", list(CALLS))
def test_two_streams_at_once(xb, call):
    want = CALLS[call](xb, "bf16")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(CALLS[call](xb, "bf16"))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for g in got for p, q in zip(g, want))


def test_captured_and_replayed(xb):
    """A training step captured twice into graphs, replayed in turn on new inputs; an uncaptured
    step between the replays does not disturb them."""
    n, k, m = 700, 96, 160
    kind, dtype = "bf16", torch.bfloat16

    def buffers(seed):
        mk = Maker(kind, seed)
        names = dict(x=(n, k), wg=(m, k), wu=(m, k), wd=(k, m), dy=(n, k))
        s = {name: mk.matrix(*shape, 0.3) for name, shape in names.items()}
        for name, shape in dict(h=(n, m), g=(n, m), u=(n, m), y=(n, k), dh=(n, m), dx=(n, k),
                                dwg=(m, k), dwu=(m, k), dwd=(k, m)).items():
            s[name] = torch.zeros(shape, device="cuda", dtype=dtype)
        s["norm"] = torch.zeros((), device="cuda")
        return s

    def step(s):
        st = stream()
        xb.gated_device(0, 3, n, k, m, ptr(s["x"]), ptr(s["wg"]), ptr(s["wu"]), ptr(s["h"]),
                        gate_ptr=ptr(s["g"]), up_ptr=ptr(s["u"]), stream=st)
        xb.linear_device(0, 3, n, m, k, ptr(s["h"]), ptr(s["wd"]), ptr(s["y"]), residual_ptr=ptr(s["x"]),
                         stream=st)
        xb.linear_backward_device(0, 3, n, m, k, ptr(s["dy"]), ptr(s["h"]), ptr(s["wd"]),
                                  dx_ptr=ptr(s["dh"]), dw_ptr=ptr(s["dwd"]), stream=st)
        xb.gated_backward_device(0, 3, n, k, m, ptr(s["dh"]), ptr(s["x"]), ptr(s["wg"]), ptr(s["wu"]),
                                 ptr(s["g"]), ptr(s["u"]), dx_ptr=ptr(s["dx"]),
                                 dgate_weight_ptr=ptr(s["dwg"]), dup_weight_ptr=ptr(s["dwu"]),
                                 stream=st)
        xb.clip_gradients_device(0, [(3, ptr(s[t]), ptr(s[t]), s[t].numel())
                                     for t in ("dwg", "dwu", "dwd")], 0.5, ptr(s["norm"]), stream=st)

    outs = ("h", "y", "dx", "dwg", "dwu", "dwd", "norm")
    graphs = []
    for seed in (1, 2):
        s = buffers(seed)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(s)
        graphs.append((g, s))
    fresh = buffers(5)
    for round_ in range(2):
        for i, (g, s) in enumerate(graphs):
            new = buffers(10 * round_ + i + 20)
            for name in ("x", "wg", "wu", "wd", "dy"):
                s[name].copy_(new[name])
            g.replay()
            step(fresh)
            step(new)
            torch.cuda.synchronize()
            for name in outs:
                assert torch.equal(s[name], new[name]), name
    graphs.clear()


FRESH = """
import sys, torch
sys.path[:0] = [{root!r}]
import xvec_b200 as xb
n, k, m = {n}, 96, 128
x, w = torch.randn(n, k, device="cuda"), torch.randn(m, k, device="cuda")
y, dw, db = torch.empty(n, m, device="cuda"), torch.empty(m, k, device="cuda"), torch.empty(m, device="cuda")
norm = torch.empty((), device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    s = torch.cuda.current_stream().cuda_stream
    xb.linear_device(0, 1, n, k, m, x.data_ptr(), w.data_ptr(), y.data_ptr(), stream=s)
    xb.linear_backward_device(0, 1, n, k, m, y.data_ptr(), x.data_ptr(), w.data_ptr(), dw_ptr=dw.data_ptr(),
                              db_ptr=db.data_ptr(), stream=s)
    xb.clip_gradients_device(0, [(1, dw.data_ptr(), dw.data_ptr(), dw.numel())], 1.0, norm.data_ptr(),
                             stream=s)
graph.replay()
torch.cuda.synchronize()
want = x.double() @ w.double().t()
assert ((y.double() - want).norm() / want.norm()).item() < 1e-6
g = want.t() @ x.double()
assert abs(norm.item() / g.norm().item() - 1) < 1e-5
assert abs(dw.double().norm().item() - 1) < 1e-5
del graph
print("captured")
"""


@pytest.mark.parametrize("n", [3, 1000])
def test_first_call_of_a_process_inside_a_capture(n):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", FRESH.format(root=root, n=n)], capture_output=True,
                       text=True, timeout=300)
    assert p.returncode == 0 and "captured" in p.stdout, p.stderr[-2000:]


def test_two_threads_at_once(xb):
    """Calls of two host threads, each on its own stream and buffers."""
    import threading
    want = {c: CALLS[c](xb, "fp32") for c in CALLS}
    torch.cuda.synchronize()
    bad = []

    def work(call):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = CALLS[call](xb, "fp32")
                torch.cuda.current_stream().synchronize()
            bad.extend(call for p, q in zip(got, want[call]) if not torch.equal(p, q))
        except Exception as e:  # reported by the main thread
            bad.append(repr(e))

    threads = [threading.Thread(target=work, args=(c,)) for c in CALLS]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_queries_through_two_layers_without_waiting(xb):
    """Calls that follow one another on a stream read what the one before wrote (their launches
    overlap at the edges), also through the same buffers again and again."""
    k = 256
    mk = Maker("fp16", 11)
    ws = [mk.matrix(k, k, k ** -0.5).contiguous() for _ in range(4)]
    for n in (1, 6, 200, 3000):
        x0 = mk.matrix(n, k).contiguous()
        a, b = x0.clone(), torch.empty_like(x0)
        for i in range(40):
            xb.linear_device(0, 2, n, k, k, ptr(a), ptr(ws[i % 4]), ptr(b), activation=xb.ACT_SILU,
                             residual_ptr=ptr(x0), stream=stream())
            a, b = b, a
        got = a.clone()
        a, b = x0.clone(), torch.empty_like(x0)
        for i in range(40):
            xb.linear_device(0, 2, n, k, k, ptr(a), ptr(ws[i % 4]), ptr(b), activation=xb.ACT_SILU,
                             residual_ptr=ptr(x0), stream=stream())
            torch.cuda.synchronize()
            a, b = b, a
        assert torch.equal(a, got)


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_through_many_layers_without_waiting(xb, kind):
    """Backward calls that follow one another without a wait: each reads the dx that the one before
    wrote, while that one's weight gradients may still be under way; all results as with a wait after
    every call."""
    k, layers = 160, 24
    mk = Maker(kind, 13)
    ws = [mk.matrix(k, k, k ** -0.5).contiguous() for _ in range(3)]
    for n in (5, 130, 1500):
        x, z, dy = mk.matrix(n, k).contiguous(), mk.matrix(n, k).contiguous(), mk.matrix(n, k).contiguous()

        def run(wait):
            d, outs = dy.clone(), []
            for i in range(layers):
                w = ws[i % 3]
                dx, dw, dw2 = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
                db = torch.empty(k, device="cuda", dtype=x.dtype)
                if i % 2:
                    xb.linear_backward_device(0, STORAGE[kind], n, k, k, ptr(d), ptr(x), ptr(w),
                                              preact_ptr=ptr(z), activation=xb.ACT_GELU,
                                              dx_ptr=ptr(dx), dw_ptr=ptr(dw), db_ptr=ptr(db),
                                              stream=stream())
                    outs += [dx, dw, db]
                else:
                    xb.gated_backward_device(0, STORAGE[kind], n, k, k, ptr(d), ptr(x), ptr(w), ptr(ws[2]),
                                             ptr(z), ptr(x), dx_ptr=ptr(dx), dgate_weight_ptr=ptr(dw),
                                             dup_weight_ptr=ptr(dw2), stream=stream())
                    outs += [dx, dw, dw2]
                if wait:
                    torch.cuda.synchronize()
                d = dx
            torch.cuda.synchronize()
            return outs

        want = run(True)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(run(False), want))


def test_gradients_against_differences(xb):
    """The gradients are the slopes of the forward pass itself: central differences of a float32
    adapter along random directions.  f(t) = <c, y(t)> in float64 of float32 outputs: rounding leaves
    2^-22 |c||y| / step, the third derivative step^2 (all values are near 1), step = 2^-6."""
    n, k, m = 24, 20, 28
    mk = Maker("fp32", 4)
    x, wg, wu, wd = mk.matrix(n, k), mk.matrix(m, k, 0.3), mk.matrix(m, k, 0.3), mk.matrix(k, m, 0.3)
    c = mk.matrix(n, k).contiguous()

    def new(*shape):
        return torch.empty(shape, device="cuda")

    def forward(x, wg, wu, wd):
        x, wg, wu, wd = (t.contiguous() for t in (x, wg, wu, wd))
        g, u, h, z, y = new(n, m), new(n, m), new(n, m), new(n, k), new(n, k)
        xb.gated_device(0, 1, n, k, m, ptr(x), ptr(wg), ptr(wu), ptr(h), gate_ptr=ptr(g), up_ptr=ptr(u),
                        stream=stream())
        xb.linear_device(0, 1, n, m, k, ptr(h), ptr(wd), ptr(y), residual_ptr=ptr(x),
                         activation=xb.ACT_GELU, preact_ptr=ptr(z), stream=stream())
        return g, u, h, z, y

    x, wg, wu, wd = (t.contiguous() for t in (x, wg, wu, wd))
    g, u, h, z, y = forward(x, wg, wu, wd)
    dh, dwd, dx, dwg, dwu = new(n, m), new(k, m), new(n, k), new(m, k), new(m, k)
    xb.linear_backward_device(0, 1, n, m, k, ptr(c), ptr(h), ptr(wd), preact_ptr=ptr(z),
                              activation=xb.ACT_GELU, dx_ptr=ptr(dh), dw_ptr=ptr(dwd), stream=stream())
    xb.gated_backward_device(0, 1, n, k, m, ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g), ptr(u),
                             dx_ptr=ptr(dx), dgate_weight_ptr=ptr(dwg), dup_weight_ptr=ptr(dwu),
                             stream=stream())
    dx = dx + c  # the residual's share
    step = 2.0 ** -6
    for i, grad in enumerate((dx, dwg, dwu, dwd)):
        base = [x, wg, wu, wd]
        d = torch.randn(base[i].shape, generator=mk.gen, device="cuda")
        d /= d.norm()
        f = []
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * step * d
            f.append((forward(*moved)[4].double() * c.double()).sum())
        slope_ = ((f[0] - f[1]) / (2 * step)).item()
        scale = (c.double().norm() * y.double().norm()).item()
        want = (grad.double() * d.double()).sum().item()
        assert abs(slope_ - want) <= scale * (2.0 ** -22 / step + 4 * step * step), i


def test_train_an_adapter_and_search_with_it(oracle, xb):
    """The operators as they are used together: queries through a gated residual adapter, the
    gradients of a loss on its outputs against automatic differentiation in 64 bits, clipped, one
    step taken; then the adapted queries search a Flat index, equal to the oracle on them."""
    n, k, m, rows = 257, 96, 200, 3000
    mk = Maker("fp32", 8)
    x, target = mk.matrix(n, k).contiguous(), mk.matrix(n, k).contiguous()
    params = [mk.matrix(m, k, k ** -0.5).contiguous(), mk.matrix(m, k, k ** -0.5).contiguous(),
              mk.matrix(k, m, m ** -0.5).contiguous(), mk.vector(m, 0.1).clone(),
              mk.vector(m, 0.1).clone(), mk.vector(k, 0.1).clone()]

    def new(*shape):
        return torch.empty(shape, device="cuda")

    def forward():
        wg, wu, wd, bg, bu, bd = params
        g, u, h, y = new(n, m), new(n, m), new(n, m), new(n, k)
        xb.gated_device(0, 1, n, k, m, ptr(x), ptr(wg), ptr(wu), ptr(h), gate_bias_ptr=ptr(bg),
                        up_bias_ptr=ptr(bu), gate_ptr=ptr(g), up_ptr=ptr(u), stream=stream())
        xb.linear_device(0, 1, n, m, k, ptr(h), ptr(wd), ptr(y), bias_ptr=ptr(bd), residual_ptr=ptr(x),
                         stream=stream())
        return g, u, h, y

    leaves = [p.double().requires_grad_() for p in params]
    a = x.double()
    h64 = torch.nn.functional.silu(a @ leaves[0].t() + leaves[3]) * (a @ leaves[1].t() + leaves[4])
    y64 = h64 @ leaves[2].t() + leaves[5] + a
    (0.5 * (y64 - target.double()).square().sum() / n).backward()

    g, u, h, y = forward()
    dy = (y - target) / n
    wg, wu, wd, bg, bu, bd = params
    grads = [torch.empty_like(p) for p in params]
    dh = new(n, m)
    xb.linear_backward_device(0, 1, n, m, k, ptr(dy), ptr(h), ptr(wd), dx_ptr=ptr(dh),
                              dw_ptr=ptr(grads[2]), db_ptr=ptr(grads[5]), stream=stream())
    xb.gated_backward_device(0, 1, n, k, m, ptr(dh), ptr(x), ptr(wg), ptr(wu), ptr(g), ptr(u),
                             dgate_weight_ptr=ptr(grads[0]), dup_weight_ptr=ptr(grads[1]),
                             dgate_bias_ptr=ptr(grads[3]), dup_bias_ptr=ptr(grads[4]), stream=stream())
    for got, leaf in zip(grads, leaves):
        # Four float32 products in a row, each within 1e-6 of its 2-norm, and the differences y - target.
        assert ((got.double() - leaf.grad).norm() / leaf.grad.norm()).item() < 1e-5
    norm = torch.zeros((), device="cuda")
    total = math.sqrt(sum(l.grad.square().sum().item() for l in leaves))
    raw = [t.clone() for t in grads]
    xb.clip_gradients_device(0, [(1, ptr(t), ptr(t), t.numel()) for t in grads], total / 2, ptr(norm),
                             stream=stream())
    assert abs(norm.item() - total) < 1e-5 * total
    for got, before in zip(grads, raw):
        assert torch.allclose(got, before * 0.5, rtol=2e-5)
    for p, t in zip(params, grads):
        p.sub_(t, alpha=0.1)

    y = forward()[3]
    base = mk.matrix(rows, k).contiguous()
    keys = np.arange(rows, dtype=np.uint64) * 3 + 1
    idx = xb.DenseFlatIndex(k, xb.METRIC_COSINE)
    idx.add(keys, base.cpu().numpy())
    opts = xb.SearchOptions(top_k=10)
    okeys = torch.zeros(n, 10, dtype=torch.int64, device="cuda")
    oscores = torch.zeros(n, 10, device="cuda")
    ocounts = torch.zeros(n, dtype=torch.int32, device="cuda")
    idx.search_device(ptr(y), n, opts, ptr(okeys), ptr(oscores), ptr(ocounts), stream=stream())
    torch.cuda.synchronize()
    st, want, scores, counts, _ = oracle.flat_search(xb.METRIC_COSINE, base.cpu().numpy(), keys,
                                                     y.cpu().numpy(), 10)
    assert st == 0 and np.array_equal(ocounts.cpu().numpy(), counts)
    assert np.array_equal(okeys.cpu().numpy().astype(np.uint64), want)
    assert np.array_equal(oscores.cpu().numpy().view(np.uint32), scores.view(np.uint32))
    idx.close()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [100, 1500])
def test_expired_device_wait(xb, kind, n):
    """A wait bound of 1 ns runs out in the matrix kernel: it sets the status, frees what it holds
    and returns; afterwards the same call is right and leaves the status alone."""
    k, m = 512, 384
    mk = Maker(kind, 6)
    x, w = mk.matrix(n, k), mk.matrix(m, k, k ** -0.5)
    y, _ = mk.out(n, m)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def call():
        xb.linear_device(0, STORAGE[kind], n, k, m, ptr(x), ptr(w), ptr(y), status_ptr=ptr(status),
                         stream=stream())
        torch.cuda.synchronize()

    assert xb.set_wait_limit_ns(1) == 2_000_000_000
    try:
        call()
        assert status.item() == 4  # XVEC_GPU_TIMEOUT
    finally:
        xb.set_wait_limit_ns(0)
    status.zero_()
    call()
    assert status.item() == 0
    want = x.double() @ w.double().t()
    close(y, want, sum_error(x.double(), w.double(), want), "y")
