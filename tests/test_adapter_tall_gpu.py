"""Sums over many terms in the adapter's products: the matrix units' additions truncate, so terms of
one sign lose a little of the sum with every addition, always in the same direction.  Long sums have to
leave the accumulators before that shows."""
import math

import pytest
import torch

from adapter_cases import STORAGE, TYPES, half_step, ptr

pytestmark = pytest.mark.gpu

# An accumulator takes at most 4096 terms, 16 in an addition: 256 additions, each off by less than 2^-23
# of a running sum that is half the final one on average (terms of one sign): 2^-16 together.  The sums
# of 4096 terms are added in float32: 2^-24 of half the sum for each, 2^-18 over 128 of them.  Terms of
# one addition are aligned before they are added: as much again.
LEAST = 2.0 ** -15


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def positive(gen, rows, cols, dtype, scale=1.0, along=1):
    """Positive values; each column's (along = 1) or row's (along = 0) of a size of its own, spread over a
    factor of two, so that the sums over the other direction lie anywhere between the type's steps."""
    t = torch.empty(rows, cols, device="cuda", dtype=dtype)
    own = (torch.rand((1, cols) if along else (rows, 1), generator=gen, device="cuda") + 1) * scale
    for i in range(0, rows, 1 << 14):  # (float32 in between, a part at a time)
        part = t[i:i + (1 << 14)]
        part.copy_((torch.rand(part.shape, generator=gen, device="cuda") * 0.5 + 0.5)
                   * (own if along else own[i:i + (1 << 14)]))
    return t


def bias_of(got, want):
    """The mean relative error.  The results' roundings are of either sign and independent: their mean
    over N exceeds 6.5 half steps / sqrt(N) with a probability below 1.4e-9 (Hoeffding).  (They are
    independent because the sums' sizes are spread, see positive.)"""
    mean = ((got.double() - want) / want).mean().item()
    return abs(mean), LEAST + 6.5 * half_step(got.dtype) / math.sqrt(got.numel())


@pytest.mark.parametrize("kind", list(TYPES))
def test_weight_gradient_of_a_tall_batch(xb, kind):
    n, k, m, dtype = 131_072, 2304, 2048, TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = positive(g, n, k, dtype), positive(g, n, m, dtype, 2.0 ** -6)
    dw = torch.empty(m, k, device="cuda", dtype=dtype)
    xb.linear_backward_device(0, STORAGE[kind], n, k, m, ptr(dy), ptr(x), 0, dw_ptr=ptr(dw),
                              stream=stream())
    want = dy[:, :512].double().t() @ x[:, :512].double()
    mean, bound = bias_of(dw[:512, :512], want)
    assert mean <= bound
    # Columns and rows at the other end, whose tiles are the last.
    want = dy[:, -64:].double().t() @ x[:, -64:].double()
    mean, bound = bias_of(dw[-64:, -64:], want)
    assert mean <= bound


@pytest.mark.parametrize("kind", list(TYPES))
def test_deep_forward_and_input_gradient(xb, kind):
    n, deep, m, dtype = 9472, 32_768, 2048, TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = positive(g, n, deep, dtype, along=0), positive(g, m, deep, dtype, 2.0 ** -6, along=0)
    y = torch.empty(n, m, device="cuda", dtype=dtype)
    xb.linear_device(0, STORAGE[kind], n, deep, m, ptr(x), ptr(w), ptr(y), stream=stream())
    mean, bound = bias_of(y[:512, :512], x[:512].double() @ w[:512].double().t())
    assert mean <= bound
    # dx of a gated block without an activation: dg = dh up, du = dh gate, two products in a row.
    wt, one = w.t().contiguous(), torch.ones(n, deep, device="cuda", dtype=dtype)
    dx = y
    xb.gated_backward_device(0, STORAGE[kind], n, m, deep, ptr(x), 0, ptr(wt), ptr(wt), ptr(one),
                             ptr(one), activation=xb.ACT_NONE, dx_ptr=ptr(dx), stream=stream())
    mean, bound = bias_of(dx[-512:, -512:], 2 * (x[-512:].double() @ w[-512:].double().t()))
    assert mean <= bound


@pytest.mark.parametrize("kind", list(TYPES))
def test_deep_gated(xb, kind):
    n, deep, m, dtype = 9472, 32_768, 1024, TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(3)
    x, wg = positive(g, n, deep, dtype, along=0), positive(g, m, deep, dtype, 2.0 ** -12, along=0)
    wu = positive(g, m, deep, dtype, 2.0 ** -10, along=0)
    h, gate, up = (torch.empty(n, m, device="cuda", dtype=dtype) for _ in range(3))
    xb.gated_device(0, STORAGE[kind], n, deep, m, ptr(x), ptr(wg), ptr(wu), ptr(h), gate_ptr=ptr(gate),
                    up_ptr=ptr(up), activation=xb.ACT_RELU, stream=stream())
    a, b = x[:512].double() @ wg[:512].double().t(), x[:512].double() @ wu[:512].double().t()
    for got, want in ((gate, a), (up, b)):
        mean, bound = bias_of(got[:512, :512], want)
        assert mean <= bound
    mean, bound = bias_of(h[:512, :512], a * b)
    assert mean <= bound + LEAST


@pytest.mark.parametrize("n", [16_384, 262_144])
def test_float32_weight_gradient_of_a_tall_batch(xb, n):
    """Terms of either sign: the 2-norm error stays below 1e-6.  In 4096 terms it is below 8e-7 (the
    products exact to 2^-23, at most 48 truncating additions in a row); the up to 64 sums of as many
    terms are added with a rounding of rms 2^-24 / sqrt(3) each of a sum that grows with the square
    root: sqrt(64 / 2) 2^-24 / sqrt(3) = 2e-7."""
    k, m = 2304, 2048
    g = torch.Generator(device="cuda").manual_seed(4)
    x, dy = (torch.randn(n, c, generator=g, device="cuda") for c in (k, m))
    dw = torch.empty(m, k, device="cuda")
    xb.linear_backward_device(0, 1, n, k, m, ptr(dy), ptr(x), 0, dw_ptr=ptr(dw), stream=stream())
    want = dy[:, :256].double().t() @ x[:, :256].double()
    assert ((dw[:256, :256].double() - want).norm() / want.norm()).item() < 1e-6


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("deep", [2048, 2049, 4095, 4096, 4097, 8192, 8193, 12_345])
def test_around_the_lengths_of_an_accumulation(xb, kind, deep):
    """Every element against 64 bits at depths around multiples of an accumulator's share, ragged
    tiles; the same bits again at the second call."""
    n, m, dtype = 2500, 1050, TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(deep)
    x = torch.randn(n, deep, generator=g, device="cuda").to(dtype)
    w = (torch.randn(m, deep, generator=g, device="cuda") * deep ** -0.5).to(dtype)
    y, again = (torch.empty(n, m, device="cuda", dtype=dtype) for _ in range(2))
    for out in (y, again):
        xb.linear_device(0, STORAGE[kind], n, deep, m, ptr(x), ptr(w), ptr(out), stream=stream())
    assert torch.equal(y, again)
    x64, w64 = x.double(), w.double()
    want = x64 @ w64.t()
    # Running sums are below R = |x|_2 |w|_2 / sqrt(deep) x 6.5 (terms of either sign): an accumulator's 256
    # truncations of 2^-23 and the float32 additions (four in a row here), 2^-24 each.
    size = 6.5 * x64.norm(dim=1)[:, None] * w64.norm(dim=1)[None] / math.sqrt(deep)
    bound = (260 * 2.0 ** -23) * size + half_step(dtype) * want.abs() * (1 + 2.0 ** -10) \
        + torch.finfo(dtype).tiny * half_step(dtype)
    assert bool(((y.double() - want).abs() <= bound).all())
    # (dW of the same depth: the operands' other order.)
    xt, wt = x.t().contiguous(), w.t().contiguous()
    dw = torch.empty(m, n, device="cuda", dtype=dtype)
    xb.linear_backward_device(0, STORAGE[kind], deep, n, m, ptr(wt), ptr(xt), 0, dw_ptr=ptr(dw),
                              stream=stream())
    assert bool(((dw.double() - want.t()).abs() <= bound.t()).all())


# Enough tiles that no depth is split, depths of several accumulations, ragged tiles.
LONG = [(9472, 2500, 1000), (5001, 4499, 1301), (9000, 6208, 515), (2600, 8195, 2304)]
LAYOUTS = [(0, 0), (8, 0), (5, 1)]  # pad, skew


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
@pytest.mark.parametrize("shape", LONG, ids=str)
def test_long_sums_with_everything_around_them(xb, kind, shape, layout):
    """Bias, activation, residual, saved pre-activations and their gradients in every layout; nothing
    around the outputs is written."""
    from test_adapter_gpu import (check_backward, check_gated, check_linear, run_gated,
                                  run_gated_backward, run_linear, run_linear_backward)
    i = LONG.index(shape)
    activation = ("silu", "gelu", "relu", "none")[i]
    n, k, m = shape
    check_linear(*run_linear(xb, kind, *shape, activation, True, True, i % 2 == 0, *layout, seed=i), activation)
    check_gated(*run_gated(xb, kind, n, k, m // 2, activation, i % 2 == 0, True, *layout, seed=i), activation)
    # The backward products' depths are the rows and the output columns.
    check_backward(kind, activation, *run_linear_backward(xb, kind, k, m, n, activation, "xwb", *layout, seed=i))
    check_backward(kind, activation,
                   *run_gated_backward(xb, kind, k, m, n, activation, "xgubc", *layout, seed=i))
