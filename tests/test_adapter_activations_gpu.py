"""The adapter's activations and their derivatives relative to their own size: far negative arguments
give small results, which an error bound relative to the argument would not see."""
import math

import pytest
import torch

from adapter_cases import ACTS, STORAGE, TYPES, half_step, ptr, tiny

pytestmark = pytest.mark.gpu

# float32: Phi's tail is a product of an exponential (2 units in the last place, its argument's rounding
# made up for), a reciprocal (2) and a polynomial of degree 7 (a rounding for each step but the last
# shrinks; 4), times z: below 12 units, 12 x 2^-24 < 2^-20.  16-bit types take a cheaper exponential, off by
# 2^-23 of its argument, at most 88 here: 88 x 2^-23 < 2^-16.
RELATIVE = {"fp32": 2.0 ** -20, "fp16": 2.0 ** -16, "bf16": 2.0 ** -16}


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2))


def values(name, z):
    return z * (phi(z) if name == "gelu" else torch.sigmoid(z))


def slopes(name, z):
    """The derivative, and the sum of its terms' sizes: where they cancel, that is what an error is
    relative to."""
    if name == "gelu":
        a, b = phi(z), z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(z)
        a, b = s, s * z * torch.sigmoid(-z)
    return a + b, a.abs() + b.abs()


def arguments(name, kind, count):
    low = -12.0 if name == "gelu" else -88.0 if kind != "fp16" else -16.0
    return torch.linspace(low, 12.0, count, device="cuda").to(TYPES[kind])[:, None].contiguous()


def check(got, want, size, kind, name):
    step, least = half_step(got.dtype), tiny(got.dtype)
    bound = RELATIVE[kind] * size * (1 + step) + step * want.abs() + least
    bad = ~((got.double() - want).abs() <= bound)
    if bool(bad.any()):
        i = int(torch.nonzero(bad)[0, 0])
        raise AssertionError(f"{name}: got {got[i].item()!r}, want {want[i].item()!r}, "
                             f"{int(bad.sum())} of {bad.numel()} off")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("name", ["gelu", "silu"])
@pytest.mark.parametrize("count", [7, 4001])  # the few-row kernel, the matrix kernel
def test_forward(xb, name, kind, count):
    for shift in range(1 if count > 100 else 60):
        z = arguments(name, kind, 4001)[shift * 67::572 if count == 7 else 1][:count].contiguous()
        n = z.shape[0]
        one, y = torch.ones(1, 1, device="cuda", dtype=z.dtype), torch.empty_like(z)
        xb.linear_device(0, STORAGE[kind], n, 1, 1, ptr(z), ptr(one), ptr(y), activation=ACTS[name],
                         stream=stream())
        want = values(name, z.double())
        check(y, want, want.abs(), kind, name)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("name", ["gelu", "silu"])
def test_derivatives(xb, name, kind):
    """dbias of single rows is the pre-activation gradient itself, rounded once."""
    z = arguments(name, kind, 4001).t().contiguous()  # one row of many columns
    m = z.shape[1]
    dy, db = torch.ones_like(z), torch.empty(m, device="cuda", dtype=z.dtype)
    xb.linear_backward_device(0, STORAGE[kind], 1, 1, m, ptr(dy), 0, 0, preact_ptr=ptr(z),
                              activation=ACTS[name], db_ptr=ptr(db), stream=stream())
    want, size = slopes(name, z[0].double())
    check(db, want, size, kind, name + "'")
    # The gated block's second gradient is the activation itself: du = dh act(gate).
    up, dub = torch.ones_like(z), torch.empty_like(db)
    xb.gated_backward_device(0, STORAGE[kind], 1, 1, m, ptr(dy), 0, 0, 0, ptr(z), ptr(up),
                             activation=ACTS[name], dgate_bias_ptr=ptr(db), dup_bias_ptr=ptr(dub),
                             stream=stream())
    check(db, want, size, kind, name + "'")
    want = values(name, z[0].double())
    check(dub, want, want.abs(), kind, name)


@pytest.mark.parametrize("kind", list(TYPES))
def test_values_that_are_not_finite(xb, kind):
    z = torch.tensor([math.inf, math.nan, -math.inf], device="cuda").to(TYPES[kind])[:, None].contiguous()
    one = torch.ones(1, 1, device="cuda", dtype=z.dtype)
    for name in ("gelu", "silu"):
        y = torch.empty_like(z)
        xb.linear_device(0, STORAGE[kind], 3, 1, 1, ptr(z), ptr(one), ptr(y), activation=ACTS[name],
                         stream=stream())
        assert y[0, 0].item() == math.inf and math.isnan(y[1, 0].item())
        # -inf times a weight of 0: a limit of 0 and the product's NaN are both taken.
        assert math.isnan(y[2, 0].item()) or y[2, 0].item() == 0
