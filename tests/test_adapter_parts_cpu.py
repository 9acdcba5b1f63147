"""What the float32 checks of the adapter's products can see: a mistake planted in a model of the
three-part product, on the CPU."""
import pytest
import torch

from adapter_parts import PRODUCTS, parts, product, relative, values

LIMIT = 1e-6  # of the GPU's checks


def two(rows, depth, cols):
    g = torch.Generator().manual_seed(1)
    return values(g, rows, depth, "cpu"), values(g, cols, depth, "cpu")


def test_the_parts_are_exact():
    for a in two(50, 60, 70):
        p = parts(a)
        assert torch.equal(p["h"] + p["m"] + p["l"], a.double())
        assert bool((p["m"] * p["h"].sign() >= 2.0 ** -10).all())
        assert bool((p["l"] * p["h"].sign() >= 2.0 ** -19).all())


@pytest.mark.parametrize("shape", [(40, 130, 90), (200, 160, 160), (60, 960, 70), (30, 20_000, 30)], ids=str)
def test_every_product_is_seen(shape):
    """All six: what is left out is at most 2 x 2^-9 x 2^-18 of the whole.  Without any one of them the
    error is beyond the limit: the least, mm, is (f 2^-8)^2 of the whole, f 1/4..1/2: 2.1e-6 on average."""
    a, b = two(*shape)
    want = a.double() @ b.double().t()
    assert relative(product(a, b), want) < 2.0 ** -26
    for p in PRODUCTS:
        assert relative(product(a, b, (p,)), want) > 1.5 * LIMIT, p
