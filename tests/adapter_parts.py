"""float32 values whose three bfloat16 parts h + m + l all count, and the six products that the adapter
makes of two such values: what a missing one costs."""
import torch

PRODUCTS = ("hh", "hm", "mh", "mm", "hl", "lh")


def values(gen, rows, cols, device="cuda", scale=0):
    """+-2^scale (1 + f 2^-8 + g 2^-17), f in [1/4, 1/2) in steps of 2^-7, g in [1/4, 1/2) in steps of
    2^-6: h = 1, m = f 2^-8 and l = g 2^-17 are exact, of one sign, and as large as parts can be within
    a factor of four.  The signs are random."""
    def pick(low, high):
        return torch.randint(low, high, (rows, cols), generator=gen, device=device)

    f, g, sign = pick(32, 64) / 128, pick(16, 32) / 64, pick(0, 2) * 2 - 1
    return (sign * (1 + f.double() * 2.0 ** -8 + g.double() * 2.0 ** -17)).float() * 2.0 ** scale


def parts(x):
    """The three bfloat16 parts in float64, each the nearest to what is left."""
    h = x.bfloat16()
    m = (x - h.float()).bfloat16()
    l = (x - h.float() - m.float()).bfloat16()
    return {"h": h.double(), "m": m.double(), "l": l.double()}


def product(a, b, without=()):
    """a b' from its six products, but for those left out."""
    a, b = parts(a), parts(b)
    return sum(a[p[0]] @ b[p[1]].t() for p in PRODUCTS if p not in without)


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()
