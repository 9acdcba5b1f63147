"""The learned adapter's formulas in 64 bits, error bounds derived from them, and
tensors laid out for the tests (strides, slack, sentinels)."""
import math

import torch

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
STORAGE = {"fp32": 1, "fp16": 2, "bf16": 3}
SENTINEL = 77.0


def half_step(dtype):
    """The most a rounding to dtype moves a value, relative to it."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """The most a rounding moves a value below the normal range, absolute."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def act(name, z):
    return {"none": lambda v: v, "relu": torch.relu,
            "gelu": lambda v: 0.5 * v * (1 + torch.erf(v / math.sqrt(2))),
            "silu": lambda v: v * torch.sigmoid(v)}[name](z)


def slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def sum_error(a, b, extra=None):
    """Bound of a float32 sum of products a [r, d] . b [c, d]: every addition is off by at most
    2^-23 of the running sum (a truncating adder included).  16 terms or fewer go into one
    addition of a matrix instruction, so truncation, which always points the same way, adds up
    over d / 16 (float32 parts: 6 d / 16) steps; the parts below 2^-24 of a float32 product that are
    left out, and roundings of either sign, grow with sqrt(d).  The running sum is of the size of
    R = sqrt(sum a^2 b^2) + |a . b| (+ |extra|)."""
    r = (a.square() @ b.square().t()).sqrt() + (a @ b.t()).abs()
    if extra is not None:
        r = r + extra.abs()
    d = a.shape[1]
    return 2.0 ** -23 * (6 * d / 16 + 8 * math.sqrt(d) + 8) * r


def rounded_terms_error(a, b, dtype):
    """Bound of sum a_i b_i where each a_i was rounded to dtype: independent errors of mean zero,
    at most c_i = half_step |a_i b_i| (+ the subnormal half step), exceed 6.5 sqrt(sum c_i^2) with a
    probability below 2 exp(-6.5^2 / 2) = 1.4e-9 (Hoeffding)."""
    c = half_step(dtype) * a.abs() + tiny(dtype)
    return 6.5 * (c.square() @ b.square().t()).sqrt()


def close(got, want, error, name=""):
    """|got - want| <= error + the rounding to got's type (of a value that is itself off by error)."""
    step = half_step(got.dtype)
    subnormal = tiny(got.dtype)
    got = got.double()
    bound = error * (1 + step) + step * want.abs() + subnormal
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        at = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{name}{list(at)}: got {got[at].item()!r}, want {want[at].item()!r}, "
                             f"bound {bound[at].item():.3g}; {int(bad.sum())} of {bad.numel()} off")


class Maker:
    """Tensors of one type from a seed.  pad: columns between the rows' ends and the next rows;
    skew: elements that the first one lies off the allocation's alignment."""

    def __init__(self, kind, seed, pad=0, skew=0, device="cuda"):
        self.dtype, self.pad, self.skew, self.device = TYPES[kind], pad, skew, device
        self.gen = torch.Generator(device=device).manual_seed(seed)

    def matrix(self, rows, cols, scale=1.0, slack=2):
        """A random [rows, cols] view; the padding and `slack` rows behind hold NaN."""
        wide = cols + self.pad
        buf = torch.full((self.skew + (rows + slack) * wide,), math.nan, dtype=self.dtype,
                         device=self.device)
        m = buf[self.skew:].view(rows + slack, wide)[:rows, :cols]
        m.copy_(torch.randn(rows, cols, generator=self.gen, device=self.device) * scale)
        return m

    def vector(self, n, scale=1.0):
        v = torch.full((self.skew + n + 2,), math.nan, dtype=self.dtype, device=self.device)
        v = v[self.skew:self.skew + n]
        v.copy_(torch.randn(n, generator=self.gen, device=self.device) * scale)
        return v

    def out(self, rows, cols=None):
        """An output and a function that checks that nothing around it was written."""
        wide = (cols if cols is not None else 1) + (self.pad if cols is not None else 0)
        count = rows * wide if cols is not None else rows
        buf = torch.full((self.skew + count + 64,), SENTINEL, dtype=self.dtype, device=self.device)
        body = buf[self.skew:self.skew + count]
        view = body.view(rows, wide)[:, :cols] if cols is not None else body

        def untouched():
            copy = buf.clone()
            c = copy[self.skew:self.skew + count]
            (c.view(rows, wide)[:, :cols] if cols is not None else c).fill_(SENTINEL)
            assert bool((copy == SENTINEL).all()), "written outside the output"

        return view, untouched


def ptr(t):
    return 0 if t is None else t.data_ptr()


def ld(t):
    return 0 if t is None else t.stride(0)
