"""Clipping gradients to a global norm on the GPU against 64 bits: types, lists of one to a thousand
tensors, empty ones, in place and not, magnitudes whose squares leave float32, norms that are not
finite, offsets past 31 bits, graphs and streams."""
import math

import pytest
import torch

from adapter_cases import SENTINEL, STORAGE, TYPES, close, half_step, ptr

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def xb():
    import xvec_b200
    assert xvec_b200.device_count() >= 1
    return xvec_b200


def stream():
    return torch.cuda.current_stream().cuda_stream


def kind_of(t):
    return {v: k for k, v in TYPES.items()}[t.dtype]


def clip(xb, tensors, max_norm, outs=None):
    norm = torch.full((3,), SENTINEL, device="cuda")
    outs = tensors if outs is None else outs
    xb.clip_gradients_device(0, [(STORAGE[kind_of(t)], ptr(t), ptr(o), t.numel())
                                 for t, o in zip(tensors, outs)], max_norm, ptr(norm[1:]),
                             stream=stream())
    assert norm[0].item() == SENTINEL and norm[2].item() == SENTINEL
    return norm[1].item()


def check(xb, tensors, ratio, in_place):
    """The norm is summed from values exact in float32 whose squares are rounded at most once to
    float32, then in float32 over few terms or in float64: 2^-20 covers it; the scale is rounded to
    float32 once more, the results to their type."""
    want_norm = math.sqrt(sum(t.double().square().sum().item() for t in tensors))
    max_norm = ratio * want_norm
    scale = min(1.0, max_norm / want_norm) if want_norm else 1.0
    want = [t.double() * scale for t in tensors]
    before = [t.clone() for t in tensors]
    outs = tensors if in_place else [torch.full_like(t, SENTINEL) for t in tensors]
    norm = clip(xb, tensors, max_norm, outs)
    assert abs(norm - want_norm) <= 2.0 ** -20 * want_norm
    for o, w, b, t in zip(outs, want, before, tensors):
        close(o, w, 2.0 ** -19 * w.abs(), "clipped")
        if not in_place:
            assert torch.equal(t, b)
        if scale == 1.0:
            assert torch.equal(o, b)


SIZES = [[1], [7, 0, 3], [16384], [16385, 1, 5000], [100_003, 333, 64], [1] * 70, [4097] * 600,
         [3] * 1300, [2_000_000, 17], [5_000_001] * 9]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kind", list(TYPES) + ["mixed"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_clip(xb, sizes, kind, in_place):
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    kinds = list(TYPES)
    tensors = []
    for i, n in enumerate(sizes):
        dtype = TYPES[kinds[i % 3] if kind == "mixed" else kind]
        # Every third tensor starts off the allocation's alignment.
        skew = i % 3
        t = torch.randn(n + skew, generator=g, device="cuda").to(dtype)[skew:]
        tensors.append(t)
    for ratio in (0.3, 2.0):
        check(xb, tensors, ratio, in_place)


@pytest.mark.parametrize("big", [1e-30, 1e-22, 1e18, 1e25, 3e37])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_squares_that_leave_float32(xb, kind, big):
    g = torch.Generator(device="cuda").manual_seed(1)
    tensors = [(torch.randn(n, generator=g, device="cuda").clamp(-3, 3) * big).to(TYPES[kind])
               for n in (40, 70_000)]
    want = math.sqrt(sum(t.double().square().sum().item() for t in tensors))
    outs = [torch.empty_like(t) for t in tensors]
    norm = clip(xb, tensors, want / 4, outs)
    if want < torch.finfo(torch.float32).max:
        assert abs(norm - want) <= 2.0 ** -20 * want
    else:
        assert norm == math.inf
    for t, o in zip(tensors, outs):
        close(o, t.double() / 4, 2.0 ** -19 * t.double().abs(), "clipped")


@pytest.mark.parametrize("limit", [1.0, 1e-3, 1e-12, 1e-30])
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_factors_below_float32(xb, kind, limit):
    """Gradients near the type's largest value and a small limit: the factor itself may lie below
    float32's normal numbers, the results do not.  The bound is test_clip's: the norm within 2^-20,
    two roundings more, and half a step of the type."""
    g = torch.Generator(device="cuda").manual_seed(3)
    sign = torch.randint(0, 2, (2051,), generator=g, device="cuda") * 2 - 1
    x = ((1 + torch.rand(2051, generator=g, device="cuda")) * 1e38 * sign).to(TYPES[kind])
    # The norm alone leaves float32 here and is written as infinity; the factor is finite.
    scale = limit / math.sqrt(x.double().square().sum().item())
    for out in (torch.full_like(x, SENTINEL), x.clone()):
        source = out if out[0] == x[0] else x
        want = x.double() * scale
        clip(xb, [source], limit, [out])
        close(out, want, 2.0 ** -19 * want.abs(), "clipped")


def test_one_large_value_among_small_ones(xb):
    t = torch.full((300_000,), 1e-21, device="cuda")
    t[123_456] = 2e-20
    want = math.sqrt(t.double().square().sum().item())
    assert abs(clip(xb, [t], 1.0) - want) <= 2.0 ** -20 * want


def test_zero_gradients_and_zero_limit(xb):
    z = torch.zeros(1000, device="cuda")
    assert clip(xb, [z], 1.0) == 0.0 and bool((z == 0).all())
    assert clip(xb, [z], 0.0) == 0.0 and bool((z == 0).all())
    t = torch.randn(1000, device="cuda")
    assert clip(xb, [t], 0.0) > 0 and bool((t == 0).all())


def test_no_tensors(xb):
    assert clip(xb, [], 1.0) == 0.0
    e = torch.empty(0, device="cuda")
    assert clip(xb, [e, e], 1.0) == 0.0


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("kind", list(TYPES))
def test_norm_that_is_not_finite(xb, kind, value):
    """The gradients are passed on unchanged and the norm says why."""
    a = torch.randn(50_000, device="cuda").to(TYPES[kind])
    b = torch.randn(33, device="cuda").to(TYPES[kind])
    b[5] = value
    before = [a.clone(), b.clone()]
    outs = [torch.empty_like(a), torch.empty_like(b)]
    for o in (outs, None):
        norm = clip(xb, [a, b], 0.1, o)
        assert math.isnan(norm) if math.isnan(value) else norm == math.inf
        for got, want in zip(o or [a, b], before):
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
            assert torch.equal(torch.isnan(got), torch.isnan(want))


def test_limit_of_infinity_leaves_the_gradients(xb):
    t = torch.randn(5000, device="cuda")
    before = t.clone()
    want = t.double().norm().item()
    assert abs(clip(xb, [t], math.inf) - want) <= 2.0 ** -20 * want and torch.equal(t, before)


def test_neighbours_stay_as_they_were(xb):
    for kind, dtype in TYPES.items():
        buf = torch.full((40_000,), SENTINEL, device="cuda", dtype=dtype)
        parts = [buf[3:10_001], buf[10_002:10_003], buf[20_000:39_999]]
        for p in parts:
            p.copy_(torch.randn(p.numel(), device="cuda"))
        check(xb, parts, 0.5, True)
        for i in (0, 2, 10_001, 10_003, 19_999, 39_999):
            assert buf[i].item() == SENTINEL


def test_offsets_past_31_bits(xb):
    n = (1 << 31) + 12_345
    t = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    t[-1], t[5], t[1 << 31] = 3.0, 4.0, 12.0
    assert abs(clip(xb, [t], 6.5) - 13.0) <= 13 * 2.0 ** -20
    assert t[-1].item() == 1.5 and t[5].item() == 2.0 and t[1 << 31].item() == 6.0
    assert int((t != 0).sum()) == 3


def test_repeats_streams_and_graphs(xb):
    g = torch.Generator(device="cuda").manual_seed(3)
    src = [torch.randn(n, generator=g, device="cuda").bfloat16() for n in (1_000_001, 40, 8192)]
    outs = [torch.empty_like(t) for t in src]
    first = clip(xb, src, 3.0, outs)
    want = [o.clone() for o in outs]
    for _ in range(3):
        assert clip(xb, src, 3.0, outs) == first
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    streams = [torch.cuda.Stream() for _ in range(3)]
    norms = torch.zeros(6, device="cuda")
    many = [[torch.empty_like(t) for t in src] for _ in range(6)]
    torch.cuda.synchronize()
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            xb.clip_gradients_device(0, [(3, ptr(a), ptr(b), a.numel()) for a, b in zip(src, many[i])],
                                     3.0, ptr(norms[i:]), stream=stream())
    torch.cuda.synchronize()
    assert norms.tolist() == [first] * 6
    assert all(torch.equal(a, b) for o in many for a, b in zip(o, want))
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            xb.clip_gradients_device(0, [(3, ptr(a), ptr(b), a.numel()) for a, b in zip(src, many[i])],
                                     3.0, ptr(norms[i:]), stream=stream())
        graphs.append(graph)
    for t in src:
        t.mul_(2)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
        clip(xb, src, 3.0, outs)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in many[:2] for a, b in zip(o, outs))
    assert norms[0].item() == norms[1].item() == 2 * first
    graphs.clear()
