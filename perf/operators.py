"""The learned-adapter operators' measured cases: one dict per case, its inputs, one pass, its work.

A learned adapter transforms embeddings before they are indexed or searched: a gated block
``h = act(x Wg' + bg) * (x Wu' + bu)``, an affine layer ``y = act(x W' + b) + r`` that brings h back
to the index's dimension, their gradients, and the clipping of all gradients to a global norm.

``own`` false: elementary torch operations in 32 bits, rounded once at the end; ``own`` true: the
library's entry points (xvec_b200).
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
MOST_FLOPS = 2.7e11   # the largest listed product
MOST_CLIP = 260_000_000  # values of the largest listed gradient list
MOST_BYTES = 1.5e9  # of a drawn product's matrices


def listed():
    return [
        # One query through a residual adapter before a search: latency.
        {"name": "linear one query", "op": "linear", "type": "fp16", "n": 1, "k": 768, "m": 768,
         "act": "none", "bias": True, "residual": True, "save": False, "pad": 0},
        # A batch of 10,000 float32 queries of 960 dimensions (the library's default storage).
        {"name": "linear query batch", "op": "linear", "type": "fp32", "n": 10_000, "k": 960, "m": 960,
         "act": "gelu", "bias": True, "residual": True, "save": False, "pad": 0},
        # Rows being added to an FP16 index, one bulk of them.
        {"name": "linear rows", "op": "linear", "type": "fp16", "n": 131_072, "k": 1024, "m": 1024,
         "act": "silu", "bias": True, "residual": True, "save": False, "pad": 0},
        # A training forward on ragged sizes: odd dimensions, rows inside wider ones, saved
        # pre-activations.
        {"name": "linear ragged", "op": "linear", "type": "bf16", "n": 4099, "k": 301, "m": 515,
         "act": "gelu", "bias": True, "residual": False, "save": True, "pad": 11},
        # The gradients of the layer that brings the hidden state back, one training batch.
        {"name": "linear backward", "op": "linear_backward", "type": "bf16", "n": 16_384, "k": 2048,
         "m": 1024, "act": "none", "bias": True, "pad": 0},
        # A small float32 adapter on odd sizes.
        {"name": "linear backward small", "op": "linear_backward", "type": "fp32", "n": 1021, "k": 100,
         "m": 129, "act": "gelu", "bias": True, "pad": 0},
        # Four float32 queries (the most that the one-pass Flat search takes) through a gated block.
        {"name": "gated four queries", "op": "gated", "type": "fp32", "n": 4, "k": 1024, "m": 2048,
         "act": "silu", "bias": False, "save": False, "pad": 0},
        # A training forward of a gated block over 768-dimensional embeddings.
        {"name": "gated rows", "op": "gated", "type": "bf16", "n": 32_768, "k": 768, "m": 2048,
         "act": "silu", "bias": True, "save": True, "pad": 0},
        # The gated block's gradients at the largest hidden width.
        {"name": "gated backward", "op": "gated_backward", "type": "fp16", "n": 8192, "k": 1024, "m": 4096,
         "act": "silu", "bias": False, "pad": 0},
        # The same in float32, odd batch, biases.
        {"name": "gated backward fp32", "op": "gated_backward", "type": "fp32", "n": 1999, "k": 960,
         "m": 1920, "act": "gelu", "bias": True, "pad": 0},
        # Clipping one adapter's gradients: three matrices and their biases.
        {"name": "clip one adapter", "op": "clip", "type": "bf16", "tensors": 6, "values": 6_300_000,
         "ratio": 0.25},
        # Clipping the gradients of an encoder trained with its adapter.
        {"name": "clip many", "op": "clip", "type": "fp32", "tensors": 48, "values": MOST_CLIP,
         "ratio": 0.5},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear_backward", "gated", "gated_backward", "clip"])
    kind = rng.choice(["fp32", "fp16", "bf16"])
    if op == "clip":
        return {"op": op, "type": kind, "tensors": _spread(rng, 1, 48),
                "values": _spread(rng, 1000, MOST_CLIP), "ratio": rng.choice([0.01, 0.3, 0.9, 2.0])}
    k, m = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
    if rng.random() < 0.5:
        k, m = -(-k // 64) * 64, -(-m // 64) * 64
    products = {"linear": 1, "linear_backward": 2, "gated": 2, "gated_backward": 4}[op]
    cap = int(min(131_072, MOST_FLOPS / (2 * k * m * products),
                  MOST_BYTES / (BYTES[kind] * (2 * k + 3 * m))))
    case = {"op": op, "type": kind, "n": _spread(rng, 1, cap), "k": k, "m": m,
            "act": rng.choice(["none", "relu", "gelu", "silu"]), "bias": rng.random() < 0.7,
            "pad": rng.choice([0, 0, 8, 5])}
    if op == "linear":
        case["residual"] = rng.random() < 0.5
    if op in ("linear", "gated"):
        case["save"] = rng.random() < 0.5
    return case


def prepare(case, seed):
    """Embeddings near N(0, 1), weights scaled by 1 / sqrt(k), gradients of a mean loss."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["type"]]

    def normal(*shape, scale=1.0):
        pad = case.get("pad", 0) if len(shape) == 2 else 0
        wide = shape[:-1] + (shape[-1] + pad,)
        t = torch.randn(wide, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)
        return t[..., : shape[-1]]

    if case["op"] == "clip":
        count, total = case["tensors"], case["values"]
        # Matrices and their biases in turn, sizes that do not divide evenly.
        share = [1 if i % 2 else 1000 + 37 * (i % 5) for i in range(count)]
        sizes = [max(1, total * s // sum(share)) for s in share]
        grads = [normal(n, scale=0.02 * (1 + i % 3)) for i, n in enumerate(sizes)]
        norm = math.sqrt(sum((0.02 * (1 + i % 3)) ** 2 * n for i, n in enumerate(sizes)))
        return {"case": case, "grads": grads, "out": [torch.empty_like(t) for t in grads],
                "max_norm": case["ratio"] * norm}
    n, k, m = case["n"], case["k"], case["m"]
    s = {"case": case, "x": normal(n, k)}
    names = ["g", "u"] if case["op"].startswith("gated") else ["z"]
    for name in names:
        s["w" + name] = normal(m, k, scale=k ** -0.5)
        s["b" + name] = normal(m, scale=0.1) if case["bias"] else None
    if case["op"].endswith("backward"):
        s["dy"] = normal(n, m, scale=0.1)
        for name in names:  # the pre-activations that the forward pass saved
            s[name] = normal(n, m)
    elif case["op"] == "linear":
        s["r"] = normal(n, m) if case["residual"] else None
    return s


# --- plain forms -------------------------------------------------------------------------------

def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z / (1 + torch.exp(-z))


def _slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    p = 1 / (1 + torch.exp(-z))
    return p * (1 + z * (1 - p))


def _affine(x, w, b):
    z = x.float() @ w.float().t()
    return z if b is None else z + b.float()


def _plain(s, case):
    op, act = case["op"], case.get("act")
    dtype = DTYPES[case["type"]]
    if op == "linear":
        z = _affine(s["x"], s["wz"], s["bz"])
        y = _act(act, z)
        y = y if s["r"] is None else y + s["r"].float()
        return {"y": y.to(dtype), **({"z": z.to(dtype)} if case["save"] else {})}
    if op == "gated":
        g, u = _affine(s["x"], s["wg"], s["bg"]), _affine(s["x"], s["wu"], s["bu"])
        h = _act(act, g) * u
        return {"h": h.to(dtype), **({"g": g.to(dtype), "u": u.to(dtype)} if case["save"] else {})}
    if op == "linear_backward":
        d = s["dy"].float()
        d = d if act == "none" else d * _slope(act, s["z"].float())
        out = {"dx": d @ s["wz"].float(), "dw": d.t() @ s["x"].float()}
        if case["bias"]:
            out["db"] = d.sum(0)
    elif op == "gated_backward":
        dh, g, u = s["dy"].float(), s["g"].float(), s["u"].float()
        dg, du = dh * u * _slope(act, g), dh * _act(act, g)
        x = s["x"].float()
        out = {"dx": dg @ s["wg"].float() + du @ s["wu"].float(), "dwg": dg.t() @ x, "dwu": du.t() @ x}
        if case["bias"]:
            out |= {"dbg": dg.sum(0), "dbu": du.sum(0)}
    else:
        norm = sum([t.double().square().sum() for t in s["grads"]]).sqrt()
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
        return {"norm": norm.float(), "clipped": [(t.float() * scale).to(dtype) for t in s["grads"]]}
    return {name: t.to(dtype) for name, t in out.items()}


# --- the library's calls -----------------------------------------------------------------------

def _own(s, case):
    import xvec_b200 as xb

    stream = torch.cuda.current_stream().cuda_stream
    storage = {"fp32": xb.STORAGE_FP32, "fp16": xb.STORAGE_FP16, "bf16": xb.STORAGE_BF16}[case["type"]]
    dtype = DTYPES[case["type"]]
    op = case["op"]
    if op == "clip":
        norm = torch.empty((), device="cuda", dtype=torch.float32)
        xb.clip_gradients_device(0, [(storage, a.data_ptr(), b.data_ptr(), a.numel())
                                     for a, b in zip(s["grads"], s["out"])],
                                 s["max_norm"], norm.data_ptr(), stream=stream)
        return {"norm": norm, "clipped": s["out"]}
    n, k, m = case["n"], case["k"], case["m"]
    act = ACTS[case["act"]]

    def new(*shape):
        return torch.empty(shape, device="cuda", dtype=dtype)

    def at(t):
        return 0 if t is None else t.data_ptr()

    x, pitch = s["x"], (lambda t: 0 if t is None else t.stride(0))
    if op == "linear":
        w, r = s["wz"], s["r"]
        y, z = new(n, m), new(n, m) if case["save"] else None
        xb.linear_device(0, storage, n, k, m, at(x), at(w), at(y), bias_ptr=at(s["bz"]),
                         residual_ptr=at(r), activation=act, preact_ptr=at(z), ldx=pitch(x),
                         ldw=pitch(w), ldr=pitch(r), stream=stream)
        return {"y": y, **({"z": z} if case["save"] else {})}
    if op == "linear_backward":
        w, z = s["wz"], None if case["act"] == "none" else s["z"]
        dx, dw, db = new(n, k), new(m, k), new(m) if case["bias"] else None
        xb.linear_backward_device(0, storage, n, k, m, at(s["dy"]), at(x), at(w), preact_ptr=at(z),
                                  activation=act, dx_ptr=at(dx), dw_ptr=at(dw), db_ptr=at(db),
                                  lddy=pitch(s["dy"]), ldx=pitch(x), ldw=pitch(w), ldz=pitch(z),
                                  stream=stream)
        return {"dx": dx, "dw": dw, **({"db": db} if case["bias"] else {})}
    wg, wu = s["wg"], s["wu"]
    if op == "gated":
        h = new(n, m)
        g, u = (new(n, m), new(n, m)) if case["save"] else (None, None)
        xb.gated_device(0, storage, n, k, m, at(x), at(wg), at(wu), at(h), gate_bias_ptr=at(s["bg"]),
                        up_bias_ptr=at(s["bu"]), activation=act, gate_ptr=at(g), up_ptr=at(u),
                        ldx=pitch(x), ldw=pitch(wg), stream=stream)
        return {"h": h, **({"g": g, "u": u} if case["save"] else {})}
    g, u, dh = s["g"], s["u"], s["dy"]
    dx, dwg, dwu = new(n, k), new(m, k), new(m, k)
    dbg, dbu = (new(m), new(m)) if case["bias"] else (None, None)
    xb.gated_backward_device(0, storage, n, k, m, at(dh), at(x), at(wg), at(wu), at(g), at(u),
                             activation=act, dx_ptr=at(dx), dgate_weight_ptr=at(dwg),
                             dup_weight_ptr=at(dwu), dgate_bias_ptr=at(dbg), dup_bias_ptr=at(dbu),
                             lddh=pitch(dh), ldx=pitch(x), ldw=pitch(wg), ldg=pitch(g), stream=stream)
    return {"dx": dx, "dwg": dwg, "dwu": dwu, **({"dbg": dbg, "dbu": dbu} if case["bias"] else {})}


def run(state):
    return _own(state, state["case"]) if own else _plain(state, state["case"])


def work(case):
    """Each input read once, each output written once; two operations for each term of a product."""
    size = BYTES[case["type"]]
    if case["op"] == "clip":
        return {"bytes": 2.0 * size * case["values"], "flops": 3.0 * case["values"]}
    n, k, m = case["n"], case["k"], case["m"]
    bias = m if case["bias"] else 0
    if case["op"] == "linear":
        values = n * k + m * k + n * m * (1 + case["residual"] + case["save"]) + bias
        flops = 2 * n * m * k
    elif case["op"] == "gated":
        values = n * k + 2 * m * k + n * m * (3 if case["save"] else 1) + 2 * bias
        flops = 4 * n * m * k
    elif case["op"] == "linear_backward":
        values = n * m * (1 if case["act"] == "none" else 2) + 2 * n * k + 2 * m * k + bias
        flops = 4 * n * m * k
    else:
        values = 3 * n * m + 2 * n * k + 4 * m * k + 2 * bias
        flops = 8 * n * m * k
    return {"bytes": float(size * values), "flops": float(flops)}


def exact(case, seed):
    """The definition in 64 bits: derivatives by automatic differentiation of the forward formula."""
    s = prepare(case, seed)
    if case["op"] == "clip":
        grads = [t.double() for t in s["grads"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t) for t in grads]))
        scale = min(1.0, s["max_norm"] / norm.item())
        return {"norm": norm, "clipped": [t * scale for t in grads]}

    act = {"none": lambda v: v, "relu": torch.nn.functional.relu, "gelu": torch.nn.functional.gelu,
           "silu": torch.nn.functional.silu}[case["act"]]
    s = {name: t.double() if torch.is_tensor(t) else t for name, t in s.items()}
    linear = torch.nn.functional.linear
    if case["op"] == "linear":
        z = linear(s["x"], s["wz"], s["bz"])
        y = act(z) if s["r"] is None else s["r"] + act(z)
        return {"y": y, **({"z": z} if case["save"] else {})}
    if case["op"] == "gated":
        g, u = linear(s["x"], s["wg"], s["bg"]), linear(s["x"], s["wu"], s["bu"])
        return {"h": u * act(g), **({"g": g, "u": u} if case["save"] else {})}
    # The pre-activations are given: the loss <dy, f(pre-activations)> differentiated by them.
    names = ["z"] if case["op"] == "linear_backward" else ["g", "u"]
    pre = [s[name].clone().requires_grad_() for name in names]
    with torch.enable_grad():
        value = act(pre[0]) if len(pre) == 1 else act(pre[0]) * pre[1]
        slopes = torch.autograd.grad((value * s["dy"]).sum(), pre)
    out = {"dx": sum(torch.einsum("nm,mk->nk", d, s["w" + name]) for d, name in zip(slopes, names))}
    for d, name in zip(slopes, names):
        tail = "" if name == "z" else name
        out["dw" + tail] = torch.einsum("nm,nk->mk", d, s["x"])
        if case["bias"]:
            out["db" + tail] = torch.sum(d, 0)
    return out
