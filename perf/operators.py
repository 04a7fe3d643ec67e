"""What surrounds the attention of an encoder layer, as measurable cases.

Four kinds, each through the package's op layer:

* ``norm``   ``ops.residual_norm`` in inference: the norm after a block, its gate, the scaled residual and the norm before the
             next block in one pass over the rows;
* ``train``  the same with its backward: gradients of the rows, the residual, the gate and both norms' parameters;
* ``int8``   ``ops.linear_int8``: a linear layer whose weight is held in 8-bit integers with a scale per output channel, over
             tokens that are scaled and rounded to 8 bits one by one, with bias and, in the first half of a feed-forward block,
             the erf GELU;
* ``clip``   ``ops.clip_grads_``: the norm over the gradients of all parameters and the gradients scaled by it.
"""
import math

import numpy as np
import torch

own = False  # true: the package's operators, false: their plain form

EPS = 1e-7
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GATES = ("none", "channel", "sequence", "element")


def listed():
    return [
        # one token of a stream: latency of a call is all there is
        {"name": "norm_token", "kind": "norm", "dtype": "bf16", "batch": 1, "seqlen": 1, "hidden": 1024, "rms": True, "post": True,
         "gate": "channel", "scale": 1.0},
        # serving a full batch of the large model, block output scaled per sequence
        {"name": "norm_batch", "kind": "norm", "dtype": "bf16", "batch": 8, "seqlen": 2048, "hidden": 1024, "rms": False, "post": True,
         "gate": "sequence", "scale": 1.0},
        # fine-tuning in half precision on ragged paragraphs packed into one row, a width that no vector divides
        {"name": "train_ragged", "kind": "train", "dtype": "fp16", "batch": 1, "seqlen": 4099, "hidden": 769, "rms": False, "post": False,
         "gate": "channel", "scale": 1.25},
        # pre-training of a deep model: norms on both sides of the block and a gate per sequence
        {"name": "train_batch", "kind": "train", "dtype": "bf16", "batch": 16, "seqlen": 2048, "hidden": 1024, "rms": True, "post": True,
         "gate": "sequence", "scale": 1.0},
        # the tail of this encoder's own blocks (residual and LayerNorm) in single precision, with the residual weighted
        {"name": "train_single", "kind": "train", "dtype": "fp32", "batch": 4, "seqlen": 2048, "hidden": 768, "rms": False, "post": False,
         "gate": "none", "scale": 1.5},
        # one token through the first half of the large model's feed-forward block
        {"name": "int8_token", "kind": "int8", "dtype": "bf16", "rows": 1, "k": 1024, "n": 4096, "bias": True, "gelu": True, "given": False},
        # a search query of 29 tokens through a projection
        {"name": "int8_query", "kind": "int8", "dtype": "fp16", "rows": 29, "k": 768, "n": 768, "bias": True, "gelu": False, "given": False},
        # a classifier's or a retriever's projection of odd sizes, single precision in and out
        {"name": "int8_ragged", "kind": "int8", "dtype": "fp32", "rows": 3001, "k": 1001, "n": 1537, "bias": False, "gelu": False, "given": False},
        # a full batch through the first half of the feed-forward block
        {"name": "int8_batch", "kind": "int8", "dtype": "bf16", "rows": 16384, "k": 1024, "n": 4096, "bias": True, "gelu": True, "given": False},
        # the second half, over tokens that the caller holds in 8 bits already
        {"name": "int8_given", "kind": "int8", "dtype": "bf16", "rows": 16384, "k": 4096, "n": 1024, "bias": True, "gelu": False, "given": True},
        # a small encoder's gradients of mixed types, within the bound as in most steps: the norm is all that changes hands
        {"name": "clip_within", "kind": "clip", "dtype": "mixed", "layers": 2, "hidden": 257, "ffn": 515, "vocab": 1009, "bound": 2.0, "out": "same"},
        # the large model's gradients in bf16, clipped into the single-precision buffers that its optimizer reads
        {"name": "clip_large", "kind": "clip", "dtype": "bf16", "layers": 24, "hidden": 1024, "ffn": 4096, "vocab": 128100, "bound": 0.1, "out": "fp32"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the same ranges."""
    kind = rng.choice(("norm", "train", "int8", "int8", "clip"))
    if kind in ("norm", "train"):
        hidden = _spread(rng, 64, 4096)
        if rng.random() < 0.6:
            hidden = (hidden + 15) // 16 * 16
        rows = min(_spread(rng, 1, 16384), (32 << 20) // hidden)
        batch = rng.choice([b for b in (1, 2, 4, 7, 16) if b <= rows])
        return {"kind": kind, "dtype": rng.choice(("bf16", "fp16", "fp32") if kind == "train" else ("bf16", "bf16", "fp16", "fp32")),
                "batch": batch, "seqlen": rows // batch, "hidden": hidden, "rms": rng.random() < 0.5, "post": rng.random() < 0.5,
                "gate": rng.choice(GATES), "scale": round(rng.uniform(0.5, 2.0), 3)}
    if kind == "int8":
        k, n = _spread(rng, 64, 4096), _spread(rng, 64, 4096)
        if rng.random() < 0.6:
            k, n = (k + 63) // 64 * 64, (n + 63) // 64 * 64
        return {"kind": kind, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "rows": _spread(rng, 1, 16384), "k": k, "n": n,
                "bias": rng.random() < 0.7, "gelu": rng.random() < 0.4, "given": rng.random() < 0.3}
    hidden = _spread(rng, 32, 1024)
    return {"kind": kind, "dtype": rng.choice(("bf16", "fp32", "mixed")), "layers": rng.randint(1, 12), "hidden": hidden,
            "ffn": hidden * 4 + rng.randint(0, 3), "vocab": _spread(rng, 100, 30000), "bound": rng.choice((0.1, 0.7, 2.0)), "out": "fp32"}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype=None):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype or TYPES[case["dtype"]])

    if case["kind"] in ("norm", "train"):
        return _prepare_norm(case, normal, gen)
    if case["kind"] == "int8":
        return _prepare_int8(case, normal)
    return _prepare_clip(case, normal)


def _prepare_norm(case, normal, gen):
    b, s, h = case["batch"], case["seqlen"], case["hidden"]
    channels = torch.exp(torch.randn(h, generator=gen, device="cuda") * 0.5)  # activations differ from channel to channel
    t = {"x": (normal(b, s, h).float() * channels).to(TYPES[case["dtype"]]),
         "residual": (normal(b, s, h, std=2.0).float() * channels + 0.1).to(TYPES[case["dtype"]]),
         "weight": normal(h, std=0.2, mean=1.0)}
    if not case["rms"]:
        t["bias"] = normal(h, std=0.2)
    if case["post"]:
        t["post_weight"] = normal(h, std=0.2, mean=1.0)
        if not case["rms"]:
            t["post_bias"] = normal(h, std=0.2)
    shape = {"channel": (h,), "sequence": (b, 1, h), "element": (b, s, h)}.get(case["gate"])
    if shape is not None:
        t["gate"] = normal(*shape, std=0.3, mean=0.5)
    state = {"case": case, "tensors": t}
    if case["kind"] == "train":
        state["grads"] = (normal(b, s, h), normal(b, s, h, std=0.5))  # of the normalised rows and of the stream
        if own:
            for v in t.values():
                v.requires_grad_()
    return state


def _int8_rows(x):
    """Rows as 8-bit integers and the scale of each: the largest magnitude becomes 127, whole numbers by rounding to the
    nearest, ties to even, of the product with the reciprocal scale in single precision."""
    x = x.float()
    top = x.abs().amax(dim=-1, keepdim=True)
    most = torch.full_like(top, 127.0)  # (divided by as a tensor: torch multiplies by the reciprocal of a number)
    inverse = torch.where(top > 0, most / top, torch.zeros_like(top))
    return torch.round(x * inverse).to(torch.int8), (top / most).squeeze(-1)


def _prepare_int8(case, normal):
    rows, k, n = case["rows"], case["k"], case["n"]
    weight, weight_scale = _int8_rows(normal(n, k, std=0.02, dtype=torch.float32))
    state = {"case": case, "x": normal(rows, k), "x_scale": None, "bias": normal(n, std=0.1) if case["bias"] else None,
             "weight": weight, "weight_scale": weight_scale}
    if case["given"]:
        state["x"], state["x_scale"] = _int8_rows(state["x"])
    if own:  # the layout that a program keeps its weight in
        from flashdeberta_b200 import ops
        state["weight"] = ops.int8_rows(weight)
    return state


def _shapes(case):
    """Shapes of an encoder's parameters."""
    h, f = case["hidden"], case["ffn"]
    layer = [(h, h), (h,)] * 4 + [(h,), (h,), (f, h), (f,), (h, f), (h,), (h,), (h,)]
    return [(case["vocab"], h), (h,), (h,), (512, h), (h,), (h,)] + layer * case["layers"]


def _prepare_clip(case, normal):
    types = {"mixed": (torch.float32, torch.bfloat16, torch.float16)}.get(case["dtype"]) or (TYPES[case["dtype"]],)
    shapes = _shapes(case)
    total = math.sqrt(sum(math.prod(s) for s in shapes))
    # gradients of about unit norm; the norms' parameters and the biases have the larger ones
    grads = [normal(*s, std=(3.0 if len(s) == 1 else 1.0) / total, dtype=types[i % len(types)]) for i, s in enumerate(shapes)]
    flat = out = None
    if case["out"] != "same":  # an optimizer's buffer: all gradients end to end
        flat = torch.empty(sum(g.numel() for g in grads), dtype=TYPES[case["out"]], device="cuda")
        out = [o.view_as(g) for o, g in zip(flat.split([g.numel() for g in grads]), grads)]
    return {"case": case, "grads": grads, "out": out, "flat": flat}


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from flashdeberta_b200 import ops
    case = state["case"]
    if case["kind"] in ("norm", "train"):
        t = state["tensors"]
        normed, stream = ops.residual_norm(
            t["x"], t["residual"], t["weight"], t.get("bias"), EPS, rms=case["rms"], post_weight=t.get("post_weight"),
            post_bias=t.get("post_bias"), gate=t.get("gate"), residual_scale=case["scale"])
        if case["kind"] == "norm":
            return normed, stream
        return (normed, stream, *torch.autograd.grad((normed, stream), tuple(t.values()), state["grads"]))
    if case["kind"] == "int8":
        return ops.linear_int8(state["x"], state["weight"], state["weight_scale"], state["bias"], x_scale=state["x_scale"],
                               gelu=case["gelu"], out_dtype=TYPES[case["dtype"]])
    norm = ops.clip_grads_(state["grads"], case["bound"], out=state["out"])
    return [norm, *(state["grads"] if state["out"] is None else [state["flat"]])]


def _run_plain(state):
    case = state["case"]
    if case["kind"] in ("norm", "train"):
        return _plain_norm(state)
    if case["kind"] == "int8":
        return _plain_int8(state)
    squares = torch.stack([(g.double() * g.double()).sum() for g in state["grads"]])
    norm = squares.sum().sqrt()
    factor = (case["bound"] / (norm + 1e-6)).clamp(max=1.0).float()
    if state["out"] is None:
        for g in state["grads"]:
            g.copy_(g.float() * factor)
        return [norm.float(), *state["grads"]]
    for g, o in zip(state["grads"], state["out"]):
        o.copy_(g.float() * factor)
    return norm.float(), state["flat"]


def _plain_normalise(x, rms, weight, bias):
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    return x if bias is None else x + bias


def _plain_norm(state):
    case, train = state["case"], state["case"]["kind"] == "train"
    given = state["tensors"]
    t = {k: v.float().detach().requires_grad_(train) for k, v in given.items()}
    u = t["x"] if not case["post"] else _plain_normalise(t["x"], case["rms"], t["post_weight"], t.get("post_bias"))
    if "gate" in t:
        u = t["gate"] * u
    stream = case["scale"] * t["residual"] + u
    normed = _plain_normalise(stream, case["rms"], t["weight"], t.get("bias"))
    kind = TYPES[case["dtype"]]
    if not train:
        return normed.to(kind), stream.to(kind)
    grads = torch.autograd.grad((normed, stream), tuple(t.values()), tuple(g.float() for g in state["grads"]))
    return (normed.detach().to(kind), stream.detach().to(kind), *(g.to(kind) for g in grads))


def _plain_int8(state):
    case = state["case"]
    x, scale = (state["x"], state["x_scale"]) if case["given"] else _int8_rows(state["x"])
    out = (x.float() @ state["weight"].float().t()) * state["weight_scale"] * scale[:, None]
    if state["bias"] is not None:
        out = out + state["bias"].float()
    if case["gelu"]:
        out = out * 0.5 * torch.erfc(out * -math.sqrt(0.5))
    return out.to(TYPES[case["dtype"]])


# ---- the operators from their definitions, in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    global own
    before, own = own, False  # the inputs alone
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["kind"] in ("norm", "train"):
        return _exact_norm(case, state)
    if case["kind"] == "int8":
        return _exact_int8(case, state)
    total = sum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in state["grads"])
    norm = math.sqrt(total)
    factor = min(1.0, case["bound"] / (norm + 1e-6))
    scaled = [g.double() * factor for g in state["grads"]]
    if state["out"] is not None:
        scaled = [torch.cat([g.flatten() for g in scaled])]
    return [torch.tensor(norm, dtype=torch.float64), *scaled]


def _exact_norm(case, state):
    t = {k: v.double() for k, v in state["tensors"].items()}
    h, one = case["hidden"], torch.ones((), dtype=torch.float64, device="cuda")

    def statistics(x):
        mean = torch.zeros_like(x[..., :1]) if case["rms"] else x.sum(-1, keepdim=True) / h
        inverse = 1.0 / torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / h + EPS)
        return (x - mean) * inverse, inverse

    def through(g, hat, inverse):  # gradient of the rows from that of their normalised form
        g = g - hat * ((g * hat).sum(-1, keepdim=True) / h) - (0.0 if case["rms"] else g.sum(-1, keepdim=True) / h)
        return g * inverse

    if case["post"]:
        hat1, inverse1 = statistics(t["x"])
        u = hat1 * t["post_weight"] + t.get("post_bias", 0.0)
    else:
        u = t["x"]
    gate = t.get("gate", one)
    stream = case["scale"] * t["residual"] + gate * u
    hat2, inverse2 = statistics(stream)
    normed = hat2 * t["weight"] + t.get("bias", 0.0)
    if case["kind"] == "norm":
        return normed, stream
    d_normed, d_stream = (g.double() for g in state["grads"])
    rows = (0, 1)
    dz = d_stream + through(d_normed * t["weight"], hat2, inverse2)
    du = dz * gate
    grads = {"residual": case["scale"] * dz, "weight": (d_normed * hat2).sum(rows), "bias": d_normed.sum(rows),
             "x": through(du * t["post_weight"], hat1, inverse1) if case["post"] else du}
    if case["post"]:
        grads["post_weight"], grads["post_bias"] = (du * hat1).sum(rows), du.sum(rows)
    if "gate" in t:
        summed = {"channel": rows, "sequence": (1,), "element": ()}[case["gate"]]
        dg = dz * u
        grads["gate"] = (dg.sum(summed) if summed else dg).reshape(t["gate"].shape)
    return (normed, stream, *(grads[k] for k in t))


def _exact_int8(case, state):
    if case["given"]:
        q, scale = state["x"].double(), state["x_scale"].double()
    else:  # the rounding to 8 bits is part of the definition, its single-precision steps included
        x = state["x"].float().cpu().numpy()
        top = np.abs(x).max(axis=1, keepdims=True)
        inverse = np.float32(127.0) / top
        q = torch.from_numpy(np.rint(x * inverse).astype(np.float64)).cuda()
        scale = torch.from_numpy((top[:, 0] / np.float32(127.0)).astype(np.float64)).cuda()
    out = torch.einsum("mk,nk->mn", q, state["weight"].double()) * state["weight_scale"].double() * scale[:, None]
    if state["bias"] is not None:
        out = out + state["bias"].double()
    if case["gelu"]:
        out = 0.5 * out * torch.special.erfc(-out / math.sqrt(2.0))
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4, "mixed": 8 / 3}[case["dtype"]]
    if case["kind"] in ("norm", "train"):
        rows, h = case["batch"] * case["seqlen"], case["hidden"]
        gate = {"none": 0, "channel": h, "sequence": case["batch"] * h, "element": rows * h}[case["gate"]]
        vectors = (1 if case["rms"] else 2) * (2 if case["post"] else 1) * h
        items = 4 * rows * h + gate + vectors  # x and residual read, both results written
        flops = (24 if case["post"] else 16) * rows * h
        if case["kind"] == "train":  # two gradients read, two written, x and residual read again
            items += 6 * rows * h + 2 * gate + 2 * vectors
            flops *= 3
        return {"bytes": size * items, "flops": flops}
    if case["kind"] == "int8":
        rows, k, n = case["rows"], case["k"], case["n"]
        read = rows * k * (1 if case["given"] else size) + (4 * rows if case["given"] else 0) + n * k + 4 * n
        return {"bytes": read + (size * n if case["bias"] else 0) + size * rows * n, "flops": 2 * rows * k * n}
    count = sum(math.prod(s) for s in _shapes(case))
    written = 0 if case["out"] == "same" else count * {"fp32": 4, "bf16": 2}[case["out"]]
    return {"bytes": size * count + written, "flops": 3 * count}
