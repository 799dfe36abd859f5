"""The training and serving operators beside the network's own layers, as a measurement sees them: the dense layer with
its epilogue (bias, activation, residual), that layer's gradient, and the clipping of a list of gradients by their global
norm.  Each in its plain form (elementary torch operations in 32 bits, `own = False`) and as this package offers it
(`own = True`), on cases that stand for what a detector's training step and a serving loop call.

A case is a dict of plain values; `prepare` turns it into tensors on the GPU from a seed alone, `run` makes one pass,
`exact` gives the same outputs in 64 bits straight from the definitions, `work` the bytes and operations of one pass.
"""
import importlib
import math

import torch

own = False

CLIP_NORM = 5.0          # the reference's training graph clips each tower's gradients to this global norm
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------------------- cases
def _dense(name, rows, cin, cout, dtype, act, bias=True, residual=False, preact=False):
    return {"name": name, "op": "dense", "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "preact": preact}


def _grad(name, rows, cin, cout, dtype, act, bias=True):
    return {"name": name, "op": "dense_grad", "rows": rows, "cin": cin, "cout": cout, "dtype": dtype, "act": act, "bias": bias}


def _clip(name, kind, tensors, largest, dtype, scale):
    return {"name": name, "op": "clip", "kind": kind, "tensors": tensors, "largest": largest, "dtype": dtype, "scale": scale}


def listed():
    return [
        # one token through a square projection with the block's input added: latency and the weights' bytes
        _dense("dense_token", 1, 4096, 4096, "bf16", "none", residual=True),
        # a few rows of odd widths (a small batch of proposals through a class head): nothing is aligned
        _dense("dense_few_rows", 13, 1027, 2051, "f16", "gelu", residual=True),
        # the detection head's first conv1d: 8 frames x 256 candidates, 512 -> 128 channels, fp32 as the network runs
        _dense("dense_head", 2048, 512, 128, "f32", "relu"),
        # layer 4's aggregation conv1d over 128 frames: 512 + 1024 pooled channels -> 512
        _dense("dense_aggregation", 32768, 1536, 512, "f32", "relu"),
        # a ragged batch through a widening layer in training: the pre-activation is kept for the backward pass
        _dense("dense_ragged", 5003, 771, 1283, "bf16", "gelu", residual=True, preact=True),
        # a long batch through the widening half of a feed-forward block
        _dense("dense_large", 8192, 4096, 16384, "bf16", "silu"),
        # the backward pass of the detection head's first conv1d
        _grad("grad_head", 2048, 512, 128, "f32", "relu"),
        # the backward pass of a ragged, odd layer in half precision
        _grad("grad_ragged", 5003, 771, 1283, "f16", "gelu"),
        # the backward pass of a feed-forward half over a long batch
        _grad("grad_large", 8192, 4096, 8192, "bf16", "silu"),
        # every convolution's gradient in the detector, most of them tiny: latency
        _clip("clip_detector", "detector", 0, 0, "f32", 1e-2),
        # a list of odd lengths in which each tensor has its own type
        _clip("clip_mixed", "ragged", 59, 3000001, "mixed", 1e-3),
        # a large model's gradients in bf16: the bytes
        _clip("clip_large", "blocks", 40, 16777216, "bf16", 1e-3),
    ]


_LARGEST_FLOPS = 2 * 8192 * 4096 * 16384


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A channel count: as drawn (often odd), or brought to a multiple of 8 or 64 as most layers have it."""
    n = _log_uniform(rng, lo, hi)
    m = rng.choice([1, 1, 8, 64])
    return max(m, n // m * m)


def draw(rng):
    op = rng.choice(["dense", "dense", "dense_grad", "dense_grad", "clip"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "clip":
        kind = rng.choice(["ragged", "ragged", "blocks"])
        dtype = rng.choice([dtype, "mixed"]) if kind == "ragged" else dtype
        scale = 10.0 ** rng.uniform(-5, -1)
        if kind == "blocks":
            return {"op": "clip", "kind": kind, "tensors": rng.randint(1, 20), "largest": _log_uniform(rng, 4096, 8388608),
                    "dtype": dtype, "scale": scale}
        return {"op": "clip", "kind": kind, "tensors": _log_uniform(rng, 1, 60), "largest": _log_uniform(rng, 2, 2000000),
                "dtype": dtype, "scale": scale}
    passes = 1 if op == "dense" else 2
    while True:
        rows, cin, cout = _log_uniform(rng, 1, 16384), _width(rng, 3, 6000), _width(rng, 1, 16384)
        if 2 * rows * cin * cout * passes <= _LARGEST_FLOPS // 2:
            break
    case = {"op": op, "rows": rows, "cin": cin, "cout": cout, "dtype": dtype,
            "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.8}
    if op == "dense":
        case["residual"] = rng.random() < 0.5
        case["preact"] = rng.random() < 0.3
    return case


# ------------------------------------------------------------------------------------------------------------ inputs
def _detector_shapes():
    """The weights of the KITTI configuration's set-abstraction layers, vote layer and head: a kernel per convolution, and
    a bias for those of the last layers that no batch norm follows."""
    layers = [(1, [[16, 16, 32], [16, 16, 32], [32, 32, 64]], 64), (64, [[64, 64, 128], [64, 64, 128], [64, 96, 128]], 128),
              (128, [[128, 128, 256], [128, 192, 256], [128, 256, 256]], 256), (256, [[256, 256, 512], [256, 512, 1024]], 512)]
    pairs = []
    for cin, mlps, aggregated in layers:
        for mlp in mlps:
            widths = [cin + 3] + mlp
            pairs += list(zip(widths[:-1], widths[1:]))
        pairs.append((sum(mlp[-1] for mlp in mlps), aggregated))
    pairs += [(256, 128), (128, 3), (512, 128), (128, 1), (512, 128), (128, 30)]
    return pairs + [(3,), (1,), (30,)]


def _clip_shapes(case):
    if case["kind"] == "detector":
        return _detector_shapes()
    if case["kind"] == "blocks":                   # matrices, half-size matrices and their vectors in turn
        side = max(1, math.isqrt(case["largest"]))
        cycle = [(side, side), (side,), (max(1, side // 2), side), (side,)]
        return [cycle[i % 4] for i in range(case["tensors"])]
    n, out = case["largest"], []
    for i in range(case["tensors"]):               # from the largest down to single elements, geometrically
        out.append((max(1, int(n ** (1.0 - i / case["tensors"]))) | 1,))
    return out


def _clip_type(case, i):
    if case["dtype"] == "mixed":
        return _TYPES[("f32", "bf16", "f16")[i % 3]]
    return _TYPES[case["dtype"]]


def _normal(shape, gen, scale=1.0):
    t = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return t.mul_(scale) if scale != 1.0 else t


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"case": case}
    if case["op"] == "clip":
        grads = []
        for i, shape in enumerate(_clip_shapes(case)):
            # gradients of different layers differ in size by an order of magnitude and more
            grads.append(_normal(shape, gen, case["scale"] * 10.0 ** (i % 3 - 1)).to(_clip_type(case, i)))
        state["grads"] = grads
    else:
        dt = _TYPES[case["dtype"]]
        rows, cin, cout = case["rows"], case["cin"], case["cout"]
        state["x"] = _normal((rows, cin), gen).to(dt)
        state["w"] = _normal((cin, cout), gen, math.sqrt(2.0 / cin)).to(dt)
        state["b"] = _normal((cout,), gen, 0.1).to(dt) if case["bias"] else None
        if case["op"] == "dense":
            state["residual"] = _normal((rows, cout), gen).to(dt) if case["residual"] else None
        else:
            state["g"] = _normal((rows, cout), gen, 0.05).to(dt)
            state["z"] = None
            if case["act"] != "none":              # what the forward pass kept
                z = state["x"].float() @ state["w"].float()
                state["z"] = (z if state["b"] is None else z + state["b"].float()).to(dt)
    if own:
        state["dense"] = importlib.import_module("3dssd_amd.utils.tf_ops.dense.tf_dense")
        state["clip"] = importlib.import_module("3dssd_amd.utils.tf_ops.gradients.tf_gradients")
    return state


# ------------------------------------------------------------------------------------------------- plain form, 32 bits
def _act32(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope32(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        return 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if act == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        s = 1.0 / (1.0 + torch.exp(-c * (z + 0.044715 * z * z * z)))
        return s + z * s * (1.0 - s) * c * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s + z * s * (1.0 - s)


def _plain(state):
    case = state["case"]
    if case["op"] == "clip":
        grads = state["grads"]
        total = torch.zeros((), dtype=torch.float64, device="cuda")
        for g in grads:
            total = total + (g.double() * g.double()).sum()
        norm = torch.sqrt(total).float()
        scale = CLIP_NORM / torch.clamp(norm, min=CLIP_NORM)
        return {"clipped": [(g.float() * scale).to(g.dtype) for g in grads], "norm": norm}
    x, w, b = state["x"], state["w"], state["b"]
    if case["op"] == "dense":
        z = x.float() @ w.float()
        if b is not None:
            z = z + b.float()
        y = _act32(z, case["act"])
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return {"out": y.to(x.dtype), "preact": z.to(x.dtype)} if case["preact"] else {"out": y.to(x.dtype)}
    dz = state["g"].float()
    if case["act"] != "none":
        dz = dz * _act_slope32(state["z"].float(), case["act"])
    out = {"inputs": (dz @ w.float().t()).to(x.dtype), "weights": (x.float().t() @ dz).to(x.dtype)}
    if b is not None:
        out["biases"] = dz.sum(0).to(x.dtype)
    return out


# ------------------------------------------------------------------------------------------------- the package's calls
def _own(state):
    case = state["case"]
    if case["op"] == "clip":
        clipped, norm = state["clip"].clip_by_global_norm(state["grads"], CLIP_NORM)
        return {"clipped": clipped, "norm": norm}
    act = None if case["act"] == "none" else case["act"]
    if case["op"] == "dense":
        got = state["dense"].dense(state["x"], state["w"], state["b"], activation=act, residual=state["residual"],
                                   return_preact=case["preact"])
        return {"out": got[0], "preact": got[1]} if case["preact"] else {"out": got}
    dx, dw, db = state["dense"].dense_grad(state["x"], state["w"], state["g"], biases=state["b"], activation=act,
                                           preact=state["z"])
    out = {"inputs": dx, "weights": dw}
    if state["b"] is not None:
        out["biases"] = db
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------- 64 bits
def _phi64(z):
    return torch.special.ndtr(z)                    # the normal distribution's integral


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(math.fsum(float(g.double().pow(2).sum()) for g in state["grads"]))
        factor = min(1.0, CLIP_NORM / norm) if norm else 1.0
        return {"clipped": [g.double() * factor for g in state["grads"]],
                "norm": torch.tensor(norm, dtype=torch.float64, device="cuda")}
    act = case["act"]
    x, w = state["x"].double(), state["w"].double()
    if case["op"] == "dense":
        z = torch.mm(x, w)
        if state["b"] is not None:
            z += state["b"].double()
        y = {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: z * _phi64(z),
             "gelu_tanh": lambda: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
             "silu": lambda: z * torch.sigmoid(z)}[act]()
        if state["residual"] is not None:
            y = y + state["residual"].double()
        return {"out": y, "preact": z} if case["preact"] else {"out": y}
    d = state["g"].double()
    if act != "none":
        z = state["z"].double()
        if act == "relu":
            d = torch.where(z > 0, d, 0.0)
        elif act == "gelu":
            d = d * (_phi64(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        elif act == "gelu_tanh":
            t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
            d = d * (0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2))
        else:
            s = torch.sigmoid(z)
            d = d * (s * (1 + z * (1 - s)))
    out = {"inputs": torch.mm(d, w.t().contiguous()), "weights": torch.mm(x.t().contiguous(), d)}
    if state["b"] is not None:
        out["biases"] = d.sum(0)
    return out


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "clip":
        n = size = 0
        for i, shape in enumerate(_clip_shapes(case)):
            n += math.prod(shape)
            size += math.prod(shape) * _clip_type(case, i).itemsize
        return {"bytes": 2 * size + 4, "flops": 3 * n}
    e = _TYPES[case["dtype"]].itemsize
    rows, cin, cout = case["rows"], case["cin"], case["cout"]
    one = rows * cout
    if case["op"] == "dense":
        n = rows * cin + cin * cout + one + (cout if case["bias"] else 0)
        n += (one if case["residual"] else 0) + (one if case["preact"] else 0)
        return {"bytes": n * e, "flops": 2 * rows * cin * cout}
    n = 2 * rows * cin + 2 * cin * cout + one + (one if case["act"] != "none" else 0) + (cout if case["bias"] else 0)
    return {"bytes": n * e, "flops": 4 * rows * cin * cout}
