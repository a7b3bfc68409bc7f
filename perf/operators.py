"""Performance cases of the 4-bit microscaled weights, through the package's public entry points.

The format is OCP MXFP4: blocks of 32 values along a row share a power-of-two scale (E8M0: one byte, 2^(byte - 127)), each
value is a 4-bit float (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign).  Three kinds of work, as a program that converts,
serves or fine-tunes such a model has them:

  quantise  a dense matrix of any float type to the format and back to BF16: ``MXFP4Weight.compress`` and ``get_weight``
  linear    y = x W^T + b on such a weight (``F.linear``), for one token to a long prompt; with ``train`` the gradient of x too
  gated     act(x G^T) * (x U^T) on a stacked weight [G; U] (``gated_mxfp4``); with ``train`` the gradient of x too

Weights are N(0, 0.02), activations N(0, 1) with a few channels twenty times as large, as decoder models have them.
"""
from __future__ import annotations

import math
import random

import torch
import torch.nn.functional as F

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a key or value projection quantised as a model is converted on its device: the smallest call
        {"name": "quantise_kv", "kind": "quantise", "m": 1024, "k": 4096, "dtype": "bf16"},
        # a gate projection of an FP32 checkpoint
        {"name": "quantise_gate_fp32", "kind": "quantise", "m": 12288, "k": 4096, "dtype": "fp32"},
        # a vocabulary-sized layer with a ragged row count, FP16 weights
        {"name": "quantise_ragged_fp16", "kind": "quantise", "m": 32003, "k": 2560, "dtype": "fp16"},
        # a key or value projection, one sequence: the launch is most of the time
        {"name": "linear_kv_1row", "kind": "linear", "m": 1024, "k": 4096, "rows": 1, "bias": False, "train": False},
        # stacked q/k/v of a 3584-wide model with its bias, three sequences
        {"name": "linear_qkv_bias_3rows", "kind": "linear", "m": 4608, "k": 3584, "rows": 3, "bias": True, "train": False},
        # an output head over 151936 tokens, eight sequences: the largest matrix of a model
        {"name": "linear_head_8rows", "kind": "linear", "m": 151936, "k": 4096, "rows": 8, "bias": False, "train": False},
        # odd sizes all over: outputs, a row length that is a multiple of 32 only, a ragged batch of short prompts
        {"name": "linear_odd_77rows", "kind": "linear", "m": 5003, "k": 2080, "rows": 77, "bias": True, "train": False},
        # down projection over a prompt of 2048 tokens
        {"name": "linear_down_prompt", "kind": "linear", "m": 4096, "k": 12288, "rows": 2048, "bias": False, "train": False},
        # an output projection while adapters are trained: the product and the gradient of its input
        {"name": "linear_train", "kind": "linear", "m": 4096, "k": 4096, "rows": 1000, "bias": False, "train": True},
        # gate and up projection of an 8B model's block, one token
        {"name": "gated_8b_1row", "kind": "gated", "m": 12288, "k": 4096, "rows": 1, "bias": False, "act": "silu", "train": False},
        # the same of a 7B model for sixteen sequences
        {"name": "gated_7b_16rows", "kind": "gated", "m": 18944, "k": 3584, "rows": 16, "bias": False, "act": "gelu_tanh", "train": False},
        # an 8B model's block in training, forward and backward: the most arithmetic
        {"name": "gated_train", "kind": "gated", "m": 12288, "k": 4096, "rows": 2048, "bias": False, "act": "silu", "train": True},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quantise", "linear", "linear", "gated"])
    k = 32 * _log_int(rng, 2, 18944 // 32)
    if kind == "quantise":
        m = min(_log_int(rng, 1, 152000), 50_000_000 // k)
        return {"kind": kind, "m": m, "k": k, "dtype": rng.choice(sorted(TYPES))}
    m = _log_int(rng, 64, 30000) if kind == "linear" else _log_int(rng, 64, 19000)
    m = min(m, 80_000_000 // k)
    train = rng.random() < 0.3
    rows = _log_int(rng, 1, 4096)
    most = 50_000_000_000 if kind == "gated" else 100_000_000_000                     # rows * m * k of the largest call
    rows = max(1, min(rows, most // (m * k), 40_000_000 // m))
    case = {"kind": kind, "m": m, "k": k, "rows": rows, "bias": rng.random() < 0.4, "train": train}
    if kind == "gated":
        case["act"] = rng.choice(["silu", "gelu", "gelu_tanh"])
    return case


# ---- the plain form ----------------------------------------------------------------------------------------------

def _quantise(x):
    """Codes (u8, a value each, sign in bit 3) and scale bytes of the rows of x.  Double precision: scaling by powers of two is
    then exact for every float type, subnormal values included."""
    m, k = x.shape
    v = x.double().view(m, k // 32, 32)
    top = v.abs().amax(-1)
    byte = (torch.frexp(top).exponent - 3 + 127).clamp(0, 254)                       # floor(log2(top)) - 2
    byte = torch.where(top == 0, 0, byte)
    a = torch.ldexp(v.abs(), (127 - byte)[..., None])
    # steps of 0.5 below 2, of 1 below 4, of 2 above; torch.round takes ties to even
    a = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code += torch.signbit(v).to(torch.uint8) * 8
    return code.view(m, k), byte.to(torch.uint8)


def _pack(code):
    """Two codes a byte, the first in the low half: how checkpoints of the format hold them."""
    return code[:, 0::2] + code[:, 1::2] * 16


def _dense(codes, scales):
    """The FP32 values of packed codes and scale bytes."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float32, device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(1).int()
    v = table[code].view(codes.shape[0], -1, 32)
    return torch.ldexp(v, (scales.int() - 127)[..., None]).flatten(1)


def _activation(g, act):
    """act(g) and its derivative, in g's type."""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * 0.044715 * g * g)


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "quantise":
        code, byte = _quantise(state["x"])
        return {"values": _dense(_pack(code), byte).to(torch.bfloat16)}
    w = _dense(state["codes"], state["scales"])
    x = state["x"].float()
    y = x @ w.T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if case["kind"] == "linear":
        out = {"y": y.to(torch.bfloat16)}
        if case["train"]:
            out["dx"] = (state["dy"].float() @ w).to(torch.bfloat16)
        return out
    g, u = y[:, :case["m"]], y[:, case["m"]:]
    a, da = _activation(g, case["act"])
    out = {"h": (a * u).to(torch.bfloat16)}
    if case["train"]:
        dh = state["dy"].float()
        out["dx"] = (torch.cat([dh * u * da, dh * a], 1) @ w).to(torch.bfloat16)
    return out


# ---- what the tools call -------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """Everything a case starts from, by the seed alone."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    m, k = case["m"], case["k"]
    if case["kind"] == "quantise":
        return {"x": (normal(m, k) * 0.02).to(TYPES[case["dtype"]])}
    rows = m if case["kind"] == "linear" else 2 * m
    step = max(1, (1 << 26) // k)
    parts = [_quantise((normal(min(step, rows - r), k) * 0.02).to(torch.bfloat16)) for r in range(0, rows, step)]
    d = {"codes": torch.cat([_pack(c) for c, _ in parts]), "scales": torch.cat([s for _, s in parts])}
    x = normal(case["rows"], k)
    x[:, torch.randint(0, k, (max(1, k // 1000),), device=dev, generator=gen)] *= 20
    d["x"] = x.to(torch.bfloat16)
    d["bias"] = (normal(rows) * 0.1).to(torch.bfloat16) if case["bias"] else None
    d["dy"] = normal(case["rows"], m).to(torch.bfloat16) if case["train"] else None
    return d


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own and case["kind"] != "quantise":
        from bf16_huffman_infer_b200 import MXFP4Weight
        state["weight"] = MXFP4Weight.from_packed(state["codes"], state["scales"])     # as a checkpoint is loaded
        if case["train"]:
            state["x"].requires_grad_()
    return state


def run(state):
    if not own:
        with torch.no_grad():
            return _run_plain(state)
    from bf16_huffman_infer_b200 import MXFP4Weight, gated_mxfp4
    case = state["case"]
    if case["kind"] == "quantise":
        return {"values": MXFP4Weight.compress(state["x"], to_cpu=False).get_weight()}
    if case["kind"] == "linear":
        name, y = "y", F.linear(state["x"], state["weight"], state["bias"])
    else:
        name, y = "h", gated_mxfp4(state["x"], state["weight"], state["bias"], activation=case["act"])
    if not case["train"]:
        return {name: y}
    dx, = torch.autograd.grad(y, state["x"], state["dy"])
    return {name: y.detach(), "dx": dx}


def work(case):
    m, k = case["m"], case["k"]
    if case["kind"] == "quantise":
        size = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
        return {"bytes": m * k * (size + 2) + m * k // 2 + m * k // 32, "flops": 4 * m * k}
    outs = m if case["kind"] == "linear" else 2 * m
    stored = outs * k // 2 + outs * k // 32 + (2 * outs if case["bias"] else 0)
    rows = case["rows"]
    passes = 2 if case["train"] else 1
    # forward: x and the weight in, the result out; backward: its gradient in, that of x out (the weight is counted once)
    return {"bytes": stored + passes * 2 * rows * (k + m), "flops": passes * 2 * rows * outs * k}


def exact(case, seed):
    """The definitions in double precision: the nearest value of the grid (ties to the even code) and sums of products."""
    d = _inputs(case, seed)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    if case["kind"] == "quantise":
        out = torch.empty(d["x"].shape, dtype=torch.float64, device="cuda")
        edges = (grid[1:] + grid[:-1]) / 2
        step = max(1, (1 << 24) // case["k"])
        for r in range(0, case["m"], step):
            v = d["x"][r:r + step].double().unflatten(1, (-1, 32))
            scale = torch.exp2(torch.floor(torch.log2(v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -125))) - 2)
            a = v.abs() / scale
            up = torch.bucketize(a, edges, right=True)              # an edge goes up ...
            tie = (a[..., None] == edges[0::2]).any(-1)             # ... but from an even code it stays
            out[r:r + step] = (grid[up - tie.int()] * scale * torch.sign(v)).flatten(1)
        return {"values": out}
    byte = d["scales"].double().repeat_interleave(32, 1)
    low, high = torch.remainder(d["codes"].int(), 16), torch.div(d["codes"].int(), 16, rounding_mode="floor")
    code = torch.empty(byte.shape, dtype=torch.int32, device="cuda")
    code[:, 0::2], code[:, 1::2] = low, high
    w = torch.where(code > 7, -1.0, 1.0).double() * grid[torch.remainder(code, 8)] * torch.exp2(byte - 127)
    y = d["x"].double().matmul(w.mT)
    if d["bias"] is not None:
        y += d["bias"].double()
    if case["kind"] == "linear":
        return {"y": y, "dx": d["dy"].double().matmul(w)} if case["train"] else {"y": y}
    g, u = y.chunk(2, 1)
    if case["act"] == "silu":
        s = torch.sigmoid(g)
        a, da = g * s, s + g * s * (1 - s)
    elif case["act"] == "gelu":
        s = torch.special.ndtr(g)
        a, da = g * s, s + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    else:
        z, dz = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3), math.sqrt(2 / math.pi) * (1 + 0.134145 * g ** 2)
        s = torch.sigmoid(2 * z)                                   # (1 + tanh z) / 2
        a, da = g * s, s + 2 * g * s * (1 - s) * dz
    if not case["train"]:
        return {"h": a * u}
    dh = d["dy"].double()
    return {"h": a * u, "dx": (dh * u * da).matmul(w[:case["m"]]) + (dh * a).matmul(w[case["m"]:])}
