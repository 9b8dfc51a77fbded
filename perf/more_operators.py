"""Steps over rows held in 8 bits, as cases that can be timed and checked.

  norm      a residual stream's next rms_norm: the rows a product left are added to
            the stream, the sum normed and weighted, and what comes out held in 8
            bits with a scale per row, then read back (rms_norm_row8, row8_read)
  quantize  rows of an attention or SwiGLU output held in 8 bits, and read back
            (row8_quantize, row8_read)
  product   rows held in 8 bits times a Q8_0 matrix, with bias, activation and
            residual in its epilogue (Q8Weights.matmul)
  gated     the same with two matrices, act(gate) * up (Q8Weights over both)

A row y is held as int8 codes and one fp32 scale: with a = max|y|, scale =
fp32(a / 127), code = rint(y * fp32(127 / a)), the product taken exactly; rows with
a < 2^-100 are zeros.  y is fp32: rms_norm's is the fp32 number nearest to
h * weight / sqrt(mean(h^2) + eps), h = fp32(x + residual).

A Q8_0 matrix is d rows of n / 32 blocks of {fp32 scale; int8 q[32]} (36 bytes).
Its codes here are uniform and its scales about 1 / (127 sqrt(n)); activations are
N(0, 1) with a few channels that are larger throughout, as a trained model's are.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # one user's token through a 7B-shaped model's layer: latency is everything
        {"name": "norm_1_4096", "kind": "norm", "rows": 1, "n": 4096, "residual": True},
        # a serving step's rows, a width that no vector divides, no residual
        {"name": "norm_333_5003", "kind": "norm", "rows": 333, "n": 5003, "residual": False},
        # prompts through a 7B-shaped model's layer: bytes are everything
        {"name": "norm_8192_4096", "kind": "norm", "rows": 8192, "n": 4096, "residual": True},
        # a decode batch's SwiGLU rows on their way to w2
        {"name": "quantize_8_11008", "kind": "quantize", "rows": 8, "n": 11008},
        # prompts' attention rows of a small model on their way to wo
        {"name": "quantize_5520_768", "kind": "quantize", "rows": 5520, "n": 768},
        # one user's wo with the stream added: the matrix's bytes are everything
        {"name": "product_1_4096x4096", "kind": "product", "rows": 1, "n": 4096, "d": 4096, "bias": False,
         "activation": "none", "residual": True},
        # a serving batch's w2 of a small model
        {"name": "product_32_2048x768", "kind": "product", "rows": 32, "n": 2048, "d": 768, "bias": False,
         "activation": "none", "residual": True},
        # a layer with biases at sizes that no tile divides
        {"name": "product_77_1056x1003", "kind": "product", "rows": 77, "n": 1056, "d": 1003, "bias": True,
         "activation": "gelu", "residual": False},
        # prompts' w2 of a 7B-shaped model: products are everything
        {"name": "product_4096_11008x4096", "kind": "product", "rows": 4096, "n": 11008, "d": 4096, "bias": True,
         "activation": "none", "residual": True},
        # a serving batch's w1 and w3 of a 7B-shaped model
        {"name": "gated_8_4096x11008", "kind": "gated", "rows": 8, "n": 4096, "d": 11008, "bias": False,
         "activation": "silu", "residual": False},
        # ragged prompts of a small model
        {"name": "gated_333_768x2048", "kind": "gated", "rows": 333, "n": 768, "d": 2048, "bias": False,
         "activation": "silu", "residual": False},
        # prompts' w1 and w3 of a 7B-shaped model
        {"name": "gated_1024_4096x11008", "kind": "gated", "rows": 1024, "n": 4096, "d": 11008, "bias": True,
         "activation": "gelu_tanh", "residual": False},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        case = {"kind": rng.choice(["norm", "quantize", "product", "product", "gated"])}
        if case["kind"] in ("norm", "quantize"):
            case["rows"] = _log_int(rng, 1, 16384)
            case["n"] = _log_int(rng, 32, 65536)
            if rng.random() < 0.5:  # widths of models
                case["n"] = (case["n"] + 63) // 64 * 64
            if case["kind"] == "norm":
                case["residual"] = rng.random() < 0.6
            if work(case)["bytes"] <= 6e8:
                return case
            continue
        case["rows"] = _log_int(rng, 1, 8192)
        case["n"] = _log_int(rng, 1, 512) * BLOCK
        case["d"] = _log_int(rng, 16, 16384)
        if rng.random() < 0.6:
            case["d"] = (case["d"] + 63) // 64 * 64
        case["bias"] = rng.random() < 0.4
        case["activation"] = rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])
        case["residual"] = rng.random() < 0.4
        if work(case)["flops"] <= 3.6e11:
            return case


def work(case):
    rows, n = case["rows"], case["n"]
    if case["kind"] in ("norm", "quantize"):  # x in, codes out, codes in, values out (residual in, sum out)
        more = 8 if case.get("residual") else 0
        return {"bytes": rows * n * (10 + more) + 8 * rows + (4 * n if case["kind"] == "norm" else 0),
                "flops": rows * n * (7 if case["kind"] == "norm" else 3)}
    mats, d = (2 if case["kind"] == "gated" else 1), case["d"]
    return {"bytes": mats * d * (n // BLOCK) * 36 + rows * (n + 4) + 4 * rows * d * (2 if case["residual"] else 1)
                     + (4 * mats * d if case["bias"] else 0),
            "flops": 2 * mats * rows * n * d}


# ------------------------------------------------------------------- inputs

def _matrix(g, d, n):
    """BlockQ8 rows, uint8 [d][n / 32][36]."""
    w = torch.empty((d, n // BLOCK, 36), dtype=torch.uint8, device="cuda")
    scale = torch.rand((d, n // BLOCK, 1), generator=g, device="cuda").add_(0.5).div_(127 * math.sqrt(n))
    w[..., :4] = scale.view(torch.uint8)
    w[..., 4:] = torch.randint(-127, 128, (d, n // BLOCK, BLOCK), generator=g, device="cuda", dtype=torch.int8).view(torch.uint8)
    return w


def prepare(case, seed):
    dev, rows, n = "cuda", case["rows"], case["n"]
    g = torch.Generator(device=dev).manual_seed(seed)
    state = {"case": case}
    channel = torch.where(torch.rand(n, generator=g, device=dev) < 0.004, 12.0, 1.0)
    x = torch.randn((rows, n), generator=g, device=dev).mul_(channel)
    if case["kind"] in ("norm", "quantize"):
        if case["kind"] == "quantize":  # a product of two, as SwiGLU's is
            x = x.mul_(torch.randn((rows, n), generator=g, device=dev))
        state["x"] = x
        if case["kind"] == "norm":
            state["residual"] = torch.randn((rows, n), generator=g, device=dev).mul_(3) if case["residual"] else None
            state["weight"] = torch.rand(n, generator=g, device=dev).add_(0.5)
            state["sum"] = torch.empty_like(x) if case["residual"] else None
        state["codes"] = torch.empty((rows, n), dtype=torch.int8, device=dev)
        state["scales"] = torch.empty(rows, device=dev)
        state["values"] = torch.empty_like(x)
        return state
    mats, d = (2 if case["kind"] == "gated" else 1), case["d"]
    codes, state["scales"] = _hold(x)
    state["codes"] = codes.to(torch.int8)
    state["w"] = [_matrix(g, d, n) for _ in range(mats)]
    state["bias"] = torch.randn(mats * d, generator=g, device=dev) if case["bias"] else None
    state["residual"] = torch.randn((rows, d), generator=g, device=dev).mul_(3) if case["residual"] else None
    state["out"] = torch.empty((rows, d), device=dev)
    if own:  # the matrix laid out once, as a program keeps it over its steps
        import nitrorag_amd as na

        state["weights"] = na.Q8Weights(*state["w"])
    return state


# --------------------------------------------------------------------- runs

def run(state):
    if own:
        return _own(state)
    return _hold_rows(state) if state["case"]["kind"] in ("norm", "quantize") else _product(state)


def _own(state):
    import nitrorag_amd as na

    case = state["case"]
    if case["kind"] == "norm":
        na.rms_norm_row8(state["x"], state["weight"], state["codes"], state["scales"], residual=state["residual"],
                         sum=state["sum"], eps=EPS)
    elif case["kind"] == "quantize":
        na.row8_quantize(state["x"], state["codes"], state["scales"])
    else:
        state["weights"].matmul(state["codes"], state["scales"], state["out"], bias=state["bias"],
                                residual=state["residual"], activation=case["activation"])
        return {"out": state["out"]}
    na.row8_read(state["codes"], state["scales"], state["values"])
    return {"values": state["values"], **({"sum": state["sum"]} if case.get("residual") else {})}


def _hold(y):
    """Codes (as fp32 numbers) and scales of fp32 rows."""
    top = y.abs().amax(-1).double()
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    scale = (top / torch.full_like(top, 127)).float()
    inverse = torch.where(top > 0, torch.full_like(top, 127) / top, 0.0).float()
    return torch.round(y.double() * inverse.double()[:, None]).float(), scale


def _hold_rows(state):
    y, out = state["x"], {}
    if state["case"]["kind"] == "norm":
        if state["residual"] is not None:
            y = out["sum"] = y + state["residual"]
        h = y.double()  # codes lie next to a border
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        y = (h * r * state["weight"].double()).float()
    codes, scales = _hold(y)
    return {"values": codes * scales[:, None], **out}


def _values(w):
    """A BlockQ8 matrix's values in fp32, [d][n]."""
    scale = w[..., :4].contiguous().view(torch.float32)
    return (w[..., 4:].contiguous().view(torch.int8).float() * scale).flatten(1)


def _activate(x, name):
    if name == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * torch.erfc(x * -math.sqrt(0.5))
    if name == "gelu_tanh":
        return x / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _product(state):
    case, d = state["case"], state["case"]["d"]
    x = state["codes"].float() * state["scales"][:, None]
    parts = [torch.matmul(x, _values(w).t()) for w in state["w"]]
    if state["bias"] is not None:
        parts = [p + state["bias"][i * d:(i + 1) * d] for i, p in enumerate(parts)]
    out = _activate(parts[0], case["activation"])
    if len(parts) > 1:
        out = out * parts[1]
    return {"out": out if state["residual"] is None else out + state["residual"]}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    """The same in 64 bits.  What is fp32 by definition (the sum, the rows that are
    held, their scales and inverse scales) is rounded to it."""
    state = prepare(case, seed)

    def fp32(t):
        return t.to(torch.float32).to(torch.float64)

    if case["kind"] in ("norm", "quantize"):
        y, out = state["x"].double(), {}
        if case["kind"] == "norm":
            if case["residual"]:
                y = out["sum"] = fp32(y + state["residual"].double())
            square = torch.linalg.vector_norm(y, dim=-1, keepdim=True).square() / case["n"]
            y = fp32(y / torch.sqrt(square + EPS) * state["weight"].double())
        top = torch.maximum(y.max(-1, keepdim=True).values, -y.min(-1, keepdim=True).values)
        most = torch.tensor(127.0, dtype=torch.float64, device=y.device).expand_as(top)
        zero = top < 2.0 ** -100
        codes = torch.round(y * fp32(torch.where(zero, 0.0, torch.div(most, top))))
        return {"values": codes * fp32(torch.where(zero, 0.0, torch.div(top, most))), **out}
    d, parts = case["d"], []
    x = state["codes"].double()
    for i, w in enumerate(state["w"]):
        blocks = w.view(d, -1, 36)
        scale = blocks[:, :, 0:4].contiguous().view(torch.float32)
        q = blocks[:, :, 4:36].contiguous().view(torch.int8)
        p = torch.matmul(x, (q.double() * scale.double()).reshape(d, -1).t()) * state["scales"].double()[:, None]
        if state["bias"] is not None:
            p += state["bias"][i * d:i * d + d].double()
        parts.append(p)
    p, name = parts[0], case["activation"]
    if name == "relu":
        p = p.clamp(min=0)
    elif name == "silu":
        p = p * torch.sigmoid(p)
    elif name == "gelu":
        p = p * torch.special.ndtr(p)
    elif name == "gelu_tanh":
        p = p * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p ** 3))
    for more in parts[1:]:
        p = p * more
    return {"out": p + state["residual"].double() if case["residual"] else p}
