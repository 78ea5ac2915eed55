"""The operators on tensors held in 8 bits with a scale for each block of 128:
weights that are multiplied as they are, and activations that a training step
keeps for its backward pass, with the sizes programs call them at.

A case is a dict of plain values.  ``listed()`` are the cases that are always
looked at, ``draw(rng)`` gives one more of the same ranges, ``prepare(case,
seed)`` makes what the program has in hand before the call, ``run(state)`` makes
the call once and returns what the program gets, ``work(case)`` is what a pass
cannot do without and ``exact(case, seed)`` the outputs in float64.  Where
``own`` is false, ``run`` computes the same in elementary torch operations.

Kinds
  quantize    ``ops.fp8_quantize`` of a matrix and the values that it then stands for
  linear      ``ops.fp8_linear``: activation rows against a weight held in 8 bits
  train       the same with a gradient: forward, and the gradient of the rows
  saved       a layer's input kept in 8 bits, and ``ops.fp8_weight_gradient`` made with it
  activation  ``ops.fp8_activation``: an activation function, which keeps its input in 8
              bits, and the gradients made with that

The format: e4m3 numbers (magnitudes up to 448) times a power of two 2^(s - 127)
that a block shares.  A block is 128 values of a row, or 128 rows of 128 columns
(weights); s is the smallest, not below 0, with which the block's largest
magnitude is at most 448 2^(s - 127).  Values are rounded to the nearest, ties to
the even code.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a 16384 x 4096 weight converted to 8 bits, as when a model is loaded
        {"name": "quantize_16384x4096", "kind": "quantize", "rows": 16384, "cols": 4096, "block": 128, "type": "bf16"},
        # ragged activations brought to 8 bits: nothing is a multiple of a block
        {"name": "quantize_509x3001_fp16", "kind": "quantize", "rows": 509, "cols": 3001, "block": 1, "type": "fp16"},
        # single-token inference through the up projection of an 8B-shaped block: latency and the weight's bytes
        {"name": "linear_token_14336x4096", "kind": "linear", "tokens": 1, "out": 14336, "in": 4096, "bias": False,
         "type": "bf16"},
        # seven speculative tokens through a ragged weight with a bias, in fp16
        {"name": "linear_7x5003x3001_fp16", "kind": "linear", "tokens": 7, "out": 5003, "in": 3001, "bias": True,
         "type": "fp16"},
        # a batch of sequences, one token each, through the down projection
        {"name": "linear_batch64_4096x14336", "kind": "linear", "tokens": 64, "out": 4096, "in": 14336,
         "bias": False, "type": "bf16"},
        # several prompts together through the up projection: the largest product
        {"name": "linear_8192_14336x4096", "kind": "linear", "tokens": 8192, "out": 14336, "in": 4096,
         "bias": False, "type": "bf16"},
        # a fine-tuning step of a GPT-2-medium-shaped feed-forward layer whose weight stays frozen, 8 x 1024 tokens
        {"name": "train_8192_4096x1024", "kind": "train", "tokens": 8192, "out": 4096, "in": 1024, "type": "bf16"},
        # the same for one short sequence through a ragged weight in fp32
        {"name": "train_333_1021x3001_fp32", "kind": "train", "tokens": 333, "out": 1021, "in": 3001, "type": "fp32"},
        # the input of that feed-forward layer kept in 8 bits while it is trained, and the gradient of its weight
        {"name": "saved_8192_4096x1024", "kind": "saved", "tokens": 8192, "out": 4096, "in": 1024, "type": "bf16"},
        # the same for one ragged sequence in fp16
        {"name": "saved_777_1021x509_fp16", "kind": "saved", "tokens": 777, "out": 1021, "in": 509, "type": "fp16"},
        # its activation function
        {"name": "activation_gelu_8192x4096", "kind": "activation", "tokens": 8192, "width": 4096,
         "function": "gelu", "gated": False, "type": "bf16"},
        # the gated one of an 8B-shaped block, one sequence
        {"name": "activation_silu_gated_2048x14336", "kind": "activation", "tokens": 2048, "width": 14336,
         "function": "silu", "gated": True, "type": "bf16"},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """a layer's width: a multiple of 64 mostly, any number otherwise"""
    n = _log_uniform(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "train", "saved", "activation"])
    type_ = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "quantize":
        cols = _width(rng, 64, 16384)
        rows = _log_uniform(rng, 1, min(16384, 16384 * 4096 // cols))
        return {"kind": kind, "rows": rows, "cols": cols, "block": rng.choice([1, 128]), "type": type_}
    if kind == "activation":
        width = _width(rng, 64, 16384)
        gated = rng.random() < 0.5
        tokens = _log_uniform(rng, 1, min(8192, 2048 * 14336 // width // (1 if type_ != "fp32" else 2)))
        return {"kind": kind, "tokens": tokens, "width": width, "function": rng.choice(["gelu", "gelu_tanh", "silu"]),
                "gated": gated, "type": type_}
    out, in_ = _width(rng, 256, 16384), _width(rng, 256, 16384)
    cap = 8192 * 14336 * 4096 // (out * in_) // (1 if kind == "linear" else 4)
    tokens = _log_uniform(rng, 1 if kind == "linear" else 32, max(32, min(8192, cap)))
    case = {"kind": kind, "tokens": tokens, "out": out, "in": in_, "type": type_}
    if kind == "linear":
        case["bias"] = rng.random() < 0.3
    return case


# -- what the program has in hand ---------------------------------------------------

def _activations(tokens, cols, type_, gen):
    """N(0, 1) with a few channels that are twenty times as large, as behind a norm"""
    x = torch.randn(tokens, cols, device="cuda", generator=gen)
    x[:, torch.randperm(cols, device="cuda", generator=gen)[:max(1, cols // 512)]] *= 20.0
    return x.to(_TYPES[type_])


def _gradients(tokens, cols, type_, gen):
    return (torch.randn(tokens, cols, device="cuda", generator=gen) * 1e-2).to(_TYPES[type_])


def _inputs(case, seed):
    """the tensors of a case, the same for every form of it; ``weight`` is dense here"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, type_, st = case["kind"], case["type"], {}
    if kind == "quantize":
        if case["block"] == 128:
            st["x"] = (torch.randn(case["rows"], case["cols"], device="cuda", generator=gen) * 0.02).to(_TYPES[type_])
        else:
            st["x"] = _activations(case["rows"], case["cols"], type_, gen)
    elif kind == "activation":
        shape = (case["tokens"], case["width"])
        st["x"] = (torch.randn(*shape, device="cuda", generator=gen) * 1.5).to(_TYPES[type_])
        st["up"] = torch.randn(*shape, device="cuda", generator=gen).to(_TYPES[type_]) if case["gated"] else None
        st["g"] = _gradients(*shape, type_, gen)
    else:
        st["x"] = _activations(case["tokens"], case["in"], type_, gen)
        if kind != "saved":
            st["weight"] = torch.randn(case["out"], case["in"], device="cuda", generator=gen).mul_(0.02).bfloat16()
        st["bias"] = None
        if case.get("bias"):
            st["bias"] = (torch.randn(case["out"], device="cuda", generator=gen) * 0.1).to(_TYPES[type_])
        if kind != "linear":
            st["g"] = _gradients(case["tokens"], case["out"], type_, gen)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if "weight" in st:
        if own:
            from neuzip_amd import ops
            st["weight"] = ops.fp8_quantize(st["weight"], 128)
        else:
            st["weight"] = _rounded(st["weight"], 128).bfloat16()  # the values that the 8 bits stand for
    if own and case["kind"] in ("train", "activation"):
        st["x"].requires_grad_(True)
        if st.get("up") is not None:
            st["up"].requires_grad_(True)
    return st


# -- the plain form ------------------------------------------------------------------

def _rounded(x, block):
    """The values that the elements of ``x`` stand for when it is held in 8 bits, float32."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % 128, 0, -rows % block))
    v = v.view(-1, block, v.shape[1] // 128, 128)
    largest = v.abs().amax((1, 3), keepdim=True).view(torch.int32)
    # the exponent, one more where the largest value is beyond 1.75 times its power of two (448 = 1.75 * 2^8)
    s = (((largest + 0x1FFFFF) >> 23) - 8).clamp_(min=0)
    up = ((254 - s) << 23).view(torch.float32)  # 2^(127 - s)
    down = torch.where(s > 0, (s << 23).view(torch.float32), 2.0 ** -127)  # 2^(s - 127)
    q = v * up
    e = ((q.view(torch.int32) >> 23) & 255).sub_(127).clamp_(min=-6)
    step = ((e - 3 + 127) << 23).view(torch.float32)
    q = torch.round(q / step).mul_(step)
    q = torch.where(largest >= 0x7F800000, math.nan, q * down)
    return q.view(-1, q.shape[2] * 128)[:rows, :cols]


def _function(kind, x):
    """f(x) and f'(x) in the type of x"""
    if kind == "gelu":
        p = torch.erfc(x * -math.sqrt(0.5)) * 0.5
        return x * p, p + x * torch.exp(x * x * -0.5) * (1 / math.sqrt(2 * math.pi))
    if kind == "gelu_tanh":
        c = 2 * math.sqrt(2 / math.pi)
        p = 1 / (1 + torch.exp(-c * (x + 0.044715 * x * x * x)))
        return x * p, p + x * p * (1 - p) * c * (1 + 3 * 0.044715 * x * x)
    p = 1 / (1 + torch.exp(-x))
    return x * p, p + x * p * (1 - p)


def run(state):
    case = state["case"]
    kind, x = case["kind"], state["x"]
    if own:
        from neuzip_amd import ops
        if kind == "quantize":
            return ops.fp8_quantize(x, case["block"]).dequantize()
        if kind == "linear":
            return ops.fp8_linear(x, state["weight"], state["bias"])
        if kind == "train":
            y = ops.fp8_linear(x, state["weight"])
            (gx,) = torch.autograd.grad(y, x, state["g"])
            return [y.detach(), gx]
        if kind == "saved":
            return ops.fp8_weight_gradient(state["g"], ops.fp8_quantize(x))
        up = state["up"]
        y = ops.fp8_activation(x, case["function"], up)
        return [y.detach(), *torch.autograd.grad(y, (x,) if up is None else (x, up), state["g"])]
    if kind == "quantize":
        return _rounded(x, case["block"]).bfloat16()
    if kind in ("linear", "train"):
        w = state["weight"].float()
        y = torch.mm(_rounded(x, 1), w.t())
        if state["bias"] is not None:
            y += state["bias"].float()
        y = y.to(x.dtype)
        if kind == "linear":
            return y
        return [y, torch.mm(state["g"].float(), w).to(x.dtype)]
    if kind == "saved":
        return torch.mm(state["g"].float().t(), _rounded(x, 1)).to(x.dtype)
    y, _ = _function(case["function"], x.float())
    f, slope = _function(case["function"], _rounded(x, 1))
    g = state["g"].float()
    if state["up"] is None:
        return [y.to(x.dtype), (g * slope).to(x.dtype)]
    y = y * state["up"].float()
    return [y.to(x.dtype), (g * _rounded(state["up"], 1) * slope).to(x.dtype), (g * f).to(x.dtype)]


# -- costs and exact values ------------------------------------------------------------

def work(case):
    kind, size = case["kind"], _SIZES[case["type"]]
    held = 1 + 1 / 128  # bytes of a value in 8 bits, with its share of the scale
    if kind == "quantize":
        # the matrix in, its codes and scales out, the values out
        block = 1 + 1 / 128 / case["block"]
        return {"bytes": int(case["rows"] * case["cols"] * (size + block + 2)), "flops": 0}
    if kind == "activation":
        # input in, result out, codes out; codes in, gradient in, gradient out; twice where there are two inputs
        inputs = 2 if case["gated"] else 1
        return {"bytes": int(case["tokens"] * case["width"] * (inputs * (2 * size + 2 * held) + 2 * size)), "flops": 0}
    m, n, k = case["tokens"], case["out"], case["in"]
    if kind == "saved":
        # input in, codes out; codes in, gradient in, gradient of the weight out
        return {"bytes": int(m * k * (size + 2 * held) + size * n * (m + k)), "flops": 2 * m * n * k}
    b = n * k * (1 + 1 / 16384) + size * m * (n + k) + (size * n if case.get("bias") else 0)
    if kind == "train":
        b += size * m * (n + k)
    return {"bytes": int(b), "flops": (2 if kind == "linear" else 4) * m * n * k}


# the non-negative e4m3 numbers in the order of their codes
_CODES = [m / 512.0 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)
                                          if (e, m) != (15, 7)]


def _held(x, block):
    """The same values as ``_rounded``, from the list of the numbers of the element type, float64."""
    table = torch.tensor(_CODES, dtype=torch.float64, device=x.device)
    between = (table[1:] + table[:-1]) / 2
    rows, cols = x.shape
    v = torch.zeros(-(-rows // block) * block, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    v[:rows, :cols] = x
    v = v.view(-1, block, v.shape[1] // 128, 128)
    part, e = torch.frexp(v.abs().amax((1, 3), keepdim=True) / 448.0)
    power = torch.where(part == 0.5, e - 1, e)  # the least with largest / 448 <= 2^power
    power = torch.where(part == 0.0, -127, power).clamp(min=-127)
    scale = (power.long() + 1023 << 52).view(torch.float64)
    size = v.abs() / scale
    below, above = torch.bucketize(size, between), torch.bucketize(size, between, right=True)
    code = torch.where(below % 2 == 0, below, above)  # they differ on a tie: the even code
    v = torch.sign(v) * table[code] * scale
    return v.view(-1, v.shape[2] * 128)[:rows, :cols]


def _exact_function(kind, x):
    if kind == "gelu":
        p = torch.exp(torch.special.log_ndtr(x))  # (ndtr itself loses its digits below -5)
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
        p = torch.sigmoid(2 * u)
        return x * p, p + x * p * torch.sigmoid(-2 * u) * 2 * math.sqrt(2 / math.pi) * (1 + 0.134145 * x * x)
    p = torch.sigmoid(x)
    return x * p, p * (1 + x * torch.sigmoid(-x))


def exact(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _held(st["x"], case["block"])
    if kind in ("linear", "train"):
        w = _held(st["weight"], 128)
        y = _held(st["x"], 1) @ w.t()
        if st["bias"] is not None:
            y = y + st["bias"].double()
        return y if kind == "linear" else [y, st["g"].double() @ w]
    if kind == "saved":
        return st["g"].double().t() @ _held(st["x"], 1)
    y, _ = _exact_function(case["function"], st["x"].double())
    f, slope = _exact_function(case["function"], _held(st["x"], 1))
    g = st["g"].double()
    if st["up"] is None:
        return [y, g * slope]
    return [y * st["up"].double(), g * _held(st["up"], 1) * slope, g * f]
