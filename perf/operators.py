"""The operators on weights held in microscaled 4 bits, and on embedding tables,
with the sizes programs call them at.

A case is a dict of plain values.  ``listed()`` are the cases that are always
looked at, ``draw(rng)`` gives one more of the same ranges, ``prepare(case,
seed)`` makes what the program has in hand before the call, ``run(state)`` makes
the call once and returns what the program gets, ``work(case)`` is what a pass
cannot do without and ``exact(case, seed)`` the outputs in float64.  Where
``own`` is false, ``run`` computes the same in elementary torch operations.

Kinds
  quantize   ``ops.mx_quantize`` of a matrix and the values that it then stands for
  linear     ``ops.mx_linear``: activation rows against a weight held in 4 bits
  train      the same with a gradient: forward, and the gradient of the rows
  lookup     ``ops.mx_embedding``: rows of a table held in 4 bits, times a scale
  gradient   ``ops.embedding_gradient``: the dense gradient of an embedding table

The format: blocks of 32 values along a row share a power of two 2^(s - 127),
s = max(exponent of the block's largest magnitude + 127 - e, 0); a value is held
as an e2m1 number (4 bits, e = 2, largest 6) or an e4m3 number (8 bits, e = 8,
largest 448) times that, rounded to the nearest, ties to the even code, larger
ones to the largest.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
# 4-bit and 8-bit elements: exponent of the largest binade, mantissa bits, smallest normal exponent, largest value
_ELEMENTS = {4: (2, 1, 0, 6.0), 8: (8, 3, -6, 448.0)}


def listed():
    return [
        # a 16384 x 4096 weight converted to 4 bits, as when a model is loaded
        {"name": "quantize_16384x4096", "kind": "quantize", "rows": 16384, "cols": 4096, "bits": 4, "type": "bf16"},
        # ragged activations brought to 8 bits: nothing is a multiple of a block
        {"name": "quantize_509x3001_8bit_fp16", "kind": "quantize", "rows": 509, "cols": 3001, "bits": 8,
         "type": "fp16"},
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
        {"name": "train_333_1021x3071_fp32", "kind": "train", "tokens": 333, "out": 1021, "in": 3071, "type": "fp32"},
        # one token looked up in an 8B-shaped model's table, scaled by the root of the width
        {"name": "lookup_token_128256x4096", "kind": "lookup", "rows": 128256, "cols": 4096, "tokens": 1,
         "scale": 64.0},
        # the tokens of a training batch in a GPT-2-medium-shaped table
        {"name": "gradient_8192_50257x1024", "kind": "gradient", "rows": 50257, "cols": 1024, "tokens": 8192,
         "scale": 32.0, "type": "bf16"},
        # a prompt's tokens in the 8B-shaped table: nearly all rows of the gradient are zeros
        {"name": "gradient_2048_128256x4096", "kind": "gradient", "rows": 128256, "cols": 4096, "tokens": 2048,
         "scale": 1.0, "type": "bf16"},
        # a batch of prompts looked up in a ragged table
        {"name": "lookup_4096_50257x1021", "kind": "lookup", "rows": 50257, "cols": 1021, "tokens": 4096,
         "scale": 32.0},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """a layer's width: a multiple of 64 mostly, any number otherwise"""
    n = _log_uniform(rng, lo, hi)
    return max(64, n // 64 * 64) if rng.random() < 0.7 else n


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "train", "lookup", "gradient"])
    type_ = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "quantize":
        cols = _width(rng, 64, 16384)
        rows = _log_uniform(rng, 1, min(16384, 16384 * 4096 // cols))
        return {"kind": kind, "rows": rows, "cols": cols, "bits": rng.choice([4, 4, 8]), "type": type_}
    if kind in ("linear", "train"):
        out, in_ = _width(rng, 256, 16384), _width(rng, 256, 16384)
        cap = 8192 * 14336 * 4096 // (out * in_) // (1 if kind == "linear" else 4)
        tokens = _log_uniform(rng, 1 if kind == "linear" else 32, max(32, min(8192, cap)))
        case = {"kind": kind, "tokens": tokens, "out": out, "in": in_, "type": type_}
        if kind == "linear":
            case["bias"] = rng.random() < 0.3
        return case
    rows, cols = _log_uniform(rng, 8000, 128256), _width(rng, 256, 4096)
    if kind == "lookup":
        return {"kind": kind, "rows": rows, "cols": cols, "tokens": _log_uniform(rng, 1, 8192),
                "scale": rng.choice([1.0, 0.1, round(math.sqrt(cols), 3)])}
    size, tokens = _SIZES[type_], _log_uniform(rng, 1, 16384)
    rows = min(rows, 128256 * 4096 * 2 // (cols * size) - tokens)  # the largest listed gradient's bytes
    return {"kind": kind, "rows": rows, "cols": cols, "tokens": tokens,
            "scale": rng.choice([1.0, round(math.sqrt(cols), 3)]), "type": type_}


# -- what the program has in hand ---------------------------------------------------

def _weight(rows, cols, gen):
    return torch.randn(rows, cols, device="cuda", generator=gen).mul_(0.02).to(torch.bfloat16)


def _activations(tokens, cols, type_, gen):
    """N(0, 1) with a few channels that are twenty times as large, as behind a norm"""
    x = torch.randn(tokens, cols, device="cuda", generator=gen)
    x[:, torch.randperm(cols, device="cuda", generator=gen)[:max(1, cols // 512)]] *= 20.0
    return x.to(_TYPES[type_])


def _ids(case, gen):
    """token ids of a text: the frequency falls with the rank, and ranks lie anywhere in the table"""
    u = torch.rand(case["tokens"], device="cuda", generator=gen, dtype=torch.float64)
    rank = (torch.exp(u * math.log(case["rows"])).long() - 1).clamp_(0, case["rows"] - 1)
    return torch.randperm(case["rows"], device="cuda", generator=gen)[rank]


def _inputs(case, seed):
    """the tensors of a case, the same for every form of it; ``weight`` is dense here"""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, st = case["kind"], {}
    if kind == "quantize":
        if case["bits"] == 4:
            st["x"] = _weight(case["rows"], case["cols"], gen).to(_TYPES[case["type"]])
        else:
            st["x"] = _activations(case["rows"], case["cols"], case["type"], gen)
    elif kind in ("linear", "train"):
        st["weight"] = _weight(case["out"], case["in"], gen)
        st["x"] = _activations(case["tokens"], case["in"], case["type"], gen)
        st["bias"] = None
        if case.get("bias"):
            st["bias"] = (torch.randn(case["out"], device="cuda", generator=gen) * 0.1).to(_TYPES[case["type"]])
        if kind == "train":
            st["g"] = (torch.randn(case["tokens"], case["out"], device="cuda", generator=gen) * 1e-2
                       ).to(_TYPES[case["type"]])
    elif kind == "lookup":
        st["weight"] = _weight(case["rows"], case["cols"], gen)
        st["ids"] = _ids(case, gen)
    else:
        st["ids"] = _ids(case, gen)
        st["g"] = (torch.randn(case["tokens"], case["cols"], device="cuda", generator=gen) * 1e-2
                   ).to(_TYPES[case["type"]])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if "weight" in st:
        if own:
            from neuzip_amd import ops
            st["weight"] = ops.mx_quantize(st["weight"], 4)
        else:
            w = st["weight"]  # the values that the 4 bits stand for, a bf16 tensor
            for at in range(0, w.shape[0], 8192):
                w[at:at + 8192] = _rounded(w[at:at + 8192], 4).to(torch.bfloat16)
    if case["kind"] == "train" and own:
        st["x"].requires_grad_(True)
    return st


# -- the plain form ------------------------------------------------------------------

def _rounded(x, bits):
    """The values that the elements of ``x`` stand for when its rows are held in 4 or 8 bits, float32."""
    top, mant, low, largest = _ELEMENTS[bits]
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)
    exponent = (v.abs().amax(-1, keepdim=True).view(torch.int32) >> 23)
    s = (exponent - top).clamp_(min=0)
    up = ((254 - s) << 23).view(torch.float32)  # 2^(127 - s)
    down = torch.where(s > 0, (s << 23).view(torch.float32), 2.0 ** -127)  # 2^(s - 127)
    q = v * up
    e = ((q.view(torch.int32) >> 23) & 255).sub_(127).clamp_(min=low)
    step = ((e - mant + 127) << 23).view(torch.float32)
    q = torch.round(q / step).mul_(step).clamp_(-largest, largest)
    return torch.where(exponent == 255, math.nan, q * down).view(rows, -1)[:, :cols]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from neuzip_amd import ops
        if kind == "quantize":
            return ops.mx_quantize(state["x"], case["bits"]).dequantize()
        if kind == "linear":
            return ops.mx_linear(state["x"], state["weight"], state["bias"])
        if kind == "train":
            y = ops.mx_linear(state["x"], state["weight"])
            (gx,) = torch.autograd.grad(y, state["x"], state["g"])
            return [y.detach(), gx]
        if kind == "lookup":
            return ops.mx_embedding(state["ids"], state["weight"], case["scale"])
        return ops.embedding_gradient(state["ids"], state["g"], case["rows"], case["scale"])
    if kind == "quantize":
        return _rounded(state["x"], case["bits"]).to(torch.bfloat16)
    if kind in ("linear", "train"):
        w = state["weight"].float()
        y = torch.mm(_rounded(state["x"], 8), w.t())
        if state["bias"] is not None:
            y += state["bias"].float()
        y = y.to(state["x"].dtype)
        if kind == "linear":
            return y
        return [y, torch.mm(state["g"].float(), w).to(state["x"].dtype)]
    if kind == "lookup":
        return (state["weight"][state["ids"]].float() * case["scale"]).to(torch.bfloat16)
    g = state["g"].float() * case["scale"]
    total = torch.zeros(case["rows"], case["cols"], device=g.device)
    return total.index_add_(0, state["ids"], g).to(state["g"].dtype)


# -- costs and exact values ------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["cols"]
        # the matrix in, its bits and scales out, the values out
        return {"bytes": int(n * (_SIZES[case["type"]] + case["bits"] / 8 + 1 / 32 + 2)), "flops": 0}
    if kind in ("linear", "train"):
        m, n, k, size = case["tokens"], case["out"], case["in"], _SIZES[case["type"]]
        b = n * k * 17 / 32 + size * m * (n + k) + (size * n if case.get("bias") else 0)
        if kind == "train":
            b += size * m * (n + k)
        return {"bytes": int(b), "flops": (2 if kind == "linear" else 4) * m * n * k}
    t, cols = case["tokens"], case["cols"]
    if kind == "lookup":
        return {"bytes": int(t * (8 + cols * (17 / 32 + 2))), "flops": 0}
    return {"bytes": int(8 * t + _SIZES[case["type"]] * cols * (t + case["rows"])), "flops": 0}


def _magnitudes(bits):
    """the non-negative numbers of the element type in the order of their codes"""
    if bits == 4:
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return [m / 512.0 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)
                                            if (e, m) != (15, 7)]


def _held(x, bits):
    """The same values as ``_rounded``, from the list of the numbers of the element type, float64."""
    table = torch.tensor(_magnitudes(bits), dtype=torch.float64, device=x.device)
    between = (table[1:] + table[:-1]) / 2
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, -1, 32)
    _, e = torch.frexp(v.abs().amax(-1, keepdim=True))
    scale = ((e - 1 - _ELEMENTS[bits][0]).clamp(min=-127).long() + 1023 << 52).view(torch.float64)
    size = v.abs() / scale
    below, above = torch.bucketize(size, between), torch.bucketize(size, between, right=True)
    code = torch.where(below % 2 == 0, below, above)  # they differ on a tie: the even code
    return (torch.sign(v) * table[code] * scale).view(rows, -1)[:, :cols]


def exact(case, seed):
    st = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _held(st["x"], case["bits"])
    if kind in ("linear", "train"):
        w = _held(st["weight"], 4)
        y = _held(st["x"], 8) @ w.t()
        if st["bias"] is not None:
            y = y + st["bias"].double()
        return y if kind == "linear" else [y, st["g"].double() @ w]
    if kind == "lookup":
        return _held(st["weight"][st["ids"]], 4) * case["scale"]
    total = torch.zeros(case["rows"], case["cols"], dtype=torch.float64, device="cuda")
    order = torch.argsort(st["ids"], stable=True)
    return total.index_put_((st["ids"][order],), st["g"][order].double(), accumulate=True) * case["scale"]
