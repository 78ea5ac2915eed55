"""Microscaled numbers in 64 bits, written from the statement of the format in
include/neuzip_hip.h, for the tests of the operators on them."""
import math

import torch

TOP = {4: 2, 8: 8}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def magnitudes(bits):
    if bits == 4:
        return [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    out = [m * 2.0 ** -9 for m in range(8)]
    for e in range(1, 16):
        out += [(1 + m / 8) * 2.0 ** (e - 7) for m in range(8)]
    return out[:-1]  # the last code is NaN


def held(x, bits):
    """float64 values that a matrix (CPU, any float type) stands for once it is held in 4 or 8 bits"""
    x = x.double()
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64)
    v[:, :cols] = x
    v = v.view(rows, -1, 32)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    w = torch.where(bad, torch.zeros_like(v), v)
    _, e = torch.frexp(w.abs().amax(-1, keepdim=True))
    power = (e - 1 - TOP[bits]).clamp(min=-127)
    power = torch.where(w.abs().amax(-1, keepdim=True) == 0, torch.full_like(power, -127), power)
    scale = torch.pow(torch.tensor(2.0, dtype=torch.float64), power.double())
    table = torch.tensor(magnitudes(bits), dtype=torch.float64)
    between = (table[1:] + table[:-1]) / 2
    size = w.abs() / scale
    low, high = torch.bucketize(size, between), torch.bucketize(size, between, right=True)
    code = torch.where(low % 2 == 0, low, high)
    out = torch.where(bad, torch.full_like(v, math.nan), torch.sign(w) * table[code] * scale)
    return out.view(rows, -1)[:, :cols]


def decoded(data, scales, cols, bits):
    """float64 values of the stored bytes (CPU uint8 tensors), padding included"""
    rows, width = data.shape[0], data.shape[1] * 8 // bits
    if bits == 4:
        codes = torch.stack((data & 15, data >> 4), -1).view(rows, width).long()
        sign, mag = codes >> 3, codes & 7
    else:
        codes = data.long()
        sign, mag = codes >> 7, codes & 127
    table = torch.tensor(magnitudes(bits) + ([math.nan] if bits == 8 else []), dtype=torch.float64)
    b = torch.arange(width // 32)
    s = scales.long()[:, (b // 16) * 16 + 4 * (b % 4) + (b % 16) // 4]
    factor = torch.where(s == 255, torch.full((), math.nan, dtype=torch.float64),
                         torch.pow(torch.tensor(2.0, dtype=torch.float64), (s - 127).double()))
    return torch.where(sign == 1, -1.0, 1.0) * table[mag] * factor.repeat_interleave(32, 1)


def round_to(x, dtype):
    """float64 -> dtype in one rounding (float32 first would round twice)"""
    if dtype == torch.float32:
        return x.float()
    keep = {torch.bfloat16: 8, torch.float16: 11}[dtype]
    low = {torch.bfloat16: -126, torch.float16: -14}[dtype]
    _, e = torch.frexp(x)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), ((e - 1).clamp(min=low) - keep + 1).double())
    return (torch.round(x / step) * step).to(dtype)
