"""Which kernels the products of tensors in 8 bits go to: the rules of csrc/nz_fp8.hip and nz_products.h once more, with
the figures read from the sources, for tests that have to reach every one of them.  On 256 compute units, a whole card
(which is what the library counts with where there is none)."""
import math
import os
import re

import numpy as np

from neuzip_amd import _build

F = np.float32


def _read(name):
    with open(os.path.join(_build.CSRC, name)) as f:
        return f.read()


def _tiles(name):
    """[(bm, bn, slots, full, half, ends, whole)] of an array of tiles"""
    text = re.search(r"constexpr Tile " + name + r"\[\] = \{(.*?)\};", _read("nz_fp8.hip"), re.S).group(1)
    out = []
    for row in re.findall(r"\{([^{}]+)\}", text):
        f = [v.strip() for v in row.split(",")]
        out.append((*(int(v) for v in f[:3]), *(F(v.rstrip("f")) for v in f[3:5]),
                    F(f[5].rstrip("f")) if len(f) > 5 else F(1), f[6:] == ["true"]))
    return out


ROWS8, ROWS16, INPUT = _tiles("kTiles"), _tiles("kTiles16"), _tiles("kTilesInput")


def up(a, b):
    return -(-a // b)


def cut(kinds, m, cols, units, steps_per_unit, least, whole=False):
    """(bm, bn, parts)"""
    best, best_time = None, None
    for bm, bn, slots, full, half, ends, only_whole in kinds:
        if only_whole and not whole:
            continue
        tiles = up(m, bm) * up(cols, bn)
        for want in range(1, min(units, 16) + 1):
            if want > 1 and (only_whole or tiles * want > 4 * slots):
                break
            length = up(units, want)
            parts = up(units, length)
            if parts != want or parts > 1 and length < least:
                continue
            groups = F(tiles * parts)
            rounds = F(math.floor(groups / F(slots)))
            rest = groups - rounds * F(slots)
            last = F(0) if rest == 0 else half if rest <= F(slots / 2) else full
            time = (rounds * full + last) * F(length * steps_per_unit) + ends * rounds + ends * F(rest > 0)
            if parts > 1:
                time += F(4) + F(parts) * F(m) * F(cols) * F(2.8e-6)
            if best is None or time < best_time:
                best, best_time = (bm, bn, parts), time
    return best


def few_inside(m, n, k, bits):
    groups = m * up(k, 512)
    return m <= 16 and groups <= 64 and (groups <= 32 or n * k <= 1 << 26 or bits == 32)


def few_rows(m, n, k, bits):
    return few_inside(m, n, k, bits) or m <= 16 and (n * k <= 1 << 25 or bits == 32)


def forward(m, n, k, bits, held=False):
    """Of a product of rows (``held``: in 8 bits already) with a result of 16 or 32 bits: ("few", groups of a wavefront's own
    rows, wavefronts for a row of the weight) or (bm, bn, parts)"""
    if few_rows(m, n, k, bits):
        groups = up(k, 512)
        waves = 8 if groups >= 8 else 4 if groups >= 4 else 2 if groups >= 2 else 1
        if up(n, 16) > 512 and waves >= 4:
            waves = 2 if m >= 4 else 4
        all_groups = m * groups
        inside = 0 if held or not few_inside(m, n, k, bits) else 1 if all_groups <= 8 else 4 if all_groups <= 32 else 8
        return "few", inside, waves
    if bits == 32:
        return cut(ROWS16, m, n, up(k, 128) * 2, 1, 8)
    return cut(ROWS8, m, n, up(k, 512), 4, 2, k % 512 == 0)


def planes(dtype):
    """bf16 numbers for a value of a gradient (of "bf16", "fp16" or "fp32")"""
    return {"bf16": 1, "fp16": 2, "fp32": 3}[dtype]


def rows_gradient(m, n, k, dtype, block_rows):
    """(bm, bn, parts) of the gradient of m rows of k values"""
    return cut(INPUT if block_rows == 128 else ROWS16, m, k, up(n, 64) * planes(dtype), 1, 8)


def weight_gradient(m, n, k, dtype):
    """(bm, bn, parts) of the gradient of n rows of k values"""
    return cut(ROWS16, n, k, up(m, 64) * planes(dtype), 1, 8)
