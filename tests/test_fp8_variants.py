"""CPU: the sizes at which products in 8 bits are tested reach every kernel that the rules choose, whole and in parts; and
the rules as the tests have them are the library's."""
import random

import pytest
import torch

import fp8_cuts
from fp8_cuts import INPUT, ROWS8, ROWS16
from neuzip_amd import _lib
from test_gpu_fp8_variants import FEW, GRADIENTS, TILES

TYPES = {"bf16": _lib.DTYPE_BF16, "fp16": _lib.DTYPE_F16, "fp32": _lib.DTYPE_F32}


def kinds(tiles):
    """every tile, whole and in parts"""
    out = set()
    for bm, bn, *_, only_whole in tiles:
        out |= {(bm, bn, False)} if only_whole else {(bm, bn, False), (bm, bn, True)}
    return out


def kind(cut):
    return cut[0], cut[1], cut[2] > 1


@pytest.mark.parametrize("bits,tiles", ((16, ROWS8), (32, ROWS16)))
@pytest.mark.parametrize("held", (False, True))
def test_products_reach_every_tile(bits, tiles, held):
    assert {kind(fp8_cuts.forward(*s, bits, held)) for s in TILES} == kinds(tiles)


def test_tiles_that_workgroups_go_through_one_after_the_other():
    """more of them than compute units, with one group of 512 values each and with several"""
    for k, several in ((512, False), (1536, True)):
        sizes = [s for s in TILES if fp8_cuts.forward(*s, 16)[:2] == (256, 256) and s[2] == k]
        assert sizes and any(several or fp8_cuts.up(m, 256) * fp8_cuts.up(n, 256) > 256 for m, n, _ in sizes)


@pytest.mark.parametrize("bits", (16, 32))
def test_few_rows_reach_every_variant(bits):
    """(groups of its own rows that a wavefront brings to 8 bits, wavefronts for a row of the weight)"""
    waves = (1, 2, 4, 8)
    want = {("few", 1, w) for w in waves} | {("few", 4, w) for w in waves} | {("few", 8, w) for w in waves[1:]}
    own = {fp8_cuts.forward(*s, bits) for s in FEW}
    assert {v for v in own if v[1]} == want and {v[2] for v in own if not v[1]} >= {2, 4}
    assert {fp8_cuts.forward(*s, bits, True) for s in FEW} == {("few", 0, w) for w in waves}
    for most in (4, 2):  # more weight rows than two rounds of workgroups: fewer wavefronts for each
        assert any(up512 > 512 and fp8_cuts.forward(*s, bits)[2] == most
                   for s in FEW for up512 in [fp8_cuts.up(s[1], 16)])


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_reach_every_tile(dtype):
    assert {kind(fp8_cuts.rows_gradient(*s, dtype, 128)) for s in GRADIENTS} == kinds(INPUT)
    assert {kind(fp8_cuts.rows_gradient(*s, dtype, 1)) for s in GRADIENTS} == kinds(ROWS16)
    assert {kind(fp8_cuts.weight_gradient(*s, dtype)) for s in GRADIENTS} == kinds(ROWS16)


@pytest.mark.skipif(torch.cuda.is_available(), reason="counts with a whole card's compute units")
def test_the_rules_are_the_librarys():
    """The library says how much room a product needs, its parts among it: the same for sizes of all kinds."""
    lib, rng = _lib.load(), random.Random(3)

    def size(most):
        n = round(most ** rng.random())
        return max(1, n // 512 * 512) if rng.random() < 0.4 else n

    def room(v):
        return fp8_cuts.up(v, 256) * 256

    def parts(cut, values):
        return room(cut[2] * values * 4) if cut[2] > 1 else 0

    for _ in range(400):
        m, n, k = size(9000), size(17000), size(17000)
        held = room(room(m * lib.nz_fp8_row_bytes(k)) + m * lib.nz_fp8_scale_bytes(k))
        for name, dtype in TYPES.items():
            bits = 32 if name == "fp32" else 16
            cut = fp8_cuts.forward(m, n, k, bits)
            if cut[0] == "few":
                want = 0 if cut[1] else held
            else:
                want = (room(m * lib.nz_fp8_row_bytes(k) * 2) if bits == 32 else held) + parts(cut, m * n)
            assert lib.nz_fp8_linear_workspace_bytes(m, n, k, dtype) == want, (m, n, k, name)
            planes = room(m * fp8_cuts.up(n, 64) * 128 * fp8_cuts.planes(name))
            for block_rows in (1, 128):
                want = 0 if name == "bf16" and n % 64 == 0 else planes
                want += parts(fp8_cuts.rows_gradient(m, n, k, name, block_rows), m * k)
                assert lib.nz_fp8_linear_grad_workspace_bytes(0, dtype, m, n, n, k, block_rows) == want, (m, n, k, name)
            want = 0 if name == "bf16" and n % 8 == 0 else planes
            want += parts(fp8_cuts.weight_gradient(m, n, k, name), n * k)
            assert lib.nz_fp8_weight_grad_workspace_bytes(0, dtype, m, n, n, k) == want, (m, n, k, name)
