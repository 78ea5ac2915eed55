"""GPU: every kernel that products of tensors in 8 bits and their gradients go to, whole and in parts, at ragged sizes,
against exact sums.  tests/test_fp8_variants.py holds that these sizes reach all of them."""
import math

import pytest
import torch

from neuzip_amd import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
DEV = "cuda"

# rows, rows and columns of the weight
FEW = [(1, 41, 45), (1, 37, 677), (1, 41, 1647), (1, 43, 3917), (9, 47, 45), (7, 39, 551), (2, 39, 2235), (1, 43, 4181),
       (16, 37, 1329), (7, 35, 2897), (4, 41, 4813), (11, 41, 2647), (9, 43, 3731), (5, 9569, 4000), (16, 9569, 2561),
       (2, 9001, 2100)]
TILES = [(21, 39, 41), (19, 43, 5667), (43, 16407, 257), (40, 5433, 12289), (4457, 997, 135), (8343, 65, 12369),
         (1643, 2481, 1747), (700, 3101, 9001), (8461, 7901, 512), (4001, 3999, 1536)]
GRADIENTS = [(39, 33, 39), (145, 155, 16461), (1251, 1417, 37), (6055, 3569, 133), (1569, 213, 4723), (1569, 256, 4723),
             (1025, 8000, 4099), (4000, 1030, 3000)]


def whole(rows, cols, seed):
    """whole numbers up to 7, which 8 bits hold at any scale; the first of each block of 128 is 7, so no block is zero"""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-7, 8, (rows, cols), generator=g, device=DEV, dtype=torch.float32)
    x[:, ::128] = 7
    return x


def powers(count, of, low):
    """a power of two for each 128 of ``count``, one of ``of`` in turn from 2^low"""
    return torch.exp2((torch.arange(count, device=DEV) // 128 % of + low).float())


def is_rounded(got, want):
    """``got`` is ``want`` (float64, exact in float32) in one rounding"""
    assert torch.equal(want.float().double(), want)
    assert got.shape == want.shape and torch.equal(got, want.float().to(got.dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", FEW + TILES)
def test_products(m, n, k, dtype):
    """The powers of the blocks of x and of w cancel: products are whole and at most 49, times the row's power of two.
    The unit of the cut behind eight of them is at most 2^(5 - 13), and sums stay below 2^24 such units in 32 bits
    whatever their order (49 k is less than 2^20)."""
    assert 49 * k + 99 * 4 < 2 ** 20
    x, wd = whole(m, k, 1), whole(n, k, 2)
    bias = whole(1, n, 3)[0] * 14
    turn, rows = powers(k, 5, -2), torch.exp2((torch.arange(m, device=DEV) % 3 - 1).float())[:, None]
    want = rows.double() * (x.double() @ wd.double().t())
    a = (x * rows * turn).to(dtype)
    held = ops.fp8_quantize(a)
    for block_rows in (1, 128):
        w = ops.fp8_quantize(wd / turn, block_rows)
        is_rounded(ops.fp8_linear(a, w), want)
        is_rounded(ops.fp8_linear(held, w, bias.to(dtype), dtype), want + bias.double())


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", GRADIENTS)
def test_gradients_of_rows(m, n, k, dtype):
    """Each block of the weight has a power of two of its own, from 2^-3 to 2^4: sums are multiples of 2^-3, and those of
    the magnitudes stay below 2^24 of that, so that every order is exact."""
    g, wd = whole(m, n, 1), whole(n, k, 2) * powers(n, 5, -2)[:, None] * powers(k, 4, -1)
    assert (g.abs().double() @ wd.abs().double()).max() < 2 ** 21
    want = g.double() @ wd.double()
    wide = torch.zeros(m, n + 64, dtype=dtype, device=DEV)  # rows that begin at whole vectors, further apart
    wide[:, :n] = g
    x = torch.zeros(m, k, dtype=dtype, device=DEV, requires_grad=True)
    for block_rows in (1, 128):
        w = ops.fp8_quantize(wd, block_rows)
        for grad in (g.to(dtype), wide[:, :n]):
            is_rounded(torch.autograd.grad(ops.fp8_linear(x, w), x, grad)[0], want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", GRADIENTS)
def test_gradients_of_weights(m, n, k, dtype):
    """each row has a power of two of its own, which the gradient's cancels: sums of whole numbers below 2^24"""
    assert 49 * m + 99 < 2 ** 24
    g, x, out = whole(m, n, 1), whole(m, k, 2), whole(n, k, 3) * 14
    turn = torch.exp2((torch.arange(m, device=DEV) % 5 - 2).float())[:, None]
    want = g.double().t() @ x.double()
    a, held = (g / turn).to(dtype), ops.fp8_quantize(x * turn)
    is_rounded(ops.fp8_weight_gradient(a, held), want)
    room = torch.full((n + 2, k), 5.0, dtype=dtype, device=DEV)
    room[1:-1] = out
    ops.fp8_weight_gradient(a, held, out=room[1:-1])
    is_rounded(room[1:-1], want + out.double())
    assert (room[0] == 5).all() and (room[-1] == 5).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(4000, 1030, 3000), (1025, 8000, 4099)])
def test_gradients_of_rows_keep_nan_and_infinities_where_they_are(m, n, k, dtype):
    """the largest tiles, whole and in parts: an infinity of the weight makes its block's columns NaN, one of the gradient
    its row infinite"""
    g, wd = whole(m, n, 1).to(dtype), whole(n, k, 2).abs() + 1
    x = torch.zeros(m, k, dtype=dtype, device=DEV, requires_grad=True)
    g[m - 1, n - 1], g[513, 3] = math.inf, math.nan
    got = torch.autograd.grad(ops.fp8_linear(x, ops.fp8_quantize(wd, 128)), x, g)[0]
    rows = torch.ones(m, dtype=torch.bool, device=DEV)
    rows[m - 1] = rows[513] = False
    assert (got[m - 1] == math.inf).all() and torch.isnan(got[513]).all() and torch.isfinite(got[rows]).all()
    wd[n - 1, 2900] = math.inf
    g[m - 1, n - 1], g[513, 3] = 1.0, 1.0
    got = torch.autograd.grad(ops.fp8_linear(x, ops.fp8_quantize(wd, 128)), x, g)[0]
    want = torch.zeros(m, k, dtype=torch.bool, device=DEV)
    want[:, 2816:2944] = True
    assert torch.equal(torch.isnan(got), want)


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,n,k", [(1643, 2481, 1747), (700, 3101, 9001), (40, 5433, 12289), (8461, 7901, 512)])
def test_products_keep_nan_where_it_is(m, n, k, dtype):
    x, wd = whole(m, k, 1).to(dtype), whole(n, k, 2)
    x[m - 2, k - 1], wd[n - 1, 5] = math.nan, math.inf
    want = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    want[m - 2] = True
    want[:, (n - 1) // 128 * 128:] = True
    assert torch.equal(torch.isnan(ops.fp8_linear(x, ops.fp8_quantize(wd, 128))), want)
