"""GPU: tensors in 8 bits with a scale for each block of 128 (quantisation, values, products and their gradients, the
gradient of a dense weight, activation functions) against float64 on the CPU."""
import math

import pytest
import torch

from neuzip_amd import ops
from fp8_oracle import cut_sums, decoded, function, held
from mx_oracle import HALF_STEP, round_to

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
DEV = "cuda"


def rnd(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def same(got, want):
    """equal values, NaN where the other has NaN"""
    got, want = got.cpu().double(), want.cpu().double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def tiny(dtype):
    """the smallest subnormal"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# -- quantisation ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("block_rows", (1, 128))
@pytest.mark.parametrize("shape", [(1, 1), (2, 31), (3, 128), (5, 129), (1, 127), (127, 640), (128, 128), (129, 257),
                                   (3, 511), (4, 512), (9, 513), (130, 1021), (257, 4096)])
def test_quantize_is_the_nearest_code(shape, block_rows, dtype):
    x = rnd(*shape, seed=shape[1], dtype=dtype) * torch.exp2(torch.arange(shape[0]) % 9 - 4.0)[:, None].to(dtype)
    q = ops.fp8_quantize(x.to(DEV), block_rows)
    assert q.shape == x.shape and q.nbytes == q.data.numel() + q.scales.numel()
    want = held(x, block_rows)
    got = decoded(q.data.cpu(), q.scales.cpu(), block_rows)
    same(got[:, :shape[1]], want)
    assert not got[:, shape[1]:].any()  # padding
    assert not q.scales.cpu()[:, -(-shape[1] // 128):].any()
    same(q.dequantize(torch.float32), want)
    for t in TYPES:
        same(q.dequantize(t), round_to(want, t))


@pytest.mark.parametrize("block_rows", (1, 128))
def test_quantize_ties_extremes_and_specials(block_rows):
    rows = []
    # every half step, and the values around the border where a block takes the next power of two
    values = [i * 2.0 ** -10 for i in range(64)] + [(1 + m / 32) * 2.0 ** e for e in range(-9, 9) for m in range(32)
                                                    if (1 + m / 32) * 2.0 ** e <= 448]
    for at in range(0, len(values), 127):
        rows.append(([448.0] + values[at:at + 127] + [0.0] * 127)[:128])
    rows.append([-v for v in rows[2]])
    for top in (447.9, 448.0, 448.1, 450.0, 511.9, 512.0):
        rows.append([top] + [top * i / 127 for i in range(127)])
    rows.append([0.0] * 128)
    rows.append([-0.0] * 127 + [1e-45])
    rows.append([1e-40 * i for i in range(128)])
    rows.append([3.4e38, -3.4e38] + [1.0] * 126)
    rows.append([2.0 ** -126 * i for i in range(128)])
    rows.append([2.0 ** -119] * 128)
    rows.append([math.nan] + [1.0] * 127)
    rows.append([1.0] * 127 + [math.inf])
    rows.append([1.0] * 7 + [-math.inf] + [2.0] * 120)
    x = torch.tensor(rows, dtype=torch.float32)
    if block_rows == 128:  # a block of its own for each row
        x = torch.nn.functional.pad(x[:, None], (0, 0, 0, 127)).reshape(-1, 128)
    for t in TYPES:
        y = x.to(t)
        q = ops.fp8_quantize(y.to(DEV), block_rows)
        same(decoded(q.data.cpu(), q.scales.cpu(), block_rows), held(y, block_rows))
        same(q.dequantize(torch.float32), held(y, block_rows).float())


@pytest.mark.parametrize("block_rows", (1, 128))
def test_quantize_special_blocks_leave_their_neighbours_alone(block_rows):
    x = rnd(300, 400)
    x[130, 140] = math.nan
    got = ops.fp8_quantize(x.to(DEV), block_rows).dequantize(torch.float32)
    same(got, held(x, block_rows))
    assert torch.isnan(got[130:130 + block_rows // 2, 128:256]).all() and torch.isnan(got).sum() == 128 * block_rows


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("block_rows", (1, 128))
def test_quantize_strides_offsets_and_shapes(block_rows, dtype):
    base = rnd(140, 700, seed=3, dtype=dtype).to(DEV)
    for view in (base[:, 1:513], base[3:135, 8:520], base[::3, :33], base.t(), base[:, ::2], base[1:2].expand(5, 700),
                 base.view(2, 70, 700), base[0], base[:0], base[:, :0], base.view(-1)[5:5 + 639 * 140].view(140, 639)):
        q = ops.fp8_quantize(view, block_rows)
        assert q.shape == view.shape
        if not view.numel():
            assert q.dequantize().shape == view.shape
            continue
        cols = view.shape[-1]
        same(q.dequantize(torch.float32).view(-1, cols), held(view.cpu().reshape(-1, cols), block_rows).float())


# -- product -----------------------------------------------------------------------------

def whole_numbers(rows, cols, most, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g).to(dtype)


SHAPES = [(1, 1, 1), (1, 16, 32), (2, 15, 31), (3, 17, 33), (1, 257, 127), (5, 33, 128), (8, 64, 129), (16, 40, 511),
          (17, 48, 512), (31, 16, 513), (33, 130, 640), (64, 31, 1040), (65, 129, 96), (130, 257, 260), (1, 300, 4096),
          (7, 100, 5003), (129, 513, 1021), (257, 300, 128), (256, 256, 512), (300, 520, 1100), (16, 2100, 16400),
          (40, 24, 9001)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_whole_numbers_is_exact(m, n, k, dtype):
    """Values up to 7 are 8-bit numbers at any scale; products are whole and at most 49, the unit of the cut behind
    eight of them is at most 2^(5 - 13), partial sums stay below 2^24: exact in any order, the result has one rounding."""
    x = whole_numbers(m, k, 7, m + k, dtype)
    wd = whole_numbers(n, k, 7, n + k)
    bias = whole_numbers(1, n, 99, 5, dtype)[0]
    assert 49 * k < 2 ** 23
    want = x.double() @ wd.double().t()
    x8 = ops.fp8_quantize(x.to(DEV))
    for block_rows in (1, 128):
        w = ops.fp8_quantize(wd.to(DEV), block_rows)
        same(ops.fp8_linear(x.to(DEV), w), round_to(want, dtype))
        same(ops.fp8_linear(x.to(DEV), w, bias.to(DEV)), round_to(want + bias.double(), dtype))
        same(ops.fp8_linear(x8, w, bias.to(DEV), dtype), round_to(want + bias.double(), dtype))


@pytest.mark.parametrize("m,n", [(1000, 1100), (4099, 2000), (300, 9000)])
def test_large_products_of_whole_numbers_are_exact(m, n):
    x, wd = whole_numbers(m, 700, 7, 1, torch.bfloat16).to(DEV), whole_numbers(n, 700, 7, 2).to(DEV)
    want = (x.double() @ wd.double().t())
    for block_rows in (1, 128):
        same(ops.fp8_linear(x, ops.fp8_quantize(wd, block_rows)), round_to(want.cpu(), torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES[:2], ids=IDS[:2])
@pytest.mark.parametrize("m,n,k", [(4096, 4096, 1024), (4097, 4101, 512), (8100, 6000, 1536), (3900, 5003, 2048)])
def test_products_of_whole_steps_are_exact(m, n, k, dtype):
    """rows of a multiple of 512 values: the tiles that workgroups go through one after the other, their ends, a scale of
    its own in every block, a bias"""
    up = torch.exp2(torch.arange(k) // 128 % 5 - 2.0).to(DEV)
    x, wd = (whole_numbers(rows, k, 7, seed).to(DEV) for rows, seed in ((m, 1), (n, 2)))
    rows = torch.exp2(torch.arange(m, device=DEV) % 3 - 1.0)[:, None]
    bias = whole_numbers(1, n, 99, 5, dtype)[0].to(DEV)
    want = (x * rows).double() @ wd.double().t() + bias.double()
    for block_rows in (1, 128):
        got = ops.fp8_linear((x * rows * up).to(dtype), ops.fp8_quantize(wd / up, block_rows), bias)
        same(got, round_to(want.cpu(), dtype))


@pytest.mark.parametrize("block_rows", (1, 128))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 200, 1024), (4, 131, 1001), (50, 60, 640), (70, 130, 300), (260, 48, 300)])
def test_product_of_random_values(m, n, k, dtype, block_rows):
    """16-bit results: eight products at a time, cut as stated; behind that each addition (k / 8 of eights, k / 128 of
    accumulators, 20 of parts) may be cut at 2^-23 of the largest it is added to.  float32 results: k 2^-23 of the sum of
    the magnitudes.  And half a step of the result."""
    x = rnd(m, k, seed=1, dtype=dtype) * torch.exp2(torch.arange(k) % 13 - 6.0).to(dtype)
    wd = rnd(n, k, seed=2, scale=0.02, dtype=torch.bfloat16)
    kept, exact, size, _ = cut_sums(x, wd, block_rows)
    want, adds = (exact, k) if dtype == torch.float32 else (kept, k / 8 + k / 128 + 20)
    got = ops.fp8_linear(x.to(DEV), ops.fp8_quantize(wd.to(DEV), block_rows)).cpu().double()
    tol = HALF_STEP[dtype] * want.abs() + adds * 2.0 ** -23 * size * (1 + HALF_STEP[dtype]) + tiny(dtype)
    assert ((got - want).abs() <= tol).all()


def test_product_of_wide_ranges_of_scales():
    """blocks whose scales are as far apart as bf16 goes: nothing overflows on the way to a result in range"""
    k = 1024
    up = torch.exp2((torch.arange(k) // 128 * 25 - 100).float())
    x, wd = torch.ones(3, k) * up, torch.ones(20, k) / up * (1 + torch.arange(20) % 15)[:, None]
    for block_rows in (1, 128):
        w = ops.fp8_quantize(wd.to(DEV), block_rows)
        for m in (3, 40):
            y = x[:1].expand(m, k).contiguous()
            same(ops.fp8_linear(y.to(DEV), w), (held(y) @ held(wd, block_rows).t()).float())
            same(ops.fp8_linear(y.bfloat16().to(DEV), w), round_to(held(y) @ held(wd, block_rows).t(), torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m", (1, 9, 70, 300))
def test_product_keeps_nan_where_it_is(m, dtype):
    k, n = 600, 140
    x, wd = rnd(m, k, dtype=dtype), rnd(n, k, seed=1)
    x[m // 2, 5] = math.nan
    wd[130, 599] = math.inf
    for block_rows in (1, 128):
        got = ops.fp8_linear(x.to(DEV), ops.fp8_quantize(wd.to(DEV), block_rows)).cpu()
        want = torch.zeros(m, n, dtype=torch.bool)
        want[m // 2] = True
        want[:, 130 if block_rows == 1 else slice(128, None)] = True
        assert torch.equal(torch.isnan(got), want)


@pytest.mark.parametrize("block_rows", (1, 128))
def test_large_tiles_keep_nan_where_it_is(block_rows):
    m, n, k = 2500, 2300, 1024
    x, wd = rnd(m, k, dtype=torch.bfloat16).to(DEV), rnd(n, k, seed=1).to(DEV)
    x[2049, 5], wd[130, 600] = math.nan, math.inf
    w = ops.fp8_quantize(wd, block_rows)
    bad = slice(130, 131) if block_rows == 1 else slice(128, 256)
    want = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    want[2049] = True
    want[:, bad] = True
    assert torch.equal(torch.isnan(ops.fp8_linear(x, w)), want)
    g = rnd(m, n, seed=2, dtype=torch.bfloat16).to(DEV)
    leaf = x.clone().requires_grad_(True)
    dx = torch.autograd.grad(ops.fp8_linear(leaf, w), leaf, g)[0]
    want = torch.zeros(m, k, dtype=torch.bool, device=DEV)
    want[:, 512:640] = True  # the block of columns that the infinity is in
    assert torch.equal(torch.isnan(dx), want)
    dw = ops.fp8_weight_gradient(g, ops.fp8_quantize(x))
    want = torch.zeros(n, k, dtype=torch.bool, device=DEV)
    want[:, :128] = True
    assert torch.equal(torch.isnan(dw), want)


def test_product_shapes_strides_and_empty():
    wd = whole_numbers(24, 96, 7, 1)
    w = ops.fp8_quantize(wd.to(DEV), 128)
    x = whole_numbers(30, 200, 7, 2, torch.bfloat16).to(DEV)
    for view in (x[:, 3:99], x[::2, 8:104], x[4, :96], x[:, :96].view(5, 6, 96), x[:2, :96].unsqueeze(1).expand(2, 3, 96),
                 x[:0, :96], x.t()[:96, :7].t()):
        same(ops.fp8_linear(view, w), round_to(view.cpu().double() @ wd.double().t(), torch.bfloat16))
    none = ops.fp8_quantize(torch.zeros(24, 0, device=DEV), 128)
    bias = torch.arange(24, device=DEV, dtype=torch.float32)
    same(ops.fp8_linear(torch.zeros(3, 0, device=DEV), none, bias), bias.expand(3, 24))
    assert ops.fp8_linear(x[:, :96], ops.fp8_quantize(torch.zeros(0, 96, device=DEV))).shape == (30, 0)
    flipped = torch.complex(torch.zeros(24), torch.arange(24.0)).conj().imag.to(DEV)  # its memory holds the other sign
    same(ops.fp8_linear(torch.zeros(3, 96, device=DEV), w, torch.complex(flipped * 0, -flipped).conj().imag),
         flipped.expand(3, 24))


# -- gradients ---------------------------------------------------------------------------

GRADIENTS = [(1, 1, 1), (3, 17, 33), (16, 130, 127), (33, 64, 128), (70, 129, 260), (64, 500, 640), (129, 257, 513),
             (300, 1021, 300), (2, 2100, 520), (520, 72, 1030)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", GRADIENTS)
def test_gradients_of_whole_numbers_are_exact(m, n, k, dtype):
    """values up to 7, sums below 2^24"""
    g, wd, xd = whole_numbers(m, n, 7, 1, dtype), whole_numbers(n, k, 7, 2), whole_numbers(m, k, 7, 3)
    out = whole_numbers(n, k, 99, 4, dtype)
    dx, dw = g.double() @ wd.double(), g.double().t() @ xd.double()
    x = xd.to(dtype).to(DEV).requires_grad_(True)
    for block_rows in (1, 128):
        y = ops.fp8_linear(x, ops.fp8_quantize(wd.to(DEV), block_rows))
        same(torch.autograd.grad(y, x, g.to(DEV))[0], round_to(dx, dtype))
        x8 = ops.fp8_quantize(xd.to(DEV), block_rows)
        same(ops.fp8_weight_gradient(g.to(DEV), x8), round_to(dw, dtype))
        room = torch.full((n + 2, k), 5.0, dtype=dtype, device=DEV)
        room[1:-1] = out.to(DEV)
        assert ops.fp8_weight_gradient(g.to(DEV), x8, out=room[1:-1]).data_ptr() == room[1:-1].data_ptr()
        same(room[1:-1], round_to(out.double() + dw, dtype))
        assert (room[0] == 5).all() and (room[-1] == 5).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(4096, 1024, 1030), (2050, 520, 2051), (1000, 6000, 300), (5000, 257, 4100)])
def test_large_gradients_of_whole_numbers_are_exact(m, n, k, dtype):
    """the larger tiles, whole and in parts, their ends, and scales of their own in every block"""
    g, xd = whole_numbers(m, n, 7, 1, dtype).to(DEV), whole_numbers(m, k, 7, 3).to(DEV)
    up = torch.exp2(torch.arange(n) // 128 % 5 - 2.0).to(DEV)[:, None] * torch.exp2(torch.arange(k) // 128 % 3 - 1.0).to(DEV)
    wd = whole_numbers(n, k, 7, 2).to(DEV) * up
    x = xd.to(dtype).requires_grad_(True)
    want = round_to((g.double() @ wd.double()).cpu(), dtype)
    for block_rows in (1, 128):
        y = ops.fp8_linear(x, ops.fp8_quantize(wd, block_rows))
        same(torch.autograd.grad(y, x, g)[0], want)
    down = torch.exp2(torch.arange(m) % 5 - 2.0).to(DEV)[:, None]
    same(ops.fp8_weight_gradient((g / down).to(dtype), ops.fp8_quantize(xd * down)),
         round_to((g.double().t() @ xd.double()).cpu(), dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(40, 300, 200), (333, 257, 130), (700, 128, 1021), (2048, 64, 128)])
def test_gradients_of_random_values(m, n, k, dtype):
    """Sums in 32 bits over as many products as the type of the gradient has planes of bf16 numbers, and half a step"""
    planes = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    g = rnd(m, n, seed=1, scale=1e-2, dtype=dtype)
    wd, xd = rnd(n, k, seed=2, scale=0.02), rnd(m, k, seed=3) * torch.exp2(torch.arange(m) % 11 - 5.0)[:, None]
    for block_rows in (1, 128):
        w64, x64, g64 = held(wd, block_rows), held(xd, block_rows), g.double()
        x = xd.to(dtype).to(DEV).requires_grad_(True)
        y = ops.fp8_linear(x, ops.fp8_quantize(wd.to(DEV), block_rows))
        got = torch.autograd.grad(y, x, g.to(DEV))[0].cpu().double()
        want, size = g64 @ w64, g64.abs() @ w64.abs()
        tol = HALF_STEP[dtype] * want.abs() + planes * n * 2.0 ** -23 * size + tiny(dtype)
        assert ((got - want).abs() <= tol).all()
        x8 = ops.fp8_quantize(xd.to(DEV), block_rows)
        got = ops.fp8_weight_gradient(g.to(DEV), x8).cpu().double()
        want, size = g64.t() @ x64, g64.t().abs() @ x64.abs()
        tol = HALF_STEP[dtype] * want.abs() + planes * m * 2.0 ** -23 * size + tiny(dtype)
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_gradients_of_strided_and_odd_places(dtype):
    m, n, k = 70, 40, 140
    base = whole_numbers(2 * m, n + 9, 7, 1, dtype).to(DEV)
    w = ops.fp8_quantize(whole_numbers(n, k, 7, 2).to(DEV), 128)
    x8 = ops.fp8_quantize(whole_numbers(m, k, 7, 3).to(DEV))
    for g in (base[:m, 1:n + 1], base[::2, :n], base[:m, 8:n + 8], base[:n, :m - 30].t()[:, :n], base[:1, :n].expand(m, n)):
        rows = g.shape[0]
        x = torch.zeros(rows, k, dtype=dtype, device=DEV, requires_grad=True)
        same(torch.autograd.grad(ops.fp8_linear(x, w), x, g)[0],
             round_to(g.cpu().double() @ w.dequantize(torch.float32).cpu().double(), dtype))
        if rows == m:
            same(ops.fp8_weight_gradient(g, x8),
                 round_to(g.cpu().double().t() @ x8.dequantize(torch.float32).cpu().double(), dtype))
    batch = ops.FP8Tensor(x8.data, x8.scales, (7, 10, k))
    g = base[:m, :n].contiguous().view(7, 10, n)
    same(ops.fp8_weight_gradient(g, batch), ops.fp8_weight_gradient(g.view(m, n), x8))


def test_gradients_of_nothing():
    none = ops.fp8_quantize(torch.zeros(0, 70, device=DEV))
    assert not ops.fp8_weight_gradient(torch.zeros(0, 5, device=DEV), none).any()
    out = torch.ones(5, 70, device=DEV)
    assert ops.fp8_weight_gradient(torch.zeros(0, 5, device=DEV), none, out=out) is out and (out == 1).all()
    x8 = ops.fp8_quantize(torch.ones(3, 70, device=DEV))
    assert ops.fp8_weight_gradient(torch.zeros(3, 0, device=DEV), x8).shape == (0, 70)
    x = torch.ones(3, 70, device=DEV, requires_grad=True)
    y = ops.fp8_linear(x, ops.fp8_quantize(torch.zeros(0, 70, device=DEV)))
    assert not torch.autograd.grad(y, x, torch.zeros(3, 0, device=DEV))[0].any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m", (70, 64))
def test_infinities_in_the_last_row_stay_in_their_row_and_column(m, dtype):
    """the last row is read again where a step of 64 rows goes beyond it; what is read again counts as zero"""
    g, xd = rnd(m, 48, seed=1, dtype=dtype), whole_numbers(m, 140, 7, 2)
    xd[m - 1] = 1.0
    g[m - 1, 5], g[m - 1, 7] = math.inf, math.nan
    got = ops.fp8_weight_gradient(g.to(DEV), ops.fp8_quantize(xd.to(DEV))).cpu()
    assert (got[5] == math.inf).all() and torch.isnan(got[7]).all()
    rest = [i for i in range(48) if i not in (5, 7)]
    assert torch.isfinite(got[rest]).all()
    xd[m - 1, 130] = math.nan
    g[m - 1, 5] = g[m - 1, 7] = 0.0
    got = ops.fp8_weight_gradient(g.to(DEV), ops.fp8_quantize(xd.to(DEV))).cpu()
    assert torch.isnan(got[:, 128:]).all() and torch.isfinite(got[:, :128]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_infinities_of_a_gradient_reach_the_rows_gradient(dtype):
    g, wd = rnd(9, 70, seed=1, dtype=dtype), whole_numbers(70, 140, 7, 2).abs() + 1
    g[4, 69], g[6, 0] = math.inf, math.nan
    x = torch.zeros(9, 140, dtype=dtype, device=DEV, requires_grad=True)
    got = torch.autograd.grad(ops.fp8_linear(x, ops.fp8_quantize(wd.to(DEV), 128)), x, g.to(DEV))[0].cpu()
    assert (got[4] == math.inf).all() and torch.isnan(got[6]).all()
    assert torch.isfinite(got[[0, 1, 2, 3, 5, 7, 8]]).all()


def test_gradients_against_differences():
    """a product of 8-bit rows that are whole numbers moves by whole numbers: differences of it are its gradient"""
    m, n, k = 5, 12, 130
    wd, g = whole_numbers(n, k, 7, 2), whole_numbers(m, n, 3, 3)
    x = whole_numbers(m, k, 6, 1).to(DEV)
    x[:, 0] = 7  # every block keeps its scale: the largest stays
    x[:, 128] = 7
    w = ops.fp8_quantize(wd.to(DEV), 128)

    def value(x):
        return (ops.fp8_linear(x, w).double() * g.to(DEV).double()).sum().item()

    leaf = x.clone().requires_grad_(True)
    dx = torch.autograd.grad(ops.fp8_linear(leaf, w), leaf, g.to(DEV))[0]
    dense = wd.to(DEV).clone()
    dw = ops.fp8_weight_gradient(g.to(DEV), ops.fp8_quantize(x))
    for i, j in ((0, 1), (2, 77), (4, 129)):
        up, down = x.clone(), x.clone()
        up[i, j] += 1
        down[i, j] -= 1
        assert (value(up) - value(down)) / 2 == dx[i, j].item()
    for i, j in ((0, 3), (11, 129), (7, 64)):
        up, down = dense.clone(), dense.clone()
        up[i, j] += 1
        down[i, j] -= 1
        move = ((x.double() @ up.double().t() - x.double() @ down.double().t()) * g.to(DEV).double()).sum() / 2
        assert move.item() == dw[i, j].item()


def test_the_same_bits_every_time():
    x, w = rnd(700, 1000, dtype=torch.bfloat16).to(DEV), ops.fp8_quantize(rnd(520, 1000, seed=1).to(DEV), 128)
    g = rnd(700, 520, seed=2, dtype=torch.bfloat16).to(DEV)
    x8 = ops.fp8_quantize(x)
    first = ops.fp8_linear(x, w), ops.fp8_weight_gradient(g, x8)
    for _ in range(3):
        assert torch.equal(ops.fp8_linear(x, w), first[0]) and torch.equal(ops.fp8_weight_gradient(g, x8), first[1])
    assert torch.equal(ops.fp8_linear(x8, w), first[0])


# -- activation functions ----------------------------------------------------------------

KINDS = ("gelu", "gelu_tanh", "silu")


def activation_tolerances(kind, x, dtype):
    """For f and f' at ``x`` (float64): half a step of the result aside, ten roundings and approximations of 2^-23 each
    (2^-19 with room), and the rounding of the exponent, of which f has the exponential: its magnitude times 2^-22.  f'
    is a sum, each of whose terms has that; where the integral is 1 - tail the same is of 1.  An exponential below the
    normal range may be lost, 2^-126, which f multiplies with x and f' with x u', both at most 1 + 3 |u|."""
    f, slope, u = function(kind, x)
    rel = 2.0 ** -19 + 2.0 ** -22 * u.clamp(max=200)
    p = torch.where(x == 0, torch.full_like(x, 0.5), f / x)
    lost = 2.0 ** -126 * (1 + 3 * u.clamp(max=200))
    return f, slope, rel * f.abs() + lost, rel * (p.abs() + (slope - p).abs()) + lost


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 127), (5, 128), (2, 513), (70, 1021), (3, 4, 640)])
def test_activation_functions(shape, kind, dtype):
    x = rnd(*shape, seed=shape[-1], scale=2.5, dtype=dtype)
    up, g = rnd(*shape, seed=1, dtype=dtype), rnd(*shape, seed=2, scale=1e-2, dtype=dtype)
    cols, half = shape[-1], HALF_STEP[dtype]
    x64, u64, g64 = (t.double().view(-1, cols) for t in (x, up, g))
    x8, u8 = held(x.view(-1, cols)), held(up.view(-1, cols))
    low = tiny(dtype) + 2.0 ** -126  # a subnormal result; the exponential below the normal range
    f, _, f_tol, _ = activation_tolerances(kind, x64, dtype)
    f8, slope, f8_tol, slope_tol = activation_tolerances(kind, x8, dtype)

    def near(got, want, tol):
        assert got.shape == x.shape
        got = got.detach().cpu().double().view(-1, cols)
        assert ((got - want).abs() <= tol * (1 + half) + half * want.abs() + low).all()

    a, b = x.to(DEV).requires_grad_(True), up.to(DEV).requires_grad_(True)
    y = ops.fp8_activation(a, kind)
    near(y, f, f_tol)
    near(torch.autograd.grad(y, a, g.to(DEV))[0], g64 * slope, g64.abs() * (slope_tol + 2.0 ** -23 * slope.abs()))
    y = ops.fp8_activation(a, kind, b)
    near(y, f * u64, (f_tol + 2.0 ** -23 * f.abs()) * u64.abs())
    da, db = torch.autograd.grad(y, (a, b), g.to(DEV))
    gu = (g64 * u8).abs()
    near(da, g64 * u8 * slope, gu * (slope_tol + 2.0 ** -22 * slope.abs()))
    near(db, g64 * f8, g64.abs() * (f8_tol + 2.0 ** -22 * f8.abs()))
    with torch.no_grad():
        assert torch.equal(ops.fp8_activation(a, kind), ops.fp8_activation(x.to(DEV), kind))
        assert torch.equal(ops.fp8_activation(a, kind, b), y)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=("bf16", "fp32"))
@pytest.mark.parametrize("kind", KINDS)
def test_activation_functions_far_out(kind, dtype):
    """finite results for every finite value, and the limits of f and f'; a block with an infinity reads as NaN"""
    x = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 12.0, -12.0, 88.0, -88.0, 100.0, -100.0, 1e10, -1e10, 1e30, -1e30, 3e38,
                       -3e38] + [0.0] * 112]).to(dtype)
    x = torch.stack([torch.cat([x[0, i:i + 1], torch.zeros(127, dtype=dtype)]) for i in range(16)])  # a block for each
    a = x.to(DEV).requires_grad_(True)
    y = ops.fp8_activation(a, kind)
    da = torch.autograd.grad(y, a, torch.ones_like(y))[0].cpu().double()
    y = y.detach().cpu().double()
    want, slope, tol, slope_tol = activation_tolerances(kind, held(x), dtype)
    full, _, full_tol, _ = activation_tolerances(kind, x.double(), dtype)
    # the oracle's own x^3 overflows to nothing for these: limits instead
    big = x.double().abs() > 1e20
    full = torch.where(big, x.double().clamp(min=0), full)
    slope = torch.where(big, (x.double() > 0).double(), slope)
    assert torch.isfinite(y).all() and torch.isfinite(da).all()
    assert ((y - full).abs() <= HALF_STEP[dtype] * full.abs() + torch.where(big, 0.0, full_tol) * 1.01 + 2.0 ** -125).all()
    assert ((da - slope).abs() <= HALF_STEP[dtype] * slope.abs() + torch.where(big, 2.0 ** -20, slope_tol) * 1.01
            + 2.0 ** -120).all()
    z = torch.zeros(3, 256, dtype=dtype)
    z[0, 3], z[1, 200], z[2, 0] = math.nan, math.inf, -math.inf
    for up in (None, torch.ones(3, 256, dtype=dtype, device=DEV)):
        a = z.to(DEV).requires_grad_(True)
        y = ops.fp8_activation(a, kind, up)
        da = torch.autograd.grad(y, a, torch.ones_like(y))[0].cpu()
        nan = torch.zeros(3, 256, dtype=torch.bool)
        nan[0, :128] = nan[1, 128:] = nan[2, :128] = True
        assert torch.equal(torch.isnan(da), nan)
        assert y[1, 200] == math.inf and torch.isnan(y[0, 3]) and torch.isnan(y[2, 0])
        assert (y.detach()[:, 5:190] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_activation_slope_against_differences(kind):
    """float32 values that 8 bits hold: f' against the differences of f at them, in float64 behind the call's rounding"""
    x = (torch.arange(128) % 15 - 7).float()[None] / 2
    x[0, 0] = 3.5
    step = 2.0 ** -6
    a = x.to(DEV).requires_grad_(True)
    da = torch.autograd.grad(ops.fp8_activation(a, kind), a, torch.ones(1, 128, device=DEV))[0].cpu().double()
    with torch.no_grad():
        up, down = (ops.fp8_activation((x + s).to(DEV), kind).cpu().double() for s in (step, -step))
    # third derivatives of these functions are below 2.5; values up to 4 with an error of 2^-18 relative, divided by 2 steps
    assert ((up - down) / (2 * step) - da).abs().max() <= 2.5 * step * step / 6 + 4 * 2.0 ** -18 / step


def test_activation_strides():
    both = rnd(9, 2 * 300, dtype=torch.bfloat16).to(DEV)
    gate, up = both[:, :300], both[:, 300:]
    assert torch.equal(ops.fp8_activation(gate, "silu", up),
                       ops.fp8_activation(gate.contiguous(), "silu", up.contiguous()))
    a = both.clone().requires_grad_(True)
    y = ops.fp8_activation(a[:, :300], "silu", a[:, 300:])
    g = rnd(9, 601, seed=1, dtype=torch.bfloat16).to(DEV)[:, 1::2]
    got = torch.autograd.grad(y, a, g)[0]
    b, c = gate.contiguous().requires_grad_(True), up.contiguous().requires_grad_(True)
    want = torch.autograd.grad(ops.fp8_activation(b, "silu", c), (b, c), g.contiguous())
    assert torch.equal(got, torch.cat(want, 1))
    same_input = gate.contiguous().requires_grad_(True)  # f(x) x: both gradients reach one leaf
    y = ops.fp8_activation(same_input, "silu", same_input)
    got = torch.autograd.grad(y, same_input, torch.ones_like(y))[0]
    b, c = (gate.contiguous().requires_grad_(True) for _ in range(2))
    want = torch.autograd.grad(ops.fp8_activation(b, "silu", c), (b, c), torch.ones_like(y))
    assert torch.equal(got, want[0] + want[1])
    wide = both[:1, :300].expand(4, 300)
    assert torch.equal(ops.fp8_activation(wide), ops.fp8_activation(wide.contiguous()))
    for empty in (both[:0], both[:, :0]):
        e = empty.detach().requires_grad_(True)
        assert torch.autograd.grad(ops.fp8_activation(e).sum(), e)[0].shape == e.shape
