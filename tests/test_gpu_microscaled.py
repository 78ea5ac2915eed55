"""GPU: weights in microscaled 4 bits (quantisation, values, products, lookup)
against float64 on the CPU."""
import math

import pytest
import torch

import neuzip_amd
from neuzip_amd import _lib, ops
from mx_oracle import HALF_STEP, decoded, held, round_to

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


# -- quantisation ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("bits", (4, 8))
@pytest.mark.parametrize("shape", [(1, 1), (2, 31), (3, 32), (5, 33), (1, 127), (7, 128), (2, 129), (3, 511), (4, 512),
                                   (9, 513), (130, 1021), (33, 4096)])
def test_quantize_is_the_nearest_code(shape, bits, dtype):
    x = rnd(*shape, seed=shape[1], dtype=dtype) * torch.exp2(torch.arange(shape[0]) % 9 - 4.0)[:, None].to(dtype)
    q = ops.mx_quantize(x.to(DEV), bits)
    assert q.shape == x.shape and q.nbytes == q.data.numel() + q.scales.numel()
    want = held(x, bits)
    got = decoded(q.data.cpu(), q.scales.cpu(), shape[1], bits)
    same(got[:, :shape[1]], want)
    assert not got[:, shape[1]:].any()  # padding
    blocks = -(-shape[1] // 32)
    used = {(b // 16) * 16 + 4 * (b % 4) + (b % 16) // 4 for b in range(blocks)}
    rest = [i for i in range(q.scales.shape[1]) if i not in used]
    assert not q.scales.cpu()[:, rest].any()
    same(q.dequantize(torch.float32), want)
    for t in TYPES:
        same(q.dequantize(t), round_to(want, t))


@pytest.mark.parametrize("bits", (4, 8))
def test_quantize_ties_extremes_and_specials(bits):
    step = {4: 0.25, 8: 2.0 ** -10}[bits]
    top = {4: 6.0, 8: 448.0}[bits]
    rows = []
    # every half step up to twice the largest value, in blocks whose largest magnitude fixes the scale at 1
    lead = {4: 4.0, 8: 256.0}[bits]
    values = [i * step for i in range(64)] + [v for e in range(-9, 9) for m in range(32)
                                              for v in [(1 + m / 32) * 2.0 ** e] if v <= 2 * lead - step]
    for at in range(0, len(values), 31):
        rows.append(([lead] + values[at:at + 31] + [0.0] * 31)[:32])
    rows.append([-v for v in rows[3]])
    rows.append([top] + [top * (1 + i / 64) for i in range(31)])  # beyond the largest code
    rows.append([0.0] * 32)
    rows.append([-0.0] * 31 + [1e-45])
    rows.append([1e-40 * i for i in range(32)])
    rows.append([3.4e38, -3.4e38] + [1.0] * 30)
    rows.append([2.0 ** -126 * i for i in range(32)])
    rows.append([math.nan] + [1.0] * 31)
    rows.append([1.0] * 31 + [math.inf])
    rows.append([1.0] * 7 + [-math.inf] + [2.0] * 24)
    x = torch.tensor(rows, dtype=torch.float32)
    for t in TYPES:
        y = x.to(t)
        q = ops.mx_quantize(y.to(DEV), bits)
        same(decoded(q.data.cpu(), q.scales.cpu(), 32, bits)[:, :32], held(y, bits))
        same(q.dequantize(torch.float32), held(y, bits).float())


def test_quantize_special_blocks_leave_their_neighbours_alone():
    x = rnd(3, 200)
    x[1, 70] = math.nan
    got = ops.mx_quantize(x.to(DEV), 4).dequantize(torch.float32)
    same(got, held(x, 4))
    assert torch.isnan(got[1, 64:96]).all() and torch.isnan(got).sum() == 32


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("bits", (4, 8))
def test_quantize_strides_offsets_and_shapes(bits, dtype):
    base = rnd(40, 700, seed=3, dtype=dtype).to(DEV)
    for view in (base[:, 1:513], base[3:11, 8:520], base[::3, :33], base.t(), base[:, ::2], base[1:2].expand(5, 700),
                 base.view(2, 20, 700), base[0], base[:0], base[:, :0], base.view(-1)[5:5 + 639 * 40].view(40, 639)):
        q = ops.mx_quantize(view, bits)
        assert q.shape == view.shape
        if not view.numel():
            assert q.dequantize().shape == view.shape
            continue
        cols = view.shape[-1]
        same(q.dequantize(torch.float32).view(-1, cols), held(view.cpu().reshape(-1, cols), bits).float())


# -- product -----------------------------------------------------------------------------

def whole_numbers(rows, cols, most, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g).to(dtype)


SHAPES = [(1, 1, 1), (1, 16, 32), (2, 15, 31), (3, 17, 33), (1, 257, 127), (5, 33, 128), (8, 64, 129), (16, 40, 511),
          (17, 48, 512), (31, 16, 513), (33, 130, 640), (64, 31, 1040), (65, 129, 96), (130, 257, 260), (1, 300, 4096),
          (7, 100, 5003), (129, 513, 1021), (257, 300, 128), (256, 256, 512), (300, 520, 1100)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_of_whole_numbers_is_exact(m, n, k, dtype):
    """Values up to 7 are 8-bit numbers; every partial sum is a multiple of 2^-1 below 2^24 (at most
    7 * 6 * k): 32-bit sums are exact in any order, the result has one rounding."""
    x = whole_numbers(m, k, 7, m + k, dtype)
    w = ops.mx_quantize(whole_numbers(n, k, 6, n + k).to(DEV), 4)
    bias = whole_numbers(1, n, 99, 5, dtype)[0]
    w64 = decoded(w.data.cpu(), w.scales.cpu(), k, 4)[:, :k]
    assert 7 * 6 * k < 2 ** 23
    want = x.double() @ w64.t()
    same(ops.mx_linear(x.to(DEV), w), round_to(want, dtype))
    same(ops.mx_linear(x.to(DEV), w, bias.to(DEV)), round_to(want + bias.double(), dtype))
    x8 = ops.mx_quantize(x.to(DEV), 8)
    same(ops.mx_linear(x8, w, bias.to(DEV), dtype), round_to(want + bias.double(), dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 1024, 4096), (4, 509, 3001), (50, 333, 2048), (150, 1021, 1000), (600, 768, 777)])
def test_product_of_random_values(m, n, k, dtype):
    """Sums of k products in 32 bits: k 2^-23 of the sum of the magnitudes (an addition may cut off instead
    of rounding), and half a step of the result."""
    x = rnd(m, k, seed=1, dtype=dtype) * torch.exp2(torch.arange(k) % 7 - 3.0).to(dtype)
    wd = rnd(n, k, seed=2, scale=0.02, dtype=torch.bfloat16)
    w = ops.mx_quantize(wd.to(DEV), 4)
    x64, w64 = held(x, 8), held(wd, 4)
    want, size = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    got = ops.mx_linear(x.to(DEV), w).cpu().double()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got - want).abs() <= HALF_STEP[dtype] * want.abs() + k * 2.0 ** -23 * size + tiny).all()


def test_product_of_wide_ranges_of_scales():
    """blocks whose scales are as far apart as bf16 goes: nothing overflows on the way to a result in range"""
    k = 512
    x = torch.ones(3, k) * torch.exp2((torch.arange(k) // 32 * 12 - 90).float())
    wd = torch.ones(20, k) * torch.exp2(-(torch.arange(k) // 32 * 12 - 90).float()) * (1 + torch.arange(20))[:, None]
    w = ops.mx_quantize(wd.to(DEV), 4)
    same(ops.mx_linear(x.to(DEV), w), held(x, 8) @ held(wd, 4).t())


@pytest.mark.parametrize("m", (1, 9, 70, 300))
def test_product_keeps_nan_where_it_is(m):
    k, n = 600, 40
    x, wd = rnd(m, k), rnd(n, k, seed=1)
    x[m // 2, 5] = math.nan
    wd[7, 599] = math.inf
    got = ops.mx_linear(x.to(DEV), ops.mx_quantize(wd.to(DEV), 4)).cpu()
    want = torch.zeros(m, n, dtype=torch.bool)
    want[m // 2] = True
    want[:, 7] = True
    assert torch.equal(torch.isnan(got), want)


def test_product_shapes_strides_and_empty():
    w = ops.mx_quantize(whole_numbers(24, 96, 6, 1).to(DEV), 4)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), 96, 4)[:, :96]
    x = whole_numbers(30, 200, 7, 2, torch.bfloat16).to(DEV)
    for view in (x[:, 3:99], x[::2, 8:104], x[4, :96], x[:, :96].view(5, 6, 96), x[:2, :96].unsqueeze(1).expand(2, 3, 96),
                 x[:0, :96], x.t()[:96, :7].t()):
        same(ops.mx_linear(view, w), round_to(view.cpu().double() @ w64.t(), torch.bfloat16))
    none = ops.mx_quantize(torch.zeros(24, 0, device=DEV), 4)
    bias = torch.arange(24, device=DEV, dtype=torch.float32)
    same(ops.mx_linear(torch.zeros(3, 0, device=DEV), none, bias), bias.expand(3, 24))
    assert ops.mx_linear(x[:, :96], ops.mx_quantize(torch.zeros(0, 96, device=DEV), 4)).shape == (30, 0)


def test_result_of_a_row_does_not_depend_on_the_rows_beside_it_by_more_than_rounding():
    k, n = 2048, 320
    x, w = rnd(200, k, dtype=torch.bfloat16).to(DEV), ops.mx_quantize(rnd(n, k, seed=1).to(DEV), 4)
    y = ops.mx_linear(x, w)
    size = held(x.cpu(), 8).abs() @ held(rnd(n, k, seed=1), 4).abs().t()
    for m in (1, 2, 16, 17, 64, 128):
        part = ops.mx_linear(x[:m], w)
        # two roundings of sums that differ by their order
        tol = 2 * 2.0 ** -8 * y[:m].cpu().double().abs() + 2 * k * 2.0 ** -23 * size[:m]
        assert ((part - y[:m]).cpu().double().abs() <= tol).all()
        assert torch.equal(part, ops.mx_linear(x[:m], w))  # the same bits every time


# -- gradient ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gradient_of_whole_numbers_is_exact(m, n, k, dtype):
    """gradients of up to 10 bits (bf16: 8): partial sums are multiples of 2^-1 below 2^24"""
    most = 127 if dtype == torch.bfloat16 else 1000
    assert most * 6 * n * 2 < 2 ** 24
    g = whole_numbers(m, n, most, m + n, dtype)
    w = ops.mx_quantize(whole_numbers(n, k, 6, n + k).to(DEV), 4)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), k, 4)[:, :k]
    x = torch.zeros(m, k, dtype=dtype, device=DEV, requires_grad=True)
    bias = torch.zeros(n, dtype=dtype, device=DEV, requires_grad=True)
    ops.mx_linear(x, w, bias).backward(g.to(DEV))
    same(x.grad, round_to(g.double() @ w64, dtype))
    want = g.double().sum(0)
    assert ((bias.grad.cpu().double() - want).abs() <= 2 * HALF_STEP[dtype] * g.double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(40, 1021, 777), (333, 512, 2048), (300, 3001, 300)])
def test_gradient_of_random_values(m, n, k, dtype):
    """Every value of the gradient is taken with all its bits (float32: three parts of 8 bits, the last of
    them rounded at 2^-24 of the value, half of which it may be off by), sums of n (three n) products in 32 bits."""
    g = rnd(m, n, seed=1, scale=0.01, dtype=dtype)
    wd = rnd(n, k, seed=2, scale=0.02, dtype=torch.bfloat16)
    w = ops.mx_quantize(wd.to(DEV), 4)
    x = torch.zeros(m, k, dtype=dtype, device=DEV, requires_grad=True)
    ops.mx_linear(x, w).backward(g.to(DEV))
    w64 = held(wd, 4)
    want, size = g.double() @ w64, g.double().abs() @ w64.abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tol = HALF_STEP[dtype] * want.abs() + (3 * n + 1) * 2.0 ** -23 * size + tiny
    assert ((x.grad.cpu().double() - want).abs() <= tol).all()


def test_gradient_against_differences():
    """x and the steps are whole numbers that 8 bits hold: the product is linear there"""
    m, n, k = 3, 70, 65
    x, g = whole_numbers(m, k, 3, 1), whole_numbers(m, n, 50, 2)
    w = ops.mx_quantize(whole_numbers(n, k, 6, 3).to(DEV), 4)
    xg = x.to(DEV).requires_grad_(True)
    ops.mx_linear(xg, w).backward(g.to(DEV))
    for seed in range(4):
        e = whole_numbers(m, k, 3, 10 + seed)
        diff = ops.mx_linear((x + e).to(DEV), w) - ops.mx_linear(x.to(DEV), w)
        assert (diff.cpu().double() * g.double()).sum() == (xg.grad.cpu().double() * e.double()).sum()


def test_gradient_of_large_and_special_values():
    w = ops.mx_quantize(whole_numbers(33, 64, 6, 1).to(DEV), 4)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), 64, 4)[:, :64]
    for dtype, big in ((torch.float32, 2.0 ** 100), (torch.float32, 2.0 ** -120), (torch.float16, 2.0 ** -24),
                       (torch.bfloat16, 2.0 ** 100)):
        g = torch.zeros(2, 33, dtype=dtype)
        g[0, 5], g[1, 32] = big, -big
        x = torch.zeros(2, 64, dtype=dtype, device=DEV, requires_grad=True)
        ops.mx_linear(x, w).backward(g.to(DEV))
        same(x.grad, round_to(g.double() @ w64, dtype))
    g = torch.zeros(3, 33)
    g[1, 4] = math.nan
    x = torch.zeros(3, 64, device=DEV, requires_grad=True)
    ops.mx_linear(x, w).backward(g.to(DEV))
    bad = torch.isnan(x.grad.cpu())
    assert bad[1].all() and not bad[0].any() and not bad[2].any()


def test_gradient_of_weights_that_read_as_nan():
    wd = whole_numbers(20, 200, 6, 1)
    wd[7, 70] = math.inf
    w = ops.mx_quantize(wd.to(DEV), 4)
    for dtype in TYPES:
        x = torch.zeros(3, 200, dtype=dtype, device=DEV, requires_grad=True)
        ops.mx_linear(x, w).backward(torch.zeros(3, 20, dtype=dtype, device=DEV))
        bad = torch.isnan(x.grad.cpu())
        assert bad[:, 64:96].all() and bad.sum() == 3 * 32


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 5, 40000), (3, 70, 20011), (2, 33000, 40), (9000, 3, 70), (1100, 530, 2600)])
def test_long_and_narrow(m, n, k, dtype):
    """whole numbers again; partial sums are multiples of 2^-1 below 2^22"""
    x = whole_numbers(m, k, 7, 1, dtype)
    w = ops.mx_quantize(whole_numbers(n, k, 6, 2).to(DEV), 4)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), k, 4)[:, :k]
    assert 7 * 6 * k < 2 ** 21 and 15 * 6 * n < 2 ** 22
    xg = x.to(DEV).requires_grad_(True)
    y = ops.mx_linear(xg, w)
    same(y.detach(), round_to(x.double() @ w64.t(), dtype))
    g = whole_numbers(m, n, 15, 3, dtype)
    y.backward(g.to(DEV))
    same(xg.grad, round_to(g.double() @ w64, dtype))


# the larger tiles, whole and in parts, each with ragged ends
LARGE = [(4100, 4099, 300), (2050, 1030, 2060), (1100, 1300, 2100), (1500, 2000, 600), (5001, 1537, 777),
         (65, 1368, 8241), (2712, 130, 11041), (2775, 1437, 8752), (140, 1129, 5803), (145, 364, 5490), (2003, 2500, 1030)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_products_of_whole_numbers(m, n, k, dtype):
    """partial sums are multiples of 2^-1 below 2^22: exact in 32 bits in any order, and in 64"""
    x = whole_numbers(m, k, 7, 1, dtype).to(DEV).requires_grad_(True)
    w = ops.mx_quantize(whole_numbers(n, k, 6, 2).to(DEV), 4)
    bias = whole_numbers(1, n, 99, 3, dtype)[0].to(DEV).requires_grad_(True)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), k, 4)[:, :k].to(DEV)
    assert 7 * 6 * k < 2 ** 21 and 15 * 6 * n < 2 ** 22
    y = ops.mx_linear(x, w, bias)
    same(y.detach(), round_to((x.detach().double() @ w64.t() + bias.detach().double()).cpu(), dtype))
    g = whole_numbers(m, n, 15, 4, dtype).to(DEV)
    y.backward(g)
    same(x.grad, round_to((g.double() @ w64).cpu(), dtype))


def test_offsets_beyond_32_bits():
    """a table of more than 2^32 bytes of codes, a result of more than 2^32 values, and an input of as many"""
    rows = 70_000_000
    table = ops.MXTensor(torch.zeros(rows, 64, dtype=torch.uint8, device=DEV),
                         torch.full((rows, 16), 127, dtype=torch.uint8, device=DEV), (rows, 100))
    table.data[-1, :50] = 0x42  # 1 and 2 in turn
    got = ops.mx_embedding(torch.tensor([0, rows - 1, rows], device=DEV), table)
    want = torch.zeros(3, 100)
    want[1] = torch.tensor([1.0, 2.0]).repeat(50)
    same(got, want)
    del table, got
    m, n = 33_001, 131_072
    x = torch.zeros(m, 32, dtype=torch.bfloat16, device=DEV)
    x[-1], x[0] = 2, 3
    w = ops.mx_quantize(torch.ones(n, 32, dtype=torch.bfloat16, device=DEV), 4)
    y = ops.mx_linear(x, w)
    assert y.numel() > 2 ** 32
    assert (y[-1] == 64).all() and (y[0] == 96).all() and not y[1:-1].any()
    q = ops.mx_quantize(y, 4)
    assert (q.data[-1] == 0x66).all() and (q.scales[-1] == 131).all() and not q.data[1:-1].any()  # 4 x 2^4
    dx = torch.autograd.grad(ops.mx_linear(x.requires_grad_(True), w), x, y)[0]
    assert (dx[-1] == 64 * n).all() and not dx[1:-1].any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n", [(1, 1), (2, 7), (31, 8), (33, 513), (64, 1024), (100, 3001), (1000, 40), (5000, 1),
                                 (8192, 1030), (40000, 9), (3, 40001)])
def test_bias_gradient_of_whole_numbers_is_exact(m, n, dtype):
    """numbers up to 30 in magnitude: 40000 of them stay below 2^24"""
    g = whole_numbers(m, n, 30, m + n, dtype)
    w = ops.mx_quantize(torch.zeros(n, 32, device=DEV), 4)
    bias = torch.zeros(n, dtype=dtype, device=DEV, requires_grad=True)
    y = ops.mx_linear(torch.zeros(m, 32, dtype=dtype, device=DEV), w, bias)
    y.backward(g.to(DEV))
    same(bias.grad, round_to(g.double().sum(0), dtype))
    wide = torch.full((m, n + 3), 7.0, dtype=dtype, device=DEV)  # rows that begin between vectors
    wide[:, 1:n + 1] = g.to(DEV)
    (gb,) = torch.autograd.grad(ops.mx_linear(torch.zeros(m, 32, dtype=dtype, device=DEV), w, bias), bias,
                                wide[:, 1:n + 1])
    same(gb, bias.grad)


def test_bias_gradient_of_no_rows_and_one_value():
    w = ops.mx_quantize(torch.zeros(70, 32, device=DEV), 4)
    bias = torch.full((70,), 3.0, device=DEV, requires_grad=True)
    ops.mx_linear(torch.zeros(0, 32, device=DEV), w, bias).sum().backward()
    same(bias.grad, torch.zeros(70))
    (gb,) = torch.autograd.grad(ops.mx_linear(torch.zeros(2, 50, 32, device=DEV), w, bias).sum(), bias)  # expanded
    same(gb, torch.full((70,), 100.0))


def test_gradient_strides_shapes_and_no_second_order():
    w = ops.mx_quantize(whole_numbers(24, 96, 6, 1).to(DEV), 4)
    w64 = decoded(w.data.cpu(), w.scales.cpu(), 96, 4)[:, :96]
    x = whole_numbers(6, 96, 7, 2).to(DEV).view(2, 3, 96).requires_grad_(True)
    ops.mx_linear(x, w).sum().backward()  # an expanded gradient
    same(x.grad, w64.sum(0).expand(2, 3, 96).float())
    g = whole_numbers(6, 50, 9, 4).to(DEV)
    (gx,) = torch.autograd.grad(ops.mx_linear(x, w), x, g[:, 7:31].view(2, 3, 24))
    same(gx.view(6, 96), (g[:, 7:31].cpu().double() @ w64).float())
    (gx,) = torch.autograd.grad(ops.mx_linear(x, w), x, torch.ones(2, 3, 24, device=DEV), create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


# -- lookup --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,count", [(1, 1, 1), (10, 31, 3), (100, 513, 77), (50, 1021, 200), (64, 4096, 1)])
def test_lookup_scales_and_rounds_once(rows, cols, count, dtype):
    table = rnd(rows, cols, seed=cols, dtype=torch.bfloat16)
    q = ops.mx_quantize(table.to(DEV), 4)
    ids = torch.randint(0, rows, (count,), generator=torch.Generator().manual_seed(1))
    for scale in (1.0, 0.1, math.sqrt(cols)):
        # a value has 2 bits, the scale 24: rounding their product to 24 bits first shows only next to ties
        want = held(table, 4)[ids] * torch.tensor(scale, dtype=torch.float32).double()
        same(ops.mx_embedding(ids.to(DEV), q, scale, dtype), round_to(want, dtype))
    same(ops.mx_embedding(ids.to(DEV).int().view(1, -1), q, 1.0, dtype), round_to(held(table, 4)[ids], dtype)[None])


def test_lookup_outside_the_table():
    q = ops.mx_quantize(rnd(10, 70).to(DEV), 4)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ids = torch.tensor([0, 9, 10, -1, 2 ** 62, 3, -2 ** 63], device=DEV)
    got = ops.mx_embedding(ids, q, 2.0, status=status)
    want = torch.zeros(7, 70, dtype=torch.bfloat16)
    full = (2 * held(rnd(10, 70), 4)).to(torch.bfloat16)
    want[0], want[1], want[5] = full[0], full[9], full[3]
    same(got, want)
    assert status.item() == 1
    status.zero_()
    ops.mx_embedding(ids[:2], q, status=status)
    assert status.item() == 0
    assert ops.mx_embedding(ids[:0], q).shape == (0, 70)
    none = ops.mx_quantize(torch.zeros(0, 70, device=DEV), 4)
    assert not ops.mx_embedding(ids, none, status=status).any() and status.item() == 1


# -- layers, streams, graphs -----------------------------------------------------------------

class Small(torch.nn.Module):
    def __init__(self, vocab=300, d=160, ffn=352):
        super().__init__()
        self.embed = torch.nn.Embedding(vocab, d)
        self.up = torch.nn.Linear(d, ffn)
        self.down = torch.nn.Linear(ffn, d, bias=False)
        self.lm_head = torch.nn.Linear(d, vocab, bias=False)

    def forward(self, ids):
        x = self.embed(ids)
        return self.lm_head(x + self.down(torch.nn.functional.silu(self.up(x))))


def test_layers_hold_compute_and_travel():
    torch.manual_seed(0)
    model = Small().to(torch.bfloat16)
    dense = {n: p.detach().clone() for n, p in model.named_parameters()}
    neuzip_amd.mx_convert(model)
    assert isinstance(model.up, neuzip_amd.nn.MXLinear) and isinstance(model.lm_head, torch.nn.Linear)
    assert isinstance(model.embed, torch.nn.Embedding) and repr(model.up).startswith("MXLinear(! in_features=160")
    model.embed = neuzip_amd.nn.MXEmbedding(model.embed, scale=3.0)
    model = model.to(DEV)
    ids = torch.randint(0, 300, (2, 9), device=DEV)
    x = model.embed(ids)
    same(x, round_to(held(dense["embed.weight"], 4)[ids.cpu()] * 3, torch.bfloat16))
    same(model.up.weight.dequantize(), held(dense["up.weight"], 4).to(torch.bfloat16))
    assert model.up.nbytes_compressed() == 352 * (128 + 16)  # 160 values: 256 codes, 16 scale bytes
    y = model.up(x).detach()
    same(y, ops.mx_linear(x, model.up.weight, model.up.bias).detach())
    same(model.embed.linear(x), ops.mx_linear(x, model.embed.weight))
    assert model.embed.linear(x).shape == (2, 9, 300)
    state = model.state_dict()
    assert {"up.weight_data", "up.weight_scales", "up.bias", "embed.weight_data"} <= set(state)
    torch.manual_seed(5)
    other = neuzip_amd.mx_convert(Small().to(torch.bfloat16))
    other.embed = neuzip_amd.nn.MXEmbedding(other.embed, scale=3.0)
    other = other.to(DEV)
    other.load_state_dict(state)
    same(other(ids).detach(), model(ids).detach())
    model.embed.check()
    model.embed(torch.tensor([300], device=DEV))
    with pytest.raises(RuntimeError, match="outside the table"):
        model.embed.check()
    model.embed.check()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert model.up(x.float()).dtype == torch.bfloat16
        assert model.embed.linear(x.float()).dtype == torch.bfloat16
    x8 = ops.mx_quantize(x, 8)
    z = model.up(x8)
    same(z, y)
    z.sum().backward()  # rows in 8 bits carry no gradient, the bias does
    same(model.up.bias.grad, torch.full((352,), 18.0))


def test_layers_that_stand_in_two_places_and_types_of_rows():
    shared = torch.nn.Linear(64, 64).to(torch.bfloat16)
    model = torch.nn.ModuleList([torch.nn.Sequential(shared, torch.nn.ReLU()), torch.nn.Sequential(shared)])
    neuzip_amd.mx_convert(model)
    assert isinstance(model[0][0], neuzip_amd.nn.MXLinear) and model[0][0] is model[1][0]
    table = neuzip_amd.nn.MXEmbedding(torch.nn.Embedding(9, 64).to(torch.bfloat16))
    ids = torch.arange(9, device=DEV)
    a = table(ids)
    b = table.half()(ids)
    assert a.dtype == torch.bfloat16 and b.dtype == torch.float16
    same(a, b)


def test_rows_of_one_quantisation_serve_several_weights():
    x = rnd(20, 256, dtype=torch.float16).to(DEV)
    x8 = ops.mx_quantize(x, 8)
    for n in (16, 100):
        w = ops.mx_quantize(rnd(n, 256, seed=n).to(DEV), 4)
        same(ops.mx_linear(x8, w, dtype=torch.float16), ops.mx_linear(x, w))


def guarded(rows, cols, dtype, past=5):
    """rows x cols that start one element behind a 16-byte boundary, and what stands round them"""
    whole = torch.full((rows * cols + 1 + past,), 9.0, dtype=dtype, device=DEV)
    return whole, whole[1:1 + rows * cols].view(rows, cols)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 33, 515), (3, 64, 512), (40, 96, 1025), (70, 128, 2048), (64, 4096, 2112),
                                   (2712, 130, 11041)])
def test_dense_pointers_need_their_elements_alignment_only(m, n, k, dtype):
    """the native calls, on memory that begins between vectors; nothing round the results is written"""
    L, code = _lib.load(), {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}.get(dtype, _lib.DTYPE_F32)
    stream = torch.cuda.current_stream().cuda_stream
    w = ops.mx_quantize(whole_numbers(n, k, 6, 2).to(DEV), 4)
    x, g, bias = (guarded(*size, dtype)[1] for size in ((m, k), (m, n), (1, n)))
    for t, most, seed in ((x, 7, 3), (g, 15, 4), (bias, 99, 5)):
        t.copy_(whole_numbers(*t.shape, most, seed, dtype))
    (y_all, y), (dx_all, dx) = guarded(m, n, dtype), guarded(m, k, dtype)

    room = torch.empty(max(16, L.nz_mx_linear_workspace_bytes(m, n, k, code)), dtype=torch.uint8, device=DEV)
    _lib.raise_for(L.nz_mx_linear(x.data_ptr(), code, m, k, k, w.data.data_ptr(), w.scales.data_ptr(), n,
                                  bias.data_ptr(), y.data_ptr(), room.data_ptr(), room.numel(), stream))
    same(y, ops.mx_linear(x.clone(), w, bias[0].clone()))

    need = L.nz_mx_linear_grad_workspace_bytes(g.data_ptr(), code, m, n, n, k)
    room = torch.empty(max(16, need), dtype=torch.uint8, device=DEV)
    _lib.raise_for(L.nz_mx_linear_grad(g.data_ptr(), code, m, n, n, w.data.data_ptr(), w.scales.data_ptr(), k,
                                       dx.data_ptr(), room.data_ptr(), room.numel(), stream))
    xg = x.clone().requires_grad_(True)
    ops.mx_linear(xg, w).backward(g.clone())
    same(dx, xg.grad)

    q_all, back = guarded(m, k, dtype)
    x4 = ops.mx_quantize(x, 4)
    _lib.raise_for(L.nz_mx_dequantize(x4.data.data_ptr(), x4.scales.data_ptr(), m, k, 4, back.data_ptr(), code, stream))
    same(back, x4.dequantize(dtype))
    for whole in (y_all, dx_all, q_all):
        assert whole[0] == 9 and (whole[-5:] == 9).all()


def test_calls_on_another_stream():
    w = ops.mx_quantize(rnd(512, 1024, seed=1).to(DEV), 4)
    x = rnd(100, 1024, dtype=torch.bfloat16).to(DEV)
    want = ops.mx_linear(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        y = x * 2
        a, b = ops.mx_linear(y, w), ops.mx_linear(x[:1], w)
    torch.cuda.current_stream().wait_stream(s)
    same(a, 2 * want.float())
    same(b, ops.mx_linear(x[:1], w))


def test_captured_calls_replay_beside_eager_ones():
    w = ops.mx_quantize(rnd(257, 640, seed=1).to(DEV), 4)
    table = ops.mx_quantize(rnd(100, 640, seed=2).to(DEV), 4)
    ids = torch.zeros(40, dtype=torch.int64, device=DEV)

    bias = torch.ones(w.shape[0], dtype=torch.bfloat16, device=DEV, requires_grad=True)

    def work():
        x = ops.mx_embedding(ids, table, 0.5)
        x.requires_grad_(True)
        y = ops.mx_linear(x, w)
        one = ops.mx_linear(x[:1].detach(), w)
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        z = ops.mx_linear(x.detach(), w, bias)
        (gb,) = torch.autograd.grad(z, bias, z.detach())
        return x.detach(), y.detach(), one, gx, gb

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = work()
        graphs.append((g, outs))
    for i in range(6):
        ids.copy_(torch.randint(0, 100, (40,), generator=torch.Generator().manual_seed(i)))
        g, outs = graphs[i % 2]
        g.replay()
        eager = work()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            same(a, b)


def test_float32_results_keep_what_is_small_beside_the_large():
    """x: multiples of 2^-2 up to 448, w: of 2^-1 up to 6, 64 of them: products are multiples of 2^-3 below 2^12,
    partial sums below 2^18, 21 bits: exact in 32 bits"""
    m, n, k = 5, 40, 64
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-15, 16, (m, k), generator=g).float() * torch.exp2(torch.randint(-2, 5, (m, k), generator=g).float())
    x[:, 3], x[:, 40] = 448.0, -448.0
    wd = whole_numbers(n, k, 6, 4)
    wd[:, 3] = wd[:, 40] = 6.0
    assert (held(x, 8) % 0.25 == 0).all() and (held(wd, 4) % 0.5 == 0).all()
    w = ops.mx_quantize(wd.to(DEV), 4)
    want = held(x, 8) @ held(wd, 4).t()
    same(ops.mx_linear(x.to(DEV), w), want)
    same(ops.mx_linear(ops.mx_quantize(x.to(DEV), 8), w, dtype=torch.float32), want)


def test_smallest_scales_of_a_weight():
    """blocks of subnormal weights: their scale is 2^-127"""
    wd = torch.arange(1, 7).repeat(64)[:64 * 5].float().view(5, 64) * 2.0 ** -127
    x = torch.full((2, 64), 2.0 ** 100)
    w = ops.mx_quantize(wd.to(DEV), 4)
    assert (w.scales[:, [0, 4]] == 0).all()
    want = held(x, 8) @ held(wd, 4).t()
    same(ops.mx_linear(x.to(DEV), w), want)
    same(ops.mx_linear(x.to(torch.bfloat16).to(DEV), w), round_to(want, torch.bfloat16))
    g = torch.full((3, 5), 2.0 ** 100, requires_grad=False)
    xg = torch.zeros(3, 64, device=DEV, requires_grad=True)
    ops.mx_linear(xg, w).backward(g.to(DEV))
    same(xg.grad, g.double() @ held(wd, 4))
