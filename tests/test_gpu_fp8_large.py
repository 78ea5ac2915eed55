"""GPU: tensors in 8 bits whose elements, codes or rows are counted beyond 32 bits, and calls of more rows than one launch
takes.  Rows repeat themselves, so that a wrong offset shows anywhere; whole numbers, so that results are exact."""
import pytest
import torch

from neuzip_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
PERIOD = 1000
MANY = 67108860 + 1300  # rows of up to 512 values: one launch takes 2^26 - 4


def room(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GiB of the GPU's memory")


def repeated(rows, cols, seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randint(-7, 8, (PERIOD, cols), generator=g, device=DEV).to(dtype)
    return x.repeat(-(-rows // PERIOD), 1)[:rows]


def repeats(t, want):
    """``t`` is ``want`` (its first PERIOD rows) over and over"""
    assert torch.equal(t[:PERIOD], want)
    for at in range(PERIOD, t.shape[0], PERIOD * 20):
        part = t[at:at + PERIOD * 20]
        assert torch.equal(part, t[at - PERIOD:at - PERIOD + part.shape[0]]), at


@pytest.mark.parametrize("block_rows", (1, 128))
def test_more_rows_than_a_launch_takes(block_rows):
    room(40)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-7, 8, (128, 1), generator=g, device=DEV).to(torch.bfloat16).repeat(-(-MANY // 128), 1)[:MANY]
    x[::128] = 7  # every block of either kind holds its values as they are
    q = ops.fp8_quantize(x, block_rows)
    assert q.data.numel() > 2 ** 32
    assert torch.equal(q.dequantize(), x)
    if block_rows == 1:
        assert torch.equal(q.data[-1300:], ops.fp8_quantize(x[-1300:]).data)
        assert torch.equal(q.scales[-1300:], ops.fp8_quantize(x[-1300:]).scales)


def test_activation_functions_of_more_rows_than_a_launch_takes():
    room(60)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randint(-7, 8, (MANY, 1), generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    up = torch.randint(-7, 8, (MANY, 1), generator=g, device=DEV).to(torch.bfloat16)
    y = ops.fp8_activation(x, "silu", up)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for at in (slice(0, 4096), slice(MANY - 4096, MANY), slice(67108860 - 50, 67108860 + 50)):
        part = x.detach()[at].clone().requires_grad_(True)
        z = ops.fp8_activation(part, "silu", up[at])
        assert torch.equal(y.detach()[at], z.detach())
        assert torch.equal(dx[at], torch.autograd.grad(z, part, torch.ones_like(z))[0])


@pytest.mark.parametrize("k", (100, 512))
def test_products_of_more_than_2_to_the_32_values(k):
    room(40)
    m, n = 70000, 65536
    x, wd = repeated(m, k, 1), repeated(n, k, 2, torch.float32)
    y = ops.fp8_linear(x, ops.fp8_quantize(wd, 128))
    assert y.numel() > 2 ** 32
    repeats(y, (x[:PERIOD].double() @ wd.double().t()).to(torch.float32).to(torch.bfloat16))


@pytest.mark.parametrize("block_rows", (1, 128))
def test_gradients_of_rows_of_more_than_2_to_the_32_values(block_rows):
    room(60)
    m, n, k = 70000, 70, 65536
    g, wd = repeated(m, n, 1), repeated(n, k, 2, torch.float32)
    x = torch.zeros(1, k, dtype=torch.bfloat16, device=DEV).expand(m, k).requires_grad_(True)
    y = ops.fp8_linear(x, ops.fp8_quantize(wd, block_rows))
    (dx,) = torch.autograd.grad(y, x, g)
    assert dx.numel() > 2 ** 32
    repeats(dx, (g[:PERIOD].double() @ wd.double()).to(torch.float32).to(torch.bfloat16))


def test_gradients_of_weights_of_more_than_2_to_the_32_values():
    room(40)
    m, n, k = 70, 70000, 65536
    g, xd = repeated(n, m, 1).t().contiguous(), repeated(m, k, 2, torch.float32)
    x8 = ops.fp8_quantize(xd)
    dw = ops.fp8_weight_gradient(g, x8)
    want = (g[:, :PERIOD].double().t() @ xd.double()).to(torch.float32)
    repeats(dw, want.to(torch.bfloat16))
    dw.fill_(3.0)
    ops.fp8_weight_gradient(g, x8, out=dw)
    repeats(dw, (want + 3).to(torch.bfloat16))


def test_a_kept_input_of_more_than_2_to_the_32_codes():
    """the rows that are summed over lie beyond 32 bits: a weight's gradient is the sum of its parts"""
    room(60)
    m, n, k = 1100000, 40, 4096
    g, x = repeated(m, n, 1), repeated(m, k, 2)
    x8 = ops.fp8_quantize(x)
    assert x8.data.numel() > 2 ** 32
    got = ops.fp8_weight_gradient(g.float(), x8)
    # 1100 periods: whole numbers below 2^24 each, so the sum may round on its way: 32 bits, m additions
    once = g[:PERIOD].double().t() @ x[:PERIOD].double()
    size = g[:PERIOD].double().abs().t() @ x[:PERIOD].double().abs()
    assert ((got.double() - 1100 * once).abs() <= m * 2.0 ** -23 * 1100 * size).all()
    tail = ops.fp8_weight_gradient(g[-2 * PERIOD:].float(), ops.fp8_quantize(x[-2 * PERIOD:]))
    assert torch.equal(tail.double(), 2 * once)
    only = torch.zeros_like(g)
    only[-PERIOD:] = g[-PERIOD:]  # the last rows alone, from their places among all
    assert torch.equal(ops.fp8_weight_gradient(only.float(), x8).double(), once)
