"""GPU: places that hold the lowest value of bfloat16 or float32, as masks do.  8 bits hold it as 2^128, which no 32 bits
do: sums with it stay sums of finite numbers, and where it meets a zero it counts for nothing."""
import pytest
import torch

from neuzip_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES, IDS = (torch.bfloat16, torch.float32), ("bf16", "fp32")
KINDS = ("gelu", "gelu_tanh", "silu")


def whole(rows, cols, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-7, 8, (rows, cols), generator=g, device=DEV, dtype=torch.float32)


def test_what_is_held():
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        x = torch.tensor([[low, -low, 0.0, 3.2e38]], device=DEV).to(dtype)
        got = ops.fp8_quantize(x).dequantize(torch.float32)[0].double()
        assert got.tolist() == [-float("inf"), float("inf"), 0.0, 240 * 2.0 ** 120]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
def test_slopes_and_gradients_of_masked_places(kind, dtype):
    """the slope is 0 below and 1 above, f(lowest) is 0; the slope at 0, a half, is off by 10 * 2^-23 at most
    (fp8_oracle.float32_tolerances) or, in 16 bits, twice that"""
    low = torch.finfo(dtype).min
    x = torch.zeros(6, 200, dtype=dtype, device=DEV)
    x[0], x[1, ::2], x[3, 150], x[4] = low, low, low, -low
    a = x.clone().requires_grad_(True)
    y = ops.fp8_activation(a, kind)
    g = torch.full_like(y, 0.25)
    (da,) = torch.autograd.grad(y, a, g)
    want = torch.where(x == low, 0.0, torch.where(x == -low, 0.25, 0.125)).to(dtype)
    far, near = x != 0, 20 * 2.0 ** -23 + torch.finfo(dtype).eps
    assert torch.equal(da[far], want[far]) and ((da - want).abs() <= near * want.abs()).all()
    assert not y.detach()[x == low].any()
    up = whole(6, 200, 1).to(dtype)
    b = up.clone().requires_grad_(True)
    da, db = torch.autograd.grad(ops.fp8_activation(a, kind, b), (a, b), g)
    want = torch.where(x == low, 0.0, want.float() * up.float()).to(dtype)
    assert torch.equal(da[far], want[far]) and ((da - want).abs() <= near * want.abs()).all()
    assert not db[:4].any() and not db[5].any()
    assert ((db[4].double() / (0.25 * 2.0 ** 128) - 1).abs() <= 2.0 ** -8).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(70, 48, 140), (1000, 1100, 700)])
def test_masked_rows_add_nothing_to_a_weights_gradient(m, n, k, dtype):
    x, g = whole(m, k, 1), whole(m, n, 2)
    hidden = torch.arange(m, device=DEV) % 7 == 3
    g[hidden] = 0
    x[hidden, ::3] = torch.finfo(torch.float32).min
    x = x.to(dtype)  # (in bfloat16 the lowest of float32 would be an infinity)
    x[hidden, ::3] = torch.finfo(dtype).min
    got = ops.fp8_weight_gradient(g.to(dtype), ops.fp8_quantize(x))
    x[hidden] = 0
    want = ops.fp8_weight_gradient(g.to(dtype), ops.fp8_quantize(x))
    assert torch.isfinite(got).all() and torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("m,n,k", [(1, 40, 300), (9, 40, 300), (16, 40, 3000), (70, 48, 640), (600, 520, 1024)])
def test_products_with_masked_places(m, n, k, dtype):
    """zeros of the weight stand against them in some columns of the result, an eighth in the others"""
    x, w = torch.zeros(m, k, dtype=dtype, device=DEV), whole(n, k, 1)
    x[0, 0] = x[m - 1, k - 1] = torch.finfo(dtype).min
    x[m // 2, 140] = 5
    w[:, 0] = w[:, k - 1] = 0
    w[::2, 0] = w[::2, k - 1] = 0.125
    # the rest of the weight counts for nothing beside the lowest value, and is exact where there is none
    rest = x.clone()
    rest[rest == torch.finfo(dtype).min] = 0
    want = rest.double() @ w.double().t()
    masked = (x == torch.finfo(dtype).min).any(1)
    held = ops.fp8_quantize(x)
    for weight in (ops.fp8_quantize(w, 1), ops.fp8_quantize(w, 128)):
        for got in (ops.fp8_linear(x, weight), ops.fp8_linear(held, weight, dtype=dtype)):
            got = got.double()
            assert torch.equal(got[~masked], want[~masked].to(dtype).double())
            assert torch.equal(got[:, 1::2], want[:, 1::2].to(dtype).double())
            times = (x == torch.finfo(dtype).min).sum(1).double()[masked][:, None] * 0.125
            assert ((got[masked][:, ::2] / (-(2.0 ** 128) * times) - 1).abs() <= 2.0 ** -8).all()
