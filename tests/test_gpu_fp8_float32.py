"""GPU: the activation functions on float32 values, which have formulas of their own, within the roundings that these
make (derived at ``fp8_oracle.float32_tolerances``; formulas for 16 bits are outside of them)."""
import pytest
import torch

from neuzip_amd import ops
from fp8_oracle import float32_tolerances, held

pytestmark = pytest.mark.gpu

DEV = "cuda"
FAR = {"gelu": (-12.5, 9.0), "gelu_tanh": (-9.9, 9.0), "silu": (-80.0, 40.0)}


def rnd(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("gated", (False, True))
@pytest.mark.parametrize("kind", FAR)
def test_float32_results_and_gradients(kind, gated):
    """Exponentials down to 2^-123 and 1 - tail above zero: values from one end to the other, in another order in every
    row, so that 8 bits hold many of them"""
    rows, cols = 40, 1021
    line = torch.linspace(*FAR[kind], rows * cols)[torch.randperm(rows * cols, generator=torch.Generator().manual_seed(1))]
    x = line.view(rows, cols) * torch.exp2(-(torch.arange(rows) % 4.0))[:, None]
    up, g = rnd(rows, cols, seed=2) if gated else None, rnd(rows, cols, seed=3)
    a = x.to(DEV).requires_grad_(True)
    b = up.to(DEV).requires_grad_(True) if gated else None
    y = ops.fp8_activation(a, kind, b)
    got = torch.autograd.grad(y, (a, b) if gated else (a,), g.to(DEV))
    u64, u8 = (up.double(), held(up)) if gated else (1.0, 1.0)
    f, _, tol, _ = float32_tolerances(kind, x.double())
    f8, slope, f8_tol, slope_tol = float32_tolerances(kind, held(x))
    g64 = g.double()

    def near(got, want, tol):
        # a product more, with another factor each, and its rounding; a subnormal product
        left = (got.detach().cpu().double() - want).abs() - (tol * (1 + 2.0 ** -20) + 2.0 ** -23 * want.abs() + 2.0 ** -149)
        assert left.max() <= 0, left.max()

    near(y, f * u64, tol * abs(u64))
    near(got[0], g64 * u8 * slope, slope_tol * (g64 * u8).abs())
    if gated:
        near(got[1], g64 * f8, f8_tol * g64.abs())


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=("bf16", "fp32"))
@pytest.mark.parametrize("kind", FAR)
def test_factors_whose_product_would_overflow(kind, dtype):
    """The slope is zero far below, however large g up is; and a small g stands beside a slope above 1 and a large factor"""
    big = 3e38
    x = torch.tensor([-1e4, 2.25, -1e4, 2.25], dtype=dtype)[:, None].expand(4, 128).contiguous()
    up = torch.tensor([-big, -big, big, big], dtype=dtype)[:, None].expand(4, 128).contiguous()
    g = torch.tensor([4.0, 0.125, -1000.0, 0.5], dtype=dtype)[:, None].expand(4, 128).contiguous()
    a, b = x.to(DEV).requires_grad_(True), up.to(DEV).requires_grad_(True)
    y = ops.fp8_activation(a, kind, b)
    da, db = (t.cpu().double() for t in torch.autograd.grad(y, (a, b), g.to(DEV)))
    assert (da[[0, 2]] == 0).all() and (db[[0, 2]] == 0).all() and (y.detach()[[0, 2]] == 0).all()
    _, slope, _, tol = float32_tolerances(kind, torch.tensor(2.25, dtype=torch.float64))
    assert slope > 1
    want = g[[1, 3]].double() * held(up[[1, 3]]) * slope
    half = torch.finfo(dtype).eps / 2
    # 16-bit formulas are off by up to 2^-19 more (their exponent's rounding is below 2^-22 of it here)
    assert ((da[[1, 3]] - want).abs() <= (half + tol / slope + 2.0 ** -19) * want.abs()).all()
