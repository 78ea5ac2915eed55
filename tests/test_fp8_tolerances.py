"""CPU: the tolerances of the activation functions in float32 are narrow enough to tell the float32 formulas from those
for results of 16 bits."""
import math

import pytest
import torch

from fp8_oracle import float32_tolerances, function


@pytest.mark.parametrize("kind,far", (("gelu", 12.5), ("silu", 80.0)))
def test_an_exponent_rounded_to_float32_is_out_of_tolerance(kind, far):
    x = torch.linspace(-far, 0, 4001, dtype=torch.float32).double()
    f, slope, f_tol, slope_tol = float32_tolerances(kind, x)
    u = function(kind, x)[2]
    binary = (u.float() * torch.tensor(math.log2(math.e))).double()  # the exponent to the base of 2, in float32
    lost = torch.expm1(u - binary * math.log(2))  # of the exponential, which below zero f has as a factor
    assert ((f * lost).abs() > f_tol).sum() > 100
    p = torch.where(x == 0, torch.full_like(x, 0.5), f / x)
    assert ((p * lost).abs() + ((slope - p) * lost).abs() > slope_tol).sum() > 100
