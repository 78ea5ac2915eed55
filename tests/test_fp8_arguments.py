"""CPU: what the operators on tensors in 8 bits refuse, at the C ABI (before any HIP call) and in Python; their oracle."""
import math

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import neuzip_amd
from neuzip_amd import _lib, ops
from neuzip_amd.ops import blocks8
from fp8_oracle import decoded, held, powers

L = _lib.load()
A, B, C, D = _lib.ERR_ARG, _lib.ERR_ALIGN, _lib.ERR_DTYPE, _lib.ERR_CAPACITY
P = 1 << 20  # an address that is never looked at


def refused(rc, code, text):
    assert rc == code
    assert text in _lib.last_error()


def test_sizes_of_the_stored_form():
    for cols, padded, scales in ((0, 0, 0), (1, 128, 4), (128, 128, 4), (129, 256, 4), (512, 512, 4), (513, 640, 8),
                                 (4096, 4096, 32)):
        assert L.nz_fp8_row_bytes(cols) == padded
        assert L.nz_fp8_scale_bytes(cols) == scales


def test_refusals_of_quantisation_and_values():
    q, v = L.nz_fp8_quantize, L.nz_fp8_dequantize
    refused(q(P, 0, 1, 1, 1, 2, P, P, None), A, "block_rows must be 1 or 128")
    refused(q(P, 3, 1, 1, 1, 1, P, P, None), C, "Unsupported data type")
    refused(q(P + 1, 0, 1, 1, 1, 1, P, P, None), B, "aligned to their elements")
    refused(q(P, 0, 1, 1, 1, 1, P + 8, P, None), B, "16-byte aligned")
    refused(q(P, 0, 1, 1, 1, 1, P, P + 4, None), B, "16-byte aligned")
    refused(q(None, 0, 1, 1, 1, 1, P, P, None), A, "null input")
    refused(q(P, 0, 1, 1, 1, 128, None, P, None), A, "null data")
    refused(q(P, 0, 1, 1 << 31, 1, 1, P, P, None), A, "2^30")
    refused(q(P, 0, 1 << 60, 512, 1, 128, P, P, None), A, "too many rows")
    assert q(None, 0, 0, 5, 1, 1, None, None, None) == _lib.OK
    assert q(None, 0, 5, 0, 1, 128, None, None, None) == _lib.OK
    refused(v(P, P, 1, 1, 1, None, 0, None), A, "null output")
    refused(v(P, None, 1, 1, 1, P, 0, None), A, "null data")
    refused(v(P, P, 1, 1, 7, P, 0, None), A, "block_rows")
    refused(v(P, P, 1, 1, 1, P + 2, 2, None), B, "aligned")
    refused(v(P, P, 1, 1 << 40, 1, P, 2, None), A, "2^30")
    assert v(None, None, 0, 5, 1, None, 0, None) == _lib.OK


def test_refusals_of_the_products():
    f, f8 = L.nz_fp8_linear, L.nz_fp8_linear_rows8
    refused(f(P, 0, 1, 0, 1, P, P, 1, 128, None, P, P, 1 << 30, None), A, "1 to 2^22")
    refused(f(P, 0, 1, 32, 32, P, P, 1, 64, None, P, P, 1 << 30, None), A, "block_rows")
    refused(f(P, 0, 1, 32, 32, None, P, 1, 128, None, P, P, 1 << 30, None), A, "null data")
    refused(f(P, 0, 1, 32, 32, P, P, 1, 128, None, None, P, 1 << 30, None), A, "null rows or output")
    refused(f(P, 0, 1, 32, 32, P, P, 1, 128, P + 1, P, P, 1 << 30, None), B, "aligned to their elements")
    refused(f(P, 0, 1 << 40, 32, 32, P, P, 1, 128, None, P, P, 1 << 30, None), A, "too many rows")
    refused(f(P, 0, 1 << 24, 32, 32, P, P, 1 << 21, 1, None, P, P, 1 << 62, None), A, "too many rows")
    need = L.nz_fp8_linear_workspace_bytes(1000, 512, 512, 0)
    assert need >= 1000 * 512
    refused(f(P, 0, 1000, 512, 512, P, P, 512, 1, None, P, P, need - 1, None), D, "workspace")
    refused(f(P, 0, 1000, 512, 512, P, P, 512, 1, None, P, P + 8, need, None), B, "workspace")
    assert f(None, 0, 0, 32, 32, None, None, 7, 1, None, None, None, 0, None) == _lib.OK
    refused(f8(P, P + 4, 1, 32, P, P, 1, 1, None, P, 0, None, 0, None), B, "16-byte aligned")
    refused(f8(P, P, 1000, 512, P, P, 512, 1, None, P, 0, P, 0, None), D, "workspace")
    refused(f8(P, P, 1, 512, P, P, 512, 1, None, None, 0, P, 0, None), A, "null output")
    g = L.nz_fp8_linear_grad
    refused(g(P, 9, 1, 1, 1, P, P, 1, 1, P, P, 1 << 30, None), C, "Unsupported data type")
    refused(g(None, 0, 1, 1, 1, P, P, 1, 1, P, P, 1 << 30, None), A, "null gradient")
    refused(g(P, 0, 1, 0, 1, P, P, 1, 1, P, P, 1 << 30, None), A, "without rows")
    refused(g(P, 0, 1, 1 << 22, 1 << 22, P, P, 1, 1, P, P, 1 << 30, None), A, "2^21")
    need = L.nz_fp8_linear_grad_workspace_bytes(P + 2, 0, 100, 512, 512, 512, 1)
    refused(g(P + 2, 0, 100, 512, 512, P, P, 512, 1, P, P, need - 1, None), D, "workspace")
    assert g(None, 0, 0, 1, 1, None, None, 1, 1, None, None, 0, None) == _lib.OK


def test_refusals_of_the_weight_gradient():
    g, room = L.nz_fp8_weight_grad, L.nz_fp8_weight_grad_workspace_bytes
    refused(g(P, 0, 1, 1, 1, P, P, 1, 1, 1, P, P, 1 << 30, None), A, "unknown flags")
    refused(g(P, 5, 1, 1, 1, P, P, 1, 1, 0, P, P, 1 << 30, None), C, "Unsupported data type")
    refused(g(P, 0, 0, 1, 1, P, P, 1, 1, 0, P, P, 1 << 30, None), A, "without rows")
    refused(g(P, 0, 1, 1, 1, P, P, 1, 3, 0, P, P, 1 << 30, None), A, "block_rows")
    refused(g(P, 0, 1, 1, 1, P, None, 1, 1, 0, P, P, 1 << 30, None), A, "null data")
    refused(g(P, 0, 1, 1, 1, P, P, 1, 1, 0, None, P, 1 << 30, None), A, "null gradient or output")
    refused(g(P, 0, 1 << 25, 8, 8, P, P, 1, 1, 0, P, P, 1 << 62, None), A, "too many rows")
    refused(g(P, 0, 8, 1 << 22, 1 << 22, P, P, 1, 1, 0, P, P, 1 << 62, None), A, "2^21")
    need = room(P, 1, 100, 512, 512, 512)
    assert need >= 2 * 2 * 100 * 512  # float16 as two bf16 numbers
    refused(g(P, 1, 100, 512, 512, P, P, 512, 1, 0, P, P, need - 1, None), D, "workspace")
    assert room(P, 0, 100, 520, 520, 512) < 100 * 512 * 2 < room(P, 0, 100, 521, 521, 512)
    assert g(None, 0, 5, 0, 1, None, None, 1, 1, 0, None, None, 0, None) == _lib.OK


def test_refusals_of_the_activation_functions():
    f, g = L.nz_fp8_activation, L.nz_fp8_activation_grad
    refused(f(3, P, 0, 1, 1, 1, None, 0, P, P, P, None, None, None), A, "unknown activation function")
    refused(f(-1, P, 0, 1, 1, 1, None, 0, P, P, P, None, None, None), A, "unknown activation function")
    refused(f(0, P, 4, 1, 1, 1, None, 0, P, P, P, None, None, None), C, "Unsupported data type")
    refused(f(0, P, 0, 1, 1, 1, None, 0, None, P, P, None, None, None), A, "null input or output")
    refused(f(0, P, 0, 1, 1, 1, None, 0, P, P, None, None, None, None), A, "null data")
    refused(f(0, P, 0, 1, 1, 1, P, 0, P, P, P, P, None, None), A, "null data")
    refused(f(0, P, 0, 1, 1, 1, P + 1, 0, P, P, P, P, P, None), B, "aligned")
    refused(f(0, P, 0, 1, 1 << 31, 1, None, 0, P, P, P, None, None, None), A, "2^30")
    assert f(0, None, 0, 0, 1, 1, None, 0, None, None, None, None, None, None) == _lib.OK
    refused(g(5, P, 0, 1, 1, 1, P, P, None, None, P, None, None), A, "unknown activation function")
    refused(g(0, P, 0, 1, 1, 1, P, P, None, None, None, None, None), A, "null gradient or output")
    refused(g(0, P, 0, 1, 1, 1, P, P, P, P, P, None, None), A, "null output")
    refused(g(0, P, 0, 1, 1, 1, P, P + 8, None, None, P, None, None), B, "16-byte aligned")
    assert g(0, None, 0, 5, 0, 1, None, None, None, None, None, None, None) == _lib.OK


def test_sizes_beyond_the_limits_have_an_answer():
    for huge in (1 << 24, 1 << 40, (1 << 63) + 5, (1 << 64) - 1):
        for m, n, k in ((huge, 5, 5), (5, huge, 5), (5, 5, huge), (huge, huge, huge)):
            L.nz_fp8_linear_workspace_bytes(m, n, k, 0), L.nz_fp8_linear_workspace_bytes(m, n, k, 2)
            L.nz_fp8_linear_grad_workspace_bytes(P, 0, m, n, n, k, 128)
            L.nz_fp8_weight_grad_workspace_bytes(P, 1, m, n, n, k)


def cpu_held(n=4, k=64, block_rows=128, shape=None):
    return ops.FP8Tensor(torch.zeros(n, L.nz_fp8_row_bytes(k), dtype=torch.uint8),
                         torch.zeros(-(-n // block_rows), L.nz_fp8_scale_bytes(k), dtype=torch.uint8), shape or (n, k),
                         block_rows)


def test_refusals_in_python():
    x, w = torch.zeros(2, 64), cpu_held()
    for call, error, text in (
            (lambda: ops.fp8_quantize(x), ValueError, "on the GPU"),
            (lambda: ops.fp8_quantize(x, 32), ValueError, "1 or 128"),
            (lambda: ops.fp8_quantize(x.double()), RuntimeError, "Unsupported data type"),
            (lambda: w.dequantize(), ValueError, "on the GPU"),
            (lambda: w.dequantize(torch.int32), RuntimeError, "Unsupported data type"),
            (lambda: ops.fp8_linear(x, torch.zeros(4, 64)), ValueError, "matrix in 8 bits"),
            (lambda: ops.fp8_linear(x, cpu_held(shape=(2, 2, 64))), ValueError, "matrix in 8 bits"),
            (lambda: ops.fp8_linear(x, cpu_held(k=96)), ValueError, "64 columns, the weight 96"),
            (lambda: ops.fp8_linear(x, w, torch.zeros(5)), ValueError, "bias must be"),
            (lambda: ops.fp8_linear(x, w, torch.zeros(4, dtype=torch.float16)), ValueError, "bias must be"),
            (lambda: ops.fp8_linear(x, w, dtype=torch.float16), ValueError, "type of x"),
            (lambda: ops.fp8_linear(w, w), ValueError, "a scale each"),
            (lambda: ops.fp8_linear(x, w), ValueError, "on the GPU"),
            (lambda: ops.fp8_linear(x.double(), w), RuntimeError, "Unsupported data type"),
            (lambda: ops.fp8_linear(x[0, 0], w), ValueError, "one dimension"),
            (lambda: ops.fp8_weight_gradient(x, x), ValueError, "held in 8 bits"),
            (lambda: ops.fp8_weight_gradient(x, w), ValueError, "dimensions of x"),
            (lambda: ops.fp8_weight_gradient(torch.zeros(4, 3).double(), w), RuntimeError, "Unsupported data type"),
            (lambda: ops.fp8_weight_gradient(torch.zeros(4, 3), w), ValueError, "on the GPU"),
            (lambda: ops.fp8_activation(x), ValueError, "on the GPU"),
            (lambda: ops.fp8_activation(x, "relu"), ValueError, "kind must be one of gelu"),
            (lambda: ops.fp8_activation(x, "silu", x[:1]), ValueError, "up must be"),
            (lambda: ops.fp8_activation(x, "silu", x.half()), ValueError, "up must be"),
            (lambda: ops.fp8_activation(x.double()), RuntimeError, "Unsupported data type"),
            (lambda: ops.fp8_activation(x[0, 0]), ValueError, "one dimension"),
            (lambda: ops.FP8Tensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), (4, 64)),
             ValueError, "shape"),
            (lambda: ops.FP8Tensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), (4, 64),
                                   128), ValueError, "shape"),
            (lambda: ops.FP8Tensor(torch.zeros(4, 128), torch.zeros(4, 4, dtype=torch.uint8), (4, 64)), ValueError,
             "shape"),
            (lambda: ops.FP8Tensor(w.data, w.scales, (4, 64), 16), ValueError, "1 or 128")):
        with pytest.raises(error, match=text):
            call()


def test_an_output_that_does_not_fit_is_refused(monkeypatch):
    monkeypatch.setattr(blocks8, "_on_gpu", lambda **tensors: 0)
    x, g = cpu_held(block_rows=1), torch.zeros(4, 3)
    for out in (torch.zeros(3, 63), torch.zeros(3, 64).half(), torch.zeros(64, 3).t(),
                torch.zeros(3, 64, dtype=torch.complex64).conj().imag.contiguous().view(64, 3)):
        with pytest.raises(ValueError, match="contiguous"):
            ops.fp8_weight_gradient(g, x, out=out)


W8, X8 = cpu_held(), cpu_held(n=2, block_rows=1)
X, G = torch.zeros(2, 64), torch.zeros(2, 4)
CALLS = [("quantize", lambda t: ops.fp8_quantize(t).data, X), ("linear", lambda t: ops.fp8_linear(t, W8), X),
         ("bias", lambda t: ops.fp8_linear(X, W8, t), G[0]),
         ("input gradient", lambda t: blocks8._input_gradient(t, W8), G),
         ("weight gradient", lambda t: ops.fp8_weight_gradient(t, X8), G),
         ("activation", lambda t: ops.fp8_activation(t), X), ("gate", lambda t: ops.fp8_activation(X, "silu", t), X)]


@pytest.mark.parametrize("call,t", [c[1:] for c in CALLS], ids=[c[0] for c in CALLS])
def test_traces_and_forward_mode_are_refused(call, t):
    for trace in (lambda: torch.jit.trace(call, t), lambda: make_fx(call)(t)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace()
    forward = torch.autograd.forward_ad
    with forward.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward.make_dual(t, torch.ones_like(t)))
    with pytest.raises(ValueError, match="on the GPU"):
        call(t)


@pytest.fixture
def without_gpu(monkeypatch):
    """the Python side alone: native calls are left out, sizes are asked for"""
    from neuzip_amd.ops import microscaled
    for module in (microscaled, blocks8):
        monkeypatch.setattr(module, "_on_gpu", lambda **tensors: 0)
        monkeypatch.setattr(module, "_call", lambda *args: None)
        monkeypatch.setattr(module, "_ask", lambda fn, index, *args: 0)


@pytest.mark.parametrize("part", ("data", "scales"))
def test_a_weight_that_is_changed_before_the_backward(without_gpu, part):
    w = cpu_held()
    x, bias = torch.zeros(2, 64, requires_grad=True), torch.zeros(4, requires_grad=True)
    y = ops.fp8_linear(x, w, bias)
    getattr(w, part).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = ops.fp8_linear(x.detach(), w, bias)  # the gradient of the bias does not use the weight
    getattr(w, part).zero_()
    y.sum().backward()
    assert bias.grad is not None


def test_inference_tensors_and_hooks_of_saved_tensors(without_gpu):
    with torch.inference_mode():
        w = cpu_held()
    x, up = torch.zeros(2, 64, requires_grad=True), torch.zeros(2, 64, requires_grad=True)
    ops.fp8_linear(x, w).sum().backward()
    assert x.grad.shape == x.shape
    w, seen = cpu_held(), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: (seen.append(t.shape), t)[1]):
        y = ops.fp8_linear(x, w)
        z = ops.fp8_activation(x, "silu", up)
    w.data.fill_(1)  # the hook keeps another tensor
    y.sum().backward()
    assert seen == [w.data.shape, w.scales.shape]
    z.sum().backward()
    assert len(seen) == 3 and up.grad.shape == up.shape


def test_writes_into_a_given_gradient_are_seen(without_gpu):
    out, p = torch.zeros(4, 64), torch.ones(4, 64, requires_grad=True)
    y = out * p
    ops.fp8_weight_gradient(G, X8, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_what_an_activation_function_keeps(without_gpu):
    """codes and scales, 129/128 bytes a value where the widths are whole groups, and nothing where nothing is recorded"""
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        x = torch.zeros(3, 512, dtype=torch.bfloat16)
        ops.fp8_activation(x)
        assert not kept
        ops.fp8_activation(x.requires_grad_(True))
        assert sum(t.numel() * t.element_size() for t in kept) == 3 * (512 + 4)
        ops.fp8_activation(x, "silu", x.detach())
        assert sum(t.numel() * t.element_size() for t in kept[1:]) == 2 * 3 * (512 + 4) + 4  # scales begin at 16 bytes


def test_the_oracle_itself():
    """hand-made bytes against the statement of the format, and the rule of the scale at its borders"""
    data = torch.zeros(1, 256, dtype=torch.uint8)
    data[0, 0], data[0, 1], data[0, 130] = 0x38, 0xB9, 0x01  # 1, -1.125, 2^-9
    scales = torch.tensor([[128, 126, 0, 0]], dtype=torch.uint8)
    v = decoded(data, scales)
    assert v[0, 0] == 2.0 and v[0, 1] == -2.25 and v[0, 130] == 2.0 ** -10 and v.abs().sum() == 4.25 + 2.0 ** -10
    for largest, power in ((448.0, 0), (448.0 + 2 ** -15, 1), (449.0, 1), (256.0, 0), (224.0, -1), (225.0, 0), (1.75, -8),
                           (0.0, -127), (1e-45, -127), (2.0 ** -119, -127), (3.4e38, 120), (3.3895e38, 120)):
        assert powers(torch.full((1, 1, 1, 1), largest, dtype=torch.float64)).item() == power, largest
    x = torch.zeros(130, 130)
    x[0, 0], x[1, 1], x[129, 129], x[128, 0] = 448.0, 1.0625, math.inf, 18.0
    h = held(x, 128)
    assert h[0, 0] == 448 and h[1, 1] == 1.0 and h[128, 0] == 18.0 and torch.isnan(h[128:, 128:]).all()
    assert not torch.isnan(h[:128]).any() and not torch.isnan(h[:, :128]).any()
    assert held(torch.tensor([[17.0, 256.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]])).tolist() == [
        [16.0, 256.0, 20.0, 0.0, 2.0 ** -8]]
    assert held(torch.tensor([[1.5 * 2.0 ** -137]])).item() == 2.0 ** -136  # steps of 2^-9 at the least scale, 2^-127


def test_layers_in_python():
    assert neuzip_amd.nn.FP8Activation("silu").kind == "silu"
    with pytest.raises(ValueError, match="kind must be one of"):
        neuzip_amd.nn.FP8Activation("relu")
