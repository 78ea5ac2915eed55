"""Calls that go through other transforms of torch: the operators write through addresses, which a trace does not
see and a tangent does not follow.  Such calls are refused, before they look for a GPU; compiled functions work."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from neuzip_amd import _lib, ops

L = _lib.load()
W = ops.MXTensor(torch.zeros(4, L.nz_mx_row_bytes(64, 4), dtype=torch.uint8),
                 torch.zeros(4, L.nz_mx_scale_bytes(64), dtype=torch.uint8), (4, 64), 4)
X, G, IDS = torch.zeros(2, 64), torch.zeros(2, 4), torch.zeros(2, dtype=torch.int64)
FLOATING = [("quantize", lambda t: ops.mx_quantize(t).data, X), ("linear", lambda t: ops.mx_linear(t, W), X),
            ("bias", lambda t: ops.mx_linear(X, W, t), G[0]),
            ("table gradient", lambda t: ops.embedding_gradient(IDS, t, 7), G),
            ("input gradient", lambda t: ops.microscaled._input_gradient(t, W), G),
            ("bias gradient", lambda t: ops.microscaled._bias_gradient(t, 4), G)]
CALLS = FLOATING + [("lookup", lambda t: ops.mx_embedding(t, W), IDS), ("values", lambda t: W.dequantize() + t, X)]


@pytest.mark.parametrize("call,t", [c[1:] for c in CALLS], ids=[c[0] for c in CALLS])
def test_traces_are_refused(call, t):
    for trace in (lambda: torch.jit.trace(call, t), lambda: make_fx(call)(t)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            trace()
    with pytest.raises(ValueError, match="on the GPU"):
        call(t)


@pytest.mark.parametrize("call,t", [c[1:] for c in FLOATING], ids=[c[0] for c in FLOATING])
def test_forward_mode_differentiation_is_refused(call, t):
    forward = torch.autograd.forward_ad
    with forward.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(forward.make_dual(t, torch.ones_like(t)))
        with pytest.raises(ValueError, match="on the GPU"):
            call(t)  # without a tangent there is none to lose


def test_rows_whose_sign_is_held_back():
    """imag of a conjugate: its memory holds the values with the other sign"""
    z = torch.arange(12.0).view(4, 3).to(torch.complex64) * 1j
    for t in (z.conj().imag, z[:, :1].conj().imag, z[1:2, :1].conj().imag):
        assert t.is_neg()
        rows, n, _ = ops.microscaled._as_rows(t, t.shape[1])
        assert not rows.is_neg() and torch.equal(rows, t) and n == t.shape[0]


@pytest.mark.gpu
def test_a_bias_and_an_output_whose_sign_is_held_back():
    bias = torch.tensor([1j], device="cuda").conj().imag
    w = ops.mx_quantize(torch.zeros(1, 64, device="cuda"), 4)
    assert ops.mx_linear(torch.zeros(1, 64, device="cuda"), w, bias).item() == -1
    with pytest.raises(ValueError, match="contiguous"):
        ops.embedding_gradient(IDS.cuda(), torch.zeros(2, 1, device="cuda"), 1, out=bias.view(1, 1))


@pytest.mark.gpu
def test_compiled_functions_make_the_calls():
    w = ops.mx_quantize(torch.randn(40, 64, device="cuda"), 4)
    x, ids = torch.randn(5, 64, device="cuda"), torch.tensor([3, 0], device="cuda")

    def work(x, ids):
        return ops.mx_linear(x * 2, w) + 1, ops.mx_embedding(ids, w), ops.embedding_gradient(ids, x[:2], 7)

    compiled = torch.compile(work, backend="eager")
    for scale in (1.0, 3.0):
        for a, b in zip(compiled(x * scale, ids), work(x * scale, ids)):
            assert torch.equal(a, b)
