"""What autograd keeps of the operators' tensors: a weight, or a tensor that gradients are added to, that is changed
between a forward pass and its backward is an error, as for torch's own layers."""
import pytest
import torch

import neuzip_amd
from neuzip_amd import _lib, ops
from neuzip_amd.ops import embedding, microscaled

L = _lib.load()


def cpu_weight(n=4, k=64):
    return ops.MXTensor(torch.zeros(n, L.nz_mx_row_bytes(k, 4), dtype=torch.uint8),
                        torch.zeros(n, L.nz_mx_scale_bytes(k), dtype=torch.uint8), (n, k), 4)


@pytest.fixture
def without_gpu(monkeypatch):
    """the Python side alone: native calls are left out, sizes are asked for"""
    for module in (microscaled, embedding):
        monkeypatch.setattr(module, "_on_gpu", lambda **tensors: 0)
        monkeypatch.setattr(module, "_call", lambda *args: None)
    monkeypatch.setattr(microscaled, "_ask", lambda fn, index, *args: 0)


@pytest.mark.parametrize("part", ("data", "scales"))
def test_a_weight_that_is_changed_before_the_backward(without_gpu, part):
    w = cpu_weight()
    x, bias = torch.zeros(2, 64, requires_grad=True), torch.zeros(4, requires_grad=True)
    y = ops.mx_linear(x, w, bias)
    getattr(w, part).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = ops.mx_linear(x.detach(), w, bias)  # the gradient of the bias does not use the weight
    getattr(w, part).zero_()
    y.sum().backward()
    assert bias.grad is not None


def test_a_weight_made_in_inference_mode_serves_a_training_step(without_gpu):
    with torch.inference_mode():
        w = cpu_weight()
    x = torch.zeros(2, 64, requires_grad=True)
    ops.mx_linear(x, w).sum().backward()
    assert x.grad.shape == x.shape


def test_weights_travel_through_the_hooks_of_saved_tensors(without_gpu):
    w, seen = cpu_weight(), []
    x = torch.zeros(2, 64, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: (seen.append(t.shape), t)[1]):
        y = ops.mx_linear(x, w)
    w.data.fill_(1)  # the hook keeps another tensor
    y.sum().backward()
    assert seen == [w.data.shape, w.scales.shape]


def test_writes_into_given_tensors_are_seen(without_gpu):
    ids = torch.zeros(2, dtype=torch.int64)
    out, p = torch.zeros(7, 4), torch.ones(7, 4, requires_grad=True)
    y = out * p
    ops.embedding_gradient(ids, torch.zeros(2, 4), 7, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    status = torch.zeros(1, dtype=torch.int32)
    before = status._version
    ops.mx_embedding(ids, cpu_weight(), status=status)
    assert status._version > before
    with torch.inference_mode():  # tensors without a version
        out = torch.zeros(7, 4)
        ops.embedding_gradient(ids, torch.zeros(2, 4), 7, out=out)


@pytest.mark.gpu
def test_a_layer_that_is_loaded_before_the_backward():
    a = neuzip_amd.nn.MXLinear(torch.nn.Linear(64, 32, device="cuda"))
    b = neuzip_amd.nn.MXLinear(torch.nn.Linear(64, 32, device="cuda"))
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    y = a(x)
    y.sum().backward()
    want = torch.ones(3, 32, device="cuda") @ a.weight.dequantize(torch.float32)
    assert torch.allclose(x.grad, want, rtol=1e-5, atol=1e-5)
    y = a(x)
    a.load_state_dict(b.state_dict())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
