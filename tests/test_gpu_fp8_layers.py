"""GPU: layers that hold weights or inputs in 8 bits, and the operators under streams and captured graphs."""
import pytest
import torch

import neuzip_amd
from neuzip_amd import nn, ops
from fp8_oracle import held
from mx_oracle import HALF_STEP

pytestmark = pytest.mark.gpu

DEV = "cuda"


def rnd(*shape, seed=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def pair(bits, rows=96, cols=200, bias=True):
    """a compressed layer (lossless) that keeps its input in ``bits``, and its dense weight"""
    manager = neuzip_amd.Manager(precision=7)
    dense = torch.nn.Linear(cols, rows, bias=bias).to(torch.bfloat16).to(DEV)
    weight = dense.weight.data.clone()
    layer = nn.Linear(manager, dense)
    layer.saved_bits = bits
    return layer, weight


def test_a_compressed_layer_that_keeps_8_bits():
    """result and the gradients of input and bias as with 16 bits kept; the weight's gradient is that of the kept values"""
    layer, weight = pair(8)
    x, g = rnd(4, 10, 200).requires_grad_(True), rnd(4, 10, 96, seed=1, scale=1e-2)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (kept.append(t), t)[1], lambda t: t):
        y = layer(x)
    assert sum(t.numel() * t.element_size() for t in kept) == 40 * (256 + 4)
    y.backward(g)
    got = layer.weight._gradient
    layer.weight._gradient = None
    gx, gb, x.grad, layer.bias.grad = x.grad, layer.bias.grad, None, None
    layer.saved_bits = 16
    z = layer(x)
    z.backward(g)
    assert torch.equal(y, z) and torch.equal(gx, x.grad) and torch.equal(gb, layer.bias.grad)
    x8, g64 = held(x.detach().cpu().view(40, 200)), g.cpu().double().view(40, 96)
    want, size = g64.t() @ x8, g64.t().abs() @ x8.abs()
    assert ((got.cpu().double() - want).abs() <= HALF_STEP[torch.bfloat16] * want.abs() + 40 * 2.0 ** -23 * size).all()
    assert got.dtype == torch.bfloat16 and got.shape == (96, 200)


def test_gradients_add_up_and_reach_the_update_hook():
    layer, weight = pair(8, bias=False)
    x, g = rnd(50, 200), rnd(50, 96, seed=1, scale=1e-2)
    layer(x.clone().requires_grad_(True)).backward(g)
    once = layer.weight._gradient.clone()
    layer(x.clone().requires_grad_(True)).backward(g)
    twice = layer.weight._gradient
    want = ops.fp8_weight_gradient(g, ops.fp8_quantize(x), out=once.clone())
    assert torch.equal(twice, want) and not torch.equal(twice, once)
    layer.weight._gradient = None
    layer.weight._gradient = torch.zeros(96, 200, device=DEV)  # another type: added to as it is
    layer(x.clone().requires_grad_(True)).backward(g)
    assert torch.equal(layer.weight._gradient, once.float())
    layer.weight._gradient = None
    sgd = torch.optim.SGD([torch.nn.Parameter(torch.zeros(1))], lr=0.5)
    scheduler = torch.optim.lr_scheduler.LambdaLR(sgd, lambda step: 1.0)
    layer.weight.register_post_accumulate_grad_hook(lambda p: neuzip_amd.compressed_lomo_hook(scheduler, p))
    layer(x.clone().requires_grad_(True)).backward(g)
    assert layer.weight._gradient is None and torch.equal(layer.weight(), weight.add(once, alpha=-0.5))


def test_autocast_and_inputs_without_a_gradient():
    layer, _ = pair(8)
    x, g = rnd(5, 200, dtype=torch.float32), rnd(5, 96, seed=1)
    with torch.autocast("cuda", torch.bfloat16):
        y = layer(x)  # no gradient for x: the weight's is made all the same
    y.backward(g)
    assert torch.equal(layer.weight._gradient, ops.fp8_weight_gradient(g, ops.fp8_quantize(x.bfloat16())))
    with torch.no_grad():
        assert not layer(x.bfloat16()).requires_grad


def test_one_row_no_rows_and_a_second_derivative():
    layer, _ = pair(8)
    x, g = rnd(200), rnd(96, seed=1)
    layer(x.clone().requires_grad_(True)).backward(g)
    want = ops.fp8_weight_gradient(g[None], ops.fp8_quantize(x[None]))
    assert torch.equal(layer.weight._gradient, want)
    layer.weight._gradient = None
    a = rnd(0, 200).requires_grad_(True)
    layer(a).sum().backward()
    assert a.grad.shape == (0, 200) and not layer.weight._gradient.any()
    a = rnd(3, 200).requires_grad_(True)
    w = ops.fp8_quantize(rnd(96, 200, seed=2), 128)
    for f in (layer, ops.fp8_activation, lambda t: ops.fp8_linear(t, w)):
        (d,) = torch.autograd.grad(f(a).float().pow(2).sum(), a, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.sum().backward()


class Block(torch.nn.Module):
    def __init__(self, d=256):
        super().__init__()
        self.up = torch.nn.Linear(d, 4 * d)
        self.act = torch.nn.GELU()
        self.down = torch.nn.Linear(4 * d, d)
        self.gate = torch.nn.SiLU()
        self.lm_head = torch.nn.Linear(d, 40)

    def forward(self, x):
        return self.lm_head(self.gate(x + self.down(self.act(self.up(x)))))


def test_a_model_with_weights_in_8_bits():
    torch.manual_seed(0)
    model = Block().to(torch.bfloat16).to(DEV)
    twin = Block().to(torch.bfloat16).to(DEV)
    twin.load_state_dict(model.state_dict())
    head = model.lm_head
    neuzip_amd.fp8_convert(model)
    assert isinstance(model.up, nn.FP8Linear) and model.lm_head is head
    x = rnd(30, 256)
    with torch.no_grad():
        for name in ("up", "down"):
            layer, dense = getattr(model, name), getattr(twin, name)
            assert torch.equal(layer.weight.dequantize().cpu().double(), held(dense.weight.detach().cpu(), 128))
            assert layer.nbytes_compressed() == dense.weight.numel() + layer.weight_scales.numel()
        h = ops.fp8_quantize(x)
        assert torch.equal(model.up(h), model.up(x))
    a = x.clone().requires_grad_(True)
    model(a).sum().backward()
    assert a.grad.shape == x.shape and model.up.bias.grad is not None and model.down.bias.grad is not None
    other = neuzip_amd.fp8_convert(Block().to(torch.bfloat16).to(DEV))
    other.load_state_dict(model.state_dict())
    with torch.no_grad():
        assert torch.equal(other(x), model(x))
        with torch.autocast("cuda", torch.bfloat16):
            assert torch.equal(model.up(x.float()), model.up(x))
    rows = nn.FP8Linear(twin.up, block_rows=1)
    assert torch.equal(rows.weight.dequantize().cpu().double(), held(twin.up.weight.detach().cpu(), 1))


def test_a_training_step_with_8_bits_kept():
    """a converted model whose layers keep 8 bits: the same result, gradients near those of the kept 16 bits"""
    torch.manual_seed(0)
    model = Block().to(torch.bfloat16)
    manager = neuzip_amd.Manager(precision=7)
    manager.convert(model)
    model = model.to(DEV)
    x, g = rnd(64, 256), rnd(64, 40, seed=1, scale=1e-2)

    def step():
        a = x.clone().requires_grad_(True)
        kept = {}

        def pack(t):
            if t.dim():
                kept[t.data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = model(a)
        y.backward(g)
        out = [y.detach(), a.grad, model.up.weight._gradient, model.down.weight._gradient, model.lm_head.weight.grad]
        model.up.weight._gradient = model.down.weight._gradient = model.lm_head.weight.grad = None
        return out, sum(kept.values())

    full, full_bytes = step()
    neuzip_amd.fp8_activations(model)
    assert model.up.saved_bits == 8 and isinstance(model.act, nn.FP8Activation)
    part, part_bytes = step()
    assert part_bytes < 0.6 * full_bytes
    for a, b in zip(part, full):
        # e4m3 keeps four bits: what passes through several such values differs by a few times 2^-4 of its size at most
        assert (a.double() - b.double()).norm() <= 2.0 ** -3 * b.double().norm()
    with neuzip_amd.DecompressAhead(manager, model):
        again, _ = step()
    for a, b in zip(again, part):
        assert torch.equal(a, b)


def test_calls_on_another_stream():
    x, w = rnd(300, 500), ops.fp8_quantize(rnd(260, 500, seed=1), 128)
    g = rnd(300, 260, seed=2)
    want = ops.fp8_linear(x, w), ops.fp8_weight_gradient(g, ops.fp8_quantize(x)), ops.fp8_activation(x, "silu", x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = ops.fp8_linear(x, w), ops.fp8_weight_gradient(g, ops.fp8_quantize(x)), ops.fp8_activation(x, "silu", x)
    other = ops.fp8_linear(x, w)  # at the same time, with a workspace of its own
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want[0])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("m,dtype", [(1, torch.bfloat16), (70, torch.bfloat16), (700, torch.float16), (40, torch.float32)])
def test_a_captured_step(m, dtype):
    """forward and backward of the operators together, captured, replayed with other values and eager work between"""
    w = ops.fp8_quantize(rnd(600, 400, seed=1, scale=0.05, dtype=torch.float32), 128)
    x, g = rnd(m, 400, dtype=dtype), rnd(m, 600, seed=2, dtype=dtype)
    total = torch.zeros(600, 400, dtype=dtype, device=DEV)
    bias = torch.zeros(600, dtype=dtype, device=DEV)

    def step(x, g, total):
        a, b = x.detach().requires_grad_(True), bias.detach().requires_grad_(True)
        h = ops.fp8_linear(ops.fp8_activation(a), w, b)
        y = ops.fp8_activation(h, "silu", h)
        da, db = torch.autograd.grad(y, (a, b), g)
        ops.fp8_weight_gradient(g, ops.fp8_quantize(x), out=total)
        return y.detach(), da, db

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, g, torch.zeros_like(total))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, g, total)
    for turn in range(4):
        x.copy_(rnd(m, 400, seed=10 + turn, dtype=dtype))
        g.copy_(rnd(m, 600, seed=20 + turn, dtype=dtype))
        total.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = torch.zeros_like(total)
        want = step(x, g, again)
        for a, b in zip((*out, total), (*want, again)):
            assert torch.equal(a, b)


def test_two_captured_calls_share_no_workspace():
    w = ops.fp8_quantize(rnd(520, 4000, seed=1), 128)
    x = [rnd(64, 4000, seed=i) for i in (2, 3)]
    want = [ops.fp8_linear(t, w) for t in x]
    graphs, out = [], []
    for t in x:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            out.append(ops.fp8_linear(t, w))
    side = torch.cuda.Stream()
    for _ in range(3):
        for t in out:
            t.zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_compiled_functions_make_the_calls():
    w = ops.fp8_quantize(rnd(40, 64, seed=1), 128)
    x = rnd(5, 64)

    def work(x):
        return ops.fp8_activation(ops.fp8_linear(x * 2, w) + 1, "gelu")

    compiled = torch.compile(work, backend="eager")
    for scale in (1.0, 3.0):
        assert torch.equal(compiled(x * scale), work(x * scale))


def test_kept_inputs_that_hooks_take_elsewhere_are_not_held():
    """A hook that moves saved tensors to the host frees their memory until the backward pass."""
    layer, _ = pair(8, rows=128, cols=4096)
    x, g = rnd(2048, 4096), rnd(2048, 128, seed=1, scale=1e-2)
    layer(x.requires_grad_(True)).backward(g)
    want, layer.weight._gradient = layer.weight._gradient, None
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        y = layer(x)
    assert torch.cuda.memory_allocated() - before < 2048 * 4096 // 2  # y alone is 2048 * 128 * 2
    y.backward(g)
    assert torch.equal(layer.weight._gradient, want)
