"""GPU: the gradient of embedding tables against float64 sums, and a compressed
table that is trained."""
import math
from functools import partial

import pytest
import torch

import neuzip_amd
from neuzip_amd import ops
from mx_oracle import HALF_STEP, held, round_to

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
IDS = ["bf16", "fp16", "fp32"]
DEV = "cuda"


def tokens(kind, count, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, rows, (count,), generator=g)
    if kind == "text":  # the frequency falls with the rank
        rank = torch.exp(torch.rand(count, generator=g, dtype=torch.float64) * math.log(rows)).long() - 1
        return torch.randperm(rows, generator=g)[rank.clamp(0, rows - 1)]
    if kind == "one":
        return torch.full((count,), rows // 2)
    if kind == "two":
        return torch.where(torch.rand(count, generator=g) < 0.1, rows - 1, 0)
    return torch.arange(count).flip(0) % rows  # "descending"


def summed(ids, g, rows, skip=None):
    """float64 sums, sums of magnitudes and counts of a table's rows"""
    ok = (ids >= 0) & (ids < rows)
    if skip is not None:
        ok &= ids != skip
    total = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    total.index_add_(0, ids[ok], g[ok].double())
    size = torch.zeros_like(total).index_add_(0, ids[ok], g[ok].double().abs())
    return total, size, torch.bincount(ids[ok], minlength=rows).double()[:, None]


CASES = [("uniform", 1, 1, 1), ("uniform", 5, 7, 3), ("text", 100, 40, 33), ("uniform", 64, 1000, 8),
         ("one", 257, 9, 64), ("text", 2000, 5003, 129), ("two", 1030, 300, 520), ("descending", 700, 350, 1021),
         ("text", 4099, 50257, 40), ("one", 3000, 2, 513), ("uniform", 9000, 1500, 24), ("text", 20000, 3001, 16),
         ("text", 16385, 900, 40), ("two", 32768, 11, 24), ("one", 70000, 3, 8), ("text", 1023, 400, 24),
         ("text", 1024, 50257, 520), ("one", 1024, 2, 100), ("two", 1025, 30, 17), ("uniform", 17, 1, 40),
         ("two", 1000, 8, 1540), ("text", 70001, 130000, 8), ("text", 10000, 600000, 9),
         ("uniform", 300, 140000, 16), ("uniform", 1, 5, 4096), ("uniform", 200001, 900, 8), ("text", 66000, 600000, 4),
         ("text", 200000, 700000, 4), ("text", 1100000, 3000, 2)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind,count,rows,cols", CASES)
def test_whole_numbers_are_exact(kind, count, rows, cols, dtype):
    """whole numbers up to 100 in magnitude: 70000 of them (200000 up to 60, 1100000 up to 15) stay below 2^24"""
    ids = tokens(kind, count, rows, seed=count)
    most = 100 if count <= 70001 else 60 if count <= 200001 else 15
    g = torch.randint(-most, most + 1, (count, cols), generator=torch.Generator().manual_seed(1)).to(dtype)
    total, _, _ = summed(ids, g, rows)
    got = ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, 0.5)
    assert got.dtype == dtype
    want = round_to(total * 0.5, dtype)
    if dtype == torch.float16:  # beyond 65504 it is an infinity in both
        want = torch.where((total * 0.5).abs() >= 65520, torch.sign(total) * math.inf, want.double()).to(dtype)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind,count,rows,cols", [("text", 3000, 700, 100), ("one", 5000, 4, 33), ("uniform", 900, 80, 256)])
def test_random_values_and_the_same_bits_every_time(kind, count, rows, cols, dtype):
    """count additions and the product with the scale, 2^-24 each, and half a step of the result"""
    ids = tokens(kind, count, rows, seed=2)
    g = torch.randn(count, cols, generator=torch.Generator().manual_seed(3)).to(dtype)
    total, size, n = summed(ids, g, rows)
    scale = 1.7
    want = total * torch.tensor(scale, dtype=torch.float32).double()
    got = ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, scale)
    tol = HALF_STEP[dtype] * want.abs() + (n + 2) * 2.0 ** -24 * size * scale * (1 + HALF_STEP[dtype])
    assert ((got.cpu().double() - want).abs() <= tol).all()
    for _ in range(3):
        assert torch.equal(got, ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, scale))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("kind,count,rows,cols", [("text", 800, 300, 65), ("two", 300, 9, 512), ("uniform", 20000, 77, 8),
                                                    ("two", 3000, 9, 512), ("text", 8192, 300, 65)])
def test_padding_frequency_and_indices_outside(kind, count, rows, cols, dtype):
    ids = tokens(kind, count, rows, seed=4)
    ids[::7] = torch.tensor([-1, rows, 2 ** 40, -2 ** 63, rows + 5])[torch.arange(len(ids[::7])) % 5]
    skip = int(ids[(ids >= 0) & (ids < rows)][0])
    g = torch.randint(-60, 61, (count, cols), generator=torch.Generator().manual_seed(5)).to(dtype)
    total, size, n = summed(ids, g, rows, skip)
    got = ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, padding_idx=skip)
    assert torch.equal(got.cpu(), round_to(total, dtype))
    assert torch.equal(got, ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, padding_idx=skip - rows))
    got = ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, 3.0, padding_idx=skip, scale_grad_by_freq=True)
    want = 3.0 * total / n.clamp(min=1)
    # the quotient of the scale, the product with it and the result are rounded
    assert ((got.cpu().double() - want).abs() <= (HALF_STEP[dtype] + 2.0 ** -22) * want.abs()).all()


@pytest.mark.parametrize("count", (900, 3000))
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_adding_to_a_gradient(dtype, count):
    rows, cols = 500, 72
    old = torch.randint(-50, 51, (rows, cols), generator=torch.Generator().manual_seed(6)).to(dtype)
    old[3] = math.nan  # a row without a token is left as it is
    ids = tokens("text", count, rows, seed=7)
    ids[ids == 3] = 4
    g = torch.randint(-60, 61, (count, cols), generator=torch.Generator().manual_seed(8)).to(dtype)
    total, _, n = summed(ids, g, rows)
    out = old.to(DEV)
    at = out.data_ptr()
    assert ops.embedding_gradient(ids.to(DEV), g.to(DEV), rows, out=out).data_ptr() == at
    want = torch.where(n > 0, round_to(torch.nan_to_num(old.double()) + total, dtype), old)
    assert torch.equal(torch.nan_to_num(out.cpu()), torch.nan_to_num(want))
    assert torch.isnan(out[3]).all() and torch.isnan(out).sum() == cols
    ops.embedding_gradient(ids[:0].to(DEV), g[:0].to(DEV), rows, out=out)
    assert torch.equal(torch.nan_to_num(out.cpu()), torch.nan_to_num(want))


def test_shapes_strides_and_empty():
    ids = tokens("uniform", 60, 11).view(3, 20)
    g = torch.randint(-9, 10, (3, 20, 50), generator=torch.Generator().manual_seed(1)).float()
    for view in (g, g[..., 3:], g[..., :33], g[..., ::2]):
        want, _, _ = summed(ids.view(-1), view.reshape(60, -1), 11)
        base = g.to(DEV)
        v = base.as_strided(view.shape, view.stride(), view.storage_offset())
        assert torch.equal(ops.embedding_gradient(ids.int().to(DEV), v, 11).cpu(), want.float())
    want, _, _ = summed(ids.view(-1), torch.ones(60, 50), 11)
    assert torch.equal(ops.embedding_gradient(ids.to(DEV), torch.ones(1, device=DEV).expand(3, 20, 50), 11).cpu(),
                       want.float())
    assert not ops.embedding_gradient(ids[:0].to(DEV), g[:0].to(DEV), 11).any()
    assert ops.embedding_gradient(ids.to(DEV), g[..., :0].to(DEV), 11).shape == (11, 0)
    assert ops.embedding_gradient(ids.to(DEV), g.to(DEV), 0).shape == (0, 50)


def test_special_values_stay_in_their_rows():
    ids = torch.tensor([1, 2, 1, 3])
    g = torch.ones(4, 40)
    g[0, 5], g[2, 6], g[3, 7] = math.inf, math.nan, -math.inf
    got = ops.embedding_gradient(ids.to(DEV), g.to(DEV), 5).cpu()
    assert got[1, 5] == math.inf and torch.isnan(got[1, 6]) and got[3, 7] == -math.inf
    assert torch.isnan(got).sum() == 1 and torch.isinf(got).sum() == 2
    ids, g = torch.cat([ids, torch.arange(3000) % 50 + 4]), torch.cat([g, torch.ones(3000, 40)])  # sorted
    more = ops.embedding_gradient(ids.to(DEV), g.to(DEV), 60).cpu()
    assert torch.equal(torch.nan_to_num(more[:4], nan=7.5), torch.nan_to_num(got[:4], nan=7.5))
    assert (more[4:54] == 60).all() and not more[54:].any()


def test_offsets_beyond_32_bits():
    rows, cols = 4_400_000, 512
    ids = torch.tensor([rows - 1, 0, rows - 1], device=DEV)
    g = torch.ones(3, cols, dtype=torch.bfloat16, device=DEV)
    got = ops.embedding_gradient(ids, g, rows, 3.0)
    assert got.numel() * 2 > 2 ** 32
    assert (got[-1] == 6).all() and (got[0] == 3).all() and not got[1:-1].any()
    wide = torch.zeros(2, 2 ** 31 + 64, dtype=torch.bfloat16, device=DEV)  # rows of g far apart
    wide[1, :8] = 5
    got = ops.embedding_gradient(ids[:2], wide[:, :8], rows)
    assert (got[0] == 5).all() and not got[1:].any()
    ids = torch.cat([ids[:2], torch.full((9000,), rows, device=DEV)])  # sorted
    got = ops.embedding_gradient(ids, wide[1, :8].expand(9002, 8), rows)
    assert (got[0] == 5).all() and (got[-1] == 5).all() and not got[1:-1].any()


def test_captured_beside_eager():
    ids = torch.zeros(900, dtype=torch.int64, device=DEV)
    g = torch.randn(900, 48, generator=torch.Generator().manual_seed(1)).to(DEV)
    acc = torch.zeros(400, 48, device=DEV)

    def work():
        acc.zero_()
        out = ops.embedding_gradient(ids, g, 400)
        ops.embedding_gradient(ids, g, 400, out=acc)
        return out

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(5):
        ids.copy_(tokens("text", 900, 400, seed=i))
        graph.replay()
        torch.cuda.synchronize()
        captured, added = out.clone(), acc.clone()
        eager = work()
        assert torch.equal(captured, eager) and torch.equal(added, eager)


class Rate:
    def get_last_lr(self):
        return [0.5]


def test_a_compressed_table_is_trained():
    torch.manual_seed(0)
    manager = neuzip_amd.Manager()
    dense = torch.nn.Embedding(120, 64, padding_idx=7).to(torch.bfloat16)
    frozen = neuzip_amd.nn.Embedding(manager, dense)
    table = dense.weight.detach().clone()
    emb = neuzip_amd.nn.Embedding(manager, dense, scale=8.0, trainable=True).to(DEV)
    assert repr(emb).endswith("scale=8.0, trainable)")
    ids = torch.randint(0, 120, (4, 30), generator=torch.Generator().manual_seed(1))
    ids[0, :3] = 7
    y = emb(ids.to(DEV))
    assert y.requires_grad and not frozen(ids.to(DEV)).requires_grad
    assert torch.equal(y.cpu(), (table[ids].float() * 8).to(torch.bfloat16))
    with torch.no_grad():
        assert torch.equal(emb(ids.to(DEV)), y) and not emb(ids.to(DEV)).requires_grad
    g = torch.randint(-4, 5, y.shape, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    y.backward(g.to(DEV))
    total, _, _ = summed(ids.view(-1), g.view(-1, 64), 120, skip=7)
    assert torch.equal(emb.weight._gradient.cpu(), (8 * total).to(torch.bfloat16))
    assert emb.weight.grad.numel() == 0
    emb(ids.to(DEV)).backward(g.to(DEV))
    assert torch.equal(emb.weight._gradient.cpu(), (16 * total).to(torch.bfloat16))
    neuzip_amd.compressed_lomo_hook(Rate(), emb.weight)
    want = table.to(DEV).add_((16 * total).to(torch.bfloat16).to(DEV), alpha=-0.5)
    assert emb.weight._gradient is None
    assert torch.equal(emb.weight(), want)
    assert torch.equal(emb(ids.to(DEV)).cpu(), (want.cpu()[ids].float() * 8).to(torch.bfloat16))


def test_embedding_linears_and_head_in_one_step():
    """tokens -> trained compressed table -> frozen 4-bit Linears -> logits of a 4-bit table, and back"""
    torch.manual_seed(0)
    vocab, d, ffn = 200, 96, 224
    manager = neuzip_amd.Manager()
    source = torch.nn.Embedding(vocab, d).to(torch.bfloat16)
    table = source.weight.detach().clone()
    head = neuzip_amd.nn.MXEmbedding(source)
    emb = neuzip_amd.nn.Embedding(manager, source, scale=2.0, trainable=True).to(DEV)
    block = torch.nn.Sequential(torch.nn.Linear(d, ffn, bias=False), torch.nn.ReLU(), torch.nn.Linear(ffn, d))
    block = block.to(torch.bfloat16)
    w1, w2, b2 = (p.detach().clone() for p in block.parameters())
    neuzip_amd.mx_convert(block)
    block = block.to(DEV)
    emb.weight.register_post_accumulate_grad_hook(partial(neuzip_amd.compressed_lomo_hook, Rate()))
    ids = torch.randint(0, vocab, (5, 13), generator=torch.Generator().manual_seed(1))
    kept = {}
    x = emb(ids.to(DEV))
    h = block(x)
    logits = head.linear(h)
    for name, t in (("x", x), ("h", h), ("logits", logits)):
        t.register_hook(lambda g, n=name: kept.__setitem__(n, g.detach().cpu().double()))
    logits.float().logsumexp(-1).sum().backward()
    # float64, from the values that each step was given
    xr = (table[ids].float() * 2).to(torch.bfloat16)
    assert torch.equal(x.detach().cpu(), xr)
    W1, W2, T = held(w1, 4), held(w2, 4), held(table, 4)
    a = held(xr.view(-1, d), 8) @ W1.t()
    a16 = a.to(torch.bfloat16).relu()
    hr = held(a16, 8) @ W2.t() + b2.double()
    # each product is half a bf16 step off; an activation that this moves over a border of its 8-bit code moves by
    # one step of it (2^-3 relative): the two runs may differ there, so the layers are compared in the mean
    got = h.detach().cpu().double().view(-1, d)
    assert (got - hr).norm() <= 2.0 ** -6 * hr.norm()
    lr = held(h.detach().cpu().view(-1, d), 8) @ T.t()
    gl = logits.detach().cpu().double().view(-1, vocab)
    size = held(h.detach().cpu().view(-1, d), 8).abs() @ T.abs().t()
    assert ((gl - lr).abs() <= 2.0 ** -8 * lr.abs() + d * 2.0 ** -23 * size).all()
    gh = kept["logits"].view(-1, vocab) @ T
    assert ((kept["h"].view(-1, d) - gh).abs() <= 2.0 ** -8 * gh.abs() + vocab * 2.0 ** -22 *
            (kept["logits"].view(-1, vocab).abs() @ T.abs())).all()
    gx = kept["x"].view(-1, d)
    total, _, _ = summed(ids.view(-1), gx.to(torch.bfloat16), vocab)
    step = round_to(2 * total, torch.bfloat16)
    want = table.to(DEV).add_(step.to(DEV), alpha=-0.5)
    # sums of a few bf16 numbers in 32 bits may round the other way than the float64 sum: one step of the gradient
    diff = (emb.weight().cpu().double() - want.cpu().double()).abs()
    assert (diff <= 0.5 * 2.0 ** -7 * (2 * total).abs() + 2.0 ** -7 * want.cpu().double().abs()).all()
    assert emb.weight._gradient is None
