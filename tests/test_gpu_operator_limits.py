"""Counts beyond what one launch may hold (2^32 - 1 threads): the operators make several, or refuse before the first."""
import pytest
import torch

from neuzip_amd import _lib, ops

DEV = "cuda"
L = _lib.load()


def test_what_is_refused():
    p, room = 1 << 20, 1 << 62  # addresses that are never looked at
    for count, cols in ((1 << 28, 4), ((1 << 28) - 31, 4),  # 32 indices to each of 2^23 workgroups of 512 threads
                        (1 << 22, 1 << 18), (1 << 30, 4)):  # 64 indices and 512 columns to each of 2^24 of 256
        rc = L.nz_embedding_gradient(p, count, p, 0, cols, 9, cols, 1.0, -1, 0, p, p, room, None)
        assert rc == _lib.ERR_ARG and "too many" in _lib.last_error()
    for call in (L.nz_mx_quantize(p, 0, (1 << 33) + 1, 512, 512, 4, p, p, None),
                 L.nz_mx_dequantize(p, p, (1 << 33) + 1, 512, 4, p, 0, None)):
        assert call == _lib.ERR_ARG and "too many" in _lib.last_error()


@pytest.fixture
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", (4, 8))
def test_more_rows_than_a_launch_holds(memory, bits):
    """67108860 rows of up to 512 values fill a launch; all values are codes"""
    rows = 70_000_000
    x = torch.tensor([-6.0, -3.0, -1.0, 0.0, 0.5, 1.5, 2.0, 4.0], dtype=torch.bfloat16, device=DEV)
    x = x[torch.randint(0, 8, (rows, 40), device=DEV, dtype=torch.int32)]
    x[:, 0], x[:, 32] = 6.0, -4.0  # the scale of both blocks is one
    q = ops.mx_quantize(x, bits)
    assert torch.equal(q.dequantize(), x)
    ids = torch.arange(rows - 1, -1, -1, device=DEV)
    ids[5], ids[-5] = rows, -1
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = ops.mx_embedding(ids, q, status=status)
    assert status.item() == 1 and not got[5].any() and not got[-5].any()
    got[5], got[-5] = x[rows - 6], x[4]
    assert torch.equal(got, x.flip(0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32), ids=("bf16", "fp32"))
def test_products_of_more_rows_than_a_launch_brings_to_8_bits(memory, dtype):
    m, n, k = 1 << 24, 3, 2100  # rows that all lie in the same place
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-7, 8, (1, k), generator=g).to(dtype)
    w = ops.mx_quantize(torch.randint(-6, 7, (n, k), generator=g).float().to(DEV), 4)
    want = (x.double() @ w.dequantize(torch.float32).cpu().double().t()).to(dtype)
    y = ops.mx_linear(x.to(DEV).expand(m, k), w)
    assert torch.equal(y[:1].cpu(), want) and (y == y[:1]).all()


@pytest.mark.gpu
def test_gradients_of_more_rows_than_a_launch_cuts(memory):
    m, n, k = 1 << 24, 2100, 32
    gen = torch.Generator().manual_seed(1)
    g = torch.randint(-9, 10, (1, n), generator=gen).to(torch.bfloat16)
    w = ops.mx_quantize(torch.randint(-6, 7, (n, k), generator=gen).float().to(DEV), 4)
    want = (g.double() @ w.dequantize(torch.float32).cpu().double()).to(torch.bfloat16)
    dx = ops.microscaled._input_gradient(g.to(DEV).expand(m, n), w)
    assert torch.equal(dx[:1].cpu(), want) and (dx == dx[:1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("count", (3, 3000))  # without sorting, and with
def test_a_table_that_one_launch_does_not_clear(memory, count):
    rows, cols = 68_000_003, 1021  # 2^23 workgroups clear 16 KB each: 137.4 GB of 138.9
    out = torch.full((rows * cols + 1,), 7.0, dtype=torch.bfloat16, device=DEV)
    ids = torch.full((count,), rows, device=DEV)  # outside, but for two
    ids[0], ids[1] = rows - 1, 0
    g = torch.ones(count, cols, dtype=torch.bfloat16, device=DEV)
    # the table of a torch tensor is aligned: this one begins between vectors
    room = max(16, L.nz_embedding_gradient_workspace_bytes(count, cols))
    ws = torch.empty(room, dtype=torch.uint8, device=DEV)
    _lib.raise_for(L.nz_embedding_gradient(ids.data_ptr(), count, g.data_ptr(), _lib.DTYPE_BF16, cols, rows, cols, 3.0,
                                           -1, 0, out.data_ptr() + 2, ws.data_ptr(), room,
                                           torch.cuda.current_stream().cuda_stream))
    assert out[0] == 7
    table = out[1:].view(rows, cols)
    assert (table[0] == 3).all() and (table[-1] == 3).all()
    for at in range(1, rows - 1, 4_000_000):
        assert not table[at:min(rows - 1, at + 4_000_000)].any()
