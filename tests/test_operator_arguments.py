"""CPU: what the operators on microscaled weights and embedding gradients refuse,
at the C ABI (before any HIP call) and in Python."""
import pytest
import torch

import neuzip_amd
from neuzip_amd import _lib, ops
from mx_oracle import decoded, held

L = _lib.load()


def refused(rc, code, text):
    assert rc == code
    assert text in _lib.last_error()


def test_sizes_of_the_stored_form():
    for cols, padded, groups in ((0, 0, 0), (1, 128, 1), (128, 128, 1), (129, 256, 1), (512, 512, 1), (513, 640, 2),
                                 (4096, 4096, 8)):
        assert L.nz_mx_row_bytes(cols, 4) == padded // 2
        assert L.nz_mx_row_bytes(cols, 8) == padded
        assert L.nz_mx_scale_bytes(cols) == 16 * groups
    assert L.nz_mx_row_bytes(100, 5) == 0


def test_refusals_of_the_abi():
    A, B, C, D = _lib.ERR_ARG, _lib.ERR_ALIGN, _lib.ERR_DTYPE, _lib.ERR_CAPACITY
    p = 1 << 20  # an address that is never looked at
    refused(L.nz_mx_quantize(p, 0, 1, 1, 1, 5, p, p, None), A, "bits must be 4 or 8")
    refused(L.nz_mx_quantize(p, 3, 1, 1, 1, 4, p, p, None), C, "Unsupported data type")
    refused(L.nz_mx_quantize(p + 1, 0, 1, 1, 1, 4, p, p, None), B, "aligned to their elements")
    refused(L.nz_mx_quantize(p, 0, 1, 1, 1, 4, p + 8, p, None), B, "16-byte aligned")
    refused(L.nz_mx_quantize(None, 0, 1, 1, 1, 4, p, p, None), A, "null input")
    refused(L.nz_mx_quantize(p, 0, 1, 1, 1, 4, None, p, None), A, "null data")
    refused(L.nz_mx_quantize(p, 0, 1, 1 << 31, 1, 4, p, p, None), A, "2^30")
    refused(L.nz_mx_quantize(p, 0, 1 << 60, 512, 1, 4, p, p, None), A, "too many rows")
    assert L.nz_mx_quantize(None, 0, 0, 5, 1, 4, None, None, None) == _lib.OK
    assert L.nz_mx_quantize(None, 0, 5, 0, 1, 4, None, None, None) == _lib.OK
    refused(L.nz_mx_dequantize(p, p, 1, 1, 4, None, 0, None), A, "null output")
    refused(L.nz_mx_lookup(p, p, 5, 1, 4, None, 3, 1.0, p, 0, None, None), A, "null indices")
    refused(L.nz_mx_lookup(p, p, 5, 1, 4, p + 4, 3, 1.0, p, 0, None, None), B, "misaligned")
    refused(L.nz_mx_lookup(p, p, 5, 1, 4, p, 3, 1.0, p, 0, p + 2, None), B, "misaligned")
    refused(L.nz_mx_linear(p, 0, 1, 0, 1, p, p, 1, None, p, p, 1 << 30, None), A, "1 to 2^22")
    refused(L.nz_mx_linear(p, 0, 1, 32, 32, None, p, 1, None, p, p, 1 << 30, None), A, "null data")
    refused(L.nz_mx_linear(p, 0, 1, 32, 32, p, p, 1, None, None, p, 1 << 30, None), A, "null rows or output")
    refused(L.nz_mx_linear(p, 0, 1, 32, 32, p, p, 1, p + 1, p, p, 1 << 30, None), B, "aligned to their elements")
    refused(L.nz_mx_linear(p, 0, 1 << 40, 32, 32, p, p, 1, None, p, p, 1 << 30, None), A, "too many rows")
    need = L.nz_mx_linear_workspace_bytes(1000, 512, 512, 0)
    assert need >= 1000 * 512
    refused(L.nz_mx_linear(p, 0, 1000, 512, 512, p, p, 512, None, p, p, need - 1, None), D, "workspace")
    refused(L.nz_mx_linear(p, 0, 1000, 512, 512, p, p, 512, None, p, p + 8, need, None), B, "workspace")
    refused(L.nz_mx_linear_rows8(p, p + 4, 1, 32, p, p, 1, None, p, 0, None, 0, None), B, "16-byte aligned")
    assert L.nz_mx_linear(None, 0, 0, 32, 32, None, None, 7, None, None, None, 0, None) == _lib.OK
    refused(L.nz_mx_linear_rows8(p, p, 1000, 512, p, p, 512, None, p, 0, p, 0, None), D, "workspace")
    refused(L.nz_mx_linear_grad(p, 9, 1, 1, 1, p, p, 1, p, p, 1 << 30, None), C, "Unsupported data type")
    refused(L.nz_mx_linear_grad(None, 0, 1, 1, 1, p, p, 1, p, p, 1 << 30, None), A, "null gradient")
    refused(L.nz_mx_linear_grad(p, 0, 1, 0, 1, p, p, 1, p, p, 1 << 30, None), A, "without rows")
    refused(L.nz_mx_linear_grad(p, 0, 1, 1 << 22, 1 << 22, p, p, 1, p, p, 1 << 30, None), A, "2^21")
    refused(L.nz_mx_linear(p, 0, 1 << 24, 32, 32, p, p, 1 << 21, None, p, p, 1 << 62, None), A, "too many rows")
    assert L.nz_mx_linear_grad_workspace_bytes(p, 0, 100, 512, 512, 512) < 100 * 512 * 2 < (
        L.nz_mx_linear_grad_workspace_bytes(p, 1, 100, 512, 512, 512))
    need = L.nz_mx_linear_grad_workspace_bytes(p + 2, 0, 100, 512, 512, 512)
    refused(L.nz_mx_linear_grad(p + 2, 0, 100, 512, 512, p, p, 512, p, p, need - 1, None), D, "workspace")
    assert L.nz_mx_linear_grad(None, 0, 0, 1, 1, None, None, 1, None, None, 0, None) == _lib.OK
    for huge in (1 << 24, 1 << 40, (1 << 63) + 5, (1 << 64) - 1):  # sizes beyond the limits: an answer, no harm
        for m, n, k in ((huge, 5, 5), (5, huge, 5), (5, 5, huge), (huge, huge, huge)):
            L.nz_mx_linear_workspace_bytes(m, n, k, 0), L.nz_mx_linear_workspace_bytes(m, n, k, 2)
            L.nz_mx_linear_grad_workspace_bytes(p, 0, m, n, n, k)
            L.nz_column_sums_workspace_bytes(m, n), L.nz_embedding_gradient_workspace_bytes(m, n)
    sums, need = L.nz_column_sums, L.nz_column_sums_workspace_bytes(5000, 100)
    assert need and not L.nz_column_sums_workspace_bytes(1, 100)
    refused(sums(p, 9, 5, 5, 5, p, p, 0, None), C, "Unsupported data type")
    refused(sums(None, 0, 5, 5, 5, p, p, 0, None), A, "null")
    refused(sums(p + 1, 0, 5, 5, 5, p, p, 0, None), B, "aligned")
    refused(sums(p, 0, 1 << 31, 5, 5, p, p, 0, None), A, "too many")
    refused(sums(p, 0, 5000, 100, 100, p, p, need - 1, None), D, "workspace")
    refused(sums(p, 0, 5000, 100, 100, p, None, need, None), B, "workspace")
    assert sums(None, 0, 5, 0, 5, None, None, 0, None) == _lib.OK
    grad = L.nz_embedding_gradient
    refused(grad(p, 1, p, 7, 1, 1, 1, 1.0, -1, 0, p, p, 1 << 30, None), C, "Unsupported data type")
    refused(grad(p, 1, p, 0, 1, 1, 1, 1.0, -1, 4, p, p, 1 << 30, None), A, "unknown flags")
    refused(grad(None, 1, p, 0, 1, 1, 1, 1.0, -1, 0, p, p, 1 << 30, None), A, "null")
    refused(grad(p + 4, 1, p, 0, 1, 1, 1, 1.0, -1, 0, p, p, 1 << 30, None), B, "aligned")
    refused(grad(p, 1 << 32, p, 0, 1, 1, 1, 1.0, -1, 0, p, p, 1 << 30, None), A, "too many")
    need = L.nz_embedding_gradient_workspace_bytes(5000, 8)
    assert need and not L.nz_embedding_gradient_workspace_bytes(1000, 8)
    refused(grad(p, 5000, p, 0, 8, 9, 8, 1.0, -1, 0, p, p, need - 1, None), D, "workspace")
    refused(grad(p, 5000, p, 0, 8, 9, 8, 1.0, -1, 0, p, p + 8, need, None), B, "workspace")
    assert grad(None, 0, None, 0, 1, 0, 5, 1.0, -1, 0, None, None, 0, None) == _lib.OK


def cpu_weight(n=4, k=64, bits=4):
    return ops.MXTensor(torch.zeros(n, L.nz_mx_row_bytes(k, bits), dtype=torch.uint8),
                        torch.zeros(n, L.nz_mx_scale_bytes(k), dtype=torch.uint8), (n, k), bits)


def test_refusals_in_python():
    x = torch.zeros(2, 64)
    w = cpu_weight()
    with pytest.raises(ValueError, match="on the GPU"):
        ops.mx_quantize(x)
    with pytest.raises(ValueError, match="4 or 8"):
        ops.mx_quantize(x, 6)
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        ops.mx_quantize(x.double())
    with pytest.raises(ValueError, match="on the GPU"):
        w.dequantize()
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        w.dequantize(torch.int32)
    with pytest.raises(ValueError, match="microscaled 4 bits"):
        ops.mx_linear(x, torch.zeros(4, 64))
    with pytest.raises(ValueError, match="microscaled 4 bits"):
        ops.mx_linear(x, cpu_weight(bits=8))
    with pytest.raises(ValueError, match="64 columns, the weight 96"):
        ops.mx_linear(x, cpu_weight(k=96))
    with pytest.raises(ValueError, match="bias must be"):
        ops.mx_linear(x, w, torch.zeros(5))
    with pytest.raises(ValueError, match="bias must be"):
        ops.mx_linear(x, w, torch.zeros(4, dtype=torch.float16))
    with pytest.raises(ValueError, match="type of x"):
        ops.mx_linear(x, w, dtype=torch.float16)
    with pytest.raises(ValueError, match="8 bits"):
        ops.mx_linear(w, w)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.mx_linear(x, w)
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        ops.mx_linear(x.double(), w)
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.mx_embedding(torch.zeros(3), w)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.mx_embedding(torch.zeros(3, dtype=torch.int64), w)
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="shape of indices"):
        ops.embedding_gradient(ids, torch.zeros(2, 5), 7)
    with pytest.raises(ValueError, match="int64 or int32"):
        ops.embedding_gradient(ids.float(), torch.zeros(3, 5), 7)
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embedding_gradient(ids, torch.zeros(3, 5), 7, padding_idx=7)
    with pytest.raises(ValueError, match="on the GPU"):
        ops.embedding_gradient(ids, torch.zeros(3, 5), 7)
    with pytest.raises(ValueError, match="shape"):
        ops.MXTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 8, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="shape"):
        ops.MXTensor(torch.zeros(4, 64), torch.zeros(4, 16, dtype=torch.uint8), (4, 64))
    with pytest.raises(ValueError, match="max_norm"):
        neuzip_amd.nn.MXEmbedding(torch.nn.Embedding(4, 8, max_norm=1.0))


def test_a_table_that_cannot_be_trained_is_refused():
    with pytest.raises(ValueError, match="max_norm"):
        neuzip_amd.nn.Embedding(None, torch.nn.Embedding(4, 8, max_norm=1.0), trainable=True)
    with pytest.raises(ValueError, match="sparse"):
        neuzip_amd.nn.Embedding(None, torch.nn.Embedding(4, 8, sparse=True), trainable=True)


def test_a_compressed_table_is_trained_on_the_gpu():
    class Held:
        def write(self, data):
            return "0"

    emb = neuzip_amd.nn.Embedding(Held(), torch.nn.Embedding(4, 8), trainable=True)
    with pytest.raises(ValueError, match="trained on the GPU"):
        emb(torch.zeros(2, dtype=torch.int64))


def test_the_oracle_itself():
    """hand-made bytes against the statement of the format, and values that are codes already"""
    data = torch.zeros(1, 64, dtype=torch.uint8)
    data[0, 0], data[0, 16] = 0x7A, 0x01  # -1 and 6 in block 0, 0.5 in block 1
    scales = torch.zeros(1, 16, dtype=torch.uint8)
    scales[0, 0], scales[0, 4] = 128, 125  # blocks 0 and 1
    v = decoded(data, scales, 64, 4)
    assert v[0, 0] == -2.0 and v[0, 1] == 12.0 and v[0, 32] == 0.125 and v.abs().sum() == 14.125
    x = torch.tensor([[0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9]])
    assert held(x, 4).tolist() == [[0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0,
                                    6.0]]
    assert held(torch.tensor([[256.0, 449.0, 17.0, 19.0, 2.0 ** -10, 3 * 2.0 ** -10]]), 8).tolist() == [
        [256.0, 448.0, 16.0, 20.0, 0.0, 2.0 ** -8]]
