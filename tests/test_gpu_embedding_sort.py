"""GPU: the sort of embedding gradients at the width of its keys: 32 bits below 2^19 rows, 64 from there on, each with
tokens that one tile holds (up to 8192) and with more."""
import pytest
import torch

from neuzip_amd import ops
from mx_oracle import round_to

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("rows", ((1 << 19) - 1, 1 << 19, 600_000, 3_000_000))
@pytest.mark.parametrize("count,cols", [(2049, 4), (4096, 8), (5000, 8), (8191, 4), (8192, 4), (8193, 4), (20000, 2)])
def test_keys_of_both_widths(rows, count, cols):
    """Tokens of few rows and of many, the first and the last row and indices outside (the largest key, at the end of
    a tile) among them.  Whole numbers up to 50: 20000 of them stay below 2^24."""
    g = torch.Generator().manual_seed(count + rows)
    ids = torch.randint(0, rows, (count,), generator=g)
    ids[::3] = torch.randint(rows - 5, rows, (len(ids[::3]),), generator=g)
    ids[1::5] = torch.randint(0, 40, (len(ids[1::5]),), generator=g)
    ids[::11] = rows
    ids[-1], ids[count // 2], ids[7] = -1, rows + 3, rows - 1
    grad = torch.randint(-50, 51, (count, cols), generator=g).float()
    for skip in (None, rows - 2):
        kept = (ids >= 0) & (ids < rows) & (ids != (-1 if skip is None else skip))
        want = torch.zeros(rows, cols, dtype=torch.float64).index_add_(0, ids[kept], grad[kept].double())
        for dtype in (torch.float32, torch.bfloat16):
            got = ops.embedding_gradient(ids.to(DEV), grad.to(dtype).to(DEV), rows, padding_idx=skip)
            assert torch.equal(got.cpu(), round_to(want, dtype))
