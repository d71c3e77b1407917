"""Rows of the adapters' operator that lie in blocks with others, and the longest ones."""
import numpy as np
import pytest
import torch

from cellerator_b200 import ops
from gpu_util import host_pack, to_dev
from row_operators import assert_within
from test_gpu_adapters import decoded, expected, weights

pytestmark = pytest.mark.gpu


def test_the_longest_row(cuda_device):
    """2^31 - 1 entries between two short rows.  Codes are 1 in one of 2,048 places, else 0, scales 1, A and B small whole numbers: every
    sum is a whole number below 2^24, so that the results are equal and not near."""
    length, genes, rank, n = 2 ** 31 - 1, 5, 4, 3
    g = torch.Generator(device=cuda_device).manual_seed(3)
    nnz = length + 7
    col = torch.randint(0, genes, (nnz,), generator=g, device=cuda_device, dtype=torch.int32)
    codes = torch.empty(nnz, dtype=torch.uint8, device=cuda_device)
    counts = torch.zeros(3, genes, dtype=torch.int64, device=cuda_device)
    edges = [0, 3, 3 + length, nnz]
    step = 1 << 27
    for lo in range(0, nnz, step):
        hi = min(nnz, lo + step)
        codes[lo:hi] = torch.randint(0, 2048, (hi - lo,), generator=g, device=cuda_device, dtype=torch.int16) == 0
    codes[-1] = codes[3 + length - 1] = codes[0] = 1              # the first place of the first row, the last of the others
    for row in range(3):
        for lo in range(edges[row], edges[row + 1], step):
            hi = min(edges[row + 1], lo + step)
            counts[row] += torch.bincount(col[lo:hi][codes[lo:hi] > 0], minlength=genes)
    down = torch.randint(1, 3, (1, genes, rank), generator=g, device=cuda_device).float()
    up = torch.randint(1, 3, (1, rank, n), generator=g, device=cuda_device).float()
    want = counts.double() @ down[0].double() @ up[0].double()
    assert float(want.max()) < 2 ** 24
    x = ops.QuantizedCsr(3, genes, 8, 1, torch.tensor(edges, device=cuda_device), col, codes, torch.ones(genes, device=cuda_device), torch.zeros(genes, device=cuda_device))
    got = ops.adapter_forward(x, torch.zeros(3, dtype=torch.int32, device=cuda_device), down, up)
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("rank,dtype", [(8, torch.float32), (16, torch.bfloat16), (12, torch.bfloat16), (5, torch.float32)])
@pytest.mark.parametrize("bits", [8, 4])
def test_rows_that_share_a_block(cuda_device, oracle, bits, rank, dtype):
    """3,000 rows of 70 entries on average: eight rows to a block, long, empty and short ones side by side and some without an adapter.  Each
    has the bits of the row alone, a block to itself, and is within the bound of the definition."""
    rng = np.random.default_rng(rank)
    rows, genes, n = 3000, 2500, 30
    lengths = rng.integers(0, 90, rows)
    lengths[rng.integers(0, rows, 300)] = 0
    lengths[::97] = rng.integers(800, genes, len(lengths[::97]))
    lengths[5], lengths[-1] = genes, 1
    row_ptr = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    assert row_ptr[-1] / rows * 8 <= 8192 and rows >= 4 * 148 * 4   # what a launch asks for before it takes eight rows to a block
    col = np.concatenate([np.sort(rng.permutation(genes)[:k]) for k in lengths]).astype(np.int32)
    c = host_pack(oracle, dict(rows=rows, cols=genes, bits=bits, policy=1, row_ptr=row_ptr, col_idx=col, scales=rng.uniform(0.01, 0.5, genes).astype(np.float32),
                               offsets=rng.uniform(-1, 1, genes).astype(np.float32), values=rng.uniform(-2, 40, len(col)).astype(np.float32)))
    down, up, scale = weights(5, genes, rank, n, dtype, cuda_device, rank)
    adapter = torch.from_numpy(rng.integers(-1, 5, rows)).int()
    x, on_device = to_dev(c, cuda_device), adapter.to(cuda_device)
    before = torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    whole = before.clone()
    ops.adapter_forward(x, on_device, down, up, scale, out=whole, beta=1.0)
    alone = before.clone()
    for lo in range(0, rows, 500):                                  # fewer than two rows to a block ask for: each has one to itself
        ops.adapter_forward(x, on_device, down, up, scale, out=alone, beta=1.0, row_begin=lo, row_end=min(rows, lo + 500))
    assert torch.equal(whole, alone)
    dense, size = decoded(oracle, c)
    want, bound = expected(dense, size, adapter, down, up, scale, beta=1.0, before=before.double().cpu())
    # rows of up to 2,500 entries: parts of 128, whose sums a lane group makes entry by entry at worst, 20 parts
    assert_within(whole.cpu(), want, bound, name="out")
    again = before.clone()
    ops.adapter_forward(x, on_device, down, up, scale, out=again, beta=1.0)
    assert torch.equal(again, whole)
