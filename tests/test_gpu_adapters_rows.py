"""Rows of the adapters' operator that lie in blocks with others, and the longest ones."""
import numpy as np
import pytest
import torch

from cellerator_b200 import ops

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
