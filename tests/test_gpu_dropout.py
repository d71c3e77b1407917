"""Dropout on the device against the generator written out: which values stay and what they become, value for value.  A kept value
is x * fp32(1 / (1 - p)) rounded once to fp32 and once more to the result's type, which is computed here, so results are equal."""
import pytest
import torch

from cellerator_b200 import ops
from row_operators import keep, matrix

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def expected(x, p, seed, sequence=0, first_row=0, dtype=None):
    scale = torch.tensor(1.0 / (1.0 - p), dtype=torch.float64).float().item()
    kept = keep(x.shape[0], x.shape[1], p, seed, sequence, first_row, x.device)
    return torch.where(kept, x.float() * scale, 0.0).to(x.dtype if dtype is None else dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3), (3, 7), (64, 32), (129, 50), (1000, 1), (5, 4099), (2, 70_000), (300, 257)])
def test_values(cuda_device, rows, cols, dtype):
    x = matrix(rows, cols, dtype, cuda_device, seed=rows + cols)
    assert torch.equal(ops.dropout(x, 0.3, seed=77, sequence=5), expected(x, 0.3, 77, 5))


@pytest.mark.parametrize("pitch,shift", [(50, 0), (52, 0), (51, 1), (64, 2), (50, 1), (53, 3)])
@pytest.mark.parametrize("dtype", TYPES)
def test_pitch_and_alignment(cuda_device, pitch, shift, dtype):
    x = matrix(33, 50, dtype, cuda_device, seed=pitch, pitch=pitch, shift=shift)
    out = matrix(33, 50, dtype, cuda_device, seed=1, pitch=61, shift=shift)
    around = out._base.clone()
    ops.dropout(x, 0.5, seed=3, out=out)
    assert torch.equal(out, expected(x, 0.5, 3))
    out.copy_(around[shift:shift + 33 * 61].view(33, 61)[:, :50])            # nothing beside the matrix was written
    assert torch.equal(out._base.view(torch.uint8), around.view(torch.uint8))


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
def test_other_type(cuda_device, dtype, out_dtype):
    x = matrix(65, 36, dtype, cuda_device, seed=4)
    out = torch.empty(65, 36, dtype=out_dtype, device=cuda_device)
    assert torch.equal(ops.dropout(x, 0.2, seed=9, out=out), expected(x, 0.2, 9, dtype=out_dtype))


@pytest.mark.parametrize("p", [0.0, 1e-9, 2.0 ** -32, 0.5, 1 - 2.0 ** -33, 0.999])
def test_probabilities(cuda_device, p):
    x = matrix(200, 100, torch.float32, cuda_device, seed=5)
    got = ops.dropout(x, p, seed=2 ** 64 - 1, sequence=2 ** 63 + 5)
    assert torch.equal(got, x if p == 0.0 else expected(x, p, 2 ** 64 - 1, 2 ** 63 + 5))


def test_share_of_dropped_values(cuda_device):
    """4 million words: the share that is dropped has a standard deviation of 0.00023 at p = 0.3; six of them."""
    got = ops.dropout(torch.ones(4000, 1000, device=cuda_device), 0.3, seed=11)
    assert abs(float((got == 0).double().mean()) - 0.3) < 6 * (0.3 * 0.7 / 4e6) ** 0.5


def test_dropped_values_are_zero_whatever_they_were(cuda_device):
    kept = keep(40, 30, 0.5, 21, 0, device=cuda_device)
    for value in (float("nan"), float("inf"), -float("inf")):
        x = torch.where(kept, torch.ones((), device=cuda_device), torch.full((), value, device=cuda_device))
        got = ops.dropout(x, 0.5, seed=21)
        assert torch.equal(got, torch.where(kept, 2.0, 0.0)) and not torch.signbit(got).any()


def test_in_place_shards_and_gradient(cuda_device):
    """A shard that names its first row drops what the whole matrix drops; the gradient of ones is mask / (1 - p)."""
    x = matrix(101, 66, torch.float32, cuda_device, seed=6)
    whole = ops.dropout(x, 0.4, seed=8, sequence=3)
    parts = [ops.dropout(x[lo:hi], 0.4, seed=8, sequence=3, first_row=lo) for lo, hi in ((0, 33), (33, 34), (34, 101))]
    assert torch.equal(torch.cat(parts), whole)
    slope = ops.dropout(torch.ones_like(x), 0.4, seed=8, sequence=3)
    assert torch.equal(slope != 0, keep(101, 66, 0.4, 8, 3, device=cuda_device))
    # differences: the operator is linear, so a step along the gradient's direction changes it by exactly that
    assert torch.equal(ops.dropout(x + 1, 0.4, seed=8, sequence=3), expected(x + 1, 0.4, 8, 3))
    last = 2 ** 32 - 101
    assert torch.equal(ops.dropout(x, 0.4, seed=8, first_row=last), expected(x, 0.4, 8, 0, last))
    assert ops.dropout(x, 0.4, seed=8, sequence=3, out=x).data_ptr() == x.data_ptr() and torch.equal(x, whole)


def test_empty(cuda_device):
    assert ops.dropout(torch.empty(0, 5, device=cuda_device), 0.1, 1).shape == (0, 5)
    assert ops.dropout(torch.empty(5, 0, device=cuda_device), 0.1, 1).shape == (5, 0)


def test_graph_replay_and_other_stream(cuda_device):
    """A captured call takes the number that stands in device_sequence when it is replayed."""
    x = matrix(70, 45, torch.float32, cuda_device, seed=9)
    number = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    out = torch.empty_like(x)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        ops.dropout(x, 0.3, seed=1, sequence=10, device_sequence=number, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.dropout(x, 0.3, seed=1, sequence=10, device_sequence=number, out=out)
        for i in range(3):
            number.fill_(i)
            graph.replay()
            assert torch.equal(out, expected(x, 0.3, 1, 10 + i))
    torch.cuda.current_stream(cuda_device).wait_stream(stream)


def test_more_than_2_to_the_32_bytes(cuda_device):
    rows, cols = 33_000, 66_000                                              # 2.2e9 values
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=cuda_device)
    ops.dropout(x, 0.25, seed=4, out=x)
    for row in (0, 16_000, rows - 1):
        assert torch.equal(x[row:row + 1] != 0, keep(1, cols, 0.25, 4, 0, row, cuda_device))
