"""Adapters of many requests on the device against the definition in 64 bits.

Bound: a part of a row (128 entries, or a 32nd of the row rounded up to whole 128s) is summed by lane groups, at worst one group
entry by entry, in segments of 128; then 5 shuffles and up to 32 parts.  With rows below 4,096 entries that is 128 + 5 + 32 = 165
roundings of the sum of magnitudes, U = 2^-24 each, and one of the decoded value; the second product has rank + 1 roundings, the
factors alpha, scale, beta and the epilogue's sums less than 8 more."""
import numpy as np
import pytest
import torch

from cellerator_b200 import ops
from conftest import random_csr
from gpu_util import host_pack, rows_of, to_dev
from row_operators import U, act, assert_within

pytestmark = pytest.mark.gpu


def decoded(oracle, c):
    """The matrix in float64, entries of a gene that a row holds twice added up and genes outside left out, and the same of
    magnitudes."""
    codes = oracle.extract_codes(c["bits"], c["row_ptr"], c["packed_row_ptr"], c["packed"]).astype(np.float64)
    row, gene = np.repeat(np.arange(c["rows"]), np.diff(c["row_ptr"])), np.clip(c["col_idx"], 0, c["cols"] - 1)
    dec = codes * c["scales"].astype(np.float64)[gene] + c["offsets"].astype(np.float64)[gene if c["policy"] == 1 else row]
    inside = (c["col_idx"] >= 0) & (c["col_idx"] < c["cols"])
    x, size = np.zeros((c["rows"], c["cols"])), np.zeros((c["rows"], c["cols"]))
    np.add.at(x, (row[inside], gene[inside]), dec[inside])
    np.add.at(size, (row[inside], gene[inside]), np.abs(dec[inside]))
    return torch.from_numpy(x), torch.from_numpy(size)


def weights(adapters, genes, rank, n, dtype, device, seed):
    g = torch.Generator().manual_seed(seed)
    down = (torch.randn(adapters, genes, rank, generator=g) * 0.1).to(dtype)
    up = (torch.randn(adapters, rank, n, generator=g) * 0.2).to(dtype)
    return down.to(device), up.to(device), (torch.rand(adapters, generator=g) + 0.5).to(device)


def expected(x, size, adapter, down, up, scale, alpha=1.0, beta=0.0, before=None, kind="none", bias=None):
    """(result, bound) in 64 bits"""
    rows, n, rank = x.shape[0], up.shape[2], up.shape[1]
    y, bound = torch.zeros(rows, n, dtype=torch.float64), torch.zeros(rows, n, dtype=torch.float64)
    down, up = down.double().cpu(), up.double().cpu()
    for a in range(down.shape[0]):
        mine = adapter == a
        s = abs(alpha) * (1.0 if scale is None else float(scale[a]))
        hidden, magnitude = x[mine] @ down[a], size[mine] @ down[a].abs()
        y[mine] = (s if alpha >= 0 else -s) * (hidden @ up[a])
        bound[mine] = s * U * ((166 * magnitude) @ up[a].abs() + (rank + 5) * (hidden.abs() @ up[a].abs()))
    if beta != 0.0:
        y = y + beta * before
        bound = bound + 4 * U * (y.abs() + (beta * before).abs())
    if bias is not None:
        y = y + bias.double()
        bound = bound + 4 * U * (y.abs() + bias.double().abs())
    out = act(y, kind)
    return out, 1.13 * bound + 20 * U * out.abs() + 20 * U * y.abs() * (kind != "none")


def case(oracle, rows, cols, most, bits, policy, seed):
    rng = np.random.default_rng(seed)
    return host_pack(oracle, random_csr(rng, rows=rows, cols=cols, max_nnz=most, bits=bits, policy=policy))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits,policy", [(8, 1), (4, 1), (8, 2), (4, 2)])
@pytest.mark.parametrize("rank,n", [(8, 32), (16, 64), (1, 7), (4, 50), (5, 33), (12, 100), (32, 128), (64, 1), (33, 300), (128, 64), (256, 16)])
def test_against_the_definition(cuda_device, oracle, rank, n, bits, policy, dtype):
    c = case(oracle, 37, 600, 400, bits, policy, rank + n)
    down, up, scale = weights(5, 600, rank, n, dtype, cuda_device, rank)
    adapter = torch.from_numpy(np.random.default_rng(rank).integers(-1, 5, 37)).int()
    got = ops.adapter_forward(to_dev(c, cuda_device), adapter.to(cuda_device), down, up, scale)
    assert_within(got.cpu(), *expected(*decoded(oracle, c), adapter, down, up, scale), name="out")


@pytest.mark.parametrize("rows,cols,most", [(1, 1, 1), (1, 5000, 4000), (3, 4000, 4000), (200, 64, 3), (50, 2000, 129)])
def test_row_lengths(cuda_device, oracle, rows, cols, most):
    c = case(oracle, rows, cols, most, 8, 1, rows)
    down, up, scale = weights(3, cols, 16, 40, torch.float32, cuda_device, 1)
    adapter = torch.arange(rows).int() % 3
    got = ops.adapter_forward(to_dev(c, cuda_device), adapter.to(cuda_device), down, up)
    assert_within(got.cpu(), *expected(*decoded(oracle, c), adapter, down, up, None), name="out")


@pytest.mark.parametrize("lengths", [[0, 1, 127, 128, 129, 0, 255, 256, 257, 4000, 0], [0], [5000, 5000]])
@pytest.mark.parametrize("bits", [8, 4])
def test_lengths_next_to_the_parts(cuda_device, oracle, lengths, bits):
    """... and rows without an entry, whose product is zero.  5,000 entries: parts of 256, two segments in turn; 128 more roundings."""
    rng = np.random.default_rng(len(lengths))
    row_ptr = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    genes = 6000
    col = np.concatenate([np.sort(rng.choice(genes, k, replace=False)) for k in lengths] + [np.zeros(0, int)]).astype(np.int32)
    c = host_pack(oracle, dict(rows=len(lengths), cols=genes, bits=bits, policy=1, row_ptr=row_ptr, col_idx=col, scales=rng.uniform(0.01, 0.5, genes).astype(np.float32),
                               offsets=rng.uniform(-1, 1, genes).astype(np.float32), values=rng.uniform(-2, 40, len(col)).astype(np.float32)))
    down, up, scale = weights(2, genes, 16, 64, torch.bfloat16, cuda_device, 2)
    adapter = (torch.arange(len(lengths)) % 2).int()
    got = ops.adapter_forward(to_dev(c, cuda_device), adapter.to(cuda_device), down, up, scale)
    want, bound = expected(*decoded(oracle, c), adapter, down, up, scale)
    assert_within(got.cpu(), want, bound * (294 / 166), name="out")
    assert not got[[i for i, k in enumerate(lengths) if k == 0]].any()


@pytest.mark.parametrize("kind", ["none", "bias", "relu", "gelu_erf", "gelu_tanh", "bias_relu", "bias_gelu_erf", "bias_gelu_tanh"])
def test_epilogue_alpha_beta(cuda_device, oracle, kind):
    c = case(oracle, 40, 300, 100, 8, 1, 7)
    down, up, scale = weights(4, 300, 8, 50, torch.float32, cuda_device, 3)
    adapter = torch.from_numpy(np.random.default_rng(7).integers(-1, 4, 40)).int()
    bias = torch.randn(50, generator=torch.Generator().manual_seed(1)) if "bias" in kind else None
    before = torch.randn(40, 50, generator=torch.Generator().manual_seed(2))
    activation = kind.replace("bias_", "").replace("bias", "none")
    for alpha, beta in ((1.0, 0.0), (-0.5, 1.0), (2.0, -0.25)):
        out = before.to(cuda_device) if beta else torch.full((40, 50), float("nan"), device=cuda_device)
        ops.adapter_forward(to_dev(c, cuda_device), adapter.to(cuda_device), down, up, scale, out=out, alpha=alpha, beta=beta, epilogue=kind,
                            bias=None if bias is None else bias.to(cuda_device))
        want, bound = expected(*decoded(oracle, c), adapter, down, up, scale, alpha, beta, before.double(), activation, bias)
        assert_within(out.cpu(), want, bound, name=kind)


def test_rows_without_an_adapter(cuda_device, oracle):
    """-1 and indices outside: out is beta times what it was, bit for bit with beta = 1, and zero with beta = 0; A and B are not read."""
    c = case(oracle, 20, 200, 50, 8, 1, 9)
    x = to_dev(c, cuda_device)
    down, up, scale = weights(2, 200, 8, 16, torch.float32, cuda_device, 4)
    down.fill_(float("nan"))
    adapter = torch.tensor([-1, 2, 2 ** 31 - 1, -2 ** 31] * 5, dtype=torch.int32, device=cuda_device)
    before = torch.randn(20, 16, device=cuda_device)
    out = before.clone()
    ops.adapter_forward(x, adapter, down, up, scale, out=out, beta=1.0)
    assert torch.equal(out, before)
    ops.adapter_forward(x, adapter, down, up, scale, out=out)
    assert torch.equal(out, torch.zeros_like(out))
    none = ops.adapter_forward(x, torch.full((20,), -1, dtype=torch.int32, device=cuda_device), down[:0], up[:0])
    assert torch.equal(none, torch.zeros_like(none))


def test_genes_outside_and_twice(cuda_device, oracle):
    """A gene outside the matrix is left out, a gene that a row holds twice counts twice, and infinities in rows of A that no
    entry names reach no result."""
    c = case(oracle, 12, 100, 60, 8, 2, 11)
    start, end = c["row_ptr"][3], c["row_ptr"][4]
    assert end - start > 6
    c["col_idx"][start], c["col_idx"][end - 1], c["col_idx"][start + 2] = -7, 100, c["col_idx"][start + 1]
    down, up, scale = weights(2, 100, 8, 16, torch.float32, cuda_device, 5)
    c["col_idx"][c["col_idx"] == 0] = 1
    down[:, 0] = float("inf")
    adapter = torch.arange(12).int() % 2
    got = ops.adapter_forward(to_dev(c, cuda_device), adapter.to(cuda_device), down, up, scale)
    finite = down.clone()
    finite[:, 0] = 0.0
    assert_within(got.cpu(), *expected(*decoded(oracle, c), adapter, finite, up, scale), name="out")


def test_a_rows_bits_follow_from_the_row(cuda_device, oracle):
    """The same bits alone, in a range of rows, in a matrix of its own, with another number of warps (longer neighbours) and at
    every call."""
    c = case(oracle, 60, 3000, 40, 8, 1, 13)
    rng = np.random.default_rng(14)
    long = host_pack(oracle, random_csr(rng, rows=60, cols=3000, max_nnz=2500, bits=8))
    # the first 30 rows of both in one matrix
    both = {}
    both.update(c, rows=60)
    head, tail = rows_of(c, 0, 30), rows_of(long, 0, 30)
    both["row_ptr"] = np.concatenate([head["row_ptr"], head["row_ptr"][-1] + tail["row_ptr"][1:]])
    both["packed_row_ptr"] = both["row_ptr"]
    both["col_idx"], both["packed"] = np.concatenate([head["col_idx"], tail["col_idx"]]), np.concatenate([head["packed"], tail["packed"]])
    down, up, scale = weights(3, 3000, 16, 64, torch.bfloat16, cuda_device, 6)
    adapter = (torch.arange(60) % 3).int().to(cuda_device)
    whole = ops.adapter_forward(to_dev(c, cuda_device), adapter, down, up, scale)
    assert torch.equal(ops.adapter_forward(to_dev(both, cuda_device), adapter, down, up, scale)[:30], whole[:30])
    out = torch.full_like(whole, 7.0)
    ops.adapter_forward(to_dev(c, cuda_device), adapter, down, up, scale, out=out, row_begin=11, row_end=47)
    assert torch.equal(out[11:47], whole[11:47]) and bool((out[:11] == 7.0).all()) and bool((out[47:] == 7.0).all())
    piece = rows_of(c, 20, 33)
    assert torch.equal(ops.adapter_forward(to_dev(piece, cuda_device), adapter[20:33].contiguous(), down, up, scale), whole[20:33])


@pytest.mark.parametrize("rows,genes,mean,rank,bits,dtype", [(2600, 2000, 900, 16, 8, torch.bfloat16), (1500, 33_538, 1500, 8, 4, torch.float32),
                                                             (3000, 1500, 800, 5, 8, torch.float32), (2400, 3000, 1000, 128, 4, torch.bfloat16)])
def test_large_batches(cuda_device, oracle, rows, genes, mean, rank, bits, dtype):
    """Two million entries and more, whose scales (and, of 33,538 genes, some zero-points) are kept in shared memory: against the
    definition on some rows, bit for bit what the same rows give in ranges of fewer entries, with empty rows by the hundred, rows
    without an adapter and one row that holds every gene."""
    rng = np.random.default_rng(rank)
    lengths = np.minimum(rng.lognormal(np.log(mean), 0.6, rows).astype(np.int64), genes)
    lengths[100:400] = 0
    lengths[-1] = 0
    lengths[500] = genes
    row_ptr = np.concatenate([[0], np.cumsum(lengths)])
    col = np.concatenate([np.sort(rng.permutation(genes)[:k]) for k in lengths]).astype(np.int32)
    c = host_pack(oracle, dict(rows=rows, cols=genes, bits=bits, policy=1, row_ptr=row_ptr, col_idx=col, scales=rng.uniform(0.01, 0.5, genes).astype(np.float32),
                               offsets=rng.uniform(-1, 1, genes).astype(np.float32), values=rng.uniform(-2, 40, len(col)).astype(np.float32)))
    assert len(col) // rows * rows >= 2_000_000
    x = to_dev(c, cuda_device)
    n = 40
    down, up, scale = weights(6, genes, rank, n, dtype, cuda_device, rank)
    adapter = torch.from_numpy(rng.integers(-1, 6, rows)).int()
    on_device = adapter.to(cuda_device)
    whole = ops.adapter_forward(x, on_device, down, up, scale)
    pieces = torch.full_like(whole, float("nan"))
    bounds = np.linspace(0, rows, 6).astype(int)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        ops.adapter_forward(x, on_device, down, up, scale, out=pieces, row_begin=int(lo), row_end=int(hi))
    assert torch.equal(whole, pieces)
    some = np.concatenate([np.arange(90, 110), [399, 400, 500, rows - 1], rng.integers(0, rows, 20)])
    for r in some:
        piece = rows_of(c, int(r), int(r) + 1)
        want, bound = expected(*decoded(oracle, piece), adapter[int(r):int(r) + 1], down, up, scale)
        # rows of up to 33,538 entries: parts of 1,152, nine segments in turn, eight of them more than counted
        assert_within(whole[int(r):int(r) + 1].cpu(), want, bound * ((166 + 8 * 128) / 166), name=str(r))


def test_pitch_of_the_output(cuda_device, oracle):
    c = case(oracle, 25, 200, 50, 4, 1, 15)
    down, up, scale = weights(2, 200, 8, 30, torch.float32, cuda_device, 7)
    adapter = (torch.arange(25) % 2).int().to(cuda_device)
    x = to_dev(c, cuda_device)
    wide = torch.full((25, 41), 3.0, device=cuda_device)
    ops.adapter_forward(x, adapter, down, up, scale, out=wide[:, 5:35])
    assert torch.equal(wide[:, 5:35], ops.adapter_forward(x, adapter, down, up, scale))
    assert bool((wide[:, :5] == 3.0).all()) and bool((wide[:, 35:] == 3.0).all())


def test_weights_that_start_anywhere(cuda_device, oracle):
    """Narrower loads where rows of A start on no 16-byte boundary; the sums are the same numbers in another order."""
    c = case(oracle, 25, 200, 50, 8, 1, 17)
    x, adapter = to_dev(c, cuda_device), (torch.arange(25) % 2).int()
    for dtype in (torch.float32, torch.bfloat16):
        down, up, scale = weights(2, 200, 16, 30, dtype, cuda_device, 8)
        buffer = torch.empty(down.numel() + 8, dtype=dtype, device=cuda_device)
        for shift in (0, 1, 2, 4):
            moved = buffer[shift:shift + down.numel()].view(down.shape).copy_(down)
            got = ops.adapter_forward(x, adapter.to(cuda_device), moved, up, scale)
            assert_within(got.cpu(), *expected(*decoded(oracle, c), adapter, down, up, scale), name=str(shift))


def test_adapters_behind_2_to_the_32_bytes(cuda_device, oracle):
    """The last of 140 adapters of 33,538 genes and rank 256 stands 4.77e9 bytes in."""
    c = case(oracle, 9, 33_538, 500, 8, 1, 19)
    down = torch.zeros(140, 33_538, 256, dtype=torch.float32, device=cuda_device)    # 4.8 GB
    up = torch.zeros(140, 256, 32, device=cuda_device)
    one_down, one_up, scale = weights(1, 33_538, 256, 32, torch.float32, cuda_device, 9)
    down[139], up[139] = one_down[0], one_up[0]
    x = to_dev(c, cuda_device)
    got = ops.adapter_forward(x, torch.full((9,), 139, dtype=torch.int32, device=cuda_device), down, up)
    assert torch.equal(got, ops.adapter_forward(x, torch.zeros(9, dtype=torch.int32, device=cuda_device), one_down, one_up)) and bool(got.any())


def test_graph_replay(cuda_device, oracle):
    c = case(oracle, 30, 200, 50, 8, 1, 21)
    down, up, scale = weights(3, 200, 8, 32, torch.float32, cuda_device, 10)
    adapter = torch.zeros(30, dtype=torch.int32, device=cuda_device)
    x, out = to_dev(c, cuda_device), torch.empty(30, 32, device=cuda_device)
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        ops.adapter_forward(x, adapter, down, up, scale, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.adapter_forward(x, adapter, down, up, scale, out=out)
        for a in (1, 2, -1):
            adapter.fill_(a)
            graph.replay()
            assert torch.equal(out, ops.adapter_forward(x, adapter, down, up, scale))
    torch.cuda.current_stream(cuda_device).wait_stream(stream)
