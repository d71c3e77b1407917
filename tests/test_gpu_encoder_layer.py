"""The first layer of an encoder as a program runs it: the shared projection, the requests' adapters on top, layer norm with its
activation and dropout; then back: the gradients of gamma and beta, and through the transposed projection that of W."""
import numpy as np
import pytest
import torch

from cellerator_b200 import capi, ops
from conftest import random_csr
from gpu_util import host_pack, to_dev
from row_operators import act, act_slope, keep

pytestmark = pytest.mark.gpu


def layer(x, w, adapter, down, up, gamma, beta, stats, kind, p):
    y = ops.spmm_forward(x, w)
    if adapter is not None:
        ops.adapter_forward(x, adapter, down, up, out=y, beta=1.0)
    return y, ops.layer_norm(y, gamma, beta, epilogue=kind, dropout=p, seed=17, sequence=4, stats=stats, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("n", [32, 50])
@pytest.mark.parametrize("with_adapters", [True, False])
def test_layer_forward_and_backward(cuda_device, oracle, n, with_adapters):
    """Against autograd in 64 bits.  Tolerances: the projection's is 1e-4 of ||row||_1 max|W| (its own tests'; observed 1e-6), and what
    follows is Lipschitz in it; here every comparison is relative to the largest value of the result, 1e-4, and half a step of bf16
    (2^-9 of twice the value) for y."""
    rows, genes, p, kind = 300, 500, 0.2, "gelu_erf"
    rng = np.random.default_rng(n)
    c = host_pack(oracle, random_csr(rng, rows=rows, cols=genes, max_nnz=200, bits=8, empty_rows=False))
    x = to_dev(c, cuda_device)
    g = torch.Generator().manual_seed(n)
    w = (torch.randn(genes, n, generator=g) * 0.05).to(cuda_device)
    gamma, beta = (torch.randn(n, generator=g) * 0.2 + 1).to(cuda_device), (torch.randn(n, generator=g) * 0.2).to(cuda_device)
    down, up = (torch.randn(4, genes, 8, generator=g) * 0.05).to(cuda_device), (torch.randn(4, 8, n, generator=g) * 0.2).to(cuda_device)
    adapter = torch.from_numpy(rng.integers(-1, 4, rows)).int().to(cuda_device) if with_adapters else None
    dy = torch.randn(rows, n, generator=g).to(cuda_device)
    stats = torch.empty(rows, 2, device=cuda_device)
    hidden, y = layer(x, w, adapter, down, up, gamma, beta, stats, kind, p)
    dh, dgamma, dbeta = ops.layer_norm_backward(hidden, dy, stats, gamma, beta, epilogue=kind, dropout=p, seed=17, sequence=4)
    dw = ops.spmm_transpose(x, dh)

    dec = oracle.unpack_csr(8, 1, c["row_ptr"], c["packed_row_ptr"], c["col_idx"], c["scales"], c["offsets"], c["packed"])
    dense = np.zeros((rows, genes))
    dense[np.repeat(np.arange(rows), np.diff(c["row_ptr"])), c["col_idx"]] = dec
    dense = torch.from_numpy(dense).to(cuda_device)
    leaves = [t.double().requires_grad_() for t in (w, gamma, beta)]
    h = dense @ leaves[0]
    if with_adapters:
        mine = adapter.long().clamp(min=0)
        low = torch.einsum("rg,rgk->rk", dense, down.double()[mine])
        h = h + torch.where((adapter >= 0)[:, None], torch.einsum("rk,rkn->rn", low, up.double()[mine]), 0.0)
    u = (h - h.mean(1, keepdim=True)) / (h.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    want = act(u * leaves[1] + leaves[2], kind) * keep(rows, n, p, 17, 4, device=cuda_device).double() / (1 - p)
    want.backward(dy.double())
    want = want.detach()
    assert float((y.double() - want).abs().max()) <= 1e-4 * float(want.abs().max()) + 2.0 ** -8 * float(want.abs().max())
    for got, leaf in zip((dw, dgamma, dbeta), leaves):
        assert float((got.double() - leaf.grad).abs().max()) <= 1e-4 * float(leaf.grad.abs().max())


def test_layer_in_a_graph(cuda_device, oracle):
    """The whole step captured once and replayed gives the bits of the eager calls."""
    rng = np.random.default_rng(3)
    rows, genes, n = 200, 400, 64
    x = to_dev(host_pack(oracle, random_csr(rng, rows=rows, cols=genes, max_nnz=100, bits=8)), cuda_device)
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(genes, n, generator=g) * 0.05).to(cuda_device)
    gamma, beta = torch.ones(n, device=cuda_device), torch.zeros(n, device=cuda_device)
    down, up = (torch.randn(2, genes, 8, generator=g) * 0.05).to(cuda_device), torch.randn(2, 8, n, generator=g).to(cuda_device)
    adapter = (torch.arange(rows) % 3 - 1).int().to(cuda_device)
    dy = torch.randn(rows, n, generator=g).to(cuda_device)
    op = ops.PreparedSpmm(capi.PROJECTION_CSR, rows, genes, n, x.nnz, 8, 1, torch.float32, cuda_device)
    hidden, stats, y = torch.empty(rows, n, device=cuda_device), torch.empty(rows, 2, device=cuda_device), torch.empty(rows, n, device=cuda_device)
    dh, dgamma, dbeta = torch.empty(rows, n, device=cuda_device), torch.empty(n, device=cuda_device), torch.empty(n, device=cuda_device)
    workspace = torch.empty(ops.layer_norm_backward_workspace(rows, n), dtype=torch.uint8, device=cuda_device)
    kw = dict(epilogue="gelu_tanh", dropout=0.1, seed=2, sequence=6)

    def step():
        op.run(x, w, hidden)
        ops.adapter_forward(x, adapter, down, up, out=hidden, beta=1.0)
        ops.layer_norm(hidden, gamma, beta, out=y, stats=stats, **kw)
        ops.dropout(y, 0.3, seed=2, sequence=7, out=y)
        ops.dropout(dy, 0.3, seed=2, sequence=7, out=dh)
        ops.layer_norm_backward(hidden, dh, stats, gamma, beta, dx=dh, dgamma=dgamma, dbeta=dbeta, workspace=workspace, **kw)

    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(stream):
        step()
        want = [t.clone() for t in (hidden, y, dh, dgamma, dbeta)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for t in (hidden, y, dh, dgamma, dbeta, stats):
            t.fill_(float("nan"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip((hidden, y, dh, dgamma, dbeta), want))
    torch.cuda.current_stream(cuda_device).wait_stream(stream)
