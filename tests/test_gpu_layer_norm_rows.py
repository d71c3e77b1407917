"""Rows of the layer norm, forward, that its other tests do not reach: rows of one value and rows far from zero, blocks that take several
wide rows, activations and odd places of wide and of the longest rows.

Bounds.  U = 2^-24.  With m a row's mean, A the mean of |x - m| and v its variance with eps: every value's distance is taken from a number
c, which is one of the row's values (up to 1,024 columns) or the mean of four neighbouring ones (above).  With B the largest |x - m|, or
|mean of four - m|, mean|x - c| <= A + B and mean (x - c)^2 <= 2 v + 2 B^2.  (Narrow rows of 16 bits take it from a first mean, which is off
by 33 U mean|x| as in norm_forward: the larger of the two stands for B.)  A distance has one rounding, a thread's sum of them at most K: 16
pairs and their sum in narrow rows, 18 in rows that stay in registers, 64 in the longest.  Then own * (c - first) + moved has two roundings
of at most 2 B and itself, 5 shuffles, a product with the reciprocal of the count, and the same again over the warps: less than 16
roundings of A + B and 20 of 2 B.  The warps' means and the row's are rounded, U |m| each.  So the mean is off by
    e = U (3 |m| + (K + 16) (A + B) + 40 B),
u by e / sigma, a rounding of |x - m| and what its deviation is off.  The squares are K fused sums of distances that have a rounding each,
U (K + 3) (2 v + 2 B^2), less what the thread's mean takes off (at most as much: three roundings more), then 5 + 5 shuffles and two products;
the thread's and the warps' distances from the mean are off by e, which makes at most 2 e / sigma of v and (e / sigma)^2; the reciprocal
root takes half of all that relative to v, rsqrtf 2 U, the sum with eps U / 2."""
import pytest
import torch

from cellerator_b200 import ops
from row_operators import U, act, assert_within, keep, matrix

pytestmark = pytest.mark.gpu


def expected(x, gamma, beta, eps, kind, factor):
    """(y, stats) and their bounds, float64"""
    rows, cols = x.shape
    m = x.mean(1, keepdim=True)
    centred = x - m
    v = centred.square().mean(1, keepdim=True) + eps
    rstd = v.rsqrt()
    u = centred * rstd
    z = u * gamma + beta
    y = act(z, kind) * factor
    spread = centred.abs().mean(1, keepdim=True)
    whole = cols // 4 * 4
    far = (centred if cols <= 1024 else centred[:, :whole].reshape(rows, -1, 4).mean(2)).abs().amax(1, keepdim=True)
    far = torch.maximum(far, 33 * U * x.abs().mean(1, keepdim=True)) if cols <= 1024 else far
    chain = 17 if cols <= 1024 else 19 if cols <= 36_864 else 65
    e_mean = U * (3 * m.abs() + (chain + 16) * (spread + far) + 40 * far)
    shift = e_mean * rstd
    e_var = 2 * U * (chain + 24) * (2 * v + 2 * far.square()) / v + 2 * shift + shift.square()
    e_rstd = 0.5 * e_var + 3 * U
    e_u = shift + u.abs() * (e_rstd + 2 * U)
    e_z = gamma.abs() * e_u + 2 * U * ((gamma * u).abs() + z.abs())
    bound = factor * (1.13 * e_z + (20 * U * z.abs() if kind.startswith("gelu") else 0.0) + 3 * U * act(z, kind).abs())
    return y, torch.cat([m, rstd], 1), bound, torch.cat([e_mean, rstd * e_rstd], 1)


def parameters(cols, device, seed):
    return matrix(1, cols, torch.float32, device, seed, 0.3, 1.0)[0], matrix(1, cols, torch.float32, device, seed + 1, 0.3, 0.1)[0]


def check(x, gamma, beta, kind="none", p=0.0, out_dtype=None, eps=1e-5, **more):
    rows, cols = x.shape
    stats = torch.full((rows, 2), float("nan"), device=x.device)
    y = ops.layer_norm(x, gamma, beta, eps, epilogue=kind, dropout=p, seed=5, sequence=9, out_dtype=out_dtype, stats=stats, **more)
    step = max(1, 16_000_000 // cols)
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        factor = keep(hi - lo, cols, p, 5, 9, lo, x.device).double() / (1 - p) if p > 0.0 else torch.ones((), dtype=torch.float64, device=x.device)
        want, want_stats, bound, stats_bound = expected(x[lo:hi].double(), gamma.double(), beta.double(), eps, kind, factor)
        assert_within(y[lo:hi], want, bound, y.dtype, f"y from row {lo}")
        assert_within(stats[lo:hi], want_stats, stats_bound, name=f"stats from row {lo}")
    return y, stats


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [1, 3, 7, 37, 50, 64, 100, 333, 700, 1000, 1024, 1025, 2049, 5000, 16_386, 33_538, 36_864, 36_868, 40_001])
def test_rows_of_one_value(cuda_device, cols, dtype):
    """... are beta, whatever the value: its mean is the value, nothing differs from it.  A third of all values, summed up and divided by the
    count, come out as one of their neighbours."""
    g = torch.Generator().manual_seed(cols)
    values = (torch.randn(200, generator=g, dtype=torch.float64) * 10 ** (torch.rand(200, generator=g, dtype=torch.float64) * 8 - 4)).to(dtype)
    values[:6] = torch.tensor([1e4, -3e4, 1e-3, 0.0, 12345.678, 0.1], dtype=torch.float64).to(dtype)
    assert torch.isfinite(values).all()
    x = values.to(cuda_device)[:, None].repeat(1, cols)
    gamma, beta = parameters(cols, cuda_device, 5)
    stats = torch.empty(200, 2, device=cuda_device)
    y = ops.layer_norm(x, gamma, beta, out_dtype=torch.float32, stats=stats)
    assert torch.equal(stats[:, 0], x[:, 0].float())
    assert torch.equal(y, beta.repeat(200, 1))
    # nothing of dy is lost to them: u is 0, so that dx = rstd (h - mean h), h = gamma dy, whose sum is off by 60 U of |h| at most
    dy = matrix(200, cols, torch.float32, cuda_device, 6)
    dx, dgamma, _ = ops.layer_norm_backward(x, dy, stats, gamma, beta, dx_dtype=torch.float32)
    assert not dgamma.any()
    h = dy.double() * gamma.double()
    rstd = stats[:, 1:].double()
    assert_within(dx, rstd * (h - h.mean(1, keepdim=True)), rstd * U * (4 * h.abs() + 64 * h.abs().mean(1, keepdim=True)), name="dx")


@pytest.mark.parametrize("cols", [37, 50, 64, 100, 700, 1000, 1025, 2049, 5000, 16_386, 33_538, 40_001])
@pytest.mark.parametrize("far", [100.0, -3e4])
def test_rows_far_from_zero(cuda_device, cols, far):
    x = matrix(90, cols, torch.float32, cuda_device, 7, 1.0, far)
    gamma, beta = parameters(cols, cuda_device, 8)
    check(x, gamma, beta)
