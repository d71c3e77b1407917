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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [3, 50, 64, 512, 1000, 1025, 2049, 5000, 16_386, 33_538, 36_868, 40_001])
def test_rows_with_a_huge_value(cuda_device, cols, dtype):
    """One value whose square is no number of fp32, first, in the middle, in a thread's first four or last: the variance is infinite, 1 / sigma
    zero, the row beta, and the mean the value's share.  Two of 3e38 have an infinite sum: their row is NaN, its neighbours are not."""
    values = [1e20, -1e30, 2e33, 1e34, -3e36, 3.3e38, float(torch.finfo(dtype).min)]
    places = sorted({0, 1 % cols, 2, cols // 2, cols - 1})
    x = matrix(len(values) * len(places) + 3, cols, dtype, cuda_device, 21)
    x[-2, :2] = 3e38
    for i, value in enumerate(values):
        for k, place in enumerate(places):
            x[i * len(places) + k, place] = value
    gamma, beta = parameters(cols, cuda_device, 22)
    stats = torch.empty(len(x), 2, device=cuda_device)
    y = ops.layer_norm(x, gamma, beta, out_dtype=torch.float32, stats=stats)
    assert torch.equal(y[:-3], beta.repeat(len(x) - 3, 1)) and not stats[:-3, 1].any()
    want = x[:-3].double().mean(1)
    assert bool(((stats[:-3, 0].double() - want).abs() <= 64 * U * x[:-3].double().abs().amax(1)).all())
    assert torch.isnan(y[-2]).all()
    for row in (-3, -1):
        assert torch.equal(y[row], ops.layer_norm(x[row:][:1].clone(), gamma, beta, out_dtype=torch.float32)[0]) and torch.isfinite(y[row]).all()


@pytest.mark.parametrize("kind,p", [("none", 0.0), ("relu", 0.0), ("gelu_erf", 0.2), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols,rows", [(1025, 2600), (2048, 1300), (2049, 1300), (4001, 700), (9000, 500), (16_384, 470), (16_386, 460), (24_576, 450), (24_577, 460), (33_538, 600),
                                       (36_864, 450), (36_865, 620), (40_002, 620), (65_535, 600)])
def test_blocks_that_take_several_rows(cuda_device, cols, rows, dtype, kind, p):
    """At least three rows for a block, whose next one is loaded, or asked for, while one is worked on: each of them against the
    definition, and with the bits that it has in shards of fewer rows than there are blocks."""
    x = matrix(rows, cols, dtype, cuda_device, cols, 1.5, 0.25)
    x[rows // 2:] -= 3.0                                            # the rows of a block are not alike
    gamma, beta = parameters(cols, cuda_device, cols + 1)
    y, stats = check(x, gamma, beta, kind, p, out_dtype=torch.float32)
    for lo in range(0, rows, 140):
        hi = min(rows, lo + 140)
        some = torch.empty(hi - lo, 2, device=cuda_device)
        assert torch.equal(ops.layer_norm(x[lo:hi], gamma, beta, epilogue=kind, dropout=p, seed=5, sequence=9, first_row=lo, out_dtype=torch.float32, stats=some), y[lo:hi])
        assert torch.equal(some, stats[lo:hi])


@pytest.mark.parametrize("kind", ["none", "relu", "gelu_erf", "gelu_tanh"])
@pytest.mark.parametrize("cols,pitch,shift", [(1237, 1240, 1), (9001, 9001, 0), (33_538, 33_539, 1), (36_601, 36_601, 0), (36_867, 36_867, 3), (36_870, 36_872, 2), (40_001, 40_004, 0),
                                              (65_533, 65_536, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_odd_places_of_wide_rows(cuda_device, cols, pitch, shift, dtype, kind):
    """Rows of any width that start anywhere, parameters that start on no 16-byte boundary, one of them or none; what lies between the rows
    stays as it was."""
    x = matrix(9, cols, dtype, cuda_device, 11, 2.0, 0.5, pitch, shift)
    buffer = matrix(1, 2 * cols + 3, torch.float32, cuda_device, 12, 0.3, 0.5)[0]
    out = matrix(9, cols, dtype, cuda_device, 13, pitch=pitch, shift=shift)
    one, zero = torch.ones(cols, device=cuda_device), torch.zeros(cols, device=cuda_device)
    around = out._base.clone()
    for gamma, beta in ((buffer[1:cols + 1], buffer[cols + 2:2 * cols + 2]), (buffer[:cols], None), (None, buffer[3:cols + 3]), (None, None)):
        stats = torch.full((9, 2), float("nan"), device=cuda_device)
        ops.layer_norm(x, gamma, beta, epilogue=kind, dropout=0.1, seed=5, sequence=9, out=out, stats=stats)
        factor = keep(9, cols, 0.1, 5, 9, device=cuda_device).double() / 0.9
        want, want_stats, bound, stats_bound = expected(x.double(), (one if gamma is None else gamma).double(), (zero if beta is None else beta).double(), 1e-5, kind, factor)
        assert_within(out, want, bound, dtype, "y")
        assert_within(stats, want_stats, stats_bound, name="stats")
    out.copy_(around[shift:shift + 9 * pitch].view(9, pitch)[:, :cols])
    assert torch.equal(out._base.view(torch.uint8), around.view(torch.uint8))


@pytest.mark.parametrize("rows,cols,dtype", [(3_000_000, 50, torch.float32), (400_000, 512, torch.bfloat16), (120_000, 2000, torch.bfloat16), (40_000, 4608, torch.float16)])
def test_gradients_of_parameters_over_many_rows(cuda_device, rows, cols, dtype):
    """Threads that add up the terms of hundreds of rows.  There are at least 148 blocks, so that no chain is longer than a 148th of the rows,
    and 64 steps more join them; terms themselves are off as in norm_backward (row_operators.py): u by 2 U |u|, a product by U.  dy and the
    terms of dgamma are not centred, so that the sums are of the size of their terms' sum."""
    x = torch.randn(rows, cols, generator=torch.Generator(device=cuda_device).manual_seed(1), device=cuda_device).to(dtype)
    dy = x.abs() + 0.25 * x                                         # dz u = |x| u + x u / 4
    gamma, beta = parameters(cols, cuda_device, 15)
    stats = torch.empty(rows, 2, device=cuda_device)
    ops.layer_norm(x, gamma, beta, stats=stats)
    _, dgamma, dbeta = ops.layer_norm_backward(x, dy, stats, gamma, beta, dx=dy.clone())
    sums = [torch.zeros(cols, dtype=torch.float64, device=cuda_device) for _ in range(4)]
    step = 32_000_000 // cols
    for lo in range(0, rows, step):
        s, d = stats[lo:lo + step].double(), dy[lo:lo + step].double()
        terms = d * ((x[lo:lo + step].double() - s[:, :1]) * s[:, 1:])
        for total, t in zip(sums, (terms, terms.abs(), d, d.abs())):
            total += t.sum(0)
    chain = rows / 148 + 64
    assert_within(dgamma, sums[0], (chain + 4) * U * sums[1], name="dgamma")
    assert_within(dbeta, sums[2], (chain + 1) * U * sums[3], name="dbeta")
