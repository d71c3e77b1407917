"""Layer norm and its gradients on the device against the formulas in 64 bits, within bounds that count fp32's roundings
(row_operators.py)."""
import pytest
import torch

from cellerator_b200 import ops
from row_operators import assert_within, keep, matrix, norm_backward, norm_forward

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one value; less than a quad; a lane; several lanes, with and without a last piece of a quad; either side of where a warp's rows end,
# backward and forward; of two and four quads to a thread, of a block's rows backward, of four, six and nine quads; the gene set; either
# side of what the registers hold; the widest
WIDTHS = [1, 2, 3, 4, 7, 16, 32, 50, 64, 100, 128, 255, 512, 513, 700, 1024, 1025, 1237, 2048, 2049, 4608, 4609, 16_384, 16_386, 24_577, 33_538, 36_864,
          36_868, 65_536]


def rows_for(cols):
    return 130 if cols <= 512 else 23 if cols <= 10_000 else 5


def parameters(cols, device, seed):
    return matrix(1, cols, torch.float32, device, seed, 0.3, 1.0)[0], matrix(1, cols, torch.float32, device, seed + 1, 0.3, 0.1)[0]


def factor_of(rows, cols, p, seed, sequence, device, first_row=0):
    if p == 0.0:
        return torch.ones((), dtype=torch.float64, device=device)
    return keep(rows, cols, p, seed, sequence, first_row, device).double() / (1 - p)


def check_forward(x, gamma, beta, eps=1e-5, kind="none", p=0.0, out_dtype=None, first_row=0, out=None):
    rows, cols = x.shape
    g = torch.ones(cols, device=x.device) if gamma is None else gamma
    b = torch.zeros(cols, device=x.device) if beta is None else beta
    factor = factor_of(rows, cols, p, 5, 9, x.device, first_row)
    want, want_stats, bound, stats_bound = norm_forward(x.double(), g.double(), b.double(), eps, kind, factor)
    stats = torch.full((rows, 2), float("nan"), device=x.device)
    y = ops.layer_norm(x, gamma, beta, eps, epilogue=kind, dropout=p, seed=5, sequence=9, first_row=first_row, out_dtype=out_dtype, stats=stats, out=out)
    assert_within(y, want, bound, y.dtype, "y")
    assert_within(stats, want_stats, stats_bound, name="stats")
    if p > 0.0:
        assert torch.equal(y != 0, (factor != 0) & (y != 0))
    return y, stats


def check_backward(x, dy, gamma, beta, kind="none", p=0.0, dx_dtype=None, eps=1e-5, stats=None, **more):
    rows, cols = x.shape
    g = torch.ones(cols, device=x.device) if gamma is None else gamma
    b = torch.zeros(cols, device=x.device) if beta is None else beta
    factor = factor_of(rows, cols, p, 5, 9, x.device)
    if stats is None:
        var, mean = torch.var_mean(x.double(), dim=1, correction=0)
        stats = torch.stack([mean, 1 / (var + eps).sqrt()], 1).float()
    want, bound, e_z, z = norm_backward(x.double(), dy.double(), stats.double(), g.double(), b.double(), kind, factor)
    if kind == "relu":
        assert bool((z.abs() > e_z).all()), "a value next to relu's corner: its side is not determined"
    got = ops.layer_norm_backward(x, dy, stats, gamma, beta, epilogue=kind, dropout=p, seed=5, sequence=9, dx_dtype=dx_dtype, **more)
    assert_within(got[0], want[0], bound[0], got[0].dtype, "dx")
    for k, name in ((1, "dgamma"), (2, "dbeta")):
        if got[k] is not None:
            assert_within(got[k], want[k], bound[k], name=name)
    assert (got[1] is None) == (gamma is None) and (got[2] is None) == (beta is None)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_forward_widths(cuda_device, cols, dtype):
    x = matrix(rows_for(cols), cols, dtype, cuda_device, cols, 2.0, 0.5)
    gamma, beta = parameters(cols, cuda_device, cols + 1)
    check_forward(x, gamma, beta)
    check_forward(x, gamma, beta, kind="gelu_erf", p=0.3, out_dtype=torch.bfloat16)


@pytest.mark.parametrize("x_dtype,dy_dtype,dx_dtype", [(torch.float32, torch.float32, None), (torch.float32, torch.bfloat16, None), (torch.bfloat16, torch.bfloat16, torch.float32),
                                                       (torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.float16, torch.float16)])
@pytest.mark.parametrize("cols", WIDTHS)
def test_backward_widths(cuda_device, cols, x_dtype, dy_dtype, dx_dtype):
    rows = rows_for(cols)
    x, dy = matrix(rows, cols, x_dtype, cuda_device, cols, 2.0, 0.5), matrix(rows, cols, dy_dtype, cuda_device, cols + 5)
    gamma, beta = parameters(cols, cuda_device, cols + 1)
    check_backward(x, dy, gamma, beta, dx_dtype=dx_dtype)
    check_backward(x, dy, gamma, beta, kind="gelu_tanh", p=0.3, dx_dtype=dx_dtype)


@pytest.mark.parametrize("kind", ["none", "relu", "gelu_erf", "gelu_tanh"])
@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("cols", [50, 700])
def test_activations_and_dropout(cuda_device, kind, p, cols):
    x, dy = matrix(97, cols, torch.float32, cuda_device, 3), matrix(97, cols, torch.float32, cuda_device, 4)
    gamma, beta = parameters(cols, cuda_device, 5)
    _, stats = check_forward(x, gamma, beta, kind=kind, p=p)
    check_backward(x, dy, gamma, beta, kind=kind, p=p, stats=stats)


@pytest.mark.parametrize("cols", [48, 2000])
@pytest.mark.parametrize("with_gamma,with_beta", [(False, False), (True, False), (False, True)])
def test_without_parameters(cuda_device, cols, with_gamma, with_beta):
    x, dy = matrix(20, cols, torch.float32, cuda_device, 13), matrix(20, cols, torch.float32, cuda_device, 14)
    gamma, beta = parameters(cols, cuda_device, 15)
    gamma, beta = gamma if with_gamma else None, beta if with_beta else None
    check_forward(x, gamma, beta, kind="gelu_tanh")
    check_backward(x, dy, gamma, beta, kind="gelu_tanh")


@pytest.mark.parametrize("rows", [0, 1, 2, 31, 33, 1000, 4099, 70_001])
@pytest.mark.parametrize("cols", [8, 50, 520])
def test_row_counts(cuda_device, rows, cols):
    if rows == 70_001 and cols == 520:
        rows = 3001
    x, dy = matrix(rows, cols, torch.float32, cuda_device, 23), matrix(rows, cols, torch.float32, cuda_device, 24)
    gamma, beta = parameters(cols, cuda_device, 25)
    check_forward(x, gamma, beta)
    dx, dgamma, dbeta = check_backward(x, dy, gamma, beta)
    if rows == 0:
        assert not dgamma.any() and not dbeta.any() and dx.shape == (0, cols)


@pytest.mark.parametrize("cols,pitch,shift", [(50, 51, 0), (50, 52, 2), (52, 60, 0), (33, 33, 1), (1030, 1031, 3), (1030, 1034, 0), (1028, 1032, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pitch_and_alignment(cuda_device, cols, pitch, shift, dtype):
    x = matrix(19, cols, dtype, cuda_device, 33, pitch=pitch, shift=shift)
    dy = matrix(19, cols, dtype, cuda_device, 34, pitch=cols + 1, shift=1)
    gamma, beta = parameters(cols, cuda_device, 35)
    out = matrix(19, cols, dtype, cuda_device, 36, pitch=pitch, shift=shift)
    around = out._base.clone()
    check_forward(x, gamma, beta, out=out)
    out.copy_(around[shift:shift + 19 * pitch].view(19, pitch)[:, :cols])
    assert torch.equal(out._base.view(torch.uint8), around.view(torch.uint8))     # nothing beside the matrix was written
    dx = matrix(19, cols, dtype, cuda_device, 37, pitch=pitch, shift=shift)
    around = dx._base.clone()
    check_backward(x, dy, gamma, beta, dx=dx)
    dx.copy_(around[shift:shift + 19 * pitch].view(19, pitch)[:, :cols])
    assert torch.equal(dx._base.view(torch.uint8), around.view(torch.uint8))


@pytest.mark.parametrize("cols", [40, 3001, 12_000])
def test_in_place(cuda_device, cols):
    x, dy = matrix(50, cols, torch.float32, cuda_device, 43), matrix(50, cols, torch.float32, cuda_device, 44)
    gamma, beta = parameters(cols, cuda_device, 45)
    stats = torch.empty(50, 2, device=cuda_device)
    y = ops.layer_norm(x, gamma, beta, stats=stats)
    want = ops.layer_norm_backward(x, dy, stats, gamma, beta)
    over = x.clone()
    assert torch.equal(ops.layer_norm(over, gamma, beta, out=over), y)
    for which in ("x", "dy"):
        xx, gg = x.clone(), dy.clone()
        got = ops.layer_norm_backward(xx, gg, stats, gamma, beta, dx=xx if which == "x" else gg)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("cols", [64, 5000, 33_538, 40_000])
def test_hard_rows(cuda_device, cols):
    """Rows of one value (with and without eps), far from zero, tiny and huge ones, and rows with an infinity or a NaN, whose
    neighbours are not touched.  A constant row whose mean is exact has u = 0 and the gradient of the formula."""
    x = matrix(12, cols, torch.float32, cuda_device, 53)
    x[1] = 4.0
    x[2] = 0.0
    x[3] += 1000.0
    x[4] *= 1e-18
    x[5] *= 1e15
    x[7, 3] = float("inf")
    x[8, cols - 1] = float("nan")
    gamma, beta = parameters(cols, cuda_device, 55)
    y, stats = ops.layer_norm(x, gamma, beta, stats=(s := torch.empty(12, 2, device=cuda_device))), s
    fine = [0, 1, 2, 3, 4, 5, 6, 9, 10, 11]
    check_forward(x[fine], gamma, beta)
    assert torch.equal(y[fine], ops.layer_norm(x[fine].contiguous(), gamma, beta))
    assert torch.equal(y[1], beta) and torch.equal(y[2], beta)
    assert torch.isnan(y[7]).all() and torch.isnan(y[8]).all()
    dy = matrix(12, cols, torch.float32, cuda_device, 56)
    dx, _, _ = ops.layer_norm_backward(x, dy, stats, gamma, beta)
    assert torch.isfinite(dx[fine]).all() and torch.isnan(dx[7]).all() and torch.isnan(dx[8]).all()
    check_backward(x[fine], dy[fine], gamma, beta, stats=stats[fine].contiguous())
    assert torch.isnan(ops.layer_norm(x, gamma, beta, 0.0)[2]).all()                # 0 / 0, as the formula has it


@pytest.mark.parametrize("kind", ["none", "relu", "gelu_erf", "gelu_tanh"])
def test_gradients_that_dropout_masks(cuda_device, kind):
    """NaN and infinities in places of dy that dropout masks reach no gradient."""
    cols = 60
    x, dy = matrix(30, cols, torch.float32, cuda_device, 63), matrix(30, cols, torch.float32, cuda_device, 64)
    gamma, beta = parameters(cols, cuda_device, 65)
    stats = torch.empty(30, 2, device=cuda_device)
    ops.layer_norm(x, gamma, beta, stats=stats)
    want = ops.layer_norm_backward(x, dy, stats, gamma, beta, epilogue=kind, dropout=0.5, seed=5, sequence=9)
    masked = ~keep(30, cols, 0.5, 5, 9, device=cuda_device)
    for value in (float("nan"), float("inf")):
        got = ops.layer_norm_backward(x, dy.masked_fill(masked, value), stats, gamma, beta, epilogue=kind, dropout=0.5, seed=5, sequence=9)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind", ["relu", "gelu_erf", "gelu_tanh"])
def test_far_activations(cuda_device, kind):
    """gamma of 1e6 and more: gelu is z or 0 there, its slope 1 or 0, with no infinity less infinity."""
    cols = 40
    x, dy = matrix(30, cols, torch.float32, cuda_device, 73), matrix(30, cols, torch.float32, cuda_device, 74)
    beta = torch.zeros(cols, device=cuda_device)
    stats = torch.empty(30, 2, device=cuda_device)
    for big in (1e6, 1e16, 1e30):
        gamma = torch.full((cols,), big, device=cuda_device)
        z = ops.layer_norm(x, gamma, beta, stats=stats)
        assert float(z.abs().min()) > 100
        y = ops.layer_norm(x, gamma, beta, epilogue=kind)
        assert torch.equal(y, torch.where(z > 0, z, 0.0 * z))
        got = ops.layer_norm_backward(x, dy, stats, gamma, beta, epilogue=kind)
        want = ops.layer_norm_backward(x, torch.where(z > 0, dy, 0.0), stats, gamma, beta)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("kind,p", [("none", 0.0), ("gelu_erf", 0.0), ("gelu_tanh", 0.3)])
def test_gradients_against_differences(cuda_device, kind, p):
    """Directional derivative of sum(w * y) from the kernels' outputs, central differences of the 64-bit form: with a step of 1e-5
    their error is the third derivative times 1e-10 / 6, and 1e-11 of cancellation: far below fp32's 1e-5 here."""
    rows, cols = 9, 37
    x, w = matrix(rows, cols, torch.float32, cuda_device, 83), matrix(rows, cols, torch.float32, cuda_device, 84)
    gamma, beta = parameters(cols, cuda_device, 85)
    stats = torch.empty(rows, 2, device=cuda_device)
    ops.layer_norm(x, gamma, beta, epilogue=kind, dropout=p, seed=5, sequence=9, stats=stats)
    grads = ops.layer_norm_backward(x, w, stats, gamma, beta, epilogue=kind, dropout=p, seed=5, sequence=9)
    factor = factor_of(rows, cols, p, 5, 9, cuda_device)
    at = [x.double(), gamma.double(), beta.double()]
    for i, grad in enumerate(grads):
        way = torch.randn(at[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64).to(cuda_device)
        def loss(t):
            moved = [v + t * way if k == i else v for k, v in enumerate(at)]
            return float((norm_forward(*moved, 1e-5, kind, factor)[0] * w.double()).sum())
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        terms = grad.double() * way
        assert abs(float(terms.sum()) - slope) <= 1e-5 * float(terms.abs().sum())


def test_rows_do_not_depend_on_their_neighbours(cuda_device):
    """The same bits in a shard as in the whole, in every call, and with any workspace."""
    for cols in (64, 50, 2000, 6000):
        x, dy = matrix(700, cols, torch.float32, cuda_device, 93), matrix(700, cols, torch.float32, cuda_device, 94)
        gamma, beta = parameters(cols, cuda_device, 95)
        stats = torch.empty(700, 2, device=cuda_device)
        kw = dict(epilogue="gelu_tanh", dropout=0.2, seed=3, sequence=1)
        y = ops.layer_norm(x, gamma, beta, stats=stats, **kw)
        grads = ops.layer_norm_backward(x, dy, stats, gamma, beta, **kw)
        again = ops.layer_norm_backward(x, dy, stats, gamma, beta, workspace=torch.full((ops.layer_norm_backward_workspace(700, cols) + 64,), 255, dtype=torch.uint8, device=cuda_device), **kw)
        assert all(torch.equal(a, b) for a, b in zip(grads, again))
        for lo, hi in ((0, 1), (1, 400), (400, 700)):
            assert torch.equal(ops.layer_norm(x[lo:hi], gamma, beta, first_row=lo, **kw), y[lo:hi])
            assert torch.equal(ops.layer_norm_backward(x[lo:hi], dy[lo:hi], stats[lo:hi].contiguous(), gamma, beta, first_row=lo, **kw)[0], grads[0][lo:hi])


@pytest.mark.parametrize("cols", [300, 3000, 5001, 40_000])
def test_some_of_the_gradients(cuda_device, cols):
    """Each gradient alone through the C entry has the bits of all together, and the others' memory is left as it was."""
    import ctypes as C
    from cellerator_b200 import capi
    rows = 90
    x, dy = matrix(rows, cols, torch.float32, cuda_device, 123), matrix(rows, cols, torch.float32, cuda_device, 124)
    gamma, beta = parameters(cols, cuda_device, 125)
    stats = torch.empty(rows, 2, device=cuda_device)
    ops.layer_norm(x, gamma, beta, stats=stats)
    want = ops.layer_norm_backward(x, dy, stats, gamma, beta, epilogue="gelu_erf")
    workspace = torch.empty(ops.layer_norm_backward_workspace(rows, cols), dtype=torch.uint8, device=cuda_device)
    for asked in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False, False, False)):
        got = [torch.full_like(t, 7.0) for t in want]
        n = capi.header(capi.LayerNorm())
        n.rows, n.columns, n.x, n.x_ld, n.dy, n.dy_ld, n.dx_ld = rows, cols, x.data_ptr(), cols, dy.data_ptr(), cols, cols
        n.x_dtype = n.dy_dtype = n.dx_dtype = capi.DTYPE_F32
        n.gamma, n.beta, n.stats, n.epilogue, n.device = gamma.data_ptr(), beta.data_ptr(), stats.data_ptr(), capi.EPILOGUE["gelu_erf"], cuda_device.index
        n.dx, n.dgamma, n.dbeta = (t.data_ptr() if a else None for t, a in zip(got, asked))
        if any(asked[1:]) or (asked[0] and cols > 4608):
            n.workspace, n.workspace_bytes = workspace.data_ptr(), workspace.numel()
        capi.check(capi.lib().cb200_layer_norm_backward(C.byref(n), torch.cuda.current_stream(cuda_device).cuda_stream))
        for g, w, a in zip(got, want, asked):
            assert torch.equal(g, w if a else torch.full_like(w, 7.0))


@pytest.mark.parametrize("rows,cols,dtype", [(20_000, 5000, torch.bfloat16), (2700, 33_538, torch.float32)])
def test_parts_of_many_rows(cuda_device, rows, cols, dtype):
    """Parts of more rows than are taken at a time: sums of 64 rows on top of each other, 64 + 3 + 8 + 16 roundings of the bound's 96."""
    x, dy = matrix(rows, cols, dtype, cuda_device, 133), matrix(rows, cols, dtype, cuda_device, 134)
    gamma, beta = parameters(cols, cuda_device, 135)
    check_backward(x, dy, gamma, beta, kind="gelu_tanh", p=0.1)


def test_graph_replay_on_another_stream(cuda_device):
    """Forward and backward captured together, eager calls in between; new inputs and a new mask at each replay."""
    for cols in (48, 2000, 5000, 40_000):
        x, dy = matrix(200, cols, torch.float32, cuda_device, 103), matrix(200, cols, torch.float32, cuda_device, 104)
        gamma, beta = parameters(cols, cuda_device, 105)
        number = torch.zeros(1, dtype=torch.int64, device=cuda_device)
        stats, y, dx, dgamma, dbeta = torch.empty(200, 2, device=cuda_device), torch.empty_like(x), torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
        workspace = torch.empty(ops.layer_norm_backward_workspace(200, cols), dtype=torch.uint8, device=cuda_device)
        kw = dict(epilogue="gelu_erf", dropout=0.2, seed=3)
        stream = torch.cuda.Stream(cuda_device)
        stream.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(stream):
            def step():
                ops.layer_norm(x, gamma, beta, out=y, stats=stats, device_sequence=number, **kw)
                ops.layer_norm_backward(x, dy, stats, gamma, beta, dx=dx, dgamma=dgamma, dbeta=dbeta, workspace=workspace, device_sequence=number, **kw)
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            for i in range(3):
                x.add_(0.5 * i)
                number.fill_(i)
                other = torch.empty(200, 2, device=cuda_device)
                want_y = ops.layer_norm(x, gamma, beta, stats=other, sequence=i, **kw)
                want = ops.layer_norm_backward(x, dy, other, gamma, beta, sequence=i, **kw)
                graph.replay()
                assert torch.equal(y, want_y) and all(torch.equal(a, b) for a, b in zip((dx, dgamma, dbeta), want))
        torch.cuda.current_stream(cuda_device).wait_stream(stream)


def test_more_than_2_to_the_32_bytes(cuda_device):
    """2.2e9 values, in place; first, middle and last rows against the rows alone."""
    for rows, cols in ((33_000, 65_536), (34_000_000, 64)):
        x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=cuda_device)
        some = [0, rows // 2, rows - 2, rows - 1]
        values = matrix(4, cols, torch.bfloat16, cuda_device, 113)
        x[some] = values
        gamma, beta = parameters(cols, cuda_device, 115)
        want = ops.layer_norm(values, gamma, beta)
        stats = torch.empty(rows, 2, device=cuda_device)
        ops.layer_norm(x, gamma, beta, out=x, stats=stats)
        assert torch.equal(x[some], want)
        x.zero_()
        x[some] = values
        dy = torch.zeros_like(x)
        dy[some] = matrix(4, cols, torch.bfloat16, cuda_device, 114)
        want = ops.layer_norm_backward(values, dy[some], stats[some], gamma, beta)
        got = ops.layer_norm_backward(x, dy, stats, gamma, beta, dx=dy)
        assert torch.equal(got[0][some], want[0])
        # four rows with a gradient: their terms, added in some order
        terms = norm_backward(values.double(), matrix(4, cols, torch.bfloat16, cuda_device, 114).double(), stats[some].double(), gamma.double(), beta.double(), "none", 1.0)
        assert_within(got[1], terms[0][1], terms[1][1], name="dgamma")
        assert_within(got[2], terms[0][2], terms[1][2], name="dbeta")
        del x, dy, got, stats


@pytest.mark.parametrize("cols", [50, 1300, 9001, 40_001])
def test_two_streams_at_once(cuda_device, cols):
    """Calls that overlap on the device, each with memory of its own, give what they give one after the other."""
    parameters_of = parameters(cols, cuda_device, 61)
    inputs = [(matrix(700, cols, torch.float32, cuda_device, 62 + k), matrix(700, cols, torch.bfloat16, cuda_device, 64 + k)) for k in range(2)]
    more = dict(epilogue="gelu_erf", dropout=0.25, seed=8)

    def both(x, dy, sequence):
        stats = torch.empty(700, 2, device=cuda_device)
        y = ops.layer_norm(x, *parameters_of, stats=stats, sequence=sequence, **more)
        return y, stats, *ops.layer_norm_backward(x, dy, stats, *parameters_of, sequence=sequence, **more)

    want = [both(*inputs[k], k) for k in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k] = both(*inputs[k], k)
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got[k], want[k]))


def test_gradients_of_parameters_that_were_not_given(cuda_device):
    """dgamma and dbeta are sums over rows whether or not there is a gamma or a beta to move."""
    for cols in (50, 1300, 5000):
        x, dy = matrix(300, cols, torch.float32, cuda_device, 71), matrix(300, cols, torch.float32, cuda_device, 72)
        stats = torch.empty(300, 2, device=cuda_device)
        ops.layer_norm(x, stats=stats)
        one, zero = torch.ones(cols, device=cuda_device), torch.zeros(cols, device=cuda_device)
        want = ops.layer_norm_backward(x, dy, stats, one, zero)
        got = ops.layer_norm_backward(x, dy, stats, dgamma=torch.full_like(one, 7.0), dbeta=torch.full_like(one, 7.0))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
