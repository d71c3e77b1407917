"""Plain forms in 64 bits of the row operators (dropout, layer norm) and bounds of what fp32 arithmetic may be off them, shared by
their tests.  Bounds count roundings: U = 2^-24 is half a step of fp32 relative to the value."""
import numpy as np
import torch

U = 2.0 ** -24


def philox_words(rows, cols, seed, sequence, first_row=0, device="cpu"):
    """Words of Philox4x32-10 for values [rows, cols]: word col % 4 of counter {col / 4, first_row + row, sequence}, key = seed."""
    low = 0xFFFFFFFF
    quads = (cols + 3) // 4
    a = torch.arange(quads, device=device).repeat(rows, 1)
    b = (torch.arange(rows, device=device) + first_row)[:, None] + 0 * a
    c, d = 0 * a + (sequence & low), 0 * a + (sequence >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57                # modulo 2^64
        a, b, c, d = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ d ^ k1, p & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([a, b, c, d], dim=2).reshape(rows, 4 * quads)[:, :cols]


def keep(rows, cols, p, seed, sequence, first_row=0, device="cpu"):
    threshold = min(int(np.floor(p * 2.0 ** 32 + 0.5)), 2 ** 32 - 1)
    return philox_words(rows, cols, seed, sequence, first_row, device) >= threshold


def act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, 0.0 * z)
    if kind == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z / 2 ** 0.5))
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    return z


def act_slope(z, kind):
    if kind == "relu":
        return (z > 0).to(z.dtype)
    if kind == "gelu_erf":
        return 0.5 * (1 + torch.erf(z / 2 ** 0.5)) + z * torch.exp(-z * z / 2) / (2 * np.pi) ** 0.5
    if kind == "gelu_tanh":
        t = torch.tanh((2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * (2 / np.pi) ** 0.5 * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def rounding(t, dtype):
    """Half a step of `dtype` at the values of t, and half its smallest number."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def norm_forward(x, gamma, beta, eps, kind, factor):
    """(y, stats, bound of y before its last rounding, bounds of the statistics), all float64; factor: what dropout multiplies by.

    A sum of N <= 65,536 values has at most 16 neighbouring values added one by one, 5 shuffles and 5 + 5 steps over the warps of
    a cluster: 32 roundings, U each, of the sum of magnitudes.  So |mean| is off by 33 U mean|x| at most; a difference from it by
    that and U of itself; the variance, a sum of squares, by 36 U of itself and twice the mean's error times the differences' mean
    (their exact sum is zero; what is left of the mean's error is squared); its reciprocal root by half that, 2 units for rsqrtf
    and 1 for the sum with eps.  u then is off by rstd 34 U mean|x| + 26 U |u|, z by that times |gamma| and 2 U (|gamma u| + |z|).
    The activations' slopes are below 1.13.  Their own error: Phi by a polynomial that is 0.75e-7 = 1.3 U off, with a reciprocal, five
    products and sums and an exponential less than 6 U; the logistic function's exponential 4 U + 2 |t| U of itself where it counts
    (sigma (1 - sigma) |t| < 0.23), a reciprocal of 2 U, four products: less than 20 U |z|."""
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1 / (centred.square().mean(1, keepdim=True) + eps).sqrt()
    u = centred * rstd
    z = u * gamma + beta
    y = act(z, kind) * factor
    size = x.abs().mean(1, keepdim=True)
    # the mean's error squared, relative to the variance with eps
    shift = (33 * U * size * rstd).square()
    du = rstd * 34 * U * size + (26 * U + shift) * u.abs()
    dz = gamma.abs() * du + 2 * U * ((gamma * u).abs() + z.abs())
    bound = factor * (1.13 * dz + (20 * U * z.abs() if kind.startswith("gelu") else 0.0) + 3 * U * act(z, kind).abs())
    return y, torch.cat([mean, rstd], 1), bound, torch.cat([33 * U * size, rstd * (24 * U + shift)], 1)


def norm_backward(x, dy, stats, gamma, beta, kind, factor):
    """(dx, dgamma, dbeta) and their bounds, float64.

    u has two roundings, z two more.  A slope is off by 20 U (1 + |z|) (as above) and, by gelu's second derivative < 1, the error of
    z.  Sums of a row have, of their magnitudes, 32 roundings as in norm_forward, or, piece by piece of 4,096 columns, 16 values of a
    thread, 5 shuffles, 8 warps and 16 pieces, 45, and one of the mean; sums over the rows of a test, one thread's rows, 5 shuffles,
    8 warps, every so many parts (14 of them) and 32 of these, at most 96."""
    mean, rstd = stats[:, :1], stats[:, 1:]
    u = (x - mean) * rstd
    z = u * gamma + beta
    dz = dy * factor * act_slope(z, kind)
    e_u = 2 * U * u.abs()
    e_z = gamma.abs() * e_u + 2 * U * ((gamma * u).abs() + z.abs())
    e_slope = 20 * U * (1 + z.abs()) + e_z if kind.startswith("gelu") else 0.0 * z
    e_dz = (dy * factor).abs() * e_slope + 3 * U * dz.abs()
    h, e_h = dz * gamma, e_dz * gamma.abs() + U * (dz * gamma).abs()
    hu, e_hu = h * u, e_h * u.abs() + h.abs() * e_u + U * (h * u).abs()
    c1, c2 = h.mean(1, keepdim=True), hu.mean(1, keepdim=True)
    e_c1 = e_h.mean(1, keepdim=True) + 47 * U * h.abs().mean(1, keepdim=True)
    e_c2 = e_hu.mean(1, keepdim=True) + 47 * U * hu.abs().mean(1, keepdim=True)
    dx = rstd * (h - c1 - u * c2)
    e_dx = rstd * (e_h + e_c1 + u.abs() * e_c2 + e_u * c2.abs() + 4 * U * (h.abs() + c1.abs() + (u * c2).abs()))
    dgamma, dbeta = (dz * u).sum(0), dz.sum(0)
    e_dgamma = (e_dz * u.abs() + dz.abs() * e_u + U * (dz * u).abs()).sum(0) + 96 * U * (dz * u).abs().sum(0)
    e_dbeta = e_dz.sum(0) + 96 * U * dz.abs().sum(0)
    return (dx, dgamma, dbeta), (e_dx, e_dgamma, e_dbeta), e_z, z


def assert_within(got, want, bound, dtype=torch.float32, name=""):
    """|got - want| <= bound and the last rounding of `dtype`; where want is not finite got is the same."""
    got = got.double()
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    same = (got == want) | torch.isnan(want)
    off = (got - want).abs() - bound - rounding(want.abs() + bound, dtype)
    bad = torch.where(finite, off > 0, ~same)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name} at {at}: {float(got[at])!r}, expected {float(want[at])!r} within {float((bound + 0 * want)[at])!r}; {int(bad.sum())} in all")


def matrix(rows, cols, dtype, device, seed, std=1.0, mean=0.0, pitch=0, shift=0):
    """Random [rows, cols] whose rows lie `pitch` elements apart, `shift` elements into their buffer; what is not the matrix is NaN."""
    g = torch.Generator().manual_seed(seed)
    values = (torch.randn(rows, cols, generator=g, dtype=torch.float64) * std + mean).to(dtype)
    pitch = max(pitch, cols)
    buffer = torch.full((rows * pitch + shift + 8,), float("nan"), dtype=dtype, device=device)
    view = buffer[shift:shift + rows * pitch].view(rows, pitch)[:, :cols] if rows else buffer[:0].view(0, cols)
    view.copy_(values.to(device))
    return view
