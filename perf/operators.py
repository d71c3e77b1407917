"""The operators behind and beside the quantized projection, as a program calls them: layer norm with its activation and
dropout, its backward pass, dropout alone, and the low-rank adapters of many requests beside the shared projection.

`run` computes them in plain torch, or, with `own`, by the calls of `cellerator_b200.ops`.  `prepare` makes what the program
holds before the call (activations, gradients, weights, a batch of cells in quantized CSR), `exact` the same results in 64 bits.

Kinds:
  norm        y = drop(act(gamma * (x - mean) / sqrt(var + eps) + beta)), row by row, and each row's {mean, 1 / sqrt(var + eps)}
  norm_back   the gradients of x, gamma and beta from y's
  drop        x / (1 - p) where the generator keeps the value, else 0
  adapt       y = s_a (deq(X) A_a) B_a, a the adapter that a cell's request brings (some bring none)

The random number of value (row, col) is word col % 4 of Philox4x32-10 with counter {col / 4, row, sequence, 0} and key = seed.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _norm(name, kind, rows, cols, x, y, epilogue="none", p=0.0):
    """x: type of the rows that are normalised (and of their gradient), y: of the result (and of the gradient that comes back)."""
    return dict(name=name, kind=kind, rows=rows, cols=cols, x=x, y=y, epilogue=epilogue, p=p)


def _adapt(name, rows, cols, median, sigma, bits, adapters, rank, n, weights):
    return dict(name=name, kind="adapt", rows=rows, cols=cols, median=median, sigma=sigma, bits=bits, adapters=adapters, rank=rank,
                n=n, weights=weights)


def listed():
    return [
        # a few dozen cells that an annotation service embeds for one request, width of the gene-panel configuration: latency
        _norm("norm_query", "norm", 64, 32, "f32", "f32", "relu"),
        # the encoder's first layer on a training mini-batch, hidden width that is no power of two
        _norm("norm_minibatch", "norm", 4_099, 50, "f32", "bf16", "gelu_erf", 0.1),
        # all cells of the million-cell configuration behind the projection, for the next layer's 16-bit product
        _norm("norm_atlas", "norm", 1_000_000, 64, "f32", "bf16", "relu"),
        # a decoder's rows over the whole gene set
        _norm("norm_genes", "norm", 4_099, 33_538, "bf16", "bf16"),
        # the gradients of the mini-batch above
        _norm("norm_back_minibatch", "norm_back", 4_099, 50, "f32", "bf16", "gelu_erf", 0.1),
        # the gradients for a million cells: what the transposed projection then takes is fp32
        _norm("norm_back_atlas", "norm_back", 1_000_000, 64, "f32", "bf16", "gelu_tanh", 0.1),
        # the gradients of a decoder's rows
        _norm("norm_back_genes", "norm_back", 1_025, 33_538, "f32", "f32"),
        # a mini-batch's hidden layer
        dict(name="drop_minibatch", kind="drop", rows=4_099, cols=50, x="f32", p=0.1),
        # the widest hidden layer that the configurations have, half a million cells
        dict(name="drop_atlas", kind="drop", rows=500_000, cols=128, x="bf16", p=0.2),
        # cells of a handful of requests against the gene panel, each with its own adapter: latency
        _adapt("adapt_query", 64, 2_000, 300, 0.5, 8, 8, 8, 32, "f32"),
        # a served batch over the full gene set, requests of ragged sizes
        _adapt("adapt_batch", 4_099, 33_538, 1_500, 0.6, 8, 16, 16, 64, "bf16"),
        # data sets mapped at once over highly variable genes, 4-bit codes
        _adapt("adapt_sets", 50_000, 4_000, 600, 0.5, 4, 12, 32, 128, "bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_back", "norm_back", "drop", "adapt", "adapt"])
    if kind == "adapt":
        cols = _spread(rng, 1_000, 33_538)
        # the more genes, the thinner the rows: 15 % at 2,000, 4.5 % at 33,538
        median = max(8, round(cols * min(0.15, 0.15 * (2_000 / cols) ** 0.43) * rng.uniform(0.5, 1.2)))
        case = _adapt("", _spread(rng, 1, min(40_000, 12_000_000 // median)), cols, median, rng.choice([0.5, 0.6]), rng.choice([8, 8, 4]),
                      rng.randint(1, 24), rng.choice([4, 8, 12, 16, 24, 32, 64]), rng.choice([16, 32, 50, 64, 100, 128]),
                      rng.choice(["f32", "bf16"]))
    else:
        # widths of hidden layers, odd ones among them, and up to the whole gene set
        cols = rng.choice([_spread(rng, 8, 512), 8 * _spread(rng, 1, 64), _spread(rng, 500, 33_538)])
        rows = _spread(rng, 16, max(64, min(1_000_000, 60_000_000 // cols)))
        if kind == "drop":
            return dict(kind=kind, rows=rows, cols=cols, x=rng.choice(["f32", "bf16", "f16"]), p=rng.choice([0.05, 0.1, 0.2, 0.5]))
        x = rng.choice(["f32", "f32", "bf16", "f16"])
        # relu has a step in its derivative: which side a value next to it falls on is no question of a kernel's
        epilogue = rng.choice(["none", "gelu_erf", "gelu_tanh"] + (["relu"] if kind == "norm" else []))
        case = _norm("", kind, rows, cols, x, rng.choice([x, "f32" if x == "f32" else x, "bf16"]), epilogue, rng.choice([0.0, 0.0, 0.1, 0.5]))
    del case["name"]
    return case


def _cells(case, g):
    """Cells x genes in quantized CSR: row lengths lognormal, genes ascending and distinct, small codes more often than large ones."""
    rows, cols, bits = case["rows"], case["cols"], case["bits"]
    device = g.device
    counts = (torch.randn(rows, generator=g, device=device, dtype=torch.float64) * case["sigma"] + math.log(case["median"])).exp().round().long()
    counts.clamp_(1, cols)
    row_ptr = torch.zeros(rows + 1, dtype=torch.int64, device=device)
    row_ptr[1:] = counts.cumsum(0)
    nnz = int(row_ptr[-1])
    row = torch.repeat_interleave(torch.arange(rows, device=device), counts, output_size=nnz)
    local = torch.arange(nnz, device=device) - row_ptr[row]
    # sorted places from sums of whole random gaps, spread over the genes that a strictly ascending row leaves
    gaps = torch.randint(1, 1_000, (nnz,), generator=g, device=device)
    upto = gaps.cumsum(0)
    begin = upto[row_ptr[:-1]] - gaps[row_ptr[:-1]]
    total = upto[row_ptr[1:] - 1] - begin + 500
    col_idx = ((upto - begin[row]) * (cols - counts[row] + 1) // (total[row] + 1) + local).int()
    codes = (torch.rand(nnz, generator=g, device=device).square_() * 2 ** bits).clamp_(max=2 ** bits - 1).to(torch.uint8)
    s = dict(row_ptr=row_ptr, col_idx=col_idx, scales=torch.rand(cols, generator=g, device=device) * 0.02 * 2 ** (8 - bits) + 0.005,
             offsets=torch.rand(cols, generator=g, device=device) * 0.5, packed=codes, packed_row_ptr=None)
    if bits == 4:
        packed_row_ptr = torch.zeros_like(row_ptr)
        packed_row_ptr[1:] = ((counts + 1) // 2).cumsum(0)
        both = torch.zeros(2 * int(packed_row_ptr[-1]), dtype=torch.uint8, device=device)
        both[2 * packed_row_ptr[row] + local] = codes
        s.update(packed=both[0::2] | both[1::2] << 4, packed_row_ptr=packed_row_ptr)
    return s


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    rows, cols, kind = case["rows"], case["cols"], case["kind"]

    def randn(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=device).mul_(std).add_(mean).to(dtype)

    s = dict(case, seed=seed * 2_654_435_761 + 12_345, sequence=seed + 7)
    if kind == "adapt":
        dtype = TYPES[case["weights"]]
        s.update(_cells(case, g))
        s["down"] = randn(case["adapters"], cols, case["rank"], std=0.02, dtype=dtype)
        s["up"] = randn(case["adapters"], case["rank"], case["n"], std=0.1, dtype=dtype)
        s["scale"] = torch.rand(case["adapters"], generator=g, device=device) + 0.5
        # requests one after the other, of ragged sizes; the first of them bring no adapter
        s["adapter"] = torch.randint(-1, case["adapters"], (rows,), generator=g, device=device).sort().values.int()
        s["out"] = torch.empty(rows, case["n"], device=device)
        if own:  # the handle that a program keeps of its matrix
            from cellerator_b200 import ops
            s["cells"] = ops.QuantizedCsr(rows, cols, case["bits"], 1, s["row_ptr"], s["col_idx"], s["packed"], s["scales"], s["offsets"],
                                          s["packed_row_ptr"])
        return s
    x = TYPES[case["x"]]
    if kind == "drop":
        s["data"] = randn(rows, cols, dtype=x)
        return s
    s["data"] = randn(rows, cols, std=2.0, mean=0.5, dtype=x)
    s["gamma"], s["beta"] = randn(cols, std=0.2, mean=1.0), randn(cols, std=0.2)
    if kind == "norm_back":
        s["dy"] = randn(rows, cols, dtype=TYPES[case["y"]])
        # the statistics that the forward pass kept
        d = s["data"].double()
        var, mean = torch.var_mean(d, dim=1, correction=0)
        s["stats"] = torch.stack([mean, (var + EPS).rsqrt()], dim=1).float()
    else:
        s["stats"] = torch.empty(rows, 2, device=device)
    return s


# ---- the plain forms ----------------------------------------------------------------------

def _round(a, b, c, d, k0, k1):
    """One round of Philox4x32 on counter words held in 64 bits."""
    p, q = a * 0xD2511F53, c * 0xCD9E8D57
    low = 0xFFFFFFFF
    return (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ d ^ k1, p & low


def _kept(rows, cols, p, seed, sequence, device):
    """Which values the generator keeps: [rows, cols] truth values."""
    low = 0xFFFFFFFF
    quads = (cols + 3) // 4
    a = torch.arange(quads, device=device).expand(rows, quads)
    b = torch.arange(rows, device=device)[:, None].expand(rows, quads)
    c, d = torch.full_like(a, sequence & low), torch.full_like(a, sequence >> 32)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b, c, d = _round(a, b, c, d, k0, k1)
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return (torch.stack([a, b, c, d], dim=2) >= int(p * 2 ** 32 + 0.5)).reshape(rows, 4 * quads)[:, :cols]


def _drop(t, s):
    if s["p"] == 0.0:
        return t
    return torch.where(_kept(s["rows"], s["cols"], s["p"], s["seed"], s["sequence"], t.device), t * (1.0 / (1.0 - s["p"])), 0.0)


def _act(z, kind):
    if kind == "relu":
        return z.clamp(min=0.0)
    if kind == "gelu_erf":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _act_slope(z, kind):
    if kind == "gelu_erf":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if kind == "gelu_tanh":
        t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 3.0 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_norm(s):
    x = s["data"].float()
    mean = x.mean(dim=1, keepdim=True)
    rstd = (x - mean).square().mean(dim=1, keepdim=True).add(EPS).rsqrt()
    y = _drop(_act((x - mean) * rstd * s["gamma"] + s["beta"], s["epilogue"]), s)
    return y.to(TYPES[s["y"]]), torch.cat([mean, rstd], dim=1)


def _plain_norm_back(s):
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    u = (s["data"].float() - mean) * rstd
    dz = _drop(s["dy"].float(), s)
    if s["epilogue"] != "none":
        dz = dz * _act_slope(u * s["gamma"] + s["beta"], s["epilogue"])
    h = dz * s["gamma"]
    dx = (h - h.mean(dim=1, keepdim=True) - u * (h * u).mean(dim=1, keepdim=True)) * rstd
    return dx.to(s["data"].dtype), (dz * u).sum(dim=0, dtype=torch.float64).float(), dz.sum(dim=0, dtype=torch.float64).float()


def _plain_adapt(s):
    rows, entries = s["rows"], s["col_idx"].numel()
    begin = s["row_ptr"][:-1]
    row = torch.repeat_interleave(torch.arange(rows, device=begin.device), s["row_ptr"][1:] - begin, output_size=entries)
    if s["packed_row_ptr"] is None:
        codes = s["packed"]
    else:
        local = torch.arange(entries, device=begin.device) - begin[row]
        codes = s["packed"][s["packed_row_ptr"][row] + local // 2] >> (4 * (local % 2)).to(torch.uint8) & 15
    genes = s["col_idx"].long()
    adapter = s["adapter"].long()
    has = adapter >= 0
    held = adapter.clamp(min=0)
    values = torch.where(has[row], codes.float() * s["scales"][genes] + s["offsets"][genes], 0.0)
    hidden = torch.zeros(rows, s["rank"], dtype=torch.float64, device=begin.device)
    hidden.index_add_(0, row, (s["down"][held[row], genes].float() * values[:, None]).double())
    return torch.einsum("rk,rkn->rn", hidden.float(), s["up"].float()[held]) * s["scale"][held][:, None]


def run(s):
    kind = s["kind"]
    if not own:
        if kind == "drop":
            return _drop(s["data"].float(), s).to(s["data"].dtype)
        return {"norm": _plain_norm, "norm_back": _plain_norm_back, "adapt": _plain_adapt}[kind](s)
    from cellerator_b200 import ops
    if kind == "drop":
        return ops.dropout(s["data"], s["p"], s["seed"], s["sequence"])
    if kind == "norm":
        y = ops.layer_norm(s["data"], s["gamma"], s["beta"], EPS, epilogue=s["epilogue"], dropout=s["p"], seed=s["seed"],
                           sequence=s["sequence"], out_dtype=TYPES[s["y"]], stats=s["stats"])
        return y, s["stats"]
    if kind == "norm_back":
        return ops.layer_norm_backward(s["data"], s["dy"], s["stats"], s["gamma"], s["beta"], epilogue=s["epilogue"], dropout=s["p"],
                                       seed=s["seed"], sequence=s["sequence"])
    return ops.adapter_forward(s["cells"], s["adapter"], s["down"], s["up"], s["scale"], out=s["out"])


def work(case):
    rows, cols, kind = case["rows"], case["cols"], case["kind"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if kind == "adapt":
        # the mean of a lognormal; clipping at the number of genes takes next to nothing off
        entries = rows * min(cols, case["median"] * math.exp(case["sigma"] ** 2 / 2))
        weights, rank, n = size[case["weights"]], case["rank"], case["n"]
        # of the adapters, the rows that some entry needs
        down = min(entries, case["adapters"] * cols) * rank * weights
        return {"bytes": entries * (4 + case["bits"] / 8) + rows * 12 + cols * 8 + down + min(rows, case["adapters"]) * rank * n * weights + rows * n * 4,
                "flops": 2 * entries * rank + 2 * rows * rank * n}
    if kind == "drop":
        return {"bytes": 2 * rows * cols * size[case["x"]], "flops": rows * cols}
    x, y = size[case["x"]], size[case["y"]]
    if kind == "norm":
        return {"bytes": rows * cols * (x + y) + rows * 8 + cols * 8, "flops": 8 * rows * cols}
    return {"bytes": rows * cols * (2 * x + y) + rows * 8 + cols * 16, "flops": 14 * rows * cols}


# ---- the definitions in 64 bits -------------------------------------------------------------

def _words(rows, cols, seed, sequence, device):
    """The random words of [rows, cols] values, ten rounds of Philox4x32 with products put together from 16-bit halves."""
    mask = 0xFFFFFFFF
    place = torch.arange((cols + 3) // 4, device=device).repeat(rows, 1)
    word = [place, torch.arange(rows, device=device).unsqueeze(1) + 0 * place, 0 * place + (sequence & mask), 0 * place + (sequence >> 32)]
    key = [seed % 2 ** 32, (seed >> 32) % 2 ** 32]

    def product(v, constant):
        """(high, low) 32 bits of v * constant"""
        lower, upper = v * (constant & 0xFFFF), v * (constant >> 16)
        middle = (lower >> 16) + (upper & 0xFFFF_FFFF_FFFF)
        return middle >> 16, (middle << 16 | lower & 0xFFFF) & mask

    for turn in range(10):
        high0, low0 = product(word[0], 0xD2511F53)
        high1, low1 = product(word[2], 0xCD9E8D57)
        word = [high1 ^ word[1] ^ key[0], low1, high0 ^ word[3] ^ key[1], low0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    return torch.stack(word, dim=-1).flatten(1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    rows, cols, kind = s["rows"], s["cols"], s["kind"]
    if kind == "adapt":
        device = s["row_ptr"].device
        result = torch.zeros(rows, s["n"], dtype=torch.float64, device=device)
        bounds = s["row_ptr"].tolist()
        step = max(1, 200_000_000 // cols)
        for lo in range(0, rows, step):  # rows of the decoded matrix, written out
            hi = min(rows, lo + step)
            b, e = bounds[lo], bounds[hi]
            lengths = s["row_ptr"][lo + 1:hi + 1] - s["row_ptr"][lo:hi]
            row = torch.arange(hi - lo, device=device).repeat_interleave(lengths)
            genes = s["col_idx"][b:e].long()
            if s["bits"] == 8:
                codes = s["packed"][b:e].double()
            else:
                bytes_ = s["packed"][int(s["packed_row_ptr"][lo]):int(s["packed_row_ptr"][hi])]
                nibbles = torch.stack([bytes_ % 16, bytes_ // 16], dim=1).flatten()
                starts = 2 * (s["packed_row_ptr"][lo:hi] - s["packed_row_ptr"][lo])
                codes = nibbles[starts[row] + torch.arange(e - b, device=device) - (s["row_ptr"][lo:hi] - b)[row]].double()
            x = torch.zeros(hi - lo, cols, dtype=torch.float64, device=device)
            x[row, genes] = codes * s["scales"].double()[genes] + s["offsets"].double()[genes]
            for a in range(s["adapters"]):
                mine = (s["adapter"][lo:hi] == a).nonzero().flatten()
                if mine.numel():
                    result[lo + mine] = s["scale"][a].double() * (x[mine] @ s["down"][a].double() @ s["up"][a].double())
        return result
    x = s["data"].double()
    factor = 1.0
    if s["p"] > 0.0:
        factor = (_words(rows, cols, s["seed"], s["sequence"], x.device) >= round(s["p"] * 2 ** 32)).double() / (1.0 - s["p"])
    if kind == "drop":
        return x * factor
    gamma, beta = s["gamma"].double(), s["beta"].double()
    if kind == "norm":
        centred = x - x.mean(1, keepdim=True)
        deviation = (centred.pow(2).mean(1, keepdim=True) + EPS).sqrt()
        z = centred / deviation * gamma + beta
        if s["epilogue"] == "relu":
            z = z * (z > 0)
        elif s["epilogue"] == "gelu_erf":
            z = z * torch.special.ndtr(z)
        elif s["epilogue"] == "gelu_tanh":
            z = z * torch.sigmoid(math.sqrt(8.0 / math.pi) * (z + 0.044715 * z.pow(3)))
        return z * factor, torch.cat([x.mean(1, keepdim=True), 1.0 / deviation], dim=1)
    kept = s["stats"].double()
    u = (x - kept[:, 0:1]) * kept[:, 1:2]
    z = u * gamma + beta
    dz = s["dy"].double() * factor
    if s["epilogue"] == "gelu_erf":
        dz = dz * (torch.special.ndtr(z) + z * torch.exp(-z.pow(2) / 2) / math.sqrt(2 * math.pi))
    elif s["epilogue"] == "gelu_tanh":
        inner = math.sqrt(8.0 / math.pi) * (z + 0.044715 * z.pow(3))
        gate = torch.sigmoid(inner)
        dz = dz * (gate + z * gate * (1 - gate) * math.sqrt(8.0 / math.pi) * (1 + 0.134145 * z.pow(2)))
    h = dz * gamma
    dx = kept[:, 1:2] * (h - h.mean(1, keepdim=True) - u * (h * u).mean(1, keepdim=True))
    return dx, (dz * u).sum(0), dz.sum(0)
