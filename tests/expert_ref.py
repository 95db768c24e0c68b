"""Plain 64-bit forms of the mixture-of-experts operators, on CPU tensors or GPU tensors alike."""
import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# Half a unit in the last place of a value in [1, 2), relative.
ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24


def route(logits, top_k, normalise):
    """Column by column, as the definition reads."""
    x = logits.double().cpu()
    experts, batch = x.shape
    expert = torch.full((top_k, batch), -1, dtype=torch.int32)
    weight = torch.zeros((top_k, batch), dtype=torch.float64)
    taken = [[] for _ in range(experts)]
    for b in range(batch):
        col = [(-v, e) for e, v in enumerate(x[:, b].tolist()) if v == v and v > -math.inf]
        col.sort()
        if not col:
            continue
        best = -col[0][0]
        t = lambda v: 1.0 if v == best else math.exp(v - best)  # noqa: E731
        chosen = col[:top_k]
        total = sum(t(-v) for v, _ in (chosen if normalise == "selected" else col))
        for j, (v, e) in enumerate(chosen):
            expert[j, b] = e
            weight[j, b] = t(-v) / total
            taken[e].append((b, j))
    row = torch.full((top_k, batch), -1, dtype=torch.int32)
    column = torch.full((top_k * batch,), -1, dtype=torch.int32)
    offset = [0]
    for e in range(experts):
        for i, (b, j) in enumerate(taken[e]):
            row[j, b], column[offset[-1] + i] = offset[-1] + i, b
        offset.append(offset[-1] + len(taken[e]))
    return expert, weight, row, column, torch.tensor(offset, dtype=torch.int32)


def route_gradient(logits, expert, d_weight, normalise):
    """Through the softmax's Jacobian, in 64 bits, for the given choices."""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    live = expert >= 0
    at = expert.clamp(min=0).long()
    chosen = torch.zeros(x.shape, dtype=torch.bool, device=x.device)
    for j in range(len(at)):
        chosen |= torch.zeros_like(chosen).scatter_(0, at[j:j + 1], live[j:j + 1])
    d = torch.zeros_like(x).scatter_add_(0, at, torch.where(live, d_weight.double(), 0.0))
    y = x if normalise == "all" else torch.where(chosen, x, -math.inf)
    best = y.max(0).values
    p = torch.where(y == -math.inf, 0.0, torch.exp(y - torch.where(best == -math.inf, 0.0, best)))
    p = p / p.sum(0).clamp(min=1e-300)
    return p * (d - (p * d).sum(0))


def gather(x, row):
    k, batch = row.shape
    out = torch.zeros((k * batch, x.shape[0]), dtype=torch.float64, device=x.device)
    for j in range(k):
        on = torch.nonzero(row[j] >= 0).flatten()
        out[row[j, on].long()] = x[:, on].double().t()
    return out


def combine(rows, row, weight):
    k, batch = row.shape
    y = torch.zeros((batch, rows.shape[1]), dtype=torch.float64, device=rows.device)
    for j in range(k):
        on = torch.nonzero(row[j] >= 0).flatten()
        w = 1.0 if weight is None else weight[j, on].double()[:, None]
        y[on] += w * rows[row[j, on].long()].double()
    return y.t()


def activate(z, name, scalars=()):
    s0, s1 = (list(scalars) + [0.0, 0.0])[:2]
    return {
        None: lambda v: v,
        "ReLU": lambda v: torch.where(v > 0, v, 0.0),
        "LeakyReLU": lambda v: torch.where(v > 0, v, s0 * v),
        "ELU": lambda v: torch.where(v > 0, v, s0 * torch.expm1(v)),
        "SELU": lambda v: 1.0507009873554804934 * torch.where(v > 0, v, 1.6732632423543772848 * torch.expm1(v)),
        "GELU": lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2.0)),
        "SiLU": lambda v: v * torch.sigmoid(v),
        "Sigmoid": torch.sigmoid,
        "Tanh": torch.tanh,
        "Softplus": lambda v: torch.logaddexp(torch.zeros_like(v), s0 * v) / s0,
        "HardSigmoid": lambda v: (s0 * v + s1).clamp(0.0, 1.0),
        "HardSwish": lambda v: v * (v + 3.0).clamp(0.0, 6.0) / 6.0,
        "Mish": lambda v: v * torch.tanh(torch.logaddexp(torch.zeros_like(v), v)),
    }[name](z)


def product(rows, weights, offset, bias=None):
    """(result before the activation, sum of |a||b| of every element)."""
    edge = offset.tolist()
    shape = (rows.shape[0], weights.shape[2])
    y = torch.zeros(shape, dtype=torch.float64, device=rows.device)
    size = torch.zeros_like(y)
    for e in range(weights.shape[0]):
        lo, hi = edge[e], edge[e + 1]
        if hi > lo:
            a, w = rows[lo:hi].double(), weights[e].double()
            y[lo:hi] = a @ w
            size[lo:hi] = a.abs() @ w.abs()
            if bias is not None:
                y[lo:hi] += bias[e].double()
                size[lo:hi] += bias[e].double().abs()
    return y, size


def product_gradient(d, rows, weights, offset):
    """((d_rows, size), (d_weights, size), (d_bias, size))."""
    edge = offset.tolist()
    zero = lambda shape: torch.zeros(shape, dtype=torch.float64, device=rows.device)  # noqa: E731
    dr, sr, dw, sw = zero(rows.shape), zero(rows.shape), zero(weights.shape), zero(weights.shape)
    db, sb = zero((weights.shape[0], weights.shape[2])), zero((weights.shape[0], weights.shape[2]))
    for e in range(weights.shape[0]):
        lo, hi = edge[e], edge[e + 1]
        if hi > lo:
            g, a, w = d[lo:hi].double(), rows[lo:hi].double(), weights[e].double()
            dr[lo:hi], sr[lo:hi] = g @ w.t(), g.abs() @ w.abs().t()
            dw[e], sw[e] = a.t() @ g, a.abs().t() @ g.abs()
            db[e], sb[e] = g.sum(0), g.abs().sum(0)
    return (dr, sr), (dw, sw), (db, sb)


def sum_bound(want, size, terms, dtype):
    """Bound of a sum of `terms` products held in fp32 and rounded once to `dtype`.

    Each product and addition is off by at most one unit of fp32 (2^-23: the
    matrix units may truncate), relative to a partial sum that is at most
    `size`; the final rounding by half a unit of the result's type.  fp16 results
    below its normal range are off by half its smallest step, 2^-25.
    """
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -140
    return ULP[dtype] * want.abs() + (1.0 + ULP[dtype]) * (2.0 * U32 * (terms + 4) * size) + tiny


def check_sum(got, want, size, terms, what=""):
    over = ((got.double() - want).abs() - sum_bound(want, size, terms, got.dtype)).max().item() if got.numel() else 0.0
    assert over <= 0.0, f"{what}: {over:.3e} over the bound of {terms} terms"
