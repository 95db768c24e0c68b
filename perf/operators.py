"""Measured cases of the mixture-of-experts operators.

Four operators, in the order a mixture uses them:

  route    softmax top-k choice of experts for every batch column of feature-major logits
           [experts, batch], with the expert-sorted row order that the product works on; gradient
  columns  feature-major columns [features, batch] to expert-sorted rows [rows, features], the weighted
           combination back to columns, and the gradients of both
  product  rows times their expert's weights [experts, inputs, outputs], ragged groups; forward with Bias and
           activation, backward with the gradients of rows, weights and biases
  clip     norm over all gradient tensors together, and the clipped gradients packed into one flat vector

With `own` false, run() computes them with elementary torch operations in 32 bits, rounded once at the end;
with `own` true it calls ponni_b200.
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_NONE = float("-inf")


# ------------------------------------------------------------------ cases ----
def listed():
    return [
        # One column of a running simulation asks for its experts: latency only.
        {"name": "route one column", "op": "route", "experts": 16, "top_k": 2, "batch": 1, "dtype": "f32",
         "normalise": "selected", "masked": False, "backward": False},
        # A training batch with some experts masked off (and columns without any), choice and gradient.
        {"name": "route training batch", "op": "route", "experts": 64, "top_k": 4, "batch": 131072, "dtype": "f32",
         "normalise": "all", "masked": True, "backward": True},
        # A large batch of 256-feature columns (the wide chain's width) is brought into expert order.
        {"name": "gather wide columns", "op": "columns", "direction": "gather", "features": 256, "batch": 1048576,
         "experts": 8, "top_k": 2, "dtype": "bf16", "masked": False},
        # The gradient of the combination, odd feature and column counts, columns that no expert took.
        {"name": "combine gradient odd", "op": "columns", "direction": "combine_backward", "features": 1001,
         "batch": 49999, "experts": 12, "top_k": 3, "dtype": "f32", "masked": True},
        # One token served by two of 64 experts: the two experts' weights are read for one row each.
        {"name": "product one token", "op": "product", "direction": "forward", "rows": 2, "experts": 64,
         "inputs": 2048, "outputs": 1024, "dtype": "bf16", "bias": False, "activation": "silu", "masked": False},
        # A serving batch: a handful of rows for each expert, bound by the weights.
        {"name": "product serving batch", "op": "product", "direction": "forward", "rows": 384, "experts": 64,
         "inputs": 1024, "outputs": 2048, "dtype": "f16", "bias": True, "activation": "gelu", "masked": False},
        # A long batch: compute-bound forward.
        {"name": "product long batch", "op": "product", "direction": "forward", "rows": 32768, "experts": 32,
         "inputs": 2048, "outputs": 2048, "dtype": "bf16", "bias": True, "activation": "silu", "masked": False},
        # A training batch's gradients of rows, weights and biases.
        {"name": "product gradient", "op": "product", "direction": "backward", "rows": 16384, "experts": 16,
         "inputs": 2048, "outputs": 1024, "dtype": "bf16", "bias": True, "activation": "none", "masked": False},
        # Emulator experts of the wide chain's width over a very large batch: bound by the rows' traffic.
        {"name": "product emulator width", "op": "product", "direction": "forward", "rows": 1048576, "experts": 8,
         "inputs": 256, "outputs": 256, "dtype": "bf16", "bias": True, "activation": "silu", "masked": False},
        # Gradients in single precision with odd widths, some rows in no group.
        {"name": "product gradient f32 odd", "op": "product", "direction": "backward", "rows": 20011, "experts": 5,
         "inputs": 301, "outputs": 257, "dtype": "f32", "bias": True, "activation": "none", "masked": True},
        # The many small tensors of a set of small networks.
        {"name": "clip small tensors", "op": "clip", "tensors": 300, "total": 2000003, "dtype": "f32", "norm": 3.0},
        # The gradients of a large mixture, weights in bfloat16 and the rest in single precision.
        {"name": "clip large mixed", "op": "clip", "tensors": 200, "total": 150000000, "dtype": "mixed", "norm": 3.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ones' ranges: sizes over their logarithm, odd ones among them."""
    most = max(max(w["bytes"] / 6e12, w["flops"] / 1e15) for w in map(work, listed()))
    while True:
        op = rng.choice(["route", "columns", "product", "product", "clip"])
        if op == "route":
            experts = _log(rng, 4, 256)
            case = {"op": op, "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                    "batch": _log(rng, 1, 262144), "dtype": rng.choice(["f32", "f16", "bf16"]),
                    "normalise": rng.choice(["selected", "all"]), "masked": rng.random() < 0.5,
                    "backward": rng.random() < 0.5}
        elif op == "columns":
            experts = _log(rng, 4, 128)
            case = {"op": op, "direction": rng.choice(["gather", "combine", "gather_backward", "combine_backward"]),
                    "features": _log(rng, 16, 4096), "batch": _log(rng, 1, 1048576), "experts": experts,
                    "top_k": rng.randint(1, min(4, experts)), "dtype": rng.choice(["f32", "f16", "bf16"]),
                    "masked": rng.random() < 0.5}
        elif op == "product":
            direction = rng.choice(["forward", "forward", "backward"])
            step = rng.choice([1, 8, 64])
            case = {"op": op, "direction": direction, "rows": _log(rng, 1, 1048576), "experts": _log(rng, 1, 64),
                    "inputs": step * max(1, _log(rng, 16, 4096) // step),
                    "outputs": step * max(1, _log(rng, 16, 4096) // step),
                    "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]), "bias": rng.random() < 0.5,
                    "activation": rng.choice(["none", "relu", "silu", "gelu"]) if direction == "forward" else "none",
                    "masked": rng.random() < 0.3}
        else:
            tensors = _log(rng, 1, 600)
            case = {"op": op, "tensors": tensors, "total": tensors * _log(rng, 1, 200000),
                    "dtype": rng.choice(["f32", "f16", "bf16", "mixed"]), "norm": rng.choice([0.5, 3.0, 3.0])}
        w = work(case)
        if 3072 in case.values():
            continue
        if max(w["bytes"] / 6e12, w["flops"] / 1e15 * (6 if case["dtype"] == "f32" else 1)) <= most:
            return case


def work(case):
    z = _SIZE.get(case["dtype"], 3)
    if case["op"] == "route":
        e, k, b = case["experts"], case["top_k"], case["batch"]
        moved = e * b * z + k * b * (3 * 4 + 4) + 4 * (e + 1)  # logits; expert, weight, row and column; offsets
        flops = 3.0 * e * b
        if case["backward"]:
            moved += 2 * e * b * z + k * b * 12
            flops += 6.0 * e * b
        return {"bytes": moved, "flops": flops}
    if case["op"] == "columns":
        f, b, k = case["features"], case["batch"], case["top_k"]
        columns, rows, index = f * b * z, f * b * k * z, 8 * k * b
        if case["direction"] == "combine_backward":
            return {"bytes": columns + 2 * rows + 2 * index, "flops": 3.0 * f * b * k}
        return {"bytes": columns + rows + index, "flops": 2.0 * f * b * k}
    if case["op"] == "product":
        r, e, n, m = case["rows"], case["experts"], case["inputs"], case["outputs"]
        used = min(e, r)  # experts whose weights are read
        if case["direction"] == "forward":
            moved = (r * n + r * m + used * n * m + (used * m if case["bias"] else 0)) * z + 4 * (e + 1)
            return {"bytes": moved, "flops": 2.0 * r * n * m}
        moved = (2 * r * n + r * m + used * n * m + e * n * m + (e * m if case["bias"] else 0)) * z + 4 * (e + 1)
        return {"bytes": moved, "flops": 4.0 * r * n * m}
    n = case["total"]
    return {"bytes": n * (z + (4 if case["dtype"] in ("f32", "mixed") else z)), "flops": 3.0 * n}


# ----------------------------------------------------------------- inputs ----
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _logits(case, g):
    x = 1.5 * torch.randn(case["experts"], case["batch"], generator=g, device="cuda")
    x = x.to(_TYPES[case["dtype"]])
    if case["masked"]:
        off = torch.rand(x.shape, generator=g, device="cuda") < 0.15
        x.masked_fill_(off, _NONE)
        x[:, 5::97] = _NONE  # columns that no expert may take
        x[:, 7::101] = torch.finfo(x.dtype).min  # masks of the type's lowest value, every expert alike
    return x


def _sizes(case):
    """Element counts of the gradient tensors: fixed by the case, spread over a factor of about a hundred."""
    rng = random.Random(case["tensors"] * 1000003 + case["total"])
    share = [math.exp(rng.uniform(0.0, 4.6)) for _ in range(case["tensors"])]
    spare = case["total"] - case["tensors"]
    sizes = [1 + int(spare * s / sum(share)) for s in share]
    sizes[-1] += case["total"] - sum(sizes)
    return sizes


def _counts(case, g):
    """Rows of each expert: uneven, the second expert without any where there are several; and the rows in a group."""
    e, rows = case["experts"], case["rows"]
    used = rows - rows // 50 if case["masked"] else rows
    share = torch.exp(0.4 * torch.randn(e, generator=g, device="cuda", dtype=torch.float64))
    if e > 2:
        share[1] = 0.0
    edge = torch.round(torch.cumsum(share, 0) / share.sum() * used).to(torch.int32)
    if rows < e:  # a few rows: each of them to an expert of its own
        took = torch.randperm(e, generator=g, device="cuda")[:used]
        edge = torch.zeros(e, dtype=torch.int32, device="cuda").index_fill_(0, took, 1).cumsum(0).to(torch.int32)
    return torch.cat([torch.zeros(1, dtype=torch.int32, device="cuda"), edge])


def prepare(case, seed):
    g = _generator(seed)
    state = {"case": case}
    if case["op"] == "route":
        state["logits"] = _logits(case, g)
        state["d_weight"] = torch.randn(case["top_k"], case["batch"], generator=g, device="cuda")
    elif case["op"] == "columns":
        t = _TYPES[case["dtype"]]
        f, b, k = case["features"], case["batch"], case["top_k"]
        routed = _route_plain(_logits(dict(case, dtype="f32"), g), k, "selected")
        state.update(routed)
        if case["direction"] in ("gather", "combine_backward"):
            state["x"] = torch.randn(f, b, generator=g, device="cuda", dtype=t)
        if case["direction"] != "gather":
            state["rows"] = torch.randn(b * k, f, generator=g, device="cuda", dtype=t)
    elif case["op"] == "product":
        t = _TYPES[case["dtype"]]
        r, e, n, m = case["rows"], case["experts"], case["inputs"], case["outputs"]
        state["offset"] = _counts(case, g)
        state["most"] = int((state["offset"][1:] - state["offset"][:-1]).max())  # the largest group, for the plain form
        state["rows"] = torch.randn(r, n, generator=g, device="cuda", dtype=t)
        state["weights"] = torch.randn(e, n, m, generator=g, device="cuda", dtype=t).mul_(n ** -0.5)
        state["bias"] = torch.randn(e, m, generator=g, device="cuda", dtype=t).mul_(0.1) if case["bias"] else None
        if case["direction"] == "backward":
            state["d_out"] = torch.randn(r, m, generator=g, device="cuda", dtype=t)
    else:
        scale = case["norm"] / math.sqrt(case["total"])
        kinds = ["bf16", "f32"] if case["dtype"] == "mixed" else [case["dtype"]]
        state["gradients"] = [(scale * torch.randn(n, generator=g, device="cuda")).to(_TYPES[kinds[i % len(kinds)]])
                              for i, n in enumerate(_sizes(case))]
        flat = torch.float32 if case["dtype"] == "mixed" else _TYPES[case["dtype"]]
        state["flat"] = torch.empty(case["total"], device="cuda", dtype=flat)
        if own:  # the handle that a training program makes once over its gradient buffers
            import ponni_b200 as pb
            state["set"] = pb.GradientSet(state["gradients"])
    return state


# ------------------------------------------------------------- plain forms ----
def _from_best(x, best):
    """exp(x - best), a value equal to the best (an infinite one too) giving 1."""
    return torch.where(x == best, 1.0, torch.exp(x - best))


def _route_plain(logits, top_k, normalise):
    experts, batch = logits.shape
    x = logits.float()
    x = torch.where(torch.isnan(x), _NONE, x)
    order = torch.sort(x, dim=0, descending=True, stable=True)
    top, expert = order.values[:top_k], order.indices[:top_k]
    live = top > _NONE
    best = top[:1]
    weight = torch.where(live, _from_best(top, best), 0.0)
    if normalise == "selected":
        total = weight.sum(0)
    else:
        total = torch.where(x > _NONE, _from_best(x, best), 0.0).sum(0)
    weight = torch.where(live, weight / total, 0.0)
    key = torch.where(live, expert, experts).t().reshape(-1)
    by_row = torch.sort(key, stable=True).indices
    n = top_k * batch
    place = torch.arange(n, device=x.device)
    row = torch.empty_like(by_row).index_copy_(0, by_row, place).reshape(batch, top_k).t()
    count = torch.zeros(experts + 1, dtype=torch.int64, device=x.device).index_add_(0, key, torch.ones_like(key))
    offset = torch.cat([count.new_zeros(1), torch.cumsum(count[:experts], 0)])
    i32 = torch.int32
    return {"expert": torch.where(live, expert, -1).to(i32), "weight": weight,
            "row": torch.where(live, row, -1).to(i32).contiguous(),
            "column": torch.where(place < offset[-1], by_row // top_k, -1).to(i32), "offset": offset.to(i32)}


def _route_backward_plain(logits, routed, d_weight, normalise):
    x = logits.float()
    x = torch.where(torch.isnan(x), _NONE, x)
    live = routed["expert"] >= 0
    w, g = routed["weight"], torch.where(live, d_weight, 0.0)
    mean = (w * g).sum(0)
    at = routed["expert"].clamp(min=0).long()
    if normalise == "selected":
        return torch.zeros_like(x).scatter_add_(0, at, w * (g - mean)).to(logits.dtype)
    best = x.max(0, keepdim=True).values
    p = torch.where(x > _NONE, _from_best(x, best), 0.0)
    p = p / p.sum(0).clamp(min=1.0)  # the best expert alone gives 1: only a column without any has less
    return (-p * mean).scatter_add_(0, at, w * g).to(logits.dtype)


def _columns_plain(s):
    direction, k = s["case"]["direction"], s["case"]["top_k"]
    column, row, weight = s["column"].long(), s["row"].long(), s["weight"]
    live = row >= 0
    if direction in ("gather", "combine_backward"):
        of_column = s["x"].float().t().contiguous()
        by_row = of_column[column.clamp(min=0)]
        by_row = torch.where((column >= 0)[:, None], by_row, 0.0)
        if direction == "gather":
            return by_row.to(s["x"].dtype)
        n = row.numel()
        of_row = torch.zeros(n + 1, device=row.device).index_copy_(0, torch.where(live, row, n).reshape(-1),
                                                                 torch.where(live, weight, 0.0).reshape(-1))
        d_rows = (by_row * of_row[:n, None]).to(s["rows"].dtype)
        took = s["rows"].float()[row.clamp(min=0)]
        d_weight = torch.where(live, (took * of_column[None]).sum(-1), 0.0)
        return {"rows": d_rows, "weight": d_weight}
    took = torch.where(live[..., None], s["rows"].float()[row.clamp(min=0)], 0.0)
    if direction == "combine":
        took = took * weight[..., None]
    return took.sum(0).t().contiguous().to(s["rows"].dtype)


def _activate(x, name):
    if name == "relu":
        return torch.where(x > 0, x, 0.0)
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    return x


def _product_plain(s):
    """The groups side by side, each filled up with zero rows to the largest one's length."""
    case, most = s["case"], max(1, s["most"])
    rows, offset, w = s["rows"].float(), s["offset"].long(), s["weights"].float()
    e, t = case["experts"], s["rows"].dtype
    place = torch.arange(case["rows"], device=rows.device)
    expert = torch.searchsorted(offset[1:].contiguous(), place, right=True)
    live = expert < e
    at = torch.where(live, expert * most + place - offset[expert], e * most)

    def grouped(v):
        v = torch.where(live[:, None], v, 0.0)
        return v.new_zeros(e * most + 1, v.shape[1]).index_copy_(0, at, v)[:-1].reshape(e, most, -1)

    def ungrouped(v):
        v = v.reshape(e * most, -1)
        return torch.where(live[:, None], v[at.clamp(max=e * most - 1)], 0.0)

    if case["direction"] == "forward":
        z = torch.bmm(grouped(rows), w)
        if s["bias"] is not None:
            z = z + s["bias"].float()[:, None, :]
        return ungrouped(_activate(z, case["activation"])).to(t)
    x, d = grouped(rows), grouped(s["d_out"].float())
    return {"rows": ungrouped(torch.bmm(d, w.transpose(1, 2))).to(t), "weights": torch.bmm(x.transpose(1, 2), d).to(t),
            "bias": d.sum(1).to(t) if case["bias"] else None}


def _clip_plain(s):
    g = [v.float() for v in s["gradients"]]
    norm = torch.sqrt(torch.stack([(v * v).sum() for v in g]).sum())
    scale = torch.where(torch.isfinite(norm) & (norm > 1.0), 1.0 / norm, 1.0)
    return {"norm": norm, "flat": torch.cat([(v * scale).to(s["flat"].dtype) for v in g])}


# -------------------------------------------------------------------- run ----
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "route":
        out = _route_plain(state["logits"], case["top_k"], case["normalise"])
        if case["backward"]:
            out["logits"] = _route_backward_plain(state["logits"], out, state["d_weight"], case["normalise"])
        return out
    return {"columns": _columns_plain, "product": _product_plain, "clip": _clip_plain}[case["op"]](state)


def _run_own(state, case):
    import ponni_b200 as pb
    if case["op"] == "route":
        r = pb.route_columns(state["logits"], case["top_k"], normalise=case["normalise"])
        out = {"expert": r.expert, "weight": r.weight, "row": r.row, "column": r.column, "offset": r.offset}
        if case["backward"]:
            out["logits"] = pb.route_columns_backward(state["logits"], r, state["d_weight"],
                                                      normalise=case["normalise"])
        return out
    if case["op"] == "columns":
        r = pb.Routing(state["expert"], state["weight"], state["row"], state["column"], state["offset"])
        direction = case["direction"]
        if direction == "gather":
            return pb.gather_columns(state["x"], r)
        if direction == "combine":
            return pb.combine_rows(state["rows"], r)
        if direction == "gather_backward":
            return pb.gather_columns_backward(state["rows"], r)
        d_rows, d_weight = pb.combine_rows_backward(state["x"], state["rows"], r)
        return {"rows": d_rows, "weight": d_weight}
    if case["op"] == "product":
        if case["direction"] == "forward":
            act = {"none": None, "relu": pb.Relu, "silu": pb.Silu, "gelu": pb.Gelu}[case["activation"]]
            return pb.expert_product(state["rows"], state["weights"], state["offset"], bias=state["bias"],
                                     activation=act(case["outputs"]) if act else None)
        d_rows, d_weights, d_bias = pb.expert_product_backward(state["d_out"], state["rows"], state["weights"],
                                                               state["offset"], bias=case["bias"])
        return {"rows": d_rows, "weights": d_weights, "bias": d_bias}
    norm = state["set"].clip(1.0, out=state["flat"])
    return {"norm": norm, "flat": state["flat"]}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    """The operators' definitions in 64 bits; whole numbers have no entry."""
    state = prepare(case, seed)
    return {"route": _route_exact, "columns": _columns_exact, "product": _product_exact, "clip": _clip_exact}[
        case["op"]](case, state)


def _softmax64(x):
    """Softmax over the first axis; a column of -inf alone gives zeros."""
    x = x.double()
    e = torch.exp(x - x.amax(0, keepdim=True).clamp(min=-1.7e308))
    return e / e.sum(0).clamp(min=1e-300)


def _route_exact(case, s):
    k, x = case["top_k"], s["logits"]
    p = _softmax64(x)
    # The chosen set: a rank counts the experts that come before this one (larger logit, or the same and a lower index).
    chosen, alive = [], torch.isfinite(x)
    rest = torch.where(alive, x.double(), _NONE)
    weight = torch.zeros(k, case["batch"], dtype=torch.float64, device=x.device)
    for i in range(k):
        top = rest.amax(0)
        first = ((rest == top) & (rest > _NONE)).double().cumsum(0)
        pick = (first == 1) & (rest == top) & (rest > _NONE)
        weight[i] = (p * pick).sum(0)
        chosen.append(pick)
        rest = rest.masked_fill(pick, _NONE)
    if case["normalise"] == "selected":
        weight = weight / weight.sum(0).clamp(min=1e-300)
    out = {"expert": None, "weight": weight, "row": None, "column": None, "offset": None}
    if case["backward"]:
        g = s["d_weight"].double()
        d_p = sum(pick * g[i] for i, pick in enumerate(chosen))  # gradient at the softmax's values
        if case["normalise"] == "selected":
            p = p * sum(c.double() for c in chosen)
            p = p / p.sum(0).clamp(min=1e-300)
        out["logits"] = p * (d_p - (p * d_p).sum(0))
    return out


def _columns_exact(case, s):
    f, b, k = case["features"], case["batch"], case["top_k"]
    direction = case["direction"]
    if f * b * k > 1e9:
        return None
    row, weight = s["row"].long(), s["weight"].double()
    if direction == "gather":
        rows = torch.zeros(b * k, f, dtype=torch.float64, device="cuda")
        for i in range(k):
            on = torch.nonzero(row[i] >= 0).flatten()
            rows[row[i, on]] = s["x"][:, on].double().t()
        return rows
    if direction == "combine_backward":
        d_rows = torch.zeros(b * k, f, dtype=torch.float64, device="cuda")
        d_weight = torch.zeros(k, b, dtype=torch.float64, device="cuda")
        for i in range(k):
            on = torch.nonzero(row[i] >= 0).flatten()
            d = s["x"][:, on].double().t()
            d_rows[row[i, on]] = d * weight[i, on, None]
            d_weight[i, on] = torch.einsum("rf,rf->r", s["rows"][row[i, on]].double(), d)
        return {"rows": d_rows, "weight": d_weight}
    y = torch.zeros(b, f, dtype=torch.float64, device="cuda")
    for i in range(k):
        on = torch.nonzero(row[i] >= 0).flatten()
        took = s["rows"][row[i, on]].double()
        y[on] += took * weight[i, on, None] if direction == "combine" else took
    return y.t().contiguous()


def _product_exact(case, s):
    if work(case)["flops"] > 6e11:
        return None
    edge = s["offset"].tolist()
    x, w = s["rows"], s["weights"]
    if case["direction"] == "forward":
        y = torch.zeros(case["rows"], case["outputs"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            lo, hi = edge[e], edge[e + 1]
            if hi > lo:
                z = x[lo:hi].double() @ w[e].double()
                if case["bias"]:
                    z += s["bias"][e].double()
                name = case["activation"]
                y[lo:hi] = {"none": lambda v: v, "relu": lambda v: v.clamp(min=0),
                            "silu": lambda v: v * torch.sigmoid(v),
                            "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2.0))}[name](z)
        return y
    d = s["d_out"]
    d_rows = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    d_w = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    d_b = torch.zeros(case["experts"], case["outputs"], dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        lo, hi = edge[e], edge[e + 1]
        if hi > lo:
            g = d[lo:hi].double()
            d_rows[lo:hi] = g @ w[e].double().t()
            d_w[e] = x[lo:hi].double().t() @ g
            d_b[e] = g.sum(0)
    return {"rows": d_rows, "weights": d_w, "bias": d_b if case["bias"] else None}


def _clip_exact(case, s):
    flat = torch.cat([v.double() for v in s["gradients"]])
    norm = torch.linalg.vector_norm(flat)
    return {"norm": norm, "flat": flat / max(1.0, float(norm))}
