"""Mixture-of-experts operators on the GPU against plain 64-bit forms (tests/expert_ref.py).

Tolerances: a sum of n products in fp32 is off by at most (n + 4) units of 2^-23
of the sum of magnitudes, plus the rounding to the result's type
(expert_ref.sum_bound).  Choices, rows and offsets are whole numbers and equal.
Routing weights: exp and the division are off by a few units (2^-22 relative) and
a sum of n exponentials by n units.
"""
import math

import pytest

torch = pytest.importorskip("torch")

import ponni_b200 as pb  # noqa: E402
from tests import expert_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DT = R.DTYPES
INF = math.inf


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)




# ------------------------------------------------------------------- route ----
def logits_of(experts, batch, dtype, seed, kind):
    g = gen(seed)
    x = randn(g, experts, batch, dtype=dtype)
    if kind == "ties":
        x = (x * 2).round() / 2
    if kind == "masked":
        x.masked_fill_(torch.rand(x.shape, generator=g, device="cuda") < 0.4, -INF)
        x[:, ::5] = -INF
        x[:, 1::7] = torch.finfo(dtype).min
        x[0, 2::9] = float("nan")
        x[:, 3::11] = float("nan")
    if kind == "infinite":
        x[experts // 2, ::2] = INF
        x[experts - 1, ::4] = INF
    if kind == "equal":
        x.zero_()
    return x


@pytest.mark.parametrize("kind", ["plain", "ties", "masked", "infinite", "equal"])
@pytest.mark.parametrize("normalise", ["selected", "all"])
@pytest.mark.parametrize("experts,top_k,batch", [(1, 1, 1), (2, 2, 3), (5, 3, 257), (8, 8, 31), (16, 2, 1000),
                                                 (130, 6, 513), (64, 4, 4099), (1024, 7, 300), (33, 5, 1)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_route(experts, top_k, batch, normalise, kind, dt):
    x = logits_of(experts, batch, DT[dt], experts * 7 + batch, kind)
    r = pb.route_columns(x, top_k, normalise=normalise)
    want = R.route(x, top_k, normalise)
    for name, got, ref in zip(("expert", "row", "column", "offset"), (r.expert, r.row, r.column, r.offset),
                              (want[0], want[2], want[3], want[4])):
        assert torch.equal(got.cpu(), ref), name
    err = (r.weight.cpu().double() - want[1]).abs()
    assert (err <= want[1] * (experts + 8) * 2.0 ** -22 + 1e-38).all()
    d_weight = randn(gen(3), top_k, batch)
    d_weight[:, ::3] *= 10
    d_weight = torch.where(r.expert >= 0, d_weight, float("nan"))  # a choice that was not made is not read
    if kind == "infinite":
        return  # the softmax has no gradient there
    d = pb.route_columns_backward(x, r, d_weight, normalise=normalise)
    ref = R.route_gradient(x, r.expert, d_weight, normalise)
    scale = ref.abs() + torch.where(r.expert >= 0, d_weight, 0.0).abs().double().sum(0)
    bound = R.ULP[x.dtype] * ref.abs() + (experts + top_k + 12) * 2.0 ** -21 * scale + 2.0 ** -25
    assert ((d.double() - ref).abs() <= bound).all()


def test_route_many_blocks_and_strides():
    g = gen(5)
    wide = randn(g, 24, 400_001)
    x = wide[:, 1:]  # row stride 400001, rows not aligned to 16 bytes
    r = pb.route_columns(x, 3)
    key = torch.where(r.expert >= 0, r.expert, 24).t().reshape(-1).long()
    by_row = torch.sort(key, stable=True).indices
    assert torch.equal(r.column.long(), by_row // 3)
    assert torch.equal(r.row.t().reshape(-1).long()[by_row], torch.arange(key.numel(), device="cuda"))
    count = torch.bincount(key, minlength=24)
    assert torch.equal(r.offset.long(), torch.cat([count.new_zeros(1), count.cumsum(0)]))
    top = torch.sort(x, dim=0, descending=True, stable=True).indices[:3]
    assert torch.equal(r.expert.long(), top)


def test_route_gradient_by_differences():
    g = gen(8)
    x = randn(g, 12, 64)
    d_weight = randn(g, 4, 64)
    for normalise in ("selected", "all"):
        r = pb.route_columns(x, 4, normalise=normalise)
        d = pb.route_columns_backward(x, r, d_weight, normalise=normalise)
        h = 1e-2
        for e in range(12):
            step = torch.zeros_like(x)
            step[e] = h
            up, down = (pb.route_columns(x + s, 4, normalise=normalise) for s in (step, -step))
            same = (up.expert == r.expert).all(0) & (down.expert == r.expert).all(0)  # the choice is not differentiable
            diff = ((up.weight - down.weight) * d_weight).sum(0) / (2 * h)
            # third derivative of a softmax entry at most 1, four entries of magnitude below 4: h^2/6 * 16, and 2^-22 / h
            assert same.float().mean() > 0.5
            assert (diff - d[e])[same].abs().max() <= 16 * h * h / 6 + 16 * 2.0 ** -22 / h


# ----------------------------------------------------------------- columns ----
def routing(experts, top_k, batch, seed, masked):
    x = logits_of(experts, batch, torch.float32, seed, "masked" if masked else "plain")
    return pb.route_columns(x, top_k)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("features,batch,top_k", [(1, 1, 1), (3, 5, 2), (64, 64, 2), (129, 65, 3), (257, 1000, 2),
                                                  (1001, 77, 8), (30, 4099, 1), (256, 3, 4), (4097, 2, 2)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_columns(features, batch, top_k, dt, masked):
    g = gen(features + batch)
    dtype = DT[dt]
    r = routing(max(top_k, 6), top_k, batch, 11, masked)
    used = int(r.offset[-1])
    x = randn(g, features, batch, dtype=dtype)
    if masked:
        x[:, ~(r.row >= 0).any(0)] = float("nan")  # columns that nobody chose
    rows = pb.gather_columns(x, r)
    assert torch.equal(rows.double(), R.gather(x, r.row))
    v = randn(g, batch * top_k, features, dtype=dtype)
    v[used:] = float("nan")  # unused rows
    y = pb.combine_rows(v, r)
    want = R.combine(v, r.row, r.weight)
    size = R.combine(v.abs(), r.row, r.weight)
    R.check_sum(y, want, size, top_k, "combine")
    back = pb.gather_columns_backward(v, r)
    R.check_sum(back, R.combine(v, r.row, None), R.combine(v.abs(), r.row, None), top_k, "gather gradient")
    d_y = randn(g, features, batch, dtype=dtype)
    if masked:
        d_y[:, ~(r.row >= 0).any(0)] = float("inf")
    d_rows, d_weight = pb.combine_rows_backward(d_y, v, r)
    by_row = R.gather(d_y, r.row)
    of_row = torch.zeros(batch * top_k, dtype=torch.float64, device="cuda")
    on = r.row >= 0
    of_row[r.row[on].long()] = r.weight[on].double()
    want = by_row * of_row[:, None]
    R.check_sum(d_rows, want, want.abs(), 1, "d_rows")
    dot = torch.zeros(top_k, batch, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(dot)
    prod = v.double() * by_row
    dot[on], mag[on] = prod.sum(1)[r.row[on].long()], prod.abs().sum(1)[r.row[on].long()]
    R.check_sum(d_weight, dot, mag, features, "d_weight")


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_columns_strided_and_offset(dt):
    g = gen(4)
    dtype = DT[dt]
    r = routing(5, 2, 333, 2, True)
    base = randn(g, 71, 337, dtype=dtype)
    x = base[1:, 3:336]  # rows of stride 337, starting off a 16-byte boundary
    want = R.gather(x, r.row)
    assert torch.equal(pb.gather_columns(x, r).double(), want)
    for pitch in (70, 71, 72, 75):
        buf = torch.full((666, pitch + 1), 7.0, dtype=dtype, device="cuda")
        out = buf[:, 1:71]
        assert pb.gather_columns(x, r, out=out) is out
        assert torch.equal(out.double(), want)
        assert (buf[:, 0] == 7).all() and (buf[:, 71:] == 7).all()  # nothing written beside the rows
    rows = randn(g, 666, 90, dtype=dtype)[:, 7:77]
    out = torch.full((70, 400), 3.0, dtype=dtype, device="cuda")
    pb.combine_rows(rows, r, out=out[:, 5:338])
    R.check_sum(out[:, 5:338], R.combine(rows, r.row, r.weight), R.combine(rows.abs(), r.row, r.weight), 2)
    assert (out[:, :5] == 3).all() and (out[:, 338:] == 3).all()


def test_columns_gradients_by_differences():
    """The combination is linear in the rows and in the weights: a finite difference has no truncation error."""
    g = gen(9)
    r = routing(6, 3, 50, 3, True)
    rows, d_y = randn(g, 150, 40), randn(g, 40, 50)
    d_rows, d_weight = pb.combine_rows_backward(d_y, rows, r)
    step = randn(g, 150, 40)
    step[int(r.offset[-1]):] = 0
    diff = ((pb.combine_rows(rows + step, r) - pb.combine_rows(rows - step, r)).double() * d_y.double()).sum() / 2
    want = (d_rows.double() * step.double()).sum()
    assert abs(diff - want) <= 1e-4 * (d_rows.double() * step.double()).abs().sum()
    dw = torch.where(r.expert >= 0, randn(g, 3, 50), 0.0)
    moved = [r._replace(weight=(r.weight + s * dw).contiguous()) for s in (1.0, -1.0)]
    diff = ((pb.combine_rows(rows, moved[0]) - pb.combine_rows(rows, moved[1])).double() * d_y.double()).sum() / 2
    want = (d_weight.double() * dw.double()).sum()
    assert abs(diff - want) <= 1e-4 * (d_weight.double() * dw.double()).abs().sum()
    x, d_r = randn(g, 40, 50), randn(g, 150, 40)
    sx = randn(g, 40, 50)
    diff = ((pb.gather_columns(x + sx, r) - pb.gather_columns(x - sx, r)).double() * d_r.double()).sum() / 2
    want = (pb.gather_columns_backward(d_r, r).double() * sx.double()).sum()
    assert abs(diff - want) <= 1e-4 * d_r.double().abs().sum()


# ----------------------------------------------------------------- product ----
def offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


GROUPS = {
    "one row": [1],
    "one group": [300],
    "empty ends": [0, 5, 0, 0, 130, 1, 0],
    "tile edges": [128, 127, 129, 256, 1, 64],
    "nothing": [0, 0, 0],
    "singles": [1] * 20,
    "long": [0, 1500, 3, 700],
}


@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("inputs,outputs", [(1, 1), (3, 5), (64, 64), (128, 256), (30, 10), (136, 72), (257, 301),
                                            (512, 384), (65, 1000)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_product(groups, inputs, outputs, dt):
    counts = GROUPS[groups]
    dtype, g = DT[dt], gen(inputs * 3 + outputs)
    e, extra = len(counts), 3
    n = sum(counts) + extra  # rows in no group
    off = offsets(counts)
    rows = randn(g, n, inputs, dtype=dtype)
    rows[n - extra:] = float("nan")
    w = randn(g, e, inputs, outputs, dtype=dtype) * inputs ** -0.5
    for i, c in enumerate(counts):
        if c == 0:
            w[i] = float("nan")  # an expert without rows is not read into any result
    b = randn(g, e, outputs, dtype=dtype)
    y = pb.expert_product(rows, w, off, bias=b)
    want, size = R.product(rows, w, off, b)
    R.check_sum(y, want, size, inputs + 1, "forward")
    y0 = pb.expert_product(rows, w, off)
    want, size = R.product(rows, w, off)
    R.check_sum(y0, want, size, inputs, "forward without bias")
    d = randn(g, n, outputs, dtype=dtype)
    d[n - extra:] = float("nan")
    got = pb.expert_product_backward(d, rows, w, off)
    ref = R.product_gradient(d, rows, w, off)
    R.check_sum(got[0], *ref[0], outputs, "d_rows")
    R.check_sum(got[1], *ref[1], max(counts), "d_weights")
    R.check_sum(got[2], *ref[2], max(counts), "d_bias")
    pb.check_operators()


@pytest.mark.parametrize("inputs,outputs", [(200, 24), (24, 200), (40, 40), (1200, 37), (128, 128), (72, 300)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_product_many_tiles_a_cta(inputs, outputs, dt):
    """Several tiles for every CTA, of widths that the tile shapes divide and do not."""
    g = gen(inputs + outputs)
    dtype = DT[dt]
    counts = [30_011, 0, 17_000, 129, 40_100]
    n, off = sum(counts), offsets(counts)
    rows, w = randn(g, n, inputs, dtype=dtype), randn(g, 5, inputs, outputs, dtype=dtype) * inputs ** -0.5
    b, d = randn(g, 5, outputs, dtype=dtype), randn(g, n, outputs, dtype=dtype)
    want, size = R.product(rows, w, off, b)
    R.check_sum(pb.expert_product(rows, w, off, bias=b), want, size, inputs + 1, "forward")
    ref = R.product_gradient(d, rows, w, off)
    for got, (want, size), terms in zip(pb.expert_product_backward(d, rows, w, off), ref, (outputs, max(counts), max(counts))):
        R.check_sum(got, want, size, terms, "gradient")
    pb.check_operators()


@pytest.mark.parametrize("counts", [[1, 2, 3, 5, 9, 16, 17, 0], [0, 33, 0], [8]])
@pytest.mark.parametrize("inputs,outputs", [(2500, 130), (1024, 128), (1027, 5), (130, 1000)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_product_few_rows(inputs, outputs, counts, dt):
    """A few rows of many inputs: sums split over K and over the blocks of a cluster."""
    g = gen(inputs)
    dtype = DT[dt]
    e, n, off = len(counts), sum(counts) + 1, offsets(counts)
    rows, w = randn(g, n, inputs, dtype=dtype), randn(g, e, inputs, outputs, dtype=dtype) * inputs ** -0.5
    b = randn(g, e, outputs, dtype=dtype)
    want, size = R.product(rows, w, off, b)
    R.check_sum(pb.expert_product(rows, w, off, bias=b), want, size, inputs + 1)
    pb.check_operators()


@pytest.mark.parametrize("layer", [pb.Relu, pb.LeakyRelu, pb.Elu, pb.Selu, pb.Gelu, pb.Silu, pb.Sigmoid, pb.Tanh,
                                   pb.Softplus, pb.HardSigmoid, pb.HardSwish, pb.Mish])
@pytest.mark.parametrize("counts", [[3, 0, 2], [200, 90, 300]])
def test_product_activation(layer, counts):
    g = gen(2)
    for dt in ("f32", "bf16"):
        dtype = DT[dt]
        rows, w = randn(g, sum(counts) + 2, 96, dtype=dtype), randn(g, 3, 96, 80, dtype=dtype) * 0.2
        b = randn(g, 3, 80, dtype=dtype)
        off = offsets(counts)
        act = layer(80)
        y = pb.expert_product(rows, w, off, bias=b, activation=act)
        z, size = R.product(rows, w, off, b)
        want = R.activate(z, act.label, act.scalar)
        want[sum(counts):] = 0.0
        # Every activation's slope is at most 1.8 (SELU); its own evaluation is off by a few units of its argument.
        bound = 1.8 * R.sum_bound(z, size, 97, torch.float32) + R.ULP[dtype] * want.abs() + 2.0 ** -20 * (1 + z.abs())
        assert ((y.double() - want).abs() <= bound).all(), (dt, ((y.double() - want).abs() - bound).max())


@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_product_strides_and_alignment(dt):
    g = gen(6)
    dtype = DT[dt]
    counts = [40, 0, 170]
    off = offsets(counts)
    for inputs, outputs in ((64, 128), (50, 70)):
        rows = randn(g, 211, inputs + 9, dtype=dtype)[1:, 3:3 + inputs]
        w = randn(g, 3, inputs + 2, outputs + 5, dtype=dtype)[:, 1:1 + inputs, 2:2 + outputs]
        b = randn(g, 3, outputs, dtype=dtype)
        buf = torch.full((210, outputs + 11), 5.0, dtype=dtype, device="cuda")
        out = buf[:, 5:5 + outputs]
        pb.expert_product(rows, w, off, bias=b, out=out)
        want, size = R.product(rows, w, off, b)
        R.check_sum(out, want, size, inputs + 1)
        assert (buf[:, :5] == 5).all() and (buf[:, 5 + outputs:] == 5).all()
        d = randn(g, 210, outputs + 3, dtype=dtype)[:, 1:1 + outputs]
        got = pb.expert_product_backward(d, rows, w, off)
        ref = R.product_gradient(d, rows, w, off)
        for a, (want, size), terms in zip(got, ref, (outputs, 170, 170)):
            R.check_sum(a, want, size, terms)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_product_keeps_groups_apart(dt):
    """NaN and infinity in one expert's rows, weights or gradients do not reach the others'."""
    g = gen(7)
    dtype = DT[dt]
    counts = [70, 60, 5, 200]
    off = offsets(counts)
    lo = [0, 70, 130, 135]
    rows, w, d = randn(g, 335, 72, dtype=dtype), randn(g, 4, 72, 88, dtype=dtype), randn(g, 335, 88, dtype=dtype)
    rows[70:130] = float("nan")
    rows[130, 0] = INF
    w[1] = INF
    d[75] = -INF
    b = torch.zeros(4, 88, dtype=dtype, device="cuda")
    y = pb.expert_product(rows, w, off, bias=b)
    dr, dw, db = pb.expert_product_backward(d, rows, w, off)
    for e in (0, 3):
        s = slice(lo[e], lo[e] + counts[e])
        want, size = R.product(rows[s], w[e:e + 1], offsets([counts[e]]))
        R.check_sum(y[s], want, size, 73)
        ref = R.product_gradient(d[s], rows[s], w[e:e + 1], offsets([counts[e]]))
        R.check_sum(dr[s], *ref[0], 88)
        R.check_sum(dw[e:e + 1], *ref[1], counts[e])
        R.check_sum(db[e:e + 1], *ref[2], counts[e])
    assert torch.isnan(y[70:130]).all()
    # an infinite value: the sums have the sign that its products give, the other rows stay finite
    assert torch.equal(y[130].float(), torch.where(w[2, 0].float() > 0, INF, -INF))
    assert torch.isfinite(y[131:135].float()).all()
    assert torch.equal(dw[2, 0].float(), torch.where(d[130].float() > 0, INF, -INF))
    assert torch.isfinite(dw[2, 1:].float()).all()


def test_product_large_values_f32():
    """Values near the ends of fp32's range."""
    off = offsets([2])
    for scale in (3.0e38, 1.0e-30):
        rows = torch.tensor([[scale, 0.0], [-scale, scale]], device="cuda").repeat(1, 8).contiguous()
        w = torch.zeros(1, 16, 24, device="cuda")
        w[0, 0, :] = torch.linspace(0.1, 0.9, 24)
        y = pb.expert_product(rows, w, off)
        want, size = R.product(rows, w, off)
        R.check_sum(y, want, size, 16)


def test_product_gradient_by_differences():
    """The product is linear in each argument: a finite difference has no truncation error."""
    g = gen(10)
    counts = [33, 0, 150, 1]
    off = offsets(counts)
    rows, w, d = randn(g, 184, 48), randn(g, 4, 48, 56), randn(g, 184, 56)
    b, sb = randn(g, 4, 56), randn(g, 4, 56)
    sr, sw = randn(g, 184, 48), randn(g, 4, 48, 56)
    dr, dw, db = pb.expert_product_backward(d, rows, w, off)
    for grad, step, up, down in ((dr, sr, (rows + sr, w, b), (rows - sr, w, b)), (dw, sw, (rows, w + sw, b), (rows, w - sw, b)),
                                 (db, sb, (rows, w, b + sb), (rows, w, b - sb))):
        f = [pb.expert_product(r_, w_, off, bias=b_).double() for r_, w_, b_ in (up, down)]
        diff = ((f[0] - f[1]) * d.double()).sum() / 2
        want = (grad.double() * step.double()).sum()
        assert abs(diff - want) <= 1e-5 * (grad.double() * step.double()).abs().sum()


def test_product_single_precision_keeps_single_precision():
    """fp32 products are as exact as fp32 arithmetic: errors near 2^-24 of the magnitudes, not bf16's or tf32's."""
    g = gen(12)
    off = offsets([500, 700])
    rows, w = randn(g, 1200, 1024), randn(g, 2, 1024, 320)
    y = pb.expert_product(rows, w, off)
    want, _ = R.product(rows, w, off)
    rms = lambda t: t.double().square().mean().sqrt().item()  # noqa: E731
    assert rms(y.double() - want) <= 1e-6 * rms(want)
    d = randn(g, 1200, 320)
    for got, (ref, _) in zip(pb.expert_product_backward(d, rows, w, off), R.product_gradient(d, rows, w, off)):
        assert rms(got.double() - ref) <= 1e-6 * rms(ref)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_product_outputs_not_needed(dt):
    g = gen(1)
    off = offsets([20, 30])
    rows, w, d = (randn(g, *s, dtype=DT[dt]) for s in ((50, 40), (2, 40, 24), (50, 24)))
    full = pb.expert_product_backward(d, rows, w, off)
    assert [v is None for v in pb.expert_product_backward(d, rows, w, off, bias=False, need_rows=False)] == [True, False, True]
    only = pb.expert_product_backward(d, rows, w, off, bias=False, need_weights=False)
    assert only[1] is None and only[2] is None and torch.equal(only[0], full[0])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_product_no_rows(dt):
    off = offsets([0, 0])
    rows, w = torch.empty(0, 32, dtype=DT[dt], device="cuda"), torch.ones(2, 32, 16, dtype=DT[dt], device="cuda")
    assert pb.expert_product(rows, w, off).shape == (0, 16)
    dr, dw, db = pb.expert_product_backward(torch.empty(0, 16, dtype=DT[dt], device="cuda"), rows, w, off)
    assert dr.shape == (0, 32) and not dw.any() and not db.any()


def test_offsets_out_of_order_are_reported():
    g = gen(1)
    rows, w = randn(g, 50, 16, dtype=torch.bfloat16), randn(g, 3, 16, 16, dtype=torch.bfloat16)
    pb.check_operators()
    for bad in ([0, 30, 20, 50], [0, 10, 20, 60], [-5, 10, 20, 50], [3, 10, 20, 50]):
        off = torch.tensor(bad, dtype=torch.int32, device="cuda")
        pb.expert_product(rows, w, off)
        with pytest.raises(pb.PonniError, match="ascending"):
            pb.check_operators()
        pb.expert_product_backward(rows, rows, w, off)
        with pytest.raises(pb.PonniError, match="ascending"):
            pb.check_operators()
        pb.check_operators()


def test_product_past_32_bit_offsets():
    """More than 2^31 elements of rows and of outputs."""
    n, f = 9_000_000, 256
    rows = torch.zeros(n, f, dtype=torch.bfloat16, device="cuda")
    g = gen(3)
    rows[-300:] = randn(g, 300, f, dtype=torch.bfloat16)
    w = randn(g, 2, f, f, dtype=torch.bfloat16)
    off = torch.tensor([0, n - 200, n], dtype=torch.int32, device="cuda")
    y = pb.expert_product(rows, w, off)
    want, size = R.product(rows[-300:], w, torch.tensor([0, 100, 300]))
    R.check_sum(y[-300:], want, size, f)
    assert not y[:-300].any()
    dr, dw, _ = pb.expert_product_backward(y, rows, w, off, bias=False)
    ref = R.product_gradient(y[-300:], rows[-300:], w, torch.tensor([0, 100, 300]))
    R.check_sum(dr[-300:], *ref[0], f)
    R.check_sum(dw, *ref[1], n)


# -------------------------------------------------------------------- clip ----
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [100_003], [7, 4096, 3, 20_000, 1] * 9, [3_000_001, 17, 2]])
@pytest.mark.parametrize("dts", [["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16", "f64"]])
def test_clip(sizes, dts):
    g = gen(sum(sizes))
    kinds = dict(DT, f64=torch.float64)
    make = lambda: [randn(g, n, dtype=kinds[dts[i % len(dts)]]) for i, n in enumerate(sizes)]  # noqa: E731
    grads = make()
    flat = torch.cat([v.double() for v in grads])
    norm = flat.norm().item()
    s = pb.GradientSet(grads)
    assert s.total == sum(sizes)
    ulp = dict(R.ULP)
    ulp[torch.float64] = 2.0 ** -53
    for max_norm in (2 * norm, norm / 3):
        scale = min(1.0, max_norm / norm)
        for dt in (torch.float32, torch.bfloat16, torch.float64):
            out = torch.full((s.total,), 9.0, dtype=dt, device="cuda")
            got = s.clip(max_norm, out=out)
            assert abs(got.item() - norm) <= 2.0 ** -22 * norm
            # the scale is held in fp32 unless both types are fp64: one unit, the product another
            assert ((out.double() - flat * scale).abs() <= (ulp[dt] + 2.0 ** -22) * flat.abs() * scale + 2.0 ** -25).all()
    assert torch.equal(torch.cat([v.double() for v in grads]), flat)  # packing leaves the gradients alone
    s.clip(2 * norm)
    assert torch.equal(torch.cat([v.double() for v in grads]), flat)
    before = [v.clone() for v in grads]
    s.clip(norm / 3)
    for a, b in zip(grads, before):
        want = b.double() / 3
        assert ((a.double() - want).abs() <= (ulp[a.dtype] + 2.0 ** -22) * want.abs() + 2.0 ** -25).all()


def test_clip_of_nothing():
    s = pb.GradientSet([torch.empty(0, device="cuda"), torch.empty(0, device="cuda", dtype=torch.float16)])
    assert s.clip(1.0).item() == 0.0
    assert s.clip(1.0, out=torch.empty(0, device="cuda")).item() == 0.0


def test_clip_unaligned_and_functional():
    g = gen(2)
    base = randn(g, 5000)
    parts = [base[1:1001].clone()[1:], base[2000:2003], base[3001:4000]]
    flat = torch.cat([p.double() for p in parts])
    keep = base.clone()
    out = torch.empty(flat.numel() + 1, device="cuda")[1:]
    norm = pb.clip_gradients(parts, 0.5, out=out)
    assert abs(norm.item() - flat.norm().item()) <= 2.0 ** -22 * flat.norm().item()
    assert ((out.double() - flat * 0.5 / flat.norm()).abs() <= 2.0 ** -21 * flat.abs()).all()
    pb.clip_gradients(parts, 0.5)
    assert torch.equal(base[:1], keep[:1]) and torch.equal(base[2003:3001], keep[2003:3001])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_clip_not_finite_and_extreme(dt):
    x = torch.ones(10_000, dtype=DT[dt], device="cuda")
    for bad in (INF, float("nan")):
        y = x.clone()
        y[77] = bad
        keep = y.clone()
        norm = pb.clip_gradients([y, x], 1.0)
        assert not math.isfinite(norm.item())
        assert torch.equal(y.view(torch.int16 if dt == "bf16" else torch.int32),
                           keep.view(torch.int16 if dt == "bf16" else torch.int32))
    for size in (1e25, 1e-25, 0.0):  # squares beyond fp32's range
        y = torch.full((10_000,), size, dtype=DT[dt], device="cuda")
        want = y.double().norm().item()
        norm = pb.clip_gradients([y], 1.0)
        assert abs(norm.item() - want) <= 2.0 ** -22 * want
        assert abs(y.double().norm().item() - min(1.0, want)) <= 0.01


def test_clip_is_the_same_every_time():
    g = gen(1)
    grads = [randn(g, n) for n in (1_000_003, 55, 700_000)]
    s = pb.GradientSet(grads)
    norms = [s.clip(1e9).item() for _ in range(5)]
    assert len(set(norms)) == 1


# ------------------------------------------------------------ as they are used ----
def test_results_are_the_same_every_time():
    g = gen(5)
    counts = [300, 0, 900, 40]
    off = offsets(counts)
    for dt in ("bf16", "f32"):
        rows, w, d = (randn(g, *s, dtype=DT[dt]) for s in ((1240, 128), (4, 128, 192), (1240, 192)))
        first = pb.expert_product_backward(d, rows, w, off)
        for _ in range(3):
            again = pb.expert_product_backward(d, rows, w, off)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_another_stream_and_capture():
    g = gen(6)
    x, logits = randn(g, 64, 500, dtype=torch.bfloat16), randn(g, 6, 500)
    w = randn(g, 6, 64, 64, dtype=torch.bfloat16) * 0.125

    def layer():
        r = pb.route_columns(logits, 2)
        return pb.combine_rows(pb.expert_product(pb.gather_columns(x, r), w, r.offset, activation=pb.Silu(64)), r)

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer()
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = layer()
    for scale in (1.0, -2.0):
        x.mul_(scale)
        logits.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, layer())


# ---------------------------------------------------------------- refusals ----
def test_refusals():
    f32, bf16 = torch.float32, torch.bfloat16
    cuda = lambda *s, dtype=f32: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    logits = cuda(4, 10)
    r = pb.route_columns(logits, 2)
    rows, w, off = cuda(20, 8), cuda(4, 8, 6), r.offset
    bad = [
        lambda: pb.route_columns(logits.cpu(), 2),
        lambda: pb.route_columns(logits.double(), 2),
        lambda: pb.route_columns(logits.t(), 2),
        lambda: pb.route_columns(logits[0], 1),
        lambda: pb.route_columns(logits, 0),
        lambda: pb.route_columns(logits, 5),
        lambda: pb.route_columns(cuda(16, 3), 9),
        lambda: pb.route_columns(cuda(1025, 3), 1),
        lambda: pb.route_columns(cuda(4, 0), 1),
        lambda: pb.route_columns(logits, 2, normalise="softmax"),
        lambda: pb.route_columns_backward(logits, r, cuda(2, 9)),
        lambda: pb.route_columns_backward(logits, r, cuda(2, 10).double()),
        lambda: pb.gather_columns(cuda(8, 11), r),
        lambda: pb.gather_columns(cuda(10, 8).t(), r),
        lambda: pb.gather_columns(cuda(8, 10), r, out=cuda(20, 9)),
        lambda: pb.gather_columns(cuda(8, 10), r, out=cuda(20, 8, dtype=bf16)),
        lambda: pb.gather_columns(cuda(8, 10).double(), r),
        lambda: pb.combine_rows(cuda(21, 8), r),
        lambda: pb.combine_rows(rows, r._replace(weight=r.weight.double())),
        lambda: pb.combine_rows(rows, r, out=cuda(8, 9)),
        lambda: pb.gather_columns_backward(cuda(19, 8), r),
        lambda: pb.combine_rows_backward(cuda(8, 10), cuda(20, 7), r),
        lambda: pb.combine_rows_backward(cuda(8, 10), rows.to(bf16), r),
        lambda: pb.expert_product(rows, w.to(bf16), off),
        lambda: pb.expert_product(rows.double(), w.double(), off),
        lambda: pb.expert_product(cuda(20, 7), w, off),
        lambda: pb.expert_product(rows, w[0], off),
        lambda: pb.expert_product(rows, w, off[:-1]),
        lambda: pb.expert_product(rows, w, off.long()),
        lambda: pb.expert_product(rows, w.transpose(1, 2), off),
        lambda: pb.expert_product(rows, w, off, bias=cuda(4, 5)),
        lambda: pb.expert_product(rows, w, off, activation=pb.Silu(5)),
        lambda: pb.expert_product(rows, w, off, activation=pb.LayerNorm(6)),
        lambda: pb.expert_product(rows, w, off, activation=pb.Bias([0.0] * 6)),
        lambda: pb.expert_product(rows, w, off, out=cuda(20, 7)),
        lambda: pb.expert_product(rows[:1].expand(20, 8), w, off),
        lambda: pb.expert_product(rows, cuda(1, 8, 6).expand(4, 8, 6), off),
        lambda: pb.expert_product_backward(cuda(20, 7), rows, w, off),
        lambda: pb.GradientSet([]),
        lambda: pb.GradientSet([torch.zeros(3)]),
        lambda: pb.GradientSet([cuda(3, dtype=torch.int32)]),
        lambda: pb.GradientSet([cuda(4, 4).t()[:2]]),
        lambda: pb.GradientSet([cuda(3)]).clip(0.0),
        lambda: pb.GradientSet([cuda(3)]).clip(float("nan")),
        lambda: pb.GradientSet([cuda(3)]).clip(1.0, out=cuda(4)),
        lambda: pb.GradientSet([cuda(3)]).clip(1.0, out=cuda(3, dtype=torch.int32)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(pb.PonniError):
            f()
            pytest.fail(f"case {i} was not refused")
    pb.check_operators()
