"""Mixture-of-experts operators at the ends of their ranges, on the GPU.

Where it can be, the data are small integers: their products and sums are exact in
fp32 in any order (below 2^24), so a result has to equal the 64-bit value rounded
to the result's type, and a lost, doubled or foreign row shows.
"""
import pytest

torch = pytest.importorskip("torch")

import ponni_b200 as pb  # noqa: E402
from tests import expert_ref as R  # noqa: E402

pytestmark = pytest.mark.gpu
DT = R.DTYPES


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def integers(g, *shape, dtype=torch.float32, most=2):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


def offsets(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


def exact_weights(d, rows, counts):
    """The weight gradient of integer data, exactly."""
    out = torch.zeros(len(counts), rows.shape[1], d.shape[1], dtype=torch.float64, device="cuda")
    lo = 0
    for e, n in enumerate(counts):
        out[e] = rows[lo:lo + n].double().t() @ d[lo:lo + n].double()
        lo += n
    return out


# ------------------------------------------------------- groups without rows ----
@pytest.mark.parametrize("experts,inputs,outputs", [(128, 2048, 64), (256, 1024, 40), (128, 2048, 130), (64, 520, 300)])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_weight_gradient_many_empty_groups(experts, inputs, outputs, dt):
    g = gen(experts + outputs)
    counts = torch.randint(1, 90, (experts,), generator=g, device="cuda").cpu()
    counts[torch.rand(experts, generator=g, device="cuda").cpu() < 0.5] = 0
    counts[experts // 3] = 3000
    counts = counts.tolist()
    n = sum(counts)
    rows, d = integers(g, n, inputs, dtype=DT[dt]), integers(g, n, outputs, dtype=DT[dt])
    w = torch.zeros(experts, inputs, outputs, dtype=DT[dt], device="cuda")
    _, dw, db = pb.expert_product_backward(d, rows, w, offsets(counts), need_rows=False)
    assert torch.equal(dw, exact_weights(d, rows, counts).to(DT[dt]))
    ones = torch.ones(n, 1, dtype=DT[dt], device="cuda")
    assert torch.equal(db, exact_weights(d, ones, counts)[:, 0].to(DT[dt]))
    pb.check_operators()


@pytest.mark.parametrize("experts,inputs,outputs", [(128, 2048, 64), (1024, 300, 17)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_weight_gradient_short_and_empty_groups(experts, inputs, outputs, dt):
    """Sums of at most one accumulator: tiles 64 columns wide, taken in turn by two halves of the epilogue."""
    g = gen(experts)
    counts = torch.randint(1, 2 * 1800 // experts, (experts,), generator=g, device="cuda").cpu()
    counts[torch.rand(experts, generator=g, device="cuda").cpu() < 0.5] = 0
    counts = counts.tolist()
    n = sum(counts)
    rows, d = integers(g, n, inputs, dtype=DT[dt]), integers(g, n, outputs, dtype=DT[dt])
    w = torch.zeros(experts, inputs, outputs, dtype=DT[dt], device="cuda")
    for _ in range(3):
        _, dw, _ = pb.expert_product_backward(d, rows, w, offsets(counts), need_rows=False)
        assert torch.equal(dw, exact_weights(d, rows, counts).to(DT[dt]))
    pb.check_operators()


def test_weight_gradient_alternating_empty_groups():
    """Long and empty groups in an order that gives one half of the epilogue four tiles in a row."""
    g = gen(3)
    counts = [4096, 0, 4096, 0, 4096, 0, 4096, 4096]
    n = sum(counts)
    rows, d = integers(g, n, 18944, dtype=torch.bfloat16, most=1), integers(g, n, 64, dtype=torch.bfloat16, most=1)
    w = torch.zeros(8, 18944, 64, dtype=torch.bfloat16, device="cuda")
    for _ in range(3):
        _, dw, _ = pb.expert_product_backward(d, rows, w, offsets(counts), bias=False, need_rows=False)
        assert torch.equal(dw, exact_weights(d, rows, counts).bfloat16())
    pb.check_operators()


# ------------------------------------------------------------- many experts ----
@pytest.mark.parametrize("experts", [640, 641, 704, 705, 1024])
@pytest.mark.parametrize("dt,each,inputs,outputs", [
    ("bf16", 3, 24, 100), ("f16", 3, 100, 40),  # 128 and 64 columns, few rows each
    ("bf16", 66, 24, 250),                      # 256 columns, one CTA
    ("bf16", 770, 130, 24), ("f16", 770, 24, 200),  # pairs
    ("f32", 50, 24, 130),                       # parts
])
def test_product_many_experts(experts, dt, each, inputs, outputs):
    g = gen(experts)
    counts = [each] * experts
    counts[5], counts[6] = 0, 2 * each
    n, off = sum(counts), offsets(counts)
    rows, w, d = (integers(g, *s, dtype=DT[dt], most=1) for s in ((n, inputs), (experts, inputs, outputs), (n, outputs)))
    b = integers(g, experts, outputs, dtype=DT[dt])
    want, _ = R.product(rows, w, off, b)
    assert torch.equal(pb.expert_product(rows, w, off, bias=b), want.to(DT[dt]))
    for got, (want, _) in zip(pb.expert_product_backward(d, rows, w, off), R.product_gradient(d, rows, w, off)):
        assert torch.equal(got, want.to(DT[dt]))
    pb.check_operators()


@pytest.mark.parametrize("experts", [641, 704])
def test_product_many_experts_f32_pairs(experts):
    g = gen(experts)
    each, inputs, outputs = 8192, 16, 130
    off = offsets([each] * experts)
    rows, w = integers(g, experts * each, inputs, most=1), integers(g, experts, inputs, outputs, most=1)
    want = torch.bmm(rows.view(experts, each, inputs), w)  # integers: exact
    assert torch.equal(pb.expert_product(rows, w, off).view_as(want), want)
    pb.check_operators()


# -------------------------------------------------------------------- errors ----
def test_a_failed_call_leaves_no_error_behind():
    """The operator check waits for its stream, which a capture forbids: the call reports it, and the runtime's error is clear."""
    import ctypes
    runtime, L = ctypes.CDLL("libcudart.so.12"), pb._abi.lib()
    pb.check_operators()
    side = torch.cuda.Stream()
    stream = ctypes.c_void_p(side.cuda_stream)
    graph = ctypes.c_void_p()
    assert runtime.cudaStreamBeginCapture(stream, 1) == 0  # 1: only this thread's calls are held to the capture
    status = L.ponni_b200_operator_check(0, stream)
    left = runtime.cudaPeekAtLastError()
    runtime.cudaStreamEndCapture(stream, ctypes.byref(graph))  # the forbidden wait has ended the capture
    runtime.cudaGetLastError()
    assert status == 4 and left == 0
    x = torch.randn(4, 10, device="cuda")
    assert pb.gather_columns(x, pb.route_columns(x, 1)).shape == (10, 4)
    pb.check_operators()


def test_offsets_out_of_order_stay_within_the_workspace():
    """Alternating offsets would make many groups of all rows: more units of the weight gradient than there is room for."""
    L = pb._abi.lib()
    g = gen(4)
    experts, n, f = 64, 200_000, 64
    rows, d = randn(g, n, f, dtype=torch.bfloat16), randn(g, n, f, dtype=torch.bfloat16)
    w = torch.zeros(experts, f, f, dtype=torch.bfloat16, device="cuda")
    dw = torch.empty_like(w)
    off = (torch.arange(experts + 1, device="cuda") % 2 * n).to(torch.int32)
    need = L.ponni_b200_expert_product_workspace(pb._abi.BF16, n, experts, f, f, 1, 1, 0)
    assert need > 0
    buf = torch.full((need + (64 << 20),), 77, dtype=torch.uint8, device="cuda")
    pb.check_operators()
    stream = pb.torch_stream_handle(rows.device)
    assert L.ponni_b200_expert_product_backward(pb._abi.BF16, d.data_ptr(), f, rows.data_ptr(), f, n, w.data_ptr(), f, f * f,
                                                off.data_ptr(), experts, f, f, None, 0, dw.data_ptr(), None, buf.data_ptr(),
                                                need, 0, stream) == 0
    with pytest.raises(pb.PonniError, match="ascending"):
        pb.check_operators()
    assert (buf[need:] == 77).all()


# --------------------------------------------------------------- activations ----
@pytest.mark.parametrize("layer", [pb.Relu, pb.LeakyRelu, pb.Elu, pb.Selu, pb.Gelu, pb.Silu, pb.Sigmoid, pb.Tanh,
                                   pb.Softplus, pb.HardSigmoid, pb.HardSwish, pb.Mish])
@pytest.mark.parametrize("rows", [1, 3, 64, 1000])  # a few rows, tiles of one CTA, pairs
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_activation_of_extreme_values(layer, rows, dt):
    """The product is value times one, so that the activation sees each value as it is; neighbours keep theirs."""
    dtype = DT[dt]
    lowest = torch.finfo(dtype).min
    values = [v for v in (0.0, -1.0, 1.0, -20.0, -41.0, -43.5, -50.0, -88.0, -100.0, -1000.0, 100.0, -1e20, 1e20, lowest,
                          float("-inf"), float("inf"), float("nan"), 0.5) if v != v or abs(v) in (0.0, float("inf")) or
              abs(v) <= -lowest]
    outputs = 130
    w = torch.tensor(values, device="cuda").repeat(20)[:outputs].to(dtype).view(1, 1, outputs)
    x = torch.ones(rows, 1, dtype=dtype, device="cuda")
    act = layer(outputs)
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    y = pb.expert_product(x, w, off, activation=act)
    want = R.activate(w.double().view(-1), act.label, act.scalar).expand(rows, outputs)
    if dt == "f16":
        want = torch.where(want.abs() >= 65520.0, want * float("inf"), want)  # beyond fp16's range
    if layer is pb.Relu:
        want = want.nan_to_num(nan=0.0, posinf=float("inf"))  # x > 0 ? x : 0
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    fine = torch.isfinite(want)
    inf = ~fine & ~torch.isnan(want)
    assert torch.equal(y[inf].double(), want[inf])
    # Each function is off by a few units of fp32, relative to its value (SiLU: and to its argument, at most 100,
    # in the exponent: 100 * 2^-24), or to one where it is a difference from one; below 2^-120 by as much.
    one = 0.0 if layer is pb.Silu else 2.0 ** -20
    bound = (R.ULP[dtype] + 2.0 ** -17) * want.abs() + one + (2.0 ** -24 if dt == "f16" else 2.0 ** -120)
    assert ((y.double() - want).abs() <= bound)[fine].all()


# ----------------------------------------------------------------- long sums ----
def check_drift(got, want, terms):
    """Sums of positive products.  The matrix units may drop up to a unit of fp32 (2^-23 of the partial sum) at each
    step of 16 terms within an accumulator's 2048, which is 2^-16; the accumulators are added in fp32, a rounding
    (2^-24) each.  Rounding the result to its type is off by half a unit, and on average, over results spread
    across a factor of four, by nothing."""
    off = (got.double() - want) / want
    held = 2.0 ** -16 + (terms / 2048 + 1) * 2.0 ** -24
    assert off.abs().max() <= R.ULP[got.dtype] * (1 + held) + held
    assert off.mean().abs() <= held + 4 * R.ULP[got.dtype] / got.numel() ** 0.5


def positive(g, *shape, dtype, scale=1.0, along=-1):
    """In [1, 4) * scale, by a factor of its own for every index of dimension `along`."""
    size = [1] * len(shape)
    size[along] = shape[along]
    spread = (1 + torch.rand(*size, generator=g, device="cuda")) * scale
    return ((1 + torch.rand(*shape, generator=g, device="cuda")) * spread).to(dtype)


@pytest.mark.parametrize("n", [40, 128, 250])
@pytest.mark.parametrize("rows", [100, 1000])  # one CTA a tile, pairs
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_long_sums_do_not_drift(dt, rows, n):
    g = gen(n)
    terms, dtype = 200_000, DT[dt]
    off = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    x = positive(g, rows, terms, dtype=dtype, scale=2.0 ** -8, along=0)
    w = positive(g, 1, terms, n, dtype=dtype, scale=2.0 ** -4)
    check_drift(pb.expert_product(x, w, off), x.double() @ w[0].double(), terms)
    wt = w.transpose(1, 2).contiguous()
    dr, _, _ = pb.expert_product_backward(x, x.new_zeros(rows, n), wt, off, bias=False, need_weights=False)
    check_drift(dr, x.double() @ wt[0].double().t(), terms)
    pb.check_operators()


@pytest.mark.parametrize("inputs,outputs", [(300, 40), (64, 128), (200, 250), (2500, 2600)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_long_weight_gradients_do_not_drift(dt, inputs, outputs):
    """(2500 x 2600 fills the SMs with whole groups, the others are split into units.)"""
    g = gen(outputs)
    n, dtype = 270_000, DT[dt]
    off = torch.tensor([0, 100, n - 50], dtype=torch.int32, device="cuda")
    x, d = positive(g, n, inputs, dtype=dtype, scale=2.0 ** -8), positive(g, n, outputs, dtype=dtype, scale=2.0 ** -4)
    w = torch.zeros(2, inputs, outputs, dtype=dtype, device="cuda")
    _, dw, _ = pb.expert_product_backward(d, x, w, off, bias=False, need_rows=False)
    take = slice(0, 300)
    check_drift(dw[1, take, take], x[100:n - 50, take].double().t() @ d[100:n - 50, take].double(), n)
    check_drift(dw[0, take, take], x[:100, take].double().t() @ d[:100, take].double(), 100)
    pb.check_operators()


@pytest.mark.parametrize("rows", [2, 100])  # a few rows, tiles
def test_single_precision_silu(rows):
    """Of an argument down to -88: exp is off by a few units, and its argument by half of one, 88 * 2^-25 in the exponent."""
    z = torch.linspace(-88.0, 20.0, 500, device="cuda")
    y = pb.expert_product(torch.ones(rows, 1, device="cuda"), z.view(1, 1, 500), offsets([rows]), activation=pb.Silu(500))
    want = R.activate(z.double(), "SiLU").expand(rows, 500)
    assert ((y.double() - want).abs() <= 2.0 ** -17 * want.abs()).all()
    near = want[0, z > -1].abs()
    assert ((y[:, z > -1].double() - want[:, z > -1]).abs() <= 2.0 ** -21 * near + 2.0 ** -140).all()


# ------------------------------------------------------------------- routing ----
@pytest.mark.parametrize("experts,batch", [(2, 1), (3, 700), (6, 5000)])
@pytest.mark.parametrize("normalise", ["selected", "all"])
def test_routing_weights_far_below_the_best(experts, batch, normalise):
    """Logits on a grid, so that their differences are exact.  exp is off by at most 2 units (2^-23), the sum of n by
    2 + (n - 1) / 2, the quotient by 1/2; the gradient takes two weights, an exponential and four roundings."""
    g = gen(batch)
    x = torch.randint(-10_000, 10_000, (experts, batch), generator=g, device="cuda").float() / 256
    k = experts if normalise == "selected" else 1
    r = pb.route_columns(x, k, normalise=normalise)
    p = torch.softmax(x.double(), 0)
    weight = torch.gather(p, 0, r.expert.long())
    unit, of_weight = 2.0 ** -23, 4 + experts / 2
    assert ((r.weight.double() - weight).abs() <= of_weight * unit * weight + 2.0 ** -148).all()
    if k == 1:
        d_w = torch.randn(1, batch, generator=g, device="cuda")
        d = pb.route_columns_backward(x, r, d_w, normalise="all")
        other = torch.ones_like(x, dtype=torch.bool).scatter_(0, r.expert.long(), False)
        want = -p * weight * d_w.double()
        assert ((d.double() - want).abs() <= (2 * of_weight + 4) * unit * want.abs() + 2.0 ** -147)[other].all()


# --------------------------------------------------------- parts of fp32 values ----
def test_single_precision_parts_are_the_nearest():
    """Factors just below two: cut-off parts would lose 2^-23 of every product, the nearest ones (2 - 2^-23) nothing."""
    value = 2.0 - 2.0 ** -23
    x = torch.full((600, 16), value, device="cuda")
    x[::2] *= -1
    w = torch.full((2, 16, 130), value, device="cuda")
    off = offsets([400, 200])
    want = (x.double() @ w[0].double()).float()
    assert torch.equal(pb.expert_product(x, w, off), want)
    d = torch.full((600, 130), value, device="cuda")
    dr, dw, _ = pb.expert_product_backward(d[:, :16].contiguous(), x, w[:, :, :16].contiguous(), off)
    assert torch.equal(dr, torch.full_like(dr, 64.0 - 2.0 ** -17))
    assert not dw.any()  # (as many rows of either sign)
    pb.check_operators()


def test_single_precision_ends_of_the_range():
    """Values that round up past the largest bf16, subnormal ones and zeros, times one; parts of a product of them."""
    top = torch.finfo(torch.float32).max
    v = torch.tensor([top, -top, top * (1 - 2.0 ** -9), top * (1 - 2.0 ** -10), 3.3961775e38, 0.0, -0.0, 1.0 + 2.0 ** -23,
                      2.0 ** -100 * (2 - 2.0 ** -23)], device="cuda")
    x = v.view(-1, 1).repeat(100, 1)
    w = torch.ones(1, 1, 24, device="cuda")
    assert torch.equal(pb.expert_product(x, w, offsets([len(x)])), x.expand(-1, 24))
    w[..., 1::2] = 0.5
    assert torch.equal(pb.expert_product(x, w, offsets([len(x)])), x * w[0])


# --------------------------------------------------- NaN and infinity in fp32 ----
@pytest.mark.parametrize("counts", [[150, 0, 300, 40], [9000, 8000]])
def test_single_precision_nan_and_infinity(counts):
    """Wherever they stand, results are NaN, infinite or finite as in plain arithmetic."""
    g = gen(len(counts))
    experts, n, off = len(counts), sum(counts), offsets(counts)
    inputs, outputs = 200, 130
    rows, w, d = randn(g, n, inputs), randn(g, experts, inputs, outputs) * inputs ** -0.5, randn(g, n, outputs)
    w[0, 5] = 1.0  # (parts that are zero)
    inf, nan = float("inf"), float("nan")
    rows[3, 5], rows[7, 9], rows[20, 5], rows[21, 0], rows[n - 1, 5] = inf, nan, -inf, 0.0, inf
    rows[20, 6] = nan
    w[0, 7, 11], w[-1, 0, 3], w[-1, 1, 3], w[0, 8, 12] = inf, inf, -inf, nan
    d[2, 5], d[30, 60], d[31, 60], d[n - 3, 129] = -inf, inf, nan, inf
    y, (dr, dw, db) = pb.expert_product(rows, w, off), pb.expert_product_backward(d, rows, w, off)
    want, size = R.product(rows, w, off)
    grads = R.product_gradient(d, rows, w, off)
    for got, ref, mag, terms in ((y, want, size, inputs), (dr, *grads[0], outputs), (dw, *grads[1], max(counts)),
                                 (db, *grads[2], max(counts))):
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        infinite = torch.isinf(ref)
        assert torch.equal(got[infinite].double(), ref[infinite]) and torch.equal(torch.isinf(got), infinite)
        fine = torch.isfinite(ref)
        R.check_sum(got[fine], ref[fine], mag[fine], terms)
    pb.check_operators()


def test_single_precision_long_sums_with_nan_and_infinity_end_in_time():
    """65536 terms in pairs of CTAs: no role's bounded wait runs out while a tile is summed again."""
    n, terms, outputs = 8400, 65536, 250
    g = gen(1)
    x, w = randn(g, n, terms), randn(g, 1, terms, outputs)
    w[0, 0] = 1.0
    x[:, -1] = 0.0
    x[5, 0], x[300:330, 0], x[8000, 7] = float("inf"), float("-inf"), float("nan")
    y = pb.expert_product(x, w, offsets([n]))
    pb.check_operators()
    assert (y[5] == float("inf")).all() and (y[300:330] == float("-inf")).all() and torch.isnan(y[8000]).all()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[5], keep[300:330], keep[8000] = False, False, False
    assert torch.isfinite(y[keep]).all()


def test_single_precision_nan_costs_little():
    g = gen(2)
    x, w, off = randn(g, 8192, 1024), randn(g, 1, 1024, 1024), offsets([8192])

    def time(x):
        pb.expert_product(x, w, off)
        begin, end = torch.cuda.Event(True), torch.cuda.Event(True)
        begin.record()
        for _ in range(3):
            pb.expert_product(x, w, off)
        end.record()
        end.synchronize()
        return begin.elapsed_time(end)

    bad = x.clone()
    bad[:, -1] = float("nan")
    assert time(bad) < 30 * time(x)  # (a sum one by one for every value that is NaN: 280 times)


# -------------------------------------------------------------- shared memory ----
def test_outputs_that_overlap_inputs_are_refused():
    g = gen(1)
    rows, w, off = randn(g, 300, 64), randn(g, 2, 64, 64), offsets([100, 200])
    r = pb.route_columns(randn(g, 2, 64), 1)
    x = randn(g, 64, 64)
    buf = randn(g, 300, 100)
    for f in (lambda: pb.expert_product(rows, w, off, out=rows),
              lambda: pb.expert_product(rows[:200], w, offsets([100, 100]), out=rows[100:]),
              lambda: pb.expert_product(buf[:, :64], w, off, out=buf[:, 36:]),
              lambda: pb.expert_product(rows[:128], w, offsets([100, 28]), out=w.view(128, 64)),
              lambda: pb.gather_columns(x, r, out=x),
              lambda: pb.combine_rows(x, r, out=x),
              lambda: pb.gather_columns_backward(x, r, out=x)):
        with pytest.raises(pb.PonniError, match="overlaps"):
            f()
    assert torch.equal(pb.gather_columns(x, r).double(), R.gather(x, r.row))


def test_outputs_beside_inputs_are_not():
    """Columns of one buffer side by side, and rows of one buffer one behind the other."""
    g = gen(2)
    w, off = randn(g, 2, 64, 64), offsets([100, 200])
    buf = randn(g, 300, 130)
    x = buf[:, 1:65].clone()
    out = buf[:, 66:]
    assert pb.expert_product(buf[:, 1:65], w, off, out=out) is out
    want, size = R.product(x, w, off)
    R.check_sum(out, want, size, 64)
    assert torch.equal(buf[:, 1:65], x)
    buf = randn(g, 600, 64)
    x = buf[300:].clone()
    pb.expert_product(buf[300:], w, off, out=buf[:300])
    want, size = R.product(x, w, off)
    R.check_sum(buf[:300], want, size, 64)


@pytest.mark.parametrize("sizes", [[5, 1000, 3], [100_001, 70_000, 2_000_003]])
def test_clip_of_views_of_the_packed_vector(sizes):
    flat = randn(gen(5), sum(sizes))
    keep = flat.double()
    parts = list(flat.split(sizes))
    norm = pb.clip_gradients(parts, 0.25, out=flat)
    assert abs(norm.item() - keep.norm().item()) <= 2.0 ** -22 * keep.norm().item()
    assert ((flat.double() - keep * 0.25 / keep.norm()).abs() <= 2.0 ** -21 * keep.abs() * 0.25 / keep.norm()).all()
    with pytest.raises(pb.PonniError, match="overlap"):
        pb.clip_gradients([parts[0], flat], 0.25)
    with pytest.raises(pb.PonniError, match="overlaps"):
        pb.clip_gradients(parts[::-1], 0.25, out=flat)


def test_routings_without_offsets_are_refused():
    x = torch.randn(4, 10, device="cuda")
    r = pb.route_columns(x, 2)
    rows = torch.zeros(20, 4, device="cuda")
    for bad in (r._replace(offset=r.offset[:0]), r._replace(offset=r.offset[:1]), r._replace(row=r.row[0]),
                r._replace(row=r.row[0, 0])):
        for f in (lambda: pb.gather_columns(x, bad), lambda: pb.combine_rows_backward(x, rows, bad)):
            with pytest.raises(pb.PonniError):
                f()
    pb.check_operators()


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("max_norm", [1.0, 1e-4, 1e-9])
def test_clip_of_gradients_near_the_largest_value(dt, max_norm):
    """A factor below fp32's normal range: it is held to a unit of fp32, and the product another."""
    for n in (1000, 3_000_000):
        x = (torch.rand(n, generator=gen(n), device="cuda") * 3e38).to(DT[dt])
        keep = x.double()
        want = keep * (max_norm / keep.norm())
        ok = want.abs() >= 2.0 ** -120  # (below, fp32 itself has fewer digits)
        out = torch.empty(n, dtype=DT[dt], device="cuda")
        pb.clip_gradients([x], max_norm, out=out)
        assert ok.sum() > n // 2
        assert ((out.double() - want).abs() <= (R.ULP[x.dtype] + 2.0 ** -22) * want.abs())[ok].all()
        pb.clip_gradients([x], max_norm)
        assert torch.equal(x, out)


# ------------------------------------------------------ long groups, exactly ----
@pytest.mark.parametrize("inputs,outputs", [(200, 24), (24, 200), (40, 40), (1200, 37), (128, 128), (72, 300), (520, 260)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_long_groups_exactly(inputs, outputs, dt):
    """Many tiles a CTA and weight gradients in units: no row lost, none taken twice, none of the next group's.

    Sums of up to 40100 products of -1, 0 and 1 are exact in fp32 (and 16-bit rows of at most 1200 terms
    of them before their rounding)."""
    g = gen(inputs + outputs)
    dtype, counts = DT[dt], [30_011, 0, 17_000, 129, 40_100, 1, 1024, 2047]
    n, off = sum(counts) + 5, offsets(counts)
    rows, w, d = (integers(g, *s, dtype=dtype, most=1) for s in ((n, inputs), (len(counts), inputs, outputs), (n, outputs)))
    b = integers(g, len(counts), outputs, dtype=dtype)
    want, _ = R.product(rows, w, off, b)
    assert torch.equal(pb.expert_product(rows, w, off, bias=b), want.to(dtype))
    for got, (want, _) in zip(pb.expert_product_backward(d, rows, w, off), R.product_gradient(d, rows, w, off)):
        assert torch.equal(got, want.to(dtype))
    pb.check_operators()


@pytest.mark.parametrize("total", [1, 63, 64, 65, 4095, 4096, 4097, 20_000, 50_001])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_edges_of_units_exactly(total, dt):
    """Rows that are not zero only beside the edges of K blocks and groups, each with a value of its own."""
    dtype, f = DT[dt], 130
    counts = [total, 7, total // 3]
    n, off = sum(counts), offsets(counts)
    at = torch.arange(n, device="cuda")
    in_group = torch.cat([torch.arange(c, device="cuda") for c in counts])
    marked = ((in_group % 64 < 2) | (in_group % 64 > 61)).to(dtype)[:, None]
    rows = marked * (1 + at[:, None] % 3).to(dtype) * torch.ones(n, f, dtype=dtype, device="cuda")
    d = marked * (1 + (at[:, None] // 3 + torch.arange(f, device="cuda")) % 2).to(dtype)
    w = torch.zeros(3, f, f, dtype=dtype, device="cuda")
    _, dw, db = pb.expert_product_backward(d, rows, w, off, need_rows=False)
    assert torch.equal(dw, exact_weights(d, rows, counts).to(dtype))
    assert torch.equal(db, exact_weights(d, torch.ones(n, 1, dtype=dtype, device="cuda"), counts)[:, 0].to(dtype))


def test_past_32_bit_offsets_exactly():
    """More than 2^31 elements of rows and of gradients; rows that are not zero on both sides of that element."""
    n, f = 9_000_000, 256
    g = gen(3)
    rows, d = (torch.zeros(n, f, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    edge = 2 ** 31 // f
    marked = [slice(0, 100), slice(edge - 150, edge + 150), slice(n - 300, n)]
    for s in marked:
        rows[s], d[s] = (integers(g, s.stop - s.start, f, dtype=torch.bfloat16) for _ in range(2))
    w = integers(g, 2, f, f, dtype=torch.bfloat16)
    counts = [n - 200, 200]
    off = offsets(counts)
    y = pb.expert_product(rows, w, off)
    dr, dw, db = pb.expert_product_backward(d, rows, w, off)
    want_w, want_b = torch.zeros(2, f, f, dtype=torch.float64, device="cuda"), torch.zeros(2, f, dtype=torch.float64, device="cuda")
    for s in marked:
        for e, (lo, hi) in enumerate(((0, n - 200), (n - 200, n))):
            a, b = max(s.start, lo), min(s.stop, hi)
            if a < b:
                x, u = rows[a:b].double(), d[a:b].double()
                assert torch.equal(y[a:b], (x @ w[e].double()).bfloat16())
                assert torch.equal(dr[a:b], (u @ w[e].double().t()).bfloat16())
                want_w[e] += x.t() @ u
                want_b[e] += u.sum(0)
    assert torch.equal(dw, want_w.bfloat16()) and torch.equal(db, want_b.bfloat16())
    for t in (y, dr):
        assert torch.count_nonzero(t[100:edge - 150]) == 0 and torch.count_nonzero(t[edge + 150:n - 300]) == 0
    pb.check_operators()


def test_columns_past_32_bit_offsets():
    """More than 2^31 elements on either side: a column's two rows, added up, are twice the column."""
    features, batch = 600, 3_700_000
    g = gen(6)
    x = integers(g, features, batch, dtype=torch.bfloat16, most=100)
    r = pb.route_columns(randn(g, 4, batch), 2)
    rows = pb.gather_columns(x, r)
    assert rows.shape[0] * rows.stride(0) > 2 ** 32
    for at in (0, batch // 2, batch - 1):
        for j in range(2):
            assert torch.equal(rows[r.row[j, at].long()], x[:, at])
    assert torch.equal(pb.gather_columns_backward(rows, r), 2 * x)
    even = r._replace(weight=torch.full_like(r.weight, 0.5))
    assert torch.equal(pb.combine_rows(rows, even), x)
    d_rows, d_weight = pb.combine_rows_backward(x, rows, even)
    assert torch.equal(d_rows, rows * 0.5)
    want = x[:, -1000:].double().square().sum(0)  # at most 600 * 100^2: exact in fp32
    assert torch.equal(d_weight[:, -1000:].double(), want.expand(2, -1))


def test_routing_past_32_bit_offsets():
    experts, batch = 1024, 2_200_000
    g = gen(7)
    x = torch.randn(experts, batch, generator=g, device="cuda", dtype=torch.float16)
    assert x.numel() > 2 ** 31
    r = pb.route_columns(x, 1, normalise="all")
    tail = x[:, -2000:].float()
    best = tail.max(0).values
    first = (tail == best).int().argmax(0)  # the lowest of equal ones
    assert torch.equal(r.expert[0, -2000:].long(), first)
    p = torch.softmax(tail.double(), 0)
    assert ((r.weight[0, -2000:].double() - p.gather(0, first[None])[0]).abs() <= 2.0 ** -13 * p.max(0).values).all()
    by_row = torch.sort(r.expert[0], stable=True).indices
    assert torch.equal(r.column.long(), by_row) and int(r.offset[-1]) == batch
    d = pb.route_columns_backward(x, r, torch.ones_like(r.weight), normalise="all")
    chosen = torch.zeros_like(p).scatter_(0, first[None], 1.0)
    want = p * (chosen - p.max(0).values)
    # of 1024 terms: (n + 8) units of 2^-22 of the weight, as for the weights; the rounding to 16 bits
    assert ((d[:, -2000:].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -11 * p + 2.0 ** -25).all()


def test_routing_weights_over_all_in_single_precision():
    """64 experts: root mean square of the weights' errors.  A rounding is 2^-24 / sqrt 3 = 3.4e-8.  A term of the sum
    passes 3 in its chunk of 8 and one for every further chunk, 11 with partial sums of a third of the square on average;
    the chosen expert's exponential (1.5 roundings) and the quotient: sqrt(11 / 3 + 1.5^2 + 1) * 3.4e-8 = 0.9e-7."""
    x = randn(gen(11), 64, 100_000) * 1.5
    r = pb.route_columns(x, 4, normalise="all")
    want = torch.softmax(x.double(), 0).gather(0, r.expert.long())
    assert ((r.weight.double() - want).norm() / want.norm()).item() <= 1e-7
