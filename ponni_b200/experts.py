"""Mixtures of experts: routing, column gather and combination, products grouped
by expert, and clipping of the gradients of many tensors.

Operators over CUDA torch tensors, on the current torch stream, backed by the
`ponni_b200_route_columns` ... `ponni_b200_gradient_set_clip` entry points of
include/ponni_b200.h.  Batches are feature-major [features, batch] as
everywhere in this package; between gather_columns and combine_rows the chosen
columns are rows [rows, features], sorted by expert.  No counterpart in the
reference, whose models are one chain of layers.

    routing = route_columns(logits, top_k=2)
    rows = gather_columns(x, routing)
    hidden = expert_product(rows, w1, routing.offset, bias=b1, activation=Silu(256))
    y = combine_rows(expert_product(hidden, w2, routing.offset, bias=b2), routing)

Every function raises PonniError on arguments that its kernels do not take.
The functions stand outside torch's autograd, as the rest of this package:
results carry no history, whatever the inputs' `requires_grad`, and gradients
come from the `_backward` calls.
Group offsets live on the device and are not read back: `check_operators`
reports afterwards whether they were in order.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

from . import _abi
from .inference import torch_stream_handle
from .layers import Layer

_NORMALISE = {"selected": _abi.ROUTE_SELECTED, "all": _abi.ROUTE_ALL}
_codes: dict = {}
_modules: list = []


def _torch():
    if not _modules:
        import torch
        _codes.update({torch.float32: _abi.F32, torch.float64: _abi.F64, torch.float16: _abi.F16,
                       torch.bfloat16: _abi.BF16})
        _modules.append(torch)
    return _modules[0]


def _empty(torch, rows: int, cols: int, dtype, device):
    """A dense matrix (empty_strided: half the call's time of empty with a shape)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def _refuse(message: str, status: int = 1):
    raise _abi.PonniError(status, message)


def _call(status: int):
    if status != _abi.OK:
        raise _abi.PonniError(status, (_abi.lib().ponni_b200_operator_error() or b"").decode())


def _real(t, what: str) -> int:
    """dtype code of a CUDA tensor of fp32, fp16 or bf16."""
    if not t.is_cuda:
        _refuse(f"{what} must be a CUDA tensor")
    code = _codes.get(t.dtype, _abi.F64)
    if code == _abi.F64:
        _refuse(f"{what} must be fp32, fp16 or bf16, not {t.dtype}", 3)
    return code


def _matrix(t, what: str) -> int:
    """Row stride of a 2-D tensor whose second index is contiguous."""
    shape = t.shape
    if len(shape) != 2:
        _refuse(f"{what} must be two-dimensional")
    rows, cols = shape
    ld, one = t.stride()
    if cols > 1 and one != 1:
        _refuse(f"{what} must be LayoutRight (second index contiguous)")
    if rows <= 1:
        return max(1, cols)
    if ld < cols:
        _refuse(f"{what} has overlapping rows")
    return ld


def _like(t, shape, dtype, device, what: str):
    """Checks a dense tensor of the given shape, type and device."""
    if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
        _refuse(f"{what} must be a dense {dtype} tensor of shape {tuple(shape)} on {device}")


def _span(t):
    """Addresses from the first element to behind the last one."""
    at = t.data_ptr()
    return at, at + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _check_apart(out, *inputs):
    """Refuses an output that shares elements with an input (the kernels read and write in no order).

    Column ranges of one buffer side by side, with the same row stride, are apart.
    """
    if out.numel() == 0:
        return
    lo, hi = _span(out)
    for t in inputs:
        if t is None or t.numel() == 0:
            continue
        a, b = _span(t)
        if a >= hi or b <= lo:
            continue
        z, ld = out.element_size(), out.stride(0)
        if t.dim() == 2 and t.element_size() == z and t.stride(0) == ld and (a - lo) % z == 0:
            at = (a - lo) // z % ld
            if at >= out.shape[1] and at + t.shape[1] <= ld:
                continue
        _refuse("out overlaps an input")


class Routing(NamedTuple):
    """What route_columns decides.

    expert, weight, row [top_k, batch]: a column's choices, largest logit first
    (int32, -1: none), their weights (fp32) and the rows they take (int32, -1:
    none).  column [batch * top_k]: the column of each row (int32, -1 past the
    last used row).  offset [experts + 1]: first row of each expert (int32).
    """
    expert: object
    weight: object
    row: object
    column: object
    offset: object


def _check_routing(r: Routing, device, batch: int):
    torch = _torch()
    shape = r.row.shape
    if len(shape) != 2 or shape[1] != batch:
        _refuse(f"the routing has rows of shape {tuple(shape)}, not of {batch} columns", 2)
    _like(r.row, shape, torch.int32, device, "routing.row")
    if r.offset.dim() != 1 or r.offset.numel() < 2:  # its last entry is read on the device
        _refuse(f"routing.offset has shape {tuple(r.offset.shape)}, not [experts + 1]", 2)
    _like(r.offset, r.offset.shape, torch.int32, device, "routing.offset")
    return shape[0]


def _output(out, shape, like, what: str):
    if out is None:
        return _empty(_torch(), *shape, like.dtype, like.device)
    if out.shape != shape or out.dtype != like.dtype or out.device != like.device:
        _refuse(f"{what} must be a {like.dtype} tensor of shape {tuple(shape)} on {like.device}", 2)
    return out


def _row_output(out, rows: int, features: int, like):
    """Rows with a stride of whole 16-byte vectors, as the tensor-core product reads them without a copy."""
    if out is not None:
        return _output(out, (rows, features), like, "out")
    pad = -features % (16 // like.element_size())
    t = _empty(_torch(), rows, features + pad, like.dtype, like.device)
    return t[:, :features] if pad else t


def route_columns(logits, top_k: int, normalise: str = "selected") -> Routing:
    """Chooses the top_k experts of every column of logits [experts, batch] (fp32, fp16 or bf16).

    Ties go to the lower expert; -inf and NaN logits are never chosen, so a
    column may have fewer choices.  `normalise`: "selected" makes the weights a
    softmax over the chosen logits, "all" takes the chosen entries of the
    softmax over all experts.
    """
    torch = _torch()
    code = _real(logits, "logits")
    ld = _matrix(logits, "logits")
    experts, batch = logits.shape
    if normalise not in _NORMALISE:
        _refuse(f"normalise must be 'selected' or 'all', not {normalise!r}")
    if batch == 0:
        _refuse("routing requires a nonzero batch size")
    top_k = int(top_k)
    if not 1 <= top_k <= min(8, experts):
        _refuse(f"top_k must be 1 to 8 and at most the {experts} experts, not {top_k}", 3)
    dev, L = logits.device, _abi.lib()
    # One allocation (five cost more than its views): expert, row, column, weight, offset, workspace.
    n = top_k * batch
    need = L.ponni_b200_route_workspace(experts, batch)
    buf = torch.empty(4 * n + experts + 1 + need // 4, dtype=torch.int32, device=dev)
    at, shape, stride = buf.data_ptr(), (top_k, batch), (batch, 1)
    space = at + 16 * n + 4 * (experts + 1)
    _call(L.ponni_b200_route_columns(code, logits.data_ptr(), ld, experts, top_k, batch, _NORMALISE[normalise], at,
                                     at + 12 * n, at + 4 * n, at + 8 * n, at + 16 * n, space, need, dev.index,
                                     torch_stream_handle(dev)))
    return Routing(buf.as_strided(shape, stride), buf.view(torch.float32).as_strided(shape, stride, 3 * n),
                   buf.as_strided(shape, stride, n), buf.as_strided((n,), (1,), 2 * n),
                   buf.as_strided((experts + 1,), (1,), 4 * n))


def route_columns_backward(logits, routing: Routing, d_weight, normalise: str = "selected"):
    """Gradient of the weights of route_columns: d_weight [top_k, batch] (fp32) -> d_logits [experts, batch]."""
    torch = _torch()
    code = _real(logits, "logits")
    ld = _matrix(logits, "logits")
    if normalise not in _NORMALISE:
        _refuse(f"normalise must be 'selected' or 'all', not {normalise!r}")
    experts, batch = logits.shape
    dev = logits.device
    top_k = _check_routing(routing, dev, batch)
    for t, dt, what in ((routing.expert, torch.int32, "routing.expert"), (routing.weight, torch.float32, "routing.weight"),
                        (d_weight, torch.float32, "d_weight")):
        _like(t, (top_k, batch), dt, dev, what)
    d = _empty(torch, experts, batch, logits.dtype, dev)
    _call(_abi.lib().ponni_b200_route_columns_backward(
        code, logits.data_ptr(), ld, experts, top_k, batch, _NORMALISE[normalise], routing.expert.data_ptr(),
        routing.weight.data_ptr(), d_weight.data_ptr(), d.data_ptr(), batch, dev.index, torch_stream_handle(dev)))
    return d


def gather_columns(x, routing: Routing, out=None):
    """Rows of the chosen columns, sorted by expert: x [features, batch] -> [batch * top_k, features].

    Rows past the last used one are zero.
    """
    _torch()
    code = _real(x, "x")
    ld = _matrix(x, "x")
    features, batch = x.shape
    dev = x.device
    top_k = _check_routing(routing, dev, batch)
    given, out = out, _row_output(out, batch * top_k, features, x)
    if given is not None:
        _check_apart(out, x, routing.row, routing.offset)
    _call(_abi.lib().ponni_b200_gather_columns(
        code, x.data_ptr(), ld, features, batch, top_k, routing.row.data_ptr(),
        routing.offset.data_ptr() + 4 * (routing.offset.numel() - 1), out.data_ptr(), _matrix(out, "out"), dev.index,
        torch_stream_handle(dev)))
    return out


def _combine(rows, routing, weight, out):
    code = _real(rows, "rows")
    ld = _matrix(rows, "rows")
    total, features = rows.shape
    dev = rows.device
    batch = routing.row.shape[-1] if routing.row.dim() else 0
    top_k = _check_routing(routing, dev, batch)
    if total != batch * top_k:
        _refuse(f"the routing has {batch * top_k} rows, not {total}", 2)
    given, out = out, _output(out, (features, batch), rows, "out")
    if given is not None:
        _check_apart(out, rows, routing.row, routing.weight)
    _call(_abi.lib().ponni_b200_combine_rows(code, rows.data_ptr(), ld, features, batch, top_k, routing.row.data_ptr(),
                                             weight, out.data_ptr(), _matrix(out, "out"), dev.index,
                                             torch_stream_handle(dev)))
    return out


def gather_columns_backward(d_rows, routing: Routing, out=None):
    """Gradient of gather_columns: the sum of a column's rows, [batch * top_k, features] -> [features, batch]."""
    _torch()
    return _combine(d_rows, routing, None, out)


def combine_rows(rows, routing: Routing, out=None):
    """Weighted sum of a column's rows: [batch * top_k, features] -> [features, batch].

    Summed in fp32 and rounded once; a column without choices gives zeros.
    """
    torch = _torch()
    _like(routing.weight, routing.row.shape, torch.float32, rows.device, "routing.weight")
    return _combine(rows, routing, routing.weight.data_ptr(), out)


def combine_rows_backward(d_y, rows, routing: Routing):
    """Gradients of combine_rows: (d_rows [batch * top_k, features], d_weight [top_k, batch] in fp32)."""
    torch = _torch()
    code = _real(d_y, "d_y")
    ld = _matrix(d_y, "d_y")
    features, batch = d_y.shape
    dev = d_y.device
    top_k = _check_routing(routing, dev, batch)
    if rows.shape != (batch * top_k, features) or rows.dtype != d_y.dtype or rows.device != dev:
        _refuse(f"rows must be a {d_y.dtype} tensor of shape {(batch * top_k, features)} on {dev}", 2)
    _like(routing.weight, routing.row.shape, torch.float32, dev, "routing.weight")
    d_rows = _row_output(None, batch * top_k, features, d_y)
    d_weight = _empty(torch, top_k, batch, torch.float32, dev)
    _call(_abi.lib().ponni_b200_combine_rows_backward(
        code, d_y.data_ptr(), ld, rows.data_ptr(), _matrix(rows, "rows"), features, batch, top_k,
        routing.row.data_ptr(), routing.weight.data_ptr(),
        routing.offset.data_ptr() + 4 * (routing.offset.numel() - 1), d_rows.data_ptr(), _matrix(d_rows, "d_rows"),
        d_weight.data_ptr(), dev.index, torch_stream_handle(dev)))
    return d_rows, d_weight


def _check_product(rows, weights, offset, what="rows"):
    torch = _torch()
    code = _real(rows, what)
    if weights.dim() != 3 or weights.dtype != rows.dtype or weights.device != rows.device:
        _refuse(f"weights must be a {rows.dtype} tensor [experts, inputs, outputs] on {rows.device}", 2)
    experts, inputs, outputs = weights.shape
    stride, ld, one = weights.stride()
    if outputs > 1 and one != 1:
        _refuse("weights must be LayoutRight (outputs contiguous)")
    if inputs == 1:
        ld = outputs
    if ld < outputs:
        _refuse("weights have overlapping rows")
    if experts == 1:
        stride = inputs * ld
    _like(offset, (experts + 1,), torch.int32, rows.device, "offset")
    return code, experts, inputs, outputs, stride, ld


def _space(L, code, total, experts, inputs, outputs, addresses, strides, backward, dev):
    """(tensor or None, bytes, address) of the product's workspace; the allocator's blocks are 512-byte aligned.

    `addresses`, `strides`: those of all operands, or-ed."""
    aligned = code != _abi.F32 and not (addresses & 15 or strides & 7)
    if aligned and not backward:
        return None, 0, None
    need = L.ponni_b200_expert_product_workspace(code, total, experts, inputs, outputs, aligned, backward, dev.index)
    if not need:
        return None, 0, None
    torch = _torch()
    t = torch.empty(need, dtype=torch.uint8, device=dev)
    return t, need, t.data_ptr()


def expert_product(rows, weights, offset, bias=None, activation: Layer | None = None, out=None):
    """out[r] = activation(rows[r] @ weights[e] + bias[e]) for the rows r in [offset[e], offset[e + 1]).

    rows [n, inputs], weights [experts, inputs, outputs] (each as in Matvec),
    bias [experts, outputs]; fp32, fp16 or bf16 alike, sums in fp32.  Rows in
    no group give zero.  `activation` is an activation layer of `outputs`
    features, such as Silu(outputs).  `out` shares no element with an input.
    """
    code, experts, inputs, outputs, stride, w_ld = _check_product(rows, weights, offset)
    ld = _matrix(rows, "rows")
    total = rows.shape[0]
    if rows.shape[1] != inputs:
        _refuse(f"rows have {rows.shape[1]} features, the weights {inputs} inputs", 2)
    dev = rows.device
    if bias is not None:
        _like(bias, (experts, outputs), rows.dtype, dev, "bias")
    kind, flags, s0, s1 = -1, 0, 0.0, 0.0
    if activation is not None:
        if not isinstance(activation, Layer) or not _abi.RELU <= activation.kind <= _abi.MISH:
            _refuse("activation must be an activation layer", 3)
        if activation.num_outputs != outputs:
            _refuse(f"the activation has {activation.num_outputs} features, the product {outputs} outputs", 2)
        kind, flags, s0, s1 = activation.kind, activation.flags, activation.scalar[0], activation.scalar[1]
    given, out = out, _row_output(out, total, outputs, rows)
    if given is not None:
        _check_apart(out, rows, weights, bias, offset)
    L = _abi.lib()
    x, w = rows.data_ptr(), weights.data_ptr()
    space, need, at = _space(L, code, total, experts, inputs, outputs, x | w, ld | w_ld | stride, 0, dev)
    _call(L.ponni_b200_expert_product(
        code, x, ld, total, w, w_ld, stride,
        None if bias is None else bias.data_ptr(), offset.data_ptr(), experts, inputs, outputs, kind, flags, s0, s1,
        out.data_ptr(), _matrix(out, "out"), at, need, dev.index, torch_stream_handle(dev)))
    return out


def expert_product_backward(d_out, rows, weights, offset, bias: bool = True, need_rows: bool = True,
                            need_weights: bool = True):
    """Gradients of expert_product without activation: (d_rows, d_weights, d_bias).

    d_out [n, outputs].  `bias`, `need_rows`, `need_weights`: a gradient that
    is not needed is None and costs nothing.  Experts without rows get zero
    gradients, rows in no group too.
    """
    torch = _torch()
    code, experts, inputs, outputs, stride, w_ld = _check_product(rows, weights, offset)
    total = rows.shape[0]
    if rows.dim() != 2 or rows.shape[1] != inputs:
        _refuse(f"rows must have the weights' {inputs} inputs", 2)
    if d_out.shape != (total, outputs) or d_out.dtype != rows.dtype or d_out.device != rows.device:
        _refuse(f"d_out must be a {rows.dtype} tensor of shape {(total, outputs)} on {rows.device}", 2)
    dev = rows.device
    d_rows = _row_output(None, total, inputs, rows) if need_rows else None
    d_weights = torch.empty((experts, inputs, outputs), dtype=rows.dtype, device=dev) if need_weights else None
    d_bias = _empty(torch, experts, outputs, rows.dtype, dev) if bias else None
    L = _abi.lib()
    d, x, w = d_out.data_ptr(), rows.data_ptr(), weights.data_ptr()
    d_ld, ld = _matrix(d_out, "d_out"), _matrix(rows, "rows")
    space, need, at = _space(L, code, total, experts, inputs, outputs, d | x | w, d_ld | ld | w_ld | stride, 1, dev)
    _call(L.ponni_b200_expert_product_backward(
        code, d, d_ld, x, ld, total, w, w_ld, stride, offset.data_ptr(), experts, inputs, outputs,
        None if d_rows is None else d_rows.data_ptr(), 0 if d_rows is None else _matrix(d_rows, "d_rows"),
        None if d_weights is None else d_weights.data_ptr(), None if d_bias is None else d_bias.data_ptr(), at, need,
        dev.index, torch_stream_handle(dev)))
    return d_rows, d_weights, d_bias


class GradientSet:
    """Gradient tensors that are clipped together by their global norm.

    Made once over buffers that keep their memory from step to step (the set
    holds references to them); dense CUDA tensors of one device, any mix of
    fp32, fp64, fp16 and bf16.
    """

    def __init__(self, tensors):
        _torch()
        self.tensors = list(tensors)
        self._set = None
        if not self.tensors:
            _refuse("a gradient set needs at least one tensor")
        dev = self.tensors[0].device
        n = len(self.tensors)
        ptrs, counts, kinds = (ctypes.c_void_p * n)(), (ctypes.c_int64 * n)(), (ctypes.c_int32 * n)()
        for i, t in enumerate(self.tensors):
            if not t.is_cuda or t.device != dev:
                _refuse(f"tensor {i} is on {t.device}; the set needs CUDA tensors of one device")
            if t.dtype not in _codes:
                _refuse(f"tensor {i} is {t.dtype}, not fp32, fp64, fp16 or bf16", 3)
            if not t.is_contiguous():
                _refuse(f"tensor {i} is not dense")
            ptrs[i], counts[i], kinds[i] = t.data_ptr(), t.numel(), _codes[t.dtype]
        self.device = dev
        L = _abi.lib()
        handle = ctypes.c_void_p()
        _call(L.ponni_b200_gradient_set_create(ptrs, counts, kinds, n, dev.index, ctypes.byref(handle)))
        self._set = handle
        self.total = int(L.ponni_b200_gradient_set_count(handle))
        self._workspace = int(L.ponni_b200_gradient_set_workspace(handle))

    def __del__(self):
        s = getattr(self, "_set", None)
        if s:
            try:
                _abi.lib().ponni_b200_gradient_set_destroy(s)
            except Exception:
                pass
            self._set = None

    def clip(self, max_norm: float, out=None):
        """The norm of all gradients together (fp32 tensor without dimensions).

        Where it is finite and above max_norm the gradients are scaled by
        max_norm / norm: in place, or into `out`, a dense vector of `total`
        values that receives all gradients in tensor order (the order of
        Inference.set_trainable_parameters_device) and leaves them as they are.
        Tensors that share elements are refused in place; `out` may share memory
        with a tensor only as the very place of its values (a view of `out`).
        """
        torch = _torch()
        kind, flat = 0, None
        if out is not None:
            if out.device != self.device or out.dim() != 1 or out.numel() != self.total or not out.is_contiguous():
                _refuse(f"out must be a dense vector of {self.total} values on {self.device}", 2)
            if out.dtype not in _codes:
                _refuse(f"out is {out.dtype}, not fp32, fp64, fp16 or bf16", 3)
            kind, flat = _codes[out.dtype], out.data_ptr()
        # The norm, then (8-byte aligned) the partial sums.
        buf = torch.empty(2 + self._workspace // 4, dtype=torch.float32, device=self.device)
        at = buf.data_ptr()
        _call(_abi.lib().ponni_b200_gradient_set_clip(self._set, float(max_norm), flat, kind, at, at + 8,
                                                      self._workspace, torch_stream_handle(self.device)))
        return buf[0]


def clip_gradients(tensors, max_norm: float, out=None):
    """GradientSet(tensors).clip(max_norm, out) for gradients whose memory changes from step to step.

    Makes the set's table and waits for the stream on every call (150 us more than a clip of a set).
    """
    s = GradientSet(tensors)
    norm = s.clip(max_norm, out)
    _torch().cuda.current_stream(s.device).synchronize()  # the set's table must outlive the kernels
    return norm


def check_operators(device=None) -> None:
    """Waits for the current stream; raises PonniError if an operator found group offsets out of order or gave up."""
    torch = _torch()
    dev = torch.device("cuda" if device is None else device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    _call(_abi.lib().ponni_b200_operator_check(dev.index, torch_stream_handle(dev)))
