"""Mixture-of-experts operators without a GPU: refusals on host tensors, workspace sizes, plain forms."""
import numpy as np
import pytest

import ponni_b200 as pb
from ponni_b200 import _abi

torch = pytest.importorskip("torch")

from tests import expert_ref as R  # noqa: E402


def test_host_tensors_are_refused():
    x = torch.zeros(4, 6)
    r = pb.Routing(*(torch.zeros(2, 6, dtype=torch.int32),) * 4, torch.zeros(5, dtype=torch.int32))
    w, off = torch.zeros(4, 6, 3), torch.zeros(5, dtype=torch.int32)
    for f in (lambda: pb.route_columns(x, 2), lambda: pb.route_columns_backward(x, r, x[:2]),
              lambda: pb.gather_columns(x, r), lambda: pb.gather_columns_backward(x, r), lambda: pb.combine_rows(x, r),
              lambda: pb.combine_rows_backward(x, x, r), lambda: pb.expert_product(x, w, off),
              lambda: pb.expert_product_backward(x, x, w, off), lambda: pb.GradientSet([x]), lambda: pb.GradientSet([])):
        with pytest.raises(pb.PonniError) as e:
            f()
        assert e.value.status == 1


def test_workspaces():
    L = _abi.lib()
    # 16-bit operands on the 16-byte grid are read in place, others through copies; fp32 as three 16-bit parts.
    assert L.ponni_b200_expert_product_workspace(_abi.BF16, 1000, 4, 64, 128, 1, 0, 0) == 0
    pad = lambda n: (n + 255) // 256 * 256  # noqa: E731
    got = L.ponni_b200_expert_product_workspace(_abi.F16, 1000, 4, 50, 70, 0, 0, 0)
    assert got == pad(1000 * 56 * 2) + pad(4 * 50 * 72 * 2)
    got = L.ponni_b200_expert_product_workspace(_abi.F32, 1000, 4, 50, 70, 1, 0, 0)
    assert got == pad(1000 * 56 * 6) + pad(4 * 50 * 72 * 6)
    assert L.ponni_b200_expert_product_workspace(_abi.F32, 3, 4, 50, 70, 1, 0, 0) == 0  # a few rows: streamed as they lie
    assert L.ponni_b200_route_workspace(16, 1) == 0
    assert L.ponni_b200_route_workspace(16, 1 << 20) > 0
    assert L.ponni_b200_gradient_set_count(None) == 0


def test_calls_without_a_device_report_it():
    if torch.cuda.is_available():
        pytest.skip("this machine has a GPU")
    L = _abi.lib()
    assert L.ponni_b200_gradient_set_create(None, None, None, 0, 0, None) == 4
    assert b"no CUDA device" in L.ponni_b200_operator_error()
    assert L.ponni_b200_operator_check(0, None) == 4


def test_plain_route_by_hand():
    x = torch.tensor([[1.0, -np.inf, 2.0], [1.0, -np.inf, np.nan], [0.0, -np.inf, -np.inf]])
    expert, weight, row, column, offset = R.route(x, 2, "selected")
    assert expert.tolist() == [[0, -1, 0], [1, -1, -1]]
    assert weight.tolist() == [[0.5, 0.0, 1.0], [0.5, 0.0, 0.0]]
    assert row.tolist() == [[0, -1, 1], [2, -1, -1]]
    assert column.tolist() == [0, 2, 0, -1, -1, -1] and offset.tolist() == [0, 2, 3, 3]
    _, weight, *_ = R.route(x, 2, "all")
    assert weight[0, 0].item() == pytest.approx(1 / (2 + np.exp(-1)))


def test_plain_gradient_by_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 4, generator=g, dtype=torch.float64)
    d = torch.randn(3, 4, generator=g, dtype=torch.float64)
    for normalise in ("selected", "all"):
        expert, *_ = R.route(x, 3, normalise)
        grad = R.route_gradient(x, expert, d, normalise)
        for e in range(6):
            step = torch.zeros_like(x)
            step[e] = 1e-5
            up, down = R.route(x + step, 3, normalise), R.route(x - step, 3, normalise)
            assert torch.equal(up[0], expert) and torch.equal(down[0], expert)
            assert torch.allclose(((up[1] - down[1]) * d).sum(0) / 2e-5, grad[e], atol=1e-8)


def test_routings_of_a_wrong_shape_are_refused():
    """The checks themselves, on host tensors (the entry points refuse those before)."""
    from ponni_b200 import experts as X
    row, none = torch.zeros(2, 6, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    good = pb.Routing(row, row.float(), row, row.view(-1), torch.zeros(5, dtype=torch.int32))
    assert X._check_routing(good, row.device, 6) == 2
    for bad in (good._replace(offset=none), good._replace(offset=none.view(0, 1)), good._replace(offset=good.offset[:1]),
                good._replace(offset=good.offset[0]), good._replace(offset=good.offset.view(5, 1)),
                good._replace(row=row[0]), good._replace(row=row[0, 0]), good._replace(row=row.long())):
        with pytest.raises(pb.PonniError):
            X._check_routing(bad, row.device, 6)
