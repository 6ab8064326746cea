"""Rows through experts in calls that lie at the edge of what is allowed: empty batches, memory that is shared, more rows than a launch has, threads."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(evt, top, dtype):
    """An empty micro-batch through all of a layer."""
    scores, x = torch.zeros(0, 7, dtype=dtype, device="cuda"), torch.zeros(0, 5, dtype=dtype, device="cuda")
    ids, w = evt.route_rows(scores, top)
    plan = evt.plan_rows(ids[:, 0].contiguous() if top == 1 else ids, 7)
    assert plan.place.shape == (0, top) and plan.offsets.tolist() == [0] * 8
    y = evt.sort_rows(x, plan)
    out = evt.combine_rows(y, plan, w, residual=x, p=0.1, seed=1)
    dy, dw = evt.combine_rows_grad(out, y, plan, w, p=0.1, seed=1)
    dx = evt.combine_rows(dy, plan, residual=out)
    assert y.shape == out.shape == dy.shape == dx.shape == (0, 5) and dw.shape == (0, top) and evt.combine_rows_grad(out, None, plan, None)[1] is None
    assert evt.route_rows_grad(scores, ids, w, dw).shape == (0, 7)
