"""What the calls on torch tensors keep for later calls is of ordinary tensors alone, whatever mode the first call was made in: no GPU needed."""
import sys
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.fixture
def modules(evt):
    rows = sys.modules[evt.RowPlan.__module__]
    kept = [(m, dict(m._makers)) for m in (rows, rows._scores)]
    for m, _ in kept:
        m._makers.clear()
    yield rows, rows._scores
    for m, makers in kept:
        m._makers.clear()
        m._makers.update(makers)


def test_a_tracers_mode(evt, modules):
    """Tensors without memory: the calls fail, in their own ways, and leave nothing of the mode behind."""
    rows, losses = modules
    with FakeTensorMode(allow_non_fake_inputs=True):
        x, w = torch.empty(4, 8, device="cuda"), torch.empty(4, 2, device="cuda")
        ids, labels = torch.empty(4, 2, dtype=torch.int32, device="cuda"), torch.empty(4, dtype=torch.int64, device="cuda")
        for call in (lambda: evt.route_rows(x, 2), lambda: evt.plan_rows(ids, 8), lambda: evt.route_rows_grad(x, ids, w, w), lambda: evt.drop_rows(x.t()[:4, :4].t(), 0.5, 1),
                     lambda: evt.class_logp(x, labels), lambda: evt.distill_loss(x, ids, w)):
            with warnings.catch_warnings(), pytest.raises(Exception):
                warnings.simplefilter("ignore")
                call()
    assert not rows._makers and not losses._makers


def test_a_function_transform(evt, modules):
    rows, losses = modules
    evt_torch = rows._torch()
    seen = []

    def f(x):
        for dtype in (torch.float32, torch.int32):
            seen.append(rows._make(0, dtype, (3,), torch.device("cpu")))  # as for a device: only those are kept
        return x.sum()
    for transform in (torch.func.functionalize, torch.func.grad):
        transform(f)(torch.ones(3))
        assert not rows._makers
    assert len(seen) == 4 and evt_torch is torch
    for dtype in (torch.float32, torch.int32):  # without one they are, and make ordinary tensors
        for mode in (torch.inference_mode, torch.enable_grad, torch.no_grad):
            with mode():
                made = rows._make(0, dtype, (3,), torch.device("cpu"))
                assert type(made) is torch.Tensor and made.data_ptr() and made.dtype == dtype and not made.requires_grad
        assert not rows._make(0, dtype, (3,), torch.device("cpu")).is_inference()
    assert set(rows._makers) == {(0, torch.float32), (0, torch.int32)}
