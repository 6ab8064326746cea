"""What rows through experts refuse, in Python and at the C entry points: no GPU needed, nothing is queued."""
import ctypes as C

import pytest
import torch


def _plan(evt, rows=4, top=2, experts=5, device=-1):
    n = rows * top
    return evt.RowPlan(rows, top, experts, device, torch.device("cpu"), torch.zeros(2 * n + experts + 1, dtype=torch.int32))


def test_scores_and_choices_are_checked(evt):
    x = torch.zeros(4, 10)
    ids, w = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for bad, error in ((x.double(), TypeError), (x.numpy(), TypeError), (x[0], ValueError), (torch.zeros(4, 4097), ValueError), (torch.zeros(10, 4).t(), ValueError)):
        with pytest.raises(error):
            evt.route_rows(bad, 2)
        with pytest.raises(error):
            evt.route_rows_grad(bad, ids, w, w)
    for top, error in ((0, ValueError), (11, ValueError), (-1, ValueError), (1.5, TypeError), (None, TypeError)):
        with pytest.raises(error, match="top"):
            evt.route_rows(x, top)
    with pytest.raises(ValueError, match="top"):
        evt.route_rows(torch.zeros(4, 100), 65)
    for T in (0.0, float("nan"), 1e5):
        with pytest.raises(ValueError, match="temperature"):
            evt.route_rows(x, 2, temperature=T)
    for bad in (ids[:3], ids.short(), ids[0], torch.zeros(4, 11, dtype=torch.int32), None):
        with pytest.raises((ValueError, TypeError)):
            evt.route_rows_grad(x, bad, w, w)
    for bad in (w[:, :1], w.double(), torch.zeros(4, 4)[:, ::2], 1.0):
        with pytest.raises((ValueError, TypeError), match="weights"):
            evt.route_rows_grad(x, ids, bad, w)
        with pytest.raises((ValueError, TypeError), match="dweights"):
            evt.route_rows_grad(x, ids, w, bad)
    with pytest.raises(ValueError, match="out"):
        evt.route_rows_grad(x, ids, w, w, out=x.half())
    for call in (lambda: evt.route_rows(x, 2), lambda: evt.route_rows_grad(x, ids, w, w), lambda: evt.plan_rows(ids, 3)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()


def test_plans_are_checked(evt):
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for bad, error in ((ids.float(), TypeError), (ids.short(), TypeError), (ids[None], ValueError), (torch.zeros(4, 0, dtype=torch.int32), ValueError), ([0], TypeError),
                       (ids.t(), ValueError), (ids[::2], ValueError), (torch.zeros((), dtype=torch.int32), ValueError)):
        with pytest.raises(error):
            evt.plan_rows(bad, 3)
    for n, error in ((0, ValueError), (4097, ValueError), (-1, ValueError), (2.0, TypeError)):
        with pytest.raises(error, match="n_experts"):
            evt.plan_rows(ids, n)
    x, y = torch.zeros(4, 6), torch.zeros(8, 6)
    plan, w = _plan(evt), torch.zeros(4, 2)
    calls = {"sort": lambda x, plan: evt.sort_rows(x, plan), "combine": lambda x, plan: evt.combine_rows(x, plan, w),
             "grad": lambda x, plan: evt.combine_rows_grad(x, y, plan, w)}
    for name, call in calls.items():
        good = y if name == "combine" else x
        for bad in (None, ids, (ids, ids, ids)):
            with pytest.raises(TypeError, match="plan"):
                call(good, bad)
        with pytest.raises(ValueError, match="plan"):
            call(good, _plan(evt, rows=5))
        with pytest.raises(ValueError, match="the plan is on"):
            call(good, _plan(evt, device=0))
        for bad, error in ((good.double(), TypeError), (good[0], ValueError), (good.tolist(), TypeError), (torch.zeros(6, good.shape[0]).t(), ValueError),
                           (good[:, :0], ValueError)):
            with pytest.raises(error):
                call(bad, plan)
        with pytest.raises(ValueError, match="on a GPU"):
            call(good, plan)


def test_rows_are_checked(evt):
    x, y, w, plan = torch.zeros(4, 6), torch.zeros(8, 6), torch.zeros(4, 2), _plan(evt)
    for bad in (w[:3], w.double(), w.half(), torch.zeros(2, 4).t(), 1.0):
        with pytest.raises((ValueError, TypeError), match="weights"):
            evt.combine_rows(y, plan, bad)
        with pytest.raises((ValueError, TypeError), match="weights"):
            evt.combine_rows_grad(x, y, plan, bad)
    with pytest.raises(ValueError, match="weights"):
        evt.combine_rows_grad(x, y, plan, None)
    for bad in (x[:3], x.double(), x.half(), torch.zeros(6, 4).t(), x[:, :5], 0):
        with pytest.raises((ValueError, TypeError), match="residual"):
            evt.combine_rows(y, plan, w, residual=bad)
        with pytest.raises((ValueError, TypeError), match="residual"):
            evt.drop_rows(x, 0.1, 1, residual=bad)
        with pytest.raises((ValueError, TypeError), match="out"):
            evt.combine_rows(y, plan, w, out=bad)
        with pytest.raises((ValueError, TypeError), match="out"):
            evt.drop_rows(x, 0.1, 1, out=bad)
    with pytest.raises(ValueError, match="out"):
        evt.drop_rows(x, 0.1, 1, out=torch.zeros(6).expand(4, 6))
    for bad in (y[:7], y.half(), y[:, :5], 0):
        with pytest.raises((ValueError, TypeError), match="y "):
            evt.combine_rows_grad(x, bad, plan, w)
        with pytest.raises((ValueError, TypeError), match="out"):
            evt.sort_rows(x, plan, out=bad)
    for p in (-0.1, 1.0, 1.5, float("nan")):
        for call in (lambda: evt.drop_rows(x, p, 1), lambda: evt.combine_rows(y, plan, w, p=p, seed=1), lambda: evt.combine_rows_grad(x, y, plan, w, p=p, seed=1)):
            with pytest.raises(ValueError, match="p must"):
                call()
    for seed, error in ((None, TypeError), (1.5, TypeError), (2 ** 64, ValueError), (-2 ** 63 - 1, ValueError), (torch.zeros(2, dtype=torch.int64), ValueError),
                        (torch.zeros(1), TypeError), (torch.zeros(1, dtype=torch.int32), TypeError)):
        with pytest.raises(error, match="seed"):
            evt.drop_rows(x, 0.1, seed)
    for layer, error in ((-1, ValueError), (2 ** 32, ValueError), (0.5, TypeError)):
        with pytest.raises(error, match="layer"):
            evt.drop_rows(x, 0.1, 1, layer=layer)
    for call in (lambda: evt.drop_rows(x, 0.1, 1), lambda: evt.drop_rows(x, 0.0, None)):
        with pytest.raises(ValueError, match="on a GPU"):
            call()


def _code(evt, name, *args):
    rc = getattr(evt._lib.load(), name)(None, *args)
    return rc, evt._lib.load().evt_last_error().decode()


def test_entry_points_refuse(evt):
    ARG, F32 = evt._lib.EVT_ERR_ARG, 0
    mem = (C.c_char * 4096)()
    at = C.addressof(mem)

    def scores(**more):
        v = dict(x=at, row_stride=8, grad=at + 1024, grad_stride=8, nrows=4, nclass=8, dtype=F32, temperature=1.0)
        v.update(more)
        return C.byref(evt._lib.EvtScores(**v))

    def rows(**more):
        v = dict(x=at, x_stride=8, out=at + 1024, out_stride=8, residual=None, residual_stride=0, nrows=4, nfeats=8, dtype=F32, p=0.0, seed=0, seed_dev=None, layer=0)
        v.update(more)
        return C.byref(evt._lib.EvtRows(**v))

    for name, args, message in (
            ("evt_route_rows", (None, 2, 1, at, at, 2), "scores"), ("evt_route_rows", (scores(nclass=4097), 2, 1, at, at, 2), "nclass"),
            ("evt_route_rows", (scores(), 9, 1, at, at, 2), "top"), ("evt_route_rows", (scores(), 0, 1, at, at, 2), "top"), ("evt_route_rows", (scores(), 2, 2, at, at, 2), "renormalize"),
            ("evt_route_rows", (scores(dtype=1), 2, 1, at, at, 2), "EVT_F32"), ("evt_route_rows", (scores(temperature=0.0), 2, 1, at, at, 2), "temperature"),
            ("evt_route_rows", (scores(x=at + 2), 2, 1, at, at, 2), "aligned"), ("evt_route_rows", (scores(), 2, 1, None, at, 2), "NULL"),
            ("evt_route_rows", (scores(), 2, 1, at, at, 1), "flags"), ("evt_route_rows", (scores(), 2, 1, at, at, 0), "device memory"),
            ("evt_route_rows_grad", (scores(), 2, 1, at, 3, at, at, 2), "EVT_I32"), ("evt_route_rows_grad", (scores(grad=at + 4), 2, 1, at, 4, at, at, 2), "own memory"),
            ("evt_route_rows_grad", (scores(grad=None), 2, 1, at, 4, at, at, 2), "NULL"), ("evt_route_rows_grad", (scores(), 2, 1, at, 4, at, at, 0), "device memory"),
            ("evt_plan_rows", (at, 4, 4, 2, 0, at, at, at, at, 2), "nexperts"), ("evt_plan_rows", (at, 4, 4, 0, 3, at, at, at, at, 2), "top"),
            ("evt_plan_rows", (at, 4, 1 << 30, 2, 3, at, at, at, at, 2), "nrows"), ("evt_plan_rows", (at, 4, 4, 2, 3, at, at, at, None, 2), "NULL"),
            ("evt_plan_rows", (at, 4, 4, 2, 3, at, at, None, at, 2), "NULL"), ("evt_plan_rows", (at, 4, 4, 2, 3, at, at, at, at, 0), "device memory"),
            ("evt_sort_rows", (None, at, at, 2, 3, 2), "rows"), ("evt_sort_rows", (rows(p=0.5), at, at, 2, 3, 2), "dropout"), ("evt_sort_rows", (rows(out=at + 64), at, at, 2, 3, 2), "apart"),
            ("evt_sort_rows", (rows(out=at), at, at, 1, 3, 2), "apart"), ("evt_sort_rows", (rows(), None, at, 2, 3, 2), "place"), ("evt_sort_rows", (rows(), at, None, 2, 3, 2), "offsets"),
            ("evt_sort_rows", (rows(out_stride=7), at, at, 2, 3, 2), "out_stride"), ("evt_sort_rows", (rows(), at, at, 2, 3, 0), "device memory"),
            ("evt_combine_rows", (rows(out=at), at, at, 1, 2), "apart"), ("evt_combine_rows", (rows(out=at + 32), at, at, 2, 2), "apart"),
            ("evt_combine_rows", (rows(residual=at + 1028, residual_stride=8), at, at, 2, 2), "residual"), ("evt_combine_rows", (rows(p=1.0), at, at, 2, 2), "p must"),
            ("evt_combine_rows", (rows(nrows=-1), at, at, 2, 2), "nrows"), ("evt_combine_rows", (rows(), at, at, 2, 0), "device memory"),
            ("evt_combine_rows_grad", (rows(), at + 2048, 8, at, at, at, None, 2, 3, 2), "together"), ("evt_combine_rows_grad", (rows(), at + 2048, 8, at, at, None, at, 2, 3, 2), "weights"),
            ("evt_combine_rows_grad", (rows(), at + 1024, 8, at, at, at, at, 2, 3, 2), "apart"), ("evt_combine_rows_grad", (rows(residual=at), at + 2048, 8, at, at, at, at, 2, 3, 2), "residual"),
            ("evt_combine_rows_grad", (rows(), at + 2050, 8, at, at, at, at, 2, 3, 2), "aligned"), ("evt_combine_rows_grad", (rows(), at + 2048, 8, at, at, at, at, 2, 3, 0), "device memory"),
            ("evt_drop_rows", (None, 2), "rows"), ("evt_drop_rows", (rows(nfeats=0), 2), "nfeats"), ("evt_drop_rows", (rows(x=None), 2), "NULL"), ("evt_drop_rows", (rows(x_stride=-1), 2), "strides"),
            ("evt_drop_rows", (rows(out=at + 4), 2), "apart"), ("evt_drop_rows", (rows(p=float("nan")), 2), "p must"), ("evt_drop_rows", (rows(), 0), "device memory")):
        rc, error = _code(evt, name, *args)
        assert rc == ARG and message in error, (name, rc, error, message)
    for name, args in (("evt_route_rows", (scores(nrows=0), 2, 1, None, None, 2)), ("evt_sort_rows", (rows(nrows=0), None, None, 2, 3, 2)),
                       ("evt_combine_rows", (rows(nrows=0), None, None, 2, 2)), ("evt_drop_rows", (rows(nrows=0, x=None, out=None), 2))):
        assert _code(evt, name, *args)[0] == 0


def test_bytes_are_the_structures(evt):
    import sys
    rows = sys.modules[evt.RowPlan.__module__]
    v = (1 << 40, 2, 1 << 41, 3, 1 << 42, 4, 5, 6, 7, 0.5, 2 ** 64 - 1, 1 << 43, 2 ** 32 - 1)
    r = evt._lib.EvtRows.from_buffer_copy(rows._rows_bytes(*v))
    assert tuple(getattr(r, f[0]) for f in r._fields_) == v and C.sizeof(r) == len(rows._rows_bytes(*v))
    v = (1 << 40, 2, 1 << 41, 3, 4, 5, 6, 0.25)
    r = evt._lib.EvtScores.from_buffer_copy(rows._scores_bytes(*v))
    assert tuple(getattr(r, f[0]) for f in r._fields_) == v and C.sizeof(r) == len(rows._scores_bytes(*v))


def test_work_of_the_tables_is_the_headers(evt):
    """plan_rows' share of its tensor, by the macro's own text."""
    import os
    import re
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "evotrees_hip.h")) as f:
        header = f.read()
    assert re.search(r"EVT_PLAN_BLOCK\(n\) \(\(n\) <= 1 << 20 \? 1024 : 4096\)", header)
    with open(evt.RowPlan.__init__.__code__.co_filename) as f:
        assert "1024 if n <= 1 << 20 else 4096" in f.read()
