"""Calls of rows through experts that are allowed or refused by what lies where: no GPU needed, nothing is queued."""
import ctypes as C

import pytest
import torch

TRUSTED = 2
MEM = (C.c_char * 8192)()
AT = (C.addressof(MEM) + 63) // 64 * 64


def rows(evt, **more):
    v = dict(x=AT, x_stride=8, out=AT + 1024, out_stride=8, residual=None, residual_stride=0, nrows=4, nfeats=8, dtype=0, p=0.0, seed=0, seed_dev=None, layer=0)
    v.update(more)
    return C.byref(evt._lib.EvtRows(**v))


def scores(evt, **more):
    v = dict(x=AT, row_stride=8, grad=AT + 1024, grad_stride=8, nrows=4, nclass=8, dtype=0, temperature=1.0)
    v.update(more)
    return C.byref(evt._lib.EvtScores(**v))


def call(evt, name, *args):
    rc = getattr(evt._lib.load(), name)(None, *args)
    return rc, evt._lib.load().evt_last_error().decode()


@pytest.mark.parametrize("top", [1, 2])
@pytest.mark.parametrize("at", [None, AT], ids=["NULL", "memory"])
def test_no_rows(evt, top, at):
    """Tensors without elements have no address: x and out are both NULL."""
    none = rows(evt, nrows=0, x=at, out=at)
    for name, args in (("evt_sort_rows", (none, None, None, top, 3, TRUSTED)), ("evt_combine_rows", (none, None, None, top, TRUSTED)),
                       ("evt_combine_rows_grad", (none, None, 8, None, None, None, None, top, 3, TRUSTED))):
        rc, error = call(evt, name, *args)
        assert rc == 0, (name, error)


def test_columns_of_one_matrix(evt):
    """Rows of equal strides side by side share no byte.  Host memory: what lies apart is refused for that, and only for that."""
    def says(name, *args):
        rc, error = call(evt, name, *args, 0)
        assert rc == evt._lib.EVT_ERR_ARG
        return error

    def apart(error):
        return "device memory" in error

    for out, stride, good in ((8, 16, True), (8, 24, True), (16, 24, True), (-8, 16, True), (-16, 24, True), (7, 16, False), (9, 16, False), (8, 15, False), (1, 16, False), (17, 24, False),
                              (16 + 8, 16, True), (16 + 4, 16, False), (-4, 16, False), (16, 16, False), (100, 16, True)):
        base = AT + 2048
        one = rows(evt, x=base, x_stride=stride, out=base + 4 * out, out_stride=stride)
        two = rows(evt, x=AT, residual=base, residual_stride=stride, out=base + 4 * out, out_stride=stride)
        assert apart(says("evt_drop_rows", one)) == good and apart(says("evt_drop_rows", two)) == good, (out, stride)
        assert apart(says("evt_sort_rows", one, AT, AT, 2, 3)) == good, (out, stride)
        three = scores(evt, x=base, row_stride=stride, grad=base + 4 * out, grad_stride=stride)
        assert apart(says("evt_route_rows_grad", three, 2, 1, AT, 4, AT, AT)) == good, (out, stride)
    base = AT + 2048
    # rows at two strides, and one row among the other's: only what is known to lie apart
    assert not apart(says("evt_drop_rows", rows(evt, x=base, x_stride=32, out=base + 32, out_stride=16)))
    assert not apart(says("evt_drop_rows", rows(evt, x=base, x_stride=0, out=base + 16, out_stride=16)))
    assert apart(says("evt_sort_rows", rows(evt, x=base + 32, x_stride=5, nrows=1, out=base, out_stride=16), AT, AT, 2, 3))
    assert not apart(says("evt_sort_rows", rows(evt, x=base + 16, x_stride=5, nrows=1, out=base, out_stride=16), AT, AT, 2, 3))
    assert not apart(says("evt_drop_rows", rows(evt, x=base + 16, x_stride=16, nrows=1, out=base, out_stride=16)))
    # half-precision columns
    assert apart(says("evt_drop_rows", rows(evt, x=base, x_stride=16, out=base + 16, out_stride=16, dtype=10)))
    assert not apart(says("evt_drop_rows", rows(evt, x=base, x_stride=16, out=base + 14, out_stride=16, dtype=10)))


def test_results_on_tables(evt):
    """A result that lies on what the call reads beside its rows would be written before another thread has read that."""
    x, out, place, w, offsets, seed, dw, y = (AT + 512 * i for i in range(8))  # 4 rows of 8 values, 2 experts each of 3; sorted rows are 256 bytes
    given = dict(x=x, out=out)

    def refused(name, *args):
        rc, error = call(evt, name, *args, TRUSTED)
        return rc == evt._lib.EVT_ERR_ARG and "apart" in error, error

    for at in (out, out - 28, out + 252):  # 8 entries of 4 bytes
        for name, args in (("evt_sort_rows", (rows(evt, **given), at, offsets, 2, 3)), ("evt_combine_rows", (rows(evt, x=x, out=out, nrows=8), at, w, 1)),
                           ("evt_combine_rows", (rows(evt, x=x, out=out, nrows=8), place, at, 1)), ("evt_combine_rows_grad", (rows(evt, **given), y, 8, at, offsets, w, dw, 2, 3)),
                           ("evt_combine_rows_grad", (rows(evt, **given), y, 8, place, offsets, at, dw, 2, 3)), ("evt_combine_rows_grad", (rows(evt, **given), y, 8, place, offsets, w, at, 2, 3)),
                           ("evt_route_rows", (scores(evt, x=out, nrows=8), 1, 1, at, w)), ("evt_route_rows", (scores(evt, x=out, nrows=8), 1, 1, place, at)),
                           ("evt_route_rows_grad", (scores(evt, x=x, grad=out, nrows=8), 1, 1, at, 4, w, dw)), ("evt_route_rows_grad", (scores(evt, x=x, grad=out, nrows=8), 1, 1, place, 4, at, dw)),
                           ("evt_route_rows_grad", (scores(evt, x=x, grad=out, nrows=8), 1, 0, place, 4, w, at))):
            no, error = refused(name, *args)
            assert no, (name, at - out, error)
    no, error = refused("evt_route_rows_grad", scores(evt, x=x, grad=out, nrows=8), 1, 1, out - 56, 5, w, dw)  # ids of 8 bytes
    assert no, error
    for at in (out - 12, out + 252):
        no, error = refused("evt_sort_rows", rows(evt, **given), place, at, 2, 3)
        assert no, error
    for at in (out, out + 120):
        for name, args in (("evt_drop_rows", (rows(evt, x=x, out=out, p=0.5, seed_dev=at),)), ("evt_combine_rows", (rows(evt, x=x, out=out, p=0.5, seed_dev=at), place, w, 2)),
                           ("evt_combine_rows_grad", (rows(evt, x=x, out=out, p=0.5, seed_dev=at), None, 0, place, offsets, w, None, 2, 3))):
            no, error = refused(name, *args)
            assert no, (name, error)
    for at in (x, x + 124, y, y + 252, place, place + 28, w - 28, offsets + 12, offsets - 28, seed + 4):
        no, error = refused("evt_combine_rows_grad", rows(evt, x=x, out=out, p=0.5, seed_dev=seed), y, 8, place, offsets, w, at, 2, 3)
        assert no and "dweights" in error, (at, error)
    no, error = refused("evt_route_rows", scores(evt, x=x), 2, 1, w + 28, w)
    assert no, error
    work = 4 * 2 * 3  # one block's counts and the totals
    tables = dict(ids=x, place=out, source=place, offsets=w, work=seed)
    for first, size in (("place", 32), ("source", 32), ("offsets", 16), ("work", work)):
        for second in tables:
            if first != second:
                for kind in (4, 5):
                    t = dict(tables)
                    t[second] = t[first] + size - (8 if second == "ids" and kind == 5 else 4)
                    no, error = refused("evt_plan_rows", t["ids"], kind, 4, 2, 3, t["place"], t["source"], t["offsets"], t["work"])
                    assert no, (first, second, error)


def test_tables_are_aligned(evt):
    """A scalar load takes the four bytes below an address that is no multiple of four."""
    x, out, place, w, offsets, source, dw, y = (AT + 512 * i for i in range(8))
    given = rows(evt, x=x, out=out)
    calls = {"evt_route_rows": ((scores(evt, x=x), 2, 1, place, w), (3, 4)), "evt_sort_rows": ((given, place, offsets, 2, 3), (1, 2)),
             "evt_combine_rows": ((rows(evt, x=x, out=out, nrows=2), place, w, 2), (1, 2)), "evt_combine_rows_grad": ((given, y, 8, place, offsets, w, dw, 2, 3), (3, 4, 5, 6)),
             "evt_plan_rows": ((x, 4, 4, 2, 3, place, source, offsets, w), (0, 5, 6, 7, 8)), "evt_route_rows_grad": ((scores(evt, x=x, grad=out), 2, 1, place, 4, w, dw), (3, 5, 6))}
    wide = {"evt_plan_rows": 1, "evt_route_rows_grad": 4}  # where a call takes the type of its ids
    for name, (args, at) in calls.items():
        for k in at:
            for off in (1, 2, 3):
                wrong = list(args)
                wrong[k] += off
                rc, error = call(evt, name, *wrong, TRUSTED)
                assert rc == evt._lib.EVT_ERR_ARG and "aligned" in error, (name, k, off, error)
        if name in wide:
            wrong = list(args)
            wrong[wide[name]], wrong[at[0]] = 5, wrong[at[0]] + 4
            rc, error = call(evt, name, *wrong, TRUSTED)
            assert rc == evt._lib.EVT_ERR_ARG and "aligned" in error, (name, error)
