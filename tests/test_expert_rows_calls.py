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
