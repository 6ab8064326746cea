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
