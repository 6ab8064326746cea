"""A plan's tables: what a copy of a plan has, and tables that are none.  No GPU needed."""
import copy
import io
import pickle

import pytest
import torch


def _plan(evt, rows=4, top=2, experts=5, more=0):
    n = rows * top
    tables = torch.arange(2 * n + experts + 1 + more, dtype=torch.int32)
    return evt.RowPlan(rows, top, experts, -1, torch.device("cpu"), tables)


@pytest.mark.parametrize("way", ["copy", "deepcopy", "pickle", "torch"])
def test_a_copy_reads_its_own_tables(evt, way):
    plan = _plan(evt, more=3)

    def saved():
        f = io.BytesIO()
        torch.save(plan, f)
        f.seek(0)
        return torch.load(f, weights_only=False)
    again = {"copy": lambda: copy.copy(plan), "deepcopy": lambda: copy.deepcopy(plan), "pickle": lambda: pickle.loads(pickle.dumps(plan)), "torch": saved}[way]()
    assert type(again) is evt.RowPlan and (again.rows, again.top, again.experts, again.device) == (4, 2, 5, -1)
    for name in ("place", "source", "offsets"):
        assert torch.equal(getattr(again, name), getattr(plan, name))
    assert again._at == again.place.data_ptr() and again.offsets_at == again.offsets.data_ptr() == again._at + 4 * 16
    if way != "copy":
        assert again._at != plan._at


def test_tables_that_are_none(evt):
    cpu, n = torch.device("cpu"), 2 * 8 + 6
    whole = torch.zeros(n + 8, dtype=torch.int32)
    evt.RowPlan(4, 2, 5, -1, cpu, whole[:n])
    for tables, error in ((whole[:n - 1], ValueError), (whole[1:n + 1], ValueError), (whole.long(), TypeError), (whole.tolist(), TypeError), (None, TypeError),
                          (torch.zeros(2 * n, dtype=torch.int32)[::2], ValueError), (torch.zeros(n, 1, dtype=torch.int32), ValueError)):
        with pytest.raises(error, match="tables"):
            evt.RowPlan(4, 2, 5, -1, cpu, tables)
    with pytest.raises(ValueError, match="the plan is on cuda:0, its tables are on cpu"):
        evt.RowPlan(4, 2, 5, 0, cpu, whole)
    for sizes in ((-1, 2, 5), (4, 0, 5), (4, 2, 0), (4, 2, 4097), (2 ** 31, 2, 5)):
        with pytest.raises(ValueError):
            evt.RowPlan(*sizes, -1, cpu, whole)
    with pytest.raises(TypeError):
        evt.RowPlan(4.0, 2, 5, -1, cpu, whole)
