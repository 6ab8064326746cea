"""A plan's tables: what a copy of a plan has, and tables that are none.  No GPU needed."""
import copy
import ctypes as C
import io
import os
import pickle
import subprocess
import sys

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


def _work_of(tmp_path):
    """EVT_PLAN_WORK as a C compiler has it."""
    source, built = tmp_path / "work.c", tmp_path / "work.so"
    source.write_text('#include "evotrees_hip.h"\nint64_t work(int64_t n, int32_t experts) { return EVT_PLAN_WORK(n, experts); }\n')
    subprocess.run(["gcc", "-shared", "-fPIC", "-I", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include"), "-o", str(built), str(source)], check=True)
    f = C.CDLL(str(built)).work
    f.argtypes, f.restype = [C.c_int64, C.c_int32], C.c_int64
    return f


def test_memory_of_a_plan(evt, monkeypatch, tmp_path):
    """What plan_rows allocates is the tables and EVT_PLAN_WORK behind them or by itself, and a plan keeps little more than its tables."""
    rows_module = sys.modules[evt.RowPlan.__module__]
    work_of, queued, made = _work_of(tmp_path), [], []

    class Memory(torch.Tensor):
        """On a GPU, as far as its checks see."""
        def get_device(self):
            return 0

    def make(device, dtype, shape, on):
        assert device == 0 and dtype == torch.int32
        made.append(torch.empty(shape, dtype=dtype))
        return made[-1]

    monkeypatch.setattr(rows_module, "_make", make)
    monkeypatch.setattr(rows_module, "_queue", lambda name, device, on, *args: queued.append((name, args)))
    for rows, top in ((0, 3), (1, 1), (16, 6), (1024, 1), (1025, 1), (341, 3), (4096, 8), (32768, 8), (131072, 8), (131072 * 8, 1), (131072 * 8 + 1, 1), (262144, 8)):
        for experts in (1, 7, 64, 128, 1000, 4096):
            del queued[:], made[:]
            n = rows * top
            plan = evt.plan_rows(torch.zeros(rows, top, dtype=torch.int32).as_subclass(Memory), experts)
            (name, args), = queued
            at, _, r, k, e, place, source, offsets, work = args
            assert name == "evt_plan_rows" and (r, k, e) == (rows, top, experts)
            first, size = made[0].data_ptr(), 4 * made[0].numel()
            assert (place, source, offsets) == (first, first + 4 * n, first + 8 * n)
            needed = 4 * work_of(n, experts)
            if len(made) == 1:
                assert work == offsets + 4 * (experts + 1) and work + needed == first + size
            else:
                assert len(made) == 2 and size == 8 * n + 4 * (experts + 1) and work == made[1].data_ptr() and needed == 4 * made[1].numel()
            kept = plan._tables.numel() * 4
            assert kept <= max(8 * n + 4 * (experts + 1) + 65536, (8 * n + 4 * (experts + 1)) * 9 // 8), (rows, top, experts, kept)
