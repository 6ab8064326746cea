"""Rows through experts (route_rows, plan_rows, sort_rows, combine_rows, drop_rows and the gradients) against their formulas in 64 bits: every type, sizes from one to many, odd
ones, rows that lie anywhere, entries without an expert, values that are none."""
import math

import pytest
import torch

import expert_rows_plain as plain

pytestmark = pytest.mark.gpu

EXPERTS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 64, 97, 128, 255, 256, 257, 511, 1000, 1024, 1025, 2048, 4095, 4096]
FEATURES = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 64, 100, 127, 130, 255, 257, 511, 1000, 1023, 1025, 2047, 2048, 4099, 8200, 16384]
DTYPES = list(plain.TYPES)


def _placed(x, pad, shift):
    """x on the GPU with rows pad elements further apart and the first one shift elements behind an aligned address."""
    N, V = x.shape
    base = torch.full((N * (V + pad) + shift + 1,), 7.0, dtype=x.dtype, device="cuda")
    view = base[shift:].as_strided((N, V), (V + pad, 1))
    view.copy_(x)
    return view


def _scores(V, dtype, seed, N=13):
    """Row 1 is masked but for one expert, row 2 altogether, row 3 holds a NaN, row 4 a +inf, row 5 equal scores, row 6 zeros of both signs, row 7 half masked, row 8 large."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=gen) * 2
    x[1, :V - 1] = -math.inf
    x[2] = -math.inf
    x[3, V // 2] = math.nan
    x[4, V - 1] = math.inf
    x[5] = 0.25
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7, :V // 2] = -math.inf
    x[8] = x[8] * 1000
    return x.to(dtype), gen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", EXPERTS)
def test_route_rows(evt, V, dtype):
    x, gen = _scores(V, plain.TYPES[dtype], V)
    for top in sorted({1, min(2, V), min(8, V), min(5, V), min(64, V)}):
        renormalize, T = (V + top) % 2 == 0, [1.0, 0.7, 2.0][(V + top) % 3]
        xg = _placed(x, V % 3, V % 5)
        ids, w = evt.route_rows(xg, top, renormalize=renormalize, temperature=T)
        want, ww, tol = plain.route(x, top, renormalize, T)
        assert torch.equal(ids.cpu(), want), (top, (ids.cpu() != want).nonzero()[:3])
        plain.close("weights", w, ww, tol)
        dw = torch.randn(13, top, generator=gen)
        dw[want < 0] = math.nan  # nobody's
        given = want.clone()
        if V > 1:
            given[9, 0] = V  # no expert
        if top > 1:
            given[10, 1] = given[10, 0]  # one expert twice
        ws = w.cpu()
        grad = evt.route_rows_grad(xg, (given if top % 2 else given.long()).cuda(), w, dw.cuda(), renormalize=renormalize, temperature=T)
        want_g, tol_g = plain.route_grad(x, given, ws, dw, renormalize, T)
        if not renormalize:
            want_g[3], want_g[4] = math.nan, math.nan
        plain.close("grad", grad, want_g, tol_g)


def _ids(rows, top, experts, seed, missing=0.1):
    gen = torch.Generator().manual_seed(seed)
    ids = (torch.rand(rows, top, generator=gen) ** 2 * experts).long().clamp(max=experts - 1)
    lost = torch.rand(rows, top, generator=gen) < missing
    ids[lost] = torch.tensor([-1, -100, experts, experts + 7, 2 ** 31 - 1])[torch.randint(0, 5, (int(lost.sum()),), generator=gen)]
    if rows > 3:
        ids[rows // 2] = -1  # a row without any
    return ids, gen


@pytest.mark.parametrize("rows,top,experts", [(0, 3, 5), (1, 1, 1), (1, 8, 256), (3, 2, 4096), (21, 3, 7), (64, 1, 64), (65, 1, 2), (1000, 8, 128), (1024, 8, 1024), (1025, 8, 1024),
                                              (1024, 4, 1025), (2000, 5, 3), (1024, 8, 4096), (16384, 8, 64), (4096, 8, 4095), (131072, 1, 33), (131073, 1, 1), (70001, 3, 1000),
                                              (200003, 2, 4096)])
def test_plan_rows(evt, rows, top, experts):
    ids, _ = _ids(rows, top, experts, rows + top)
    place, source, offsets = plain.plan(ids, experts)
    for kind in (torch.int32, torch.int64):
        for _ in range(2):
            plan = evt.plan_rows(ids.to(kind).cuda(), experts)
            assert plan.place.cpu().reshape(-1).tolist() == place
            assert plan.source.tolist() == source
            assert plan.offsets.tolist() == offsets
            assert plan.place.shape == (rows, top) and plan.place.dtype == plan.source.dtype == plan.offsets.dtype == torch.int32
    if top == 1:
        assert torch.equal(evt.plan_rows(ids[:, 0].cuda(), experts).place.cpu().reshape(-1), torch.tensor(place, dtype=torch.int32))


def test_ids_of_64_bits_beyond_32(evt):
    ids = torch.tensor([[2 ** 32, 1], [2 ** 32 + 1, 0], [-2 ** 40, 1]])
    plan = evt.plan_rows(ids.cuda(), 2)
    assert plan.place.tolist() == [[-1, 1], [-1, 0], [-1, 2]] and plan.offsets.tolist() == [0, 1, 3]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", FEATURES)
def test_rows_there_and_back(evt, H, dtype):
    rows, top, experts = 19, [1, 2, 3, 8, 9, 17][H % 6], 11
    ids, gen = _ids(rows, top, experts, H)
    place = torch.tensor(plain.plan(ids, experts)[0]).view(rows, top)
    t = plain.TYPES[dtype]
    x = torch.randn(rows, H, generator=gen).to(t)
    plan = evt.plan_rows(ids.cuda(), experts)
    n = rows * top
    out = _placed(torch.full((n, H), 5.0).to(t), 3, H % 3)
    got = evt.sort_rows(_placed(x, H % 4, (H + 1) % 5), plan, out=out)
    want = torch.zeros(n, H, dtype=t)
    for r in range(rows):
        for j in range(top):
            if place[r, j] >= 0:
                want[place[r, j]] = x[r]
    assert got is out and torch.equal(got.cpu(), want)
    beyond = out.as_strided((n, 3), (H + 3, 1), out.storage_offset() + H)
    assert torch.equal(beyond, torch.full_like(beyond, 7.0))  # between the rows
    assert torch.equal(evt.sort_rows(x.cuda(), plan).cpu(), want)

    y = torch.randn(n, H, generator=gen).to(t)
    w = torch.rand(rows, top, generator=gen)
    used = torch.zeros(n, dtype=torch.bool)
    used[place[place >= 0]] = True
    y[~used] = math.nan  # nobody's rows
    w[place < 0] = math.nan
    res, dout = torch.randn(rows, H, generator=gen).to(t), torch.randn(rows, H, generator=gen).to(t)
    yg, wg = _placed(y, (H + 1) % 4, H % 5), w.cuda()
    for p, layer, residual, weights in ((0.0, 0, None, None), (0.0, 0, res, w), (0.3, 5, res, w), (0.1, 0, None, w)):
        seed = 1234567 * H + layer
        got = evt.combine_rows(yg, plan, None if weights is None else wg, residual=None if residual is None else _placed(residual, 1, 1), p=p, seed=seed, layer=layer)
        plain.close("combine", got, *plain.combine(y, place, weights, residual, p, seed, layer))
        dy, dw = evt.combine_rows_grad(_placed(dout, 2, 1), None if weights is None else yg, plan, None if weights is None else wg, p=p, seed=seed, layer=layer)
        want_y, want_w = plain.combine_grad(dout, None if weights is None else y, place, weights, p, seed, layer)
        plain.close("dy", dy, *want_y)
        if weights is None:
            assert dw is None
        else:
            plain.close("dweights", dw, *want_w)
            again = evt.combine_rows_grad(dout.cuda(), None, plan, wg, p=p, seed=seed, layer=layer)
            assert torch.equal(again[0], dy) and again[1] is None
    onto = res.cuda()
    assert evt.combine_rows(yg, plan, wg, residual=onto, p=0.3, seed=9, layer=1, out=onto) is onto
    plain.close("onto the residual", onto, *plain.combine(y, place, w, res, 0.3, 9, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H", FEATURES)
def test_drop_rows(evt, H, dtype):
    rows, t = 23, plain.TYPES[dtype]
    gen = torch.Generator().manual_seed(H)
    x, res = torch.randn(rows, H, generator=gen).to(t), torch.randn(rows, H, generator=gen).to(t)
    for p, seed, layer in ((0.25, 0, 0), (0.1, -1, 1), (0.5, 2 ** 64 - 1, 2 ** 32 - 1), (0.9999, 77, 3), (0.0, None, 0), (1e-9, 5, 5)):
        xg = _placed(x, H % 3, H % 4)
        want, tol = plain.drop(x, p, seed or 0, layer, None)
        got = evt.drop_rows(xg, p, seed, layer=layer)
        plain.close("drop", got, want, tol)
        if p:
            as_int = (seed + 2 ** 63) % 2 ** 64 - 2 ** 63
            held = torch.tensor([as_int], device="cuda")
            assert torch.equal(evt.drop_rows(xg, p, held, layer=layer), got) and torch.equal(evt.drop_rows(xg, p, held[0], layer=layer), got)
        want, tol = plain.drop(x, p, seed or 0, layer, res)
        plain.close("residual", evt.drop_rows(xg, p, seed, layer=layer, residual=_placed(res, 2, 1)), want, tol)
        onto, held = x.cuda(), res.cuda()
        version = onto._version
        assert evt.drop_rows(onto, p, seed, layer=layer, residual=held, out=onto) is onto and onto._version > version
        plain.close("in place", onto, want, tol)
        assert evt.drop_rows(x.cuda(), p, seed, layer=layer, residual=held, out=held) is held
        plain.close("onto the residual", held, want, tol)
