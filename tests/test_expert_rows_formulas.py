"""The 64-bit gradients that rows through experts are tested against, against differences of the 64-bit formulas: no GPU needed."""
import math

import pytest
import torch

import expert_rows_plain as plain


def _slope(f, x, at, step=1e-5):
    """Central difference of f by x[at]: off by step^2 times a third derivative, and the rounding of f over the step."""
    keep = float(x[at])
    x[at] = keep + step
    up = f()
    x[at] = keep - step
    down = f()
    x[at] = keep
    return (up - down) / (2 * step)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("top,T", [(1, 1.0), (3, 0.7), (7, 2.0)])
def test_choice(renormalize, top, T):
    gen = torch.Generator().manual_seed(top)
    x = torch.randn(4, 9, generator=gen, dtype=torch.float64)
    x[1, 2:] = -math.inf  # fewer than are asked for
    dw = torch.randn(4, top, generator=gen, dtype=torch.float64)
    ids, w, _ = plain.route(x, top, renormalize, T)
    grad = plain.route_grad(x, ids, w, dw, renormalize, T)[0]

    def f():
        return float((plain.route(x, top, renormalize, T)[1] * dw).sum())
    for i in range(4):
        for c in range(9):
            if x[i, c] != -math.inf:
                assert abs(_slope(f, x, (i, c)) - float(grad[i, c])) < 1e-8, (i, c)


@pytest.mark.parametrize("p", [0.0, 0.3])
def test_combination(p):
    gen = torch.Generator().manual_seed(5)
    ids = torch.tensor([[0, 2], [1, -1], [-1, -1], [2, 0]])
    place = torch.tensor(plain.plan(ids, 3)[0]).view(4, 2)
    y, w, dout = (torch.randn(s, generator=gen, dtype=torch.float64) for s in ((8, 6), (4, 2), (4, 6)))
    (dy, _), (dw, _) = plain.combine_grad(dout, y, place, w, p, 11, 2)

    def f():
        return float((plain.combine(y, place, w, None, p, 11, 2)[0] * dout).sum())
    for at in [(i, c) for i in range(8) for c in range(6)]:
        assert abs(_slope(f, y, at) - float(dy[at])) < 1e-8
    for at in [(i, j) for i in range(4) for j in range(2)]:
        assert abs(_slope(f, w, at) - float(dw[at])) < 1e-8


def test_sorting_and_dropout():
    gen = torch.Generator().manual_seed(6)
    ids = torch.tensor([[0, 2], [1, -1], [-1, -1], [2, 0]])
    place = torch.tensor(plain.plan(ids, 3)[0]).view(4, 2)
    x, dsorted = torch.randn(4, 5, generator=gen, dtype=torch.float64), torch.randn(8, 5, generator=gen, dtype=torch.float64)

    def f():
        return float(sum((x[r] * dsorted[place[r, j]]).sum() for r in range(4) for j in range(2) if place[r, j] >= 0))
    want = plain.combine(dsorted, place, None, None, 0.0, 0, 0)[0]
    for at in [(i, c) for i in range(4) for c in range(5)]:
        assert abs(_slope(f, x, at) - float(want[at])) < 1e-8

    dout = torch.randn(4, 5, generator=gen, dtype=torch.float64)

    def g():
        return float((plain.drop(x, 0.4, 3, 1, None)[0] * dout).sum())
    want = plain.drop(dout, 0.4, 3, 1, None)[0]
    for at in [(i, c) for i in range(4) for c in range(5)]:
        assert abs(_slope(g, x, at) - float(want[at])) < 1e-8


def test_bits_are_the_row_samples(evt):
    """The generator is the one that row samples are drawn with: splitmix_mask's bytes."""
    key = plain.splitmix(77, 4)
    halves = evt.splitmix_mask(key, 8 * 3 * 2).view("<u2").reshape(3, 8)[:, :7].astype("int64")
    low = evt.splitmix_mask(~key & plain.M, 8 * 3 * 2).view("<u2").reshape(3, 8)[:, :7].astype("int64")
    assert torch.equal(plain.bits(3, 7, 77, 4), torch.from_numpy(halves << 16 | low))
