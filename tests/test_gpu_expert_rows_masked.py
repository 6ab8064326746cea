"""The gradient of the choice of experts in rows that a mask leaves nothing of: what its documentation makes NaN is NaN there too, and no other row is."""
import math

import pytest
import torch

import expert_rows_plain as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V,top", [(1, 1), (3, 2), (16, 4), (40, 6), (97, 64), (256, 8), (1000, 9), (2048, 2), (4096, 8)])
def test_no_score_and_no_number(evt, V, top, dtype, renormalize):
    rows, t = 11, plain.TYPES[dtype]
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(rows, V, generator=gen)
    x[:8] = -math.inf  # 0 to 7: no expert that can be chosen
    x = x.to(t)
    ids = torch.full((rows, top), -1, dtype=torch.int64)
    ids[8:] = torch.arange(top) % V
    w, dw = torch.rand(rows, top, generator=gen) / top, torch.randn(rows, top, generator=gen)
    ids[0, 0] = V  # no class
    ids[1, top - 1] = 2 ** 31 - 1
    ids[2, 0], w[2, 0] = V - 1, math.nan
    ids[3, top - 1], dw[3, top - 1] = 0, math.nan
    ids[4, 0] = V // 2  # a row without scores whose entry counts: no share of others is taken from it
    w[5], dw[5] = math.nan, math.nan  # nobody's
    ids[9, 0] = V
    dw[10, 0] = math.nan
    want, tol = plain.route_grad(x, ids, w, dw, renormalize, 0.5)
    assert want[[0, 1, 2, 3, 9, 10]].isnan().all() and want[[4, 5, 6, 7, 8]].isfinite().all()
    for kind in (torch.int32, torch.int64):
        got = evt.route_rows_grad(x.cuda(), ids.to(kind).cuda(), w.cuda(), dw.cuda(), renormalize=renormalize, temperature=0.5)
        plain.close("grad", got, want, tol)
