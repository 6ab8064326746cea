"""The losses over rows of class scores where a value is at the end of its range, is none, or stands in more than one sequence: against their formulas in
64 bits."""
import math

import pytest
import torch

import class_losses_plain as plain

pytestmark = pytest.mark.gpu


def _log1p_exp(h):
    """log(1 + exp(h)), infinite where h is."""
    return max(h, 0.0) + math.log1p(math.exp(-abs(h)))


@pytest.mark.parametrize("V,N", [(7, 24), (130, 24), (130, 3000), (33_000, 600)])  # slopes and losses in one launch, and in two
@pytest.mark.parametrize("soft", [0.0, 0.1])
def test_preference_of_impossible_answers(evt, V, N, soft):
    """An answer with a label that cannot be (a score of -inf): the chosen one, the rejected one, of a pair without weight."""
    gen = torch.Generator().manual_seed(V + N)
    x = torch.randn(N, V, generator=gen)
    lab = torch.randint(1, V, (N,), generator=gen)
    off = torch.tensor([0, 3, 6, 9, 12, 15, 18, 21, 24], dtype=torch.int32)  # pairs (0, 4), (1, 5), (2, 6), (3, 7)
    for row in (1, 16, 8):  # sequences 0, 5 and 2
        lab[row] = 0
        x[row, 0] = -math.inf
    ref = torch.randn(8, generator=gen) - 20
    w = torch.tensor([1.5, 0.5, 0.0, 2.0])
    beta, margin = 0.3, 0.2
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda(), beta=beta, label_smoothing=soft, margin=margin, weights=w.cuda())
    lp, lp_off, rows = plain.logp(x, lab, 1.0)
    want, tol = torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.float64)
    slope, slope_off = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    for p in range(4):
        c, r = slice(3 * p, 3 * p + 3), slice(12 + 3 * p, 15 + 3 * p)
        h = beta * (float(lp[c].sum()) - float(lp[r].sum()) - (float(ref[p]) - float(ref[4 + p]))) - margin
        wp, o = float(w[p]), beta * float(lp_off[c].sum() + lp_off[r].sum())
        if wp:
            want[p] = wp * ((1 - soft) * _log1p_exp(-h) + (soft * _log1p_exp(h) if soft else 0.0))
            tol[p] = wp * o  # a loss's derivative by h is under 1
            win, lose = (1.0, 0.0) if h == math.inf else (0.0, 1.0) if h == -math.inf else (1 / (1 + math.exp(-h)), 1 / (1 + math.exp(h)))
            dh = wp * beta * (soft * win - (1 - soft) * lose)
            slope[c], slope[r] = dh, -dh
            slope_off[c] = slope_off[r] = (wp * beta * 2 * win * lose * o if math.isfinite(h) else 0.0) + 2 * plain.U * abs(dh)
    assert want[0] == math.inf and (want[1] == math.inf) == (soft != 0) and want[2] == 0 and math.isfinite(want[3])
    plain.close("loss", loss, want, tol + plain.U * want.abs().nan_to_num(0, 0, 0) + 2.0 ** -149)
    assert seq[0] == -math.inf and seq[5] == -math.inf and seq[2] == -math.inf
    plain.close("grad", grad, *plain.label_grad(rows, lab, slope, 1.0, x.dtype, slope_off))
