"""The losses over rows of class scores where a value is at the end of its range, is none, or stands in more than one sequence: against their formulas in
64 bits."""
import ctypes as C
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


def _pair_slopes(x, lab, off, ref, beta):
    """(slope, what it may be off by) that each sequence's pair gives its rows: NaN for both of a pair one of which is no sequence."""
    lp, lp_off, rows = plain.logp(x, lab, 1.0)
    half = (len(off) - 1) // 2
    ok = [0 <= a <= b <= len(lab) and a >= off[0] and b <= off[-1] for a, b in zip(off, off[1:])]
    slopes, offs, seen = [0.0] * (2 * half), [0.0] * (2 * half), ok
    for p in range(half):
        c, r = slice(off[p], off[p + 1]), slice(off[half + p], off[half + p + 1])
        if not (ok[p] and ok[half + p]):
            slopes[p] = slopes[half + p] = math.nan
            continue
        h = beta * (float(lp[c].sum() - lp[r].sum()) - (float(ref[p]) - float(ref[half + p])))
        win, lose = 1 / (1 + math.exp(-h)), 1 / (1 + math.exp(h))
        slopes[p], slopes[half + p] = -beta * lose, beta * lose
        offs[p] = offs[half + p] = beta * 2 * win * lose * beta * float(lp_off[c].sum() + lp_off[r].sum()) + 2 * plain.U * beta * lose
    return slopes, offs, seen, rows


@pytest.mark.parametrize("V,N", [(130, 24), (130, 3000), (33_000, 600)])  # slopes and losses in one launch, and in two
def test_preference_gradient_where_offsets_descend(evt, V, N):
    """Rows of a sequence that is none take the gradient of another that has them, whatever the form; rows of no other take none."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(N, V, generator=gen)
    lab = torch.randint(0, V, (N,), generator=gen)
    for off in ([0, 20, 2, 4, 6, 8, 10],  # sequence 0 ends behind the last, 1 descends; pairs (0, 3), (1, 4), (2, 5)
                [6, 9, 0, 3, 12],  # sequence 1 descends, 2 begins in front of the first
                [4, 7, 3, 12, 9, 12, 20]):  # 1 descends, 2 begins in front, 3 descends
        ref = torch.randn(len(off) - 1, generator=gen) - 20
        slopes, offs, ok, rows = _pair_slopes(x, lab, off, ref, 0.1)
        slope, slope_off = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
        owned = torch.zeros(N, dtype=torch.int32)
        for k, (a, b) in enumerate(zip(off, off[1:])):
            if ok[k]:
                slope[a:b], slope_off[a:b] = slopes[k], offs[k]
                owned[a:b] += 1
        assert owned.max() == 1
        loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), torch.tensor(off, dtype=torch.int32).cuda(), ref.cuda())
        plain.close("grad", grad, *plain.label_grad(rows, lab, slope, 1.0, x.dtype, slope_off))


@pytest.mark.parametrize("V,N", [(130, 24), (130, 3000), (33_000, 600)])
def test_preference_rows_of_two_sequences(evt, V, N):
    """Two sequences that both have a row (the offsets descend between them): one of their gradients, the same one in every call and in every form."""
    gen = torch.Generator().manual_seed(V + 1)
    x = torch.randn(N, V, generator=gen)
    lab = torch.randint(0, V, (N,), generator=gen)
    off = [0, 5, 3, 8, 10, 12, 14, 16, 18]  # 1 descends; 0 and 2 share rows 3 and 4; pairs (0, 4), (1, 5), (2, 6), (3, 7)
    ref = torch.randn(8, generator=gen) - 20
    ref[0] -= 40  # the slope of pair 2 is the larger by far
    slopes, offs, ok, rows = _pair_slopes(x, lab, off, ref, 0.1)
    assert abs(slopes[2]) > 1.2 * abs(slopes[0])
    args = x.cuda(), lab.cuda(), torch.tensor(off, dtype=torch.int32).cuda(), ref.cuda()
    loss, seq, grad = evt.preference_loss(*args)
    slope, slope_off = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    for k in (0, 3, 4, 5, 6, 7, 2):  # the larger slope's last
        slope[off[k]:off[k + 1]], slope_off[off[k]:off[k + 1]] = slopes[k], offs[k]
    plain.close("grad", grad, *plain.label_grad(rows, lab, slope, 1.0, x.dtype, slope_off))
    for _ in range(20):
        for a, b in zip(evt.preference_loss(*args), (loss, seq, grad)):
            assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))


@pytest.mark.parametrize("V,N,pairs,dtype", [(2100, 500, 300, "f32"), (2100, 1000, 1000, "bf16"), (16, 9000, 5000, "f32")])  # one launch; one launch; two, many pairs
def test_preference_many_pairs(evt, V, N, pairs, dtype):
    """More sequences than a wavefront looks at: each row's gradient is its own pair's; of two sequences that descending offsets give a row one's, whichever place they have."""
    gen = torch.Generator().manual_seed(pairs)
    x = torch.randn(N, V, generator=gen).to(plain.TYPES[dtype])
    lab = torch.randint(0, V, (N,), generator=gen)
    ref = torch.randn(2 * pairs, generator=gen)
    off = torch.randint(0, N + 1, (2 * pairs + 1,), generator=gen).sort().values.to(torch.int32)
    want = plain.preference(x, lab, off, ref, 0.1, 0.0, 0.0, False, 1.0, None)
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda())
    plain.close("loss", loss, *want[0])
    plain.close("grad", grad, *want[2])
    # sequences k and m > k + 1 (the one between descends) both have rows 40 to 59, and no other has
    for k, m in ((3, 70), (10, 12), (100, pairs + 200), (pairs - 1, 2 * pairs - 2)):
        bounds = [0] * (k + 1) + [60] * (m - k - 1) + [40] + [100] * (2 * pairs - m)
        lab[40:60] = 1
        slopes, offs, ok, rows = _pair_slopes(x, lab, bounds, ref, 0.1)
        assert len(bounds) == 2 * pairs + 1 and ok[k] and ok[m] and not ok[m - 1]
        slope, slope_off = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
        def bits(s):  # of a slope's float, as an unsigned number
            return int(torch.tensor([s], dtype=torch.float32).view(torch.int32)) & 0xFFFFFFFF
        for j in sorted((k, m), key=lambda j: bits(slopes[j])):
            slope[bounds[j]:bounds[j + 1]], slope_off[bounds[j]:bounds[j + 1]] = slopes[j], offs[j]
        loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), torch.tensor(bounds, dtype=torch.int32).cuda(), ref.cuda())
        plain.close("grad", grad, *plain.label_grad(rows, lab, slope, 1.0, x.dtype, slope_off))


@pytest.mark.parametrize("V,N", [(130, 24), (130, 3000)])
def test_preference_rows_shared_with_a_pair_without_slope(evt, V, N):
    """A row takes the gradient of the sequence whose pair has one, not that of a pair of weight 0, on whichever side."""
    gen = torch.Generator().manual_seed(V + 2)
    x = torch.randn(N, V, generator=gen)
    lab = torch.randint(0, V, (N,), generator=gen)
    off = [0, 2, 4, 6, 8, 14, 11, 18, 20]  # pairs (0, 4), (1, 5), (2, 6), (3, 7); 5 descends, 4 and 6 share rows 11 to 13
    ref = torch.randn(8, generator=gen) - 20
    for without in (0, 2):
        w = torch.ones(4)
        w[without] = 0.0
        loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), torch.tensor(off, dtype=torch.int32).cuda(), ref.cuda(), weights=w.cuda())
        slopes, offs, ok, rows = _pair_slopes(x, lab, off, ref, 0.1)
        slope, slope_off = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
        for k in range(8):
            if ok[k] and k % 4 != without:
                slope[off[k]:off[k + 1]], slope_off[off[k]:off[k + 1]] = slopes[k], offs[k]
        plain.close("grad", grad, *plain.label_grad(rows, lab, slope, 1.0, x.dtype, slope_off))


@pytest.mark.parametrize("V,N", [(3, 9), (7, 9), (100, 9), (1500, 300), (3001, 300), (50_021, 9)])  # every form
@pytest.mark.parametrize("dtype", list(plain.TYPES))
def test_teacher_scores_that_are_no_numbers(evt, V, N, dtype):
    """A NaN or +inf among the teacher's scores of a row that counts: its loss is NaN and all of its gradient; the other rows are as they were."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(N, V, generator=gen).to(plain.TYPES[dtype])
    ids = torch.stack([torch.randperm(V, generator=gen)[:3] for _ in range(N)])
    top = torch.randn(N, 3, generator=gen)
    want = plain.distill(x, ids, top, 1.0, None)
    top[2, 1], top[5, 0] = math.nan, math.inf
    for k in (2, 5):
        want[0][0][k] = want[1][0][k] = math.nan
    loss, grad = evt.distill_loss(x.cuda(), ids.cuda(), top.cuda())
    plain.close("loss", loss, *want[0])
    plain.close("grad", grad, *want[1])


@pytest.mark.parametrize("V", [3, 7, 40, 700, 9001, 140_001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_policies_far_apart(evt, V, dtype):
    """exp(logp - old) and exp(ref - logp) beyond float's range, with advantages, weights and a kl_coef that bring the loss back into it: the loss
    and the gradient are finite, and 0 at a class that cannot be."""
    gen = torch.Generator().manual_seed(V)
    gaps = torch.tensor([90.0, 120.0, 170.0, -95.0, -120.0, 0.1, 80.5, 88.9])
    adv = torch.tensor([-1e-3, -1e-10, -1e-25, 1e20, 1e30, 1.0, -1e-4, -0.1])
    w = torch.tensor([1.0, 1e-7, 1e-30, 1.0, 0.5, 1.0, 1.0, 1.0])
    N = len(gaps)
    x = torch.randn(N, V, generator=gen)
    x[:, 1] = -math.inf
    x = x.to(plain.TYPES[dtype])
    lab = torch.randint(0, V, (N,), generator=gen)
    lab[lab == 1] = 2
    lp = plain.logp(x, lab, 1.0)[0]
    old = (lp - gaps).float()
    loss, logp, grad = evt.policy_loss(x.cuda(), lab.cuda(), old.cuda(), adv.cuda(), weights=w.cuda())
    want = plain.policy(x, lab, old, adv, None, 0.2, 0.2, 0.0, 1.0, w)
    assert torch.isfinite(want[0][0]).all() and (want[0][0] != 0).all() and not want[2][0][:, 1].any()
    plain.close("loss", loss, *want[0])
    plain.close("grad", grad, *want[2])
    # the KL term alone: 0.05 exp(90) is 6e37
    ref = (lp + torch.tensor([90.0, 88.8, 100.0, 150.0, -90.0, -300.0, 81.0, 0.2])).float()
    w = torch.tensor([1.0, 1.0, 1e-6, 1e-30, 1.0, 1.0, 1.0, 1.0])
    none = torch.zeros(N)
    loss, logp, grad = evt.policy_loss(x.cuda(), lab.cuda(), old.cuda(), none.cuda(), ref.cuda(), kl_coef=0.05, weights=w.cuda())
    want = plain.policy(x, lab, old, none, ref, 0.2, 0.2, 0.05, 1.0, w)
    assert torch.isfinite(want[0][0]).all() and torch.isfinite(want[2][0]).all()
    plain.close("kl loss", loss, *want[0])
    plain.close("kl grad", grad, *want[2])


@pytest.mark.parametrize("V", [3, 40, 9001])
def test_advantage_that_is_no_number(evt, V):
    """Its row's loss and gradient are NaN on either side of the bounds and between them; no other row's are."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(6, V, generator=gen)
    lab = torch.randint(0, V, (6,), generator=gen)
    old = (plain.logp(x, lab, 1.0)[0] - torch.tensor([-1.0, 0.0, 1.0, -1.0, 0.0, 1.0])).float()
    adv = torch.tensor([math.nan, math.nan, math.nan, 1.0, 1.0, 1.0])
    loss, logp, grad = evt.policy_loss(x.cuda(), lab.cuda(), old.cuda(), adv.cuda())
    assert torch.isnan(loss).tolist() == [True] * 3 + [False] * 3 and not torch.isnan(logp).any()
    assert torch.isnan(grad[:3]).all() and torch.isfinite(grad[3:]).all()


def test_out_counts_as_a_change(evt):
    """A gradient written over a tensor that a recorded operation kept: its backward pass says so and does not compute with the gradient."""
    N, V = 12, 50
    lab = torch.randint(0, V, (N,)).cuda()
    v = torch.randn(N).cuda()
    off = torch.tensor([0, 5, 12], dtype=torch.int32).cuda()
    stats = torch.ones(N, 2).cuda()
    leaf = torch.randn(N, V).cuda().requires_grad_()
    for call in (lambda y: evt.class_logp_grad(y, lab, stats, v, out=y), lambda y: evt.distill_loss(y, lab[:, None], v[:, None], out=y),
                 lambda y: evt.policy_loss(y, lab, v, v, out=y), lambda y: evt.preference_loss(y, lab, off, v[:2].contiguous(), out=y)):
        y = leaf.exp()
        before = y._version
        call(y)
        assert y._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
        box = torch.zeros(N, V + 3).cuda()
        before = box._version
        call_out = box[:, 1:V + 1]
        call_out.copy_(leaf.detach())
        assert box._version == before + 1
        call(call_out)
        assert box._version == before + 2
    with torch.inference_mode():  # tensors made here have no such count
        z = leaf.detach() * 2.0
        assert evt.policy_loss(z, lab, v, v, out=z)[2] is z
    z = evt.policy_loss(z, lab, v, v, out=z)[2]


def test_results_are_not_recorded(evt):
    """Scores that require a gradient: no result does, and the returned gradient goes on by hand."""
    N, V = 12, 50
    leaf = torch.randn(N, V).cuda().requires_grad_()
    lab, v = torch.randint(0, V, (N,)).cuda(), torch.randn(N).cuda()
    logits = leaf * 2.0
    loss, logp, grad = evt.policy_loss(logits, lab, v - 4, v)
    logits.backward(grad)
    assert not loss.requires_grad and not logp.requires_grad and not grad.requires_grad and torch.equal(leaf.grad, grad * 2.0)
    assert not any(t.requires_grad for t in evt.class_logp(logits, lab))


def test_host_memory_is_refused(evt):
    """The C entry points ask where a pointer lies unless the caller vouches for it: pinned host memory is not device memory."""
    L, E = evt._lib.load(), evt._lib
    x, lab = torch.zeros(4, 10).cuda(), torch.zeros(4, dtype=torch.int64).cuda()
    out = torch.zeros(4, 2).cuda()
    host = [torch.zeros(4, 10).pin_memory(), torch.zeros(4, dtype=torch.int64).pin_memory(), torch.zeros(4, 2).pin_memory()]

    def call(x, lab, out):
        s = E.EvtScores(x.data_ptr(), 10, None, 0, 4, 10, 0, 1.0)
        return L.evt_class_logp(None, C.byref(s), lab.data_ptr(), 5, out.data_ptr(), stats.data_ptr(), 0)

    stats = torch.zeros(4, 2).cuda()
    torch.cuda.synchronize()
    assert call(x, lab, out) == E.EVT_OK
    torch.cuda.synchronize()
    for args in ((host[0], lab, out), (x, host[1], out), (x, lab, host[2])):
        assert call(*args) == E.EVT_ERR_ARG and b"device memory" in L.evt_last_error()
    torch.cuda.synchronize()
