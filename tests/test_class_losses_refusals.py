"""What the losses over rows of class scores refuse, in Python and at the C entry points: no GPU needed, nothing is queued."""
import ctypes as C

import pytest
import torch


def _good(N=4, V=10):
    x = torch.zeros(N, V)
    lab = torch.zeros(N, dtype=torch.int64)
    v = torch.zeros(N)
    ids = torch.zeros(N, 3, dtype=torch.int32)
    off = torch.tensor([0, 2, 4], dtype=torch.int32)
    return x, lab, v, ids, off


def _all(evt, x, **more):
    """Every operator on x, with arguments that fit it."""
    N = x.shape[0] if isinstance(x, torch.Tensor) and x.dim() else 4
    _, lab, v, ids, off = _good(N)
    st = torch.zeros(N, 2)
    return [lambda: evt.class_logp(x, lab, **more), lambda: evt.class_logp_grad(x, lab, st, v, **more),
            lambda: evt.distill_loss(x, ids, torch.zeros(N, 3), **more), lambda: evt.policy_loss(x, lab, v, v, **more),
            lambda: evt.preference_loss(x, lab, off, torch.zeros(2), **more)]


def test_scores_are_checked(evt):
    x, lab, v, ids, off = _good()
    for bad, error in ((x.double(), TypeError), (x.long(), TypeError), (x.numpy(), TypeError), (x[0], ValueError), (x[None], ValueError),
                       (torch.zeros(4, 0), ValueError), (torch.zeros(4, 1).expand(4, (1 << 30) + 1), ValueError), (torch.zeros(10, 4).t(), ValueError), (torch.zeros(4, 20)[:, ::2], ValueError)):
        for call in _all(evt, bad):
            with pytest.raises(error):
                call()
    for call in _all(evt, x):  # nothing else is wrong with these: the scores are on no GPU
        with pytest.raises(ValueError, match="on a GPU"):
            call()
    for T in (0.0, -1.0, 0.9e-4, 1.1e4, float("inf"), float("nan")):
        for call in _all(evt, x, temperature=T):
            with pytest.raises(ValueError, match="temperature"):
                call()


def test_labels_and_values_are_checked(evt):
    x, lab, v, ids, off = _good()
    st, two = torch.zeros(4, 2), torch.zeros(2)
    for bad in (lab[:3], lab.short(), lab.float(), lab[:, None], torch.zeros(8, dtype=torch.int64)[::2], [0, 0, 0, 0]):
        for call in (lambda: evt.class_logp(x, bad), lambda: evt.class_logp_grad(x, bad, st, v), lambda: evt.policy_loss(x, bad, v, v),
                     lambda: evt.preference_loss(x, bad, off, two)):
            with pytest.raises((ValueError, TypeError), match="labels|actions"):
                call()
    for bad in (v[:3], v.double(), v[:, None], torch.zeros(8)[::2], 1.0):
        for name, call in (("dlogp", lambda: evt.class_logp_grad(x, lab, st, bad)), ("old_logp", lambda: evt.policy_loss(x, lab, bad, v)),
                           ("advantages", lambda: evt.policy_loss(x, lab, v, bad)), ("ref_logp", lambda: evt.policy_loss(x, lab, v, v, bad)),
                           ("weights", lambda: evt.policy_loss(x, lab, v, v, weights=bad)),
                           ("weights", lambda: evt.distill_loss(x, ids, torch.zeros(4, 3), weights=bad)),
                           ("weights", lambda: evt.preference_loss(x, lab, off, two, weights=bad)),
                           ("ref_logp", lambda: evt.preference_loss(x, lab, off, bad))):
            with pytest.raises((ValueError, TypeError), match=name):
                call()
    with pytest.raises(ValueError, match="stats"):
        evt.class_logp_grad(x, lab, torch.zeros(2, 4), v)


def test_teachers_and_pairs_are_checked(evt):
    x, lab, v, ids, off = _good()
    top, two = torch.zeros(4, 3), torch.zeros(2)
    for bad in (ids[:3], ids.short(), ids[0], torch.zeros(4, 0, dtype=torch.int32), torch.zeros(4, 1025, dtype=torch.int32), None):
        with pytest.raises((ValueError, TypeError)):
            evt.distill_loss(x, bad, top)
    for bad in (top[:, :2], top.double(), torch.zeros(3, 4).t()):
        with pytest.raises((ValueError, TypeError), match="top_logits"):
            evt.distill_loss(x, ids, bad)
    for bad in (off.long(), off[:2], torch.zeros(4, dtype=torch.int32), off[None], torch.zeros(1, dtype=torch.int32), [0, 2, 4]):
        with pytest.raises((ValueError, TypeError), match="offsets"):
            evt.preference_loss(x, lab, bad, two)
    for name, value in (("beta", 0.0), ("beta", float("inf")), ("label_smoothing", 0.6), ("label_smoothing", -0.1), ("margin", float("nan")), ("margin", float("inf"))):
        with pytest.raises(ValueError, match=name):
            evt.preference_loss(x, lab, off, two, **{name: value})
    for name, value in (("clip_low", -0.1), ("clip_low", 1.1), ("clip_high", -0.1), ("clip_high", float("inf")), ("kl_coef", -1.0), ("kl_coef", float("nan"))):
        with pytest.raises(ValueError, match=name):
            evt.policy_loss(x, lab, v, v, v, **{name: value})
    with pytest.raises(ValueError, match="ref_logp"):
        evt.policy_loss(x, lab, v, v, kl_coef=0.1)


def test_out_is_checked(evt):
    x, lab, v, ids, off = _good()
    for bad in (x[:3], x.half(), torch.zeros(10, 4).t(), torch.zeros(10).expand(4, 10), 0):
        for call in _all(evt, x, out=bad)[1:]:
            with pytest.raises(ValueError, match="out"):
                call()
    with pytest.raises(ValueError, match="no gradient"):
        evt.policy_loss(x, lab, v, v, grad=False, out=x)


def test_c_entry_points_refuse(evt):
    """Null pointers, sizes, types, strides and overlaps, before any pointer is followed."""
    L, S, E = evt._lib.load(), evt._lib.EvtScores, evt._lib
    p, q = 0x10000, 0x90000  # never followed

    def scores(x=p, xs=10, g=q, gs=10, n=4, v=10, dtype=0, t=1.0):
        return C.byref(S(x, xs, g, gs, n, v, dtype, t))

    def logp(s, lab=p, kind=5, out=p, st=p, flags=2):
        return L.evt_class_logp(None, s, lab, kind, out, st, flags)

    def grad(s, lab=p, kind=5, st=p, d=p, flags=2):
        return L.evt_class_logp_grad(None, s, lab, kind, st, d, flags)

    def distill(s, ids=p, kind=4, top=p, tt=0, n=3, w=None, loss=p, flags=2):
        return L.evt_distill_loss(None, s, ids, kind, top, tt, n, w, loss, flags)

    def policy(s, lab=p, kind=5, old=p, adv=p, ref=None, w=None, lo=0.2, hi=0.2, kl=0.0, loss=p, lp=p, flags=2):
        return L.evt_policy_loss(None, s, lab, kind, old, adv, ref, w, lo, hi, kl, loss, lp, flags)

    def pref(s, lab=p, kind=5, off=p, n=1, ref=p, w=None, beta=0.1, soft=0.0, margin=0.0, avg=0, loss=p, seq=p, work=p, flags=2):
        return L.evt_preference_loss(None, s, lab, kind, off, n, ref, w, beta, soft, margin, avg, loss, seq, work, flags)

    every = (logp, grad, distill, policy, pref)
    wrong = [None, scores(x=None), scores(xs=-1), scores(gs=9), scores(n=-1), scores(n=1 << 31), scores(v=0), scores(v=(1 << 30) + 1, gs=1 << 31), scores(v=-5), scores(dtype=1), scores(dtype=9),
             scores(t=0.0), scores(t=9e-5), scores(t=11000.0), scores(t=float("nan")), scores(t=float("inf")), scores(x=p + 1), scores(g=q + 2), scores(g=p + 4), scores(g=p, gs=12), scores(g=p + 40),
             scores(g=p - 4)]
    for call in every:
        for s in wrong:
            assert call(s) == E.EVT_ERR_ARG and L.evt_last_error()
        assert call(scores(), flags=1) == E.EVT_ERR_ARG
    for call in every[:-1]:  # no rows, nothing to do (a pair of empty sequences has a loss)
        assert call(scores(n=0, x=None, g=None)) == E.EVT_OK
    for call in (logp, grad, policy, pref):
        assert call(scores(), lab=None) == E.EVT_ERR_ARG and call(scores(), kind=6) == E.EVT_ERR_ARG
    assert grad(scores(g=None)) == E.EVT_ERR_ARG
    for call, names in ((logp, ("out", "st")), (grad, ("st", "d")), (distill, ("ids", "top", "loss")), (policy, ("old", "adv", "loss", "lp")),
                        (pref, ("off", "ref", "loss", "seq", "work"))):
        for name in names:
            assert call(scores(), **{name: None}) == E.EVT_ERR_ARG, name
    for more in (dict(kind=0), dict(tt=1), dict(n=0), dict(n=1025)):
        assert distill(scores(), **more) == E.EVT_ERR_ARG
    for more in (dict(lo=-0.1), dict(lo=1.5), dict(hi=-1.0), dict(hi=float("nan")), dict(kl=-1.0), dict(kl=float("inf")), dict(kl=0.1)):
        assert policy(scores(), **more) == E.EVT_ERR_ARG
    for more in (dict(n=0), dict(n=1 << 22), dict(beta=0.0), dict(beta=float("inf")), dict(soft=0.7), dict(margin=float("inf")), dict(avg=2)):
        assert pref(scores(), **more) == E.EVT_ERR_ARG


def test_a_teacher_needs_a_classifier(evt):
    import numpy as np
    with pytest.raises(ValueError, match="mlogloss"):
        evt.init(evt.EvoTreeRegressor(), np.zeros((4, 1)), np.zeros(4), teacher=evt.Teacher(np.zeros((4, 1), int), np.zeros((4, 1))))
    assert evt._lib.load().evt_set_teacher(None, None, None, 0, 1.0) == evt._lib.EVT_ERR_ARG
