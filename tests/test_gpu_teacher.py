"""A classifier fitted to a teacher (evt_set_teacher): its gradients are distill_loss's on the handle's predictions, bit for bit, and the formula's in 64
bits; they follow the predictions through the trees, and labels come back when the teacher goes."""
import numpy as np
import pytest
import torch

import class_losses_plain as plain

pytestmark = pytest.mark.gpu


def _handle(evt, N, K, weights, rng, F=6, B=16, D=4):
    x_bin = rng.integers(1, B + 1, size=(F, N), dtype=np.uint8)
    y = rng.integers(1, K + 1, size=N).astype(np.float32)
    h = evt.Handle(N, F, B, K, D, "mlogloss")
    h.set_xbin(x_bin)
    mu = rng.standard_normal(K).astype(np.float32)
    h.set_target(y, weights, mu - mu.max(), rng.standard_normal((N, K)).astype(np.float32))
    return h


def _teacher(rng, N, K, n_top):
    ids = np.stack([rng.permutation(K)[:n_top] for _ in range(N)]) if n_top <= K else rng.integers(0, K, size=(N, n_top))
    ids[rng.random((N, n_top)) < 0.2] = -1
    ids[1] = -1
    return ids, (rng.standard_normal((N, n_top)) * 2).astype(np.float32)


def _check(h, ids, scores, T, weights):
    K = h.K
    pred, grad = h.get_pred(), h.get_grads()
    x = torch.from_numpy(pred)
    w = None if weights is None else torch.from_numpy(weights)
    (_, _), (want, tol) = plain.distill(x, torch.from_numpy(ids), torch.from_numpy(scores), T, w)
    plain.close("gradient", torch.from_numpy(grad[:, :K].copy()), want, tol)
    rows = plain.Rows(x, T)
    ww = torch.ones(h.N, dtype=torch.float64) if w is None else w.double()
    # q (1 - q) w: off by q's own share twice, and the roundings of expf (2 U), the quotient and the products
    plain.close("curvature", torch.from_numpy(grad[:, K:2 * K].copy()), ww[:, None] * rows.q * (1 - rows.q),
                ww[:, None] * rows.q * (2 * rows.off + 16 * plain.U) + 2.0 ** -126)
    assert np.array_equal(grad[:, 2 * K], np.ones(h.N, np.float32) if weights is None else weights)
    return pred, grad


@pytest.mark.parametrize("K,n_top", [(2, 1), (3, 3), (5, 2), (7, 3), (8, 8), (16, 5), (16, 40), (4, 1024)])
def test_gradients(evt, K, n_top):
    rng = np.random.default_rng(K * 100 + n_top)
    N = 3001 if n_top < 100 else 70
    T = [1.0, 1.5][K % 2]
    weights = (rng.random(N) + 0.5).astype(np.float32) if K % 3 else None
    h = _handle(evt, N, K, weights, rng)
    try:
        ids, scores = _teacher(rng, N, K, n_top)
        h.update_grads()
        labels = h.get_grads()
        h.set_teacher(ids, scores, T)
        h.update_grads()
        pred, grad = _check(h, ids, scores, T, weights)
        loss, same = evt.distill_loss(torch.from_numpy(pred).cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(scores).cuda(), T,
                                      weights=None if weights is None else torch.from_numpy(weights).cuda())
        assert np.array_equal(same.cpu().numpy(), grad[:, :K])
        h.set_teacher(None, None)
        h.update_grads()
        assert np.array_equal(h.get_grads(), labels)
    finally:
        h.close()


@pytest.mark.parametrize("ahead", [0, 1])
def test_gradients_follow_the_trees(evt, ahead):
    rng = np.random.default_rng(4)
    N, K, T = 20_000, 6, 2.0
    h = _handle(evt, N, K, None, rng)
    try:
        ids, scores = _teacher(rng, N, K, 3)
        h.set_teacher(ids, scores, T)
        h.set_option("grads_ahead", ahead)
        js = np.arange(1, 7, dtype=np.uint32)
        h.update_grads()
        before = h.get_pred()
        for _ in range(3):
            h.grow_tree(js, evt.make_params(eta=0.3))
            h.update_grads()
            after, _ = _check(h, ids, scores, T, None)
            assert not np.array_equal(before, after)
            before = after
    finally:
        h.close()


def test_fit(evt):
    rng = np.random.default_rng(9)
    N, K = 4000, 4
    x = rng.standard_normal((N, 5))
    y = rng.integers(0, K, N)
    ids, scores = _teacher(rng, N, K, 2)
    config = evt.EvoTreeClassifier(nrounds=6, max_depth=4, eta=0.2)
    m = evt.fit(config, x_train=x, y_train=y, teacher=evt.Teacher(ids, scores, 1.5), x_eval=x[:500], y_eval=y[:500], verbosity=0)
    p = m(x)
    assert p.shape == (N, K) and np.isfinite(p).all() and len(m.trees) == 7 and len(m.info["logger"]["metrics"]) == 7
    other = evt.fit(config, x_train=x, y_train=y, verbosity=0)
    assert not np.array_equal(other(x), p)
    # the same through a table, and rounds added to a kept handle
    table = {"c%d" % j: x[:, j] for j in range(5)}
    m2, cache = evt.fit(evt.EvoTreeClassifier(nrounds=3, max_depth=4, eta=0.2), dict(table, y=y), target_name="y", teacher=evt.Teacher(ids, scores, 1.5),
                        return_cache=True, verbosity=0)
    m2, cache = evt.update(config, m2, cache)
    assert len(m2.trees) == 7
    cache.handle.close()


def test_refusals(evt):
    rng = np.random.default_rng(3)
    N, K = 50, 3
    h = _handle(evt, N, K, None, rng)
    try:
        ids, scores = _teacher(rng, N, K, 2)
        h.set_teacher(ids, scores)
        h.update_grads()
        want = h.get_grads()
        for bad in ((ids[:-1], scores[:-1]), (ids, scores[:, :1]), (ids.astype(float), scores), (ids[0], scores[0]), (np.full_like(ids, K), scores)):
            with pytest.raises(ValueError):
                h.set_teacher(*bad)
        for s in (np.nan, np.inf):
            worse = np.array(scores)
            worse[7] = s
            good = np.array(ids)
            good[7] = 1
            with pytest.raises(evt.EvtError):
                h.set_teacher(good, worse)
        for T in (0.0, -1.0, float("nan"), float("inf")):
            with pytest.raises(evt.EvtError):
                h.set_teacher(ids, scores, T)
        with pytest.raises(evt.EvtError):
            h.set_teacher(np.zeros((N, 1025), int), np.zeros((N, 1025)))
        L = evt._lib.load()
        flat = np.full((N, 2), K, np.int32)  # past the classes, by the C entry point
        assert L.evt_set_teacher(h._h, evt._lib.ptr(flat), evt._lib.ptr(scores), 2, 1.0) == evt._lib.EVT_ERR_ARG
        assert L.evt_set_teacher(h._h, None, None, 2, 1.0) == evt._lib.EVT_ERR_ARG
        assert L.evt_set_teacher(h._h, None, None, -1, 1.0) == evt._lib.EVT_ERR_ARG
        h.update_grads()  # the teacher there was stays
        assert np.array_equal(h.get_grads(), want)
    finally:
        h.close()
    mse = evt.Handle(10, 2, 8, 1, 3, "mse")
    try:
        with pytest.raises(evt.EvtError, match="mlogloss"):
            mse.set_teacher(np.zeros((10, 1), int), np.zeros((10, 1)))
    finally:
        mse.close()


def test_unsigned_ids(evt):
    rng = np.random.default_rng(5)
    N, K = 60, 4
    h = _handle(evt, N, K, None, rng)
    try:
        ids, scores = rng.integers(0, K, (N, 2)), rng.standard_normal((N, 2)).astype(np.float32)
        grads = []
        for kind in (np.int64, np.uint8, np.uint32, np.uint64):
            h.set_teacher(ids.astype(kind), scores)
            h.update_grads()
            grads.append(h.get_grads())
        assert all(np.array_equal(g, grads[0]) for g in grads[1:])
    finally:
        h.close()


def test_update_with_another_teacher(evt):
    rng = np.random.default_rng(11)
    N, K = 3000, 3
    x, y = rng.standard_normal((N, 4)), rng.integers(0, K, N)
    first, second = evt.Teacher(*_teacher(rng, N, K, 2)), evt.Teacher(*_teacher(rng, N, K, 2), 2.0)
    kw = dict(max_depth=3, eta=0.3)

    def grown(*teachers):
        m, cache = evt.fit(evt.EvoTreeClassifier(nrounds=2, **kw), x_train=x, y_train=y, teacher=first, return_cache=True, verbosity=0)
        m, cache = evt.update(evt.EvoTreeClassifier(nrounds=4, **kw), m, cache, *teachers)
        p = m(x)
        cache.handle.close()
        return p

    kept = grown()
    assert np.array_equal(kept, evt.fit(evt.EvoTreeClassifier(nrounds=4, **kw), x_train=x, y_train=y, teacher=first, verbosity=0)(x))
    assert np.array_equal(kept, grown(None, None, None, first))
    assert not np.array_equal(kept, grown(None, None, None, second))
    m, cache = evt.fit(evt.EvoTreeRegressor(nrounds=1), x_train=x, y_train=x[:, 0], return_cache=True, verbosity=0)
    with pytest.raises(ValueError, match="mlogloss"):
        evt.update(evt.EvoTreeRegressor(nrounds=2), m, cache, teacher=first)
    cache.handle.close()
