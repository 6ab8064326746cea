"""What a classifier's teacher may be given as: arrays, torch tensors of any type and device, at least one entry a row."""
import types

import numpy as np
import pytest
import torch


def test_no_entries_are_refused(evt):
    """A teacher of no entries is no way back to the labels."""
    handle = types.SimpleNamespace(N=4, K=3, _h=None)
    for ids in (np.zeros((4, 0), int), torch.zeros(4, 0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="n_top"):
            evt.Handle.set_teacher(handle, ids, np.zeros((4, 0)))
    with pytest.raises(ValueError, match="whole numbers"):
        evt.Handle.set_teacher(handle, torch.zeros(4, 1), torch.zeros(4, 1))


def test_tensors_are_read_as_arrays(evt):
    from_host = evt._lib.host_array
    for t in (torch.arange(6).reshape(3, 2), torch.ones(2, 2, dtype=torch.bfloat16) / 3, torch.ones(2, 2, dtype=torch.float16) / 3, torch.randn(4, 3, requires_grad=True)):
        assert np.array_equal(from_host(t), t.detach().double().numpy())
    assert from_host([[1, 2]]).tolist() == [[1, 2]] and from_host(np.float32(2)).dtype == np.float32


@pytest.mark.gpu
def test_gradients_from_tensors(evt):
    rng = np.random.default_rng(5)
    N, K = 500, 4
    h = evt.Handle(N, 3, 8, K, 3, "mlogloss")
    try:
        h.set_xbin(rng.integers(1, 9, size=(3, N), dtype=np.uint8))
        h.set_target(rng.integers(1, K + 1, size=N).astype(np.float32), None, np.zeros(K, np.float32), None)
        ids = torch.from_numpy(rng.integers(-1, K, (N, 2)))
        scores = torch.from_numpy(rng.standard_normal((N, 2))).to(torch.bfloat16)
        grads = []
        for i, s in ((ids.numpy(), scores.float().numpy()), (ids, scores), (ids.cuda(), scores.cuda()), (ids.int().cuda(), scores.cuda().float().requires_grad_())):
            h.set_teacher(i, s, 1.5)
            h.update_grads()
            grads.append(h.get_grads())
        assert all(np.array_equal(g, grads[0]) for g in grads[1:]) and grads[0][:, :K].any()
    finally:
        h.close()


@pytest.mark.gpu
def test_fit_to_tensors(evt):
    rng = np.random.default_rng(6)
    N, K = 1000, 3
    x, y = rng.standard_normal((N, 4)), rng.integers(0, K, N)
    ids, logits = torch.from_numpy(rng.integers(0, K, (N, 2))), torch.from_numpy(rng.standard_normal((N, 2))).float()
    config = evt.EvoTreeClassifier(nrounds=3, max_depth=3)
    want = evt.fit(config, x_train=x, y_train=y, teacher=evt.Teacher(ids.numpy(), logits.numpy()), verbosity=0)(x)
    assert np.array_equal(want, evt.fit(config, x_train=x, y_train=y, teacher=evt.Teacher(ids.cuda(), logits.cuda()), verbosity=0)(x))
