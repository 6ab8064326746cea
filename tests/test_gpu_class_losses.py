"""The losses over rows of class scores (class_logp, distill_loss, policy_loss, preference_loss and their gradients) against their formulas in 64
bits: every type, numbers of classes from one to many, odd ones, rows that lie anywhere, masks that leave a row nothing, values that are none."""
import math

import pytest
import torch

import class_losses_plain as plain

pytestmark = pytest.mark.gpu

CLASSES = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 33, 64, 100, 127, 128, 129, 255, 511, 513, 1000, 1024, 1025, 2047, 2049, 4097, 8191, 8200, 16385, 32768, 50021,
           65537, 70001, 131072, 170003]
WIDE = [3, 100, 1025, 50021]


def _scores(V, dtype, seed, N=13, spread=3.0, special=True):
    """(N, V) on the CPU.  Row 1 is masked but for one class, row 2 altogether, row 3 holds a NaN, row 4 a +inf, row 5 is large, row 6 half masked."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=gen) * spread
    if special:
        x[1, : V - 1] = -math.inf
        x[2] = -math.inf
        x[3, V // 2] = math.nan
        x[4, V - 1] = math.inf
        x[5] = x[5] * 100 + 1000
        x[6, : V // 2] = -math.inf
    return x.to(dtype), gen


def _labels(N, V, gen, wide=torch.int64):
    lab = torch.randint(0, V, (N,), generator=gen)
    lab[1] = V - 1
    lab[7] = -100
    lab[8] = -1
    lab[9] = V  # none of the classes
    return lab.to(wide)


def _placed(x, pad, shift):
    """x on the GPU with rows pad elements further apart and the first one shift elements behind an aligned address."""
    N, V = x.shape
    base = torch.full((N * (V + pad) + shift,), 7.0, dtype=x.dtype, device="cuda")
    view = base[shift:].as_strided((N, V), (V + pad, 1)) if shift else base.as_strided((N, V), (V + pad, 1))
    view.copy_(x)
    return view


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", CLASSES)
def test_class_logp(evt, V, dtype):
    x, gen = _scores(V, plain.TYPES[dtype], V)
    lab = _labels(13, V, gen)
    T = [1.0, 0.7, 2.0][V % 3]
    g = torch.randn(13, generator=gen)
    g[10] = 0.0
    want, tol, rows = plain.logp(x, lab, T)
    xg = _placed(x, V % 2, V % 5)
    lp, stats = evt.class_logp(xg, lab.cuda(), temperature=T)
    plain.close("logp", lp, want, tol)
    m = torch.where(lab < 0, 0.0, torch.where(rows.bad, stats[:, 0].cpu().double(), rows.m))
    s = torch.where(lab < 0, 0.0, torch.where(rows.bad, math.nan, rows.s))
    plain.close("max", stats[:, 0], m, torch.zeros(()))
    plain.close("sum", stats[:, 1], s, s.nan_to_num(0) * plain.chain(V))
    grad = evt.class_logp_grad(xg, lab.cuda(), stats, g.cuda(), temperature=T)
    plain.close("grad", grad, *plain.label_grad(rows, lab, g.double(), T, x.dtype))


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", CLASSES)
def test_policy_loss(evt, V, dtype):
    x, gen = _scores(V, plain.TYPES[dtype], V + 1)
    N = 13
    lab = _labels(N, V, gen, torch.int32)
    T = [1.0, 2.0, 0.7][V % 3]
    lp = plain.logp(x, lab, T)[0].nan_to_num(0, 0, -3)
    # ratios well inside and outside the bounds of 0.8 and 1.3, and equal policies
    old = (lp - torch.tensor([0.0, 0.1, -0.1, 0.5, -0.5, 0.0, 0.1, 0.2, 0.5, -0.5, 0.05, -0.6, 0.7])).float()
    adv = torch.tensor([1.0, -1.0, 0.5, 1.0, 1.0, 0.0, 2.0, 1.0, 1.0, 1.0, -0.3, -1.5, 1.5])
    ref = (lp + torch.randn(N, generator=gen) * 0.5).float()
    w = torch.rand(N, generator=gen) + 0.5
    w[10] = 0.0
    kl = 0.1 if V % 2 else 0.0
    loss, logp, grad = evt.policy_loss(_placed(x, 3, V % 3), lab.cuda(), old.cuda(), adv.cuda(), ref_logp=ref.cuda() if kl else None, clip_low=0.2,
                                       clip_high=0.3, kl_coef=kl, temperature=T, weights=w.cuda())
    want = plain.policy(x, lab, old, adv, ref, 0.2, 0.3, kl, T, w)
    plain.close("loss", loss, *want[0])
    plain.close("logp", logp, *want[1])
    plain.close("grad", grad, *want[2])


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", CLASSES)
def test_distill_loss(evt, V, dtype):
    x, gen = _scores(V, plain.TYPES[dtype], V + 2)
    N, k = 13, [1, 5, 64, 130][V % 4]
    ids = torch.randint(0, V, (N, k), generator=gen)  # many come twice
    ids[:, k // 2:][torch.rand(N, k - k // 2, generator=gen) < 0.3] = -1
    ids[1] = V - 1
    ids[7] = -1
    ids[9, k - 1] = V
    top = torch.randn(N, k, generator=gen) * 3
    top[8] = -math.inf
    top[11, 0] = -math.inf
    w = torch.rand(N, generator=gen) + 0.5
    w[10] = 0.0
    T = [1.0, 2.0, 0.7][V % 3]
    loss, grad = evt.distill_loss(_placed(x, V % 4, 1), ids.cuda().to([torch.int64, torch.int32][V % 2]), top.cuda(), temperature=T, weights=w.cuda())
    want = plain.distill(x, ids, top, T, w)
    plain.close("loss", loss, *want[0])
    plain.close("grad", grad, *want[1])


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", [2, 7, 16, 17, 100, 1025, 4097, 32768, 70001])
def test_preference_loss(evt, V, dtype, average):
    N, T = 41, [1.0, 0.7][V % 2]
    x, gen = _scores(V, plain.TYPES[dtype], V + 3, N)
    x[2:5] = torch.randn(3, V, generator=gen).to(x.dtype)
    lab = torch.randint(0, V, (N,), generator=gen)
    lab[5:9] = -100
    lab[x.float().gather(1, lab.clamp(min=0)[:, None])[:, 0] == -math.inf] = V - 1
    lab[20] = -1  # a sequence without a label, and one without a row
    off = torch.tensor([2, 9, 20, 21, 21, 30, 38], dtype=torch.int32)
    ref = torch.randn(6, generator=gen) * 2
    w = torch.tensor([1.0, 0.5, 2.0])
    lp = plain.logp(x, lab, T)[0]
    for k, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:])):  # near what the sequences have
        ref[k] += float(lp[a:b].sum()) / (max(1, int((lab[a:b] >= 0).sum())) if average else 1)
    args = dict(beta=0.3, label_smoothing=0.1 if V % 2 else 0.0, margin=0.2)
    loss, seq, grad = evt.preference_loss(_placed(x, 1, 1), lab.cuda(), off.cuda(), ref.cuda(), average=average, temperature=T, weights=w.cuda(), **args)
    want = plain.preference(x, lab, off, ref, args["beta"], args["label_smoothing"], args["margin"], average, T, w)
    plain.close("loss", loss, *want[0])
    plain.close("seq_logp", seq, *want[1])
    plain.close("grad", grad, *want[2])
    assert not grad[:2].any() and not grad[38:].any()


@pytest.mark.parametrize("V,N,dtype", [(5, 2600, "f32"), (7, 2500, "bf16"), (130, 2400, "f16"), (1300, 2300, "f32"), (4100, 2200, "bf16")])
def test_preference_many_rows(evt, V, N, dtype):
    """More rows than one launch finds the pairs of: the slopes come from a kernel of their own.  An odd number of pairs, sequences of no rows among them."""
    x, gen = _scores(V, plain.TYPES[dtype], V, N, special=False)
    lab = torch.randint(-1, V, (N,), generator=gen)
    cuts = torch.randint(3, N - 5, (9,), generator=gen).sort().values
    off = torch.cat([torch.tensor([3]), cuts[:4], cuts[3:4], cuts[4:], torch.tensor([N - 5])])[:11].to(torch.int32)
    lp = torch.cat([torch.zeros(1, dtype=torch.float64), plain.logp(x, lab, 1.0)[0].cumsum(0)])
    ref = (lp[off[1:].long()] - lp[off[:-1].long()] + torch.randn(10, generator=gen) * 3).float()
    w = torch.tensor([1.0, 0.0, 0.5, 2.0, 1.0])
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda(), beta=0.2, weights=w.cuda())
    want = plain.preference(x, lab, off, ref, 0.2, 0.0, 0.0, False, 1.0, w)
    plain.close("loss", loss, *want[0])
    plain.close("seq_logp", seq, *want[1])
    plain.close("grad", grad, *want[2])


def test_preference_bad_rows_and_offsets(evt):
    """A NaN score or a label past the classes spoils its own pair, offsets that do not ascend theirs; the others are as they are alone."""
    V, N = 130, 24
    x, gen = _scores(V, torch.float32, 5, N, special=False)
    lab = torch.randint(0, V, (N,), generator=gen)
    ref = torch.randn(8, generator=gen) - 20
    off = torch.tensor([0, 3, 6, 9, 12, 15, 18, 21, 24], dtype=torch.int32)
    x[4, 7] = math.nan  # pair 1
    lab[20] = V  # pair 2 (its rejected one)
    want = plain.preference(x, lab, off, ref, 0.1, 0.0, 0.0, False, 1.0, None)
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda())
    plain.close("loss", loss, *want[0])
    plain.close("seq_logp", seq, *want[1])
    plain.close("grad", grad, *want[2])
    assert torch.isnan(loss).tolist() == [False, True, True, False]
    off[4] = 40  # past the rows: sequences 3 and 4, pairs 3 and 0
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda())
    assert torch.isnan(loss).all() and torch.isnan(seq).tolist() == [True, True, False, True, True, False, True, True]
    off = torch.tensor([-3, 3, 6, 9, 12, 15, 18, 21, 24], dtype=torch.int32)
    x[4, 7], lab[20] = 0.0, 0
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda())
    assert torch.isnan(loss).tolist() == [True, False, False, False]
    want = plain.preference(x, lab, torch.tensor([0, 3, 6, 9, 12, 15, 18, 21, 24]), ref, 0.1, 0.0, 0.0, False, 1.0, None)
    plain.close("loss", loss[1:], want[0][0][1:], want[0][1][1:])
    plain.close("grad", grad[3:12], want[2][0][3:12], want[2][1][3:12])


@pytest.mark.parametrize("V,N", [(2, 100_003), (7, 60_013), (16, 4097), (54, 20_001), (300, 5003), (1999, 1201)])
@pytest.mark.parametrize("dtype", list(plain.TYPES))
def test_many_rows(evt, V, N, dtype):
    x, gen = _scores(V, plain.TYPES[dtype], V, N, special=False)
    lab = torch.randint(-1, V, (N,), generator=gen)
    want, tol_lp, rows = plain.logp(x, lab, 1.0)
    lp, stats = evt.class_logp(x.cuda(), lab.cuda())
    plain.close("logp", lp, want, tol_lp)
    d = torch.randn(N, generator=gen)
    grad = evt.class_logp_grad(x.cuda(), lab.cuda(), stats, d.cuda()).cpu().double()
    one = torch.zeros(N, V, dtype=torch.float64).scatter_(1, lab.clamp(min=0)[:, None], 1.0)
    due = torch.where(lab[:, None] < 0, 0.0, d.double()[:, None] * (one - rows.q))
    tol = d.abs().double()[:, None] * (rows.q * rows.off + 4 * plain.U * (one + rows.q))
    plain.close("grad", grad, due, tol + plain.half_step(x.dtype) * (due.abs() + tol) + plain.LEAST[x.dtype] * 5)
    adv = torch.randn(N, generator=gen)
    old = torch.where(lab < 0, 0.0, want).float()  # r = 1: between the bounds
    loss, lp2, grad = evt.policy_loss(x.cuda(), lab.cuda(), old.cuda(), adv.cuda())
    assert torch.equal(lp, lp2)
    plain.close("policy loss", loss, torch.where(lab < 0, 0.0, -adv.double()), adv.abs().double() * (1.1 * tol_lp + plain.U))


def _calls(evt, x, gen, out=None):
    """One call of each operator on x (on the GPU): their outputs, gradients last."""
    N, V = x.shape
    lab = torch.randint(-1, V, (N,), generator=gen).cuda()
    ids = torch.randint(-1, V, (N, 6), generator=gen, dtype=torch.int32).cuda()
    top = torch.randn(N, 6, generator=gen).cuda().to(torch.bfloat16)
    v = [torch.randn(N, generator=gen).cuda() for _ in range(4)]
    off = torch.tensor([1, N // 3, N // 2, N - 2, N - 1], dtype=torch.int32).cuda()

    def logp_grad():
        lp, st = evt.class_logp(x, lab)
        return lp, st, evt.class_logp_grad(x, lab, st, v[0], out=out() if out else None)

    return [logp_grad, lambda: evt.distill_loss(x, ids, top, 1.5, out=out() if out else None),
            lambda: evt.policy_loss(x, lab, v[0] - 5, v[1], v[2] - 5, kl_coef=0.1, weights=v[3].abs(), out=out() if out else None),
            lambda: evt.preference_loss(x, lab, off, v[0][:4].contiguous(), out=out() if out else None)]


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", [1, 5, 16, 40, 1000, 8191, 50021, 131072, 170003])
def test_in_place_strided_and_repeated(evt, V, dtype):
    """The gradient in the scores' own memory, between other values, and twice over: the same bits."""
    x, gen = _scores(V, plain.TYPES[dtype], V, 9)
    state = gen.get_state()
    xg = _placed(x, 2, 1)
    first = [[t.clone() for t in f()] for f in _calls(evt, xg, gen)]
    gen.set_state(state)
    again = [f() for f in _calls(evt, xg, gen)]
    for a, b in zip(first, again):
        for u, v in zip(a, b):
            assert torch.equal(u.nan_to_num(9.0), v.nan_to_num(9.0))
    gen.set_state(state)
    box = torch.full((9, V + 5), 3.0, dtype=x.dtype, device="cuda")
    for f, a in zip(_calls(evt, xg, gen, lambda: box[:, 2:V + 2]), first):
        assert torch.equal(f()[-1].nan_to_num(9.0), a[-1].nan_to_num(9.0))
        assert (box[:, :2] == 3).all() and (box[:, V + 2:] == 3).all()
    gen.set_state(state)
    target = _placed(x, 2, 1)
    for f, a in zip(_calls(evt, target, gen, lambda: target), first):
        target.copy_(x)
        got = f()
        assert got[-1].data_ptr() == target.data_ptr()
        for u, v in zip(got, a):
            assert torch.equal(u.nan_to_num(9.0), v.nan_to_num(9.0))


def test_rows_far_apart(evt):
    """Rows whose elements' numbers pass 32 bits, scores and gradient."""
    N, V, step = 20, 1000, 1 << 28
    x, gen = _scores(V, torch.bfloat16, 3, N, special=False)
    state = gen.get_state()
    want = [f() for f in _calls(evt, x.cuda(), gen)]
    far = torch.empty(step * (N - 1) + V, dtype=torch.bfloat16, device="cuda").as_strided((N, V), (step, 1))
    far.copy_(x)
    out = torch.empty(step * (N - 1) + V, dtype=torch.bfloat16, device="cuda").as_strided((N, V), (step, 1))
    gen.set_state(state)
    for f, a in zip(_calls(evt, far, gen, lambda: out), want):
        for u, v in zip(f(), a):
            assert torch.equal(u, v)


def test_one_row_for_all(evt):
    """Scores whose rows are one row (a stride of 0)."""
    x, gen = _scores(333, torch.float32, 4, 1, special=False)
    state = gen.get_state()
    want = [f() for f in _calls(evt, x.cuda().repeat(12, 1), gen)]
    gen.set_state(state)
    for f, a in zip(_calls(evt, x.cuda().expand(12, 333), gen), want):
        for u, v in zip(f(), a):
            assert torch.equal(u, v)


@pytest.mark.parametrize("N,V,dtype", [(17_000_100, 4200, torch.bfloat16), (68_000_000, 1100, torch.float16), (34_000_000, 700, torch.float32)])
def test_rows_of_several_launches(evt, N, V, dtype):
    """More rows than one launch has threads for; all of them one row in memory."""
    x, gen = _scores(V, dtype, 8, 1, special=False)
    lab = torch.full((N,), 3, dtype=torch.int32)
    lab[-1], lab[N // 2], lab[-2] = V - 1, -1, 0
    lp, stats = evt.class_logp(x.cuda().expand(N, V), lab.cuda())
    # other numbers of rows may take other forms, whose sums are in another order: held against 64 bits, and all the rows alike against each other
    want, tol, _ = plain.logp(x.expand(4, V), torch.tensor([3, V - 1, -1, 0]), 1.0)
    plain.close("logp", torch.stack([lp[0], lp[-1], lp[N // 2], lp[-2]]), want, tol)
    lp[-1] = lp[N // 2] = lp[-2] = lp[0].clone()
    assert (lp == lp[0]).all() and (stats[:, 1] == stats[0, 1]).sum() == N - 1


def test_extreme_scores_and_temperatures(evt):
    """Scores at the ends of their type - masks of its lowest value - and the least and greatest temperature."""
    for dtype in plain.TYPES.values():
        top = torch.finfo(dtype).max
        for T in (1e-4, 1.0, 1e4):
            for V in (5, 20, 600, 9000):
                x = torch.zeros(6, V, dtype=dtype)
                x[0] = -top  # every class as likely as the next
                x[1, 1:] = -top
                x[2] = top
                x[3, : V // 2] = -top
                x[4, 0], x[4, 1] = top, -top
                lab = torch.tensor([1, 0, V - 1, V - 1, 0, 2])
                want, tol, rows = plain.logp(x, lab, T)
                lp, stats = evt.class_logp(x.cuda(), lab.cuda(), T)
                plain.close("logp", lp, want, tol)
                d = torch.ones(6)
                plain.close("grad", evt.class_logp_grad(x.cuda(), lab.cuda(), stats, d.cuda(), T), *plain.label_grad(rows, lab, d.double(), T, dtype))


def test_no_rows_and_no_gradient(evt):
    x = torch.zeros(0, 50, device="cuda")
    lab = torch.zeros(0, dtype=torch.int64, device="cuda")
    v = torch.zeros(0, device="cuda")
    lp, st = evt.class_logp(x, lab)
    assert lp.shape == (0,) and st.shape == (0, 2) and evt.class_logp_grad(x, lab, st, v).shape == (0, 50)
    loss, grad = evt.distill_loss(x, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, device="cuda"))
    assert loss.shape == (0,) and grad.shape == (0, 50)
    assert evt.policy_loss(x, lab, v, v)[2].shape == (0, 50)
    loss, seq, grad = evt.preference_loss(x, lab, torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda"))
    assert abs(loss.item() - math.log(2)) < 1e-6 and not seq.any() and grad.shape == (0, 50)
    y, gen = _scores(77, torch.float32, 6, 30, special=False)
    y = y.cuda()
    lab = torch.randint(0, 77, (30,), generator=gen).cuda()
    v = torch.randn(30, generator=gen).cuda()
    ids = torch.randint(0, 77, (30, 4), generator=gen).cuda()
    off = torch.tensor([0, 10, 30], dtype=torch.int32, device="cuda")
    for with_grad, without in ((evt.distill_loss(y, ids, torch.ones(30, 4, device="cuda")), evt.distill_loss(y, ids, torch.ones(30, 4, device="cuda"), grad=False)),
                               (evt.policy_loss(y, lab, v, v), evt.policy_loss(y, lab, v, v, grad=False)),
                               (evt.preference_loss(y, lab, off, v[:2].contiguous()), evt.preference_loss(y, lab, off, v[:2].contiguous(), grad=False))):
        assert without[-1] is None
        for a, b in zip(with_grad[:-1], without[:-1]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n_top", [1, 2, 63, 64, 65, 200, 1024])
@pytest.mark.parametrize("kind", list(plain.TYPES))
def test_teachers_of_any_length(evt, n_top, kind):
    V, N = 1500, 6
    x, gen = _scores(V, torch.float32, n_top, N, special=False)
    ids = torch.randint(0, V, (N, n_top), generator=gen)
    ids[3] = 11  # all one class
    top = (torch.randn(N, n_top, generator=gen) * 2).to(plain.TYPES[kind])
    loss, grad = evt.distill_loss(x.cuda(), ids.cuda(), top.cuda(), temperature=1.3)
    want = plain.distill(x, ids, top, 1.3, None)
    plain.close("loss", loss, *want[0])
    plain.close("grad", grad, *want[1])


def test_gradients_against_differences(evt):
    """The gradients against central differences of the 64-bit losses: (f(x + h) - f(x - h)) / 2h is off by f''' h^2 / 6, third derivatives of
    these losses are below 40 here and h = 1e-4: 1e-7, and by the losses' own 64-bit rounding over h, 1e-11; the gradients, of at most about 1, by
    chain(9) = 6e-6."""
    V, N, h = 9, 6, 1e-4
    x, gen = _scores(V, torch.float32, 12, N, 1.0, special=False)
    lab = torch.randint(0, V, (N,), generator=gen)
    old = plain.logp(x, lab, 1.0)[0].float() - torch.tensor([0.0, 0.1, -0.1, 0.5, -0.5, 0.05])
    adv = torch.randn(N, generator=gen)
    ref = old + 0.3
    ids = torch.randint(0, V, (N, 3), generator=gen)
    top = torch.randn(N, 3, generator=gen)
    off = torch.tensor([0, 2, 3, 4, 6], dtype=torch.int32)
    seq_ref = torch.randn(4, generator=gen)
    T = 1.5

    def losses(z):
        return [plain.distill(z, ids, top, T, None)[0][0].sum(), plain.policy(z, lab, old, adv, ref, 0.2, 0.2, 0.1, 1.0, None)[0][0].sum(),
                plain.preference(z, lab, off, seq_ref, 0.5, 0.1, 0.1, False, T, None)[0][0].sum(), plain.logp(z, lab, T)[0].sum()]

    xg, labg = x.cuda(), lab.cuda()
    stats = evt.class_logp(xg, labg, T)[1]
    grads = [evt.distill_loss(xg, ids.cuda(), top.cuda(), T)[1],
             evt.policy_loss(xg, labg, old.cuda(), adv.cuda(), ref.cuda(), kl_coef=0.1)[2],
             evt.preference_loss(xg, labg, off.cuda(), seq_ref.cuda(), 0.5, 0.1, 0.1, temperature=T)[2],
             evt.class_logp_grad(xg, labg, stats, torch.ones(N, device="cuda"), T)]
    for i in range(N):
        for c in range(V):
            z = x.double().clone()
            z[i, c] += h
            up = losses(z)
            z[i, c] -= 2 * h
            down = losses(z)
            for name, g, a, b in zip(("distill", "policy", "preference", "logp"), grads, up, down):
                assert abs(float(g[i, c]) - float(a - b) / (2 * h)) < 1e-5, (name, i, c)


def test_streams_and_graphs(evt):
    """On another stream; recorded into two graphs that are replayed in turn with eager work between: every replay equals the eager result."""
    x, gen = _scores(5003, torch.bfloat16, 21, 40, special=False)
    xg = x.cuda()
    calls = _calls(evt, xg, gen)
    want = [[t.clone() for t in f()] for f in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        later = xg * 1.0  # made on that stream
        xg.record_stream(side)
        got = [f() for f in calls]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for u, v in zip(a, b):
            assert torch.equal(u, v)
    assert torch.equal(later, xg)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = [f() for f in calls]
        graphs.append((graph, outs))
    for turn in range(3):
        for graph, outs in graphs:
            for o in outs:
                for t in o:
                    t.fill_(5)
        torch.cuda.synchronize()
        graphs[0][0].replay()
        graphs[1][0].replay()
        eager = [f() for f in calls]
        torch.cuda.synchronize()
        for outs in (graphs[0][1], graphs[1][1], eager):
            for a, b in zip(outs, want):
                for u, v in zip(a, b):
                    assert torch.equal(u, v), turn
    xg.copy_(xg.flip(0))  # the graphs read what is there when they run
    for graph, _ in graphs:
        graph.replay()
    eager = [f() for f in calls]
    for graph, outs in graphs:
        for a, b in zip(outs, eager):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_preference_training_step(evt):
    """The run of a preference step: the reference model scores the answers, the policy's loss falls to log 2 where it is that model, its gradient
    is class_logp's with the pairs' slopes, and a policy step on the same rows agrees with both."""
    V, N = 777, 60
    x, gen = _scores(V, torch.float32, 31, N, special=False)
    lab = torch.randint(0, V, (N,), generator=gen)
    lab[:5] = -100
    off = torch.tensor([0, 14, 30, 41, 60], dtype=torch.int32)
    xg, labg, offg = x.cuda(), lab.cuda(), off.cuda()
    lp, stats = evt.class_logp(xg, labg)
    sums = torch.cat([torch.zeros(1, device="cuda", dtype=torch.float64), lp.double().cumsum(0)])[off.long().cuda()]
    ref = (sums[1:] - sums[:-1]).float()
    loss, seq, grad = evt.preference_loss(xg, labg, offg, ref, beta=0.1)
    # seq - ref: off by the roundings of two sums of some 130 to 32 bits, 2 * 2^-17; times beta / 2
    assert (loss - math.log(2)).abs().max() < 0.1 * 2.0 ** -16 + 2 * plain.U and (seq - ref).abs().max() <= 2.0 ** -16
    slope = torch.zeros(N, device="cuda")
    for k in range(4):
        slope[off[k]:off[k + 1]] = (-0.05, -0.05, 0.05, 0.05)[k]
    same = evt.class_logp_grad(xg, labg, stats, slope)
    # the slope itself is off by beta / 4 of the difference above, 0.1 / 4 * 0.1 * 2^-15
    assert (grad - same).abs().max() < 0.0025 * 2.0 ** -15 + 8 * plain.U * 0.05
    _, lp2, pg = evt.policy_loss(xg, labg, lp, -slope)
    assert torch.equal(lp, lp2) and (pg - same).abs().max() < 40 * plain.U * 0.05  # r = 1 but for the rounding of lp, of at most 32


@pytest.mark.parametrize("V,dtype", [(1100, "f32"), (2050, "bf16"), (2100, "f32"), (3001, "f16"), (4099, "bf16"), (4097, "f32"), (8193, "bf16"), (9000, "f32"), (16390, "f16"),
                                     (16385, "bf16"), (20000, "f32"), (32770, "bf16"), (33000, "f32"), (65537, "f16"), (66001, "f32"), (131075, "bf16"), (140001, "f16")])
def test_more_rows_than_units(evt, V, dtype):
    """The forms that many rows take, in blocks of every size, rows at odd addresses, some left out."""
    N = 263
    x, gen = _scores(V, plain.TYPES[dtype], V + 9, N)
    lab = _labels(N, V, gen)
    xg = _placed(x, V % 3, V % 2)
    want, tol, rows = plain.logp(x, lab, 1.0)
    lp, stats = evt.class_logp(xg, lab.cuda())
    plain.close("logp", lp, want, tol)
    adv = torch.randn(N, generator=gen)
    adv[20] = 0.0
    old = want.nan_to_num(0, 0, -3).float()  # r = 1 but for the roundings: between the bounds
    w = torch.rand(N, generator=gen) + 0.5
    w[30] = 0.0
    case = plain.policy(x, lab, old, adv, None, 0.2, 0.2, 0.0, 1.0, w)
    loss, lp2, grad = evt.policy_loss(xg, lab.cuda(), old.cuda(), adv.cuda(), weights=w.cuda())
    plain.close("policy loss", loss, *case[0])
    plain.close("policy grad", grad, *case[2])
    plain.close("logp grad", evt.class_logp_grad(xg, lab.cuda(), stats, adv.cuda()), *plain.label_grad(rows, lab, adv.double(), 1.0, x.dtype))
    ids = torch.randint(-1, V, (N, 7), generator=gen, dtype=torch.int32)
    ids[40, 2] = ids[40, 5] = 3
    top = torch.randn(N, 7, generator=gen) * 2
    case = plain.distill(x, ids, top, 1.0, w)
    loss, grad = evt.distill_loss(xg, ids.cuda(), top.cuda(), weights=w.cuda())
    plain.close("distill loss", loss, *case[0])
    plain.close("distill grad", grad, *case[1])
    plain.close("distill loss alone", evt.distill_loss(xg, ids.cuda(), top.cuda(), weights=w.cuda(), grad=False)[0], *case[0])
    target = _placed(x, V % 3, V % 2)  # in place
    assert torch.equal(evt.distill_loss(target, ids.cuda(), top.cuda(), weights=w.cuda(), out=target)[1].nan_to_num(9.0), grad.nan_to_num(9.0))


def test_rows_left_out_hold_anything(evt):
    """NaN and infinities in the rows, entries and values of what is left out reach nothing."""
    for V in (3, 40, 700, 9001):
        N = 12
        x, gen = _scores(V, torch.bfloat16, V, N, special=False)
        clean = x.clone()
        lab = torch.randint(0, V, (N,), generator=gen)
        lab[2:5] = -1
        x[2], x[3], x[4, 0] = math.nan, math.inf, math.nan
        v = torch.randn(N, generator=gen)
        bad = v.clone()
        bad[2:5] = math.nan
        calls = []
        for z, u in ((x, bad), (clean, v)):
            z, u, l = z.cuda(), u.cuda(), lab.cuda()
            lp, st = evt.class_logp(z, l)
            ids = torch.zeros(N, 3, dtype=torch.int64)
            ids[:, 1] = V - 1
            ids[:, 2] = -1
            ids[2:5] = -5
            top = torch.ones(N, 3)
            if u[2] != u[2]:
                top[:, 2], top[2:5] = math.nan, math.inf
            off = torch.tensor([0, 6, N], dtype=torch.int32)
            calls.append([lp, st, evt.class_logp_grad(z, l, st, u), *evt.policy_loss(z, l, u, u, u, kl_coef=0.1, weights=u.abs()),
                          *evt.distill_loss(z, ids.cuda(), top.cuda(), weights=v.abs().cuda()), *evt.preference_loss(z, l, off.cuda(), v[:2].cuda())])
        for a, b in zip(*calls):
            assert torch.equal(a, b) and not torch.isnan(a).any()


def test_threads_on_streams_of_their_own(evt):
    """Calls of several threads at once, each on its own stream."""
    import threading
    x, gen = _scores(6007, torch.float16, 44, 50, special=False)
    calls = _calls(evt, x.cuda(), gen)
    want = [[t.clone() for t in f()] for f in calls]
    torch.cuda.synchronize()
    wrong = []

    def work():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = [f() for f in calls]
                stream.synchronize()
                for a, b in zip(got, want):
                    for u, v in zip(a, b):
                        if not torch.equal(u, v):
                            wrong.append(1)
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("V,N", [(130, 24), (33_000, 600)])  # one launch for slopes and losses, and two
def test_preference_offsets_past_the_last(evt, V, N):
    """A sequence behind the last offset has rows that no loss counts: its pair is NaN, not the loss of no rows."""
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(N, V, generator=gen)
    lab = torch.randint(0, V, (N,), generator=gen)
    ref = torch.randn(6, generator=gen) - 20
    off = torch.tensor([0, 3, 18, 6, 6, 9, 12], dtype=torch.int32)  # sequence 1 ends behind row 11, 2 descends; pairs are (0, 3), (1, 4), (2, 5)
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref.cuda())
    assert torch.isnan(loss).tolist() == [False, True, True]
    assert torch.isnan(seq).tolist() == [False, True, True, False, True, True]
    alone, tol = plain.preference(x, lab, torch.tensor([0, 3, 3]), ref[[0, 3]], 0.1, 0.0, 0.0, False, 1.0, None)[0]
    plain.close("loss", loss[:1], alone, tol)
    off = torch.tensor([6, 9, 0, 3, 12], dtype=torch.int32)  # sequence 1 descends, 2 begins in front of the first: pairs (0, 2), (1, 3)
    loss, seq, grad = evt.preference_loss(x.cuda(), lab.cuda(), off.cuda(), ref[:4].cuda())
    assert torch.isnan(loss).all() and torch.isnan(seq).all()
