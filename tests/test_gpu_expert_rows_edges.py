"""Rows through experts as a program uses them: a layer and its backward pass, the leaves of a tree as experts, other streams, threads and graphs, padded batches, rows that are
one in memory, offsets beyond 32 bits and more rows than a launch has."""
import math
import threading

import numpy as np
import pytest
import torch

import expert_rows_plain as plain

pytestmark = pytest.mark.gpu


class Layer:
    """A router and experts that scale their rows, with the calls of a training step."""

    def __init__(self, evt, rows=37, experts=6, top=3, H=20, dtype=torch.float32, seed=1, p=0.25, pad=2, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        self.evt, self.experts, self.top, self.p, self.layer = evt, experts, top, p, 5
        self.scores = torch.randn(rows, experts, generator=gen)
        self.scores[rows - pad:] = -math.inf  # padded rows: no expert
        self.x, self.dout = (torch.randn(rows, H, generator=gen).to(dtype) for _ in range(2))
        self.scale = (torch.rand(experts, generator=gen) + 0.5).to(dtype)
        self.seed = torch.tensor([seed * 7919])
        if device != "cpu":
            for name in ("scores", "x", "dout", "scale", "seed"):
                setattr(self, name, getattr(self, name).to(device))

    def expert_of_place(self, plan):
        e = torch.bucketize(torch.arange(plan.rows * plan.top, device=self.x.device, dtype=torch.int32), plan.offsets[1:], right=True)
        return self.scale[e.clamp(max=self.experts - 1)][:, None]

    def step(self):
        evt = self.evt
        experts, weights = evt.route_rows(self.scores, self.top, temperature=0.8)
        plan = evt.plan_rows(experts, self.experts)
        scale = self.expert_of_place(plan)
        y = evt.sort_rows(self.x, plan) * scale
        out = evt.combine_rows(y, plan, weights, residual=self.x, p=self.p, seed=self.seed, layer=self.layer)
        dy, dweights = evt.combine_rows_grad(self.dout, y, plan, weights, p=self.p, seed=self.seed, layer=self.layer)
        dx = evt.combine_rows(dy * scale, plan, residual=self.dout)
        dscores = evt.route_rows_grad(self.scores, experts, weights, dweights, temperature=0.8)
        return out, dx, dscores, weights, dweights, experts, plan.place, plan.source, plan.offsets, dy, y


def test_layer_and_its_backward_pass(evt):
    L = Layer(evt)
    out, dx, dscores, weights, dweights, experts, place, source, offsets, dy, y = [t.cpu() for t in L.step()]
    scores, x, dout, scale, seed = (getattr(L, n).cpu().double() if n != "seed" else int(L.seed) for n in ("scores", "x", "dout", "scale", "seed"))
    rows, H = x.shape

    def forward(scores, x):
        ids, w, _ = plain.route(scores, L.top, True, 0.8)
        assert torch.equal(ids, experts)
        total = torch.zeros_like(x)
        for j in range(L.top):
            has = ids[:, j] >= 0
            total[has] += w[has, j, None] * scale[ids[has, j].long()][:, None] * x[has]
        return x + plain.dropped(total, L.p, seed, L.layer)

    # some two hundred roundings on the way to a gradient, of what its terms are in size
    d = plain.dropped(dout, L.p, seed, L.layer).abs()
    by_expert = (d * x.abs()).sum(1, keepdim=True) * scale.max()
    plain.close("out", out, forward(scores, x), 50 * plain.U * (x.abs() + 3 * scale.max() * x.abs()))
    for i, c in [(i, c) for i in (0, 11, 36) for c in range(H)]:
        e = torch.zeros_like(x)
        e[i, c] = 1e-4
        slope = float(((forward(scores, x + e) - forward(scores, x - e)) * dout).sum()) / 2e-4
        assert abs(slope - float(dx[i, c])) < 200 * plain.U * float(dout[i, c].abs() + d[i, c] * scale.max()) + 1e-9
    for i, c in [(i, c) for i in (0, 11, 20) for c in range(L.experts)]:
        e = torch.zeros_like(scores)
        e[i, c] = 1e-4
        slope = float(((forward(scores + e, x) - forward(scores - e, x)) * dout).sum()) / 2e-4
        # a difference's own error: its step squared over six of a third derivative
        assert abs(slope - float(dscores[i, c])) < (200 * plain.U + 1e-7) * float(by_expert[i]) / 0.8 + 1e-9
    assert (dscores[35:] == 0).all() and torch.equal(out[35:], L.x[35:].cpu()) and torch.equal(dx[35:], L.dout[35:].cpu()) and (dweights[35:] == 0).all()


def test_leaves_of_a_tree_as_experts(evt):
    rng = np.random.default_rng(0)
    X = rng.normal(size=(3000, 5))
    target = (X[:, 0] > 0) * 2.0 + X[:, 1]
    m = evt.fit(evt.EvoTreeRegressor(nrounds=1, max_depth=4, nbins=16), x_train=X, y_train=target)
    leaf = evt.predict_leaf_idx(m, X)[:, -1].astype(np.int64)  # the first tree is the bias
    n = int(leaf.max()) + 1
    assert len(set(leaf.tolist())) > 3
    plan = evt.plan_rows(torch.from_numpy(leaf).cuda(), n)
    place, source, offsets = plain.plan(torch.from_numpy(leaf)[:, None], n)
    assert plan.source.tolist() == source and plan.offsets.tolist() == offsets
    x = torch.from_numpy(X.astype(np.float32)).cuda()
    rows = evt.sort_rows(x, plan)
    assert torch.equal(rows.cpu(), torch.from_numpy(X.astype(np.float32))[source])
    bounds = plan.offsets.tolist()
    means = torch.cat([rows[a:b].mean(0, keepdim=True).expand(b - a, -1) for a, b in zip(bounds, bounds[1:]) if b > a])  # a model of each leaf
    back = evt.combine_rows(means.contiguous(), plan)
    for k in set(leaf.tolist()):
        at = torch.from_numpy(np.nonzero(leaf == k)[0]).cuda()
        plain.close("leaf's mean", back[at], x[at].double().mean(0, keepdim=True).expand(len(at), -1).cpu(), x[at].double().abs().mean(0).cpu() * len(at) * plain.U)


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_equal_calls_give_equal_bits(evt):
    for dtype in (torch.float32, torch.bfloat16):
        L = Layer(evt, rows=1500, experts=100, top=9, H=333, dtype=dtype)
        first = [t.clone() for t in L.step()]
        for _ in range(3):
            assert _same(L.step(), first)


def test_streams_and_graphs(evt):
    """On another stream; recorded into two graphs that are replayed in turn, with eager work and another seed between: every replay equals the eager result."""
    layers = [Layer(evt, rows=300, experts=12, top=4, H=70, seed=3), Layer(evt, rows=5000, experts=300, top=2, H=1000, dtype=torch.bfloat16, seed=4)]
    eager = [[t.clone() for t in L.step()] for L in layers]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [L.step() for L in layers]
    side.synchronize()
    assert all(_same(a, b) for a, b in zip(got, eager))
    graphs = []
    for L in layers:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = L.step()
        graphs.append((g, outs))
    for turn in range(4):
        for L, (g, outs), e in zip(layers, graphs, eager):
            for t in outs:
                t.zero_()
            g.replay()
            assert _same(outs, L.step())
            if turn == 0:
                assert _same(outs, e)
        for L in layers:
            L.seed += 1
            L.scores.mul_(-1.0 if turn == 1 else 1.1).masked_fill_(L.scores == math.inf, -math.inf)
    graphs[0][0].replay()
    graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(_same(outs, L.step()) for L, (g, outs) in zip(layers, graphs))


def test_threads_on_their_own_streams(evt):
    layers = [Layer(evt, rows=r, experts=e, top=k, H=h, dtype=t, seed=r) for r, e, k, h, t in
              ((20000, 64, 4, 130, torch.bfloat16), (100, 8, 2, 4096, torch.float32), (3000, 1000, 8, 65, torch.float16), (9000, 5, 1, 512, torch.float32))]
    want = [[t.clone() for t in L.step()] for L in layers]
    torch.cuda.synchronize()
    wrong = []

    def work(L, w):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = L.step()
                s.synchronize()
                if not _same(got, w):
                    wrong.append(L)
    threads = [threading.Thread(target=work, args=a) for a in zip(layers, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", list(plain.TYPES))
def test_a_batch_of_padding(evt, dtype):
    t = plain.TYPES[dtype]
    for rows, top, H in ((1, 1, 1), (5, 3, 100), (700, 2, 1000)):
        scores = torch.full((rows, 9), -math.inf, dtype=t, device="cuda")
        ids, w = evt.route_rows(scores, top)
        assert (ids == -1).all() and (w == 0).all()
        assert (evt.route_rows_grad(scores, ids, w, torch.full_like(w, math.nan), renormalize=False) == 0).all()
        plan = evt.plan_rows(ids, 9)
        assert (plan.place == -1).all() and (plan.source == -1).all() and (plan.offsets == 0).all()
        x, res = torch.randn(rows, H, device="cuda").to(t), torch.randn(rows, H, device="cuda").to(t)
        y = torch.full((rows * top, H), math.nan, dtype=t, device="cuda")
        assert (evt.sort_rows(x, plan) == 0).all()
        none = torch.full((rows, top), math.nan, device="cuda")
        assert torch.equal(evt.combine_rows(y, plan, none, residual=res, p=0.5, seed=3), res) and (evt.combine_rows(y, plan, none) == 0).all()
        dy, dw = evt.combine_rows_grad(x, y, plan, none)
        assert (dy == 0).all() and (dw == 0).all()


def test_no_rows(evt):
    scores = torch.zeros(0, 7, device="cuda")
    ids, w = evt.route_rows(scores, 3)
    assert ids.shape == w.shape == (0, 3) and evt.route_rows_grad(scores, ids, w, w).shape == (0, 7)
    plan = evt.plan_rows(ids, 7)
    assert plan.place.shape == (0, 3) and plan.source.shape == (0,) and plan.offsets.tolist() == [0] * 8
    x = torch.zeros(0, 5, device="cuda")
    assert evt.sort_rows(x, plan).shape == evt.combine_rows(x, plan, w, residual=x, p=0.1, seed=1).shape == evt.drop_rows(x, 0.1, 1).shape == (0, 5)
    dy, dw = evt.combine_rows_grad(x, x, plan, w)
    assert dy.shape == (0, 5) and dw.shape == (0, 3)


@pytest.mark.parametrize("H", [7, 64, 513, 2048])
def test_values_that_are_none(evt, H):
    """What is dropped is 0 whatever it was; what is not stays as arithmetic has it, and no other element's."""
    rows, p, seed, layer = 40, 0.4, 99, 1
    x = torch.randn(rows, H)
    x[::3] = math.nan
    x[1::3] = math.inf
    out = evt.drop_rows(x.cuda(), p, seed, layer=layer).cpu()
    gone = plain.bits(rows, H, seed, layer) < plain.threshold(p)
    assert (out[gone] == 0).all() and out[::3][~gone[::3]].isnan().all() and (out[1::3][~gone[1::3]] == math.inf).all() and out[2::3].isfinite().all()
    ids = torch.arange(rows)[:, None] % 4
    plan = evt.plan_rows(ids.cuda(), 4)
    place = plan.place.cpu()[:, 0].long()
    y = torch.randn(rows, H)
    y[place[5]] = math.nan
    y[place[9], H // 2] = -math.inf
    w = torch.rand(rows, 1) + 0.5
    out = evt.combine_rows(y.cuda(), plan, w.cuda()).cpu()
    assert out[5].isnan().all() and out[9, H // 2] == -math.inf and int((~out.isfinite()).sum()) == H + 1
    dy, dw = evt.combine_rows_grad(x.cuda(), y.cuda(), plan, w.cuda(), p=p, seed=seed, layer=layer)
    want_y, want_w = plain.combine_grad(x, y, place[:, None], w, p, seed, layer)
    plain.close("dy", dy, *want_y)
    plain.close("dweights", dw, *want_w)


@pytest.mark.parametrize("H", [5, 100, 1025])
def test_one_row_for_all(evt, H):
    """Rows that are only read may be one in memory."""
    rows, top = 50, 2
    ids, gen = torch.arange(rows * top).view(rows, top) % 7, torch.Generator().manual_seed(H)
    plan = evt.plan_rows(ids.cuda(), 7)
    one, w = torch.randn(1, H, generator=gen), torch.rand(rows, top, generator=gen)
    many = one.cuda().expand(rows, H)
    place = plan.place.cpu()
    assert torch.equal(evt.sort_rows(many, plan).cpu(), one.expand(rows * top, H))
    plain.close("combine", evt.combine_rows(one.cuda().expand(rows * top, H), plan, w.cuda(), residual=many, p=0.2, seed=4),
                *plain.combine(one.expand(rows * top, H), place, w, one.expand(rows, H), 0.2, 4, 0))
    dy, dw = evt.combine_rows_grad(many, one.cuda().expand(rows * top, H), plan, w.cuda(), p=0.2, seed=4)
    want_y, want_w = plain.combine_grad(one.expand(rows, H), one.expand(rows * top, H), place, w, 0.2, 4, 0)
    plain.close("dy", dy, *want_y)
    plain.close("dweights", dw, *want_w)
    plain.close("drop", evt.drop_rows(many, 0.2, 4, residual=many), *plain.drop(one.expand(rows, H), 0.2, 4, 0, one.expand(rows, H)))


def test_offsets_beyond_32_bits(evt):
    """2.6e9 values of sorted rows."""
    rows, top, H = 40000, 8, 8192
    ids = (torch.arange(rows, device="cuda")[:, None] * 3 + torch.arange(top, device="cuda") * 5) % 64
    plan = evt.plan_rows(ids, 64)
    x = torch.randn(rows, H, device="cuda").bfloat16()
    y = evt.sort_rows(x, plan)
    for at in range(0, rows * top, 20000):
        part = plan.source[at:at + 20000].long() // top
        assert torch.equal(y[at:at + 20000], x[part]), at
    assert torch.equal(evt.combine_rows(y, plan), x * 8)  # seven exact sums in 32 bits
    w = torch.ones(rows, top, device="cuda")
    dy, dw = evt.combine_rows_grad(x, y, plan, w)
    assert torch.equal(dy, y)
    size = (x.double() ** 2).sum(1, keepdim=True)
    assert ((dw.double() - size).abs() <= 1.01 * plain.U * (8 + H // 256 + 14) * size).all()


@pytest.mark.parametrize("rows,H", [(17_000_000, 3), (17_000_000, 9), (8_500_000, 520)])
def test_more_rows_than_a_launch_has(evt, rows, H):
    """In place: a row done twice would show."""
    x = torch.ones(rows, H, dtype=torch.float16, device="cuda")
    assert evt.drop_rows(x, 0.25, 5, out=x) is x
    scale = torch.tensor(2.0 ** 32 / (2 ** 32 - plain.threshold(0.25))).half().cuda()
    for first in (0, rows // 2, rows - 1000, 1 << 23, (1 << 24) - 500):
        first = min(first, rows - 1000)
        keep = plain.bits(1000, H, 5, 0, first) >= plain.threshold(0.25)
        assert torch.equal(x[first:first + 1000].cpu(), torch.where(keep, scale.cpu(), torch.zeros((), dtype=torch.float16)))
    for a in range(0, rows, 1 << 20):
        part = x[a:a + (1 << 20)]
        assert bool(((part == 0) | (part == scale)).all())


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("V,top", [(5, 5), (40, 6), (256, 8), (100, 40), (3000, 64)])
def test_one_expert_several_times_in_a_row(evt, V, top, renormalize):
    """Its shares are added up, in the same order in every call."""
    rows, gen = 21, torch.Generator().manual_seed(V)
    x = torch.randn(rows, V, generator=gen)
    ids = torch.randint(0, V, (rows, top), generator=gen)
    ids[3] = 2
    ids[4, ::2] = 1
    ids[5, 1:] = -1
    w, dw = torch.rand(rows, top, generator=gen), torch.randn(rows, top, generator=gen) * 10
    w /= w.sum(1, keepdim=True)
    got = evt.route_rows_grad(x.cuda(), ids.cuda(), w.cuda(), dw.cuda(), renormalize=renormalize, temperature=0.5)
    plain.close("grad", got, *plain.route_grad(x, ids, w, dw, renormalize, 0.5))
    for _ in range(3):
        assert torch.equal(evt.route_rows_grad(x.cuda(), ids.cuda(), w.cuda(), dw.cuda(), renormalize=renormalize, temperature=0.5), got)
    place, source, offsets = plain.plan(ids, V)
    plan = evt.plan_rows(ids.cuda(), V)
    assert plan.place.reshape(-1).tolist() == place and plan.source.tolist() == source and plan.offsets.tolist() == offsets


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", [6, 64, 200, 1030])
def test_scores_at_the_ends_of_their_type(evt, V, dtype):
    """The lowest number is a score like others, -inf is none; several that are no numbers come first, in their order, then +inf."""
    t = plain.TYPES[dtype]
    info, gen = torch.finfo(t), torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=gen)
    x[0] = -math.inf
    x[0, V // 2], x[0, 1] = info.min, info.min
    x[1] = info.min
    x[1, V - 1] = info.max
    x[2, ::2], x[2, 1::2] = info.max, info.min
    x[3, 1] = x[3, V - 1] = math.nan
    x[3, 2] = math.inf
    x[4, 0] = x[4, V - 2] = math.inf
    x[5] = info.smallest_normal
    x[5, ::2] = -info.smallest_normal
    x[6] = 0.0
    x[6, V - 1] = info.smallest_normal * info.eps  # the least number above 0
    x[6, 0] = -0.0
    x = x.to(t)
    for top in (1, 2, 4, 6):
        for renormalize in (True, False):
            ids, w = evt.route_rows(x.cuda(), top, renormalize=renormalize)
            want, ww, tol = plain.route(x, top, renormalize, 1.0)
            assert torch.equal(ids.cpu(), want), (top, ids.cpu(), want)
            plain.close("weights", w, ww, tol.nan_to_num(0, 0, 0) + plain.U)


@pytest.mark.parametrize("rows", [1, 2])
@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("H", [1, 8, 100, 2048, 5003])
def test_single_rows(evt, H, dtype, rows):
    """A service's step: one token or two through all of it, without dropout."""
    experts, top, t = 64, 6, plain.TYPES[dtype]
    gen = torch.Generator().manual_seed(H + rows)
    scores, x, res = (torch.randn(rows, n, generator=gen).to(t) for n in (experts, H, H))
    ids, w = evt.route_rows(scores.cuda(), top)
    want, ww, tol = plain.route(scores, top, True, 1.0)
    assert torch.equal(ids.cpu(), want)
    plain.close("weights", w, ww, tol)
    plan = evt.plan_rows(ids, experts)
    place, source, offsets = plain.plan(want, experts)
    assert plan.place.reshape(-1).tolist() == place and plan.source.tolist() == source and plan.offsets.tolist() == offsets
    y = evt.sort_rows(x.cuda(), plan)
    assert torch.equal(y.cpu(), x[torch.tensor(source) // top])
    out = evt.combine_rows(y, plan, w, residual=res.cuda())
    plain.close("combine", out, *plain.combine(y.cpu(), plan.place.cpu(), w.cpu(), res, 0.0, 0, 0))


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("V", [40, 48, 49, 70, 96, 130, 160, 192, 193, 300, 384, 385, 600, 768, 769, 1200, 1536, 1537, 3000])
def test_choices_of_every_length(evt, V, dtype):
    """Every number of lanes and of scores a lane, lists of 2, 4, 8 and 16 and longer choices, with many equal scores."""
    gen = torch.Generator().manual_seed(V)
    x = (torch.randn(9, V, generator=gen) * 3).round() / 2
    x[1, V // 3:] = -math.inf
    x[2, :V - 3] = -math.inf
    x = x.to(plain.TYPES[dtype])
    for top in (1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 33):
        ids, w = evt.route_rows(x.cuda(), top, renormalize=top % 2 == 0, temperature=0.9)
        want, ww, tol = plain.route(x, top, top % 2 == 0, 0.9)
        assert torch.equal(ids.cpu(), want), (top, ids.cpu(), want)
        plain.close("weights", w, ww, tol)


@pytest.mark.parametrize("dtype", list(plain.TYPES))
@pytest.mark.parametrize("H", [70_001, 1_000_003])
def test_very_long_rows(evt, H, dtype):
    rows, top, t = 3, 2, plain.TYPES[dtype]
    gen = torch.Generator().manual_seed(H)
    ids = torch.tensor([[1, 0], [-1, 1], [0, 2]])
    plan = evt.plan_rows(ids.cuda(), 3)
    place = plan.place.cpu()
    x, res, y = (torch.randn(n, H, generator=gen).to(t) for n in (rows, rows, rows * top))
    w = torch.rand(rows, top, generator=gen)
    want = torch.zeros(rows * top, H, dtype=t)
    for r in range(rows):
        for j in range(top):
            if place[r, j] >= 0:
                want[place[r, j]] = x[r]
    assert torch.equal(evt.sort_rows(x.cuda(), plan).cpu(), want)
    plain.close("combine", evt.combine_rows(y.cuda(), plan, w.cuda(), residual=res.cuda(), p=0.2, seed=8, layer=1), *plain.combine(y, place, w, res, 0.2, 8, 1))
    dy, dw = evt.combine_rows_grad(x.cuda(), y.cuda(), plan, w.cuda(), p=0.2, seed=8, layer=1)
    want_y, want_w = plain.combine_grad(x, y, place, w, 0.2, 8, 1)
    plain.close("dy", dy, *want_y)
    plain.close("dweights", dw, *want_w)
    plain.close("drop", evt.drop_rows(x.cuda(), 0.2, 8, layer=1), *plain.drop(x, 0.2, 8, 1, None))


def test_many_experts_a_row(evt):
    """A model's trees as routers: two hundred entries a row."""
    rows, top, experts, H = 40, 203, 31, 37
    ids, gen = torch.randint(-1, experts, (rows, top), generator=torch.Generator().manual_seed(1)), torch.Generator().manual_seed(2)
    plan = evt.plan_rows(ids.cuda(), experts)
    place, source, offsets = plain.plan(ids, experts)
    assert plan.place.reshape(-1).tolist() == place and plan.source.tolist() == source and plan.offsets.tolist() == offsets
    place = plan.place.cpu()
    x, y, w = torch.randn(rows, H, generator=gen), torch.randn(rows * top, H, generator=gen), torch.rand(rows, top, generator=gen)
    n = offsets[-1]
    sorted_rows = evt.sort_rows(x.cuda(), plan).cpu()
    assert torch.equal(sorted_rows[:n], x[torch.tensor(source[:n]) // top]) and (sorted_rows[n:] == 0).all()
    plain.close("combine", evt.combine_rows(y.cuda(), plan, w.cuda()), *plain.combine(y, place, w, None, 0.0, 0, 0))
    dy, dw = evt.combine_rows_grad(x.cuda(), y.cuda(), plan, w.cuda())
    want_y, want_w = plain.combine_grad(x, y, place, w, 0.0, 0, 0)
    plain.close("dy", dy, *want_y)
    plain.close("dweights", dw, *want_w)


@pytest.mark.parametrize("n", [1 << 20, (1 << 20) + 1, (1 << 20) + 4097])
@pytest.mark.parametrize("experts", [5, 700, 2049])
def test_tables_around_the_large_blocks(evt, n, experts):
    """Both block sizes, joined sources and single ones, entries without an expert; against a stable sort."""
    gen = torch.Generator().manual_seed(n + experts)
    ids = (torch.rand(n, generator=gen) ** 3 * experts).long()
    ids[torch.rand(n, generator=gen) < 0.05] = -1
    plan = evt.plan_rows(ids.cuda(), experts)
    key = torch.where(ids < 0, experts, ids)
    order = torch.argsort(key, stable=True)
    count = int((ids >= 0).sum())
    place = torch.empty_like(order)
    place[order] = torch.arange(n)
    assert torch.equal(plan.place.cpu()[:, 0].long(), torch.where(ids < 0, -1, place))
    assert torch.equal(plan.source.cpu().long(), torch.where(torch.arange(n) < count, order, -1))
    assert plan.offsets.tolist() == [0] + torch.bincount(key, minlength=experts + 1)[:experts].cumsum(0).tolist()
