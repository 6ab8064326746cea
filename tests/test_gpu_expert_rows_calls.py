"""Rows through experts in calls that lie at the edge of what is allowed: empty batches, memory that is shared, more rows than a launch has, threads."""
import threading

import pytest
import torch

import expert_rows_plain as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(evt, top, dtype):
    """An empty micro-batch through all of a layer."""
    scores, x = torch.zeros(0, 7, dtype=dtype, device="cuda"), torch.zeros(0, 5, dtype=dtype, device="cuda")
    ids, w = evt.route_rows(scores, top)
    plan = evt.plan_rows(ids[:, 0].contiguous() if top == 1 else ids, 7)
    assert plan.place.shape == (0, top) and plan.offsets.tolist() == [0] * 8
    y = evt.sort_rows(x, plan)
    out = evt.combine_rows(y, plan, w, residual=x, p=0.1, seed=1)
    dy, dw = evt.combine_rows_grad(out, y, plan, w, p=0.1, seed=1)
    dx = evt.combine_rows(dy, plan, residual=out)
    assert y.shape == out.shape == dy.shape == dx.shape == (0, 5) and dw.shape == (0, top) and evt.combine_rows_grad(out, None, plan, None)[1] is None
    assert evt.route_rows_grad(scores, ids, w, dw).shape == (0, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,top", [(1, 2), (5, 3), (64, 2), (201, 8), (513, 1), (4099, 2)])
def test_columns_of_one_matrix(evt, H, top, dtype):
    """x, residual and result side by side in the same rows: the results of tensors of their own, and nothing else is written."""
    rows, experts, gen = 37, 7, torch.Generator().manual_seed(H)
    n = rows * top
    ids = torch.randint(-1, experts, (rows, top), generator=gen).cuda()
    plan = evt.plan_rows(ids, experts)
    w = torch.rand(rows, top, generator=gen).cuda()
    first = torch.randn(n, 3 * H + 2, generator=gen).to(dtype).cuda()

    def columns():
        buf = first.clone()
        return buf, buf[:, :H], buf[:, H:2 * H], buf[:, 2 * H + 1:3 * H + 1]

    def check(call, *shapes):
        """call(a, b, out) with rows that these tensors have, out one of the three places."""
        for at in range(3):
            buf, *cols = columns()
            a, b = (c[:m] for c, m in zip([c for i, c in enumerate(cols) if i != at], shapes))
            out = cols[at][:shapes[2]]
            want = call(a.clone(), b.clone(), None)
            expected = buf.clone()
            expected[:shapes[2], out.storage_offset():out.storage_offset() + H] = want
            assert call(a, b, out) is out and torch.equal(buf, expected)

    check(lambda a, b, out: evt.sort_rows(a, plan, out=out), rows, rows, n)
    check(lambda a, b, out: evt.combine_rows(a, plan, w, residual=b, p=0.3, seed=2, out=out), n, rows, rows)
    check(lambda a, b, out: evt.drop_rows(a, 0.3, 2, residual=b, out=out), n, n, n)
    if 1 < H <= 4096:
        shape = (n, min(H, 3))
        e, we = torch.randint(0, H, shape, generator=gen).cuda(), torch.rand(shape, generator=gen).cuda()
        for renormalize in (True, False):
            check(lambda a, b, out: evt.route_rows_grad(a, e, we, we, renormalize=renormalize, out=out), n, n, n)


def test_results_on_tables(evt):
    """Refused where they lie on what the call reads, taken where they only touch it."""
    rows, top, H, experts = 40, 8, 8, 11
    n = rows * top
    gen = torch.Generator().manual_seed(1)
    memory = torch.zeros(3 * n * H + 64, device="cuda")
    at = [0]

    def place(*shape):
        """A tensor that starts where the last one ended."""
        size = torch.Size(shape).numel()
        at[0] += size
        return memory[at[0] - size:at[0]].view(shape)

    w, out, x, y, seed = place(rows, top), place(rows, H), place(rows, H), place(n, H), memory[-2:].view(torch.int64)
    for t in (w, x, y):
        t.copy_(torch.randn(t.shape, generator=gen))
    seed.fill_(77)
    ids = torch.randint(-1, experts, (rows, top), generator=gen).cuda()
    plan = evt.plan_rows(ids, experts)
    assert evt.combine_rows(y, plan, w, residual=x, p=0.3, seed=seed, out=out) is out
    assert torch.equal(out, evt.combine_rows(y.clone(), plan, w.clone(), residual=x.clone(), p=0.3, seed=77))
    assert torch.equal(evt.drop_rows(x, 0.3, seed, out=out), evt.drop_rows(x, 0.3, 77))
    scores = torch.randn(rows, H, generator=gen).cuda()
    e, v = evt.route_rows(scores, top)
    tables = plan._tables[:2 * n].view(torch.float32)
    for call in (lambda: evt.combine_rows(y, plan, w, out=w), lambda: evt.combine_rows(y, plan, w, out=memory[n - 1:n - 1 + rows * H].view(rows, H)),
                 lambda: evt.combine_rows(y, plan, w, p=0.5, seed=seed, out=memory[-1 - rows * H:-1].view(rows, H)),
                 lambda: evt.drop_rows(x[:1], 0.5, seed, out=memory[-H - 1:-1].view(1, H)), lambda: evt.combine_rows(y, plan, w, out=tables[:rows * H].view(rows, H)),
                 lambda: evt.route_rows_grad(scores, e, v, v.clone(), out=v), lambda: evt.route_rows_grad(scores, e, v.clone(), v, renormalize=False, out=v),
                 lambda: evt.route_rows_grad(scores, e, v, v, out=e.view(torch.float32))):
        before = memory.clone()
        with pytest.raises(evt.EvtError, match="apart"):
            call()
        assert torch.equal(memory, before)


def test_memory_of_a_plan(evt):
    """Tables of many experts, eagerly and in a graph: what the call works in goes to the next one, and the plan keeps its tables alone."""
    rows, top, experts, H = 20000, 2, 4096, 33
    gen = torch.Generator().manual_seed(3)
    ids, x = torch.randint(-1, experts, (rows, top), generator=gen).cuda(), torch.randn(rows, H, generator=gen).cuda()
    other = torch.randint(0, experts, (rows, top), generator=gen).cuda()
    evt.plan_rows(ids, experts)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    plan = evt.plan_rows(ids, experts)
    tables = 4 * (2 * rows * top + experts + 1)
    assert torch.cuda.memory_allocated() - before <= tables + 65536
    wanted = [[t.clone() for t in (p.place, p.source, p.offsets, evt.sort_rows(x, p))] for p in (evt.plan_rows(ids, experts), evt.plan_rows(other, experts))]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plans = [evt.plan_rows(i, experts) for i in (ids, other)]
        outs = [[p.place, p.source, p.offsets, evt.sort_rows(x, p)] for p in plans]
    for _ in range(4):
        for out in outs:
            for t in out:
                t.zero_()
        g.replay()
        eager = [evt.plan_rows(i, experts) for i in (other, ids)]
        for out, want in zip(outs, wanted):
            assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert torch.equal(eager[0].source, wanted[1][1]) and torch.equal(eager[1].source, wanted[0][1])
    assert torch.equal(plan.place, wanted[0][0]) and torch.equal(plan.source, wanted[0][1])


@pytest.mark.parametrize("H,top", [(3, 1), (9, 2)])
def test_more_rows_than_a_launch_has(evt, H, top):
    """Places and weights by the absolute row, what no entry has cleared once: rows on both sides of the 2^24th, where the second launch begins, with and without experts."""
    rows, experts = 17_000_000, 5
    gen = torch.Generator(device="cuda").manual_seed(H)
    ids = torch.randint(0, experts, (rows, top), generator=gen, device="cuda")
    ids[(1 << 24) - 700:(1 << 24) + 300] = -1
    ids[rows - 1000:] = -1
    plan = evt.plan_rows(ids, experts)
    place, n = plan.place.long(), rows * top
    valid, count = place >= 0, int(plan.offsets[-1])
    assert count == n - 2000 * top and torch.equal(valid, ids >= 0)
    x = torch.randn(rows, H, generator=gen, device="cuda").half()
    out = torch.full((n, H), 7.0, dtype=torch.float16, device="cuda")
    evt.sort_rows(x, plan, out=out)
    source = plan.source.long()
    assert torch.equal(out[:count], x[source[:count] // top]) and bool((out[count:] == 0).all())
    y = torch.randn(n, H, generator=gen, device="cuda").half()
    w = torch.rand(rows, top, generator=gen, device="cuda")
    sums, sizes = torch.zeros(rows, H, dtype=torch.float64, device="cuda"), torch.zeros(rows, H, dtype=torch.float64, device="cuda")
    for j in range(top):
        part = torch.where(valid[:, j, None], w[:, j, None].double() * y[place[:, j].clamp(min=0)].double(), 0.0)
        sums += part
        sizes += part.abs()
    got = evt.combine_rows(y, plan, w).double()
    # two 32-bit steps an entry, and the result's half step, the smallest numbers' included
    assert bool(((got - sums).abs() <= sums.abs() * 2.0 ** -11 + 2.0 ** -25 + 2 * top * 1.01 * 2.0 ** -24 * sizes).all())
    del sums, sizes, got
    dy, dw = evt.combine_rows_grad(x, y, plan, w)
    assert bool((dy[count:] == 0).all()) and bool((dw[~valid] == 0).all())
    for j in range(top):
        at = place[:, j].clamp(min=0)
        assert torch.equal(dy[at][valid[:, j]], (w[:, j, None] * x.float()).half()[valid[:, j]])  # one product, one rounding
        terms = x.double() * y[at].double()
        assert bool(((dw[:, j].double() - terms.sum(1)).abs() <= 1.01 * 2.0 ** -24 * (H + 6) * terms.abs().sum(1))[valid[:, j]].all())


def test_threads(evt):
    """Four threads on their own streams, twenty turns each, all of which have to come to an end."""
    gen = torch.Generator().manual_seed(8)
    given = []
    for rows, experts, top, H, dtype in ((9000, 64, 4, 130, torch.bfloat16), (100, 8, 2, 4096, torch.float32), (1500, 1000, 8, 65, torch.float16), (3000, 4096, 1, 512, torch.float32)):
        given.append((torch.randn(rows, experts, generator=gen).cuda(), torch.randn(rows, H, generator=gen).to(dtype).cuda(), top, experts))

    def step(scores, x, top, experts):
        ids, w = evt.route_rows(scores, top)
        plan = evt.plan_rows(ids, experts)
        y = evt.sort_rows(x, plan)
        out = evt.combine_rows(y, plan, w, residual=x, p=0.2, seed=4)
        dy, dw = evt.combine_rows_grad(out, y, plan, w, p=0.2, seed=4)
        return ids, w, plan.place, plan.source, y, out, dy, dw, evt.route_rows_grad(scores, ids, w, dw)

    wanted = [[t.clone() for t in step(*g)] for g in given]
    torch.cuda.synchronize()
    turns, wrong = [0] * len(given), []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = step(*given[k])
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, wanted[k])):
                        wrong.append("another result in thread %d" % k)
                    turns[k] += 1
        except BaseException as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(given))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and turns == [20] * len(given), (wrong, turns)


def test_in_autograd_functions(evt):
    """The gradients that the calls return, as a program records them: those of a composition of plain operations in 64 bits, at every leaf."""
    rows, experts, top, H, p, seed = 23, 6, 2, 17, 0.25, 12

    class Route(torch.autograd.Function):
        @staticmethod
        def forward(ctx, scores):
            ids, w = evt.route_rows(scores, top)
            ctx.save_for_backward(scores, ids, w)
            ctx.mark_non_differentiable(ids)
            return ids, w

        @staticmethod
        def backward(ctx, _, dw):
            scores, ids, w = ctx.saved_tensors
            return evt.route_rows_grad(scores, ids, w, dw.contiguous())

    class Sort(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, plan):
            ctx.plan = plan
            return evt.sort_rows(x, plan)

        @staticmethod
        def backward(ctx, dy):
            return evt.combine_rows(dy.contiguous(), ctx.plan), None

    class Combine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, w, x, plan):
            ctx.plan = plan
            ctx.save_for_backward(y, w)
            return evt.combine_rows(y, plan, w, residual=x, p=p, seed=seed)

        @staticmethod
        def backward(ctx, dout):
            y, w = ctx.saved_tensors
            return (*evt.combine_rows_grad(dout.contiguous(), y, ctx.plan, w, p=p, seed=seed), dout, None)

    gen = torch.Generator().manual_seed(5)
    leaves = [torch.randn(s, generator=gen) for s in ((rows, experts), (rows, H), (experts, H))]
    dout = torch.randn(rows, H, generator=gen)
    scores, x, scale = (t.cuda().requires_grad_() for t in leaves)
    assert not any(t.requires_grad for t in (*evt.route_rows(scores, top), evt.drop_rows(x, p, seed)))
    ids, w = Route.apply(scores)
    plan = evt.plan_rows(ids, experts)
    expert = ids.reshape(-1)[plan.source.long()].long()
    out = Combine.apply(Sort.apply(x, plan) * scale[expert], w, x, plan)
    got = torch.autograd.grad(out, (scores, x, scale), dout.cuda())

    s64, x64, k64 = (t.double().requires_grad_() for t in leaves)
    chosen = ids.cpu().long()
    w64 = torch.softmax(s64.gather(1, chosen), 1)
    total = sum(w64[:, j, None] * k64[chosen[:, j]] * x64 for j in range(top))
    gone = plain.bits(rows, H, seed, 0) < plain.threshold(p)
    want_out = x64 + torch.where(gone, 0.0, total * (2.0 ** 32 / (2 ** 32 - plain.threshold(p))))
    want = torch.autograd.grad(want_out, (s64, x64, k64), dout.double())
    # two hundred 32-bit roundings of sums whose terms' sizes add up to less than 40: 46 of dout w x / (1 - p) at most, or a row's 17 of dout scale x / (1 - p)
    for name, a, b in (("out", out, want_out.detach()), ("scores", got[0], want[0]), ("x", got[1], want[1]), ("scale", got[2], want[2])):
        plain.close(name, a, b, torch.full_like(b, 200 * plain.U * 40))


def test_leaves_of_a_tree(evt):
    """A column of predict_leaf_idx, as the module's documentation takes it to the GPU."""
    gen = torch.Generator().manual_seed(6)
    X = torch.randn(500, 3, generator=gen, dtype=torch.float64).numpy()
    m = evt.fit(evt.EvoTreeRegressor(nrounds=2, max_depth=3, nbins=16), x_train=X, y_train=X[:, 0] + X[:, 1])
    leaf = evt.predict_leaf_idx(m, X)
    k = leaf.shape[1] - 1
    ids = torch.from_numpy(leaf[:, k].astype("int64")).cuda()
    plan = evt.plan_rows(ids, int(leaf[:, k].max()) + 1)
    place, source, offsets = plain.plan(ids.cpu()[:, None], plan.experts)
    assert plan.place.reshape(-1).tolist() == place and plan.source.tolist() == source and plan.offsets.tolist() == offsets and offsets[-1] == 500


@pytest.mark.parametrize("mode", [torch.inference_mode, torch.no_grad])
def test_a_layer_without_gradients(evt, mode):
    """Scores that are one row in memory, results in place, tensors made in that mode and read outside of it."""
    rows, experts, top, H = 30, 20, 3, 50
    gen = torch.Generator().manual_seed(9)
    one, x = torch.randn(1, experts, generator=gen), torch.randn(rows, H, generator=gen)
    with mode():
        scores, held = one.cuda().expand(rows, experts), x.cuda()
        ids, w = evt.route_rows(scores, top, renormalize=False)
        plan = evt.plan_rows(ids, experts)
        y = evt.sort_rows(held, plan)
        out = evt.combine_rows(y, plan, w, residual=held, out=held)
        grads = evt.route_rows_grad(scores, ids, w, w, renormalize=False)
    assert out is held
    want, ww, tol = plain.route(one.expand(rows, experts), top, False, 1.0)
    assert torch.equal(ids.cpu(), want)
    plain.close("weights", w, ww, tol)
    plain.close("out", out, *plain.combine(y.cpu(), plan.place.cpu(), w.cpu(), x, 0.0, 0, 0))
    plain.close("grad", grads, *plain.route_grad(one.expand(rows, experts), want, w.cpu(), w.cpu(), False, 1.0))
    again = evt.plan_rows(ids.clone(), experts)  # outside
    assert torch.equal(again.place, plan.place) and not again.place.is_inference()
