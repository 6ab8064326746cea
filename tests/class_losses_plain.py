"""The losses over rows of class scores in 64 bits on the CPU, row by row from their formulas, with what a row's log-probabilities may be off by
in 32-bit arithmetic.

U is half a step of float32.  A kernel finds a row's sum S of exponentials from differences d = x - max (off by U |d|), times log2(e) / T (two
roundings more), through the hardware's exp2 (within 2 U), added up in some order of its own.  The exponent's error of 3 U |d| / T weighs
with exp(-|d| / T) and so stays under 1.2 U of the largest term; a term passes through at most V / 256 + 40 sums and rescalings, each off by U or
by 2 U.  So S, and with it log S, is off by less than CHAIN(V) = (2 V / 256 + 90) U, and a log-probability by that and 4 U of its own two terms."""
import math

import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# half the least step of a type: what is left of values under its normal range.  The exponentials' own denormals are lost as well
LEAST = {torch.float64: 0.0, torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def chain(V):
    return (2.0 * V / 256 + 90) * U


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Rows:
    """q, log q and statistics of every row in 64 bits; d: what a row's log q may be off by, per class."""

    def __init__(self, x, T):
        z = x.double()
        self.N, self.V = z.shape
        self.bad = (torch.isnan(z) | (z == math.inf)).any(1)
        clean = torch.where(self.bad[:, None], 0.0, z)
        self.m = clean.amax(1)
        self.empty = self.m == -math.inf
        base = torch.where(self.empty, 0.0, self.m)
        d = (clean - base[:, None]) / T
        self.e = torch.exp(d)
        self.s = self.e.sum(1)
        self.q = torch.where(self.empty[:, None], 0.0, self.e / torch.where(self.empty, 1.0, self.s)[:, None])
        self.lq = torch.where(self.empty[:, None], -math.inf, d - torch.log(self.s)[:, None])
        self.q[self.bad], self.lq[self.bad] = math.nan, math.nan
        far = torch.where(torch.isfinite(d), d.abs(), 0.0)
        self.off = chain(self.V) + 4 * U * (far + math.log(self.V + 1))

    def at(self, table, labels):
        """table[i, labels[i]], NaN for a label past the classes; 0 for one below 0."""
        out = torch.zeros(self.N, dtype=torch.float64)
        for i, c in enumerate(labels.tolist()):
            if c >= self.V:
                out[i] = math.nan
            elif c >= 0:
                out[i] = table[i, c]
        return out


def label_grad(rows, labels, slope, T, dtype, slope_off=None):
    """(gradient, what it may be off by) of rows whose loss has the slope dloss / dlogp; 0 for a slope of 0."""
    g = torch.zeros(rows.N, rows.V, dtype=torch.float64)
    tol = torch.zeros_like(g)
    for i, c in enumerate(labels.tolist()):
        if c < 0 or slope[i] == 0:
            if slope_off is not None and c >= 0:
                tol[i] = slope_off[i] / T
            continue
        if c >= rows.V or rows.bad[i] or math.isnan(slope[i]):
            g[i] = math.nan
            continue
        one = torch.zeros(rows.V, dtype=torch.float64)
        one[c] = 1
        k = float(slope[i]) / T
        g[i] = k * (one - rows.q[i])
        tol[i] = abs(k) * (rows.q[i] * rows.off[i] + 4 * U * (one + rows.q[i]))
        if slope_off is not None:
            tol[i] += float(slope_off[i]) / T * (one + rows.q[i])
    tol += half_step(dtype) * (g.abs() + tol) + LEAST[dtype] * (1 + slope.abs().nan_to_num(0, 0, 0)[:, None] / T)
    return g, tol


def logp(x, labels, T):
    rows = Rows(x, T)
    out = rows.at(rows.lq, labels)
    off = rows.at(rows.off, labels).nan_to_num(0)
    return out, off + U * out.abs().nan_to_num(0, 0, 0), rows


def distill(x, ids, top, T, w):
    rows = Rows(x, T)
    dtype = x.dtype
    loss = torch.zeros(rows.N, dtype=torch.float64)
    loss_tol = torch.zeros_like(loss)
    g = torch.zeros(rows.N, rows.V, dtype=torch.float64)
    tol = torch.zeros_like(g)
    for i in range(rows.N):
        wi = 1.0 if w is None else float(w[i])
        have = ids[i] >= 0
        t = torch.where(have, top[i].double(), -math.inf)
        if wi == 0 or not (t > -math.inf).any():
            continue
        if (ids[i] >= rows.V).any():
            loss[i], g[i] = math.nan, math.nan
            continue
        lp = torch.log_softmax(t / T, 0)
        p = torch.exp(lp)
        target = torch.zeros(rows.V, dtype=torch.float64)
        lead = (t.amax() - t) / T
        lead = torch.where(torch.isfinite(lead), lead, 0.0)
        p_off = chain(len(t)) + 4 * U * (lead + math.log(len(t) + 1))  # a teacher's probability, relative
        total, off = 0.0, 0.0
        target_off = torch.zeros_like(target)
        for j, c in enumerate(ids[i].tolist()):
            if c < 0 or p[j] == 0:
                continue
            target[c] += p[j]
            target_off[c] += p[j] * p_off[j]
            gap = lp[j] - rows.lq[i, c]
            total += p[j] * gap
            if rows.bad[i] or not math.isfinite(gap):
                continue
            off += p[j] * (p_off[j] * (abs(gap) + 1) + rows.off[i, c] + 4 * U * (abs(lp[j]) + abs(rows.lq[i, c])) + len(t) / 64 * U * abs(gap))
        loss[i] = wi * T * T * total
        loss_tol[i] = abs(wi) * T * T * (off + 8 * U * abs(total)) if math.isfinite(total) else 0.0
        g[i] = wi * T * (rows.q[i] - target)
        tol[i] = abs(wi) * T * (rows.q[i] * rows.off[i] + target_off + 8 * U * (rows.q[i] + target))
    tol += half_step(dtype) * (g.abs() + tol).nan_to_num(0) + LEAST[dtype] * (1 + T * (1.0 if w is None else w.abs().max().item()))
    return (loss, loss_tol + U * loss.abs().nan_to_num(0, 0, 0)), (g, tol)


def policy(x, labels, old, adv, ref, lo, hi, kl, T, w):
    lp, off, rows = logp(x, labels, T)
    n = rows.N
    loss, loss_tol, slope, slope_off = (torch.zeros(n, dtype=torch.float64) for _ in range(4))
    for i in range(n):
        wi = 1.0 if w is None else float(w[i])
        if labels[i] < 0 or wi == 0:
            continue
        v, o = float(lp[i]), float(off[i])
        a = float(adv[i])
        if a != 0:
            if math.isnan(v):
                l = d = math.nan
            else:
                r = math.exp(min(700.0, v - float(old[i])))
                held = min(max(r, 1 - lo), 1 + hi) * a
                l, d = (-r * a, -r * a) if r * a <= held else (-held, 0.0)
            loss[i], slope[i] = l, d
            loss_tol[i] = slope_off[i] = abs(d) * 2 * o
        if kl:
            b = float(ref[i]) - v
            e = math.exp(b) if math.isfinite(b) else (math.inf if b > 0 else math.nan)
            loss[i] += kl * (e - b - 1)
            slope[i] -= kl * (e - 1)
            if math.isfinite(e):
                loss_tol[i] += kl * abs(e - 1) * 2 * o + kl * o * o * e
                slope_off[i] += kl * e * 2 * o
        loss[i] *= wi
        slope[i] *= wi
        loss_tol[i] *= abs(wi)
        slope_off[i] = abs(wi) * slope_off[i] + 2 * U * abs(slope[i])
    loss_tol += U * loss.abs().nan_to_num(0, 0, 0) + 2.0 ** -149
    slope_off = slope_off.nan_to_num(0, 0, 0)
    return (loss, loss_tol), (lp, off), label_grad(rows, labels, slope, T, x.dtype, slope_off)


def preference(x, labels, offsets, ref, beta, soft, margin, average, T, w):
    lp, off, rows = logp(x, labels, T)
    bounds = offsets.tolist()
    half = (len(bounds) - 1) // 2
    seq, seq_off, count = [], [], []
    for a, b in zip(bounds, bounds[1:]):
        if not 0 <= a <= b <= rows.N:
            seq.append(math.nan), seq_off.append(0.0), count.append(1)
            continue
        n = max(1, int((labels[a:b] >= 0).sum())) if average else 1
        seq.append(float(lp[a:b].sum()) / n)
        seq_off.append(float(off[a:b].sum()) / n)
        count.append(n)
    loss, loss_tol = torch.zeros(half, dtype=torch.float64), torch.zeros(half, dtype=torch.float64)
    slope, slope_off = torch.zeros(rows.N, dtype=torch.float64), torch.zeros(rows.N, dtype=torch.float64)
    for p in range(half):
        wp = 1.0 if w is None else float(w[p])
        if wp == 0:
            if math.isnan(seq[p] + seq[half + p]) and not (0 <= bounds[p] <= bounds[p + 1] <= rows.N):
                loss[p] = math.nan
            continue
        h = beta * ((seq[p] - seq[half + p]) - (float(ref[p]) - float(ref[half + p]))) - margin
        o = beta * (seq_off[p] + seq_off[half + p])
        up = math.log1p(math.exp(-abs(h))) + max(-h, 0.0) if not math.isnan(h) else math.nan
        sig = 1 / (1 + math.exp(-h)) if h >= -700 else 0.0
        lose = 1 / (1 + math.exp(h)) if h <= 700 else 0.0
        if math.isnan(h):
            sig = lose = math.nan
        loss[p] = wp * (up + (soft * h if soft else 0.0))
        loss_tol[p] = abs(wp) * o
        dh = wp * beta * (soft * sig - (1 - soft) * lose)
        dh_off = abs(wp) * beta * min(0.25, 2 * sig * lose) * o if not math.isnan(h) else 0.0
        for k, sign in ((p, 1.0), (half + p, -1.0)):
            a, b = bounds[k], bounds[k + 1]
            if 0 <= a <= b <= rows.N:
                slope[a:b] = sign * dh / count[k]
                slope_off[a:b] = dh_off / count[k] + 2 * U * abs(dh) / count[k]
    loss_tol += U * loss.abs().nan_to_num(0, 0, 0) + 2.0 ** -149
    seq = torch.tensor(seq, dtype=torch.float64)
    seq_off = torch.tensor(seq_off, dtype=torch.float64) + U * seq.abs().nan_to_num(0, 0, 0)
    return (loss, loss_tol), (seq, seq_off), label_grad(rows, labels, slope, T, x.dtype, slope_off.nan_to_num(0, 0, 0))


def close(name, got, want, tol):
    """NaN where a NaN is due, the same infinities, everything else within its tolerance."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "%s: NaN at %s, due at %s" % (
        name, torch.isnan(got).nonzero()[:4].tolist(), torch.isnan(want).nonzero()[:4].tolist())
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and not torch.isinf(got[~inf]).any(), name
    some = torch.isfinite(want)
    over = (got - want).abs()[some] - tol.expand_as(want)[some]
    if over.numel() and over.max() > 0:
        k = int(over.argmax())
        raise AssertionError("%s: %r for %r, off by %.3g of %.3g allowed (%d values of %d)" % (
            name, got[some][k].item(), want[some][k].item(), (got - want).abs()[some][k], tol.expand_as(want)[some][k], int((over > 0).sum()), over.numel()))
