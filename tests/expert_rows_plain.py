"""Rows through experts in 64 bits on the CPU, row by row where that is plainer, with what the library's results may be off by.

A rounding to a type is off by at most half a step, eps / 2 relative to the value.  Single precision has u = 2^-24: a chain of n sums and products is off by at most
n u times the sum of its terms' sizes (1 % more for the squares, and the smallest normal numbers where a product is smaller)."""
import math

import numpy as np
import torch

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
U = 2.0 ** -24
TINY = 2.0 ** -120


def half_step(v, dtype):
    """Half a step of a type at v, its smallest numbers' steps included."""
    return v.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def close(name, got, want, tol):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, "%s: shape %s, not %s" % (name, tuple(got.shape), tuple(want.shape))
    same = (got == want) | (got.isnan() & want.isnan())
    off = (got - want).abs() > tol
    wrong = ~same & (off | got.isnan() | want.isnan() | got.isinf() | want.isinf())
    if wrong.any():
        at = tuple(int(v) for v in wrong.nonzero()[0])
        raise AssertionError("%s: %d of %d wrong, first at %s: got %r, want %r" % (name, int(wrong.sum()), wrong.numel(), at, float(got[at]), float(want[at])))


def route(scores, top, renormalize, temperature):
    """experts, weights, and the weights' tolerance."""
    x = scores.double()
    rows, classes = x.shape
    ids, w, tol = torch.full((rows, top), -1, dtype=torch.int32), torch.zeros(rows, top, dtype=torch.float64), torch.zeros(rows, top, dtype=torch.float64)
    for i in range(rows):
        values = x[i].tolist()
        order = sorted((c for c in range(classes) if values[c] != -math.inf), key=lambda c: (0 if values[c] != values[c] else 1, -values[c] if values[c] == values[c] else 0, c))
        chosen = order[:top]
        if not chosen:
            continue
        ids[i, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        m = values[chosen[0]]
        if m != m or m == math.inf:
            w[i, :len(chosen)] = math.nan
            continue
        d = (x[i] - m) / temperature
        share = d[chosen] if renormalize else d[order]
        e = share.exp()
        total = e.sum()
        # an exponent is off by 3 u of itself (difference, factor, product), its exponential by two steps
        each = 1.01 * (3 * U * share.abs() + 4 * U)
        of_sum = (e * each).sum() / total + 1.01 * U * (64 + 8)
        w[i, :len(chosen)] = d[chosen].exp() / total
        tol[i, :len(chosen)] = w[i, :len(chosen)] * (1.01 * (3 * U * d[chosen].abs() + 4 * U) + of_sum + 4 * U) + TINY
    return ids, w, tol


def route_grad(scores, ids, w, dw, renormalize, temperature):
    """The gradient and its tolerance."""
    x, w, dw = scores.double(), w.double(), dw.double()
    rows, classes = x.shape
    top = ids.shape[1]
    grad, size = torch.zeros_like(x), torch.zeros_like(x)
    for i in range(rows):
        has = ids[i] >= 0
        at = ids[i][has].long()
        if (at >= classes).any():
            grad[i] = math.nan
            continue
        wi, di = w[i][has], dw[i][has]
        m, m_size = (wi * di).sum(), (wi * di).abs().sum()
        if m != m:
            grad[i] = math.nan
            continue
        if renormalize:
            for j in range(len(at)):
                grad[i, at[j]] += wi[j] * (di[j] - m)
                size[i, at[j]] += (wi[j] * (di[j].abs() + m_size)).abs()
        else:
            z = x[i] / temperature
            d = z - z.max() if (z > -math.inf).any() else z
            q = torch.softmax(z, 0) if (z > -math.inf).any() else torch.zeros_like(z)
            grad[i] = -q * m
            # the exponent's 3 u, as of the choice, and the sum's
            size[i] = q * m_size * (1 + 0.2 * torch.where(q > 0, d.abs(), 0.0) + 0.2 * (q * torch.where(q > 0, d.abs(), 0.0)).sum())
            for j in range(len(at)):
                grad[i, at[j]] += wi[j] * di[j]
                size[i, at[j]] += (wi[j] * di[j]).abs()
    grad, size = grad / temperature, size / temperature
    # the mean's chain of `top`, a class's of up to `top` more, the exponentials' sum of 64 a lane over 64 lanes, and a few
    return grad, half_step(grad, scores.dtype) + 1.02 * U * (2 * top + 64 + 20) * size + TINY


def plan(ids, experts):
    """place, source, offsets as lists, by going through the entries."""
    flat = ids.reshape(-1).tolist()
    by = [[] for _ in range(experts)]
    for i, e in enumerate(flat):
        if 0 <= e < experts:
            by[e].append(i)
    place, source, offsets = [-1] * len(flat), [], [0]
    for entries in by:
        for i in entries:
            place[i] = len(source)
            source.append(i)
        offsets.append(len(source))
    return place, source + [-1] * (len(flat) - len(source)), offsets


M = (1 << 64) - 1


def splitmix(start, n):
    """Output n (from 0) of SplitMix64 (Steele, Lea, Flood 2014), in whole numbers."""
    z = (start + (n + 1) * 0x9E3779B97F4A7C15) & M
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
    return z ^ (z >> 31)


def threshold(p):
    return min(int(round(p * 2 ** 32)), 2 ** 32 - 1)


def bits(rows, features, seed, layer, first=0):
    """The 32 bits of every element of rows first to first + rows - 1."""
    key = splitmix(seed & M, layer)
    words = (features + 3) // 4

    def outputs(start):
        z = np.arange(first * words + 1, (first + rows) * words + 1, dtype=np.uint64)
        with np.errstate(over="ignore"):
            z = np.uint64(start) + z * np.uint64(0x9E3779B97F4A7C15)
            z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
            z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
            z = z ^ (z >> np.uint64(31))
        return z.astype("<u8").view("<u2").reshape(rows, 4 * words)[:, :features].astype(np.int64)

    return torch.from_numpy(outputs(key) << 16 | outputs(~key & M))


def dropped(v, p, seed, layer):
    """drop(v) of a matrix."""
    if not p:
        return v.double()
    t = threshold(p)
    return torch.where(bits(v.shape[0], v.shape[1], seed, layer) < t, 0.0, v.double() * (2.0 ** 32 / (2 ** 32 - t)))


def drop(x, p, seed, layer, residual):
    v = dropped(x, p, seed, layer)
    size = v.abs()
    if residual is not None:
        v = v + residual.double()
        size = size + residual.double().abs()
    return v, half_step(v, x.dtype) + 1.01 * U * 3 * size


def combine(y, place, w, residual, p, seed, layer):
    rows, top = place.shape
    v, size = torch.zeros(rows, y.shape[1], dtype=torch.float64), torch.zeros(rows, y.shape[1], dtype=torch.float64)
    for j in range(top):
        has = (place[:, j] >= 0).nonzero()[:, 0]
        part = y[place[has, j].long()].double() * (1.0 if w is None else w[has, j, None].double())
        v[has] += part
        size[has] += part.abs()
    v, size = dropped(v, p, seed, layer), dropped(size, p, seed, layer)
    if residual is not None:
        v = v + residual.double()
        size = size + residual.double().abs()
    return v, half_step(v, y.dtype) + 1.01 * U * (top + 4) * size.nan_to_num(0, 0, 0) + TINY


def combine_grad(dout, y, place, w, p, seed, layer):
    """(dy, tolerance), (dweights, tolerance)"""
    rows, top = place.shape
    d = dropped(dout, p, seed, layer)
    dy = torch.zeros(rows * top, dout.shape[1], dtype=torch.float64)
    dw, size = torch.zeros(rows, top, dtype=torch.float64), torch.zeros(rows, top, dtype=torch.float64)
    for j in range(top):
        has = (place[:, j] >= 0).nonzero()[:, 0]
        at = place[has, j].long()
        dy[at] = d[has] * (1.0 if w is None else w[has, j, None].double())
        if y is not None:
            dw[has, j] = (d[has] * y[at].double()).sum(1)
            size[has, j] = (d[has] * y[at].double()).abs().sum(1)
    # a thread's chain: a piece's 4 or 8 values, one piece in 64 of the row's, then a tree over 1024 threads
    chain = 8 + (dout.shape[1] + 255) // 256 + 12
    return (dy, half_step(dy, dout.dtype) + 1.01 * U * 3 * dy.abs() + TINY), (dw, 1.01 * U * (chain + 2) * size.nan_to_num(0, 0, 0) + TINY)
