"""Rows through experts, as cases that can be timed: the choice of each row's experts from its scores, rows sorted by expert and combined again with
weights, dropout from a counter-based generator, and the gradients of these.

A case is a dict of plain values.  "op" is the operator:

  route         the best experts of every row and their weights
  route_grad    the gradient of these weights by the scores
  sort          the tables that order rows by expert, and the rows in that order
  combine       every row's weighted sum of what its experts returned, with dropout and a residual
  combine_grad  the gradients of that by the experts' rows and by the weights
  drop          dropout of rows, and a residual added

"rows" rows (tokens, or training rows) of "features" values of type "dtype", "top" of "experts" experts each.  The last "pad" rows are a padded batch's
and have no expert.  With "masked" a tenth of the experts has -inf for a score, as one that is switched off.  `run` computes the plain form, or with
`own` calls this repository's package."""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOST = 32768 * 8 * 4096  # values of the experts' rows in the largest case
GAMMA, MIX1, MIX2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB  # SplitMix64


def _package():
    """This repository's package: its folder's name is no module name, so it is loaded from its path, as bench.py does."""
    name = "evotrees_jl_amd"
    if name in sys.modules:
        return sys.modules[name]
    folder = os.path.join(os.getcwd(), "evotrees.jl_amd")
    spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
    module = importlib.util.module_from_spec(spec)
    sys.modules[name] = module
    spec.loader.exec_module(module)
    return module


def _case(name, op, rows, dtype, **more):
    case = dict(name=name, op=op, rows=rows, dtype=dtype, experts=0, top=0, features=0, pad=0, masked=False, renormalize=True, temperature=1.0, p=0.0,
                layer=0, residual=False)
    case.update(more)
    return case


def listed():
    return [
        # one step of eight sequences that a service answers: the smallest choice
        _case("route_step", "route", 8, "bfloat16", experts=64, top=6),
        # a training batch's choice of 8 of 256 experts
        _case("route_batch", "route", 131072, "bfloat16", experts=256, top=8),
        # its backward pass where the weights are shares of all experts' probabilities, an odd number of them, some switched off
        _case("route_grad_odd", "route_grad", 50_021, "float32", experts=97, top=4, renormalize=False, masked=True, temperature=1.5),
        # the backward pass of a batch's choice, weights that sum to one
        _case("route_grad_batch", "route_grad", 131072, "bfloat16", experts=256, top=8),
        # the rows of one step to their experts
        _case("sort_step", "sort", 16, "bfloat16", experts=64, top=6, features=2048),
        # the rows of a training batch, the last of them padding
        _case("sort_batch", "sort", 32768, "bfloat16", experts=128, top=8, features=4096, pad=1000),
        # the step's way back: no dropout in service
        _case("combine_step", "combine", 16, "bfloat16", experts=64, top=6, features=2048, residual=True),
        # a training batch's, with dropout in front of the residual
        _case("combine_batch", "combine", 32768, "bfloat16", experts=128, top=8, features=4096, pad=1000, p=0.1, layer=3, residual=True),
        # rows of a table at the leaves of one tree: single precision, an odd number of leaves
        _case("combine_grad_leaves", "combine_grad", 200_003, "float32", experts=1023, top=1, features=100),
        # a training batch's backward pass
        _case("combine_grad_batch", "combine_grad", 32768, "bfloat16", experts=128, top=8, features=4096, pad=1000, p=0.1, layer=3),
        # a short sequence's rows, fine-tuned in half precision
        _case("drop_few", "drop", 64, "float16", features=4099, p=0.05, layer=1, residual=True),
        # a training batch's rows
        _case("drop_batch", "drop", 65536, "bfloat16", features=8192, p=0.1, layer=7, residual=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same kinds: 1 to 262 144 rows of 16 to 16 384 features, 2 to 1024 experts, up to a quarter of the largest listed case's values."""
    op = rng.choice(["route", "route_grad", "sort", "combine", "combine_grad", "drop"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    experts = _log_uniform(rng, 2, 1024)
    top = min(experts, rng.choice([1, 2, 2, 3, 4, 6, 8, 8, 12]))
    more = dict(layer=rng.randint(0, 100))
    if op in ("route", "route_grad"):
        rows = _log_uniform(rng, 1, min(262_144, (1 << 25) // experts))
        more.update(experts=experts, top=top, masked=rng.choice([False, False, True]), renormalize=rng.choice([True, True, False]),
                    temperature=rng.choice([1.0, 1.0, 0.5]))
    elif op == "drop":
        features = _log_uniform(rng, 16, 16384)
        rows = _log_uniform(rng, 1, min(262_144, (1 << 27) // features))
        more.update(features=features, p=rng.choice([0.05, 0.1, 0.25, 0.5]), residual=rng.choice([False, True]))
    else:
        features = _log_uniform(rng, 16, 16384)
        rows = _log_uniform(rng, 1, min(262_144, MOST // 4 // (features * top)))
        more.update(experts=experts, top=top, features=features, pad=rng.choice([0, rng.randint(0, rows // 4)]))
        if op != "sort":
            more["p"] = rng.choice([0.0, 0.1])
        if op == "combine":
            more["residual"] = rng.choice([False, True])
    case = _case("", op, rows, dtype, **more)
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------

def prepare(case, seed):
    rows, experts, top, features, dtype = case["rows"], case["experts"], case["top"], case["features"], TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        out = torch.empty(shape, dtype=dtype, device="cuda")
        step = max(1, (1 << 27) // max(1, shape[1]))
        for a in range(0, shape[0], step):
            part = out[a:a + step]
            part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * scale)
        return out

    state = dict(case=case, pkg=_package() if own else None)
    # one of an optimizer step's draws; a training program keeps it on the device
    state["seed"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=gen, device="cuda")
    if case["op"] in ("route", "route_grad"):
        x = normal(rows, experts, scale=2.0)
        if case["masked"]:
            x[:, 1:][:, torch.rand(experts - 1, generator=gen, device="cuda") < 0.1] = -math.inf
        state["scores"] = x
        if case["op"] == "route_grad":
            state["experts"], state["weights"] = _plain_route(case, x)
            state["dweights"] = torch.randn(rows, top, generator=gen, device="cuda")
        return state
    if case["op"] == "drop":
        state["x"] = normal(rows, features)
        state["residual"] = normal(rows, features) if case["residual"] else None
        return state
    # distinct experts a row, the first ones far more often than the last
    first = (torch.rand(rows, 1, generator=gen, device="cuda") ** 2 * experts).long().clamp(max=experts - 1)
    step = 1 + (torch.rand(rows, 1, generator=gen, device="cuda") * (experts // top)).long().clamp(max=experts // top - 1)
    chosen = (first + torch.arange(top, device="cuda") * step) % experts
    if case["pad"]:
        chosen[rows - case["pad"]:] = -1
    state["experts"] = chosen.int()
    if case["op"] == "sort":
        state["x"] = normal(rows, features)
        return state
    state["place"] = _plain_plan(case, state["experts"])[0]
    if own:  # made when the rows were sorted
        state["plan"] = state["pkg"].plan_rows(state["experts"], experts)
    state["weights"] = torch.softmax(torch.randn(rows, top, generator=gen, device="cuda"), 1)
    state["y"] = normal(rows * top, features)
    if case["op"] == "combine":
        state["residual"] = normal(rows, features) if case["residual"] else None
    else:
        state["dout"] = normal(rows, features)
    return state


# ---- plain forms ----------------------------------------------------------------------------

def _signed(v):
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def _mixed(z):
    """SplitMix64's output for the states z, int64 in place of its unsigned words: products wrap alike, shifts have their upper bits cleared."""
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * _signed(MIX1)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * _signed(MIX2)
    return z ^ ((z >> 31) & ((1 << 33) - 1))


def _threshold(p):
    return int(round(p * 2 ** 32))


def _plain_kept(case, seed):
    """Which of the values stay: element (r, c) has the 16 bits c % 4 of word r ceil(features / 4) + c // 4 of SplitMix64 started at key as the upper half of
    a number of 32, and those of SplitMix64 started at ~key as the lower.  key: output `layer` of SplitMix64 started at the seed."""
    rows, features = case["rows"], case["features"]
    words = (features + 3) // 4
    key = _mixed(seed + _signed((case["layer"] + 1) * GAMMA))
    step = (torch.arange(rows * words, device=seed.device) + 1) * _signed(GAMMA)
    high, low = _mixed(step + key).view(rows, words), _mixed(step + ~key).view(rows, words)
    kept = torch.empty((rows, words, 4), dtype=torch.bool, device=seed.device)
    for j in range(4):
        kept[:, :, j] = ((high >> (16 * j)) & 0xFFFF) * 65536 + ((low >> (16 * j)) & 0xFFFF) >= _threshold(case["p"])
    return kept.view(rows, 4 * words)[:, :features]


def _plain_drop(case, seed, x):
    if not case["p"]:
        return x
    return torch.where(_plain_kept(case, seed), x * (2.0 ** 32 / (2.0 ** 32 - _threshold(case["p"]))), 0.0)


def _plain_route(case, x):
    top, experts = case["top"], x.shape[1]
    x = x.float()
    left, number = x.clone(), torch.arange(experts, device=x.device)
    ids, best = [], []
    for _ in range(top):
        most = left.amax(1, keepdim=True)
        at = torch.where(left == most, number, experts).amin(1, keepdim=True)
        left.scatter_(1, at, -math.inf)
        ids.append(torch.where(most > -math.inf, at, -1))
        best.append(most)
    ids, best = torch.cat(ids, 1), torch.cat(best, 1)
    e = torch.exp((best - best[:, :1]) / case["temperature"])
    total = e.sum(1, keepdim=True) if case["renormalize"] else torch.exp((x - best[:, :1]) / case["temperature"]).sum(1, keepdim=True)
    return ids.int(), torch.where(ids >= 0, e / total, 0.0)


def _plain_plan(case, experts):
    ids = experts.reshape(-1).long()
    n = ids.numel()
    order = torch.argsort(torch.where(ids < 0, case["experts"], ids), stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(n, device=ids.device)
    count = (ids >= 0).sum()
    place = torch.where(ids < 0, -1, position).view(experts.shape).int()
    source = torch.where(torch.arange(n, device=ids.device) < count, order, -1).int()
    bounds = torch.zeros(case["experts"] + 1, dtype=torch.int64, device=ids.device)
    bounds[1:] = torch.zeros(case["experts"] + 1, dtype=torch.int64, device=ids.device).scatter_add_(
        0, torch.where(ids < 0, case["experts"], ids), torch.ones_like(ids))[:-1].cumsum(0)
    return place, source, bounds.int()


def _run_own(state):
    case, pkg = state["case"], state["pkg"]
    if case["op"] == "route":
        return pkg.route_rows(state["scores"], case["top"], renormalize=case["renormalize"], temperature=case["temperature"])
    if case["op"] == "route_grad":
        return pkg.route_rows_grad(state["scores"], state["experts"], state["weights"], state["dweights"], renormalize=case["renormalize"],
                                   temperature=case["temperature"])
    if case["op"] == "sort":
        plan = pkg.plan_rows(state["experts"], case["experts"])
        return plan.place, plan.source, plan.offsets, pkg.sort_rows(state["x"], plan)
    if case["op"] == "combine":
        return pkg.combine_rows(state["y"], state["plan"], state["weights"], residual=state["residual"], p=case["p"], seed=state["seed"], layer=case["layer"])
    if case["op"] == "combine_grad":
        return pkg.combine_rows_grad(state["dout"], state["y"], state["plan"], state["weights"], p=case["p"], seed=state["seed"], layer=case["layer"])
    return pkg.drop_rows(state["x"], case["p"], state["seed"], layer=case["layer"], residual=state["residual"])


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    rows, top = case["rows"], case["top"]
    if case["op"] == "route":
        return _plain_route(case, state["scores"])
    if case["op"] == "route_grad":
        x, ids, w, dw = state["scores"].float(), state["experts"].long(), state["weights"], state["dweights"]
        valid = ids >= 0
        own_part = torch.where(valid, w * dw, 0.0)
        mean = own_part.sum(1, keepdim=True)
        if case["renormalize"]:
            grad = torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0), own_part - torch.where(valid, w * mean, 0.0))
        else:
            e = torch.exp((x - x.amax(1, keepdim=True)) / case["temperature"])
            grad = (e / e.sum(1, keepdim=True) * -mean).scatter_add_(1, ids.clamp(min=0), own_part)
        return (grad / case["temperature"]).to(state["scores"].dtype)
    if case["op"] == "sort":
        place, source, bounds = _plain_plan(case, state["experts"])
        out = torch.where((source >= 0)[:, None], state["x"][(source.long() // top).clamp(min=0)], 0.0)
        return place, source, bounds, out
    if case["op"] == "drop":
        out = _plain_drop(case, state["seed"], state["x"].float())
        if case["residual"]:
            out = out + state["residual"].float()
        return out.to(state["x"].dtype)
    place, y, w = state["place"].long(), state["y"], state["weights"]
    valid = place >= 0
    at = place.clamp(min=0)
    if case["op"] == "combine":
        out = torch.zeros((rows, case["features"]), device=y.device)
        for j in range(top):
            out += torch.where(valid[:, j, None], w[:, j, None] * y[at[:, j]].float(), 0.0)
        out = _plain_drop(case, state["seed"], out)
        if case["residual"]:
            out = out + state["residual"].float()
        return out.to(y.dtype)
    d = _plain_drop(case, state["seed"], state["dout"].float())
    dy, dw = y.new_zeros((rows * top + 1, case["features"])), torch.zeros_like(w)
    for j in range(top):  # what has no place goes to a row behind the last
        dy[torch.where(valid[:, j], at[:, j], rows * top)] = (w[:, j, None] * d).to(y.dtype)
        dw[:, j] = torch.where(valid[:, j], (d * y[at[:, j]].float()).sum(1), 0.0)
    return dy[:-1], dw


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    """Bytes: inputs read once, outputs written once, experts' rows that nobody has neither.  Operations: a score's comparison and the exponential's three,
    a product and a sum for each value of an expert's row, four for each 64 random bits' value and two for one that dropout scales."""
    rows, top, features, op = case["rows"], case["top"], case["features"], case["op"]
    size = 4 if case["dtype"] == "float32" else 2
    if op == "route":
        return {"bytes": rows * case["experts"] * size + 8 * rows * top, "flops": rows * case["experts"] * (1 if case["renormalize"] else 4)}
    if op == "route_grad":
        read = 0 if case["renormalize"] else rows * case["experts"] * size
        return {"bytes": read + rows * case["experts"] * size + 12 * rows * top, "flops": rows * top * 4 + (0 if case["renormalize"] else rows * case["experts"] * 4)}
    whole, mask = rows * features * size, (6 if case["p"] else 0) * rows * features
    if op == "drop":
        return {"bytes": whole * (3 if case["residual"] else 2), "flops": mask + rows * features}
    used = (rows - case["pad"]) * top
    if op == "sort":
        return {"bytes": (rows - case["pad"]) * features * size + rows * top * features * size + 12 * rows * top + 4 * case["experts"], "flops": rows * top}
    if op == "combine":
        return {"bytes": used * features * size + whole * (2 if case["residual"] else 1) + 8 * rows * top, "flops": mask + 2 * used * features}
    return {"bytes": used * features * size + rows * top * features * size + (rows - case["pad"]) * features * size + 12 * rows * top,
            "flops": mask + 3 * used * features}


# ---- the definition in 64 bits ------------------------------------------------------------------

def _exact_kept(case, seed):
    rows, features = case["rows"], case["features"]
    with np.errstate(over="ignore"):
        def words(start, first, n):
            z = np.arange(first + 1, first + n + 1, dtype=np.uint64)
            z *= np.uint64(GAMMA)
            z += start
            for shift, factor in ((30, MIX1), (27, MIX2)):
                z ^= z >> np.uint64(shift)
                z *= np.uint64(factor)
            z ^= z >> np.uint64(31)
            return z

        key = words(np.uint64(seed), case["layer"], 1)[0]
        n = (features + 3) // 4
        kept = np.empty((rows, features), dtype=bool)
        step = max(1, (1 << 22) // n)
        for a in range(0, rows, step):
            b = min(rows, a + step)
            halves = [words(start, a * n, (b - a) * n).view(np.uint16).reshape(b - a, 4 * n)[:, :features] for start in (key, ~key)]
            kept[a:b] = halves[0].astype(np.uint32) * np.uint32(65536) + halves[1] >= np.uint32(_threshold(case["p"]))
    return torch.from_numpy(kept).cuda()


def exact(case, seed):
    state = prepare(case, seed)
    op, rows, top = case["op"], case["rows"], case["top"]
    if op in ("route", "route_grad"):
        x = state["scores"].double()
        q = torch.softmax(x / case["temperature"], 1)
        if op == "route":
            order = torch.sort(x, dim=1, descending=True, stable=True)
            ids = order.indices[:, :top]
            chosen = order.values[:, :top]
            w = torch.softmax(chosen / case["temperature"], 1) if case["renormalize"] else q.gather(1, ids)
            return torch.where(chosen == -math.inf, -1, ids).int(), torch.where(chosen == -math.inf, 0.0, w)
        ids, w, dw = state["experts"].long(), state["weights"].double(), state["dweights"].double()
        share = torch.zeros_like(x)
        slope = torch.zeros_like(x)
        for j in range(top):  # no expert twice in a row
            has = (ids[:, j] >= 0).nonzero()[:, 0]
            share[has, ids[has, j]] = w[has, j]
            slope[has, ids[has, j]] = dw[has, j]
        mean = (share * slope).sum(1, keepdim=True)
        if case["renormalize"]:
            return share * (slope - mean) / case["temperature"]
        return (share * slope - q * mean) / case["temperature"]
    if op == "drop":
        out = state["x"].double()
        out *= _exact_kept(case, state["seed"].cpu().numpy().view(np.uint64)[0])
        out /= 1.0 - _threshold(case["p"]) / 2 ** 32
        return out + state["residual"].double() if case["residual"] else out
    chosen = state["experts"].cpu().numpy().reshape(-1).astype(np.int64)
    n = chosen.size
    live = np.nonzero(chosen >= 0)[0]
    order = np.sort(chosen[live] * n + live) % n  # ascending by expert, then by place in the batch
    place = np.full(n, -1, dtype=np.int32)
    place[order] = np.arange(order.size)
    if op == "sort":
        source = np.full(n, -1, dtype=np.int32)
        source[:order.size] = order
        bounds = np.searchsorted(np.sort(chosen[live]), np.arange(case["experts"] + 1)).astype(np.int32)
        out = torch.zeros((n, case["features"]), dtype=torch.float64, device="cuda")
        out[:order.size] = state["x"].double()[torch.from_numpy(order // top).cuda()]
        return torch.from_numpy(place).cuda().view(rows, top), torch.from_numpy(source).cuda(), torch.from_numpy(bounds).cuda(), out
    place = torch.from_numpy(place).cuda().view(rows, top).long()
    w = state["weights"].double()
    scale = 1.0
    if case["p"]:
        scale = _exact_kept(case, state["seed"].cpu().numpy().view(np.uint64)[0]).double() / (1.0 - _threshold(case["p"]) / 2 ** 32)
    if op == "combine":
        out = torch.zeros((rows, case["features"]), dtype=torch.float64, device="cuda")
        for j in range(top):
            has = (place[:, j] >= 0).nonzero()[:, 0]
            out[has] += w[has, j, None] * state["y"][place[has, j]].double()
        out = out * scale
        return out + state["residual"].double() if case["residual"] else out
    d = state["dout"].double() * scale
    dy = torch.zeros((n, case["features"]), dtype=torch.float64, device="cuda")
    dw = torch.zeros_like(w)
    for j in range(top):
        has = (place[:, j] >= 0).nonzero()[:, 0]
        dy[place[has, j]] = w[has, j, None] * d[has]
        dw[has, j] = (d[has] * state["y"][place[has, j]].double()).sum(1)
    return dy, dw
