"""The losses over rows of class scores, with their gradients, as cases that can be timed: log-probabilities of chosen classes, distillation
from a teacher's top logits, the preference loss of paired sequences and the clipped policy loss.

A case is a dict of plain values.  "op" is the operator:

  logp         log-probabilities of the rows' labels (scoring with a reference model), and each row's maximum and sum of exponentials
  logp_grad    the gradient of these, from what the forward call kept
  distill      loss and gradient against the top logits of a teacher
  preference   loss of every pair, log-probabilities of the sequences, gradient
  policy       loss and log-probability of every token, gradient

"rows" tokens (or training rows) of "classes" scores of type "dtype".  Rows without a label, of weight zero or behind the last
sequence are among them as in a padded batch, and with "masked" a tenth of the classes has -inf for a score, as constrained decoding leaves it.
`run` computes the plain form, or with `own` calls this repository's package."""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOST = 8192 * 131072  # scores of the largest case


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


def _case(name, op, rows, classes, dtype, **more):
    case = dict(name=name, op=op, rows=rows, classes=classes, dtype=dtype, temperature=1.0, masked=False, top=0, pairs=0, pad=0, average=False,
                smoothing=0.0, kl=0.0)
    case.update(more)
    return case


def listed():
    return [
        # one step of eight sequences scored by a service: the smallest call there is
        _case("logp_step", "logp", 8, 32768, "bfloat16"),
        # a batch scored by the reference model before training
        _case("logp_batch", "logp", 8192, 131072, "bfloat16"),
        # the rows of a multi-class model's validation set
        _case("logp_seven_classes", "logp", 200_003, 7, "float32"),
        # the backward pass of a summed log-probability, an odd number of classes
        _case("logp_grad_odd", "logp_grad", 4096, 50_021, "bfloat16"),
        # a few tokens distilled in half precision
        _case("distill_few", "distill", 4, 32768, "float16", top=16, temperature=2.0),
        # a training batch against the 64 best logits a teacher stored for each token
        _case("distill_batch", "distill", 8192, 131072, "bfloat16", top=64),
        # a teacher's three best classes as the target of a seven-class model of a million rows
        _case("distill_seven_classes", "distill", 1_000_000, 7, "float32", top=3, temperature=1.5),
        # eight pairs of answers of different lengths
        _case("preference_batch", "preference", 5003, 32768, "bfloat16", pairs=8, pad=17),
        # one pair, single precision, scores of an odd number of classes, some of them masked
        _case("preference_pair", "preference", 700, 100_003, "float32", pairs=1, masked=True, average=True, smoothing=0.1),
        # the tokens of sixteen answers, one each: a first step, latency counts
        _case("policy_few", "policy", 16, 32768, "bfloat16", kl=0.05),
        # a step over sampled answers, with the KL term
        _case("policy_batch", "policy", 8192, 131072, "bfloat16", kl=0.05),
        # a smaller vocabulary of odd size in single precision, sampled at a temperature, some classes masked
        _case("policy_odd", "policy", 12_007, 1999, "float32", temperature=0.7, masked=True, kl=0.02),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same kinds: 2 to 131072 classes, 1 to a million rows, up to half as many scores as the largest listed case has."""
    op = rng.choice(["logp", "logp_grad", "distill", "distill", "preference", "preference", "policy", "policy"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    classes = _log_uniform(rng, 2, 131072)
    most = MOST // (4 if dtype == "float32" else 2)
    rows = _log_uniform(rng, 1, min(1_000_000, most // classes))
    more = dict(temperature=rng.choice([1.0, 1.0, 0.7, 2.0]), masked=rng.choice([False, False, True]) and classes >= 16)
    if op == "distill":
        more["top"] = _log_uniform(rng, 1, min(classes, 128))
    elif op == "preference":
        rows = max(2, min(rows, 60_000))
        more["pairs"] = _log_uniform(rng, 1, max(1, min(rows // 2, 256)))
        more["pad"] = rng.randint(0, min(40, rows - 2 * more["pairs"]))
        more["average"] = rng.choice([False, True])
        more["smoothing"] = rng.choice([0.0, 0.1])
    elif op == "policy":
        more["kl"] = rng.choice([0.0, 0.05])
    case = _case("", op, rows, classes, dtype, **more)
    del case["name"]
    return case


def _lengths(case):
    """Lengths of the case's sequences, the chosen ones first: at least one row each, all rows but `pad`."""
    rng = random.Random(case["rows"] * 1009 + case["pairs"])
    n = 2 * case["pairs"]
    share = [rng.uniform(0.2, 1.0) for _ in range(n)]
    free = case["rows"] - case["pad"] - n
    lengths = [1 + int(free * v / sum(share)) for v in share]
    lengths[-1] += case["rows"] - case["pad"] - sum(lengths)
    return lengths


def _chunks(case, limit=1 << 27):
    step = max(1, limit // case["classes"])
    return [(a, min(case["rows"], a + step)) for a in range(0, case["rows"], step)]


def _logp32(case, x, labels):
    """Log-probabilities of the labels as an earlier model of the program would have found them, in pieces."""
    out = torch.zeros(case["rows"], device="cuda")
    for a, b in _chunks(case):
        z = torch.log_softmax(x[a:b].float() / case["temperature"], 1)
        out[a:b] = z.gather(1, labels[a:b].clamp(min=0)[:, None])[:, 0]
    return out


def prepare(case, seed):
    rows, classes = case["rows"], case["classes"]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device="cuda")

    x = torch.empty((rows, classes), dtype=TYPES[case["dtype"]], device="cuda")
    hidden = uniform(classes) < 0.1 if case["masked"] else None
    for a, b in _chunks(case):
        z = normal(b - a, classes) * 2.0
        if hidden is not None:
            z[:, hidden] = -math.inf
        x[a:b] = z
    state = dict(case=case, logits=x, pkg=_package() if own else None)
    if case["op"] == "distill":
        top = case["top"]
        first = torch.randint(0, classes, (rows, 1), generator=gen, device="cuda")
        step = 1 + (uniform(rows, 1) * (classes // top)).long().clamp(max=classes // top - 1)
        rank = torch.arange(top, device="cuda")
        ids = (first + rank * step) % classes  # no class twice in a row
        x.scatter_(1, ids, (5.0 - 0.1 * rank + normal(rows, top)).to(x.dtype))
        state["top_logits"] = (8.0 - 0.3 * rank + 0.3 * normal(rows, top)).contiguous()
        if top > 1:  # teachers that stored fewer
            ids = torch.where((rank >= (top + 1) // 2) & (uniform(rows, 1) < 0.1), -1, ids)
        state["top_ids"] = ids.to(torch.int32)
        state["weights"] = torch.where(uniform(rows) < 0.05, 0.0, 0.5 + uniform(rows))
        return state
    labels = torch.randint(0, classes, (rows,), generator=gen, device="cuda")
    x.scatter_(1, labels[:, None], (6.0 + 2.0 * normal(rows, 1)).to(x.dtype))
    if case["op"] in ("logp", "logp_grad"):
        state["labels"] = torch.where(uniform(rows) < 0.05, -100, labels)
        if case["op"] == "logp_grad":
            state["dlogp"] = normal(rows)
            if own:  # the forward pass has been made
                state["stats"] = state["pkg"].class_logp(x, state["labels"], temperature=case["temperature"])[1]
        return state
    if case["op"] == "preference":
        lengths = _lengths(case)
        bounds = [0]
        for n in lengths:
            labels[bounds[-1]:bounds[-1] + n // 4] = -100  # the question
            bounds.append(bounds[-1] + n)
        state["labels"] = labels
        state["offsets"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        logp = torch.where(labels < 0, 0.0, _logp32(case, x, labels)).double()
        total = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), logp.cumsum(0)])
        sums = total[bounds[1:]] - total[bounds[:-1]]
        if case["average"]:
            sums = sums / torch.tensor([n - n // 4 for n in lengths], device="cuda")
        state["ref_logp"] = (sums + normal(len(lengths)) * (0.3 if case["average"] else 8.0)).float()
        state["weights"] = 0.5 + uniform(case["pairs"])
        state["beta"] = 2.0 if case["average"] else 0.1
        return state
    logp = _logp32(case, x, labels)
    state["labels"] = labels
    state["old_logp"] = logp + 0.15 * normal(rows)
    state["ref_logp"] = logp + 0.3 * normal(rows) if case["kl"] else None
    state["advantages"] = torch.where(uniform(rows) < 0.1, 0.0, normal(rows))
    state["weights"] = torch.where(uniform(rows) < 0.1, 0.0, 0.5 + uniform(rows))
    return state


def _run_own(state):
    case, pkg, x = state["case"], state["pkg"], state["logits"]
    temperature = case["temperature"]
    if case["op"] == "logp":
        return pkg.class_logp(x, state["labels"], temperature=temperature)
    if case["op"] == "logp_grad":
        return pkg.class_logp_grad(x, state["labels"], state["stats"], state["dlogp"], temperature=temperature)
    if case["op"] == "distill":
        return pkg.distill_loss(x, state["top_ids"], state["top_logits"], temperature=temperature, weights=state["weights"])
    if case["op"] == "preference":
        return pkg.preference_loss(x, state["labels"], state["offsets"], state["ref_logp"], beta=state["beta"], label_smoothing=case["smoothing"],
                                   average=case["average"], temperature=temperature, weights=state["weights"])
    return pkg.policy_loss(x, state["labels"], state["old_logp"], state["advantages"], ref_logp=state["ref_logp"], clip_low=0.2, clip_high=0.28,
                           kl_coef=case["kl"], temperature=temperature, weights=state["weights"])


def run(state):
    if own:
        return _run_own(state)
    case, x = state["case"], state["logits"]
    temperature = case["temperature"]
    most = x.float().amax(1, keepdim=True)
    d = (x.float() - most) / temperature
    e = d.exp()
    total = e.sum(1, keepdim=True)
    if case["op"] == "distill":
        ids, w = state["top_ids"].long(), state["weights"][:, None]
        valid = ids >= 0
        at = ids.clamp(min=0)
        t = torch.where(valid, state["top_logits"] / temperature, -math.inf)
        t = t - t.amax(1, keepdim=True)
        te = t.exp()
        ts = te.sum(1, keepdim=True)
        p = te / ts
        gap = torch.where(valid, (t - ts.log()) - (d.gather(1, at) - total.log()), 0.0)
        loss = (w * temperature * temperature * p * gap).sum(1)
        grad = (e / total).scatter_add_(1, at, -p)
        return loss, (grad * (w * temperature)).to(x.dtype)
    labels = state["labels"]
    live = labels >= 0
    at = labels.clamp(min=0)[:, None]
    logp = torch.where(live, (d.gather(1, at) - total.log())[:, 0], 0.0)
    if case["op"] == "logp":
        return logp, torch.where(live[:, None], torch.cat([most, total], 1), 0.0)
    if case["op"] == "logp_grad":
        slope = state["dlogp"]
    elif case["op"] == "preference":
        bounds = state["offsets"].long()
        n = bounds.numel() - 1
        sums = torch.cat([torch.zeros(1, dtype=torch.float64, device=x.device), logp.double().cumsum(0)])[bounds]
        seq = sums[1:] - sums[:-1]
        scale = torch.ones(n, dtype=torch.float64, device=x.device)
        if case["average"]:
            count = torch.cat([torch.zeros(1, dtype=torch.int64, device=x.device), live.long().cumsum(0)])[bounds]
            scale = 1.0 / (count[1:] - count[:-1]).clamp(min=1).double()
        seq = seq * scale
        half = n // 2
        ratio = seq - state["ref_logp"].double()
        h = state["beta"] * (ratio[:half] - ratio[half:])
        soft, w = case["smoothing"], state["weights"].double()
        up = torch.log1p(torch.exp(-h.abs())) + torch.relu(-h)  # -log sigmoid(h)
        loss = (w * ((1.0 - soft) * up + soft * (up + h))).float()
        dh = w * (1.0 / (1.0 + torch.exp(-h)) - 1.0 + soft) * state["beta"]
        each = (torch.cat([dh, -dh]) * scale).float()
        place = torch.searchsorted(bounds, torch.arange(x.shape[0], device=x.device), right=True) - 1
        slope = torch.where((place >= 0) & (place < n), each[place.clamp(0, n - 1)], 0.0)
        logp = seq.float()
    else:
        ratio = (logp.double() - state["old_logp"].double()).exp()  # next to a border of the clipping
        a, w = state["advantages"].double(), state["weights"].double()
        free, held = ratio * a, ratio.clamp(0.8, 1.28) * a
        loss = -torch.minimum(free, held)
        slope = torch.where(free <= held, -free, 0.0)
        if case["kl"]:
            back = state["ref_logp"].double() - logp.double()
            loss = loss + case["kl"] * (back.exp() - back - 1.0)
            slope = slope + case["kl"] * (1.0 - back.exp())
        loss = (w * loss).float()
        slope = (w * slope).float()
    slope = torch.where(live, slope / temperature, 0.0)[:, None]
    grad = (e / total) * -slope
    grad.scatter_add_(1, at, slope)
    grad = grad.to(x.dtype)
    if case["op"] == "logp_grad":
        return grad
    return loss, logp, grad


def _bytes(case):
    """Scores of the rows that count are read once and every gradient is written once, and the rows' own values."""
    rows, classes = case["rows"], case["classes"]
    size = 4 if case["dtype"] == "float32" else 2
    live = {"logp": 0.95, "logp_grad": 0.95, "distill": 0.95, "policy": 0.9, "preference": 1.0}[case["op"]] * rows
    if case["op"] == "preference":
        live = sum(n - n // 4 for n in _lengths(case))
    each = {"logp": 20, "logp_grad": 20, "distill": 8 + 8 * case["top"], "preference": 8, "policy": 28 + (4 if case["kl"] else 0)}[case["op"]]
    out = 0 if case["op"] == "logp" else rows * classes * size
    return live, live * classes * size + out + rows * each


def work(case):
    """Operations: a difference, a product, an exponential and a sum for each score, and a second exponential's three for each gradient."""
    live, moved = _bytes(case)
    return {"bytes": moved, "flops": live * case["classes"] * (4 if case["op"] == "logp" else 3 if case["op"] == "logp_grad" else 7)}


def exact(case, seed):
    state = prepare(case, seed)
    x, rows = state["logits"], case["rows"]
    beta = 1.0 / case["temperature"]
    grad = None if case["op"] == "logp" else torch.empty((rows, case["classes"]), dtype=torch.float64, device="cuda")

    def log_q(a, b):
        return torch.log_softmax(x[a:b].double() * beta, 1)

    if case["op"] == "distill":
        loss = torch.empty(rows, dtype=torch.float64, device="cuda")
        for a, b in _chunks(case, 1 << 26):
            lq = log_q(a, b)
            ids = state["top_ids"][a:b].long()
            scores = (state["top_logits"][a:b].double() * beta).masked_fill(ids < 0, -math.inf)
            lp = torch.log_softmax(scores, 1)
            ids = ids.clamp(min=0)
            p = lp.exp()
            w = state["weights"][a:b].double()
            kl = torch.where(p > 0, p * (lp - lq.gather(1, ids)), 0.0)
            loss[a:b] = w / beta ** 2 * kl.sum(1)
            target = torch.zeros_like(lq).scatter_add_(1, ids, p)
            grad[a:b] = (w / beta)[:, None] * (lq.exp() - target)
        return loss, grad
    labels = state["labels"]
    index = torch.arange(rows, device="cuda")
    logp = torch.empty(rows, dtype=torch.float64, device="cuda")
    stats = torch.zeros((rows, 2), dtype=torch.float64, device="cuda")
    for a, b in _chunks(case, 1 << 26):
        lq = log_q(a, b)
        if grad is None:  # the greatest probability is one over the sum of exponentials
            stats[a:b, 0] = x[a:b].double().amax(1)
            stats[a:b, 1] = torch.exp(-lq.amax(1))
        logp[a:b] = lq[index[:b - a], labels[a:b].clamp(min=0)]
        if grad is not None:
            grad[a:b] = lq.exp_()
    logp[labels < 0] = 0.0
    if case["op"] == "logp":
        stats[labels < 0] = 0.0
        return logp, stats
    if case["op"] == "logp_grad":
        slope = state["dlogp"].double()
    elif case["op"] == "preference":
        bounds = state["offsets"].tolist()
        pairs = case["pairs"]
        value, length = [], []
        for a, b in zip(bounds, bounds[1:]):
            length.append(max(1, int((labels[a:b] >= 0).sum())) if case["average"] else 1)
            value.append(logp[a:b].sum().item() / length[-1])
        ref, w = state["ref_logp"].tolist(), state["weights"].tolist()
        loss, slope = [], torch.zeros(rows, dtype=torch.float64, device="cuda")
        for i in range(pairs):
            h = state["beta"] * ((value[i] - value[pairs + i]) - (ref[i] - ref[pairs + i]))
            win = 1.0 / (1.0 + math.exp(-h)) if h >= 0 else math.exp(h) / (1.0 + math.exp(h))
            lose = 1.0 / (1.0 + math.exp(h)) if h < 0 else math.exp(-h) / (1.0 + math.exp(-h))
            log_win = -math.log1p(math.exp(-h)) if h >= 0 else h - math.log1p(math.exp(h))
            loss.append(w[i] * (-(1.0 - case["smoothing"]) * log_win - case["smoothing"] * (log_win - h)))
            dh = w[i] * state["beta"] * (case["smoothing"] * win - (1.0 - case["smoothing"]) * lose)
            slope[bounds[i]:bounds[i + 1]] = dh / length[i]
            slope[bounds[pairs + i]:bounds[pairs + i + 1]] = -dh / length[pairs + i]
        loss = torch.tensor(loss, dtype=torch.float64, device="cuda")
        logp = torch.tensor(value, dtype=torch.float64, device="cuda")
    else:
        w, adv = state["weights"].double(), state["advantages"].double()
        r = torch.exp(logp - state["old_logp"].double())
        clipped = ((r > 1.28) & (adv > 0)) | ((r < 0.8) & (adv < 0))
        kept = torch.where(clipped, torch.where(adv > 0, 1.28, 0.8).double(), r)
        loss = -kept * adv
        slope = torch.where(clipped, 0.0, -r * adv)
        if case["kl"]:
            delta = state["ref_logp"].double() - logp
            loss = loss + case["kl"] * (torch.expm1(delta) - delta)
            slope = slope - case["kl"] * torch.expm1(delta)
        loss, slope = w * loss, w * slope
    slope = (slope * beta).masked_fill(labels < 0, 0.0)
    grad.mul_(-slope[:, None])
    grad[index, labels.clamp(min=0)] += slope
    if case["op"] == "logp_grad":
        return grad
    return loss, logp, grad
