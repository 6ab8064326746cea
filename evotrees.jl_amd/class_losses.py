"""Losses over rows of class scores with their gradients, on torch tensors in device memory: log-probabilities of chosen classes, distillation
from a teacher's top scores, the clipped policy loss and the preference loss of paired sequences (the C entry points evt_class_logp,
evt_class_logp_grad, evt_distill_loss, evt_policy_loss and evt_preference_loss; include/evotrees_hip.h has the formulas).

They stand beside the multi-class log loss that EvoTreeClassifier is fitted with (mlogloss_grad_hess, src/loss.jl:93-98, :113-128) for models of any number of
classes, a language model's vocabulary as well as a classifier's levels, and have no counterpart in the reference.

Scores are a (rows, classes) tensor of float32, bfloat16 or float16 whose classes lie side by side (`scores.stride(1) == 1`); rows may be
any distance apart.  Labels and class ids count from 0 and are int32 or int64; a negative one stands for none.  Values that
belong to a row, an entry or a pair are contiguous float32.  Temperatures are from 1e-4 to 1e4.  All tensors of a call are on one GPU; the work is queued on that GPU's current
stream and nothing waits for it.  As the gradients of this package's other losses, these are returned, not recorded: results never require a
gradient, also where the scores do, so that a loss added to a recorded one has no part in its backward pass.  The returned gradient goes on from there
(`logits.backward(grad)`), and a loss's weights stand in for what a chain rule would multiply it by.  `out` takes the gradient: a tensor like the scores, or the scores
themselves, which the gradient then replaces - a change of that tensor as any operation in place is, which a recorded operation that kept it reports.

Wrong arguments raise ValueError or TypeError before anything is queued; what a call refuses in the library raises EvtError."""
import ctypes as C

from . import _lib

__all__ = ["class_logp", "class_logp_grad", "distill_loss", "policy_loss", "preference_loss"]

_F32, _I32, _I64, _BF16, _F16 = 0, 4, 5, 10, 11
_TRUSTED = 2  # EVT_STATIC_TRUSTED: the tensors say where they are
_INF = float("inf")
_torch = None
_makers = {}  # by device
_entries = {}  # by name


def _load():
    """torch, the codes of its types and what a call needs of it; imported with the first call, a fit needs none."""
    global _torch, _FLOATS, _INTS, _F32S, _I32S, _like, _device, _stream, _changed, _wrapped
    import torch
    _F32S = {torch.float32: _F32}
    _FLOATS = {torch.float32: _F32, torch.bfloat16: _BF16, torch.float16: _F16}
    _I32S = {torch.int32: _I32}
    _INTS = {torch.int32: _I32, torch.int64: _I64}
    _like = torch.empty_like
    _device = torch.cuda.current_device
    _changed = torch.autograd.graph.increment_version
    # the current stream's handle without a Stream object around it, 1.1 us less a call
    _stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)
    _wrapped = getattr(getattr(torch._C, "_functorch", None), "is_functorch_wrapped_tensor", lambda t: False)
    _torch = torch


def _lasts(t):
    """Whether a tensor can make others for later calls: one that a tracer's mode or a function transform made is theirs, and has no memory when they have ended."""
    return type(t) is _torch.Tensor and not _wrapped(t)


def _bad(name, v, x, shape, kinds):
    """Says what is wrong with a tensor that is not as its call needs it."""
    if not isinstance(v, _torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(v).__name__))
    if v.dtype not in kinds:
        raise TypeError("%s must be %s, got %s" % (name, " or ".join(str(k)[6:] for k in kinds), v.dtype))
    if tuple(v.shape) != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, shape, tuple(v.shape)))
    if v.device != x.device:
        raise ValueError("%s is on %s, the scores are on %s" % (name, v.device, x.device))
    raise ValueError("%s must be contiguous" % name)


class _Call:
    """A call on some scores: the checks of what belongs to them, and the launch on their device's current stream."""
    __slots__ = ("x", "kind", "rows", "classes", "device", "temperature", "out")

    def __init__(self, x, temperature):
        if _torch is None:
            _load()
        if not isinstance(x, _torch.Tensor):
            raise TypeError("the scores must be a torch tensor, got %s" % type(x).__name__)
        kind = _FLOATS.get(x.dtype)
        if kind is None:
            raise TypeError("the scores must be float32, bfloat16 or float16, got %s" % x.dtype)
        if x.dim() != 2:
            raise ValueError("the scores must be a (rows, classes) matrix, got shape %s" % (tuple(x.shape),))
        rows, classes = x.shape
        if not 1 <= classes <= 1 << 30 or rows > 0x7FFFFFFF:
            raise ValueError("the scores must have 1 to 2^30 classes and at most 2^31 - 1 rows, got shape %s" % (tuple(x.shape),))
        if x.stride(1) != 1 and classes > 1:
            raise ValueError("the scores of a row must lie side by side, got strides %s" % (x.stride(),))
        self.x, self.kind, self.rows, self.classes, self.device, self.temperature = x, kind, rows, classes, x.get_device(), float(temperature)
        if not 1e-4 <= self.temperature <= 1e4:
            raise ValueError("temperature must be in [1e-4, 1e4], got %s" % temperature)

    def check(self, name, v, shape, kinds):
        """v's address, and its type's code by way of `kinds`."""
        try:
            if v.dtype in kinds and v.shape == shape and v.is_contiguous() and v.get_device() == self.device:
                return v.data_ptr()
        except AttributeError:
            pass
        _bad(name, v, self.x, shape, kinds)

    def floats(self, name, v):
        return self.check(name, v, (self.rows,), _F32S)

    def optional(self, name, v, n):
        return None if v is None else self.check(name, v, (n,), _F32S)

    def gradient(self, want, out):
        """The tensor the gradient goes to, None for none."""
        x = self.x
        self.out = out
        if out is None:
            if not want:
                return None
            return _like(x, memory_format=_torch.contiguous_format)
        if not want:
            raise ValueError("out was given, but no gradient is asked for")
        if not isinstance(out, _torch.Tensor) or out.dtype != x.dtype or out.shape != x.shape or out.device != x.device:
            raise ValueError("out must be a tensor like the scores: %s, %s, on %s" % (tuple(x.shape), x.dtype, x.device))
        if (out.stride(1) != 1 and out.shape[1] > 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
            raise ValueError("the rows of out must lie side by side or apart, got strides %s" % (out.stride(),))
        return out

    def values(self, *shape):
        """A float32 tensor on the call's device, by way of one that is there: 0.3 us less than torch.empty with a type and a device."""
        make = _makers.get(self.device)
        if make is None:
            one = _torch.empty(0, dtype=_torch.float32, device=self.x.device)
            make = one.new_empty
            if self.device >= 0 and _lasts(one):
                _makers[self.device] = make
        return make(shape)

    def run(self, name, grad, *args):
        x, dev, rows, classes = self.x, self.device, self.rows, self.classes
        if dev < 0:
            raise ValueError("the scores must be on a GPU, got %s" % x.device)
        s = _lib.EvtScores(x.data_ptr(), x.stride(0) if rows > 1 else classes, None if grad is None else grad.data_ptr(),
                           0 if grad is None else grad.stride(0) if rows > 1 else classes, rows, classes, self.kind, self.temperature)
        call = _entries.get(name)
        if call is None:
            call = _entries[name] = getattr(_lib.load(), name)
        if dev == _device():
            rc = call(_stream(dev), C.byref(s), *args, _TRUSTED)
        else:
            with _torch.cuda.device(dev):
                rc = call(_stream(dev), C.byref(s), *args, _TRUSTED)
        if rc:
            _lib.check(rc)
        if grad is not None and self.out is not None and not grad.is_inference():
            _changed(grad)


def class_logp(logits, labels, temperature=1.0):
    """Log-probability of every row's label under softmax(logits / temperature), and each row's maximum and sum of exponentials, which
    class_logp_grad takes: tensors (rows,) and (rows, 2), both float32.  Both are 0 for a row whose label is negative.  Nothing is recorded for a backward
    pass: class_logp_grad is it."""
    call = _Call(logits, temperature)
    rows = call.rows
    at = call.check("labels", labels, (rows,), _INTS)
    logp, stats = call.values(rows), call.values(rows, 2)
    call.run("evt_class_logp", None, at, _INTS[labels.dtype], logp.data_ptr(), stats.data_ptr())
    return logp, stats


def class_logp_grad(logits, labels, stats, dlogp, temperature=1.0, out=None):
    """Gradient of sum(dlogp * class_logp(logits, labels, temperature)[0]) by the logits, of the logits' type.  stats: what class_logp
    returned for the same logits and temperature."""
    call = _Call(logits, temperature)
    at = call.check("labels", labels, (call.rows,), _INTS)
    stats_at, dlogp_at = call.check("stats", stats, (call.rows, 2), _F32S), call.floats("dlogp", dlogp)
    grad = call.gradient(True, out)
    call.run("evt_class_logp_grad", grad, at, _INTS[labels.dtype], stats_at, dlogp_at)
    return grad


def distill_loss(logits, top_ids, top_logits, temperature=1.0, weights=None, grad=True, out=None):
    """Distillation from a teacher's best classes: for every row weights * temperature^2 * KL(softmax(top_logits / temperature) over the row's entries ||
    softmax(logits / temperature)), and the gradient of the sum of all rows' losses by the logits (None with grad=False), which is returned, not recorded.

    top_ids, top_logits: (rows, n_top), at most 1024 entries; a negative id is no entry.  top_logits may be float32, bfloat16 or float16."""
    call = _Call(logits, temperature)
    rows = call.rows
    if not isinstance(top_ids, _torch.Tensor) or top_ids.dim() != 2 or not 1 <= top_ids.shape[1] <= 1024:
        raise ValueError("top_ids must be a (rows, n_top) tensor with n_top from 1 to 1024")
    shape = (rows, top_ids.shape[1])
    ids_at, top_at = call.check("top_ids", top_ids, shape, _INTS), call.check("top_logits", top_logits, shape, _FLOATS)
    weights_at = call.optional("weights", weights, rows)
    g = call.gradient(grad, out)
    loss = call.values(rows)
    call.run("evt_distill_loss", g, ids_at, _INTS[top_ids.dtype], top_at, _FLOATS[top_logits.dtype], shape[1], weights_at, loss.data_ptr())
    return loss, g


def policy_loss(logits, actions, old_logp, advantages, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, temperature=1.0, weights=None, grad=True,
                out=None):
    """The clipped policy loss of every token, its log-probability, and the gradient of the sum of all losses by the logits (None with grad=False), which is
    returned, not recorded.

    With r = exp(logp - old_logp) the loss is weights * (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(b) - b - 1)), A the
    advantage and b = ref_logp - logp.  A negative action marks a padded row: its loss, log-probability and gradient are 0.  A weight of 0 leaves
    the log-probability."""
    call = _Call(logits, temperature)
    at = call.check("actions", actions, (call.rows,), _INTS)
    old_at, advantages_at = call.floats("old_logp", old_logp), call.floats("advantages", advantages)
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not (0.0 <= clip_low <= 1.0 and 0.0 <= clip_high < _INF and 0.0 <= kl_coef < _INF):
        raise ValueError("clip_low must be in [0, 1], clip_high and kl_coef finite and at least 0, got %s, %s and %s" % (clip_low, clip_high, kl_coef))
    ref_at, weights_at = call.optional("ref_logp", ref_logp, call.rows), call.optional("weights", weights, call.rows)
    if ref_at is None and kl_coef:
        raise ValueError("kl_coef needs ref_logp")
    g = call.gradient(grad, out)
    loss, logp = _like(old_logp), _like(old_logp)
    call.run("evt_policy_loss", g, at, _INTS[actions.dtype], old_at, advantages_at, ref_at, weights_at, clip_low, clip_high, kl_coef,
             loss.data_ptr(), logp.data_ptr())
    return loss, logp, g


def preference_loss(logits, labels, offsets, ref_logp, beta=0.1, label_smoothing=0.0, margin=0.0, average=False, temperature=1.0, weights=None,
                    grad=True, out=None):
    """The preference loss of pairs of sequences packed one behind the other, the log-probability of every sequence (summed over its labelled
    rows, their mean with `average`), and the gradient of the sum of all losses by the logits (None with grad=False), which is returned, not recorded.

    offsets: int32, sequence k has the rows offsets[k] to offsets[k + 1] - 1; the first half of the sequences are the chosen ones, the second half,
    in the same order, the rejected.  ref_logp: the reference model's log-probability of every sequence.  weights: one for each pair.
    With h = beta ((chosen - rejected) - (ref chosen - ref rejected)) - margin a pair's loss is weights * (-(1 - label_smoothing) log sigmoid(h)
    - label_smoothing log sigmoid(-h)).  Rows of no sequence get a gradient of 0.  Offsets that do not ascend, leave the rows or
    lie outside the first and the last are no sequence: its pair's loss and the gradient of its partner's rows are NaN.  A row that two sequences
    have, where offsets descend, takes the gradient of one of them, the same one in every call."""
    call = _Call(logits, temperature)
    at = call.check("labels", labels, (call.rows,), _INTS)
    if not isinstance(offsets, _torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 3 or offsets.shape[0] % 2 == 0:
        raise ValueError("offsets must be a vector of an odd number of row numbers, at least 3: one more than there are sequences")
    seqs = offsets.shape[0] - 1
    offsets_at, ref_at = call.check("offsets", offsets, (seqs + 1,), _I32S), call.check("ref_logp", ref_logp, (seqs,), _F32S)
    beta, label_smoothing, margin = float(beta), float(label_smoothing), float(margin)
    if not (0.0 < beta < _INF and 0.0 <= label_smoothing <= 0.5 and -_INF < margin < _INF):
        raise ValueError("beta must be positive and finite, label_smoothing in [0, 0.5], margin finite, got %s, %s and %s" % (beta, label_smoothing, margin))
    weights_at = call.optional("weights", weights, seqs // 2)
    g = call.gradient(grad, out)
    loss, seq_logp, work = call.values(seqs // 2), _like(ref_logp), call.values(4 * call.rows)
    call.run("evt_preference_loss", g, at, _INTS[labels.dtype], offsets_at, seqs // 2, ref_at, weights_at, beta, label_smoothing, margin,
             1 if average else 0, loss.data_ptr(), seq_logp.data_ptr(), work.data_ptr())
    return loss, seq_logp, g
