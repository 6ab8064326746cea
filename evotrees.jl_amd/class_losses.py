"""Losses over rows of class scores with their gradients, on torch tensors in device memory: log-probabilities of chosen classes, distillation
from a teacher's top scores, the clipped policy loss and the preference loss of paired sequences (the C entry points evt_class_logp,
evt_class_logp_grad, evt_distill_loss, evt_policy_loss and evt_preference_loss; include/evotrees_hip.h has the formulas).

They stand beside the multi-class log loss that EvoTreeClassifier is fitted with (mlogloss_grad_hess, src/loss.jl:93-98, :113-128) for models of any number of
classes, a language model's vocabulary as well as a classifier's levels, and have no counterpart in the reference.

Scores are a (rows, classes) tensor of float32, bfloat16 or float16 whose classes lie side by side (`scores.stride(1) == 1`); rows may be
any distance apart.  Labels and class ids count from 0 and are int32 or int64; a negative one stands for none.  Values that
belong to a row, an entry or a pair are contiguous float32.  All tensors of a call are on one GPU; the work is queued on that GPU's current
stream and nothing waits for it.  As the gradients of this package's other losses, these are returned, not recorded: there is no autograd
graph, and a loss's weights stand in for what a chain rule would multiply it by.  `out` takes the gradient: a tensor like the scores, or the scores
themselves, which the gradient then replaces.

Wrong arguments raise ValueError or TypeError before anything is queued; what a call refuses in the library raises EvtError."""
import ctypes as C

from . import _lib

__all__ = ["class_logp", "class_logp_grad", "distill_loss", "policy_loss", "preference_loss"]

_F32, _I32, _I64, _BF16, _F16 = 0, 4, 5, 10, 11
_TRUSTED = 2  # EVT_STATIC_TRUSTED: the tensors say where they are
_torch = None


def _load():
    """torch and the codes of its types; imported with the first call, a fit needs none."""
    global _torch, _FLOATS, _INTS, _new
    if _torch is None:
        import torch
        _FLOATS = {torch.float32: _F32, torch.bfloat16: _BF16, torch.float16: _F16}
        _INTS = {torch.int32: _I32, torch.int64: _I64}
        _new = torch.empty
        _torch = torch
    return _torch


def _scores(name, x):
    torch = _load()
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(x).__name__))
    if x.dtype not in _FLOATS:
        raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, x.dtype))
    if x.dim() != 2:
        raise ValueError("%s must be a (rows, classes) matrix, got shape %s" % (name, tuple(x.shape)))
    if x.shape[1] < 1 or x.shape[1] > 0x7FFFFFFF or x.shape[0] > 0x7FFFFFFF:
        raise ValueError("%s must have 1 to 2^31 - 1 classes and at most 2^31 - 1 rows, got shape %s" % (name, tuple(x.shape)))
    if x.stride(1) != 1 and x.shape[1] > 1:
        raise ValueError("the classes of %s must lie side by side, got strides %s" % (name, x.stride()))


def _check(name, v, x, shape, kinds, what):
    if not isinstance(v, _torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(v).__name__))
    if v.dtype not in kinds:
        raise TypeError("%s must be %s, got %s" % (name, what, v.dtype))
    if tuple(v.shape) != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, shape, tuple(v.shape)))
    if not v.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    if v.device != x.device:
        raise ValueError("%s is on %s, the scores are on %s" % (name, v.device, x.device))


def _floats(name, v, x, n):
    _check(name, v, x, (n,), (_torch.float32,), "float32")


def _labels(name, v, x):
    _check(name, v, x, (x.shape[0],), _INTS, "int32 or int64")


def _number(name, v, low, high, open_low=False):
    v = float(v)
    if not (low < v if open_low else low <= v) or not v <= high or v == float("inf"):
        raise ValueError("%s must be finite and in %s%s, %s], got %s" % (name, "(" if open_low else "[", low, high, v))
    return v


def _gradient(x, want, out):
    """The tensor the gradient goes to, None for none."""
    if out is None:
        return _new(x.shape, dtype=x.dtype, device=x.device) if want else None
    if not want:
        raise ValueError("out was given, but no gradient is asked for")
    if not isinstance(out, _torch.Tensor) or out.dtype != x.dtype or out.shape != x.shape or out.device != x.device:
        raise ValueError("out must be a tensor like the scores: %s, %s, on %s" % (tuple(x.shape), x.dtype, x.device))
    if (out.stride(1) != 1 and out.shape[1] > 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError("the rows of out must lie side by side or apart, got strides %s" % (out.stride(),))
    return out


class _Call:
    """The scores as the library takes them, and the device and stream of the call."""

    def __init__(self, x, temperature):
        self.x, self.temperature = x, _number("temperature", temperature, 0.0, float("inf"), True)

    def run(self, name, grad, *args):
        x = self.x
        if not x.is_cuda:
            raise ValueError("the scores must be on a GPU, got %s" % x.device)
        s = _lib.EvtScores(x.data_ptr(), x.stride(0) if x.shape[0] > 1 else x.shape[1], None if grad is None else grad.data_ptr(),
                           0 if grad is None else grad.stride(0) if x.shape[0] > 1 else x.shape[1], x.shape[0], x.shape[1], _FLOATS[x.dtype], self.temperature)
        call = getattr(_lib.load(), name)
        dev = x.device.index
        if dev == _torch.cuda.current_device():
            _lib.check(call(_torch.cuda.current_stream(dev).cuda_stream, C.byref(s), *args, _TRUSTED))
        else:
            with _torch.cuda.device(dev):
                _lib.check(call(_torch.cuda.current_stream(dev).cuda_stream, C.byref(s), *args, _TRUSTED))


def _at(v):
    return None if v is None else v.data_ptr()


def _made(x, *shape):
    return _new(shape, dtype=_torch.float32, device=x.device)


def class_logp(logits, labels, temperature=1.0):
    """Log-probability of every row's label under softmax(logits / temperature), and each row's maximum and sum of exponentials, which
    class_logp_grad takes: tensors (rows,) and (rows, 2), both float32.  Both are 0 for a row whose label is negative."""
    _scores("logits", logits)
    call = _Call(logits, temperature)
    _labels("labels", labels, logits)
    rows = logits.shape[0]
    logp, stats = _made(logits, rows), _made(logits, rows, 2)
    call.run("evt_class_logp", None, labels.data_ptr(), _INTS[labels.dtype], logp.data_ptr(), stats.data_ptr())
    return logp, stats


def class_logp_grad(logits, labels, stats, dlogp, temperature=1.0, out=None):
    """Gradient of sum(dlogp * class_logp(logits, labels, temperature)[0]) by the logits, of the logits' type.  stats: what class_logp
    returned for the same logits and temperature."""
    _scores("logits", logits)
    call = _Call(logits, temperature)
    _labels("labels", labels, logits)
    rows = logits.shape[0]
    _check("stats", stats, logits, (rows, 2), (_torch.float32,), "float32")
    _floats("dlogp", dlogp, logits, rows)
    grad = _gradient(logits, True, out)
    call.run("evt_class_logp_grad", grad, labels.data_ptr(), _INTS[labels.dtype], stats.data_ptr(), dlogp.data_ptr())
    return grad


def distill_loss(logits, top_ids, top_logits, temperature=1.0, weights=None, grad=True, out=None):
    """Distillation from a teacher's best classes: for every row weights * temperature^2 * KL(softmax(top_logits / temperature) over the row's entries ||
    softmax(logits / temperature)), and the gradient of the sum of all rows' losses by the logits (None with grad=False).

    top_ids, top_logits: (rows, n_top), at most 1024 entries; a negative id is no entry.  top_logits may be float32, bfloat16 or float16."""
    _scores("logits", logits)
    call = _Call(logits, temperature)
    rows = logits.shape[0]
    if not isinstance(top_ids, _torch.Tensor) or top_ids.dim() != 2 or not 1 <= top_ids.shape[1] <= 1024:
        raise ValueError("top_ids must be a (rows, n_top) tensor with n_top from 1 to 1024")
    shape = (rows, top_ids.shape[1])
    _check("top_ids", top_ids, logits, shape, _INTS, "int32 or int64")
    _check("top_logits", top_logits, logits, shape, _FLOATS, "float32, bfloat16 or float16")
    if weights is not None:
        _floats("weights", weights, logits, rows)
    g = _gradient(logits, grad, out)
    loss = _made(logits, rows)
    call.run("evt_distill_loss", g, top_ids.data_ptr(), _INTS[top_ids.dtype], top_logits.data_ptr(), _FLOATS[top_logits.dtype], shape[1], _at(weights),
             loss.data_ptr())
    return loss, g


def policy_loss(logits, actions, old_logp, advantages, ref_logp=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, temperature=1.0, weights=None, grad=True,
                out=None):
    """The clipped policy loss of every token, its log-probability, and the gradient of the sum of all losses by the logits (None with grad=False).

    With r = exp(logp - old_logp) the loss is weights * (-min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(b) - b - 1)), A the
    advantage and b = ref_logp - logp.  A negative action marks a padded row: its loss, log-probability and gradient are 0.  A weight of 0 leaves
    the log-probability."""
    _scores("logits", logits)
    call = _Call(logits, temperature)
    rows = logits.shape[0]
    _labels("actions", actions, logits)
    _floats("old_logp", old_logp, logits, rows)
    _floats("advantages", advantages, logits, rows)
    clip_low, clip_high = _number("clip_low", clip_low, 0.0, 1.0), _number("clip_high", clip_high, 0.0, float("inf"))
    kl_coef = _number("kl_coef", kl_coef, 0.0, float("inf"))
    if ref_logp is not None:
        _floats("ref_logp", ref_logp, logits, rows)
    elif kl_coef:
        raise ValueError("kl_coef needs ref_logp")
    if weights is not None:
        _floats("weights", weights, logits, rows)
    g = _gradient(logits, grad, out)
    loss, logp = _made(logits, rows), _made(logits, rows)
    call.run("evt_policy_loss", g, actions.data_ptr(), _INTS[actions.dtype], old_logp.data_ptr(), advantages.data_ptr(), _at(ref_logp), _at(weights),
             clip_low, clip_high, kl_coef, loss.data_ptr(), logp.data_ptr())
    return loss, logp, g


def preference_loss(logits, labels, offsets, ref_logp, beta=0.1, label_smoothing=0.0, margin=0.0, average=False, temperature=1.0, weights=None,
                    grad=True, out=None):
    """The preference loss of pairs of sequences packed one behind the other, the log-probability of every sequence (summed over its labelled
    rows, their mean with `average`), and the gradient of the sum of all losses by the logits (None with grad=False).

    offsets: int32, sequence k has the rows offsets[k] to offsets[k + 1] - 1; the first half of the sequences are the chosen ones, the second half,
    in the same order, the rejected.  ref_logp: the reference model's log-probability of every sequence.  weights: one for each pair.
    With h = beta ((chosen - rejected) - (ref chosen - ref rejected)) - margin a pair's loss is weights * (-(1 - label_smoothing) log sigmoid(h)
    - label_smoothing log sigmoid(-h)).  Rows of no sequence get a gradient of 0; offsets that do not ascend or leave the rows
    make their pair's results NaN."""
    _scores("logits", logits)
    call = _Call(logits, temperature)
    rows = logits.shape[0]
    _labels("labels", labels, logits)
    if not isinstance(offsets, _torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 3 or offsets.shape[0] % 2 == 0:
        raise ValueError("offsets must be a vector of an odd number of row numbers, at least 3: one more than there are sequences")
    _check("offsets", offsets, logits, tuple(offsets.shape), (_torch.int32,), "int32")
    seqs = offsets.shape[0] - 1
    _floats("ref_logp", ref_logp, logits, seqs)
    beta = _number("beta", beta, 0.0, float("inf"), True)
    label_smoothing = _number("label_smoothing", label_smoothing, 0.0, 0.5)
    margin = _number("margin", margin, -float("inf"), float("inf"))
    if weights is not None:
        _floats("weights", weights, logits, seqs // 2)
    g = _gradient(logits, grad, out)
    loss, seq_logp, work = _made(logits, seqs // 2), _made(logits, seqs), _made(logits, 4 * rows)
    call.run("evt_preference_loss", g, labels.data_ptr(), _INTS[labels.dtype], offsets.data_ptr(), seqs // 2, ref_logp.data_ptr(), _at(weights),
             beta, label_smoothing, margin, 1 if average else 0, loss.data_ptr(), seq_logp.data_ptr(), work.data_ptr())
    return loss, seq_logp, g
