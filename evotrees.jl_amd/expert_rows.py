"""Rows through experts, on torch tensors in device memory: the choice of each row's experts from their scores, rows sorted by expert and combined again with weights,
dropout, and the gradients of these (the C entry points evt_route_rows, evt_route_rows_grad, evt_plan_rows, evt_sort_rows, evt_combine_rows, evt_combine_rows_grad and
evt_drop_rows; include/evotrees_hip.h has the formulas).

They stand beside the losses over rows of class scores, the partition of rows by node (update_nodes_idx!, src/fit-utils.jl) and the random sample of rows: an expert may be
a layer's that a router chooses for a language model's token, or a model of its own at a leaf that predict_leaf_idx finds for a table's row: a column of what that returns, uint32
on the host, goes to the GPU as int32 or int64, torch.from_numpy(leaf[:, k].astype("int64")).cuda().  They have no counterpart in the reference.

    experts, weights = route_rows(scores, 8)                    # (rows, 8) each
    plan = plan_rows(experts, n_experts)
    y = ...experts' products of sort_rows(x, plan), expert e's rows plan.offsets[e] to plan.offsets[e + 1] - 1...
    out = combine_rows(y, plan, weights, residual=x, p=0.1, seed=seed, layer=3)

    dy, dweights = combine_rows_grad(dout, y, plan, weights, p=0.1, seed=seed, layer=3)
    dx = combine_rows(...the products' gradient from dy..., plan, residual=dout)   # sort_rows' gradient, and the residual's
    dscores = route_rows_grad(scores, experts, weights, dweights)

Rows are (rows, features) tensors of float32, bfloat16 or float16 whose features lie side by side (`x.stride(1) == 1`); rows may be any distance apart.  Weights and
their gradients are contiguous float32.  All tensors of a call are on one GPU; the work is queued on that GPU's current stream and nothing waits for it.  As the gradients of
this package's losses, these are returned, not recorded: a call reads the values of its tensors, whether they require a gradient or carry a tangent or not, its results never do, and
the backward pass is the program's to write, as shown above or in a torch.autograd.Function.  `out` takes
a result: a tensor like it, which counts as changed in place.  It shares no memory with what the call reads but where a call says so; columns of one matrix, with equal
strides, share none.

Wrong arguments raise ValueError or TypeError before anything is queued; what a call refuses in the library raises EvtError."""
import operator
import struct

from . import _lib
from . import class_losses as _scores

__all__ = ["RowPlan", "route_rows", "route_rows_grad", "plan_rows", "sort_rows", "combine_rows", "combine_rows_grad", "drop_rows"]

_TRUSTED = 2  # EVT_STATIC_TRUSTED: the tensors say where they are
_MOST = 4096  # experts
# an evt_rows (_lib.EvtRows) and an evt_scores (_lib.EvtScores) as bytes, a third of the time that a ctypes structure takes
_rows_bytes = struct.Struct("@PqPqPqqiidQPI4x").pack
_scores_bytes = struct.Struct("@PqPqqiid").pack
_NONE = (0, 0)  # no residual
_makers = {}  # by device and type
_entries = {}  # by name


def _torch():
    if _scores._torch is None:
        _scores._load()
    return _scores._torch


def _make(device, dtype, shape, on):
    """A tensor by way of one that is there: less time than torch.empty with a type and a device."""
    make = _makers.get((device, dtype))
    if make is None:
        one = _scores._torch.empty(0, dtype=dtype, device=on)
        make = one.new_empty
        if device >= 0 and _scores._lasts(one):
            _makers[(device, dtype)] = make
    return make(shape)


def _queue(name, device, on, *args):
    if device < 0:
        raise ValueError("the rows must be on a GPU, got %s" % on)
    call = _entries.get(name)
    if call is None:
        call = _entries[name] = getattr(_lib.load(), name)
    if device == _scores._device():
        rc = call(_scores._stream(device), *args, _TRUSTED)
    else:
        with _scores._torch.cuda.device(device):
            rc = call(_scores._stream(device), *args, _TRUSTED)
    if rc:
        _lib.check(rc)


def _whole(name, v, least, most):
    try:
        n = operator.index(v)
    except TypeError:
        raise TypeError("%s must be a whole number, got %s" % (name, type(v).__name__)) from None
    if not least <= n <= most:
        raise ValueError("%s must be in [%d, %d], got %d" % (name, least, most, n))
    return n


def _bad(name, v, shape, kinds, on):
    """Says what is wrong with a tensor that is not as its call needs it."""
    if not isinstance(v, _scores._torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(v).__name__))
    if v.dtype not in kinds:
        raise TypeError("%s must be %s, got %s" % (name, " or ".join(str(k)[6:] for k in kinds), v.dtype))
    if tuple(v.shape) != shape:
        raise ValueError("%s must have shape %s, got %s" % (name, shape, tuple(v.shape)))
    if v.device != on:
        raise ValueError("%s is on %s, the rows are on %s" % (name, v.device, on))
    raise ValueError("%s must be contiguous" % name)


def _check(name, v, shape, kinds, device, on):
    """v's address."""
    try:
        if v.dtype in kinds and v.shape == shape and v.is_contiguous() and v.get_device() == device:
            return v.data_ptr()
    except AttributeError:
        pass
    _bad(name, v, shape, kinds, on)


class RowPlan:
    """The tables that order rows by expert, from plan_rows.  place: (rows, top), where each entry of `experts` stands among the sorted rows, -1 if it is no
    expert's; source: (rows * top,), row * top + column of the entry at each place, -1 behind the last; offsets: (n_experts + 1,), expert e has the places
    offsets[e] to offsets[e + 1] - 1.  All are int32 on the device of `experts`."""
    __slots__ = ("rows", "top", "experts", "device", "offsets_at", "_on", "_tables", "_at")

    def __init__(self, rows, top, experts, device, on, tables):
        torch = _torch()
        if not isinstance(tables, torch.Tensor) or tables.dtype != torch.int32:
            raise TypeError("the tables must be one int32 tensor")
        if tables.get_device() != device:
            raise ValueError("the plan is on %s, its tables are on %s" % ("cuda:%d" % device if device >= 0 else on, tables.device))
        rows, top, experts = _whole("rows", rows, 0, 0x7FFFFFFF), _whole("top", top, 1, 0x7FFFFFFF), _whole("experts", experts, 1, _MOST)
        if tables.dim() != 1 or not tables.is_contiguous() or tables.storage_offset() or tables.shape[0] < 2 * rows * top + experts + 1:
            raise ValueError("the tables must be a vector of its own memory, place, source and offsets one behind the other, got shape %s" % (tuple(tables.shape),))
        self._hold(rows, top, experts, device, on, tables)

    def _hold(self, rows, top, experts, device, on, tables):
        self.rows, self.top, self.experts, self.device, self._on, self._tables = rows, top, experts, device, on, tables
        self._at = tables.data_ptr()
        self.offsets_at = self._at + 8 * rows * top

    def __reduce__(self):
        """A copy has its own tables, at their own address."""
        return _plan_again, (self.rows, self.top, self.experts, self._tables)

    @property
    def place(self):
        return self._tables.as_strided((self.rows, self.top), (self.top, 1), 0)

    @property
    def source(self):
        n = self.rows * self.top
        return self._tables.as_strided((n,), (1,), n)

    @property
    def offsets(self):
        return self._tables.as_strided((self.experts + 1,), (1,), 2 * self.rows * self.top)


def _plan_again(rows, top, experts, tables):
    return RowPlan(rows, top, experts, tables.get_device(), tables.device, tables)


class _Rows:
    """A call on some rows: the checks of what belongs to them, and the launch."""
    __slots__ = ("x", "kind", "rows", "feats", "device", "changed")

    def __init__(self, name, x):
        torch = _torch()
        if not isinstance(x, torch.Tensor):
            raise TypeError("%s must be a torch tensor, got %s" % (name, type(x).__name__))
        self.kind = _scores._FLOATS.get(x.dtype)
        if self.kind is None:
            raise TypeError("%s must be float32, bfloat16 or float16, got %s" % (name, x.dtype))
        if x.dim() != 2:
            raise ValueError("%s must be a (rows, features) matrix, got shape %s" % (name, tuple(x.shape)))
        self.rows, self.feats = x.shape
        if not 1 <= self.feats <= 1 << 24 or self.rows > 0x7FFFFFFF:
            raise ValueError("%s must have 1 to 2^24 features and at most 2^31 - 1 rows, got shape %s" % (name, tuple(x.shape)))
        if x.stride(1) != 1 and self.feats > 1:
            raise ValueError("the features of a row of %s must lie side by side, got strides %s" % (name, x.stride()))
        self.x, self.device, self.changed = x, x.get_device(), None

    def like(self, name, v, rows):
        """Address and row stride of other rows of the call."""
        x = self.x
        if not isinstance(v, _scores._torch.Tensor):
            raise TypeError("%s must be a torch tensor, got %s" % (name, type(v).__name__))
        if v.dtype != x.dtype:
            raise TypeError("%s must be %s as the other rows are, got %s" % (name, x.dtype, v.dtype))
        if v.dim() != 2 or v.shape[0] != rows or v.shape[1] != self.feats:
            raise ValueError("%s must have shape %s, got %s" % (name, (rows, self.feats), tuple(v.shape)))
        if v.get_device() != self.device:
            raise ValueError("%s is on %s, the other rows are on %s" % (name, v.device, x.device))
        if v.stride(1) != 1 and self.feats > 1:
            raise ValueError("the features of a row of %s must lie side by side, got strides %s" % (name, v.stride()))
        return v.data_ptr(), v.stride(0) if rows > 1 else self.feats

    def result(self, out, rows, like=None):
        """The tensor that a result goes to; `like`, where it is contiguous, makes one sooner."""
        if out is None:
            if like is not None and like.is_contiguous():
                return _scores._like(like)
            return _make(self.device, self.x.dtype, (rows, self.feats), self.x.device)
        self.like("out", out, rows)
        if rows > 1 and out.stride(0) < self.feats:
            raise ValueError("the rows of out must lie side by side or apart, got strides %s" % (out.stride(),))
        self.changed = out
        return out

    def plan(self, plan, sorted_rows):
        if not isinstance(plan, RowPlan):
            raise TypeError("plan must be what plan_rows returned, got %s" % type(plan).__name__)
        n = plan.rows * plan.top
        if self.rows != (n if sorted_rows else plan.rows):
            raise ValueError("the plan has %d rows of %d experts, %d sorted ones; got %d" % (plan.rows, plan.top, n, self.rows))
        if plan.device != self.device:
            raise ValueError("the plan is on %s, the rows are on %s" % (plan._on, self.x.device))
        return n

    def args(self, out, rows, res, p, seed, layer):
        """The call's evt_rows; res: address and row stride of the residual."""
        x, n = self.x, self.rows
        p = float(p)
        if not 0.0 <= p < 1.0:
            raise ValueError("p must be in [0, 1), got %s" % p)
        at = seed_at = 0
        if p:
            if isinstance(seed, _scores._torch.Tensor):
                seed_at = _check("seed", seed if seed.dim() else seed.view(1), (1,), (_scores._torch.int64,), self.device, x.device)
            else:
                at = _whole("seed", seed, -2 ** 63, 2 ** 64 - 1) & 0xFFFFFFFFFFFFFFFF
            layer = _whole("layer", layer, 0, 0xFFFFFFFF)
        else:
            layer = 0
        return _rows_bytes(x.data_ptr(), x.stride(0) if n > 1 else self.feats, out.data_ptr(), out.stride(0) if out.shape[0] > 1 else self.feats, res[0], res[1],
                           rows, self.feats, self.kind, p, at, seed_at, layer)

    def run(self, name, *args):
        _queue(name, self.device, self.x.device, *args)
        if self.changed is not None and not self.changed.is_inference():
            _scores._changed(self.changed)


def _route(scores, top, temperature):
    call = _scores._Call(scores, temperature)
    if call.classes > _MOST:
        raise ValueError("the scores must have at most %d experts, got %d" % (_MOST, call.classes))
    return call, _whole("top", top, 1, min(64, call.classes))


def _evt_scores(call, grad):
    x, rows = call.x, call.rows
    return _scores_bytes(x.data_ptr(), x.stride(0) if rows > 1 else call.classes, 0 if grad is None else grad.data_ptr(),
                         0 if grad is None else grad.stride(0) if rows > 1 else call.classes, rows, call.classes, call.kind, call.temperature)


def route_rows(scores, top, renormalize=True, temperature=1.0):
    """The `top` best of every row's experts, the best first and of equal scores the lower expert first, and their weights: tensors (rows, top), int32 and float32.

    scores: (rows, experts), at most 4096 experts; top: 1 to 64.  A weight is the expert's probability under softmax(scores / temperature) over the row's chosen experts, or with
    renormalize=False over all of them.  A score of -inf is an expert that cannot be chosen: a row with too few others has expert -1 with weight 0 in what is left."""
    call, top = _route(scores, top, temperature)
    torch = _scores._torch
    experts = _make(call.device, torch.int32, (call.rows, top), call.x.device)
    weights = _make(call.device, torch.float32, (call.rows, top), call.x.device)
    _queue("evt_route_rows", call.device, call.x.device, _evt_scores(call, None), top, 1 if renormalize else 0, experts.data_ptr(), weights.data_ptr())
    return experts, weights


def route_rows_grad(scores, experts, weights, dweights, renormalize=True, temperature=1.0, out=None):
    """Gradient of sum(dweights * weights) by the scores, of the scores' type, from what route_rows returned for the same scores, renormalize and temperature.  An expert of -1
    has no part in it, whatever stands at its weight's gradient.  `out` may be the scores themselves."""
    if not isinstance(experts, _torch().Tensor) or experts.dim() != 2:
        raise ValueError("experts must be a (rows, top) tensor")
    call, top = _route(scores, experts.shape[1], temperature)
    shape = (call.rows, top)
    ids_at = call.check("experts", experts, shape, _scores._INTS)
    w_at, dw_at = call.check("weights", weights, shape, _scores._F32S), call.check("dweights", dweights, shape, _scores._F32S)
    grad = call.gradient(True, out)
    _queue("evt_route_rows_grad", call.device, call.x.device, _evt_scores(call, grad), top, 1 if renormalize else 0, ids_at, _scores._INTS[experts.dtype],
           w_at, dw_at)
    if out is not None and not out.is_inference():
        _scores._changed(out)
    return grad


def plan_rows(experts, n_experts):
    """The tables that order rows by expert, a RowPlan: entries of one expert stand together, those of lower rows first.

    experts: (rows, top) or, of one expert a row, (rows,), int32 or int64, on a GPU; what is outside 0 to n_experts - 1 is no expert and has no place.  n_experts: at most
    4096."""
    torch = _torch()
    if not isinstance(experts, torch.Tensor):
        raise TypeError("experts must be a torch tensor, got %s" % type(experts).__name__)
    if experts.dim() not in (1, 2) or (experts.dim() == 2 and experts.shape[1] < 1):
        raise ValueError("experts must be a (rows, top) or (rows,) tensor, got shape %s" % (tuple(experts.shape),))
    n_experts = _whole("n_experts", n_experts, 1, _MOST)
    rows, top = experts.shape[0], experts.shape[1] if experts.dim() == 2 else 1
    n = rows * top
    if n > 0x7FFFFFFF:
        raise ValueError("experts must have at most 2^31 - 1 entries, got %d" % n)
    device, on = experts.get_device(), experts.device
    at = _check("experts", experts, experts.shape, _scores._INTS, device, on)
    if device < 0:
        raise ValueError("experts must be on a GPU, got %s" % on)
    # The tables, and what the call works in behind them: a second tensor costs a call 1.5 us.  A large one would stay as long as the plan, which a layer's backward pass still needs, and
    # goes when the work is queued.
    kept, block = 2 * n + n_experts + 1, 1024 if n <= 1 << 20 else 4096
    more = ((n + block - 1) // block + 1) * n_experts
    plan = RowPlan.__new__(RowPlan)
    if more <= 16384 or more <= kept >> 3:
        plan._hold(rows, top, n_experts, device, on, _make(device, torch.int32, (kept + more,), on))
        work_at = plan._at + 4 * kept
    else:
        plan._hold(rows, top, n_experts, device, on, _make(device, torch.int32, (kept,), on))
        work = _make(device, torch.int32, (more,), on)
        work_at = work.data_ptr()
    _queue("evt_plan_rows", device, on, at, _scores._INTS[experts.dtype], rows, top, n_experts, plan._at, plan._at + 4 * n, plan.offsets_at, work_at)
    return plan


def sort_rows(x, plan, out=None):
    """The rows in the plan's order, (rows * top, features): each row once for each of its experts, and 0 behind the last of them.  The gradient by x is
    combine_rows(dsorted, plan)."""
    call = _Rows("x", x)
    n = call.plan(plan, False)
    y = call.result(out, n)
    call.run("evt_sort_rows", call.args(y, call.rows, _NONE, 0.0, 0, 0), plan._at, plan.offsets_at, plan.top, plan.experts)
    return y


def combine_rows(y, plan, weights=None, residual=None, p=0.0, seed=None, layer=0, out=None):
    """residual + dropout(sum over a row's experts of weights * y), (rows, features): what the experts returned for the plan's sorted rows, back in the rows' order.

    weights: (rows, top), None for ones; an entry without an expert has no part whatever its weight.  p, seed and layer: dropout of the sum, see drop_rows.  `out` may be
    the residual."""
    call = _Rows("y", y)
    call.plan(plan, True)
    w_at = None if weights is None else _check("weights", weights, (plan.rows, plan.top), _scores._F32S, call.device, y.device)
    res = _NONE if residual is None else call.like("residual", residual, plan.rows)
    z = call.result(out, plan.rows, residual)
    call.run("evt_combine_rows", call.args(z, plan.rows, res, p, seed, layer), plan._at, w_at, plan.top)
    return z


def combine_rows_grad(dout, y, plan, weights, p=0.0, seed=None, layer=0):
    """Gradients of sum(dout * combine_rows(y, plan, weights, p=p, seed=seed, layer=layer)) by y, (rows * top, features) with 0 in rows that no entry has, and by the
    weights, (rows, top) with 0 for entries without an expert.  The residual's is dout.  With y None the weights' is not computed (None), and weights may be None for ones."""
    call = _Rows("dout", dout)
    n = call.plan(plan, False)
    w_at = dw_at = None
    y_at = (None, 0)
    dweights = None
    if weights is not None:
        w_at = _check("weights", weights, (plan.rows, plan.top), _scores._F32S, call.device, dout.device)
    if y is not None:
        if weights is None:
            raise ValueError("the weights' gradient needs weights")
        y_at = call.like("y", y, n)
        dweights = _make(call.device, _scores._torch.float32, (plan.rows, plan.top), dout.device)
        dw_at = dweights.data_ptr() if n else None
        if not n:
            y_at = (None, 0)
    dy = call.result(None, n)
    call.run("evt_combine_rows_grad", call.args(dy, call.rows, _NONE, p, seed, layer), y_at[0], y_at[1], plan._at, plan.offsets_at, w_at, dw_at, plan.top,
             plan.experts)
    return dy, dweights


def drop_rows(x, p, seed, layer=0, residual=None, out=None):
    """residual + dropout(x): each value is 0 with probability p and x / (1 - p) otherwise (p in multiples of 2^-32).

    seed: a whole number, or an int64 tensor of one element on the rows' GPU, read when the work runs, so that a replayed graph draws anew when its program changed it.
    layer: a whole number that keeps a program's uses of one seed apart.  Which values are dropped depends on seed, layer, row, column and the number of features alone (include/evotrees_hip.h
    says how); no mask is stored, and the gradient by x is drop_rows(dout, p, seed, layer).  What is dropped is 0 also where x is infinite or no number.  `out` may be x or the residual."""
    call = _Rows("x", x)
    res = _NONE if residual is None else call.like("residual", residual, call.rows)
    z = call.result(out, call.rows, x)
    call.run("evt_drop_rows", call.args(z, call.rows, res, p, seed, layer))
    return z
