"""Row operators that stand around the sparse ones in a layer with several experts, node types or relations.

The reference covers the sparse half of a graph layer (aggregation and edge scores); these cover what such a layer
computes densely before and after it, with their gradients:

    y, h = rms_norm(x, weight, residual=res)            # pre-norm on a residual stream
    r    = route(logits, k)                             # k of G experts a row, and the rows' lists by expert
    z    = grouped_matmul(y, W, r.groups, gather=True)  # one weight [out, in] an expert
    out  = combine_rows(z, r.groups, r.weights)         # weighted sum back, row order

A relation- or type-specific transform is the same with ``groups = group_rows(types, num_types)`` in the place of the
router.  ``rms_norm(..., quantize=True)`` gives 8-bit rows with a scale each (``QuantizedRows``), which
``grouped_matmul`` takes together with 8-bit weights.

All functions run on the current stream, allocate their outputs and workspaces there, never synchronise, and may be
captured into a CUDA graph (``featgraph_b200.graph_capture``).  A captured backward pass goes through
``torch.autograd.grad`` and returns detached outputs: torch ties a leaf's gradient accumulation to the stream of its
first live graph, so no graph of an eager step on the same leaves may be alive while a step is captured.

Types: float32, float16, bfloat16; sums are 32-bit and each output is rounded once.  No atomics on values: the same bits on
every run.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _device as dev

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.float8_e4m3fn: 3}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_SCORING = {"softmax": 0, "sigmoid": 1}
MAX_WIDTH, MAX_GROUPS, MAX_CHOICES = 16384, 1024, 32
MAX_COLUMNS = 2 ** 31 - 1025  # of products and sums: counted in 32 bits, up to the end of the last tile


class QuantizedRows(NamedTuple):
    """8-bit rows: ``values`` (float8_e4m3fn) [..., d] times ``scales`` (float32) [...]."""
    values: torch.Tensor
    scales: torch.Tensor


class RowGroups:
    """The lists of ``group_rows``: slots ``offsets[g] .. offsets[g + 1]`` belong to group g, ``order[slot]`` is the
    entry (row * k + choice) that a slot holds, ``position`` [n, k] the slot of each entry.  Entries in no group have
    position -1; the slots from ``offsets[-1]`` on hold -1.  All int32, on one device.  The lists are trusted to
    be such a pair of permutations; values out of range are treated as -1.  A backward pass needs them as they were in the
    forward pass: lists that were written to in between raise, as other saved tensors do."""
    __slots__ = ("offsets", "order", "position")

    def __init__(self, offsets, order, position):
        for name, t in (("offsets", offsets), ("order", order), ("position", position)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_contiguous() or t.device != offsets.device:
                raise ValueError("%s must be a contiguous int32 tensor, on one device with the others" % name)
        if offsets.dim() != 1 or not 2 <= offsets.numel() <= MAX_GROUPS + 1:
            raise ValueError("offsets must have 2 to %d values" % (MAX_GROUPS + 1))
        if position.dim() != 2 or order.dim() != 1 or order.numel() != position.numel() or not 1 <= position.shape[1] <= MAX_CHOICES:
            raise ValueError("order [n k] and position [n, k], 1 <= k <= %d, must list the same entries" % MAX_CHOICES)
        self.offsets, self.order, self.position = offsets, order, position

    @property
    def num_groups(self):
        return self.offsets.numel() - 1

    @property
    def num_entries(self):
        return self.order.numel()

    @property
    def num_rows(self):
        return self.position.shape[0]

    @property
    def choices(self):
        return self.position.shape[1]


class Routing(NamedTuple):
    """``weights`` [n, k] (float32, differentiable), ``experts`` [n, k] (int32, -1 where a row ran out of open
    experts) and the ``RowGroups`` of the experts."""
    weights: torch.Tensor
    experts: torch.Tensor
    groups: RowGroups


_entries = {}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, index, *args):
    """One library call on the current stream of device ``index``.  A small call's time is mostly spent on the way to it,
    so the way is short: entry points are looked up once, the stream's address is read without a Stream object."""
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(dev.lib(), name)
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        dev.check(rc)


def _size(name, *args):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(dev.lib(), name)
    return fn(*args)


def check_waits(device=None):
    """Waits for the current stream of ``device`` (the current one unless stated) and raises ``FeatGraphError`` if a row
    operator on that device ever gave up waiting for its own copies, which it does after some four seconds instead of
    hanging.  What that call returned is undefined.  For points where a program synchronises anyway; not for capture."""
    device = dev.resolve_device(device)
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("check_waits() synchronises: it cannot be captured")
    _call("fg_wait_status", device.index)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _tensor(t, what, dtypes, dims=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s: expected a torch.Tensor, got %r" % (what, type(t)))
    if t.dtype not in dtypes:
        raise TypeError("%s must be %s, got %s" % (what, " or ".join(str(d).replace("torch.", "") for d in dtypes), t.dtype))
    if dims is not None and t.dim() != dims:
        raise ValueError("%s must have %d dimensions, has shape %s" % (what, dims, tuple(t.shape)))
    return t


def _on(x, *others):
    """The rows' device index; the tensors of ``others`` (name, tensor or None, ...) must be there too."""
    if not x.is_cuda:
        dev.resolve_device(x.device)
    index = x.get_device()
    for i in range(1, len(others), 2):
        t = others[i]
        if t is not None and (not t.is_cuda or t.get_device() != index):
            raise ValueError("%s lives on %s, the rows on %s" % (others[i - 1], t.device, x.device))
    return index


def _as_rows(t):
    """t as a 2-D tensor whose rows are dense (a row stride of its own is kept), and that stride."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    n, d = t.shape
    ld, step = t.stride()
    if d > 1 and step != 1 or n > 1 and ld < d:
        t = t.contiguous()
        ld = d
    return t, (ld if n > 1 else d)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- norm ----

def _norm_forward(x, weight, residual, eps, quantize):
    xr, ldx = _as_rows(x)
    n, d = xr.shape
    device, kind = x.device, _TYPES[x.dtype]
    rr, ldr, h = None, 0, None
    if residual is not None:
        rr, ldr = _as_rows(residual)
        h = torch.empty(n, d, dtype=x.dtype, device=device)
    scales = None
    if quantize:
        y = torch.empty(n, d, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty(n, dtype=torch.float32, device=device)
    else:
        y = torch.empty(n, d, dtype=x.dtype, device=device)
    _call("fg_rms_norm", x.get_device(), xr.data_ptr(), ldx, _ptr(rr), ldr, _ptr(weight), _ptr(h), y.data_ptr(), _ptr(scales), n, d, eps, kind,
          kind if weight is None else _TYPES[weight.dtype], 3 if quantize else kind)
    if x.dim() != 2:
        shape = x.shape
        y, h, scales = y.view(shape), None if h is None else h.view(shape), None if scales is None else scales.view(shape[:-1])
    return y, h, scales


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, _ = _norm_forward(x, weight, residual, eps, False)
        ctx.eps = eps
        ctx.save_for_backward(x if h is None else h, weight)
        ctx.set_materialize_grads(False)
        return (y, h) if h is not None else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        if dy is None:  # only the sum was used
            return (dh if ctx.needs_input_grad[0] else None, None if weight is None else torch.zeros_like(weight),
                    dh if ctx.needs_input_grad[2] else None, None)
        d = h.shape[-1]
        hr, ldh = _as_rows(h)
        gr, ldg = _as_rows(dy)
        sr, lds = (None, 0) if dh is None else _as_rows(dh)
        n = hr.shape[0]
        dx = torch.empty(n, d, dtype=h.dtype, device=h.device)
        dw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        partial = None
        blocks = _size("fg_rms_norm_backward_blocks", n, d)
        if dw is not None:
            partial = torch.empty(blocks, d, dtype=torch.float32, device=h.device)
        kind = _TYPES[h.dtype]
        _call("fg_rms_norm_backward", h.get_device(), hr.data_ptr(), ldh, _ptr(weight), gr.data_ptr(), ldg, _ptr(sr), lds, dx.data_ptr(), _ptr(dw),
              _ptr(partial), blocks, n, d, ctx.eps, kind, kind if weight is None else _TYPES[weight.dtype])
        dx = dx.view(h.shape)
        return dx if ctx.needs_input_grad[0] else None, dw, dx if ctx.needs_input_grad[2] else None, None


def rms_norm(x, weight=None, residual=None, eps=1e-6, quantize=False):
    """Root-mean-square norm of the rows of ``x`` [..., d], d <= 16384, with the residual's addition:

        h = x + residual (in x's type; h = x without one)      y = h / sqrt(mean(h^2) + eps) * weight

    Returns ``y``, or ``(y, h)`` with a residual: h is the stream that the next layer adds to.  ``weight`` [d] is of
    x's type or float32 (None: ones).  ``quantize``: y as ``QuantizedRows`` (scale = max|y| / 448 a row, 1 where
    that quotient is 0 in 32 bits, as for a row of zeros; a row with an infinity or NaN has a scale that says so) - the
    form for serving, which has no gradient and refuses inputs that want one."""
    _tensor(x, "x", _FLOATS)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError("x must have rows of 1 to %d values, has shape %s" % (MAX_WIDTH, tuple(x.shape)))
    if weight is not None:
        _tensor(weight, "weight", (x.dtype, torch.float32), 1)
        if weight.shape[0] != x.shape[-1]:
            raise ValueError("weight has %d values, the rows %d" % (weight.shape[0], x.shape[-1]))
    if residual is not None:
        _tensor(residual, "residual", (x.dtype,))
        if residual.shape != x.shape:
            raise ValueError("residual has shape %s, x %s" % (tuple(residual.shape), tuple(x.shape)))
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("eps must be >= 0, got %r" % eps)
    _on(x, "weight", weight, "residual", residual)
    if weight is not None:
        weight = weight.contiguous()
    if _wants_grad(x, weight, residual):
        if quantize:
            raise ValueError("the 8-bit output has no gradient: call it under torch.no_grad() or on detached tensors")
        return _Norm.apply(x, weight, residual, eps)
    y, h, scales = _norm_forward(x, weight, residual, eps, bool(quantize))
    if quantize:
        y = QuantizedRows(y, scales)
    return y if h is None else (y, h)


def quantize_rows(x):
    """``x`` [..., d] as ``QuantizedRows``, the values that ``rms_norm(quantize=True)`` would give for y = x.  For a weight
    [groups, out, in] that is a scale for each output of each group.  No gradient."""
    _tensor(x, "x", _FLOATS)
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError("x must have rows of 1 to %d values, has shape %s" % (MAX_WIDTH, tuple(x.shape)))
    _on(x)
    if _wants_grad(x):
        raise ValueError("the 8-bit output has no gradient: call it under torch.no_grad() or on detached tensors")
    xr, ldx = _as_rows(x)
    n, d = xr.shape
    y = torch.empty(n, d, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(n, dtype=torch.float32, device=x.device)
    _call("fg_quantize_rows", x.get_device(), xr.data_ptr(), ldx, y.data_ptr(), scales.data_ptr(), n, d, _TYPES[x.dtype])
    return QuantizedRows(y.view(x.shape), scales.view(x.shape[:-1]))


# ---- routing ----

def group_rows(keys, num_groups):
    """``RowGroups`` of entries with ``keys`` [n] or [n, k] (int32 or int64): entry row * k + j belongs to group
    keys[row, j]; any value outside [0, num_groups) means no group.  Slots of a group hold its entries in ascending
    order.  num_groups <= 1024, k <= 32, n k < 2^31."""
    _tensor(keys, "keys", (torch.int32, torch.int64))
    if keys.dim() == 1:
        keys = keys.unsqueeze(1)
    if keys.dim() != 2 or not 1 <= keys.shape[1] <= MAX_CHOICES:
        raise ValueError("keys must be [n] or [n, k] with 1 <= k <= %d, have shape %s" % (MAX_CHOICES, tuple(keys.shape)))
    num_groups = int(num_groups)
    if not 1 <= num_groups <= MAX_GROUPS:
        raise ValueError("num_groups must be 1 to %d, got %d" % (MAX_GROUPS, num_groups))
    if keys.numel() >= 2 ** 31:
        raise ValueError("%d entries: fewer than 2^31 are wanted" % keys.numel())
    _on(keys)
    if keys.dtype == torch.int64:
        keys = keys.clamp(-1, num_groups).int()
    return _group(keys.contiguous(), num_groups)


def _lists(n, k, num_groups, device):
    """Unfilled lists, and the workspace that filling them takes."""
    m = n * k
    g = object.__new__(RowGroups)  # by construction what RowGroups() checks
    g.offsets = torch.empty(num_groups + 1, dtype=torch.int32, device=device)
    g.order = torch.empty(m, dtype=torch.int32, device=device)
    g.position = torch.empty(n, k, dtype=torch.int32, device=device)
    size = _size("fg_group_rows_workspace", m, num_groups)
    return g, (torch.empty(size, dtype=torch.uint8, device=device) if size else None), size


def _group(keys, num_groups):
    g, work, size = _lists(keys.shape[0], keys.shape[1], num_groups, keys.device)
    _call("fg_group_rows", keys.get_device(), keys.data_ptr(), g.num_entries, num_groups, g.offsets.data_ptr(), g.order.data_ptr(), g.position.data_ptr(),
          _ptr(work), size)
    return g


def _choose(logits, k, scoring, normalize):
    x, ld = _as_rows(logits)
    n, experts = x.shape
    device = x.device
    weights = torch.empty(n, k, dtype=torch.float32, device=device)
    chosen = torch.empty(n, k, dtype=torch.int32, device=device)
    g, work, size = _lists(n, k, experts, device)
    _call("fg_route", x.get_device(), x.data_ptr(), ld, weights.data_ptr(), chosen.data_ptr(), g.offsets.data_ptr(), g.order.data_ptr(),
          g.position.data_ptr(), n, experts, k, _TYPES[x.dtype], scoring, normalize, _ptr(work), size)
    return weights, chosen, g


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, scoring, normalize, lists):
        weights, chosen, g = _choose(logits, k, scoring, normalize)
        lists.append(chosen)  # what has no gradient does not pass through autograd
        lists.append(g)
        ctx.save_for_backward(logits, weights, chosen)
        ctx.args = (k, scoring, normalize)
        return weights

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights):
        logits, weights, chosen = ctx.saved_tensors
        x, ld = _as_rows(logits)
        dweights = dweights.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        k, scoring, normalize = ctx.args
        _call("fg_route_backward", x.get_device(), x.data_ptr(), ld, weights.data_ptr(), chosen.data_ptr(), dweights.data_ptr(), dx.data_ptr(),
              x.shape[0], x.shape[1], k, _TYPES[x.dtype], scoring, normalize)
        return dx, None, None, None, None


def route(logits, k, scoring="softmax", normalize=True):
    """The k largest logits of each row of ``logits`` [n, experts] in descending order, ties to the lowest index, as a
    ``Routing``.  Weights: softmax over the row, or sigmoid; ``normalize``: divided by their sum over the choice.
    A logit of -inf or NaN is closed: never chosen and without weight; where fewer than k are open, the remaining
    choices are -1 with weight 0.  experts <= 1024, k <= 32.  The weights are differentiable."""
    _tensor(logits, "logits", _FLOATS, 2)
    n, experts = logits.shape
    k = int(k)
    if scoring not in _SCORING:
        raise ValueError("scoring must be 'softmax' or 'sigmoid', got %r" % (scoring,))
    if not 1 <= experts <= MAX_GROUPS:
        raise ValueError("1 to %d experts are possible, got %d" % (MAX_GROUPS, experts))
    if not 1 <= k <= min(experts, MAX_CHOICES):
        raise ValueError("k must be 1 to %d, got %d" % (min(experts, MAX_CHOICES), k))
    if n * k >= 2 ** 31:
        raise ValueError("%d entries: fewer than 2^31 are wanted" % (n * k))
    _on(logits)
    args = (k, _SCORING[scoring], 1 if normalize else 0)
    if _wants_grad(logits):
        lists = []
        weights = _Route.apply(logits, *args, lists)
        return Routing(weights, *lists)
    return Routing(*_choose(logits, *args))


# ---- products ----

def _save(ctx, groups, *tensors):
    """Keeps ``tensors`` and the lists for the backward pass.  The lists count as saved tensors, so that ones that are refilled
    before it raise - but for lists made in inference mode, which autograd does not save (nor sees written to)."""
    lists = (groups.offsets, groups.order, groups.position)
    ctx.lists = lists if any(t.is_inference() for t in lists) else ()
    ctx.save_for_backward(*tensors, *(() if ctx.lists else lists))


def _saved(ctx):
    return (*ctx.saved_tensors, *ctx.lists)


def _product(x, ldx, x_scales, w, strides, w_scales, groups, gather, x_rows, inner, outer, out_dtype):
    device, kind, m, g = x.device, _TYPES[x.dtype], groups.order.numel(), groups.offsets.numel() - 1
    y = torch.empty(m, outer, dtype=out_dtype, device=device)
    xp, wp, order = x.data_ptr(), w.data_ptr(), groups.order.data_ptr() if gather else None
    size = _size("fg_grouped_matmul_workspace", xp, ldx, wp, *strides, order, m, g, inner, outer, kind)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _call("fg_grouped_matmul", x.get_device(), xp, ldx, _ptr(x_scales), wp, *strides, _ptr(w_scales), groups.offsets.data_ptr(), order,
          groups.position.shape[1], x_rows, y.data_ptr(), m, g, inner, outer, kind, _TYPES[out_dtype], _ptr(work), size)
    return y


class _Product(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, groups, gather):
        xr, ldx = _as_rows(x)
        ctx.gather = gather
        _save(ctx, groups, x, w)
        return _product(xr, ldx, None, w, w.stride(), None, groups, gather, x.shape[0], w.shape[2], w.shape[1], x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets, slots, places = _saved(ctx)
        outer, inner = w.shape[1], w.shape[2]
        want_dx, want_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        dyr, ldy = _as_rows(dy)
        xr, ldx = _as_rows(x)
        device, kind, m, g = x.device, _TYPES[x.dtype], slots.numel(), offsets.numel() - 1
        dx = torch.empty(x.shape, dtype=x.dtype, device=device) if want_dx else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=device) if want_dw else None
        order, position = (slots.data_ptr(), places.data_ptr()) if ctx.gather else (None, None)
        operands = (xr.data_ptr(), ldx, w.data_ptr(), *w.stride())
        size = _size("fg_grouped_matmul_backward_workspace", *operands, order, dyr.data_ptr(), ldy, want_dx, want_dw, m, g, inner, outer, kind)
        work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _call("fg_grouped_matmul_backward", x.get_device(), *operands, offsets.data_ptr(), order, position, places.shape[1],
              x.shape[0], dyr.data_ptr(), ldy, _ptr(dx), _ptr(dw), m, g, inner, outer, kind, _ptr(work), size)
        return dx, dw, None, None


def grouped_matmul(x, weight, groups, gather=False, out_dtype=None):
    """One product for each group: ``y[p] = weight[g] @ row`` for the slots p of group g; y is [entries, out], slots in
    no group are 0.  ``weight`` [groups, out, in] (any strides).  ``x`` [entries, in] holds a row for each slot, or, with
    ``gather``, [n, in] the rows in their own order, of which slot p reads row order[p] // k.  The groups' sizes stay on
    the device.  Differentiable in x and weight.

    An infinity or NaN stays in the rows (of ``weight``: the groups and outputs) that it belongs to.  In float32 an
    infinity gives NaN there, as operands are cut into parts; up to 32 slots of a weight with a dense inner axis of at most
    6144 values, and the other types, give what the sum gives.

    ``x`` and ``weight`` may both be ``QuantizedRows`` (scales [rows] and [groups, out]): products of the 8-bit values
    in 32-bit sums, scaled at the end, in ``out_dtype`` (bfloat16 unless stated); no gradient."""
    if not isinstance(groups, RowGroups):
        raise TypeError("groups: expected RowGroups (group_rows, route), got %r" % (type(groups),))
    eight = isinstance(x, QuantizedRows)
    if eight != isinstance(weight, QuantizedRows):
        raise TypeError("x and weight must both be QuantizedRows, or neither")
    x_scales = w_scales = None
    if eight:
        (x, x_scales), (weight, w_scales) = x, weight
        _tensor(x, "x.values", (torch.float8_e4m3fn,), 2)
        _tensor(weight, "weight.values", (torch.float8_e4m3fn,), 3)
        _tensor(x_scales, "x.scales", (torch.float32,), 1)
        _tensor(w_scales, "weight.scales", (torch.float32,), 2)
        if x_scales.shape != x.shape[:1] or w_scales.shape != weight.shape[:2]:
            raise ValueError("a scale for each row of x and for each output of weight is wanted")
        out_dtype = torch.bfloat16 if out_dtype is None else out_dtype
        if out_dtype not in _FLOATS:
            raise TypeError("out_dtype must be float32, float16 or bfloat16, got %s" % (out_dtype,))
    else:
        _tensor(x, "x", _FLOATS, 2)
        _tensor(weight, "weight", (x.dtype,), 3)
        if out_dtype not in (None, x.dtype):
            raise TypeError("out_dtype is x's type (%s) unless the inputs are 8-bit" % (x.dtype,))
        out_dtype = x.dtype
    if weight.shape[0] != groups.num_groups:
        raise ValueError("weight has %d groups, the rows %d" % (weight.shape[0], groups.num_groups))
    if weight.shape[2] != x.shape[1]:
        raise ValueError("weight takes %d values, the rows have %d" % (weight.shape[2], x.shape[1]))
    if not 1 <= weight.shape[1] <= MAX_COLUMNS or not 1 <= weight.shape[2] <= MAX_COLUMNS:
        raise ValueError("weight has shape %s" % (tuple(weight.shape),))
    want = groups.num_rows if gather else groups.num_entries
    if x.shape[0] != want:
        raise ValueError("x has %d rows, the groups %d%s" % (x.shape[0], want, "" if gather else " slots"))
    _on(x, "weight", weight, "groups", groups.offsets, "scales", x_scales, "weight_scales", w_scales)
    gather = bool(gather)
    if not eight and _wants_grad(x, weight):
        return _Product.apply(x, weight, groups, gather)
    xr, ldx = _as_rows(x)
    if eight:
        x_scales, w_scales = x_scales.contiguous(), w_scales.contiguous()
    return _product(xr, ldx, x_scales, weight, weight.stride(), w_scales, groups, gather, x.shape[0], weight.shape[2], weight.shape[1], out_dtype)


# ---- weighted sum back ----

def _combine(y, groups, weights):
    yr, ldy = _as_rows(y)
    n, k, d = groups.num_rows, groups.choices, y.shape[1]
    out = torch.empty(n, d, dtype=y.dtype, device=y.device)
    _call("fg_combine_rows", y.get_device(), yr.data_ptr(), ldy, _ptr(weights), groups.position.data_ptr(), out.data_ptr(), n, k, d, _TYPES[y.dtype])
    return out


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, groups, weights):
        _save(ctx, groups, y, weights)
        return _combine(y, groups, weights)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, weights, offsets, _, position = _saved(ctx)
        yr, ldy = _as_rows(y)
        gr, ldd = _as_rows(dout)
        (n, k), d = position.shape, y.shape[1]
        dy = torch.empty(n * k, d, dtype=y.dtype, device=y.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(n, k, dtype=torch.float32, device=y.device) if weights is not None and ctx.needs_input_grad[2] else None
        _call("fg_combine_rows_backward", y.get_device(), yr.data_ptr(), ldy, _ptr(weights), position.data_ptr(), offsets.data_ptr(),
              offsets.numel() - 1, gr.data_ptr(), ldd, _ptr(dy), _ptr(dw), n, k, d, _TYPES[y.dtype])
        return dy, None, dw


def combine_rows(y, groups, weights=None):
    """``out[t] = sum over j of weights[t, j] * y[position[t, j]]`` for ``y`` [entries, d] in slot order: the rows of
    ``grouped_matmul`` summed back into row order, [n, d].  Entries in no group add nothing.  ``weights`` [n, k] float32
    (None: ones).  Differentiable in y and weights."""
    if not isinstance(groups, RowGroups):
        raise TypeError("groups: expected RowGroups (group_rows, route), got %r" % (type(groups),))
    _tensor(y, "y", _FLOATS, 2)
    if y.shape[0] != groups.num_entries or not 1 <= y.shape[1] <= MAX_COLUMNS:
        raise ValueError("y must have a row for each of %d slots, has shape %s" % (groups.num_entries, tuple(y.shape)))
    if weights is not None:
        _tensor(weights, "weights", (torch.float32,), 2)
        if weights.shape != groups.position.shape:
            raise ValueError("weights have shape %s, the choices %s" % (tuple(weights.shape), tuple(groups.position.shape)))
    _on(y, "groups", groups.offsets, "weights", weights)
    if weights is not None:
        weights = weights.contiguous()
    if _wants_grad(y, weights):
        return _Combine.apply(y, groups, weights)
    return _combine(y, groups, weights)
