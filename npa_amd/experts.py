"""Mixtures of experts over rows: particles (or tokens) of several kinds, each
with an update rule of its own (no reference counterpart: its models have one
MLP for every particle, models/npa.py:63-78).

A row has k entries, each of which names an expert, or none: any number outside
0 .. experts - 1.

* ``sort_rows``: a stable sort of the entries by expert, as a ``Routing``.
* ``dispatch`` / ``combine``: rows to their entries' places, and the results back
  as the sum over a row's entries of weight times result.
* ``linear`` / ``mlp``: one layer, or Linear, ReLU, Linear, of every expert over
  the sorted rows, in one kernel a layer.  They need nothing but the experts'
  first places, so rows that are sorted already (clouds of different kinds one
  after another) need no routing.
* ``ExpertMlp``: a router and experts as a module, which ``npa_amd.mlp.mlp`` and
  ``step_euler`` run like any other.

Everything stays on the device: no count is read on the host, so all of it can be
captured into a HIP graph.  Rows are float32, bfloat16 or float16; sums are
float32, in a fixed order, and each result is rounded once.  float32 factors keep
their 24 bits.  Gradients throughout; a second derivative raises, and so does a
forward-mode one.
"""
import math
from typing import NamedTuple

import torch

from . import _rows
from . import mlp as _mlp
from ._rows import TYPES, address
from .sphops import _native

_lib = _native.lib

MAX_EXPERTS, MAX_CHOICES, MAX_SLOTS, MAX_FEATURES = 1024, 64, 1 << 30, 65536


class Routing(NamedTuple):
    """Where entries stand (int32, on the GPU): ``offsets`` (experts + 1), each
    expert's first place and then the first place behind them all; ``slot``, of the
    index's shape, each entry's place, ~place for an entry without an expert;
    ``source``, each place's entry (row * k + choice)."""
    offsets: torch.Tensor
    slot: torch.Tensor
    source: torch.Tensor


def sort_rows(index, experts):
    """The ``Routing`` of ``index`` (..., k), int32 or int64: entries stand expert
    after expert, each one's in their order, those without one behind the last."""
    if not index.is_cuda or index.dtype not in (torch.int32, torch.int64):
        raise TypeError("index must be an int32 or int64 GPU tensor")
    if index.dim() < 1 or not 1 <= index.shape[-1] <= MAX_CHOICES:
        raise RuntimeError(f"index must have 1 to {MAX_CHOICES} entries a row, got shape {tuple(index.shape)}")
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"experts must be 1 to {MAX_EXPERTS}, got {experts}")
    n, choices, dev = index.numel(), index.shape[-1], index.device
    if n > MAX_SLOTS:
        raise RuntimeError(f"index must have at most {MAX_SLOTS} entries")
    index = index if index.is_contiguous() else index.contiguous()
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    slot = torch.empty(index.shape, dtype=torch.int32, device=dev)
    source = torch.empty(n, dtype=torch.int32, device=dev)
    nbytes = _lib.sphops_sort_rows_workspace_bytes(n // choices, choices, experts)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _rows.call(_lib.sphops_sort_rows, dev, index.data_ptr(), int(index.dtype == torch.int64), n // choices, choices,
               experts, offsets.data_ptr(), slot.data_ptr(), source.data_ptr(), address(work))
    return Routing(offsets, slot, source)


def _check_slot(routing, device):
    """slot, source, rows and entries a row."""
    slot, source = routing.slot, routing.source
    if slot.dtype != torch.int32 or slot.device != device:
        raise TypeError(f"routing must hold int32 tensors on {device}")
    if slot.dim() < 1 or not 1 <= slot.shape[-1] <= MAX_CHOICES or not slot.is_contiguous():
        raise RuntimeError(f"routing.slot must be contiguous with 1 to {MAX_CHOICES} entries a row, got shape "
                           f"{tuple(slot.shape)}")
    if source.dtype != torch.int32 or source.device != device:
        raise TypeError(f"routing must hold int32 tensors on {device}")
    if source.shape != (slot.numel(),) or not source.is_contiguous():
        raise RuntimeError(f"routing.source must be contiguous and have shape {(slot.numel(),)}, got "
                           f"{tuple(source.shape)}")
    return slot, source, slot.numel() // slot.shape[-1], slot.shape[-1]


def _check_features(t, what):
    _rows.check_rows(t, what)
    if t.shape[-1] > MAX_FEATURES:
        raise RuntimeError(f"{what} must have rows of at most {MAX_FEATURES} values")


def _spread(x, slot, source):
    rows, choices, cols = slot.numel() // slot.shape[-1], slot.shape[-1], x.shape[-1]
    v, _, stride = _rows.rows_view(x)
    out = torch.empty(rows * choices, cols, dtype=x.dtype, device=x.device)
    _rows.call(_lib.sphops_dispatch_rows, x.device, v.data_ptr(), TYPES[x.dtype], stride, slot.data_ptr(),
               source.data_ptr(), out.data_ptr(), rows, choices, cols)
    return out


def _gather(results, weight, slot):
    rows, choices, cols = slot.numel() // slot.shape[-1], slot.shape[-1], results.shape[-1]
    results = results if results.is_contiguous() else results.contiguous()
    y = torch.empty(*slot.shape[:-1], cols, dtype=results.dtype, device=results.device)
    _rows.call(_lib.sphops_combine_rows, results.device, results.data_ptr(), TYPES[results.dtype], address(weight),
               slot.data_ptr(), y.data_ptr(), rows, choices, cols)
    return y


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, slot, source):
        ctx.save_for_backward(slot)
        return _spread(x, slot, source)

    @staticmethod
    def backward(ctx, d_out):
        slot, = ctx.saved_tensors
        return (*_rows.first_order("dispatch", _gather(d_out, None, slot)), None, None)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, results, weight, slot, source):
        ctx.save_for_backward(results, weight, slot, source)
        return _gather(results, weight, slot)

    @staticmethod
    def backward(ctx, dy):
        results, weight, slot, source = ctx.saved_tensors
        need_r, need_w = ctx.needs_input_grad[:2]
        results = results if results.is_contiguous() else results.contiguous()
        u, rows, stride = _rows.rows_view(dy)
        d_results = torch.empty_like(results) if need_r else None
        dw = torch.empty(slot.shape, dtype=torch.float32, device=dy.device) if need_w else None
        _rows.call(_lib.sphops_combine_rows_backward, dy.device, u.data_ptr(), TYPES[dy.dtype], stride,
                   results.data_ptr(), address(weight), slot.data_ptr(), source.data_ptr(), address(d_results),
                   address(dw), rows, slot.shape[-1], dy.shape[-1])
        return (*_rows.first_order("combine", d_results, dw), None, None)


def dispatch(x, routing):
    """Rows at their entries' places: x (..., cols) to (places, cols), a row k
    times; places of entries without an expert hold zeros."""
    _check_features(x, "x")
    slot, source, _, _ = _check_slot(routing, x.device)
    if x.shape[:-1] != slot.shape[:-1]:
        raise RuntimeError(f"x must have shape {tuple(slot.shape[:-1])} + (cols,), got {tuple(x.shape)}")
    return _Dispatch.apply(x, slot, source) if _rows.wants_grad(x) else _spread(x, slot, source)


def combine(results, weight, routing):
    """The places' rows back: y[r] is the sum over the row's entries, in their
    order, of ``weight`` (float32, of the index's shape; None: 1) times the
    place's row of ``results`` (places, cols).  Entries without an expert are left
    out, whatever their weight and place hold."""
    _check_features(results, "results")
    slot, source, rows, choices = _check_slot(routing, results.device)
    if results.dim() != 2 or results.shape[0] != rows * choices:
        raise RuntimeError(f"results must have {rows * choices} rows, got shape {tuple(results.shape)}")
    weight = _rows.check_weight(weight, slot.shape, (torch.float32,), results.device, "weight")
    if _rows.wants_grad(results, weight):
        return _Combine.apply(results, weight, slot, source)
    return _gather(results, weight, slot)


def _work(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear(x, w, b, offsets, relu=False):
    (experts, outs, cols), slots, kind = w.shape, x.shape[0], TYPES[x.dtype]
    v, _, stride = _rows.rows_view(x)
    y = torch.empty(slots, outs, dtype=x.dtype, device=x.device)
    work = _work(_lib.sphops_expert_linear_workspace_bytes(kind, slots, experts, cols, outs), x.device)
    _rows.call(_lib.sphops_expert_linear, x.device, v.data_ptr(), kind, stride, w.data_ptr(), address(b),
               offsets.data_ptr(), y.data_ptr(), slots, experts, cols, outs, int(relu), address(work))
    return y


def _gradients(dy, x, w, offsets, need_x, need_w, need_b, h=None):
    """dx (zero where h is not above 0), dW and db, those that are needed."""
    (experts, outs, cols), slots, kind, dev = w.shape, x.shape[0], TYPES[x.dtype], x.device
    if not (need_x or need_w or need_b):
        return None, None, None
    u, _, dy_stride = _rows.rows_view(dy)
    v, _, stride = _rows.rows_view(x)
    dx = torch.empty(slots, cols, dtype=x.dtype, device=dev) if need_x else None
    dw = torch.empty(w.shape, dtype=x.dtype, device=dev) if need_w else None
    db = torch.empty(experts, outs, dtype=x.dtype, device=dev) if need_b else None
    work = _work(_lib.sphops_expert_linear_backward_workspace_bytes(kind, slots, experts, cols, outs), dev)
    _rows.call(_lib.sphops_expert_linear_backward, dev, u.data_ptr(), dy_stride, v.data_ptr(), kind, stride,
               w.data_ptr(), address(h), offsets.data_ptr(), address(dx), address(dw), address(db), slots, experts, cols,
               outs, address(work))
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, offsets):
        ctx.save_for_backward(x, w, offsets)
        return _linear(x, w, b, offsets)

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        return (*_rows.first_order("the experts' layer", *_gradients(dy, x, w, offsets, *ctx.needs_input_grad[:3])), None)


class _Mlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, offsets):
        h = _linear(x, w1, b1, offsets, relu=True)
        ctx.save_for_backward(x, h, w1, w2, offsets)
        return _linear(h, w2, b2, offsets)

    @staticmethod
    def backward(ctx, dy):
        x, h, w1, w2, offsets = ctx.saved_tensors
        need_x, need_w1, need_b1, need_w2, need_b2, _ = ctx.needs_input_grad
        first = need_x or need_w1 or need_b1
        da, dw2, db2 = _gradients(dy, h, w2, offsets, first, need_w2, need_b2, h)
        dx, dw1, db1 = _gradients(da, x, w1, offsets, need_x, need_w1, need_b1) if first else (None, None, None)
        return (*_rows.first_order("the experts' MLP", dx, dw1, db1, dw2, db2), None)


def _fused_forward(x, w1, b1, w2, b2, offsets, keep):
    """y, and what the input gradient reads of the hidden values (a bit of each)."""
    (experts, hidden, cols), outs, slots = w1.shape, w2.shape[1], x.shape[0]
    y = torch.empty(slots, outs, dtype=torch.float32, device=x.device)
    mask = torch.empty(slots, 4, dtype=torch.int32, device=x.device) if keep else None
    _rows.call(_lib.sphops_expert_mlp_forward, x.device, x.data_ptr(), w1.data_ptr(), address(b1), w2.data_ptr(),
               address(b2), offsets.data_ptr(), y.data_ptr(), address(mask), slots, experts, cols, hidden, outs)
    return y, mask


class _FusedMlp(torch.autograd.Function):
    """``_Mlp`` of 128 hidden units in float32: x and a bit of each hidden value are kept."""

    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, offsets):
        x = x if x.is_contiguous() else x.contiguous()
        y, mask = _fused_forward(x, w1, b1, w2, b2, offsets, ctx.needs_input_grad[0])
        ctx.save_for_backward(x, mask, w1, b1, w2, offsets)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, mask, w1, b1, w2, offsets = ctx.saved_tensors
        need_x, need_w1, need_b1, need_w2, need_b2, _ = ctx.needs_input_grad
        (experts, hidden, cols), outs, slots, dev = w1.shape, w2.shape[1], x.shape[0], x.device
        dy = dy if dy.is_contiguous() else dy.contiguous()
        dx = dw1 = db1 = dw2 = db2 = None
        if need_x:
            dx = torch.empty_like(x)
            _rows.call(_lib.sphops_expert_mlp_input_grad, dev, dy.data_ptr(), w1.data_ptr(), w2.data_ptr(),
                       mask.data_ptr(), offsets.data_ptr(), dx.data_ptr(), slots, experts, cols, hidden, outs)
        if need_w1 or need_b1 or need_w2 or need_b2:
            dw1 = torch.empty_like(w1) if need_w1 else None
            db1 = torch.empty(experts, hidden, dtype=torch.float32, device=dev) if need_b1 else None
            dw2 = torch.empty_like(w2) if need_w2 else None
            db2 = torch.empty(experts, outs, dtype=torch.float32, device=dev) if need_b2 else None
            work = torch.empty(max(_lib.sphops_expert_mlp_workspace_bytes(slots, experts, cols, hidden, outs), 1),
                               dtype=torch.uint8, device=dev)
            _rows.call(_lib.sphops_expert_mlp_weight_grad, dev, x.data_ptr(), dy.data_ptr(), w1.data_ptr(), address(b1),
                       w2.data_ptr(), offsets.data_ptr(), address(dw1), address(db1), address(dw2), address(db2), slots,
                       experts, cols, hidden, outs, work.data_ptr())
        return (*_rows.first_order("the experts' MLP", dx, dw1, db1, dw2, db2), None)


def _check_layer(x, weight, bias, slots, experts, cols, what):
    if weight.dim() != 3 or not 1 <= weight.shape[1] <= MAX_FEATURES:
        raise RuntimeError(f"{what} must have shape (experts, out, in), got {tuple(weight.shape)}")
    outs = weight.shape[1]
    weight = _rows.check_weight(weight, (experts, outs, cols), (x.dtype,), x.device, what)
    bias = _rows.check_weight(bias, (experts, outs), (x.dtype,), x.device, f"the bias beside {what}")
    if _lib.sphops_expert_linear_workspace_bytes(TYPES[x.dtype], slots, experts, cols, outs) < 0:
        raise RuntimeError(f"no layer of {experts} experts for {slots} rows of {cols} inputs and {outs} outputs")
    return weight, bias


def _check_sorted(x, offsets):
    _check_features(x, "x")
    if x.dim() != 2:
        raise RuntimeError(f"x must have shape (places, in), got {tuple(x.shape)}")
    if offsets.dtype != torch.int32 or offsets.device != x.device:
        raise TypeError(f"offsets must be an int32 tensor on {x.device}")
    if offsets.dim() != 1 or not 2 <= offsets.shape[0] <= MAX_EXPERTS + 1 or not offsets.is_contiguous():
        raise RuntimeError(f"offsets must be contiguous and have 2 to {MAX_EXPERTS + 1} words, got shape "
                           f"{tuple(offsets.shape)}")
    return x.shape[0], offsets.shape[0] - 1, x.shape[1]


def linear(x, weight, bias, offsets):
    """x (places, in) through the linear layer of each place's expert: rows
    ``offsets[e]`` to ``offsets[e + 1] - 1`` give x W_e^T + b_e, rows behind the
    last expert's zeros.  ``weight`` (experts, out, in) and ``bias`` (experts,
    out; may be None) are of x's type; ``offsets`` (int32, as in a ``Routing``)
    starts at 0 and does not decrease.  The gradients of an expert without rows
    are zeros.  A layer whose launch would pass 2^32 threads raises (from about 2^37,
    float32 2^38, of places times inputs or outputs).

    Large float32 products run on bfloat16 pieces of their factors: there a value
    that is not finite may give NaN where float32 gives an infinity, and factors below
    2^-110 lose their last bits."""
    slots, experts, cols = _check_sorted(x, offsets)
    weight, bias = _check_layer(x, weight, bias, slots, experts, cols, "weight")
    if _rows.wants_grad(x, weight, bias):
        return _Linear.apply(x, weight, bias, offsets)
    return _linear(x, weight, bias, offsets)


def mlp(x, w1, b1, w2, b2, offsets):
    """``linear(relu(linear(x, w1, b1, offsets)), w2, b2, offsets)``.  float32 rows
    of 4 to 168 values with 128 hidden units and 4 to 64 outputs, the shapes of an
    automaton's update rule, take one kernel each way, which keeps the hidden
    values in registers; the weights' gradients compute them again, and where one
    lies within rounding of 0 they may take the ReLU's other side than y and x's
    gradient.  Elsewhere the ReLU is in the first layer's kernel and its
    mask in the second one's input gradient, and the hidden values, and their
    gradient, are kept in x's type.  float32 as in ``linear``."""
    slots, experts, cols = _check_sorted(x, offsets)
    w1, b1 = _check_layer(x, w1, b1, slots, experts, cols, "w1")
    hidden = w1.shape[1]
    w2, b2 = _check_layer(x, w2, b2, slots, experts, hidden, "w2")
    fused = (x.dtype == torch.float32
             and _lib.sphops_expert_mlp_workspace_bytes(slots, experts, cols, hidden, w2.shape[1]) >= 0)
    if _rows.wants_grad(x, w1, b1, w2, b2):
        return (_FusedMlp if fused else _Mlp).apply(x, w1, b1, w2, b2, offsets)
    if fused:
        return _fused_forward(x if x.is_contiguous() else x.contiguous(), w1, b1, w2, b2, offsets, False)[0]
    return _linear(_linear(x, w1, b1, offsets, relu=True), w2, b2, offsets)


class ExpertMlp(torch.nn.Module):
    """Linear, ReLU, Linear of ``experts`` experts, of which a router (a linear
    layer and a softmax) chooses ``choices`` for each row; the row's result is the
    sum of theirs, weighted with the router's probabilities.  Rows are of the
    parameters' type; under autocast they may be of any, the router runs as autocast
    runs a ``torch.nn.Linear`` and the experts in the parameters' type."""

    def __init__(self, in_features, hidden, out_features, experts, choices=1, bias=True, device=None, dtype=None):
        super().__init__()
        if not 1 <= choices <= min(experts, MAX_CHOICES) or experts > MAX_EXPERTS:
            raise ValueError(f"{choices} choices of {experts} experts")
        kind = dict(device=device, dtype=dtype)
        self.experts, self.choices = experts, choices
        self.router = torch.nn.Linear(in_features, experts, **kind)
        self.w1 = torch.nn.Parameter(torch.empty(experts, hidden, in_features, **kind))
        self.w2 = torch.nn.Parameter(torch.empty(experts, out_features, hidden, **kind))
        self.b1 = torch.nn.Parameter(torch.empty(experts, hidden, **kind)) if bias else None
        self.b2 = torch.nn.Parameter(torch.empty(experts, out_features, **kind)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        """Each expert as ``torch.nn.Linear`` starts its weights and biases."""
        self.router.reset_parameters()
        for w, b in ((self.w1, self.b1), (self.w2, self.b2)):
            for t in (w, b):
                if t is not None:
                    torch.nn.init.uniform_(t, -1 / math.sqrt(w.shape[2]), 1 / math.sqrt(w.shape[2]))

    def forward(self, x):
        logits = _mlp.linear(x, self.router) if x.dtype == torch.float32 else self.router(x)
        if torch.is_autocast_enabled():
            x = x.to(self.w1.dtype)
        weight, index = torch.softmax(logits.float(), -1).topk(self.choices, dim=-1)
        routing = sort_rows(index, self.experts)
        results = mlp(dispatch(x, routing), self.w1, self.b1, self.w2, self.b2, routing.offsets)
        return combine(results, weight, routing)
