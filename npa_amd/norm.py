"""Layer norm over rows (no reference counterpart: its models normalise
perception's gradients by their logarithm only, models/npa.py:83-85).

With m = mean x and v = mean (x - m)^2 over a row (one particle's or token's
vector),

    y = (x - m) / sqrt(v + eps) * weight + bias

in float32 whatever the rows' type, rounded once.  A row that holds a NaN or an
infinity is NaN.  The gradients of weight and bias are sums over the rows in a
fixed order.  In front of an automaton's MLP,
``torch.nn.Sequential(LayerNorm(66), Linear(66, 128), ReLU(), Linear(128, 18))``
runs through ``npa_amd.mlp.mlp`` and ``step_euler`` like any module.
"""
import torch

from . import _rows
from ._rows import TYPES, address
from .sphops import _native

_lib = _native.lib


def _forward(x, weight, bias, eps, keep):
    """y, and what the backward reads: x's rows with their stride, and two floats a row."""
    cols = x.shape[-1]
    v, rows, stride = _rows.rows_view(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep else None
    wide = any(t is not None and t.dtype == torch.float32 for t in (weight, bias))
    _rows.call(_lib.sphops_layer_norm, x.device, v.data_ptr(), TYPES[x.dtype], stride, address(weight), address(bias),
               int(wide), y.data_ptr(), address(stats), rows, cols, eps)
    return y, v, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, v, stats = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(v, weight, stats)
        ctx.wtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        v, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        cols, dev = dy.shape[-1], dy.device
        u, rows, dy_stride = _rows.rows_view(dy)
        stride = v.stride(0) if v.dim() == 2 and rows > 1 else cols
        dx = torch.empty(dy.shape, dtype=dy.dtype, device=dev) if need_x else None
        dw, db = (torch.empty(cols, dtype=ctx.wtype, device=dev) if n else None for n in (need_w, need_b))
        work = torch.empty(max(_lib.sphops_layer_norm_workspace_bytes(TYPES[dy.dtype], rows, cols), 1),
                           dtype=torch.uint8, device=dev)
        _rows.call(_lib.sphops_layer_norm_backward, dev, v.data_ptr(), stride, u.data_ptr(), dy_stride,
                   TYPES[dy.dtype], address(weight), int(ctx.wtype == torch.float32), stats.data_ptr(), address(dx),
                   address(dw), address(db), rows, cols, work.data_ptr())
        return (*_rows.first_order("layer norm", dx, dw, db), None)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm over x's last dimension, of x's type (float32, bfloat16 or
    float16; autocast changes nothing).  ``weight`` and ``bias`` have its length
    and are both float32 or both of x's type; either may be None.  Gradients of
    all three; a second derivative and a forward-mode one raise.  A finite row the
    squares of whose deviations pass float32's range (deviations of about 1e19, masks
    of the lowest value among them) gives the bias, and no gradient to x."""
    _rows.check_rows(x, "x")
    types = (torch.float32,) if x.dtype == torch.float32 else (torch.float32, x.dtype)
    weight = _rows.check_weight(weight, x.shape[-1:], types, x.device, "weight")
    bias = _rows.check_weight(bias, x.shape[-1:], types, x.device, "bias")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    if not eps >= 0:
        raise ValueError("eps must not be negative")
    if _rows.wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, weight, bias, float(eps), False)[0]


class LayerNorm(torch.nn.LayerNorm):
    """``torch.nn.LayerNorm`` over the last dimension through ``layer_norm``: the
    same parameters under the same names."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm takes rows, one dimension, got {tuple(self.normalized_shape)}")

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise RuntimeError(f"x must have rows of {self.normalized_shape[0]} values, got shape {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
