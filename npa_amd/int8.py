"""Rows in 8 bits: activations kept between forward and backward, and layers
as products of 8-bit integers (no reference counterpart: its models run
``torch.nn.Linear`` in float32, models/npa.py:63-78).

A row x (one particle's or token's vector) has one float32 scale and one int8
code a value: with m = max(max |x|, 2^-100),

    scale = m / 127        code = round(x * (127 / m))        value = code * scale

in float32 steps, ties to the even code, so a value is off by at most half a
scale (with ``relu`` by less than one: see ``quantize_rows``).  A row that holds a NaN or an infinity gets a NaN scale: whatever is
computed from it is NaN.

* ``quantize_rows`` / ``restore_rows``: a tensor to a ``Rows8`` and back;
  ``checkpoint(function, x)`` runs a function of rows that keeps x in 8 bits and
  runs again in the backward.
* ``weight_grad``: a linear layer's dW and db from its saved input;
  ``npa_amd.mlp.mlp(module, z, checkpoint="int8")`` trains a module's layers
  that way, and NPA's Linear, ReLU, Linear keeps nothing but z in 8 bits (88
  bytes a particle instead of 844 at 83 inputs).
* ``linear`` / ``mlp`` and their modules ``Int8Linear`` / ``Int8Mlp``: inference
  with integer products, a scale for each row and each output channel.
"""
import ctypes
import functools
from typing import NamedTuple, Tuple

import torch

from .sphops import _native

_lib = _native.lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # SPHOPS_F32, _BF16, _F16
MAX_COLS = 65536
MAX_ROWS = 1 << 30
WEIGHT_ALIGN = 16  # bytes a row of a weight's codes is padded to
MLP_HIDDEN, MLP_MIN, MLP_MAX_IN, MLP_MAX_OUT = 128, 4, 168, 64


class Rows8(NamedTuple):
    """A tensor's rows in 8 bits: int8 ``codes`` (rows, ld), the columns from
    the row's length on zero; float32 ``scale`` (rows,); the ``shape`` of the
    tensor they stand for, rows along its last dimension."""
    codes: torch.Tensor
    scale: torch.Tensor
    shape: Tuple[int, ...]


def _ptr(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _stream(t):
    return ctypes.c_void_p(torch._C._cuda_getCurrentRawStream(t.device.index))


def _check_rows(x, what):
    if not x.is_cuda or x.dtype not in TYPES:
        raise TypeError(f"{what} must be a float32, bfloat16 or float16 GPU tensor")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLS:
        raise RuntimeError(f"{what} must have rows of 1 to {MAX_COLS} values, got shape {tuple(x.shape)}")
    if x.numel() // x.shape[-1] > MAX_ROWS:
        raise RuntimeError(f"{what} must have at most {MAX_ROWS} rows")


def _check_saved(r, what):
    rows = 1
    for n in r.shape[:-1]:
        rows *= n
    if r.codes.dtype != torch.int8 or r.scale.dtype != torch.float32 or not r.codes.is_cuda:
        raise TypeError(f"{what} must hold int8 codes and float32 scales on the GPU")
    if r.scale.device != r.codes.device:
        raise TypeError(f"{what}'s codes and scales must be on one device")
    if (r.codes.dim() != 2 or not r.codes.is_contiguous() or not r.scale.is_contiguous() or r.codes.shape[0] != rows
            or r.scale.shape != (rows,) or not 1 <= r.shape[-1] <= r.codes.shape[1] or r.shape[-1] > MAX_COLS
            or r.codes.shape[1] % 4 or r.codes.data_ptr() % 4):
        raise RuntimeError(f"{what}: codes {tuple(r.codes.shape)} and scales {tuple(r.scale.shape)} do not hold a "
                           f"tensor of shape {tuple(r.shape)} (contiguous, rows padded to a multiple of 4)")


def _check_weight(w, what):
    _check_saved(w, what)
    if len(w.shape) != 2 or w.codes.shape[1] % WEIGHT_ALIGN or w.codes.data_ptr() % WEIGHT_ALIGN:
        raise RuntimeError(f"{what} must be a matrix whose rows of codes are padded and aligned to {WEIGHT_ALIGN} "
                           f"bytes (quantize_rows(weight, align={WEIGHT_ALIGN}))")


def _check_bias(b, outs, device, what):
    if b is None:
        return
    if b.dtype != torch.float32 or b.device != device:
        raise TypeError(f"{what} must be a float32 tensor on {device}")
    if b.shape != (outs,) or not b.is_contiguous():
        raise RuntimeError(f"{what} must be contiguous and have shape {(outs,)}, got {tuple(b.shape)}")


def _no_backward(x, what):
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{what} is for inference and has no backward: call it under torch.no_grad()")


def _rows_view(x):
    """x as (tensor, rows, row stride): its rows where one stride leads from
    each to the next and a row is contiguous, else those of a copy."""
    cols = x.shape[-1]
    rows = x.numel() // cols
    if x.dim() == 1:
        return (x if x.stride(0) == 1 or cols == 1 else x.contiguous()), rows, cols
    if cols == 1 or x.stride(-1) == 1:
        v = x
        if x.dim() != 2:
            try:
                v = x.view(rows, cols)
            except RuntimeError:
                v = x.reshape(rows, cols)
        return v, rows, (v.stride(0) if rows > 1 else cols)
    return x.contiguous(), rows, cols


def quantize_rows(x, relu=False, align=4):
    """x's rows (last dimension) in 8 bits.  With ``relu`` the rows kept are
    relu(x), and in finite rows a code is positive exactly where x is: positive
    values below half a scale have the code 1, not 0, and stand for up to a
    scale more than they are.  That is little where rows have no outliers; in a
    row whose largest value is hundreds of times the others' it is most of them.
    ``align``: bytes a row of codes is padded to (a multiple of 4)."""
    _check_rows(x, "x")
    if align < 4 or align % 4:
        raise ValueError("align must be a multiple of 4")
    x = x.detach()
    cols = x.shape[-1]
    v, rows, stride = _rows_view(x)
    ld = -(-cols // align) * align
    codes = torch.empty(rows, ld, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, device=x.device)
    _native.check(_lib.sphops_quantize_rows(_ptr(v), TYPES[x.dtype], stride, _ptr(codes), ld, _ptr(scale), rows, cols,
                                            int(relu), _stream(x)))
    return Rows8(codes, scale, tuple(x.shape))


def restore_rows(r, dtype=torch.float32):
    """The tensor that ``r`` stands for, code * scale rounded once to dtype (a
    row's float32 largest or lowest value, as masks hold, comes back as it was)."""
    _check_saved(r, "r")
    if dtype not in TYPES:
        raise TypeError("dtype must be float32, bfloat16 or float16")
    out = torch.empty(r.shape, dtype=dtype, device=r.codes.device)
    _native.check(_lib.sphops_restore_rows(_ptr(r.codes), r.codes.shape[1], _ptr(r.scale), _ptr(out), TYPES[dtype],
                                           r.codes.shape[0], r.shape[-1], _stream(out)))
    return out


def weight_grad(r, dy, bias=True):
    """(dW, db) of a linear layer whose input was saved as ``r``: dW = dy^T x
    (out, in) and db the column sums of dy (None without ``bias``), float32 and
    in a fixed order of summation."""
    _check_saved(r, "r")
    if dy.dtype != torch.float32 or dy.device != r.codes.device:
        raise TypeError(f"dy must be a float32 tensor on {r.codes.device}")
    if dy.dim() < 1 or dy.shape[:-1] != tuple(r.shape[:-1]):
        raise RuntimeError(f"dy must have shape {tuple(r.shape[:-1])} + (out,), got {tuple(dy.shape)}")
    dy = dy.contiguous()
    rows, nin, nout = r.codes.shape[0], r.shape[-1], dy.shape[-1]
    nbytes = _lib.sphops_rows8_weight_grad_workspace_bytes(rows, nin, nout)
    if nbytes < 0:
        raise RuntimeError(f"no weight gradient for {rows} rows of {nin} inputs and {nout} outputs")
    dw = torch.empty(nout, nin, device=dy.device)
    db = torch.empty(nout, device=dy.device) if bias else None
    work = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dy.device)
    _native.check(_lib.sphops_rows8_weight_grad(_ptr(r.codes), r.codes.shape[1], _ptr(r.scale), _ptr(dy), _ptr(dw),
                                                _ptr(db), rows, nin, nout, _ptr(work), _stream(dy)))
    return dw, db


def linear(x, w, bias=None):
    """x W^T + bias in 8-bit integers, of x's dtype: the rows of x are put into
    8 bits, ``w`` is the weight as ``quantize_rows(weight, align=16)`` gives it.
    Inference only."""
    _check_rows(x, "x")
    _no_backward(x, "int8.linear")
    _check_weight(w, "w")
    outs, cols = w.shape
    if w.codes.device != x.device:
        raise TypeError("x and w must be on one device")
    if x.shape[-1] != cols:
        raise RuntimeError(f"x must have rows of {cols} values, got shape {tuple(x.shape)}")
    _check_bias(bias, outs, x.device, "bias")
    v, rows, stride = _rows_view(x)
    nbytes = _lib.sphops_linear8_workspace_bytes(rows, cols, outs)
    if nbytes < 0:
        raise RuntimeError(f"no integer product for {rows} rows of {cols} inputs and {outs} outputs")
    y = torch.empty(*x.shape[:-1], outs, dtype=x.dtype, device=x.device)
    work = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=x.device)
    _native.check(_lib.sphops_linear8(
        v.data_ptr(), TYPES[x.dtype], stride, w.codes.data_ptr(), w.codes.shape[1], w.scale.data_ptr(),
        None if bias is None else bias.data_ptr(), y.data_ptr(), rows, cols, outs, work.data_ptr(),
        torch._C._cuda_getCurrentRawStream(x.device.index)))
    return y


def mlp(z, w1, b1, w2, b2):
    """relu(z W1^T + b1) W2^T + b2 in 8-bit integers over float32 rows, 128
    hidden units, in one kernel: z and then the hidden row are put into 8 bits,
    the weights are given as ``quantize_rows(weight, align=16)`` gives them.
    Inference only."""
    if not z.is_cuda or z.dtype != torch.float32:
        raise TypeError("z must be a float32 GPU tensor")
    _no_backward(z, "int8.mlp")
    _check_weight(w1, "w1")
    _check_weight(w2, "w2")
    (hidden, nin), (nout, second) = w1.shape, w2.shape
    if not (hidden == second == MLP_HIDDEN and MLP_MIN <= nin <= MLP_MAX_IN and MLP_MIN <= nout <= MLP_MAX_OUT):
        raise RuntimeError(f"int8.mlp takes {MLP_HIDDEN} hidden units, {MLP_MIN} to {MLP_MAX_IN} inputs and {MLP_MIN} "
                           f"to {MLP_MAX_OUT} outputs, got weights {tuple(w1.shape)} and {tuple(w2.shape)}")
    if w1.codes.device != z.device or w2.codes.device != z.device:
        raise TypeError("z and the weights must be on one device")
    if z.dim() < 1 or z.shape[-1] != nin:
        raise RuntimeError(f"z must have rows of {nin} values, got shape {tuple(z.shape)}")
    _check_bias(b1, hidden, z.device, "b1")
    _check_bias(b2, nout, z.device, "b2")
    zc = z.contiguous()
    rows = zc.numel() // nin
    if rows > MAX_ROWS:
        raise RuntimeError(f"z must have at most {MAX_ROWS} rows")
    y = torch.empty(*z.shape[:-1], nout, device=z.device)
    _native.check(_lib.sphops_mlp8_forward(
        zc.data_ptr(), w1.codes.data_ptr(), w1.codes.shape[1], w1.scale.data_ptr(),
        None if b1 is None else b1.data_ptr(), w2.codes.data_ptr(), w2.codes.shape[1], w2.scale.data_ptr(),
        None if b2 is None else b2.data_ptr(), y.data_ptr(), rows, nin, hidden, nout,
        torch._C._cuda_getCurrentRawStream(z.device.index)))
    return y


class _Once(torch.autograd.Function):
    """Gradients as they are; differentiated again they raise."""

    @staticmethod
    def forward(ctx, what, anchor, *grads):
        ctx.what = what
        return grads

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} has no second derivative")


def first_order(what, *grads):
    """What a backward without a graph returns.  Under create_graph these
    gradients would count as constants and a second derivative would lose their
    part silently; they raise there instead (whether or not the upstream requires
    a gradient, which ``once_differentiable`` goes by)."""
    some = [g for g in grads if g is not None]
    if not torch.is_grad_enabled() or not some:
        return grads
    held = iter(_Once.apply(what, torch.zeros((), requires_grad=True), *some))
    return tuple(None if g is None else next(held) for g in grads)


def _leaves(t):
    """The leaf tensors that t's graph leads to."""
    todo, seen = [t.grad_fn], set()
    while todo:
        node = todo.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        if isinstance(getattr(node, "variable", None), torch.Tensor):
            yield node.variable
        todo.extend(n for n, _ in node.next_functions)


class _Checkpoint(torch.autograd.Function):
    """tensors: ``count`` params, then the parameters of ``function``'s own."""

    @staticmethod
    def forward(ctx, function, count, x, *tensors):
        r = quantize_rows(x)
        ctx.function, ctx.shape, ctx.dtype = function, r.shape, x.dtype
        ctx.count, ctx.own = count, tensors[count:]
        # without its cache, which would keep casts of params made here without a graph
        ctx.autocast = functools.partial(torch.autocast, "cuda", torch.get_autocast_dtype("cuda"),
                                         torch.is_autocast_enabled("cuda"), cache_enabled=False)
        ctx.save_for_backward(r.codes, r.scale, *tensors)
        with torch.no_grad(), ctx.autocast():
            return function(x, *tensors[:count])

    @staticmethod
    def backward(ctx, dy):
        codes, scale, *tensors = ctx.saved_tensors
        needs = ctx.needs_input_grad[2:]
        with torch.enable_grad(), ctx.autocast():
            x = restore_rows(Rows8(codes, scale, ctx.shape), ctx.dtype).requires_grad_(needs[0])
            params = [p.detach().requires_grad_(n) for p, n in zip(tensors[:ctx.count], needs[1:])]
            y = ctx.function(x, *params)
        inputs = [x, *params, *ctx.own]
        needs = [n and t.requires_grad for t, n in zip(inputs, needs)]  # own ones may have been frozen since
        wanted = [t for t, n in zip(inputs, needs) if n]
        known = {id(t) for t in wanted}
        if any(id(t) not in known for t in _leaves(y)):
            raise RuntimeError("int8.checkpoint: the function reads a tensor that requires a gradient and is neither an "
                               "argument nor a parameter of a module that it is: pass it as one of params")
        grads = iter(torch.autograd.grad(y, wanted, dy, allow_unused=True))
        return (None, None, *first_order("int8.checkpoint", *(next(grads) if n else None for n in needs)))


def checkpoint(function, x, *params):
    """``function(x, *params)``, one tensor, that keeps x in 8 bits for its
    backward: there x is restored and the function runs again with gradients,
    under the forward's autocast; it must not draw random numbers.
    The rounding of x is passed straight through.  ``params``: the tensors
    besides x that gradients are wanted of.  Where ``function`` is a module, or
    a method of one, the module's parameters get theirs without being named; any
    other tensor that it reads and that requires a gradient makes the backward
    raise."""
    _check_rows(x, "x")
    module = function if isinstance(function, torch.nn.Module) else getattr(function, "__self__", None)
    own = [p for p in module.parameters() if p.requires_grad] if isinstance(module, torch.nn.Module) else []
    if not torch.is_grad_enabled() or not any(t.requires_grad for t in (x, *params, *own)):
        return function(x, *params)
    return _Checkpoint.apply(function, len(params), x, *params, *own)


def _kept_weight(layer):
    if layer.weight.dtype not in TYPES or not layer.weight.is_cuda:
        raise TypeError("the layer's weight must be a float32, bfloat16 or float16 GPU tensor")
    bias = None if layer.bias is None else layer.bias.detach().float().contiguous().clone()
    return quantize_rows(layer.weight, align=WEIGHT_ALIGN), bias


class Int8Linear(torch.nn.Module):
    """A ``torch.nn.Linear`` for inference in 8-bit integers: its weight is laid
    out once, here."""

    def __init__(self, layer):
        super().__init__()
        w, bias = _kept_weight(layer)
        self.in_features, self.out_features = layer.in_features, layer.out_features
        self.register_buffer("codes", w.codes)
        self.register_buffer("scale", w.scale)
        self.register_buffer("bias", bias)

    @property
    def rows(self):
        return Rows8(self.codes, self.scale, (self.out_features, self.in_features))

    def forward(self, x):
        return linear(x, self.rows, self.bias)


class Int8Mlp(torch.nn.Module):
    """A ``Sequential`` of Linear and ReLU for inference in 8-bit integers, for
    instance an NPA model's ``model.model``: Linear, ReLU, Linear with 128
    hidden units in one kernel, any other through ``Int8Linear``."""

    def __init__(self, module):
        super().__init__()
        layers = list(module) if isinstance(module, torch.nn.Sequential) else [module]
        for m in layers:
            if type(m) not in (torch.nn.Linear, torch.nn.ReLU):
                raise TypeError(f"Int8Mlp takes Linear and ReLU layers, got {type(m).__name__}")
        self.layers = torch.nn.ModuleList(Int8Linear(m) if type(m) is torch.nn.Linear else m for m in layers)
        first, last = self.layers[0], self.layers[-1]
        self.fused = ([type(m) for m in layers] == [torch.nn.Linear, torch.nn.ReLU, torch.nn.Linear]
                      and first.out_features == MLP_HIDDEN and MLP_MIN <= first.in_features <= MLP_MAX_IN
                      and MLP_MIN <= last.out_features <= MLP_MAX_OUT)

    def forward(self, z):
        if self.fused and z.dtype == torch.float32:
            first, last = self.layers[0], self.layers[2]
            return mlp(z, first.rows, first.bias, last.rows, last.bias)
        for layer in self.layers:
            z = layer(z)
        return z
