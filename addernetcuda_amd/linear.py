"""Linear layers with what surrounds them in one call: ``act(x w' + bias) + residual``.

The reference's VGG classifiers are ``nn.Linear`` - ReLU stacks (vgg.py) and leave them to the framework; the blocks of linear
layers that networks put beside adder layers add a GELU or SiLU and a shortcut.  csrc/linear*.hip computes the product on the
matrix cores and bias, activation and shortcut on its way out, so that the product's result crosses memory once; the backward
is one pass for ``dy * act'(z)`` and the bias's gradient, then the two products.

float32 and bfloat16, all tensors of a call alike (the module rounds float32 parameters for a bfloat16 input).  CPU tensors and
other types go through torch's own operators.
"""
import ctypes
import functools

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._lib import lib, check, ptr, stream_ptr, on_device, plain_call

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}   # adder_act
TYPES = {torch.float32: 0, torch.bfloat16: 1}         # adder_type


@functools.lru_cache(maxsize=4096)
def _fwd_bytes(rows, k, n, kind):
    need = ctypes.c_size_t(0)
    check(lib.adder_linear_fwd_workspace_bytes(rows, k, n, kind, ctypes.byref(need)), "adder_linear_fwd_workspace_bytes")
    return need.value


@functools.lru_cache(maxsize=4096)
def _bwd_bytes(rows, k, n, act, kind):
    need = ctypes.c_size_t(0)
    check(lib.adder_linear_bwd_workspace_bytes(rows, k, n, act, kind, ctypes.byref(need)), "adder_linear_bwd_workspace_bytes")
    return need.value


def as_rows(t, width):
    """``t`` as (rows, width) with neighbouring values side by side, and the stride of its rows: a view where it is one."""
    rows = t.numel() // width
    if t.dim() != 2:
        t = t.reshape(rows, width)
    stride = t.stride(0)
    if (t.stride(1) != 1 and width > 1) or (stride < width and stride != 0 and rows > 1):
        t = t.contiguous()
        stride = width
    return t, stride if rows > 1 else width


def _forward(x, w, bias, residual, act, keep):
    """y and, with ``keep``, the values before the activation, as (rows, out_features)."""
    n, k = w.shape
    rows = x.numel() // k
    dev, kind = x.device, TYPES[x.dtype]
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    pre = torch.empty((rows, n), dtype=x.dtype, device=dev) if keep else None
    if rows == 0:
        return y, pre
    x, ldx = as_rows(x, k)
    ldr = 0
    if residual is not None:
        residual, ldr = as_rows(residual, n)
    need = _fwd_bytes(rows, k, n, kind)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with on_device(dev):
        check(lib.adder_linear_fwd(x.data_ptr(), ldx, w.data_ptr(), ptr(bias), ptr(residual), ldr, y.data_ptr(), ptr(pre), act, rows, k, n,
                                   kind, ptr(ws), need, stream_ptr(dev)), "adder_linear_fwd")
    return y, pre


class _linear_act(Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act):
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, pre = _forward(x, w, bias, residual, act, keep)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, w if ctx.needs_input_grad[0] else None, pre)
        ctx.act, ctx.dims, ctx.x_shape = act, (x.numel() // w.shape[1], w.shape[1], w.shape[0]), x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, pre = ctx.saved_tensors
        rows, k, n = ctx.dims
        dev, dtype = dy.device, dy.dtype
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        gr = dy if want_r else None
        if not (want_x or want_w or want_b):
            return None, None, None, gr, None
        make = torch.zeros if rows == 0 else torch.empty
        gx = make(ctx.x_shape, dtype=dtype, device=dev) if want_x else None
        gw = make((n, k), dtype=dtype, device=dev) if want_w else None
        gb = make(n, dtype=dtype, device=dev) if want_b else None
        if rows == 0:
            return gx, gw, gb, gr, None
        dy, ldd = as_rows(dy, n)
        ldx = k
        if want_w:
            x, ldx = as_rows(x, k)
        kind = TYPES[dtype]
        need = _bwd_bytes(rows, k, n, ctx.act, kind)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        with on_device(dev):
            check(lib.adder_linear_bwd(dy.data_ptr(), ldd, ptr(pre), ptr(x), ldx, ptr(w), ptr(gx), ptr(gw), ptr(gb), ctx.act, rows, k, n,
                                       kind, ptr(ws), need, stream_ptr(dev)), "adder_linear_bwd")
        return gx, gw, gb, gr, None


def _torch_linear_act(x, weight, bias, residual, act):
    y = F.linear(x, weight, bias)
    y = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}[act](y)
    return y if residual is None else y + residual


def linear_act(x, weight, bias=None, residual=None, act="none"):
    """``act(x @ weight.T + bias) + residual`` with ``x`` (..., in_features), ``weight`` (out_features, in_features), ``bias``
    (out_features) or None, ``residual`` None or of any shape that broadcasts to the result's, and ``act`` one of "none", "relu",
    "gelu" (by the error function) and "silu"."""
    if act not in ACTS:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    if weight.dim() != 2:
        raise RuntimeError(f"weight must have two dimensions, got {tuple(weight.shape)}")
    n, k = weight.shape
    if x.dim() == 0 or x.shape[-1] != k:
        raise RuntimeError(f"x has shape {tuple(x.shape)} but the weight expects {k} features")
    if bias is not None and tuple(bias.shape) != (n,):
        raise RuntimeError(f"bias must have shape ({n},), got {tuple(bias.shape)}")
    tensors = [t for t in (x, weight, bias, residual) if t is not None]
    for t in tensors:
        if t.device != x.device:
            raise RuntimeError("all tensors must be on the same device")
        if t.dtype != x.dtype:
            raise RuntimeError(f"all tensors must have the type of x, {x.dtype}, got {t.dtype}")
    shape = x.shape[:-1] + (n,)
    if residual is not None and residual.shape != shape:
        try:
            residual = residual.expand(shape)
        except RuntimeError:
            raise RuntimeError(f"residual of shape {tuple(residual.shape)} does not broadcast to {tuple(shape)}") from None
    if not x.is_cuda or x.dtype not in TYPES or n == 0 or k == 0:
        return _torch_linear_act(x, weight, bias, residual, act)
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if plain_call(x):
        return _forward(x, weight, bias, residual, ACTS[act], False)[0]
    return _linear_act.apply(x, weight, bias, residual, ACTS[act])


class LinearAct(nn.Linear):
    """``nn.Linear`` (same parameters and state_dict keys) with the activation behind it and, in the call, a shortcut that is added to
    the result: ``layer(x, residual=shortcut)``.  float32 parameters are rounded to bfloat16 for a bfloat16 input."""

    def __init__(self, in_features, out_features, bias=True, act="none", device=None, dtype=None):
        if act not in ACTS:
            raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.act = act

    def forward(self, x, residual=None):
        w, b = self.weight, self.bias
        if x.dtype == torch.bfloat16 and w.dtype == torch.float32:
            w, b = w.to(x.dtype), None if b is None else b.to(x.dtype)
        return linear_act(x, w, b, residual=residual, act=self.act)

    def extra_repr(self):
        return f"{super().extra_repr()}, act={self.act}"
