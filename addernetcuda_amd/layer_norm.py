"""Layer normalisation over the last dimensions of a tensor, forward and backward in one pass over the rows each
(csrc/layer_norm.hip); the gradients of weight and bias come out of the backward's pass as sums per workgroup that a second
launch adds up in a fixed order.

float32, or bfloat16 with a bfloat16 or float32 weight; sums and statistics are 32 bits.  CPU tensors and other types go through
torch's own operator.
"""
import ctypes
import functools
import math

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from ._lib import lib, check, ptr, stream_ptr, on_device, plain_call
from .linear import TYPES, as_rows


@functools.lru_cache(maxsize=4096)
def _bwd_bytes(rows, width, kind):
    need = ctypes.c_size_t(0)
    check(lib.adder_layer_norm_bwd_workspace_bytes(rows, width, kind, ctypes.byref(need)), "adder_layer_norm_bwd_workspace_bytes")
    return need.value


def _forward(x, weight, bias, width, eps, keep):
    rows = x.numel() // width
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean = torch.empty(rows, dtype=torch.float32, device=dev) if keep else None
    rstd = torch.empty(rows, dtype=torch.float32, device=dev) if keep else None
    if rows:
        x, ldx = as_rows(x, width)
        of = weight if weight is not None else bias
        with on_device(dev):
            check(lib.adder_layer_norm_fwd(x.data_ptr(), ldx, ptr(weight), ptr(bias), y.data_ptr(), ptr(mean), ptr(rstd), eps, rows, width,
                                           TYPES[x.dtype], TYPES[x.dtype if of is None else of.dtype], stream_ptr(dev)),
                  "adder_layer_norm_fwd")
    return y, mean, rstd


class _layer_norm(Function):
    @staticmethod
    def forward(ctx, x, weight, bias, width, eps):
        y, mean, rstd = _forward(x, weight, bias, width, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.width, ctx.bias = width, None if bias is None else (bias.shape, bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        width, dev = ctx.width, dy.device
        rows = x.numel() // width
        want_x, want_w, want_b = ctx.needs_input_grad[:3]
        make = torch.zeros if rows == 0 else torch.empty
        gx = make(x.shape, dtype=x.dtype, device=dev) if want_x else None
        gw = make(weight.shape, dtype=weight.dtype, device=dev) if want_w else None
        gb = make(ctx.bias[0], dtype=ctx.bias[1], device=dev) if want_b else None
        if rows:
            kind = TYPES[x.dtype]
            x, ldx = as_rows(x, width)
            dy, ldd = as_rows(dy, width)
            need = _bwd_bytes(rows, width, kind) if want_w or want_b else 0
            ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
            of = weight.dtype if weight is not None else x.dtype if ctx.bias is None else ctx.bias[1]
            with on_device(dev):
                check(lib.adder_layer_norm_bwd(dy.data_ptr(), ldd, x.data_ptr(), ldx, ptr(weight), mean.data_ptr(), rstd.data_ptr(), ptr(gx),
                                               ptr(gw), ptr(gb), rows, width, kind, TYPES[of], ptr(ws), need, stream_ptr(dev)),
                      "adder_layer_norm_bwd")
        return gx, gw, gb, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` with mean and (biased) variance over the last dimension of ``x``; over as many
    as ``weight`` (or ``bias``) has, where one is given."""
    of = weight if weight is not None else bias
    shape = tuple(of.shape) if of is not None else tuple(x.shape[-1:])
    if not shape or tuple(x.shape[-len(shape):]) != shape:
        raise RuntimeError(f"x has shape {tuple(x.shape)} but the last dimensions are to be {shape}")
    if not eps >= 0:
        raise RuntimeError(f"eps must not be negative, got {eps}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if tuple(t.shape) != shape:
            raise RuntimeError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if t.device != x.device:
            raise RuntimeError("all tensors must be on the same device")
        if t.dtype != of.dtype or not (t.dtype == x.dtype or (x.dtype, t.dtype) == (torch.bfloat16, torch.float32)):
            raise RuntimeError(f"{name} must have the type of x (or float32 beside bfloat16), {x.dtype}, got {t.dtype}")
    width = math.prod(shape)
    if not x.is_cuda or x.dtype not in TYPES or width == 0:
        if of is not None and of.dtype != x.dtype:
            return F.layer_norm(x.to(of.dtype), shape, weight, bias, eps).to(x.dtype)
        return F.layer_norm(x, shape, weight, bias, eps)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if plain_call(x):
        return _forward(x, weight, bias, width, eps, False)[0]
    return _layer_norm.apply(x, weight, bias, width, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same arguments, parameters and state_dict keys) through the kernels above."""

    def forward(self, x):
        if self.weight is None and self.bias is None and len(self.normalized_shape) > 1:
            k = len(self.normalized_shape)
            if tuple(x.shape[-k:]) != tuple(self.normalized_shape):
                raise RuntimeError(f"x has shape {tuple(x.shape)} but the last dimensions are to be {tuple(self.normalized_shape)}")
            return layer_norm(x.flatten(-k), eps=self.eps).view(x.shape)
        if self.weight is None and self.bias is None and tuple(x.shape[-1:]) != tuple(self.normalized_shape):
            raise RuntimeError(f"x has shape {tuple(x.shape)} but the last dimension is to be {self.normalized_shape[0]}")
        return layer_norm(x, self.weight, self.bias, self.eps)
