"""Root-mean-square normalisation over the last dimension of a tensor, with the addition of a shortcut in front of it: the sum, its norm and, in
the backward, the shortcut's own gradient in one pass over the rows each (csrc/rms_norm.hip).  Arguments, outputs and the autograd node are
csrc/nodes_blocks.cpp; the same norm with a result of 8-bit codes is ``fp8.rms_norm_fp8``.

float32, or bfloat16 with a bfloat16 or float32 weight; sums and statistics are 32 bits.  Inside ``torch.autocast`` too the result has the type of
``x`` (as torch's own), or of its sum with a residual of another type.  CPU tensors, other types, tensor subclasses and calls that something records, traces or transforms go through torch's own
operators.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ._lib import nodes, plain_tensors
from .linear import TYPES, _plus


def _check(x, weight, eps):
    if not eps >= 0:
        raise RuntimeError(f"eps must not be negative, got {eps}")
    if x.dim() == 0:
        raise RuntimeError("x must have a dimension")
    if weight is not None and tuple(weight.shape) != tuple(x.shape[-1:]):
        raise RuntimeError(f"weight must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")


def _torch_rms_norm(x, weight, eps, residual):
    _check(x, weight, eps)
    s = x if residual is None else _plus(x, residual)
    if weight is not None and weight.dtype != s.dtype:
        y = F.rms_norm(s.to(weight.dtype), s.shape[-1:], weight, eps).to(s.dtype)
    else:
        y = F.rms_norm(s, s.shape[-1:], weight, eps)
    return y if residual is None else (y, s)


def _in_autocast(x, weight, residual):
    """Inside ``torch.autocast`` types may differ: ``x`` and the residual meet in the wider, a narrower weight beside them."""
    if residual is not None and residual.dtype != x.dtype and x.is_floating_point() and residual.is_floating_point():
        wider = torch.promote_types(x.dtype, residual.dtype)
        x, residual = x.to(wider), residual.to(wider)
    if weight is not None and x.dtype == torch.float32:
        weight = weight.float()
    return x, weight, residual


def _eps(eps, x):
    """A norm's ``eps``; None: of the type that it computes in (as ``F.rms_norm``)."""
    return eps if eps is not None else torch.finfo(torch.float64 if x.dtype == torch.float64 else torch.float32).eps


def rms_norm(x, weight=None, eps=1e-6, residual=None):
    """``s / sqrt(mean(s^2) + eps) * weight`` over the last dimension of ``s``, which is ``x`` or, where a ``residual`` is given that broadcasts
    to its shape, ``x + residual``; then the result is the pair of this and ``s``.  ``eps=None``: the machine epsilon of the type that the norm is
    computed in, as ``F.rms_norm``'s."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        x, weight, residual = _in_autocast(x, weight, residual)
    eps = _eps(eps, x)
    if plain_tensors(x, weight, residual) and x.is_cuda and x.dtype in TYPES and x.shape[-1:] != (0,):
        return nodes().rms_norm(x, weight, eps, residual)
    return _torch_rms_norm(x, weight, eps, residual)


class RMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` over the last dimension, of ``width`` values (same parameters and state_dict keys; ``eps`` is 1e-6 where ``nn.RMSNorm``'s is
    None unless it is given), through the kernels above; in the call, a shortcut that is added first: ``y, s = norm(x, residual=shortcut)``."""

    def __init__(self, width, eps=1e-6, elementwise_affine=True, device=None, dtype=None):
        super().__init__(width, eps=eps, elementwise_affine=elementwise_affine, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"RMSNorm is over the last dimension, got {tuple(self.normalized_shape)}")

    def forward(self, x, residual=None):
        if tuple(x.shape[-1:]) != tuple(self.normalized_shape):
            raise RuntimeError(f"x has shape {tuple(x.shape)} but the last dimension is to be {self.normalized_shape[0]}")
        return rms_norm(x, self.weight, self.eps, residual)
