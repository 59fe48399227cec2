"""Layer normalisation over the last dimensions of a tensor, forward and backward in one pass over the rows each
(csrc/layer_norm.hip); the gradients of weight and bias come out of the backward's pass as sums per workgroup that a second
launch adds up in a fixed order.  Arguments, outputs and the autograd node are csrc/nodes.cpp.

float32, or bfloat16 with a bfloat16 or float32 weight; sums and statistics are 32 bits.  Inside ``torch.autocast`` the result is float32,
as torch's own is.  CPU tensors, other types, tensor subclasses and calls that something records, traces or transforms go through torch's own
operator.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ._lib import nodes, plain_tensors
from .linear import TYPES

_BELOW_F32 = (torch.bfloat16, torch.float16)


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` with mean and (biased) variance over the last dimension of ``x``; over as many
    as ``weight`` (or ``bias``) has, where one is given."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):   # (torch casts everything below float32 to it)
        x, weight, bias = (t.float() if t is not None and t.dtype in _BELOW_F32 else t for t in (x, weight, bias))
    of = weight if weight is not None else bias
    if plain_tensors(x, weight, bias) and x.is_cuda and x.dtype in TYPES and (of is None or of.numel()) and x.shape[-1:] != (0,):
        return nodes().layer_norm(x, weight, bias, eps)
    if not eps >= 0:
        raise RuntimeError(f"eps must not be negative, got {eps}")
    shape = tuple(of.shape) if of is not None else tuple(x.shape[-1:])
    if of is not None and of.dtype != x.dtype:
        return F.layer_norm(x.to(of.dtype), shape, weight, bias, eps).to(x.dtype)
    return F.layer_norm(x, shape, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` (same arguments, parameters and state_dict keys) through the kernels above."""

    def forward(self, x):
        if self.weight is not None or self.bias is not None:
            return layer_norm(x, self.weight, self.bias, self.eps)
        shape = tuple(self.normalized_shape)
        if tuple(x.shape[-len(shape):]) != shape:
            raise RuntimeError(f"x has shape {tuple(x.shape)} but the last dimension{'s are' if len(shape) > 1 else ' is'} to be {shape}")
        return layer_norm(x.flatten(-len(shape)), eps=self.eps).view(x.shape)
