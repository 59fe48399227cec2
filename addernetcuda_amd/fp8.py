"""Layers that serve in 8 bits: values as e4m3 codes (``torch.float8_e4m3fn``) with a float32 scale for each block of 128 neighbouring values of a row,
and of 128 x 128 values of a weight.  A code stands for ``code * scale``; a block's largest magnitude (at least 2^-100) has the largest code, 448.

    codes, scales = quantize(x)                        # of activations; quantize(z, gate="silu"): of silu(first half) * second half
    codes, scales, s = rms_norm_fp8(x, w, residual=r)  # of the RMS norm of s = x + r
    w8, w8_scales = quantize_weight(weight)
    y = linear_fp8(codes, scales, w8, w8_scales, bias, residual=r)
    serve_fp8(net)                                     # the gated blocks of a network (models.GatedMLP), in place

The product is csrc/fp8_product.hip (the 8-bit matrix instructions; block sums are scaled and added up in 32 bits), the codes csrc/fp8.hip and
csrc/rms_norm.hip.  There are no gradients through codes: a call that would need one raises.  float32 and bfloat16 values; CPU tensors, other
types, tensor subclasses and calls that something records, traces or transforms go through torch's own operators.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ._lib import nodes, plain_tensors
from .gated import _TORCH_ACTS, GatedLinear
from .linear import ACTS, TYPES, _torch_linear_act
from .rms_norm import RMSNorm, _eps, _in_autocast, _torch_rms_norm

BLOCK = 128   # ADDER_CODE_BLOCK
TOP, LEAST = 448.0, 2.0 ** -100
CODES = torch.float8_e4m3fn


def _no_gradients(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or on detached tensors")


def _largest(v, dims):
    """Of the magnitudes that are numbers."""
    return torch.where(v.isnan(), 0.0, v.abs()).amax(dims)


def _torch_codes(v, largest, spread):
    top = largest.float().clamp(min=LEAST)
    most = torch.full_like(top, TOP)   # (a number over a tensor is rounded twice, and a tensor on the GPU over a number multiplied by the reciprocal)
    return (v.float() * spread(most / top)).to(CODES), top / most


def _torch_quantize(x):
    b = F.pad(x, (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    q, s = _torch_codes(b, _largest(b, -1), lambda t: t.unsqueeze(-1))
    return q.flatten(-2)[..., :x.shape[-1]].contiguous(), s


def quantize(x, gate=None):
    """Codes of ``x`` (..., width) and scales (..., ceil(width / 128)).  ``gate``: an activation; the codes are of ``act(first half) * second half`` of the last
    dimension."""
    if gate is not None and gate not in ACTS:
        raise ValueError(f"gate must be None or one of {tuple(ACTS)}, got {gate!r}")
    if x.dim() == 0 or (gate is not None and x.shape[-1] % 2):
        raise RuntimeError(f"x must have a last dimension{'' if gate is None else ' of two halves'}, got {tuple(x.shape)}")
    if plain_tensors(x) and x.is_cuda and x.dtype in TYPES and x.shape[-1]:
        return nodes().quantize(x, -1 if gate is None else ACTS[gate])
    _no_gradients("quantize", x)
    if gate is not None:
        a, b = x.float().chunk(2, -1)
        x = _TORCH_ACTS[gate](a) * b
    return _torch_quantize(x)


def quantize_weight(weight):
    """Codes of ``weight`` (out_features, in_features) and scales (ceil(out_features / 128), ceil(in_features / 128))."""
    if weight.dim() != 2 or not weight.numel():
        raise RuntimeError(f"weight must have two dimensions that are not empty, got {tuple(weight.shape)}")
    if plain_tensors(weight) and weight.is_cuda and weight.dtype in TYPES:
        return nodes().quantize_weight(weight)
    _no_gradients("quantize_weight", weight)
    n, k = weight.shape
    b = F.pad(weight, (0, -k % BLOCK, 0, -n % BLOCK)).unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
    q, s = _torch_codes(b, _largest(b, (1, 3)), lambda t: t[:, None, :, None])
    return q.flatten(2).flatten(0, 1)[:n, :k].contiguous(), s


def _spread(scale, n):
    return scale.repeat_interleave(BLOCK, -1)[..., :n]


def values(codes, scale):
    """The float32 values that codes stand for; ``scale`` as ``quantize`` gives it, or as ``quantize_weight`` does."""
    width = codes.shape[-1]
    if scale.dim() == 2 and codes.dim() == 2 and scale.shape[0] != codes.shape[0]:
        scale = scale.repeat_interleave(BLOCK, 0)[:codes.shape[0]]
    return codes.float() * _spread(scale, width)


def rms_norm_fp8(x, weight=None, eps=1e-6, residual=None):
    """``rms_norm.rms_norm`` with its result as codes: ``(codes, scales)``, or with a residual ``(codes, scales, x + residual)``."""
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        x, weight, residual = _in_autocast(x, weight, residual)
    eps = _eps(eps, x)
    if plain_tensors(x, weight, residual) and x.is_cuda and x.dtype in TYPES and x.shape[-1:] != (0,):
        return nodes().rms_norm_fp8(x, weight, eps, residual)
    _no_gradients("rms_norm_fp8", x, weight, residual)
    if residual is None:
        return _torch_quantize(_torch_rms_norm(x, weight, eps, None))
    y, s = _torch_rms_norm(x, weight, eps, residual)
    return (*_torch_quantize(y), s)


def linear_fp8(x, x_scale, weight, weight_scale, bias=None, residual=None, act="none", dtype=torch.bfloat16):
    """``act(x @ weight.T + bias) + residual`` of the values that codes stand for: ``x`` (..., in_features) with ``x_scale`` as ``quantize`` gives them,
    ``weight`` (out_features, in_features) with ``weight_scale`` as ``quantize_weight`` does; ``bias``, ``residual`` (of any shape that broadcasts to
    the result's) and the result have ``dtype``, bfloat16 or float32."""
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    if dtype not in TYPES:
        raise ValueError(f"dtype must be one of {tuple(TYPES)}, got {dtype}")
    if plain_tensors(x, x_scale, weight, weight_scale, bias, residual) and x.is_cuda and weight.numel():
        return nodes().linear_fp8(x, x_scale, weight, weight_scale, bias, residual, code, TYPES[dtype])
    _no_gradients("linear_fp8", x, x_scale, weight, weight_scale, bias, residual)
    if weight.dim() != 2 or tuple(x.shape[-1:]) != tuple(weight.shape[1:]):
        raise RuntimeError(f"x has shape {tuple(x.shape)} but the weight has {tuple(weight.shape)}")
    blocks = -(-weight.shape[1] // BLOCK)
    if tuple(x_scale.shape) != (*x.shape[:-1], blocks) or tuple(weight_scale.shape) != (-(-weight.shape[0] // BLOCK), blocks):
        raise RuntimeError(f"scales of shape {tuple(x_scale.shape)} and {tuple(weight_scale.shape)} do not fit {tuple(x.shape)} and {tuple(weight.shape)}")
    w = weight.float() * _spread(weight_scale.repeat_interleave(BLOCK, 0)[:weight.shape[0]], weight.shape[1])
    y = _torch_linear_act(x.float() * _spread(x_scale, x.shape[-1]), w, None if bias is None else bias.float(), None, act)
    return (y if residual is None else y + residual.float()).to(dtype)


class LinearFp8(nn.Module):
    """A linear layer that serves in 8 bits: ``linear.LinearAct``'s arguments and call.  The weight is held as codes and scales (buffers), rounded once by
    ``LinearFp8.of(layer)``; the input is rounded in the call, or comes as the pair ``(codes, scales)`` that ``quantize`` or ``rms_norm_fp8`` gave.
    ``gate``: an activation; the input has 2 in_features values, and ``act(first half) * second half`` is what the layer takes.  The
    result has the type of the residual, of the input, or bfloat16 where that comes as codes: 2^-8, on the way to the next codes' 2^-4.  Types that the
    product does not have are rounded from its float32."""

    def __init__(self, in_features, out_features, bias=True, act="none", gate=None, device=None):
        for name, value in (("act", act), ("gate", gate)):
            if value not in ACTS and (name, value) != ("gate", None):
                raise ValueError(f"{name} must be one of {tuple(ACTS)}, got {value!r}")
        super().__init__()
        self.in_features, self.out_features, self.act, self.gate = in_features, out_features, act, gate
        self.register_buffer("weight", torch.zeros(out_features, in_features, device=device).to(CODES))
        self.register_buffer("weight_scale", torch.ones(-(-out_features // BLOCK), -(-in_features // BLOCK), device=device))
        self.register_buffer("bias", torch.zeros(out_features, device=device) if bias else None)

    def _apply(self, fn, recurse=True):
        """``to(...)``, ``half()`` and the like move codes and scales and leave their types: a code of another type would be another number."""
        def moved(t):
            r = fn(t)
            return r if r.dtype == t.dtype else t.to(r.device)
        return super()._apply(moved, recurse)

    @classmethod
    def of(cls, layer, gate=None):
        """From an ``nn.Linear`` or ``LinearAct`` (its activation is kept)."""
        if isinstance(layer, GatedLinear):
            raise ValueError("a gated layer's halves meet where the layer behind it takes its input: serve_fp8 makes both")
        return cls._holding(layer, getattr(layer, "act", "none"), gate)

    @classmethod
    @torch.no_grad()
    def _holding(cls, layer, act, gate=None):
        made = cls(layer.in_features, layer.out_features, layer.bias is not None, act, gate, device=layer.weight.device)
        made.weight, made.weight_scale = quantize_weight(layer.weight.detach())
        if layer.bias is not None:
            made.bias = layer.bias.detach().float().clone()
        return made.train(layer.training)

    def forward(self, x, residual=None):
        if isinstance(x, tuple):
            codes, scale = x
            dtype = torch.bfloat16 if residual is None else residual.dtype
        else:
            codes, scale = quantize(x, self.gate)
            dtype = x.dtype if residual is None else residual.dtype
        made = dtype if dtype in TYPES else torch.float32   # (the product has no others)
        bias = None if self.bias is None else self.bias.to(made)
        return linear_fp8(codes, scale, self.weight, self.weight_scale, bias, None if residual is None else residual.to(made), self.act, made).to(dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, act={self.act}, gate={self.gate}"


class RMSNormFp8(nn.Module):
    """``rms_norm.RMSNorm`` whose result is codes: ``(codes, scales)``, what ``LinearFp8`` takes; with a residual ``((codes, scales), x + residual)``."""

    def __init__(self, norm):
        super().__init__()
        self.eps, self.width = norm.eps, norm.normalized_shape[0]
        self.register_buffer("weight", None if norm.weight is None else norm.weight.detach().clone())

    def forward(self, x, residual=None):
        w = self.weight if self.weight is None or x.dtype == torch.bfloat16 else self.weight.to(x.dtype)   # (as RMSNorm: float32 beside bfloat16 too)
        got = rms_norm_fp8(x, w, self.eps, residual)
        return got if residual is None else (got[:2], got[2])


def serve_fp8(net):
    """The gated blocks (``models.GatedMLP``) of a network in 8 bits, in place: the norm gives codes, the products take codes and give values, the gate's
    product becomes codes on its way to the second.  For inference: call the network under ``torch.no_grad()``.  Returns the network."""
    from .models import GatedMLP
    blocks = [m for m in net.modules() if isinstance(m, GatedMLP) and isinstance(m.norm, RMSNorm)]
    if not blocks:
        raise ValueError("serve_fp8: no gated block in this network")
    for block in blocks:
        gate = block.gated.act
        # (the first product gives both halves' sums: the gate is applied where they become codes)
        block.norm, block.gated, block.down = RMSNormFp8(block.norm), LinearFp8._holding(block.gated, "none"), LinearFp8.of(block.down, gate=gate)
    return net
