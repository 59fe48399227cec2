"""Linear layers with what surrounds them in one call: ``act(x w' + bias) + residual``.

The reference's VGG classifiers are ``nn.Linear`` - ReLU stacks (vgg.py) and leave them to the framework; the blocks of linear
layers that networks put beside adder layers add a GELU or SiLU and a shortcut.  csrc/linear*.hip computes the product on the
matrix cores and bias, activation and shortcut on its way out, so that the product's result crosses memory once; the backward
is one pass for ``dy * act'(z)`` and the bias's gradient, then the two products.  Arguments, outputs and the autograd node are
csrc/nodes.cpp.

float32 and bfloat16, all tensors of a call alike (the module rounds float32 parameters for a bfloat16 input, ``torch.autocast`` all
that the product reads).  CPU tensors, other
types, tensor subclasses and calls that something records, traces or transforms go through torch's own operators.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ._lib import nodes, plain_tensors

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}   # adder_act
TYPES = {torch.float32: 0, torch.bfloat16: 1}         # adder_type


def _plus(y, residual):
    try:
        residual = residual.expand(y.shape)
    except RuntimeError:
        raise RuntimeError(f"residual of shape {tuple(residual.shape)} does not broadcast to {tuple(y.shape)}") from None
    return y + residual


def _torch_linear_act(x, weight, bias, residual, act):
    if weight.dim() != 2:
        raise RuntimeError(f"weight must have two dimensions, got {tuple(weight.shape)}")
    y = F.linear(x, weight, bias)
    if act != "none":
        y = {"relu": F.relu, "gelu": F.gelu, "silu": F.silu}[act](y)
    return y if residual is None else _plus(y, residual)


def _autocast_linear_act(x, weight, bias, residual, act):
    """Inside ``torch.autocast``: the product in its type, as ``F.linear``'s there; a residual of another type is added behind it."""
    dtype = torch.get_autocast_dtype("cuda")
    if dtype not in TYPES or any(t is not None and t.dtype not in TYPES for t in (x, weight, bias)):
        return _torch_linear_act(x, weight, bias, residual, act)
    own = residual is None or residual.dtype == dtype
    with torch.autocast("cuda", enabled=False):
        y = linear_act(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype), residual if own else None, act)
        return y if own else _plus(y, residual)


def linear_act(x, weight, bias=None, residual=None, act="none"):
    """``act(x @ weight.T + bias) + residual`` with ``x`` (..., in_features), ``weight`` (out_features, in_features), ``bias``
    (out_features) or None, ``residual`` None or of any shape that broadcasts to the result's, and ``act`` one of "none", "relu",
    "gelu" (by the error function) and "silu".  As with torch's, the backward of "relu" without a residual reads the result: it is not
    to be edited in place before that."""
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    if plain_tensors(x, weight, bias, residual) and x.is_cuda:
        if torch.is_autocast_enabled("cuda"):
            return _autocast_linear_act(x, weight, bias, residual, act)
        if x.dtype in TYPES and weight.numel():
            return nodes().linear_act(x, weight, bias, residual, code)
    return _torch_linear_act(x, weight, bias, residual, act)


class LinearAct(nn.Linear):
    """``nn.Linear`` (same parameters and state_dict keys) with the activation behind it and, in the call, a shortcut that is added to
    the result: ``layer(x, residual=shortcut)``.  float32 parameters are rounded to bfloat16 for a bfloat16 input (inside ``torch.autocast`` to
    its type, as by ``nn.Linear``)."""

    def __init__(self, in_features, out_features, bias=True, act="none", device=None, dtype=None):
        if act not in ACTS:
            raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.act = act

    def forward(self, x, residual=None):
        w, b = self.weight, self.bias
        kind = x.device.type
        if x.dtype == torch.bfloat16 and w.dtype == torch.float32 and not (kind in ("cuda", "cpu") and torch.is_autocast_enabled(kind)):
            w, b = w.to(x.dtype), None if b is None else b.to(x.dtype)
        return linear_act(x, w, b, residual=residual, act=self.act)

    def extra_repr(self):
        return f"{super().extra_repr()}, act={self.act}"
