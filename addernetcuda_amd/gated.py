"""Gated linear layers: ``act(x wg' + bg) * (x wu' + bu)``, the first half of a gated feed-forward block, as one product whose epilogue holds both
sums (csrc/linear*.hip; the backward's pass over dy is csrc/gated.hip, the products behind it the linear layers').  Arguments, outputs and the
autograd node are csrc/nodes_blocks.cpp.

float32 and bfloat16, all tensors of a call alike (the module rounds float32 parameters for a bfloat16 input, ``torch.autocast`` all that the
product reads).  CPU tensors, other types, tensor subclasses and calls that something records, traces or transforms go through torch's own
operators.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from ._lib import nodes, plain_tensors
from .linear import ACTS, TYPES

_TORCH_ACTS = {"none": lambda t: t, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def _torch_gated_linear(x, weight, bias, act):
    if weight.dim() != 2 or weight.shape[0] % 2:
        raise RuntimeError(f"weight must have two dimensions, the first of two halves, got {tuple(weight.shape)}")
    gate, up = F.linear(x, weight, bias).chunk(2, -1)
    return _TORCH_ACTS[act](gate) * up


def gated_linear(x, weight, bias=None, act="silu"):
    """``act(x @ gate.T + bg) * (x @ up.T + bu)`` with ``x`` (..., in_features), ``weight`` (2 hidden, in_features) holding ``gate`` and behind it ``up``,
    ``bias`` (2 hidden) or None, and ``act`` one of "none", "relu", "gelu" (by the error function) and "silu"."""
    code = ACTS.get(act)
    if code is None:
        raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
    if plain_tensors(x, weight, bias) and x.is_cuda:
        if torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            if dtype in TYPES and all(t is None or t.dtype in TYPES for t in (x, weight, bias)):
                with torch.autocast("cuda", enabled=False):
                    return gated_linear(x.to(dtype), weight.to(dtype), None if bias is None else bias.to(dtype), act)
        elif x.dtype in TYPES and weight.numel():
            return nodes().gated_linear(x, weight, bias, code)
    return _torch_gated_linear(x, weight, bias, act)


class GatedLinear(nn.Linear):
    """``nn.Linear(in_features, 2 * hidden)`` (its parameters and state_dict keys; the gate's rows first) whose halves make ``hidden`` values.
    float32 parameters are rounded to bfloat16 for a bfloat16 input (inside ``torch.autocast`` to its type, as by ``nn.Linear``)."""

    def __init__(self, in_features, hidden, bias=False, act="silu", device=None, dtype=None):
        if act not in ACTS:
            raise ValueError(f"act must be one of {tuple(ACTS)}, got {act!r}")
        super().__init__(in_features, 2 * hidden, bias=bias, device=device, dtype=dtype)
        self.act = act

    def forward(self, x):
        w, b = self.weight, self.bias
        kind = x.device.type
        if x.dtype == torch.bfloat16 and w.dtype == torch.float32 and not (kind in ("cuda", "cpu") and torch.is_autocast_enabled(kind)):
            w, b = w.to(x.dtype), None if b is None else b.to(x.dtype)
        return gated_linear(x, w, b, act=self.act)

    def extra_repr(self):
        return f"{super().extra_repr()}, act={self.act}"
