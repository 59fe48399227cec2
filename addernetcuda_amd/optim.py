"""``torch.optim.SGD`` (main.py:67 of the reference: momentum 0.9, weight decay 5e-4) with the update of all
parameters of a group in one launch.

A network of adder layers has many small parameters (ResNet-20: 65 tensors, 272 000 values); the framework's
fused update takes two launches of 15 us for them, csrc/sgd.hip one of 5 us.  Same update rule, same
``state_dict`` (``momentum_buffer`` per parameter), same constructor; what the kernel does not cover (Nesterov,
dampening, ``maximize``, no momentum, parameters that are not contiguous float32 GPU tensors, sparse gradients) is
left to ``torch.optim.SGD.step``.  As with the framework's fused update, a float learning rate is frozen into a
captured graph; pass the rate as a one-element float32 device tensor to change it between replays.

``AdamW`` does the same for ``torch.optim.AdamW`` (csrc/adamw.hip), with its state in 32 or in 8 bits.
"""
import ctypes

import torch

from ._lib import lib, check, nodes, stream_ptr, on_device

_MAX = 96   # ADDER_SGD_BATCH_MAX


def _torch_step(kind, optimizer, groups):
    """``kind.step`` for these groups alone.  Hooks belong to the step that this one is part of: the framework wraps a class's ``step`` once one of its
    own has been made, and would run them again."""
    step = kind.step
    if getattr(step, "hooked", False):
        step = step.__wrapped__
    kept = optimizer.param_groups
    try:
        optimizer.param_groups = groups
        step(optimizer)
    finally:
        optimizer.param_groups = kept


class SGD(torch.optim.SGD):
    def __init__(self, params, lr=1e-3, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False, *,
                 maximize=False):
        super().__init__(params, lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                         nesterov=nesterov, maximize=maximize, foreach=False, fused=False)

    @staticmethod
    def _kernel_takes(group, params):
        if group["momentum"] <= 0 or group["dampening"] != 0 or group["nesterov"] or group["maximize"]:
            return False
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and not (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1):
            return False
        dev = params[0].device
        for p in params:
            g = p.grad
            if not (p.is_cuda and p.device == dev and p.dtype == torch.float32 and p.is_contiguous()
                    and g.dtype == torch.float32 and g.device == dev and not g.is_sparse and g.is_contiguous()
                    and p.numel() > 0):
                return False
        return True

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        rest = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if not self._kernel_takes(group, params):
                rest.append(group)
                continue
            bufs = []
            for p in params:
                state = self.state[p]
                if state.get("momentum_buffer") is None:
                    # (zeros: the first update then leaves buf = grad + weight_decay * p, as torch.optim.SGD does)
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                bufs.append(state["momentum_buffer"])
            lr = group["lr"]
            lr_ptr, lr_val = (lr.data_ptr(), 0.0) if isinstance(lr, torch.Tensor) else (None, float(lr))
            dev = params[0].device
            with on_device(dev):
                for i in range(0, len(params), _MAX):
                    ps, bs = params[i:i + _MAX], bufs[i:i + _MAX]
                    k = len(ps)
                    pa = (ctypes.c_void_p * k)(*[p.data_ptr() for p in ps])
                    ga = (ctypes.c_void_p * k)(*[p.grad.data_ptr() for p in ps])
                    ba = (ctypes.c_void_p * k)(*[b.data_ptr() for b in bs])
                    na = (ctypes.c_long * k)(*[p.numel() for p in ps])
                    check(lib.adder_sgd_momentum_step_f32(k, pa, ga, ba, na, lr_ptr, lr_val, float(group["momentum"]),
                                                          float(group["weight_decay"]), stream_ptr(dev)),
                          "adder_sgd_momentum_step_f32")
        if rest:   # the groups the kernel does not take: the framework's own update, group by group
            _torch_step(torch.optim.SGD, self, rest)
        return loss


STATE_BLOCK = 256   # ADDER_STATE_BLOCK
_PIECE = 1 << 30    # values of one entry of the kernel's table; longer tensors take several
_GROUPS = (1 << 24) - 1   # workgroups, of 1024 values at least, that the entry points take in one launch
_CODES = {"exp_avg": torch.int8, "exp_avg_sq": torch.uint8}
_MOMENTS = ("exp_avg", "exp_avg_sq", "max_exp_avg_sq")   # that the framework's step holds in the parameter's type


def state_values(codes, scales, dtype=torch.float32):
    """The values that an 8-bit moment of ``AdamW`` stands for: ``codes`` int8 (``exp_avg``) or uint8 (``exp_avg_sq``), ``scales`` one float32
    per ``STATE_BLOCK`` codes; a float32 or bfloat16 tensor shaped like ``codes``."""
    if codes.dtype not in (torch.int8, torch.uint8):
        raise RuntimeError(f"codes must be int8 or uint8, got {codes.dtype}")
    if dtype not in _ADAMW_TYPES:
        raise RuntimeError(f"dtype must be float32 or bfloat16, got {dtype}")
    if not (codes.is_cuda and scales.device == codes.device):
        raise RuntimeError("codes and scales must be CUDA tensors on one device")
    n = codes.numel()
    if scales.dtype != torch.float32 or scales.numel() != -(-n // STATE_BLOCK):
        raise RuntimeError(f"scales must be {-(-n // STATE_BLOCK)} float32 values, got {scales.numel()} of {scales.dtype}")
    codes, scales = codes.contiguous(), scales.contiguous()
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    if n:
        with on_device(codes.device):
            check(lib.adder_state_values(codes.data_ptr(), int(codes.dtype == torch.int8), scales.data_ptr(), out.data_ptr(), n,
                                         _ADAMW_TYPES[dtype], stream_ptr(codes.device)), "adder_state_values")
    return out


_ADAMW_TYPES = {torch.float32: 0, torch.bfloat16: 1}   # adder_type


class AdamW(torch.optim.AdamW):
    """``torch.optim.AdamW`` with the update of all parameters of a group in one launch (csrc/adamw.hip; up to 96 tensors, or 64 with
    8-bit state), and its two moments in 32 bits or, with ``state_bits=8``, as 8-bit codes: 16 instead of 28 bytes of memory traffic a
    float32 parameter and 2 instead of 8 bytes of memory.

    Parameters: float32 or bfloat16, with gradients of their type.  With ``state_bits=32`` the state is that of ``torch.optim.AdamW``
    (float32 ``exp_avg``, ``exp_avg_sq`` whatever the parameter's type; ``step``), and what the kernel does not cover (``amsgrad``,
    ``maximize``, CPU or non-contiguous tensors, other types, sparse gradients) is left to ``torch.optim.AdamW.step``.  With
    ``state_bits=8`` tensors of at least ``min_8bit_size`` values hold ``exp_avg`` (int8) and ``exp_avg_sq`` (uint8) with float32
    ``exp_avg_scale`` and ``exp_avg_sq_scale``, one per ``STATE_BLOCK`` values (``state_values`` decodes them); smaller ones, whose state costs
    nothing, keep 32 bits, and what the kernel does not cover is an error.

    ``capturable=True`` keeps the step count on the device, so that a captured HIP graph counts on; the learning rate may then be a
    one-element float32 device tensor."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False, *, maximize=False,
                 capturable=False, state_bits=32, min_8bit_size=4096):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if state_bits == 8 and (amsgrad or maximize):
            raise ValueError("state_bits=8 takes neither amsgrad nor maximize")
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad, maximize=maximize,
                         foreach=False, fused=False, capturable=capturable)
        self.state_bits, self.min_8bit_size = state_bits, min_8bit_size

    def __getstate__(self):   # (copies and pickles: the framework's optimizer keeps its own three parts and nothing else)
        return {**super().__getstate__(), "state_bits": self.state_bits, "min_8bit_size": self.min_8bit_size}

    @staticmethod
    def _kernel_takes(group, params):
        if group["amsgrad"] or group["maximize"]:
            return False
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and not (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1):
            return False
        if any(isinstance(b, torch.Tensor) for b in group["betas"]):
            return False
        dev = params[0].device
        for p in params:
            g = p.grad
            if not (p.is_cuda and p.device == dev and g.device == dev and p.dtype in _ADAMW_TYPES and g.dtype == p.dtype
                    and p.layout == g.layout == torch.strided and p.is_contiguous() and g.is_contiguous()):
                return False
        return True

    def _new_state(self, p, step):
        state = self.state[p]
        state["step"] = step
        if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
            blocks = -(-p.numel() // STATE_BLOCK)
            for name, dtype in _CODES.items():
                state[name] = torch.zeros(p.shape, dtype=dtype, device=p.device)
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        else:
            for name in _CODES:
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state

    def load_state_dict(self, state_dict):
        """As ``torch.optim.Optimizer.load_state_dict``, but 8-bit moments stay codes, and those of parameters that the kernel takes are
        float32."""
        super().load_state_dict(state_dict)
        for group in self.param_groups:   # (the framework's fused step wants counts on the device, which the kernel's numbers are not)
            group["fused"] = group["fused"] and False
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(saved, own):
            for name, value in state_dict["state"].get(i, {}).items():
                if not isinstance(value, torch.Tensor) or name == "step":
                    continue
                if value.dtype in (torch.int8, torch.uint8):
                    self.state[p][name] = value.to(device=p.device, copy=True)
                elif (p.is_cuda and p.dtype in _ADAMW_TYPES) or name.endswith("_scale"):   # (the others have their parameter's type by now)
                    self.state[p][name] = value.to(device=p.device, dtype=torch.float32, copy=True)
        for group in self.param_groups:   # parameters of one count share its tensor again (see _kernel_step)
            if group["capturable"] and not (group["amsgrad"] or group["maximize"]):
                shared = {}
                for p in group["params"]:
                    if self.state.get(p):
                        step = float(self.state[p]["step"])
                        if step not in shared:
                            shared[step] = torch.tensor(step, dtype=torch.float32, device=p.device)
                        self.state[p]["step"] = shared[step]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        rest = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if not group["capturable"] and params[0].is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: a captured step counts on only where capturable=True keeps its count on the device")
            if self._kernel_step(group, params):
                continue
            if self._kernel_takes(group, params):
                self._make_states(group, params)
                if not self._kernel_step(group, params):
                    raise RuntimeError("AdamW: the state does not fit its parameters")
            elif self.state_bits == 8 or any(self.state[p]["exp_avg"].dtype == torch.int8 for p in params if self.state.get(p)):
                raise RuntimeError("state_bits=8 needs contiguous float32 or bfloat16 GPU parameters with gradients of their type, on one device")
            else:
                rest.append(group)
        if rest:   # the groups the kernel does not take: the framework's own update, group by group
            shared = [pair for group in rest for pair in self._as_torchs(group)]
            _torch_step(torch.optim.AdamW, self, rest)
            for count, states in shared:
                count.add_(1)
                for state in states:
                    state["step"] = count
        return loss

    def _as_torchs(self, group):
        """Prepares the states of a group for the framework's step: moments in the parameter's type, and a count of its own for each parameter, which
        the framework raises one by one.  Returns the counts on the device that were shared, with the states that go back to them."""
        self._part_counts(group)
        users = {}
        for p in group["params"]:
            state = self.state.get(p)
            if not state or p.grad is None:
                continue
            for name in _MOMENTS:
                if name in state and state[name].dtype != p.dtype:
                    state[name] = state[name].to(p.dtype)
            step = state["step"]
            if not isinstance(step, torch.Tensor):
                state["step"] = torch.tensor(float(step), device=p.device if group["capturable"] else "cpu")
            else:
                users.setdefault(id(step), (step, []))[1].append(state)
        shared = [(step, states) for step, states in users.values() if len(states) > 1]
        for step, states in shared:
            for state in states:
                state["step"] = step.clone()
        return shared if group["capturable"] else []

    def _part_counts(self, group):
        """Parameters without a gradient now do not count on with the others: those of one count have a copy of it together from here on."""
        of = self.state
        used = {id(of[p]["step"]) for p in group["params"] if p.grad is not None and of.get(p)}
        left = {}
        for p in group["params"]:
            if p.grad is None and of.get(p) and id(of[p]["step"]) in used and isinstance(of[p]["step"], torch.Tensor):
                step = of[p]["step"]
                if id(step) not in left:
                    left[id(step)] = step.clone()
                of[p]["step"] = left[id(step)]

    def _make_states(self, group, params):
        """The states of ``params`` as the kernel wants them: moments as float32 or codes, and the step count as an int or, with
        ``capturable``, as a tensor on the device that the parameters of one count share (one tiny launch counts them all)."""
        of, capturable, dev = self.state, group["capturable"], params[0].device
        fresh = torch.zeros((), dtype=torch.float32, device=dev) if capturable else 0
        counts = {}   # made here, by their value
        for p in params:
            state = of[p] or self._new_state(p, fresh)
            step = state["step"]
            if not capturable:
                state["step"] = int(step)
            elif not (isinstance(step, torch.Tensor) and step.is_cuda and step.dtype == torch.float32):
                step = float(step)
                if step not in counts:
                    counts[step] = torch.tensor(step, dtype=torch.float32, device=dev)
                state["step"] = counts[step]
            for name in _CODES:   # (what torch.optim.AdamW made for a group that it had to take before)
                if state[name].dtype not in (torch.float32, _CODES[name]):
                    state[name] = state[name].float()
        if capturable:
            self._part_counts(group)

    def _kernel_step(self, group, params):
        """The launches of one step, by csrc/nodes.cpp: False, and nothing done, where something is not as the kernels want it."""
        lr, capturable, of = group["lr"], group["capturable"], self.state
        if group["amsgrad"] or group["maximize"] or not params[0].is_cuda:
            return False
        states = [of[p] for p in params]
        if not all(states):
            return False
        if capturable and len(params) < len(group["params"]):
            used = {id(state["step"]) for state in states}
            if any(p.grad is None and of.get(p) and id(of[p]["step"]) in used for p in group["params"]):
                return False
        rate, rate_at = lr, 0
        if isinstance(lr, torch.Tensor):
            if not (lr.is_cuda and lr.dtype == torch.float32 and lr.numel() == 1 and lr.device == params[0].device):
                return False
            rate, rate_at = 0.0, lr.data_ptr()
        b1, b2 = group["betas"]
        if isinstance(b1, torch.Tensor) or isinstance(b2, torch.Tensor):
            return False
        return nodes().adamw_step(params, states, capturable, rate, rate_at, b1, b2, group["eps"], group["weight_decay"], _PIECE, _GROUPS)
