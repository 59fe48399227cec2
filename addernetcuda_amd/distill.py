"""The loss against a teacher's top logits: a student learns from the K largest logits that a teacher had for a row, and from the row's label.

    q = softmax(logits / T),  o = softmax(logits),  p = softmax(top_logits / T) over the K
    row = alpha T^2 sum_k p_k (log p_k - log q[top_classes_k]) - (1 - alpha) log o[label],   loss = mean over the rows that count

csrc/distill.hip: the logits are read once for the loss and, where rows are many, its gradient.  Arguments and the autograd node are
csrc/nodes_blocks.cpp.  float32 and bfloat16 logits (the loss is float32); CPU tensors, other types, tensor subclasses, more than 1024 top
logits and calls that something records, traces or transforms go through torch's own operators.
"""
import torch
import torch.nn.functional as F

from ._lib import nodes, plain_tensors
from .linear import TYPES

TOP_MOST = 1024   # ADDER_DISTILL_TOP_MAX


def _at(values, classes, exist):
    """``values`` (rows, classes) at ``classes``; not a number, for the row's gradient too, where one of a row's does not exist."""
    found = values.gather(1, torch.where(exist, classes, 0))
    return found * torch.where(exist.all(1, keepdim=True), 1.0, torch.nan).to(values.dtype)


def _torch_distillation_loss(logits, top_logits, top_classes, labels, temperature, alpha, ignore_index):
    logits, top = logits.float() if logits.dtype in (torch.bfloat16, torch.float16) else logits, top_logits.detach()
    top = top.to(logits.dtype)
    keep = torch.ones(logits.shape[0], dtype=torch.bool, device=logits.device) if labels is None else labels != ignore_index
    exists = lambda classes: (classes >= 0) & (classes < logits.shape[1])
    counts = keep.unsqueeze(1)
    logits = torch.where(counts, logits, 0.0)   # (whatever a row that does not count holds reaches neither the loss nor a gradient)
    there = counts & (top != -torch.inf)        # (one that is no number is)
    top = torch.where(there.any(1, keepdim=True), torch.where(counts, top, 0.0), 0.0)
    log_p = F.log_softmax(top / temperature, 1)
    p = torch.where(there, log_p.exp(), 0.0)
    log_q = _at(F.log_softmax(logits / temperature, 1), torch.where(there, top_classes, 0), exists(top_classes) | ~there)
    rows = temperature ** 2 * torch.where(p == 0, torch.zeros_like(p), p * (log_p - log_q)).sum(1)
    if labels is not None:
        of = torch.where(keep, labels, torch.zeros_like(labels)).unsqueeze(1)
        hard = -_at(F.log_softmax(logits, 1), of, exists(of)).squeeze(1)
        rows = hard if alpha == 0 else rows if alpha == 1 else alpha * rows + (1 - alpha) * hard
    return torch.where(keep, rows, torch.zeros_like(rows)).sum() / keep.sum().clamp(min=1)


def distillation_loss(logits, top_logits, top_classes, labels=None, temperature=1.0, alpha=0.5, ignore_index=-100):
    """The loss above of ``logits`` (rows, classes) against ``top_logits`` (rows, K; no gradient goes there) at ``top_classes`` (rows, K; int64) and, where
    given, ``labels`` (rows; int64); without labels it is the teacher's part alone, whatever ``alpha``.

    Rows with the label ``ignore_index`` do not count; where none does the loss is zero.  A top logit of -infinity adds nothing, and a row whose
    top logits all are has no teacher's part.  A class may be among the K twice.  A class that does not exist (but beside a top logit
    of -infinity, where any number may stand) makes its row's loss and gradient not a number, and so does a top logit of +infinity or one that is none."""
    if logits.dim() != 2 or top_logits.dim() != 2 or not logits.shape[1] or not top_logits.shape[1] or top_logits.shape[0] != logits.shape[0]:
        raise RuntimeError(f"logits and top_logits must be matrices of as many rows, got {tuple(logits.shape)} and {tuple(top_logits.shape)}")
    if tuple(top_classes.shape) != tuple(top_logits.shape) or top_classes.dtype != torch.int64:
        raise RuntimeError(f"top_classes must be int64 of shape {tuple(top_logits.shape)}, got {top_classes.dtype} of {tuple(top_classes.shape)}")
    if labels is not None and (tuple(labels.shape) != tuple(logits.shape[:1]) or labels.dtype != torch.int64):
        raise RuntimeError(f"labels must be int64 of shape {tuple(logits.shape[:1])}, got {labels.dtype} of {tuple(labels.shape)}")
    if any(t is not None and t.device != logits.device for t in (top_logits, top_classes, labels)):
        raise RuntimeError("all tensors must be on the same device")
    if not 0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive, got {temperature}")
    if not 0 <= alpha <= 1:
        raise ValueError(f"alpha must be between 0 and 1, got {alpha}")
    if (plain_tensors(logits, top_logits, top_classes, labels) and logits.is_cuda and logits.dtype in TYPES and top_logits.dtype in TYPES
            and top_logits.shape[1] <= TOP_MOST and logits.shape[0]):
        return nodes().distillation_loss(logits, top_logits, top_classes, labels, float(temperature), float(alpha), ignore_index)
    return _torch_distillation_loss(logits, top_logits, top_classes, labels, temperature, alpha, ignore_index)
