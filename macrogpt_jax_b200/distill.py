"""Distillation from a teacher's top logits: the divergence of a student's full distribution from the
teacher's distribution over its top entries, and the gradient (csrc/logprob.cu).

  topk_distillation_loss(logits, teacher_ids, teacher_logits, temperature=..., mask=...)

The teacher's entries are what logprobs.token_logprobs(teacher_logits, top_k=...) returns (ids, and log
probabilities, which serve as logits).  `OutputHead.distillation_loss` calls it on the head's logits.
The reference has no counterpart; the loss stands next to that of ueaj/opt/next_token_loss.py:99-174.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import ops
from .logprobs import check_ids, check_logits, check_mask, check_tangents, check_temperature, first_order

MAX_ENTRIES = 1024


def check_teacher(teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, logits: torch.Tensor, who: str):
    """(ids, teacher values), contiguous, for logits (or activations) of the leading shape."""
    if teacher_ids.dim() < 1 or teacher_ids.shape[-1] > MAX_ENTRIES:
        raise ValueError(f"{who}: teacher_ids {tuple(teacher_ids.shape)}: at most {MAX_ENTRIES} entries per row")
    shape = (*logits.shape[:-1], teacher_ids.shape[-1])
    ids = check_ids(teacher_ids, shape, logits, "teacher_ids", who)
    if teacher_logits.shape != shape or teacher_logits.device != logits.device:
        raise ValueError(f"{who}: teacher_logits {tuple(teacher_logits.shape)} on {teacher_logits.device}, expected "
                         f"{shape} on {logits.device}")
    if teacher_logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{who}: expected bfloat16 or float32 teacher_logits, got {teacher_logits.dtype}")
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise ValueError(f"{who}: the teacher gets no gradient; detach teacher_logits")
    check_tangents(who, teacher_logits)
    return ids, teacher_logits.detach().contiguous()


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, mask, temperature):
        loss, stats = ops.distill_forward(logits, ids, teacher, mask, temperature, True)
        ctx.save_for_backward(logits, ids, teacher, mask, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @first_order
    def backward(ctx, dloss):
        logits, ids, teacher, mask, stats = ctx.saved_tensors
        dlogits = ops.distill_backward(logits, stats, ids, teacher, mask, ctx.temperature, dloss)
        return dlogits, None, None, None, None


def topk_distillation_loss(logits: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                           temperature: float = 1.0, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Per row of `logits` [..., V] (bf16 or f32, CUDA; strides as for token_logprobs) the f32 loss
      sum_j q_j (log q_j - log p[id_j]),   p = softmax(logits / temperature) over all V columns,
                                           q = softmax(teacher_logits / temperature) over the entries present,
    with `teacher_ids` [..., K] (integers, K <= 1024; an id < 0 marks an absent entry) and
    `teacher_logits` [..., K] (bf16 or f32; log probabilities serve as well, since q does not change
    with a constant per row).  An entry of -inf has q = 0; a row without any weight has loss 0 and
    gradient 0, and so has a row whose `mask` [...] (bool or integer) is 0, which is not read.  An id >= V
    with q > 0 gives NaN, while the gradient, which has no column for it, stays finite with the other entries'
    part: look at the loss.  A column given twice counts twice.  The gradient reaches `logits` only, in
    their type: (p_v - sum of q_j with id_j == v) / temperature; multiply the loss by temperature^2 to
    keep gradients of one size across temperatures."""
    who = "topk_distillation_loss"
    check_logits(logits, who)
    check_tangents(who, logits)
    temperature = check_temperature(temperature, who)
    ids, teacher = check_teacher(teacher_ids, teacher_logits, logits, who)
    mask = check_mask(mask, logits, who)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillFn.apply(logits, ids, teacher, mask, temperature)
    return ops.distill_forward(logits, ids, teacher, mask, temperature, False)[0]
