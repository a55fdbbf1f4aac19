"""Log probabilities of given tokens, with the entropy of every row and its top alternatives, from
logits: one kernel that reads the logits once (csrc/logprob.cu), and its gradient.

  token_logprobs(logits, tokens, top_k=..., temperature=..., mask=..., entropy=...)

scores a prompt, records what a sampler chose and among what, gives a teacher's targets for
distill.topk_distillation_loss, and is the differentiable log probability (and entropy bonus) of
training on sampled tokens.  `OutputHead.token_logprobs` calls it on the head's logits.  The reference
has no counterpart (its only use of the logits is the loss of ueaj/opt/next_token_loss.py:99-174).
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import ops

MAX_TOP_K = 256


class TokenLogprobs(NamedTuple):
    """Results over the leading shape of the logits; None where not asked for."""
    logprob: Optional[torch.Tensor]       # f32 [...]
    entropy: Optional[torch.Tensor]       # f32 [...]
    top_logprobs: Optional[torch.Tensor]  # f32 [..., top_k], descending
    top_ids: Optional[torch.Tensor]       # int64 [..., top_k]


def check_logits(logits: torch.Tensor, who: str) -> None:
    if not logits.is_cuda:
        raise ValueError(f"{who}: expected CUDA logits (this library has no CPU path)")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{who}: expected bfloat16 or float32 logits, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{who}: logits of shape {tuple(logits.shape)} have no columns")


def check_temperature(temperature: float, who: str) -> float:
    t = float(temperature)
    if not (t > 0.0) or math.isinf(t):
        raise ValueError(f"{who}: temperature must be finite and > 0, got {temperature}")
    return t


def check_score(tokens, top_k: int, V: int, temperature: float, entropy: bool, who: str) -> float:
    """What is asked of token_logprobs over V columns; returns the temperature."""
    if not 0 <= top_k <= MAX_TOP_K or top_k > V:
        raise ValueError(f"{who}: top_k must be 0..{min(MAX_TOP_K, V)}, got {top_k}")
    if tokens is None and not entropy and not top_k:
        raise ValueError(f"{who}: nothing asked for (no tokens, no entropy, top_k 0)")
    return check_temperature(temperature, who)


def check_mask(mask: Optional[torch.Tensor], logits: torch.Tensor, who: str) -> Optional[torch.Tensor]:
    """The mask as contiguous bytes, one per row: 0 leaves the row out."""
    if mask is None:
        return None
    if mask.shape != logits.shape[:-1] or mask.device != logits.device:
        raise ValueError(f"{who}: mask {tuple(mask.shape)} on {mask.device} for logits {tuple(logits.shape)} on "
                         f"{logits.device}")
    if mask.dtype not in (torch.bool, torch.uint8):
        if mask.dtype.is_floating_point or mask.dtype.is_complex:
            raise TypeError(f"{who}: the mask selects rows (bool or integer), got {mask.dtype}")
        mask = mask != 0
    return mask.contiguous()


def check_ids(ids: torch.Tensor, shape, logits: torch.Tensor, name: str, who: str) -> torch.Tensor:
    """Contiguous int32 or int64 ids of the given shape on the logits' device."""
    if ids.shape != shape or ids.device != logits.device:
        raise ValueError(f"{who}: {name} {tuple(ids.shape)} on {ids.device}, expected {tuple(shape)} on "
                         f"{logits.device}")
    if ids.dtype not in (torch.int32, torch.int64):
        if ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
            raise TypeError(f"{who}: {name} must be integers, got {ids.dtype}")
        ids = ids.to(torch.int64)
    return ids.contiguous()


def check_tangents(who: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses forward-mode derivatives, as an autograd function without one does; without the function
    (nothing requires a gradient) the results would carry no tangent, that is, a derivative of zero."""
    if forward_ad._current_level < 0:  # no dual tensors; unpack_dual says so too, in 0.9 us a tensor
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{who}: forward-mode derivatives are not implemented")


def first_order(backward):
    """once_differentiable, without its host time where no graph of the gradient is asked for."""
    once = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, top_k, temperature, entropy):
        lp, ent, top_lp, top_id, stats = ops.token_logprobs_forward(logits, tokens, mask, top_k, temperature, entropy,
                                                                    True)
        if top_k:
            ctx.mark_non_differentiable(top_id)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, mask, stats, top_id)
        ctx.temperature = temperature
        return lp, ent, top_lp, top_id

    @staticmethod
    @first_order
    def backward(ctx, dlp, dent, dtop, _):
        logits, tokens, mask, stats, top_id = ctx.saved_tensors
        if dlp is None and dent is None and dtop is None:
            return None, None, None, None, None, None
        dlogits = ops.token_logprobs_backward(logits, stats, tokens, mask, ctx.temperature, dlp, dent, dtop, top_id)
        return dlogits, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0, mask: Optional[torch.Tensor] = None,
                   entropy: bool = True) -> TokenLogprobs:
    """Of every row of `logits` [..., V] (bf16 or f32, CUDA; any strides), under the distribution
    p = softmax(logits / temperature):
      logprob       log p[token] for `tokens` [...] (integers; a negative token counts from the end, one
                    outside [-V, V) gives NaN, and its gradient is that of -log sum exp alone, as the
                    next-token loss's is: finite, so look at the result); None without tokens
      entropy       -sum_v p_v log p_v (None with entropy=False)
      top_logprobs, top_ids   the top_k (at most 256) largest logits, descending: log p and column; NaN
                    first, ties to the lowest column
    `mask` [...] (bool or integer): a row whose mask is 0 is not read; it gives 0, 0, (-inf, -1) and a
    gradient of 0.  A logit of -inf has probability 0; a row of only -inf, or holding +inf or NaN, gives
    NaN.  Arithmetic is f32; gradients reach `logits` through logprob, entropy and top_logprobs, in the
    logits' type.  Rows are read in place for up to two levels of row strides (logits[:, :-1], a padded
    pitch); logits of more levels, or with a column stride, are copied, in the forward and in the backward.
    For a next-token shift under autograd a mask of the last position is cheaper than logits[:, :-1], whose
    own backward writes the whole gradient once more.  The same call gives the same bits; the last bits of a row may differ between calls
    with other numbers of rows or another alignment, which group its sums differently."""
    who = "token_logprobs"
    check_logits(logits, who)
    check_tangents(who, logits)
    lead, V = logits.shape[:-1], logits.shape[-1]
    temperature = check_score(tokens, top_k, V, temperature, entropy, who)
    if tokens is not None:
        tokens = check_ids(tokens, lead, logits, "tokens", who)
    mask = check_mask(mask, logits, who)
    if torch.is_grad_enabled() and logits.requires_grad:
        return TokenLogprobs(*_TokenLogprobsFn.apply(logits, tokens, mask, top_k, temperature, entropy))
    return TokenLogprobs(*ops.token_logprobs_forward(logits, tokens, mask, top_k, temperature, entropy, False)[:4])
