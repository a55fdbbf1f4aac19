"""The output head of the reference's LlamaModel (ueaj/model/model.py:84-97 and get_logits,
140-165): final RMSNorm, the lm_head Einsum "bnd,dv->bnv" (zeros_init, sharding (None, 'tensor'))
and the optional soft cap 15 * tanh(logits / 15), with the next-token loss fused behind it.

`get_logits` computes what the reference's does (norm -> FP8 lm_head -> cap), bf16 logits out.
`token_loss` is the fused path chunked_softmax_cross_entropy takes for this head: one autograd node
that never hands the logits to the caller:
  forward   ufp8_rmsnorm_quant (norm output written straight as the e4m3 GEMM operand), e4m3
            quantisation of the weight, the lm_head GEMM with the XENT epilogue (bf16 logits, soft
            cap, per-row softmax partials), ufp8_xent_combine (lse, masked loss);
  backward  ufp8_xent_backward (fp8 logit gradient, scale from the per-row results), the two FP8
            GEMMs dX = dL W^T and dW = X^T dL, ufp8_rmsnorm_backward.
The logits are kept from the forward for the backward (2 bytes per logit in HBM) instead of being
recomputed, which the reference's rematerialised chunks do (one GEMM of 2 T d V FLOPs fewer).

`token_logprobs` and `distillation_loss` put the operators of logprobs.py and distill.py behind the
same head (the teacher's targets, the scores of sampled tokens, the student's step): one node of the
same kind, whose backward writes the operator's logit gradient straight as fp8 (e5m2: scale from the
rows' results; an e4m3 bwd_dtype: from the gradient's largest value, one more pass over the logits) and
runs the two FP8 GEMMs and the norm's backward.
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional

import torch

from . import ops
from .configurator import config
from .einsum import Einsum, Rngs, zeros_init
from .distill import check_teacher, topk_distillation_loss
from .logprobs import (TokenLogprobs, check_ids, check_logits, check_mask, check_score, check_tangents,
                       check_temperature, first_order, token_logprobs)
from .rmsnorm import RMSNorm

HEAD_CAP = 15.0  # the constant of ueaj/model/model.py:163


class _HeadXentFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2d, scale, w, labels, mask, centered, eps, cap, bwd_fmt):
        loss, saved = ops.head_xent_forward(x2d, scale, centered, eps, w, labels, mask, cap)
        ctx.saved = saved
        ctx.save_for_backward(x2d, labels, mask)
        ctx.scale, ctx.centered, ctx.cap, ctx.bwd_fmt = scale, centered, cap, bwd_fmt
        return loss

    @staticmethod
    def backward(ctx, dloss):
        x2d, labels, mask = ctx.saved_tensors
        rstd = ctx.saved[1]
        need_dw = ctx.needs_input_grad[2]
        dxn, dw = ops.head_xent_backward(dloss.to(torch.float32).contiguous(), ctx.saved, labels, mask, ctx.cap,
                                         need_dw, ctx.bwd_fmt)
        ctx.saved = None
        need_ds = ctx.scale is not None and ctx.needs_input_grad[1]
        dx, ds = ops.rmsnorm_backward(x2d, ctx.scale, ctx.centered, rstd, dxn, need_ds)
        dscale = ds.reshape(ctx.scale.shape).to(torch.bfloat16) if need_ds else None
        return dx, dscale, dw, None, None, None, None, None, None


class _HeadRowsFn(torch.autograd.Function):
    """Head -> operator on its logits.  `op` is a _Score or _Distill: forward(logits, want_stats) ->
    (outputs, stats), backward(logits, stats, ids, grads, head) with the integer outputs `ids`."""

    @staticmethod
    def forward(ctx, x2d, scale, w, op, centered, eps, cap, bwd_fmt):
        logits, (qx, rstd, qw) = ops.head_rows_forward(x2d, scale, centered, eps, w, cap)
        out, stats = op.forward(logits[:, :w.shape[1]], True)
        ids = [t for t in out if t is not None and not t.is_floating_point()]
        ctx.mark_non_differentiable(*ids)
        ctx.set_materialize_grads(False)
        # all tensors through autograd, which frees them after the backward, notices a change in place and
        # lets saved-tensor hooks move them; ctx.op keeps none
        ctx.save_for_backward(x2d, scale, logits, stats, rstd, qx.q, qx.inv_scale, qx.amax, qw.q, qw.inv_scale, qw.amax,
                              *ids, *op.tensors())
        ctx.op, ctx.n_ids, ctx.V = op.with_tensors(*(None,) * len(op.tensors())), len(ids), w.shape[1]
        ctx.centered, ctx.cap, ctx.bwd_fmt = centered, cap, bwd_fmt
        return out

    @staticmethod
    @first_order
    def backward(ctx, *grads):
        if all(g is None for g in grads):
            return (None,) * 8
        x2d, scale, logits, stats, rstd, *rest = ctx.saved_tensors
        qx, qw, ids = ops.Fp8Tensor(*rest[:3]), ops.Fp8Tensor(*rest[3:6]), rest[6:6 + ctx.n_ids]
        op = ctx.op.with_tensors(*rest[6 + ctx.n_ids:])
        dxn, dw = ops.head_rows_backward(lambda lg, head: op.backward(lg, stats, ids, grads, head), logits,
                                         (qx, rstd, qw), ctx.V, ctx.cap, ctx.needs_input_grad[2], ctx.bwd_fmt)
        need_ds = scale is not None and ctx.needs_input_grad[1]
        dx, ds = ops.rmsnorm_backward(x2d, scale, ctx.centered, rstd, dxn, need_ds)
        dscale = ds.reshape(scale.shape).to(torch.bfloat16) if need_ds else None
        return dx, dscale, dw, None, None, None, None, None


class _Score(NamedTuple):
    tokens: Optional[torch.Tensor]
    mask: Optional[torch.Tensor]
    top_k: int
    temperature: float
    entropy: bool

    def tensors(self):
        return self.tokens, self.mask

    def with_tensors(self, tokens, mask):
        return self._replace(tokens=tokens, mask=mask)

    def forward(self, logits, want_stats):
        *out, stats = ops.token_logprobs_forward(logits, self.tokens, self.mask, self.top_k, self.temperature,
                                                 self.entropy, want_stats)
        return tuple(out), stats

    def backward(self, logits, stats, ids, grads, head):
        dlp, dent, dtop, _ = grads
        return ops.token_logprobs_backward(logits, stats, self.tokens, self.mask, self.temperature, dlp, dent, dtop,
                                           ids[0] if ids else None, head)


class _Distill(NamedTuple):
    ids: torch.Tensor
    teacher: torch.Tensor
    mask: Optional[torch.Tensor]
    temperature: float

    def tensors(self):
        return self.ids, self.teacher, self.mask

    def with_tensors(self, ids, teacher, mask):
        return self._replace(ids=ids, teacher=teacher, mask=mask)

    def forward(self, logits, want_stats):
        loss, stats = ops.distill_forward(logits, self.ids, self.teacher, self.mask, self.temperature, want_stats)
        return (loss,), stats

    def backward(self, logits, stats, ids, grads, head):
        return ops.distill_backward(logits, stats, self.ids, self.teacher, self.mask, self.temperature, grads[0], head)


@config
class OutputHead(torch.nn.Module):
    """Final norm + lm_head + soft cap of LlamaModel (ueaj/model/model.py:84-97, 140-165)."""

    def __init__(self, model_d: int, vocab_size: int, norm: Callable = RMSNorm, lm_head: Callable = Einsum,
                 head_cap: Optional[str] = "tanh", *, rngs: Rngs, mesh=None):
        super().__init__()
        if head_cap not in (None, "tanh"):
            raise ValueError(f"head_cap must be None or 'tanh', got {head_cap!r}")
        self.model_d, self.vocab_size, self.head_cap = model_d, vocab_size, head_cap
        self.norm = norm(model_d=model_d, rngs=rngs, mesh=mesh)
        self.lm_head = lm_head("bnd,dv->bnv", size_dict={"d": model_d, "v": vocab_size}, initializer=zeros_init,
                               rngs=rngs, dtype=torch.bfloat16, mesh=mesh, sharding=(None, "tensor"))

    def get_logits(self, activations: torch.Tensor) -> torch.Tensor:
        """LlamaModel.get_logits: norm -> lm_head -> 15 * tanh(logits / 15) (bf16 arithmetic)."""
        logits = self.lm_head(self.norm(activations))
        if self.head_cap == "tanh":
            logits = HEAD_CAP * torch.tanh(logits / HEAD_CAP)
        return logits

    def forward(self, activations: torch.Tensor) -> torch.Tensor:
        return self.get_logits(activations)

    def fused(self) -> bool:
        """True when token_loss can run the fused norm -> FP8 lm_head -> loss node."""
        lm, nm = self.lm_head, self.norm
        return (isinstance(nm, RMSNorm) and (nm.scale is None or nm.scale.dtype == torch.bfloat16) and
                isinstance(lm, Einsum) and lm.einsum_expr == "bnd,dv->bnv" and lm.static_scale is None and
                lm.fwd_dtype == torch.float8_e4m3fn and getattr(lm, "shard", None) is None)

    def token_loss(self, activations: torch.Tensor, targets: torch.Tensor,
                   mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Per-token loss (f32 [batch, seq]) = softmax_cross_entropy(get_logits(a), targets) * mask,
        through the fused node (fused() must hold)."""
        if not self.fused():
            raise ValueError("token_loss: this head is not the fused RMSNorm + FP8 Einsum combination")
        lead = activations.shape[:-1]
        self._check_width(activations, "token_loss")
        x2d = activations.to(torch.bfloat16).reshape(-1, self.model_d).contiguous()
        labels = targets.reshape(-1).to(torch.int32).contiguous()
        mk = None if mask is None else mask.reshape(-1).to(torch.uint8).contiguous()
        w = self.lm_head.w if self.lm_head.w.dtype == torch.bfloat16 else self.lm_head.w.to(torch.bfloat16)
        cap = HEAD_CAP if self.head_cap == "tanh" else 0.0
        loss = _HeadXentFn.apply(x2d, self.norm.scale, w, labels, mk, self.norm.recenter, self.norm.eps, cap,
                                 ops.FMT_OF_DTYPE[self.lm_head.bwd_dtype])
        return loss.reshape(lead)

    def check_whole(self, who: str) -> None:
        """With the lm_head's columns split over ranks (Einsum.reshard) the logits here are this rank's part."""
        shard = getattr(self.lm_head, "shard", None)
        if shard is not None:
            raise NotImplementedError(f"{who}: the lm_head holds part {shard[1]} of {shard[2]} of the vocabulary; "
                                      f"results over all of it are not implemented")

    def _check_width(self, activations: torch.Tensor, who: str) -> None:
        """Another width flattens to another number of rows than the tokens, ids and masks have."""
        if activations.shape[-1:] != (self.model_d,):
            raise ValueError(f"{who}: activations {tuple(activations.shape)}, expected [..., {self.model_d}]")

    def _rows(self, activations: torch.Tensor, op, who: str):
        """op's outputs on the logits of the flattened activations, through the fused node."""
        x2d = activations.to(torch.bfloat16).reshape(-1, self.model_d).contiguous()
        w = self.lm_head.w if self.lm_head.w.dtype == torch.bfloat16 else self.lm_head.w.to(torch.bfloat16)
        cap = HEAD_CAP if self.head_cap == "tanh" else 0.0
        scale = self.norm.scale
        check_tangents(who, x2d, scale, w)
        if any(t is not None and t.device != x2d.device for t in (scale, w)):
            raise ValueError(f"{who}: activations on {x2d.device}, the head on {w.device}")
        if x2d.device.index != torch.cuda.current_device():  # the norm and the GEMMs launch on the current device
            with torch.cuda.device(x2d.device):
                return self._rows(activations, op, who)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x2d, scale, w)):
            return _HeadRowsFn.apply(x2d, scale, w, op, self.norm.recenter, self.norm.eps, cap,
                                     ops.FMT_OF_DTYPE[self.lm_head.bwd_dtype])
        logits, _ = ops.head_rows_forward(x2d, scale, self.norm.recenter, self.norm.eps, w, cap)
        return op.forward(logits[:, :self.vocab_size], False)[0]

    def token_logprobs(self, activations: torch.Tensor, tokens: Optional[torch.Tensor] = None, *, top_k: int = 0,
                       temperature: float = 1.0, mask: Optional[torch.Tensor] = None,
                       entropy: bool = True) -> TokenLogprobs:
        """logprobs.token_logprobs(self.get_logits(activations), ...), through the fused node when
        fused() holds (then the gradients reach the activations, the norm and the lm_head)."""
        who, lead = "OutputHead.token_logprobs", activations.shape[:-1]
        self.check_whole(who)
        self._check_width(activations, who)
        if not self.fused():
            return token_logprobs(self.get_logits(activations), tokens, top_k=top_k, temperature=temperature, mask=mask,
                                  entropy=entropy)
        check_logits(activations, who)
        temperature = check_score(tokens, top_k, self.vocab_size, temperature, entropy, who)
        if tokens is not None:
            tokens = check_ids(tokens, lead, activations, "tokens", who).reshape(-1)
        mask = check_mask(mask, activations, who)
        op = _Score(tokens, None if mask is None else mask.reshape(-1), top_k, temperature, entropy)
        lp, ent, top_lp, top_id = self._rows(activations, op, who)
        return TokenLogprobs(None if lp is None else lp.reshape(lead), None if ent is None else ent.reshape(lead),
                             None if top_lp is None else top_lp.reshape(*lead, top_k),
                             None if top_id is None else top_id.reshape(*lead, top_k))

    def distillation_loss(self, activations: torch.Tensor, teacher_ids: torch.Tensor, teacher_logits: torch.Tensor, *,
                          temperature: float = 1.0, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """distill.topk_distillation_loss(self.get_logits(activations), ...), through the fused node when
        fused() holds."""
        who, lead = "OutputHead.distillation_loss", activations.shape[:-1]
        self.check_whole(who)
        self._check_width(activations, who)
        if not self.fused():
            return topk_distillation_loss(self.get_logits(activations), teacher_ids, teacher_logits,
                                          temperature=temperature, mask=mask)
        check_logits(activations, who)
        temperature = check_temperature(temperature, who)
        ids, teacher = check_teacher(teacher_ids, teacher_logits, activations, who)
        mask = check_mask(mask, activations, who)
        rows = (lead.numel(), ids.shape[-1])  # no -1, which fits any number of rows of no entries
        op = _Distill(ids.reshape(rows), teacher.reshape(rows), None if mask is None else mask.reshape(-1),
                      temperature)
        return self._rows(activations, op, who)[0].reshape(lead)
