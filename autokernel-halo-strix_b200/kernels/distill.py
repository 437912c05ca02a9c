"""Distillation from a teacher's top-K log-probabilities on B200.

`distill_topk` is the loss of a student's logits against what a teacher's
`kernels.token_logprobs.token_logprobs(..., top_k=K, temperature=T)` answered: per row the K most
likely tokens and their log-probabilities.  It reads the student's logits once; with the default
mode the same pass writes their gradient, as `kernels.ce_fused` does for hard labels.

The reference trains on hard labels only (kernels/ce_fused.py:557-785).
"""
from typing import Optional

import torch

from kernels import _ak
from kernels.token_logprobs import check_scales, once

KERNEL_TYPE = "distill_topk"
BACKEND = "cuda_sm100a"

MAX_TOP_K = 128


def _distill_backward(ctx, g_loss):
    if ctx.fused:
        if ctx.consumed:
            raise RuntimeError("distill_topk: backward through the same graph twice needs mode='tiny' (the "
                               "gradient made in the forward is consumed by the first backward)")
        ctx.consumed = True
        (grad,) = ctx.saved_tensors
        _ak.scale_by_device_scalar_(grad, g_loss)
    else:
        logits, idx, rest, gk, mask, inv_n = ctx.saved_tensors
        grad = _ak.distill_topk_bwd(logits, idx, rest, gk, mask, inv_n, g_loss, *ctx.args)
    return (grad,) + (None,) * 7


class _DistillTopK(torch.autograd.Function):
    """`fused` writes the gradient in the forward and keeps it instead of the logits; `tiny` keeps the
    logits with 2 + K numbers a row and recomputes in the backward."""

    @staticmethod
    def forward(ctx, logits, idx, lp, mask, temperature, softcap, tail, fused):
        loss, _, inv_n, grad, rest, gk = _ak.distill_topk_fwd(logits, idx, lp, mask, temperature, softcap, tail,
                                                              want_grad=fused, want_stats=not fused)
        ctx.fused, ctx.args, ctx.consumed = fused, (temperature, softcap), False
        if fused:
            ctx.save_for_backward(grad)
        else:
            ctx.save_for_backward(logits, idx, rest, gk, mask, inv_n)
        return loss

    @staticmethod
    def backward(ctx, g_loss):
        return once(_distill_backward, ctx, g_loss)


def distill_topk(logits: torch.Tensor, teacher_indices: torch.Tensor, teacher_logprobs: torch.Tensor, *,
                 mask: Optional[torch.Tensor] = None, temperature: float = 1.0, softcap: float = 0.0,
                 tail: bool = False, mode: Optional[str] = None) -> torch.Tensor:
    """temperature^2 * mean over the rows of sum_k q_k (log q_k - log p_k), a scalar: KL(teacher ||
    student) where a row's tokens are all different.

    logits (..., V): the student's, fp32, bf16 or fp16 on the GPU; p = softmax(softcap(logits) /
    temperature).  Row views are read in place, as in `token_logprobs`.
    teacher_indices, teacher_logprobs (..., K), K <= 128: the teacher's tokens and their
    log-probabilities at the same temperature.  A negative index is padding; a row of padding alone
    has loss 0 and no gradient.  An index outside the vocabulary makes its row NaN.  Several entries
    of one token have a term each; their masses add up in the gradient (a constant away from the KL
    of the merged teacher).
    tail: False renormalises the teacher over its K entries; True takes exp(teacher_logprobs) as they
    are and compares the rest of both distributions as one bucket, left out where the student has
    masked it (no logit outside the teacher's tokens within 30000 of its largest) and where the
    entries' mass exceeds 1.  The gradient is that of the terms that are there, whatever mass they have.
    mask (...), bool: rows that count; the others have no gradient, whatever they hold.
    mode: "fused" writes the gradient in the forward (one read of the logits, one write) and its
    backward scales it in place, once per forward (a graph of the backward alone is replayed once per
    replay of the forward); "tiny" keeps the logits and recomputes in the backward, which rounds once
    whatever the upstream gradient is and can run twice.  Default: "tiny" for fp16, whose gradient of a mean would underflow before
    a loss scale reaches it, else "fused".
    """
    what = "distill_topk"
    _ak.dtype_code(logits)
    _ak.refuse_tangents(what, logits, teacher_logprobs)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., V) with V >= 1, got {tuple(logits.shape)}")
    lead = logits.shape[:-1]
    if teacher_indices.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: teacher_indices must be int64 or int32, got {teacher_indices.dtype}")
    _ak.dtype_code(teacher_logprobs)
    if teacher_indices.dim() < 1 or teacher_indices.shape[:-1] != lead or teacher_logprobs.shape != teacher_indices.shape:
        raise ValueError(f"{what}: teacher {tuple(teacher_indices.shape)} / {tuple(teacher_logprobs.shape)} do not match "
                         f"the rows {tuple(lead)}")
    if not 1 <= teacher_indices.shape[-1] <= MAX_TOP_K:
        raise ValueError(f"{what}: 1..{MAX_TOP_K} teacher entries a row, got {teacher_indices.shape[-1]}")
    if teacher_logprobs.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: the teacher gets no gradient; detach teacher_logprobs")
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError(f"{what}: mask must be bool, got {mask.dtype}")
        if mask.shape != lead:
            raise ValueError(f"{what}: mask {tuple(mask.shape)} does not match the rows {tuple(lead)}")
        mask = mask.contiguous()
    temperature, softcap = check_scales(what, temperature, softcap)
    if mode not in (None, "fused", "tiny"):
        raise ValueError(f"{what}: mode must be 'fused' or 'tiny', got {mode!r}")
    idx = teacher_indices.to(torch.int64).contiguous()
    lp = _ak.f32_dense(teacher_logprobs)
    if logits.requires_grad and torch.is_grad_enabled():
        fused = mode == "fused" or (mode is None and logits.dtype != torch.float16)
        return _DistillTopK.apply(logits, idx, lp, mask, temperature, softcap, bool(tail), fused)
    return _ak.distill_topk_fwd(logits, idx, lp, mask, temperature, softcap, bool(tail))[0]


def kernel_fn(logits: torch.Tensor, teacher_indices: torch.Tensor, teacher_logprobs: torch.Tensor) -> torch.Tensor:
    """The loss with its defaults: the teacher renormalised over its entries, temperature 1."""
    return distill_topk(logits, teacher_indices, teacher_logprobs)
