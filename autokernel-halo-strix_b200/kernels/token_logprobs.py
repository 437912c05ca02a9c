"""Log-probabilities of given tokens on B200, with entropies and top alternatives.

`token_logprobs` reads logit rows once and answers, per row: how likely the target token was,
how uncertain the distribution is, and which tokens were most likely.  It serves scoring and
decoding (no gradient is kept then), a teacher's pass over a batch for `kernels.distill`, and
policy-gradient losses: `logprobs` and `entropy` are differentiable.  The cross-entropy in
`kernels.ce_fused` is the loss over the same rows.

`linear_token_logprobs` answers the same (without alternatives) from hidden states and the output
projection on the tensor cores; logits are never stored, as in `ChunkedLinearCrossEntropyLoss`.

The reference has only the losses (kernels/ce_fused.py:557-785,
kernels/hip/chunked_linear_cross_entropy.py:50-229).
"""
import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from kernels import _ak

KERNEL_TYPE = "token_logprobs"
BACKEND = "cuda_sm100a"

MAX_TOP_K = 128
LOWEST_TEMPERATURE = LOWEST_SOFTCAP = 2.0 ** -100


class TokenLogprobs(NamedTuple):
    """Per row of the input; fp32, indices int64.  Fields that were not asked for are None."""
    logprobs: Optional[torch.Tensor]
    entropy: Optional[torch.Tensor]
    lse: torch.Tensor
    top_logprobs: Optional[torch.Tensor] = None
    top_indices: Optional[torch.Tensor] = None


def once(backward, ctx, *grads):
    """`backward(ctx, *grads)` as torch's `once_differentiable` runs it; its bookkeeping (several
    microseconds) is only needed where a graph of the backward is built."""
    if torch.is_grad_enabled():
        return once_differentiable(backward)(ctx, *grads)
    return backward(ctx, *grads)


def _token_logprobs_backward(ctx, g_lp, g_ent):
    if g_lp is None and g_ent is None:
        return (None,) * 7
    logits, targets, stats = ctx.saved_tensors
    return (_ak.token_logprobs_bwd(logits, targets, stats, g_lp, g_ent, *ctx.args),) + (None,) * 6


class _TokenLogprobs(torch.autograd.Function):
    """Saves the logits and four numbers a row; the backward recomputes the softmax from them."""

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature, softcap, ignore_index, entropy):
        lp, ent, lse, top_lp, top_idx, stats = _ak.token_logprobs_fwd(
            logits, targets, top_k, temperature, softcap, ignore_index, want_entropy=entropy, want_stats=True)
        ctx.save_for_backward(logits, targets, stats)
        ctx.args = (temperature, softcap, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (lse, top_lp, top_idx) if t is not None))
        return lp, ent, lse, top_lp, top_idx

    @staticmethod
    def backward(ctx, g_lp, g_ent, *rest):
        return once(_token_logprobs_backward, ctx, g_lp, g_ent)


def check_scales(what: str, temperature: float, softcap: float):
    if temperature == 1.0 and softcap == 0.0:
        return 1.0, 0.0
    temperature, softcap = float(temperature), float(softcap)
    if not (temperature >= LOWEST_TEMPERATURE and math.isfinite(temperature)):
        raise ValueError(f"{what}: temperature must be at least 2^-100 and finite, got {temperature}")
    if not (softcap == 0.0 or (softcap >= LOWEST_SOFTCAP and math.isfinite(softcap))):
        raise ValueError(f"{what}: softcap must be 0 (none), or at least 2^-100 and finite, got {softcap}")
    return temperature, softcap


def check_targets(what: str, targets: torch.Tensor, lead) -> torch.Tensor:
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"{what}: targets must be int64 or int32, got {targets.dtype}")
    if targets.shape != lead:
        raise ValueError(f"{what}: targets {tuple(targets.shape)} do not match the rows {tuple(lead)}")
    if targets.dtype is torch.int64 and targets.is_contiguous():
        return targets
    return targets.to(torch.int64).contiguous()


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0, softcap: float = 0.0, ignore_index: int = -100,
                   entropy: bool = False) -> TokenLogprobs:
    """Log-probabilities under softmax(softcap(logits) / temperature) over the last dimension.

    logits (..., V): fp32, bf16 or fp16 on the GPU.  Row views (logits[:, :-1], logits[..., :V]) are
    read in place; an input whose last dimension is strided, or with more than two uneven leading
    dimensions, is copied.
    targets (...): the tokens whose `logprobs` are wanted, or None.  Where a target is `ignore_index`
    its log-probability and entropy are 0 and its row gets no gradient, whatever the row holds; a
    target outside the vocabulary gives NaN.
    top_k: alternatives per row, at most 128 (of at most 1,048,320 tokens): `top_logprobs` and `top_indices` (..., top_k), most
    likely first, equal logits by lowest index.  They and `lse` carry no gradient.
    entropy: whether to compute the entropy (nats).
    temperature: at least 2^-100; softcap: 0 for none, or at least 2^-100.

    -inf logits are tokens without probability.  A row of nothing else has log-probabilities -inf,
    entropy 0 and no gradient; a row with NaN is NaN.
    """
    what = "token_logprobs"
    _ak.dtype_code(logits)
    _ak.refuse_tangents(what, logits)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits must be (..., V) with V >= 1, got {tuple(logits.shape)}")
    if targets is not None:
        targets = check_targets(what, targets, logits.shape[:-1])
    if top_k:
        top_k = int(top_k)
        if not 0 <= top_k <= min(MAX_TOP_K, logits.shape[-1]):
            raise ValueError(f"{what}: top_k must be in 0..{min(MAX_TOP_K, logits.shape[-1])}, got {top_k}")
    else:
        top_k = 0
    temperature, softcap = check_scales(what, temperature, softcap)
    ignore_index = int(ignore_index)
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*_TokenLogprobs.apply(logits, targets, top_k, temperature, softcap, ignore_index,
                                                   bool(entropy)))
    return TokenLogprobs(*_ak.token_logprobs_fwd(logits, targets, top_k, temperature, softcap, ignore_index,
                                                 want_entropy=bool(entropy))[:5])


def _linear_token_logprobs_backward(ctx, g_lp, g_ent):
    if g_lp is None and g_ent is None:
        return (None,) * 7
    hidden, w, targets, stats = ctx.saved_tensors
    # a weight of another type than hidden's has its gradient rounded from fp32 to that type, if at all
    dh, dw = _ak.linear_logprobs_bwd(hidden, w, targets, stats, g_lp, g_ent, *ctx.args,
                                     need_dh=ctx.needs_input_grad[0], need_dw=ctx.needs_input_grad[1],
                                     dw_dtype=w.dtype if ctx.weight_dtype == w.dtype else torch.float32)
    return (dh, dw.to(ctx.weight_dtype) if dw is not None else None) + (None,) * 5


class _LinearTokenLogprobs(torch.autograd.Function):
    """Saves its operands and four numbers a row; the backward forms the logits again, chunk by chunk."""

    @staticmethod
    def forward(ctx, hidden, weight, targets, temperature, softcap, ignore_index, entropy):
        w = weight.to(hidden.dtype)
        lp, ent, lse, stats = _ak.linear_logprobs_fwd(hidden, w, targets, temperature, softcap, ignore_index,
                                                      want_entropy=entropy, want_stats=True)
        ctx.save_for_backward(hidden, w, targets, stats)
        ctx.args, ctx.weight_dtype = (temperature, softcap, ignore_index), weight.dtype
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(lse)
        return lp, ent, lse

    @staticmethod
    def backward(ctx, g_lp, g_ent, *rest):
        return once(_linear_token_logprobs_backward, ctx, g_lp, g_ent)


def _dense16(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and on a 16-byte boundary (a TMA operand)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def linear_token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, targets: Optional[torch.Tensor] = None, *,
                          temperature: float = 1.0, softcap: float = 0.0, ignore_index: int = -100,
                          entropy: bool = False) -> TokenLogprobs:
    """`token_logprobs(hidden @ weight.T, targets, ...)` without the logits and without alternatives.

    hidden (..., D): bf16 or fp16 on the GPU, D a multiple of 8; weight (V, D): cast to hidden's type
    if it has another (its gradient is rounded to its own type only; an fp32 weight's is not).  The log-probabilities are of the fp32 accumulators: nothing between the
    products and the result is rounded to 16 bits.  In the backward the gradient of the logits is, as
    the operand of the two products that follow.  The hidden states of ignored rows have to be
    finite where a gradient of weight is wanted (they enter it times 0).
    """
    what = "linear_token_logprobs"
    _ak.refuse_tangents(what, hidden, weight)
    if hidden.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{what}: hidden must be bfloat16 or float16, got {hidden.dtype}")
    _ak.dtype_code(weight)
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[0] < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden (..., D) and weight (V, D), got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    D = hidden.shape[-1]
    if D < 8 or D % 8:
        raise ValueError(f"{what}: the hidden size must be a multiple of 8, got {D}")
    lead = hidden.shape[:-1]
    if targets is not None:
        targets = check_targets(what, targets, lead).view(-1)
    temperature, softcap = check_scales(what, temperature, softcap)
    ignore_index = int(ignore_index)
    h = _dense16(hidden if hidden.dim() == 2 else hidden.reshape(-1, D))
    w = _dense16(weight)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        lp, ent, lse = _LinearTokenLogprobs.apply(h, w, targets, temperature, softcap, ignore_index, bool(entropy))
    else:
        lp, ent, lse, _ = _ak.linear_logprobs_fwd(h, w.to(h.dtype), targets, temperature, softcap, ignore_index,
                                                  want_entropy=bool(entropy))
    if len(lead) != 1:
        lp, ent, lse = (t.view(lead) if t is not None else None for t in (lp, ent, lse))
    return TokenLogprobs(lp, ent, lse)


def kernel_fn(logits: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    """Log-probability of each row's target (0 where it is -100)."""
    return token_logprobs(logits, targets).logprobs
