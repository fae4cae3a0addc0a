"""Clipped policy loss with a KL term over per-token log-probabilities.

Per token where ``mask`` holds, with r = logps - old_logps, advantage A and d = ref_logps - logps,

    clipped = (A > 0 and r > log(1 + clip_high)) or (A < 0 and r < log(1 - clip_low))
    loss = -A * (the passed bound, 1 + clip_high or 1 - clip_low, if clipped else exp(r))
           + kl_coef * (exp(d) - 1 - d)

which is -min(exp(r) A, clip(exp(r)) A) with the comparison made on the logarithms (the
subtraction of two close fp32 numbers is exact, an exponential is not), and the always
positive estimate of KL(policy || reference). ``reduction="token"`` averages over all
tokens, ``"sequence"`` over the sequences with tokens of their means over tokens.

CUDA path (csrc/objective.cu): a pass over the mask counts the tokens, then one pass over
the inputs gives the loss and its finished gradient; the backward multiplies the stored
gradient by the incoming one in place, and leaves it untouched when that is 1. CPU tensors
take the same math in eager torch.
"""

from __future__ import annotations

import math

import torch

from pluggy_b200.ops._ext import ext
from pluggy_b200.ops.preference import check_no_grad, check_tokens, tokens_contiguous


class _KlTerm(torch.autograd.Function):
    """e^d - 1 - d with its gradient formed as expm1(d), not as the difference e^d - 1."""

    @staticmethod
    def forward(ctx, d):
        em1 = torch.expm1(d)
        ctx.save_for_backward(em1)
        return em1 - d

    @staticmethod
    def backward(ctx, g):
        return g * ctx.saved_tensors[0]


def policy_loss_reference(logps, old_logps, advantages, mask, ref_logps=None, clip_low=0.2,
                          clip_high=0.2, kl_coef=0.0, reduction="token"):
    # outside the mask every input is replaced first, so that nothing there has a gradient
    def at(x):
        return torch.where(mask, x.float(), 0.0)

    lp = at(logps)
    adv = at(advantages.unsqueeze(1) if advantages.dim() == 1 else advantages)
    r = lp - (lp.detach() if old_logps is None else at(old_logps))
    up = (adv > 0) & (r > math.log1p(clip_high))
    dn = (adv < 0) & (r < math.log1p(-clip_low))
    bound = torch.where(up, 1 + clip_high, 1 - clip_low)
    # an advantage of 0 gives 0 also where e^r overflows
    flat = up | dn | ((adv == 0) & (r > 0))
    per = -torch.where(up | dn, bound, torch.exp(torch.where(flat, 0.0, r))) * adv
    kl = torch.zeros_like(lp)
    if ref_logps is not None:
        kl = _KlTerm.apply(at(ref_logps) - lp)
        if kl_coef:
            per = per + kl_coef * kl
    n = mask.sum(1)
    tokens = n.sum().clamp_min(1)
    if reduction == "token":
        w = mask / tokens
    else:
        w = mask / n.clamp_min(1).unsqueeze(1) / (n > 0).sum().clamp_min(1)
    loss = (torch.where(mask, per, 0.0) * w).sum()
    return (loss, (torch.where(mask, kl, 0.0).sum() / tokens).detach(),
            ((up | dn) & mask).sum() / tokens)


def policy_loss(logps: torch.Tensor, old_logps: torch.Tensor | None, advantages: torch.Tensor,
                mask: torch.Tensor, *, ref_logps: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, reduction: str = "token"):
    """``(loss, mean KL estimate, clipped share of the tokens)``; see the module's formulas.

    ``logps`` fp32, ``old_logps`` and ``ref_logps`` fp32 or bf16 and ``mask`` bool are [R, S],
    ``advantages`` is fp32 [R] or [R, S]; any row strides. ``old_logps`` None stands for
    ``logps.detach()`` (one update for each rollout: exp(r) = 1), ``ref_logps`` None for no KL
    term. Only ``logps`` has a gradient. Places outside the mask may hold anything."""
    if mask.dim() != 2 or mask.dtype != torch.bool:
        raise ValueError(f"policy_loss: mask must be bool [R, S], got {mask.dtype} {tuple(mask.shape)}")
    if not 0 <= clip_low < 1 or not clip_high >= 0:
        raise ValueError("policy_loss: clip_low in [0, 1) and clip_high >= 0")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"policy_loss: reduction must be 'token' or 'sequence', got {reduction!r}")
    if kl_coef and ref_logps is None:
        raise ValueError("policy_loss: kl_coef needs ref_logps")
    check_no_grad("policy_loss", old_logps=old_logps, ref_logps=ref_logps, advantages=advantages)
    if not mask.is_cuda or mask.shape[0] == 0:
        fp32 = (torch.float32,)
        check_tokens("policy_loss", mask, logps=(logps, fp32),
                     old_logps=(old_logps, (torch.float32, torch.bfloat16)),
                     ref_logps=(ref_logps, (torch.float32, torch.bfloat16)))
        check_tokens("policy_loss", mask.any(1) if advantages.dim() == 1 else mask,
                     advantages=(advantages, fp32))
        return policy_loss_reference(logps, old_logps, advantages, mask, ref_logps, clip_low, clip_high,
                                     kl_coef, reduction)
    return tuple(ext().policy_loss(logps, old_logps, advantages, tokens_contiguous(mask), ref_logps,
                                   float(clip_low), float(clip_high), float(kl_coef),
                                   reduction == "sequence"))
