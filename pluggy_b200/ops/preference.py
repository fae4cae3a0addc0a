"""Paired preference loss over per-token log-probabilities.

For pair ``i`` with a chosen (side 0) and a rejected (side 1) sequence, over the tokens
where ``mask`` holds,

    s[side, i] = sum_t (logps - ref_logps)       (their mean with ``length_normalized``)
    h[i] = s[0, i] - s[1, i]
    sigmoid:  (1 - eps) softplus(-beta h) + eps softplus(beta h)   (eps = label_smoothing)
    hinge:    max(0, 1 - beta h)
    ipo:      (h - 1 / (2 beta))^2
    loss = mean_i of these

and the implicit rewards are ``beta * s``. A sequence without tokens has s = 0.

CUDA path (csrc/objective.cu): one pass over the log-probabilities, then one small kernel
over the pairs that leaves one number per row, the gradient of each of its tokens; the
backward spreads it over the mask. CPU tensors take the same math in eager torch.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from pluggy_b200.ops._ext import ext

KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


def preference_loss_reference(logps, ref_logps, mask, beta=0.1, kind="sigmoid", label_smoothing=0.0,
                              length_normalized=False):
    d = logps.float() if ref_logps is None else logps.float() - ref_logps.float()
    s = torch.where(mask, d, 0.0).sum(-1)
    if length_normalized:
        s = s / mask.sum(-1).clamp_min(1)
    h = s[0] - s[1]
    if kind == "sigmoid":
        per = -(1 - label_smoothing) * F.logsigmoid(beta * h)
        if label_smoothing:
            per = per - label_smoothing * F.logsigmoid(-beta * h)
    elif kind == "hinge":
        per = torch.relu(1 - beta * h)
    else:
        per = (h - 0.5 / beta).square()
    loss = per.sum() / max(1, h.numel())
    return loss, (beta * s[0]).detach(), (beta * s[1]).detach()


def check_tokens(op: str, mask: torch.Tensor, **tensors) -> None:
    """Shapes, devices and types of (tensor or None, allowed types) against the mask's, for CPU
    tensors; the CUDA entry points check the same."""
    for name, (t, types) in tensors.items():
        if t is None:
            continue
        if t.shape != mask.shape or t.device != mask.device:
            raise ValueError(f"{op}: {name} must have mask's shape {tuple(mask.shape)} and device, got "
                             f"{tuple(t.shape)} on {t.device}")
        if t.dtype not in types:
            raise TypeError(f"{op}: {name} is {t.dtype}, expected one of {types}")


def tokens_contiguous(t: torch.Tensor) -> torch.Tensor:
    """``t`` or a copy whose last dimension is contiguous (what the kernels stream)."""
    return t if t.shape[-1] < 2 or t.stride(-1) == 1 else t.contiguous()


def check_no_grad(op: str, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{op}: {name} takes no gradient here; detach it or compute it under no_grad")


def preference_loss(logps: torch.Tensor, ref_logps: torch.Tensor | None, mask: torch.Tensor, *,
                    beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                    length_normalized: bool = False):
    """``(loss, chosen_rewards [P], rejected_rewards [P])``; see the module's formulas.

    ``logps`` fp32, ``ref_logps`` fp32 or bf16 (None: no reference model) and ``mask`` bool are
    ``[2, P, S]`` with the chosen sequences at index 0 and the rejected ones at 1, any outer
    strides (a batch of alternating sequences is ``x.view(P, 2, S).transpose(0, 1)``). Only
    ``logps`` has a gradient. Places outside the mask may hold anything."""
    if mask.dim() != 3 or mask.shape[0] != 2 or mask.dtype != torch.bool:
        raise ValueError(f"preference_loss: mask must be bool [2, P, S], got {mask.dtype} "
                         f"{tuple(mask.shape)}")
    if kind not in KINDS:
        raise ValueError(f"preference_loss: kind must be one of {sorted(KINDS)}, got {kind!r}")
    if not beta > 0:
        raise ValueError("preference_loss: beta must be positive")
    if not 0 <= label_smoothing < 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError("preference_loss: label_smoothing in [0, 0.5), for kind 'sigmoid' only")
    if ref_logps is not None and ref_logps.requires_grad:
        check_no_grad("preference_loss", ref_logps=ref_logps)
    if not mask.is_cuda or mask.shape[1] == 0:
        check_tokens("preference_loss", mask, logps=(logps, (torch.float32,)),
                     ref_logps=(ref_logps, (torch.float32, torch.bfloat16)))
        return preference_loss_reference(logps, ref_logps, mask, beta, kind, label_smoothing,
                                         length_normalized)
    return tuple(ext().preference_loss(logps, ref_logps, tokens_contiguous(mask), KINDS[kind], float(beta),
                                       float(label_smoothing), bool(length_normalized)))
