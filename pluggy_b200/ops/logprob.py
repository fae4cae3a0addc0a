"""Log-probabilities of given tokens under a linear head (the LM head), without its logits.

``linear_token_logprobs(hidden, weight, labels)`` returns, for every token,

    z = softcap(hidden @ weight^T) / temperature
    out = z[label] - log(sum(exp(z)))             (0 where the label is ignore_index)

in fp32, differentiable in ``hidden`` and ``weight``. It is what a preference or a policy
loss reads of the policy, and with gradients off it scores tokens under a frozen
reference model or one sampled token at a time.

CUDA path (csrc/logprob.cu): the product's tcgen05 epilogue reduces every accumulator
tile to a (maximum, sum of exponentials) pair per row, so no logits are written; the
backward recomputes them one vocabulary range at a time as the bf16 matrix
``-g_t * softmax``, whose two products give the gradients; the labels' own entries, most of a
gradient, never leave fp32. Ranges are split over
the vocabulary rather than over the tokens so that each row of the weight's gradient is
written once, in its final type, instead of being summed over chunks of tokens. Large
problems save that second product of hidden and weight: the forward stores bf16
exponentials, which are the gradient's rows up to a factor for each row. Tokens with ignored
labels are packed away on the device first: they cost no products, and values in their
hidden rows reach no output.
"""

from __future__ import annotations

import math

import torch

from pluggy_b200.ops._ext import ext, status_word

# Bytes of the bf16 matrix that a call keeps from its forward to its backward, or recomputes at a
# time: two for each token, rounded up to 256 of them, and vocabulary entry. Ignored tokens are
# among them, because how many there are is known on the device alone.
WORKSPACE = 8 << 30
# tokens * vocabulary * D from which the matrix is kept: below it the product that this saves
# takes less than 0.1 ms, and recomputing rounds a term of the weight's gradient once less
KEEP_PRODUCT = 1 << 36
# bytes of the k splits' fp32 sums of the hidden rows' gradient
SPLIT_WORKSPACE = 512 << 20
# Scoring at most this many tokens skips the packing of the kept ones: up to 256 tokens
# are one row of tiles, whose time is the head's one pass through memory.
UNPACKED_ROWS = 256


def token_logprobs_reference(hidden, weight, labels, ignore_index=-100, softcap=None,
                             temperature=1.0):
    """fp32 math in eager torch on [T, D] rows; ignored rows and those whose label is outside the
    vocabulary (NaN) take no part in the graph."""
    outside = (labels != ignore_index) & ((labels < 0) | (labels >= weight.shape[0]))
    keep = ((labels != ignore_index) & ~outside).nonzero().squeeze(1)
    z = hidden[keep].float() @ weight.float().t()
    if softcap:
        z = torch.tanh(z / softcap) * softcap
    z = z / temperature
    lp = z.gather(1, labels[keep].unsqueeze(1)).squeeze(1) - torch.logsumexp(z, dim=-1)
    out = torch.zeros(labels.shape, dtype=torch.float32, device=hidden.device)
    return out.masked_fill_(outside, float("nan")).index_put((keep,), lp)


def _rows_aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` or a copy whose rows start on 16-byte boundaries and do not overlap, as those of an
    expanded row do (what the TMA loads need)."""
    if t.stride(1) == 1 and t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


def linear_token_logprobs(hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor,
                          ignore_index: int = -100, *, weight_lowp: torch.Tensor | None = None,
                          softcap: float | None = None, temperature: float = 1.0,
                          workspace_bytes: int | None = None) -> torch.Tensor:
    """fp32 log-probability of every label under ``softmax(softcap(hidden weight^T) / temperature)``.

    ``hidden`` [..., D] and ``weight`` [V, D] are bf16 or fp32, ``labels`` [...] int64 (already
    shifted: ``labels[t]`` is scored against ``hidden[t]``). The result has labels' shape and is
    0 where the label is ``ignore_index``; a label outside [0, V) gives NaN and no gradient.
    On CUDA the products are bf16 with fp32 accumulation, as everywhere in this package (an
    fp32 ``weight`` is cast, or ``weight_lowp``, its cached bf16 copy, is read instead), and D
    must be a multiple of 8. The gradients have the inputs' types. ``workspace_bytes`` (8 GiB
    when None) bounds the bf16 matrix that a training call keeps for its backward: two bytes for
    each token, ignored ones included, and vocabulary entry, recomputed in parts where that is
    more. Not in it: the hidden rows in bf16, kept, too; 16 bytes for each token and 128 to 256
    vocabulary entries during the forward; in the backward 4 bytes for each token and column of
    either gradient asked for, and for the hidden states' gradient several such parts, up to
    512 MiB of them."""
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_token_logprobs: hidden [..., D] and weight [V, D], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if labels.shape != hidden.shape[:-1] or labels.dtype != torch.int64:
        raise ValueError(f"linear_token_logprobs: labels must be int64 {tuple(hidden.shape[:-1])}, got "
                         f"{labels.dtype} {tuple(labels.shape)}")
    if not temperature > 0 or (softcap is not None and not 0 <= softcap < math.inf):
        raise ValueError("linear_token_logprobs: temperature must be positive, softcap finite and not negative")
    if weight.shape[0] == 0:
        raise ValueError("linear_token_logprobs: an empty vocabulary")
    for name, t in (("hidden", hidden), ("weight", weight)):
        if t.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"linear_token_logprobs: {name} must be bf16 or fp32, got {t.dtype}")
    if weight.device != hidden.device or labels.device != hidden.device:
        raise ValueError("linear_token_logprobs: hidden, weight and labels must be on one device")
    if weight_lowp is not None and (weight_lowp.shape != weight.shape
                                    or weight_lowp.dtype != torch.bfloat16
                                    or weight_lowp.device != weight.device):
        raise ValueError("linear_token_logprobs: weight_lowp must be weight's bf16 copy")
    D = hidden.shape[-1]
    if not hidden.is_cuda:
        flat = labels.reshape(-1)
        return token_logprobs_reference(hidden.reshape(-1, D), weight, flat, ignore_index, softcap,
                                        temperature).view(labels.shape)
    if D % 8 or D == 0:
        raise ValueError(f"linear_token_logprobs: D must be a multiple of 8 on CUDA, got {D}")
    if labels.numel() == 0:
        return (hidden.sum() + weight.sum()) * torch.zeros(labels.shape, device=hidden.device)
    w = weight_lowp if weight_lowp is not None else weight.detach().to(torch.bfloat16)
    h = hidden.reshape(-1, D)
    h, w = _rows_aligned(h), _rows_aligned(w)
    T, V = h.shape[0], w.shape[0]
    workspace = WORKSPACE if workspace_bytes is None else int(workspace_bytes)
    keep = 2 * _round_up(T, 256) * V <= workspace and T * V * D >= KEEP_PRODUCT
    out = ext().token_logprobs(h, weight, w, labels.reshape(-1).contiguous(), int(ignore_index),
                               float(softcap or 0.0), float(temperature), T > UNPACKED_ROWS, keep,
                               workspace, SPLIT_WORKSPACE, status_word(h.device))
    return out.view(labels.shape)
