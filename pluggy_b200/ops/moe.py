"""Dropless top-k MoE expert FFN.

Parity: reference ``pluggy/kernels/moe.py:38-168`` (``moe_expert_ffn``: sort the
(token, expert) pairs by expert, per-expert SwiGLU FFN with packed weights
``gate_up_proj (E, 2I, H)`` / ``down_proj (E, H, I)``, scale by the routing
weight, scatter-add back). The loop and grouped forms give identical results.

CUDA path: pairs are sorted once by expert; each of the FFN's projections is
ONE launch of this package's grouped tcgen05 GEMM over all experts
(:func:`pluggy_b200.ops.grouped.grouped_swiglu_ffn`: a device-computed padded
per-expert row layout, no host synchronisation) and the GLU is the sm_100a
kernel; the combine is a scatter-add of the route-weighted rows.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from pluggy_b200.ops.elementwise import swiglu_mul


def expert_histogram(idx: torch.Tensor, n: int) -> torch.Tensor:
    """int64 [n]: how many entries of ``idx`` (values in [0, n)) equal each value.
    A scatter-add, so it stays on the device: ``torch.bincount`` on CUDA reads the
    input's minimum and maximum back to the host to size its output."""
    flat = idx.reshape(-1).to(torch.int64)
    out = torch.zeros(n, dtype=torch.int64, device=idx.device)
    return out.scatter_add_(0, flat, torch.ones_like(flat))


def _expert_ffn_loop(hidden, top_indices, top_weights, gate_up_proj, down_proj):
    T, H = hidden.shape
    E = gate_up_proj.shape[0]
    out = torch.zeros(T, H, device=hidden.device, dtype=hidden.dtype)
    mask = F.one_hot(top_indices, num_classes=E).permute(2, 1, 0)  # (E, K, T)
    hit = mask.sum(dim=(-1, -2)).nonzero(as_tuple=False).flatten()
    gu = gate_up_proj.to(hidden.dtype)
    dn = down_proj.to(hidden.dtype)
    for e in hit.tolist():
        k_pos, tok = torch.where(mask[e])
        if tok.numel() == 0:
            continue
        g, u = F.linear(hidden[tok], gu[e]).chunk(2, dim=-1)
        y = F.linear(swiglu_mul(g, u), dn[e]) * top_weights[tok, k_pos, None]
        out.index_add_(0, tok, y.to(out.dtype))
    return out


def _expert_ffn_sorted(hidden, top_indices, top_weights, gate_up_proj, down_proj, gu_lowp=None,
                       dn_lowp=None):
    from pluggy_b200.ops.grouped import grouped_swiglu_ffn

    T, H = hidden.shape
    E = gate_up_proj.shape[0]
    K = top_indices.shape[1]
    tok = torch.arange(T, device=hidden.device).unsqueeze(1).expand(T, K).reshape(-1)
    exp = top_indices.reshape(-1)
    w = top_weights.reshape(-1)
    order = torch.argsort(exp, stable=True)
    s_tok, s_w, s_exp = tok[order], w[order], exp[order]
    counts = expert_histogram(exp, E)
    x = hidden[s_tok]
    y = grouped_swiglu_ffn(x, s_exp, counts, gate_up_proj, down_proj, gu_lowp, dn_lowp)
    y = y * s_w.unsqueeze(1).to(y.dtype)
    out = torch.zeros(T, H, device=hidden.device, dtype=y.dtype)
    out.index_add_(0, s_tok, y)
    return out.to(hidden.dtype)


def moe_expert_ffn(hidden, top_indices, top_weights, gate_up_proj, down_proj, *,
                   use_grouped_mm: bool | None = None, gu_lowp=None, dn_lowp=None):
    """Dropless top-k expert FFN; ``use_grouped_mm`` None = auto (CUDA -> sorted grouped path)."""
    assert hidden.dim() == 2 and top_indices.shape == top_weights.shape
    assert top_indices.shape[0] == hidden.shape[0]
    assert gate_up_proj.dim() == 3 and down_proj.dim() == 3
    if use_grouped_mm is None:
        use_grouped_mm = hidden.is_cuda
    if use_grouped_mm:
        return _expert_ffn_sorted(hidden, top_indices, top_weights, gate_up_proj, down_proj,
                                  gu_lowp, dn_lowp)
    return _expert_ffn_loop(hidden, top_indices, top_weights, gate_up_proj, down_proj)


# ------------------------------------------------------------------ router losses
def router_balance_loss_reference(router_logits, top_indices, balance_coef=1.0, z_coef=0.0, mask=None):
    """fp32 math in eager torch on lists of [T, E] logits and [T, k] indices."""
    E = router_logits[0].shape[1]
    x = torch.cat([g.float() for g in router_logits])
    idx = torch.cat(list(top_indices))
    if mask is not None:
        keep = mask.repeat(len(router_logits)).nonzero().squeeze(1)
        x, idx = x[keep], idx[keep]
    n = max(1, x.shape[0])
    inside = (idx >= 0) & (idx < E)
    counts = expert_histogram(idx[inside], E)
    lse = torch.logsumexp(x, dim=-1)
    probs = torch.exp(x - lse.unsqueeze(1))
    loss = balance_coef * E * (counts / n * probs.sum(0) / n).sum()
    if z_coef:
        loss = loss + z_coef * lse.square().sum() / n
    # the fractions are unknown where a choice lies outside: NaN, in the gradient too
    return (loss if inside.all() else loss * float("nan")), counts


def router_balance_loss(router_logits, top_indices, *, balance_coef: float = 1.0, z_coef: float = 0.0,
                        mask: torch.Tensor | None = None):
    """Balance and z loss of one or several MoE routers, and the tokens sent to each expert.

    ``router_logits`` is [T, E] (bf16 or fp32) or a list of them, one for each layer, and
    ``top_indices`` the routers' own choices, int64 [T, k] alike. Over the n tokens of all
    layers (those where ``mask``, bool [T], holds), with p = softmax(logits) in fp32 and
    counts[e] = how often expert e was chosen,

        loss = balance_coef * E * sum_e (counts[e] / n) * mean(p[:, e]) + z_coef * mean(logsumexp^2)

    Returns ``(loss, counts int64 [E])``; the gradient goes to the logits (the counts are
    constants, as in the models' auxiliary loss). An index outside [0, E) is not counted and makes
    the loss and the gradient of every kept row NaN. On CUDA at most 128 layers of 1024 experts in one call.

    CUDA path (csrc/objective.cu): all layers in one launch that keeps a row's probabilities
    in registers and writes only its log-sum-exp, one small kernel for the loss, one launch
    for all gradients; no probabilities and no concatenated logits in memory."""
    single = isinstance(router_logits, torch.Tensor)
    logits = [router_logits] if single else list(router_logits)
    idx = [top_indices] if single else list(top_indices)
    if not logits or len(idx) != len(logits):
        raise ValueError(f"router_balance_loss: one index tensor for each router, got {len(logits)} and "
                         f"{len(idx)}")
    x0 = logits[0]
    if x0.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"router_balance_loss: logits must be bf16 or fp32, got {x0.dtype}")
    if x0.dim() != 2 or x0.shape[1] == 0:
        raise ValueError(f"router_balance_loss: logits must be [T, E] with E > 0, got {tuple(x0.shape)}")
    if x0.is_cuda:  # the extension checks every layer
        from pluggy_b200.ops._ext import ext

        return tuple(ext().router_balance_loss(logits, idx, mask, float(balance_coef), float(z_coef)))
    for x, i in zip(logits, idx):
        if x.shape != x0.shape or x.dtype != x0.dtype or x.device != x0.device:
            raise ValueError("router_balance_loss: the routers' logits must be [T, E], alike")
        if i.shape != (x.shape[0], idx[0].shape[-1]) or i.dtype != torch.int64 or i.device != x.device:
            raise ValueError(f"router_balance_loss: indices must be int64 [T, k], got {i.dtype} "
                             f"{tuple(i.shape)}")
    if mask is not None and (mask.shape != x0.shape[:1] or mask.dtype != torch.bool
                             or mask.device != x0.device):
        raise ValueError(f"router_balance_loss: mask must be bool [{x0.shape[0]}]")
    return router_balance_loss_reference(logits, idx, balance_coef, z_coef, mask)
