"""Measured cases of the post-training operators: per-token log-probabilities of a linear
head, the paired preference loss, the clipped policy loss with a KL term, and the MoE
router's balance and z losses.

``run`` computes a case either in its plain form (elementary torch operations in fp32) or,
with ``own`` true, through the package's public operators; both take what ``prepare`` made.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # ---- log-probabilities of given tokens under hidden @ weight^T
        # the newest sampled token of one sequence: latency, bound by reading the head
        dict(name="logprob-one-token", op="logprob", train=False, T=1, D=1024, V=151936, ignored=0.0,
             softcap=0.0, temperature=1.0),
        # a frozen reference model scoring a batch whose prompts are masked out
        dict(name="logprob-score", op="logprob", train=False, T=4096, D=2560, V=151936, ignored=0.4,
             softcap=0.0, temperature=1.0),
        # a small byte-level-like head with odd sizes, softcapped logits, tempered policy
        dict(name="logprob-odd-train", op="logprob", train=True, T=777, D=256, V=8191, ignored=0.3,
             softcap=30.0, temperature=0.8),
        # the policy's own pass over a training micro-batch, prompts masked out
        dict(name="logprob-train", op="logprob", train=True, T=8192, D=2048, V=128256, ignored=0.35,
             softcap=0.0, temperature=1.0),
        # the largest: every token of a packed batch trains
        dict(name="logprob-train-large", op="logprob", train=True, T=16384, D=1024, V=151936,
             ignored=0.0, softcap=0.0, temperature=1.0),
        # ---- paired preference loss over per-token log-probabilities
        # two pairs, the micro-batch of a large model: latency
        dict(name="preference-small", op="preference", P=2, S=512, kind="sigmoid", smoothing=0.0,
             normalized=False, ref="float32"),
        # many long ragged pairs, length-normalised, reference stored in bf16
        dict(name="preference-large", op="preference", P=511, S=8192, kind="ipo", smoothing=0.0,
             normalized=True, ref="bfloat16"),
        # ---- clipped policy loss with a KL term
        # one micro-batch of rollouts, one advantage for each sequence: latency
        dict(name="policy-small", op="policy", R=8, S=1023, reduction="token", per_token=False,
             stored="float32", kl=0.05),
        # a whole rollout batch with per-token advantages, averaged by sequence
        dict(name="policy-large", op="policy", R=1024, S=16384, reduction="sequence", per_token=True,
             stored="float32", kl=0.02),
        # ---- balance and z loss of MoE routers, with the per-expert counts
        # one layer, a short odd batch, an expert count that is no power of two
        dict(name="router-small", op="router", L=1, T=257, E=60, k=4, masked=0.0),
        # the routers of a 24-layer step, 128 experts, top 8, 2 x 4096 tokens
        dict(name="router-step", op="router", L=24, T=8192, E=128, k=8, masked=0.0),
        # more experts, more tokens, padded rows left out
        dict(name="router-large", op="router", L=24, T=32768, E=256, k=8, masked=0.2),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(max(n, lo), hi)
    return n - 1 if n == 3072 else n


def draw(rng):
    """One more case of the listed ranges."""
    op = rng.choice(["logprob", "logprob", "preference", "policy", "router"])
    if op == "logprob":
        train = rng.random() < 0.6
        while True:
            T = _log_int(rng, 1, 16384)
            D = 8 * _log_int(rng, 8, 320)
            V = _log_int(rng, 500, 152000)
            if D != 3072 and T * D * V <= 16384 * 1024 * 151936:
                break
        return dict(op=op, train=train, T=T, D=D, V=V, ignored=rng.choice([0.0, 0.3, 0.7]),
                    softcap=rng.choice([0.0, 0.0, 30.0]), temperature=rng.choice([1.0, 1.0, 0.7]))
    if op == "preference":
        while True:
            P, S = _log_int(rng, 1, 512), _log_int(rng, 1, 32768)
            if P * S <= 511 * 8192:
                break
        kind = rng.choice(["sigmoid", "hinge", "ipo"])
        return dict(op=op, P=P, S=S, kind=kind, smoothing=rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0,
                    normalized=rng.random() < 0.3, ref=rng.choice(["float32", "bfloat16", "none"]))
    if op == "policy":
        while True:
            R, S = _log_int(rng, 1, 2048), _log_int(rng, 1, 32768)
            if R * S <= 1024 * 16384:
                break
        return dict(op=op, R=R, S=S, reduction=rng.choice(["token", "sequence"]),
                    per_token=rng.random() < 0.5, stored=rng.choice(["float32", "bfloat16"]),
                    kl=rng.choice([0.0, 0.05]))
    while True:
        L, T, E = _log_int(rng, 1, 48), _log_int(rng, 1, 32768), _log_int(rng, 4, 512)
        if L * T * E <= 24 * 32768 * 256:
            break
    return dict(op=op, L=L, T=T, E=E, k=min(E, rng.choice([1, 2, 4, 8])), masked=rng.choice([0.0, 0.2]))


# ------------------------------------------------------------------------- inputs
def _lengths(gen, rows, S):
    """Ragged lengths 0..S: mostly spread, some sequences full and some empty."""
    u = torch.rand(rows, generator=gen, device=DEV)
    n = (0.2 + 0.8 * u) * S
    n = torch.where(u < 0.05, torch.zeros_like(n), n)
    n = torch.where(u > 0.9, torch.full_like(n, float(S)), n)
    return n.round().long()


def _mask(gen, rows, S):
    return torch.arange(S, device=DEV)[None, :] < _lengths(gen, rows, S)[:, None]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    st = {"case": dict(case)}
    op = case["op"]
    if op == "logprob":
        T, D, V = case["T"], case["D"], case["V"]
        w = torch.empty(V, D, dtype=torch.bfloat16, device=DEV)
        for r in range(0, V, 16384):  # logits of a trained head: spread of a few units
            w[r:r + 16384] = randn(min(16384, V - r), D) * (2.0 / math.sqrt(D))
        labels = (V * rand(T).pow(3)).long().clamp_(max=V - 1)  # frequent ids are low ids
        h = randn(T, D)
        # a share of the tokens is likely under the model, the rest is not
        wy = w[labels].float()
        h += wy * (15.0 * rand(T, 1) / wy.square().sum(1, keepdim=True).clamp_min(1e-3))
        if case["ignored"]:
            labels[rand(T) < case["ignored"]] = -100
        st.update(hidden=h.to(torch.bfloat16), weight=w, labels=labels)
        if case["train"]:
            st["hidden"].requires_grad_(True)
            st["weight"].requires_grad_(True)
            st["grad"] = randn(T)  # of the loss that reads the log-probabilities
    elif op == "preference":
        P, S = case["P"], case["S"]
        mask = _mask(gen, 2 * P, S).view(2, P, S)
        logps = -(0.05 + 2.0 * rand(2, P, S).square()) * mask
        st.update(logps=logps.requires_grad_(True), mask=mask, ref=None)
        if case["ref"] != "none":
            st["ref"] = ((logps.detach() + 0.1 * randn(2, P, S)) * mask).to(getattr(torch, case["ref"]))
    elif op == "policy":
        R, S = case["R"], case["S"]
        mask = _mask(gen, R, S)
        logps = -(0.01 + 2.0 * rand(R, S).square()) * mask
        dt = getattr(torch, case["stored"])
        st.update(logps=logps.requires_grad_(True), mask=mask,
                  old=((logps.detach() + 0.15 * randn(R, S)) * mask).to(dt),
                  ref=((logps.detach() + 0.3 * randn(R, S)) * mask).to(dt),
                  adv=randn(R, S) if case["per_token"] else randn(R))
    else:
        L, T, E, k = case["L"], case["T"], case["E"], case["k"]
        bias = randn(L, 1, E)  # some experts are more popular
        logits, idx = [], []
        for i in range(L):
            x = (1.2 * randn(T, E) + 0.5 * bias[i]).to(torch.bfloat16)
            # the router's own choice (distinct scores, so it is the same on every run)
            idx.append(torch.topk(x.float() + 1e-4 * rand(T, E), k, dim=-1).indices.contiguous())
            logits.append(x.requires_grad_(True))
        st.update(logits=logits, idx=idx, mask=None)
        if case["masked"]:
            st["mask"] = rand(T) >= case["masked"]
    return st


# ------------------------------------------------------------------ plain forms
ROWS = 4096  # rows of fp32 logits that the plain form holds at a time


def _plain_logprob(st, c):
    h, w, labels = st["hidden"].detach(), st["weight"].detach(), st["labels"]
    rows = (labels != -100).nonzero().squeeze(1)
    out = torch.zeros(labels.shape, dtype=torch.float32, device=h.device)
    wf = w.float()
    if c["train"]:
        dh = torch.zeros(h.shape, dtype=torch.float32, device=h.device)
        dw = torch.zeros(w.shape, dtype=torch.float32, device=h.device)
    for s in range(0, rows.numel(), ROWS):
        r = rows[s:s + ROWS]
        hf, y = h[r].float(), labels[r].unsqueeze(1)
        z = hf @ wf.t()
        if c["softcap"]:
            z = torch.tanh(z / c["softcap"])
            slope = 1.0 - z * z if c["train"] else None
            z = z * c["softcap"]
        z = z / c["temperature"]
        m = z.max(dim=1, keepdim=True).values
        e = torch.exp(z - m)
        total = e.sum(dim=1, keepdim=True)
        out[r] = (z.gather(1, y) - m - torch.log(total)).squeeze(1)
        if c["train"]:
            g = st["grad"][r].unsqueeze(1)
            dz = e * (-g / total)
            dz.scatter_add_(1, y, g)
            dz = dz / c["temperature"]
            if c["softcap"]:
                dz = dz * slope
            dh[r] = dz @ wf
            dw += dz.t() @ hf
    if not c["train"]:
        return {"logps": out}
    return {"logps": out, "dhidden": dh.to(h.dtype), "dweight": dw.to(w.dtype)}


BETA = 0.1


def _plain_preference(st, c):
    lp, mask = st["logps"].detach(), st["mask"]
    m = mask.float()
    d = lp if st["ref"] is None else lp - st["ref"].float()
    s = torch.where(mask, d, torch.zeros_like(d)).sum(-1)  # [2, P]
    n = m.sum(-1).clamp_min(1.0) if c["normalized"] else torch.ones_like(s)
    s = s / n
    h = s[0] - s[1]
    P = h.numel()
    if c["kind"] == "sigmoid":
        eps, x = c["smoothing"], BETA * h
        soft = torch.log1p(torch.exp(-x.abs()))
        loss = (1 - eps) * (soft + (-x).clamp_min(0)) + eps * (soft + x.clamp_min(0))
        dl = BETA * (1.0 / (1.0 + torch.exp(-x)) - (1 - eps))
    elif c["kind"] == "hinge":
        loss = (1.0 - BETA * h).clamp_min(0)
        dl = torch.where(BETA * h < 1.0, -BETA, 0.0)
    else:
        loss = (h - 0.5 / BETA).square()
        dl = 2.0 * (h - 0.5 / BETA)
    dl = dl / P
    grad = torch.stack((dl, -dl)).div(n).unsqueeze(-1) * m
    return {"loss": loss.sum() / P, "chosen": BETA * s[0], "rejected": BETA * s[1], "dlogps": grad}


CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _plain_policy(st, c):
    lp, mask = st["logps"].detach(), st["mask"]
    adv = st["adv"] if st["adv"].dim() == 2 else st["adv"].unsqueeze(1)
    m = mask.float()
    logr = lp - st["old"].float()
    ratio = torch.exp(logr)
    up = (adv > 0) & (logr > math.log1p(CLIP_HIGH))
    dn = (adv < 0) & (logr < math.log1p(-CLIP_LOW))
    bound = torch.where(up, 1.0 + CLIP_HIGH, torch.where(dn, 1.0 - CLIP_LOW, ratio))
    pg = -bound * adv
    d = st["ref"].float() - lp
    e1 = torch.expm1(d)
    kl = e1 - d
    n = m.sum(1)
    if c["reduction"] == "token":
        w = m / n.sum().clamp_min(1.0)
    else:
        w = m / n.clamp_min(1.0).unsqueeze(1) / (n > 0).sum().clamp_min(1)
    zero = torch.zeros_like(lp)
    loss = torch.where(mask, (pg + c["kl"] * kl) * w, zero).sum()
    tokens = n.sum().clamp_min(1.0)
    grad = torch.where(up | dn, zero, -adv * ratio) - c["kl"] * e1
    return {"loss": loss, "kl": torch.where(mask, kl, zero).sum() / tokens,
            "clipped": (mask & (up | dn)).float().sum() / tokens,
            "dlogps": torch.where(mask, grad * w, zero)}


BALANCE, ZCOEF = 1e-2, 1e-3


def _plain_router(st, c):
    E = c["E"]
    counts = torch.zeros(E, dtype=torch.int64, device=DEV)
    psum = torch.zeros(E, dtype=torch.float32, device=DEV)
    z2 = torch.zeros((), dtype=torch.float32, device=DEV)
    m = st["mask"]
    n = 0.0
    probs, lses = [], []
    for x, idx in zip(st["logits"], st["idx"]):
        x = x.detach().float()
        top = x.max(-1, keepdim=True).values
        e = torch.exp(x - top)
        tot = e.sum(-1, keepdim=True)
        p, lse = e / tot, (top + torch.log(tot)).squeeze(-1)
        keep = torch.ones_like(lse) if m is None else m.float()
        one = keep.long().unsqueeze(1).expand_as(idx)
        counts.scatter_add_(0, idx.reshape(-1), one.reshape(-1))
        psum += (p * keep.unsqueeze(1)).sum(0)
        z2 += (lse.square() * keep).sum()
        n = n + keep.sum()
        probs.append(p)
        lses.append(lse)
    n = n.clamp_min(1.0)
    frac = counts.float() / n
    loss = BALANCE * E * (frac * (psum / n)).sum() + ZCOEF * z2 / n
    grads = []
    for p, lse, x in zip(probs, lses, st["logits"]):
        keep = torch.ones_like(lse) if m is None else m.float()
        a = frac - (p * frac).sum(-1, keepdim=True)
        g = p * (BALANCE * E / n * a + 2.0 * ZCOEF / n * lse.unsqueeze(1)) * keep.unsqueeze(1)
        grads.append(g.to(x.dtype))
    return {"loss": loss, "counts": counts, "dlogits": grads}


# ------------------------------------------------------------------------- run
def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return {"logprob": _plain_logprob, "preference": _plain_preference, "policy": _plain_policy,
                "router": _plain_router}[op](st, c)
    from pluggy_b200 import ops

    if op == "logprob":
        kw = dict(softcap=c["softcap"] or None, temperature=c["temperature"])
        if not c["train"]:
            with torch.no_grad():
                return {"logps": ops.linear_token_logprobs(st["hidden"], st["weight"], st["labels"], **kw)}
        lp = ops.linear_token_logprobs(st["hidden"], st["weight"], st["labels"], **kw)
        dh, dw = torch.autograd.grad(lp, (st["hidden"], st["weight"]), st["grad"])
        return {"logps": lp.detach(), "dhidden": dh, "dweight": dw}
    if op == "preference":
        loss, chosen, rejected = ops.preference_loss(
            st["logps"], st["ref"], st["mask"], beta=BETA, kind=c["kind"],
            label_smoothing=c["smoothing"], length_normalized=c["normalized"])
        (g,) = torch.autograd.grad(loss, st["logps"])
        return {"loss": loss.detach(), "chosen": chosen, "rejected": rejected, "dlogps": g}
    if op == "policy":
        loss, kl, clipped = ops.policy_loss(
            st["logps"], st["old"], st["adv"], st["mask"], ref_logps=st["ref"], clip_low=CLIP_LOW,
            clip_high=CLIP_HIGH, kl_coef=c["kl"], reduction=c["reduction"])
        (g,) = torch.autograd.grad(loss, st["logps"])
        return {"loss": loss.detach(), "kl": kl, "clipped": clipped, "dlogps": g}
    loss, counts = ops.router_balance_loss(st["logits"], st["idx"], balance_coef=BALANCE, z_coef=ZCOEF,
                                           mask=st["mask"])
    return {"loss": loss.detach(), "counts": counts,
            "dlogits": list(torch.autograd.grad(loss, st["logits"]))}


# ------------------------------------------------------------------------ work
def work(case):
    c = case
    if c["op"] == "logprob":
        n = c["T"] * (1.0 - c["ignored"])
        b = 2.0 * n * c["D"] + 2.0 * c["V"] * c["D"] + 12.0 * c["T"]
        f = 2.0 * n * c["V"] * c["D"]
        if c["train"]:  # both gradients written; dhidden and dweight are one product each
            return {"bytes": b + 2.0 * c["T"] * c["D"] + 2.0 * c["V"] * c["D"] + 4.0 * c["T"], "flops": 3 * f}
        return {"bytes": b, "flops": f}
    if c["op"] == "preference":
        n = 2.0 * c["P"] * c["S"]
        ref = {"none": 0, "float32": 4, "bfloat16": 2}[c["ref"]]
        return {"bytes": n * (4 + ref + 1 + 4) + 8.0 * c["P"], "flops": 4 * n}
    if c["op"] == "policy":
        n = 1.0 * c["R"] * c["S"]
        s = 4 if c["stored"] == "float32" else 2
        return {"bytes": n * (4 + 2 * s + 1 + (4 if c["per_token"] else 0) + 4) + 4.0 * c["R"], "flops": 20 * n}
    n = 1.0 * c["L"] * c["T"]
    # the logits read for the sums and again for the gradient, which needs those sums
    return {"bytes": n * (c["E"] * 2 * 2 + c["k"] * 8) + 8.0 * c["E"], "flops": 10 * n * c["E"]}


# ----------------------------------------------------------------------- exact
def exact(case, seed):
    """What ``run`` returns, from the definitions, in 64 bits."""
    c = dict(case)
    st = prepare(case, seed)
    f64 = torch.float64
    with torch.no_grad():
        if c["op"] == "logprob":
            tau, cap = c["temperature"], c["softcap"]
            H, W, y = st["hidden"].detach().to(f64), st["weight"].detach().to(f64), st["labels"]
            T = H.shape[0]
            lp = torch.zeros(T, dtype=f64, device=DEV)
            dH = torch.zeros_like(H)
            dW = torch.zeros_like(W) if c["train"] else None
            for s in range(0, T, 1024):
                e = min(T, s + 1024)
                ok = y[s:e] >= 0
                if not bool(ok.any()):
                    continue
                a = torch.matmul(H[s:e], W.T)
                z = (cap * torch.tanh(a / cap) if cap else a) / tau
                lse = torch.logsumexp(z, dim=1)
                at = y[s:e].clamp_min(0)
                pick = torch.arange(e - s, device=DEV)
                lp[s:e] = torch.where(ok, z[pick, at] - lse, torch.zeros_like(lse))
                if c["train"]:
                    G = torch.exp(z - lse[:, None]).neg_()
                    G[pick, at] += 1.0
                    G *= (st["grad"][s:e].to(f64) * ok)[:, None] / tau
                    if cap:
                        G *= 1.0 - torch.tanh(a / cap) ** 2
                    dH[s:e] = torch.matmul(G, W)
                    dW += torch.matmul(G.T, H[s:e])
            return {"logps": lp, "dhidden": dH, "dweight": dW} if c["train"] else {"logps": lp}
        if c["op"] == "preference":
            lp = st["logps"].detach().to(f64)
            keep = st["mask"]
            diff = lp - (0 if st["ref"] is None else st["ref"].to(f64))
            n = keep.sum(-1).to(f64)
            scale = 1.0 / n.clamp(min=1) if c["normalized"] else torch.ones_like(n)
            ratio = diff.masked_fill(~keep, 0.0).sum(-1) * scale
            margin = ratio[0] - ratio[1]
            P = margin.shape[0]
            if c["kind"] == "sigmoid":
                sp = torch.nn.functional.softplus
                per = (1 - c["smoothing"]) * sp(-BETA * margin) + c["smoothing"] * sp(BETA * margin)
                slope = BETA * (torch.sigmoid(BETA * margin) - 1 + c["smoothing"])
            elif c["kind"] == "hinge":
                per = torch.relu(1 - BETA * margin)
                slope = -BETA * (BETA * margin < 1).to(f64)
            else:
                per = (margin - 1 / (2 * BETA)) ** 2
                slope = 2 * (margin - 1 / (2 * BETA))
            signed = torch.stack([slope, -slope]) * scale / P
            return {"loss": per.mean(), "chosen": BETA * ratio[0], "rejected": BETA * ratio[1],
                    "dlogps": signed[:, :, None] * keep}
        if c["op"] == "policy":
            lp, old, ref, adv = (st[k].detach().to(f64) for k in ("logps", "old", "ref", "adv"))
            keep = st["mask"]
            if adv.dim() == 1:
                adv = adv[:, None].expand_as(lp)
            r = (lp - old).exp()
            hi = (adv > 0) & (lp - old > math.log1p(CLIP_HIGH))
            lo = (adv < 0) & (lp - old < math.log1p(-CLIP_LOW))
            value = -torch.where(hi, (1 + CLIP_HIGH) * adv, torch.where(lo, (1 - CLIP_LOW) * adv, r * adv))
            slope = torch.where(hi | lo, torch.zeros_like(r), -r * adv)
            k3 = torch.expm1(ref - lp) - (ref - lp)
            n = keep.sum(1).to(f64)
            total = n.sum().clamp(min=1)
            if c["reduction"] == "token":
                weight = keep / total
            else:
                weight = keep / n.clamp(min=1)[:, None] / max(1, int((n > 0).sum()))
            return {"loss": ((value + c["kl"] * k3) * weight).sum(), "kl": (k3 * keep).sum() / total,
                    "clipped": ((hi | lo) & keep).sum() / total,
                    "dlogps": (slope - c["kl"] * torch.expm1(ref - lp)) * weight}
        E, keep = c["E"], st["mask"]
        keep = torch.ones(c["T"], dtype=torch.bool, device=DEV) if keep is None else keep
        n = max(1, int(keep.sum()) * c["L"])
        counts = sum(torch.bincount(i[keep].reshape(-1), minlength=E) for i in st["idx"])
        f = counts.to(f64) / n
        mean_p, z = torch.zeros(E, dtype=f64, device=DEV), torch.zeros((), dtype=f64, device=DEV)
        for x in st["logits"]:
            x = x.detach().to(f64)[keep]
            mean_p += torch.softmax(x, -1).sum(0) / n
            z += torch.logsumexp(x, -1).square().sum() / n
        grads = []
        for x in st["logits"]:
            x = x.detach().to(f64)
            p, l = torch.softmax(x, -1), torch.logsumexp(x, -1)
            g = BALANCE * E / n * p * (f - (p @ f)[:, None]) + 2 * ZCOEF / n * p * l[:, None]
            grads.append(g * keep[:, None])
        return {"loss": BALANCE * E * (f * mean_p).sum() + ZCOEF * z, "counts": counts, "dlogits": grads}
