"""Preference, policy and router losses against their formulas in 64 bits.

Tolerances: u = 2^-24. A sum over tokens is formed in fp32 over at most 32 values per lane and
5 shuffle steps, then in fp64, so it errs by less than 64 u times the sum of magnitudes (2^-18);
exponentials, logarithms and the remaining operations add a few u of a result's size, for
which 2^-20 stands. bf16 results are rounded once more (2^-8 of the result).
"""

import math

import pytest
import torch

from pluggy_b200.ops import policy_loss, preference_loss, router_balance_loss

GPU = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        from pluggy_b200.ops import _ext

        torch.cuda.synchronize()
        _ext.check_status()


def gen_for(*key):
    return torch.Generator().manual_seed(sum((i + 1) * int(k) for i, k in enumerate(key)))


def ragged(g, rows, S):
    n = torch.randint(0, S + 1, (rows,), generator=g)
    n[0] = S
    n[-1] = 0 if rows > 2 else n[-1]
    m = torch.arange(S)[None, :] < n[:, None]
    return m & (torch.rand(rows, S, generator=g) < 0.9)  # holes, too


# ------------------------------------------------------------------- preference
def pref_inputs(P, S, dev, ref):
    g = gen_for(P, S)
    lp = -torch.rand(2, P, S, generator=g).square() * 3
    mask = ragged(g, 2 * P, S).view(2, P, S)
    r = None if ref is None else (lp + 0.2 * torch.randn(2, P, S, generator=g)).to(ref).to(dev)
    return lp.to(dev), r, mask.to(dev)


def pref_exact(lp, ref, mask, beta, kind, eps, norm):
    """loss, rewards [2, P], gradient, error bounds of the rewards / beta [2, P]"""
    d = (lp.double() - (0 if ref is None else ref.double())).masked_fill(~mask, 0.0)
    n = mask.sum(-1).clamp_min(1).double() if norm else torch.ones(lp.shape[:2], device=lp.device).double()
    s, bound = d.sum(-1) / n, d.abs().sum(-1) / n * 2.0 ** -18
    h = s[0] - s[1]
    if kind == "sigmoid":
        sp = torch.nn.functional.softplus
        per, dl = (1 - eps) * sp(-beta * h) + eps * sp(beta * h), beta * (torch.sigmoid(beta * h) - 1 + eps)
    elif kind == "hinge":
        per, dl = torch.relu(1 - beta * h), torch.where(beta * h < 1, -beta, 0.0).double()
    else:
        per, dl = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta)
    P = h.numel()
    grad = torch.stack((dl, -dl)) / n / P
    return per.sum() / P, beta * s, grad[..., None] * mask, bound, h, n


def check_pref(lp, ref, mask, beta=0.1, kind="sigmoid", eps=0.0, norm=False, scale=1.0):
    lp = lp.detach().requires_grad_(True)
    loss, ch, rj = preference_loss(lp, ref, mask, beta=beta, kind=kind, label_smoothing=eps,
                                   length_normalized=norm)
    (grad,) = torch.autograd.grad(loss * scale, lp)
    assert not ch.requires_grad and not rj.requires_grad
    eloss, rew, egrad, bound, h, n = pref_exact(lp.detach(), ref, mask, beta, kind, eps, norm)
    dh = bound[0] + bound[1] + 2.0 ** -22 * h.abs()
    for got, want, b in ((ch, rew[0], bound[0]), (rj, rew[1], bound[1])):
        assert ((got - want).abs() <= beta * b + 2.0 ** -20 * want.abs()).all()
    x = (h - 0.5 / beta).abs()
    # the losses' slopes: beta, beta, 2 |x|; their curvatures: beta^2 / 4, none (no pair of
    # these inputs lies within dh of the corner), 2
    per_err = 2 * x * dh + dh ** 2 + 2.0 ** -20 * x ** 2 if kind == "ipo" else beta * dh + 2.0 ** -20
    assert (loss - eloss).abs() <= per_err.mean() + 2.0 ** -20 * eloss.abs()
    if kind == "hinge":
        assert ((1 - beta * h).abs() > beta * dh + 1e-6).all(), "an input on the corner"
    curve = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    tol = (curve * dh / n / h.numel())[..., None] + 2.0 ** -19 * egrad.abs() / 1.0 + beta * 2.0 ** -24 / h.numel()
    assert ((grad - scale * egrad).abs() <= abs(scale) * tol).all()
    assert (grad[~mask] == 0).all()
    return loss.detach(), ch, rj, grad


PREF = [(1, 1), (1, 5), (2, 31), (3, 128), (2, 1023), (5, 1024), (4, 1025), (1, 20000), (33, 260), (700, 3)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("P,S", PREF)
@pytest.mark.parametrize("kind,eps,norm,ref", [
    ("sigmoid", 0.0, False, torch.float32), ("sigmoid", 0.2, True, torch.bfloat16),
    ("hinge", 0.0, False, torch.bfloat16), ("ipo", 0.0, True, torch.float32), ("sigmoid", 0.1, False, None)])
def test_preference(P, S, kind, eps, norm, ref, dev):
    check_pref(*pref_inputs(P, S, dev, ref), kind=kind, eps=eps, norm=norm)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_empty_sequences_and_masked_garbage(dev):
    lp, ref, mask = pref_inputs(4, 600, dev, torch.float32)
    mask[:, 1] = False   # a pair without any token
    mask[1, 2] = False   # one side only
    clean = check_pref(lp, ref, mask)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min):
        dirty = check_pref(torch.where(mask, lp, bad), torch.where(mask, ref, bad), mask)
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)
    assert (clean[3][:, 1] == 0).all()
    mask[:] = False
    loss, ch, rj, grad = check_pref(lp, ref, mask)
    assert abs(loss.item() - math.log(2)) < 1e-6 and (grad == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_extreme_margins(dev):
    """Margins of +-1e4: the sigmoid loss is 0 or linear, never infinite or NaN."""
    lp = torch.zeros(2, 2, 4, device=dev)
    lp[0, 0], lp[1, 1] = -2.5e5, -2.5e5
    mask = torch.ones(2, 2, 4, dtype=torch.bool, device=dev)
    check_pref(lp, None, mask, beta=0.01)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_views_and_streams(dev):
    """Alternating sequences, a sliced token range, transposed tokens and an expanded mask."""
    lp, ref, mask = pref_inputs(6, 515, dev, torch.float32)
    inter = torch.stack((lp[0], lp[1]), 1).reshape(12, 515)
    a = check_pref(inter.view(6, 2, 515).transpose(0, 1), ref, mask)
    wide = torch.full((2, 6, 520), float("nan"), device=dev)
    wide[..., 3:518] = lp
    b = check_pref(wide[..., 3:518], ref, mask)
    c = check_pref(lp.transpose(1, 2).contiguous().transpose(1, 2), ref, mask)
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
    check_pref(lp, ref, mask[:1, :1].expand(2, 6, 515))
    if dev == "cuda":
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            d = check_pref(lp, ref, mask)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(a[0], d[0]) and torch.equal(a[3], d[3])


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_incoming_gradient(dev):
    check_pref(*pref_inputs(3, 700, dev, torch.float32), scale=-0.25)


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_gradient_matches_differences(dev):
    """Perturbing one row's tokens by +-step moves the loss by 2 step times the row's gradient."""
    lp, ref, mask = pref_inputs(2, 64, dev, torch.float32)
    *_, grad = check_pref(lp, ref, mask, beta=0.5)
    step = 2.0 ** -6
    for side in (0, 1):
        e = torch.zeros_like(lp)
        e[side, 0] = step
        up = preference_loss(lp + e, ref, mask, beta=0.5)[0].double()
        dn = preference_loss(lp - e, ref, mask, beta=0.5)[0].double()
        n = int(mask[side, 0].sum())
        # third derivative of softplus(beta h) <= beta^3 / 10 in h, h moves by n step
        tol = (n * step) ** 3 * 0.5 ** 3 / 10 + 2.0 ** -20 * 10
        assert abs((up - dn).item() - 2 * step * grad[side, 0].sum().item()) <= tol


# ----------------------------------------------------------------------- policy
def policy_inputs(R, S, dev, stored=torch.float32, per_token=True):
    g = gen_for(R, S, 3)
    lp = -torch.rand(R, S, generator=g).square() * 3
    old = (lp + 0.2 * torch.randn(R, S, generator=g)).to(stored)
    ref = (lp + 0.4 * torch.randn(R, S, generator=g)).to(stored)
    adv = torch.randn(R, S, generator=g) if per_token else torch.randn(R, generator=g)
    return [t.to(dev) for t in (lp, old, adv, ragged(g, R, S), ref)]


def policy_exact(lp, old, adv, mask, ref, lo, hi, klc, reduction):
    """loss, kl, share, gradient, sum of |terms| of the loss, |terms| of the gradient"""
    f = torch.float64
    lpd = lp.to(f).masked_fill(~mask, 0.0)
    A = (adv.to(f)[:, None].expand(lp.shape) if adv.dim() == 1 else adv.to(f)).masked_fill(~mask, 0.0)
    r = torch.zeros_like(lpd) if old is None else (lp.to(f) - old.to(f)).masked_fill(~mask, 0.0)
    # the comparison is made on fp32 numbers: r and the bounds' logarithms
    r32 = r.float().to(f)
    up = (A > 0) & (r32 > torch.tensor(math.log1p(hi)).float().item())
    dn = (A < 0) & (r32 < torch.tensor(math.log1p(-lo)).float().item())
    ratio = torch.where(up, 1 + hi, torch.where(dn, 1 - lo, r.exp()))
    pg = -ratio * A
    g1 = torch.where(up | dn, 0.0, -r.exp() * A)
    kl = torch.zeros_like(lpd)
    g2 = torch.zeros_like(lpd)
    if ref is not None:
        d = (ref.to(f) - lp.to(f)).masked_fill(~mask, 0.0)
        kl, g2 = torch.expm1(d) - d, -klc * torch.expm1(d)
    n = mask.sum(1).to(f)
    tok = n.sum().clamp_min(1)
    w = mask / tok if reduction == "token" else mask / n.clamp_min(1)[:, None] / (n > 0).sum().clamp_min(1)
    return (((pg + klc * kl) * w).sum(), (kl * mask).sum() / tok, ((up | dn) & mask).sum() / tok,
            (g1 + g2) * w, ((pg.abs() + klc * kl) * w).sum(), (g1.abs() + g2.abs()) * w)


def check_policy(lp, old, adv, mask, ref=None, lo=0.2, hi=0.25, klc=0.0, reduction="token", scale=1.0):
    lp = lp.detach().requires_grad_(True)
    loss, kl, share = policy_loss(lp, old, adv, mask, ref_logps=ref, clip_low=lo, clip_high=hi, kl_coef=klc,
                                  reduction=reduction)
    (grad,) = torch.autograd.grad(loss * scale, lp)
    assert not kl.requires_grad and not share.requires_grad
    eloss, ekl, eshare, egrad, mag, gmag = policy_exact(lp.detach(), old, adv, mask, ref, lo, hi, klc, reduction)
    # kl on the CPU is expm1(d) - d, off by 2^-24 |d| ~ 2^-24 each
    assert (loss - eloss).abs() <= 2.0 ** -18 * mag + 2.0 ** -23 * (1 + klc)
    assert (kl - ekl).abs() <= 2.0 ** -18 * ekl + 2.0 ** -23
    assert (share - eshare).abs() <= 2.0 ** -22
    assert ((grad - scale * egrad).abs() <= abs(scale) * (2.0 ** -20 * gmag + 1e-30)).all()
    assert (grad[~mask] == 0).all()
    return loss.detach(), kl, share, grad


POLICY = [(1, 1), (3, 7), (2, 128), (8, 1023), (5, 1024), (4, 1025), (3, 2049), (2, 9001), (300, 33), (2000, 1)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("R,S", POLICY)
@pytest.mark.parametrize("reduction,per_token,stored,klc", [
    ("token", True, torch.float32, 0.1), ("sequence", False, torch.bfloat16, 0.0),
    ("sequence", True, torch.bfloat16, 0.3), ("token", False, torch.float32, 0.0)])
def test_policy(R, S, reduction, per_token, stored, klc, dev):
    lp, old, adv, mask, ref = policy_inputs(R, S, dev, stored, per_token)
    check_policy(lp, old, adv, mask, ref if klc else None, klc=klc, reduction=reduction)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_policy_empty_rows_and_masked_garbage(dev, reduction):
    lp, old, adv, mask, ref = policy_inputs(6, 700, dev)
    mask[2] = False
    kw = dict(klc=0.2, reduction=reduction)
    clean = check_policy(lp, old, adv, mask, ref, **kw)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(torch.float32).min):
        dirty = check_policy(*(torch.where(mask, t, bad) for t in (lp, old, adv)), mask,
                             torch.where(mask, ref, bad), **kw)
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)
    # an advantage of a row without tokens may be NaN, too
    rowadv = adv[:, 0].clone()
    rowadv[2] = float("nan")
    assert torch.isfinite(check_policy(lp, old, rowadv.nan_to_num(0.0), mask, ref, **kw)[0])
    got = policy_loss(lp, old, rowadv, mask, ref_logps=ref, kl_coef=0.2, reduction=reduction)
    assert all(torch.isfinite(t).all() for t in got)
    mask[:] = False
    assert all((t == 0).all() for t in check_policy(lp, old, adv, mask, ref, **kw))


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_first_update_and_reference_statistics(dev):
    """Without old log-probabilities the ratio is 1; with kl_coef 0 the KL is only reported."""
    lp, old, adv, mask, ref = policy_inputs(5, 333, dev)
    a = check_policy(lp, None, adv, mask)
    b = check_policy(lp, lp.clone(), adv, mask)
    assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3]) and a[2] == 0
    assert check_policy(lp, old, adv, mask, ref, klc=0.0)[1] > 0


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_far_ratios(dev):
    """Ratios of e^+-30 and reference gaps of +-20 stay finite; a passed bound has no gradient."""
    lp = torch.tensor([[-1.0, -31.0, -1.0, -31.0], [-1.0, -21.0, -1.0, -1.0]], device=dev)
    old = torch.tensor([[-31.0, -1.0, -31.0, -1.0], [-1.0, -1.0, -1.0, -1.0]], device=dev)
    ref = torch.tensor([[-1.0, -31.0, -1.0, -31.0], [-21.0, -1.0, -1.0, -1.0 - 1e-4]], device=dev)
    adv = torch.tensor([[1.0, -1.0, -1.0, 1.0], [0.0, 1.0, -1.0, 1.0]], device=dev)
    mask = torch.ones(2, 4, dtype=torch.bool, device=dev)
    grad = check_policy(lp, old, adv, mask, ref, klc=0.0)[3]
    assert grad[0, 0] == 0 and grad[0, 1] == 0
    check_policy(lp, old, adv, mask, ref, klc=0.5)


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_views_and_incoming_gradient(dev):
    lp, old, adv, mask, ref = policy_inputs(7, 515, dev)
    kw = dict(klc=0.1, reduction="sequence")
    a = check_policy(lp, old, adv, mask, ref, **kw)
    wide = torch.full((7, 1 + 2 * 515), float("nan"), device=dev)
    wide[:, 1:516], wide[:, 516:] = lp, old
    b = check_policy(wide[:, 1:516], wide[:, 516:], adv.t().contiguous().t(), mask, ref, **kw)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    check_policy(lp, old, adv[:1, :1].expand(7, 515), mask[:1].expand(7, 515), ref, scale=0.125, **kw)
    check_policy(lp, old, adv[:, 3], mask, ref, scale=-3.0, **kw)


@GPU
def test_policy_second_backward_is_refused():
    lp, old, adv, mask, _ = policy_inputs(2, 64, "cuda")
    loss = policy_loss(lp.requires_grad_(True), old, adv, mask)[0]
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        loss.backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_gradient_matches_differences(dev):
    """Per-token central differences of tokens at least `step` away from a bound."""
    step = 2.0 ** -7
    lp, old, adv, mask, ref = policy_inputs(1, 40, dev)
    r = lp - old
    near = ((r - math.log1p(0.25)).abs() < 2 * step) | ((r - math.log1p(-0.2)).abs() < 2 * step)
    mask = mask & ~near
    grad = check_policy(lp, old, adv, mask, ref, klc=0.3)[3]
    n = int(mask.sum())
    for t in range(40):
        e = torch.zeros_like(lp)
        e[0, t] = step
        f = [policy_loss(lp + s * e, old, adv, mask, ref_logps=ref, clip_low=0.2, clip_high=0.25,
                         kl_coef=0.3)[0].double() for s in (1, -1)]
        # third derivative <= |A| e^r + 0.3 e^d < 20 over these inputs; fp32 rounding of the mean
        tol = step ** 3 / 3 * 20 / n + 2.0 ** -21
        assert abs((f[0] - f[1]).item() - 2 * step * grad[0, t].item()) <= tol


# ----------------------------------------------------------------------- router
def router_inputs(L, T, E, k, dev, dtype, masked):
    g = gen_for(L, T, E, k)
    xs, idx = [], []
    for _ in range(L):
        x = (torch.randn(T, E, generator=g) * 1.5).to(dtype)
        idx.append(torch.topk(x.float() + 1e-3 * torch.rand(T, E, generator=g), k).indices.to(dev))
        xs.append(x.to(dev))
    return xs, idx, (torch.rand(T, generator=g) < 0.7).to(dev) if masked else None


def check_router(xs, idx, mask=None, cb=0.7, cz=0.3, scale=1.0):
    xs = [x.detach().requires_grad_(True) for x in xs]
    T, E = xs[0].shape
    L = len(xs)
    loss, counts = router_balance_loss(xs, idx, balance_coef=cb, z_coef=cz, mask=mask)
    grads = torch.autograd.grad(loss * scale, xs)
    assert counts.dtype == torch.int64 and counts.shape == (E,)
    keep = torch.ones(T, dtype=torch.bool, device=xs[0].device) if mask is None else mask
    n = max(1, L * int(keep.sum()))
    ec = sum(torch.bincount(i[keep].reshape(-1), minlength=E) for i in idx)
    assert torch.equal(counts, ec)
    f = ec.double() / n
    x = torch.stack([v.detach().double() for v in xs])
    x = torch.where(keep[None, :, None], x, 0.0)
    p, lse = torch.softmax(x, -1), torch.logsumexp(x, -1)
    kf = keep.double()
    P = (p * kf[None, :, None]).sum((0, 1)) / n
    bal, z = E * (f * P).sum(), (lse.square() * kf).sum() / n
    # a probability errs by a few u (exponent arguments up to |x| ~ 2^3); sums as above
    assert (loss - (cb * bal + cz * z)).abs() <= 2.0 ** -18 * (cb * bal + cz * z) + 1e-30
    dot = (p * f).sum(-1, keepdim=True)
    want = cb * E / n * p * (f - dot) + 2 * cz / n * p * lse[..., None]
    size = cb * E / n * p * (f + dot) + 2 * cz / n * p * lse[..., None].abs()
    bf = 2.0 ** -8 if xs[0].dtype == torch.bfloat16 else 0.0
    for l in range(L):
        assert grads[l].dtype == xs[l].dtype
        w = scale * want[l] * kf[:, None]
        tol = abs(scale) * 2.0 ** -18 * size[l] + bf * w.abs() + 1e-30
        assert ((grads[l] - w).abs() <= tol).all()
        assert (grads[l][~keep] == 0).all()
    return loss.detach(), counts, torch.stack(grads)


ROUTER = [(1, 1, 1, 1), (1, 3, 5, 2), (2, 65, 8, 2), (1, 257, 60, 4), (3, 100, 64, 8), (24, 33, 128, 8),
          (2, 1000, 128, 8), (1, 70, 160, 6), (2, 90, 256, 8), (1, 50, 257, 3), (1, 40, 512, 10),
          (2, 31, 1000, 8), (1, 20, 1024, 40), (5, 2, 33, 1), (1, 5000, 16, 2)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("L,T,E,k", ROUTER)
@pytest.mark.parametrize("dtype,masked", [(torch.bfloat16, False), (torch.float32, True), (torch.bfloat16, True),
                                          (torch.float32, False)])
def test_router(L, T, E, k, dtype, masked, dev):
    check_router(*router_inputs(L, T, E, k, dev, dtype, masked))


@pytest.mark.parametrize("dev", DEVICES)
def test_router_masked_garbage_empty_and_tied(dev):
    xs, idx, mask = router_inputs(2, 300, 64, 4, dev, torch.bfloat16, True)
    clean = check_router(xs, idx, mask)
    for bad in (float("nan"), float("inf"), float("-inf")):
        dirty = check_router([torch.where(mask[:, None], x, bad) for x in xs], idx, mask)
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)
    loss, counts, grads = check_router(xs, idx, torch.zeros_like(mask))
    assert loss == 0 and (counts == 0).all() and (grads == 0).all()
    # zero logits (a router at its initialisation): every token on the same experts
    zero = [torch.zeros_like(x) for x in xs]
    same = [torch.arange(4, device=dev).expand(300, 4).contiguous() for _ in idx]
    check_router(zero, same)
    # one expert far ahead: probabilities of 0 and 1
    far = [x.clone() for x in xs]
    for x in far:
        x[:, 3] = 300.0
    check_router(far, idx)


@pytest.mark.parametrize("dev", DEVICES)
def test_router_single_tensor_views_and_coefficients(dev):
    xs, idx, _ = router_inputs(1, 130, 128, 8, dev, torch.float32, False)
    a = router_balance_loss(xs[0], idx[0], balance_coef=0.5, z_coef=0.1)
    b = router_balance_loss(xs, idx, balance_coef=0.5, z_coef=0.1)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    wide = torch.zeros(130, 300, device=dev)
    for off in (0, 1, 8):  # rows of a wider projection, on and off a 16-byte boundary
        wide[:, off:off + 128] = xs[0]
        check_router([wide[:, off:off + 128]], [idx[0].t().contiguous().t()])
    check_router([xs[0].t().contiguous().t()], idx)
    check_router(xs, idx, cz=0.0)
    check_router(xs, idx, cb=0.0, scale=-2.5)


@pytest.mark.parametrize("dev", DEVICES)
def test_router_equals_the_models_auxiliary_loss(dev):
    """Balance and z loss of the MoE model, whose own top-k are the given indices."""
    from pluggy_b200.models.qwen3_moe import load_balancing_loss, router_z_loss

    xs, _, _ = router_inputs(3, 200, 64, 4, dev, torch.float32, False)
    idx = [torch.topk(torch.softmax(x, -1), 4).indices for x in xs]
    loss, counts = router_balance_loss(xs, idx, balance_coef=0.01, z_coef=0.001)
    want = 0.01 * load_balancing_loss(xs, 64, 4) + 0.001 * router_z_loss(xs)
    assert (loss - want).abs() <= 2.0 ** -17 * want
    assert counts.sum() == 3 * 200 * 4


@pytest.mark.parametrize("dev", DEVICES)
def test_router_gradient_matches_differences(dev):
    xs, idx, _ = router_inputs(1, 16, 24, 2, dev, torch.float32, False)
    g = check_router(xs, idx, cb=1.0, cz=0.5)[2][0].double()
    u = torch.randn(16, 24, generator=gen_for(9)).to(dev)
    step = 2.0 ** -6
    f = [router_balance_loss(xs[0] + s * step * u, idx[0], balance_coef=1.0, z_coef=0.5)[0].double()
         for s in (1, -1)]
    # |u| < 4: third derivatives of p and lse^2 along u below 4^3 (2 + 2 lse), lse < 8; fp32 noise
    tol = step ** 2 / 6 * 4 ** 3 * 18 + 2.0 ** -18 * 30 / step
    assert abs((f[0] - f[1]).item() / (2 * step) - (g * u).sum().item()) <= tol


@GPU
def test_router_index_outside_is_nan():
    xs, idx, _ = router_inputs(1, 64, 60, 2, "cuda", torch.bfloat16, False)
    idx[0][5, 0] = 60
    assert torch.isnan(router_balance_loss(xs, idx, z_coef=0.0)[0])
    idx[0][5, 0] = -1
    assert torch.isnan(router_balance_loss(xs, idx, z_coef=0.1)[0])


@GPU
def test_losses_repeat_bitwise():
    a = [check_pref(*pref_inputs(40, 5000, "cuda", torch.float32)) for _ in range(2)]
    lp, old, adv, mask, ref = policy_inputs(40, 5000, "cuda")
    b = [check_policy(lp, old, adv, mask, ref, klc=0.1) for _ in range(2)]
    c = [check_router(*router_inputs(4, 5000, 128, 8, "cuda", torch.bfloat16, True)) for _ in range(2)]
    for x, y in (a, b, c):
        for p, q in zip(x, y):
            assert torch.equal(p, q)


# --------------------------------------------------------------------- refusals
def test_preference_refusals():
    lp, m = torch.zeros(2, 3, 4), torch.ones(2, 3, 4, dtype=torch.bool)
    for bad, err in (((lp, None, m.float()), ValueError), ((lp, None, m[0]), ValueError),
                     ((lp[:, :2], None, m), ValueError), ((lp.double(), None, m), TypeError),
                     ((lp, lp.half(), m), TypeError), ((lp, lp.clone().requires_grad_(True), m), ValueError)):
        with pytest.raises(err):
            preference_loss(*bad)
    for kw in (dict(kind="best"), dict(beta=0.0), dict(label_smoothing=0.5),
               dict(kind="ipo", label_smoothing=0.1)):
        with pytest.raises(ValueError):
            preference_loss(lp, None, m, **kw)


def test_policy_refusals():
    lp, m, a = torch.zeros(3, 4), torch.ones(3, 4, dtype=torch.bool), torch.zeros(3)
    for bad, err in (((lp, None, a, m.float()), ValueError), ((lp, lp[:2], a, m), ValueError),
                     ((lp, None, torch.zeros(4), m), ValueError), ((lp.bfloat16(), None, a, m), TypeError),
                     ((lp, lp.half(), a, m), TypeError), ((lp, None, a.double(), m), TypeError),
                     ((lp, lp.clone().requires_grad_(True), a, m), ValueError)):
        with pytest.raises(err):
            policy_loss(*bad)
    for kw in (dict(clip_low=1.0), dict(clip_high=-0.1), dict(reduction="mean"), dict(kl_coef=0.1)):
        with pytest.raises(ValueError):
            policy_loss(lp, None, a, m, **kw)


def test_router_refusals():
    x, i = torch.zeros(5, 8), torch.zeros(5, 2, dtype=torch.int64)
    for bad, err in ((([], []), ValueError), (([x], [i, i]), ValueError), ((x, i.int()), ValueError),
                     ((x, i[:4]), ValueError), (([x, x[:, :4]], [i, i]), ValueError),
                     ((x.double(), i), TypeError), ((x[:, :0], i), ValueError)):
        with pytest.raises(err):
            router_balance_loss(*bad)
    with pytest.raises(ValueError):
        router_balance_loss(x, i, mask=torch.ones(5))


@GPU
def test_refusals_on_the_gpu():
    m = torch.ones(2, 3, 4, dtype=torch.bool, device="cuda")
    with pytest.raises(ValueError):
        preference_loss(torch.zeros(2, 3, 4), None, m)
    with pytest.raises(ValueError):
        policy_loss(torch.zeros(3, 4), None, torch.zeros(3, device="cuda"), m[0])
    x = torch.zeros(2, 1025, device="cuda")
    with pytest.raises(ValueError, match="1024"):
        router_balance_loss(x, torch.zeros(2, 1, dtype=torch.int64, device="cuda"))
    x = torch.zeros(2, 8, device="cuda")
    i = torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="128 layers"):
        router_balance_loss([x] * 129, [i] * 129)


@pytest.mark.parametrize("dev", DEVICES)
def test_nothing_to_do(dev):
    """No pairs, no tokens, no rows."""
    z = torch.zeros(2, 0, 5, device=dev, requires_grad=True)
    assert preference_loss(z, None, z.bool())[0] == 0
    z = torch.zeros(2, 3, 0, device=dev, requires_grad=True)
    loss = preference_loss(z, None, z.bool())[0]
    assert abs(loss.item() - math.log(2)) < 1e-6
    loss.backward()
    for shape in ((0, 4), (3, 0)):
        z = torch.zeros(shape, device=dev, requires_grad=True)
        loss, kl, share = policy_loss(z, None, torch.zeros(shape[0], device=dev), z.bool())
        assert loss == 0 and kl == 0 and share == 0
        loss.backward()
    x = torch.zeros(0, 16, device=dev, requires_grad=True)
    loss, counts = router_balance_loss(x, torch.zeros(0, 2, dtype=torch.int64, device=dev))
    assert loss == 0 and (counts == 0).all()
    loss.backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_reported_kl_may_overflow(dev):
    """With kl_coef 0 a KL estimate beyond fp32 is reported and reaches neither loss nor gradient."""
    lp = torch.tensor([[-100.0, -1.0, -2.0]], device=dev, requires_grad=True)
    adv, mask = torch.ones(1, device=dev), torch.ones(1, 3, dtype=torch.bool, device=dev)
    want = policy_loss(lp, None, adv, mask)[0]
    (egrad,) = torch.autograd.grad(want, lp, retain_graph=True)
    for far in (-1.0, float("-inf")):
        ref = torch.tensor([[far, -1.5, -1.0]], device=dev)
        loss, kl, _ = policy_loss(lp, None, adv, mask, ref_logps=ref)
        (grad,) = torch.autograd.grad(loss, lp)
        assert torch.isinf(kl) and torch.equal(loss, want) and torch.equal(grad, egrad)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("per_token", [False, True])
def test_policy_zero_advantage_and_overflowing_ratio(per_token, dev):
    """exp(99) is beyond fp32, its product with an advantage of 0 is 0; a NaN ratio stays NaN."""
    lp = torch.tensor([[-1.0, -1.0, -1.0], [-1.0, -2.0, -1.0]], device=dev, requires_grad=True)
    old = torch.tensor([[-100.0, -1.5, -100.0], [-1.0, -1.5, -1.0]], device=dev)
    mask = torch.ones(2, 3, dtype=torch.bool, device=dev)
    adv = torch.tensor([0.0, 0.5], device=dev)
    adv = adv[:, None].expand(2, 3).contiguous() if per_token else adv
    loss, _, share = policy_loss(lp, old, adv, mask)
    (grad,) = torch.autograd.grad(loss, lp)
    want, _, _, egrad, mag, gmag = policy_exact(lp.detach(), old, adv, mask, None, 0.2, 0.2, 0.0, "token")
    assert (loss - want).abs() <= 2.0 ** -18 * mag and share == 0
    assert ((grad - egrad).abs() <= 2.0 ** -20 * gmag).all() and (grad[0] == 0).all()
    bad = old.clone()
    bad[0, 1] = float("nan")
    assert torch.isnan(policy_loss(lp, bad, adv, mask)[0])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("op", ["preference", "policy", "router"])
def test_results_may_be_changed_in_place(op, grad, dev):
    """`loss /= n`, `loss += aux` and the like, as on any other tensor."""
    m = torch.ones(2, 3, 40, dtype=torch.bool, device=dev)
    z = torch.randn(2, 3, 40, generator=gen_for(5)).to(dev)
    run = {"preference": lambda x: preference_loss(x, None, m),
           "policy": lambda x: policy_loss(x[0], None, torch.ones(3, device=dev), m[0]),
           "router": lambda x: router_balance_loss(x[0], torch.zeros(3, 2, dtype=torch.int64, device=dev))}[op]
    x = z.clone().requires_grad_(grad)
    want = run(x)
    got = run(x)
    loss = got[0]
    loss /= 4
    loss += 1
    for a, b in zip(got[1:], want[1:]):
        a *= 2
        assert torch.equal(a, 2 * b)
    assert torch.equal(loss, want[0] / 4 + 1)
    if grad:
        assert torch.equal(4 * torch.autograd.grad(loss, x)[0], torch.autograd.grad(want[0], x)[0])


@GPU
@pytest.mark.parametrize("cb,cz", [(0.5, 0.1), (0.5, 0.0), (0.0, 0.1)])
def test_router_index_outside_has_no_finite_gradient(cb, cz):
    """The fractions are unknown then: NaN in the loss and in every kept row's gradient. NaN logits
    stay in their own row."""
    xs, idx, mask = router_inputs(2, 300, 60, 2, "cuda", torch.bfloat16, True)
    mask[5], mask[6] = True, False
    idx[1][5, 0] = 60
    for x in xs:
        x.requires_grad_(True)
    loss, _ = router_balance_loss(xs, idx, balance_coef=cb, z_coef=cz, mask=mask)
    assert torch.isnan(loss)
    for g in torch.autograd.grad(loss, xs):
        assert torch.isnan(g[mask]).all() and (g[~mask] == 0).all()
    idx[1][5, 0] = 0
    xs = [x.detach().clone() for x in xs]
    xs[0][5, 3] = float("nan")
    for x in xs:
        x.requires_grad_(True)
    a, b = torch.autograd.grad(router_balance_loss(xs, idx, balance_coef=cb, z_coef=cz, mask=mask)[0], xs)
    assert torch.isnan(a[5]).all() and torch.isfinite(b).all() and torch.isfinite(a).sum() == a.numel() - 60


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bad", [60, -1, 1 << 40])
def test_router_index_outside_on_every_device(bad, dev):
    xs, idx, mask = router_inputs(2, 100, 60, 2, dev, torch.float32, True)
    mask[5], mask[6] = True, False
    want = router_balance_loss(xs, idx, mask=mask)[1].clone()
    want[idx[0][5, 1]] -= 1
    idx[0][5, 1] = bad
    idx[0][6, 1] = bad  # of a masked token: not looked at
    for x in xs:
        x.requires_grad_(True)
    loss, counts = router_balance_loss(xs, idx, z_coef=0.1, mask=mask)
    assert torch.isnan(loss) and torch.equal(counts, want)
    for g in torch.autograd.grad(loss, xs):
        assert torch.isnan(g[mask]).all() and (g[~mask] == 0).all()
    idx[0][5, 1] = 0
    assert torch.isfinite(router_balance_loss(xs, idx, z_coef=0.1, mask=mask)[0])
