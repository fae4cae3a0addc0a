"""Token log-probabilities of a linear head against the definition in 64 bits.

Tolerances. The kernel's operands are the bf16 values that the reference reads too, so a
logit is off by its fp32 accumulation alone: at most D additions of relative error 2^-23
in the order of sum_k |h_k w_k|, which random signs keep near sqrt(D); 2^-22 sqrt(D)
sum|h w| bounds it and its use in the log-sum-exp with room to spare, and the result's own
rounding and exponentials add a few 2^-23 of its size. The gradients' operand G is rounded
to bf16, whose 8-bit significand makes that 2^-8 of each term at most, and so are gradients of
bf16 inputs (2^-8 of the result): |d grad| <= 2^-7 |G| |operand| per element covers both.
"""

import pytest
import torch

from pluggy_b200.ops import linear_token_logprobs

GPU = pytest.mark.gpu
IGN = -100


@pytest.fixture
def status():
    yield
    if torch.cuda.is_available():
        from pluggy_b200.ops import _ext

        torch.cuda.synchronize()
        _ext.check_status()


def make(T, D, V, dev, ignored=0.3, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed + T + 7 * D + 13 * V)
    h = torch.randn(T, D, generator=g).to(dtype).to(dev)
    w = (torch.randn(V, D, generator=g) * (3.0 / D ** 0.5)).to(dtype).to(dev)
    y = torch.randint(0, V, (T,), generator=g)
    y[torch.rand(T, generator=g) < ignored] = IGN
    return h, w, y.to(dev), torch.randn(T, generator=g).to(dev)


def exact(h, w, y, gout, softcap=None, tau=1.0):
    """(logps, dh, dw, |G| |w|, |G|^T |h|, logit bound) in 64 bits; ignored rows left out."""
    keep = y != IGN
    H = torch.where(keep[:, None], h.double(), 0.0)
    W = w.double()
    a = H @ W.t()
    z = (softcap * torch.tanh(a / softcap) if softcap else a) / tau
    lse = torch.logsumexp(z, 1)
    at = y.clamp_min(0)
    r = torch.arange(len(y), device=y.device)
    lp = torch.where(keep, z[r, at] - lse, 0.0)
    G = -torch.exp(z - lse[:, None])
    G[r, at] += 1.0
    G *= (torch.where(keep, gout.double(), 0.0) / tau)[:, None]
    if softcap:
        G *= 1 - torch.tanh(a / softcap) ** 2
    bound = (H.abs() @ W.abs().t()).max() / tau
    return lp, G @ W, G.t() @ H, G.abs() @ W.abs(), G.abs().t() @ H.abs(), bound


def check_case(h, w, y, gout, softcap=None, tau=1.0, dw_slack=1.0, **kw):
    D = h.shape[1]
    h = h.requires_grad_(True)
    w = w.requires_grad_(True)
    lp = linear_token_logprobs(h, w, y, softcap=softcap, temperature=tau, **kw)
    assert lp.dtype == torch.float32 and lp.shape == y.shape
    dh, dw = torch.autograd.grad(lp, (h, w), gout)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    with torch.no_grad():
        lp2 = linear_token_logprobs(h, w, y, softcap=softcap, temperature=tau, **kw)
        ref, rdh, rdw, bdh, bdw, bound = exact(h, w, y, gout, softcap, tau)
    tol = 2.0 ** -22 * D ** 0.5 * bound + 2.0 ** -20 * ref.abs()
    assert ((lp - ref).abs() <= tol).all()
    assert ((lp2 - ref).abs() <= tol).all()
    assert (lp[y == IGN] == 0).all()
    assert ((dh - rdh).abs() <= 2.0 ** -7 * bdh + 1e-6).all()
    assert ((dw - rdw).abs() <= dw_slack * 2.0 ** -7 * bdw + 1e-6).all()
    return lp, dh, dw


@pytest.mark.parametrize("softcap,tau", [(None, 1.0), (5.0, 0.7)])
@pytest.mark.parametrize("T,D,V", [(1, 8, 1), (7, 24, 33), (40, 64, 301)])
def test_cpu_matches_definition(T, D, V, softcap, tau):
    check_case(*make(T, D, V, "cpu", dtype=torch.float32), softcap, tau)


CASES = [(1, 64, 1), (1, 1024, 4099), (2, 8, 33), (31, 72, 255), (127, 256, 1000), (128, 64, 256),
         (129, 520, 257), (256, 128, 511), (257, 128, 513), (700, 256, 8191), (1025, 136, 2049),
         (3000, 64, 5001)]


@GPU
@pytest.mark.parametrize("T,D,V", CASES)
@pytest.mark.parametrize("softcap,tau", [(None, 1.0), (4.0, 0.6)])
def test_kernel_matches_definition(T, D, V, softcap, tau, status):
    check_case(*make(T, D, V, "cuda"), softcap, tau)


@GPU
@pytest.mark.parametrize("ignored", [0.0, 1.0])
@pytest.mark.parametrize("T", [1, 300])
def test_kernel_all_or_no_rows_ignored(T, ignored, status):
    lp, dh, dw = check_case(*make(T, 128, 700, "cuda", ignored=ignored))
    if ignored == 1.0:
        assert (lp == 0).all() and (dh == 0).all() and (dw == 0).all()


@GPU
@pytest.mark.parametrize("softcap", [None, 4.0])
@pytest.mark.parametrize("workspace", [0, 512 * 2 * 600, 512 * 2 * 2099])
def test_kernel_vocabulary_ranges(workspace, softcap, status):
    """Less workspace than the exponentials take: they are recomputed by vocabulary ranges."""
    check_case(*make(512, 128, 2100, "cuda"), softcap, 0.9, workspace_bytes=workspace)


@pytest.fixture
def kept(monkeypatch):
    """The forward keeps its exponentials at any size."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0)


# With kept exponentials the hidden rows of dW are rounded to bf16 once more, after their scaling
KEPT_DW = 1.5


@GPU
@pytest.mark.parametrize("T,D,V", CASES)
@pytest.mark.parametrize("softcap,tau", [(None, 1.0), (4.0, 0.6)])
def test_kernel_with_kept_exponentials(T, D, V, softcap, tau, kept, status):
    check_case(*make(T, D, V, "cuda"), softcap, tau, dw_slack=KEPT_DW)


@GPU
def test_kernel_kept_exponentials_with_long_sums(kept, status):
    """D above 512: several accumulator pieces for each logit."""
    for D in (520, 1024, 2056):
        check_case(*make(300, D, 1500, "cuda"), dw_slack=KEPT_DW)


@GPU
@pytest.mark.parametrize("fallback", [True, False])
def test_kernel_unlikely_labels(fallback, monkeypatch, status):
    """Labels at log-probabilities of -20 to -1000 and beyond, out of the range of the kept
    exponentials: the gradient is recomputed, as exact as any other."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if fallback else 1 << 62)
    h, w, y, g = make(300, 64, 700, "cuda", ignored=0.2)
    h2 = (h.float() * torch.linspace(2, 300, 300, device="cuda")[:, None]).bfloat16()
    lp, dh, dw = check_case(h2, w, y, g)
    assert lp.min() < -1000
    # within the range, but far from the usual one
    h3 = (h.float() * torch.linspace(1, 5, 300, device="cuda")[:, None]).bfloat16()
    lp, dh, dw = check_case(h3, w, y, g, dw_slack=KEPT_DW if fallback else 1.0)
    assert -97 < lp.min() < -30


@GPU
def test_kernel_backward_twice(kept, status):
    """A second backward through the same call gives the same gradients."""
    h, w, y, g = make(300, 64, 900, "cuda")
    h.requires_grad_(True)
    w.requires_grad_(True)
    lp = linear_token_logprobs(h, w, y)
    a = torch.autograd.grad(lp, (h, w), g, retain_graph=True)
    torch.autograd.grad(lp, (h, w), -3.0 * g, retain_graph=True)
    b = torch.autograd.grad(lp, (h, w), g)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@GPU
def test_kernel_kept_masked_vocabulary_and_garbage(kept, status):
    """Entries at -inf first in the vocabulary, NaN hidden rows where labels are ignored."""
    D, V = 64, 900
    h, w, y, g = make(300, D, V, "cuda")
    h = h.abs()
    y = torch.where(y == IGN, y, y.clamp_min(400))
    ref = exact(h, w[300:], torch.where(y == IGN, y, y - 300), g)
    h2 = h.clone()
    h2[y == IGN] = float("nan")
    w2 = w.clone()
    w2[:300] = float("-inf")
    h2.requires_grad_(True)
    lp = linear_token_logprobs(h2, w2, y)
    assert ((lp - ref[0]).abs() <= 2.0 ** -22 * 8 * ref[-1] + 2.0 ** -20 * ref[0].abs()).all()
    # the weight's gradient needs no product with the -inf rows
    wr = w2.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(linear_token_logprobs(h2.detach(), wr, y), wr, g)
    assert (dw[:300] == 0).all()
    assert ((dw[300:] - ref[2]).abs() <= KEPT_DW * 2.0 ** -7 * ref[4] + 1e-6).all()


@GPU
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_ignored_rows_do_not_reach_anything(bad, status):
    """NaN and infinities in the hidden rows of ignored tokens change nothing."""
    h, w, y, g = make(600, 128, 1000, "cuda")
    clean = check_case(h.clone(), w.clone(), y, g)
    h2 = h.clone()
    h2[y == IGN] = bad
    h2.requires_grad_(True)
    w2 = w.clone().requires_grad_(True)
    gb = torch.where(y == IGN, torch.full_like(g, float("nan")), g)
    lp = linear_token_logprobs(h2, w2, y)
    dh, dw = torch.autograd.grad(lp, (h2, w2), gb)
    for a, b in zip((lp, dh, dw), clean):
        assert torch.equal(a, b)


@GPU
def test_kernel_extreme_logits(status):
    """Logits of +-1e4 keep finite log-probabilities; equal logits give -log V."""
    D, V = 64, 500
    h = torch.zeros(3, D, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    h[0, 0], h[1, 0], w[7, 0] = 100.0, -100.0, 100.0
    y = torch.tensor([7, 7, 3], device="cuda")
    lp = linear_token_logprobs(h, w, y)
    ref = exact(h, w, y, torch.ones(3, device="cuda"))[0]
    assert ((lp - ref).abs() <= 2.0 ** -20 * (1 + ref.abs())).all()


@GPU
def test_kernel_minus_infinity_logits(status):
    """A vocabulary entry at -inf (a masked logit) has probability 0 and gradient 0."""
    D, V = 64, 300
    h, w, y, g = make(200, D, V, "cuda", ignored=0.0)
    h = h.abs()  # positive, so that a weight row of -inf gives -inf logits
    y = y.clamp_max(V - 2)
    w2 = w.clone()
    w2[V - 1] = float("-inf")
    lp = linear_token_logprobs(h, w2, y)
    ref, *_, bound = exact(h, w[:V - 1], y, g)
    assert ((lp - ref).abs() <= 2.0 ** -22 * 8 * bound + 2.0 ** -20 * ref.abs()).all()


@GPU
def test_kernel_types_views_and_shapes(status):
    """fp32 inputs (cast to bf16 for the products), a cached bf16 weight, [B, S] labels and
    strided hidden states."""
    h, w, y, g = make(6 * 50, 128, 900, "cuda")
    hf = h.float().view(6, 50, 128).requires_grad_(True)
    wf = w.float().requires_grad_(True)
    lp = linear_token_logprobs(hf, wf, y.view(6, 50), weight_lowp=w)
    dh, dw = torch.autograd.grad(lp, (hf, wf), g.view(6, 50))
    assert dh.dtype == dw.dtype == torch.float32 and dh.shape == hf.shape
    ref, rdh, rdw, bdh, bdw, bound = exact(h, w, y, g)
    assert ((lp.view(-1) - ref).abs() <= 2.0 ** -22 * 12 * bound + 2.0 ** -20 * ref.abs()).all()
    assert ((dh.view(-1, 128) - rdh).abs() <= 2.0 ** -7 * bdh + 1e-6).all()
    assert ((dw - rdw).abs() <= 2.0 ** -7 * bdw + 1e-6).all()
    big = torch.zeros(300, 3, 128, device="cuda", dtype=torch.bfloat16)
    big[:, 1] = h
    assert torch.equal(linear_token_logprobs(big[:, 1], w, y), lp.view(-1).detach())
    odd = torch.zeros(300 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(300, 128)
    odd.copy_(h)
    assert torch.equal(linear_token_logprobs(odd, w, y), lp.view(-1).detach())


@GPU
def test_kernel_only_one_gradient_asked(status):
    h, w, y, g = make(400, 64, 700, "cuda")
    both = check_case(h.clone(), w.clone(), y, g)
    hr = h.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_token_logprobs(hr, w, y), hr, g)[0], both[1])
    wr = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_token_logprobs(h, wr, y), wr, g)[0], both[2])


@GPU
def test_kernel_gradient_matches_differences(status):
    """Central differences along a direction. hidden and weight lie on a grid of 2^-4 (below
    2) and the step is 2^-6, so every perturbed value is a bf16 value. The difference's own
    error is step^2 / 6 times a third derivative of order |u|^3 ~ (step-scaled logit change)^3."""
    gen = torch.Generator().manual_seed(5)
    T, D, V, step = 64, 32, 200, 2.0 ** -6
    h = (torch.randint(-16, 17, (T, D), generator=gen) / 16).cuda()
    w = (torch.randint(-16, 17, (V, D), generator=gen) / 16).cuda()
    y = torch.randint(0, V, (T,), generator=gen).cuda()
    u = (torch.randint(0, 2, (T, D), generator=gen) * 2.0 - 1.0).cuda()
    u *= torch.rand(T, D, generator=gen).cuda() < 0.25
    hb, wb = h.bfloat16().requires_grad_(True), w.bfloat16()
    lp = linear_token_logprobs(hb, wb, y)
    (dh,) = torch.autograd.grad(lp.sum(), hb)
    up = linear_token_logprobs((h + step * u).bfloat16(), wb, y).double()
    dn = linear_token_logprobs((h - step * u).bfloat16(), wb, y).double()
    diff = (up - dn) / (2 * step)
    want = (dh.double() * u).sum(1)
    # |u w| <= 8 per logit: third derivative of log-sum-exp <= 8^3; plus fp32 noise / step and
    # bf16 rounding of the gradient (2^-7 of sum |dh|, |G| |W| <= 2 x 8)
    tol = step ** 2 / 6 * 8.0 ** 3 + 2.0 ** -20 * 10 / step + 2.0 ** -7 * 16
    assert ((diff - want).abs() <= tol).all()


@GPU
def test_kernel_is_repeatable(status):
    h, w, y, g = make(900, 256, 3000, "cuda")
    a = check_case(h.clone(), w.clone(), y, g)
    b = check_case(h.clone(), w.clone(), y, g)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


@GPU
def test_kernel_on_another_stream(status):
    h, w, y, g = make(500, 128, 1000, "cuda")
    a = check_case(h.clone(), w.clone(), y, g)[0].detach()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = linear_token_logprobs(h, w, y)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a, b)


@GPU
def test_label_outside_the_vocabulary_is_nan(status):
    h, w, y, g = make(300, 64, 100, "cuda", ignored=0.0)
    y2 = y.clone()
    y2[5], y2[6] = 100, -7
    for kw in ({}, {"train": True}):
        hr = h.clone().requires_grad_(bool(kw))
        lp = linear_token_logprobs(hr, w, y2)
        assert torch.isnan(lp[5:7]).all() and torch.isfinite(lp[7:]).all() and torch.isfinite(lp[:5]).all()
    (dh,) = torch.autograd.grad(lp, hr, g)
    assert (dh[5:7] == 0).all() and torch.isfinite(dh).all()
    assert torch.isnan(linear_token_logprobs(h[5:7], w, y2[5:7])).all()


def test_refusals():
    h, w, y = torch.zeros(4, 16), torch.zeros(9, 16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="hidden"):
        linear_token_logprobs(h, torch.zeros(9, 8), y)
    with pytest.raises(ValueError, match="labels"):
        linear_token_logprobs(h, w, y[:3])
    with pytest.raises(ValueError, match="labels"):
        linear_token_logprobs(h, w, y.int())
    with pytest.raises(ValueError, match="temperature"):
        linear_token_logprobs(h, w, y, temperature=0.0)
    with pytest.raises(ValueError, match="softcap"):
        linear_token_logprobs(h, w, y, softcap=-1.0)
    with pytest.raises(ValueError, match="empty"):
        linear_token_logprobs(h, torch.zeros(0, 16), y)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        linear_token_logprobs(h.double(), w, y)
    with pytest.raises(ValueError, match="weight_lowp"):
        linear_token_logprobs(h, w, y, weight_lowp=w)


def test_no_tokens():
    lp = linear_token_logprobs(torch.zeros(2, 0, 16, requires_grad=True), torch.zeros(9, 16),
                               torch.zeros(2, 0, dtype=torch.int64))
    assert lp.shape == (2, 0)


@GPU
def test_refusals_on_the_gpu(status):
    y = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="multiple of 8"):
        linear_token_logprobs(torch.zeros(4, 12, device="cuda"), torch.zeros(9, 12, device="cuda"), y)
    with pytest.raises(ValueError, match="one device"):
        linear_token_logprobs(torch.zeros(4, 16, device="cuda"), torch.zeros(9, 16), y)
    lp = linear_token_logprobs(torch.zeros(0, 16, device="cuda", requires_grad=True),
                               torch.zeros(9, 16, device="cuda"), y[:0])
    assert lp.shape == (0,)
    lp.sum().backward()


@GPU
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kernel_kept_repeated_labels(dtype, kept, status):
    """Long runs of one label (more than one block lists at a time), an ignore_index that is a
    vocabulary entry, and labels outside the vocabulary."""
    h, w, y, g = make(700, 648, 300, "cuda", ignored=0.0)
    y[100:500] = 7
    y[3:40] = 299
    y[600:650] = 11
    for ign in (-100, 11):
        z = torch.where(y == 11, IGN, y) if ign == 11 else y
        hr, wr = h.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
        lp = linear_token_logprobs(hr, wr, y, ign)
        dh, dw = torch.autograd.grad(lp, (hr, wr), g)
        ref, rdh, rdw, bdh, bdw, bound = exact(h, w, z, g)
        assert ((lp - ref).abs() <= 2.0 ** -22 * 648 ** 0.5 * bound + 2.0 ** -20 * ref.abs()).all()
        assert ((dh - rdh).abs() <= 2.0 ** -7 * bdh + 1e-6).all()
        assert ((dw - rdw).abs() <= KEPT_DW * 2.0 ** -7 * bdw + 1e-6).all()
    y2 = y.clone()
    y2[5], y2[6] = 1 << 40, -5
    lp = linear_token_logprobs(h.requires_grad_(True), w.requires_grad_(True), y2)
    dh, dw = torch.autograd.grad(lp, (h, w), g)
    assert torch.isnan(lp[5:7]).all() and torch.isfinite(dh).all() and torch.isfinite(dw).all()


@GPU
@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("T,D,V", [(1, 64, 300), (300, 128, 700), (1500, 520, 900), (5000, 64, 2000)])
def test_kernel_label_entries_are_not_rounded(T, D, V, keep, monkeypatch, status):
    """The labels' entries of G, most of a gradient, stay in fp32; bf16 rounds the others (2^-8 of
    a term; with kept exponentials twice in dW) and the results (2^-8). 2^-14 of all terms covers
    G's own error in fp32 (logits of order 10 that are 1e-6 off). Labels repeat: low ids are
    frequent."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if keep else 1 << 62)
    h, w, y, g = make(T, D, V, "cuda", ignored=0.2)
    frequent = (V * torch.rand(T, generator=torch.Generator().manual_seed(T)).pow(3)).long().cuda()
    y = torch.where(y == IGN, y, frequent)
    h.requires_grad_(True)
    w.requires_grad_(True)
    dh, dw = torch.autograd.grad(linear_token_logprobs(h, w, y), (h, w), g)
    with torch.no_grad():
        H, W = torch.where((y != IGN)[:, None], h.double(), 0.0), w.double()
        go = torch.where(y != IGN, g.double(), 0.0)[:, None]
        G = -torch.softmax(H @ W.t(), 1) * go
        own = torch.zeros_like(G).scatter_(1, y.clamp_min(0)[:, None], 1.0)
        rest, G = (G * (1 - own)).abs(), G + own * go
        A = G.abs()
        rdh, rdw = G @ W, G.t() @ H
        tol_h = 2.0 ** -8 * (rdh.abs() + rest @ W.abs()) + 2.0 ** -14 * (A @ W.abs()) + 1e-6
        tol_w = (2.0 ** -8 * (rdw.abs() + (2.01 if keep else 1) * (rest.t() @ H.abs()))
                 + 2.0 ** -14 * (A.t() @ H.abs()) + 1e-6)
    assert ((dh - rdh).abs() <= tol_h).all()
    assert ((dw - rdw).abs() <= tol_w).all()


@GPU
@pytest.mark.parametrize("V", [904, 901])
@pytest.mark.parametrize("keep", [True, False])
def test_kernel_saved_tensors_on_the_host(V, keep, monkeypatch, status):
    """Saved-tensor hooks that hand back contiguous copies, vocabularies of no whole 16 bytes too."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if keep else 1 << 62)
    h, w, y, g = make(300, 64, V, "cuda")
    h.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(linear_token_logprobs(h, w, y), (h, w), g)
    with torch.autograd.graph.save_on_cpu():
        lp = linear_token_logprobs(h, w, y)
    for a, b in zip(torch.autograd.grad(lp, (h, w), g), want):
        assert torch.equal(a, b)


@GPU
def test_kernel_status_word_is_not_a_saved_tensor(status):
    """Saved-tensor hooks would hand the backward a copy, and its reports would be lost."""
    from pluggy_b200.ops._ext import status_word

    h, w, y, g = make(300, 64, 90, "cuda")
    seen = []

    def pack(t):
        seen.append(t.data_ptr())
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        lp = linear_token_logprobs(h.requires_grad_(True), w, y)
    assert seen and status_word().data_ptr() not in seen
    torch.autograd.grad(lp, h, g)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
def test_label_outside_is_nan_on_every_device(dev):
    h, w, _, g = make(6, 16, 9, dev, dtype=torch.float32)
    y = torch.tensor([0, 9, -3, IGN, 8, 1 << 40], device=dev)
    h.requires_grad_(True)
    w.requires_grad_(True)
    lp = linear_token_logprobs(h, w, y)
    assert torch.isnan(lp[[1, 2, 5]]).all() and torch.isfinite(lp[[0, 3, 4]]).all() and lp[3] == 0
    dh, dw = torch.autograd.grad(lp, (h, w), g)
    assert (dh[[1, 2, 3, 5]] == 0).all() and torch.isfinite(dh).all() and torch.isfinite(dw).all()
    assert (dh[[0, 4]] != 0).any(1).all()
    # ignore_index may be a vocabulary entry
    assert (linear_token_logprobs(h, w, y, ignore_index=8)[4] == 0)


def test_overlapping_rows_are_copied():
    """Rows expanded from one and sliding windows: their stride is no row stride of a tensor map."""
    from pluggy_b200.ops.logprob import _rows_aligned

    x = torch.randn(1, 64)
    for t in (x.expand(5, 64), x.view(-1).as_strided((4, 32), (8, 1)), x.view(8, 8).t()):
        c = _rows_aligned(t)
        assert c.is_contiguous() and torch.equal(c, t)
    y = torch.randn(6, 128)[:, :64]
    assert _rows_aligned(y) is y or y.data_ptr() % 16


@GPU
@pytest.mark.parametrize("T", [1, 5, 200, 300])
def test_kernel_overlapping_rows(T, status):
    """Hidden rows expanded from one, a sliding window over one buffer, one weight row for all."""
    h, w, y, g = make(T, 64, 500, "cuda", ignored=0.0)
    for hv in (h[:1].expand(T, 64), h.new_empty(8 * T + 56).copy_(torch.randn(8 * T + 56)).as_strided((T, 64), (8, 1))):
        lp = linear_token_logprobs(hv, w, y)
        assert torch.equal(lp, linear_token_logprobs(hv.contiguous(), w, y))
        ref, *_, bound = exact(hv.contiguous(), w, y, g)
        assert ((lp - ref).abs() <= 2.0 ** -22 * 8 * bound + 2.0 ** -20 * ref.abs()).all()
        a, b = hv.detach().requires_grad_(True), hv.contiguous().requires_grad_(True)
        (da,) = torch.autograd.grad(linear_token_logprobs(a, w, y), a, g)
        (db,) = torch.autograd.grad(linear_token_logprobs(b, w, y), b, g)
        assert torch.equal(da, db)
    lp = linear_token_logprobs(h, w[:1].expand(500, 64), y)
    assert ((lp + torch.log(torch.tensor(500.0))).abs() <= 2.0 ** -22 * 8 * bound + 2.0 ** -20 * 7).all()


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=GPU)])
@pytest.mark.parametrize("softcap", [float("nan"), float("inf")])
def test_softcap_that_is_no_number_is_refused(softcap, dev):
    """NaN read as no softcap on CUDA, infinity as 0 * inf."""
    h, w, y, _ = make(3, 16, 9, dev, dtype=torch.float32)
    with pytest.raises(ValueError, match="softcap"):
        linear_token_logprobs(h, w, y, softcap=softcap)


@GPU
@pytest.mark.parametrize("far", [-95.0, -71.0, -67.0, -40.0])
def test_kernel_unlikely_labels_with_small_gradients(far, kept, status):
    """Labels at log-probability `far`, incoming gradients of 1e-8 and hidden values of 0.02: no
    factor of dW leaves bf16's range, so that the bound holds relative to the terms. 1e-30 stands
    for entries of probability below 1e-20."""
    gen = torch.Generator().manual_seed(0)
    T, D, V = 300, 64, 700
    h = (0.02 * torch.randn(T, D, generator=gen)).bfloat16().cuda()
    w = (156 * torch.randn(V, D, generator=gen)).bfloat16().cuda()
    y = (torch.log_softmax(h.double() @ w.double().t(), 1) - far).abs().argmin(1)
    g = torch.full((T,), 1e-8, device="cuda")
    lp, rdh, rdw, bdh, bdw, _ = exact(h, w, y, g)
    assert (lp.median() - far).abs() < 1  # near -40 single rows have no label this close
    h.requires_grad_(True)
    w.requires_grad_(True)
    dh, dw = torch.autograd.grad(linear_token_logprobs(h, w, y), (h, w), g)
    # 2^-14: G's own error in fp32 (logits of order 100 that are 1e-5 off)
    assert ((dh - rdh).abs() <= (2.0 ** -7 + 2.0 ** -14) * bdh + 1e-30).all()
    assert ((dw - rdw).abs() <= KEPT_DW * (2.0 ** -7 + 2.0 ** -14) * bdw + 1e-30).all()


@GPU
@pytest.mark.parametrize("D", [1032, 2056, 2560])
@pytest.mark.parametrize("softcap,tau", [(4.0, 0.6), (None, 1.0)])
@pytest.mark.parametrize("keep", [False, True])
def test_kernel_long_sums_with_softcap(D, softcap, tau, keep, monkeypatch, status):
    """D above 1024: a logit is summed in several accumulator pieces (above 512 where at most 128
    rows are scored), with and without a softcap, scoring and both gradients."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if keep else 1 << 62)
    for T, V in ((300, 1500), (100, 700)):
        check_case(*make(T, D, V, "cuda"), softcap, tau, dw_slack=KEPT_DW if keep else 1.0)


@GPU
@pytest.mark.parametrize("softcap,tau", [(4.0, 0.6), (None, 1.0)])
@pytest.mark.parametrize("keep", [False, True])
def test_kernel_many_tokens_of_wide_rows(softcap, tau, keep, monkeypatch, status):
    """More tokens than the search through all labels takes (they are sorted), rows wider than a
    block's 1024 columns."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if keep else 1 << 62)
    check_case(*make(4500, 1288, 600, "cuda"), softcap, tau, dw_slack=KEPT_DW if keep else 1.0)
