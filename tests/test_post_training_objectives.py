"""The post-training objectives on models, and the MoE model's fused router losses."""

import gc
import importlib.util
import os

import pytest
import torch

from pluggy_b200.models.builder import build_model
from pluggy_b200.objectives.builder import build_objective

GPU = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=GPU)]
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IGN = -100


def small(name="qwen3_dense", dev="cpu", **kw):
    cfg = dict(num_layers=2, num_heads=2, num_kv_heads=1, emb_dim=128, head_dim=64, vocab_size=200)
    cfg.update({"qwen3_moe": dict(moe_ffn_dim=128, num_experts=32, top_k=4, router_init_std=0.02),
                "gemma4": dict(ffn_dim=128, global_head_dim=64, sliding_window=16,
                               final_logit_softcapping=3.0)}.get(name, dict(ffn_dim=256)))
    cfg.update(kw)
    torch.manual_seed(0)
    m = build_model(name, cfg)
    m.init_weights(0.2) if name == "gemma4" else m.init_weights()
    return m.to(dev)


def pairs(dev, P=3, S=128, V=200):
    g = torch.Generator().manual_seed(1)
    out = {}
    for side in ("chosen", "rejected"):
        ids = torch.randint(0, V, (P, S), generator=g)
        labels = ids.clone()
        labels[:, :4] = IGN
        labels[1, 70:] = IGN
        out[f"{side}_ids"], out[f"{side}_labels"] = ids.to(dev), labels.to(dev)
    return out


def logits_logps(model, ids, labels):
    """[B, S] log-probabilities from the model's full logits, shifted like the objectives'."""
    lp = torch.log_softmax(model(ids).float(), -1)
    y = torch.cat((labels[:, 1:], torch.full_like(labels[:, :1], IGN)), 1)
    return torch.where(y == IGN, 0.0, lp.gather(2, y.clamp_min(0)[..., None])[..., 0])


@pytest.mark.parametrize("name", ["qwen3_dense", "gemma4", "qwen3_moe"])
def test_scores_are_the_models_log_probabilities(name):
    """On CPU in fp32: the same numbers as from the logits, the logit softcap included."""
    m = small(name)
    b = pairs("cpu")
    got = build_objective("PREFERENCE", {}).score(m, b)
    assert not got.requires_grad
    with torch.no_grad():
        for i, side in enumerate(("chosen", "rejected")):
            want = logits_logps(m, b[f"{side}_ids"], b[f"{side}_labels"])
            assert torch.allclose(got[i], want, atol=1e-5, rtol=1e-5)


@GPU
def test_scores_on_the_gpu_match_the_cpu():
    """bf16 forward and head against fp32: log-probabilities of about -5 to 2^-6 of that."""
    b = pairs("cpu")
    cpu = build_objective("PREFERENCE", {}).score(small(), b)
    gpu = build_objective("PREFERENCE", {}).score(small(dev="cuda"), {k: v.cuda() for k, v in b.items()})
    assert ((gpu.cpu() - cpu).abs() <= 0.08).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_preference_objective_at_the_reference(dev):
    """Policy = reference: loss log 2, no rewards, and a gradient that favours the chosen."""
    m = small(dev=dev)
    obj = build_objective("PREFERENCE", dict(beta=0.5))
    b = pairs(dev)
    b["ref_logps"] = obj.score(m, b)
    loss = obj.compute_loss(m, b)
    assert abs(loss.item() - 0.6931472) < 1e-5
    assert obj.metrics["chosen_reward"] == 0 and obj.metrics["rejected_reward"] == 0
    loss.backward()
    with torch.no_grad():
        for p in m.parameters():
            if p.grad is not None:
                p -= 0.05 * p.grad
        assert obj.compute_loss(m, b) < loss
        assert obj.metrics["chosen_reward"] > obj.metrics["rejected_reward"]


@pytest.mark.parametrize("dev", DEVICES)
def test_policy_objective_first_update(dev):
    """Without old log-probabilities the gradient is that of -sum A log p / n."""
    m = small(dev=dev)
    obj = build_objective("POLICY", {})
    b = pairs(dev)
    batch = {"input_ids": b["chosen_ids"], "labels": b["chosen_labels"],
             "advantages": torch.tensor([1.0, -2.0, 0.5], device=dev)}
    loss = obj.compute_loss(m, batch)
    (g,) = torch.autograd.grad(loss, m.lm_head.weight)
    from pluggy_b200.objectives.post_training import token_logprobs

    lp, mask = token_logprobs(m, batch["input_ids"], batch["labels"])
    want = -(lp * batch["advantages"][:, None] * mask).sum() / mask.sum()
    (gw,) = torch.autograd.grad(want, m.lm_head.weight)
    assert (g - gw).norm() <= 2.0 ** -7 * gw.norm()
    assert obj.metrics["clipped"] == 0


def test_objectives_refuse_what_they_cannot_use():
    m = small()
    b = pairs("cpu")
    pref, pol = build_objective("PREFERENCE", {}), build_objective("POLICY", dict(kl_coef=0.1))
    with pytest.raises(ValueError, match="ref_logps"):
        pref.compute_loss(m, b)
    with pytest.raises(ValueError, match="chosen_ids"):
        build_objective("PREFERENCE", dict(reference_free=True)).compute_loss(m, {"input_ids": b["chosen_ids"]})
    with pytest.raises(ValueError, match="advantages"):
        pol.compute_loss(m, {"input_ids": b["chosen_ids"], "labels": b["chosen_labels"]})
    build_objective("PREFERENCE", dict(reference_free=True)).compute_loss(m, b)

    class Split:
        dim = "tp"

        class mesh:
            size = staticmethod(lambda dim: 2)

    m.tp = Split()
    with pytest.raises(NotImplementedError, match="tp"):
        build_objective("PREFERENCE", dict(reference_free=True)).compute_loss(m, b)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("padded", [False, True])
def test_fused_router_losses_match_the_default(dev, padded):
    """Same loss, gradients and counts; with a padding mask, those of the tokens that count."""
    ids = torch.randint(0, 200, (2, 128), generator=torch.Generator().manual_seed(3)).to(dev)
    mask = None
    if padded:
        mask = torch.ones(2, 128, dtype=torch.long, device=dev)
        mask[0, 100:] = 0
    got = []
    # both read one forward pass: on the GPU two passes differ in the last bits of the logits
    # (the model's split sums add in any order)
    m = small("qwen3_moe", dev, router_aux_loss_coef=0.1)
    m(ids, attention_mask=mask)
    for fused in (False, True):
        m.fused_router_losses = fused
        aux = m.aux_loss()
        if padded and not fused:  # the default counts padded tokens: restate it without them
            from pluggy_b200.models.qwen3_moe import load_balancing_loss, router_z_loss

            keep = mask.bool().reshape(-1)
            logits = [x[keep] for x in m._router_logits]
            aux = 0.1 * load_balancing_loss(logits, 32, 4) + 0.001 * router_z_loss(logits)
        grads = torch.autograd.grad(aux, [b.ffn.router.weight for b in m.blocks], retain_graph=True)
        got.append((aux.detach(), grads, m.last_tokens_per_expert))
    (a, ga, ca), (b, gb, cb) = got
    assert abs(a - b) <= 2.0 ** -16 * a
    for x, y in zip(ga, gb):
        # on the GPU the routers' logits, and so their gradients, are bf16
        assert (x - y).norm() <= (2.0 ** -7 if dev == "cuda" else 1e-4) * x.norm()
    if not padded:
        assert torch.equal(ca, cb)
    assert cb.sum() == (228 if padded else 256) * 4 * 2


@pytest.mark.parametrize("dev", DEVICES)
def test_example_runs(dev):
    spec = importlib.util.spec_from_file_location("post_training_example",
                                                  os.path.join(ROOT, "examples", "post_training.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    assert ex.main(["--device", dev, "--steps", "3"]) == 0


@GPU
@pytest.mark.parametrize("keep", [False, True])
def test_operators_replay_from_a_cuda_graph(keep, monkeypatch):
    """Forward and backward captured once: a replay on new inputs, other rows ignored among them,
    gives what eager calls give."""
    from pluggy_b200.ops import linear_token_logprobs, logprob, policy_loss, preference_loss, router_balance_loss

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0 if keep else 1 << 62)
    g = torch.Generator(device="cuda").manual_seed(0)

    def inputs():
        y = torch.randint(0, 700, (8, 40), generator=g, device="cuda")
        y[torch.rand(8, 40, generator=g, device="cuda") < 0.3] = IGN
        return [torch.randn(8, 40, 64, generator=g, device="cuda").bfloat16(),
                torch.randn(700, 64, generator=g, device="cuda").bfloat16() * 0.2, y,
                torch.randn(8, generator=g, device="cuda"),
                torch.randn(300, 64, generator=g, device="cuda").bfloat16()]

    def step(h, w, y, adv, x):
        h, w, x = (t.detach().requires_grad_(True) for t in (h, w, x))
        lp = linear_token_logprobs(h, w, y)
        mask = y != IGN
        pol = policy_loss(lp, None, adv, mask, reduction="sequence")[0]
        pref = preference_loss(lp.view(2, 4, 40), None, mask.view(2, 4, 40))[0]
        idx = (torch.arange(600, device="cuda") % 64).view(300, 2)
        bal, counts = router_balance_loss(x, idx, balance_coef=0.1, z_coef=0.1)
        return [lp.detach(), pol.detach(), counts, *torch.autograd.grad(pol + 0.5 * pref + bal, (h, w, x))]

    static = inputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for _ in range(2):
        new = inputs()
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step(*new)):
            assert torch.equal(a, b)


@GPU
def test_gradients_are_not_differentiated_again():
    """With a graph of the backward pass asked for, the first gradient is as ever and a second
    one is refused, not zero."""
    from pluggy_b200.ops import linear_token_logprobs, policy_loss, preference_loss, router_balance_loss

    def leaf(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda").to(dtype).requires_grad_(True)

    h, w = leaf(40, 64, dtype=torch.bfloat16), leaf(300, 64, dtype=torch.bfloat16)
    lp, x = leaf(2, 4, 40), leaf(50, 16)
    mask = torch.ones(2, 4, 40, dtype=torch.bool, device="cuda")
    y = torch.randint(0, 300, (40,), device="cuda")
    idx = torch.arange(100, device="cuda").view(50, 2) % 16
    for leaves, run in (((h, w), lambda: linear_token_logprobs(h, w, y).sum()),
                        ((lp,), lambda: preference_loss(lp, None, mask)[0]),
                        ((lp,), lambda: policy_loss(lp[0], None, torch.ones(4, device="cuda"), mask[0])[0]),
                        ((x,), lambda: router_balance_loss(x, idx, z_coef=0.1)[0])):
        plain = torch.autograd.grad(run(), leaves)
        again = torch.autograd.grad(run(), leaves, create_graph=True)
        for a, b in zip(plain, again):
            assert torch.equal(a, b)
            with pytest.raises(RuntimeError, match="differentiated again"):
                b.float().sum().backward()


@GPU
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", ["hidden", "weight", "pref_logps", "pref_ref", "logps", "old", "advantages", "ref",
                                   "router"])
def test_forward_mode_is_refused(which, grad):
    """A tangent on any input raises; it is never dropped, whether gradients are on or off."""
    import torch.autograd.forward_ad as fw

    from pluggy_b200.ops import linear_token_logprobs, policy_loss, preference_loss, router_balance_loss

    m = torch.ones(2, 3, 40, dtype=torch.bool, device="cuda")
    x, a = torch.randn(2, 3, 40, device="cuda"), torch.ones(3, device="cuda")
    h, w = torch.randn(5, 64, device="cuda"), torch.randn(30, 64, device="cuda")
    y = torch.zeros(5, dtype=torch.int64, device="cuda")

    def dual(t):
        return fw.make_dual(t, torch.ones_like(t))

    run = {"hidden": lambda: linear_token_logprobs(dual(h), w, y),
           "weight": lambda: linear_token_logprobs(h, dual(w), y),
           "pref_logps": lambda: preference_loss(dual(x), None, m),
           "pref_ref": lambda: preference_loss(x, dual(x), m),
           "logps": lambda: policy_loss(dual(x[0]), None, a, m[0]),
           "old": lambda: policy_loss(x[0], dual(x[0]), a, m[0]),
           "advantages": lambda: policy_loss(x[0], None, dual(a), m[0]),
           "ref": lambda: policy_loss(x[0], None, a, m[0], ref_logps=dual(x[0])),
           "router": lambda: router_balance_loss(dual(h), torch.zeros(5, 2, dtype=torch.int64, device="cuda"))}
    with fw.dual_level(), torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
        run[which]()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("name", ["PREFERENCE", "POLICY"])
def test_padding_does_not_reach_the_router_losses(name, fused, dev):
    """The auxiliary loss, the routers' gradients and the experts' counts are those of the tokens
    before the padding, of the same forward pass; on the CPU, where two passes agree, longer padding
    and other ids in it leave them as they are."""
    from pluggy_b200.models.qwen3_moe import load_balancing_loss, router_z_loss

    lengths = [64, 40, 64, 10, 0, 33]
    P, S = len(lengths) // 2, 64

    def batch(total, pad):
        g = torch.Generator().manual_seed(1)
        ids, labels = torch.full((2 * P, total), pad), torch.full((2 * P, total), IGN)
        full = torch.randint(0, 200, (2 * P, S), generator=g)
        for i, n in enumerate(lengths):
            ids[i, :n] = full[i, :n]
            labels[i, 4:n] = full[i, 4:n]
        if name == "POLICY":
            out = {"input_ids": ids, "labels": labels, "advantages": torch.linspace(-1, 1, 2 * P)}
        else:
            out = {f"{side}_{k}": t[i * P:(i + 1) * P] for i, side in enumerate(("chosen", "rejected"))
                   for k, t in (("ids", ids), ("labels", labels))}
        return {k: t.to(dev) for k, t in out.items()}

    m = small("qwen3_moe", dev, router_aux_loss_coef=0.1, router_z_loss_coef=0.01, fused_router_losses=fused)
    obj = build_objective(name, dict(reference_free=True) if name == "PREFERENCE" else {})
    got = []
    for total, pad in ((S, 0), (2 * S, 0), (2 * S, 7)):
        loss = obj.compute_loss(m, batch(total, pad))
        aux = m.aux_loss()
        assert abs(loss - obj.metrics["loss"] - aux) <= 1e-5 * loss.abs()
        keep = (torch.arange(total)[None, :] < torch.tensor(lengths)[:, None]).reshape(-1).to(dev)
        logits = [x[keep] for x in m._router_logits]
        want = 0.1 * load_balancing_loss(logits, 32, 4) + 0.01 * router_z_loss(logits)
        weights = [b.ffn.router.weight for b in m.blocks]
        grads = torch.autograd.grad(aux, weights, retain_graph=True)
        assert abs(aux - want) <= 2.0 ** -16 * want
        for x, y in zip(grads, torch.autograd.grad(want, weights)):
            # on the GPU the routers' logits, and so their gradients, are bf16
            assert (x - y).norm() <= (2.0 ** -7 if dev == "cuda" else 1e-4) * y.norm()
        got.append((aux.detach(), grads, m.last_tokens_per_expert))
        assert got[-1][2].sum() == sum(lengths) * 4 * 2
    for aux, grads, counts in got[1:] if dev == "cpu" else ():
        assert abs(aux - got[0][0]) <= 1e-5 * got[0][0] and torch.equal(counts, got[0][2])
        for x, y in zip(grads, got[0][1]):
            assert (x - y).norm() <= 2e-5 * y.norm()


def test_token_mask_argument():
    """Checked against the ids; an all-true mask is no mask; nothing left gives 0."""
    m = small("qwen3_moe", router_aux_loss_coef=0.1)
    ids = torch.randint(0, 200, (2, 16), generator=torch.Generator().manual_seed(3))
    with pytest.raises(ValueError, match="token_mask"):
        m(ids, token_mask=torch.ones(2, 15, dtype=torch.bool))
    with pytest.raises(ValueError, match="token_mask"):
        m(ids, token_mask=torch.ones(2, 16))
    m(ids)
    want, counts = m.aux_loss(), m.last_tokens_per_expert
    m(ids, token_mask=torch.ones(2, 16, dtype=torch.bool))
    for fused in (False, True):
        m.fused_router_losses = fused
        assert abs(m.aux_loss() - want) <= 1e-5 * want
        assert torch.equal(m.last_tokens_per_expert, counts)
    m(ids, token_mask=torch.zeros(2, 16, dtype=torch.bool))
    for fused in (False, True):
        m.fused_router_losses = fused
        assert m.aux_loss() == 0
    # padding of the attention and of the losses together
    am = torch.ones(2, 16, dtype=torch.long)
    am[0, 12:] = 0
    tm = torch.ones(2, 16, dtype=torch.bool)
    tm[1, 10:] = False
    m(ids, attention_mask=am, token_mask=tm)
    m.aux_loss()
    assert m.last_tokens_per_expert.sum() == (12 + 10) * 4 * 2


@GPU
def test_launch_counts(monkeypatch):
    """The counted launches are the package's kernels and memsets that the profiler sees, forward and
    backward."""
    from torch.profiler import ProfilerActivity, profile

    from pluggy_b200.ops import linear_token_logprobs, logprob, policy_loss, preference_loss, router_balance_loss
    from pluggy_b200.utils.launch_count import count_launches

    m = torch.ones(2, 3, 40, dtype=torch.bool, device="cuda")
    x = torch.randn(2, 3, 40, device="cuda").requires_grad_(True)
    h = torch.randn(300, 64, device="cuda").bfloat16().requires_grad_(True)
    w = torch.randn(700, 64, device="cuda").bfloat16().requires_grad_(True)
    y, g = torch.zeros(300, dtype=torch.int64, device="cuda"), torch.ones(300, device="cuda")
    idx = torch.zeros(300, 2, dtype=torch.int64, device="cuda")
    ones, one = torch.ones(3, device="cuda"), torch.ones((), device="cuda")

    def logprobs(*wrt, **kw):
        return lambda: torch.autograd.grad(linear_token_logprobs(h, w, y, **kw), wrt, g)

    def score(n):
        def run():
            with torch.no_grad():
                linear_token_logprobs(h[:n], w, y[:n])
        return run

    def loss(fn, leaf):
        return lambda: torch.autograd.grad(fn()[0], leaf, one)

    recompute, keep_all = 1 << 62, 0
    # kernels and memsets; the last gradient of the head takes three vocabulary ranges
    cases = [(score(5), 2, 0, recompute), (score(200), 2, 0, recompute), (score(300), 4, 0, recompute),
             (logprobs(h, w), 9, 1, recompute), (logprobs(h, w), 10, 1, keep_all), (logprobs(h), 7, 0, recompute),
             (logprobs(w, workspace_bytes=512 * 2 * 256), 5 + 2 * 3, 1, keep_all),
             (loss(lambda: preference_loss(x, None, m), x), 3, 0, recompute),
             (loss(lambda: policy_loss(x[0], None, ones, m[0]), x), 3, 0, recompute),
             (loss(lambda: router_balance_loss(h, idx), h), 3, 0, recompute)]
    for run, kernels, memsets, keep in cases:
        monkeypatch.setattr(logprob, "KEEP_PRODUCT", keep)
        run()
        torch.cuda.synchronize()
        with count_launches() as cnt, profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as prof:
            run()
            torch.cuda.synchronize()
        # torch's own kernels live in the namespaces at:: and c10::, and the gradient of x[0] has a memset
        seen = [e.name for e in prof.events() if e.device_type == torch.autograd.DeviceType.CUDA
                and not any(s in e.name for s in ("at::", "c10::", "Memcpy", "Memset"))]
        assert cnt.count == kernels + memsets and len(seen) == kernels, (cnt.count, kernels, memsets, seen)


@GPU
@pytest.mark.parametrize("name", ["PREFERENCE", "POLICY"])
def test_objectives_bound_what_they_keep(name, monkeypatch):
    """``workspace_bytes`` reaches the head: a step that keeps nothing holds less until its backward,
    and its gradients are the same up to the kept rows' rounding."""
    from pluggy_b200.ops import logprob

    monkeypatch.setattr(logprob, "KEEP_PRODUCT", 0)
    V = 4000
    m = small(dev="cuda", vocab_size=V)
    b = pairs("cuda", P=4, S=512, V=V)
    batch = b if name == "PREFERENCE" else {"input_ids": b["chosen_ids"].repeat(2, 1),
                                            "labels": b["chosen_labels"].repeat(2, 1),
                                            "advantages": torch.linspace(-1, 1, 8, device="cuda")}
    held, grads = [], []
    for ws in (None, 1 << 20):
        cfg = dict(workspace_bytes=ws, **(dict(reference_free=True) if name == "PREFERENCE" else {}))
        obj = build_objective(name, cfg)
        obj.compute_loss(m, batch)  # caches and workspaces of a first call
        gc.collect()
        before = torch.cuda.memory_allocated()
        loss = obj.compute_loss(m, batch)
        held.append(torch.cuda.memory_allocated() - before)
        grads.append(torch.autograd.grad(loss, m.lm_head.weight)[0])
        del loss
    kept = 2 * 8 * 512 * V  # bytes of the matrix
    assert held[0] - held[1] >= kept - (2 << 20)
    # c_t h_t is rounded to bf16 once more (2^-8 of a term); the passes' hidden states differ in bf16's last bits
    assert (grads[0] - grads[1]).norm() <= 2.0 ** -6 * grads[1].norm()


def test_before_padding():
    from pluggy_b200.objectives.post_training import before_padding

    y = torch.tensor([[IGN, 5, IGN, 7, IGN], [IGN] * 5, [1, 2, 3, 4, 0], [9, IGN, IGN, IGN, IGN]])
    assert before_padding(y).sum(1).tolist() == [4, 0, 5, 1]
    assert before_padding(y)[0].tolist() == [True] * 4 + [False]
    assert before_padding(y, 0)[2].tolist() == [True] * 4 + [False]
    assert before_padding(y[:, :0]).shape == (4, 0)


def test_models_without_a_token_mask():
    """A model whose forward has no token_mask, a MoE subclass with the older signature among them,
    runs as it did."""
    from pluggy_b200.models.qwen3_moe import Qwen3Moe

    class Own(Qwen3Moe):
        def forward(self, x, attention_mask=None, return_hidden_states=False, return_final_hidden=False,
                    position_ids=None):
            return super().forward(x, attention_mask, return_hidden_states, return_final_hidden, position_ids)

    torch.manual_seed(0)
    m = Own(num_layers=1, num_heads=2, num_kv_heads=1, emb_dim=128, head_dim=64, vocab_size=200, moe_ffn_dim=128,
            num_experts=8, top_k=2)
    m.init_weights()
    build_objective("PREFERENCE", dict(reference_free=True)).compute_loss(m, pairs("cpu"))
    assert m.last_tokens_per_expert.sum() == 6 * 128 * 2


def test_masked_router_rows_may_hold_anything():
    from pluggy_b200.models.qwen3_moe import load_balancing_loss, router_z_loss

    keep = torch.tensor([True, False, True, False, True])
    x = torch.randn(5, 8, generator=torch.Generator().manual_seed(0))
    want = load_balancing_loss([x[keep]] * 2, 8, 2) + router_z_loss([x[keep]] * 2)
    x[~keep] = float("nan")
    x.requires_grad_(True)
    got = load_balancing_loss([x] * 2, 8, 2, keep) + router_z_loss([x] * 2, keep)
    (g,) = torch.autograd.grad(got, x)
    assert abs(got - want) <= 1e-6 * want and (g[~keep] == 0).all() and torch.isfinite(g).all()
