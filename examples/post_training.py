"""Preference tuning and a clipped policy update of a small MoE decoder on synthetic data.

    python examples/post_training.py [--device cuda] [--steps 4]

1. A frozen copy of the model scores every pair (no gradients, no logits).
2. Preference steps move the model towards the chosen sequences.
3. "Rollouts" are scored under the tuned model, given one advantage for each sequence (here:
   how many tokens of a favoured range they hold), and a few clipped updates with a KL term
   against the frozen copy follow.

The router's balance and z loss joins every step's loss through the model's ``aux_loss()``.
Every step prints the objective's metrics; the exit code is 0 if they moved the right way.
"""

import argparse
import copy
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pluggy_b200.models.builder import build_model  # noqa: E402
from pluggy_b200.objectives.builder import build_objective  # noqa: E402
from pluggy_b200.optimizer.builder import build_optimizer  # noqa: E402

IGNORE = -100


def sequences(n, S, vocab, low, high, gen):
    """[n, S] ids with tokens of [low, high) after a prompt of 8, right-padded to S; labels ignore
    the prompt and the padding."""
    ids = torch.randint(low, high, (n, S), generator=gen)
    ids[:, :8] = torch.randint(0, vocab, (1, 8), generator=gen)
    labels = ids.clone()
    labels[:, :8] = IGNORE
    lengths = torch.randint(S // 2, S + 1, (n,), generator=gen)
    pad = torch.arange(S)[None, :] >= lengths[:, None]
    ids[pad], labels[pad] = 0, IGNORE
    return ids, labels


def show(step, kind, objective):
    print(f"{kind} step {step}: " + ", ".join(f"{k} {float(v):.4f}" for k, v in objective.metrics.items()),
          flush=True)


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--steps", type=int, default=4)
    p.add_argument("--seq", type=int, default=128)
    p.add_argument("--vocab", type=int, default=512)
    a = p.parse_args(argv)
    dev = torch.device(a.device)
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(0)
    # head_dim 64 and widths of whole 128s: on a GPU the model runs on the fused kernels
    model = build_model("qwen3_moe", dict(num_layers=2, num_heads=4, num_kv_heads=2, emb_dim=256, head_dim=64,
                                          vocab_size=a.vocab, moe_ffn_dim=128, num_experts=32, top_k=4,
                                          router_init_std=0.02, fused_router_losses=True))
    model.init_weights()
    model.to(dev)
    frozen = copy.deepcopy(model).requires_grad_(False)
    opt = build_optimizer(model, "adamw", dict(lr=1e-3, weight_decay=0.0))

    # ---- preference pairs: tokens of the lower half of the vocabulary over those of the upper
    chosen, chosen_labels = sequences(8, a.seq, a.vocab, 0, a.vocab // 2, gen)
    rejected, rejected_labels = sequences(8, a.seq, a.vocab, a.vocab // 2, a.vocab, gen)
    batch = {k: v.to(dev) for k, v in dict(chosen_ids=chosen, chosen_labels=chosen_labels, rejected_ids=rejected,
                                           rejected_labels=rejected_labels).items()}
    pref = build_objective("PREFERENCE", dict(beta=0.1))
    batch["ref_logps"] = pref.score(frozen, batch)
    losses = []
    for i in range(a.steps):
        loss = pref.compute_loss(model, batch)
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(float(pref.metrics["loss"]))
        show(i, "preference", pref)
    ok = losses[-1] < losses[0] and float(pref.metrics["ranked_right"]) > 0.5

    # ---- policy: sequences of any tokens, rewarded for those of the first quarter
    ids, labels = sequences(16, a.seq, a.vocab, 0, a.vocab, gen)
    reward = ((ids < a.vocab // 4) & (labels != IGNORE)).sum(1) / (labels != IGNORE).sum(1)
    adv = (reward - reward.mean()) / reward.std()
    roll = {"input_ids": ids.to(dev), "labels": labels.to(dev), "advantages": adv.to(dev)}
    policy = build_objective("POLICY", dict(clip_low=0.2, clip_high=0.28, kl_coef=0.02, reduction="sequence"))
    roll["old_logps"] = policy.score(model, roll)
    roll["ref_logps"] = policy.score(frozen, roll)
    losses = []
    for i in range(a.steps):
        loss = policy.compute_loss(model, roll)
        loss.backward()
        opt.step()
        opt.zero_grad(set_to_none=True)
        losses.append(float(policy.metrics["loss"]))
        show(i, "policy", policy)
    ok = ok and losses[-1] < losses[0]
    counts = model.last_tokens_per_expert
    print(f"tokens per expert: min {int(counts.min())}, max {int(counts.max())}")
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
