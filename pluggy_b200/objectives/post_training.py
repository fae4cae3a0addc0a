"""Post-training objectives: preference pairs and clipped policy updates.

Both read per-token log-probabilities of the model's own head
(:func:`pluggy_b200.ops.linear_token_logprobs`, no logits in memory) and add the model's
``aux_loss()`` (MoE router losses) when it has one, as the AR objective does. Sequences are
right-padded: under causal attention nothing before the padding sees it, so the packed
forward serves them, and padded positions carry ``ignore_index`` labels. What follows a
sequence's last label is taken for padding and counts neither in the router losses nor in
the experts' token counts (models whose ``forward`` takes a ``token_mask``).

The data sources of the trainer make no such batches, so its config check refuses these
objectives: a program calls them from its own loop (``examples/post_training.py``).

``score(model, ...)`` gives the same log-probabilities without gradients: the reference
model's, or the policy's before its update.
"""

from __future__ import annotations

import inspect

import torch
import torch.nn as nn

from pluggy_b200.objectives.autoregressive import shift_labels
from pluggy_b200.ops.logprob import linear_token_logprobs
from pluggy_b200.ops.policy import policy_loss
from pluggy_b200.ops.preference import preference_loss


def before_padding(labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """bool [B, S]: positions up to each row's last label."""
    kept = labels != ignore_index
    if labels.shape[1] == 0:
        return kept
    at = torch.arange(1, labels.shape[1] + 1, device=labels.device)
    return at <= torch.where(kept, at, 0).amax(1, keepdim=True)


def token_logprobs(model: nn.Module, ids: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                   temperature: float = 1.0, workspace_bytes: int | None = None):
    """``(logps [B, S] fp32, mask [B, S])``: position t holds the log-probability of ``labels[t + 1]``
    given ``ids[:t + 1]``; the mask is False where that label is ``ignore_index`` and at the end.
    ``workspace_bytes`` is :func:`linear_token_logprobs`'s."""
    core = getattr(model, "module", model)
    for axis in ("tp", "cp"):
        par = getattr(core, axis, None)
        if par is not None and par.mesh.size(par.dim) > 1:
            raise NotImplementedError(f"post-training objectives do not split the model over {axis}")
    if ids.shape != labels.shape or ids.dim() != 2:
        raise ValueError(f"ids and labels must be [B, S] alike, got {tuple(ids.shape)} and "
                         f"{tuple(labels.shape)}")
    masks = "token_mask" in inspect.signature(core.forward).parameters
    kw = {"token_mask": before_padding(labels, ignore_index)} if masks else {}
    hidden = model(ids, return_final_hidden=True, **kw)
    labels = shift_labels(labels, ignore_index)
    lowp_fn = getattr(core, "lm_head_lowp", None)
    lowp = lowp_fn() if callable(lowp_fn) and hidden.is_cuda else None
    logps = linear_token_logprobs(hidden, core.lm_head.weight, labels, ignore_index, weight_lowp=lowp,
                                  softcap=getattr(core, "final_logit_softcapping", None),
                                  temperature=temperature, workspace_bytes=workspace_bytes)
    return logps, labels != ignore_index


def _need(batch: dict, keys, what: str) -> None:
    missing = [k for k in keys if k not in batch]
    if missing:
        raise ValueError(f"{what} needs the batch keys {list(keys)}, missing {missing}")


def _with_aux(model: nn.Module, loss: torch.Tensor) -> torch.Tensor:
    aux_fn = getattr(getattr(model, "module", model), "aux_loss", None)
    aux = aux_fn() if callable(aux_fn) else None
    return loss if aux is None else loss + aux


class PreferenceObjective:
    """Preference pairs (sigmoid, hinge or squared loss on the paired log-ratios).

    Batch: ``chosen_ids``, ``chosen_labels``, ``rejected_ids``, ``rejected_labels`` [P, S], and
    ``ref_logps`` [2, P, S] from :meth:`score` of the reference model unless ``reference_free``.
    ``metrics`` holds the last call's mean rewards and the share of pairs ranked right.
    ``workspace_bytes`` bounds what a step keeps of its head for the backward (8 GiB when None)."""

    KEYS = ("chosen_ids", "chosen_labels", "rejected_ids", "rejected_labels")
    batch_keys = KEYS  # what every batch must hold

    def __init__(self, ignore_index: int = -100, beta: float = 0.1, kind: str = "sigmoid",
                 label_smoothing: float = 0.0, length_normalized: bool = False,
                 reference_free: bool = False, workspace_bytes: int | None = None):
        self.workspace_bytes = workspace_bytes
        self.ignore_index, self.beta, self.kind = ignore_index, beta, kind
        self.label_smoothing, self.length_normalized = label_smoothing, length_normalized
        self.reference_free = reference_free
        self.metrics: dict[str, torch.Tensor] = {}

    def _logps(self, model: nn.Module, batch: dict):
        _need(batch, self.KEYS, "PREFERENCE")
        ids = torch.cat((batch["chosen_ids"], batch["rejected_ids"]))
        labels = torch.cat((batch["chosen_labels"], batch["rejected_labels"]))
        lp, mask = token_logprobs(model, ids, labels, self.ignore_index, workspace_bytes=self.workspace_bytes)
        shape = (2, *batch["chosen_ids"].shape)
        return lp.view(shape), mask.view(shape)

    @torch.no_grad()
    def score(self, model: nn.Module, batch: dict) -> torch.Tensor:
        """``ref_logps`` [2, P, S] of ``batch`` under ``model``."""
        return self._logps(model, batch)[0]

    def compute_loss(self, model: nn.Module, batch: dict[str, torch.Tensor]) -> torch.Tensor:
        if not self.reference_free:
            _need(batch, ("ref_logps",), "PREFERENCE without reference_free")
        lp, mask = self._logps(model, batch)
        ref = None if self.reference_free else batch["ref_logps"]
        loss, chosen, rejected = preference_loss(
            lp, ref, mask, beta=self.beta, kind=self.kind, label_smoothing=self.label_smoothing,
            length_normalized=self.length_normalized)
        self.metrics = {"loss": loss.detach(), "chosen_reward": chosen.mean(),
                        "rejected_reward": rejected.mean(),
                        "ranked_right": (chosen > rejected).float().mean()}
        return _with_aux(model, loss)


class PolicyObjective:
    """Clipped policy update with a KL term against a reference model.

    Batch: ``input_ids``, ``labels`` [R, S] (``ignore_index`` on the prompt and the padding),
    ``advantages`` [R] or [R, S]; ``old_logps`` [R, S] from :meth:`score` of the policy that sampled
    (left out for the first update after sampling); ``ref_logps`` [R, S] where ``kl_coef`` is set.
    [R, S] entries belong to the position that predicts the token, as :meth:`score` gives them.
    ``metrics`` holds the last call's loss, KL estimate and clipped share.
    ``workspace_bytes`` bounds what a step keeps of its head for the backward (8 GiB when None)."""

    batch_keys = ("input_ids", "labels", "advantages")  # what every batch must hold

    def __init__(self, ignore_index: int = -100, clip_low: float = 0.2, clip_high: float = 0.2,
                 kl_coef: float = 0.0, reduction: str = "token", temperature: float = 1.0,
                 workspace_bytes: int | None = None):
        self.workspace_bytes = workspace_bytes
        self.ignore_index, self.clip_low, self.clip_high = ignore_index, clip_low, clip_high
        self.kl_coef, self.reduction, self.temperature = kl_coef, reduction, temperature
        self.metrics: dict[str, torch.Tensor] = {}

    @torch.no_grad()
    def score(self, model: nn.Module, batch: dict) -> torch.Tensor:
        """``old_logps`` or ``ref_logps`` [R, S] of ``batch`` under ``model``."""
        _need(batch, ("input_ids", "labels"), "POLICY")
        return token_logprobs(model, batch["input_ids"], batch["labels"], self.ignore_index,
                              self.temperature, self.workspace_bytes)[0]

    def compute_loss(self, model: nn.Module, batch: dict[str, torch.Tensor]) -> torch.Tensor:
        _need(batch, self.batch_keys + (("ref_logps",) if self.kl_coef else ()), "POLICY")
        lp, mask = token_logprobs(model, batch["input_ids"], batch["labels"], self.ignore_index,
                                  self.temperature, self.workspace_bytes)
        loss, kl, clipped = policy_loss(
            lp, batch.get("old_logps"), batch["advantages"], mask, ref_logps=batch.get("ref_logps"),
            clip_low=self.clip_low, clip_high=self.clip_high, kl_coef=self.kl_coef,
            reduction=self.reduction)
        self.metrics = {"loss": loss.detach(), "kl": kl, "clipped": clipped}
        return _with_aux(model, loss)
