"""Objectives of the device engine other than cross-entropy: preference pairs and sampled answers.

``PipelineTrainer(..., objective=PreferenceObjective(beta=0.1))`` replaces the LM head's loss; the
objective's per-token tensors come with each step, batched as the targets::

    ref = frozen.logprobs(x, y)                     # a trainer that holds the reference model
    stats = trainer.step(step, x, y, extras={"ref_logps": ref, "mask": answer_tokens})

The loss of a step is the mean over its microbatches, each the mean over its pairs or marked tokens.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import ClassVar

import torch


class Objective:
    """``needs`` / ``takes``: names and types of the per-token [batch, S] tensors that must / may come along."""

    needs: ClassVar[dict[str, torch.dtype]] = {}
    takes: ClassVar[dict[str, torch.dtype]] = {}

    def split(self, extras, targets: torch.Tensor, microbatches: int, device) -> list[dict[str, torch.Tensor]]:
        """The step's tensors checked, on the device and cut into microbatches."""
        extras = {k: v for k, v in (extras or {}).items() if v is not None}
        known = {**self.needs, **self.takes}
        missing, unknown = set(self.needs) - set(extras), set(extras) - set(known)
        if missing or unknown:
            raise ValueError(f"{type(self).__name__}: missing {sorted(missing)}, unknown {sorted(unknown)}")
        for name, t in extras.items():
            if t.shape != targets.shape or t.dtype != known[name]:
                raise ValueError(f"{type(self).__name__}: {name} must be {known[name]} {tuple(targets.shape)}, "
                                 f"got {t.dtype} {tuple(t.shape)}")
        cut = {k: v.to(device, non_blocking=True).chunk(microbatches) for k, v in extras.items()}
        return [{k: v[i] for k, v in cut.items()} for i in range(microbatches)]

    def apply(self, head, x, targets, extras, saved, grads, loss_sum, grad_scale) -> None:
        raise NotImplementedError


@dataclass(frozen=True)
class PreferenceObjective(Objective):
    """Pairs of answers: rows 2i and 2i + 1 of a batch are the preferred and the rejected one, ``mask`` marks
    their tokens, ``ref_logps`` are the log probabilities under the reference model (``ops.preference_loss``)."""

    beta: float = 0.1
    form: str = "sigmoid"
    label_smoothing: float = 0.0
    needs = {"ref_logps": torch.float32, "mask": torch.bool}

    def apply(self, head, x, targets, extras, saved, grads, loss_sum, grad_scale) -> None:
        head.fwd_preference_loss(x, targets, saved, grads, loss_sum, grad_scale, beta=self.beta, form=self.form,
                                 label_smoothing=self.label_smoothing, **extras)


@dataclass(frozen=True)
class PolicyObjective(Objective):
    """Sampled answers with advantages: ``old_logps`` under the policy that sampled them, ``ref_logps`` for the
    KL term, ``mask`` marks the sampled tokens (``ops.policy_loss_chunk``)."""

    clip_low: float = 0.2
    clip_high: float = 0.2
    kl_coef: float = 0.0
    needs = {"old_logps": torch.float32, "advantages": torch.float32, "mask": torch.bool}
    takes = {"ref_logps": torch.float32}

    def apply(self, head, x, targets, extras, saved, grads, loss_sum, grad_scale) -> None:
        head.fwd_policy_loss(x, targets, saved, grads, loss_sum, grad_scale, clip_low=self.clip_low,
                             clip_high=self.clip_high, kl_coef=self.kl_coef, **extras)


__all__ = ["Objective", "PreferenceObjective", "PolicyObjective"]
