"""Training objectives other than next-token cross entropy, for
``StreamedLoraTrainer.train_step(ids, labels, objective=...)``.

The reference trains on shifted cross entropy alone (src/lema/_trainer.py:
151-157). These take its place at the same point of the step: each is called
with the head's logits [batch, seq, vocab], the targets aligned with them
(``next_targets``) and a factor for the gradient, and returns (loss, gradient
of the logits). The gradient is computed in the same pass as the loss and
written over the logits (``lema_b200.ops``: ``preference_loss_grad``,
``policy_loss_grad``, ``distill_loss_grad``), so a step holds one [batch, seq,
vocab] tensor. Per-token inputs are aligned like the targets, as
``StreamedLoraTrainer.token_logprobs`` returns them.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch

from . import ops

IGNORE = -100


def next_targets(labels: torch.Tensor) -> torch.Tensor:
    """Targets of each position of [batch, seq] labels: the next label, and none
    (-100) at the last. Labels of -100 (prompts, padding) stay out of the loss."""
    return torch.nn.functional.pad(labels[:, 1:], (0, 1), value=IGNORE)


@dataclass
class Preference:
    """Pairs of answers: the first half of the batch chosen, the second half the
    rejected ones of the same prompts. ``ref_logps`` [batch, seq] are the frozen
    model's (``token_logprobs(ids, labels, adapters=False)``, before the first step where
    whole layers are fine-tuned; None: reference-free).
    ``rewards`` [batch] of the last call: beta * summed log ratios."""

    ref_logps: torch.Tensor | None = None
    beta: float = 0.1
    label_smoothing: float = 0.0
    rewards: torch.Tensor | None = field(default=None, init=False)

    def __call__(self, logits, targets, grad_scale):
        loss, self.rewards, dlogits = ops.preference_loss_grad(
            logits, targets, self.ref_logps, beta=self.beta, label_smoothing=self.label_smoothing,
            grad_scale=grad_scale, out=logits)
        return loss, dlogits


@dataclass
class Policy:
    """Clipped policy optimisation over sampled tokens: ``old_logps`` [batch, seq] of
    the policy that sampled them (None: the current one), ``advantages`` [batch] or
    [batch, seq], ``ref_logps`` for the KL term. ``logps`` and ``kl`` of the last
    call."""

    advantages: torch.Tensor
    old_logps: torch.Tensor | None = None
    ref_logps: torch.Tensor | None = None
    clip: tuple[float, float] = (0.2, 0.2)
    kl_coef: float = 0.0
    temperature: float = 1.0
    reduction: str = "token"
    logps: torch.Tensor | None = field(default=None, init=False)
    kl: torch.Tensor | None = field(default=None, init=False)

    def __call__(self, logits, targets, grad_scale):
        loss, self.logps, self.kl, dlogits = ops.policy_loss_grad(
            logits, targets, self.old_logps, self.advantages, self.ref_logps, clip=self.clip,
            kl_coef=self.kl_coef, temperature=self.temperature, reduction=self.reduction,
            grad_scale=grad_scale, out=logits)
        return loss, dlogits


@dataclass
class Distill:
    """A teacher's K best tokens of each position: ``teacher_ids`` and
    ``teacher_logits`` [batch, seq, K] (``torch.topk`` of its logits, say). Positions
    without a target are left out."""

    teacher_ids: torch.Tensor
    teacher_logits: torch.Tensor
    temperature: float = 1.0

    def __call__(self, logits, targets, grad_scale):
        return ops.distill_loss_grad(logits, self.teacher_ids, self.teacher_logits,
                                     targets != IGNORE, temperature=self.temperature,
                                     grad_scale=grad_scale, out=logits)
