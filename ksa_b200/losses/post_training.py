"""Losses of a post-training step as modules: the clipped policy loss with a KL term, and the preference loss of pairs.

Both take log probabilities of answer tokens (``ops.linear_log_probs``, or a model called with ``log_probs=True``) as rows or packed behind one
another; :mod:`ksa_b200.ops.token_losses` has the formulas."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from .. import ops


class PolicyLoss(nn.Module):
    """``(loss, stats)`` of :func:`ksa_b200.ops.policy_loss`."""

    def __init__(self, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, reduction: str = "token"):
        super().__init__()
        self.clip_low, self.clip_high, self.kl_coef, self.reduction = clip_low, clip_high, kl_coef, reduction

    def forward(self, log_probs: torch.Tensor, old_log_probs: torch.Tensor, advantages: torch.Tensor, ref_log_probs: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return ops.policy_loss(log_probs, old_log_probs, advantages, ref_log_probs, mask, cu_seqlens, clip_low=self.clip_low,
                               clip_high=self.clip_high, kl_coef=self.kl_coef, reduction=self.reduction)


class PreferenceLoss(nn.Module):
    """``(loss, rewards)`` of :func:`ksa_b200.ops.preference_loss`; sequences ``2 i`` and ``2 i + 1`` are a pair's preferred and rejected answer."""

    def __init__(self, beta: float = 0.1, label_smoothing: float = 0.0):
        super().__init__()
        self.beta, self.label_smoothing = beta, label_smoothing

    def forward(self, log_probs: torch.Tensor, ref_log_probs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        return ops.preference_loss(log_probs, ref_log_probs, mask, cu_seqlens, beta=self.beta, label_smoothing=self.label_smoothing)
