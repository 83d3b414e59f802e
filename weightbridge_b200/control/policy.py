"""Comparison of the rollout's log probabilities with the trainer's: whether a sync arrived as a policy.

The planner's checks, flags and digests say that every byte was delivered; whether the rollout then
serves the trainer's policy (an fp8 rollout holds other bytes by design, a wrong mapping of names
delivers the wrong ones faithfully) shows in the tokens: the rollout returns the log probability of
every token it sampled, and the trainer recomputes them with the weights that it sent.  Where both
hold the same weights the two differ by their kernels' rounding only.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from ..ops.logprobs import token_logprobs


@dataclass
class PolicyGap:
    """Over the tokens that were compared (``tokens`` of them): the mean and largest
    ``|trainer - rollout|`` of their log probabilities, and the estimate ``mean(r - 1 - ln r)``,
    r = p_trainer / p_rollout, of KL(rollout || trainer) on tokens that the rollout sampled."""
    tokens: int
    mean_abs: float
    max_abs: float
    kl: float
    version: int | None = None

    def within(self, tolerance: float) -> bool:
        """Whether the mean difference is at most ``tolerance`` (False where it is NaN)."""
        return self.mean_abs <= tolerance


def policy_gap(logits: torch.Tensor, tokens: torch.Tensor, rollout_logprobs: torch.Tensor, *, vocab: int | None = None,
               temperature: float = 1.0, ignore_index: int = -100) -> PolicyGap:
    """The gap between ``rollout_logprobs`` and the log probabilities of ``tokens`` under ``logits``
    (the trainer's, one row a token; arguments as in ``token_logprobs``).  Waits for the GPU.
    Tokens that both sides give probability 0 differ by nothing; one side alone, without bound."""
    if rollout_logprobs.shape != tokens.shape:
        raise ValueError(f"policy_gap: {tuple(rollout_logprobs.shape)} rollout log probabilities for tokens of shape {tuple(tokens.shape)}")
    with torch.no_grad():
        mine = token_logprobs(logits.detach(), tokens, vocab=vocab, temperature=temperature, ignore_index=ignore_index).logprobs.double()
        keep = tokens != ignore_index
        theirs = rollout_logprobs.detach().to(mine.device, torch.float64)
        log_r = torch.where((mine == theirs) | ~keep, 0.0, mine - theirs)
        n = keep.sum()
        gap = torch.stack([n.double(), log_r.abs().sum(), log_r.abs().amax() if log_r.numel() else n.double(),
                           (log_r.exp() - 1 - log_r).sum()]).tolist()
    if gap[0] == 0:
        return PolicyGap(0, 0.0, 0.0, 0.0)
    return PolicyGap(int(gap[0]), gap[1] / gap[0], gap[2], math.inf if math.isinf(gap[1]) else gap[3] / gap[0])
