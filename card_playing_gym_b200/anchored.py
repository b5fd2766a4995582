"""A policy update on this library's training operators: a residual policy head, the anchored objective, AdamW.

The head is one MLP block of the trunk's shape on its final hidden state (up, GELU, down onto the residual; the reference's
blocks are cardgym/nn/trunk.py:124-157) and the policy layer, three ``dense.linear`` products; its loss is
``ppo.anchored_objective`` against a frozen reference head (the magnet of a regularised self-play update, or the
supervised policy that fine-tuning must not leave), and ``optim.AdamW`` clips and steps. Nothing of an update is read by the
host until its totals are.

    python -m card_playing_gym_b200.anchored [--rows 4096] [--steps 20] [--dtype bfloat16]

runs it on synthetic decisions over 52 cards and prints the totals of each step.
"""

from __future__ import annotations

import argparse
import copy
from dataclasses import dataclass

import torch

from . import ppo
from .dense import linear
from .optim import AdamW


class PolicyHead(torch.nn.Module):
    """hidden [N, d] -> logits [N, actions]: act(hidden W1 + b1) W2 + b2 + hidden, then the policy layer."""

    def __init__(self, d_model: int = 240, d_ff: int = 720, actions: int = 52, *, device="cuda",
                 dtype: torch.dtype = torch.float32, generator: torch.Generator | None = None) -> None:
        super().__init__()
        def weight(rows: int, cols: int) -> torch.nn.Parameter:
            start = torch.randn((rows, cols), generator=generator, device=device) / cols ** 0.5
            return torch.nn.Parameter(start.to(dtype))

        def bias(rows: int) -> torch.nn.Parameter:
            return torch.nn.Parameter(torch.zeros(rows, device=device, dtype=dtype))

        self.up, self.up_bias = weight(d_ff, d_model), bias(d_ff)
        self.down, self.down_bias = weight(d_model, d_ff), bias(d_model)
        self.policy, self.policy_bias = weight(actions, d_model), bias(actions)

    def forward(self, hidden: torch.Tensor) -> torch.Tensor:
        block = linear(hidden, self.up, self.up_bias, activation="gelu")
        block = linear(block, self.down, self.down_bias, hidden)
        return linear(block, self.policy, self.policy_bias)


@dataclass
class Decisions:
    """Recorded decisions: the trunk's hidden state, the legal actions, the action taken, the behaviour's log-probability of
    it, its advantage and its weight."""

    hidden: torch.Tensor
    legal: torch.Tensor
    actions: torch.Tensor
    old_log_probs: torch.Tensor
    advantages: torch.Tensor
    weights: torch.Tensor


class AnchoredUpdate:
    """One update of ``head`` per call, anchored to a frozen copy of it taken here (or to ``reference``).

    ``loss_scale`` multiplies the objective for the backward pass, None: 1024 for a float16 head (whose gradients of a mean
    over many rows would fall below float16's least step) and 1 for the others. AdamW's step is the same for scaled
    gradients with ``eps`` and ``max_norm`` scaled alike, so nothing is scaled back: the optimizer's moments and
    ``grad_norm`` are those of the scaled objective.
    """

    def __init__(self, head: PolicyHead, *, reference: PolicyHead | None = None, lr: float = 1e-3,
                 weight_decay: float = 0.0, state_bits: int = 32, max_norm: float = 1.0, clip_ratio: float = 0.2,
                 beta: float = 0.05, alpha: float = 0.01, loss_scale: float | None = None) -> None:
        self.head = head
        self.reference = copy.deepcopy(head) if reference is None else reference
        self.reference.requires_grad_(False)
        if loss_scale is None:
            loss_scale = 1024.0 if head.up.dtype is torch.float16 else 1.0
        self.loss_scale = loss_scale
        self._scale = torch.full((), loss_scale, device=head.up.device)
        self.optimizer = AdamW(head.parameters(), lr=lr, eps=1e-8 * loss_scale, weight_decay=weight_decay,
                               state_bits=state_bits, max_norm=max_norm * loss_scale)
        self.clip_ratio, self.beta, self.alpha = clip_ratio, beta, alpha

    def __call__(self, batch: Decisions) -> torch.Tensor:
        """Returns the totals (fp32 [9], ``ppo.ANCHORED_KEYS``) of the policy before the step, on the device."""

        self.optimizer.zero_grad(set_to_none=True)
        with torch.no_grad():
            reference = self.reference(batch.hidden)
        objective, totals = ppo.anchored_objective(
            self.head(batch.hidden), batch.actions, batch.old_log_probs, batch.advantages, batch.weights,
            clip_ratio=self.clip_ratio, beta=self.beta, alpha=self.alpha, reference_logits=reference, legal=batch.legal)
        objective.backward(self._scale)
        self.optimizer.step()
        return totals


def synthetic_decisions(head: PolicyHead, rows: int, seed: int = 0) -> Decisions:
    """Decisions that ``head`` takes on random hidden states, with advantages that prefer low cards."""

    device, dtype = head.up.device, head.up.dtype
    g = torch.Generator(device=device).manual_seed(seed)
    hidden = torch.randn((rows, head.up.shape[1]), generator=g, device=device).to(dtype)
    width = head.policy.shape[0]
    legal = torch.rand((rows, width), generator=g, device=device) < 0.4
    legal[:, 0] = True
    with torch.no_grad():
        logits = head(hidden)
        noise = torch.rand((rows, width), generator=g, device=device).clamp_(1e-20, 1 - 1e-7)
        actions = torch.argmax(logits.float().masked_fill(~legal, -torch.inf) - torch.log(-torch.log(noise)), dim=1)
        old = ppo.action_log_probs(logits, actions, legal=legal)
    advantages = 1.0 - 2.0 * actions.float() / width
    weights = torch.full((rows,), 1.0 / rows, device=device)
    return Decisions(hidden, legal, actions, old, advantages, weights)


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--rows", type=int, default=4096)
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--dtype", choices=("float32", "float16", "bfloat16"), default="bfloat16")
    parser.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    args = parser.parse_args(argv)
    head = PolicyHead(dtype=getattr(torch, args.dtype), generator=torch.Generator(device="cuda").manual_seed(0))
    batch = synthetic_decisions(head, args.rows)
    update = AnchoredUpdate(head, state_bits=args.state_bits)
    for step in range(args.steps):
        totals = dict(zip(ppo.ANCHORED_KEYS, update(batch).tolist()))
        print(f"step {step:3d} " + " ".join(f"{key} {totals[key]:+.5f}" for key in
                                           ("objective", "policy_loss", "reference_kl", "entropy", "clip")))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
