"""The policy update of anchored.py: its first step against torch autograd and the AdamW formula in float64, and runs in every
type that lower the objective, with either state width."""

from __future__ import annotations

import math

import pytest
import torch

from card_playing_gym_b200 import anchored, ppo
from card_playing_gym_b200 import _native as nat


def plain_step(head, reference, batch, *, lr, clip_ratio, beta, alpha, max_norm):
    """Objective and stepped weights in float64, from the definitions."""

    names = [name for name, _ in head.named_parameters()]
    w = {name: p.detach().double().requires_grad_() for name, p in head.named_parameters()}
    r = {name: p.detach().double() for name, p in reference.named_parameters()}
    hidden = batch.hidden.double()

    def logits(v):
        block = torch.nn.functional.gelu(hidden @ v["up"].t() + v["up_bias"]) @ v["down"].t() + v["down_bias"] + hidden
        return block @ v["policy"].t() + v["policy_bias"]

    hide = ~batch.legal
    lp = torch.log_softmax(logits(w).masked_fill(hide, -1e30), 1)
    lr_ = torch.log_softmax(logits(r).masked_fill(hide, -1e30), 1)
    p = lp.exp()
    picked = lp.gather(1, batch.actions[:, None])[:, 0]
    ratio = torch.exp(picked - batch.old_log_probs.double())
    advantage = batch.advantages.double()
    surrogate = -torch.minimum(ratio * advantage, ratio.clamp(1 - clip_ratio, 1 + clip_ratio) * advantage)
    kl = (p * (lp - lr_)).sum(1)
    entropy = -(p * lp).sum(1)
    count = batch.legal.sum(1).double()
    norm = torch.where(count > 1, 1 / torch.log(count.clamp(min=2)), 0.0)
    objective = ((surrogate + beta * kl - alpha * norm * entropy) * batch.weights.double()).sum()
    grads = torch.autograd.grad(objective, [w[n] for n in names])
    size = math.sqrt(sum(float((g * g).sum()) for g in grads))
    scale = min(1.0, max_norm / (size + 1e-6))
    stepped = {}
    for name, g in zip(names, grads):
        g = g * scale
        # t = 1: both bias corrections leave g / (|g| + eps)
        stepped[name] = w[name].detach() - lr * g / (g.abs() + 1e-8), g
    return objective.detach(), stepped


@pytest.mark.gpu
def test_the_first_step_against_the_definitions():
    """fp32: an entry whose gradient is far above eps and its rounding moves by lr; the bound is the update's change for a
    relative gradient error of 1e-3, where the gradient is over 1e-6 (its fp32 error is below 1e-9)."""

    g = torch.Generator(device="cuda").manual_seed(1)
    head = anchored.PolicyHead(generator=g)
    reference = anchored.PolicyHead(generator=g)
    batch = anchored.synthetic_decisions(head, 500)
    options = dict(lr=1e-2, clip_ratio=0.2, beta=0.1, alpha=0.02, max_norm=0.5)
    want, stepped = plain_step(head, reference, batch, **options)
    totals = anchored.AnchoredUpdate(head, reference=reference, **options)(batch)
    assert float(totals[-1]) == pytest.approx(float(want), abs=2e-6)
    for name, p in head.named_parameters():
        moved, gradient = stepped[name]
        clear = gradient.abs() > 1e-6
        assert clear.any()
        assert (p.detach().double() - moved).abs()[clear].max() <= 1e-2 * 1e-3 + 1e-6, name
    assert nat.fault_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_updates_lower_the_objective(dtype, bits):
    head = anchored.PolicyHead(dtype=getattr(torch, dtype), generator=torch.Generator(device="cuda").manual_seed(0))
    batch = anchored.synthetic_decisions(head, 1000)
    if dtype == "float16":
        batch.weights = batch.weights * 64  # half-precision gradients of a mean over rows are scaled, as any loss in it
    update = anchored.AnchoredUpdate(head, state_bits=bits, max_norm=64.0 if dtype == "float16" else 1.0)
    history = torch.stack([update(batch) for _ in range(8)])
    scale = float(history[0][ppo.ANCHORED_KEYS.index("row_weight")])
    first, last = float(history[0][-1]) / scale, float(history[-1][-1]) / scale
    assert last < first - 0.02
    kl = history[:, ppo.ANCHORED_KEYS.index("reference_kl")] / scale
    assert abs(float(kl[0])) < 1e-5 and 1e-4 < float(kl[-1]) < 1.0
    assert nat.fault_status() == 0


@pytest.mark.gpu
def test_the_command_runs(capsys):
    assert anchored.main(["--rows", "256", "--steps", "2", "--state-bits", "8"]) == 0
    assert capsys.readouterr().out.count("objective") == 2


@pytest.mark.gpu
def test_half_precision_gradients_of_a_mean_over_many_rows_keep_their_small_entries():
    """A power of two on the weights only moves float16 exponents, so the first moment of an update with weights of 2^-18 is
    2^-12 of that with weights of 2^-6, but for the entries that either loses below float16's least step: together less
    than a rounding of the whole, 2^-11 of its size. (Unscaled, three quarters of the logits' gradient are zero.)"""

    moments = []
    for weight in (2.0 ** -18, 2.0 ** -6):
        head = anchored.PolicyHead(dtype=torch.float16, generator=torch.Generator(device="cuda").manual_seed(0))
        batch = anchored.synthetic_decisions(head, 4096)
        batch.weights = torch.full_like(batch.weights, weight)
        reference = anchored.PolicyHead(dtype=torch.float16, generator=torch.Generator(device="cuda").manual_seed(3))
        update = anchored.AnchoredUpdate(head, reference=reference, max_norm=1e6)
        update(batch)
        assert int(update.optimizer.steps) == 1
        moments.append(update.optimizer.flat["exp_avg"].double() / (weight * update.loss_scale))
    assert (moments[0] - moments[1]).norm() <= 2.0 ** -11 * moments[1].norm()


@pytest.mark.gpu
def test_a_loss_scale_leaves_the_update_as_it_is():
    """In float32 a power of two on the objective changes exponents alone: eps and the clip move with it, all but the
    1e-6 beside the norm (2^-20 of the clip's factor at a norm of 1)."""

    heads = []
    for scale in (1.0, 256.0):
        head = anchored.PolicyHead(generator=torch.Generator(device="cuda").manual_seed(0))
        batch = anchored.synthetic_decisions(head, 500)
        update = anchored.AnchoredUpdate(head, lr=1e-2, max_norm=1e-3, loss_scale=scale)
        for _ in range(2):
            update(batch)
        heads.append(head)
    for p, q in zip(*(h.parameters() for h in heads)):
        assert (p - q).abs().max() <= 1e-2 * 1e-2
