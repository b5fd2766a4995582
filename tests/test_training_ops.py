"""The training operators' custom ops: shapes a trace sees without a GPU, and on the GPU each op against its wrapper."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from card_playing_gym_b200 import ops  # noqa: F401  (registers the ops)

OPS = torch.ops.cardgym_b200


def test_fake_kernels_give_the_output_shapes():
    with FakeTensorMode():
        logits, rows = torch.empty((5, 300), dtype=torch.bfloat16), torch.empty(5)
        actions = torch.empty(5, dtype=torch.int64)
        grad, totals = OPS.anchored_objective(logits, logits, None, None, actions, rows, rows, rows, 0.2, 0.1, 0.0)
        assert grad.shape == (5, 300) and grad.dtype == torch.bfloat16 and totals.shape == (9,)
        assert OPS.action_log_probs(logits, actions, None).dtype == torch.float32
        y = OPS.linear(torch.empty((2, 7, 24)), torch.empty((40, 24)), torch.empty(40), None, "gelu")
        assert y.shape == (2, 7, 40)


@pytest.mark.gpu
def test_ops_match_the_wrappers():
    from card_playing_gym_b200 import dense, ppo

    g = torch.Generator(device="cuda").manual_seed(2)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    logits, reference = normal(40, 300), normal(40, 300)
    legal = torch.rand((40, 300), generator=g, device="cuda") < 0.7
    actions = torch.randint(0, 300, (40,), generator=g, device="cuda")
    legal[torch.arange(40, device="cuda"), actions] = True
    old = ppo.action_log_probs(logits, actions, legal=legal) + 0.1
    assert torch.equal(OPS.action_log_probs(logits, actions, legal) + 0.1, old)
    rest = (old, normal(40), torch.rand(40, generator=g, device="cuda"))
    grad, totals = OPS.anchored_objective(logits, reference, None, legal, actions, *rest, 0.2, 0.1, 0.01)
    leaf = logits.clone().requires_grad_()
    objective, want = ppo.anchored_objective(leaf, actions, *rest, clip_ratio=0.2, beta=0.1, alpha=0.01,
                                             reference_logits=reference, legal=legal)
    objective.backward()
    assert torch.equal(grad, leaf.grad) and torch.equal(totals, want)
    torch.library.opcheck(OPS.anchored_objective, (logits, reference, None, legal, actions, *rest, 0.2, 0.1, 0.01))
    x, weight, bias, residual = normal(50, 24), normal(40, 24), normal(40), normal(50, 40)
    assert torch.equal(OPS.linear(x, weight, bias, residual, "silu"),
                       dense.linear(x, weight, bias, residual, activation="silu"))
    torch.library.opcheck(OPS.linear, (x, weight, bias, residual, "silu"))
