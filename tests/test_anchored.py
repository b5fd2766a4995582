"""ppo.anchored_objective and ppo.action_log_probs against their formulas in 64 bits: widths from one entry to past what
a cluster's shared memory holds, types, both references, masks (rows with nothing legal, what a mask hides being NaN,
infinite or the type's lowest value), strides, ignored rows, and their refusals.

Tolerances. With n entries summed by partial sums of at most m = max(32, n / 256) sequential fp32 additions, a row's
probabilities are within (m + 64) * 2^-24 of theirs relatively (the exponent's argument rounds at 2^-24 of at most 40,
the fast exponential at 2^-22). An entry of the gradient is a probability times a sum of terms, each rounded a few times
at 2^-24 of the largest: the same factor times the row's scale, w (|c| + beta (|z| + |r| + KL) + alpha'), bounds it. A 16-bit
gradient rounds once more: 2^-8 or 2^-11 of the entry, and fp16's least step."""

from __future__ import annotations

import math

import pytest
import torch

from card_playing_gym_b200 import _native as nat
from card_playing_gym_b200 import ppo

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CLIP, BETA, ALPHA = 0.2, 0.3, 0.02


def factor(width: int) -> float:
    return (max(32, width / 256) + 64) * 2.0 ** -24


def inputs(rows, width, dtype, *, reference="logits", legal=False, pad=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    logits = (2 * normal(rows, width + pad)).to(dtype)[:, :width]
    data = dict(logits=logits, legal=None, advantages=normal(rows),
                weights=torch.rand(rows, generator=g, device="cuda") + 0.1)
    if legal:
        data["legal"] = torch.rand((rows, width), generator=g, device="cuda") < 0.6
        data["legal"][:, width // 2] = True
    data["actions"] = torch.randint(0, width, (rows,), generator=g, device="cuda")
    if legal:
        data["actions"] = torch.where(data["legal"].gather(1, data["actions"][:, None])[:, 0], data["actions"], width // 2)
    lp = log_softmax(logits, data["legal"]).gather(1, data["actions"][:, None])[:, 0]
    shift = 0.3 * torch.randn(rows, generator=g, device="cuda", dtype=torch.float64)
    for bound in (math.log(1 - CLIP), math.log(1 + CLIP)):  # away from the kinks, where two roundings may part
        shift = torch.where((shift - bound).abs() < 1e-3, bound + 3e-3, shift)
    data["old"] = (lp - shift).float()
    if reference == "logits":
        data["reference_logits"] = (logits.float() + 0.4 * normal(rows, width)).to(dtype)
    elif reference == "log-probs":
        data["reference_log_probs"] = (lp + 0.3 * normal(rows)).float()
    return data


def log_softmax(z, legal):
    z = z.double()
    if legal is None:
        return z - torch.logsumexp(z, 1, keepdim=True)
    z = torch.where(legal.bool(), z, -math.inf)
    return torch.where(legal.bool(), z - torch.logsumexp(z, 1, keepdim=True), 0.0)


def formula(data, beta=BETA, alpha=ALPHA, clip=CLIP, counted=None):
    """(objective, totals, gradient, scale of each row) in 64 bits, the gradient by autograd."""

    rows, width = data["logits"].shape
    counted = torch.ones(rows, dtype=torch.bool, device="cuda") if counted is None else counted
    keep = counted.nonzero()[:, 0]
    legal = data["legal"]
    legal = torch.ones((rows, width), dtype=torch.bool, device="cuda") if legal is None else legal.bool()
    legal = legal[keep]
    z = torch.where(legal, data["logits"][keep].double(), -1e30).requires_grad_()
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(lp)
    action = data["actions"][keep][:, None]
    picked = lp.gather(1, action)[:, 0]
    log_ratio = picked - data["old"][keep].double()
    ratio = torch.exp(log_ratio)
    advantage, weight = data["advantages"][keep].double(), data["weights"][keep].double()
    surrogate = -torch.minimum(ratio * advantage, ratio.clamp(1 - clip, 1 + clip) * advantage)
    entropy = -(p * lp).sum(1)
    count = legal.sum(1).double()
    norm = torch.where(count > 1, 1 / torch.log(count.clamp(min=2)), 0.0)
    kl = torch.zeros_like(ratio)
    reach = z.detach().abs().masked_fill(~legal, 0).amax(1)
    if "reference_logits" in data:
        r = torch.where(legal, data["reference_logits"][keep].double(), -1e30)
        reach = reach + r.abs().masked_fill(~legal, 0).amax(1)
        kl = (p * (lp - (r - torch.logsumexp(r, 1, keepdim=True)))).sum(1)
    elif "reference_log_probs" in data:
        u = data["reference_log_probs"][keep].double() - picked
        kl = torch.expm1(u) - u
    rows_l = surrogate + beta * kl - alpha * norm * entropy
    terms = torch.stack([surrogate, torch.ones_like(ratio), entropy, norm * entropy, (count > 1).double(),
                         ((ratio - 1).abs() > clip).double(), ratio - 1 - log_ratio, kl, rows_l])
    totals = (terms * weight).sum(1)
    totals[-1].backward()
    gradient = torch.zeros((rows, width), dtype=torch.float64, device="cuda")
    gradient[keep] = torch.where(legal, z.grad, 0.0)
    scale = torch.zeros(rows, dtype=torch.float64, device="cuda")
    scale[keep] = weight * (ratio.detach() * advantage.abs() + beta * (reach + kl.detach() + 4) + alpha * norm * 40)
    magnitude = (terms.abs() * weight).sum(1) + (weight * (reach + 4)).sum()
    return totals[-1].detach(), totals.detach(), gradient, scale, magnitude.detach()


def run(data, beta=BETA, alpha=ALPHA, clip=CLIP):
    logits = data["logits"].detach().requires_grad_()
    extra = {k: data[k] for k in ("reference_logits", "reference_log_probs") if k in data}
    objective, totals = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"],
                                               data["weights"], clip_ratio=clip, beta=beta, alpha=alpha,
                                               legal=data["legal"], **extra)
    objective.backward()
    return objective.detach(), totals, logits.grad


def check(data, counted=None, beta=BETA, alpha=ALPHA):
    objective, totals, gradient = run(data, beta, alpha)
    want, want_totals, want_gradient, scale, magnitude = formula(data, beta, alpha, counted=counted)
    width, dtype = data["logits"].shape[1], data["logits"].dtype
    k = factor(width)
    assert gradient.dtype == dtype and gradient.shape == data["logits"].shape
    assert ((totals.double() - want_totals).abs() <= k * magnitude).all()
    assert abs(float(objective) - float(want)) <= k * float(magnitude[-1])
    bound = k * scale[:, None] + (1 + k) * HALF_STEP[dtype] * want_gradient.abs()
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25
    assert ((gradient.double() - want_gradient).abs() <= bound).all()
    assert nat.fault_status() == 0


WIDTHS = [1, 2, 3, 8, 31, 52, 64, 65, 250, 256, 257, 511, 1000, 1024, 1025, 2056, 4099, 16384, 50021, 131072]


@pytest.mark.gpu
@pytest.mark.parametrize("legal", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", WIDTHS)
def test_exact_divergence(width, dtype, legal):
    check(inputs(5 if width > 10000 else 37, width, TYPES[dtype], legal=legal))


@pytest.mark.gpu
@pytest.mark.parametrize("reference", ["log-probs", "none"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [1, 52, 100, 700, 5003, 60000])
def test_sampled_divergence_and_none(width, dtype, reference):
    check(inputs(9, width, TYPES[dtype], reference=reference, legal=width == 100),
          beta=BETA if reference == "log-probs" else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [230000, 400001])
def test_rows_wider_than_a_cluster_holds(width, dtype):
    check(inputs(3, width, TYPES[dtype], legal=True))


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 3, 8, 100])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [13, 52, 300, 1500, 9001])
def test_padded_rows(width, dtype, pad):
    check(inputs(11, width, TYPES[dtype], legal=True, pad=pad))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [52, 1025, 20000])
def test_other_layouts(width):
    """Transposed logits, a reference and a mask of other strides and offsets than the logits'."""

    data = inputs(6, width, torch.bfloat16, legal=True)
    data["logits"] = data["logits"].t().contiguous().t()
    check(data)
    data = inputs(6, width, torch.bfloat16, legal=True)
    wide = torch.zeros((6, width + 7), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:width + 3] = data["reference_logits"]
    data["reference_logits"] = wide[:, 3:width + 3]
    mask = torch.zeros((6, width + 5), dtype=torch.uint8, device="cuda")
    mask[:, 1:width + 1] = data["legal"]
    data["legal"] = mask[:, 1:width + 1]
    check(data)
    data["reference_logits"] = data["reference_logits"][:1].expand(6, width)  # one reference for every row
    check(data)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 33, 5000, 70001])
def test_row_counts(rows):
    check(inputs(rows, 52, torch.float32, legal=True))
    check(inputs(min(rows, 5000), 1300, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [52, 600, 3001, 40000])
def test_rows_that_count_for_nothing(width, dtype):
    data = inputs(12, width, TYPES[dtype], legal=True)
    counted = torch.ones(12, dtype=torch.bool, device="cuda")
    data["actions"][1] = -1
    data["actions"][2] = -100
    data["legal"][3] = False
    data["weights"][4] = 0.0
    data["logits"][4] = math.nan
    data["logits"][5] = -math.inf
    data["logits"][6, ::2] = math.nan
    data["actions"][6] = -1
    counted[[1, 2, 3, 4, 5, 6]] = False
    objective, totals, gradient = run(data)
    assert torch.isfinite(totals).all() and not gradient[~counted].any()
    data["logits"][~counted] = 0  # the formula drops them
    data["legal"][3] = True
    check_against = formula(data, counted=counted)
    assert ((totals.double() - check_against[1]).abs() <= factor(width) * check_against[4]).all()
    assert nat.fault_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [math.nan, math.inf, -math.inf, "lowest", "highest"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [52, 500, 2000, 30001])
def test_what_a_mask_hides_may_hold_anything(width, dtype, hidden):
    data = inputs(8, width, TYPES[dtype], legal=True)
    want = run(data)
    info = torch.finfo(TYPES[dtype])
    fill = {"lowest": info.min, "highest": info.max}.get(hidden, hidden)
    data["logits"] = data["logits"].masked_fill(~data["legal"], fill)
    data["reference_logits"] = data["reference_logits"].masked_fill(~data["legal"], fill)
    for a, b in zip(run(data), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [52, 500, 2000, 30000])
def test_masking_by_the_lowest_logit_or_minus_infinity(width, dtype):
    """Without a mask tensor, entries at minus infinity or the type's lowest value have probability zero."""

    data = inputs(8, width, TYPES[dtype], legal=True)
    hide = ~data["legal"]
    data["legal"] = None
    for fill in (-math.inf, torch.finfo(TYPES[dtype]).min):
        filled = dict(data, logits=data["logits"].masked_fill(hide, fill),
                      reference_logits=data["reference_logits"].masked_fill(hide, fill))
        objective, totals, gradient = run(filled, alpha=0.0)
        want = formula(dict(data, legal=~hide), alpha=0.0)
        assert abs(float(objective) - float(want[0])) <= factor(width) * float(want[4][-1])
        assert not gradient[hide].any()
        bound = factor(width) * want[3][:, None] + 1.01 * HALF_STEP[TYPES[dtype]] * want[2].abs() + 2.0 ** -25
        assert ((gradient.double() - want[2]).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("width", [52, 300, 3000])
def test_a_legal_nan_reaches_the_objective(width):
    data = inputs(6, width, torch.float32)
    data["logits"][2, width // 3] = math.nan
    objective, totals, gradient = run(data)
    assert math.isnan(float(objective)) and torch.isnan(gradient[2]).any()
    assert torch.isfinite(gradient[[0, 1, 3, 4, 5]]).all()
    data = inputs(6, width, torch.float32)
    data["logits"][2] = math.nan
    assert math.isnan(float(run(data)[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("width", [52, 3000])
def test_bad_actions_set_the_fault_word(width):
    data = inputs(4, width, torch.float32, legal=True)
    data["actions"][1] = width
    _, _, gradient = run(data)
    assert nat.fault_status() == 0x420 and not gradient[1].any()
    data = inputs(4, width, torch.float32, legal=True)
    data["legal"][2, data["actions"][2]] = False
    data["legal"][2, (data["actions"][2] + 1) % width] = True
    _, _, gradient = run(data)
    assert nat.fault_status() == 0x421 and not gradient[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("reference", ["logits", "log-probs"])
@pytest.mark.parametrize("width", [20, 1200])
def test_the_gradient_against_differences(width, reference):
    """Central differences of the fp32 objective: (2^-22 |L|) / h of rounding, h^2 of curvature, at h = 2^-6."""

    data = inputs(1, width, torch.float32, reference=reference)
    data["weights"][:] = 1.0
    objective, _, gradient = run(data)
    h = 2.0 ** -6
    largest = gradient[0].abs().argmax()
    for j in {int(data["actions"][0]), int(largest), width // 2}:
        ends = []
        for sign in (1, -1):
            moved = dict(data, logits=data["logits"].clone())
            moved["logits"][0, j] += sign * h
            ends.append(float(run(moved)[0]))
        difference = (ends[0] - ends[1]) / (2 * h)
        assert difference == pytest.approx(float(gradient[0, j]), abs=8 * 2.0 ** -22 / h + 4 * h * h)


@pytest.mark.gpu
def test_backward_scales_and_repeats():
    data = inputs(16, 300, torch.float32)
    _, _, once = run(data)
    logits = data["logits"].detach().requires_grad_()
    objective, _ = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                          clip_ratio=CLIP, beta=BETA, alpha=ALPHA,
                                          reference_logits=data["reference_logits"])
    (first,) = torch.autograd.grad(3.0 * objective, logits, retain_graph=True)
    (second,) = torch.autograd.grad(objective, logits)
    assert torch.equal(second, once) and torch.equal(first, 3.0 * once)
    with torch.no_grad():
        value, _ = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                          clip_ratio=CLIP, beta=BETA, alpha=ALPHA,
                                          reference_logits=data["reference_logits"])
    assert torch.equal(value, objective.detach())


@pytest.mark.gpu
def test_agrees_with_the_policy_objective_where_both_apply():
    """Without a KL term it is the per-head objective on the behaviour's distribution."""

    data = inputs(200, 52, torch.float32, legal=True, reference="none")
    old = torch.softmax(data["logits"].float().masked_fill(~data["legal"], -math.inf), 1)
    old_lp = torch.log(old.gather(1, data["actions"][:, None])[:, 0])
    logits = (data["logits"] + 0.1 * torch.sin(torch.arange(52, device="cuda"))).requires_grad_()
    a, _ = ppo.policy_objective(logits, old, data["actions"], data["advantages"], data["weights"], clip_ratio=CLIP, alpha=ALPHA)
    (ga,) = torch.autograd.grad(a, logits)
    b, _ = ppo.anchored_objective(logits, data["actions"], old_lp, data["advantages"], data["weights"], clip_ratio=CLIP,
                                  beta=0.0, alpha=ALPHA, legal=data["legal"])
    (gb,) = torch.autograd.grad(b, logits)
    scale = float((data["weights"] * (data["advantages"].abs() + 1)).sum())
    assert abs(float(a.detach()) - float(b.detach())) <= 256 * 2.0 ** -24 * scale
    assert (ga - gb).abs().max() <= 256 * 2.0 ** -24 * float((data["weights"] * (1 + data["advantages"].abs())).max())


@pytest.mark.gpu
@pytest.mark.parametrize("legal", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", WIDTHS + [400001])
def test_action_log_probs(width, dtype, legal):
    data = inputs(7, width, TYPES[dtype], legal=legal, pad=3 if width % 2 else 0)
    got = ppo.action_log_probs(data["logits"], data["actions"], legal=data["legal"])
    want = log_softmax(data["logits"], data["legal"]).gather(1, data["actions"][:, None])[:, 0]
    reach = data["logits"].double().abs().amax(1) + 20
    assert ((got.double() - want).abs() <= factor(width) * reach).all()
    data["actions"][0] = -1
    if legal and width > 1:
        data["legal"][1] = False
        data["legal"][2, data["actions"][2]] = False
        data["legal"][2, (data["actions"][2] + 1) % width] = True
    again = ppo.action_log_probs(data["logits"], data["actions"], legal=data["legal"])
    assert float(again[0]) == 0.0 and torch.equal(again[3:], got[3:])
    if legal and width > 1:
        assert float(again[1]) == 0.0 and float(again[2]) == -math.inf
    assert nat.fault_status() == 0


@pytest.mark.gpu
def test_empty_batches_and_streams():
    empty = inputs(4, 52, torch.float32)
    empty = {k: None if v is None else v[:0] for k, v in empty.items()}
    objective, totals, gradient = run(empty)
    assert float(objective) == 0 and not totals.any() and gradient.shape == (0, 52)
    assert ppo.action_log_probs(empty["logits"], empty["actions"]).shape == (0,)
    data = inputs(64, 3000, torch.bfloat16)
    want = run(data)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(data)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_refusals():
    data = inputs(4, 52, torch.float32, legal=True)
    base = dict(clip_ratio=CLIP, beta=BETA, reference_logits=data["reference_logits"], legal=data["legal"])
    rows = (data["actions"], data["old"], data["advantages"], data["weights"])
    with pytest.raises(ValueError, match="one of the two"):
        ppo.anchored_objective(data["logits"], *rows, clip_ratio=CLIP, beta=BETA)
    with pytest.raises(ValueError, match="not both"):
        ppo.anchored_objective(data["logits"], *rows, **{**base, "beta": 0.0}, reference_log_probs=data["old"])
    with pytest.raises(ValueError, match="clip_ratio"):
        ppo.anchored_objective(data["logits"], *rows, **{**base, "clip_ratio": -0.1})
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ppo.anchored_objective(data["logits"].double(), *rows, **base)
    with pytest.raises(ValueError, match="reference_logits must be"):
        ppo.anchored_objective(data["logits"].bfloat16(), *rows, **base)
    with pytest.raises(ValueError, match="legal must be"):
        ppo.anchored_objective(data["logits"], *rows, **{**base, "legal": data["legal"].float()})
    with pytest.raises(ValueError, match="legal must be"):
        ppo.anchored_objective(data["logits"], *rows, **{**base, "legal": data["legal"][:, :50]})
    with pytest.raises(ValueError, match="old_log_probs"):
        ppo.anchored_objective(data["logits"], data["actions"], data["old"][:3], *rows[2:], **base)
    with pytest.raises(ValueError, match="integers"):
        ppo.action_log_probs(data["logits"], data["old"])
    with pytest.raises(ValueError, match="width"):
        ppo.action_log_probs(data["logits"][:, :0], data["actions"])
    with pytest.raises(ValueError, match="CUDA"):
        ppo.action_log_probs(data["logits"].cpu(), data["actions"].cpu())


def test_the_library_refuses_bad_arguments():
    with pytest.raises(nat.NativeError, match="dtype"):
        nat.call("cg_action_log_probs", None, 7, 1, 1, 1, None, 0, None, None, None)
    with pytest.raises(nat.NativeError, match="stride"):
        nat.call("cg_action_log_probs", None, 0, 1, 4, 3, None, 0, None, None, None)
    with pytest.raises(nat.NativeError, match="totals"):
        nat.call("cg_anchored_objective", None, 0, 0, 4, 4, None, 0, None, None, 0, None, None, None, None, 0.2, 0.0,
                 0.0, None, 4, None, None, 0, None)


def _moved(plane, before, after):
    """The plane as columns of a wider store: its rows start `before` entries in."""

    store = torch.zeros((plane.shape[0], before + plane.shape[1] + after), dtype=plane.dtype, device=plane.device)
    store[:, before:before + plane.shape[1]] = plane
    return store[:, before:before + plane.shape[1]]


@pytest.mark.gpu
@pytest.mark.parametrize("legal", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [2, 17, 31, 32, 33, 61, 64, 65, 125, 128, 129, 250, 256, 257, 509, 512, 513, 777, 1017, 1018,
                                   1024, 1025])
def test_the_edges_of_a_rows_registers_at_any_alignment(width, dtype, legal):
    data = inputs(70, width, TYPES[dtype], legal=legal, seed=width)
    check(data)
    data["logits"] = _moved(data["logits"], 1, 2)
    data["reference_logits"] = _moved(data["reference_logits"], 3, 1)
    if legal:
        data["legal"] = _moved(data["legal"], 1, 0)
    check(data)
    assert nat.fault_status() == 0


@pytest.mark.gpu
def test_the_objective_may_be_added_to_in_place():
    """As other losses are: autograd takes it as a tensor of its own, and the totals keep their values."""

    data = inputs(16, 300, torch.float32)
    _, want_totals, once = run(data)
    logits = data["logits"].detach().requires_grad_()
    other = torch.ones(3, device="cuda", requires_grad=True)
    objective, totals = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                               clip_ratio=CLIP, beta=BETA, alpha=ALPHA,
                                               reference_logits=data["reference_logits"])
    objective += 5.0 * other.sum()
    objective /= 4.0
    objective.backward()
    assert torch.equal(logits.grad, 0.25 * once) and torch.equal(other.grad, torch.full_like(other, 1.25))
    assert torch.equal(totals, want_totals)
    with torch.no_grad():
        value, totals = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                               clip_ratio=CLIP, beta=BETA, alpha=ALPHA,
                                               reference_logits=data["reference_logits"])
        value += 1.0
    assert torch.equal(totals, want_totals)


@pytest.mark.gpu
@pytest.mark.parametrize("weight,beta,alpha", [(4.0, 1.0, 0.0), (-4.0, 1.0, 0.0), (1.0, -4.0, 0.0), (1.0, 0.1, 40.0),
                                               (1.0, 0.1, -40.0), (-3.0, 0.3, 2.0)])
@pytest.mark.parametrize("width", [52, 2000, 30000])
def test_the_lowest_logit_has_no_gradient_under_large_coefficients_of_either_sign(width, weight, beta, alpha):
    """A probability of zero times a coefficient times the lowest logit's distance, which passes the largest float."""

    data = inputs(8, width, torch.float32, legal=True)
    hide = ~data["legal"]
    data["weights"][:] = weight
    filled = dict(data, legal=None, logits=data["logits"].masked_fill(hide, torch.finfo(torch.float32).min),
                  reference_logits=data["reference_logits"].masked_fill(hide, -1e5))
    objective, totals, gradient = run(filled, beta=beta, alpha=alpha)
    assert torch.isfinite(gradient).all() and not gradient[hide].any()


@pytest.mark.gpu
def test_the_inputs_are_released_with_the_graph():
    """What the backward pass may need is held by autograd: hooks see it, and the first backward lets go of it."""

    data = inputs(64, 5000, torch.float32, legal=True)
    logits = data["logits"].detach().requires_grad_()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t, lambda t: t):
        objective, _ = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                              clip_ratio=CLIP, beta=BETA, alpha=ALPHA,
                                              reference_logits=data["reference_logits"], legal=data["legal"])
    assert seen.count(torch.Size([64, 5000])) == 3  # logits, reference, mask
    objective.backward()
    held = torch.cuda.memory_allocated()
    del data["reference_logits"], data["legal"]
    assert torch.cuda.memory_allocated() <= held - 64 * 5000 * 5 and objective.grad_fn is not None


@pytest.mark.gpu
def test_a_second_backward_refuses_inputs_that_have_changed():
    data = inputs(8, 300, torch.float32)
    logits = data["logits"].detach().requires_grad_()
    objective, _ = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                          clip_ratio=CLIP, beta=BETA, reference_logits=data["reference_logits"])
    objective.backward(retain_graph=True)
    data["advantages"].add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        objective.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("factor_of_loss", [65536.0, 3.0, 0.37])
@pytest.mark.parametrize("legal", [False, True])
@pytest.mark.parametrize("reference", ["logits", "log-probs"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [52, 700, 3000, 20000])
def test_a_loss_scale_comes_before_the_gradients_rounding(width, dtype, reference, legal, factor_of_loss):
    """With weights of a mean over many rows a 16-bit gradient is small: (factor * objective).backward() is the scaled
    objective's gradient rounded once, not the factor times a gradient that was rounded, to zero in part, before it."""

    data = inputs(24, width, TYPES[dtype], reference=reference, legal=legal)
    data["weights"] = data["weights"] / 2.0 ** 18
    _, _, want, scale, _ = formula(data)
    logits = data["logits"].detach().requires_grad_()
    extra = {k: data[k] for k in ("reference_logits", "reference_log_probs") if k in data}
    objective, totals = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                               clip_ratio=CLIP, beta=BETA, alpha=ALPHA, legal=data["legal"], **extra)
    before = totals.clone()
    (got,) = torch.autograd.grad(factor_of_loss * objective, logits, retain_graph=True)
    k = factor(width)
    for by, gradient in ((factor_of_loss, got), (0.5, torch.autograd.grad(0.5 * objective, logits)[0])):
        bound = by * (k * scale[:, None] + (1 + 2 * k) * HALF_STEP[TYPES[dtype]] * want.abs())
        if TYPES[dtype] == torch.float16:
            bound = bound + 2.0 ** -25
        assert gradient.dtype == TYPES[dtype]
        assert ((gradient.double() - by * want).abs() <= bound).all()
    assert torch.equal(totals, before) and nat.fault_status() == 0


@pytest.mark.gpu
def test_a_gradient_scaler_trains_half_precision_logits():
    """GradScaler's scale reaches the gradient before its rounding, and its unscaled gradient is the formula's."""

    data = inputs(64, 52, torch.float16, legal=True)
    data["weights"] = data["weights"] / 2.0 ** 20
    _, _, want, scale, _ = formula(data)
    logits = data["logits"].detach().requires_grad_()
    objective, _ = ppo.anchored_objective(logits, data["actions"], data["old"], data["advantages"], data["weights"],
                                          clip_ratio=CLIP, beta=BETA, alpha=ALPHA, legal=data["legal"],
                                          reference_logits=data["reference_logits"])
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 20)
    scaler.scale(objective).backward()
    k = factor(52)
    bound = 2.0 ** 20 * (k * scale[:, None] + (1 + 2 * k) * 2.0 ** -11 * want.abs()) + 2.0 ** -25
    assert ((logits.grad.double() - 2.0 ** 20 * want).abs() <= bound).all()


def test_the_library_refuses_a_gradient_without_its_scale():
    fill = [None, 0, 0, 4, 4, None, 0, None, None, 0, None, None, None, None, 0.2, 0.0, 0.0]
    with pytest.raises(nat.NativeError, match="NULL pointer"):
        nat.call("cg_anchored_gradient", None, 0, 1, *fill[3:], None, 0, None, 4, None)
    with pytest.raises(nat.NativeError, match="dtype"):
        nat.call("cg_anchored_gradient", None, 9, *fill[2:], None, 0, None, 4, None)


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [0.0, 1e-4, -1e-3, 0.01, 0.3, -0.49, 0.51, -1.0, 2.0])
@pytest.mark.parametrize("width", [2, 52, 700, 2000])
def test_the_sampled_divergences_do_not_cancel_near_the_reference(width, apart):
    """exp(u) - u - 1 is u^2 / 2 near zero, far below the rounding of 1. Of uniform logits log pi = -log(width) is off by
    2^-21 at most (4 units in the last place of 7.6), which moves the estimate by |exp(u) - 1| times it; its own
    arithmetic takes 2^-20 of itself, and past the series 2^-22 of exp(u) + |u| + 1."""

    rows = 40
    logits = torch.zeros((rows, width), device="cuda", requires_grad=True)
    level = -math.log(width)
    log_probs = torch.full((rows,), level + apart, device="cuda")
    ones = torch.ones(rows, device="cuda")
    actions = torch.arange(rows, device="cuda") % width
    objective, totals = ppo.anchored_objective(logits, actions, log_probs, 0.0 * ones, ones, clip_ratio=CLIP, beta=1.0,
                                               reference_log_probs=log_probs)
    objective.backward()
    u = float(log_probs[0].double()) - level
    for key, v in (("reference_kl", u), ("behavior_kl", -u)):
        want = math.expm1(v) - v
        bound = abs(math.expm1(v)) * 2.0 ** -21 + 2.0 ** -20 * want + (2.0 ** -22 * (math.exp(v) + abs(v) + 1) if abs(v) >= 0.49 else 0)
        got = float(totals[ppo.ANCHORED_KEYS.index(key)]) / rows
        assert abs(got - want) <= bound + 2.0 ** -42, key
    slope = -math.expm1(u) * (1.0 - 1.0 / width)  # d KL / d logit of the action
    assert abs(float(logits.grad[0, 0]) - slope) <= 2.0 ** -20 * abs(slope) + 2.0 ** -20 * math.exp(u)


def test_rows_past_32_bits_are_refused():
    """By the wrapper, which would hand the library a width cut to 32 bits, and by the library."""

    wide = torch.zeros((1, 1)).expand(1, (1 << 32) + 52)
    with pytest.raises(ValueError, match="width of at most"):
        ppo.action_log_probs(wide, torch.zeros(1, dtype=torch.int64))
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="width of at most"):
        ppo.anchored_objective(wide, torch.zeros(1, dtype=torch.int64), one, one, one, clip_ratio=CLIP, beta=0.0)
    with pytest.raises(nat.NativeError, match="bad shape"):
        nat.call("cg_action_log_probs", None, 0, 1, (1 << 30) + 1, (1 << 30) + 1, None, 0, None, None, None)
