"""The policy update's operators on real work: the anchored policy objective, the fused linear layer, the AdamW step.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the
end) or, where ``own`` is set, through card_playing_gym_b200's public entry points. ``exact`` restates each
definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CLIP, BETA, ALPHA = 0.2, 0.05, 0.01
LR, BETAS, EPS, DECAY, STEPS_BEFORE = 3e-4, (0.9, 0.999), 1e-8, 0.01, 100
BLOCK = 256  # entries of one scale of an 8-bit state; every tensor starts on a multiple of it
E4M3_MAX = 448.0

LARGEST_ROWS, LARGEST_VOCABULARY = 4096, 131072
LARGEST_PRODUCT = 8192 * 4096 * 4096
LARGEST_MODEL = 1 << 28


# -- cases ------------------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # One small minibatch of card plays: 52 cards, a legal mask, the magnet policy's logits beside it.
        dict(name="objective cards small", op="objective", rows=96, width=52, type="float32", reference="logits",
             legal=True, grad=True, pad=0),
        # The update's full batch of decisions (the PPO step's 262,144 rows of 52 cards).
        dict(name="objective cards batch", op="objective", rows=262144, width=52, type="float32", reference="logits",
             legal=True, grad=True, pad=0),
        # Token log-probabilities of a recorded batch under the current policy, odd width, no gradient.
        dict(name="objective log-probs", op="objective", rows=1500, width=50021, type="float16", reference="none",
             legal=False, grad=False, pad=3),
        # Fine-tuning a sequence model on its own samples against a frozen reference: the full vocabulary's logits.
        dict(name="objective vocabulary", op="objective", rows=4096, width=131072, type="bfloat16",
             reference="logits", legal=False, grad=True, pad=0),
        # One game's next decision through a trunk MLP's up projection.
        dict(name="linear single token", op="linear", rows=1, inner=240, outer=720, type="bfloat16",
             activation="gelu", bias=True, residual=False, grad=False),
        # A few sequences' next token through a wide layer: the weights are what is read.
        dict(name="linear decode", op="linear", rows=24, inner=4096, outer=8192, type="bfloat16", activation="silu",
             bias=True, residual=False, grad=False),
        # A training microbatch through a trunk MLP's down projection onto the residual, in full precision.
        dict(name="linear trunk down", op="linear", rows=16384, inner=720, outer=240, type="float32",
             activation="none", bias=True, residual=True, grad=True),
        # A training microbatch through a wide layer with its activation and residual.
        dict(name="linear wide", op="linear", rows=8192, inner=4096, outer=4096, type="bfloat16", activation="gelu",
             bias=True, residual=True, grad=True),
        # The smallest configuration's trunk (d 32, two layers), no clipping.
        dict(name="adamw small", op="adamw", layout="trunk", d=32, ff=64, layers=2, type="float32", bits=32,
             clip=False),
        # The rl-v6 trunk (d 240, 16 layers) in 32-bit states with the trainer's global-norm clip.
        dict(name="adamw trunk", op="adamw", layout="trunk", d=240, ff=720, layers=16, type="float32", bits=32,
             clip=True),
        # The same trunk widened and deepened, states in 8 bits.
        dict(name="adamw deep trunk 8-bit", op="adamw", layout="trunk", d=1024, ff=2048, layers=24, type="float32",
             bits=8, clip=True),
        # A model of a quarter of a billion weights trained in bfloat16 with 32-bit master copies.
        dict(name="adamw large 8-bit", op="adamw", layout="split", elements=LARGEST_MODEL, tensors=120, spread=1,
             type="bfloat16", bits=8, clip=True),
    ]


def _log_uniform(rng: random.Random, low: float, high: float) -> int:
    return max(int(low), min(int(high), round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("objective", "linear", "adamw"))
    if op == "objective":
        width = _log_uniform(rng, 2, LARGEST_VOCABULARY)
        rows = _log_uniform(rng, 1, min(1 << 18, LARGEST_ROWS * LARGEST_VOCABULARY // (2 * width)))
        grad = rng.random() < 0.8
        return dict(op=op, rows=rows, width=width, type=rng.choice(list(TYPES)),
                    reference=rng.choice(("logits", "log-probs")) if grad else "none", legal=rng.random() < 0.5,
                    grad=grad, pad=rng.choice((0, 0, 3, 8)))
    if op == "linear":
        inner, outer = _log_uniform(rng, 1, 8192), _log_uniform(rng, 1, 8192)
        rows = _log_uniform(rng, 1, min(1 << 17, LARGEST_PRODUCT // (2 * inner * outer)))
        return dict(op=op, rows=rows, inner=inner, outer=outer, type=rng.choice(list(TYPES)),
                    activation=rng.choice(("none", "relu", "gelu", "silu")), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.5, grad=rng.random() < 0.7)
    tensors = _log_uniform(rng, 1, 200)
    return dict(op=op, layout="split", elements=_log_uniform(rng, 1e4, LARGEST_MODEL // 2), tensors=tensors,
                spread=rng.randrange(1 << 20), type=rng.choice(list(TYPES)), bits=rng.choice((8, 32)),
                clip=rng.random() < 0.7)


def _sizes(case: dict) -> list[int]:
    """Entries of each parameter: a trunk's (per layer: qkv, out, up, down, their biases and two norms), or a split."""

    if case["layout"] == "trunk":
        d, ff = case["d"], case["ff"]
        return [d] + [d * d + d * d // 2, d * d, ff * d, ff, d * ff, d, d, d, d, d] * case["layers"]
    rng = random.Random(case["spread"])
    share = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(case["tensors"])]
    scale = case["elements"] / sum(share)
    return [max(1, int(s * scale)) for s in share]


def work(case: dict) -> dict:
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        size = TYPES[case["type"]].itemsize
        weight = 2 * 4 + (size if size < 4 else 0)  # the fp32 weight read and written, and its 16-bit copy written
        moments = 4 * (1 + 4 / BLOCK) if case["bits"] == 8 else 16
        return {"bytes": n * (size + weight + moments), "flops": n * (20 + (2 if case["clip"] else 0))}
    size = TYPES[case["type"]].itemsize
    if case["op"] == "objective":
        n = case["rows"] * case["width"]
        planes = size * (1 + (case["reference"] == "logits") + case["grad"]) + case["legal"]
        return {"bytes": n * planes + case["rows"] * 24, "flops": n * (25 if case["grad"] else 4)}
    m, k, n = case["rows"], case["inner"], case["outer"]
    bias, residual = case["bias"], case["residual"]
    nbytes = m * k + n * k + n * bias + m * n * residual + m * n
    flops = 2 * m * n * k
    if case["grad"]:  # dy in; dx, dw, db out (the residual's gradient is dy)
        nbytes += m * n + m * k + n * k + n * bias
        flops += 4 * m * n * k
    return {"bytes": nbytes * size, "flops": flops}


# -- inputs -----------------------------------------------------------------------------------------------------------
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(generator, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=generator, device=DEVICE)


def _objective_inputs(case: dict, seed: int) -> dict:
    """Logits of a trained policy, a reference near it, sampled actions, and the behaviour's log-probabilities."""

    g = _generator(seed)
    rows, width = case["rows"], case["width"]
    kind = TYPES[case["type"]]
    store = (2.0 * _normal(g, rows, width + case["pad"])).to(kind)
    logits = store[:, :width]
    legal = None
    if case["legal"]:
        legal = torch.rand((rows, width), generator=g, device=DEVICE) < 0.6
        if rows >= 8:
            legal[3] = False  # a padding row: nothing is legal
    z = logits.float() if legal is None else logits.float().masked_fill(~legal, -math.inf)
    noise = torch.rand((rows, width), generator=g, device=DEVICE).clamp_(1e-20, 1 - 1e-7)
    actions = torch.argmax(z - torch.log(-torch.log(noise)), dim=1)
    del noise
    log_probs = z.gather(1, actions[:, None])[:, 0] - torch.logsumexp(z, dim=1)
    log_probs = torch.where(torch.isfinite(log_probs), log_probs, torch.zeros_like(log_probs))
    if rows >= 8:
        actions[5::32] = -1  # positions that are not the policy's own: they count for nothing
    # The new policy has moved a little from the one that acted. No ratio lies within rounding of the clip's
    # bounds, where two correct roundings may fall on either side of the kink.
    log_ratio = 0.15 * _normal(g, rows)
    for bound in (math.log(1 - CLIP), math.log(1 + CLIP)):
        near = (log_ratio - bound).abs() < 1e-3
        log_ratio = torch.where(near, torch.full_like(log_ratio, bound + 2e-3), log_ratio)
    state = dict(logits=logits, legal=legal, actions=actions, old=log_probs - log_ratio,
                 advantages=_normal(g, rows),
                 weights=torch.rand(rows, generator=g, device=DEVICE).add_(0.5).div_(rows))
    if case["reference"] == "logits":
        reference = z.new_empty((rows, width)).normal_(generator=g).mul_(0.3)
        state["reference"] = reference.add_(logits.float()).to(kind)
    elif case["reference"] == "log-probs":
        state["reference"] = log_probs + 0.2 * _normal(g, rows)
    return state


def _linear_inputs(case: dict, seed: int) -> dict:
    g = _generator(seed)
    kind = TYPES[case["type"]]
    m, k, n = case["rows"], case["inner"], case["outer"]
    state = dict(x=_normal(g, m, k).to(kind), weight=(_normal(g, n, k) / math.sqrt(k)).to(kind), bias=None,
                 residual=None, dy=None)
    if case["bias"]:
        state["bias"] = (0.1 * _normal(g, n)).to(kind)
    if case["residual"]:
        state["residual"] = _normal(g, m, n).to(kind)
    if case["grad"]:
        state["dy"] = _normal(g, m, n).to(kind)
    return state


def _adamw_inputs(case: dict, seed: int) -> dict:
    """One step in the middle of training: parameters, gradients and moments in flat storage with a view per tensor."""

    g = _generator(seed)
    kind = TYPES[case["type"]]
    sizes = _sizes(case)
    starts, total = [], 0
    for size in sizes:
        starts.append(total)
        total += -(-size // BLOCK) * BLOCK
    starts_gpu = torch.tensor(starts, device=DEVICE)
    ends_gpu = starts_gpu + torch.tensor(sizes, device=DEVICE)
    at = torch.arange(0, total, BLOCK, device=DEVICE)
    which = torch.searchsorted(starts_gpu, at, right=True) - 1
    live = (at[:, None] + torch.arange(BLOCK, device=DEVICE)) < ends_gpu[which][:, None]
    # Gradients of one magnitude per tensor; a tenth of the blocks got none and have no history (rows of an
    # embedding that no token of the run has named).
    scale = torch.exp(1.5 * _normal(g, len(sizes)))[which][:, None] * 1e-3
    touched = (torch.rand(len(at), 1, generator=g, device=DEVICE) > 0.1) & live
    del at, which

    def blocks(factor) -> torch.Tensor:
        return _normal(g, total // BLOCK, BLOCK).mul_(factor).mul_(touched)

    grad = blocks(scale).view(-1).to(kind)
    first = blocks(0.3 * scale)
    second = blocks(scale).square_().mul_(0.5).add_(0.5 * scale.square() * touched)
    master = _normal(g, total // BLOCK, BLOCK).mul_(0.02).mul_(live).view(-1)
    state = dict(sizes=sizes, starts=starts, grad=grad, steps=STEPS_BEFORE, live=live)
    state["weights"] = master.to(kind) if kind != torch.float32 else master
    if kind != torch.float32:
        state["master"] = master
    if case["bits"] == 32:
        state["moments"] = dict(exp_avg=first.view(-1), exp_avg_sq=second.view(-1))
    else:
        state["moments"] = {}
        for name, value in (("exp_avg", first), ("exp_avg_sq_root", second.sqrt_())):
            peak = value.abs().amax(dim=1)
            unit = torch.where(peak > 0, E4M3_MAX / peak, torch.zeros_like(peak))
            state["moments"][name] = (value * unit[:, None]).to(torch.float8_e4m3fn).view(-1)
            state["moments"][name + "_scale"] = peak
    return state


_INPUTS = {"objective": _objective_inputs, "linear": _linear_inputs, "adamw": _adamw_inputs}


def prepare(case: dict, seed: int) -> dict:
    state = _INPUTS[case["op"]](case, seed)
    state["case"] = case
    if own and case["op"] == "adamw":
        from card_playing_gym_b200.optim import AdamW

        parameters = []
        for start, size in zip(state["starts"], state["sizes"]):
            p = torch.nn.Parameter(state["weights"][start:start + size])
            p.grad = state["grad"][start:start + size]
            parameters.append(p)
        optimizer = AdamW(parameters, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                          max_norm=1.0 if case["clip"] else None)
        for name, value in state.pop("moments").items():
            optimizer.flat[name].copy_(value)
        if "master" in state:
            optimizer.flat["master"].copy_(state.pop("master"))
        optimizer.steps.fill_(STEPS_BEFORE)
        state["optimizer"] = optimizer
    return state


# -- the plain forms --------------------------------------------------------------------------------------------------
def _plain_objective(state: dict):
    case, actions = state["case"], state["actions"]
    logits, legal = state["logits"], state["legal"]
    z = logits.float()
    if legal is not None:
        z = z.masked_fill(~legal, -math.inf)
    peak = z.amax(dim=1, keepdim=True)
    peak = torch.where(torch.isfinite(peak), peak, torch.zeros_like(peak))
    exps = torch.exp(z - peak)
    total = exps.sum(dim=1, keepdim=True)
    used = (actions >= 0) & (total[:, 0] > 0)
    total = torch.where(total > 0, total, torch.ones_like(total))
    log_p = z - peak - torch.log(total)
    picked = log_p.gather(1, actions.clamp(min=0)[:, None])[:, 0]
    zero = torch.zeros((), device=z.device)
    if not case["grad"]:
        return torch.where(used, picked, zero)
    p = exps / total
    inside = p > 0
    picked = torch.where(used, picked, zero)
    old, advantages = state["old"], state["advantages"]
    weights = torch.where(used, state["weights"], zero)
    log_ratio = torch.where(used, picked - old, zero)
    ratio = torch.exp(log_ratio)
    clipped = ratio.clamp(1 - CLIP, 1 + CLIP)
    surrogate = -torch.minimum(ratio * advantages, clipped * advantages)
    held = clipped * advantages < ratio * advantages
    slope = torch.where(held, zero, -advantages * ratio)
    plogp = torch.where(inside, p * log_p, zero)
    entropy = -plogp.sum(dim=1)
    count = torch.full_like(weights, z.shape[1]) if legal is None else legal.sum(dim=1).float()
    eligible = (count > 1) & used
    norm = torch.where(eligible, 1 / torch.log(count.clamp(min=2)), zero)
    gradient = torch.where(inside, ALPHA * norm[:, None] * p * (log_p + entropy[:, None]), zero)
    if case["reference"] == "logits":
        r = state["reference"].float()
        if legal is not None:
            r = r.masked_fill(~legal, -math.inf)
        r_peak = r.amax(dim=1, keepdim=True)
        r_peak = torch.where(torch.isfinite(r_peak), r_peak, torch.zeros_like(r_peak))
        r_total = torch.exp(r - r_peak).sum(dim=1, keepdim=True)
        apart = torch.where(inside, log_p - (r - r_peak - torch.log(r_total)), zero)
        divergence = (p * apart).sum(dim=1)
        gradient = gradient + BETA * p * (apart - divergence[:, None]) * inside
    else:
        u = torch.where(used, state["reference"] - picked, zero)
        divergence = torch.exp(u) - u - 1
        slope = slope + BETA * (1 - torch.exp(u))
    gradient = gradient - p * slope[:, None]
    gradient.scatter_add_(1, actions.clamp(min=0)[:, None], torch.where(used, slope, zero)[:, None])
    gradient = gradient * weights[:, None]
    gradient = torch.where(used[:, None], gradient, zero)
    normalised = entropy * norm
    outside = (ratio - 1).abs() > CLIP
    row_objective = surrogate + BETA * divergence - ALPHA * normalised
    terms = torch.stack([surrogate, torch.ones_like(ratio), entropy, normalised, eligible.float(), outside.float(),
                         ratio - 1 - log_ratio, divergence, row_objective])
    totals = (torch.where(used, terms, zero) * weights).sum(dim=1)
    return {"objective": totals[8], "totals": totals, "gradient": gradient.to(logits.dtype)}


def _activation(pre: torch.Tensor, name: str):
    """The activation and its derivative."""

    if name == "relu":
        return pre.clamp(min=0), (pre > 0).to(pre.dtype)
    if name == "gelu":
        cumulative = 0.5 * (1 + torch.erf(pre * math.sqrt(0.5)))
        return pre * cumulative, cumulative + pre * torch.exp(-0.5 * pre * pre) / math.sqrt(2 * math.pi)
    if name == "silu":
        gate = 1 / (1 + torch.exp(-pre))
        return pre * gate, gate * (1 + pre * (1 - gate))
    return pre, torch.ones_like(pre)


def _plain_linear(state: dict):
    case = state["case"]
    kind = state["x"].dtype
    x, weight = state["x"].float(), state["weight"].float()
    pre = x @ weight.t()
    if state["bias"] is not None:
        pre = pre + state["bias"].float()
    y, slope = _activation(pre, case["activation"])
    if state["residual"] is not None:
        y = y + state["residual"].float()
    if not case["grad"]:
        return y.to(kind)
    dpre = state["dy"].float() * slope
    out = {"y": y.to(kind), "dx": (dpre @ weight).to(kind), "dweight": (dpre.t() @ x).to(kind)}
    if state["bias"] is not None:
        out["dbias"] = dpre.sum(dim=0).to(kind)
    if state["residual"] is not None:
        out["dresidual"] = state["dy"]
    return out


def _plain_adamw(state: dict):
    case, moments, live = state["case"], state["moments"], state["live"]
    state["steps"] += 1
    lr, (b1, b2) = LR, BETAS
    grad = state["grad"].float().view(-1, BLOCK)
    if case["clip"]:
        norm = torch.sqrt((grad * grad).sum())
        grad = grad * torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    if case["bits"] == 32:
        first, second = (moments[name].view(-1, BLOCK) for name in ("exp_avg", "exp_avg_sq"))
    else:
        first = moments["exp_avg"].float().view(-1, BLOCK) * (moments["exp_avg_scale"] / E4M3_MAX)[:, None]
        root = moments["exp_avg_sq_root"].float().view(-1, BLOCK)
        second = (root * (moments["exp_avg_sq_root_scale"] / E4M3_MAX)[:, None]).square()
    first = b1 * first + (1 - b1) * grad
    second = b2 * second + (1 - b2) * (grad * grad)
    root = torch.sqrt(second)
    denominator = root * (1 / math.sqrt(1 - b2 ** state["steps"])) + EPS
    step = first / denominator * (lr / (1 - b1 ** state["steps"]))
    master = state.get("master", state["weights"])
    master.copy_((master.view(-1, BLOCK) * (1 - lr * DECAY) - step).view(-1))
    if "master" in state:
        state["weights"].copy_(master)
    if case["bits"] == 32:
        moments["exp_avg"].copy_(first.view(-1))
        moments["exp_avg_sq"].copy_(second.view(-1))
    else:
        for name, value in (("exp_avg", first), ("exp_avg_sq_root", root)):
            peak = value.abs().amax(dim=1)
            unit = torch.where(peak > 0, E4M3_MAX / peak, torch.zeros_like(peak))[:, None]
            scaled = value * unit
            if name == "exp_avg_sq_root":  # what is not zero keeps at least the smallest code
                scaled = torch.where((value > 0) & (scaled < 2.0 ** -9), torch.full_like(scaled, 2.0 ** -9), scaled)
            moments[name].copy_(scaled.to(torch.float8_e4m3fn).view(-1))
            moments[name + "_scale"].copy_(peak)
    return {"weights": state["weights"], **({"master": state["master"]} if "master" in state else {}), **moments}


# -- one pass ---------------------------------------------------------------------------------------------------------
def run(state: dict):
    case = state["case"]
    if not own:
        return {"objective": _plain_objective, "linear": _plain_linear, "adamw": _plain_adamw}[case["op"]](state)
    if case["op"] == "objective":
        from card_playing_gym_b200 import ppo

        if not case["grad"]:
            return ppo.action_log_probs(state["logits"], state["actions"], legal=state["legal"])
        logits = state["logits"].detach().requires_grad_()
        name = "reference_logits" if case["reference"] == "logits" else "reference_log_probs"
        objective, totals = ppo.anchored_objective(
            logits, state["actions"], state["old"], state["advantages"], state["weights"], clip_ratio=CLIP, beta=BETA,
            alpha=ALPHA, legal=state["legal"], **{name: state["reference"]})
        (gradient,) = torch.autograd.grad(objective, logits)
        return {"objective": objective.detach(), "totals": totals, "gradient": gradient}
    if case["op"] == "linear":
        from card_playing_gym_b200 import dense

        if not case["grad"]:
            with torch.no_grad():
                return dense.linear(state["x"], state["weight"], state["bias"], state["residual"],
                                    activation=case["activation"])
        leaves = {name: state[name].detach().requires_grad_() for name in ("x", "weight", "bias", "residual")
                  if state[name] is not None}
        y = dense.linear(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("residual"),
                         activation=case["activation"])
        grads = torch.autograd.grad(y, list(leaves.values()), state["dy"])
        return {"y": y.detach(), **{"d" + name: grad for name, grad in zip(leaves, grads)}}
    optimizer = state["optimizer"]
    optimizer.step()
    return {"weights": state["weights"], **optimizer.flat}


# -- the definitions in 64 bits ---------------------------------------------------------------------------------------
def _exact_objective(case: dict, s: dict):
    rows, width = s["logits"].shape
    step = max(1, (1 << 26) // width)
    pieces, gradient = [], []
    for at in range(0, rows, step):
        cut = slice(at, at + step)
        z, actions = s["logits"][cut].double(), s["actions"][cut]
        legal = torch.ones_like(z, dtype=torch.bool) if s["legal"] is None else s["legal"][cut]
        counted = (actions >= 0) & legal.any(dim=1)
        legal = legal | ~legal.any(dim=1, keepdim=True)  # an empty row is computed over everything, then dropped
        log_pi = torch.where(legal, z - torch.logsumexp(torch.where(legal, z, -math.inf), dim=1, keepdim=True), 0.0)
        pi = torch.where(legal, torch.exp(log_pi), 0.0)
        chosen = torch.nn.functional.one_hot(actions.clamp(min=0), width).double()
        lp = (log_pi * chosen).sum(dim=1)
        if not case["grad"]:
            pieces.append(torch.where(counted, lp, 0.0))
            continue
        advantage = s["advantages"][cut].double()
        log_ratio = lp - s["old"][cut].double()
        ratio = torch.exp(log_ratio)
        bounded = torch.clamp(ratio, 1 - CLIP, 1 + CLIP)
        loss = -torch.minimum(ratio * advantage, bounded * advantage)
        d_lp = torch.where(ratio * advantage <= bounded * advantage, -advantage * ratio, 0.0)
        entropy = -(pi * log_pi).sum(dim=1)
        number = legal.sum(dim=1)
        norm = torch.where(number > 1, 1 / torch.log(number.clamp(min=2).double()), 0.0)
        d_logits = ALPHA * norm[:, None] * pi * (log_pi + entropy[:, None])
        if case["reference"] == "logits":
            ref = s["reference"][cut].double()
            log_rho = ref - torch.logsumexp(torch.where(legal, ref, -math.inf), dim=1, keepdim=True)
            gap = torch.where(legal, log_pi - log_rho, 0.0)
            kl = (pi * gap).sum(dim=1)
            d_logits += BETA * pi * (gap - kl[:, None])
        else:
            u = s["reference"][cut].double() - lp
            kl = torch.expm1(u) - u
            d_lp = d_lp - BETA * torch.expm1(u)
        d_logits += d_lp[:, None] * (chosen - pi)
        w = torch.where(counted, s["weights"][cut].double(), 0.0)
        gradient.append(torch.where(counted[:, None], d_logits * w[:, None], 0.0))
        full = loss + BETA * kl - ALPHA * norm * entropy
        terms = torch.stack([loss, torch.ones_like(loss), entropy, norm * entropy, (number > 1).double(),
                             ((ratio - 1).abs() > CLIP).double(), ratio - 1 - log_ratio, kl, full])
        pieces.append((torch.where(counted, terms, 0.0) * w).sum(dim=1))
    if not case["grad"]:
        return torch.cat(pieces)
    totals = torch.stack(pieces).sum(dim=0)
    return {"objective": totals[8], "totals": totals, "gradient": torch.cat(gradient)}


def _exact_linear(case: dict, s: dict):
    wide = {name: None if s[name] is None else s[name].double() for name in ("x", "weight", "bias", "residual", "dy")}
    pre = torch.einsum("mk,nk->mn", wide["x"], wide["weight"])
    if wide["bias"] is not None:
        pre += wide["bias"]
    pre.requires_grad_(case["grad"])
    functional = torch.nn.functional
    post = {"none": lambda t: t * 1.0, "relu": functional.relu, "gelu": functional.gelu,
            "silu": functional.silu}[case["activation"]](pre)
    y = post.detach() if wide["residual"] is None else post.detach() + wide["residual"]
    if not case["grad"]:
        return y
    (dpre,) = torch.autograd.grad(post, pre, wide["dy"])
    out = {"y": y, "dx": torch.einsum("mn,nk->mk", dpre, wide["weight"]),
           "dweight": torch.einsum("mn,mk->nk", dpre, wide["x"])}
    if wide["bias"] is not None:
        out["dbias"] = torch.einsum("mn->n", dpre)
    if wide["residual"] is not None:
        out["dresidual"] = wide["dy"]
    return out


def _exact_adamw(case: dict, s: dict):
    moments, t = s["moments"], STEPS_BEFORE + 1
    g = s["grad"].double()
    if case["clip"]:
        g *= min(1.0, 1.0 / (float(torch.linalg.vector_norm(g)) + 1e-6))

    def held(name):
        return moments[name].double() * moments[name + "_scale"].double().repeat_interleave(BLOCK) / E4M3_MAX

    m = moments["exp_avg"].double() if case["bits"] == 32 else held("exp_avg")
    v = moments["exp_avg_sq"].double() if case["bits"] == 32 else held("exp_avg_sq_root") ** 2
    m = m.mul_(BETAS[0]).add_(g, alpha=1 - BETAS[0])
    v = v.mul_(BETAS[1]).addcmul_(g, g, value=1 - BETAS[1])
    m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    w = s.get("master", s["weights"]).double()
    w = w - LR * DECAY * w - LR * m_hat / (v_hat.sqrt() + EPS)
    out = {"weights": w, **({"master": w} if "master" in s else {})}
    if case["bits"] == 32:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    # The 8-bit codes are steps of the scales, which have values in 64 bits; the codes themselves do not.
    return {**out, "exp_avg": None, "exp_avg_sq_root": None,
            "exp_avg_scale": m.abs().view(-1, BLOCK).amax(dim=1),
            "exp_avg_sq_root_scale": v.sqrt().view(-1, BLOCK).amax(dim=1)}


def exact(case: dict, seed: int):
    s = _INPUTS[case["op"]](case, seed)
    return {"objective": _exact_objective, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](case, s)
