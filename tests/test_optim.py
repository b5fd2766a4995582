"""optim.AdamW against its formula in 64 bits: types, state widths, odd and unaligned tensors, the clip, skipped steps,
groups, missing gradients, the state's round trip, and its refusals.

Tolerances. fp32 arithmetic on k rounded operations is within k * 2^-24 of the operands' magnitudes: the moments take at
most 4, the weight 12 (its update is divided and scaled, and the clip's norm is summed in fp32 over 8 entries, +8).
An 8-bit code is within half a step of the value it stands for: 2^-4 of it, or 2^-10 of the block's unit where e4m3 is
subnormal. A 16-bit weight is its master rounded once."""

from __future__ import annotations

import math

import pytest
import torch

from card_playing_gym_b200 import dense
from card_playing_gym_b200 import optim

EPS32 = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = [(1,), (7,), (256,), (3, 257), (8192,), (8193,), (0,), (64, 515)]


def parameters(sizes, dtype, offset=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for size in sizes:
        n = math.prod(size)
        store = (0.05 * torch.randn(n + offset, generator=g, device="cuda")).to(dtype)
        grad = (1e-2 * torch.randn(n + offset, generator=g, device="cuda")).to(dtype)
        p = torch.nn.Parameter(store[offset:].view(size))
        p.grad = grad[offset:].view(size)
        out.append(p)
    return out


class Formula:
    """The step in float64 over a list of tensors, with 32-bit moments or the block-scaled 8-bit codes of another state."""

    def __init__(self, params, lr, betas, eps, decay, max_norm):
        self.p = [p.detach().double().clone() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.t, self.max_norm = 0, max_norm
        self.lr, self.betas, self.eps, self.decay = lr, betas, eps, decay

    def step(self, grads):
        self.t += 1
        clip = 1.0
        if self.max_norm is not None:
            norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads if g is not None))
            clip = min(1.0, self.max_norm / (norm + 1e-6))
        b1, b2 = self.betas
        for i, g in enumerate(grads):
            if g is None:
                continue
            g = g.double() * clip
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            update = self.m[i] / (1 - b1 ** self.t) / ((self.v[i] / (1 - b2 ** self.t)).sqrt() + self.eps)
            self.p[i] = self.p[i] * (1 - self.lr * self.decay) - self.lr * update


def decoded(state, name):
    codes = state[name].float().double().reshape(-1)
    scale = state[name + "_scale"].double().repeat_interleave(optim.BLOCK)[: codes.numel()]
    return (codes * scale / 448.0).reshape(state[name].shape)


def check_codes(state, name, value):
    """Every code is the nearest one to `value` at the block's scale, which is the block's largest magnitude."""

    flat = value.reshape(-1)
    for block, scale in enumerate(state[name + "_scale"].double().tolist()):
        piece = flat[block * optim.BLOCK:(block + 1) * optim.BLOCK]
        assert scale == pytest.approx(float(piece.abs().max()), rel=8 * EPS32, abs=1e-38)
        codes = state[name].reshape(-1)[block * optim.BLOCK:(block + 1) * optim.BLOCK].double()
        if scale == 0:
            assert not codes.any()
            continue
        scaled = piece * 448.0 / scale
        half = torch.maximum(scaled.abs() * 2.0 ** -4, torch.full_like(scaled, 2.0 ** -10)) * (1 + 1e-5)
        if name == "exp_avg_sq_root":
            small = (scaled > 0) & (scaled < 2.0 ** -9)
            assert (codes[small] == 2.0 ** -9).all()
            codes, scaled, half = codes[~small], scaled[~small], half[~small]
        assert ((codes - scaled).abs() <= half).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_32_bit_moments(dtype, offset, max_norm):
    params = parameters(SIZES, TYPES[dtype], offset)
    want = Formula(params, 3e-3, (0.9, 0.99), 1e-8, 0.1, max_norm)
    opt = optim.AdamW(params, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.1, max_norm=max_norm)
    g = torch.Generator(device="cuda").manual_seed(9)
    for _ in range(3):
        for p in params:
            p.grad.copy_(1e-2 * torch.randn(p.shape, generator=g, device="cuda"))
        grads = [p.grad.clone() for p in params]
        opt.step()
        want.step(grads)
    assert int(opt.steps) == 3
    for p, m, v, w in zip(params, want.m, want.v, want.p):
        state = opt.state[p]
        if not p.numel():
            continue
        assert (state["exp_avg"].double() - m).abs().max() <= 3 * 12 * EPS32 * m.abs().max()
        assert (state["exp_avg_sq"].double() - v).abs().max() <= 3 * 20 * EPS32 * v.abs().max()
        held = state["master"] if dtype != "fp32" else p.detach()
        bound = 3 * 20 * EPS32 * (w.abs().max() + 3e-3 * 10)
        assert (held.double() - w).abs().max() <= bound
        if dtype != "fp32":
            assert torch.equal(p.detach(), held.to(p.dtype))
    if max_norm is not None:
        norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in grads))
        assert float(opt.grad_norm) == pytest.approx(norm, rel=8 * EPS32)


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("offset", [0, 5])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_8_bit_moments(dtype, offset, max_norm):
    params = parameters(SIZES, TYPES[dtype], offset)
    params[4].grad.zero_()  # a tensor without gradient entries: no history, no blow-up
    params[5].grad[:300] = 0
    want = Formula(params, 3e-3, (0.9, 0.99), 1e-8, 0.1, max_norm)
    opt = optim.AdamW(params, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.1, max_norm=max_norm, state_bits=8)
    for _ in range(3):
        for i, p in enumerate(params):  # the formula starts from the values the codes stand for
            want.m[i] = decoded(opt.state[p], "exp_avg")
            want.v[i] = decoded(opt.state[p], "exp_avg_sq_root") ** 2
            want.p[i] = (opt.state[p]["master"] if dtype != "fp32" else p.detach()).double().clone()
        want.step([p.grad for p in params])
        opt.step()
        for i, p in enumerate(params):
            if not p.numel():
                continue
            state = opt.state[p]
            check_codes(state, "exp_avg", want.m[i])
            check_codes(state, "exp_avg_sq_root", want.v[i].sqrt())
            held = state["master"] if dtype != "fp32" else p.detach()
            assert (held.double() - want.p[i]).abs().max() <= 20 * EPS32 * (want.p[i].abs().max() + 3e-3 * 10)
            if dtype != "fp32":
                assert torch.equal(p.detach(), held.to(p.dtype))


@pytest.mark.gpu
def test_a_magnitude_too_small_for_a_scale_is_held_as_zero():
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.full((300,), 1e-37, device="cuda")
    opt = optim.AdamW([p], lr=1e-3, state_bits=8)
    opt.step()
    assert torch.isfinite(p).all()
    assert not opt.state[p]["exp_avg"].float().any() and not opt.state[p]["exp_avg_sq_root"].float().any()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_norm_that_is_not_finite_skips_the_step(bits, bad):
    params = parameters([(300,), (5, 77)], torch.float32)
    opt = optim.AdamW(params, max_norm=1.0, state_bits=bits)
    opt.step()
    before = [p.detach().clone() for p in params] + [v.clone().view(torch.uint8) for v in opt.flat.values()]
    params[1].grad[2, 3] = bad
    opt.step()
    after = [p.detach() for p in params] + [v.view(torch.uint8) for v in opt.flat.values()]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    assert int(opt.steps) == 1 and not math.isfinite(float(opt.grad_norm))
    params[1].grad[2, 3] = 0.1
    opt.step()
    assert int(opt.steps) == 2 and not torch.equal(before[0], params[0].detach())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("count", [3, 65, 700])
def test_many_tensors_match_one_at_a_time(count, bits):
    """The tables of few and many tensors and several launches: every tensor steps as it does alone."""

    sizes = [((i * 37) % 611 + 1,) for i in range(count)]
    together = parameters(sizes, torch.float32)
    alone = parameters(sizes, torch.float32)
    for i in range(0, count, 5):
        together[i].grad = None
        alone[i].grad = None
    both = optim.AdamW(together, lr=1e-2, state_bits=bits)
    both.step()
    for p, q in zip(alone, together):
        optim.AdamW([p], lr=1e-2, state_bits=bits).step()
        assert torch.equal(p, q)
    clipped = parameters(sizes, torch.float32)
    opt = optim.AdamW(clipped, max_norm=1.0, state_bits=bits)
    opt.step()
    norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in clipped))
    assert float(opt.grad_norm) == pytest.approx(norm, rel=8 * EPS32)


@pytest.mark.gpu
def test_groups_have_their_own_hyperparameters_and_schedulers_drive_them():
    params = parameters([(500,), (400,)], torch.float32)
    want = [Formula([params[0]], 1e-2, (0.9, 0.999), 1e-8, 0.1, None), Formula([params[1]], 2e-3, (0.8, 0.95), 1e-6, 0.0, None)]
    opt = optim.AdamW([dict(params=[params[0]], lr=1e-2, weight_decay=0.1),
                       dict(params=[params[1]], lr=2e-3, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.0)])
    halve = torch.optim.lr_scheduler.StepLR(opt, step_size=1, gamma=0.5)
    for _ in range(2):
        opt.step()
        for w, p in zip(want, params):
            w.step([p.grad])
            w.lr *= 0.5
        halve.step()
    for w, p in zip(want, params):
        assert (p.detach().double() - w.p[0]).abs().max() <= 2 * 20 * EPS32 * (w.p[0].abs().max() + 0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_state_round_trip_continues_the_run(bits):
    a = parameters([(300,), (9, 33)], torch.bfloat16)
    opt = optim.AdamW(a, lr=1e-2, max_norm=1.0, state_bits=bits)
    opt.step()
    b = parameters([(300,), (9, 33)], torch.bfloat16)
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    other = optim.AdamW(b, lr=1.0, max_norm=1.0, state_bits=bits)
    other.load_state_dict(opt.state_dict())
    opt.step()
    other.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert int(other.steps) == 2 and other.param_groups[0]["lr"] == 1e-2
    with pytest.raises(ValueError, match="bits"):
        optim.AdamW(b, state_bits=40 - bits).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError, match="shapes"):
        optim.AdamW(parameters([(300,), (9, 34)], torch.bfloat16), state_bits=bits).load_state_dict(opt.state_dict())


@pytest.mark.gpu
def test_the_step_runs_on_the_current_stream_and_in_a_graph():
    params = parameters([(4000,)], torch.float32)
    opt = optim.AdamW(params, lr=1e-2, max_norm=1.0)
    twin = parameters([(4000,)], torch.float32)
    eager = optim.AdamW(twin, lr=1e-2, max_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        eager.step()
    assert torch.equal(params[0], twin[0]) and int(opt.steps) == 4


@pytest.mark.gpu
def test_refusals_on_the_device():
    p = torch.nn.Parameter(torch.ones(8, 8, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        optim.AdamW([torch.nn.Parameter(torch.ones(8, 8, device="cuda").t())])
    with pytest.raises(ValueError, match="one dtype"):
        optim.AdamW([p, torch.nn.Parameter(torch.ones(3, device="cuda", dtype=torch.bfloat16))])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        optim.AdamW([torch.nn.Parameter(torch.ones(3, device="cuda", dtype=torch.float64))])
    opt = optim.AdamW([p])
    with pytest.raises(ValueError, match="constructor"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.ones(2, device="cuda"))]))
    p.grad = torch.ones(8, 8, device="cuda").t()
    with pytest.raises(ValueError, match="dense and contiguous"):
        opt.step()
    p.data = torch.ones(4, device="cuda")
    p.grad = torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="changed its size"):
        opt.step()


def test_refusals_without_a_gpu():
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([p])
    with pytest.raises(ValueError, match="state_bits"):
        optim.AdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="max_norm"):
        optim.AdamW([p], max_norm=0.0)
    with pytest.raises(ValueError, match="betas"):
        optim.AdamW([p], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="negative"):
        optim.AdamW([p], lr=-1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_a_backward_pass_through_stepped_weights_is_refused(bits):
    """As with torch's optimizers: a graph from before the step has saved the weights, which the step has changed."""

    weight, still = (torch.nn.Parameter(torch.randn(40, 24, device="cuda")) for _ in range(2))
    x = torch.randn(50, 24, device="cuda", requires_grad=True)
    opt = optim.AdamW([weight, still], state_bits=bits)
    loss = dense.linear(x, weight).square().sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert still._version == 0  # no gradient: the step left it as it was
    loss = dense.linear(x, weight).square().sum()
    loss.backward()
    opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("size", [1e-18, 3e-19])
def test_a_second_moment_below_the_normal_range_counts_without_eps(size, bits):
    """v = 1e-3 g^2 is subnormal here, within 2^-150 of its value (1e-5 of it at least); the first step moves by lr all the same."""

    p = torch.nn.Parameter(torch.zeros(700, device="cuda"))
    sign = torch.where(torch.arange(700, device="cuda") % 3 == 0, -1.0, 1.0)
    p.grad = size * sign
    opt = optim.AdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=bits)
    opt.step()
    assert (p.detach() + 1e-2 * sign).abs().max() <= 1e-2 * 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("size", [1e-20, 1e-22, 1e-24, 1e-30, 1e-38, 0.0])
def test_without_eps_a_vanishing_gradient_moves_a_weight_by_a_few_learning_rates_at_most(size, bits):
    """Adam's update is at most about (1 - b1) / sqrt(1 - b2) learning rates, 3.2, before the bias correction by 1 / (1 - b1)
    of a first step, 32 in all; a v that float32 cannot hold must not make more of it."""

    p = torch.nn.Parameter(torch.zeros(700, device="cuda"))
    p.grad = torch.full_like(p, size)
    opt = optim.AdamW([p], lr=1e-2, eps=0.0, weight_decay=0.0, state_bits=bits)
    for _ in range(3):
        opt.step()
        assert torch.isfinite(p).all() and p.detach().abs().max() <= 3 * 33 * 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("count", [1, 16, 17, 32, 33, 70, 700])
def test_any_number_of_groups(count, max_norm):
    """Learning rates by layer: each group's own hyperparameters at every step, past one launch's share of them."""

    params = parameters([(40 + i % 7,) for i in range(count)], torch.float32)
    groups = [dict(params=[p], lr=1e-3 * (1 + i % 40), betas=(0.8 + 0.001 * (i % 90), 0.99), eps=1e-8, weight_decay=0.01 * (i % 3))
              for i, p in enumerate(params)]
    clip = 1.0
    if max_norm is not None:
        clip = min(1.0, max_norm / (math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in params)) + 1e-6))
    want = [Formula([p], g["lr"], g["betas"], g["eps"], g["weight_decay"], None) for p, g in zip(params, groups)]
    opt = optim.AdamW(groups, max_norm=max_norm)
    for _ in range(2):
        opt.step()
        for w, p in zip(want, params):
            w.step([p.grad.double() * clip])
    assert int(opt.steps) == 2
    for w, p in zip(want, params):
        assert (p.detach().double() - w.p[0]).abs().max() <= 2 * 20 * EPS32 * (w.p[0].abs().max() + 0.4)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [8, 32])
def test_gradients_whose_squares_pass_the_largest_float_are_clipped(bits, dtype, offset):
    """Entries of 1e25: the norm is finite, so the step is taken, with gradients of 1e25 times the clip's 1e-27."""

    params = parameters([(20000,), (77,)], TYPES[dtype], offset)
    for p in params:
        p.grad.mul_(1e27)
    norm = math.sqrt(sum(float((p.grad.double() ** 2).sum()) for p in params))
    opt = optim.AdamW(params, lr=1e-2, weight_decay=0.0, max_norm=1.0, state_bits=bits)
    before = [p.detach().float().clone() for p in params]
    opt.step()
    assert int(opt.steps) == 1 and float(opt.grad_norm) == pytest.approx(norm, rel=8 * EPS32)
    for p, old in zip(params, before):
        held = (opt.state[p]["master"] if dtype != "fp32" else p.detach()).double()
        g = p.grad.double() / norm
        want = old.double() - 1e-2 * g / (g.abs() + 1e-8)
        assert (held - want).abs().max() <= 1e-2 * 1e-4 + 20 * EPS32


@pytest.mark.gpu
def test_a_norm_past_the_largest_float_skips_the_step():
    params = parameters([(300,)], torch.float32)
    params[0].grad.fill_(3e38)
    before = params[0].detach().clone()
    opt = optim.AdamW(params, max_norm=1.0)
    opt.step()
    assert int(opt.steps) == 0 and float(opt.grad_norm) == math.inf and torch.equal(params[0].detach(), before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_weights_loaded_after_the_optimizer_was_made_are_the_ones_that_step(dtype):
    """A checkpoint loaded into the model, an edit in place, another tensor under the parameter: 16-bit masters follow."""

    kind = TYPES[dtype]
    params = parameters([(300,), (9, 33)], kind)
    opt = optim.AdamW(params, lr=1e-3)
    opt.step()
    fresh = parameters([(300,), (9, 33)], kind, seed=5)
    model = torch.nn.ParameterList(params)
    model.load_state_dict(torch.nn.ParameterList(fresh).state_dict())
    for edit in (None, lambda p: p.mul_(0.5), lambda p: p.add_(1.0)):
        if edit is not None:
            with torch.no_grad():
                edit(params[1])
        before = [p.detach().double() for p in params]
        opt.step()
        for p, old in zip(params, before):
            moved = (p.detach().double() - old).abs()
            assert moved.max() <= 4e-3 + 2.0 ** -7 * old.abs().max() and (dtype != "fp32" or moved.max() > 0)
    params[0].data = torch.full_like(params[0].data, 3.0)
    opt.step()
    assert (params[0].detach().double() - 3.0).abs().max() <= 4e-3 + 2.0 ** -7 * 3


@pytest.mark.gpu
@pytest.mark.parametrize("model_first", [False, True])
def test_masters_keep_their_low_bits_when_a_checkpoint_is_loaded(model_first):
    params = parameters([(700,)], torch.bfloat16)
    opt = optim.AdamW(params, lr=1e-4, max_norm=1.0)
    for _ in range(3):
        opt.step()
    others = parameters([(700,)], torch.bfloat16, seed=7)
    others[0].grad.copy_(params[0].grad)
    again = optim.AdamW(others, lr=1e-4, max_norm=1.0)
    loads = [lambda: again.load_state_dict(opt.state_dict()),
             lambda: torch.nn.ParameterList(others).load_state_dict(torch.nn.ParameterList(params).state_dict())]
    for load in reversed(loads) if model_first else loads:
        load()
    for _ in range(3):
        opt.step()
        again.step()
    assert torch.equal(opt.flat["master"], again.flat["master"]) and torch.equal(params[0], others[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_8_bit_first_moment_is_the_formulas_own_in_fp32(dtype):
    """b1 m + (1 - b1) g with every operation rounded to fp32, over the block's largest magnitude: the same scales and the same
    codes, step after step. (A product fused with the sum gives neighbouring codes at an edge, and a scale that follows
    such a code is off by a code's step later.)"""

    n = 1 << 21
    params = parameters([(n,)], TYPES[dtype])
    opt = optim.AdamW(params, lr=1e-3, betas=(0.9, 0.999), state_bits=8)
    codes = torch.zeros(n // optim.BLOCK, optim.BLOCK, device="cuda")
    scale = torch.zeros(n // optim.BLOCK, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    for _ in range(4):
        params[0].grad.copy_(1e-2 * torch.randn(n, generator=g, device="cuda"))
        grad = params[0].grad.float().view(-1, optim.BLOCK)
        first = 0.9 * (codes * (scale * torch.tensor(1.0 / 448.0, device="cuda"))[:, None]) + (1 - 0.9) * grad
        scale = first.abs().amax(dim=1)
        codes = (first * (448.0 * (1.0 / scale))[:, None]).to(torch.float8_e4m3fn).float()
        opt.step()
        assert torch.equal(opt.flat["exp_avg_scale"], scale)
        assert torch.equal(opt.flat["exp_avg"].float().view(-1, optim.BLOCK), codes)
