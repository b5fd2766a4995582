"""dense.linear against its formula in 64 bits: types, activations, odd sizes from one entry to past a tile, strides,
missing biases and residuals, empty extents, gradients (the formula's and differences), and its refusals.

Tolerances. A product's sum of K fp32 terms is within 2^-24 sqrt-to-linear of sum |a||b|: 2^-21 of it covers any order of
addition of exact products up to these depths (the float32 operands' three bfloat16 parts leave 2^-23 of it). The activation's
derivative is at most 1.13, its curvature at most 1.1. 16-bit results round once (2^-8, 2^-11); the sum kept for the
backward pass and the gradient entering its products round once more each."""

from __future__ import annotations

import math
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

import pytest
import torch

from card_playing_gym_b200 import dense
from card_playing_gym_b200 import _native as nat

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ACC = 2.0 ** -21
LEAST = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}

ACT = {"none": lambda z: z * 1.0, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def case(m, k, n, dtype, bias=True, residual=True):
    return dict(x=normal((m, k), dtype, 1), weight=normal((n, k), dtype, 2, 1 / math.sqrt(max(k, 1))),
                bias=normal((n,), dtype, 3, 0.5) if bias else None,
                residual=normal((m, n), dtype, 4) if residual else None, dy=normal((m, n), dtype, 5))


def check(data, activation, backward=True):
    dtype = data["x"].dtype
    leaves = {name: data[name].detach().requires_grad_(backward) for name in ("x", "weight", "bias", "residual")
              if data[name] is not None}
    y = dense.linear(leaves["x"], leaves["weight"], leaves.get("bias"), leaves.get("residual"), activation=activation)
    wide = {name: value.detach().double().requires_grad_(backward) for name, value in leaves.items()}
    pre = wide["x"] @ wide["weight"].t()
    reach = wide["x"].abs().detach() @ wide["weight"].abs().t().detach()
    if "bias" in wide:
        pre = pre + wide["bias"]
        reach = reach + wide["bias"].abs().detach()
    want = ACT[activation](pre)
    if "residual" in wide:
        want = want + wide["residual"]
    half, least = HALF_STEP[dtype], LEAST[dtype]
    assert y.dtype == dtype and y.shape == want.shape
    near = 1.2 * ACC * reach + 2.0 ** -20 * (pre.detach().abs() + want.detach().abs())
    assert ((y.double() - want).abs() <= near + (half + ACC) * want.abs() + least).all()
    if not backward:
        return y
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), data["dy"])))
    expected = dict(zip(wide, torch.autograd.grad(want, list(wide.values()), data["dy"].double())))
    pre, dy = pre.detach(), data["dy"].double()
    dpre_bound = dy.abs() * 1.2  # |dpre|, and what a rounding of pre and of dpre moves it by
    off = dy.abs() * (1.2 * half * (activation != "none") + 1.1 * (half * pre.abs() + 1.2 * ACC * reach) * (activation not in ("none", "relu"))
                      + 2.0 ** -20)
    if activation == "relu":  # the kink: a sum within its error of zero may fall on either side
        off = off + dy.abs() * (pre.abs() <= 1.2 * ACC * reach + least)
    bounds = {"x": off @ wide["weight"].detach().abs() + ACC * (dpre_bound @ wide["weight"].detach().abs()),
              "weight": off.t() @ wide["x"].detach().abs() + ACC * (dpre_bound.t() @ wide["x"].detach().abs()),
              "bias": off.sum(0) + ACC * dpre_bound.sum(0), "residual": torch.zeros_like(dy)}
    for name, grad in grads.items():
        assert grad.dtype == dtype
        bound = bounds[name] + (half + ACC) * expected[name].abs() + least
        assert ((grad.double() - expected[name]).abs() <= bound).all(), name
    return y


SHAPES = [(1, 1, 1), (1, 240, 720), (2, 7, 3), (5, 64, 64), (17, 33, 129), (64, 240, 720), (129, 720, 240), (127, 65, 257),
          (300, 1001, 515), (257, 128, 1), (1000, 1, 300), (515, 2050, 130), (2048, 256, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("activation", list(ACT))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(shape, dtype, activation):
    check(case(*shape, TYPES[dtype]), activation)
    assert nat.fault_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 7, 8, 9, 16, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("inner,outer", [(240, 720), (4096, 1000), (77, 33), (3000, 4097)])
def test_few_tokens(rows, dtype, inner, outer):
    with torch.no_grad():
        check(case(rows, inner, outer, TYPES[dtype]), "gelu", backward=False)
        check(case(rows, inner, outer, TYPES[dtype], bias=False, residual=False), "none", backward=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_parts_may_be_missing(dtype, bias, residual):
    check(case(200, 96, 160, TYPES[dtype], bias, residual), "silu")
    check(case(200, 96, 160, TYPES[dtype], bias, residual), "none")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(4000, 24, 40), (40000, 32, 16), (20000, 240, 720)])
def test_tall_batches_join_their_slices(dtype, shape):
    check(case(*shape, TYPES[dtype]), "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_strided_and_unaligned_inputs(dtype, pad):
    """Rows longer than the matrix, matrices that start inside a row, transposed and expanded ones."""

    data = case(150, 72, 136, TYPES[dtype])
    for name in ("x", "weight", "residual", "dy"):
        m, k = data[name].shape
        store = torch.full((m, k + 2 * pad), math.nan, dtype=data[name].dtype, device="cuda")
        store[:, pad:pad + k] = data[name]
        data[name] = store[:, pad:pad + k]
    store = torch.zeros(136 + pad, dtype=TYPES[dtype], device="cuda")
    store[pad:] = data["bias"]
    data["bias"] = store[pad:]
    check(data, "gelu")
    data = case(150, 72, 136, TYPES[dtype])
    for name in ("x", "weight", "residual", "dy"):
        data[name] = data[name].t().contiguous().t()
    check(data, "gelu")
    data["dy"] = data["dy"][:1].expand(150, 136)
    data["x"] = data["x"][:1].expand(150, 72)
    check(data, "silu")


@pytest.mark.gpu
def test_leading_dimensions():
    x, weight, bias = normal((3, 5, 48), torch.bfloat16, 1), normal((32, 48), torch.bfloat16, 2), normal((32,), torch.bfloat16, 3)
    y = dense.linear(x, weight, bias, normal((3, 5, 32), torch.bfloat16, 4), activation="relu")
    flat = dense.linear(x.view(15, 48), weight, bias, normal((3, 5, 32), torch.bfloat16, 4).view(15, 32), activation="relu")
    assert y.shape == (3, 5, 32) and torch.equal(y.view(15, 32), flat)
    one = dense.linear(x[0, 0], weight, bias, activation="relu")
    assert one.shape == (32,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(0, 16, 8), (4, 0, 8), (4, 16, 0)])
def test_empty_extents(dtype, shape):
    """No rows: nothing; no depth: the epilogue of zero; no outputs: zero gradients."""

    data = case(*shape, TYPES[dtype])
    leaves = {k: data[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual")}
    y = dense.linear(*leaves.values(), activation="gelu")
    grads = torch.autograd.grad(y, list(leaves.values()), data["dy"])
    assert all(g.shape == leaf.shape for g, leaf in zip(grads, leaves.values()))
    if shape[1] == 0:
        want = torch.nn.functional.gelu(data["bias"].double()) + data["residual"].double()
        assert ((y.double() - want).abs() <= 2 * HALF_STEP[TYPES[dtype]] * (want.abs() + 1)).all()
    assert not grads[0].any() and not grads[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinities_and_nan_stay_in_their_rows(dtype, activation):
    data = case(140, 64, 96, TYPES[dtype], residual=False)
    want = dense.linear(data["x"], data["weight"], data["bias"], activation=activation)
    data["x"][7, 3] = math.nan
    data["x"][9] = 0.0
    data["x"][9, 5] = math.inf
    got = dense.linear(data["x"], data["weight"], data["bias"], activation=activation)
    assert torch.isnan(got[7]).all()
    assert not torch.isfinite(got[9]).all() or activation != "none"
    rest = [i for i in range(140) if i not in (7, 9)]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("activation", list(ACT))
def test_the_gradient_against_differences(activation):
    """Central differences of sum(dy * y) in fp32 at h = 2^-5: rounding 2^-22 |L| / h, curvature h^2."""

    data = case(6, 9, 5, torch.float32)
    if activation == "relu":  # away from the kink
        data["bias"] = data["bias"].sign() * 4
    leaves = {k: data[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual")}
    grads = dict(zip(leaves, torch.autograd.grad(dense.linear(*leaves.values(), activation=activation), list(leaves.values()),
                                                 data["dy"])))

    def value(inputs):
        with torch.no_grad():
            return float((dense.linear(*inputs.values(), activation=activation).double() * data["dy"].double()).sum())

    h = 2.0 ** -5
    for name, at in (("x", (2, 3)), ("weight", (4, 8)), ("bias", (1,)), ("residual", (5, 2))):
        ends = []
        for sign in (1, -1):
            moved = {k: v.detach().clone() for k, v in leaves.items()}
            moved[name][at] += sign * h
            ends.append(value(moved))
        assert (ends[0] - ends[1]) / (2 * h) == pytest.approx(float(grads[name][at]), abs=30 * 2.0 ** -22 / h + 30 * h * h)


@pytest.mark.gpu
def test_only_what_needs_a_gradient_gets_one():
    data = case(64, 48, 32, torch.bfloat16)
    full = {k: data[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual")}
    every = torch.autograd.grad(dense.linear(*full.values(), activation="gelu"), list(full.values()), data["dy"])
    for name, want in zip(full, every):
        some = {k: data[k].detach().requires_grad_(k == name) for k in full}
        (got,) = torch.autograd.grad(dense.linear(*some.values(), activation="gelu"), [some[name]], data["dy"])
        assert torch.equal(got, want), name


@pytest.mark.gpu
def test_streams_and_repeats_agree():
    data = case(500, 240, 720, torch.bfloat16)
    want = check(data, "gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = check(data, "gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w = normal((4, 8), torch.float32, 1), normal((6, 8), torch.float32, 2)
    with pytest.raises(ValueError, match="weight must be"):
        dense.linear(x, w.bfloat16())
    with pytest.raises(ValueError, match="bias must be"):
        dense.linear(x, w, normal((5,), torch.float32, 3))
    with pytest.raises(ValueError, match="residual must be"):
        dense.linear(x, w, None, normal((4, 5), torch.float32, 3))


def test_refusals_without_a_gpu():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="CUDA"):
        dense.linear(x, w)
    with pytest.raises(ValueError, match="activation"):
        dense.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="does not multiply"):
        dense.linear(x, torch.zeros(6, 7))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        dense.linear(x.double(), w.double())
    with pytest.raises(nat.NativeError, match="activation"):
        nat.call("cg_linear_forward", None, 8, None, 8, None, None, 0, 0, 4, 8, 6, 9, None, None, None, 0, None)
    with pytest.raises(nat.NativeError, match="shape"):
        nat.query("cg_linear_workspace_bytes", None, 8, None, 8, None, 0, 0, -1, 8, 8, 0, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(4800, 520, 1000), (4800, 520, 500), (2000, 300, 1000), (5000, 100, 1001), (700, 720, 240)])
def test_rounds_of_tiles_that_do_not_fill_the_chip(shape, dtype):
    check(case(*shape, TYPES[dtype]), "gelu")
    assert nat.fault_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("outer", [36, 40, 68, 72, 100, 160])
def test_results_whose_rows_start_off_a_sector(outer, dtype):
    data = case(300, 64, outer, TYPES[dtype])
    check(data, "silu")
    wide = torch.zeros((300, outer + 12), dtype=TYPES[dtype], device="cuda")
    for offset in (1, 4, 8):
        wide[:, offset:offset + outer] = data["residual"]
        check({**data, "residual": wide[:, offset:offset + outer]}, "relu")


def test_every_kernel_with_large_shared_memory_is_set_up_on_each_device():
    """The permission for more than 48 KB of dynamic shared memory belongs to a device: a host function that asks for it
    keeps its record of having asked by device."""

    for path in sorted((Path(dense.__file__).parent / "csrc").glob("*.cu")):
        lines = path.read_text().splitlines()
        for at, line in enumerate(lines):
            if "cudaFuncSetAttribute(" in line:
                assert any("[device & 63]" in before for before in lines[at - 4:at]), f"{path.name}:{at + 1}"


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_second_device_of_the_process(dtype):
    data = case(300, 64, 96, TYPES[dtype])
    want = dense.linear(data["x"], data["weight"], data["bias"], data["residual"], activation="gelu")
    other = {name: value.to("cuda:1") for name, value in data.items()}
    got = dense.linear(other["x"], other["weight"], other["bias"], other["residual"], activation="gelu")
    assert torch.equal(got.to("cuda:0"), want)


def same_kind(got, want):
    """Both NaN, both an infinity of one sign, or both finite."""

    return (torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isposinf(got), torch.isposinf(want))
            and torch.equal(torch.isneginf(got), torch.isneginf(want)))


@pytest.mark.gpu
@pytest.mark.parametrize("activation", list(ACT))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,inner,outer", [(20, 64, 96), (32, 300, 100), (33, 64, 96), (140, 64, 96), (140, 700, 131),
                                              (64, 4000, 72)])
def test_an_infinity_is_one_whatever_the_row_count(rows, inner, outer, dtype, activation):
    """One infinity in a row makes every sum of it an infinity of the weight's sign, two of them a NaN where the signs
    differ, in the formula as in the layer."""

    data = case(rows, inner, outer, TYPES[dtype], residual=False)
    data["x"][7, 5] = math.inf
    data["x"][9] = 0.0
    data["x"][9, 5] = -math.inf
    data["x"][11, 3], data["x"][11, inner - 1] = math.inf, -math.inf
    data["weight"][4, 2] = math.inf
    data["x"][13, 2] = 0.0
    got = dense.linear(data["x"], data["weight"], data["bias"], activation=activation)
    want = ACT[activation](data["x"].double() @ data["weight"].double().t() + data["bias"].double())
    assert torch.isinf(want[7]).sum() >= outer // 4 and torch.isnan(want[13, 4])
    assert same_kind(got.double(), want)
    assert nat.fault_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [20, 140, 3000])
def test_an_infinity_in_the_backward_pass(rows, dtype):
    data = case(rows, 72, 100, TYPES[dtype], residual=False)
    data["dy"][3, 8] = math.inf
    data["x"][6, 2] = -math.inf
    leaves = {k: data[k].detach().requires_grad_() for k in ("x", "weight", "bias")}
    grads = torch.autograd.grad(dense.linear(*leaves.values()), list(leaves.values()), data["dy"])
    dy = data["dy"].double()
    for got, want in zip(grads, (dy @ data["weight"].double(), dy.t() @ data["x"].double(), dy.sum(0))):
        assert torch.isinf(want).any() and same_kind(got.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 24, 32, 33, 4096])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_gelu_left_of_zero_is_rounded_once(dtype, rows):
    """Products by one are exact, so a 16-bit GELU is its value's nearest one, but for 3% of the spacing there (1e-5 of the
    value is 2% of float16's), down to z = -13; the slope too, with 2^-20 where its terms cancel. Few rows or many."""

    kind = TYPES[dtype]
    x = torch.linspace(-13, 4, 8192, device="cuda").to(kind).view(-1, 1)[:: 8192 // rows][:rows] if rows > 1 else \
        torch.full((1, 1), -4.0, dtype=kind, device="cuda")
    x = x.contiguous().requires_grad_()
    one = torch.ones((1, 1), dtype=kind, device="cuda")
    y = dense.linear(x, one, activation="gelu")
    (slope,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    cumulative = 0.5 * torch.special.erfc(-z / math.sqrt(2))
    least = torch.finfo(kind).smallest_normal
    for got, want, extra in ((y, z * cumulative, 0.0),
                             (slope, cumulative + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 2.0 ** -20)):
        spacing = 2.0 ** torch.floor(torch.log2(want.abs().clamp(min=least))) * 2 * HALF_STEP[kind]
        assert ((got.double() - want).abs() <= 0.53 * spacing + extra).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(2, 3, 0), (0,), (0, 4, 0), (2, 0, 5), (3, 1, 0)])
def test_leading_dimensions_of_empty_extents(shape, dtype):
    kind = TYPES[dtype]
    x = torch.zeros(shape, dtype=kind, device="cuda", requires_grad=True)
    weight = torch.ones((6, shape[-1]), dtype=kind, device="cuda", requires_grad=True)
    bias = normal((6,), kind, 3).requires_grad_()
    residual = normal((*shape[:-1], 6), kind, 4).requires_grad_()
    y = dense.linear(x, weight, bias, residual, activation="relu")
    want = torch.relu(bias.double()) + residual.double()
    assert y.shape == (*shape[:-1], 6)
    assert ((y.double() - want).abs() <= 2 * HALF_STEP[kind] * (want.abs() + 1)).all()
    grads = torch.autograd.grad(y, (x, weight, bias, residual), torch.ones_like(y))
    rows = math.prod(shape[:-1])
    assert [g.shape for g in grads] == [x.shape, weight.shape, bias.shape, residual.shape]
    assert torch.equal(grads[2].double(), rows * (bias > 0).double()) and torch.equal(grads[3], torch.ones_like(residual))


@pytest.mark.gpu
def test_a_product_of_no_depth_past_32_bits_of_entries():
    """2^33 outputs (17 GB), all of them the bias."""

    x = torch.zeros((1 << 20, 0), dtype=torch.bfloat16, device="cuda")
    bias = normal((8192,), torch.bfloat16, 1)
    torch.full((1 << 33,), math.nan, dtype=torch.bfloat16, device="cuda")  # what the output's memory may hold
    y = dense.linear(x, torch.zeros((8192, 0), dtype=torch.bfloat16, device="cuda"), bias)
    assert all(torch.equal(piece, bias.expand_as(piece)) for piece in y.split(1 << 16))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 20, 32, 33, 5000])
def test_float32_silu_in_full_precision(rows):
    """Products by one are exact. An exponential, a sum and a quotient of at most two units in the last place each: 2^-21 of
    the value, and for the slope of its larger term, g and z g (1 - g)."""

    x = torch.linspace(-80, 20, 5000, device="cuda")[:: 5000 // rows][:rows].reshape(-1, 1).requires_grad_()
    one = torch.ones((1, 1), device="cuda")
    y = dense.linear(x, one, activation="silu")
    (slope,) = torch.autograd.grad(y, x, torch.ones_like(y))
    z = x.detach().double()
    gate = 1 / (1 + torch.exp(-z))
    assert ((y.double() - z * gate).abs() <= 2.0 ** -21 * (z * gate).abs()).all()
    assert ((slope.double() - gate * (1 + z * (1 - gate))).abs() <= 2.0 ** -21 * gate * (1 + z.abs())).all()


@pytest.mark.gpu
def test_a_threads_first_cuda_call_may_be_a_product():
    """Memory from torch's cache leaves a new thread without a current context until its first launch, and a 16-bit layer
    begins with a tensor map, a driver call that needs one."""

    data = case(64, 64, 64, torch.bfloat16, bias=False, residual=False)
    with torch.no_grad():
        want = dense.linear(data["x"], data["weight"])
        torch.cuda.synchronize()
        with ThreadPoolExecutor(1) as pool:
            got = pool.submit(lambda: dense.linear(data["x"], data["weight"])).result()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_a_programs_first_backward_pass_may_be_a_product():
    """The autograd worker's first call, with neither a bias nor an activation to launch anything before it."""

    code = ("import torch; from card_playing_gym_b200 import dense\n"
            "x, w, dy = (torch.ones(64, 64, dtype=torch.bfloat16, device='cuda') for _ in range(3))\n"
            "w.requires_grad_()\n"
            "torch.autograd.grad(dense.linear(x, w), w, dy); grad, = torch.autograd.grad(dense.linear(x, w), w, dy)\n"
            "assert (grad == 64).all()")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(dense.__file__).parents[1], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("inner,outer", [(2304, 2304), (300, 200)])
def test_the_weight_gradient_of_a_long_batch(inner, outer, dtype):
    """The tensor cores cut a running sum toward zero, by some 1.7e-7 of it every 16 rows where its terms have one sign, which
    moves the whole gradient: over 262,144 rows in one sum by 1.5e-3. Sums of 16,384 rows (float16) and 65,536 (bfloat16)
    leave 9e-5 and 3.9e-4 of it; the bounds are 2^-13 and 2^-11. Factors of 1 to 2 a column spread the entries over a
    binade, so that their own rounding averages out."""

    rows, kind = 1 << 18, TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(3)
    uniform = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    x = (uniform(rows, inner).add_(0.5) * torch.exp2(uniform(inner))).to(kind)
    dy = (uniform(rows, outer).add_(0.5) * torch.exp2(uniform(outer) - 6)).to(kind)
    weight = torch.zeros((outer, inner), dtype=kind, device="cuda", requires_grad=True)
    (got,) = torch.autograd.grad(dense.linear(x, weight), weight, dy)
    some = list(range(0, outer, outer // 8))
    want = torch.stack([(dy[:, j:j + 1].double() * x.double()).sum(0) for j in some])
    off = got[some].double() / want - 1
    shift = 2.0 ** -13 if dtype == "fp16" else 2.0 ** -11
    assert abs(float(off.mean())) <= shift + HALF_STEP[kind] / off.numel() ** 0.5
    assert float(off.abs().max()) <= HALF_STEP[kind] + 1.5 * shift


def test_float32_tokens_go_where_they_are_faster():
    """Up to 24 tokens the weights are read in place; more of them through a large float32 layer are packed for the tensor
    cores, which takes a workspace."""

    def workspace(rows, inner, outer, dtype):
        return nat.query("cg_linear_workspace_bytes", None, inner, None, inner, None, 0, nat.DTYPE_CODES[dtype], rows, inner,
                         outer, 0, 0)

    for rows in (1, 24):
        assert workspace(rows, 8192, 4096, torch.float32) == 0
    assert workspace(25, 8192, 4096, torch.float32) > 0 and workspace(32, 1 << 16, 128, torch.float32) > 0
    assert workspace(32, 512, 4096, torch.float32) == 0 and workspace(33, 512, 4096, torch.float32) > 0
    assert workspace(32, 8192, 4096, torch.bfloat16) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [24, 25, 32, 33])
def test_many_float32_tokens_through_a_large_layer(rows):
    check(case(rows, 2048, 4100, torch.float32), "gelu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("activation", ["relu", "gelu", "silu"])
def test_slopes_at_infinite_sums_are_their_limits(activation, dtype):
    """A float16 sum past 65,504 is kept as an infinity for the backward pass: its slope is 1 (or 0 on the left), not a NaN."""

    kind = TYPES[dtype]
    big = math.inf if dtype != "fp16" else 60000.0
    x = torch.full((40, 1), big, dtype=kind, device="cuda")
    x[20:] = -big
    x.requires_grad_()
    two = torch.full((1, 1), 2.0, dtype=kind, device="cuda")
    bias = torch.zeros(1, dtype=kind, device="cuda", requires_grad=True)
    y = dense.linear(x, two, bias, activation=activation)
    dx, dbias = torch.autograd.grad(y, (x, bias), torch.ones_like(y))
    assert torch.equal(dx[:20], torch.full_like(dx[:20], 2.0)) and not dx[20:].any() and float(dbias) == 20.0
