"""A linear layer with its bias, activation and residual in the product's epilogue, differentiable.

``linear(x, weight, bias, residual, activation=...)`` is ``activation(x @ weight.T + bias) + residual`` in one product
(csrc/dense.cu), in float32, float16 or bfloat16 with fp32 sums: the shapes of the reference trunk's MLP and projections
(cardgym/nn/trunk.py:124-157) in training, where gradients flow to every input, and for single tokens.
"""

from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import _native as nat

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def _unit_rows(matrix: torch.Tensor) -> torch.Tensor:
    """The matrix with adjacent row entries and rows that do not overlap (a copy only where it has neither)."""

    if matrix.is_contiguous():
        return matrix
    if matrix.shape[1] > 1 and matrix.stride(1) != 1 or matrix.shape[0] > 1 and matrix.stride(0) < matrix.shape[1]:
        return matrix.contiguous()
    return matrix


def _row_stride(matrix: torch.Tensor) -> int:
    return max(matrix.stride(0), matrix.shape[1]) if matrix.shape[0] > 1 else matrix.shape[1]


@lru_cache(maxsize=4096)
def _workspace_bytes(*layout: int) -> int:
    return nat.query("cg_linear_workspace_bytes", *layout)


def _workspace(x, weight, dy, activation: int) -> torch.Tensor | None:
    # Of the addresses only their places within sixteen bytes count.
    need = _workspace_bytes(nat.ptr(x) & 15, _row_stride(x), nat.ptr(weight) & 15, _row_stride(weight),
                            0 if dy is None else nat.ptr(dy) & 15, 0 if dy is None else _row_stride(dy),
                            nat.DTYPE_CODES[x.dtype], x.shape[0], x.shape[1], weight.shape[0], activation,
                            0 if dy is None else 1)
    return torch.empty(need, dtype=torch.uint8, device=x.device) if need else None


def _empty(matrix: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(matrix) if matrix.is_contiguous() else matrix.new_empty(matrix.shape)


def _forward(x, weight, bias, residual, activation: int, keep: bool):
    """(y, the sum before the activation where it is to be kept)."""

    rows, inner = x.shape
    outer = weight.shape[0]
    with nat.on_device(x.device):
        y = x.new_empty((rows, outer))
        pre = torch.empty_like(y) if keep else None
        workspace = _workspace(x, weight, None, activation)
        nat.call("cg_linear_forward", nat.ptr(x), _row_stride(x), nat.ptr(weight), _row_stride(weight), nat.ptr(bias),
                 nat.ptr(residual), 0 if residual is None else _row_stride(residual), nat.DTYPE_CODES[x.dtype], rows,
                 inner, outer, activation, nat.ptr(y), nat.ptr(pre), nat.ptr(workspace),
                 0 if workspace is None else workspace.numel(), nat.stream_handle(x.device))
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        trains = any(ctx.needs_input_grad[:3])
        y, pre = _forward(x, weight, bias, residual, activation, trains and activation != 0)
        if trains:
            ctx.save_for_backward(x, weight, pre)
        ctx.activation = activation
        return y

    @staticmethod
    @nat.backward_once
    def backward(ctx, dy):
        dx = dweight = dbias = None
        needs_x, needs_weight, needs_bias, needs_residual, _ = ctx.needs_input_grad
        if needs_x or needs_weight or needs_bias:
            x, weight, pre = ctx.saved_tensors
            rows, inner = x.shape
            outer = weight.shape[0]
            g = _unit_rows(dy)
            with nat.on_device(x.device):
                dx = _empty(x) if needs_x else None
                dweight = _empty(weight) if needs_weight else None
                dbias = x.new_empty(outer) if needs_bias else None
                workspace = _workspace(x, weight, g, ctx.activation)
                nat.call("cg_linear_backward", nat.ptr(g), _row_stride(g), nat.ptr(pre), nat.ptr(x), _row_stride(x),
                         nat.ptr(weight), _row_stride(weight), nat.DTYPE_CODES[x.dtype], rows, inner, outer,
                         ctx.activation, nat.ptr(dx), nat.ptr(dweight), nat.ptr(dbias), nat.ptr(workspace),
                         0 if workspace is None else workspace.numel(), nat.stream_handle(x.device))
        return dx, dweight, dbias, dy if needs_residual else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, activation: str = "none") -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual``: x [..., K], weight [N, K], bias [N], residual [..., N] -> [..., N].

    All share one dtype (float32, float16, bfloat16) and one CUDA device; rows may be strided. ``activation``: "none",
    "relu", "gelu" (exact, by erf) or "silu". Products are summed in fp32 and rounded once, after the residual.

    Differentiable in x, weight, bias and residual. In training the sum before the activation is kept in the inputs'
    dtype, as is the gradient that enters the two backward products: each a rounding of 2^-8 (bfloat16) or 2^-11
    (float16) beside the results' own, which halves what the pass reads and writes.
    """

    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {activation!r}")
    if x.dtype not in nat.DTYPE_CODES:
        raise ValueError(f"x must be float32, float16 or bfloat16, not {x.dtype}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} does not multiply a weight of {tuple(weight.shape)}")
    outer = weight.shape[0]
    shape = (*x.shape[:-1], outer)
    if bias is not None and bias.shape != (outer,):
        raise ValueError(f"bias must be [{outer}], not {tuple(bias.shape)}")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must be {shape}, not {tuple(residual.shape)}")
    for name, tensor in (("weight", weight), ("bias", bias), ("residual", residual)):
        if tensor is not None and (tensor.dtype != x.dtype or tensor.device != x.device):
            raise ValueError(f"{name} must be {x.dtype} on {x.device}, as x is, not {tensor.dtype} on {tensor.device}")
    nat.ptr(x)  # refuses CPU tensors
    if x.dim() != 2:
        rows = math.prod(shape[:-1])  # -1 is ambiguous where a row has no entries
        x = x.reshape(rows, x.shape[-1])
        residual = None if residual is None else residual.reshape(rows, outer)
    inputs = (_unit_rows(x), _unit_rows(weight), None if bias is None else bias.contiguous(),
              None if residual is None else _unit_rows(residual))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        y = _Linear.apply(*inputs, ACTIVATIONS[activation])
    else:
        y, _ = _forward(*inputs, ACTIVATIONS[activation], False)
    return y if len(shape) == 2 else y.view(shape)
