"""Token rows sorted by expert and back: the exchange around a mixture-of-experts block's products.

    order = expert_order(ids, num_experts)      # ids [T, k]: pairs (token, choice) -> rows sorted by expert
    rows = gather(x, order)                     # [T k, H]: the token of every row   (gather_mx: MXFP8 rows)
    y = ...                                     # the experts' products on offsets-delimited rows (ops/grouped.py)
    out = combine(y, order, weights, residual)  # [T, H]: residual + sum_k w_k y_k

`gather` and `combine` are differentiable.  All calls run on the current stream without waiting for the host;
the row count of every expert stays on the device (`order.offsets`).  CUDA: csrc/expert_dispatch.cu; CPU
tensors: the same arithmetic in PyTorch.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._ext import ext

MAX_EXPERTS = 4096  # of a sort; the products of ops/grouped.py take 1024 on CUDA


class ExpertOrder(NamedTuple):
    """Rows sorted by expert, earlier pairs first, as `expert_order` makes them (a slice of offsets is for the products
    alone: `gather` and `combine` go by the whole table).  A pair whose expert is not in [base, base + E) - masked
    tokens use -1 - has no row.  Rows past offsets[E] belong to no pair."""

    offsets: torch.Tensor  # int32 [E + 1]: expert e owns rows offsets[e] .. offsets[e + 1]
    slots: torch.Tensor    # int32 [T, k]: row of the pair, -1 if it has none
    pairs: torch.Tensor    # int32 [T k]: pair t k + j of the row, -1 past the last row


def expert_order(ids: torch.Tensor, num_experts: int, expert_base: int = 0) -> ExpertOrder:
    """Stable sort of the pairs of ids [T, k] (int32 or int64) by expert, for experts [base, base + num_experts)."""
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {MAX_EXPERTS}]")
    if ids.dim() != 2 or ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("ids must be an int32 or int64 [tokens, topk] tensor")
    if ids.is_cuda:
        return ExpertOrder(*ext().expert_order(ids, num_experts, expert_base))
    flat = ids.reshape(-1).long() - expert_base
    key = torch.where((flat >= 0) & (flat < num_experts), flat, num_experts)
    pairs = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=num_experts + 1)[:num_experts]
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    place = torch.arange(flat.numel())
    slots = torch.empty_like(place)
    slots[pairs] = place
    slots = torch.where(key < num_experts, slots, -1)
    pairs = torch.where(place < offsets[-1], pairs, -1)
    return ExpertOrder(offsets.int(), slots.int().view(ids.shape), pairs.int())


def _check_tokens(x: torch.Tensor, order: ExpertOrder, name: str) -> None:
    if x.dim() != 2 or x.shape[0] != order.slots.shape[0]:
        raise ValueError(f"{name} must be [{order.slots.shape[0]}, width]: one row per token of the order")


def _gather(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    token = order.pairs.clamp_min(0).long() // max(1, order.slots.shape[1])
    zero = torch.zeros((), dtype=x.dtype)
    return torch.where((order.pairs >= 0)[:, None], x[token], zero)


def gather_mx(codes: torch.Tensor, scales: torch.Tensor, order: ExpertOrder) -> tuple[torch.Tensor, torch.Tensor]:
    """`gather` of MXFP8 rows: codes [T, n] and their scale bytes [T, n / 32], both uint8, in one launch."""
    _check_tokens(codes, order, "codes")
    _check_tokens(scales, order, "scales")
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("codes and scales must be uint8")
    if codes.is_cuda:
        return ext().expert_gather_mx(codes, scales, order.slots, order.offsets)
    return _gather(codes, order), _gather(scales, order)


def gather_backward(drows: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """Gradient of `gather`: dx[t] = sum over the token's rows of drows (fp32 sum, one rounding)."""
    return combine(drows, order)


def _combine(y, order, weights, residual, out_dtype):
    here = order.slots >= 0
    rows = y[order.slots.clamp_min(0).long()].float() if y.shape[0] else y.new_zeros((*order.slots.shape, y.shape[1])).float()
    w = torch.where(here, weights if weights is not None else torch.ones(()), 0.0)
    out = (torch.where(here[..., None], rows, 0.0) * w[..., None]).sum(1)
    if residual is not None:
        out = out + residual.float()
    return out.to(out_dtype)


def combine_backward(dout: torch.Tensor, y: torch.Tensor, order: ExpertOrder, weights: torch.Tensor,
                     need_dy: bool = True, need_dweights: bool = True):
    """Gradients of `combine`: dy[row of (t, j)] = w[t, j] dout[t] (rows of no pair: 0) and
    dweights[t, j] = <dout[t], y[row]> in fp32 (0 for a pair without a row); each None if not needed."""
    if y.is_cuda:
        return ext().expert_combine_backward(dout, y, weights, order.slots, order.offsets, need_dy, need_dweights)
    here, at, g = order.slots >= 0, order.slots.clamp_min(0).long(), dout.float()
    dy = dw = None
    if need_dy:
        dy = torch.zeros(y.shape, dtype=torch.float32)
        dy[at[here]] = (weights[..., None] * g[:, None])[here]
        dy = dy.to(y.dtype)
    if need_dweights:
        dw = torch.where(here, (y[at].float() * g[:, None]).sum(-1), 0.0)
    return dy, dw


class _Gather(torch.autograd.Function):  # CPU tensors; the extension has its own nodes
    @staticmethod
    def forward(ctx, x, *order):
        ctx.order = ExpertOrder(*order)
        return _gather(x, ctx.order)

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        return gather_backward(drows, ctx.order), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, residual, out_dtype, *order):
        ctx.order = ExpertOrder(*order)
        ctx.save_for_backward(y if weights is not None else None, weights)  # unweighted: no gradient reads the rows
        ctx.dtype = y.dtype
        return _combine(y, ctx.order, weights, residual, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        y, weights = ctx.saved_tensors
        need = ctx.needs_input_grad
        dy = dw = None
        if weights is None:
            dy = _gather(dout, ctx.order).to(ctx.dtype) if need[0] else None
        elif need[0] or need[1]:
            dy, dw = combine_backward(dout, y, ctx.order, weights, need[0], need[1])
        return (dy, dw, dout if need[2] else None) + (None,) * 4


def gather(x: torch.Tensor, order: ExpertOrder) -> torch.Tensor:
    """Rows [T k, H]: row r holds its pair's token row x[pairs[r] // k]; rows of no pair are zero.

    x [T, H] of any type and strides.  Differentiable where x is BF16, FP16 or FP32."""
    _check_tokens(x, order, "x")
    if x.is_cuda:
        return ext().expert_gather(x, order.slots, order.offsets)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Gather.apply(x, *order)
    return _gather(x, order)


def combine(y: torch.Tensor, order: ExpertOrder, weights: torch.Tensor | None = None,
            residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """[T, H]: residual[t] + sum_j weights[t, j] y[slots[t, j]], summed in fp32 in choice order, rounded once.

    y [T k, H] BF16, FP16 or FP32; weights fp32 [T, k] (None: 1); `out_dtype` y's type (default) or fp32;
    residual [T, H] of the output's type.  A pair without a row adds nothing, whatever its weight holds.
    Differentiable in y, weights and residual."""
    out_dtype = out_dtype or y.dtype
    if y.dim() != 2 or y.shape[0] != order.pairs.shape[0]:
        raise ValueError(f"y must be [{order.pairs.shape[0]}, width]: one row per pair of the order")
    if y.dtype not in (torch.bfloat16, torch.float16, torch.float32) or out_dtype not in (y.dtype, torch.float32):
        raise ValueError("y must be BF16, FP16 or FP32, and out_dtype y's type or FP32")
    if weights is not None and (weights.shape != order.slots.shape or weights.dtype != torch.float32):
        raise ValueError(f"weights must be fp32 {list(order.slots.shape)}")
    if residual is not None and (residual.shape != (order.slots.shape[0], y.shape[1]) or residual.dtype != out_dtype):
        raise ValueError("residual must be [tokens, width] of the output's type")
    if y.is_cuda:
        return ext().expert_combine(y, weights, residual, order.slots, order.offsets, out_dtype == torch.float32)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, weights, residual)):
        return _Combine.apply(y, weights, residual, out_dtype, *order)
    return _combine(y, order, weights, residual, out_dtype)
