"""Matrix products of every expert's rows in one launch, with SwiGLU in the epilogue, and their gradients.

Rows are sorted by expert (`ops/dispatch.py`): expert e owns rows offsets[e] .. offsets[e + 1] of x, and its
weight is w[e] [N, K] (K contiguous, the convention of the model's `w13` = [gate rows | up rows] and `w2`).
The offsets ascend and stay on the device.  Rows before offsets[0] and past offsets[E] give zero rows, so a slice
offsets[a : b + 1] with w[a : b] computes some of a larger table's experts.  CUDA: csrc/expert_mm.cu (tcgen05, BF16
or FP16 operands, fp32 accumulators, one rounding), at most 1024 experts a call (the tile table lies in shared memory);
CPU tensors: the same products in fp32.

The tensor cores take 16-bit operands: a gated product keeps its operands for the backward pass in x's type, and their
gradient is rounded to it before dx and dw are formed from it.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from ._ext import error_word, ext

ACTIVATIONS = (None, "swiglu")


def _check(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, n: int, name: str) -> None:
    if w.dim() != 3 or w.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("w must be a BF16 or FP16 [experts, n, k] tensor")
    if w.shape[1] % 8 or w.shape[2] % 8 or not w.shape[1] or not w.shape[2]:
        raise ValueError("n and k must be multiples of 8")
    if x.dim() != 2 or x.shape[1] != n or x.dtype != w.dtype:
        raise ValueError(f"{name} must be [rows, {n}] of w's type")
    if offsets.dtype != torch.int32 or offsets.shape != (w.shape[0] + 1,):
        raise ValueError("offsets must be int32 [experts + 1]")


def _spans(offsets: torch.Tensor, rows: int):
    off = offsets.clamp(0, rows).cummax(0).values.tolist()
    return list(zip(off, off[1:]))


def _silu_grad(z: torch.Tensor, da: torch.Tensor) -> torch.Tensor:
    g, u = z.float().chunk(2, dim=-1)
    s = torch.sigmoid(g)
    return torch.cat((da.float() * u * s * (1 + g * (1 - s)), da.float() * g * s), -1)


def _linear(x, w, offsets, gated: bool, save_pre: bool):
    z = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float32)
    for e, (a, b) in enumerate(_spans(offsets, x.shape[0])):
        z[a:b] = x[a:b].float() @ w[e].float().T
    if not gated:
        return z.to(x.dtype), None
    g, u = z.chunk(2, dim=-1)
    return (g * torch.sigmoid(g) * u).to(x.dtype), z.to(x.dtype) if save_pre else None


def expert_linear_backward(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
                           need_dx: bool = True, need_dw: bool = True):
    """Gradients of the products y_e = x_e w_e^T: dx_e = dy_e w_e [P, K] and dw_e = dy_e^T x_e [E, N, K] (zero for an
    expert without rows), in w's type; each None if not needed.  For a gated product pass `swiglu_backward`'s result."""
    _check(x, w, offsets, w.shape[2], "x")
    _check(dy, w, offsets, w.shape[1], "dy")
    if w.is_cuda:
        return ext().expert_linear_backward(dy, x, w, offsets, need_dx, need_dw, error_word(w.device))
    dx = torch.zeros(x.shape, dtype=torch.float32) if need_dx else None
    dw = torch.zeros(w.shape, dtype=torch.float32) if need_dw else None
    for e, (a, b) in enumerate(_spans(offsets, x.shape[0])):
        if need_dx:
            dx[a:b] = dy[a:b].float() @ w[e].float()
        if need_dw:
            dw[e] = dy[a:b].float().T @ x[a:b].float()
    return (dx.to(x.dtype) if need_dx else None), (dw.to(w.dtype) if need_dw else None)


def swiglu_backward(dy: torch.Tensor, pre: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """Gradient [P, N] of silu(gate) * up with respect to pre = [gate | up], from dy [P, N / 2]; rows
    before offsets[0] and past offsets[E] are zero."""
    if pre.dim() != 2 or pre.shape[1] % 16 or pre.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("pre must be a BF16 or FP16 [rows, n] tensor, n a multiple of 16")
    if dy.shape != (pre.shape[0], pre.shape[1] // 2) or dy.dtype != pre.dtype:
        raise ValueError("dy must be [rows, n / 2] of pre's type")
    if pre.is_cuda:
        return ext().swiglu_backward(dy, pre, offsets)
    dz = _silu_grad(pre, dy)
    spans = _spans(offsets, pre.shape[0])
    dz[:spans[0][0]] = 0
    dz[spans[-1][1]:] = 0
    return dz.to(pre.dtype)


class _ExpertLinear(torch.autograd.Function):  # CPU tensors; the extension has its own node
    @staticmethod
    def forward(ctx, x, w, offsets, gated):
        y, pre = _linear(x, w, offsets, gated, gated)
        ctx.save_for_backward(x, w, offsets, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, offsets, pre = ctx.saved_tensors
        dz = swiglu_backward(dy, pre, offsets) if pre is not None else dy
        dx, dw = expert_linear_backward(dz, x, w, offsets, *ctx.needs_input_grad[:2])
        return dx, dw, None, None


def expert_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, activation: str | None = None) -> torch.Tensor:
    """y_e = x_e w_e^T for every expert's rows: [P, N], or with activation "swiglu" [P, N / 2] =
    silu(first half) * second half of each row's products.

    x [P, K] and w [E, N, K] BF16 or FP16 (N, K multiples of 8; N of 16 with "swiglu"), offsets int32 [E + 1] on the
    same device.  Differentiable in x and w: a gated product keeps its [P, N] operands, rounded to x's type, for
    the backward pass, and rounds their gradient likewise."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {ACTIVATIONS}")
    _check(x, w, offsets, w.shape[2] if w.dim() == 3 else 0, "x")
    gated = activation == "swiglu"
    if gated and w.shape[1] % 16:
        raise ValueError("a gated product needs n a multiple of 16")
    if w.is_cuda:
        return ext().expert_linear(x, w, offsets, gated, error_word(w.device))
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        return _ExpertLinear.apply(x, w, offsets, gated)
    return _linear(x, w, offsets, gated, False)[0]
