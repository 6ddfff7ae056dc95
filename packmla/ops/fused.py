"""Fused element-wise / reduction ops of the decode step (csrc/fused_ops.cu); PyTorch on CPU."""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from ..formats import abi, codec
from ._ext import ext


def add_rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, d: torch.Tensor | None = None,
                dfp32: torch.Tensor | None = None, inplace: bool = False):
    """Returns (x_new, h): x_new = bf16(x + d + dfp32) (x itself if no addend), h = bf16(rmsnorm(x_new) * w)."""
    has_add = d is not None or dfp32 is not None
    if x.is_cuda and x.shape[1] % 2 == 0 and x.shape[1] <= 8192:
        h = torch.empty_like(x)
        x_out = (x if inplace else torch.empty_like(x)) if has_add else None
        ext().add_rmsnorm(x, d, dfp32, x_out, w, float(eps), h)
        return (x_out if has_add else x), h
    xf = x.float()
    if d is not None:
        xf = xf + d.float()
    if dfp32 is not None:
        xf = xf + dfp32.float()
    if has_add:
        xn = xf.to(torch.bfloat16)
        xf = xn.float()
    else:
        xn = x
    h = (xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + eps) * w).to(torch.bfloat16)
    return xn, h


def rope_q(q: torch.Tensor, pos: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """Rotate coords 448..511 of q [B, H, 512] bf16 by freqs[pos] (in place on CUDA)."""
    if q.is_cuda:
        ext().rope_q(q, pos.to(torch.int64).contiguous(), freqs)
        return q
    fr = freqs[pos.long()]
    c, s = fr[:, None, :, 0], fr[:, None, :, 1]
    tail = q[..., abi.NOPE_DIM:].float().unflatten(-1, (abi.ROPE_PAIRS, 2))
    re, im = tail[..., 0], tail[..., 1]
    rot = torch.stack((re * c - im * s, re * s + im * c), -1).flatten(-2)
    return torch.cat((q[..., :abi.NOPE_DIM], rot.to(torch.bfloat16)), -1)


def comp_pool(proj: torch.Tensor, off: int, D: int, ape: torch.Tensor, state: torch.Tensor, req: torch.Tensor,
              pos: torch.Tensor) -> torch.Tensor:
    """One token per row of online-softmax pooling; returns raw fp32 [B, D] (valid where the group completes)."""
    ratio = ape.shape[0]
    if proj.is_cuda:
        raw = torch.empty(proj.shape[0], D, dtype=torch.float32, device=proj.device)
        ext().comp_pool(proj, off, D, ape, state, req.to(torch.int64).contiguous(), pos.to(torch.int64).contiguous(), raw)
        return raw
    val = proj[:, off:off + D].float()
    slot = pos.long() % ratio
    gate = proj[:, off + D:off + 2 * D].float() + ape[slot]
    st = state[req.long()]
    m, l, acc = st[:, 0], st[:, 1], st[:, 2]
    mn = torch.maximum(m, gate)
    a = torch.exp(m - mn)
    e = torch.exp(gate - mn)
    l2 = l * a + e
    acc2 = acc * a + e * val
    raw = acc2 / l2
    done = (slot == ratio - 1)[:, None]
    state[req.long()] = torch.stack((torch.where(done, torch.full_like(mn, float("-inf")), mn),
                                     torch.where(done, torch.zeros_like(l2), l2),
                                     torch.where(done, torch.zeros_like(acc2), acc2)), 1)
    return raw


def route_topk(logits: torch.Tensor, bias: torch.Tensor | None, k: int, scaling: float):
    """Sigmoid scores of bf16 logits; top-k of score + bias (ties: lower expert); weights normalized over the k."""
    T, E = logits.shape
    if logits.is_cuda and E <= 512:
        ids = torch.empty(T, k, dtype=torch.int32, device=logits.device)
        w = torch.empty(T, k, dtype=torch.float32, device=logits.device)
        ext().route_topk(logits, bias, k, float(scaling), ids, w)
        return ids, w
    scores = torch.sigmoid(logits.float())
    key = scores + (bias if bias is not None else 0.0)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    w = scores.gather(1, order)
    return order.int(), w / w.sum(-1, keepdim=True) * scaling


def silu_mul(gu: torch.Tensor) -> torch.Tensor:
    I = gu.shape[1] // 2
    if gu.is_cuda:
        out = torch.empty(gu.shape[0], I, dtype=torch.bfloat16, device=gu.device)
        ext().silu_mul(gu, out)
        return out
    return (F.silu(gu[:, :I].float()) * gu[:, I:].float()).to(torch.bfloat16)


MX_GROUP = 32  # columns that share one UE8M0 scale of an MXFP8 row


def _norm_oracle(s: torch.Tensor, w: torch.Tensor, eps: float):
    """(s r, r) of fp32 rows s: the normalized rows before the weight, and r = (mean(s^2) + eps)^-1/2."""
    r = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
    return s * r, r


def mx_quantize(h: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows [T, n] -> (E4M3 codes [T, n], UE8M0 scale bytes [T, n / 32]), uint8: the rule of `add_rmsnorm_mx`.

    A NaN is a NaN code and counts for no scale; an infinity has the largest scale and code, which stand for infinity in
    BF16 and fp32 (finite values beside it come out as zero)."""
    b = h.float().unflatten(-1, (h.shape[1] // MX_GROUP, MX_GROUP))
    amax = torch.where(b.isnan(), 0.0, b.abs()).amax(-1)
    e = codec.ue8m0_exponent(amax.clamp_max(torch.finfo(torch.float32).max))
    codes = codec.e4m3_encode((b * codec.exp2_int(-e)[..., None]).clamp(-448, 448))
    return codes.reshape(h.shape), (e + 127).to(torch.uint8)


def mx_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """MXFP8 rows -> code x 2^(scale - 127), NaN for scale byte 255.  E4M3 has four significant bits: exact for scale
    bytes 3 to 246 in BF16 and 0 to 246 in fp32, rounded once beyond them (to zero, a subnormal or infinity)."""
    if codes.is_cuda and dtype == torch.bfloat16:
        return ext().mx_dequantize(codes, scales)
    v = codec.e4m3_decode(codes).unflatten(-1, (codes.shape[1] // MX_GROUP, MX_GROUP))
    s = torch.where(scales == 255, float("nan"), codec.exp2_int(scales.to(torch.int32) - 127))
    return (v * s[..., None]).reshape(codes.shape).to(dtype)


def _check_norm(x: torch.Tensor, w: torch.Tensor) -> None:
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("x must be a BF16 or FP16 [rows, n] tensor")
    if x.shape[1] % MX_GROUP or not 0 < x.shape[1] <= 8192:
        raise ValueError(f"n = {x.shape[1]} must be a multiple of {MX_GROUP} and at most 8192")
    if w.shape != (x.shape[1],) or w.dtype != torch.float32:
        raise ValueError("w must be fp32 [n]")


def _add_rmsnorm_mx(x, w, eps, d, dfp32, inplace, return_h):
    _check_norm(x, w)
    s = x
    if d is not None or dfp32 is not None:
        s = x.float()
        for t in (d, dfp32):
            if t is not None:
                s = s + t.float()
        s = x.copy_(s) if inplace else s.to(x.dtype)
    h = _norm_oracle(s.float(), w, eps)[0] * w
    return (s, *mx_quantize(h), h.to(x.dtype) if return_h else None)


def add_rmsnorm_backward(dh: torch.Tensor, x: torch.Tensor, w: torch.Tensor, eps: float,
                         dres: torch.Tensor | None = None, fp32_dx: bool = False):
    """Gradients of `add_rmsnorm` / `add_rmsnorm_mx` at the stored stream x, from dh (of h) and dres (of x itself).

    Returns (dx, dw) - dx in x's type is also the gradient of the addend d, dw is fp32 and does not depend on
    timing (fixed summation order) - or (dx, dw, fp32 dx) with `fp32_dx`, the gradient of the fp32 addend."""
    if x.is_cuda:
        dx, dw, dxf = ext().rmsnorm_backward(dh, x, w, eps, dres, fp32_dx)
        return (dx, dw, dxf) if fp32_dx else (dx, dw)
    _check_norm(x, w)
    n, r = _norm_oracle(x.float(), w, eps)
    g = dh.float() * w
    dxf = r * (g - n * (g * n).mean(-1, keepdim=True))
    if dres is not None:
        dxf = dxf + dres.float()
    dw = (dh.float() * n).sum(0)
    return (dxf.to(x.dtype), dw, dxf) if fp32_dx else (dxf.to(x.dtype), dw)


class _AddRmsNormMx(torch.autograd.Function):  # CPU tensors; the extension has its own node
    @staticmethod
    def forward(ctx, x, w, d, dfp32, eps, return_h):
        s, codes, scales, h = _add_rmsnorm_mx(x, w, eps, d, dfp32, False, return_h)
        if s is x:
            s = x.view_as(x)
        ctx.save_for_backward(s, w)
        ctx.eps = eps
        ctx.addends = d is not None, dfp32 is not None
        ctx.mark_non_differentiable(codes, scales)
        ctx.set_materialize_grads(False)
        return s, codes, scales, h

    @staticmethod
    @once_differentiable
    def backward(ctx, ds, _codes, _scales, dh):
        s, w = ctx.saved_tensors
        need = ctx.needs_input_grad
        has_d, has_f = ctx.addends
        if dh is None:  # only the stream was used
            dx, dw, dxf = ds, None, ds.float() if ds is not None and has_f else None
        else:
            dx, dw, *rest = add_rmsnorm_backward(dh, s, w, ctx.eps, ds, fp32_dx=has_f and need[3])
            dxf = rest[0] if rest else None
        return (dx if need[0] else None, dw if need[1] else None, dx if has_d and need[2] else None,
                dxf if has_f and need[3] else None, None, None)


def add_rmsnorm_mx(x: torch.Tensor, w: torch.Tensor, eps: float, d: torch.Tensor | None = None,
                   dfp32: torch.Tensor | None = None, inplace: bool = False, return_h: bool = False):
    """Residual add + RMSNorm with MXFP8 rows out: (x_new, codes, scales, h).

    x_new = x + d + dfp32 in x's type (x itself without an addend; written over x with `inplace`,
    where d may be x and every other operand has to lie apart from x);
    h = x_new * rsqrt(mean(x_new^2) + eps) * w in fp32; codes [T, n] are the E4M3 codes of h (uint8) and scales
    [T, n / 32] its UE8M0 scale bytes, one per 32 columns; with `return_h`, h rounded to x's type (the router's and
    the shared expert's input), else None.  x, d: BF16 or FP16 [T, n], n a multiple of 32 up to 8192; w fp32 [n].

    Differentiable in x, w, d and dfp32 through x_new and h; the codes carry no gradient (a trainer that feeds
    them to its products uses h's gradient for them)."""
    if x.is_cuda and not inplace:
        return ext().add_rmsnorm_mx(x, w, eps, d, dfp32, False, return_h)
    wanted = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, d, dfp32))
    if not wanted:
        if x.is_cuda:
            return ext().add_rmsnorm_mx(x, w, eps, d, dfp32, True, return_h)
        return _add_rmsnorm_mx(x, w, eps, d, dfp32, inplace, return_h)
    if inplace:
        raise ValueError("inplace is not available where a gradient is recorded")
    return _AddRmsNormMx.apply(x, w, d, dfp32, eps, return_h)
