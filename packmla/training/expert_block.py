"""A trainable mixture-of-experts block on packmla's kernels, and a small fit that runs it end to end.

    python -m packmla.training.expert_block --tokens 2048 --hidden 1024 --inter 512 --experts 16 --steps 20

`ExpertBlock` is one block from the residual stream to the residual stream: residual add + RMSNorm
(`ops.fused.add_rmsnorm_mx`, whose h feeds the router and the experts and whose MXFP8 rows are what a served
model would send to its experts), router (sigmoid scores of the chosen top-k, normalized: the served model's
rule), rows sorted by expert, gate/up products with SwiGLU, down products, weighted sum.  Every step has a
gradient.  The command fits a block to a teacher block of other weights on Gaussian tokens with AdamW and prints
one JSON line: first and last loss, and milliseconds per step on the device.  Runs on CPU tensors as well.
"""
from __future__ import annotations

import argparse
import json

import torch
from torch import nn

from ..ops import dispatch, fused, grouped


class ExpertBlock(nn.Module):
    def __init__(self, hidden: int, inter: int, experts: int, topk: int, eps: float = 1e-6,
                 dtype: torch.dtype = torch.bfloat16, device: str | torch.device = "cpu", seed: int = 0):
        super().__init__()
        if hidden % 32 or inter % 8:
            raise ValueError("hidden must be a multiple of 32 and inter of 8")
        if not 1 <= topk <= experts:
            raise ValueError("topk must be in [1, experts]")
        g = torch.Generator(device=device).manual_seed(seed)

        def normal(*shape, scale):
            return nn.Parameter((torch.randn(*shape, generator=g, device=device) * scale).to(dtype))

        self.norm = nn.Parameter(torch.ones(hidden, device=device))
        self.gate = normal(experts, hidden, scale=hidden ** -0.5)
        self.w13 = normal(experts, 2 * inter, hidden, scale=hidden ** -0.5)
        self.w2 = normal(experts, hidden, inter, scale=inter ** -0.5)
        self.topk, self.eps = topk, eps

    def route(self, h: torch.Tensor, mask: torch.Tensor | None = None):
        """(ids [T, k] int32, weights fp32 [T, k]): top-k of the sigmoid scores, normalized over the k.  Tokens
        where `mask` is false get id -1: no expert sees them."""
        scores = torch.sigmoid((h @ self.gate.T).float())
        top = scores.topk(self.topk, dim=-1)
        ids = top.indices.int()
        if mask is not None:
            ids = torch.where(mask[:, None], ids, -1)
        return ids, top.values / top.values.sum(-1, keepdim=True)

    def forward(self, x: torch.Tensor, d: torch.Tensor | None = None, mask: torch.Tensor | None = None):
        """(stream, out): stream = x + d, out = stream + the routed experts' sum of its normed rows, x's type."""
        stream, _, _, h = fused.add_rmsnorm_mx(x, self.norm, self.eps, d, return_h=True)
        ids, weights = self.route(h, mask)
        order = dispatch.expert_order(ids, self.w13.shape[0])
        act = grouped.expert_linear(dispatch.gather(h, order), self.w13, order.offsets, activation="swiglu")
        y = grouped.expert_linear(act, self.w2, order.offsets)
        return stream, dispatch.combine(y, order, weights, stream)


def fit(tokens: int, hidden: int, inter: int, experts: int, topk: int, steps: int, lr: float,
        device: str, seed: int = 0) -> dict:
    block = ExpertBlock(hidden, inter, experts, topk, device=device, seed=seed)
    teacher = ExpertBlock(hidden, inter, experts, topk, device=device, seed=seed + 1)
    teacher.gate.data.copy_(block.gate.data)  # the same routing: the experts are what is learned
    optimizer = torch.optim.AdamW(block.parameters(), lr=lr, weight_decay=0.0)
    g = torch.Generator(device=device).manual_seed(seed + 2)
    losses, times = [], []
    cuda = torch.device(device).type == "cuda"
    for _ in range(steps):
        x, d = (torch.randn(tokens, hidden, generator=g, device=device).bfloat16() for _ in range(2))
        with torch.no_grad():
            want = teacher(x, d)[1].float()
        if cuda:
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
        optimizer.zero_grad(set_to_none=True)
        stream, out = block(x, d)
        loss = (out.float() - want).square().mean() / (want - stream.float()).square().mean()
        loss.backward()
        optimizer.step()
        if cuda:
            end.record()
            times.append((start, end))
        losses.append(loss.detach())
    out = {"tokens": tokens, "hidden": hidden, "inter": inter, "experts": experts, "topk": topk, "steps": steps,
           "first_loss": round(losses[0].item(), 5), "last_loss": round(losses[-1].item(), 5)}
    if cuda:
        from ..ops import check_errors

        check_errors(torch.device(device))
        out["ms_per_step"] = round(sorted(a.elapsed_time(b) for a, b in times)[len(times) // 2], 3)
    return out


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=2048)
    ap.add_argument("--hidden", type=int, default=1024)
    ap.add_argument("--inter", type=int, default=512)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--topk", type=int, default=4)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--lr", type=float, default=1e-3)
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    print(json.dumps(fit(a.tokens, a.hidden, a.inter, a.experts, a.topk, a.steps, a.lr, a.device, a.seed)), flush=True)


if __name__ == "__main__":
    main()
