"""Expert block operators on CPU tensors (the arithmetic the kernels are held to) against 64-bit references."""
import pytest
import torch

import expert_block_reference as ref
from expert_block_reference import ACC, F64
from packmla.ops import dispatch, fused, grouped

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


@pytest.mark.parametrize("rows,n,dtype,addends", [(1, 32, BF16, 0), (5, 96, F16, 1), (7, 416, BF16, 2), (0, 64, BF16, 1)])
def test_norm_mx(rows, n, dtype, addends):
    g = torch.Generator().manual_seed(rows + n)
    x, w = randn(g, rows, n, dtype=dtype, scale=3.0), 1 + 0.3 * randn(g, n)
    d = randn(g, rows, n, dtype=dtype) if addends else None
    df = randn(g, rows, n) if addends > 1 else None
    s, codes, scales, h = fused.add_rmsnorm_mx(x, w, 1e-6, d, df, return_h=True)
    rs, rh, _ = ref.norm(x, w, 1e-6, d, df)
    assert torch.equal(s.to(F64), rs)
    rel = ACC * (n + 8)
    ref.check(h, rh, rh.abs() * rel, "h")
    if rows:
        ref.check_mx(codes, scales, rh, rel)
        back = fused.mx_dequantize(codes, scales)
        again = fused.mx_quantize(back.float())
        assert torch.equal(fused.mx_dequantize(*again), back)  # quantizing the values a row stands for keeps them
    dh, dres = randn(g, rows, n, dtype=dtype), randn(g, rows, n, dtype=dtype)
    dx, dw, dxf = fused.add_rmsnorm_backward(dh, s, w, 1e-6, dres, fp32_dx=True)
    rdx, rdw = ref.norm_grads(rs, w, 1e-6, dh, dres)
    scale = (rdx.abs().max() if rows else 0) * 1e-4
    ref.check(dx, rdx, scale)
    ref.check(dxf, rdx, scale)
    ref.check(dw, rdw, rdw.abs().max() * 1e-4)


def test_norm_mx_gradients_flow_and_refusals():
    g = torch.Generator().manual_seed(1)
    x, d, w = (t.requires_grad_(True) for t in (randn(g, 3, 64, dtype=BF16), randn(g, 3, 64, dtype=BF16), 1 + 0.1 * randn(g, 64)))
    s, _, _, h = fused.add_rmsnorm_mx(x, w, 1e-6, d, return_h=True)
    dh = randn(g, 3, 64, dtype=BF16)
    dx, dd, dw = torch.autograd.grad(h, [x, d, w], dh)
    rdx, rdw = ref.norm_grads(s.detach().to(F64), w.detach(), 1e-6, dh)
    ref.check(dx, rdx, 1e-4)
    assert torch.equal(dx, dd)
    ref.check(dw, rdw, 1e-4)
    with pytest.raises(ValueError, match="multiple of 32"):
        fused.add_rmsnorm_mx(torch.zeros(1, 40, dtype=BF16), torch.ones(40), 1e-6)
    with pytest.raises(ValueError, match="BF16 or FP16"):
        fused.add_rmsnorm_mx(torch.zeros(1, 64), torch.ones(64), 1e-6)


@pytest.mark.parametrize("T,k,E,base", [(0, 2, 3, 0), (1, 1, 1, 0), (7, 3, 5, 2), (40, 8, 64, 0)])
def test_order_gather_combine(T, k, E, base):
    g = torch.Generator().manual_seed(T + E)
    ids = torch.randint(base - 1, base + E + 1, (T, k), generator=g)
    order = dispatch.expert_order(ids, E, base)
    for a, b in zip(order, ref.order(ids, E, base)):
        assert torch.equal(a, b)
    x = randn(g, T, 24, dtype=BF16).requires_grad_(True)
    rows = dispatch.gather(x, order)
    for r, p in enumerate(order.pairs.tolist()):
        assert torch.equal(rows[r], x[p // k] if p >= 0 else torch.zeros(24, dtype=BF16))
    y = rows.detach().clone().requires_grad_(True)
    w = torch.rand(T, k, generator=g).requires_grad_(True)
    out = dispatch.combine(y, order, w, out_dtype=F32)
    want = torch.zeros(T, 24, dtype=F64)
    for t in range(T):
        for j in range(k):
            if order.slots[t, j] >= 0:
                want[t] += w[t, j].to(F64) * y[order.slots[t, j]].to(F64)
    ref.check(out, want.detach(), 1e-5)
    if T:
        dout = randn(g, T, 24)
        dy, dw = torch.autograd.grad(out, [y, w], dout)
        dx, = torch.autograd.grad(rows, x, dy)
        for t in range(T):
            total = torch.zeros(24, dtype=F64)
            for j in range(k):
                r = int(order.slots[t, j])
                if r >= 0:
                    ref.check(dy[r], w[t, j].detach().to(F64) * dout[t].to(F64), 1e-6)
                    ref.check(dw[t, j], (dout[t].to(F64) * y[r].detach().to(F64)).sum(), 1e-4)
                    total += dy[r].to(F64)
                else:
                    assert dw[t, j] == 0
            ref.check(dx[t], total, 1e-5)


@pytest.mark.parametrize("counts,tail,K,N,gated", [([1], 0, 8, 16, False), ([3, 0, 5], 2, 24, 32, True), ([0, 0], 3, 16, 16, True)])
def test_products(counts, tail, K, N, gated):
    g = torch.Generator().manual_seed(K + N)
    offsets = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32)
    P = int(offsets[-1]) + tail
    x, w = randn(g, P, K, dtype=F16).requires_grad_(True), randn(g, len(counts), N, K, dtype=F16, scale=K ** -0.5).requires_grad_(True)
    y = grouped.expert_linear(x, w, offsets, activation="swiglu" if gated else None)
    z, s = ref.linear(x.detach(), w.detach(), offsets)
    z = z.requires_grad_(True)
    want = ref.swiglu(z) if gated else z
    ref.check(y, want.detach(), 1e-4 if gated else s * ACC * K)
    dy = randn(g, *y.shape, dtype=F16)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    dz, = torch.autograd.grad(want, z, dy.to(F64))
    dz[P - tail:] = 0
    rdx, _ = ref.linear(dz, w.detach().transpose(1, 2), offsets)
    ref.check(dx, rdx, 2e-2)
    for e in range(len(counts)):
        a, b = int(offsets[e]), int(offsets[e + 1])
        ref.check(dw[e], dz[a:b].T @ x.detach()[a:b].to(F64), 2e-2)


def test_products_refusals():
    x, w, off = torch.zeros(2, 16, dtype=BF16), torch.zeros(1, 8, 16, dtype=BF16), torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(ValueError, match="multiple of 16"):
        grouped.expert_linear(x, w, off, activation="swiglu")
    with pytest.raises(ValueError, match="w's type"):
        grouped.expert_linear(x.float(), w, off)
    with pytest.raises(ValueError, match="offsets"):
        grouped.expert_linear(x, w, off.long())
