"""Expert block kernels (csrc/norm_mx.cu, expert_dispatch.cu, expert_mm.cu) against 64-bit references."""
import pytest
import torch

import expert_block_reference as ref
from expert_block_reference import ACC, F64
from packmla.ops import check_errors, dispatch, fused, grouped

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ norm
def norm_inputs(rows, n, dtype, addends, seed=0):
    g = gen(seed + rows * 7 + n)
    x = randn(g, rows, n, dtype=dtype, scale=3.0)
    w = 1 + 0.3 * randn(g, n)
    d = randn(g, rows, n, dtype=dtype) if addends else None
    df = randn(g, rows, n, scale=0.5) if addends > 1 else None
    return g, x, w, d, df


@pytest.mark.parametrize("rows,n,dtype,addends", [
    (1, 32, BF16, 0), (1, 4096, BF16, 2), (3, 64, F16, 1), (17, 2080, BF16, 2), (5, 8192, F16, 2), (130, 544, BF16, 1),
    (9, 256, F16, 0), (0, 64, BF16, 1),
])
def test_norm_mx(cuda, rows, n, dtype, addends):
    _, x, w, d, df = norm_inputs(rows, n, dtype, addends)
    s, codes, scales, h = fused.add_rmsnorm_mx(x, w, 1e-6, d, df, return_h=True)
    rs, rh, _ = ref.norm(x, w, 1e-6, d, df)
    assert torch.equal(s.to(F64), rs)  # fp32 additions in the same order, one rounding
    assert (s is x) == (addends == 0)
    rel = ACC * (n ** 0.5 + 8)  # fp32 sum of n squares (tree), root and two products
    ref.check(h, rh, rh.abs() * rel, "h")
    if rows:
        ref.check_mx(codes, scales, rh, rel)
    a = fused.add_rmsnorm_mx(x.clone(), w, 1e-6, d, df)
    assert a[3] is None and torch.equal(a[1], codes) and torch.equal(a[2], scales)
    if addends:
        x2 = x.clone()
        a = fused.add_rmsnorm_mx(x2, w, 1e-6, d, df, inplace=True)
        assert a[0].data_ptr() == x2.data_ptr() and torch.equal(x2, s) and torch.equal(a[1], codes)


def test_norm_mx_strided_and_unaligned_rows(cuda):
    g = gen(3)
    wide = randn(g, 6, 3 * 96, dtype=BF16)
    w = randn(g, 96)
    for x in (wide[:, 96:192], wide[:, 1:97], wide[::2, :96], wide.t()[:96, :6].contiguous().t()):
        got = fused.add_rmsnorm_mx(x, w, 1e-6, x, return_h=True)
        want = fused.add_rmsnorm_mx(x.contiguous(), w, 1e-6, x.contiguous(), return_h=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_norm_mx_special_values(cuda):
    x = torch.ones(5, 64, device="cuda", dtype=BF16)
    x[0, 3] = float("nan")
    x[1] = 0
    x[2, 5] = float("inf")
    x[3] = 1e-30
    x[4] = 3e38
    w = torch.ones(64, device="cuda")
    s, codes, scales, h = fused.add_rmsnorm_mx(x, w, 1e-6, return_h=True)
    hf = h.float()
    assert hf[0].isnan().all() and (codes[0] & 127 == 127).all()
    assert (hf[1] == 0).all() and (codes[1] == 0).all()
    assert hf[2, 5].isnan() and (hf[2, :5] == 0).all() and codes[2, 5] & 127 == 127
    assert hf[3].isfinite().all() and hf[4].isfinite().all()
    # a group of zeros, or below the floor, keeps the floor's scale: 448 2^e >= 1e-4
    assert scales[1].tolist() == [127 - 22, 127 - 22]


@pytest.mark.parametrize("rows,n,dtype,res,f32", [
    (1, 32, BF16, False, False), (7, 64, F16, True, True), (333, 2080, BF16, True, False), (41, 8192, F16, True, False),
    (2500, 256, BF16, False, True), (0, 96, BF16, True, False),
])
def test_norm_backward(cuda, rows, n, dtype, res, f32):
    g, x, w, _, _ = norm_inputs(rows, n, dtype, 0, seed=9)
    dh = randn(g, rows, n, dtype=dtype)
    dres = randn(g, rows, n, dtype=dtype) if res else None
    out = fused.add_rmsnorm_backward(dh, x, w, 1e-5, dres, fp32_dx=f32)
    s = x.to(F64)
    rdx, rdw = ref.norm_grads(s, w, 1e-5, dh, dres)
    r = (s.square().mean(-1, keepdim=True) + 1e-5) ** -0.5
    size = r * (dh.to(F64) * w.to(F64)).abs() + s.abs() * r ** 3 / n * (dh.to(F64) * w.to(F64) * s).abs().sum(-1, keepdim=True)
    slack = (size + (dres.to(F64).abs() if res else 0)) * ACC * (n ** 0.5 + 16)
    ref.check(out[0], rdx, slack, "dx")
    if f32:
        ref.check(out[2], rdx, slack, "dx fp32")
    mag = (dh.to(F64) * s * r).abs().sum(0)
    ref.check(out[1], rdw, mag * ACC * (rows ** 0.5 + n ** 0.5 + 16), "dw")
    again = fused.add_rmsnorm_backward(dh, x, w, 1e-5, dres, fp32_dx=f32)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_norm_autograd_matches_formula_and_differences(cuda):
    g, x, w, d, df = norm_inputs(6, 128, BF16, 2, seed=4)
    leaves = [t.requires_grad_(True) for t in (x, w, d, df)]
    s, codes, scales, h = fused.add_rmsnorm_mx(x, w, 1e-6, d, df, return_h=True)
    assert not codes.requires_grad and not scales.requires_grad
    dh, ds = randn(g, 6, 128, dtype=BF16), randn(g, 6, 128, dtype=BF16)
    grads = torch.autograd.grad([h, s], leaves, [dh, ds])
    rdx, rdw = ref.norm_grads(s.detach().to(F64), w.detach(), 1e-6, dh, ds)
    for t in (grads[0], grads[2]):
        ref.check(t, rdx, rdx.abs().max() * 1e-4, "dx")
    ref.check(grads[3], rdx, rdx.abs().max() * 1e-4, "ddf")
    ref.check(grads[1], rdw, rdw.abs().max() * 1e-4, "dw")
    # central differences of the loss <dh, h> + <ds, s> along a direction, at the stored stream
    v = randn(g, 6, 128, dtype=F64)
    s0, w64 = s.detach().to(F64), w.detach().to(F64)

    def loss(t):
        q = s0 + t * v
        return (dh.to(F64) * q * (q.square().mean(-1, keepdim=True) + 1e-6) ** -0.5 * w64).sum() + (ds.to(F64) * q).sum()

    step = 1e-5
    diff = (loss(step) - loss(-step)) / (2 * step)
    # each rounded gradient is off by at most 2^-8 of itself
    assert abs(diff - (grads[0].to(F64) * v).sum()) <= 1.01 * 2 ** -8 * (rdx * v).abs().sum()
    # the stream alone
    s, _, _, h = fused.add_rmsnorm_mx(x, w, 1e-6, d, df, return_h=True)
    only = torch.autograd.grad(s, [x, d, df], ds)
    assert torch.equal(only[0], ds) and torch.equal(only[1], ds) and torch.equal(only[2], ds.float())


def test_norm_refusals(cuda):
    x, w = torch.zeros(2, 64, device="cuda", dtype=BF16), torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="multiple of 32"):
        fused.add_rmsnorm_mx(x[:, :48].contiguous(), w[:48].contiguous(), 1e-6)
    with pytest.raises(RuntimeError, match="BF16 or FP16"):
        fused.add_rmsnorm_mx(x.float(), w, 1e-6)
    with pytest.raises(RuntimeError, match="fp32"):
        fused.add_rmsnorm_mx(x, w.bfloat16(), 1e-6)
    with pytest.raises(RuntimeError, match="d must be"):
        fused.add_rmsnorm_mx(x, w, 1e-6, x[:1])
    with pytest.raises(RuntimeError, match="d must be on"):
        fused.add_rmsnorm_mx(x, w, 1e-6, x.cpu())
    with pytest.raises(RuntimeError, match="at most 8192"):
        fused.add_rmsnorm_mx(torch.zeros(1, 8224, device="cuda", dtype=BF16), torch.ones(8224, device="cuda"), 1e-6)
    with pytest.raises(ValueError, match="inplace"):
        fused.add_rmsnorm_mx(x.requires_grad_(True), w, 1e-6, x.detach(), inplace=True)


# ------------------------------------------------------------------------------------------------ order
@pytest.mark.parametrize("T,k,E,base,dtype", [
    (1, 1, 1, 0, torch.int32), (1, 8, 256, 0, torch.int32), (8, 8, 256, 0, torch.int64), (33, 3, 7, 2, torch.int32),
    (513, 8, 64, 64, torch.int64), (700, 6, 1000, 0, torch.int32), (1024, 4, 4096, 0, torch.int32), (1400, 6, 12, -3, torch.int32),
    (2100, 8, 40, 0, torch.int64),
])
def test_order(cuda, T, k, E, base, dtype):
    g = torch.Generator().manual_seed(T + k + E)
    ids = torch.randint(base - 2, base + E + 2, (T, k), generator=g).to(dtype)
    ids[:, 0] = base  # one crowded expert
    got = dispatch.expert_order(ids.cuda(), E, base)
    if T * k * E <= 1 << 21:
        want = ref.order(ids, E, base)
    else:
        want = dispatch.expert_order(ids, E, base)
    for a, b in zip(got, want):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)


@pytest.mark.parametrize("T", [511, 513, 1025, 2049, 70000])
def test_order_agrees_with_host_across_cluster_sizes(cuda, T):
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-1, 33, (T, 8), generator=g).int()
    for a, b in zip(dispatch.expert_order(ids.cuda(), 32), dispatch.expert_order(ids, 32)):
        assert torch.equal(a.cpu(), b)


def test_order_empty_masked_and_strided(cuda):
    o = dispatch.expert_order(torch.zeros(0, 4, device="cuda", dtype=torch.int32), 3)
    assert o.offsets.tolist() == [0] * 4 and o.slots.shape == (0, 4) and o.pairs.numel() == 0
    o = dispatch.expert_order(torch.full((5, 2), -1, device="cuda", dtype=torch.int64), 3)
    assert o.offsets.tolist() == [0] * 4 and (o.slots == -1).all() and (o.pairs == -1).all()
    far = torch.tensor([[1 << 40, 2], [-(1 << 40), 0]], device="cuda")
    o = dispatch.expert_order(far, 3)
    assert o.slots.tolist() == [[-1, 1], [-1, 0]] and o.pairs.tolist() == [3, 1, -1, -1]
    wide = torch.randint(0, 5, (40, 6), device="cuda")
    for ids in (wide[:, 2:5], wide[::2], wide.t()):
        for a, b in zip(dispatch.expert_order(ids, 5), dispatch.expert_order(ids.contiguous(), 5)):
            assert torch.equal(a, b)


def routed(T, k, E, masked, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(max(E, k), generator=g)[:k] for _ in range(T)]).int() if T else torch.zeros(0, k).int()
    if masked:
        ids[torch.rand(T, k, generator=g) < masked] = -1
    return dispatch.expert_order(ids.cuda(), max(E, k))


# ------------------------------------------------------------------------------------------------ gather
@pytest.mark.parametrize("T,k,E,H,dtype,masked", [
    (1, 1, 1, 1, BF16, 0), (1, 8, 16, 4096, BF16, 0), (37, 3, 9, 129, BF16, 0.3), (65, 6, 32, 2050, F16, 0.5),
    (20, 2, 4, 77, F32, 0.2), (300, 8, 64, 520, BF16, 0.1), (9, 4, 8, 24, torch.uint8, 0.4), (9, 4, 8, 27, torch.uint8, 1.0),
    (0, 2, 4, 64, BF16, 0),
])
def test_gather_and_gradient(cuda, T, k, E, H, dtype, masked):
    g = gen(T + H)
    order = routed(T, k, E, masked, T)
    x = torch.randint(0, 256, (T, H), device="cuda", generator=g, dtype=torch.uint8) if dtype == torch.uint8 else randn(g, T, H, dtype=dtype)
    rows = dispatch.gather(x, order)
    pairs = order.pairs.long()
    want = torch.where((pairs >= 0)[:, None], x[pairs.clamp_min(0) // k], torch.zeros((), dtype=dtype, device="cuda")) if T else x
    assert torch.equal(rows, want)
    if dtype == torch.uint8:
        return
    x.requires_grad_(True)
    drows = randn(g, T * k, H, dtype=dtype)
    dx, = torch.autograd.grad(dispatch.gather(x, order), x, drows)
    here = (order.slots >= 0)[..., None]
    parts = torch.where(here, drows.to(F64)[order.slots.clamp_min(0).long()], 0.0) if T else drows.to(F64).view(0, k, H)
    ref.check(dx, parts.sum(1), parts.abs().sum(1) * ACC * k, "dx")


def test_gather_strided_unaligned_and_mx(cuda):
    g = gen(5)
    order = routed(50, 4, 8, 0.2, 1)
    wide = randn(g, 100, 300, dtype=BF16)
    for x in (wide[:50, 8:136], wide[:50, 1:130], wide[::2, :128], wide[:50].t().contiguous().t()):
        assert torch.equal(dispatch.gather(x, order), dispatch.gather(x.contiguous(), order))
    for n in (32, 96, 128, 544):
        codes = torch.randint(0, 256, (50, n), device="cuda", dtype=torch.uint8)
        scales = torch.randint(0, 256, (50, n // 32), device="cuda", dtype=torch.uint8)
        a, b = dispatch.gather_mx(codes, scales, order)
        assert torch.equal(a, dispatch.gather(codes, order)) and torch.equal(b, dispatch.gather(scales, order))


# ------------------------------------------------------------------------------------------------ combine
def combine_reference(y, order, weights, residual):
    here = order.slots >= 0
    rows = torch.where(here[..., None], y.to(F64)[order.slots.clamp_min(0).long()], 0.0)
    w = torch.where(here, weights.to(F64) if weights is not None else 1.0, 0.0)[..., None]
    out, mag = (rows * w).sum(1), (rows * w).abs().sum(1)
    if residual is not None:
        out, mag = out + residual.to(F64), mag + residual.to(F64).abs()
    return out, mag, rows, w


@pytest.mark.parametrize("T,k,E,H,dtype,out,masked,weighted,res", [
    (1, 1, 1, 1, BF16, None, 0, True, False), (8, 8, 64, 4096, BF16, F32, 0, True, True), (37, 3, 9, 129, F16, None, 0.3, True, True),
    (64, 6, 32, 2048, BF16, None, 0.5, True, False), (20, 2, 4, 77, F32, None, 0.2, False, True), (33, 11, 16, 264, BF16, F32, 0.1, True, False),
    (40, 4, 8, 512, F16, F32, 1.0, True, True), (5, 20, 32, 40, F16, None, 0, True, False),
])
def test_combine_and_gradients(cuda, T, k, E, H, dtype, out, masked, weighted, res):
    g = gen(T * 3 + H)
    order = routed(T, k, E, masked, T + 1)
    y = randn(g, T * k, H, dtype=dtype)
    weights = torch.rand(T, k, device="cuda", generator=g) if weighted else None
    residual = randn(g, T, H, dtype=out or dtype) if res else None
    want, mag, rows, w = combine_reference(y, order, weights, residual)
    got = dispatch.combine(y, order, weights, residual, out)
    assert got.dtype == (out or dtype)
    ref.check(got, want, mag * ACC * (k + 1), "out")
    leaves = [t.requires_grad_(True) for t in (y, weights, residual) if t is not None]
    dout = randn(g, T, H, dtype=out or dtype)
    grads = dict(zip([n for n, t in (("y", y), ("w", weights), ("r", residual)) if t is not None],
                     torch.autograd.grad(dispatch.combine(y, order, weights, residual, out), leaves, dout)))
    dy = torch.zeros(T * k, H, dtype=F64, device="cuda")
    here = order.slots >= 0
    dy[order.slots[here].long()] = (w * dout.to(F64)[:, None])[here]
    ref.check(grads["y"], dy, dy.abs() * ACC, "dy")
    if weighted:
        prod = rows * dout.to(F64)[:, None]
        ref.check(grads["w"], prod.sum(-1), prod.abs().sum(-1) * ACC * (H ** 0.5 + 8), "dw")
        # difference quotient: the sum is linear in the weights
        v = torch.randn(T, k, device="cuda", dtype=F64, generator=g)
        shift = lambda t: ((rows * (w + t * torch.where(here, v, 0.0)[..., None])).sum(1) * dout.to(F64)).sum()  # noqa: E731
        diff = (shift(1e-3) - shift(-1e-3)) / 2e-3
        assert abs(diff - (grads["w"].to(F64) * v).sum()) <= 1e-4 * (prod.abs().sum(-1) * v.abs()).sum() + 1e-9
    if res:
        assert torch.equal(grads["r"], dout)


def test_combine_ignores_what_masked_pairs_hold(cuda):
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]], device="cuda", dtype=torch.int32)
    order = dispatch.expert_order(ids, 2)
    y = torch.ones(6, 64, device="cuda", dtype=BF16)
    y[3:] = float("nan")  # rows of no pair
    w = torch.ones(3, 2, device="cuda")
    w[0, 1] = w[1, 0] = float("nan")
    w[1, 1] = float("inf")
    out = dispatch.combine(y, order, w)
    assert out.float().tolist() == [[1.0] * 64, [0.0] * 64, [2.0] * 64]
    dy, dw = dispatch.combine_backward(torch.ones(3, 64, device="cuda", dtype=BF16), y, order, w)
    assert (dy[:3] == 1).all() and (dy[3:] == 0).all()
    assert dw.tolist() == [[64.0, 0.0], [0.0, 0.0], [64.0, 64.0]]


def test_combine_strided_rows_repeat_bits(cuda):
    g = gen(8)
    order = routed(60, 4, 8, 0.1, 3)
    wide = randn(g, 480, 400, dtype=BF16)
    w = torch.rand(60, 8, device="cuda", generator=g)
    for y in (wide[:240, 8:264], wide[::2, 1:258], wide[:240].t().contiguous().t()):
        for ww in (w[:, :4], w[:, ::2]):
            a = dispatch.combine(y, order, ww)
            assert torch.equal(a, dispatch.combine(y.contiguous(), order, ww.contiguous()))
            b = dispatch.combine_backward(a, y, order, ww)
            c = dispatch.combine_backward(a, y.contiguous(), order, ww.contiguous())
            # a wide row is summed by other threads than a narrow one: the same values to fp32 rounding
            assert torch.equal(b[0], c[0])
            torch.testing.assert_close(b[1], c[1], rtol=1e-5, atol=1e-4)


def test_dispatch_refusals(cuda):
    ids = torch.zeros(4, 2, device="cuda", dtype=torch.int32)
    with pytest.raises(ValueError, match="num_experts"):
        dispatch.expert_order(ids, 5000)
    with pytest.raises(ValueError, match="int32 or int64"):
        dispatch.expert_order(ids.float(), 4)
    order = dispatch.expert_order(ids, 4)
    x = torch.zeros(4, 64, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="one row per token"):
        dispatch.gather(x[:3], order)
    with pytest.raises(ValueError, match="one row per pair"):
        dispatch.combine(x, order)
    y = torch.zeros(8, 64, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="weights"):
        dispatch.combine(y, order, torch.ones(4, 2, device="cuda", dtype=BF16))
    with pytest.raises(ValueError, match="residual"):
        dispatch.combine(y, order, residual=x.float())
    with pytest.raises(ValueError, match="out_dtype"):
        dispatch.combine(y, order, out_dtype=F16)
    with pytest.raises(RuntimeError, match="must be on"):
        dispatch.combine(y, order, torch.ones(4, 2))
    # a table that no order made reaches no memory outside
    bad = dispatch.ExpertOrder(order.offsets, torch.full_like(order.slots, 1 << 30), order.pairs)
    assert (dispatch.combine(y + 1, bad) == 0).all()


# ------------------------------------------------------------------------------------------------ products
def spread(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


MM = [
    # rows per expert, rows past the last, K, N, type
    ([1], 0, 64, 16, BF16),
    ([5, 0, 3], 0, 8, 8, F16),
    ([128, 128], 0, 256, 512, BF16),
    ([1, 127, 0, 129, 300], 0, 200, 264, BF16),
    ([64, 65, 63, 16, 17, 15], 9, 136, 528, F16),
    ([0, 0, 0], 5, 64, 64, BF16),
    ([700, 1100], 130, 328, 1040, BF16),
    ([2, 0, 1, 0, 0, 4, 1, 0, 33, 70], 0, 512, 256, F16),
    ([1300], 0, 72, 2064, BF16),
]


def mm_inputs(counts, tail, K, N, dtype, seed=0):
    g = gen(seed + K + N + len(counts))
    offsets = spread(counts)
    P = int(offsets[-1]) + tail
    x, w = randn(g, P, K, dtype=dtype), randn(g, len(counts), N, K, dtype=dtype, scale=K ** -0.5)
    return g, x, w, offsets, P


@pytest.mark.parametrize("counts,tail,K,N,dtype", MM)
def test_expert_linear(cuda, counts, tail, K, N, dtype):
    _, x, w, offsets, P = mm_inputs(counts, tail, K, N, dtype)
    if tail:
        x[-tail:] = float("nan")  # rows of no expert reach nothing
    y = grouped.expert_linear(x, w, offsets)
    check_errors(cuda)
    z, s = ref.linear(x, w, offsets)
    ref.check(y, z, s * ACC * K, "y")
    if N % 16 == 0:
        y = grouped.expert_linear(x, w, offsets, activation="swiglu")
        check_errors(cuda)
        I = N // 2
        # |d silu| <= 1.1; exp and the division are within 2^-20
        err = s * ACC * K
        g, u = z[:, :I], z[:, I:]
        sil = ref.swiglu(torch.cat((g, torch.ones_like(g)), 1))
        slack = 1.1 * (u.abs() + err[:, I:]) * err[:, :I] + sil.abs() * err[:, I:] + (sil * u).abs() * 2 ** -20
        ref.check(y, sil * u, slack, "gated")


@pytest.mark.parametrize("counts,tail,K,N,dtype", MM)
def test_expert_linear_backward(cuda, counts, tail, K, N, dtype):
    g, x, w, offsets, P = mm_inputs(counts, tail, K, N, dtype, seed=1)
    dy = randn(g, P, N, dtype=dtype)
    if tail:
        x[-tail:] = float("nan")
        dy[-tail:] = float("inf")
    dx, dw = grouped.expert_linear_backward(dy, x, w, offsets)
    check_errors(cuda)
    rdx, s = ref.linear(dy, w.transpose(1, 2), offsets)
    ref.check(dx, rdx, s * ACC * N, "dx")
    off = offsets.tolist()
    for e in range(len(counts)):
        a, b = off[e], off[e + 1]
        d, v = dy[a:b].to(F64), x[a:b].to(F64)
        ref.check(dw[e], d.T @ v, (d.abs().T @ v.abs()) * ACC * max(1, b - a), f"dw[{e}]")
    only = grouped.expert_linear_backward(dy, x, w, offsets, need_dx=False)
    assert only[0] is None and torch.equal(only[1], dw)


@pytest.mark.parametrize("counts,tail,K,N,dtype", [MM[i] for i in (0, 2, 4, 6)])
def test_gated_autograd(cuda, counts, tail, K, N, dtype):
    g, x, w, offsets, P = mm_inputs(counts, tail, K, N, dtype, seed=2)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = grouped.expert_linear(x, w, offsets, activation="swiglu")
    with torch.no_grad():
        assert torch.equal(y, grouped.expert_linear(x, w, offsets, activation="swiglu"))
    dy = randn(g, P, N // 2, dtype=dtype)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    check_errors(cuda)
    z, s = ref.linear(x.detach(), w.detach(), offsets)
    z = z.requires_grad_(True)
    out = ref.swiglu(z)
    dz, = torch.autograd.grad(out, z, dy.to(F64))
    dz[int(offsets[-1]):] = 0
    rdx, mx = ref.linear(dz, w.detach().transpose(1, 2), offsets)
    u = ref.ROUND[dtype]
    # pre and dz are each rounded to the type (their gradient's slope in pre is at most 1.1 |dy| (1 + |z|)), then the sum
    zz = z.detach().abs()
    slope = 1.1 * torch.cat((dy.to(F64).abs(),) * 2, 1) * (1 + torch.cat((zz[:, N // 2:], zz[:, :N // 2]), 1) + zz)
    off_by = u * dz.abs() + slope * (u * zz + s * ACC * K) * 2
    off_by[int(offsets[-1]):] = 0
    err, _ = ref.linear(off_by, w.detach().abs().transpose(1, 2), offsets)
    ref.check(dx, rdx, err + mx * ACC * N, "dx")
    spans = offsets.tolist()
    for e, (a, b) in enumerate(zip(spans, spans[1:])):
        v = x.detach()[a:b].to(F64)
        ref.check(dw[e], dz[a:b].T @ v, off_by[a:b].T @ v.abs() + dz[a:b].abs().T @ v.abs() * ACC * max(1, b - a), f"dw[{e}]")


@pytest.mark.parametrize("P,I,dtype", [(1, 8, BF16), (37, 136, F16), (700, 2048, BF16), (3, 4104, BF16)])
def test_swiglu_backward(cuda, P, I, dtype):
    g = gen(P)
    pre, dy = randn(g, P, 2 * I, dtype=dtype, scale=3.0), randn(g, P, I, dtype=dtype)
    pre[0, 0], pre[0, 1] = -60000.0, 60000.0
    have = max(1, P - 2)
    offsets = torch.tensor([0, have // 2, have], dtype=torch.int32, device="cuda")
    dz = grouped.swiglu_backward(dy, pre, offsets)
    z = pre.to(F64).requires_grad_(True)
    want, = torch.autograd.grad(ref.swiglu(z), z, dy.to(F64))
    want[have:] = 0
    mag = torch.cat([dy.to(F64).abs() * (1 + pre.to(F64).abs()[:, I:] * (1 + pre.to(F64).abs()[:, :I].clamp_max(30))),
                     dy.to(F64).abs() * pre.to(F64).abs()[:, :I]], 1)
    ref.check(dz, want, mag * 2 ** -20, "dz")
    # central differences along a direction, rows of an expert only
    v = randn(g, have, 2 * I, dtype=F64)
    v[0, :2] = 0
    f = lambda t: (ref.swiglu(pre[:have].to(F64) + t * v) * dy[:have].to(F64)).sum()  # noqa: E731
    diff = (f(1e-5) - f(-1e-5)) / 2e-5
    assert abs(diff - (dz[:have].to(F64) * v).sum()) <= 1.01 * ref.ROUND[dtype] * (want[:have] * v).abs().sum() + 1e-6 * (mag[:have] * v.abs()).sum()


def test_products_strided_rows_and_streams(cuda):
    g = gen(6)
    offsets = spread([70, 3, 200])
    wide = randn(g, 273, 400, dtype=BF16)
    w = randn(g, 3, 64, 128, dtype=BF16)
    want = None
    for x in (wide[:, 8:136], wide[:, 8:136].contiguous(), wide[:, 8:136].t().contiguous().t()):
        y = grouped.expert_linear(x, w, offsets)
        assert want is None or torch.equal(y, want)
        want = y
    odd = wide[:, 1:129]
    assert torch.equal(grouped.expert_linear(odd, w, offsets), grouped.expert_linear(odd.contiguous(), w, offsets))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = grouped.expert_linear(wide[:, 8:136], w, offsets)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, want)
    check_errors(cuda)


def test_products_repeat_and_capture(cuda):
    g, x, w, offsets, P = mm_inputs([300, 0, 45, 129], 0, 256, 512, BF16)
    y = grouped.expert_linear(x, w, offsets, activation="swiglu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg = grouped.expert_linear(x, w, offsets, activation="swiglu")
    for counts in ([300, 0, 45, 129], [0, 474, 0, 0], [1, 1, 1, 471]):
        offsets.copy_(spread(counts))
        graph.replay()
        assert torch.equal(yg, grouped.expert_linear(x, w, offsets, activation="swiglu"))
    offsets.copy_(spread([300, 0, 45, 129]))
    graph.replay()
    assert torch.equal(yg, y)
    check_errors(cuda)


def test_wrong_offsets_stay_inside(cuda):
    """Offsets that decrease or pass the rows are clamped: no row outside x or y is touched."""
    _, x, w, _, P = mm_inputs([100, 60], 0, 64, 64, BF16)
    for bad in ([0, 500, 700], [-5, 80, 60], [90, 10, 160]):
        offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
        assert grouped.expert_linear(x, w, offsets).shape == (P, 64)
        grouped.expert_linear_backward(x, x, w, offsets)
    check_errors(cuda)


def test_products_refusals(cuda):
    x, w = torch.zeros(4, 64, device="cuda", dtype=BF16), torch.zeros(2, 32, 64, device="cuda", dtype=BF16)
    offsets = spread([2, 2])
    with pytest.raises(ValueError, match="activation"):
        grouped.expert_linear(x, w, offsets, activation="gelu")
    with pytest.raises(ValueError, match="multiples of 8"):
        grouped.expert_linear(x[:, :60].contiguous(), w[:, :, :60].contiguous(), offsets)
    with pytest.raises(ValueError, match="multiple of 16"):
        grouped.expert_linear(x, w[:, :24].contiguous(), offsets, activation="swiglu")
    with pytest.raises(ValueError, match="w's type"):
        grouped.expert_linear(x.half(), w, offsets)
    with pytest.raises(ValueError, match="offsets"):
        grouped.expert_linear(x, w, offsets.long())
    with pytest.raises(ValueError, match="offsets"):
        grouped.expert_linear(x, w, offsets[:2])
    with pytest.raises(RuntimeError, match="contiguous"):
        grouped.expert_linear(x, w.transpose(0, 1).contiguous().transpose(0, 1), offsets)
    with pytest.raises(RuntimeError, match="must be on"):
        grouped.expert_linear(x, w, offsets.cpu())
    with pytest.raises(ValueError, match="dy"):
        grouped.expert_linear_backward(x, x, w, offsets)
    assert grouped.expert_linear(x[:0], w, spread([0, 0])).shape == (0, 32)
    dx, dw = grouped.expert_linear_backward(torch.zeros(0, 32, device="cuda", dtype=BF16), x[:0], w, spread([0, 0]))
    assert dx.shape == (0, 64) and (dw == 0).all()


# ------------------------------------------------------------------------------------------------ paths
@pytest.mark.parametrize("rows,n", [(1, 32), (7, 96), (300, 4096), (0, 64)])
def test_mx_dequantize_is_exact(cuda, rows, n):
    codes = torch.randint(0, 256, (rows, n), device="cuda", dtype=torch.uint8)
    codes[codes & 127 == 127] = 0  # no NaN codes
    scales = torch.randint(100, 150, (rows, n // 32), device="cuda", dtype=torch.uint8)
    got = fused.mx_dequantize(codes, scales)
    assert got.dtype == BF16
    assert torch.equal(got.cpu(), fused.mx_dequantize(codes.cpu(), scales.cpu()))


def test_grouped_experts_match_the_expert_loop(cuda):
    from packmla.ops import moe

    g = gen(11)
    T, k, E, H, I = 130, 3, 12, 256, 192
    h = randn(g, T, H, dtype=BF16)
    lw = {"w13": randn(g, E, 2 * I, H, dtype=BF16, scale=H ** -0.5), "w2": randn(g, E, H, I, dtype=BF16, scale=I ** -0.5)}
    ids = torch.rand(T, 2 * E, device="cuda", generator=g).topk(k).indices.int()  # half of them on other ranks
    w = torch.rand(T, k, device="cuda", generator=g)
    ref_out = moe.experts(h, ids, w, lw, 0, E, "bf16")
    got = moe.experts(h, ids, w, lw, 0, E, "bf16", precision="grouped")
    check_errors(cuda)
    assert (got - ref_out).norm() <= 2 ** -7 * ref_out.norm()


def test_block_on_the_gpu_matches_the_cpu(cuda):
    from packmla.training.expert_block import ExpertBlock, fit

    dev = ExpertBlock(128, 64, 8, 2, device="cuda", seed=1)
    cpu = ExpertBlock(128, 64, 8, 2, device="cpu", seed=1)
    for a, b in zip(cpu.parameters(), dev.parameters()):
        a.data.copy_(b.data)
    g = torch.Generator().manual_seed(5)
    x, d, v = (torch.randn(70, 128, generator=g).bfloat16() for _ in range(3))
    grads = []
    for block, where in ((dev, "cuda"), (cpu, "cpu")):
        xr = x.to(where).requires_grad_(True)
        stream, out = block(xr, d.to(where), (torch.arange(70) % 9 != 0).to(where))
        grads.append([t.cpu().double() for t in (out.detach(), *torch.autograd.grad(out, [xr, *block.parameters()], v.to(where)))])
    check_errors(cuda)
    for a, b in zip(*grads):  # both sides round BF16 rows at the same places; sums differ in order
        assert (a - b).norm() <= 2e-2 * b.norm()
    r = fit(tokens=512, hidden=128, inter=64, experts=8, topk=2, steps=30, lr=3e-3, device="cuda")
    assert r["last_loss"] < 0.9 * r["first_loss"]


@pytest.mark.parametrize("E", [376, 384, 385, 500, 750, 768, 1500, 1536, 3000])
def test_order_counters_around_the_shared_memory_default(cuda, E):
    """Counter tables just below, at and above 48 KB (the size a launch may use without asking)."""
    g = torch.Generator().manual_seed(E)
    for T in (70, 1100):
        ids = torch.randint(-1, E, (T, 8), generator=g).int()
        for a, b in zip(dispatch.expert_order(ids.cuda(), E), dispatch.expert_order(ids, E)):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("T,k", [(10000, 1000), (9000, 300), (3, 1024)])
def test_combine_with_many_choices(cuda, T, k):
    """A block's slots and weights stay within the shared memory of a launch at any topk."""
    g = gen(k)
    ids = torch.randint(-1, 40, (T, k), device="cuda", generator=g)
    order = dispatch.expert_order(ids, 40)
    y = randn(g, T * k, 8, dtype=BF16)
    w = torch.rand(T, k, device="cuda", generator=g)
    got = dispatch.combine(y, order, w, out_dtype=F32)
    here = order.slots >= 0
    part = torch.where(here[..., None], y[order.slots.clamp_min(0).long()].to(F64), 0.0) * torch.where(here, w, 0).to(F64)[..., None]
    ref.check(got, part.sum(1), part.abs().sum(1) * ACC * (k + 1), "out")
    with pytest.raises(RuntimeError, match="1024"):
        dispatch.expert_order(torch.zeros(2, 1025, device="cuda", dtype=torch.int32), 4)


def test_broadcast_rows(cuda):
    """One row expanded over many (stride 0): operands are read as the rows they stand for."""
    g = gen(12)
    row, w = randn(g, 1, 64, dtype=BF16), randn(g, 2, 32, 64, dtype=BF16)
    offsets = spread([40, 5])
    x = row.expand(45, 64)
    assert torch.equal(grouped.expert_linear(x, w, offsets), grouped.expert_linear(x.contiguous(), w, offsets))
    dy = randn(g, 1, 32, dtype=BF16).expand(45, 32)
    for a, b in zip(grouped.expert_linear_backward(dy, x, w, offsets),
                    grouped.expert_linear_backward(dy.contiguous(), x.contiguous(), w, offsets)):
        assert torch.equal(a, b)
    norm = torch.ones(64, device="cuda")
    for a, b in zip(fused.add_rmsnorm_mx(x, norm, 1e-6, x, return_h=True),
                    fused.add_rmsnorm_mx(x.contiguous(), norm, 1e-6, x.contiguous(), return_h=True)):
        assert torch.equal(a, b)
    order = routed(45, 2, 4, 0.1, 2)
    assert torch.equal(dispatch.gather(x, order), dispatch.gather(x.contiguous(), order))
    y = row.expand(90, 64)
    out = dispatch.combine(y, order)
    assert torch.equal(out, dispatch.combine(y.contiguous(), order))
    # the gradient of a broadcast input is the sum over its rows
    leaf = row.clone().requires_grad_(True)
    grad, = torch.autograd.grad(dispatch.gather(leaf.expand(45, 64), order), leaf, torch.ones(90, 64, device="cuda", dtype=BF16))
    count = float((order.slots >= 0).sum())
    assert ((grad.float() - count).abs() <= 2 ** -7 * count).all()
    check_errors(cuda)


def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements and 2^32 bytes in the rows: the last rows are where they belong."""
    T, k, H = 70000, 8, 4096
    ids = (torch.arange(T * k, device="cuda") % 11).view(T, k)
    order = dispatch.expert_order(ids, 11)
    x = torch.empty(T, H, device="cuda", dtype=BF16)
    x[:] = (torch.arange(T, device="cuda") % 251)[:, None].to(BF16)
    x[:, -1] = 7
    rows = dispatch.gather(x, order)
    assert rows.numel() > 1 << 31
    for r in (0, 1, T * k // 2, T * k - 2, T * k - 1):
        assert torch.equal(rows[r], x[int(order.pairs[r]) // k])
    out = dispatch.combine(rows, order)
    for t in (0, 1, T // 2, T - 1):
        assert torch.equal(out[t].float(), 8 * x[t].float())
    dy, dw = dispatch.combine_backward(x, rows, order, torch.full((T, k), 2.0, device="cuda"))
    assert torch.equal(dy[T * k - 1], 2 * x[int(order.pairs[-1]) // k])
    last = x[T - 1].double()
    assert abs(dw[T - 1, 0].double() - (last * last).sum()) <= 1e-5 * (last * last).sum()
    del dy, dw, out, x
    # products: rows x outputs past 2^31 elements
    w = torch.zeros(2, H, 64, device="cuda", dtype=BF16)
    w[0, :, 0], w[1, :, 1] = 1, 2
    P = T * k
    offsets = torch.tensor([0, P - 5, P], dtype=torch.int32, device="cuda")
    y = grouped.expert_linear(rows[:, :64], w, offsets)
    check_errors(cuda)
    assert y.numel() > 1 << 31
    for r in (0, P // 2, P - 6, P - 5, P - 1):
        want = rows[r, 0] if r < P - 5 else 2 * rows[r, 1]
        assert (y[r] == want).all()


@pytest.mark.parametrize("activation", [None, "swiglu"])
def test_error_check_between_the_passes(cuda, activation):
    """`check_errors` clears the error word in place; a backward pass after it still runs."""
    g = gen(21)
    x, w = randn(g, 40, 64, dtype=BF16).requires_grad_(True), randn(g, 2, 32, 64, dtype=BF16).requires_grad_(True)
    out = grouped.expert_linear(x, w, spread([30, 10]), activation)
    v = randn(g, *out.shape, dtype=BF16)
    want = torch.autograd.grad(out, (x, w), v, retain_graph=True)
    check_errors(cuda)
    for a, b in zip(torch.autograd.grad(out, (x, w), v), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("E", [2049, 3011, 3012, 3600, 4096])
def test_order_of_many_pairs_and_experts(cuda, E):
    """Where the counters of all sixteen blocks and warps would not fit, fewer of them sort the pairs."""
    g = torch.Generator().manual_seed(E)
    for T in (300, 600, 1100, 9000):
        ids = torch.randint(-1, E, (T, 8), generator=g).int()
        for a, b in zip(dispatch.expert_order(ids.cuda(), E), dispatch.expert_order(ids, E)):
            assert torch.equal(a.cpu(), b)


def test_one_column_of_any_stride(cuda):
    """A [rows, 1] view (top-1 weights, one-wide rows) is dense whatever stride its column reports."""
    order = routed(37, 1, 4, 0.2, 5)
    g = gen(31)
    y, dout = randn(g, 37, 24, dtype=BF16), randn(g, 37, 24, dtype=BF16)
    w = randn(g, 3, 37)[:1].t()
    assert w.stride(1) != 1
    assert torch.equal(dispatch.combine(y, order, w), dispatch.combine(y, order, w.clone(memory_format=torch.contiguous_format)))
    for a, b in zip(dispatch.combine_backward(dout, y, order, w), dispatch.combine_backward(dout, y, order, w.reshape(37).clone()[:, None])):
        assert torch.equal(a, b)
    x = randn(g, 3, 37)[:1].t()
    assert torch.equal(dispatch.gather(x, order), dispatch.gather(x.reshape(37).clone()[:, None], order))


def test_norm_inplace_is_seen_and_checked(cuda):
    """An in-place sum counts as a change of x: a gradient that saved x's old values refuses; overlapping rows are refused."""
    g = gen(41)
    w, d = torch.ones(64, device="cuda"), randn(g, 8, 64, dtype=BF16)
    x = randn(g, 8, 64, dtype=BF16)
    scale = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    y = x * scale  # saves x
    new, *_ = fused.add_rmsnorm_mx(x, w, 1e-6, d, inplace=True)
    assert new.data_ptr() == x.data_ptr()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="apart"):
        fused.add_rmsnorm_mx(x[:1].expand(8, 64), w, 1e-6, d, inplace=True)
    with pytest.raises(RuntimeError, match="apart"):
        fused.add_rmsnorm_mx(torch.as_strided(x, (8, 64), (32, 1)), w, 1e-6, d, inplace=True)
    flat = randn(g, 9 * 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(flat[:512].view(8, 64), w, 1e-6, flat[64:].view(8, 64), inplace=True)
    with torch.inference_mode():
        a = randn(g, 8, 64, dtype=BF16)
        b = a.clone()
        new, *_ = fused.add_rmsnorm_mx(a, w, 1e-6, d, inplace=True)
        assert torch.equal(new, fused.add_rmsnorm_mx(b, w, 1e-6, d)[0])


def test_exchange_and_norm_gradient_repeat_in_a_graph(cuda):
    """Calls whose second kernel starts ahead of the first one's end, captured and replayed on changing inputs."""
    g = gen(51)
    T, k, E, H = 700, 4, 16, 544
    ids = torch.randint(-1, E, (T, k), device="cuda", generator=g)
    x, dh = randn(g, T, H, dtype=BF16), randn(g, T, H, dtype=BF16)
    weights, w = torch.rand(T, k, device="cuda", generator=g), 1 + 0.1 * randn(g, H)

    def run():
        order = dispatch.expert_order(ids, E)
        out = dispatch.combine(dispatch.gather(x, order), order, weights)
        return (*order, out, *dispatch.combine_backward(dh, dispatch.gather(dh, order), order, weights),
                *fused.add_rmsnorm_backward(dh, x, w, 1e-6, out))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for _ in range(20):
        ids.copy_(torch.randint(-1, E, (T, k), device="cuda", generator=g))
        x.copy_(randn(g, T, H, dtype=BF16))
        graph.replay()
        for a, b in zip(got, run()):
            assert torch.equal(a, b)
    check_errors(cuda)


def test_unweighted_combine_keeps_no_rows(cuda):
    """Without weights the gradient does not read the rows: they may be written over before it runs."""
    g = gen(61)
    order = routed(30, 2, 4, 0.2, 7)
    y = randn(g, 60, 40, dtype=F16)
    leaf = y.clone().requires_grad_(True)
    rows = leaf * 1
    out = dispatch.combine(rows, order, out_dtype=F32)
    with torch.no_grad():
        rows.zero_()
    v = randn(g, 30, 40)
    got, = torch.autograd.grad(out, leaf, v)
    assert got.dtype == F16 and torch.equal(got, dispatch.gather(v, order).half())
