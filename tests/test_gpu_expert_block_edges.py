"""Expert block kernels at the edges of their contracts, against 64-bit references."""
import sys
from concurrent.futures import ThreadPoolExecutor

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


# ------------------------------------------------------------------------------------------------ tables
def check_products(dy, x, w, offsets, rows):
    """Products and gradients against the reference on `rows`, the table they have to follow."""
    N, K = w.shape[1:]
    z, s = ref.linear(x, w, rows)
    ref.check(grouped.expert_linear(x, w, offsets), z, s * ACC * K, "y")
    dx, dw = grouped.expert_linear_backward(dy, x, w, offsets)
    rdx, s = ref.linear(dy, w.transpose(1, 2), rows)
    ref.check(dx, rdx, s * ACC * N, "dx")
    for e, (a, b) in enumerate(zip(rows.tolist(), rows.tolist()[1:])):
        d, v = dy[a:b].to(F64), x[a:b].to(F64)
        ref.check(dw[e], d.T @ v, (d.abs().T @ v.abs()) * ACC * max(1, b - a), f"dw[{e}]")
    check_errors(x.device)


TABLES = [[4, 10], [1, 1, 340], [130, 130, 300, 333], [300, 300, 300], [7, 263, 270, 300], [340, 340]]


@pytest.mark.parametrize("K,N,dtype", [(64, 32, BF16), (200, 528, F16)])
@pytest.mark.parametrize("table", TABLES)
def test_rows_before_the_first_expert(cuda, table, K, N, dtype):
    """A table that starts past row 0 (some experts of a larger one): the rows before it belong to nobody."""
    P, E = 340, len(table) - 1
    g = gen(len(table) + K)
    offsets = torch.tensor(table, dtype=torch.int32, device="cuda")
    x, dy = randn(g, P, K, dtype=dtype), randn(g, P, N, dtype=dtype)
    w = randn(g, E, N, K, dtype=dtype, scale=K ** -0.5)
    nobody = torch.ones(P, dtype=torch.bool, device="cuda")
    nobody[table[0]:table[-1]] = False
    x[nobody] = float("nan")
    dy[nobody] = float("inf")
    check_products(dy, x, w, offsets, offsets)
    y = grouped.expert_linear(x, w, offsets, activation="swiglu")
    assert (y[nobody] == 0).all() and y.isfinite().all()
    assert (grouped.swiglu_backward(dy[:, :N // 2], dy, offsets)[nobody] == 0).all()


def test_experts_of_a_larger_table(cuda):
    """offsets[a : b + 1] is the table of experts a .. b: their rows give what the whole table gives, with gradients."""
    g = gen(3)
    table = torch.tensor([0, 40, 300, 300, 420, 500], dtype=torch.int32, device="cuda")
    x, w = randn(g, 500, 96, dtype=BF16), randn(g, 5, 64, 96, dtype=BF16, scale=0.1)
    part = table[1:5]
    for activation in (None, "swiglu"):
        whole = grouped.expert_linear(x, w, table, activation)
        xr, wr = x.clone().requires_grad_(True), w[1:4].clone().requires_grad_(True)
        y = grouped.expert_linear(xr, wr, part, activation)
        assert torch.equal(y[40:420], whole[40:420])
        assert (y[:40] == 0).all() and (y[420:] == 0).all()
        dx, dw = torch.autograd.grad(y, [xr, wr], torch.ones_like(y))
        assert (dx[:40] == 0).all() and (dx[420:] == 0).all()
        full = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        want = torch.autograd.grad(grouped.expert_linear(*full, table, activation), full, torch.ones_like(whole))
        assert torch.equal(dx[40:420], want[0][40:420]) and torch.equal(dw, want[1][1:4])
    check_errors(cuda)


@pytest.mark.parametrize("K,N,dtype", [(64, 64, BF16), (136, 264, F16)])
@pytest.mark.parametrize("bad", [[0, 500, 700], [-5, 80, 60], [90, 10, 160], [30, -3, 400], [900, 0, 7], [-9, -8, -7]])
def test_wrong_tables_are_clamped(cuda, bad, K, N, dtype):
    """A table that decreases or leaves the rows acts as its running maximum within them; no row around x or dy is read."""
    P, pad = 160, 300
    g = gen(K)
    big_x = torch.full((P + 2 * pad, K), float("nan"), device="cuda", dtype=dtype)
    big_dy = torch.full((P + 2 * pad, N), float("nan"), device="cuda", dtype=dtype)
    x, dy = big_x[pad:pad + P], big_dy[pad:pad + P]
    x.copy_(randn(g, P, K, dtype=dtype))
    dy.copy_(randn(g, P, N, dtype=dtype))
    w = randn(g, 2, N, K, dtype=dtype, scale=K ** -0.5)
    offsets = torch.tensor(bad, dtype=torch.int32, device="cuda")
    check_products(dy, x, w, offsets, offsets.clamp(0, P).cummax(0).values)


def test_accumulators_handed_back_tile_after_tile(cuda):
    """Many short tiles a CTA pair, each in the columns that the one before last left: the same bits every time."""
    g = gen(9)
    E, P, K, N = 64, 64 * 70 + 11, 64, 2048
    offsets = (torch.arange(E + 1, device="cuda") * 70).int()
    x, w = randn(g, P, K, dtype=BF16), randn(g, E, N, K, dtype=BF16, scale=K ** -0.5)
    z, s = ref.linear(x, w, offsets)
    want = grouped.expert_linear(x, w, offsets)
    ref.check(want, z, s * ACC * K, "y")
    for _ in range(200):
        assert torch.equal(grouped.expert_linear(x, w, offsets), want)
    check_errors(cuda)


# ------------------------------------------------------------------------------------------------ host threads
def together(*calls, times=20000):
    """Every call from a thread and on a stream of its own, many times and closely interleaved; raises what any raised."""
    def loop(call):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(times):
                call()
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)
    try:
        with ThreadPoolExecutor(len(calls)) as pool:
            for done in [pool.submit(loop, c) for c in calls]:
                done.result()
    finally:
        sys.setswitchinterval(interval)


def test_calls_of_two_threads_with_other_sizes(cuda):
    """A launch's shared memory limit belongs to the kernel, not to the call: a smaller call of another thread must
    not lower it between the larger one's request and its launch."""
    ids = torch.zeros(4096, 8, dtype=torch.int32, device="cuda")
    together(lambda: dispatch.expert_order(ids[:64], 4000), lambda: dispatch.expert_order(ids[:512], 500))
    g = gen(1)
    wide, narrow = randn(g, 4, 8192, dtype=BF16), randn(g, 4, 4096, dtype=BF16)
    w = torch.ones(8192, device="cuda")
    together(lambda: fused.add_rmsnorm_backward(wide, wide, w, 1e-6, wide),
             lambda: fused.add_rmsnorm_backward(narrow, narrow, w[:4096], 1e-6))
    x = randn(g, 8, 8, dtype=BF16)
    many, one = torch.zeros(1024, 8, 8, device="cuda", dtype=BF16), torch.zeros(1, 8, 8, device="cuda", dtype=BF16)
    table = torch.zeros(1025, device="cuda", dtype=torch.int32)
    together(lambda: grouped.expert_linear(x, many, table), lambda: grouped.expert_linear(x, one, table[:2]))
    check_errors(cuda)


# ------------------------------------------------------------------------------------------------ in place
def test_inplace_norm_and_operands_in_its_memory(cuda):
    """Rows of a wider buffer: addends in other columns or rows of it are read, ones that x writes over are refused, and
    where the strides do not tell, the addend is copied first."""
    g = gen(5)
    w = 1 + 0.1 * randn(g, 64)

    def both(make):
        """make(buffer) -> x, d, df, w: in place against the same sums on copies."""
        buf = randn(g, 40, 256, dtype=BF16)
        want = fused.add_rmsnorm_mx(*call_args(*(t.clone() if t is not None else None for t in make(buf))))
        x, *rest = make(buf)
        keep = buf.clone()
        new, codes, scales, _ = fused.add_rmsnorm_mx(*call_args(x, *rest), inplace=True)
        assert new.data_ptr() == x.data_ptr()
        assert torch.equal(x, want[0]) and torch.equal(codes, want[1]) and torch.equal(scales, want[2])
        changed = buf != keep
        x.fill_(7)
        keep[buf == 7] = 7
        assert not (changed & (keep != 7)).any()  # nothing but x was written

    def call_args(x, d, df, weight):
        return x, weight, 1e-6, d, df

    def floats(t):  # the same memory as fp32 rows
        return t.view(F32)

    both(lambda b: (b[:, :64], b[:, 64:128], None, w))
    both(lambda b: (b[::2, :64], b[1::2, :64], None, w))
    both(lambda b: (b[:, 64:128], b[:, :64], floats(b)[:, 64:], w))
    both(lambda b: (b[:20, 8:72], b[20:, 8:72], floats(b)[20:, 64:], w))
    both(lambda b: (b[:10, :64], b[::4, 128:192], None, w))       # other steps: copied
    both(lambda b: (b[::4, :64], b[:10, 128:192], None, w))
    both(lambda b: (b[:, :64], b[:, 64:128], None, floats(b)[3, 64:]))
    both(lambda b: (b[3:4, :64], b[3:4, 64:128], floats(b)[3:4, 64:], w))

    buf = randn(g, 40, 256, dtype=BF16)
    keep = buf.clone()
    x = buf[1:-1, :64]
    for d in (buf[:-2, :64], buf[2:, :64], buf[1:-1, 32:96], buf[2:, 56:120], buf[1:-1, 8:72]):
        with pytest.raises(RuntimeError, match="overlap"):
            fused.add_rmsnorm_mx(x, w, 1e-6, d, inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(x, w, 1e-6, None, floats(buf)[1:-1, :64], inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(x, w, 1e-6, None, floats(buf)[:-2, 16:80], inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(x[:1], floats(buf)[1, 16:80], 1e-6, x[:1], inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(x[:1], w, 1e-6, buf[1:2, 8:72], inplace=True)
    wrap = torch.as_strided(buf, (30, 64), (256, 1), 256 + 224)  # columns 224 .. 287: the next row's first 32
    with pytest.raises(RuntimeError, match="overlap"):
        fused.add_rmsnorm_mx(buf[1:31, :64], w, 1e-6, wrap, inplace=True)
    assert torch.equal(buf, keep)
    want = fused.add_rmsnorm_mx(x.clone(), w, 1e-6, x.clone())
    new, codes, *_ = fused.add_rmsnorm_mx(x, w, 1e-6, x, inplace=True)  # x on itself
    assert torch.equal(new, want[0]) and torch.equal(codes, want[1])


# ------------------------------------------------------------------------------------------------ tangents
def test_tangents_are_refused(cuda):
    """No operator has a forward-mode derivative: an input with a tangent is refused, not answered without one."""
    from torch.autograd import forward_ad

    g = gen(2)
    x, w = randn(g, 6, 64, dtype=BF16), torch.ones(64, device="cuda")
    d, df = randn(g, 6, 64, dtype=BF16), randn(g, 6, 64)
    order = dispatch.expert_order(torch.arange(6, device="cuda").view(3, 2), 6)
    weights, residual = torch.rand(3, 2, device="cuda", generator=g), randn(g, 3, 64, dtype=BF16)
    mats = randn(g, 6, 32, 64, dtype=BF16)
    dy, pre, da = randn(g, 6, 32, dtype=BF16), randn(g, 6, 64, dtype=BF16), randn(g, 6, 32, dtype=BF16)
    calls = [
        (lambda *t: fused.add_rmsnorm_mx(t[0], t[1], 1e-6, t[2], t[3]), (x, w, d, df)),
        (lambda *t: fused.add_rmsnorm_mx(t[0].clone(), t[1], 1e-6, t[2], t[3], inplace=True), (x, w, d, df)),
        (lambda *t: fused.add_rmsnorm_backward(t[0], t[1], t[2], 1e-6, t[3]), (d, x, w, d)),
        (lambda t: dispatch.gather(t, order), (residual,)),
        (lambda *t: dispatch.combine(t[0], order, t[1], t[2]), (x, weights, residual)),
        (lambda *t: dispatch.combine_backward(t[0], t[1], order, t[2]), (residual, x, weights)),
        (lambda *t: grouped.expert_linear(t[0], t[1], order.offsets), (x, mats)),
        (lambda *t: grouped.expert_linear_backward(t[0], t[1], t[2], order.offsets), (dy, x, mats)),
        (lambda *t: grouped.swiglu_backward(t[0], t[1], order.offsets), (da, pre)),
    ]
    for call, inputs in calls:
        call(*inputs)
        with forward_ad.dual_level():
            call(*inputs)  # a level alone changes nothing
            for i, t in enumerate(inputs):
                dual = [forward_ad.make_dual(u, torch.ones_like(u)) if j == i else u for j, u in enumerate(inputs)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
    with forward_ad.dual_level():  # where a gradient is recorded too
        dual = forward_ad.make_dual(residual.clone().requires_grad_(True), torch.ones_like(residual))
        for call in (lambda t: dispatch.gather(t, order), lambda t: dispatch.combine(x, order, weights, t)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)


# ------------------------------------------------------------------------------------------------ MXFP8 values
def test_mx_dequantize_over_every_code_and_scale(cuda):
    """code x 2^(scale - 127), rounded once where BF16 cannot hold it (scale bytes 0 to 2 and from 247); 255 is NaN."""
    codes = torch.arange(256, device="cuda", dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, device="cuda", dtype=torch.uint8)[:, None].repeat(1, 8)
    value = codes.view(torch.float8_e4m3fn).to(F64) * torch.exp2(torch.arange(256, device="cuda", dtype=F64) - 127)[:, None]
    value[255] = float("nan")
    want = value.float().bfloat16()
    for got in (fused.mx_dequantize(codes, scales), fused.mx_dequantize(codes.cpu(), scales.cpu()).cuda()):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    held = ~value[3:247].isnan()
    assert torch.equal(want[3:247][held].to(F64), value[3:247][held])  # exact there


def test_rows_with_infinities_and_nan_match_the_host(cuda):
    """Groups that hold infinities or NaN: finite values keep their codes beside a NaN, and infinities stay infinite."""
    h = 1 + (torch.arange(96).float().view(1, 96) + 0.3) / 64
    w = h[0].clone()
    w[5], w[40], w[70], w[71] = float("nan"), float("inf"), -float("inf"), float("nan")
    x = torch.ones(3, 96, dtype=BF16)
    x[2, 9] = float("nan")
    got = fused.add_rmsnorm_mx(x.cuda(), w.cuda(), 0.0)
    want = fused.add_rmsnorm_mx(x, w, 0.0)
    nan = want[1] & 127 == 127
    assert torch.equal(got[1].cpu() & 127 == 127, nan) and torch.equal(got[1].cpu()[~nan], want[1][~nan])
    assert torch.equal(got[2].cpu(), want[2])


# ------------------------------------------------------------------------------------------------ paths
def test_exchange_of_mx_rows_matches_the_host(cuda):
    """`EPMoE.forward_mx` of one rank, its experts through the served path ("grouped" products), with masked tokens."""
    from packmla.parallel.ep import EPMoE, local_expert_fn

    g = torch.Generator().manual_seed(4)
    T, E, k, H, I = 70, 6, 2, 128, 64
    lw = {"w13": (torch.randn(E, 2 * I, H, generator=g) * H ** -0.5).to(BF16), "w2": (torch.randn(E, H, I, generator=g) * I ** -0.5).to(BF16)}
    h = torch.randn(T, H, generator=g)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    ids[::7] = -1
    weights, residual = torch.rand(T, k, generator=g), torch.randn(T, H, generator=g)
    codes, scales = fused.mx_quantize(h)
    out = []
    for dev in ("cpu", "cuda"):
        ep = EPMoE(E)
        fn = local_expert_fn({n: t.to(dev) for n, t in lw.items()}, 0, E, "bf16", precision="grouped")
        out.append(ep.forward_mx(codes.to(dev), scales.to(dev), ids.to(dev), weights.to(dev), fn, residual.to(dev)).cpu())
    check_errors(cuda)
    assert torch.equal(out[1][::7], residual[::7])
    # both sides round rows to BF16 at the same places; the products' sums differ in order
    assert (out[1] - out[0]).norm() <= 2 ** -7 * (out[0] - residual).norm()


def test_engine_with_grouped_experts_in_a_decode_graph(cuda):
    """The grouped products in the served model: captured decode steps give the eager ones' tokens."""
    from helpers import small_gpu_config
    from packmla.config import EngineConfig
    from packmla.engine.engine import Engine, SamplingParams
    from packmla.models.weights import init_weights

    cfg = small_gpu_config(expert_format="bf16")
    W = init_weights(cfg, device=cuda, seed=7)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (90, 33)]
    outs = []
    for graphs in (False, True):
        ecfg = EngineConfig(kv_cache_format="direct", max_running_requests=2, cuda_graph_bs=[1, 2], chunked_prefill_size=64,
                            moe_precision="grouped", disable_cuda_graph=not graphs)
        eng = Engine.build(cfg, ecfg, cuda, max_context=1024, max_requests=2, kv_bytes=64 << 20, weights=W)
        if graphs:
            eng.runner.capture()
        outs.append(eng.generate(prompts, SamplingParams(max_new_tokens=6)))
        eng.runner.release()
    check_errors(cuda)
    assert outs[0] == outs[1]
