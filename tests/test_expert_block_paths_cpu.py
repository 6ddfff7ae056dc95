"""The paths that use the expert block operators: grouped BF16 experts, MXFP8 expert parallelism, the trainable block."""
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

from packmla.config import EngineConfig, ModelConfig
from packmla.models.weights import init_weights
from packmla.ops import fused, moe
from packmla.training.expert_block import ExpertBlock, fit


def inputs(cfg, T, seed):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, cfg.hidden_size, generator=g).bfloat16()
    ids = torch.stack([torch.randperm(cfg.n_routed_experts, generator=g)[:cfg.moe_topk] for _ in range(T)]).int()
    return h, ids, torch.rand(T, cfg.moe_topk, generator=g)


@pytest.mark.parametrize("base,local", [(0, 8), (4, 4)])
def test_grouped_experts_match_the_expert_loop(base, local):
    cfg = ModelConfig.tiny(num_layers=2)
    lw = init_weights(cfg)["layers"][1]
    lw = {"w13": lw["w13"][base:base + local], "w2": lw["w2"][base:base + local]}
    h, ids, w = inputs(cfg, 41, 3)
    ref = moe.experts(h, ids, w, lw, base, local, "bf16")
    got = moe.experts(h, ids, w, lw, base, local, "bf16", precision="grouped")
    assert got.dtype == torch.float32
    # the loop rounds the same intermediate rows; the grouped products also round the outputs to BF16
    assert (got - ref).norm() <= 2 ** -7 * ref.norm()


def test_grouped_precision_is_refused_where_it_cannot_run():
    from packmla.engine.engine import Engine

    cfg = ModelConfig.tiny(num_layers=2)
    lw = init_weights(cfg)["layers"][1]
    h, ids, w = inputs(cfg, 3, 0)
    with pytest.raises(ValueError, match="BF16 experts"):
        moe.experts(h, ids, w, lw, 0, 8, "mxfp4", precision="grouped")
    EngineConfig(kv_cache_format="direct", device="cpu", moe_precision="grouped").validate()
    with pytest.raises(ValueError, match="moe_precision"):
        EngineConfig(kv_cache_format="direct", device="cpu", moe_precision="fp8").validate()
    cfg.expert_format = "mxfp4"
    with pytest.raises(ValueError, match="BF16 experts"):
        Engine.build(cfg, EngineConfig(kv_cache_format="direct", device="cpu", moe_precision="grouped"), device="cpu")


def _mx_rows(h):
    return fused.mx_quantize(h.float())


def _worker(rank, world, port, out_path):
    import torch.distributed as dist

    from packmla.parallel.ep import EPMoE, local_expert_fn

    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        cfg = ModelConfig.tiny(num_layers=2)
        lw = init_weights(cfg, rank, world)["layers"][1]
        h, ids, w = inputs(cfg, 29 + 8 * rank, 50 + rank)
        codes, scales = _mx_rows(h)
        ep = EPMoE(cfg.n_routed_experts, combine_dtype=torch.float32)
        fn = local_expert_fn(lw, ep.expert_base, ep.local_experts, cfg.expert_format)
        got = ep.forward_mx(codes, scales, ids, w, fn, residual=h.float())
        same = ep.forward(fused.mx_dequantize(codes, scales), ids, w, fn)
        masked = ids.clone()
        masked[::3] = -1
        torch.save({"got": got, "same": same, "masked": ep.forward_mx(codes, scales, masked, w, fn),
                    "counts": ep.last_counts}, f"{out_path}.{rank}")
    finally:
        dist.destroy_process_group()


def test_mxfp8_expert_parallelism_equals_bf16_exchange_of_the_same_values(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    out = str(tmp_path / "ep")
    mp.spawn(_worker, args=(2, port, out), nprocs=2, join=True)
    cfg = ModelConfig.tiny(num_layers=2)
    for rank in range(2):
        r = torch.load(f"{out}.{rank}")
        h, ids, w = inputs(cfg, 29 + 8 * rank, 50 + rank)
        torch.testing.assert_close(r["got"], r["same"] + h.float(), rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(r["masked"][1::3], r["same"][1::3], rtol=1e-5, atol=1e-5)
        assert (r["masked"][::3] == 0).all()
        kept = (h.shape[0] - len(range(0, h.shape[0], 3))) * cfg.moe_topk
        assert sum(r["counts"]["sent"]) == kept


def test_mxfp8_experts_find_the_same_codes():
    """The served experts quantize their inputs by the rule of the norm's rows: quantizing the values that MXFP8 rows
    stand for gives those values again, so an MXFP8 exchange changes nothing for them."""
    g = torch.Generator().manual_seed(0)
    h = torch.randn(64, 256, generator=g) * torch.exp(3 * torch.randn(64, 1, generator=g))
    h[5] = 0
    rows = fused.mx_dequantize(*_mx_rows(h))
    assert torch.equal(moe.mx_quant(rows.float()), rows.float())


def plain_block(block, x, d, ids):
    """The block's forward in 64 bits for fixed routing ids, from its parameters."""
    f = torch.float64
    s = x + d
    h = s * (s.square().mean(-1, keepdim=True) + block.eps) ** -0.5 * block.norm.to(f)
    score = torch.sigmoid(h @ block.gate.to(f).T).gather(1, ids.long().clamp_min(0))
    wts = score / score.sum(-1, keepdim=True)
    out = s.clone()
    I = block.w2.shape[2]
    for t in range(x.shape[0]):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if e >= 0:
                z = block.w13[e].to(f) @ h[t]
                out[t] = out[t] + wts[t, j] * (block.w2[e].to(f) @ (z[:I] * torch.sigmoid(z[:I]) * z[I:]))
    return out


def test_block_gradients_match_the_formula_and_differences():
    block = ExpertBlock(32, 16, 4, 2, dtype=torch.float16, seed=1)
    g = torch.Generator().manual_seed(2)
    x, d = (torch.randn(6, 32, generator=g).half() for _ in range(2))
    mask = torch.tensor([True, True, False, True, True, True])
    v = torch.randn(6, 32, generator=g, dtype=torch.float64)
    xr = x.clone().requires_grad_(True)
    stream, out = block(xr, d, mask)
    grads = torch.autograd.grad(out, [xr, *block.parameters()], v.half())
    with torch.no_grad():
        _, _, _, h = fused.add_rmsnorm_mx(x, block.norm, block.eps, d, return_h=True)
        ids, _ = block.route(h, mask)
        s = (x.float() + d.float()).half().double()
        assert torch.allclose(out.double(), plain_block(block, s, torch.zeros_like(s), ids), rtol=2e-2, atol=2e-2)
        assert torch.equal(out[2], stream[2])
        # central difference along a random direction of the stream
        u = torch.randn(6, 32, generator=g, dtype=torch.float64)
        f = lambda t: (plain_block(block, s + t * u, torch.zeros_like(s), ids) * v.half().double()).sum()  # noqa: E731
        diff = (f(1e-6) - f(-1e-6)) / 2e-6
    got = (grads[0].double() * u).sum()
    # FP16 rows (2^-11) through three products and their gradients
    assert abs(got - diff) <= 2e-2 * (grads[0].double().abs() * u.abs()).sum()
    s64 = s.clone().requires_grad_(True)
    params = [p.detach().double().requires_grad_(True) for p in block.parameters()]
    twin = ExpertBlock(32, 16, 4, 2, dtype=torch.float64, seed=1)
    for p, q in zip(twin.parameters(), params):
        p.data = q.data.to(p.dtype) if p.dtype == torch.float32 else q.data
    exact = torch.autograd.grad(plain_block(twin, s64, torch.zeros_like(s64), ids), [s64, *twin.parameters()], v.half().double())
    for a, b in zip(grads, exact):
        assert (a.double() - b.double()).norm() <= 1e-2 * b.double().norm()


def test_fit_lowers_the_loss():
    r = fit(tokens=256, hidden=64, inter=32, experts=4, topk=2, steps=30, lr=3e-3, device="cpu")
    assert r["last_loss"] < 0.8 * r["first_loss"]


def test_block_refusals():
    with pytest.raises(ValueError, match="multiple of 32"):
        ExpertBlock(40, 16, 4, 2)
    with pytest.raises(ValueError, match="topk"):
        ExpertBlock(32, 16, 4, 5)
