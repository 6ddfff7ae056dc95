"""Cases of the mixture-of-experts block operators: residual add + RMSNorm to MXFP8 rows, rows sorted by
expert and back, and the experts' matrix products, forward and backward.

`run` computes a case in elementary torch operations in 32 bits (`own` false) or through packmla.ops
(`own` true); `exact` computes it in 64 bits from the definitions.  Geometry is the served model's
(hidden 4096, expert intermediate 2048, 256 experts, top 8; 32 local experts on one of 8 ranks) or generic.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6
GROUP = 32          # values that share one MXFP8 scale
TINY = 1e-4         # smallest magnitude an MXFP8 scale covers


def listed():
    return [
        # one decode step of eight requests: the launch is all there is
        {"name": "norm_decode", "op": "norm", "rows": 8, "width": 4096, "type": "bf16", "addends": 2, "train": False},
        # one prefill chunk: the residual, an attention output (bf16) and a routed sum (fp32) into the next block's rows
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "width": 4096, "type": "bf16", "addends": 2, "train": False},
        # a training step on packed sequences: odd row count, a width that fills no power of two, half precision
        {"name": "norm_train_odd", "op": "norm", "rows": 4999, "width": 2080, "type": "f16", "addends": 1, "train": True},
        # routing of one decode step over all experts
        {"name": "dispatch_decode", "op": "dispatch", "tokens": 8, "topk": 8, "experts": 256, "width": 4096, "type": "bf16", "masked": 0.0, "train": False},
        # a rank's 4096 tokens as MXFP8 rows with their scales, to all experts
        {"name": "dispatch_mx_prefill", "op": "dispatch", "tokens": 4096, "topk": 8, "experts": 256, "width": 4096, "type": "mx", "masked": 0.0, "train": False},
        # a training step with padding tokens masked out of the routing; odd token count
        {"name": "dispatch_train_masked", "op": "dispatch", "tokens": 6001, "topk": 6, "experts": 64, "width": 2048, "type": "bf16", "masked": 0.07, "train": True},
        # expert outputs of a decode step back to their tokens, onto the shared expert's output
        {"name": "combine_decode", "op": "combine", "tokens": 8, "topk": 8, "experts": 256, "width": 4096, "type": "bf16", "masked": 0.0, "residual": True, "train": False},
        # a rank's 4096 tokens, weighted sum and the gradients of the rows and of the routing weights
        {"name": "combine_train", "op": "combine", "tokens": 4096, "topk": 8, "experts": 256, "width": 4096, "type": "bf16", "masked": 0.0, "residual": False, "train": True},
        # gate and up products of a decode step on one of eight ranks: a few rows an expert, weights read once
        {"name": "experts_decode", "op": "experts", "rows": 64, "experts": 32, "k": 4096, "n": 4096, "type": "bf16", "gated": True, "train": False},
        # gate and up products of the rows that eight ranks' 4096 tokens send to one rank
        {"name": "experts_prefill", "op": "experts", "rows": 32768, "experts": 32, "k": 4096, "n": 4096, "type": "bf16", "gated": True, "train": False},
        # a plain product with widths that end inside every tile, half precision
        {"name": "experts_ragged", "op": "experts", "rows": 7001, "experts": 24, "k": 1416, "n": 2088, "type": "f16", "gated": False, "train": False},
        # the backward pass of the gate and up products: gradients of the rows and of every expert's weights
        {"name": "experts_train", "op": "experts", "rows": 16384, "experts": 32, "k": 4096, "n": 4096, "type": "bf16", "gated": True, "train": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "dispatch", "combine", "experts", "experts"])
    if op == "norm":
        width = 32 * _log(rng, 2, 256)
        rows = _log(rng, 1, min(16384, 8192 * 4096 // width))
        train = rng.random() < 0.4
        return {"op": op, "rows": rows, "width": width, "type": rng.choice(["bf16", "f16"]), "addends": rng.randint(1 if train else 0, 2),
                "train": train}
    if op in ("dispatch", "combine"):
        train = rng.random() < 0.4
        topk, experts = rng.randint(1, 8), _log(rng, 8, 256)
        kind = rng.choice(["bf16", "f16", "f32"] if op == "combine" or train else ["bf16", "f16", "f32", "mx"])
        width = 32 * _log(rng, 4, 192) if kind == "mx" else _log(rng, 100, 6000)
        if kind != "mx" and rng.random() < 0.7:
            width = -(-width // 8) * 8
        most = 4096 * 8 * 4096 // (topk * width * (2 if kind == "f32" else 1))
        case = {"op": op, "tokens": _log(rng, 1, max(1, min(16384, most))), "topk": topk, "experts": experts, "width": width,
                "type": kind, "masked": rng.choice([0.0, 0.0, rng.uniform(0.01, 0.5)]), "train": train}
        if op == "combine":
            case["residual"] = rng.random() < 0.5
        return case
    gated = rng.random() < 0.5
    k, n = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 512)
    n = n // 16 * 16 if gated else n
    return {"op": op, "rows": _log(rng, 1, 16384), "experts": _log(rng, 1, 32), "k": k, "n": n, "type": rng.choice(["bf16", "f16"]),
            "gated": gated, "train": rng.random() < 0.4}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _route(tokens, topk, experts, masked, g):
    """Distinct experts per token, some far more popular than others; masked tokens have expert -1."""
    logits = torch.randn(tokens, experts, device="cuda", generator=g) + 0.3 * torch.randn(experts, device="cuda", generator=g)
    top = logits.topk(min(topk, experts), dim=-1)
    ids = top.indices.int()
    ids[torch.rand(tokens, device="cuda", generator=g) < masked] = -1
    return ids.contiguous(), torch.softmax(top.values, -1).contiguous()


def _order(ids, experts):
    """(offsets [E + 1], slots [T, k], pairs [T k]): pairs sorted by expert, earlier pairs first; -1 where there is none."""
    flat = ids.reshape(-1)
    key = torch.where(flat >= 0, flat, experts)
    pairs = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=key.device)).sum(0) if key.numel() * experts < (1 << 24) else torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.arange(flat.numel(), device=key.device)
    slots = torch.empty_like(place)
    slots[pairs] = place
    slots = torch.where(flat >= 0, slots, -1)
    pairs = torch.where(place < offsets[-1], pairs, -1)
    return offsets.int(), slots.int().view(ids.shape), pairs.int()


def prepare(case, seed):
    g, op, kind = _generator(seed), case["op"], TYPES.get(case["type"])

    def normal(*shape, scale=1.0, dtype=kind):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    s = {"case": case}
    if op == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = normal(rows, width, scale=4.0)
        s["w"] = 1.0 + 0.2 * normal(width, dtype=torch.float32)
        s["d"] = normal(rows, width) if case["addends"] > 0 else None
        s["df"] = normal(rows, width, scale=0.5, dtype=torch.float32) if case["addends"] > 1 else None
        if case["train"]:
            s["dres"], s["dh"] = normal(rows, width, scale=0.1), normal(rows, width, scale=0.1)
            for name in ("x", "w", "d", "df"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    if op in ("dispatch", "combine"):
        T, E, H = case["tokens"], case["experts"], case["width"]
        s["ids"], s["wts"] = _route(T, case["topk"], E, case["masked"], g)
        k = s["ids"].shape[1]
        if op == "dispatch":
            if case["type"] == "mx":
                s["codes"] = (torch.randn(T, H, device="cuda", generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                s["scales"] = torch.randint(118, 124, (T, H // GROUP), device="cuda", generator=g, dtype=torch.uint8)
            else:
                s["x"] = normal(T, H)
        else:
            s["order"] = _order(s["ids"], E)
            s["y"] = normal(T * k, H)
            s["residual"] = normal(T, H) if case["residual"] else None
        if case["train"]:
            s["grad"] = normal(T * k, H, scale=0.1) if op == "dispatch" else normal(T, H, scale=0.1)
            for name in ("x",) if op == "dispatch" else ("y", "wts", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    P, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
    ids, _ = _route(P, 1, E, 0.0, g)
    s["offsets"], _, pairs = _order(ids, E)
    s["x"] = normal(P, K)
    s["w"] = normal(E, N, K, scale=K ** -0.5)
    # where each row stands in a table with one page of rows per expert (the plain form's layout of the batch)
    owner = ids.reshape(-1)[pairs.long()].long()
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    s["at"] = owner * s["most"] + torch.arange(P, device="cuda") - s["offsets"].long()[owner]
    if case["train"]:
        s["dy"] = normal(P, N // 2 if case["gated"] else N, scale=0.1)
        if case["gated"]:
            s["pre"] = normal(P, N)  # the products that the forward pass kept
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _mx(v, to):
    """Rows [T, n] -> (codes, scales): the smallest power of two that brings each group of 32 within 448."""
    b = v.reshape(v.shape[0], -1, GROUP)
    m, e = torch.frexp(b.abs().amax(-1).clamp_min(TINY))     # m 2^e, m in [0.5, 1)
    e = e - 9 + (m > 0.875).int()                            # 448 = 0.875 * 2^9
    q = torch.ldexp(b, -e[..., None]).reshape(v.shape)
    return (q.to(torch.float8_e4m3fn) if to is None else q), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _norm(s, f, to=None):
    x, w, d, df = s["x"].detach(), s["w"].detach(), s["d"], s["df"]
    r = x.to(f)
    if d is not None:
        r = r + d.detach().to(f)
    if df is not None:
        r = r + df.detach().to(f)
    res = r.to(x.dtype)
    v = res.to(f)
    inv = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = v * inv
    h = n * w.to(f)
    codes, scales = _mx(h, to)
    out = {"stream": res, "codes": codes, "scales": scales, "h": h.to(x.dtype if to is None else f)}
    if s["case"]["train"]:
        gh = s["dh"].to(f)
        gn = gh * w.to(f)
        dx = inv * (gn - n * (gn * n).mean(-1, keepdim=True)) + s["dres"].to(f)
        out["dx"] = dx.to(x.dtype if to is None else f)
        out["dw"] = (gh * n).sum(0)
        if d is not None:
            out["dd"] = out["dx"]
        if df is not None:
            out["ddf"] = dx
    return out


def _table(v, at, pages, most, f):
    t = torch.zeros(pages * most, v.shape[1], dtype=f, device=v.device)
    t[at] = v.to(f)
    return t.view(pages, most, -1)


def _gate(z):
    g, u = z.chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u


def _gate_grad(z, da):
    g, u = z.chunk(2, dim=-1)
    sg = torch.sigmoid(g)
    return torch.cat([da * u * sg * (1 + g * (1 - sg)), da * g * sg], -1)


def _dispatch(s, f, to):
    case = s["case"]
    offsets, slots, pairs = _order(s["ids"], case["experts"])
    k, there = slots.shape[1], (pairs >= 0)[:, None]
    token = pairs.clamp_min(0).long() // k
    out = {"offsets": offsets, "slots": slots, "pairs": pairs}
    if case["type"] == "mx":
        zero = torch.zeros((), dtype=torch.uint8, device=token.device)
        out["codes"] = torch.where(there, s["codes"][token], zero).view(torch.float8_e4m3fn)
        out["scales"] = torch.where(there, s["scales"][token], zero).view(torch.float8_e8m0fnu)
        return out
    x = s["x"].detach()
    out["rows"] = torch.where(there, x.to(f)[token], 0.0).to(to or x.dtype)
    if case["train"]:
        got = s["grad"].to(f)[slots.clamp_min(0).long()]
        out["dx"] = torch.where((slots >= 0)[..., None], got, 0.0).sum(1).to(to or x.dtype)
    return out


def _combine(s, f, to):
    offsets, slots, pairs = s["order"]
    y, wts = s["y"].detach(), s["wts"].detach()
    at = slots.clamp_min(0).long()
    here = slots >= 0
    weight = torch.where(here, wts.to(f), 0.0)
    got = torch.where(here[..., None], y.to(f)[at], 0.0)
    out = (got * weight[..., None]).sum(1)
    if s["residual"] is not None:
        out = out + s["residual"].detach().to(f)
    res = {"out": out.to(to or y.dtype)}
    if s["case"]["train"]:
        grad = s["grad"].to(f)
        dy = torch.zeros(y.shape, dtype=f, device=y.device)
        dy[at[here]] = (weight[..., None] * grad[:, None])[here]
        res["dy"] = dy.to(to or y.dtype)
        res["dweights"] = (got * grad[:, None]).sum(-1)
        if s["residual"] is not None:
            res["dresidual"] = grad.to(to or y.dtype)
    return res


def _experts(s, f, to):
    case = s["case"]
    x, w, at, most = s["x"], s["w"], s["at"], s["most"]
    E, P = w.shape[0], x.shape[0]
    to = to or x.dtype
    xt, wf = _table(x, at, E, most, f), w.to(f)
    if not case["train"]:
        z = torch.bmm(xt, wf.transpose(1, 2)).view(E * most, -1)[at]
        return {"y": (_gate(z) if case["gated"] else z).to(to)}
    dz = _gate_grad(s["pre"].to(f), s["dy"].to(f)) if case["gated"] else s["dy"].to(f)
    zt = _table(dz, at, E, most, f)
    out = {"dx": torch.bmm(zt, wf).view(E * most, -1)[at].to(to), "dw": torch.bmm(zt.transpose(1, 2), xt).to(to)}
    if case["gated"]:
        out["dz"] = dz.to(to)
    return out


PLAIN = {"dispatch": _dispatch, "combine": _combine, "experts": _experts}


def run(state):
    case = state["case"]
    if own:
        return OWN[case["op"]](state)
    with torch.no_grad():
        if case["op"] == "norm":
            return _norm(state, torch.float32)
        return PLAIN[case["op"]](state, torch.float32, None)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    from packmla.ops import fused

    case, x, d, df, w = s["case"], s["x"], s["d"], s["df"], s["w"]
    res, codes, scales, h = fused.add_rmsnorm_mx(x, w, EPS, d, df, return_h=True)
    out = {"stream": res.detach(), "codes": codes.view(torch.float8_e4m3fn), "scales": scales.view(torch.float8_e8m0fnu), "h": h.detach()}
    if case["train"]:
        wanted = [x, w] + [t for t in (d, df) if t is not None]
        out.update(dict(zip(("dx", "dw", "dd", "ddf"), torch.autograd.grad([h, res], wanted, [s["dh"], s["dres"]]))))
    return out


def _own_dispatch(s):
    from packmla.ops import dispatch

    case = s["case"]
    order = dispatch.expert_order(s["ids"], case["experts"])
    out = {"offsets": order.offsets, "slots": order.slots, "pairs": order.pairs}
    if case["type"] == "mx":
        codes, scales = dispatch.gather_mx(s["codes"], s["scales"], order)
        out["codes"], out["scales"] = codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)
        return out
    rows = dispatch.gather(s["x"], order)
    out["rows"] = rows.detach()
    if case["train"]:
        out["dx"], = torch.autograd.grad(rows, s["x"], s["grad"])
    return out


def _own_combine(s):
    from packmla.ops import dispatch

    order = dispatch.ExpertOrder(*s["order"])
    y, wts, residual = s["y"], s["wts"], s["residual"]
    out = dispatch.combine(y, order, wts, residual)
    res = {"out": out.detach()}
    if s["case"]["train"]:
        wanted = [y, wts] + ([residual] if residual is not None else [])
        res.update(dict(zip(("dy", "dweights", "dresidual"), torch.autograd.grad(out, wanted, s["grad"]))))
    return res


def _own_experts(s):
    from packmla.ops import grouped

    case, x, w, offsets = s["case"], s["x"], s["w"], s["offsets"]
    if not case["train"]:
        return {"y": grouped.expert_linear(x, w, offsets, activation="swiglu" if case["gated"] else None)}
    dz = grouped.swiglu_backward(s["dy"], s["pre"], offsets) if case["gated"] else s["dy"]
    dx, dw = grouped.expert_linear_backward(dz, x, w, offsets)
    out = {"dx": dx, "dw": dw}
    if case["gated"]:
        out["dz"] = dz
    return out


OWN = {"norm": _own_norm, "dispatch": _own_dispatch, "combine": _own_combine, "experts": _own_experts}


# ------------------------------------------------------------------------------------------------ what cannot be done without
def work(case):
    op, e = case["op"], {"bf16": 2, "f16": 2, "f32": 4, "mx": 1}[case["type"]]
    if op == "norm":
        v, a = case["rows"] * case["width"], case["addends"]
        b = v * (e + (e if a > 0 else 0) + (4 if a > 1 else 0)) + 4 * case["width"]     # x, d, df, w
        b += v * ((e if a else 0) + 1 + e) + v // GROUP                                  # stream, codes, h, scales
        f = 8 * v
        if case["train"]:
            b += v * (2 * e + e + (4 if a > 1 else 0)) + 4 * case["width"]               # dh, dres, dx (also dd's), ddf, dw
            f += 10 * v
        return {"bytes": b, "flops": f}
    if op in ("dispatch", "combine"):
        T, k, E, H = case["tokens"], min(case["topk"], case["experts"]), case["experts"], case["width"]
        row = H + H // GROUP if case["type"] == "mx" else H * e
        one, all_ = T * row, T * k * row
        if op == "dispatch":
            b = 4 * T * k * 3 + 4 * (E + 1) + one + all_                                 # ids, slots, pairs, offsets, x, rows
            return {"bytes": b + (all_ + one if case["train"] else 0), "flops": T * k * H if case["train"] else T * k}
        b = all_ + one * (2 if case["residual"] else 1) + 8 * T * k                      # y, residual, out, slots, weights
        f = 2 * T * k * H
        if case["train"]:
            b += one + all_ + 4 * T * k                                                  # grad, dy, dweights
            f += 3 * T * k * H
        return {"bytes": b, "flops": f}
    P, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
    used = min(E, P)                                                                     # experts that rows can reach
    if not case["train"]:
        return {"bytes": e * (P * K + used * N * K + P * (N // 2 if case["gated"] else N)), "flops": 2 * P * N * K}
    dy = P * (N // 2 + 2 * N) if case["gated"] else P * N                                # dact, pre, dz; or dy
    return {"bytes": e * (dy + 2 * P * K + used * N * K + E * N * K), "flops": 4 * P * N * K}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_mx(h):
    """Codes before their rounding, and the scales: the least e with amax <= 448 * 2^e, amax at least 1e-4."""
    T, n = h.shape
    amax = h.view(T, n // GROUP, GROUP).abs().max(-1).values
    amax = torch.maximum(amax, torch.full_like(amax, TINY))
    e = torch.ceil(torch.log2(amax / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e)  # a logarithm that came out just above a whole number
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1, e)
    return h / torch.exp2(e).repeat_interleave(GROUP, 1), torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    op, f = case["op"], torch.float64
    with torch.no_grad():
        if op == "norm":
            stream = s["x"].to(f)
            for name in ("d", "df"):
                if s[name] is not None:
                    stream = stream + s[name].to(f)
            stored = stream.to(s["x"].dtype).to(f)
            n, w = case["width"], s["w"].to(f)
            rms = torch.sqrt((stored * stored).sum(1) / n + EPS)[:, None]
            h = stored / rms * w
            codes, scales = _exact_mx(h)
            out = {"stream": stream, "codes": codes, "scales": scales, "h": h}
            if case["train"]:
                a = s["dh"].to(f)
                dot = (a * w * stored).sum(1, keepdim=True)
                dx = a * w / rms - stored * dot / (n * rms ** 3) + s["dres"].to(f)
                out["dx"], out["dw"] = dx, (a * stored / rms).sum(0)
                if s["d"] is not None:
                    out["dd"] = dx
                if s["df"] is not None:
                    out["ddf"] = dx
            return out
        if op == "dispatch":
            if case["type"] == "mx" or not case["train"]:
                return None  # whole numbers and copies
            T, k = s["ids"].shape
            _, slots, _ = _order(s["ids"], case["experts"])
            dx = torch.zeros(T, case["width"], dtype=f, device="cuda")
            for j in range(k):
                here = torch.nonzero(slots[:, j] >= 0)[:, 0]
                dx[here] += s["grad"][slots[here, j].long()].to(f)
            return {"offsets": None, "slots": None, "pairs": None, "rows": None, "dx": dx}
        if op == "combine":
            _, slots, _ = s["order"]
            T, k = slots.shape
            out = s["residual"].to(f) if s["residual"] is not None else torch.zeros(T, case["width"], dtype=f, device="cuda")
            out = out.clone()
            grad = s["grad"].to(f) if case["train"] else None
            dy = torch.zeros(s["y"].shape, dtype=f, device="cuda") if case["train"] else None
            dw = torch.zeros(T, k, dtype=f, device="cuda")
            for j in range(k):
                here = torch.nonzero(slots[:, j] >= 0)[:, 0]
                at, a = slots[here, j].long(), s["wts"][here, j].to(f)[:, None]
                rows = s["y"][at].to(f)
                out[here] += a * rows
                if case["train"]:
                    dw[here, j] = (rows * grad[here]).sum(1)
                    dy[at] = a * grad[here]
            res = {"out": out}
            if case["train"]:
                res.update(dy=dy, dweights=dw)
                if s["residual"] is not None:
                    res["dresidual"] = grad
            return res
        off = s["offsets"].tolist()
        P, E, K, N = case["rows"], case["experts"], case["k"], case["n"]
        x, w = s["x"], s["w"]
        if not case["train"]:
            y = torch.empty(P, N // 2 if case["gated"] else N, dtype=f, device="cuda")
            for i in range(E):
                z = x[off[i]:off[i + 1]].to(f) @ w[i].to(f).T
                y[off[i]:off[i + 1]] = z[:, :N // 2] / (1 + torch.exp(-z[:, :N // 2])) * z[:, N // 2:] if case["gated"] else z
            return {"y": y}
        dz = s["dy"].to(f)
        if case["gated"]:
            gate, up = s["pre"][:, :N // 2].to(f), s["pre"][:, N // 2:].to(f)
            sg = 1 / (1 + torch.exp(-gate))
            dz = torch.cat([dz * up * (sg + gate * sg * (1 - sg)), dz * gate * sg], 1)
        dx = torch.empty(P, K, dtype=f, device="cuda")
        dw = torch.empty(E, N, K, dtype=f, device="cuda")
        for i in range(E):
            part = dz[off[i]:off[i + 1]]
            dx[off[i]:off[i + 1]] = part @ w[i].to(f)
            dw[i] = part.T @ x[off[i]:off[i + 1]].to(f)
        out = {"dx": dx, "dw": dw}
        if case["gated"]:
            out["dz"] = dz
        return out
