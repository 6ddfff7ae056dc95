"""64-bit references of the expert block operators and the error bounds their tests use."""
import torch

F64 = torch.float64
# unit roundoff 2^-p of a type with p significant bits, and half the spacing below the normal range
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
ACC = 2.0 ** -22  # relative error of one fp32 addition or product, truncation included


def check(got, exact, slack, what=""):
    """|got - exact| <= one rounding of the (perturbed) exact value + slack, element by element."""
    u, tiny = ROUND[got.dtype], TINY[got.dtype]
    got, exact = got.detach().to(F64).cpu(), exact.detach().to(F64).cpu()
    assert got.shape == exact.shape, what
    slack = slack.cpu() if isinstance(slack, torch.Tensor) else slack
    bound = u * 1.01 * (exact.abs() + slack) + tiny + slack
    bad = ~((got - exact).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - exact).abs() - bound).max():.3g}"


def norm(x, w, eps, d=None, df=None):
    """(stored stream in f64, h in f64, r)"""
    s = x.float()
    for t in (d, df):
        if t is not None:
            s = s + t.float()
    s = s.to(x.dtype).to(F64)
    r = (s.square().mean(-1, keepdim=True) + eps) ** -0.5
    return s, s * r * w.to(F64), r


def norm_grads(s, w, eps, dh, dres=None):
    n = s.shape[1]
    r = (s.square().mean(-1, keepdim=True) + eps) ** -0.5
    g = dh.to(F64) * w.to(F64)
    dx = r * g - s * r ** 3 / n * (g * s).sum(-1, keepdim=True)
    if dres is not None:
        dx = dx + dres.to(F64)
    return dx, (dh.to(F64) * s * r).sum(0)


def check_mx(codes, scales, h, rel):
    """Codes and scale bytes stand for h (f64) within half an E4M3 step; the scale is the least that holds the
    group's largest magnitude.  `rel`: relative error of the fp32 h they were made from."""
    codes, scales, h = codes.cpu(), scales.cpu(), h.cpu()
    T, n = h.shape
    amax = h.abs().view(T, n // 32, 32).amax(-1).clamp_min(1e-4)
    step = torch.exp2(scales.to(F64) - 127)
    assert (448 * step >= amax * (1 - rel)).all() and (224 * step < amax * (1 + rel)).all()
    v = codes.view(torch.float8_e4m3fn).to(F64)
    want = h / step.repeat_interleave(32, 1)
    # spacing of E4M3: 2^(exponent - 3), subnormals 2^-9; a value that rounds across a binade has the lower spacing
    exponent = torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -6)))
    half = torch.exp2(exponent - 4)
    assert ((v - want).abs() <= half * (1 + 1e-6) + rel * want.abs()).all()


def order(ids, E, base=0):
    """(offsets, slots, pairs) by counting in Python."""
    T, k = ids.shape
    flat = [int(i) - base for i in ids.reshape(-1).tolist()]
    pairs = [p for e in range(E) for p in range(T * k) if flat[p] == e]
    offsets = [0]
    for e in range(E):
        offsets.append(offsets[-1] + sum(1 for f in flat if f == e))
    slots = [-1] * (T * k)
    for r, p in enumerate(pairs):
        slots[p] = r
    pairs = pairs + [-1] * (T * k - len(pairs))
    i32 = dict(dtype=torch.int32)
    return torch.tensor(offsets, **i32), torch.tensor(slots, **i32).view(T, k), torch.tensor(pairs, **i32)


def linear(x, w, offsets):
    """(y, sum of |x w| per output) in f64, rows past the last expert zero."""
    off = offsets.tolist()
    y = torch.zeros(x.shape[0], w.shape[1], dtype=F64, device=x.device)
    s = torch.zeros_like(y)
    for e in range(w.shape[0]):
        a, b = off[e], off[e + 1]
        y[a:b] = x[a:b].to(F64) @ w[e].to(F64).T
        s[a:b] = x[a:b].to(F64).abs() @ w[e].to(F64).abs().T
    return y, s


def swiglu(z):
    g, u = z.chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u  # finite, and of finite slope, at any finite g
