"""Expert block operators on CPU tensors at the edges of their contracts."""
import pytest
import torch

import expert_block_reference as ref
from expert_block_reference import ACC, F64
from packmla.ops import fused, grouped

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("table", [[4, 10], [3, 3, 8, 11], [12, 12]])
def test_rows_before_the_first_expert(table):
    """A table that starts past row 0 (some experts of a larger one): the rows before it belong to nobody."""
    g = torch.Generator().manual_seed(len(table))
    P, E, K, N = 12, len(table) - 1, 24, 32
    offsets = torch.tensor(table, dtype=torch.int32)
    x, dy, w = (torch.randn(*s, generator=g).to(BF16) for s in ((P, K), (P, N), (E, N, K)))
    nobody = torch.ones(P, dtype=torch.bool)
    nobody[table[0]:table[-1]] = False
    x[nobody], dy[nobody] = float("nan"), float("inf")
    z, s = ref.linear(x, w, offsets)
    ref.check(grouped.expert_linear(x, w, offsets), z, s * ACC * K, "y")
    dx, dw = grouped.expert_linear_backward(dy, x, w, offsets)
    rdx, s = ref.linear(dy, w.transpose(1, 2), offsets)
    ref.check(dx, rdx, s * ACC * N, "dx")
    for e, (a, b) in enumerate(zip(table, table[1:])):
        ref.check(dw[e], dy[a:b].to(F64).T @ x[a:b].to(F64), (dy[a:b].to(F64).abs().T @ x[a:b].to(F64).abs()) * ACC * P, "dw")
    assert (grouped.expert_linear(x, w, offsets, activation="swiglu")[nobody] == 0).all()
    assert (grouped.swiglu_backward(dy[:, :N // 2], dy, offsets)[nobody] == 0).all()


@pytest.mark.parametrize("dtype,first", [(BF16, 3), (F32, 0)])
def test_mx_dequantize_over_every_code_and_scale(dtype, first):
    """code x 2^(scale - 127), rounded once where the type cannot hold it; scale byte 255 is NaN."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 8)
    value = codes.view(torch.float8_e4m3fn).to(F64) * torch.exp2(torch.arange(256, dtype=F64) - 127)[:, None]
    value[255] = float("nan")
    want = value.float().to(dtype)
    got = fused.mx_dequantize(codes, scales, dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    held = ~value[first:247].isnan()
    assert torch.equal(want[first:247][held].to(F64), value[first:247][held])  # exact there


def test_mx_quantize_of_infinities_and_nan():
    """Beside a NaN the finite values keep their codes and scale; infinities stay infinite."""
    g = torch.Generator().manual_seed(1)
    h = 3 * torch.randn(4, 96, generator=g)
    codes, scales = fused.mx_quantize(h)
    bad = h.clone()
    bad[0, 5], bad[1, 40], bad[2, 70], bad[2, 71] = float("nan"), float("inf"), -float("inf"), float("nan")
    bad[3] = float("nan")
    got, gs = fused.mx_quantize(bad)
    small = h[0, :32].abs().amax() == h[0, 5].abs()  # the NaN took the group's largest value away
    assert not small and gs[0, 0] == scales[0, 0]
    keep = torch.arange(96) != 5
    assert torch.equal(got[0, keep], codes[0, keep]) and got[0, 5] & 127 == 127
    v = fused.mx_dequantize(got, gs)
    assert v[1, 40] == float("inf") and (v[1, 32:40] == 0).all() and torch.equal(got[1, :32], codes[1, :32])
    assert v[2, 70] == -float("inf") and v[2, 71].isnan() and v[2, 72:].eq(0).all()
    assert (got[3] & 127 == 127).all()


def test_requantizing_keeps_values_not_codes():
    """What MXFP8 rows stand for is kept when quantized again; a maximum rounded down to 224 2^e takes the next smaller
    scale then, and every code of its group changes."""
    h = torch.zeros(2, 32)
    h[0, 0], h[0, 1] = 225.0, 3.0
    h[1] = torch.linspace(-300, 300, 32)
    codes, scales = fused.mx_quantize(h)
    values = fused.mx_dequantize(codes, scales)
    again, smaller = fused.mx_quantize(values.float())
    assert torch.equal(fused.mx_dequantize(again, smaller), values)
    assert scales.tolist() == [[127], [127]] and smaller.tolist() == [[126], [127]]
    assert (again[0, :2] != codes[0, :2]).all() and torch.equal(again[1], codes[1])
