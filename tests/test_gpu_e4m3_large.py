"""The 8-bit norm, the projections over codes and the codes' read-back where results have more than 2^31 elements, and the
same call twice."""

import pytest
import torch

from forgeserve_amd import ops
from test_gpu_linear_e4m3 import BF16, DEV, F16, block_half, close, close_codes, decoded, operands, wanted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gated", [False, True])
def test_products(gated):
    m, n, k = 70001, 32768, 128
    x, w, bias, _ = operands(16, n, k, gated, BF16)
    x = x.repeat(-(-m // 16), 1)[:m] * torch.randn(m, 1, device=DEV).bfloat16()
    a, s = ops.quantize_e4m3(x)
    some = torch.tensor([0, 1, 40000, 65535, 65536, m - 2, m - 1], device=DEV)
    want = wanted(decoded(a[some], s[:, some]), decoded(*w), bias, "silu", gated, None)
    y = ops.linear_e4m3(a, *w, a_scales=s, bias=bias, activation="silu", gated=gated)
    close(y[some], *want)
    del y
    codes, scales = ops.linear_e4m3_codes(a, *w, a_scales=s, bias=bias, activation="silu", gated=gated)
    close_codes(codes[some], scales[:, some], *want)
    values = ops.dequantize_e4m3(codes, scales, BF16)
    assert torch.equal(values[some].double(), decoded(codes[some], scales[:, some]))


def test_norm():
    m, n = (1 << 19) + 12, 4096
    x = torch.randn(64, n, device=DEV).bfloat16().repeat(m // 64 + 1, 1)[:m] * torch.randn(m, 1, device=DEV).bfloat16()
    delta, w = torch.randn(m, 1, device=DEV).bfloat16().expand(m, n).contiguous(), torch.randn(n, device=DEV).bfloat16()
    v = torch.empty_like(x)
    codes, scales = ops.add_rmsnorm_e4m3(x, w, 1e-5, delta=delta, x_out=v)
    some = torch.tensor([0, 1 << 18, 1 << 19, m - 1], device=DEV)
    assert torch.equal(v[some], (x[some].float() + delta[some].float()).to(BF16))
    again, same = ops.add_rmsnorm_e4m3(v[some], w, 1e-5)
    assert torch.equal(codes[some].view(torch.uint8), again.view(torch.uint8)) and torch.equal(scales[:, some], same)


@pytest.mark.parametrize("m,n,k,gated,codes_out", [
    (8, 6144, 4096, False, False), (64, 4096, 4096, False, False), (333, 8192, 2048, False, True), (448, 14336, 4096, True, True),
    (448, 4096, 14336, False, False), (160, 2048, 8192, False, False), (1, 14336, 4096, True, True), (2777, 4096, 14336, False, False),
    (2050, 14336, 4096, True, False)])
def test_the_same_call_twice(m, n, k, gated, codes_out):
    """Bit for bit, whatever its workspace held before."""
    x, w, bias, r = operands(m, n, k, gated, BF16)
    a, s = ops.quantize_e4m3(x)
    for rows, rows_s in ((a, s), (x, None)):
        first = None
        for fill in (0.0, float("nan"), 1e30):
            blocks = [torch.full((1 << 22,), fill, device=DEV) for _ in range(12)]
            del blocks
            if codes_out:
                got = ops.linear_e4m3_codes(rows, *w, a_scales=rows_s, bias=bias, activation="gelu", gated=gated)
            else:
                got = (ops.linear_e4m3(rows, *w, a_scales=rows_s, bias=bias, activation="gelu", gated=gated, residual=r),)
            got = [t.view(torch.uint8) for t in got]
            first = first or got
            assert all(torch.equal(p, q) for p, q in zip(first, got))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_block_half_twice(dtype):
    half = block_half(1024, 4096, dtype, 5)[3]
    x, delta = torch.randn(700, 1024, device=DEV).to(dtype), torch.randn(700, 1024, device=DEV).to(dtype)
    first = half(x, delta)
    for _ in range(3):
        assert all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(first, half(x, delta)))
