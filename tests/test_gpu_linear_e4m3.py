"""Projections over 8-bit codes with bias, activation, gate and residual, and their results in codes, against the definition
in 64 bits."""

import ctypes
import math

import pytest
import torch

import e4m3_reference as ref
from forgeserve_amd import _lib, ops

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
gpu = pytest.mark.gpu
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]


def plan(m, n, k, gated, codes):
    """(tile rows, tile columns, K splits, through memory) of a call over codes."""
    out = (ctypes.c_int32 * 4)()
    call = _lib.Linear(m=m, n=n, k=k, gated=gated, x_scales=16, out_scales=16 if codes else None)
    assert _lib.load().fs_linear_e4m3_plan(call, out) == 0
    return tuple(out)


# ------------------------------------------------------------------------------------------------
# the definition
# ------------------------------------------------------------------------------------------------
def decoded(codes, scales):
    """The values of a matrix in codes, in 64 bits, on its device."""
    k = codes.shape[1]
    e = scales.transpose(0, 1).flatten(1)[:, : k // 128]
    two = (e.long() - 127 + 1023 << 52).view(torch.float64)
    v = ref.VALUES.to(codes.device)[codes.contiguous().view(torch.uint8).long()]
    return (v.unflatten(1, (-1, 128)) * two[..., None]).flatten(1)


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(z * -math.sqrt(0.5))   # (ndtr loses the tail below -1 on the GPU)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))   # ((1 + tanh y) / 2 without its loss)
    return z


def wanted(x, w, bias, act, gated, residual):
    """The result in 64 bits and how far the sums and what follows may take it in 32. The sums: 2^-14 of the products'
    absolute sum (the matrix instruction aligns eights of products before it adds them; measured at a twentieth of that),
    and 2^-22 of that and the bias for the additions behind. An activation's slope is at most 1.13, and its own value is
    within 2^-15 = 3.1e-5 of itself: its exponential's argument is at most 85 where the result is above 1e-36 (below, 1e-36
    bounds what is lost), and has 4.5 roundings of 2^-24 for gelu_tanh (square, multiply-add, product, log2 e and that
    constant's own): 2.3e-5; 2.5 for gelu, with its polynomial 1.3e-5 + 8e-6; 1.5 for silu; the rest are a few of 2^-23. A
    product or sum of the results is two roundings more."""
    z, mag = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs() * 2.0 ** -8
    dz = (2.0 ** -14 + 2.0 ** -22) * mag
    n = z.shape[1] // 2 if gated else z.shape[1]
    y = act64(z[:, :n], act)
    dy = (1.13 * dz[:, :n] + 2.0 ** -15 * y.abs() + 1e-36) if act else dz[:, :n]
    if gated:
        up, du = z[:, n:], dz[:, n:]
        dy = dy * up.abs() + du * y.abs() + dy * du + 2.0 ** -23 * (y * up).abs()
        y = y * up
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -23 * y.abs()
    return y, dy


def close(got, y, dy):
    """16-bit results: half a step on top (of f16's smallest ones 2^-25)."""
    eps = torch.finfo(got.dtype).eps / 2
    tol = dy + eps * (y.abs() + dy) + (2.0 ** -25 if got.dtype == F16 else 0)
    err = (got.double() - y).abs()
    assert (err <= tol).all(), (err / tol).max()


def close_codes(codes, scales, y, dy):
    """Codes: half a step, 2^-4 of the value or 2^-10 of the scale, which is at most 2 / 448 of the largest."""
    top = (y.abs() + dy).unflatten(1, (-1, 128)).amax(2, keepdim=True).expand(-1, -1, 128).flatten(1)
    tol = dy + 2.0 ** -4 * (y.abs() + dy) + 2.0 ** -10 * (2.0 / 448) * 1.001 * top
    err = (decoded(codes, scales) - y).abs()
    assert (err <= tol).all(), (err / tol).max()
    used = y.shape[1] // 128
    assert (scales.transpose(0, 1).flatten(1)[:, used:] == 0).all()


def operands(m, n, k, gated, dtype, seed=0, bias_dtype=None):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * m + n + k)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    rows = (2 if gated else 1) * n
    x = (normal(m, k) * normal(k).mul_(0.5).exp_()).to(dtype)
    w = ops.quantize_e4m3(normal(rows, k).mul_(k ** -0.5))
    return x, w, normal(rows).to(bias_dtype or dtype), normal(m, n).to(dtype)


# ------------------------------------------------------------------------------------------------
# every kernel
# ------------------------------------------------------------------------------------------------
# (m, n, k, gated, codes out) -> its plan; tiles that the rows and columns end inside of
SIZES = {
    (5, 1, 512, False, False): (16, 16, 1, 0), (1, 7, 128, False, False): (16, 16, 1, 0),
    (1, 3, 128, True, False): (16, 16, 1, 0), (5, 1, 512, True, False): (16, 16, 1, 0),
    (5, 128, 512, False, True): (16, 16, 1, 1), (13, 640, 4096, False, True): (16, 16, 1, 1),
    (5, 128, 512, True, True): (16, 16, 1, 1), (5, 4305, 512, False, False): (16, 32, 1, 0),
    (5, 2441, 512, True, False): (16, 32, 1, 0), (9, 2050, 896, True, False): (16, 32, 1, 0),
    (6, 4224, 512, False, True): (16, 32, 1, 1), (5, 2176, 512, True, True): (16, 32, 1, 1),
    (5, 8444, 512, False, False): (16, 64, 1, 0), (5, 4420, 512, True, False): (16, 64, 1, 0),
    (16, 5003, 512, True, False): (16, 64, 1, 0), (6, 8448, 512, False, True): (16, 64, 1, 1),
    (6, 4352, 512, True, True): (16, 64, 1, 1), (5, 16852, 512, False, False): (16, 112, 1, 0),
    (5, 8954, 512, True, False): (16, 112, 1, 0), (5, 17024, 640, False, True): (16, 112, 1, 1),
    (16, 14336, 512, True, True): (16, 112, 1, 1), (5, 8704, 512, True, True): (16, 112, 1, 1),
    (31, 1537, 640, False, False): (32, 16, 1, 0), (17, 1, 512, False, False): (32, 16, 1, 0),
    (17, 1, 512, True, False): (32, 16, 1, 0), (17, 128, 512, False, True): (32, 16, 1, 1),
    (17, 128, 512, True, True): (32, 16, 1, 1), (17, 4443, 512, False, False): (32, 32, 1, 0),
    (19, 2097, 512, True, False): (32, 32, 1, 0), (17, 4864, 512, False, True): (32, 32, 1, 1),
    (17, 2432, 512, True, True): (32, 32, 1, 1), (17, 9604, 512, False, False): (32, 64, 1, 0),
    (17, 4204, 512, True, False): (32, 64, 1, 0), (18, 8576, 512, False, True): (32, 64, 1, 1),
    (20, 4224, 512, True, True): (32, 64, 1, 1), (17, 17300, 512, False, False): (32, 112, 1, 0),
    (19, 8301, 512, True, False): (32, 112, 1, 0), (17, 16640, 512, False, True): (32, 112, 1, 1),
    (19, 9088, 512, True, True): (32, 112, 1, 1), (34, 1, 512, False, False): (64, 16, 1, 0),
    (33, 1, 512, True, False): (64, 16, 1, 0), (33, 128, 512, False, True): (64, 16, 1, 1),
    (33, 128, 512, True, True): (64, 16, 1, 1), (36, 4126, 512, False, False): (64, 32, 1, 0),
    (35, 2105, 512, True, False): (64, 32, 1, 0), (36, 4736, 512, False, True): (64, 32, 1, 1),
    (36, 2176, 512, True, True): (64, 32, 1, 1), (134, 1, 512, False, False): (64, 64, 1, 0),
    (134, 1, 512, True, False): (64, 64, 1, 0), (65, 128, 4864, False, True): (64, 64, 1, 1),
    (129, 128, 1152, True, True): (64, 64, 1, 1), (35, 4, 11264, False, False): (64, 64, 2, 1),
    (65, 128, 5120, False, True): (64, 64, 2, 1), (73, 4, 5120, True, False): (64, 64, 2, 1),
    (129, 128, 1024, True, True): (64, 64, 2, 1), (135, 4, 2048, False, False): (64, 64, 4, 1),
    (129, 128, 2048, False, True): (64, 64, 4, 1), (134, 4, 2048, True, False): (64, 64, 4, 1),
    (129, 128, 2048, True, True): (64, 64, 4, 1), (129, 4, 4096, False, False): (64, 64, 8, 1),
    (33, 128, 12288, False, True): (64, 64, 8, 1), (129, 4, 4096, True, False): (64, 64, 8, 1),
    (33, 128, 12288, True, True): (64, 64, 8, 1), (71, 16420, 512, False, False): (64, 128, 1, 0),
    (129, 128, 512, False, True): (64, 128, 1, 0), (65, 8605, 512, True, False): (64, 128, 1, 0),
    (36, 17292, 4096, False, False): (64, 128, 2, 1), (33, 16768, 4096, False, True): (64, 128, 2, 1),
    (36, 8724, 4096, True, False): (64, 128, 2, 1), (35, 9644, 4096, False, False): (64, 128, 4, 1),
    (34, 10240, 2048, False, True): (64, 128, 4, 1), (37, 4244, 4096, True, False): (64, 128, 4, 1),
    (37, 4356, 16384, False, False): (64, 128, 8, 1), (39, 4608, 12288, False, True): (64, 128, 8, 1),
    (40, 2068, 16384, True, False): (64, 128, 8, 1), (129, 128, 512, True, True): (64, 256, 1, 0),
    (65, 1, 512, False, False): (128, 16, 1, 0), (65, 1, 512, True, False): (128, 16, 1, 0),
    (65, 128, 512, False, True): (128, 16, 1, 1), (65, 128, 512, True, True): (128, 16, 1, 1),
    (67, 4172, 512, False, False): (128, 32, 1, 0), (66, 2074, 512, True, False): (128, 32, 1, 0),
    (72, 4224, 512, False, True): (128, 32, 1, 1), (72, 2176, 512, True, True): (128, 32, 1, 1),
    (75, 16940, 1536, False, False): (128, 128, 1, 0), (130, 12032, 1408, False, True): (128, 128, 1, 0),
    (70, 9399, 1664, True, False): (128, 128, 1, 0), (79, 8320, 5248, True, True): (128, 128, 1, 1),
    (72, 8204, 4096, False, False): (128, 128, 2, 1), (66, 8320, 4096, False, True): (128, 128, 2, 1),
    (76, 4164, 4096, True, False): (128, 128, 2, 1), (70, 5120, 2048, True, True): (128, 128, 2, 1),
    (133, 2836, 4096, False, False): (128, 128, 4, 1), (132, 2816, 4096, False, True): (128, 128, 4, 1),
    (2754, 68, 4096, True, False): (128, 128, 4, 1), (135, 1408, 4096, True, True): (128, 128, 4, 1),
    (2052, 68, 8192, False, False): (128, 128, 8, 1), (69, 2176, 8192, False, True): (128, 128, 8, 1),
    (2073, 36, 8192, True, False): (128, 128, 8, 1), (75, 1280, 8192, True, True): (128, 128, 8, 1),
    (71, 17024, 512, True, True): (128, 256, 1, 0), (394, 9433, 1152, False, False): (256, 128, 1, 0),
    (258, 13184, 1152, False, True): (256, 128, 1, 0), (134, 12083, 1152, True, False): (256, 128, 1, 0),
    (158, 13364, 9216, False, False): (256, 128, 2, 1), (173, 12288, 7168, False, True): (256, 128, 2, 1),
    (732, 1372, 7168, True, False): (256, 128, 2, 1), (131, 5632, 4096, True, True): (256, 128, 2, 1),
    (140, 6116, 8192, False, False): (256, 128, 4, 1), (220, 4352, 6144, False, True): (256, 128, 4, 1),
    (263, 1652, 8192, True, False): (256, 128, 4, 1), (134, 3200, 8192, True, True): (256, 128, 4, 1),
    (146, 2884, 16384, False, False): (256, 128, 8, 1), (135, 2816, 16384, False, True): (256, 128, 8, 1),
    (2797, 68, 16384, True, False): (256, 128, 8, 1), (130, 1408, 16384, True, True): (256, 128, 8, 1),
    (1713, 4893, 1408, False, False): (256, 256, 1, 0), (1689, 4864, 1408, False, True): (256, 256, 1, 0),
    (259, 14221, 1408, True, False): (256, 256, 1, 0), (200, 17920, 512, True, True): (256, 256, 1, 0),
    (1848, 2180, 7168, False, False): (256, 256, 2, 1), (468, 9216, 6144, False, True): (256, 256, 2, 1),
    (366, 5524, 6144, True, False): (256, 256, 2, 1), (138, 11392, 5120, True, True): (256, 256, 2, 1),
    (138, 10996, 8192, False, False): (256, 256, 4, 1), (141, 11008, 8192, False, True): (256, 256, 4, 1),
    (193, 4108, 8192, True, False): (256, 256, 4, 1), (132, 4608, 8192, True, True): (256, 256, 4, 1),
    (2711, 260, 16384, False, False): (256, 256, 8, 1), (137, 5760, 16384, False, True): (256, 256, 8, 1),
    (2797, 132, 16384, True, False): (256, 256, 8, 1), (131, 2176, 16384, True, True): (256, 256, 8, 1),
}


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@gpu
def test_linear(size, dtype):
    m, n, k, gated, codes_out = size
    act = ACTS[(m + n + k) % 5]
    x, w, bias, r = operands(m, n, k, gated, dtype)
    a, a_scales = ops.quantize_e4m3(x)
    xv, wv = decoded(a, a_scales), decoded(*w)
    if codes_out:
        for b in (None, bias):
            want = wanted(xv, wv, b, act, gated, None)
            close_codes(*ops.linear_e4m3_codes(a, *w, a_scales=a_scales, bias=b, activation=act, gated=gated), *want)
            close_codes(*ops.linear_e4m3_codes(x, *w, bias=b, activation=act, gated=gated), *want)
        return
    want = wanted(xv, wv, None, act, gated, None)
    y = ops.linear_e4m3(a, *w, a_scales=a_scales, activation=act, gated=gated, dtype=dtype)
    close(y, *want)
    assert torch.equal(ops.linear_e4m3(x, *w, activation=act, gated=gated), y)
    # results and residuals with strides and alignments of their own; the space between is left alone
    want = wanted(xv, wv, bias, act, gated, r)
    for shift in (0, 3):
        back = torch.full((m, n + 20), 3.0, dtype=dtype, device=DEV)
        rs = torch.zeros(m, n + 8, dtype=dtype, device=DEV)[:, shift: shift + n].copy_(r)
        bs = torch.zeros(bias.numel() + 8, dtype=dtype, device=DEV)[shift: shift + bias.numel()].copy_(bias)
        y = ops.linear_e4m3(a, *w, a_scales=a_scales, bias=bs, activation=act, gated=gated, residual=rs,
                            out=back[:, 8 + shift: 8 + shift + n])
        close(y, *want)
        assert (back[:, : 8 + shift] == 3).all() and (back[:, 8 + shift + n:] == 3).all()


@pytest.mark.parametrize("m,n,k,gated", [(3, 4100, 8320, False), (17, 20000, 1792, False), (8, 12000, 2944, True), (33, 4096, 8192, False),
                                         (100, 8192, 4096, False), (2, 9000, 128, False), (2, 9000, 640, False), (1, 9003, 1152, True)])
@gpu
def test_wide_and_large_weights_of_short_batches(m, n, k, gated):
    """Weights of more than 32 MB are read past the caches; where a workgroup has many rows of W its waves begin at different
    stages, with one more stage for some waves, or none for some."""
    assert plan(m, n, k, gated, False)[0] in (16, 32, 64, 128)
    x, w, bias, r = operands(m, n, k, gated, BF16)
    a, a_scales = ops.quantize_e4m3(x)
    want = wanted(decoded(a, a_scales), decoded(*w), bias, "silu", gated, r)
    y = ops.linear_e4m3(a, *w, a_scales=a_scales, bias=bias, activation="silu", gated=gated, residual=r)
    close(y, *want)
    # rows do not depend on which of the batch they are, nor on what lies behind them
    assert torch.equal(ops.linear_e4m3(a.flip(0), *w, a_scales=a_scales.flip(1).contiguous(), bias=bias, activation="silu",
                                       gated=gated, residual=r.flip(0)).flip(0), y)


def test_the_sizes_take_every_kernel():
    assert {size: plan(*size) for size in SIZES} == SIZES


def test_no_other_kernel_is_chosen():
    """Over the shapes of projections and odd ones besides, the rule gives what the list above has."""
    seen = set()
    for m in [1, 2, 7, 8, 16, 17, 40, 64, 100, 129, 200, 256, 300, 448, 513, 700, 1000, 1500, 2050, 4097, 8005, 20000]:
        for n in (1, 7, 64, 128, 130, 512, 1024, 1540, 2048, 3001, 4096, 6144, 9000, 14336, 16384, 28672, 128256):
            for k in (128, 384, 1024, 2048, 4096, 6144, 8192, 10240, 14336, 16384):
                for gated in (False, True):
                    for codes in (False, True):
                        if not codes or n % 128 == 0:
                            seen.add((gated, codes) + plan(m, n, k, gated, codes))
    assert seen <= {(gated, codes) + p for (m, n, k, gated, codes), p in SIZES.items()}


# ------------------------------------------------------------------------------------------------
# what else a call may hold
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ACTS[1:])
@pytest.mark.parametrize("m", [3, 40])
@gpu
def test_activations(act, m):
    """An activation over all of its range: sums of zero, and a float32 bias that is its argument."""
    n = 8192
    z = torch.cat([torch.linspace(-110, 110, n // 2), torch.randn(n // 2 - 8, generator=torch.Generator().manual_seed(1)) * 3,
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 3e4, -3e4, 1e-6, -1e-6])]).to(DEV)
    w, w_scales = torch.zeros(n, 128, dtype=torch.uint8, device=DEV), torch.full((1, n, 4), 127, dtype=torch.uint8, device=DEV)
    x = torch.randn(m, 128, device=DEV, dtype=BF16)
    y = act64(z.double(), act)
    for dtype in (BF16, F16):
        close(ops.linear_e4m3(x, w, w_scales, bias=z, activation=act, dtype=dtype), y.expand(m, n), (2.0 ** -15 * y.abs() + 1e-36))
    one = torch.cat([z, torch.full_like(z, -1.5)])
    got = ops.linear_e4m3_codes(x, w.repeat(2, 1), w_scales.repeat(1, 2, 1), bias=one, activation=act, gated=True)
    close_codes(*got, (-1.5 * y).expand(m, n), (2.0 ** -14 * y.abs() + 2e-36).expand(m, n))
    # at the ends
    z = torch.tensor([float("inf"), float("nan")], device=DEV)
    got = ops.linear_e4m3(x, w[:2], w_scales[:, :2].contiguous(), bias=z, activation=act, dtype=BF16)
    assert (got[:, 0] == float("inf")).all() and got[:, 1].isnan().all()


@pytest.mark.parametrize("bias_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n,k,gated", [(4, 203, 256, False), (4, 203, 256, True), (77, 260, 1024, True), (900, 516, 384, False)])
@gpu
def test_bias_of_any_type(bias_dtype, m, n, k, gated):
    x, w, bias, _ = operands(m, n, k, gated, BF16, bias_dtype=bias_dtype)
    a, s = ops.quantize_e4m3(x)
    close(ops.linear_e4m3(a, *w, a_scales=s, bias=bias, activation="silu", gated=gated),
          *wanted(decoded(a, s), decoded(*w), bias, "silu", gated, None))


@gpu
def test_rows_of_any_type():
    """float32 rows, and the dtype of a result that nobody names."""
    x, w, _, r = operands(20, 130, 384, False, F16)
    got = ops.linear_e4m3(x.float(), *w)
    assert got.dtype == BF16
    close(got, *wanted(decoded(*ops.quantize_e4m3(x)), decoded(*w), None, None, False, None))
    a, s = ops.quantize_e4m3(x)
    assert ops.linear_e4m3(x, *w).dtype == F16 and ops.linear_e4m3(a, *w, a_scales=s, residual=r).dtype == F16
    assert ops.linear_e4m3(a, *w, a_scales=s).dtype == BF16 and ops.linear_e4m3(x, *w, dtype=BF16).dtype == BF16


@pytest.mark.parametrize("m", [1, 16, 40, 300, 1100])
@gpu
def test_codes_with_wide_rows(m):
    x, w, _, _ = operands(m, 256, 640, False, BF16)
    a, s = ops.quantize_e4m3(x)
    want = ops.linear_e4m3(a, *w, a_scales=s)
    wide = [torch.full((t.shape[0], 640 + 48), 255, dtype=torch.uint8, device=DEV) for t in (a, w[0])]
    for t, v in zip(wide, (a, w[0])):
        t[:, 16: 16 + 640] = v.view(torch.uint8)
    assert torch.equal(ops.linear_e4m3(wide[0][:, 16: 656], wide[1][:, 16: 656], w[1], a_scales=s), want)


@pytest.mark.parametrize("m", [4, 40, 300])
@gpu
def test_what_is_not_finite_stays_in_its_row(m):
    x, w, _, _ = operands(m, 256, 1024, True, BF16)
    clean = ops.linear_e4m3(x, *w, activation="silu", gated=True)
    codes = ops.linear_e4m3_codes(x, *w, activation="silu", gated=True)
    x[1, 700], x[2, 3] = float("nan"), float("-inf")
    got = ops.linear_e4m3(x, *w, activation="silu", gated=True)
    keep = [i for i in range(m) if i not in (1, 2)]
    assert got[1:3].isnan().all() and torch.equal(got[keep], clean[keep])
    got = ops.linear_e4m3_codes(x, *w, activation="silu", gated=True)
    assert ops.dequantize_e4m3(*got, F32)[1:3].isnan().all()
    assert torch.equal(got[0].view(torch.uint8)[keep], codes[0].view(torch.uint8)[keep]) and torch.equal(got[1][:, keep], codes[1][:, keep])


@pytest.mark.parametrize("m,n,k", [(3, 640, 512), (50, 512, 2048), (448, 520, 3584), (2050, 2048, 1024)])
@gpu
def test_result_over_its_residual(m, n, k):
    x, w, b, r = operands(m, n, k, False, BF16)
    want = ops.linear_e4m3(x, *w, bias=b, residual=r)
    got = ops.linear_e4m3(x, *w, bias=b, residual=r, out=r)
    assert got is r and torch.equal(got, want)


@gpu
def test_no_rows():
    w = ops.quantize_e4m3(torch.randn(256, 128, device=DEV))
    x = torch.empty(0, 128, dtype=BF16, device=DEV)
    assert ops.linear_e4m3(x, *w, gated=True).shape == (0, 128)
    codes, scales = ops.linear_e4m3_codes(x, *w)
    assert codes.shape == (0, 256) and scales.shape == (1, 0, 4)
    assert ops.linear_e4m3(codes, *ops.quantize_e4m3(torch.randn(9, 256, device=DEV)), a_scales=scales).shape == (0, 9)


@pytest.mark.parametrize("m", [1, 16, 17, 100, 448, 1500])
@gpu
def test_the_same_as_the_product_alone(m):
    """Without a bias, a gate and an activation: gemm_e4m3's result, up to the order of the sums over K."""
    x, w, _, r = operands(m, 1024, 4096, False, BF16)
    close(ops.linear_e4m3(x, *w, residual=r), *wanted(decoded(*ops.quantize_e4m3(x)), decoded(*w), None, None, False, r))
    want = ops.gemm_e4m3(x, *w, residual=r)
    assert ((ops.linear_e4m3(x, *w, residual=r).double() - want.double()).norm() <= 2.0 ** -8 * want.double().norm())


# ------------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------------
def block_half(d, f, dtype, seed):
    """A block's MLP half: its weights, and a call of it."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    w1 = ops.quantize_e4m3(torch.randn(2 * f, d, generator=g, device=DEV).mul_(d ** -0.5))
    w2 = ops.quantize_e4m3(torch.randn(d, f, generator=g, device=DEV).mul_(f ** -0.5))
    norm = (1 + 0.1 * torch.randn(d, generator=g, device=DEV)).to(dtype)

    def half(x, delta):
        v = torch.empty_like(x)
        c, s = ops.add_rmsnorm_e4m3(x, norm, 1e-5, delta=delta, x_out=v)
        h, hs = ops.linear_e4m3_codes(c, *w1, a_scales=s, activation="silu", gated=True)
        return v, c, s, h, hs, ops.linear_e4m3(h, *w2, a_scales=hs, residual=v)

    return w1, w2, norm, half


@pytest.mark.parametrize("m,d,f", [(1, 512, 1408), (16, 1024, 1024), (40, 512, 1536), (300, 640, 2048), (1300, 2048, 4096)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@gpu
def test_a_block_half(dtype, m, d, f):
    """Norm, gated product and product with the residual, each step against 64 bits from its own inputs; then captured, and
    replayed with new rows between eager calls."""
    w1, w2, norm, half = block_half(d, f, dtype, m)
    x, delta = (torch.randn(m, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)).to(dtype) for i in (1, 2))
    v, c, s, h, hs, y = half(x, delta)
    assert torch.equal(v, (x.float() + delta.float()).to(dtype))
    n64 = v.double() / (v.double().square().mean(1, keepdim=True) + 1e-5).sqrt() * norm.double()
    close_codes(c, s, n64, 2.0 ** -18 * n64.abs())
    close_codes(h, hs, *wanted(decoded(c, s), decoded(*w1), None, "silu", True, None))
    close(y, *wanted(decoded(h, hs), decoded(*w2), None, None, False, v))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = half(x, delta)
    for i in range(4):
        x.copy_(torch.randn(m, d, device=DEV))
        delta.copy_(torch.randn(m, d, device=DEV))
        graph.replay()
        want = half(x, delta)
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))


@gpu
def test_calls_on_two_streams():
    """Calls that hold encoded rows and sums in memory, in flight together."""
    w1, w2, norm, half = block_half(1024, 2048, BF16, 3)
    xs = [torch.randn(200, 1024, device=DEV).bfloat16() for _ in range(2)]
    want = [half(x, x)[-1] for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(half(xs[i], xs[i])[-1])
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)
