"""The RMS norm with its output in 8-bit codes, and codes as values, against their definition in 64 bits."""

import math

import pytest
import torch

import e4m3_reference as ref
from forgeserve_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ALL = (10, 246)


def values(codes, scales):
    k = codes.shape[1]
    e = scales.cpu().transpose(0, 1).flatten(1)[:, : k // 128]
    return ref.decode(codes.view(torch.uint8).cpu().unflatten(1, (k // 128, 128)), e).flatten(1)


def check(codes, scales, v, w, eps):
    """codes against the norm of v (CPU, in its type). The kernel's r: a sum of squares of at most 40 additions in a thread and
    40 across them (half of them between sums of 512 columns), a mean, a root and a quotient, then two products: 64 roundings
    of 2^-24 at most with the halving by the root, 2^-18. A code is off by
    half a step, 2^-4 of the value or 2^-10 of the scale, which is at most 2 / 448 of the group's largest."""
    m, n = v.shape
    assert codes.shape == (m, n) and codes.dtype == torch.float8_e4m3fn and scales.shape == (-(-n // 512), m, 4)
    x = v.double()
    y = x / (x.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    top = y.abs().unflatten(1, (-1, 128)).amax(2, keepdim=True).expand(-1, -1, 128).flatten(1)
    tol = (2.0 ** -4 + 2.0 ** -17) * y.abs() + 2.0 ** -10 * (2 / 448) * 1.001 * top
    err = (values(codes, scales) - y).abs()
    assert (err <= tol).all(), (err / tol).max()
    assert (scales.cpu().transpose(0, 1).flatten(1)[:, n // 128:] == 0).all()
    # the definition's own codes, but where 2^-18 may turn one: of a value near the middle between two, some 2^-13 of
    # them, or a group whose largest is next to a scale's border
    c, e = ref.encode(y.unflatten(1, (-1, 128)), ALL)
    same = (codes.view(torch.uint8).cpu() == c.flatten(1)).double().mean()
    assert same > 1 - 2.0 ** -7, same


def rows(m, n, dtype, seed, spread=0.7):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g) * torch.exp(spread * torch.randn(n, generator=g)) * torch.exp(torch.randn(m, 1, generator=g))
    return x.to(dtype), torch.randn(m, n, generator=g).to(dtype), (1 + 0.1 * torch.randn(n, generator=g)).to(dtype)


SIZES = [(1, 128), (3, 256), (6, 512), (5, 640), (2, 1024), (9, 1152), (7, 2048), (1, 2176), (65, 4096), (3, 4224), (2, 8192),
         (3, 8320), (2, 14336), (1, 16384), (2, 16512), (1, 40960), (3001, 384)]


@pytest.mark.parametrize("m,n", SIZES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_norm(dtype, m, n):
    x, d, w = rows(m, n, dtype, m + n)
    check(*ops.add_rmsnorm_e4m3(x.to(DEV), w.to(DEV), 1e-5), x, w, 1e-5)
    v = (x.float() + d.float()).to(dtype)
    for shift in (0, 1):   # aligned rows, and others with space between them that is left alone
        wide = [torch.full((m, n + 16), 3.0, dtype=dtype, device=DEV)[:, 8 + shift: 8 + shift + n] for _ in range(3)]
        xs, ds, out = wide[0].copy_(x), wide[1].copy_(d), wide[2]
        ws = torch.zeros(n + 8, dtype=dtype, device=DEV)[shift: shift + n].copy_(w)
        got = ops.add_rmsnorm_e4m3(xs, ws, 1e-6, delta=ds, x_out=out)
        assert torch.equal(out.cpu(), v)
        assert (out._base[:, : 8 + shift] == 3).all() and (out._base[:, 8 + shift + n:] == 3).all()
        check(*got, v, w, 1e-6)
        # the sum in the place of either
        for over in (xs, ds):
            keep = over.clone()
            again = ops.add_rmsnorm_e4m3(xs, ws, 1e-6, delta=ds, x_out=over)
            assert torch.equal(over, out) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, again))
            over.copy_(keep)


@pytest.mark.parametrize("n", [384, 1024, 2048, 2176, 4096, 8192, 14336, 16512])
def test_a_row_does_not_depend_on_its_batch(n):
    """Short batches and long ones, whose threads hold other pieces of a row."""
    x, _, w = (t.to(DEV) for t in rows(37, n, BF16, n))
    x = x.repeat(40, 1)
    codes, scales = ops.add_rmsnorm_e4m3(x, w, 1e-5)
    for i in (0, 20, 36, 1400):
        c, s = ops.add_rmsnorm_e4m3(x[i: i + 1], w, 1e-5)
        assert torch.equal(c.view(torch.uint8), codes[i: i + 1].view(torch.uint8)) and torch.equal(s[:, 0], scales[:, i])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [256, 2048, 20480])
def test_rows_of_zeros_and_what_is_not_finite(dtype, n):
    x, _, w = rows(6, n, dtype, n)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, n - 1] = float("nan")
    x[4] = 0
    x[4, 130] = torch.finfo(dtype).tiny
    codes, scales = ops.add_rmsnorm_e4m3(x.to(DEV), w.to(DEV), 1e-5)
    got = values(codes, scales)
    check(codes[[0, 5]], scales[:, [0, 5]].contiguous(), x[[0, 5]], w, 1e-5)
    assert (got[1] == 0).all() and got[3].isnan().all()
    # an infinite sum of squares: r = 0, so that finite values are zeros and the infinite one is NaN
    assert got[2, 5].isnan() and (got[2, torch.arange(n) != 5] == 0).all()
    tiny = float(x[4, 130].double() / math.sqrt(x[4, 130].double() ** 2 / n + 1e-5) * w[130].double())
    if abs(tiny) > 448 * 2.0 ** -117:   # (the smallest scale keeps less of what is smaller)
        assert abs(got[4, 130] - tiny) <= (2.0 ** -4 + 2.0 ** -16) * abs(tiny)
    assert (got[4, torch.arange(n) != 130] == 0).all()


@pytest.mark.parametrize("other", [None, float("nan"), float("inf"), 2.0 ** 127 * 1.9])
def test_every_value_is_encoded_by_its_definition(other):
    """Rows of ones leave the weight itself (1 / sqrt(mean) = 1), so its codes are those of any 32-bit value, exactly:
    subnormal ones, ties, what the smallest and the largest scale leave. `other`: in another group of the same wave."""
    g = torch.Generator().manual_seed(5)
    n = 16384
    w = torch.randint(0, 1 << 23, (n,), generator=g, dtype=torch.int32)
    w = torch.where(torch.rand(n, generator=g) < 0.5, w & ~0x7ffff, w)                        # ties and whole codes
    top = torch.randint(0, 254, (n // 128, 1), generator=g)                                     # a group's largest exponent
    ex = (top - torch.randint(0, 20, (n // 128, 128), generator=g)).clamp(min=0).flatten().int()
    w = (w | ex << 23 | torch.randint(0, 2, (n,), generator=g, dtype=torch.int32) << 31).view(F32)
    if other is not None:
        w[128 * 3 + 7 :: 512] = other
    c, e = ref.encode(w.view(-1, 128), ALL)
    for m in (1, 1030):
        codes, scales = ops.add_rmsnorm_e4m3(torch.ones(m, n, device=DEV), w.to(DEV), 0.0)
        got = codes.view(torch.uint8)
        assert torch.equal(got, got[:1].expand(m, -1)) and torch.equal(scales, scales[:, :1].expand(-1, m, -1))
        assert torch.equal(scales[:, 0].cpu().flatten(), e)
        nan = (c.flatten() & 127) == 127
        assert torch.equal(torch.where(nan, c.flatten(), got[0].cpu()), c.flatten())
        assert (got[0].cpu()[nan] & 127 == 127).all()


def test_single_rows_of_any_stride():
    x, w = torch.randn(512, 1, device=DEV).t(), torch.randn(512, device=DEV)
    want = ops.add_rmsnorm_e4m3(x.contiguous(), w, 1e-5)
    got = ops.add_rmsnorm_e4m3(x, w, 1e-5)
    assert x.stride() == (1, 1) and torch.equal(got[0].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(got[1], want[1])
    out = torch.zeros(512, 1, device=DEV).t()
    assert torch.equal(ops.dequantize_e4m3(*want, F32, out=out), ops.dequantize_e4m3(*want, F32))


def test_no_rows():
    w = torch.ones(256, device=DEV)
    codes, scales = ops.add_rmsnorm_e4m3(torch.empty(0, 256, device=DEV), w, 1e-5)
    assert codes.shape == (0, 256) and scales.shape == (1, 0, 4)
    assert ops.dequantize_e4m3(codes, scales, BF16).shape == (0, 256)
    x = torch.empty(0, 256, device=DEV)
    assert ops.add_rmsnorm_e4m3(x, w, 1e-5, delta=x, x_out=torch.empty_like(x))[0].shape == (0, 256)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k", [(1, 128), (3, 640), (70, 512), (5, 1152), (2001, 256)])
def test_dequantize(dtype, m, k):
    """Random codes under random scales (every code, all exponents): the value itself, in f16 rounded to it."""
    g = torch.Generator().manual_seed(m + k)
    codes = torch.randint(0, 256, (m, k), generator=g, dtype=torch.uint8)
    e = torch.randint(10, 247, (m, k // 128), generator=g)
    want = ref.decode(codes.unflatten(1, (-1, 128)), e).flatten(1).to(F32).to(dtype)   # (f32 holds each exactly)
    wide = torch.zeros(m, k + 32, dtype=torch.uint8, device=DEV)[:, 16: 16 + k].copy_(codes)
    scales = ref.packed_scales(e.to(torch.uint8)).to(DEV)
    for c in (codes.to(DEV), wide.view(torch.float8_e4m3fn)):
        for shift in (0, 1):
            back = torch.full((m, k + 16), 3.0, dtype=dtype, device=DEV)
            out = back[:, 8 + shift: 8 + shift + k]
            got = ops.dequantize_e4m3(c, scales, dtype, out=out)
            assert got is out and torch.equal(got.cpu().nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))
            assert torch.equal(got.isnan().cpu(), want.isnan())
            assert (back[:, : 8 + shift] == 3).all() and (back[:, 8 + shift + k:] == 3).all()
    assert torch.equal(ops.dequantize_e4m3(codes.to(DEV), scales, dtype).cpu().nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))


def test_there_and_back():
    """Values that codes hold come back as they were, and the second coding changes nothing."""
    x = rows(50, 768, BF16, 3)[0].to(DEV)
    codes, scales = ops.quantize_e4m3(x)
    y = ops.dequantize_e4m3(codes, scales, BF16)
    c2, s2 = ops.quantize_e4m3(y)
    assert torch.equal(ops.dequantize_e4m3(c2, s2, BF16), y)
