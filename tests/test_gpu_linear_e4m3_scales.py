"""The scales of results that projections over codes leave in codes: the smallest power of two for the group's own largest
magnitude, on every path that writes codes. Bit for bit where the result is known exactly; where sums round, between what
the largest may be at least and at most."""

import pytest
import torch

import e4m3_reference as ref
from forgeserve_amd import ops
from test_gpu_linear_e4m3 import ACTS, BF16, DEV, SIZES, decoded, operands, wanted

gpu = pytest.mark.gpu
ALL = (10, 246)
CODES_OUT = [size for size in SIZES if size[4]]


def unpacked(scales, n):
    """Exponent bytes (rows, n / 128) of packed scales, on the CPU; the bytes past them are zeros."""
    e = scales.cpu().transpose(0, 1).flatten(1)
    assert (e[:, n // 128:] == 0).all()
    return e[:, : n // 128].long()


def check_scales(scales, y, dy):
    """Each exponent byte is what some amax between the least and the greatest that y +- dy may have asks for."""
    y, dy = y.cpu().abs(), dy.cpu()
    least, most = (ref.exponents(v.unflatten(1, (-1, 128)), ALL).long() for v in ((y - dy).clamp(min=0), y + dy))
    e = unpacked(scales, y.shape[1])
    assert ((least <= e) & (e <= most)).all(), (e - most).max()
    return (least == most).double().mean()


def test_the_check_itself():
    """It takes the definition's exponents and none that is one off, though results have come through sums that round."""
    g = torch.Generator().manual_seed(9)
    y = torch.randn(20, 640, generator=g, dtype=torch.float64) * torch.exp(torch.randn(20, 5, generator=g)).repeat_interleave(128, 1)
    dy = 2.0 ** -14 * 20 * torch.ones_like(y)
    _, e = ref.encode(y.unflatten(1, (-1, 128)), ALL)
    assert check_scales(ref.packed_scales(e), y, dy) > 0.95
    for off in (-1, 1, 2):
        with pytest.raises(AssertionError):
            check_scales(ref.packed_scales((e.int() + off).to(torch.uint8)), y, dy)
    with pytest.raises(AssertionError):   # the row beside it
        check_scales(ref.packed_scales(e.roll(1, 0)), y, dy)


@pytest.mark.parametrize("size", CODES_OUT)
@gpu
def test_scales_of_sums(size):
    m, n, k, gated, _ = size
    act = ACTS[(m + n + k) % 5]
    x, w, bias, _ = operands(m, n, k, gated, BF16, seed=1)
    a, a_scales = ops.quantize_e4m3(x)
    pinned = check_scales(ops.linear_e4m3_codes(a, *w, a_scales=a_scales, bias=bias, activation=act, gated=gated)[1],
                          *wanted(decoded(a, a_scales), decoded(*w), bias, act, gated, None))
    assert pinned > 0.9


@pytest.mark.parametrize("size", CODES_OUT)
@gpu
def test_codes_and_scales_of_known_results(size):
    """Rows of x with one value that is not zero pick a column of w, so that a sum is one product of two codes, which float32
    holds; a float32 bias, relu and the gate's product round as float32 does. Magnitudes differ by up to 2^40 from a row to
    the next and from a group of columns to the next."""
    m, n, k, gated, _ = size
    g = torch.Generator().manual_seed(m + n + k)
    rows = (2 if gated else 1) * n

    def draw(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g)

    act = None if (m + k // 128) % 2 else "relu"
    col = draw(0, k, m)
    x = torch.zeros(m, k, dtype=torch.uint8)
    x[torch.arange(m), col] = (draw(1, 127, m) | draw(0, 2, m) << 7).to(torch.uint8)
    xe = draw(107, 148, m, 1).expand(m, k // 128)
    w = torch.randint(0, 256, (rows, k), generator=g, dtype=torch.uint8)
    w ^= (w & 127) == 127                                                # (no NaN)
    level = draw(107, 148, rows // 128).repeat_interleave(128)          # of a group of results
    we = level[:, None] + draw(-2, 3, rows, k // 128)
    bias = (torch.randn(rows, generator=g) * torch.exp2(level - 127.0 + draw(-6, 7, rows // 128).repeat_interleave(128))).float()
    packed = [ref.packed_scales(e.to(torch.uint8)).to(DEV) for e in (xe, we)]
    codes, scales = ops.linear_e4m3_codes(x.to(DEV), w.to(DEV), packed[1], a_scales=packed[0], bias=bias.to(DEV), activation=act,
                                          gated=gated)

    some = torch.unique(torch.cat([torch.tensor([0, m - 1, m // 2, min(m - 1, 63), min(m - 1, 64), min(m - 1, 127)]), draw(0, m, 24)]))
    at = col[some]
    xv = ref.decode(x[some, at][:, None], xe[some, 0])
    wv = ref.decode(w[:, at, None], we[:, at // 128])[..., 0].T
    z = (xv * wv).float()
    assert torch.equal(z.double(), xv * wv)
    z = z + bias
    y = z[:, :n].relu() if act else z[:, :n]
    y = y * z[:, n:] if gated else y
    c, e = ref.encode(y.unflatten(1, (-1, 128)), ALL)
    assert torch.equal(unpacked(scales, n)[some], e.long())
    got, c = codes.view(torch.uint8).cpu()[some], c.flatten(1)
    assert torch.equal(got & 127, c & 127) and torch.equal(got[c & 127 != 0], c[c & 127 != 0])   # (zeros of either sign)
