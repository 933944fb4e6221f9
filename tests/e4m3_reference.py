"""The 8-bit pool and matrices in 64 bits on the CPU, from their definition: what the kernels are compared with."""

import torch

LIMITS = {torch.float32: (10, 246), torch.bfloat16: (10, 246), torch.float16: (112, 134)}


def _table():
    c = torch.arange(256)
    ex, man = (c >> 3) & 15, (c & 7).double()
    v = torch.where(ex == 0, torch.ldexp(man, torch.tensor(-9)), torch.ldexp(1 + man / 8, ex - 7))
    v[(c & 127) == 127] = float("nan")
    return torch.where(c >= 128, -v, v)


VALUES = _table()                 # what each of the 256 codes stands for, unscaled
_POSITIVE = VALUES[:127]          # 0 .. 448, increasing


def decode(codes, e):
    """codes (.., n) uint8 and exponent bytes (..) -> values (.., n) in 64 bits."""
    return torch.ldexp(VALUES[codes.long()], (e.long() - 127)[..., None])


def exponents(x, limits):
    """The exponent byte of each group x (.., n): the smallest power of two s with max |x| <= 448 s, of the finite x."""
    amax = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    m, ex = torch.frexp(amax / 448.0)
    e = torch.where(m > 0.5, ex, ex - 1) + 127
    return torch.where(amax > 0, e, limits[0]).clamp(*limits)


def encode(x, limits):
    """(codes (.., n) uint8, exponent bytes (..)) of groups x (.., n) in 64 bits: the nearest code, ties to the even
    one; NaN for what is not finite."""
    x = x.double()
    e = exponents(x, limits)
    y = torch.ldexp(x, (127 - e)[..., None])
    a = y.abs().clamp(max=448.0).nan_to_num(0.0)
    hi = torch.searchsorted(_POSITIVE, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    d_hi, d_lo = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = torch.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = torch.where(torch.isfinite(x), code + 128 * torch.signbit(x), 127)
    return code.to(torch.uint8), e.to(torch.uint8)


def value_order(hd):
    """Place of each dim in a tile of values."""
    d = torch.arange(hd)
    n = torch.clamp(hd // 16 - 4 * (d // 64), max=4)
    return (d // 64) * 64 + (d % 16) * n + (d // 16) % 4


def rows_of(k, v, scales):
    """Tiles (blocks, heads, ..) as codes (blocks, heads, block, hd) of keys and of values, and exponents (.., 2, block)."""
    kr = k.view(torch.uint8).transpose(2, 3).flatten(-2)
    vr = v.view(torch.uint8)[:, :, :, value_order(v.shape[3])].transpose(-1, -2).flatten(2, 3)
    return kr, vr, scales


def tiles_of(kr, vr):
    """Codes (blocks, heads, block, hd) as tiles."""
    nb, h, bs, hd = kr.shape
    k = kr.view(nb, h, bs, hd // 16, 16).transpose(2, 3).contiguous()
    at = torch.empty(hd, dtype=torch.long)
    at[value_order(hd)] = torch.arange(hd)
    v = vr.view(nb, h, bs // 4, 4, hd).transpose(-1, -2)[:, :, :, at].contiguous()
    return k, v


def attention(q, k, v, positions, scale):
    """q (T, H, hd), k and v (KV heads, n, hd) in 64 bits, positions (T,): (out, sum of p |v|), zeros where position < 0."""
    t, h, hd = q.shape
    hkv, n, _ = k.shape
    out, mag = torch.zeros(t, h, hd, dtype=torch.float64), torch.zeros(t, h, hd, dtype=torch.float64)
    for i in range(t):
        m = min(int(positions[i]) + 1, n)
        if m <= 0:
            continue
        for kvh in range(hkv):
            g = slice(kvh * (h // hkv), (kvh + 1) * (h // hkv))
            p = torch.softmax(q[i, g].double() @ k[kvh, :m].T * scale, -1)
            out[i, g], mag[i, g] = p @ v[kvh, :m], p @ v[kvh, :m].abs()
    return out, mag


def packed_scales(e):
    """Exponent bytes (rows, K / 128) as a matrix's (ceil(K / 512), rows, 4)."""
    rows, n = e.shape
    return torch.nn.functional.pad(e, (0, -n % 4)).view(rows, -1, 4).transpose(0, 1).contiguous()
