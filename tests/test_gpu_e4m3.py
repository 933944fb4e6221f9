"""The 8-bit pool on the GPU against its definition in 64 bits: writes, reading back, attention, and the model, the
Engine and speculation over it."""

import math

import pytest
import torch

import e4m3_reference as ref
import forgeserve_amd as fa
from forgeserve_amd import ModelConfig, PagedKVPool, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make_pool(hd, kv, bs, blocks, dtype, heads=None, layers=1, seed=None):
    heads = heads or kv
    cfg = ModelConfig(vocab_size=32, d_model=hd * heads, n_layers=layers, n_heads=heads, n_kv_heads=kv, ffn_dim=64,
                      max_seq_len=1 << 20)
    pool = PagedKVPool(cfg, blocks, bs, dtype=dtype, device=DEV, cache_dtype=E4M3)
    if seed is not None:   # something in every slot, NaN codes among it
        g = torch.Generator().manual_seed(seed)
        for s in (pool.k_store, pool.v_store):
            s.view(torch.uint8).copy_(torch.randint(0, 256, s.shape, generator=g, dtype=torch.uint8))
        lo, hi = ref.LIMITS[dtype]
        pool.scale_store.copy_(torch.randint(max(lo, 118), min(hi, 130), pool.scale_store.shape, generator=g))
    return pool


def stored(pool, layer=0):
    """(keys, values) of every slot in 64 bits, (blocks, heads, block, hd), and the exponents (blocks, heads, 2, block)."""
    k, v, s = ref.rows_of(pool.k[layer].cpu(), pool.v[layer].cpu(), pool.scales[layer].cpu())
    return ref.decode(k, s[:, :, 0]), ref.decode(v, s[:, :, 1]), s


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-7.125), torch.nan_to_num(b, nan=-7.125))


def special_rows(x):
    """Rows with zeros, what is not finite, and magnitudes at both ends of the scales' range."""
    x = x.clone()
    n = x.shape[0]
    big = {F32: 3e38, BF16: 3e38, F16: 65504.0}[x.dtype]
    x[0] = 0
    x[1 % n, ..., 3] = float("nan")
    x[2 % n, ..., 5] = float("inf")
    x[3 % n, ..., :] = float("-inf")
    x[4 % n, ..., 1] = big
    x[5 % n] *= 1e-6
    x[6 % n] *= 2.0 ** -120 if x.dtype != F16 else 2.0 ** -20
    x[7 % n, ..., 0] = 448.0
    return x


# ------------------------------------------------------------------------------------------------
# the plain write and reading back
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,kv,bs", [(64, 2, 16), (128, 3, 16), (16, 1, 4), (48, 2, 20), (96, 2, 12), (256, 1, 32), (32, 4, 16)])
def test_write_and_read_back(dtype, hd, kv, bs):
    b, t, nb = 3, 5, 6
    pool = make_pool(hd, kv, bs, 3 * nb + 2, dtype, seed=1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, b * t, kv, hd, generator=g).mul_(3).to(dtype)
    x = torch.stack([special_rows(x[0]), special_rows(x[1].flip(0))])
    k, v = (y.view(b, t, kv, hd).transpose(1, 2).to(DEV) for y in x)   # strided rows, head_dim contiguous
    tables = torch.randperm(3 * nb, generator=g).view(3, nb).int()
    tables[2, 1] = -1 if hd != 48 else 999        # an unmapped block: its tokens are not written, it reads as zeros
    pos = torch.tensor([[0, 1, 2, 3, 4], [bs - 1, bs, -1, 3 * bs + 1, nb * bs], [bs, 2 * bs + 3, 5 * bs, -1, 0]], dtype=torch.int32)
    before = stored(pool)
    lay, td = pool.layout(0), tables.to(DEV)
    ops.paged_kv_write(k, v, pos.to(DEV), td, lay)
    want_k, want_v, want_s = (y.clone() for y in before)
    for i in range(b):
        for j in range(t):
            p = int(pos[i, j])
            blk = int(tables[i, p // bs]) if 0 <= p < nb * bs else -1
            if not 0 <= blk < 3 * nb + 2:
                continue
            for side, want in ((0, want_k), (1, want_v)):
                c, e = ref.encode(x[side, i * t + j], ref.LIMITS[dtype])
                want[blk, :, p % bs], want_s[blk, :, side, p % bs] = ref.decode(c, e), e
    got = stored(pool)
    assert torch.equal(got[2], want_s)
    assert same(got[0], want_k) and same(got[1], want_v)
    # every table block in table order, exactly what the codes stand for
    ka, va = ops.paged_gather(lay, td, dtype, DEV)
    ok = ((tables >= 0) & (tables < 3 * nb + 2))[:, :, None, None, None]
    for out, want in ((ka, got[0]), (va, got[1])):
        w = torch.where(ok, want[tables.clamp(0, 3 * nb + 1).long()], 0.0)      # (b, nb, kv, bs, hd)
        assert out.dtype == dtype and same(out.cpu().double(), w.transpose(1, 2).reshape(b, kv, nb * bs, hd))


def test_view_update_is_write_and_gather():
    pool = make_pool(64, 2, 16, 8, BF16)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, 2, 7, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    table, pos = torch.tensor([[0, 3], [5, 1]]), torch.arange(12, 19)[None].expand(2, 7)
    ka, va = pool.views(table, pos)[0].update(k, v)
    for x, out in ((k, ka), (v, va)):
        c, e = ref.encode(x.cpu(), ref.LIMITS[BF16])
        assert torch.equal(out[:, :, 12:19].cpu().double(), ref.decode(c, e))
        assert not out[:, :, :12].any() and not out[:, :, 19:].any()


def test_far_blocks():
    """A pool of more than 4 GiB: a block's place takes 64 bits."""
    nb = (1 << 32) // (8 * 16 * 128) + 40
    pool = make_pool(128, 8, 16, nb, BF16)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(1, 8, 1, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    table = torch.tensor([[nb - 1]], dtype=torch.int32, device=DEV)
    ops.paged_kv_write(k, v, torch.tensor([[3]], dtype=torch.int32, device=DEV), table, pool.layout(0))
    ka, va = ops.paged_gather(pool.layout(0), table, BF16, DEV)
    c, e = ref.encode(k.cpu(), ref.LIMITS[BF16])
    assert torch.equal(ka[:, :, 3:4].cpu().double(), ref.decode(c, e)) and int(ka.ne(0).sum()) <= 8 * 128
    q = torch.randn(1, 1, 8, 128, generator=g).bfloat16().to(DEV)
    out = ops.paged_attention(q, pool.layout(0), table, torch.tensor([[3]], dtype=torch.int32, device=DEV), 0.1)
    want, mag = ref.attention(q[0].cpu(), ka[0].cpu().double(), va[0].cpu().double(), [3], 0.1)
    assert ((out[0].cpu().double() - want).abs() <= 0.01 * mag + 0.004 * want.abs()).all()


# ------------------------------------------------------------------------------------------------
# the fused rotation and write
# ------------------------------------------------------------------------------------------------
def rope_tables(hd, n, g):
    a = torch.rand(n, hd // 2, generator=g) * 2 * math.pi
    return a.cos(), a.sin()


def rotate64(x, pos, cos, sin):
    a, b = x.double().chunk(2, -1)
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def check_codes(got, e, want, limits):
    """got: decoded values with exponents e of groups whose 64-bit values are `want`. The kernel's float32 value is
    within two roundings of a product and one of a sum, 3 * 2^-24 of |x1 c| + |x2 s| <= sqrt(2) max |x|; its code is
    the nearest to that, so a value lies within half a code step of `want` plus that distance, and the scale is the
    definition's but where the largest magnitude is that near to its border."""
    amax = want.abs().amax(-1)
    slack = amax * 2.0 ** -20
    e_lo, e_hi = (ref.exponents((amax + d)[..., None], limits) for d in (-slack, slack))
    assert ((e >= e_lo) & (e <= e_hi)).all()
    s = torch.ldexp(torch.ones_like(want), (e.long() - 127)[..., None])
    _, ex = torch.frexp((want.abs() + slack[..., None]) / s)
    step = torch.ldexp(s, (ex - 1).clamp(min=-6) - 3)
    assert ((got - want).abs() <= step / 2 + slack[..., None]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("hd,heads,kv", [(128, 8, 2), (64, 6, 3), (96, 4, 2), (32, 3, 1), (256, 2, 2), (16, 5, 5)])
@pytest.mark.parametrize("form", ["decode", "window", "packed", "slots"])
def test_rope_write(dtype, hd, heads, kv, form):
    g = torch.Generator().manual_seed(hd + heads)
    bs, nb, rows, rope_len = 16, 5, 3, 70
    pool = make_pool(hd, kv, bs, rows * nb + 1, dtype, seed=5)
    tables = torch.randperm(rows * nb, generator=g).view(rows, nb).int()
    tables[1, 2] = -1
    cos, sin = rope_tables(hd, rope_len, g)
    token_row, slots, T = None, None, 1
    if form == "decode":
        pos = torch.tensor([17, -1, 69], dtype=torch.int32)
        row = torch.arange(3)
    elif form == "window":   # runs that cross 4-key groups and blocks, padding, a position past the rotary table
        T = 7
        pos = torch.stack([torch.arange(13, 20), torch.tensor([4, 5, 6, 7, -1, -1, -1]), torch.arange(66, 73)]).int().view(-1)
        row = torch.arange(3).repeat_interleave(7)
    elif form == "slots":    # rotated at one position, stored at another
        T = 5
        pos = torch.stack([torch.arange(40, 45), torch.arange(5), torch.arange(60, 65)]).int().view(-1)
        slots = torch.stack([torch.arange(0, 5), torch.arange(14, 19), torch.arange(3, 8)]).int().view(-1)
        row = torch.arange(3).repeat_interleave(5)
    else:                    # prompts back to back, a row that is none, one that starts inside a group
        lens, starts = [37, 1, 22, 2], [0, 9, 6, 0]
        pos = torch.cat([torch.arange(s, s + n) for s, n in zip(starts, lens)]).int()
        token_row = torch.tensor([0, 1, 2, 7]).repeat_interleave(torch.tensor(lens)).int()
        row = token_row.long()
    m = pos.numel()
    x = torch.randn(m, (heads + 2 * kv) * hd, generator=g).mul_(2).to(dtype)
    lay = pool.layout(0)
    before = stored(pool)

    def call(qkv):
        d = lambda t: None if t is None else t.to(DEV)
        if token_row is not None:
            return ops.qkv_rope_write_varlen(qkv, d(pos), d(token_row), heads, d(cos), d(sin), d(tables), lay)
        return ops.qkv_rope_write(qkv, d(pos), T, heads, d(cos), d(sin), d(tables), lay, slots=d(slots))

    q = call(x.to(DEV)).cpu().double().view(m, heads, hd)
    got_k, got_v, got_s = stored(pool)
    ok = (pos >= 0) & (pos < rope_len) & (row < rows)
    h3 = x.view(m, heads + 2 * kv, hd)
    turned = rotate64(h3[:, : heads + kv], pos.long().clamp(0, rope_len - 1), cos, sin)
    # queries: one rounding to the dtype of a float32 value within 3 * 2^-24 (sqrt 2 max) of it
    eps = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    want_q = torch.where(ok[:, None, None], turned[:, :heads], 0.0)
    tol = eps * want_q.abs() + 2.0 ** -21 * want_q.abs().amax(-1, keepdim=True) + (2.0 ** -25 if dtype == F16 else 0)
    assert ((q - want_q).abs() <= tol).all()
    # the pool: the written slots hold their tokens, every other one what it held
    at = (slots if slots is not None else pos).long()
    seen = torch.zeros(before[0].shape[0], bs, dtype=torch.bool)
    for i in range(m):
        blk = int(tables[row[i], at[i] // bs]) if ok[i] and at[i] < nb * bs else -1
        if blk < 0:
            continue
        sl = int(at[i]) % bs
        seen[blk, sl] = True
        check_codes(got_k[blk, :, sl], got_s[blk, :, 0, sl], turned[i, heads:], ref.LIMITS[dtype])
        c, e = ref.encode(h3[i, heads + kv:], ref.LIMITS[dtype])
        assert torch.equal(got_s[blk, :, 1, sl], e) and torch.equal(got_v[blk, :, sl], ref.decode(c, e))
    for got, old in ((got_k, before[0]), (got_v, before[1])):
        assert same(got.transpose(1, 2)[~seen], old.transpose(1, 2)[~seen])
    assert torch.equal(got_s.permute(0, 3, 1, 2)[~seen], before[2].permute(0, 3, 1, 2)[~seen])
    if dtype != F32:   # rows that are not 16-byte aligned take the other kernel: the same codes and queries
        codes = [s.clone() for s in (pool.k_store.view(torch.uint8), pool.v_store.view(torch.uint8), pool.scale_store)]
        wide = torch.zeros(m, x.shape[1] + 3, dtype=dtype, device=DEV)
        wide[:, 1: 1 + x.shape[1]] = x.to(DEV)
        q2 = call(wide[:, 1: 1 + x.shape[1]]).cpu().double().view(m, heads, hd)
        assert torch.equal(q, q2)
        for old, s in zip(codes, (pool.k_store.view(torch.uint8), pool.v_store.view(torch.uint8), pool.scale_store)):
            assert torch.equal(old, s)


def test_rope_write_what_is_not_finite():
    """A key's or value's element that is not finite is a NaN code; its neighbours keep the scale of the finite ones."""
    pool = make_pool(64, 1, 16, 1, BF16)
    x = torch.randn(1, 3 * 64, generator=torch.Generator().manual_seed(6)).bfloat16()
    x[0, 128 + 9] = float("inf")
    x[0, 128 + 10] = float("nan")
    x[0, 64 + 3] = float("nan")
    cos, sin = torch.ones(1, 32, device=DEV), torch.zeros(1, 32, device=DEV)
    z = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.qkv_rope_write(x.to(DEV), z, 1, 1, cos, sin, z[None], pool.layout(0))
    k, v, s = stored(pool)
    c, e = ref.encode(x[0, 128:], ref.LIMITS[BF16])
    assert same(v[0, 0, 0], ref.decode(c, e)) and v[0, 0, 0].isnan().sum() == 2
    assert k[0, 0, 0].isnan().nonzero().view(-1).tolist() == [3, 35]


@pytest.mark.parametrize("m", [64, 320])
def test_split_projection_into_the_pool(m):
    """A projection that splits K hands its partials to the write: the same codes and queries as written from its output."""
    g = torch.Generator().manual_seed(7)
    d, hd, heads, kv = 2048, 64, 32, 8
    n = (heads + 2 * kv) * hd
    h = torch.randn(m, d, generator=g).bfloat16().to(DEV)
    w = torch.randn(n, d, generator=g).mul_(0.02).bfloat16().to(DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(hd, 64, g))
    T = 5
    pos = torch.arange(T, dtype=torch.int32).repeat(m // T + 1)[: m // T * T].to(DEV)
    h = h[: m // T * T]
    b = h.shape[0] // T
    tables = torch.arange(b, dtype=torch.int32, device=DEV)[:, None].contiguous()
    pools = [make_pool(hd, kv, 16, b, BF16, heads=heads) for _ in range(2)]
    from forgeserve_amd import _lib
    assert _lib.load().fs_gemm_splits(n, d, _lib.BF16) > 1
    q1 = ops.qkv_rope_gemm(h, w, pos, T, heads, cos, sin, tables, pools[0].layout(0))
    q2 = ops.qkv_rope_write(ops.gemm(h, w), pos, T, heads, cos, sin, tables, pools[1].layout(0))
    assert torch.equal(q1, q2)
    for a, c in zip((pools[0].k_store, pools[0].v_store, pools[0].scale_store),
                    (pools[1].k_store, pools[1].v_store, pools[1].scale_store)):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
def fill(pool, g, spread=0.5):
    """Finite random keys and values in every slot of layer 0; returns them in 64 bits."""
    nb, kv, bs, hd = pool.num_blocks, pool.cfg.n_kv_heads, pool.block_size, pool.cfg.head_dim
    lim = ref.LIMITS[pool.dtype]
    rows = [torch.randn(nb, kv, bs, hd, generator=g) * torch.exp(spread * torch.randn(nb, kv, bs, 1, generator=g))
            for _ in range(2)]
    (kc, ke), (vc, ve) = (ref.encode(x.double(), lim) for x in rows)
    k, v = ref.tiles_of(kc, vc)
    pool.k[0].view(torch.uint8).copy_(k)
    pool.v[0].view(torch.uint8).copy_(v)
    pool.scales[0].copy_(torch.stack([ke, ve], 2))
    return ref.decode(kc, ke), ref.decode(vc, ve)


def row_keys(x, table, bs):
    """Keys or values (KV heads, n, hd) of a table row in 64 bits."""
    kv, hd = x.shape[1], x.shape[3]
    return x[table.long()].transpose(0, 1).reshape(kv, -1, hd)


def check_attention(out, want, mag, dtype):
    """Error of an output: p is rounded to the operands' 16-bit type (half a step of sum p |v|), scores and sums are
    float32 (1e-4 of sum p |v| covers scores of magnitude 100 and 2^15 keys), and the output is rounded once."""
    eps = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    tol = (eps * 1.02 + 1e-4) * mag + eps * want.abs() + (2.0 ** -24 if dtype == F16 else 1e-30)
    bad = (out.double() - want).abs() > tol
    assert not bad.any(), ((out.double() - want).abs() / tol).max()


CASES = [  # dtype, hd, heads, kv, bs, T, contexts (a row's furthest position + 1)
    (BF16, 128, 8, 2, 16, 1, [1, 2, 15, 16, 17, 31, 33, 300, 1000]),
    (BF16, 128, 8, 1, 16, 7, [7, 40, 290, 700]),
    (BF16, 64, 32, 4, 32, 5, [5, 6, 64, 511, 1300]),
    (F16, 64, 8, 2, 16, 1, [1, 16, 17, 200, 900]),
    (F16, 128, 12, 4, 48, 3, [3, 50, 333]),
    (F16, 128, 8, 1, 16, 7, [9, 100, 600]),
    (BF16, 64, 3, 3, 16, 1, [5, 77]),
    (F32, 64, 4, 2, 16, 3, [3, 30, 600]),
    (BF16, 96, 4, 2, 16, 2, [2, 70]),
    (BF16, 128, 4, 2, 20, 2, [2, 70, 555]),
    (F16, 256, 4, 2, 4, 1, [1, 9, 65]),
    (F32, 16, 2, 1, 8, 4, [4, 90]),
    (BF16, 128, 40, 1, 16, 1, [1, 100, 513]),
    (BF16, 128, 8, 2, 16, 50, [50, 120, 333]),
    (F16, 64, 8, 2, 32, 90, [90, 130]),
    (BF16, 64, 16, 2, 16, 41, [41, 64, 300]),
    (BF16, 128, 4, 1, 32, 200, [200, 201, 700]),
]


@pytest.mark.parametrize("dtype,hd,heads,kv,bs,T,ctx", CASES)
def test_attention(dtype, hd, heads, kv, bs, T, ctx):
    g = torch.Generator().manual_seed(hd + heads + T)
    nb = -(-max(ctx) // bs) + 1
    pool = make_pool(hd, kv, bs, len(ctx) * nb + 1, dtype, heads=heads)
    k, v = fill(pool, g)
    tables = torch.randperm(len(ctx) * nb, generator=g).view(len(ctx), nb).int()
    pos = torch.stack([torch.arange(n - T, n) for n in ctx]).int()
    pos[-1, T // 2:] = -1 if T > 1 else pos[-1, 0]     # a window shorter than the others'
    q = torch.randn(len(ctx), T, heads, hd, generator=g).to(dtype)
    # queries and outputs with strides of their own
    qd = torch.zeros(len(ctx), T, heads, hd + 8, dtype=dtype, device=DEV)[..., :hd].copy_(q)
    out = torch.full((len(ctx), heads, T, hd), 9.0, dtype=dtype, device=DEV).transpose(1, 2)
    scale = 1 / math.sqrt(hd)
    ops.paged_attention(qd, pool.layout(0), tables.to(DEV), pos.to(DEV), scale, out=out)
    for i in range(len(ctx)):
        want, mag = ref.attention(q[i], row_keys(k, tables[i], bs), row_keys(v, tables[i], bs), pos[i], scale)
        check_attention(out[i].cpu(), want, mag, dtype)
    assert not out[-1, T // 2:].any() or T == 1


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_scales(dtype, scale):
    g = torch.Generator().manual_seed(11)
    pool = make_pool(64, 2, 16, 20, dtype, heads=4)
    k, v = fill(pool, g)
    tables = torch.randperm(20, generator=g).view(1, 20).int()
    pos = torch.tensor([[300]], dtype=torch.int32)
    q = torch.randn(1, 1, 4, 64, generator=g).to(dtype)
    out = ops.paged_attention(q.to(DEV), pool.layout(0), tables.to(DEV), pos.to(DEV), scale)
    want, mag = ref.attention(q[0], row_keys(k, tables[0], 16), row_keys(v, tables[0], 16), pos[0], scale)
    check_attention(out[0].cpu(), want, mag, dtype)


@pytest.mark.parametrize("dtype,hd,heads,kv,T", [(BF16, 128, 8, 2, 7), (F16, 64, 8, 2, 7), (BF16, 64, 4, 2, 1), (F32, 64, 4, 2, 5),
                                                 (BF16, 128, 8, 2, 60), (F16, 128, 8, 2, 60)])
def test_attention_ignores_what_a_row_may_not_see(dtype, hd, heads, kv, T):
    """NaN codes behind a row's position (never written, or written by a later token of its window), in unmapped
    blocks' place and in blocks past the table change nothing; one that a row sees makes that row NaN, no other."""
    g = torch.Generator().manual_seed(12)
    bs, nb = 16, 12
    pool = make_pool(hd, kv, bs, nb + 2, dtype, heads=heads)
    fill(pool, g)
    tables = torch.randperm(nb, generator=g).view(1, nb).int().to(DEV)
    tables[0, 2] = -1
    last = 100 if T < 50 else 120
    pos = torch.arange(last - T + 1, last + 1).int()[None].to(DEV)
    q = torch.randn(1, T, heads, hd, generator=g).to(dtype).to(DEV)
    lay, scale = pool.layout(0), 0.1
    clean = ops.paged_attention(q, lay, tables, pos, scale).clone()
    assert not clean.isnan().any()

    def poison(p, side):
        blk, sl = int(tables[0, p // bs]), p % bs
        if side == 0:
            pool.k[0].view(torch.uint8)[blk, :, 0, sl, 3] = 0x7f
        else:
            pool.v[0].view(torch.uint8)[blk, :, sl // 4, int(ref.value_order(hd)[5]), sl % 4] = 0xff

    for p in range(last + 1, last + 40):   # behind every row
        poison(p, 0), poison(p, 1)
    pool.scales[0][int(tables[0, (last + 1) // bs]), :, :, (last + 1) % bs:] = 255
    assert torch.equal(ops.paged_attention(q, lay, tables, pos, scale), clean)
    if T > 1:   # a value that only the window's later tokens see: dim 5 of theirs is NaN
        cut = last - T // 2
        poison(cut, 1)
        got = ops.paged_attention(q, lay, tables, pos, scale)
        first = T - 1 - T // 2
        assert torch.equal(got[:, :first], clean[:, :first])
        assert got[:, first:, :, 5].isnan().all()
        keep = [d for d in range(hd) if d != 5]
        assert torch.equal(got[:, first:][..., keep], clean[:, first:][..., keep])
        poison(cut, 0)   # and a key: all of theirs
        got = ops.paged_attention(q, lay, tables, pos, scale)
        assert torch.equal(got[:, :first], clean[:, :first]) and got[:, first:].isnan().all()
    # the only key that a row sees
    poison(0, 0)
    one = ops.paged_attention(q[:, :1], lay, tables, torch.zeros(1, 1, dtype=torch.int32, device=DEV), scale)
    assert one.isnan().all()


@pytest.mark.parametrize("dtype,hd,bs", [(BF16, 128, 16), (BF16, 64, 32), (F16, 128, 16), (F16, 64, 16), (F32, 64, 16)])
def test_a_query_has_the_same_bits_whoever_computes_it(dtype, hd, bs):
    """One token, a window, a padded batch and a packed prompt give a query at a position the same output."""
    g = torch.Generator().manual_seed(13)
    heads, kv, n = 8, 2, 400
    nb = -(-n // bs)
    pool = make_pool(hd, kv, bs, 2 * nb, dtype, heads=heads)
    fill(pool, g)
    tables = torch.randperm(2 * nb, generator=g).view(2, nb).int().to(DEV)
    q = torch.randn(n, heads, hd, generator=g).to(dtype).to(DEV)
    lay, scale = pool.layout(0), 1 / math.sqrt(hd)
    pos = torch.full((2, n), -1, dtype=torch.int32)
    pos[0], pos[1, :100] = torch.arange(n), torch.arange(200, 300)
    cu = torch.tensor([0, n, n + 100], dtype=torch.int32, device=DEV)
    packed = ops.paged_attention_varlen(torch.cat([q, q[200:300]]), lay, tables, pos.to(DEV), cu, scale)
    whole = ops.paged_attention(q[None], lay, tables[:1], pos[:1].to(DEV), scale)[0]
    assert torch.equal(packed[:n], whole)
    for p in (0, 1, 15, 16, 17, 100, 255, 256, 300, n - 1):
        one = ops.paged_attention(q[None, p: p + 1], lay, tables[:1], torch.tensor([[p]], dtype=torch.int32, device=DEV), scale)
        assert torch.equal(one[0, 0], whole[p]), p
    for p in (0, 30, 250, n - 7):
        w = ops.paged_attention(q[None, p: p + 7], lay, tables[:1], torch.arange(p, p + 7, dtype=torch.int32, device=DEV)[None], scale)
        assert torch.equal(w[0], whole[p: p + 7]), p
    one = ops.paged_attention(q[None, 250:251], lay, tables[1:], torch.tensor([[250]], dtype=torch.int32, device=DEV), scale)
    assert torch.equal(one[0, 0], packed[n + 50])
    # queries in a larger batch
    many = ops.paged_attention(q[250:251].expand(70, -1, -1, -1).contiguous(), lay, tables[:1].expand(70, -1).contiguous(),
                               torch.full((70, 1), 250, dtype=torch.int32, device=DEV), scale)
    assert torch.equal(many, whole[250].expand(70, 1, -1, -1))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_context(dtype):
    """More keys than a chunk: the chunks are joined."""
    g = torch.Generator().manual_seed(14)
    n, bs, hd, heads, kv = 40000, 16, 128, 4, 1
    nb = -(-n // bs)
    pool = make_pool(hd, kv, bs, nb, dtype, heads=heads)
    k, v = fill(pool, g)
    tables = torch.randperm(nb, generator=g).view(1, nb).int()
    pos = torch.tensor([[n - 3, n - 1, 16383, 16384]], dtype=torch.int32)
    q = torch.randn(1, 4, heads, hd, generator=g).to(dtype)
    out = ops.paged_attention(q.to(DEV), pool.layout(0), tables.to(DEV), pos.to(DEV), 0.3)
    want, mag = ref.attention(q[0], row_keys(k, tables[0], bs), row_keys(v, tables[0], bs), pos[0], 0.3)
    check_attention(out[0].cpu(), want, mag, dtype)


@pytest.mark.parametrize("dtype,hd,heads,T", [(BF16, 128, 4, 1), (F16, 64, 8, 1), (BF16, 128, 8, 4)])
def test_lengths_about_a_chunk(dtype, hd, heads, T):
    """Rows that end just before, at and behind the borders of the chunks of keys, alone and in a batch."""
    g = torch.Generator().manual_seed(15)
    bs, kv = 16, 1
    ends = [2047, 2048, 2049, 4096, 4097, 8191, 8192, 8193, 8256, 16384, 16385]
    nb = -(-max(ends) // bs)
    pool = make_pool(hd, kv, bs, nb, dtype, heads=heads)
    k, v = fill(pool, g)
    table = torch.randperm(nb, generator=g).view(1, nb).int()
    pos = torch.stack([torch.arange(n - T, n) for n in ends]).int()
    q = torch.randn(len(ends), T, heads, hd, generator=g).to(dtype)
    scale = 1 / math.sqrt(hd)
    out = ops.paged_attention(q.to(DEV), pool.layout(0), table.expand(len(ends), -1).contiguous().to(DEV), pos.to(DEV), scale)
    kr, vr = row_keys(k, table[0], bs), row_keys(v, table[0], bs)
    for i, n in enumerate(ends):
        want, mag = ref.attention(q[i], kr, vr, pos[i], scale)
        check_attention(out[i].cpu(), want, mag, dtype)
        short = table[:, : -(-n // bs)].contiguous().to(DEV)       # a table no longer than the row
        one = ops.paged_attention(q[i: i + 1].to(DEV), pool.layout(0), short, pos[i: i + 1].to(DEV), scale)
        assert torch.equal(one[0], out[i]), n


@pytest.mark.parametrize("dtype,hd", [(F32, 64), (BF16, 128), (F16, 64), (BF16, 96), (F32, 16)])
@pytest.mark.parametrize("n", [6, 32, 700])
def test_a_nan_value_without_weight_is_still_seen(dtype, hd, n):
    """0 * NaN: a visible key's NaN reaches the output however small the key's probability, in its dim alone."""
    g = torch.Generator().manual_seed(hd + n)
    bs = 16
    nb = -(-n // bs)
    pool = make_pool(hd, 1, bs, nb, dtype, heads=2)
    k, v = fill(pool, g)
    pool.v[0].view(torch.uint8)[0, 0, 0, 5, 3] = 0xff    # slot 3 of block 0
    d = int((ref.value_order(hd) == 5).nonzero())
    tables = torch.arange(nb, dtype=torch.int32, device=DEV)[None]
    q = (row_keys(k, tables[0].cpu(), bs)[0, 5] * 60).to(dtype).expand(1, 1, 2, hd).contiguous()
    pos = torch.tensor([[n - 1]], dtype=torch.int32)
    out = ops.paged_attention(q.to(DEV), pool.layout(0), tables, pos.to(DEV), 1.0).cpu()
    assert out[..., d].isnan().all()
    out[..., d] = 0
    v[0, 0, 3, d] = 0
    want, mag = ref.attention(q[0], row_keys(k, tables[0].cpu(), bs), row_keys(v, tables[0].cpu(), bs), pos[0], 1.0)
    want[..., d] = 0
    check_attention(out[0], want, mag, dtype)


@pytest.mark.parametrize("dtype,hd,heads,kv,T", [(BF16, 128, 8, 2, 6), (F16, 64, 8, 2, 6), (BF16, 64, 8, 1, 40), (F16, 128, 4, 1, 70)])
@pytest.mark.parametrize("n", [40, 700, 9000])
def test_padding_between_the_tokens_of_a_window(dtype, hd, heads, kv, T, n):
    """Padding rows anywhere in a window give zeros, whatever their neighbours see (NaN among it), and change nothing of
    theirs; a window of padding alone gives zeros."""
    g = torch.Generator().manual_seed(n + T)
    bs = 16
    nb = -(-(n + T) // bs)
    pool = make_pool(hd, kv, bs, 3 * nb, dtype, heads=heads)
    k, v = fill(pool, g)
    pool.v[0].view(torch.uint8)[0, 0, 0, 5, 1] = 0x7f    # NaN: slot 1 of block 0
    d = int((ref.value_order(hd) == 5).nonzero())
    v[0, 0, 1, d] = float("nan")
    tables = torch.arange(3 * nb).view(3, nb).int()      # row 0 sees the NaN
    pos = torch.stack([torch.arange(n, n + T)] * 3).int()
    pad = torch.rand(3, T, generator=g) < 0.4
    pad[1, 0] = pad[0, -1] = True
    pad[2] = True
    pos[pad] = -1
    q = torch.randn(3, T, heads, hd, generator=g).to(dtype)
    scale = 1 / math.sqrt(hd)
    out = ops.paged_attention(q.to(DEV), pool.layout(0), tables.to(DEV), pos.to(DEV), scale)
    assert not out[pad.to(DEV)].any()
    for i in range(2):
        want, mag = ref.attention(q[i], row_keys(k, tables[i], bs), row_keys(v, tables[i], bs), pos[i], scale)
        there = ~pad[i]
        got = out[i].cpu()
        nan = want.isnan()
        assert torch.equal(got.isnan()[there], nan[there])
        check_attention(torch.where(nan, 0.0, got.float())[there].to(dtype), torch.where(nan, 0.0, want)[there],
                        torch.where(nan, 0.0, mag)[there], dtype)
    # a row alone has the same bits
    one = ops.paged_attention(q[1:2].to(DEV), pool.layout(0), tables[1:2].to(DEV), pos[1:2].to(DEV), scale)
    assert torch.equal(one[0], out[1])


def test_packed_rows_behind_the_last_sequence_are_left_alone():
    g = torch.Generator().manual_seed(15)
    pool = make_pool(128, 2, 16, 40, BF16, heads=8)
    fill(pool, g)
    tables = torch.randperm(40, generator=g).view(2, 20).int().to(DEV)
    lens = [300, 70]
    pos = torch.full((2, 300), -1, dtype=torch.int32)
    pos[0], pos[1, :70] = torch.arange(300), torch.arange(70)
    q = torch.randn(390, 8, 128, generator=g).bfloat16().to(DEV)
    out = torch.full((390, 8, 128), 5.0, dtype=BF16, device=DEV)
    ops.paged_attention_varlen(q, pool.layout(0), tables, pos.to(DEV), torch.tensor([0, 300, 370], dtype=torch.int32, device=DEV),
                               0.1, out=out)
    assert (out[370:] == 5.0).all() and not (out[:370] == 5.0).all(-1).any()


# ------------------------------------------------------------------------------------------------
# the calls together: graphs, streams, the model
# ------------------------------------------------------------------------------------------------
def test_captured_steps_replay():
    """A step (rotary write, attention, reading back) captured in a graph, replayed with new inputs between eager ones."""
    g = torch.Generator().manual_seed(16)
    b, heads, kv, hd, nb = 6, 8, 2, 128, 30
    pools = [make_pool(hd, kv, 16, b * nb, BF16, heads=heads) for _ in range(2)]
    fill(pools[0], g)
    for name in ("k_store", "v_store", "scale_store"):
        getattr(pools[1], name).view(torch.uint8).copy_(getattr(pools[0], name).view(torch.uint8))
    tables = torch.randperm(b * nb, generator=g).view(b, nb).int().to(DEV)
    cos, sin = (t.to(DEV) for t in rope_tables(hd, 480, g))
    qkv = torch.randn(b, (heads + 2 * kv) * hd, generator=g).bfloat16().to(DEV)
    pos = torch.tensor([3, 100, 200, 300, 400, 470], dtype=torch.int32, device=DEV)

    def step(pool):
        lay = pool.layout(0)
        q = ops.qkv_rope_write(qkv, pos, 1, heads, cos, sin, tables, lay)
        o = ops.paged_attention(q.view(b, 1, heads, hd), lay, tables, pos[:, None], 0.1)
        return (q, o, *ops.paged_gather(lay, tables, BF16, DEV))

    step(pools[0]), step(pools[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(pools[0])
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        pos.sub_(1)
        graph.replay()
        want = step(pools[1])
        torch.cuda.synchronize()
        for a, c in zip(captured, want):
            assert torch.equal(a, c), i


def test_another_stream():
    g = torch.Generator().manual_seed(17)
    pool = make_pool(64, 2, 16, 8, BF16, heads=4)
    k, v = (torch.randn(1, 2, 100, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    tables, pos = torch.arange(8, dtype=torch.int32, device=DEV)[None], torch.arange(100, dtype=torch.int32, device=DEV)[None]
    q = torch.randn(1, 1, 4, 64, generator=g).bfloat16().to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.paged_kv_write(k, v, pos, tables, pool.layout(0))
        out = ops.paged_attention(q, pool.layout(0), tables, pos[:, -1:], 0.125)
    side.synchronize()
    assert torch.equal(out, ops.paged_attention(q, pool.layout(0), tables, pos[:, -1:].contiguous(), 0.125))
    assert not out.isnan().any() and out.any()


MODEL = dict(vocab_size=300, d_model=512, n_layers=3, n_heads=8, n_kv_heads=2, ffn_dim=1024, max_seq_len=256)


def small_model(dtype, seed=0, **kw):
    torch.manual_seed(seed)
    return fa.ForgeModel(ModelConfig(**{**MODEL, **kw})).eval().to(device=DEV, dtype=dtype)


@pytest.mark.parametrize("dtype,kw", [(BF16, {}), (F16, {}), (F32, {}), (BF16, dict(n_heads=4)), (BF16, dict(d_model=384, n_heads=4))])
def test_model_over_the_pool(dtype, kw):
    """The model's forward over an 8-bit pool equals its own blocks run over the values that the pool holds: prompt and
    decode steps agree with one another bit for bit, and with the 16-bit pool within what the codes' rounding moves."""
    model = small_model(dtype, **kw)
    g = torch.Generator().manual_seed(18)
    ids = torch.randint(0, 300, (2, 60), generator=g)
    tables = torch.randperm(8, generator=g).view(2, 4)
    pools = [PagedKVPool(model.cfg, 8, 16, dtype=dtype, device=DEV, cache_dtype=c) for c in (E4M3, E4M3, None)]
    pos = torch.arange(60).expand(2, 60)
    whole = [model(ids, pos, p.views(tables, pos)) for p in (pools[0], pools[2])]
    steps = [model(ids[:, :40], pos[:, :40], pools[1].views(tables, pos[:, :40]))]
    steps += [model(ids[:, i: i + 1], pos[:, i: i + 1], pools[1].views(tables, pos[:, i: i + 1])) for i in range(40, 60)]
    assert torch.equal(torch.cat(steps, 1), whole[0])
    assert torch.equal(pools[0].k_store.view(torch.uint8), pools[1].k_store.view(torch.uint8))
    assert torch.equal(pools[0].v_store.view(torch.uint8), pools[1].v_store.view(torch.uint8))
    assert torch.equal(pools[0].scale_store, pools[1].scale_store)
    # a weighted mean of values that moved by up to 2^-4 each, mostly at random: far below a tenth of the logits' size
    rel = (whole[0].float() - whole[1].float()).norm() / whole[1].float().norm()
    assert 0 < rel < 0.1, rel


def test_blocks_one_by_one_and_in_a_run():
    """The native run of blocks over an 8-bit pool launches what the blocks launch one by one."""
    model = small_model(BF16)
    ids, tables, pos = torch.arange(24).view(2, 12), torch.tensor([[0, 1], [2, 3]]), torch.arange(12).expand(2, 12)
    pools = [PagedKVPool(model.cfg, 4, 16, dtype=BF16, device=DEV, cache_dtype=E4M3) for _ in range(2)]
    a = model(ids, pos, pools[0].views(tables, pos))
    for layer in model.layers:
        layer.step = layer.step   # a step of the object's own: no native run
    b = model(ids, pos, pools[1].views(tables, pos))
    assert torch.equal(a, b) and torch.equal(pools[0].k_store.view(torch.uint8), pools[1].k_store.view(torch.uint8))


def test_packed_prefill_over_the_pool():
    model = small_model(BF16)
    g = torch.Generator().manual_seed(19)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (70, 1, 33)]
    lists = [[4, 0, 7, 2, 9], [1], [3, 5, 6]]
    pools = [PagedKVPool(model.cfg, 10, 16, dtype=BF16, device=DEV, cache_dtype=E4M3) for _ in range(2)]
    got = fa.prefill_packed(model, pools[0], prompts, lists)
    for i, p in enumerate(prompts):
        pos = torch.arange(len(p))[None]
        want = model(torch.tensor([p]), pos, pools[1].views(torch.tensor([lists[i]]), pos))[0, -1]
        assert torch.equal(got[i], want), i
    assert torch.equal(pools[0].v_store.view(torch.uint8), pools[1].v_store.view(torch.uint8))


@pytest.mark.parametrize("graphs", [False, True])
def test_engine_and_speculation_over_the_pool(graphs):
    """Greedy tokens of the one-token Engine, the speculative Engine and the speculative batch over 8-bit pools are the
    same: a verify pass computes each position as a decode step does."""
    model = small_model(BF16)
    draft = fa.early_exit_draft(model, 1)
    prompts = [[1, 2, 3, 4, 5], [9, 8, 7], list(range(40))]

    def engine(**kw):
        e = fa.Engine(model, 60, cache_dtype=E4M3, **kw)
        ids = [e.add_request(p, 20) for p in prompts]
        e.run()
        return [e.requests[i].output for i in ids]

    plain = engine()
    assert plain == engine(draft=draft, k=3, graphs=graphs) == engine(draft=draft, k=3, graphs=graphs, share_kv=False)
    sb = fa.SpeculativeBatch(model, draft, 60, k=3, graphs=graphs, cache_dtype=E4M3)
    assert sb.pool_t.cache_dtype == E4M3


@pytest.mark.parametrize("dtype,hd,T", [(F16, 64, 1), (F16, 128, 7), (F16, 64, 60), (BF16, 64, 1), (BF16, 128, 60)])
@pytest.mark.parametrize("n", [100, 700, 9000])
def test_keys_far_below_the_largest(dtype, hd, T, n):
    """Many keys whose probabilities are 2^-25.3 of one key's: their share counts in full where that key's value is 0."""
    pool = make_pool(hd, 1, 16, -(-n // 16), dtype, heads=2)
    rows = torch.zeros(2, pool.num_blocks * 16, hd, dtype=torch.float64)
    rows[0, 0, 0], rows[1, 1:] = 8.0, 1.0
    rows[1, 1:, 5] = 3.0
    coded = [ref.encode(x, ref.LIMITS[dtype]) for x in rows]
    kc, vc = (c.view(pool.num_blocks, 1, 16, hd) for c, _ in coded)
    k, v = ref.tiles_of(kc, vc)
    pool.k[0].view(torch.uint8).copy_(k)
    pool.v[0].view(torch.uint8).copy_(v)
    pool.scales[0].copy_(torch.stack([e.view(-1, 1, 16) for _, e in coded], 2))
    q = torch.zeros(1, T, 2, hd, dtype=dtype)
    q[..., 0] = 2.0
    scale = 25.3 * math.log(2) / 16
    pos = torch.arange(n - T, n).int()[None]
    table = torch.arange(pool.num_blocks, dtype=torch.int32)[None]
    out = ops.paged_attention(q.to(DEV), pool.layout(0), table.to(DEV), pos.to(DEV), scale)
    want, mag = ref.attention(q[0], rows[0, None], rows[1, None], pos[0], scale)
    check_attention(out[0].cpu(), want, mag, dtype)
