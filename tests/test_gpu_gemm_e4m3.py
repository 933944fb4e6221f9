"""Projections in 8-bit floating point against their definition in 64 bits."""

import math

import pytest
import torch

import e4m3_reference as ref
from forgeserve_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ALL = (10, 246)   # a matrix's scales have the same limits whatever its dtype


def values(codes, scales, k):
    """A matrix's values in 64 bits from its codes (rows, K) and packed scales."""
    e = scales.cpu().transpose(0, 1).flatten(1)[:, : k // 128]
    return ref.decode(codes.view(torch.uint8).cpu().unflatten(1, (k // 128, 128)), e).flatten(1)


def encoded(x):
    """x's values as the definition encodes them, in 64 bits."""
    c, e = ref.encode(x.double().unflatten(1, (-1, 128)), ALL)
    return ref.decode(c, e).flatten(1)


def check(got, x, w, residual=None):
    """got against x w^T (+ residual), x and w in 64 bits. The result is rounded once, half a step. Below that lie the
    matrix instruction's own sums: it aligns 128 products before it adds them; 2^-14 of the products' absolute sum is
    twenty times what it was measured to be off (2.5e-5 of a random result's norm, some 3e-6 of that sum)."""
    want, mag = x @ w.T, x.abs() @ w.abs().T
    if residual is not None:
        want = want + residual.double()
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -14 * mag + (2.0 ** -25 if got.dtype == F16 else 0)
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,k", [(1, 128), (5, 384), (33, 512), (3, 640), (130, 2048)])
def test_quantize(dtype, rows, k):
    g = torch.Generator().manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(3 * torch.randn(rows, k, generator=g))).to(dtype)
    x[0, :128] = 0
    x[-1, 5], x[-1, 6], x[-1, 127] = float("inf"), float("nan"), 448.0
    c, e = ref.encode(x.double().unflatten(1, (-1, 128)), ALL)
    want = ref.decode(c, e).flatten(1)
    wide = torch.zeros(rows, k + 5, dtype=dtype, device=DEV)
    wide[:, 3: 3 + k] = x.to(DEV)
    for y in (x.to(DEV), wide[:, 3: 3 + k]):   # aligned rows and others
        codes, scales = ops.quantize_e4m3(y)
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == (rows, k) and scales.shape == (-(-k // 512), rows, 4)
        assert torch.equal(scales.cpu(), ref.packed_scales(e))
        got = values(codes, scales, k)
        assert torch.equal(got.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_quantize_every_value(dtype):
    """Every 16-bit pattern under scales from its own magnitude up: the one conversion is the definition's rounding."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(65536, 128, dtype=dtype)
    top = torch.finfo(dtype).max
    x[:, 0] = bits
    for i, f in enumerate((1.0, 1.7, 33.0, 1000.0, 3e4)):
        x[:, 1] = (bits.double().abs() * f).clamp(max=top).nan_to_num(1.0).to(dtype)
        codes, scales = ops.quantize_e4m3(x.to(DEV))
        c, e = ref.encode(x.double(), ALL)
        assert torch.equal(scales[0, :, 0].cpu(), e)
        got, want = values(codes, scales, 128)[:, :2], ref.decode(c, e)[:, :2]
        assert torch.equal(got.nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))


SIZES = [(1, 16, 128), (1, 7, 384), (3, 130, 640), (8, 6144, 4096), (16, 70, 2048), (16, 9001, 512), (2, 8193, 1024),
         (17, 64, 128), (64, 130, 512), (33, 7, 1536), (64, 2048, 2048), (65, 64, 256), (130, 300, 640), (300, 128, 4096),
         (448, 520, 3584), (257, 4100, 1024), (1000, 260, 384), (520, 1, 512), (700, 1537, 896)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gemm(dtype, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    x = (torch.randn(m, k, generator=g) * torch.exp(0.7 * torch.randn(k, generator=g))).to(dtype)
    w = torch.randn(n, k, generator=g).mul_(0.02).to(BF16)
    codes, scales = ops.quantize_e4m3(w.to(DEV))
    xv, wv = encoded(x), values(codes, scales, k)
    check(ops.gemm_e4m3(x.to(DEV), codes, scales), xv, wv)
    # rows, results and residuals with strides and alignments of their own; the space between is left alone
    for shift in (0, 3):
        xs = torch.zeros(m, k + 8, dtype=dtype, device=DEV)[:, shift: shift + k].copy_(x)
        back = torch.full((m, n + 12), 3.0, dtype=dtype, device=DEV)
        r = torch.randn(m, n, generator=g).to(dtype)
        rs = torch.zeros(m, n + 5, dtype=dtype, device=DEV)[:, shift: shift + n].copy_(r)
        out = ops.gemm_e4m3(xs, codes, scales, out=back[:, 4 + shift: 4 + shift + n], residual=rs)
        check(out, xv, wv, r)
        assert (back[:, : 4 + shift] == 3).all() and (back[:, 4 + shift + n:] == 3).all()


@pytest.mark.parametrize("m", [1, 16, 40, 200])
def test_codes_with_wide_rows(m):
    g = torch.Generator().manual_seed(m)
    k, n = 256, 200
    x = torch.randn(m, k, generator=g).bfloat16()
    codes, scales = ops.quantize_e4m3(torch.randn(n, k, generator=g).to(DEV))
    wide = torch.zeros(n, k + 48, dtype=torch.uint8, device=DEV)
    wide[:, 16: 16 + k] = codes.view(torch.uint8)
    check(ops.gemm_e4m3(x.to(DEV), wide[:, 16: 16 + k], scales), encoded(x), values(codes, scales, k))


@pytest.mark.parametrize("m", [4, 40, 300])
def test_what_is_not_finite_stays_in_its_row(m):
    g = torch.Generator().manual_seed(m)
    k, n = 1024, 96
    x, w = torch.randn(m, k, generator=g).bfloat16(), torch.randn(n, k, generator=g).to(DEV)
    codes, scales = ops.quantize_e4m3(w)
    clean = ops.gemm_e4m3(x.to(DEV), codes, scales)
    x[1, 700], x[2, 3] = float("nan"), float("-inf")
    got = ops.gemm_e4m3(x.to(DEV), codes, scales)
    assert got[1].isnan().all() and got[2].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    bad = codes.view(torch.uint8).clone()
    bad[5, 300] = 0x7f
    got = ops.gemm_e4m3(x.to(DEV)[keep].contiguous(), bad, scales)
    assert got[:, 5].isnan().all() and not got[:, :5].isnan().any() and not got[:, 6:].isnan().any()


@pytest.mark.parametrize("m", [3, 64, 200])
def test_extreme_magnitudes(m):
    """Rows of the largest and of the smallest bf16 values, and zeros."""
    g = torch.Generator().manual_seed(m)
    k, n = 256, 64
    x = torch.randn(m, k, generator=g)
    x[0] = 0
    x[1] *= 1e30
    x[2] *= 1e-30
    x = x.bfloat16()
    codes, scales = ops.quantize_e4m3(torch.randn(n, k, generator=g).to(DEV))
    check(ops.gemm_e4m3(x.to(DEV), codes, scales), encoded(x), values(codes, scales, k))


def test_no_rows():
    codes, scales = ops.quantize_e4m3(torch.randn(32, 128, device=DEV))
    assert ops.gemm_e4m3(torch.empty(0, 128, dtype=BF16, device=DEV), codes, scales).shape == (0, 32)
    assert ops.quantize_e4m3(torch.empty(0, 128, dtype=BF16, device=DEV))[0].shape == (0, 128)


@pytest.mark.parametrize("m", [5, 50, 300])
def test_captured(m):
    """Replays with new rows between eager calls; two captured calls share the workspace one after the other."""
    g = torch.Generator().manual_seed(m)
    k, n = 1024, 512
    codes, scales = ops.quantize_e4m3(torch.randn(n, k, generator=g).to(DEV))
    back, bscales = ops.quantize_e4m3(torch.randn(k, n, generator=g).to(DEV))
    x = torch.randn(m, k, generator=g).bfloat16().to(DEV)
    step = lambda: ops.gemm_e4m3(ops.gemm_e4m3(x, codes, scales), back, bscales, residual=x)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.copy_(torch.randn(m, k, generator=g))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_an_mlp_of_8_bit_projections():
    """gate | up, the SwiGLU and down with its residual, as a decoder block runs them, against the same chain in 64 bits
    from each step's own inputs."""
    g = torch.Generator().manual_seed(21)
    d, f = 512, 1024
    wgu, wd = torch.randn(2 * f, d, generator=g).mul_(0.05).to(DEV), torch.randn(d, f, generator=g).mul_(0.05).to(DEV)
    (cgu, sgu), (cd, sd) = ops.quantize_e4m3(wgu), ops.quantize_e4m3(wd)
    for m in (1, 20, 90):
        x = torch.randn(m, d, generator=g).bfloat16().to(DEV)
        gu = ops.gemm_e4m3(x, cgu, sgu)
        check(gu, encoded(x.cpu()), values(cgu, sgu, d))
        h = ops.silu_mul(gu)
        y = ops.gemm_e4m3(h, cd, sd, residual=x)
        check(y, encoded(h.cpu()), values(cd, sd, f), x.cpu())


# tiles of 256 whole and cut off, with and without a split of K, and what the smaller tiles take of large calls
@pytest.mark.parametrize("m,n,k", [(700, 4096, 14336), (2050, 2048, 8192), (4097, 1100, 640), (1100, 9000, 256), (2300, 3001, 384),
                                   (512, 6144, 4096), (448, 16384, 1024), (300, 16301, 640)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_calls(dtype, m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    x = (torch.randn(m, k, generator=g, device=DEV) * torch.exp(0.7 * torch.randn(k, generator=g, device=DEV))).to(dtype)
    w = torch.randn(n, k, generator=g, device=DEV).mul_(0.02)
    codes, scales = ops.quantize_e4m3(w)
    xv, wv = (t.to(DEV) for t in (encoded(x.cpu()), values(codes, scales, k)))
    want, mag = xv @ wv.t().contiguous(), xv.abs() @ wv.abs().t().contiguous()

    # What the matrix instruction drops: it adds eight products at a time (of eight neighbours in K), aligned to the
    # largest, and of each of the other seven loses less than 2^-13 of the largest's power of two (found with a pair
    # that cancels beside products of every smaller size: those 13 places below count in full, those 14 below not at all
    # where they share its eight, in full elsewhere). So an element is off by less than 7 * 2^-13 max |x| max |w| of each
    # eight, plus 2^-23 of mag for each float32 sum on its way (an instruction takes 64 of K or more and adds 8 to 16
    # eights), plus its rounding. That bound grows as K where the errors grow as its root, so the whole result's norm is
    # held to more: rounding is off by at most eps / sqrt(12) of it, and the dropped parts were measured at 2.5e-5 of it, a
    # fifth of the 2^-13 allowed here.
    eights = [t.abs().unflatten(1, (k // 8, 8)).amax(2) for t in (xv, wv)]
    dropped = 7 * 2.0 ** -13 * (eights[0] @ eights[1].t().contiguous()) + (k // 64 + 16) * 2.0 ** -23 * mag
    eps = torch.finfo(dtype).eps

    def close(got, plus):
        y = want + plus
        err = (got.double() - y).abs()
        assert (err <= (1 + eps) * dropped + eps / 2 * y.abs() + (2.0 ** -25 if dtype == F16 else 0)).all()
        assert err.norm() <= (1.02 * eps / math.sqrt(12)) * y.norm() + 2.0 ** -13 * want.norm()

    close(ops.gemm_e4m3(x, codes, scales), 0)
    r = torch.randn(m, n, generator=g, device=DEV).to(dtype)
    back = torch.full((m, n + 12), 3.0, dtype=dtype, device=DEV)
    close(ops.gemm_e4m3(x, codes, scales, out=back[:, 5: 5 + n], residual=r), r.double())
    assert (back[:, :5] == 3).all() and (back[:, 5 + n:] == 3).all()


@pytest.mark.parametrize("m,n,k", [(3, 640, 512), (50, 512, 2048), (448, 520, 3584), (2050, 2048, 1024)])
def test_result_over_its_residual(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn(m, k, generator=g, device=DEV).bfloat16()
    codes, scales = ops.quantize_e4m3(torch.randn(n, k, generator=g, device=DEV))
    r = torch.randn(m, n, generator=g, device=DEV).bfloat16()
    want = ops.gemm_e4m3(x, codes, scales, residual=r)
    got = ops.gemm_e4m3(x, codes, scales, out=r, residual=r)
    assert got is r and torch.equal(got, want)


def test_calls_on_two_streams():
    """Calls that split K and hold encoded rows, in flight together."""
    g = torch.Generator(device=DEV).manual_seed(5)
    k, n, m = 8192, 1024, 200
    codes, scales = ops.quantize_e4m3(torch.randn(n, k, generator=g, device=DEV))
    xs = [torch.randn(m, k, generator=g, device=DEV).bfloat16() for _ in range(2)]
    want = [ops.gemm_e4m3(x, codes, scales) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.gemm_e4m3(xs[i], codes, scales))
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


@pytest.mark.parametrize("dtype,T", [(BF16, 1), (BF16, 5), (F16, 3), (BF16, 40)])
def test_a_block_in_8_bits(dtype, T):
    """The attention half of a decoder block, all of it over codes: the fused projection, its rotation and write into the
    pool, the attention over it and the output projection with its residual; each step against 64 bits from its own
    inputs, eagerly and replayed from a graph."""
    from forgeserve_amd import ModelConfig, PagedKVPool

    g = torch.Generator().manual_seed(T)
    heads, kv, hd, b, bs, ctx = 8, 2, 64, 3, 16, 90
    d = heads * hd
    pool = PagedKVPool(ModelConfig(vocab_size=32, d_model=d, n_layers=1, n_heads=heads, n_kv_heads=kv, ffn_dim=64,
                                   max_seq_len=1024), b * 9, bs, dtype=dtype, device=DEV, cache_dtype=torch.float8_e4m3fn)
    tables = torch.randperm(b * 9, generator=g).view(b, 9).int().to(DEV)
    angle = torch.rand(256, hd // 2, generator=g) * 6.28
    cos, sin = angle.cos().to(DEV), angle.sin().to(DEV)
    (cq, sq), (co, so) = (ops.quantize_e4m3(torch.randn(n, d, generator=g).mul_(0.05).to(DEV)) for n in ((heads + 2 * kv) * hd, d))
    old = torch.randn(b * ctx, (heads + 2 * kv) * hd, generator=g).to(dtype).to(DEV)     # what the pool holds already
    ops.qkv_rope_write(old, torch.arange(ctx, dtype=torch.int32).repeat(b).to(DEV), ctx, heads, cos, sin, tables, pool.layout(0))
    x = torch.randn(b * T, d, generator=g).to(dtype).to(DEV)
    pos = (ctx + torch.arange(T, dtype=torch.int32)).repeat(b, 1).to(DEV)

    def step():
        qkv = ops.gemm_e4m3(x, cq, sq)
        q = ops.qkv_rope_write(qkv, pos.view(-1), T, heads, cos, sin, tables, pool.layout(0))
        a = ops.paged_attention(q.view(b, T, heads, hd), pool.layout(0), tables, pos, hd ** -0.5)
        return qkv, q, a, ops.gemm_e4m3(a.view(b * T, d), co, so, residual=x)

    qkv, q, a, y = step()
    check(qkv, encoded(x.cpu()), values(cq, sq, d))
    k_all, v_all = (t.cpu().double() for t in ops.paged_gather(pool.layout(0), tables, dtype, DEV))
    for i in range(b):
        want, mag = ref.attention(q.view(b, T, heads, hd)[i].cpu(), k_all[i], v_all[i], pos[i].cpu(), hd ** -0.5)
        eps = torch.finfo(dtype).eps / 2       # p and the result rounded to the type, scores and sums in float32
        assert ((a[i].cpu().double() - want).abs() <= (1.02 * eps + 1e-4) * mag + eps * want.abs() + 2.0 ** -24).all()
    check(y, encoded(a.view(b * T, d).cpu()), values(co, so, d), x.cpu())
    # the keys as written: rotated in float32, then within half a step of a code (2^-4 of it, or 2^-10 of the scale,
    # which is less than 2^-17 of the largest)
    k1, k2 = (t.double().cpu() for t in qkv.view(b, T, -1, hd)[:, :, heads: heads + kv].chunk(2, -1))
    c, s = (t[ctx: ctx + T, None].double().cpu() for t in (cos, sin))
    rot = torch.cat([k1 * c - k2 * s, k2 * c + k1 * s], -1).transpose(1, 2)
    near = 2.0 ** -4 * rot.abs() + 2.0 ** -17 * rot.abs().amax(-1, keepdim=True)
    assert ((k_all[:, :, ctx: ctx + T] - rot).abs() <= near * 1.001).all()

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        x.copy_(torch.randn(b * T, d, generator=g))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(u, w) for u, w in zip(captured, eager))
