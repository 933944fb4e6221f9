"""The 8-bit pool's layout and what the calls refuse, on the CPU: nothing is launched."""

import ctypes
import os

import pytest
import torch

import e4m3_reference as ref
from forgeserve_amd import ModelConfig, PagedKVPool, _lib, ops
from forgeserve_amd.build import LIB

E4M3 = torch.float8_e4m3fn


def config(hd=64, heads=4, kv=2, layers=2):
    return ModelConfig(vocab_size=32, d_model=hd * heads, n_layers=layers, n_heads=heads, n_kv_heads=kv, ffn_dim=64,
                       max_seq_len=64)


def tensors(nb=3, h=2, hd=64, bs=16):
    u8 = dict(dtype=torch.uint8)
    return torch.zeros(nb, h, hd // 16, bs, 16, **u8), torch.zeros(nb, h, bs // 4, hd, 4, **u8), torch.zeros(nb, h, 2, bs, **u8)


def test_reference_codes():
    """The definition's own corners: every code is its own nearest, ties go to the even code, the scale's border is
    448 itself, what is not finite is NaN."""
    finite = ref.VALUES[~torch.isnan(ref.VALUES)]
    one = torch.tensor([448.0])
    for v in finite.tolist():
        c, e = ref.encode(torch.cat([one.double(), torch.tensor([v], dtype=torch.float64)]), (10, 246))
        assert int(e) == 127 and ref.VALUES[int(c[1])] == v
    c, e = ref.encode(torch.tensor([448.0, 17.0, 19.0, -17.0, 2.0 ** -10, float("inf"), float("nan")]), (10, 246))
    assert ref.decode(c, e)[:5].tolist() == [448.0, 16.0, 20.0, -16.0, 0.0] and ref.decode(c, e)[5:].isnan().all()
    assert int(ref.exponents(torch.tensor([448.5]).double(), (10, 246))) == 128
    assert int(ref.exponents(torch.tensor([224.0]).double(), (10, 246))) == 126
    assert int(ref.exponents(torch.tensor([0.0]).double(), (112, 134))) == 112


def test_codes_agree_with_torch():
    x = torch.randn(4000, generator=torch.Generator().manual_seed(1)).mul_(60).clamp_(-448, 448)
    x[0] = 448.0
    c, _ = ref.encode(x.double(), (10, 246))
    assert torch.equal(c, x.to(E4M3).view(torch.uint8))


@pytest.mark.parametrize("hd", [16, 48, 64, 96, 128, 256])
def test_value_order_is_a_permutation(hd):
    p = ref.value_order(hd)
    assert sorted(p.tolist()) == list(range(hd))
    if hd % 64 == 0:   # the 16 bytes at a place: four keys of dims d, d + 16, d + 32, d + 48
        assert p[16] == p[0] + 1 and p[32] == p[0] + 2 and p[1] == p[0] + 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_pool_layout(dtype):
    pool = PagedKVPool(config(), 6, 16, dtype=dtype, device="cpu", cache_dtype=E4M3)
    for layer in range(2):
        lay = pool.layout(layer)
        assert lay.dtype == _lib.DTYPE_CODE[dtype] | _lib.STORE_E4M3
        assert (lay.k, lay.v) == (pool.k[layer].data_ptr(), pool.v[layer].data_ptr())
        assert lay.k + lay.k_group == pool.scales[layer].data_ptr()
        assert (lay.k_block, lay.k_head, lay.v_block, lay.v_head) == (2 * 1024, 1024, 2 * 1024, 1024)
        assert (lay.k_slot, lay.k_dim) == pool.scales[layer].stride()[:2] == (32, 6 * 32)
        assert (lay.v_slot, lay.v_dim, lay.block_size, lay.n_kv_heads, lay.head_dim, lay.num_blocks) == (0, 0, 16, 2, 64, 6)
    assert pool.k[0].dtype == E4M3 and pool.dtype == dtype and pool.cache_dtype == E4M3
    plain = PagedKVPool(config(), 6, 16, dtype=dtype, device="cpu")
    assert plain.cache_dtype == dtype and plain.scales is None and plain.layout(0).dtype == _lib.DTYPE_CODE[dtype]


def test_pool_refusals():
    with pytest.raises(ValueError, match="8-bit pool"):
        PagedKVPool(config(hd=40), 6, 16, device="cpu", cache_dtype=E4M3)
    with pytest.raises(ValueError, match="8-bit pool"):
        PagedKVPool(config(), 6, 6, device="cpu", cache_dtype=E4M3)
    with pytest.raises(ValueError, match="cache_dtype"):
        PagedKVPool(config(), 6, 16, device="cpu", cache_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="key_layout"):
        PagedKVPool(config(), 6, 16, device="cpu", cache_dtype=E4M3, key_layout="rows")


def test_layout_refusals():
    k, v, s = tensors()
    assert ops.kv_layout_e4m3(k, v.view(E4M3), s, torch.bfloat16).num_blocks == 3
    bad = [(k.int(), v, s), (k, v.float(), s), (k, v, s.int()), (k[0], v, s), (k, v[:, :, :, :32], s), (k[:, :, :, :8], v, s),
           (k, v, s[:, :, :1]), (k, v, s[:, :1]), (k[:2], v, s), (k.transpose(2, 3).contiguous().transpose(2, 3), v, s),
           (k, v, torch.zeros(3, 2, 2, 32, dtype=torch.uint8)[..., ::2]), tensors(hd=272), tensors(bs=6)]
    for args in bad:
        with pytest.raises(ValueError, match="8-bit pool"):
            ops.kv_layout_e4m3(*args, torch.bfloat16)
    with pytest.raises(ValueError, match="dtype"):
        ops.kv_layout_e4m3(k, v, s, torch.int8)


def test_calls_refuse_bad_layouts():
    """The C calls check a pool of codes before anything is launched."""
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    lib = _lib.load()
    k, v, s = tensors()
    good = ops.kv_layout_e4m3(k, v, s, torch.bfloat16)

    def calls(lay):
        p = ctypes.byref(lay)
        return [lib.fs_paged_kv_write(16, 16, 0, 0, 0, 0, 1, 16, 16, 4, 4, p, None),
                lib.fs_paged_gather(p, 16, 4, 0, 4, 16, 16, None),
                lib.fs_qkv_rope_write(16, 4096, 0, 1, 4, 16, None, 16, 16, 8, 16, 4, 4, p, 16, 4096, None),
                lib.fs_paged_attention(16, 0, 0, 0, p, 16, 4, 4, 16, 1, 1, 4, 1.0, 16, 0, 0, 0, 256, 0, None)]

    assert calls(good)[:3] == [0, 0, 0]   # (nothing to do: no rows)
    for field, value in [("dtype", 19), ("head_dim", 72), ("head_dim", 272), ("block_size", 6), ("k_block", 8), ("v_head", 4),
                         ("k_group", 0), ("k_slot", 2), ("v_dim", 4), ("v_slot", 1), ("num_blocks", 0),
                         ("k", good.k + 8), ("v", good.v + 4), ("k_group", good.k_group + 2)]:
        lay = _lib.KVLayout.from_buffer_copy(good)
        setattr(lay, field, value)
        assert calls(lay) == [-1] * 4, field
    # an aligned gather's outputs must be aligned too; the workspace is still checked
    assert lib.fs_paged_gather(ctypes.byref(good), 16, 4, 1, 4, 8, 16, None) == -1 and b"aligned" in lib.fs_last_error()
    assert calls(good)[3] == -1 and b"workspace" in lib.fs_last_error()


def test_rows_of_another_dtype_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "require_device", lambda *t: None)
    k, v, s = tensors()
    lay = ops.kv_layout_e4m3(k, v, s, torch.bfloat16)
    x, i = torch.zeros(1, 512, dtype=torch.float16), torch.zeros(1, 4, dtype=torch.int32)
    f = torch.zeros(8, 32)
    with pytest.raises(ValueError, match="another dtype"):
        ops.qkv_rope_write(x, i[0, :1], 1, 4, f, f, i, lay)
    with pytest.raises(ValueError, match="another dtype"):
        ops.qkv_rope_write_varlen(x, i[0, :1], i[0, :1], 4, f, f, i, lay)
    with pytest.raises(ValueError, match="another dtype"):
        ops.paged_kv_write(x.view(1, 2, 4, 64), x.view(1, 2, 4, 64), i, i, lay)
    with pytest.raises(ValueError, match="another dtype"):
        ops.paged_gather(lay, i, torch.float32, "cpu")
    with pytest.raises(ValueError, match="another dtype"):
        ops.paged_attention(x.view(1, 1, 8, 64), lay, i, i[:, :1], 1.0)
    with pytest.raises(ValueError, match="another dtype"):
        ops.paged_attention_varlen(x.view(1, 8, 64), lay, i, i[:, :1], i[0, :2], 1.0)


def test_projection_refusals():
    """The C calls check their arguments before anything is launched."""
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    lib = _lib.load()
    need = lib.fs_gemm_e4m3_workspace_size(100, 64, 256)
    assert need >= 100 * 256 + 100 * 4 and lib.fs_gemm_e4m3_workspace_size(1, 64, 200) == 0

    def gemm(x=256, ldx=256, w=256, ldw=256, ws=256, c=256, ldc=64, r=None, ldr=0, m=0, n=64, k=256, dt=_lib.BF16, work=256,
             size=1 << 40):
        return lib.fs_gemm_e4m3(x, ldx, w, ldw, ws, c, ldc, r, ldr, m, n, k, dt, work, size, None)

    assert gemm() == 0   # (no rows)
    for bad in [dict(x=None), dict(w=None), dict(ws=None), dict(c=None), dict(dt=_lib.F32), dict(dt=7), dict(k=200), dict(k=0),
                dict(m=-1), dict(n=0), dict(ldx=255), dict(ldw=255), dict(ldw=264), dict(ldc=63), dict(r=256, ldr=63),
                dict(w=264), dict(ws=258), dict(m=100, work=None), dict(m=100, size=need - 1), dict(m=100, work=128),
                dict(m=1 << 29), dict(n=1 << 29, ldc=1 << 30), dict(k=1 << 23, ldx=1 << 23, ldw=1 << 23), dict(ldw=1 << 23)]:
        assert gemm(**bad) == -1, bad

    def quantize(x=256, ldx=256, rows=0, k=256, dt=_lib.BF16, codes=256, ldc=256, scales=256):
        return lib.fs_quantize_e4m3(x, ldx, rows, k, dt, codes, ldc, scales, None)

    assert quantize() == 0
    for bad in [dict(x=None), dict(codes=None), dict(scales=None), dict(dt=5), dict(k=100), dict(k=0), dict(rows=-1), dict(ldx=255),
                dict(ldc=255), dict(ldc=264), dict(codes=264), dict(scales=257), dict(rows=1 << 31)]:
        assert quantize(**bad) == -1, bad


def test_projection_wrappers_refuse(monkeypatch):
    monkeypatch.setattr(ops, "require_device", lambda *t: None)
    x, w, s = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(8, 256, dtype=torch.uint8), torch.zeros(1, 8, 4, dtype=torch.uint8)
    for bad in [(x.float(), w, s), (x[:, :128], w, s), (x, w.int(), s), (x, w, s.int()), (x, w, s[:, :7]),
                (x, w, torch.zeros(2, 8, 4, dtype=torch.uint8)), (x, w, torch.zeros(1, 8, 8, dtype=torch.uint8)[..., ::2]),
                (x.t(), w, s)]:
        with pytest.raises(ValueError):
            ops.gemm_e4m3(*bad)
    with pytest.raises(ValueError, match="out"):
        ops.gemm_e4m3(x, w, s, out=torch.zeros(2, 9, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_e4m3(x, w, s, residual=torch.zeros(2, 8))
    with pytest.raises(ValueError, match="128"):
        ops.quantize_e4m3(torch.zeros(3, 200))


def test_empty_layouts_are_refused():
    for kw in (dict(nb=0), dict(h=0), dict(hd=0), dict(bs=0)):
        with pytest.raises(ValueError, match="8-bit pool"):
            ops.kv_layout_e4m3(*tensors(**kw), torch.bfloat16)


def test_projection_refuses_tensors_of_two_devices(monkeypatch):
    monkeypatch.setattr(ops, "require_device", lambda *t: None)
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w, s = torch.zeros(32, 128, dtype=torch.uint8), torch.zeros(1, 32, 4, dtype=torch.uint8)
    y = torch.zeros(2, 32, dtype=torch.bfloat16)
    for kw in (dict(w=w.to("meta")), dict(w_scales=s.to("meta")), dict(out=y.to("meta")), dict(residual=y.to("meta"))):
        with pytest.raises(ValueError, match="devices"):
            ops.gemm_e4m3(x, **(dict(w=w, w_scales=s) | kw))


def test_tensors_of_another_device_than_the_current_are_refused(monkeypatch):
    class Elsewhere:
        device = torch.device("cuda", 1)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="current device"):
        ops._check_current("gemm_e4m3", Elsewhere())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    ops._check_current("gemm_e4m3", Elsewhere())


@pytest.mark.parametrize("limits", [(10, 246), (112, 134)])
def test_how_far_a_code_is_from_its_value(limits):
    """Half a step: 2^-4 of the value from 2^-6 of the scale on, 2^-10 of the scale below. A group's largest may be as low
    as 224 scales, which puts these at 2^-13.8 and 2^-17.8 of it, and not lower."""
    g = torch.Generator().manual_seed(22)
    tops = torch.tensor([224.0000001, 225.0, 300.0, 448.0], dtype=torch.float64)
    x = torch.exp2(-22 * torch.rand(4, 200000, generator=g, dtype=torch.float64)) * tops[:, None]
    x[:, 0] = tops
    c, e = ref.encode(x, limits)
    assert (e == 127).all()   # the scale is 1
    err, top = (ref.decode(c, e) - x).abs(), tops[:, None]
    normal = x >= 2.0 ** -6
    assert (err <= 2.0 ** -4 * x)[normal].all() and (err <= 2.0 ** -10)[~normal].all()
    assert (err <= 2.0 ** -4 * x)[x >= 2.0 ** -13.8 * top].all() and (err <= 2.0 ** -17.8 * top)[x < 2.0 ** -13.8 * top].all()
    # a bound that took the largest for 448 scales would be too small for the first two groups
    low = x < 2.0 ** -14.5 * top
    assert (err > 2.0 ** -18.5 * top)[:2][low[:2]].any() and (err > 2.0 ** -4 * x)[:2][(x >= 2.0 ** -14.5 * top)[:2]].any()


def test_the_smallest_float16_values_are_kept_exactly():
    """float16's scale is at least 2^-15: below 2^-21 the codes are its own smallest steps of 2^-24."""
    x = torch.arange(8, dtype=torch.float64) * 2.0 ** -24
    c, e = ref.encode(x, ref.LIMITS[torch.float16])
    assert int(e) == 112 and torch.equal(ref.decode(c, e), x)
