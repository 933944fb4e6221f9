"""What the 8-bit norm, the projections over codes and the codes' read-back refuse, on the CPU: nothing is launched."""

import os

import pytest
import torch

from forgeserve_amd import _lib, ops
from forgeserve_amd.build import LIB

BF16, F16, U8 = torch.bfloat16, torch.float16, torch.uint8


@pytest.fixture
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    return _lib.load()


@pytest.fixture
def on_cpu(monkeypatch):
    monkeypatch.setattr(ops, "require_device", lambda *t: None)


def test_linear_refusals(lib):
    """The C call checks its arguments before anything is launched."""
    good = dict(x=256, x_scales=256, w=256, w_scales=256, out=256, ldx=256, ldw=256, ldo=128, m=0, n=128, k=256, dtype=_lib.BF16)

    def call(size=1 << 40, work=256, **kw):
        return lib.fs_linear_e4m3(_lib.Linear(**(good | kw)), work, size, None)

    assert call() == 0 and call(x_scales=None, x_dtype=_lib.F32) == 0 and call(out_scales=256) == 0   # (no rows)
    assert call(gated=1, bias=256, residual=256, ldr=128) == 0
    for bad in [dict(x=None), dict(w=None), dict(w_scales=None), dict(out=None), dict(dtype=_lib.F32), dict(dtype=9),
                dict(x_scales=None, x_dtype=5), dict(bias=256, bias_dtype=3), dict(activation=5), dict(activation=-1),
                dict(out_scales=256, residual=256, ldr=128), dict(out_scales=256, n=120), dict(k=200), dict(k=0), dict(n=0),
                dict(m=-1), dict(ldx=255), dict(ldw=240), dict(ldw=264), dict(ldo=127), dict(residual=256, ldr=127), dict(w=264),
                dict(x=264), dict(ldx=264), dict(out_scales=256, out=264), dict(out_scales=256, ldo=136), dict(w_scales=258),
                dict(x_scales=257), dict(out_scales=258), dict(m=1 << 29), dict(n=1 << 28, ldo=1 << 29),
                dict(m=1 << 26, x_scales=None, x_dtype=_lib.F32),
                dict(m=1 << 28, n=1 << 20, ldo=1 << 20), dict(k=1 << 23, ldx=1 << 23, ldw=1 << 23), dict(ldw=1 << 23), dict(ldx=1 << 23)]:
        assert call(**bad) == -1, bad
        assert b"linear_e4m3" in lib.fs_last_error()
    assert lib.fs_linear_e4m3(None, 256, 1 << 30, None) == -1
    # a workspace of what the call needs: encoded rows, and sums that go through memory
    for kw in (dict(m=100, x_scales=None, x_dtype=_lib.BF16), dict(m=5, out_scales=256)):
        need = lib.fs_linear_e4m3_workspace_size(_lib.Linear(**(good | kw)))
        assert need > 0
        for ws in (dict(work=None), dict(size=need - 1), dict(work=128)):
            assert call(**kw, **ws) == -1
    assert lib.fs_linear_e4m3_workspace_size(_lib.Linear(**(good | dict(m=5)))) == 0
    assert lib.fs_linear_e4m3_workspace_size(None) == 0
    assert lib.fs_linear_e4m3_plan(_lib.Linear(**good), None) == -1


def test_norm_and_values_refusals(lib):
    def norm(x=256, ldx=256, d=None, ldd=0, xo=None, ldxo=0, w=256, c=256, ldc=256, s=256, m=0, n=256, dt=_lib.BF16):
        return lib.fs_add_rmsnorm_e4m3(x, ldx, d, ldd, xo, ldxo, w, c, ldc, s, m, n, 1e-5, dt, None)

    assert norm() == 0 and norm(d=256, ldd=256, xo=256, ldxo=256) == 0
    for bad in [dict(x=None), dict(w=None), dict(c=None), dict(s=None), dict(d=256, ldd=256), dict(dt=5), dict(m=-1), dict(n=200),
                dict(n=0), dict(ldx=255), dict(ldc=255), dict(ldc=264), dict(c=264), dict(s=258), dict(m=1 << 31),
                dict(m=1 << 26), dict(m=1 << 22, n=2048, ldx=2048, ldc=2048),
                dict(d=256, ldd=255, xo=256, ldxo=256), dict(d=256, ldd=256, xo=256, ldxo=255)]:
        assert norm(**bad) == -1, bad

    def values(c=256, ldc=256, s=256, rows=0, k=256, dt=_lib.BF16, out=256, ldo=256):
        return lib.fs_dequantize_e4m3(c, ldc, s, rows, k, dt, out, ldo, None)

    assert values() == 0
    for bad in [dict(c=None), dict(s=None), dict(out=None), dict(dt=5), dict(k=100), dict(k=0), dict(rows=-1), dict(ldc=255),
                dict(ldo=255), dict(ldc=264), dict(c=264), dict(s=257), dict(rows=1 << 26),
                dict(rows=1 << 62), dict(rows=1 << 25, k=1024, ldc=1024, ldo=1024)]:
        assert values(**bad) == -1, bad


def test_wrappers_refuse(on_cpu):
    x, w, s = torch.zeros(2, 256, dtype=BF16), torch.zeros(128, 256, dtype=U8), torch.zeros(1, 128, 4, dtype=U8)
    codes, cs = torch.zeros(2, 256, dtype=U8), torch.zeros(1, 2, 4, dtype=U8)
    for f in (ops.linear_e4m3, ops.linear_e4m3_codes):
        for bad in [(x[:, :128], w, s), (x, w.int(), s), (x, w, s.int()), (x, w, s[:, :7]), (x.t(), w, s), (x[0], w, s), (x, w[0], s),
                    (x, w, torch.zeros(2, 128, 4, dtype=U8)), (x, w, torch.zeros(1, 128, 8, dtype=U8)[..., ::2]), (codes, w, s),
                    (codes, w, s, cs[:, :1]), (codes, w, s, cs.int()), (x, w, s, cs), (x.double(), w, s), (x[:, :0], w[:, :0], s[:0]),
                    (x, w[:0], s[:, :0])]:
            with pytest.raises(ValueError):
                f(*bad)
        with pytest.raises(ValueError, match="activation"):
            f(x, w, s, activation="tanh")
        for b in (torch.zeros(127), torch.zeros(128, dtype=torch.float64), torch.zeros(1, 128), torch.zeros(256)[::2]):
            with pytest.raises(ValueError, match="bias"):
                f(x, w, s, bias=b)
    for kw in (dict(dtype=torch.float32), dict(out=torch.zeros(2, 128)), dict(out=torch.zeros(2, 127, dtype=BF16)),
               dict(out=torch.zeros(2, 128, dtype=BF16), dtype=F16), dict(residual=torch.zeros(2, 128)),
               dict(residual=torch.zeros(2, 128, dtype=F16), dtype=BF16), dict(residual=torch.zeros(3, 128, dtype=BF16)),
               dict(gated=True, residual=torch.zeros(2, 128, dtype=BF16)), dict(out=torch.zeros(128, 2, dtype=BF16).t())):
        with pytest.raises(ValueError):
            ops.linear_e4m3(x, w, s, **kw)
    with pytest.raises(ValueError, match="even"):
        ops.linear_e4m3(x, w[:127], s[:, :127].contiguous(), gated=True)
    with pytest.raises(ValueError, match="128"):
        ops.linear_e4m3_codes(x, w, s, gated=True)   # 64 columns
    with pytest.raises(ValueError, match="128"):
        ops.linear_e4m3_codes(x, w[:120], s[:, :120].contiguous())

    g = torch.ones(256, dtype=BF16)
    for bad in [dict(x=x[:, :200], weight=g[:200]), dict(weight=g[:128]), dict(weight=g.float()), dict(delta=x), dict(x_out=x),
                dict(delta=x[:1], x_out=x), dict(delta=x, x_out=x.float()), dict(x=x.int()), dict(x=x.t()),
                dict(weight=torch.ones(512, dtype=BF16)[::2])]:
        with pytest.raises(ValueError):
            ops.add_rmsnorm_e4m3(**(dict(x=x, weight=g, eps=1e-5) | bad))
    for bad in [dict(codes=codes[:, :200]), dict(codes=codes.int()), dict(scales=cs[:, :1]), dict(dtype=torch.int8),
                dict(out=torch.zeros(2, 256)), dict(out=torch.zeros(2, 255, dtype=BF16))]:
        with pytest.raises(ValueError):
            ops.dequantize_e4m3(**(dict(codes=codes, scales=cs, dtype=BF16) | bad))


def test_tensors_of_two_devices_are_refused(on_cpu):
    x, w, s = torch.zeros(2, 256, dtype=BF16), torch.zeros(128, 256, dtype=U8), torch.zeros(1, 128, 4, dtype=U8)
    y, cs = torch.zeros(2, 128, dtype=BF16), torch.zeros(1, 2, 4, dtype=U8)
    g = torch.ones(256, dtype=BF16)
    base = dict(a=x, w=w, w_scales=s)
    for kw in (dict(w=w.to("meta")), dict(w_scales=s.to("meta")), dict(a_scales=cs.to("meta")), dict(bias=g[:128].to("meta"))):
        for f in (ops.linear_e4m3, ops.linear_e4m3_codes):
            with pytest.raises(ValueError, match="devices"):
                f(**(base | kw))
    for kw in (dict(out=y.to("meta")), dict(residual=y.to("meta"))):
        with pytest.raises(ValueError, match="devices"):
            ops.linear_e4m3(**(base | kw))
    for kw in (dict(weight=g.to("meta")), dict(delta=x.to("meta"), x_out=x), dict(delta=x, x_out=x.to("meta"))):
        with pytest.raises(ValueError, match="devices"):
            ops.add_rmsnorm_e4m3(**(dict(x=x, weight=g, eps=1e-5) | kw))
    with pytest.raises(ValueError, match="devices"):
        ops.dequantize_e4m3(w, s.to("meta"), BF16)


def test_host_tensors_are_refused():
    x, w, s = torch.zeros(2, 256, dtype=BF16), torch.zeros(128, 256, dtype=U8), torch.zeros(1, 128, 4, dtype=U8)
    for call in (lambda: ops.linear_e4m3(x, w, s), lambda: ops.linear_e4m3_codes(x, w, s), lambda: ops.dequantize_e4m3(w, s, BF16),
                 lambda: ops.add_rmsnorm_e4m3(x, torch.ones(256, dtype=BF16), 1e-5)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()
