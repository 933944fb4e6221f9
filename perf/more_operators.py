"""The 8-bit half of a decoder block as its users call it: the RMS norm with the residual's addition whose output is
8-bit floating point, products over such codes with bias, activation, gate and residual in their epilogue (16-bit
results, or codes again for the next product), codes read back as values, and a block's MLP half made of them.

Format: e4m3 codes (4 exponent and 3 mantissa bits, largest value 448) with a scale for each 128 columns of a row, the
smallest power of two that brings the group's largest magnitude to 448 or less, kept as its biased exponent byte e
(10 to 246): a code stands for value(code) * 2^(e - 127). Scales lie as (ceil(K / 512), rows, 4).

 * norm: v = round(x + delta), y = v / sqrt(mean(v^2) + eps) * weight, in codes; v is returned too where delta is given
 * linear: y = act(x w^T + bias) + residual, or with a gate (w and bias hold the gate's rows, then the others')
   y = act(gate) * up + residual
 * mlp: norm, gate and up product with the gate, in codes, down product with the residual

Sizes come from the package's own configurations: the 1B shape (d 2048, 32/8 heads of 64, ffn 8192), the 8B shape (d 4096,
32/8 heads of 128, ffn 14336), the tiny float32 model (d 256), with the batches and windows that the benchmark and
the tests run. Codes are returned as the values they stand for.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E4M3 = torch.float8_e4m3fn
GROUP = 128                  # columns per scale
LOW, HIGH = 10, 246          # exponent bytes of the scales
EPS = 1e-5


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def _linear(name, m, n, k, dtype="bf16", act="none", gated=False, bias=False, residual=False, codes_out=False, codes_in=True):
    """n: columns of the result."""
    return dict(name=name, kind="linear", dtype=dtype, m=m, n=n, k=k, act=act, gated=gated, bias=bias, residual=residual,
                codes_in=codes_in, codes_out=codes_out)


def listed():
    return [
        # one token through the tiny float32 model's norm: the smallest call, where latency counts
        dict(name="norm_tiny_f32", kind="norm", dtype="f32", m=1, n=256, delta=False),
        # a decode step of a full batch: the attention's output is added, the next product reads codes
        dict(name="norm_step_8b", kind="norm", dtype="bf16", m=64, n=4096, delta=True),
        # an admission's packed prompts (an odd number of tokens)
        dict(name="norm_prompts_8b", kind="norm", dtype="bf16", m=8005, n=4096, delta=True),
        # a small decoding batch's QKV projection with its bias: the weights' bytes
        _linear("qkv_bias_step", 8, 6144, 4096, bias=True),
        # a full decode batch's output projection with bias and residual
        _linear("wo_step", 64, 4096, 4096, bias=True, residual=True),
        # a plain two-layer MLP's first product at the 1B shape in half precision, an odd batch, from 16-bit rows
        _linear("fc_gelu_1b_f16", 333, 8192, 2048, dtype="f16", act="gelu", bias=True, codes_in=False),
        # the same left in codes for the second product
        _linear("fc_codes_1b", 333, 8192, 2048, act="gelu_tanh", bias=True, codes_out=True),
        # a verify pass (64 windows of 7): gate and up in one product, the gated result left in codes
        _linear("gate_up_verify", 448, 14336, 4096, act="silu", gated=True, codes_out=True),
        # the same of a long packed prefill, 16-bit result: the matrix cores' rate
        _linear("gate_up_prompts", 8005, 14336, 4096, act="silu", gated=True),
        # a block's MLP half: one request's token, verify windows at the 1B shape in half precision, packed prompts
        dict(name="mlp_one_8b", kind="mlp", dtype="bf16", m=1, d=4096, f=14336),
        dict(name="mlp_verify_1b_f16", kind="mlp", dtype="f16", m=160, d=2048, f=8192),
        dict(name="mlp_prompts_8b", kind="mlp", dtype="bf16", m=2777, d=4096, f=14336),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "linear", "mlp"])
    if kind == "norm":
        n = rng.choice([256, 2048, 4096, 8192, 14336, GROUP * _log_int(rng, 1, 120)])
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), m=_log_int(rng, 1, 8000), n=n,
                    delta=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "mlp":
        d, f = rng.choice([(2048, 8192), (4096, 14336), (GROUP * _log_int(rng, 2, 32), GROUP * _log_int(rng, 2, 100))])
        return dict(kind=kind, dtype=dtype, m=_log_int(rng, 1, 2700), d=d, f=f)
    codes_out = rng.random() < 0.35
    # the shapes' projections, and sizes of no configuration (any number of columns; whole groups where codes are written)
    n, k = rng.choice([(6144, 4096), (4096, 4096), (14336, 4096), (4096, 14336), (8192, 2048), (2048, 8192),
                       (GROUP * _log_int(rng, 1, 60) if codes_out else _log_int(rng, 70, 9000), GROUP * _log_int(rng, 1, 60))])
    gated = n * k <= 14336 * 4096 and rng.random() < 0.4
    return dict(kind=kind, dtype=dtype, m=_log_int(rng, 1, 8000 if k <= 4096 else 4000), n=n, k=k, gated=gated,
                act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"] if gated else
                               ["none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                bias=rng.random() < 0.6, residual=not codes_out and rng.random() < 0.4, codes_in=rng.random() < 0.7,
                codes_out=codes_out)


# ------------------------------------------------------------------------------------------------
# what a program has in hand
# ------------------------------------------------------------------------------------------------
def _scale_byte(amax):
    """The exponent byte of the smallest power of two s with amax / s <= 448."""
    m, ex = torch.frexp(amax)                       # amax = m 2^ex, 0.5 <= m < 1; 448 = 0.875 * 2^9
    return torch.where(amax > 0, ex + 118 + (m > 0.875), 0).clamp(LOW, HIGH)


def _encode(x):
    """Rows x (rows, K) in 32 bits as codes (uint8) and exponent bytes (rows, K / 128)."""
    x = x.unflatten(1, (-1, GROUP))
    e = _scale_byte(x.abs().amax(-1))
    inv = ((254 - e).int() << 23).view(torch.float32)     # 2^(127 - e), from its bits
    return (x * inv[..., None]).clamp(-448, 448).to(E4M3).view(torch.uint8).flatten(1), e


def _values(codes, e):
    """What codes (rows, K) with exponent bytes (rows, K / 128) stand for, in 32 bits."""
    scale = (e.int() << 23).view(torch.float32)[..., None]
    return (codes.view(E4M3).unflatten(1, (-1, GROUP)).float() * scale).flatten(1)


def _packed(e):
    """Exponent bytes (rows, K / 128) as (ceil(K / 512), rows, 4)."""
    rows, n = e.shape
    return torch.nn.functional.pad(e, (0, -n % 4)).view(rows, -1, 4).transpose(0, 1).contiguous().to(torch.uint8)


def _unpacked(scales, k):
    return scales.transpose(0, 1).flatten(1)[:, : k // GROUP]


def _weight(g, n, k):
    codes, e = _encode(torch.randn(n, k, device=DEV, generator=g).mul_(k ** -0.5))
    return codes.view(E4M3), _packed(e)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case, "dtype": dtype}
    if kind in ("norm", "mlp"):
        m, n = case["m"], case["n"] if kind == "norm" else case["d"]
        # a residual stream with channels of different size, and rows too
        s["x"] = (normal(m, n) * normal(n).mul_(0.7).exp_() * normal(m, 1).mul_(0.5).exp_()).to(dtype)
        s["delta"] = normal(m, n).to(dtype) if kind == "mlp" or case["delta"] else None
        s["norm"] = normal(n).mul_(0.1).add_(1.0).to(dtype)
        if kind == "mlp":
            s["w1"], s["w2"] = _weight(g, 2 * case["f"], n), _weight(g, n, case["f"])
        return s
    m, n, k = case["m"], case["n"], case["k"]
    rows = (2 if case["gated"] else 1) * n
    # activations with channels of different size, as after a norm or a gate
    x = normal(m, k) * normal(k).mul_(0.5).exp_()
    if case["codes_in"]:
        codes, e = _encode(x)
        s["x"], s["x_scales"] = codes.view(E4M3), _packed(e)
    else:
        s["x"], s["x_scales"] = x.to(dtype), None
    s["w"], s["w_scales"] = _weight(g, rows, k)
    s["bias"] = normal(rows).mul_(0.3).to(dtype) if case["bias"] else None
    s["residual"] = normal(m, n).to(dtype) if case["residual"] else None
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _act(z, name):
    if name == "relu":
        return torch.where(z < 0, 0.0, z)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if name == "gelu_tanh":
        return z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _norm(x, delta, weight):
    """The sum rounded to the rows' type, and its norm in 32 bits."""
    v = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    f = v.float()
    return v, f / torch.sqrt((f * f).mean(-1, keepdim=True) + EPS) * weight.float()


def _product(x, x_e, w, w_scales, bias, act, gated):
    """act(x w^T + bias) in 32 bits, x in codes with exponent bytes x_e."""
    z = torch.matmul(_values(x, x_e), _values(w, _unpacked(w_scales, w.shape[1])).t())
    if bias is not None:
        z = z + bias.float()
    if gated:
        gate, up = z.chunk(2, -1)
        return _act(gate, act) * up
    return _act(z, act)


def _plain(s):
    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind == "norm":
        v, y = _norm(s["x"], s["delta"], s["norm"])
        y = _values(*_encode(y)).to(torch.bfloat16)
        return y if s["delta"] is None else (v, y)
    if kind == "mlp":
        v, y = _norm(s["x"], s["delta"], s["norm"])
        h = _product(*_encode(y), *s["w1"], None, "silu", True)
        return (_product(*_encode(h), *s["w2"], None, "none", False) + v.float()).to(dtype)
    x = (s["x"], _unpacked(s["x_scales"], case["k"])) if case["codes_in"] else _encode(s["x"].float())
    y = _product(*x, s["w"], s["w_scales"], s["bias"], case["act"], case["gated"])
    if case["codes_out"]:
        return _values(*_encode(y)).to(torch.bfloat16)
    return (y if s["residual"] is None else y + s["residual"].float()).to(dtype)


def _own(s):
    from forgeserve_amd import ops

    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind == "linear":
        act = None if case["act"] == "none" else case["act"]
        if case["codes_out"]:
            codes = ops.linear_e4m3_codes(s["x"], s["w"], s["w_scales"], a_scales=s["x_scales"], bias=s["bias"], activation=act,
                                          gated=case["gated"])
            return ops.dequantize_e4m3(*codes, torch.bfloat16)
        return ops.linear_e4m3(s["x"], s["w"], s["w_scales"], a_scales=s["x_scales"], bias=s["bias"], activation=act,
                               gated=case["gated"], residual=s["residual"], dtype=dtype)
    v = None if s["delta"] is None else torch.empty_like(s["x"])
    codes, scales = ops.add_rmsnorm_e4m3(s["x"], s["norm"], EPS, delta=s["delta"], x_out=v)
    if kind == "norm":
        y = ops.dequantize_e4m3(codes, scales, torch.bfloat16)
        return y if v is None else (v, y)
    h, h_scales = ops.linear_e4m3_codes(codes, *s["w1"], a_scales=scales, activation="silu", gated=True)
    return ops.linear_e4m3(h, *s["w2"], a_scales=h_scales, residual=v, dtype=dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    es, kind, m = torch.finfo(DTYPES[case["dtype"]]).bits // 8, case["kind"], case["m"]

    def codes(rows, k):
        return rows * k + rows * k // GROUP

    if kind == "norm":   # codes are written, then read back as two-byte values
        n = case["n"]
        return {"bytes": m * n * es * (3 if case["delta"] else 1) + n * es + 2 * codes(m, n) + 2 * m * n, "flops": 8 * m * n}
    if kind == "mlp":
        d, f = case["d"], case["f"]
        return {"bytes": 3 * m * d * es + d * es + codes(2 * f, d) + codes(d, f), "flops": 6 * m * d * f}
    n, k = case["n"], case["k"]
    rows = (2 if case["gated"] else 1) * n
    out = 2 * codes(m, n) + 2 * m * n if case["codes_out"] else m * n * es * (2 if case["residual"] else 1)
    x = codes(m, k) if case["codes_in"] else m * k * es
    return {"bytes": x + codes(rows, k) + (rows * es if case["bias"] else 0) + out, "flops": 2 * m * rows * k}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _pow2(n):
    """2^n in 64 bits, from its bits."""
    return (n.long() + 1023 << 52).view(torch.float64)


def _rounded(x):
    """x (rows, K) in 64 bits rounded to the nearest values that e4m3 with its groups' scales has (ties to even)."""
    x = x.view(x.shape[0], -1, GROUP)
    m, ex = torch.frexp(x.abs().amax(-1, keepdim=True) / 448.0)
    s = _pow2(torch.where(m > 0.5, ex, ex - 1).clamp(LOW - 127, HIGH - 127))    # 2^ceil(log2(amax / 448))
    y = (x / s).clamp(-448, 448)
    step = _pow2((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)                     # eight steps a binade, down to 2^-6
    return (torch.round(y / step) * step * s).flatten(1)


def _decoded(codes, scales):
    """Codes (rows, K) with packed scales in 64 bits, from their bits."""
    c = torch.arange(256)
    ex, man = (c >> 3) & 15, (c & 7).double()
    v = torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * _pow2(ex - 7))
    look = torch.where(c >= 128, -v, v).to(DEV)
    rows, k = codes.shape
    e = scales.permute(1, 0, 2).reshape(rows, -1)[:, : k // GROUP].long()
    return (look[codes.view(torch.uint8).long()].view(rows, -1, GROUP) * _pow2(e - 127)[:, :, None]).view(rows, k)


def _act64(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return z * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "linear":
        x = _decoded(s["x"], s["x_scales"]) if case["codes_in"] else _rounded(s["x"].double())
        z = x @ _decoded(s["w"], s["w_scales"]).T
        if case["bias"]:
            z += s["bias"].double()
        n = case["n"]
        y = _act64(z[:, :n], case["act"]) * z[:, n:] if case["gated"] else _act64(z, case["act"])
        if case["codes_out"]:
            return _rounded(y)
        return y + s["residual"].double() if case["residual"] else y
    v = s["x"]
    if s["delta"] is not None:   # the sum is held in the rows' type; in 64 bits it has one rounding, as in 32
        v = (v.double() + s["delta"].double()).to(s["dtype"])
    y = v.double() * s["norm"].double() / (v.double().square().mean(-1, keepdim=True) + EPS).sqrt()
    if kind == "norm":
        return _rounded(y) if s["delta"] is None else (v.double(), _rounded(y))
    z = _rounded(y) @ _decoded(*s["w1"]).T
    h = _act64(z[:, : case["f"]], "silu") * z[:, case["f"]:]
    return _rounded(h) @ _decoded(*s["w2"]).T + v.double()
