"""The 8-bit serving operators as their users call them: a key/value cache held in 8-bit floating point as it
is written (with the rotation of the queries and keys) and read back, the paged attention that reads it (one
token per row, speculative windows, packed prompts), and projections whose weights and activations are 8-bit
floating point with a scale for each 128 of K.

Formats (both hold e4m3 codes, 4 exponent and 3 mantissa bits, largest value 448, with a power of two as scale,
kept as its biased exponent byte e: the scale is 2^(e - 127), the smallest one that brings the group's largest
magnitude to 448 or less, between LO and HI of the type that the values are used in):
 * cache: one scale per token, KV head and side (key, value). A (block, head) tile of keys is
   (head_dim / 16, block_size, 16), a tile of values (block_size / 4, head_dim, 4) with the dims of each group of
   64 ordered by d % 16 first, and the scales are (2, block_size): keys', values'.
 * matrices: one scale per row and 128 columns, (ceil(K / 512), rows, 4).

Sizes come from the package's own configurations: the 1B shape (d 2048, 32/8 heads of 64, ffn 8192), the 8B
shape (d 4096, 32/8 heads of 128, ffn 14336), the tiny float32 model (8/4 heads of 32), with the batches,
windows and contexts that the benchmark and the tests run. Lengths that differ from row to row are drawn from
the case's `sizes` number; the values are drawn from the seed.
"""

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 16
E4M3 = torch.float8_e4m3fn
GROUP = 128                                             # columns per scale of a matrix
LIMITS = {"f32": (10, 246), "bf16": (10, 246), "f16": (112, 134)}   # scale exponents: values stay normal, finite


# ------------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # one layer's cache update of a small float32 model through a layer's view: a few tokens are written,
        # the whole cache is read back (the smallest call, where latency counts)
        dict(name="update_tiny_f32", kind="update", dtype="f32", kv_heads=4, hd=32, batch=4, t=3, lo=40, hi=200, sizes=1),
        # the same for a batch with long contexts: what a caller with an attention of its own reads
        dict(name="update_8b", kind="update", dtype="bf16", kv_heads=8, hd=128, batch=16, t=1, lo=512, hi=4096, sizes=2),
        # one decode step's rotation and cache write of 64 rows, and the blocks it wrote read back
        dict(name="write_step_8b", kind="write", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=64, t=1, lo=512,
             hi=8192, sizes=3),
        # an admission's packed ragged prompts, written and read back
        dict(name="write_prompts_8b", kind="write_packed", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=4, lo=300,
             hi=4096, sizes=4),
        # one request decoding a token at an ordinary context: the smallest attention call
        dict(name="attn_one", kind="attn", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=1, t=1, lo=1000, hi=1000,
             pad=False, sizes=5),
        # a decode step of a full batch
        dict(name="attn_decode_8b", kind="attn", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=64, t=1, lo=1024,
             hi=8192, pad=False, sizes=6),
        # a few requests with long contexts
        dict(name="attn_long", kind="attn", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=3, t=1, lo=8000, hi=30000,
             pad=False, sizes=7),
        # the verify windows of a half-precision model at the 1B shape, some rows' windows shorter than the others'
        dict(name="attn_verify_1b_f16", kind="attn", dtype="f16", heads=32, kv_heads=8, hd=64, batch=32, t=5, lo=128,
             hi=2048, pad=True, sizes=8),
        # the attention of an admission's packed ragged prompts
        dict(name="attn_prompts", kind="attn_packed", dtype="bf16", heads=32, kv_heads=8, hd=128, batch=4, lo=300,
             hi=4096, sizes=9),
        # the QKV projection of a small decoding batch at the 8B shape: the weights' bytes
        dict(name="proj_qkv_step", kind="proj", dtype="bf16", m=8, n=6144, k=4096, residual=False),
        # the down projection of a verify pass (64 rows, windows of 7) with its residual
        dict(name="proj_down_verify", kind="proj", dtype="bf16", m=448, n=4096, k=14336, residual=True),
        # the gate and up projection of a long packed prefill (an odd number of tokens): the matrix cores' rate
        dict(name="proj_gate_up_prompts", kind="proj", dtype="bf16", m=8005, n=28672, k=4096, residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["update", "write", "write_packed", "attn", "attn", "attn_packed", "proj", "proj"])
    sizes = rng.randrange(1000)
    if kind == "proj":
        # the projections of the two shapes, and sizes of no configuration (any number of columns)
        n, k = rng.choice([(6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336), (2048, 2048), (16384, 2048),
                           (2048, 8192), (_log_int(rng, 70, 9000), 128 * _log_int(rng, 1, 60))])
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), m=_log_int(rng, 1, 8000), n=n, k=k,
                    residual=rng.random() < 0.4)
    hd, kv_heads, rep = rng.choice([64, 128]), rng.choice([4, 8]), rng.choice([1, 4, 4, 8])
    if kind == "update":
        hi = _log_int(rng, 40, 4096)
        return dict(kind=kind, dtype=rng.choice(["f32", "bf16", "f16"]), kv_heads=kv_heads, hd=rng.choice([32, 64, 128]),
                    batch=_log_int(rng, 1, max(1, min(32, 60000 // hi))), t=rng.choice([1, 1, 5, 7]), lo=hi // 4 + 8, hi=hi,
                    sizes=sizes)
    if kind == "write":
        hi = _log_int(rng, 100, 8192)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * rep, kv_heads=kv_heads, hd=hd,
                    batch=_log_int(rng, 1, 64), t=rng.choice([1, 1, 5, 7]), lo=hi // 8 + 8, hi=hi, sizes=sizes)
    if kind == "write_packed":
        hi = _log_int(rng, 60, 4096)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * 4, kv_heads=kv_heads, hd=hd,
                    batch=max(1, min(8, 12000 // hi)), lo=hi // 8 + 1, hi=hi, sizes=sizes)
    if kind == "attn":
        hi = _log_int(rng, 60, 30000)
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * rep, kv_heads=kv_heads, hd=hd,
                    batch=max(1, min(_log_int(rng, 1, 64), 250000 // hi)), t=rng.choice([1, 1, 1, 3, 5, 7]), lo=hi // 8 + 9,
                    hi=hi, pad=rng.random() < 0.3, sizes=sizes)
    hi = _log_int(rng, 200, 4096)
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16"]), heads=kv_heads * 4, kv_heads=kv_heads, hd=hd,
                batch=max(1, min(8, 10000 // hi)), lo=hi // 8 + 40, hi=hi, sizes=sizes)


# ------------------------------------------------------------------------------------------------
# what a case's sizes and seed stand for
# ------------------------------------------------------------------------------------------------
def _lengths(case):
    """The rows' context or prompt lengths in lo..hi (the first is hi)."""
    r = random.Random(case["sizes"])
    return [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"] - 1)]


def _window_lengths(case):
    """How many of a window's tokens each row has (the first has them all; with `pad` a row may have none)."""
    r = random.Random(case["sizes"] + 1)
    return [case["t"]] + [r.randint(0, case["t"]) if case.get("pad") else case["t"] for _ in range(case["batch"] - 1)]


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g)


def _scale_byte(amax, limits):
    """The exponent byte of the smallest power of two s with amax / s <= 448, between the limits."""
    m, ex = torch.frexp(amax)                       # amax = m 2^ex, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(amax > 0, ex + 118 + (m > 0.875), 0)
    return e.clamp(*limits)


def _encode(x, limits):
    """Codes (uint8) and exponent bytes of x's last dimension as one group each, in 32 bits."""
    e = _scale_byte(x.abs().amax(-1), limits)
    inv = ((254 - e).int() << 23).view(torch.float32)     # 2^(127 - e), from its bits
    codes = (x * inv[..., None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
    return codes, e.to(torch.uint8)


def _value_order(hd):
    """Place of dim d in a tile of values: within each 64 dims (or what is left of them) by d % 16 first."""
    d = torch.arange(hd)
    n = torch.clamp(hd // 16 - 4 * (d // 64), max=4)
    return ((d // 64) * 64 + (d % 16) * n + (d // 16) % 4).to(DEV)


def _decode(codes, e):
    """What codes (.., n) with exponent bytes (..) stand for, in 32 bits."""
    return codes.view(E4M3).float() * (e.int() << 23).view(torch.float32)[..., None]


def _key_rows(tiles):
    """Key tiles (.., hd / 16, block, 16) as rows (.., block, hd)."""
    return tiles.transpose(-2, -3).flatten(-2)


def _value_rows(tiles):
    """Value tiles (.., block / 4, hd, 4) as rows (.., block, hd)."""
    return tiles.index_select(-2, _value_order(tiles.shape[-2])).transpose(-1, -2).flatten(-3, -2)


def _cache(g, case, blocks):
    """A cache of `blocks` blocks with something in every slot: its tiles of keys and of values and its scales."""
    h, d = case["kv_heads"], case["hd"]
    limits = LIMITS[case["dtype"]]

    def side():
        x = _normal(g, blocks, h, BLOCK, d).mul_(_normal(g, blocks, h, BLOCK, 1).mul_(0.5).exp_())
        return _encode(x, limits)

    k, ek = side()
    v, ev = side()
    k = k.unflatten(-1, (d // 16, 16)).transpose(2, 3).contiguous()
    at = torch.empty(d, dtype=torch.long, device=DEV)
    at[_value_order(d)] = torch.arange(d, device=DEV)
    v = v.unflatten(2, (BLOCK // 4, 4)).transpose(-1, -2).index_select(-2, at).contiguous()
    scales = torch.stack([ek, ev], 2).transpose(0, 1).contiguous().transpose(0, 1)   # a head's blocks side by side
    return {"k": k, "v": v, "scales": scales}


def _tables(case, lengths, extra=8):
    """Shuffled block tables of rows of these lengths (zero padded), and the pool's number of blocks."""
    need = [-(-n // BLOCK) for n in lengths]
    ids = list(range(sum(need) + extra))
    random.Random(case["sizes"] + 2).shuffle(ids)
    width, rows, at = max(need), [], 0
    for n in need:
        rows.append(ids[at: at + n] + [0] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device=DEV), len(ids)


def _rope(hd, length, theta=10000.0):
    a = torch.outer(torch.arange(length).double(), theta ** (-torch.arange(0, hd, 2).double() / hd))
    return a.cos().float().to(DEV), a.sin().float().to(DEV)


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    dtype = DTYPES[case["dtype"]]
    s = {"case": case, "dtype": dtype}
    if kind == "proj":
        m, n, k = case["m"], case["n"], case["k"]
        # activations with channels of different size, as after a norm or a gate
        s["x"] = (_normal(g, m, k) * _normal(g, k).mul_(0.7).exp_()).to(dtype)
        w = _normal(g, n, k).mul_(0.02)
        codes, e = _encode(w.unflatten(1, (k // GROUP, GROUP)), LIMITS["f32"])
        s["w"] = codes.flatten(1).view(E4M3)
        s["w_scales"] = _packed_scales(e)
        s["residual"] = _normal(g, m, n).to(dtype) if case["residual"] else None
        return s
    lengths = _lengths(case)
    b, hkv, d = case["batch"], case["kv_heads"], case["hd"]
    tables, blocks = _tables(case, lengths)
    s |= _cache(g, case, blocks) | {"tables": tables}
    if kind in ("update", "write", "attn"):
        t, have = case["t"], torch.tensor(_window_lengths(case), device=DEV)
        first = torch.tensor([max(n - t, 0) for n in lengths], device=DEV)
        step = torch.arange(t, device=DEV)
        s["positions"] = torch.where(step < have[:, None], first[:, None] + step, -1).int().contiguous()
    else:
        n = torch.tensor(lengths, device=DEV)
        step = torch.arange(max(lengths), device=DEV)
        s["positions"] = torch.where(step < n[:, None], step, -1).int().contiguous()
        s["cu"] = torch.cat([n.new_zeros(1), n.cumsum(0)]).int()
        s["token_row"] = torch.arange(b, device=DEV).repeat_interleave(n).int()
        s["token_position"] = s["positions"][s["positions"] >= 0].contiguous()
    if kind == "update":   # new keys and values of one layer, (B, KV heads, T, head_dim)
        s["k_new"], s["v_new"] = (_normal(g, b, hkv, case["t"], d).to(dtype) for _ in range(2))
    elif kind in ("write", "write_packed"):   # rows of the fused projection's output
        rows = sum(lengths) if kind == "write_packed" else b * case["t"]
        s["qkv"] = _normal(g, rows, (case["heads"] + 2 * hkv) * d).to(dtype)
        s["cos"], s["sin"] = _rope(d, case["hi"] + 8)
        s["read"] = tables
        if kind == "write":   # the blocks that hold the window
            last = ((s["positions"][:, -1:].long() // BLOCK))
            s["read"] = tables.gather(1, last).contiguous()
    else:
        rows = sum(lengths) if kind == "attn_packed" else b * case["t"]
        q = _normal(g, rows, case["heads"], d).to(dtype)
        s["q"] = q if kind == "attn_packed" else q.view(b, case["t"], case["heads"], d)
    return s


def _packed_scales(e):
    """Exponent bytes (rows, K / 128) as (ceil(K / 512), rows, 4)."""
    rows, n = e.shape
    return torch.nn.functional.pad(e, (0, -n % 4)).view(rows, -1, 4).transpose(0, 1).contiguous()


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _write(s, k, v, row, position):
    """Encode keys and values (tokens, KV heads, head_dim) and put them into the cache at (row, position)."""
    limits = LIMITS[s["case"]["dtype"]]
    there = position >= 0
    blk = s["tables"][row, position.clamp(min=0) // BLOCK].long()[there]
    slot = (position % BLOCK)[there].long()
    (k, ek), (v, ev) = _encode(k[there], limits), _encode(v[there], limits)
    s["k"].transpose(2, 3)[blk, :, slot] = k.unflatten(-1, (-1, 16))
    to = torch.empty_like(v)
    to[..., _value_order(v.shape[-1])] = v
    s["v"].permute(0, 2, 4, 1, 3)[blk, slot // 4, slot % 4] = to
    s["scales"].permute(0, 3, 1, 2)[blk, slot] = torch.stack([ek, ev], -1)


def _read(s, tables):
    """Every block of the tables in table order, (B, KV heads, blocks * block, head_dim) each, in 32 bits."""
    t = tables.long()
    e = s["scales"][t]                                   # (B, blocks, heads, 2, block)
    k = _decode(_key_rows(s["k"][t]), e[:, :, :, 0])     # (B, blocks, heads, block, hd)
    v = _decode(_value_rows(s["v"][t]), e[:, :, :, 1])
    return tuple(x.transpose(1, 2).flatten(2, 3) for x in (k, v))


def _rotate(x, position, cos, sin):
    """Half-split rotation of x (tokens, heads, head_dim) at positions (tokens,), in 32 bits; zeros at -1."""
    p = position.clamp(min=0).long()
    c, sn = cos[p][:, None], sin[p][:, None]
    a, b = x.float().chunk(2, -1)
    out = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    return torch.where((position >= 0)[:, None, None], out, 0.0)


def _attend(s, q, positions):
    """q (B, T, heads, hd), positions (B, T) -> softmax(q k^T / sqrt(hd)) v over the keys 0..position."""
    b, t, h, d = q.shape
    k, v = _read(s, s["tables"])
    hkv, n = k.shape[1], k.shape[2]
    q = q.float().view(b, t, hkv, h // hkv, d).transpose(1, 2).flatten(2, 3)    # (B, KV heads, T * group, hd)
    scores = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    seen = torch.arange(n, device=DEV) <= positions[:, :, None]
    seen = seen.repeat_interleave(h // hkv, 1)[:, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.matmul(w, v) / torch.where(total == 0, 1.0, total)
    return out.view(b, hkv, t, h // hkv, d).transpose(1, 2).flatten(2, 3)


def _plain(s):
    case, dtype, kind = s["case"], s["dtype"], s["case"]["kind"]
    if kind == "proj":
        k = case["k"]
        x, ex = _encode(s["x"].float().unflatten(1, (k // GROUP, GROUP)), LIMITS["f32"])
        ew = s["w_scales"].transpose(0, 1).flatten(1)[:, : k // GROUP]
        w = _decode(s["w"].view(torch.uint8).unflatten(1, (k // GROUP, GROUP)), ew).flatten(1)
        y = torch.matmul(_decode(x, ex).flatten(1), w.t())
        return (y if s["residual"] is None else y + s["residual"].float()).to(dtype)
    hkv, d, pos = case["kv_heads"], case["hd"], s["positions"]
    if kind == "update":
        row = torch.arange(pos.shape[0], device=DEV)[:, None].expand_as(pos).flatten()
        new = (x.float().transpose(1, 2).flatten(0, 1) for x in (s["k_new"], s["v_new"]))
        _write(s, *new, row, pos.flatten().long())
        return tuple(x.to(dtype) for x in _read(s, s["tables"]))
    if kind in ("write", "write_packed"):
        if kind == "write":
            row, at = torch.arange(pos.shape[0], device=DEV)[:, None].expand_as(pos).flatten(), pos.flatten()
        else:
            row, at = s["token_row"], s["token_position"]
        qkv = s["qkv"].unflatten(1, (-1, d))
        qk = _rotate(qkv[:, : -hkv], at, s["cos"], s["sin"])
        _write(s, qk[:, case["heads"]:], qkv[:, -hkv:].float(), row.long(), at.long())
        return (qk[:, : case["heads"]].flatten(1).to(dtype), *(x.to(dtype) for x in _read(s, s["read"])))
    if kind == "attn":
        return _attend(s, s["q"], pos).to(dtype)
    there = pos >= 0
    q = torch.zeros(*pos.shape, *s["q"].shape[1:], dtype=dtype, device=DEV)
    q[there] = s["q"]
    return _attend(s, q, pos)[there].to(dtype)


def _own(s):
    from forgeserve_amd import ops

    case, kind = s["case"], s["case"]["kind"]
    if kind == "proj":
        return ops.gemm_e4m3(s["x"], s["w"], s["w_scales"], residual=s["residual"])
    if "layout" not in s:   # the handle that a program keeps for a layer of its cache
        s["layout"] = ops.kv_layout_e4m3(s["k"], s["v"], s["scales"], s["dtype"])
    lay, scale = s["layout"], 1.0 / math.sqrt(case["hd"])
    if kind == "update":
        ops.paged_kv_write(s["k_new"], s["v_new"], s["positions"], s["tables"], lay)
        return ops.paged_gather(lay, s["tables"], s["dtype"], s["q"].device if "q" in s else s["k_new"].device)
    if kind == "write":
        q = ops.qkv_rope_write(s["qkv"], s["positions"].view(-1), case["t"], case["heads"], s["cos"], s["sin"], s["tables"],
                               lay)
        return (q, *ops.paged_gather(lay, s["read"], s["dtype"], s["qkv"].device))
    if kind == "write_packed":
        q = ops.qkv_rope_write_varlen(s["qkv"], s["token_position"], s["token_row"], case["heads"], s["cos"], s["sin"],
                                      s["tables"], lay)
        return (q, *ops.paged_gather(lay, s["read"], s["dtype"], s["qkv"].device))
    if kind == "attn":
        return ops.paged_attention(s["q"], lay, s["tables"], s["positions"], scale)
    return ops.paged_attention_varlen(s["q"], lay, s["tables"], s["positions"], s["cu"], scale)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    es, kind = torch.finfo(DTYPES[case["dtype"]]).bits // 8, case["kind"]
    if kind == "proj":
        m, n, k = case["m"], case["n"], case["k"]
        out = m * n * es * (2 if case["residual"] else 1)
        return {"bytes": m * k * es + n * k + n * k // GROUP + out, "flops": 2 * m * n * k}
    hkv, d, lengths = case["kv_heads"], case["hd"], _lengths(case)
    slot = 2 * hkv * (d + 1)            # a token's codes and scales
    if kind in ("update", "write", "write_packed"):
        tokens = sum(lengths) if kind == "write_packed" else sum(_window_lengths(case))
        width = max(-(-n // BLOCK) for n in lengths)
        read = case["batch"] * (1 if kind == "write" else width) * BLOCK
        new = tokens * 2 * hkv * d * es
        q = 0 if kind == "update" else 2 * tokens * case["heads"] * d * es + tokens * d * 4
        return {"bytes": new + q + tokens * slot + read * (slot + 2 * hkv * d * es), "flops": 4 * (tokens + read) * hkv * d}
    if kind == "attn":
        seen = [(max(n - case["t"], 0) + w, w) for n, w in zip(lengths, _window_lengths(case))]
        keys = sum(n for n, w in seen if w)
        pairs = sum(w * n - w * (w - 1) // 2 for n, w in seen)
        tokens = case["batch"] * case["t"]
    else:
        keys, tokens = sum(lengths), sum(lengths)
        pairs = sum(n * (n + 1) // 2 for n in lengths)
    return {"bytes": keys * slot + 2 * tokens * case["heads"] * d * es, "flops": 4 * pairs * case["heads"] * d}


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------
def _pow2(n):
    """2^n in 64 bits, from its bits."""
    return (n.long() + 1023 << 52).view(torch.float64)


def _round_e4m3(x, limits):
    """x (.., n) in 64 bits rounded to the nearest multiples that e4m3 with the group's scale has (ties to even)."""
    m, ex = torch.frexp(x.abs().amax(-1, keepdim=True) / 448.0)
    ex = torch.where(m > 0.5, ex, ex - 1)                    # ceil(log2(amax / 448))
    s = _pow2(ex.clamp(limits[0] - 127, limits[1] - 127))
    y = (x / s).clamp(-448, 448)
    _, ey = torch.frexp(y)
    step = _pow2((ey - 1).clamp(min=-6) - 3)   # eight steps a binade, down to 2^-6
    return torch.round(y / step) * step * s


def _table_values():
    """The 256 codes' values in 64 bits, from their bits."""
    c = torch.arange(256)
    ex, man = (c >> 3) & 15, (c & 7).double()
    v = torch.where(ex == 0, man * 2.0 ** -9, (1 + man / 8) * _pow2(ex - 7))
    v[(c & 127) == 127] = math.nan
    return torch.where(c >= 128, -v, v).to(DEV)


def _slot_values(s, blocks):
    """Blocks (n,) of the cache in 64 bits: (heads, n * block, hd) of keys and of values."""
    look, d = _table_values(), s["case"]["hd"]
    sc = _pow2(s["scales"][blocks].long() - 127)       # (n, heads, 2, block)
    k = look[s["k"][blocks].long()]                                # (n, heads, hd / 16, block, 16)
    k = k.movedim(3, 2).reshape(*k.shape[:2], BLOCK, d) * sc[:, :, 0, :, None]
    v = look[s["v"][blocks].long()]                                # (n, heads, block / 4, hd, 4)
    v = v[:, :, :, _value_order(d)].movedim(4, 3).reshape(*v.shape[:2], BLOCK, d) * sc[:, :, 1, :, None]
    return tuple(x.transpose(0, 1).reshape(x.shape[1], -1, d) for x in (k, v))


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "proj":
        m, n, k = case["m"], case["n"], case["k"]
        x = _round_e4m3(s["x"].double().view(m, k // GROUP, GROUP), LIMITS["f32"]).view(m, k)
        e = s["w_scales"].permute(1, 0, 2).reshape(n, -1)[:, : k // GROUP].long()
        w = _table_values()[s["w"].view(torch.uint8).long()].view(n, k // GROUP, GROUP)
        w = (w * _pow2(e - 127)[:, :, None]).view(n, k)
        y = x @ w.T
        return y if s["residual"] is None else y + s["residual"].double()
    d, hkv, limits = case["hd"], case["kv_heads"], LIMITS[case["dtype"]]
    tables, pos = s["tables"].long(), s["positions"].long()
    if kind in ("attn", "attn_packed"):
        rep, outs = case["heads"] // hkv, []
        for r in range(case["batch"]):
            here = pos[r][pos[r] >= 0]
            q = s["q"][r] if kind == "attn" else s["q"][int(s["cu"][r]): int(s["cu"][r + 1])]
            out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
            if here.numel():
                n = int(here.max()) + 1
                k, v = _slot_values(s, tables[r, : -(-n // BLOCK)])
                hidden = torch.arange(n, device=DEV)[None, :] > here[:, None]
                for h in range(case["heads"]):
                    z = (q[: here.numel(), h].double() @ k[h // rep, :n].T) * d ** -0.5
                    out[: here.numel(), h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[h // rep, :n]
            outs.append(out)
        return torch.stack(outs) if kind == "attn" else torch.cat(outs)
    # the new tokens, in the order of the calls' rows
    if kind == "update":
        k, v = (x.double().permute(0, 2, 1, 3).reshape(-1, hkv, d) for x in (s["k_new"], s["v_new"]))
        q = None
    else:
        at = (pos if kind == "write" else s["token_position"].long()).reshape(-1)
        rows = s["qkv"].double().view(-1, case["heads"] + 2 * hkv, d)
        c, sn = (x.double()[at.clamp(min=0)][:, None] for x in (s["cos"], s["sin"]))
        a, b = rows[:, : case["heads"] + hkv, : d // 2], rows[:, : case["heads"] + hkv, d // 2:]
        turned = torch.cat([a * c - b * sn, a * sn + b * c], -1)
        q, k, v = turned[:, : case["heads"]].reshape(len(at), -1), turned[:, case["heads"]:], rows[:, case["heads"] + hkv:]
    k, v = _round_e4m3(k, limits), _round_e4m3(v, limits)
    at = (s["token_position"].long() if kind == "write_packed" else pos.reshape(-1))
    row = (s["token_row"].long() if kind == "write_packed" else
           torch.arange(case["batch"], device=DEV).repeat_interleave(case["t"]))
    blk, slot = tables[row, at // BLOCK], at % BLOCK
    read = (s["read"] if "read" in s else s["tables"]).long()
    place = torch.full((s["k"].shape[0] * BLOCK,), -1, dtype=torch.long, device=DEV)   # the token now in a slot
    place[blk * BLOCK + slot] = torch.arange(len(at), device=DEV)
    ks, vs = [], []
    for r in range(read.shape[0]):
        old_k, old_v = _slot_values(s, read[r])
        new = place[(read[r][:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).reshape(-1)]
        is_new = (new >= 0)[None, :, None]
        ks.append(torch.where(is_new, k[new.clamp(min=0)].transpose(0, 1), old_k))
        vs.append(torch.where(is_new, v[new.clamp(min=0)].transpose(0, 1), old_v))
    k, v = torch.stack(ks), torch.stack(vs)
    return (k, v) if q is None else (q, k, v)
