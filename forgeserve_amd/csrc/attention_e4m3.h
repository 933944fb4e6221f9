// Attention over a pool of e4m3 codes on the matrix cores: bf16 and f16 rows, head_dim 64 or 128, block_size a
// multiple of 16 (attention.hip includes this file and says how the work is split, planned, folded and joined).
//
// The same transposed products as over a 16-bit pool, S^T = K.Q^T and O^T += V^T.P^T, with the codes turned into 16-bit
// operands in registers. Both conversions are exact: a key's scale is applied by the conversion itself; a value's, which
// differs from key to key within an operand, goes into the probabilities (bf16: p is rounded once, after the exact
// product with the power of two) or multiplies the operand (f16, whose range p times a scale would leave). So the only
// roundings are p's to 16 bits, which the product of 16-bit operands needs and the bf16 pool's attention has too (the f16
// pool's scalar kernel keeps p in f32: f16 rows give up that much for the matrix cores, 2.1e-4 -> 2.3e-4 of the output's
// norm), the output's, and the sums', in f32; l sums p unrounded.
//
// The tiles are stored so that a wave's loads are whole: 16 bytes a lane are dims 16c .. 16c+15 of a key (lane l16 = key,
// c = g, g + 4), which makes k-step 2j + h of the product dims 16 (g + 4j) + 8h .. +7 of lane group g, for the keys as
// for the queries; and of the values dims r, r + 16, r + 32, r + 48 of four keys.
//
// A pair of tiles is 64 conversions a lane at 128 dims, as many vector instructions again for its softmax (T = 1, four
// heads a KV head) and 16 products, about 1 us for a wave alone on its SIMD: a large batch's 2,048 waves draw 6.1 TB/s
// (64 rows of 1024-8192 keys, 32/8 heads: 109 us; the 16-bit pool's kernel 188 us for twice the bytes), a few long rows
// are bound by their longest wave (3 rows of 8000-30000 keys: 34-38 us in 140 workgroups, 127 MB; one row of 1000 keys:
// 10.4 us, most of it the launch and one load after another).
//
// A score that is NaN makes its row's output NaN, and so does a value that is NaN in its dim, for the rows that see it
// and for no other.

namespace {

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8_t;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2_t;

template <bool B> struct Flag { static constexpr bool value = B; };

// Operand bits of the two row dtypes.
template <int DT> struct Operand;
template <> struct Operand<FS_BF16> {
  static constexpr uint32_t ONES = 0x3f803f80u, EXPONENTS = 0x7f807f80u;   // pairs of 1.0, and of all exponent bits
  static FS_DEVICE float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  template <bool HI>
  static FS_DEVICE uint32_t pair(uint32_t codes, float scale) {   // two codes times the scale
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
  }
  static FS_DEVICE uint32_t round2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, bf16x2_t));
  }
};
template <> struct Operand<FS_F16> {
  static constexpr uint32_t ONES = 0x3c003c00u, EXPONENTS = 0x7c007c00u;
  static FS_DEVICE float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  template <bool HI>
  static FS_DEVICE uint32_t pair(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HI));
  }
  static FS_DEVICE uint32_t round2(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_t));
  }
  static FS_DEVICE uint32_t times(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, a) * __builtin_bit_cast(f16x2_t, b));
  }
};

// Eight codes as an operand: eight dims of a key with its scale, or (scale 1) four values of one dim from each tile.
template <int DT>
FS_DEVICE u32x4 operand8(uint32_t a, uint32_t b, float scale) {
  typedef Operand<DT> O;
  return u32x4{O::template pair<false>(a, scale), O::template pair<true>(a, scale), O::template pair<false>(b, scale),
               O::template pair<true>(b, scale)};
}

// The scales of a lane's four keys of a tile, from their exponent bytes.
FS_DEVICE void four_scales(uint32_t bytes, float (&s)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = scale_value((bytes >> (8 * e)) & 0xffu);
}
// f16: those of two tiles as operand bits, key by key.
FS_DEVICE u32x4 scale_operand(const float (&a)[4], const float (&b)[4]) {
  typedef Operand<FS_F16> O;
  return u32x4{O::round2(a[0], a[1]), O::round2(a[2], a[3]), O::round2(b[0], b[1]), O::round2(b[2], b[3])};
}
FS_DEVICE u32x4 times8(u32x4 v, u32x4 s) {
  typedef Operand<FS_F16> O;
  return u32x4{O::times(v[0], s[0]), O::times(v[1], s[1]), O::times(v[2], s[2]), O::times(v[3], s[3])};
}

FS_DEVICE u32x4 signed_query_bits(u32x4 q, float scale_log2) {
  return __builtin_bit_cast(u32x4, signed_query(__builtin_bit_cast(bf16x8_t, q), scale_log2));   // (the same bits in f16)
}

template <int DT, int D, bool TWO>
FS_DEVICE void tile_scores_e4m3(const u32x4 (&kf)[D / 32], const u32x4 (&qf)[2][D / 32], float4_t (&sc)[2]) {
  sc[0] = float4_t{0.f, 0.f, 0.f, 0.f};
  sc[1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) {
    sc[0] = Operand<DT>::mfma(kf[ks], qf[0][ks], sc[0]);
    if (TWO) sc[1] = Operand<DT>::mfma(kf[ks], qf[1][ks], sc[1]);
  }
}

// f16 holds p times 2^7 (as do l and the sums, of every partial, so that it leaves the quotient): the largest, 2^REF_SLACK
// of it, still fits, and eleven bits are kept down to 2^-21 of the reference, within 2^-32 of it below, where p as it is
// would have lost them below 2^-14 and been nothing below 2^-25. (bf16: p times the value's scale, at least 2^-117, is
// below a normal number only for values of 1e-30 and less.)
template <int DT> constexpr float P_LOG2 = DT == FS_F16 ? 7.f : 0.f;

// pair_probs with a value's scale in its probability (bf16). A score that is NaN moves no reference; its p, l and
// sums are NaN (and partial_reference keeps such a partial from counting as empty).
template <int DT, bool TWO, class Scales>
FS_DEVICE bool pair_probs_e4m3(const float (&sc)[2][2][4], Scales scales, float scale, float (&m_run)[2], float (&l_run)[2],
                               float (&alpha)[2], u32x4 (&pf)[2]) {
  constexpr int NT = TWO ? 2 : 1;
  typedef Operand<DT> O;
  float x[2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float a[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) a[e] = __builtin_elementwise_maximum(sc[0][nt][e], sc[1][nt][e]);
    x[nt] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(a[0], a[1]), __builtin_elementwise_maximum(a[2], a[3]));
  }
  const bool moved = __any(x[0] * scale > m_run[0] + REF_SLACK || (TWO && x[1] * scale > m_run[1] + REF_SLACK));
  if (moved) {
    float tmax[2];
    max_across_groups2(x[0], x[TWO ? 1 : 0], tmax[0], tmax[1]);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float t = tmax[nt] * scale;
      const bool mv = t > m_run[nt] + REF_SLACK;
      const float m_new = mv ? t : m_run[nt];
      alpha[nt] = mv ? fast_exp2(m_run[nt] - m_new) : 1.f;
      l_run[nt] *= alpha[nt];
      m_run[nt] = m_new;
    }
  }
  float ref[2], sum[2] = {0.f, 0.f};
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) ref[nt] = (m_run[nt] == -INFINITY ? 0.f : m_run[nt]) - P_LOG2<DT>;   // (a row that has seen nothing yet: every p is 0)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float vs[4];
    if (DT == FS_BF16) scales(u, vs);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float pv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) pv[e] = fast_exp2(fmaf(sc[u][nt][e], scale, -ref[nt]));
      sum[nt] += (pv[0] + pv[1]) + (pv[2] + pv[3]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x = pv[2 * c], y = pv[2 * c + 1];
        pf[nt][2 * u + c] = DT == FS_BF16 ? O::round2(x * vs[2 * c], y * vs[2 * c + 1]) : O::round2(x, y);
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) l_run[nt] += sum[nt];
  return moved;
}

// The reference of a finished partial: one that saw NaN alone has none yet, and would pass for an empty one.
FS_DEVICE float partial_reference(float m, float l) { return __builtin_isnan(l) ? 0.f : m; }

// The bytes of four codes that are NaN: 0x80 there, 0 elsewhere.
FS_DEVICE uint32_t nan_codes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// pair_step over codes: value(mt) is the pair's values of dims 16 mt .. as an operand, scales(u, s) the scales of the
// lane's four keys of tile u (bf16; f16's value has them), nans() not 0 if one of the lane's codes of values is NaN. In a
// pair that some row sees only in part, a value that is NaN is zeroed in the operand, and a product of two indicators
// (which values are NaN, which keys a row sees) says which sums it belongs to: 0 * NaN would reach the rows that may not
// see it. (The search runs over the codes, four at a time: over the operands it took longer than the rest of the pair.)
// again() makes the compiler take the values for new ones: else it would keep all of a pair's operands in registers from
// the search for NaN to the products, and from there to the indicators.
template <int DT, int D, bool TWO, bool SEEN = false, class Value, class Nans, class Again, class Scales>
FS_DEVICE void pair_step_e4m3(const float4_t (&sc)[2][2], Value value, Nans nans, Again again, Scales scales, int j0, const bool (&ok)[2],
                              bool fresh, int qmax, const int (&rpos)[2], int rmin, float scale, float4_t (&acc)[D / 16][2],
                              float (&m_run)[2], float (&l_run)[2]) {
  constexpr int MT = D / 16;
  constexpr int NT = TWO ? 2 : 1;
  typedef Operand<DT> O;
  const int g = (threadIdx.x & 63) >> 4;
  const bool full = SEEN || (ok[0] && ok[1] && j0 + 31 <= rmin);   // wave-uniform
  float s[2][2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][nt][e] = sc[u][nt][e];
  // the row sees the lane's keys e <= last_key(u, row's position)
  auto last_key = [&](int u, int pos) { return (ok[u] ? pos : -1) - j0 - 16 * u - 4 * g; };
  if (!full) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int last = last_key(u, rpos[nt]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] = e <= last ? s[u][nt][e] : -INFINITY;
      }
  }
  u32x4 pf[2];
  float alpha[2];
  const bool moved = pair_probs_e4m3<DT, TWO>(s, scales, scale, m_run, l_run, alpha, pf);
  if (moved && !fresh) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mt][nt][e] *= alpha[nt];
  }
  // all bits of an operand's keys that a row at `pos` sees
  auto seen_bits = [&](int pos) {
    u32x4 k;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int last = last_key(c >> 1, pos), e = 2 * (c & 1);   // keys e, e + 1
      k[c] = (e <= last ? 0xffffu : 0u) | (e < last ? 0xffff0000u : 0u);
    }
    return k;
  };
  // all bits of an operand's values that are NaN (codes have no infinities)
  auto nan_bits = [](u32x4 v) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t x = ~v[c] & O::EXPONENTS;
      v[c] = ((x & 0xffffu) == 0 ? 0xffffu : 0u) | ((x >> 16) == 0 ? 0xffff0000u : 0u);
    }
    return v;
  };
  bool any_nan = false;
  u32x4 keep = {~0u, ~0u, ~0u, ~0u};
  if (!full) {
    keep = seen_bits(qmax);
    // a probability is 0 where its key is hidden, whatever the scale there
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) pf[nt] &= seen_bits(rpos[nt]);
    any_nan = __any(nans() != 0);
    again();
  }
  __builtin_amdgcn_sched_barrier(0);
  u32x4 v[2][2];
  v[0][0] = value(0);
  v[0][1] = value(1);
#pragma unroll
  for (int mt = 0; mt < MT; mt += 2) {
    u32x4(&now)[2] = v[mt / 2 & 1], (&next)[2] = v[(mt / 2 & 1) ^ 1];
    if (mt + 2 < MT) {
      next[0] = value(mt + 2);
      next[1] = value(mt + 3);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!full && any_nan) {
#pragma unroll
      for (int i = 0; i < 2; ++i) now[i] &= keep & ~nan_bits(now[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      acc[mt + i][0] = O::mfma(now[i], pf[0], acc[mt + i][0]);
      if (TWO) acc[mt + i][1] = O::mfma(now[i], pf[1], acc[mt + i][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (!full && any_nan) {
    again();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const u32x4 seen = seen_bits(rpos[nt]) & O::ONES;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const float4_t n = O::mfma(nan_bits(value(mt)) & keep & O::ONES, seen, float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mt][nt][e] = n[e] > 0.f ? __uint_as_float(0x7fc00000u) : acc[mt][nt][e];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// The smallest position of a tile's queries, padding apart (rows_min_pos's -1 would send every pair of a padded window
// through the masks: 32 padded windows of 5 over 128-2048 keys, 64 dims, took 24 us for 16). What a padding row sums over
// pairs that all others see is never looked at: attn_emit gives it zeros.
FS_DEVICE int rows_min_seen(const int (&rpos)[2], int nrows) {
  const int l16 = threadIdx.x & 15;
  int v = 0x7ffffffe;
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) v = 16 * nt + l16 < nrows && rpos[nt] >= 0 ? min(v, rpos[nt]) : v;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

// The queries of a wave's 32-row tile as operands: Q[row][16 (g + 4j) + 8h .. +8] in k-step 2j + h.
template <int DT, int D, int NT>
FS_DEVICE void load_queries_e4m3(const AttnParams& P, int b, int hkv, int row0, int nrows, u32x4 (&qf)[2][D / 32]) {
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const uint16_t* qbase = reinterpret_cast<const uint16_t*>(P.q);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = row0 + 16 * nt + l16;
    const bool ok = (16 * nt + l16) < nrows && token_exists(P, b, r / P.G);
    const int t = ok ? r / P.G : 0;
    const int h = hkv * P.G + (ok ? r - (r / P.G) * P.G : 0);
    const uint16_t* qr = qbase + q_offset(P, b, t) + (int64_t)h * P.q_sh;
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
      qf[nt][ks] = ok ? signed_query_bits(*reinterpret_cast<const u32x4*>(qr + 16 * (g + 4 * (ks >> 1)) + 8 * (ks & 1)), P.scale_log2)
                      : u32x4{};
  }
}

// ------------------------------------------------------------------------------------------------
// unit kernels' tiles
// ------------------------------------------------------------------------------------------------
// A wave's share of a unit, as attn_wave_tiles. A pair of tiles is 8 loads of 16 bytes a lane (128 dims), a byte of the
// key's scale and a word of four values' per tile. NP pairs are in registers.
template <int DT, int D, int BSZ, bool TWO, int NP>
__device__ __attribute__((always_inline)) inline void attn_wave_tiles_e4m3(const AttnParams& P, int b, int kbeg, int kend,
                                                                           int qmax, int row0, int nrows,
                                                                           const int (&rpos)[2], int hkv, int w,
                                                                           float4_t (*red_acc)[64], float* red_m,
                                                                           float* red_l) {
  constexpr int KS = D / 32, MT = D / 16, NT = TWO ? 2 : 1;
  constexpr int C = D / 64;   // 16-byte loads of keys, and of values, per tile
  const int lane = threadIdx.x & 63;
  const int l16 = lane & 15, g = lane >> 4;
  const int ntiles = (kend - kbeg + 15) >> 4;
  const int npairs = (ntiles + 1) >> 1;
  const int np_w = npairs > w ? (npairs - w + UNIT_WAVES - 1) / UNIT_WAVES : 0;   // <= 64 pairs
  auto pair_key = [&](int i) { return kbeg + 32 * (w + UNIT_WAVES * i); };
  const int BS = BSZ ? BSZ : P.kv.block_size;

  // lane i: where the tiles of the wave's pair i start, in bytes (64 bits), and which of them are there
  const uint8_t* kpool = key_tile(P.kv, 0, hkv);
  const uint8_t* vpool = value_tile(P.kv, 0, hkv);
  const uint8_t* spool = tile_scales(P.kv, 0, hkv);
  uint64_t k_at[2], v_at[2], s_at[2];
  uint64_t mapped[2];
  bool all_mapped = true;
  {
    int phys[2] = {-1, -1}, slot0[2] = {0, 0};
    bool exists[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int j0 = pair_key(lane) + 16 * u, blk = j0 / BS;
      exists[u] = lane < np_w && j0 < kend;
      if (exists[u]) {
        slot0[u] = j0 - blk * BS;
        if (blk < P.max_blocks) phys[u] = P.table[(int64_t)b * P.table_stride + blk];
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const bool ok = phys[u] >= 0 && phys[u] < P.kv.num_blocks;
      mapped[u] = __ballot(ok);
      all_mapped &= mapped[u] == __ballot(exists[u]);
      const int64_t pb = ok ? phys[u] : 0;
      k_at[u] = (uint64_t)(pb * P.kv.k_block + 16 * slot0[u]);
      v_at[u] = (uint64_t)(pb * P.kv.v_block + D * slot0[u]);
      s_at[u] = (uint64_t)(pb * P.kv.k_slot + slot0[u]);
    }
    if (!exists[1]) {
      k_at[1] = k_at[0];
      v_at[1] = v_at[0];
      s_at[1] = s_at[0];
    }
  }

  u32x4 qf[2][KS];
  load_queries_e4m3<DT, D, NT>(P, b, hkv, row0, nrows, qf);

  static_assert(NP * 2 * (2 * C + 2) < 64, "vmcnt counts every load in flight");
  struct Keys {
    u32x4 k[2][C];
    uint32_t s[2];
  } kb[NP];
  struct Values {
    u32x4 v[2][C];
    uint32_t s[2];
  } vb[NP];
  uint32_t k_lane[C];
#pragma unroll
  for (int j = 0; j < C; ++j) k_lane[j] = (uint32_t)((g + 4 * j) * 16 * BS + 16 * l16);
  const uint32_t v_lane = (uint32_t)(4 * D * g + 16 * l16);
  auto tile_at = [&](const uint8_t* pool, uint64_t at, int i) {
    const int l = max(min(i, np_w - 1), 0);
    const uint32_t lo = __builtin_amdgcn_readlane((int)at, l), hi = __builtin_amdgcn_readlane((int)(at >> 32), l);
    uint64_t t = reinterpret_cast<uint64_t>(pool) + ((uint64_t)hi << 32 | lo);
    asm("" : "+s"(t));   // a scalar base and 32-bit lane offsets: no 64-bit vector adds per load
    return (__attribute__((address_space(1))) const char*)t;
  };
  typedef __attribute__((address_space(1))) const u32x4 GCodes;
  typedef __attribute__((address_space(1))) const uint8_t GByte;
  typedef __attribute__((address_space(1))) const uint32_t GWord;
  auto load_keys = [&](int pair, Keys& x) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      auto kt = tile_at(kpool, k_at[u], pair);
#pragma unroll
      for (int j = 0; j < C; ++j) x.k[u][j] = __builtin_nontemporal_load((GCodes*)(kt + k_lane[j]));
      x.s[u] = *(GByte*)(tile_at(spool, s_at[u], pair) + l16);
    }
  };
  auto load_values = [&](int pair, Values& x) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      auto vt = tile_at(vpool, v_at[u], pair);
#pragma unroll
      for (int j = 0; j < C; ++j) x.v[u][j] = __builtin_nontemporal_load((GCodes*)(vt + (v_lane + 256 * j)));
      x.s[u] = *(GWord*)(tile_at(spool, s_at[u], pair) + (BS + 4 * g));
    }
  };
#pragma unroll
  for (int j = 0; j < NP; ++j) {   // in the order that the loops' waits count
    load_keys(j, kb[j]);
    __builtin_amdgcn_sched_barrier(0);
    load_values(j, vb[j]);
    __builtin_amdgcn_sched_barrier(0);
  }

  float4_t acc[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    acc[mt][0] = float4_t{0.f, 0.f, 0.f, 0.f};
    acc[mt][1] = float4_t{0.f, 0.f, 0.f, 0.f};
  }
  float m_run[2] = {-INFINITY, -INFINITY};
  float l_run[2] = {0.f, 0.f};

  const int rmin = rows_min_seen(rpos, nrows);
  const int n_seen = rmin + 1 > kbeg ? min((rmin + 1 - kbeg) >> 5, ntiles >> 1) : 0;   // pairs all rows see
  const int n_full = all_mapped && n_seen > w ? (n_seen - w + UNIT_WAVES - 1) / UNIT_WAVES : 0;
  const float scale = positive_scale(P.scale_log2);
  auto there = [&](int i, int u) { return i < np_w && ((mapped[u] >> (i & 63)) & 1) != 0; };
  int i = 0;
  auto scores = [&](const Keys& x, float4_t (&sc)[2][2]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float s = scale_value(x.s[u]);
      u32x4 kf[KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        kf[ks] = operand8<DT>(x.k[u][ks >> 1][2 * (ks & 1)], x.k[u][ks >> 1][2 * (ks & 1) + 1], s);
      tile_scores_e4m3<DT, D, TWO>(kf, qf, sc[u]);
    }
  };
  auto pair = [&](int j, auto seen, bool refill) {
    const int p = i + j;
    float4_t sc[2][2];
    scores(kb[j], sc);
    if (refill) {
      __builtin_amdgcn_sched_barrier(0);
      load_keys(p + NP, kb[j]);
    }
    auto scales = [&](int u, float (&vs)[4]) { four_scales(vb[j].s[u], vs); };
    u32x4 vso = {};
    if (DT == FS_F16) {
      float a[4], c[4];
      scales(0, a);
      scales(1, c);
      if constexpr (!decltype(seen)::value) {   // (a slot that was never written may hold any byte: it must stay finite)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = fminf(a[e], scale_value(ScaleRange<FS_F16>::HI));
          c[e] = fminf(c[e], scale_value(ScaleRange<FS_F16>::HI));
        }
      }
      vso = scale_operand(a, c);
    }
    auto value = [&](int mt) {
      const u32x4 o = operand8<DT>(vb[j].v[0][mt >> 2][mt & 3], vb[j].v[1][mt >> 2][mt & 3], 1.f);
      return DT == FS_F16 ? times8(o, vso) : o;
    };
    auto nans = [&]() {
      uint32_t n = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) n |= nan_codes(vb[j].v[u][c][e]);
      return n;
    };
    auto again = [&]() {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c) asm volatile("" : "+v"(vb[j].v[u][c]));
    };
    if constexpr (decltype(seen)::value)
      pair_step_e4m3<DT, D, TWO, true>(sc, value, nans, again, scales, 0, {true, true}, p == 0, 0, rpos, rmin, scale, acc, m_run, l_run);
    else
      pair_step_e4m3<DT, D, TWO>(sc, value, nans, again, scales, pair_key(p), {there(p, 0), there(p, 1)}, p == 0, qmax, rpos, rmin, scale, acc,
                                 m_run, l_run);
    if (refill) {
      __builtin_amdgcn_sched_barrier(0);
      load_values(p + NP, vb[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (; i + NP <= n_full && i + NP < np_w; i += NP) {
#pragma unroll
    for (int j = 0; j < NP; ++j) pair(j, Flag<true>{}, true);
  }
  for (; i + NP < np_w; i += NP) {
#pragma unroll
    for (int j = 0; j < NP; ++j) pair(j, Flag<false>{}, true);
  }
#pragma unroll
  for (int j = 0; j < NP; ++j) pair(j, Flag<false>{}, false);   // the last pairs, or absent ones: nothing is left to load
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) red_acc[nt * MT + mt][lane] = acc[mt][nt];
    const float lsum = sum_across_groups(l_run[nt]);
    if (g == 0) {
      red_m[16 * nt + l16] = partial_reference(m_run[nt], lsum);
      red_l[16 * nt + l16] = lsum;
    }
  }
}

}  // namespace
