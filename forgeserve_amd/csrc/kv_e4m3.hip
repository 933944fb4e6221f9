// The paged pool held as e4m3 codes (fs_kv_layout with FS_STORE_E4M3): the fused rotary + write, the plain write and
// the gather that reads it back.
//
// A token's keys and values of one KV head are a group with one scale each: code = rne(x / s), s the smallest power
// of two with max |x| <= 448 s. The rotation runs in f32 on unrounded cos and sin and is rounded once (queries to the
// row dtype, keys to their codes): out[i] = x1 c - x2 s, out[i + D/2] = x2 c + x1 s, two products and one sum each.
#include "e4m3.h"
#include "kv.h"

namespace {

// One wave per head of a token: lane i holds dims i, i + 64, ... (or pairs i and i + 64 of a rotation).
template <int DT>
FS_DEVICE void store_key(const fs_kv_layout& kv, int64_t blk, int h, int slot, const float (&a)[2], const float (&b)[2]) {
  const int lane = threadIdx.x & 63, half = kv.head_dim / 2;
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < half) m = fmaxf(m, fmaxf(finite_magnitude(a[c]), finite_magnitude(b[c])));
  const int e = scale_exponent<DT>(wave_max(m));
  const float inv = scale_inverse(e);
  uint8_t* t = key_tile(kv, blk, h);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int p = lane + 64 * c;
    if (p >= half) break;
    t[key_code(kv, slot, p)] = encode1(a[c], inv);
    t[key_code(kv, slot, p + half)] = encode1(b[c], inv);
  }
  if (lane == 0) tile_scales(kv, blk, h)[slot] = (uint8_t)e;
}

template <int DT>
FS_DEVICE void store_value(const fs_kv_layout& kv, int64_t blk, int h, int slot, const float (&x)[4]) {
  const int lane = threadIdx.x & 63, D = kv.head_dim;
  float m = 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < D) m = fmaxf(m, finite_magnitude(x[c]));
  const int e = scale_exponent<DT>(wave_max(m));
  const float inv = scale_inverse(e);
  uint8_t* t = value_tile(kv, blk, h);
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < D) t[value_code(kv, slot, lane + 64 * c)] = encode1(x[c], inv);
  if (lane == 0) tile_scales(kv, blk, h)[kv.block_size + slot] = (uint8_t)e;
}

// Any row dtype and alignment: a wave per head of a token, four to a workgroup.
template <int DT>
__global__ void __launch_bounds__(256) rope_write_e4m3_kernel(
    const typename Elem<DT>::T* __restrict__ qkv, int64_t qkv_stride, int32_t T, int32_t H,
    const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, const int32_t* __restrict__ token_row,
    int32_t n_rows, const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, int32_t rope_len,
    const int32_t* __restrict__ table, int64_t table_stride, int32_t max_blocks, fs_kv_layout kv,
    typename Elem<DT>::T* __restrict__ q_out, int64_t q_stride) {
  typedef Elem<DT> E;
  typedef typename E::T T_;
  const int64_t m = blockIdx.x;
  int b = token_row ? token_row[m] : (int)(m / T);
  const bool row_ok = token_row == nullptr || (b >= 0 && b < n_rows);
  b = row_ok ? b : 0;
  const int D = kv.head_dim, half = D / 2, Hkv = kv.n_kv_heads;
  const int pos = row_ok ? positions[m] : -1;
  const bool rot_ok = pos >= 0 && pos < rope_len;
  int64_t blk = 0;
  int slot = 0;
  const int wpos = slots ? slots[m] : pos;
  const bool write_ok = rot_ok && slot_of(wpos, table, table_stride, b, max_blocks, kv, blk, slot);
  const T_* row = qkv + m * qkv_stride;
  const int lane = threadIdx.x & 63;
  const int head = 4 * blockIdx.y + (threadIdx.x >> 6);   // (wave-uniform)
  if (head >= H + 2 * Hkv) return;
  const T_* x = row + (int64_t)head * D;
  if (head >= H + Hkv) {
    if (!write_ok) return;
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = lane + 64 * c < D ? E::load(x, lane + 64 * c) : 0.f;
    store_value<DT>(kv, blk, head - H - Hkv, slot, v);
    return;
  }
  float o1[2] = {0.f, 0.f}, o2[2] = {0.f, 0.f};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int p = lane + 64 * c;
    if (p >= half || !rot_ok) break;
    const float x1 = E::load(x, p), x2 = E::load(x, p + half);
    const float cs = rope_cos[(int64_t)pos * half + p], sn = rope_sin[(int64_t)pos * half + p];
    o1[c] = x1 * cs - x2 * sn;
    o2[c] = x2 * cs + x1 * sn;
  }
  if (head < H) {
    T_* qo = q_out + m * q_stride + (int64_t)head * D;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int p = lane + 64 * c;
      if (p >= half) break;
      E::store(qo, p, o1[c]);
      E::store(qo, p + half, o2[c]);
    }
  } else if (write_ok) {
    store_key<DT>(kv, blk, head - H, slot, o1, o2);
  }
}

// 16-bit rows that split into aligned 16-byte groups, D / 16 a power of two: a thread rotates 8 pairs of a head (dims
// p0 .. and p0 + D/2 ..) or takes 8 dims of a head's values, and the D/16 (values: D/8) neighbouring lanes of a head
// share its maximum. PART: the rows are the sums of the projection's split-K partials (load8).
//
// A key's codes go out 8 bytes at a time. A value's lie four keys to a word (16 bytes from dim to dim in the
// thread's order), so a single token's are byte stores; where four consecutive tokens of a call fill the four slots of
// such a group (prompts, long windows), the first one's threads write them all, as words, and the others' do nothing.
//
// Bound by HBM for prompts (7626 tokens, 32/8 heads of 128: 45 us for 176 MB, 3.9 TB/s; workgroups of 256 and 448 threads
// 49 and 52, 16 neighbouring tokens on one XCD 47), by the launch and three loads one after the other for a step (64
// tokens: 4.2 us).
template <int DT, int PART>
__global__ void __launch_bounds__(128) rope_write_e4m3_vec_kernel(
    const uint16_t* __restrict__ qkv, QkvPart pp, int64_t qkv_stride, int64_t n_tokens, int32_t T, int32_t H,
    const int32_t* __restrict__ positions, const int32_t* __restrict__ slots, const int32_t* __restrict__ token_row,
    int32_t n_rows, const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, int32_t rope_len,
    const int32_t* __restrict__ table, int64_t table_stride, int32_t max_blocks, fs_kv_layout kv,
    uint16_t* __restrict__ q_out, int64_t q_stride) {
  const int64_t m = blockIdx.x;
  const int D = kv.head_dim, half = D / 2, Hkv = kv.n_kv_heads;
  const int ng = half / 8;                                      // lanes per head of the rotation
  const int n_rot = (H + Hkv) * ng, v0 = n_rot + (n_rot & ng);   // the values' lanes start at a multiple of 2 ng
  const int gi = blockIdx.y * blockDim.x + threadIdx.x;
  const bool rot = gi < n_rot, val = gi >= v0 && gi < v0 + Hkv * 2 * ng;
  const int head = rot ? gi / ng : 0, p0 = rot ? 8 * (gi - head * ng) : 0;
  const int e0 = val ? 8 * (gi - v0) : 0;
  const int64_t row0 = m * qkv_stride;
  const int64_t val0 = (int64_t)(H + Hkv) * D + e0;
  float x1[8], x2[8];
  if (rot) {
    load8<DT, PART>(qkv, pp, row0 + (int64_t)head * D + p0, x1);
    load8<DT, PART>(qkv, pp, row0 + (int64_t)head * D + p0 + half, x2);
  } else if (val) {
    load8<DT, PART>(qkv, pp, row0 + val0, x1);
  }
  int b = token_row ? token_row[m] : (int)(m / T);
  const bool row_ok = token_row == nullptr || (b >= 0 && b < n_rows);
  b = row_ok ? b : 0;
  const int pos = row_ok ? positions[m] : -1;
  const bool rot_ok = pos >= 0 && pos < rope_len;
  const int64_t cs = rot_ok ? (int64_t)pos * half : 0;
  float4_t c4[2] = {}, s4[2] = {};
  if (rot) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c4[i] = *reinterpret_cast<const float4_t*>(rope_cos + cs + p0 + 4 * i);
      s4[i] = *reinterpret_cast<const float4_t*>(rope_sin + cs + p0 + 4 * i);
    }
  }
  int64_t blk = 0;
  int slot = 0;
  const int wpos = slots ? slots[m] : pos;
  const bool write_ok = rot_ok && slot_of(wpos, table, table_stride, b, max_blocks, kv, blk, slot);
  auto group_max = [](float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
  };
  if (rot) {
    float o1[8], o2[8], mx = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = c4[j >> 2][j & 3], sn = s4[j >> 2][j & 3];
      o1[j] = rot_ok ? x1[j] * c - x2[j] * sn : 0.f;
      o2[j] = rot_ok ? x2[j] * c + x1[j] * sn : 0.f;
    }
    if (head < H) {
      uint16_t* qo = q_out + m * q_stride + (int64_t)head * D + p0;
      *reinterpret_cast<u32x4_t*>(qo) = pack8<DT>(o1);
      *reinterpret_cast<u32x4_t*>(qo + half) = pack8<DT>(o2);
      return;
    }
    if (!write_ok) return;   // (the same for every lane of the token)
#pragma unroll
    for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fmaxf(finite_magnitude(o1[j]), finite_magnitude(o2[j])));
    const int e = scale_exponent<DT>(group_max(mx, ng)), h = head - H;
    const float inv = scale_inverse(e);
    uint8_t* t = key_tile(kv, blk, h);
    *reinterpret_cast<u32x2_t*>(t + key_code(kv, slot, p0)) =
        u32x2_t{encode4(o1[0], o1[1], o1[2], o1[3], inv), encode4(o1[4], o1[5], o1[6], o1[7], inv)};
    *reinterpret_cast<u32x2_t*>(t + key_code(kv, slot, p0 + half)) =
        u32x2_t{encode4(o2[0], o2[1], o2[2], o2[3], inv), encode4(o2[4], o2[5], o2[6], o2[7], inv)};
    if (p0 == 0) tile_scales(kv, blk, h)[slot] = (uint8_t)e;
    return;
  }
  if (!val || !write_ok) return;
  const int h = e0 / D, d0 = e0 - h * D;
  uint8_t* t = value_tile(kv, blk, h);
  uint8_t* sc = tile_scales(kv, blk, h) + kv.block_size;
  // whether tokens first .. first + 3 fill the slots of this token's 4-key group in order
  const int64_t first = m - (slot & 3);
  bool quad = (token_row || T >= 4) && first >= 0 && first + 3 < n_tokens;
  if (quad) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t mi = first + i;
      const int pi = positions[mi], wi = slots ? slots[mi] : pi, bi = token_row ? token_row[mi] : (int)(mi / T);
      quad &= bi == b && pi >= 0 && pi < rope_len && wi == wpos - (slot & 3) + i;
    }
  }
  float mx = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) mx = fmaxf(mx, finite_magnitude(x1[j]));
  if (!quad) {
    const int e = scale_exponent<DT>(group_max(mx, 2 * ng));
    const float inv = scale_inverse(e);
    const uint32_t w[2] = {encode4(x1[0], x1[1], x1[2], x1[3], inv), encode4(x1[4], x1[5], x1[6], x1[7], inv)};
#pragma unroll
    for (int j = 0; j < 8; ++j) t[value_code(kv, slot, d0 + j)] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    if (d0 == 0) sc[slot] = (uint8_t)e;
    return;
  }
  if (slot & 3) return;
  float x[4][8], y[4][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[0][j] = x1[j];
#pragma unroll
  for (int i = 1; i < 4; ++i) load8<DT, PART>(qkv, pp, row0 + i * qkv_stride + val0, x[i]);
  uint32_t es = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float mi = mx;
    if (i) {
      mi = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) mi = fmaxf(mi, finite_magnitude(x[i][j]));
    }
    const int e = scale_exponent<DT>(group_max(mi, 2 * ng));
    const float inv = scale_inverse(e);
    es |= (uint32_t)e << (8 * i);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[i][j] = to_code_range(x[i][j], inv);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0][j], y[1][j], 0, false);
    *reinterpret_cast<uint32_t*>(t + value_code(kv, slot, d0 + j)) =
        (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2][j], y[3][j], w, true);
  }
  if (d0 == 0) *reinterpret_cast<uint32_t*>(sc + slot) = es;
}

// A wave per head of k_new[b, :, t, :], then of v_new[b, :, t, :], four to a workgroup (four heads one after the other per
// wave took 16 tokens of 8 heads of 128 dims 8.9 us for 5.1).
template <int DT>
__global__ void __launch_bounds__(256) kv_write_e4m3_kernel(const typename Elem<DT>::T* __restrict__ k_new,
                                                            const typename Elem<DT>::T* __restrict__ v_new, int64_t s_b,
                                                            int64_t s_h, int64_t s_t, int32_t T,
                                                            const int32_t* __restrict__ positions,
                                                            const int32_t* __restrict__ table, int64_t table_stride,
                                                            int32_t max_blocks, fs_kv_layout kv) {
  typedef Elem<DT> E;
  const int bt = blockIdx.x;
  const int b = bt / T, t = bt - b * T;
  int64_t blk = 0;
  int slot = 0;
  if (!slot_of(positions[bt], table, table_stride, b, max_blocks, kv, blk, slot)) return;
  const int lane = threadIdx.x & 63, D = kv.head_dim, half = D / 2, Hkv = kv.n_kv_heads;
  const int i = 4 * blockIdx.y + (threadIdx.x >> 6);
  if (i >= 2 * Hkv) return;
  const int h = i < Hkv ? i : i - Hkv;
  const int64_t at = (int64_t)b * s_b + (int64_t)h * s_h + (int64_t)t * s_t;
  if (i < Hkv) {
    float x1[2], x2[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int p = lane + 64 * c;
      x1[c] = p < half ? E::load(k_new, at + p) : 0.f;
      x2[c] = p < half ? E::load(k_new, at + p + half) : 0.f;
    }
    store_key<DT>(kv, blk, h, slot, x1, x2);
  } else {
    float v[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = lane + 64 * c < D ? E::load(v_new, at + lane + 64 * c) : 0.f;
    store_value<DT>(kv, blk, h, slot, v);
  }
}

template <int DT>
FS_DEVICE void store8(typename Elem<DT>::T* p, const float (&v)[8]) {   // 16-byte aligned
  if constexpr (DT == FS_F32) {
    *reinterpret_cast<float4_t*>(p) = float4_t{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4_t*>(p + 4) = float4_t{v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<u32x4_t*>(p) = pack8<DT>(v);
  }
}

// Two waves per tile, one for its keys and one for its values: (row b, table entry j, head h) in the outputs' order of
// heads. Keys: 8 consecutive dims of a slot per lane; values: four keys of 8 consecutive dims per lane, so that both sides'
// stores are 8 consecutive elements and a row's lanes lie side by side. A block id outside the pool reads as zeros. Bound
// by HBM: 16 rows of 256 blocks, 8 heads of 128, 16-bit outputs: 404 MB in 77-86 us, 4.7-5.2 TB/s; small calls by one load
// after another (64 blocks: 5.7 us; with one wave a tile 7.7).
template <int DT>
__global__ void __launch_bounds__(256) gather_e4m3_kernel(fs_kv_layout kv, const int32_t* __restrict__ table,
                                                          int64_t table_stride, int32_t max_blocks,
                                                          typename Elem<DT>::T* __restrict__ k_out,
                                                          typename Elem<DT>::T* __restrict__ v_out, uint32_t tiles) {
  const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const uint32_t tile = unit >> 1;
  if (tile >= tiles) return;
  const int lane = threadIdx.x & 63, D = kv.head_dim, BS = kv.block_size, Hkv = kv.n_kv_heads;
  const uint32_t bj = tile / (uint32_t)Hkv, row = bj / (uint32_t)max_blocks;
  const int h = (int)(tile - bj * (uint32_t)Hkv);
  const int64_t b = row, j = bj - row * (uint32_t)max_blocks;
  const int64_t blk = table[b * table_stride + j];
  const bool ok = blk >= 0 && blk < kv.num_blocks;
  const int64_t out0 = ((b * Hkv + h) * max_blocks + j) * BS * (int64_t)D;
  const uint8_t* kt = key_tile(kv, ok ? blk : 0, h);
  const uint8_t* vt = value_tile(kv, ok ? blk : 0, h);
  const uint8_t* sc = tile_scales(kv, ok ? blk : 0, h);
  const int c8 = D / 8;
  for (int i0 = unit & 1 ? BS * c8 : lane; i0 < BS * c8; i0 += 256) {   // four at a time, their loads together
    u32x2_t w[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = min(i0 + 64 * u, BS * c8 - 1), slot = i / c8, d = 8 * (i - slot * c8);
      w[u] = *reinterpret_cast<const u32x2_t*>(kt + key_code(kv, slot, d));
      s[u] = ok ? scale_value(sc[slot]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 64 * u, slot = i / c8, d = 8 * (i - slot * c8);
      if (i >= BS * c8) break;
      float v[8];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float f[4];
        decode4(w[u][q], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = ok ? f[e] * s[u] : 0.f;
      }
      store8<DT>(k_out + out0 + (int64_t)slot * D + d, v);
    }
  }
  for (int i = unit & 1 ? lane : BS / 4 * c8; i < BS / 4 * c8; i += 64) {
    const int g = i / c8, d = 8 * (i - g * c8);
    float v[4][8];
    float s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = ok ? scale_value(sc[BS + 4 * g + e]) : 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float f[4];
      decode4(*reinterpret_cast<const uint32_t*>(vt + value_code(kv, 4 * g, d + c)), f);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e][c] = ok ? f[e] * s[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) store8<DT>(v_out + out0 + (int64_t)(4 * g + e) * D + d, v[e]);
  }
}

}  // namespace

namespace fs {

int qkv_rope_write_e4m3(const void* qkv, const float* part, int32_t splits, int64_t part_stride, int64_t qkv_stride,
                        int64_t n_tokens, int32_t T, int32_t n_heads, const int32_t* positions, const int32_t* slots,
                        const int32_t* token_row, int32_t n_rows, const float* rope_cos, const float* rope_sin,
                        int32_t rope_len, const int32_t* tables, int64_t table_stride, int32_t max_blocks,
                        const fs_kv_layout& kv, void* q_out, int64_t q_stride, hipStream_t s) {
  auto al16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int ng = kv.head_dim / 16;
  const bool vec = row_dtype(kv) != FS_F32 && (ng & (ng - 1)) == 0 && qkv_stride % 8 == 0 && q_stride % 8 == 0 &&
                   al16(part ? (const void*)part : qkv) && al16(q_out) && al16(rope_cos) && al16(rope_sin) &&
                   (kv.head_dim / 2) % 8 == 0;
  FS_CHECK_ARG(part == nullptr || (vec && splits >= 1 && part_stride >= n_tokens * qkv_stride),
               "qkv_rope_write_partials: needs 16-bit data, head_dim / 16 a power of two, 16-byte aligned rows");
  if (vec) {
    const int lanes = (n_heads + kv.n_kv_heads + 1) / 2 * 2 * ng + kv.n_kv_heads * 2 * ng;
    const dim3 vgrid((unsigned)n_tokens, (unsigned)((lanes + 127) / 128));
    const QkvPart pp{part, splits, part_stride};
#define FS_VEC(DT, P)                                                                                              \
  rope_write_e4m3_vec_kernel<DT, P><<<vgrid, 128, 0, s>>>((const uint16_t*)qkv, pp, qkv_stride, n_tokens, T, n_heads, \
                                                          positions, slots, token_row, n_rows, rope_cos, rope_sin,     \
                                                          rope_len, tables, table_stride, max_blocks, kv,              \
                                                          (uint16_t*)q_out, q_stride)
#define FS_VEC_DT(DT)                    \
  switch (part ? splits : 0) {           \
    case 0: FS_VEC(DT, 0); break;        \
    case 2: FS_VEC(DT, 2); break;        \
    case 4: FS_VEC(DT, 4); break;        \
    case 8: FS_VEC(DT, 8); break;        \
    default: FS_VEC(DT, -1); break;      \
  }
    if (row_dtype(kv) == FS_BF16) FS_VEC_DT(FS_BF16)
    else FS_VEC_DT(FS_F16)
#undef FS_VEC_DT
#undef FS_VEC
    return launch_status("qkv_rope_write");
  }
  const dim3 grid((unsigned)n_tokens, (unsigned)((n_heads + 2 * kv.n_kv_heads + 3) / 4));
#define FS_LAUNCH(DT)                                                                                                 \
  rope_write_e4m3_kernel<DT><<<grid, 256, 0, s>>>((const typename Elem<DT>::T*)qkv, qkv_stride, T, n_heads, positions, \
                                                  slots, token_row, n_rows, rope_cos, rope_sin, rope_len, tables,      \
                                                  table_stride, max_blocks, kv, (typename Elem<DT>::T*)q_out, q_stride)
  switch (row_dtype(kv)) {
    case FS_F32: FS_LAUNCH(FS_F32); break;
    case FS_BF16: FS_LAUNCH(FS_BF16); break;
    default: FS_LAUNCH(FS_F16); break;
  }
#undef FS_LAUNCH
  return launch_status("qkv_rope_write");
}

int paged_kv_write_e4m3(const void* k_new, const void* v_new, int64_t s_b, int64_t s_h, int64_t s_t, int32_t B, int32_t T,
                        const int32_t* positions, const int32_t* tables, int64_t table_stride, int32_t max_blocks,
                        const fs_kv_layout& kv, hipStream_t s) {
  const dim3 grid((unsigned)(B * T), (unsigned)((2 * kv.n_kv_heads + 3) / 4));
#define FS_LAUNCH(DT)                                                                                             \
  kv_write_e4m3_kernel<DT><<<grid, 256, 0, s>>>((const typename Elem<DT>::T*)k_new, (const typename Elem<DT>::T*)v_new, \
                                                s_b, s_h, s_t, T, positions, tables, table_stride, max_blocks, kv)
  switch (row_dtype(kv)) {
    case FS_F32: FS_LAUNCH(FS_F32); break;
    case FS_BF16: FS_LAUNCH(FS_BF16); break;
    default: FS_LAUNCH(FS_F16); break;
  }
#undef FS_LAUNCH
  return launch_status("paged_kv_write");
}

int paged_gather_e4m3(const fs_kv_layout& kv, const int32_t* tables, int64_t table_stride, int32_t B, int32_t max_blocks,
                      void* k_out, void* v_out, hipStream_t s) {
  FS_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) == 0,
               "paged_gather: outputs of an 8-bit pool must be 16-byte aligned");
  const int64_t tiles = (int64_t)B * max_blocks * kv.n_kv_heads;
  FS_CHECK_ARG(tiles < 0x3fffffff, "paged_gather: %lld tiles", (long long)tiles);
  const dim3 grid((unsigned)((tiles + 1) / 2));
#define FS_LAUNCH(DT)                                                                                       \
  gather_e4m3_kernel<DT><<<grid, 256, 0, s>>>(kv, tables, table_stride, max_blocks, (typename Elem<DT>::T*)k_out, \
                                              (typename Elem<DT>::T*)v_out, (uint32_t)tiles)
  switch (row_dtype(kv)) {
    case FS_F32: FS_LAUNCH(FS_F32); break;
    case FS_BF16: FS_LAUNCH(FS_BF16); break;
    default: FS_LAUNCH(FS_F16); break;
  }
#undef FS_LAUNCH
  return launch_status("paged_gather");
}

}  // namespace fs
