// What the kernels that write a paged pool share: a token's place in the pool, and the loads of the fused
// projection's rows.
#pragma once

#include "common.h"

namespace {

FS_DEVICE bool slot_of(int pos, const int32_t* table, int64_t table_stride, int b, int max_blocks,
                       const fs_kv_layout& kv, int64_t& blk, int& slot) {
  if (pos < 0) return false;
  int bi = pos / kv.block_size;
  if (bi >= max_blocks) return false;
  blk = table[(int64_t)b * table_stride + bi];
  if (blk < 0 || blk >= kv.num_blocks) return false;
  slot = pos - bi * kv.block_size;
  return true;
}

typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4_t;

template <int DT>
FS_DEVICE void unpack8(const u32x4_t& w, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = Elem<DT>::to_f32((uint16_t)(w[j] & 0xffffu));
    v[2 * j + 1] = Elem<DT>::to_f32((uint16_t)(w[j] >> 16));
  }
}

template <int DT>
FS_DEVICE u32x4_t pack8(const float (&v)[8]) {
  u32x4_t w;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = (uint32_t)Elem<DT>::store_bits(v[2 * j]) | ((uint32_t)Elem<DT>::store_bits(v[2 * j + 1]) << 16);
  return w;
}

// Eight consecutive qkv elements as floats: the 16-bit row itself, or (PART) the split-K partials of
// the QKV projection [splits][rows][cols] added in increasing split order and rounded to DT, exactly the
// values the GEMM's own reduction would have stored.
struct QkvPart {
  const float* part;   // null: read the 16-bit qkv rows
  int32_t splits;
  int64_t stride;      // elements between consecutive splits (rows * cols)
};

// PART: 0 reads the 16-bit row; > 0 adds that many partials, all loaded before the first add; < 0
// adds pp.splits partials one at a time.
template <int DT, int PART>
FS_DEVICE void load8(const uint16_t* qkv, const QkvPart& pp, int64_t e, float (&v)[8]) {
  if (PART == 0) {
    unpack8<DT>(*reinterpret_cast<const u32x4_t*>(qkv + e), v);
    return;
  }
  float4_t a, b;
  if (PART > 0) {
    constexpr int NS = PART > 0 ? PART : 1;
    float4_t qa[NS], qb[NS];
#pragma unroll
    for (int sp = 0; sp < NS; ++sp) {
      qa[sp] = *reinterpret_cast<const float4_t*>(pp.part + sp * pp.stride + e);
      qb[sp] = *reinterpret_cast<const float4_t*>(pp.part + sp * pp.stride + e + 4);
    }
    a = qa[0];
    b = qb[0];
#pragma unroll
    for (int sp = 1; sp < NS; ++sp)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] += qa[sp][j];
        b[j] += qb[sp][j];
      }
  } else {
    a = *reinterpret_cast<const float4_t*>(pp.part + e);
    b = *reinterpret_cast<const float4_t*>(pp.part + e + 4);
    for (int sp = 1; sp < pp.splits; ++sp) {
      const float4_t a2 = *reinterpret_cast<const float4_t*>(pp.part + sp * pp.stride + e);
      const float4_t b2 = *reinterpret_cast<const float4_t*>(pp.part + sp * pp.stride + e + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        a[j] += a2[j];
        b[j] += b2[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[j] = Elem<DT>::round(a[j]);
    v[j + 4] = Elem<DT>::round(b[j]);
  }
}

}  // namespace
