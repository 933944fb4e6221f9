// Rows of a matrix in 8-bit floating point (e4m3.h has the format): groups of 128 columns, their encoding from 16-bit and
// 32-bit values, and finished results of four columns.
//
// The scales of a matrix of r rows lie as [ceil(K / 512)][r][4]: a word per row holds four groups' bytes, one per stage
// of 128, and the words of consecutive rows lie side by side.
#pragma once

#include "e4m3.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2_t;

constexpr int GROUP = 128;        // K per scale

// Largest |x| of N words of two 16-bit values each, as bits (both types' magnitudes order as integers do).
template <int N>
FS_DEVICE uint32_t magnitude_bits(const uint32_t (&w)[N]) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
  return m[0] > m[1] ? m[0] : m[1];
}
template <int DT>
FS_DEVICE float half_of(uint32_t w, int hi) { return Elem<DT>::to_f32((uint16_t)(w >> (16 * hi))); }

// Magnitudes above this are not finite, or (bf16) more than the largest scale's 448.
template <int DT> constexpr uint32_t LARGEST = DT == FS_BF16 ? 0x7f60u : 0x7bffu;

// The exponent byte of a group whose largest magnitude has these bits (at most LARGEST).
template <int DT>
FS_DEVICE int exponent_of_bits(uint32_t m) {
  return scale_exponent<FS_F32>(Elem<DT>::to_f32((uint16_t)m));
}

// Two 16-bit values' codes under the scale 2^(e - 127) = s: one conversion, which divides by the scale and rounds to
// nearest even (each bf16 and f16 gives the definition's code).
template <int DT, bool HI>
FS_DEVICE s16x2_t encode_pair(s16x2_t old, uint32_t w, float s) {
  typedef short v2s __attribute__((ext_vector_type(2)));
  if constexpr (DT == FS_BF16) {
    typedef __bf16 v2b __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(s16x2_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(v2s, old),
                                                                                 __builtin_bit_cast(v2b, w), s, HI));
  } else {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(s16x2_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(v2s, old),
                                                                                __builtin_bit_cast(v2h, w), s, HI));
  }
}
// Four values' codes. FAR: some of the wave's are above LARGEST (saturated, or NaN where not finite).
template <int DT>
FS_DEVICE uint32_t encode_words(uint32_t a, uint32_t b, int e, bool far) {
  if (far) return encode4(half_of<DT>(a, 0), half_of<DT>(a, 1), half_of<DT>(b, 0), half_of<DT>(b, 1), scale_inverse(e));
  const float s = scale_value(e);
  s16x2_t c = {0, 0};
  c = encode_pair<DT, false>(c, a, s);
  c = encode_pair<DT, true>(c, b, s);
  return __builtin_bit_cast(uint32_t, c);
}
// Largest finite magnitude of N words.
template <int DT, int N>
FS_DEVICE float finite_max(const uint32_t (&w)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fmaxf(finite_magnitude(half_of<DT>(w[i], 0)), finite_magnitude(half_of<DT>(w[i], 1))));
  return m;
}

// The largest over a lane's LANES neighbours, 8 or 16, in each of them (within a row of lanes: no trip through LDS):
// lanes 1 and 2 apart, then mirrored within 8, then within 16.
template <int LANES>
FS_DEVICE uint32_t group_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xf, 0xf, false));
  return LANES == 8 ? m : max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xf, 0xf, false));
}
// (magnitudes order as their bits do)
template <int LANES>
FS_DEVICE float group_max(float m) { return __uint_as_float(group_max<LANES>(__float_as_uint(m))); }

// A group of 128 values, 2 NW in each of 64 / NW lanes: the exponent byte of its scale, and the lane's codes.
template <int DT, int NW>
FS_DEVICE void encode_group(const uint32_t (&w)[NW], int& e, uint32_t (&c)[NW / 2]) {
  constexpr int LANES = 64 / NW;
  const uint32_t m = group_max<LANES>(magnitude_bits(w));
  const bool far = __any(m > LARGEST<DT>);
  e = far ? scale_exponent<FS_F32>(group_max<LANES>(finite_max<DT>(w))) : exponent_of_bits<DT>(m);
#pragma unroll
  for (int i = 0; i < NW / 2; ++i) c[i] = encode_words<DT>(w[2 * i], w[2 * i + 1], e, far);
}

// A group of 128 values in 32 bits, eight in each of 16 lanes: the exponent byte of its scale, and the lane's codes. One
// conversion divides by the scale and rounds to nearest even; what is not finite, or more than the largest scale's 448, takes
// the way of encode4, for all of the wave.
FS_DEVICE u32x2_t encode_eight(const float (&v)[8], int& e) {
  typedef short v2s __attribute__((ext_vector_type(2)));
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = group_max<16>(m);
  if (__any(m > 0x7f600000u)) {   // 448 * 2^119
    float f = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f = fmaxf(f, finite_magnitude(v[i]));
    e = scale_exponent<FS_F32>(group_max<16>(f));
    const float inv = scale_inverse(e);
    return u32x2_t{encode4(v[0], v[1], v[2], v[3], inv), encode4(v[4], v[5], v[6], v[7], inv)};
  }
  e = scale_exponent<FS_F32>(__uint_as_float(m));
  const float s = scale_value(e);
  u32x2_t c;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v2s w = {0, 0};
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[4 * h], v[4 * h + 1], s, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[4 * h + 2], v[4 * h + 3], s, true);
    c[h] = __builtin_bit_cast(uint32_t, w);
  }
  return c;
}

// ------------------------------------------------------------------------------------------------
// results
// ------------------------------------------------------------------------------------------------
// Four finished columns col0 .. of a row C of `cols`, rounded once.
template <int DT>
FS_DEVICE void store_row4(float4_t a, uint16_t* C, int64_t col0, int64_t cols, bool vec) {
  if (vec && col0 + 4 <= cols) {
    *reinterpret_cast<u32x2_t*>(C + col0) =
        u32x2_t{(uint32_t)Elem<DT>::store_bits(a[0]) | ((uint32_t)Elem<DT>::store_bits(a[1]) << 16),
                (uint32_t)Elem<DT>::store_bits(a[2]) | ((uint32_t)Elem<DT>::store_bits(a[3]) << 16)};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col0 + e < cols) C[col0 + e] = Elem<DT>::store_bits(a[e]);
}
// Whether rows of C (and R) can be stored and read eight bytes at a time.
inline bool rows_by_8(const void* C, int64_t ldc, const void* R, int64_t ldr) {
  return ((reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(R)) & 7) == 0 && ldc % 4 == 0 && (!R || ldr % 4 == 0);
}

inline int64_t scale_bytes(int64_t rows, int64_t K) { return (K + 511) / 512 * rows * 4; }
// Whether a launch of so many waves, four a workgroup, stays below 2^32 threads.
inline bool waves_fit(int64_t waves) { return waves <= (1 << 26) - 4; }
inline int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }
inline bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

namespace fs {
// fs_quantize_e4m3 without its checks (gemm_e4m3.hip).
void quantize_rows_e4m3(const void* X, int64_t ldx, int64_t rows, int64_t K, int32_t dtype, uint8_t* codes, int64_t ldc,
                        uint32_t* scales, hipStream_t s);
}  // namespace fs
