// 8-bit floating point (e4m3: 4 exponent and 3 mantissa bits, OCP, largest value 448) with a power of two as the
// scale of a group of values, kept as its biased exponent byte e: a code c stands for value(c) * 2^(e - 127).
//
// A power of two moves no mantissa bit: both the encoding x * 2^(127 - e) and the decoding are exact but for one rounding,
// which is within half a step: 2^-4 of the value where the code is normal, from 2^-6 of the scale s on, and 2^-10 s below
// that. The group's largest is above 224 s (unless s is the smallest there is), so these are at most 2^-13.8 and 2^-17.8
// of it; another scale would put it at 448 s and gain a factor of two there. It is also what the hardware takes: the
// conversions to bf16 and f16 and the matrix instructions apply such a scale by themselves.
#pragma once

#include "common.h"

namespace {

typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2_t;

// The exponents a group's scale may have. f32 and bf16: every value a code stands for is normal and finite in
// bf16. f16: every one is an f16 (down to its smallest step, 2^-24, which is all the precision that smaller inputs had).
template <int DT> struct ScaleRange { static constexpr int LO = 10, HI = 246; };
template <> struct ScaleRange<FS_F16> { static constexpr int LO = 112, HI = 134; };

FS_DEVICE bool is_finite(float x) { return fabsf(x) < INFINITY; }   // (false for NaN)
FS_DEVICE float finite_magnitude(float x) { return is_finite(x) ? fabsf(x) : 0.f; }

// The exponent byte of the smallest power of two s with amax / s <= 448 = 1.75 * 2^8, between LO and HI.
template <int DT>
FS_DEVICE int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, ScaleRange<DT>::LO), ScaleRange<DT>::HI);
}
FS_DEVICE float scale_value(int e) { return __uint_as_float((uint32_t)e << 23); }
FS_DEVICE float scale_inverse(int e) { return __uint_as_float((uint32_t)(254 - e) << 23); }

// The value to encode under 1 / scale: at most 448 (only the largest scale leaves more), NaN for what is not finite.
FS_DEVICE float to_code_range(float x, float inv) {
  return is_finite(x) ? __builtin_amdgcn_fmed3f(x * inv, -448.f, 448.f) : __uint_as_float(0x7fc00000u);
}
// Four values' codes (round to nearest even), the first in the low byte.
FS_DEVICE uint32_t encode4(float a, float b, float c, float d, float inv) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(to_code_range(a, inv), to_code_range(b, inv), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(to_code_range(c, inv), to_code_range(d, inv), w, true);
}
FS_DEVICE uint8_t encode1(float a, float inv) {
  return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(to_code_range(a, inv), 0.f, 0, false);
}
// The four codes of a word as floats, unscaled.
FS_DEVICE void decode4(uint32_t w, float (&v)[4]) {
  const f32x2_t a = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false));
  const f32x2_t b = __builtin_bit_cast(f32x2_t, __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true));
  v[0] = a[0];
  v[1] = a[1];
  v[2] = b[0];
  v[3] = b[1];
}

// ------------------------------------------------------------------------------------------------
// the pool of codes (fs_kv_layout with FS_STORE_E4M3)
// ------------------------------------------------------------------------------------------------
__host__ __device__ inline bool stores_e4m3(const fs_kv_layout& kv) { return (kv.dtype & FS_STORE_E4M3) != 0; }
__host__ __device__ inline int32_t row_dtype(const fs_kv_layout& kv) { return kv.dtype & ~FS_STORE_E4M3; }

FS_DEVICE int64_t key_code(const fs_kv_layout& kv, int slot, int d) {   // inside a tile of keys
  return (int64_t)(d >> 4) * 16 * kv.block_size + slot * 16 + (d & 15);
}
// Place of dim d among a 4-key group's dims: each 64 dims (or what is left of them) by d % 16 first, so that the
// 16 bytes at a place are four keys of dims d, d + 16, d + 32 and d + 48: what a lane of a matrix instruction wants.
FS_DEVICE int value_place(int head_dim, int d) {
  const int left = (head_dim >> 4) - ((d >> 6) << 2), n = left < 4 ? left : 4;
  return (d & ~63) + (d & 15) * n + ((d >> 4) & 3);
}
FS_DEVICE int64_t value_code(const fs_kv_layout& kv, int slot, int d) {   // inside a tile of values
  return (int64_t)(slot >> 2) * 4 * kv.head_dim + value_place(kv.head_dim, d) * 4 + (slot & 3);
}
FS_DEVICE uint8_t* key_tile(const fs_kv_layout& kv, int64_t blk, int h) {
  return reinterpret_cast<uint8_t*>(kv.k) + blk * kv.k_block + h * kv.k_head;
}
FS_DEVICE uint8_t* value_tile(const fs_kv_layout& kv, int64_t blk, int h) {
  return reinterpret_cast<uint8_t*>(kv.v) + blk * kv.v_block + h * kv.v_head;
}
FS_DEVICE uint8_t* tile_scales(const fs_kv_layout& kv, int64_t blk, int h) {   // keys', then values'
  return reinterpret_cast<uint8_t*>(kv.k) + kv.k_group + blk * kv.k_slot + h * kv.k_dim;
}

// What every entry point asks of such a layout.
inline int check_e4m3_layout(const fs_kv_layout& kv, const char* what) {
  const int32_t dt = row_dtype(kv);
  FS_CHECK_ARG(dt == FS_F32 || dt == FS_BF16 || dt == FS_F16, "%s: 8-bit pool: bad dtype %d", what, kv.dtype);
  FS_CHECK_ARG(kv.head_dim > 0 && kv.head_dim % 16 == 0 && kv.head_dim <= 256 && kv.block_size > 0 &&
                   kv.block_size % 4 == 0 && kv.n_kv_heads > 0 && kv.num_blocks > 0,
               "%s: 8-bit pool: head_dim %d (a multiple of 16, at most 256), block_size %d (a multiple of 4), %d heads, "
               "%lld blocks",
               what, kv.head_dim, kv.block_size, kv.n_kv_heads, (long long)kv.num_blocks);
  const uintptr_t k = reinterpret_cast<uintptr_t>(kv.k), v = reinterpret_cast<uintptr_t>(kv.v);
  FS_CHECK_ARG(((k | v | (uintptr_t)kv.k_block | (uintptr_t)kv.k_head | (uintptr_t)kv.v_block | (uintptr_t)kv.v_head) & 15) == 0,
               "%s: 8-bit pool: tiles not 16-byte aligned", what);
  FS_CHECK_ARG(kv.k_group != 0 && kv.v_slot == 0 && kv.v_dim == 0 &&
                   (((uintptr_t)kv.k_group | (uintptr_t)kv.k_slot | (uintptr_t)kv.k_dim) & 3) == 0,
               "%s: 8-bit pool: scales missing or not 4-byte aligned", what);
  return 0;
}

}  // namespace

namespace fs {
// kv.hip's calls on a pool of codes (kv_e4m3.hip); the arguments they share have been checked. qkv null: `part` holds
// `splits` partials of the projection, `part_stride` elements apart.
int qkv_rope_write_e4m3(const void* qkv, const float* part, int32_t splits, int64_t part_stride, int64_t qkv_stride,
                        int64_t n_tokens, int32_t T, int32_t n_heads, const int32_t* positions, const int32_t* slots,
                        const int32_t* token_row, int32_t n_rows, const float* rope_cos, const float* rope_sin,
                        int32_t rope_len, const int32_t* tables, int64_t table_stride, int32_t max_blocks,
                        const fs_kv_layout& kv, void* q_out, int64_t q_stride, hipStream_t s);
int paged_kv_write_e4m3(const void* k_new, const void* v_new, int64_t s_b, int64_t s_h, int64_t s_t, int32_t B, int32_t T,
                        const int32_t* positions, const int32_t* tables, int64_t table_stride, int32_t max_blocks,
                        const fs_kv_layout& kv, hipStream_t s);
int paged_gather_e4m3(const fs_kv_layout& kv, const int32_t* tables, int64_t table_stride, int32_t B, int32_t max_blocks,
                      void* k_out, void* v_out, hipStream_t s);
}  // namespace fs
