// Projections in 8-bit floating point: C[M,N] = X[M,K] . W[N,K]^T (+ R), W held as e4m3 codes with a power of two per row
// and 128 of K as their scale, X (bf16 or f16) brought to the same form within the call (e4m3.h has the format).
//
//   C[m][n] = round(sum over groups g of 2^(ex[m][g] + ew[n][g] - 254) * sum over k in g of cx[m][k] cw[n][k] (+ R[m][n]))
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 128 of K at a time and applies both scales itself, so a group is one
// instruction's depth, the chain of a sum over K stays in one f32 accumulator, and the only roundings are the codes', the
// sum's and the result's (product and residual together, once). The sum's: the matrix core adds eight neighbours' products
// at a time, aligned to the largest, and drops what lies more than 13 binary places below that one's power of two (found
// with pairs that cancel); from there on it keeps f32's places. So an element is off by less than 7 * 2^-13 of each
// eight's largest product, and a random result by 2.5e-5 of its norm (measured), a tenth of f16's rounding, which is why
// 32-bit results are not offered.
//
// The scales of a matrix of r rows lie as [ceil(K / 512)][r][4]: a word per row holds four groups' bytes, one per stage
// of 128, and the words of consecutive rows lie side by side.
//
// The kernel depends on M (the sums' order over K with it, so a row's last bit may differ between a short and a long
// batch): up to 16 rows one launch does everything; beyond that X is encoded first, then multiplied in LDS-fed tiles.
#include "e4m3.h"

namespace {

typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t u32x4;
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((__vector_size__(2 * sizeof(short)))) short s16x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(_Float16)))) _Float16 f16x2_t;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2_t;

constexpr int GROUP = 128;        // K per scale
constexpr int SHORT_ROWS = 16;    // rows that one launch takes
constexpr int SHORT_BYTES = 64 * 1024;   // and their codes
template <int I> struct Int { static constexpr int value = I; };

// D = A . B^T of 16 x 128 codes each: a lane holds 32 of its row's (two 16-byte chunks: any two, the same for A and B).
// BYTE: which of the four groups in the scale words.
template <int BYTE>
FS_DEVICE float4_t mfma_codes(i32x8 a, i32x8 b, float4_t c, uint32_t sa, uint32_t sb) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, __builtin_bit_cast(f32x4, c), 0, 0,
                                                                                       BYTE, (int)sa, BYTE, (int)sb));
}
// The same of 32 x 64 codes each: a lane holds 32 of row lane % 32.
template <int BYTE>
FS_DEVICE f32x16 mfma_codes32(i32x8 a, i32x8 b, f32x16 c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, BYTE, (int)sa, BYTE, (int)sb);
}
FS_DEVICE i32x8 both_chunks(u32x4 a, u32x4 b) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// A stage's rows in LDS are 128 bytes, eight 16-byte chunks, chunk c at place c ^ swap_of(row): an operand read's 16
// lanes take one chunk of 16 consecutive rows, which must differ in their place within 256 bytes, two rows' worth.
// (Swapped by row & 7, as 128-byte banks would have it, half of the LDS port's time went to conflicts.)
FS_DEVICE int swap_of(int row) { return (row >> 1) & 7; }

// ------------------------------------------------------------------------------------------------
// encoding rows of 16-bit values
// ------------------------------------------------------------------------------------------------
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

// A wave per 512 columns of a row: 16 lanes of 8 values share a group. VEC: rows of aligned 16-byte pieces.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) quantize_e4m3_kernel(const typename Elem<DT>::T* __restrict__ X, int64_t ldx,
                                                            int64_t rows, int64_t K, uint8_t* __restrict__ codes,
                                                            int64_t ldc, uint32_t* __restrict__ scales, int64_t kw) {
  typedef Elem<DT> E;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= rows * kw) return;
  const int lane = threadIdx.x & 63;
  const int64_t row = unit / kw, k4 = unit - row * kw, k = k4 * 512 + lane * 8;
  const bool in = k < K;   // (whole groups: K % 128 == 0)
  float v[8];
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  int e;
  u32x2_t out;
  if constexpr (DT == FS_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = in ? E::load(X, row * ldx + k + j) : 0.f;
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_magnitude(v[j]));
    e = scale_exponent<FS_F32>(group_max<16>(m));
    const float inv = scale_inverse(e);
    out = u32x2_t{encode4(v[0], v[1], v[2], v[3], inv), encode4(v[4], v[5], v[6], v[7], inv)};
  } else {
    if (in) {
      if (VEC) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(X + row * ldx + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = x[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = (uint32_t)X[row * ldx + k + 2 * j] | ((uint32_t)X[row * ldx + k + 2 * j + 1] << 16);
      }
    }
    uint32_t c[2];
    encode_group<DT>(w, e, c);
    out = u32x2_t{c[0], c[1]};
  }
  if (in) *reinterpret_cast<u32x2_t*>(codes + row * ldc + k) = out;
  // the row's word: lane 16 g holds byte g (zeros past K)
  uint32_t word = (lane & 15) == 0 && in ? (uint32_t)e << (8 * (lane >> 4)) : 0u;
  word |= (uint32_t)__shfl_xor((int)word, 16, 64);
  word |= (uint32_t)__shfl_xor((int)word, 32, 64);
  if (lane == 0) scales[k4 * rows + row] = word;
}

// ------------------------------------------------------------------------------------------------
// results
// ------------------------------------------------------------------------------------------------
// Four finished columns C[row][col0 ..]: the residual added in f32, rounded once.
template <int DT>
FS_DEVICE void store_row4(float4_t a, int64_t row, int64_t col0, uint16_t* C, int64_t ldc, const uint16_t* R, int64_t ldr,
                          int64_t N, bool vec) {
  if (vec && col0 + 4 <= N) {
    if (R) {
      const u32x2_t r = *reinterpret_cast<const u32x2_t*>(R + row * ldr + col0);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += half_of<DT>(r[e >> 1], e & 1);
    }
    *reinterpret_cast<u32x2_t*>(C + row * ldc + col0) =
        u32x2_t{(uint32_t)Elem<DT>::store_bits(a[0]) | ((uint32_t)Elem<DT>::store_bits(a[1]) << 16),
                (uint32_t)Elem<DT>::store_bits(a[2]) | ((uint32_t)Elem<DT>::store_bits(a[3]) << 16)};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col0 + e < N) C[row * ldc + col0 + e] = Elem<DT>::store_bits(R ? a[e] + Elem<DT>::to_f32(R[row * ldr + col0 + e]) : a[e]);
}
// Whether rows of C (and R) can be stored and read eight bytes at a time.
inline bool rows_by_8(const void* C, int64_t ldc, const void* R, int64_t ldr) {
  return ((reinterpret_cast<uintptr_t>(C) | reinterpret_cast<uintptr_t>(R)) & 7) == 0 && ldc % 4 == 0 && (!R || ldr % 4 == 0);
}

// ------------------------------------------------------------------------------------------------
// up to 16 rows: one launch, bound by the weights' bytes
// ------------------------------------------------------------------------------------------------
// A workgroup takes 16 TN columns of C; its eight waves split K and are joined in order through LDS. Weights go straight
// from HBM to registers in the instruction's own shape (a lane's two 16-byte chunks of a row's 128; a wave's load covers
// whole lines), DEPTH stages ahead. While the first of them are on their way the workgroup encodes the rows into LDS,
// eight lanes to a group: M K bytes of codes (XB at most, which bounds the rows) and a byte per
// row and group.
template <int DT, int TN, int DEPTH, int XB>
__global__ void __launch_bounds__(512) gemm_e4m3_short_kernel(const uint16_t* __restrict__ X, int64_t ldx,
                                                              const uint8_t* __restrict__ W, int64_t ldw,
                                                              const uint8_t* __restrict__ wsc, uint16_t* __restrict__ C,
                                                              int64_t ldc, const uint16_t* __restrict__ R, int64_t ldr,
                                                              int M, int64_t N, int nk, bool vec) {
  static_assert(XB >= 8 * TN * 1024, "the sums take the codes' place");
  __shared__ __attribute__((aligned(1024))) char xcodes[XB];   // [stage][row][128], chunk c of a row at c ^ swap_of(row)
  __shared__ uint8_t xexp[XB / GROUP];                          // [stage][row]
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t n0 = (int64_t)blockIdx.x * (16 * TN);
  const int k0 = (int)((int64_t)w * nk / 8), k1 = (int)((int64_t)(w + 1) * nk / 8);

  // The rows in pieces of 16 values (a chunk of codes), thread t's being t, t + 512, ...: one batch of them ahead of the
  // weights' loads, and always one on its way while another is encoded.
  constexpr int BATCH = 2;
  const int per_row = 8 * nk, pieces = M * per_row, row_step = 512 / per_row, piece_step = 512 - row_step * per_row;
  int lrow = tid / per_row, lpiece = tid - lrow * per_row;   // the next piece to load
  auto load_pieces = [&](u32x4 (&xp)[BATCH][2]) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const u32x4* p = reinterpret_cast<const u32x4*>(X + min(lrow, M - 1) * ldx + 16 * lpiece);
      xp[i][0] = p[0];
      xp[i][1] = p[1];
      lrow += row_step;
      lpiece += piece_step;
      if (lpiece >= per_row) lpiece -= per_row, ++lrow;
    }
  };
  u32x4 xa[BATCH][2], xb[BATCH][2];
  load_pieces(xa);

  struct Stage {
    u32x4 c[TN][2];
    uint32_t s[TN];
  } ring[DEPTH];
  const uint8_t* wrow[TN];
  int64_t srow[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    const int64_t n = min(n0 + 16 * j + l16, N - 1);
    wrow[j] = W + n * ldw + 16 * g;
    srow[j] = 4 * n;
  }
  auto load = [&](int k, Stage& x) {
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      x.c[j][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wrow[j] + (int64_t)k * GROUP));
      x.c[j][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wrow[j] + (int64_t)k * GROUP + 64));
      x.s[j] = wsc[(int64_t)(k >> 2) * 4 * N + srow[j] + (k & 3)];
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (k0 + d < k1) load(k0 + d, ring[d]);

  int row = tid / per_row, piece = tid - row * per_row;   // the next piece to encode
  auto encode_pieces = [&](const u32x4 (&xp)[BATCH][2], int first) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (first + i * 512 + 64 * w >= pieces) return;   // (wave-uniform; a group's 8 lanes are in or out together)
      uint32_t x[8], c[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = xp[i][j >> 2][j & 3];
      int e;
      encode_group<DT>(x, e, c);
      if (row < M) {
        const int at = (piece >> 3) * M + row;
        *reinterpret_cast<u32x4*>(xcodes + at * GROUP + 16 * ((piece & 7) ^ swap_of(row))) = u32x4{c[0], c[1], c[2], c[3]};
        if ((piece & 7) == 0) xexp[at] = (uint8_t)e;
      }
      row += row_step;
      piece += piece_step;
      if (piece >= per_row) piece -= per_row, ++row;
    }
  };
  for (int first = 0; first < pieces; first += 2 * BATCH * 512) {
    if (first + BATCH * 512 < pieces) load_pieces(xb);
    encode_pieces(xa, first);
    if (first + BATCH * 512 >= pieces) break;
    if (first + 2 * BATCH * 512 < pieces) load_pieces(xa);
    encode_pieces(xb, first + BATCH * 512);
  }
  __syncthreads();

  const int xrow = l16 < M ? l16 : 0;   // (lanes past the last row: results nobody stores)
  const int c0 = 16 * (g ^ swap_of(xrow)), c1 = 16 * ((4 + g) ^ swap_of(xrow));
  float4_t acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = float4_t{0.f, 0.f, 0.f, 0.f};
  for (int kt = k0; kt < k1; kt += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (kt + d >= k1) break;   // (wave-uniform)
      const char* row = xcodes + ((kt + d) * M + xrow) * GROUP;
      const i32x8 xf = both_chunks(*reinterpret_cast<const u32x4*>(row + c0), *reinterpret_cast<const u32x4*>(row + c1));
      const uint32_t xe = xexp[(kt + d) * M + xrow];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[j] = mfma_codes<0>(both_chunks(ring[d].c[j][0], ring[d].c[j][1]), xf, acc[j], ring[d].s[j], xe);
      if (kt + d + DEPTH < k1) load(kt + d + DEPTH, ring[d]);
    }
  }
  __syncthreads();   // every wave has read its codes
  float4_t(*red)[TN][64] = reinterpret_cast<float4_t(*)[TN][64]>(xcodes);
#pragma unroll
  for (int j = 0; j < TN; ++j) red[w][j][lane] = acc[j];
  __syncthreads();
  if (w >= TN) return;
  // wave j joins its columns' eight sums in order: lane (l16, g) has row l16, columns 16 j + 4 g ..
  float4_t a = red[0][w][lane];
#pragma unroll
  for (int v = 1; v < 8; ++v) {
    const float4_t b = red[v][w][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] += b[r];
  }
  if (l16 < M) store_row4<DT>(a, l16, n0 + 16 * w + 4 * g, C, ldc, R, ldr, N, vec);
}

// ------------------------------------------------------------------------------------------------
// LDS-fed tiles
// ------------------------------------------------------------------------------------------------
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Copies straight into LDS, 16 or 4 bytes a lane at a wave-uniform base plus the lane's offset; lane l lands at
// lds + 16 l (4 l). Counted by vmcnt; the waits are explicit.
FS_DEVICE void dma16_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
FS_DEVICE void dma4_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
FS_DEVICE void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Which tile a workgroup takes: workgroup ids go round the 8 XCDs; each gets a contiguous range of tiles, rows fastest
// inside groups of at most 8 row tiles, so that the tiles it runs at once share their panels through its L2.
FS_DEVICE bool tile_of(int tiles_m, int ntiles, int bm, int bn, int64_t& m0, int64_t& n0) {
  const int per_xcd = (ntiles + 7) / 8;
  const int tile = (blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (tile >= ntiles) return false;
  const int tiles_n = ntiles / tiles_m;
  const int grp = tile / (8 * tiles_n), first = 8 * grp, gm = min(tiles_m - first, 8);
  const int in_grp = tile - grp * 8 * tiles_n;
  m0 = (int64_t)(first + in_grp % gm) * bm;
  n0 = (int64_t)(in_grp / gm) * bn;
  return true;
}

struct Operands {
  const uint8_t *x, *w;          // codes
  const uint8_t *xs, *ws;        // scale words
  int64_t ldx, ldw;              // bytes from row to row
  int64_t M, N;
  int nk;                        // stages of 128
  int tiles_m, ntiles;
};

// BM x BN tiles, WGM x WGN waves, NS stages of 128 in LDS, NS - 1 of them on their way. The words of the rows'
// scales come with every fourth stage (one copy per 64 rows), into one of two places.
template <int DT, int BM, int BN, int WGM, int WGN, int NS>
__global__ void __launch_bounds__(64 * WGM * WGN) gemm_e4m3_tile_kernel(Operands P, uint16_t* __restrict__ C, int64_t ldc,
                                                                        const uint16_t* __restrict__ R, int64_t ldr,
                                                                        bool vec, float* __restrict__ part) {
  constexpr int NW = WGM * WGN, XB = BM * GROUP, STAGE = (BM + BN) * GROUP;
  constexpr int TM = BM / WGM / 16, TN = BN / WGN / 16;
  constexpr int CPW = STAGE / 1024 / NW;               // copies of codes per wave and stage
  constexpr int SW = (BM + BN) / 64;                   // copies of scale words per four stages
  static_assert(STAGE / 1024 % NW == 0 && SW <= NW && BM % 64 == 0, "whole copies, evenly");
  static_assert(NS >= 2 && NS <= 4, "wait_stages covers two stages behind the awaited one; scale words have two places");
  __shared__ __attribute__((aligned(1024))) char smem[NS * STAGE];
  __shared__ __attribute__((aligned(256))) uint32_t words[2][BM + BN];
  int64_t m0, n0;
  if (!tile_of(P.tiles_m, P.ntiles, BM, BN, m0, n0)) return;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem, words0 = (uint32_t)(uintptr_t)words;
  const int split = blockIdx.y, nk = P.nk / (int)gridDim.y, first = split * nk;   // (nk % 4 == 0 where K is split)
  // copy q of a stage: rows 8 q .. of the X block, then of the W block; lane l takes row l >> 3, physical chunk l & 7
  const int cr = lane >> 3;
  const char* base[CPW];
  uint32_t off[CPW];
#pragma unroll
  for (int i = 0; i < CPW; ++i) {
    const int q = i * NW + wave, row = 8 * q + cr, c = (lane & 7) ^ swap_of(row);
    const bool in_x = 8 * q < BM;
    const int64_t lead = in_x ? m0 : n0, last = (in_x ? P.M : P.N) - 1, ld = in_x ? P.ldx : P.ldw;
    const int64_t r = min(lead + (in_x ? row : row - BM), last) - lead;
    base[i] = reinterpret_cast<const char*>((in_x ? P.x : P.w) + lead * ld);
    off[i] = (uint32_t)(r * ld + 16 * c);
  }
  const char* sbase = nullptr;
  uint32_t soff = 0;
  if (wave < SW) {
    const bool in_x = 64 * wave < BM;
    const int64_t lead = in_x ? m0 : n0, rows = in_x ? P.M : P.N;
    const int64_t r = min(lead + (in_x ? 64 * wave : 64 * wave - BM) + lane, rows - 1);
    sbase = reinterpret_cast<const char*>(in_x ? P.xs : P.ws);
    soff = (uint32_t)(4 * r);
  }
  auto issue = [&](int kt) {   // kt: the split's stage
    const int k = first + kt;
    if ((k & 3) == 0 || kt == 0) {
      if (wave < SW)
        dma4_at(sbase + (int64_t)(k >> 2) * 4 * (64 * wave < BM ? P.M : P.N), soff,
                words0 + (uint32_t)(4 * ((k >> 2 & 1) * (BM + BN) + 64 * wave)));
    }
    const uint32_t to = lds0 + (uint32_t)((kt % NS) * STAGE);
#pragma unroll
    for (int i = 0; i < CPW; ++i) dma16_at(base[i] + (int64_t)k * GROUP, off[i], to + (uint32_t)((i * NW + wave) * 1024));
  };
  auto wait_stages = [&](int later) {   // (a copy of scale words among the later ones only makes the wait longer)
    if (later >= 2) wait_vm<2 * CPW>();
    else if (later == 1) wait_vm<CPW>();
    else wait_vm<0>();
  };
  float4_t acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
  uint32_t xs[TM], ws[TN];
#pragma unroll
  for (int s = 0; s < NS - 1; ++s)
    if (s < nk) issue(s);
  for (int kt = 0; kt < nk; ++kt) {
    wait_stages(min(NS - 2, nk - 1 - kt));
    __syncthreads();   // stage kt has landed for every wave; stage kt-1 is no longer being read
    if (kt + NS - 1 < nk) issue(kt + NS - 1);
    const int k = first + kt;
    if ((k & 3) == 0 || kt == 0) {
      const uint32_t* p = words[k >> 2 & 1];
#pragma unroll
      for (int i = 0; i < TM; ++i) xs[i] = p[wm * (BM / WGM) + 16 * i + l16];
#pragma unroll
      for (int j = 0; j < TN; ++j) ws[j] = p[BM + wn * (BN / WGN) + 16 * j + l16];
    }
    const char* st = smem + (kt % NS) * STAGE;
    auto fragment = [&](const char* rows, int r) {
      return both_chunks(*reinterpret_cast<const u32x4*>(rows + r * GROUP + 16 * (g ^ swap_of(r))),
                         *reinterpret_cast<const u32x4*>(rows + r * GROUP + 16 * ((4 + g) ^ swap_of(r))));
    };
    i32x8 xf[TM], wf[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) xf[i] = fragment(st, wm * (BM / WGM) + 16 * i + l16);
#pragma unroll
    for (int j = 0; j < TN; ++j) wf[j] = fragment(st + XB, wn * (BN / WGN) + 16 * j + l16);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
        acc[i][j] = mfma_codes<0>(wf[j], xf[i], acc[i][j], ws[j], xs[i]);
#pragma unroll
    for (int i = 0; i < TM; ++i) xs[i] >>= 8;   // the next group's byte
#pragma unroll
    for (int j = 0; j < TN; ++j) ws[j] >>= 8;
  }
  // acc[i][j]: lane (l16, g) holds C[16i + l16][16j + 4g + r]
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m0 + wm * (BM / WGM) + 16 * i + l16;
    if (row >= P.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t col0 = n0 + wn * (BN / WGN) + 16 * j + 4 * g;
      if (part) {   // (N % 4 == 0)
        if (col0 < P.N) *reinterpret_cast<float4_t*>(part + ((int64_t)split * P.M + row) * P.N + col0) = acc[i][j];
      } else {
        store_row4<DT>(acc[i][j], row, col0, C, ldc, R, ldr, P.N, vec);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// long batches: 256 x 256 tiles, 8 waves of 128 x 64 in two alternating groups
// ------------------------------------------------------------------------------------------------
// A stage of 128 is 2048 cycles of products a SIMD (16 instructions of 64 cycles in each of its two waves), 192 KB of
// operand reads and 64 KB of copies, and all three have to overlap. Waves w and w + 4 share a SIMD; waves 4..7 run half a
// phase behind waves 0..3, so that one multiplies while the other reads and copies. A phase is one 64 x 64 half of the
// wave's tile: its first half reads the operands (in a stage's first phase the W's for both) and issues copies, its
// second, behind a barrier, multiplies. Two stages live in LDS. In halves from a stage's start (in brackets the second
// group, one later):
//   phase of stage kt     reads        they are back   copies                     waits for its copies of
//   0: halves 0, 1 (1, 2) W, X0        in half 0 (1)   X1 of kt + 1               X1 of kt
//   1: halves 2, 3 (3, 4) X1           in half 2 (3)   W and X0 of kt + 2         W and X0 of kt + 1
// (X0: rows 0-63 of each group of 128.) Both orders of a place in LDS hold by the barriers that end the first halves:
//  - what a copy overwrites has been read. A wave waits for its own reads before that barrier, so W and X0 of kt are in
//    every wave's registers behind the one that ends half 1, and X1 behind the one that ends half 3; the copies into
//    their places are issued in halves 2 (3) and, by the next stage's first phase, 4 (5).
//  - what is read has landed. A wave waits there too, until only its eight youngest copies are on their way: for W and
//    X0 of kt + 1 in half 2 (3), read in half 4 (5); for X1 of kt in half 0 (1), read in half 2 (3).
// The scale words of four stages (2 KB) are one more copy per wave, issued four stages before they are read, into the
// place of words that were read four stages earlier, and counted in that stage's waits; a lane keeps its six words in
// registers and each stage's instructions pick their byte.
//
// Measured, 8005 x 28672 x 4096 with the rows' encoding (21 us): 1,230 us in 128 x 128 tiles, 999 in four phases of 64 x 32
// quadrants a stage (the order of the 16-bit kernel, on 32 x 32 products: on 16 x 16 ones the compiler moves the sums from
// register to register and spills), 803 in two (2.40 PFLOP/s). With the copies issued one half later in place of the wait
// for the reads 830. What bounds it: with the reads not yet waited for (795-825), the loop without its copies took 675,
// without the operand reads 640, with neither 597, all tiles the same one (copies from L2 alone) 700.
template <int DT, bool PARTIAL>
__global__ void __launch_bounds__(512, 2) gemm_e4m3_long_kernel(Operands P, uint16_t* __restrict__ C, int64_t ldc,
                                                                const uint16_t* __restrict__ R, int64_t ldr, bool vec,
                                                                float* __restrict__ part) {
  constexpr int BUF = 256 * GROUP;      // one operand's stage
  constexpr int PITCH = 64 * 2 + 16;    // a row of a wave's rounded results
  constexpr int SMEM = 8 * 128 * PITCH;
  static_assert(SMEM >= 4 * BUF, "the ring fits: X stages 0, 1, then W stages 0, 1");
  __shared__ __attribute__((aligned(1024))) char smem[SMEM];
  __shared__ __attribute__((aligned(256))) uint32_t words[2][512];   // X rows', then W rows'
  int64_t m0, n0;
  if (!tile_of(P.tiles_m, P.ntiles, 256, 256, m0, n0)) return;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem, words0 = (uint32_t)(uintptr_t)words;

  // Copies: 8 rows of 128 bytes each; lane l takes row l >> 3, physical chunk l & 7 of it, which holds logical chunk
  // (l & 7) ^ swap_of(row). A wave's rows of either operand are 64 i + 8 wave ..; half q of X has i = q and q + 2.
  const int cr = lane >> 3, cc = (lane & 7) ^ swap_of(8 * (wave & 1) + cr);
  uint32_t xo[4], wo[4];
  const int crow = 8 * wave;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    xo[i] = (uint32_t)((min(m0 + 64 * i + crow + cr, P.M - 1) - m0) * P.ldx + 16 * cc);
    wo[i] = (uint32_t)((min(n0 + 64 * i + crow + cr, P.N - 1) - n0) * P.ldw + 16 * cc);
  }
  const int split = blockIdx.y, nk = P.nk / (int)gridDim.y, first = split * nk;   // (nk % 4 == 0 where K is split)
  const char* xb = reinterpret_cast<const char*>(P.x + m0 * P.ldx + (int64_t)first * GROUP);
  const char* wb = reinterpret_cast<const char*>(P.w + n0 * P.ldw + (int64_t)first * GROUP);
  auto copy_x = [&](int q, int kt, int buf) {
#pragma unroll
    for (int i = q; i < 4; i += 2)
      dma16_at(xb + (int64_t)kt * GROUP, xo[i], lds0 + (uint32_t)(buf * BUF + (64 * i + crow) * GROUP));
  };
  auto copy_w = [&](int kt, int buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      dma16_at(wb + (int64_t)kt * GROUP, wo[i], lds0 + (uint32_t)((2 + buf) * BUF + (64 * i + crow) * GROUP));
  };
  // 64 rows' words of the four stages from kt (a multiple of 4) on: waves 0..3 X's, 4..7 W's
  const int64_t srows = wm ? P.N : P.M;
  const uint32_t so = (uint32_t)(4 * min((wm ? n0 : m0) + 64 * (wave & 3) + lane, srows - 1));
  const char* sb = reinterpret_cast<const char*>(wm ? P.ws : P.xs) + (int64_t)(first >> 2) * 4 * srows;
  auto copy_s = [&](int kt) {
    dma4_at(sb + (int64_t)(kt >> 2) * 4 * srows, so, words0 + (uint32_t)(4 * ((kt >> 2 & 1) * 512 + 64 * wave)));
  };

  // Operands: lane l holds row l % 32 of a tile of 32 and, of k-step ks, chunks 4 ks + 2 (l / 32) and the next.
  typedef __attribute__((address_space(3))) const u32x4 LdsFrag;
  const int l32 = lane & 31, half = lane >> 5;
  uint32_t xl[4], wl[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t at = 16 * ((4 * (c >> 1) + 2 * half + (c & 1)) ^ swap_of(l32));
    xl[c] = lds0 + (uint32_t)((wm * 128 + l32) * GROUP) + at;
    wl[c] = lds0 + 2 * BUF + (uint32_t)((wn * 64 + l32) * GROUP) + at;
  }

  f32x16 acc[4][2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
  i32x8 xf[2][2], wf[2][2];   // [tile][k-step]
  uint32_t xs[4], ws[2];

  auto read_x = [&](int q, int buf) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t at = (uint32_t)(buf * BUF + q * 64 * GROUP + i * 32 * GROUP);
        xf[i][ks] = both_chunks(*(LdsFrag*)(uintptr_t)(xl[2 * ks] + at), *(LdsFrag*)(uintptr_t)(xl[2 * ks + 1] + at));
      }
  };
  auto read_w = [&](int buf) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t at = (uint32_t)(buf * BUF + j * 32 * GROUP);
        wf[j][ks] = both_chunks(*(LdsFrag*)(uintptr_t)(wl[2 * ks] + at), *(LdsFrag*)(uintptr_t)(wl[2 * ks + 1] + at));
      }
  };
  auto read_s = [&](int kt) {
    const uint32_t* p = words[kt >> 2 & 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) xs[i] = p[wm * 128 + 32 * i + l32];
#pragma unroll
    for (int j = 0; j < 2; ++j) ws[j] = p[256 + wn * 64 + 32 * j + l32];
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // the end of a phase's first half, its reads back, and the second half: 8 products
  auto mul = [&](auto byte, int q) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    barrier();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[2 * q + i][j] = mfma_codes32<decltype(byte)::value>(wf[j][ks], xf[i][ks], acc[2 * q + i][j], ws[j], xs[2 * q + i]);
    __builtin_amdgcn_s_setprio(0);
    barrier();
  };
  // stage kt, whose groups are byte kt % 4 of the words. inner: two more stages follow it, and four behind its group's
  // first (no branches: the compiler moves these products past them, barriers or not, to the stage's end)
  auto stage = [&](int kt, auto byte, auto inner) {
    constexpr int buf = decltype(byte)::value & 1;   // kt & 1
    constexpr bool IN = decltype(inner)::value != 0;
    const bool next = IN || kt + 1 < nk, next2 = IN || kt + 2 < nk;
    const bool scales = decltype(byte)::value == 0 && (IN || kt + 4 < nk);   // this stage's waits count one copy more
    if (decltype(byte)::value == 0) read_s(kt);
    read_w(buf);
    read_x(0, buf);
    if (scales) copy_s(kt + 4);
    if (next) {
      copy_x(1, kt + 1, buf ^ 1);
      if (scales) wait_vm<9>();
      else wait_vm<8>();
    } else {
      wait_vm<0>();
    }
    mul(byte, 0);
    read_x(1, buf);
    if (next2) {
      copy_w(kt + 2, buf);
      copy_x(0, kt + 2, buf);
      if (scales) wait_vm<9>();
      else wait_vm<8>();
    } else if (next) {
      wait_vm<2>();
    }
    mul(byte, 1);
  };

  copy_s(0);
  copy_w(0, 0);
  copy_x(0, 0, 0);
  copy_x(1, 0, 0);
  if (nk > 1) {
    copy_w(1, 1);
    copy_x(0, 1, 1);
    wait_vm<8>();
  } else {
    wait_vm<2>();
  }
  barrier();
  if (wm) barrier();   // the second group runs one barrier behind
  int kt = 0;
  for (; kt + 5 < nk; kt += 4) {
    stage(kt, Int<0>{}, Int<1>{});
    stage(kt + 1, Int<1>{}, Int<1>{});
    stage(kt + 2, Int<2>{}, Int<1>{});
    stage(kt + 3, Int<3>{}, Int<1>{});
  }
  for (; kt < nk; kt += 4) {
    stage(kt, Int<0>{}, Int<0>{});
    if (kt + 1 < nk) stage(kt + 1, Int<1>{}, Int<0>{});
    if (kt + 2 < nk) stage(kt + 2, Int<2>{}, Int<0>{});
    if (kt + 3 < nk) stage(kt + 3, Int<3>{}, Int<0>{});
  }
  if (!wm) barrier();

  // acc[i][j][4 t + r]: the lane holds C[32 i + l32][32 j + 8 t + 4 half + r]
  auto four = [&](int i, int j, int t) { return float4_t{acc[i][j][4 * t], acc[i][j][4 * t + 1], acc[i][j][4 * t + 2], acc[i][j][4 * t + 3]}; };
  if (PARTIAL) {   // (N % 4 == 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = m0 + wm * 128 + 32 * i + l32;
      float* prow = part + ((int64_t)split * P.M + row) * P.N;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int64_t col0 = n0 + wn * 64 + 32 * j + 8 * t + 4 * half;
          if (row < P.M && col0 < P.N) *reinterpret_cast<float4_t*>(prow + col0) = four(i, j, t);
        }
    }
    return;
  }
  // The wave's rounded results (the residual added before) to LDS, then out by whole rows, 16 bytes a lane. Every copy
  // has landed and, past this barrier, every wave has read its last operands: the ring's space is free.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  char* out = smem + wave * 128 * PITCH;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = m0 + wm * 128 + 32 * i + l32;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float4_t a = four(i, j, t);
        const int64_t col0 = n0 + wn * 64 + 32 * j + 8 * t + 4 * half;
        if (R && row < P.M) {
          if (vec && col0 + 4 <= P.N) {
            const u32x2_t r = *reinterpret_cast<const u32x2_t*>(R + row * ldr + col0);
#pragma unroll
            for (int e = 0; e < 4; ++e) a[e] += half_of<DT>(r[e >> 1], e & 1);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col0 + e < P.N) a[e] += Elem<DT>::to_f32(R[row * ldr + col0 + e]);
          }
        }
        *reinterpret_cast<u32x2_t*>(out + (32 * i + l32) * PITCH + 2 * (32 * j + 8 * t + 4 * half)) =
            u32x2_t{(uint32_t)Elem<DT>::store_bits(a[0]) | ((uint32_t)Elem<DT>::store_bits(a[1]) << 16),
                    (uint32_t)Elem<DT>::store_bits(a[2]) | ((uint32_t)Elem<DT>::store_bits(a[3]) << 16)};
      }
  }
  const int64_t col = n0 + wn * 64 + 8 * (lane & 7);
  const bool wide = col + 8 <= P.N && (ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
#pragma unroll 4
  for (int it = 0; it < 16; ++it) {
    const int lr = it * 8 + (lane >> 3);
    const int64_t row = m0 + wm * 128 + lr;
    const u32x4 o = *reinterpret_cast<const u32x4*>(out + lr * PITCH + 16 * (lane & 7));
    if (row >= P.M) continue;
    if (wide) {
      *reinterpret_cast<u32x4*>(C + row * ldc + col) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < P.N) C[row * ldc + col + e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
    }
  }
}

// C = round(sum of the splits' partials in order (+ R)), four columns a thread.
template <int DT>
__global__ void __launch_bounds__(256) gemm_e4m3_join_kernel(const float* __restrict__ part, int splits, int64_t M, int64_t N,
                                                             uint16_t* __restrict__ C, int64_t ldc,
                                                             const uint16_t* __restrict__ R, int64_t ldr, bool vec) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= M * N) return;
  const int64_t row = e / N;
  float4_t a = *reinterpret_cast<const float4_t*>(part + e);
  for (int s = 1; s < splits; ++s) {
    const float4_t b = *reinterpret_cast<const float4_t*>(part + (int64_t)s * M * N + e);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] += b[r];
  }
  store_row4<DT>(a, row, e - row * N, C, ldc, R, ldr, N, vec);
}

struct Plan {
  int bm, bn, splits;
};
// The tile and the K splits of a shape: the cheapest of what a sweep over the 8B and 1B projections and 17 to 8000 rows
// fits (us): each round of 256 workgroups takes its stages at `stage` and `fixed` on top (of 64 x 64 tiles two share a
// CU, at half the rate each), and a split writes and reads its partials at 4.5 TB/s and joins them in a launch of 3.
// What the sweep's best would have saved over these choices is 1-2 us of 15-50, 5% beyond. Without the 256 x 128 tiles,
// which copy three quarters of 128 x 128's bytes for a product, 256 x 28672 x 4096 took 53.8 us for 45.1, 1000 x 6144 x 4096
// 52.1 for 42.3, 448 x 16384 x 2048 33.0 for 28.1, 2000 x 4096 x 4096 55.6 for 46.0.
Plan plan_for(int64_t M, int64_t N, int64_t K) {
  struct Cand {
    int bm, bn;
    double stage, fixed;
  };
  static const Cand cands[] = {{64, 64, 0.43, 3.0}, {128, 128, 0.66, 5.0}, {256, 128, 1.05, 7.0}, {256, 256, 1.5, 10.0}};
  const int64_t nk = K / GROUP;
  Plan best{64, 64, 1};
  double least = 1e30;
  for (const Cand& c : cands) {
    const int64_t tiles = ((M + c.bm - 1) / c.bm) * ((N + c.bn - 1) / c.bn);
    for (int s = 1; s <= 8; s *= 2) {
      // (a split starts at a whole word of scales; partials are stored four columns at a time)
      if (s > 1 && (nk % (4 * s) != 0 || N % 4 != 0)) break;
      const double us = (double)((tiles * s + 255) / 256) * ((double)(nk / s) * c.stage + c.fixed) +
                        (s > 1 ? 3.0 + (double)s * (double)M * (double)N * 8.0 / 4.5e6 : 0.0);
      if (us < least) least = us, best = Plan{c.bm, c.bn, s};
    }
  }
  return best;
}

int64_t scale_bytes(int64_t rows, int64_t K) { return (K + 511) / 512 * rows * 4; }
int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Whether one launch takes a call: few rows, in aligned pieces. Every workgroup encodes them for itself, 0.06 us per KB of
// codes and round of workgroups, where the other way's two more launches cost 4.5 us: 16 x 4096 x 4096 12.0 us against
// 14.3, 8 x 2048 x 8192 13.5 against 14.9, 8 x 4096 x 14336 22.8 against 18.8; in two rounds 4 x 28672 x 4096 32.7 against
// 31.2, 1 x 31.1.
bool short_size(int64_t M, int64_t N, int64_t K) { return M <= SHORT_ROWS && M * K <= (N <= 16384 ? SHORT_BYTES : 8 * 1024); }
bool short_call(int64_t M, int64_t N, int64_t K, const void* X, int64_t ldx) {
  return short_size(M, N, K) && al16(X) && ldx % 8 == 0;
}
// So many 16-column tiles a workgroup of it that the grid is one round of the CUs where it can be.
int short_tiles(int64_t N) {
  const int64_t tiles = (N + 15) / 16;
  return tiles <= 256 ? 1 : tiles <= 512 ? 2 : 4;
}

void quantize(const void* X, int64_t ldx, int64_t rows, int64_t K, int32_t dtype, uint8_t* codes, int64_t ldc, uint32_t* scales,
              hipStream_t s) {
  const int64_t kw = (K + 511) / 512;
  const dim3 grid((unsigned)((rows * kw + 3) / 4));
  const bool vec = al16(X) && ldx % 8 == 0;
  if (dtype == FS_F32)
    quantize_e4m3_kernel<FS_F32, false><<<grid, 256, 0, s>>>((const float*)X, ldx, rows, K, codes, ldc, scales, kw);
  else if (dtype == FS_BF16 && vec)
    quantize_e4m3_kernel<FS_BF16, true><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, rows, K, codes, ldc, scales, kw);
  else if (dtype == FS_BF16)
    quantize_e4m3_kernel<FS_BF16, false><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, rows, K, codes, ldc, scales, kw);
  else if (vec)
    quantize_e4m3_kernel<FS_F16, true><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, rows, K, codes, ldc, scales, kw);
  else
    quantize_e4m3_kernel<FS_F16, false><<<grid, 256, 0, s>>>((const uint16_t*)X, ldx, rows, K, codes, ldc, scales, kw);
}

template <int DT>
int gemm(const uint16_t* X, int64_t ldx, const uint8_t* W, int64_t ldw, const uint8_t* ws, uint16_t* C, int64_t ldc,
         const uint16_t* R, int64_t ldr, int64_t M, int64_t N, int64_t K, char* work, hipStream_t s) {
  const bool vec = rows_by_8(C, ldc, R, ldr);
  const int nk = (int)(K / GROUP);
  if (short_call(M, N, K, X, ldx)) {
    const int64_t tiles = (N + 15) / 16;
    const int tn = short_tiles(N);
#define FS_SHORT_XB(TN, DEPTH, XB)                                                                                     \
  gemm_e4m3_short_kernel<DT, TN, DEPTH, XB><<<dim3((unsigned)((tiles + TN - 1) / TN)), 512, 0, s>>>(X, ldx, W, ldw, ws, C, ldc, \
                                                                                                    R, ldr, (int)M, N, nk, vec)
#define FS_SHORT(TN, DEPTH)                                          \
  do {                                                               \
    if (M * K <= 32 * 1024) FS_SHORT_XB(TN, DEPTH, 32 * 1024);        \
    else FS_SHORT_XB(TN, DEPTH, SHORT_BYTES);                        \
  } while (0)
    if (tn == 1) FS_SHORT(1, 7);
    else if (tn == 2) FS_SHORT(2, 4);
    else FS_SHORT(4, 2);
#undef FS_SHORT_XB
#undef FS_SHORT
    return fs::launch_status("gemm_e4m3");
  }
  uint8_t* codes = reinterpret_cast<uint8_t*>(work);
  uint8_t* xs = codes + align256(M * K);
  float* part = reinterpret_cast<float*>(xs + align256(scale_bytes(M, K)));
  quantize(X, ldx, M, K, DT, codes, K, reinterpret_cast<uint32_t*>(xs), s);
  const Plan p = plan_for(M, N, K);
  Operands P{codes, W, xs, ws, K, ldw, M, N, nk, (int)((M + p.bm - 1) / p.bm), 0};
  P.ntiles = P.tiles_m * (int)((N + p.bn - 1) / p.bn);
  const dim3 grid((unsigned)(8 * ((P.ntiles + 7) / 8)), (unsigned)p.splits);
  float* out = p.splits > 1 ? part : nullptr;
  if (p.bm == 64)
    gemm_e4m3_tile_kernel<DT, 64, 64, 2, 2, 4><<<grid, 256, 0, s>>>(P, C, ldc, R, ldr, vec, out);
  else if (p.bn == 256 && out)
    gemm_e4m3_long_kernel<DT, true><<<grid, 512, 0, s>>>(P, C, ldc, R, ldr, vec, out);
  else if (p.bn == 256)
    gemm_e4m3_long_kernel<DT, false><<<grid, 512, 0, s>>>(P, C, ldc, R, ldr, vec, nullptr);
  else if (p.bm == 256)
    gemm_e4m3_tile_kernel<DT, 256, 128, 4, 2, 3><<<grid, 512, 0, s>>>(P, C, ldc, R, ldr, vec, out);
  else
    gemm_e4m3_tile_kernel<DT, 128, 128, 2, 4, 4><<<grid, 512, 0, s>>>(P, C, ldc, R, ldr, vec, out);
  if (p.splits > 1) {
    const int64_t n4 = M * N / 4;
    gemm_e4m3_join_kernel<DT><<<dim3((unsigned)((n4 + 255) / 256)), 256, 0, s>>>(part, p.splits, M, N, C, ldc, R, ldr, vec);
  }
  return fs::launch_status("gemm_e4m3");
}

}  // namespace

extern "C" int fs_quantize_e4m3(const void* X, int64_t ldx, int64_t rows, int64_t K, int32_t dtype, void* codes, int64_t ldc,
                                void* scales, void* stream) {
  FS_CHECK_ARG(X && codes && scales, "quantize_e4m3: null pointer");
  FS_CHECK_ARG(dtype == FS_F32 || dtype == FS_BF16 || dtype == FS_F16, "quantize_e4m3: dtype %d", dtype);
  FS_CHECK_ARG(rows >= 0 && K > 0 && K % GROUP == 0 && ldx >= K && ldc >= K, "quantize_e4m3: rows %lld K %lld (a multiple of %d)",
               (long long)rows, (long long)K, GROUP);
  FS_CHECK_ARG(ldc % 16 == 0 && al16(codes) && (reinterpret_cast<uintptr_t>(scales) & 3) == 0,
               "quantize_e4m3: codes need 16-byte aligned rows, scales whole words");
  FS_CHECK_ARG(rows * ((K + 511) / 512) < 0x7fffffffLL, "quantize_e4m3: rows %lld K %lld", (long long)rows, (long long)K);
  if (rows == 0) return 0;
  quantize(X, ldx, rows, K, dtype, reinterpret_cast<uint8_t*>(codes), ldc, reinterpret_cast<uint32_t*>(scales), fs::as_stream(stream));
  return fs::launch_status("quantize_e4m3");
}

extern "C" int64_t fs_gemm_e4m3_workspace_size(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || K % GROUP) return 0;
  const Plan p = plan_for(M, N, K);
  return align256(M * K) + align256(scale_bytes(M, K)) + (p.splits > 1 ? (int64_t)p.splits * M * N * (int64_t)sizeof(float) : 0);
}

extern "C" int fs_gemm_e4m3_plan(int64_t M, int64_t N, int64_t K, int32_t* plan) {
  FS_CHECK_ARG(plan && M > 0 && N > 0 && K > 0 && K % GROUP == 0, "gemm_e4m3_plan: M %lld N %lld K %lld (K a multiple of %d)",
               (long long)M, (long long)N, (long long)K, GROUP);
  Plan p = plan_for(M, N, K);
  if (short_size(M, N, K)) p = Plan{SHORT_ROWS, 16 * short_tiles(N), 1};
  plan[0] = p.bm;
  plan[1] = p.bn;
  plan[2] = p.splits;
  return 0;
}

extern "C" int fs_gemm_e4m3(const void* X, int64_t ldx, const void* W, int64_t ldw, const void* w_scales, void* C, int64_t ldc,
                            const void* R, int64_t ldr, int64_t M, int64_t N, int64_t K, int32_t dtype, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  FS_CHECK_ARG(X && W && w_scales && C, "gemm_e4m3: null pointer");
  FS_CHECK_ARG(dtype == FS_BF16 || dtype == FS_F16, "gemm_e4m3: bf16 and f16 rows (dtype %d)", dtype);
  FS_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K % GROUP == 0, "gemm_e4m3: M %lld N %lld K %lld (K a multiple of %d)", (long long)M,
               (long long)N, (long long)K, GROUP);
  FS_CHECK_ARG(ldx >= K && ldw >= K && ldc >= N && (!R || ldr >= N), "gemm_e4m3: leading dimensions");
  FS_CHECK_ARG(ldw % 16 == 0 && al16(W) && (reinterpret_cast<uintptr_t>(w_scales) & 3) == 0,
               "gemm_e4m3: codes need 16-byte aligned rows, scales whole words");
  // a copy's offset inside its tile of rows, and a row's scale word inside its group of K, are 32 bits
  FS_CHECK_ARG(K <= (1 << 22) && ldw < (1 << 23) && M < (1 << 29) && N < (1 << 29), "gemm_e4m3: M %lld N %lld K %lld ldw %lld",
               (long long)M, (long long)N, (long long)K, (long long)ldw);
  if (M == 0) return 0;
  const int64_t need = fs_gemm_e4m3_workspace_size(M, N, K);
  FS_CHECK_ARG(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
               "gemm_e4m3: workspace %lld < %lld bytes (or not 256-byte aligned)", (long long)workspace_bytes, (long long)need);
  hipStream_t s = fs::as_stream(stream);
  char* work = reinterpret_cast<char*>(workspace);
  const auto call = dtype == FS_BF16 ? gemm<FS_BF16> : gemm<FS_F16>;
  return call((const uint16_t*)X, ldx, (const uint8_t*)W, ldw, (const uint8_t*)w_scales, (uint16_t*)C, ldc, (const uint16_t*)R,
              ldr, M, N, K, work, s);
}
