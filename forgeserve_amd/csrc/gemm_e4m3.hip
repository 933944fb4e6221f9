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
#include "gemm_e4m3.h"

namespace {

constexpr int SHORT_ROWS = 16;    // rows that one launch takes
constexpr int SHORT_BYTES = 64 * 1024;   // and their codes

// ------------------------------------------------------------------------------------------------
// encoding rows
// ------------------------------------------------------------------------------------------------
// A wave per 512 columns of a row: 16 lanes of 8 values share a group. VEC: rows of aligned 16-byte pieces (8005 x 4096 bf16
// 19.4 us); 32-bit rows come value by value (60.7), for weights are encoded once and activations have 16 bits.
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
  const ResidualOut<DT> out{C, ldc, R, ldr, vec, nullptr};
  put4(out, a, row, e - row * N, N);
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
// Whether a call's launches stay below 2^32 threads: a wave for a row's 512 columns that are encoded, a workgroup a tile
// (these in eights), a thread for four columns of joined splits.
bool launches_fit(int64_t M, int64_t N, int64_t K, bool in_one) {
  constexpr int64_t LIMIT = 1LL << 32;
  if (in_one) return ((N + 15) / 16 + short_tiles(N) - 1) / short_tiles(N) * 512 < LIMIT;
  const Plan p = plan_for(M, N, K);
  const int64_t tiles = ((M + p.bm - 1) / p.bm) * ((N + p.bn - 1) / p.bn);
  return waves_fit(M * ((K + 511) / 512)) && (tiles + 7) / 8 * 8 * (p.bm == 64 ? 256 : 512) < LIMIT &&
         (p.splits == 1 || M * N / 4 + 256 <= LIMIT);
}

}  // namespace

void fs::quantize_rows_e4m3(const void* X, int64_t ldx, int64_t rows, int64_t K, int32_t dtype, uint8_t* codes, int64_t ldc, uint32_t* scales,
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

namespace {

template <int DT>
int gemm(const uint16_t* X, int64_t ldx, const uint8_t* W, int64_t ldw, const uint8_t* ws, uint16_t* C, int64_t ldc,
         const uint16_t* R, int64_t ldr, int64_t M, int64_t N, int64_t K, char* work, hipStream_t s) {
  typedef ResidualOut<DT> Out;
  Out out{C, ldc, R, ldr, rows_by_8(C, ldc, R, ldr), nullptr};
  const int nk = (int)(K / GROUP);
  if (short_call(M, N, K, X, ldx)) {
    const int64_t tiles = (N + 15) / 16;
    const int tn = short_tiles(N);
#define FS_SHORT_XB(TN, DEPTH, XB)                                                                                     \
  gemm_e4m3_short_kernel<Out, TN, DEPTH, XB>                                                                           \
      <<<dim3((unsigned)((tiles + TN - 1) / TN)), 512, 0, s>>>(X, ldx, W, ldw, ws, out, (int)M, N, nk)
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
  fs::quantize_rows_e4m3(X, ldx, M, K, DT, codes, K, reinterpret_cast<uint32_t*>(xs), s);
  const Plan p = plan_for(M, N, K);
  Operands P{codes, W, xs, ws, K, ldw, M, N, nk, (int)((M + p.bm - 1) / p.bm), 0};
  P.ntiles = P.tiles_m * (int)((N + p.bn - 1) / p.bn);
  const dim3 grid((unsigned)(8 * ((P.ntiles + 7) / 8)), (unsigned)p.splits);
  out.part = p.splits > 1 ? part : nullptr;
  if (p.bm == 64)
    gemm_e4m3_tile_kernel<Out, 64, 64, 2, 2, 4><<<grid, 256, 0, s>>>(P, out);
  else if (p.bn == 256 && out.part)
    gemm_e4m3_long_kernel<Out, true><<<grid, 512, 0, s>>>(P, out);
  else if (p.bn == 256)
    gemm_e4m3_long_kernel<Out, false><<<grid, 512, 0, s>>>(P, out);
  else if (p.bm == 256)
    gemm_e4m3_tile_kernel<Out, 256, 128, 4, 2, 3><<<grid, 512, 0, s>>>(P, out);
  else
    gemm_e4m3_tile_kernel<Out, 128, 128, 2, 4, 4><<<grid, 512, 0, s>>>(P, out);
  if (p.splits > 1) {
    const int64_t n4 = M * N / 4;
    gemm_e4m3_join_kernel<DT><<<dim3((unsigned)((n4 + 255) / 256)), 256, 0, s>>>(part, p.splits, M, N, C, ldc, R, ldr, out.vec);
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
  FS_CHECK_ARG(rows < (1 << 26) && waves_fit(rows * ((K + 511) / 512)), "quantize_e4m3: rows %lld K %lld", (long long)rows, (long long)K);
  if (rows == 0) return 0;
  fs::quantize_rows_e4m3(X, ldx, rows, K, dtype, reinterpret_cast<uint8_t*>(codes), ldc, reinterpret_cast<uint32_t*>(scales), fs::as_stream(stream));
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
  FS_CHECK_ARG(launches_fit(M, N, K, short_call(M, N, K, X, ldx)), "gemm_e4m3: M %lld N %lld K %lld", (long long)M, (long long)N,
               (long long)K);
  const int64_t need = fs_gemm_e4m3_workspace_size(M, N, K);
  FS_CHECK_ARG(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0,
               "gemm_e4m3: workspace %lld < %lld bytes (or not 256-byte aligned)", (long long)workspace_bytes, (long long)need);
  hipStream_t s = fs::as_stream(stream);
  char* work = reinterpret_cast<char*>(workspace);
  const auto call = dtype == FS_BF16 ? gemm<FS_BF16> : gemm<FS_F16>;
  return call((const uint16_t*)X, ldx, (const uint8_t*)W, ldw, (const uint8_t*)w_scales, (uint16_t*)C, ldc, (const uint16_t*)R,
              ldr, M, N, K, work, s);
}
