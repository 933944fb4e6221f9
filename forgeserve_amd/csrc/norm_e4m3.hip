// Rows between projections over codes: the residual's addition and RMS norm with the output in codes, and codes as values.
//
//   v = x, or round(x + delta) (written too);  codes of v r w,  r = 1 / sqrt(mean(v^2) + eps)
//
// Everything behind v is f32 and rounded once, to the code: where the norm's 16-bit output is encoded afterwards it has been
// rounded twice before. A row is held in registers between the sum of its squares and its codes, so each byte is read once:
// HBM bounds long batches, the chain of one row's loads, sum and stores short ones. A row's result depends on its length
// only, not on the batch.
#include "rows_e4m3.h"

namespace {

template <int DT>
struct Eight {   // eight values of a row as loaded
  u32x4 w[DT == FS_F32 ? 2 : 1];
};
template <int DT, bool VEC>
FS_DEVICE Eight<DT> load8(const typename Elem<DT>::T* p) {
  Eight<DT> r;
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < (DT == FS_F32 ? 2 : 1); ++h) r.w[h] = reinterpret_cast<const u32x4*>(p)[h];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (DT == FS_F32) r.w[e >> 2][e & 3] = __float_as_uint(p[e]);
      else if (e & 1) r.w[0][e >> 1] |= (uint32_t)p[e] << 16;
      else r.w[0][e >> 1] = p[e];
    }
  }
  return r;
}
template <int DT>
FS_DEVICE float value_of(const Eight<DT>& r, int e) {
  if constexpr (DT == FS_F32) return __uint_as_float(r.w[e >> 2][e & 3]);
  else return half_of<DT>(r.w[0][e >> 1], e & 1);
}
// PAST: past the caches.
template <bool PAST, class T>
FS_DEVICE void store16(T* p, T v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <int DT, bool VEC, bool PAST>
FS_DEVICE void store8(typename Elem<DT>::T* p, const float (&v)[8]) {
  if constexpr (VEC && DT == FS_F32) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      store16<PAST>(reinterpret_cast<float4_t*>(p) + h, float4_t{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]});
  } else if constexpr (VEC) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = (uint32_t)Elem<DT>::store_bits(v[2 * j]) | ((uint32_t)Elem<DT>::store_bits(v[2 * j + 1]) << 16);
    store16<PAST>(reinterpret_cast<u32x4*>(p), w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) Elem<DT>::store(p, e, v[e]);
  }
}

// The codes of eight normed values a lane, 16 lanes a group, a wave 512 columns: the row's word k4 with them. `in`: whether
// the lane's columns exist (whole groups).
FS_DEVICE void store_codes(const float (&y)[8], bool in, uint8_t* codes, uint32_t* word, int lane) {
  int e;
  const u32x2_t c = encode_eight(y, e);
  if (in) *reinterpret_cast<u32x2_t*>(codes) = c;
  uint32_t w = (lane & 15) == 0 && in ? (uint32_t)e << (8 * (lane >> 4)) : 0u;   // lane 16 g holds byte g, zeros past the row
  w |= (uint32_t)__shfl_xor((int)w, 16, 64);
  w |= (uint32_t)__shfl_xor((int)w, 32, 64);
  if (lane == 0) *word = w;
}

struct NormArgs {
  const void* x;
  const void* delta;
  void* x_out;
  const void* w;
  uint8_t* codes;
  uint32_t* scales;
  int64_t ldx, ldd, ldxo, ldc, M;
  int N;
  float eps;
};

// T threads a row, WG / T rows a workgroup, a thread's pieces of eight columns t, t + T, ... (G of them). The squares of 512
// columns, a wave's, are added across it and these sums in order, whatever T and G. G == 0: rows of any length, v read again
// for the codes.
// x_out is written past the caches: what reads it next comes two products later, and the codes, read first, stay in them
// (1000 x 4096 bf16 8.6 -> 7.7 us, 8005 x 4096 40.1 -> 38.7, 8005 x 8192 83.6 -> 81.0; with the products and the next norm
// behind it 1000 rows 197.2 -> 196.2, 2777 rows 451.4 -> 450.2; a read-back's values, which are read next, lose by it: 2777 rows
// and a norm of them 20.3 -> 23.4).
template <int DT, bool VEC, bool DELTA, int T, int WG, int G>
__global__ void __launch_bounds__(WG) add_rmsnorm_e4m3_kernel(NormArgs a) {
  typedef typename Elem<DT>::T E;
  static_assert(T == 64 || T == WG, "a wave or a workgroup a row");
  constexpr int SUMS = G > 0 ? G * (T / 64) : WG / 64;   // of 512 columns each, or a wave's
  __shared__ float red[T > 64 ? SUMS : 1];
  const int t = threadIdx.x % T, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (WG / T) + threadIdx.x / T;
  if (T == 64 && row >= a.M) return;
  const E* x = static_cast<const E*>(a.x) + row * a.ldx;
  const E* delta = DELTA ? static_cast<const E*>(a.delta) + row * a.ldd : nullptr;
  E* xo = DELTA ? static_cast<E*>(a.x_out) + row * a.ldxo : nullptr;
  const E* w = static_cast<const E*>(a.w);
  const int np = a.N / 8;
  uint8_t* codes = a.codes + row * a.ldc;

  auto sum_piece = [&](int p, const Eight<DT>& xr, const Eight<DT>& dr, float (&v)[8]) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = value_of<DT>(xr, e);
      if (DELTA) v[e] = Elem<DT>::round(v[e] + value_of<DT>(dr, e));
      sq += v[e] * v[e];
    }
    if (DELTA) store8<DT, VEC, (G > 0)>(xo + 8 * p, v);
    return sq;
  };
  auto scale_of = [&](float sum) { return 1.0f / sqrtf(sum / (float)a.N + a.eps); };
  auto added = [&]() {
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < SUMS; ++i) sum += red[i];
    return sum;
  };
  auto codes_of = [&](int p, const float (&v)[8], const Eight<DT>& wr, float r) {   // p: all of a wave's in turn
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = v[e] * r * value_of<DT>(wr, e);
    store_codes(y, p < np, codes + 8 * p, a.scales + (int64_t)(p >> 6) * a.M + row, lane);
  };

  if constexpr (G > 0) {
    Eight<DT> xr[G], dr[G], wr[G];
#pragma unroll
    for (int u = 0; u < G; ++u) {   // every load in flight before any arithmetic
      const int p = min(t + T * u, np - 1);
      xr[u] = load8<DT, VEC>(x + 8 * p);
      if (DELTA) dr[u] = load8<DT, VEC>(delta + 8 * p);
    }
#pragma unroll
    for (int u = 0; u < G; ++u) wr[u] = load8<DT, VEC>(w + 8 * min(t + T * u, np - 1));
    __builtin_amdgcn_sched_barrier(0);   // (the compiler would wait for each piece's before it loads the next)
    float v[G][8], sum = 0.f;
#pragma unroll
    for (int u = 0; u < G; ++u) {
      float sq = 0.f;
      if (t + T * u < np) {
        sq = sum_piece(t + T * u, xr[u], dr[u], v[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
      }
      sq = wave_sum(sq);
      if (T == 64) sum += sq;
      else if (lane == 0) red[(t >> 6) + (T / 64) * u] = sq;
    }
    const float r = scale_of(T == 64 ? sum : added());
#pragma unroll
    for (int u = 0; u < G; ++u)
      if (((t & ~63) + T * u) < np) codes_of(t + T * u, v[u], wr[u], r);   // (wave-uniform)
  } else {
    float sq = 0.f;
    for (int p = t; p < np; p += T) {
      float v[8];
      const Eight<DT> xr = load8<DT, VEC>(x + 8 * p), dr = DELTA ? load8<DT, VEC>(delta + 8 * p) : xr;
      sq += sum_piece(p, xr, dr, v);
    }
    sq = wave_sum(sq);
    if (lane == 0) red[t >> 6] = sq;
    const float r = scale_of(added());
    const E* again = DELTA ? xo : x;   // (a thread reads what it wrote itself)
    for (int p = t; (p & ~63) < np; p += T) {
      float v[8];
      const int at = 8 * min(p, np - 1);
      const Eight<DT> vr = load8<DT, VEC>(p < np ? again + at : x), wr = load8<DT, VEC>(w + at);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = value_of<DT>(vr, e);
      codes_of(p, v, wr, r);
    }
  }
}

// A wave per 512 columns of a row, eight codes a lane. Bound by HBM: 8005 x 4096 to bf16 in 18.4 us, 5.4 TB/s; by its latency
// where rows are few (64 x 4096 2.8).
template <int DT, bool VEC>
__global__ void __launch_bounds__(256) dequantize_e4m3_kernel(const uint8_t* __restrict__ codes, int64_t ldc,
                                                              const uint32_t* __restrict__ scales, int64_t rows, int64_t K,
                                                              int64_t kw, typename Elem<DT>::T* __restrict__ out, int64_t ldo) {
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= rows * kw) return;
  const int lane = threadIdx.x & 63;
  const int64_t row = unit / kw, k4 = unit - row * kw, k = k4 * 512 + lane * 8;
  if (k >= K) return;
  const u32x2_t c = *reinterpret_cast<const u32x2_t*>(codes + row * ldc + k);
  const float s = scale_value((int)(scales[k4 * rows + row] >> (8 * (lane >> 4)) & 255u));
  float a[4], b[4];
  decode4(c[0], a);
  decode4(c[1], b);
  const float v[8] = {a[0] * s, a[1] * s, a[2] * s, a[3] * s, b[0] * s, b[1] * s, b[2] * s, b[3] * s};
  store8<DT, VEC, false>(out + row * ldo + k, v);
}

bool dtype_ok(int32_t dt) { return dt == FS_F32 || dt == FS_BF16 || dt == FS_F16; }

// Up to four rows a CU are held by their latency: one piece a thread (64 x 4096 bf16 with delta 3.7 us, two pieces 4.2; 64 x
// 8192 4.5, four pieces 5.7); longer batches by HBM, where fewer, larger threads draw more (8005 x 4096 21.0 us without delta,
// one piece 25.9; with delta 38.7, 5.9 TB/s). The results are the same. Rows of more than 16384 columns, which no configuration
// here has, are not held and read twice (2000 x 20480 bf16 with delta 60.7 us, 4.7 TB/s of the bytes that it cannot do without;
// 2000 x 16384 39.3, 5.8).
template <int DT, bool VEC, bool DELTA>
void launch_norm(const NormArgs& a, hipStream_t s) {
  const unsigned rows = (unsigned)a.M, rows4 = (unsigned)((a.M + 3) / 4);
  const bool few = a.M <= 1024;
#define FS_LAUNCH(T, WG, G) add_rmsnorm_e4m3_kernel<DT, VEC, DELTA, T, WG, G><<<T == 64 ? rows4 : rows, WG, 0, s>>>(a)
  if (a.N <= 512) FS_LAUNCH(64, 256, 1);
  else if (a.N <= 1024) FS_LAUNCH(64, 256, 2);
  else if (a.N <= 2048) FS_LAUNCH(256, 256, 1);
  else if (a.N <= 4096) few ? FS_LAUNCH(512, 512, 1) : FS_LAUNCH(256, 256, 2);
  else if (a.N <= 8192) few ? FS_LAUNCH(1024, 1024, 1) : FS_LAUNCH(256, 256, 4);
  else if (a.N <= 16384) few ? FS_LAUNCH(1024, 1024, 2) : FS_LAUNCH(512, 512, 4);
  else FS_LAUNCH(1024, 1024, 0);
#undef FS_LAUNCH
}
template <int DT>
void launch_norm(const NormArgs& a, bool vec, hipStream_t s) {
  if (a.delta) vec ? launch_norm<DT, true, true>(a, s) : launch_norm<DT, false, true>(a, s);
  else vec ? launch_norm<DT, true, false>(a, s) : launch_norm<DT, false, false>(a, s);
}

}  // namespace

extern "C" int fs_add_rmsnorm_e4m3(const void* x, int64_t ldx, const void* delta, int64_t ldd, void* x_out, int64_t ldxo,
                                   const void* weight, void* codes, int64_t ldc, void* scales, int64_t M, int64_t N, float eps,
                                   int32_t dtype, void* stream) {
  FS_CHECK_ARG(x && weight && codes && scales && (!delta || x_out), "add_rmsnorm_e4m3: null pointer");
  FS_CHECK_ARG(dtype_ok(dtype), "add_rmsnorm_e4m3: dtype %d", dtype);
  FS_CHECK_ARG(M >= 0 && N > 0 && N % GROUP == 0 && N < 0x7fff0000, "add_rmsnorm_e4m3: M %lld N %lld (a multiple of %d)",
               (long long)M, (long long)N, GROUP);
  // (below 2^32 threads: a wave a row, or up to 1024 threads)
  FS_CHECK_ARG(N <= 1024 ? waves_fit(M) : M < (1 << 22), "add_rmsnorm_e4m3: M %lld N %lld", (long long)M, (long long)N);
  FS_CHECK_ARG(ldx >= N && ldc >= N && (!delta || (ldd >= N && ldxo >= N)), "add_rmsnorm_e4m3: leading dimensions");
  FS_CHECK_ARG(ldc % 16 == 0 && al16(codes) && (reinterpret_cast<uintptr_t>(scales) & 3) == 0,
               "add_rmsnorm_e4m3: codes need 16-byte aligned rows, scales whole words");
  if (M == 0) return 0;
  hipStream_t s = fs::as_stream(stream);
  const NormArgs a{x, delta, x_out, weight, reinterpret_cast<uint8_t*>(codes), reinterpret_cast<uint32_t*>(scales), ldx, ldd, ldxo,
                   ldc, M, (int)N, eps};
  const int64_t per = dtype == FS_F32 ? 4 : 8;
  const bool vec = al16(x) && al16(weight) && ldx % per == 0 &&
                   (!delta || (al16(delta) && al16(x_out) && ldd % per == 0 && ldxo % per == 0));
  if (dtype == FS_F32) launch_norm<FS_F32>(a, vec, s);
  else if (dtype == FS_BF16) launch_norm<FS_BF16>(a, vec, s);
  else launch_norm<FS_F16>(a, vec, s);
  return fs::launch_status("add_rmsnorm_e4m3");
}

extern "C" int fs_dequantize_e4m3(const void* codes, int64_t ldc, const void* scales, int64_t rows, int64_t K, int32_t dtype,
                                  void* out, int64_t ldo, void* stream) {
  FS_CHECK_ARG(codes && scales && out, "dequantize_e4m3: null pointer");
  FS_CHECK_ARG(dtype_ok(dtype), "dequantize_e4m3: dtype %d", dtype);
  FS_CHECK_ARG(rows >= 0 && K > 0 && K % GROUP == 0 && ldc >= K && ldo >= K, "dequantize_e4m3: rows %lld K %lld (a multiple of %d)",
               (long long)rows, (long long)K, GROUP);
  FS_CHECK_ARG(ldc % 16 == 0 && al16(codes) && (reinterpret_cast<uintptr_t>(scales) & 3) == 0,
               "dequantize_e4m3: codes need 16-byte aligned rows, scales whole words");
  FS_CHECK_ARG(rows < (1 << 26) && waves_fit(rows * ((K + 511) / 512)), "dequantize_e4m3: rows %lld K %lld", (long long)rows, (long long)K);
  if (rows == 0) return 0;
  const int64_t kw = (K + 511) / 512;
  const dim3 grid((unsigned)((rows * kw + 3) / 4));
  const bool vec = al16(out) && ldo % (dtype == FS_F32 ? 4 : 8) == 0;
  hipStream_t s = fs::as_stream(stream);
#define FS_LAUNCH(DT, VEC)                                                                                                \
  dequantize_e4m3_kernel<DT, VEC><<<grid, 256, 0, s>>>(reinterpret_cast<const uint8_t*>(codes), ldc,                      \
                                                       reinterpret_cast<const uint32_t*>(scales), rows, K, kw,            \
                                                       reinterpret_cast<Elem<DT>::T*>(out), ldo)
  if (dtype == FS_F32) vec ? FS_LAUNCH(FS_F32, true) : FS_LAUNCH(FS_F32, false);
  else if (dtype == FS_BF16) vec ? FS_LAUNCH(FS_BF16, true) : FS_LAUNCH(FS_BF16, false);
  else vec ? FS_LAUNCH(FS_F16, true) : FS_LAUNCH(FS_F16, false);
#undef FS_LAUNCH
  return fs::launch_status("dequantize_e4m3");
}
