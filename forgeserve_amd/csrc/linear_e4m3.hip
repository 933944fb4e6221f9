// Projections over codes with what follows them in one call: with z = x w^T + b,
//
//   y = act(z) + R, or with a gate (W and b hold the gate's F rows, then the others')  y = act(z_gate) * z_up + R
//
// x and w in e4m3 codes (rows_e4m3.h; 16-bit or 32-bit rows of x are encoded first), the sums as gemm_e4m3.hip's, everything
// behind them in f32 and rounded once: to 16-bit rows, or to codes with a scale for each 128 columns, which is what the next
// product reads. The products are gemm_e4m3.h's kernels; where a tile holds what its results need (a gate's column beside its
// other's: the tile's columns are drawn from both halves of W; for codes whole groups of 128 columns), the workgroup finishes
// them from LDS, else the sums go through memory and a second kernel finishes them.
#include "gemm_e4m3.h"

namespace {

// Rows that the streaming kernels may take, and, of more than 32, the bytes of their codes: every workgroup copies them all,
// beside one or two tiles of W. us, streamed and in tiles, of one weight called again and again / of 1 GB of weights in turn:
// 64 x 4096 x 4096 8.2 and 10.4 / 9.5 and 11.3; 100 x 4096 x 4096 10.7 and 12.6 / 11.5 and 14.3; 128 x 6144 x 4096 13.8 and 15.3 /
// 15.3 and 14.5; 64 x 2048 x 8192 10.6 and 10.4 / 12.6 and 11.3; over the limit 64 x 4096 x 14336 23.3 and 17.3 / 22.2 and 18.9, 96
// x 2048 x 8192 14.7 and 12.4 / 16.6 and 12.4; with four tiles 64 x 16384 x 2048 11.1 and 9.8.
constexpr int STREAM_ROWS = 128;
constexpr int64_t STREAM_BYTES = 600 * 1024;
// Bytes of W from which they are read past the caches (`nt`): of a weight's size several pass between two calls that read the
// same one, and then the caches have none of it. us, past them and through them, of one weight called again and again / of 1 GB
// of weights in turn: 1 x 4096 x 14336 11.5 and 12.5 / 12.1 and 13.0; 1 x 28672 x 4096 20.3 and 21.8 / 21.5 and 23.8; 1 x 128256 x
// 4096 82.6 and 91.9 / 81.4 and 89.5. Smaller ones are read through them, for they may still be there; that wins nothing to speak
// of (64 x 4096 x 4096 8.8 and 8.5, 8 x 6144 x 4096 5.8 both), and costs 4 to 8 % where a model's other layers pass in between, as
// in its decode steps (9.0 and 9.4; 7.7 and 8.3).
constexpr int64_t READ_ONCE = 32 << 20;

// ------------------------------------------------------------------------------------------------
// what is done with the sums
// ------------------------------------------------------------------------------------------------
// z / (1 + e^-y). The factor 2^-6 keeps the reciprocal a normal number up to e^-y = 2^128, where z's share of the result is
// less than 2^-120; the hardware's exponential and reciprocal are within two f32 steps, and y's rounding times log2(e)
// adds |y| 2^-24: nothing against 16 bits.
FS_DEVICE float over_one_plus_exp(float z, float y) {
  const float e = __builtin_amdgcn_exp2f(y * -1.4426950408889634f);
  return (z * 0x1p-6f) * __builtin_amdgcn_rcpf(fmaf(e, 0x1p-6f, 0x1p-6f));
}
// z Phi(z) with Phi(-a) = erfc(a / sqrt 2) / 2 = e^(-a^2 / 2) t Q(t) / 2, t = 1 / (1 + 0.4 a / sqrt 2): Q, of degree 6, is
// the polynomial whose largest relative error over 0 <= a <= 19.8 is least (3.5e-6, fitted to scipy's erfcx). The result is
// within 8e-6 of itself in both tails, a thirtieth of f16's rounding. About 22 instructions of a lane, 2.5 us of 333 x 8192's
// 17.2, which the vector units set.
FS_DEVICE float gelu_erf(float z) {
  const float a = fabsf(z), t = __builtin_amdgcn_rcpf(fmaf(a, 0.282842712f, 1.f));
  float q = -0.0880692603f;
  q = fmaf(q, t, 0.161608521f);
  q = fmaf(q, t, 0.102756314f);
  q = fmaf(q, t, 0.158245978f);
  q = fmaf(q, t, 0.215523985f);
  q = fmaf(q, t, 0.224155506f);
  q = fmaf(q, t, 0.225775499f);
  const float phi = 0.5f * t * q * __builtin_amdgcn_exp2f(a * a * -0.72134752f);   // Phi(-a)
  return z * (z < 0.f ? phi : 1.f - phi);
}

template <bool GATED_, bool CODES_>
struct LinearOut {
  static constexpr bool GATED = GATED_, CODES = CODES_, STAGED = true;
  uint16_t* C;            // rows, or codes
  int64_t ldc;            // in elements
  const uint16_t* R;
  int64_t ldr;
  const void* bias;
  int64_t up;             // where the others' bias begins
  int32_t dtype, bias_dtype, act;
  bool whole;             // eight columns of C, R and the bias at a time, all there
  uint8_t* scales;        // of codes
  int64_t rows;
  float* part;

  // a 16-bit value of the results' type
  FS_DEVICE float value(uint32_t h) const { return dtype == FS_BF16 ? bf16_to_f32((uint16_t)h) : f16_to_f32((uint16_t)h); }
  // two results rounded to it
  FS_DEVICE uint32_t pair(float a, float b) const {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return dtype == FS_BF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b16x2))
                            : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h16x2));
  }
  FS_DEVICE float bias_at(int64_t i) const {
    return bias_dtype == FS_F32 ? static_cast<const float*>(bias)[i]
                                : bias_dtype == FS_BF16 ? bf16_to_f32(static_cast<const uint16_t*>(bias)[i])
                                                        : f16_to_f32(static_cast<const uint16_t*>(bias)[i]);
  }
  // WHOLE: `whole`, and so no bounds and no single elements: little code, for it is fetched when every CU comes to need it
  template <bool WHOLE, int NC>
  FS_DEVICE void add_bias(float (&v)[NC], int64_t at, int64_t left) const {
    if (WHOLE && bias_dtype == FS_F32) {
#pragma unroll
      for (int h = 0; h < NC / 4; ++h) {
        const float4_t b = *reinterpret_cast<const float4_t*>(static_cast<const float*>(bias) + at + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] += b[e];
      }
    } else if (WHOLE) {
      uint32_t b[NC / 2];
#pragma unroll
      for (int h = 0; h < NC / 4; ++h) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(bias) + at + 4 * h);
        b[2 * h] = w[0];
        b[2 * h + 1] = w[1];
      }
#pragma unroll
      for (int e = 0; e < NC; ++e) {
        const uint32_t w = b[e >> 1] >> (16 * (e & 1));
        v[e] += bias_dtype == FS_BF16 ? bf16_to_f32((uint16_t)w) : f16_to_f32((uint16_t)w);
      }
    } else {
#pragma unroll 1
      for (int e = 0; e < NC; ++e) {
        if (e >= left) break;
        const float b = bias_at(at + e);
#pragma unroll
        for (int f = 0; f < NC; ++f) v[f] += f == e ? b : 0.f;
      }
    }
  }
  // NC columns' sums from col on, of `cols`, to what is rounded
  template <bool WHOLE, int NC>
  FS_DEVICE void compute(float (&v)[NC], float (&u)[NC], int64_t row, int64_t col, int64_t cols) const {
    if (bias) {
      add_bias<WHOLE>(v, col, cols - col);
      if (GATED) add_bias<WHOLE>(u, up + col, cols - col);
    }
    switch (act) {
      case FS_ACT_RELU:
#pragma unroll
        for (int e = 0; e < NC; ++e) v[e] = v[e] < 0.f ? 0.f : v[e];
        break;
      case FS_ACT_SILU:
#pragma unroll
        for (int e = 0; e < NC; ++e) v[e] = over_one_plus_exp(v[e], v[e]);
        break;
      case FS_ACT_GELU:
#pragma unroll
        for (int e = 0; e < NC; ++e) v[e] = gelu_erf(v[e]);
        break;
      case FS_ACT_GELU_TANH:   // (1 + tanh y) / 2 = 1 / (1 + e^-2y), y = sqrt(2 / pi) (z + 0.044715 z^3)
#pragma unroll
        for (int e = 0; e < NC; ++e)
          v[e] = over_one_plus_exp(v[e], v[e] * fmaf(v[e] * v[e], 0.0713548163f, 1.59576912f));
        break;
      default: break;
    }
    if (GATED) {
#pragma unroll
      for (int e = 0; e < NC; ++e) v[e] *= u[e];
    }
    if (!CODES && R) {
      const uint16_t* r = R + row * ldr + col;
      if (WHOLE) {
#pragma unroll
        for (int h = 0; h < NC / 4; ++h) {
          const u32x2_t w = *reinterpret_cast<const u32x2_t*>(r + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[4 * h + e] += value(w[e >> 1] >> (16 * (e & 1)));
        }
      } else {
#pragma unroll 1
        for (int e = 0; e < NC; ++e) {
          if (col + e >= cols) break;
          const float b = value(r[e]);
#pragma unroll
          for (int f = 0; f < NC; ++f) v[f] += f == e ? b : 0.f;
        }
      }
    }
  }
  // Four columns' sums (the others' in b where gated) finished and stored.
  FS_DEVICE void four(const float4_t& a, const float4_t& b, int64_t row, int64_t col, int64_t cols) const {
    float v[4] = {a[0], a[1], a[2], a[3]}, u[4] = {b[0], b[1], b[2], b[3]};
    uint16_t* c = C + row * ldc + col;
    if (whole) {
      compute<true>(v, u, row, col, cols);
      *reinterpret_cast<u32x2_t*>(c) = u32x2_t{pair(v[0], v[1]), pair(v[2], v[3])};
    } else {
      compute<false>(v, u, row, col, cols);
      const uint32_t o[2] = {pair(v[0], v[1]), pair(v[2], v[3])};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < cols) c[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
    }
  }
  // Eight columns' sums finished and stored. For codes 16 lanes side by side hold a row's group (all in range, or none).
  template <bool WHOLE>
  FS_DEVICE void piece(float (&v)[8], float (&u)[8], int64_t row, int64_t col, int64_t cols) const {
    compute<WHOLE>(v, u, row, col, cols);
    if constexpr (CODES) {
      int e;
      *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint8_t*>(C) + row * ldc + col) = encode_eight(v, e);
      if ((col & (GROUP - 1)) == 0) {
        const int g = (int)(col / GROUP);
        uint8_t* word = scales + ((int64_t)(g >> 2) * rows + row) * 4;
        word[g & 3] = (uint8_t)e;
        if (col + GROUP >= cols)
          for (int b = (g & 3) + 1; b < 4; ++b) word[b] = 0;
      }
    } else {
      uint16_t* c = C + row * ldc + col;
      const u32x4 o = {pair(v[0], v[1]), pair(v[2], v[3]), pair(v[4], v[5]), pair(v[6], v[7])};
      if (WHOLE) {
        *reinterpret_cast<u32x4*>(c) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < cols) c[e] = (uint16_t)(o[e >> 1] >> (16 * (e & 1)));
      }
    }
  }
};

// The SPLITS sums in memory added in order and finished, eight columns of the results a thread (N % 4 == 0: rows of W); every
// load ahead of the first addition, for what it takes is their latency: 160 x 2048 of eight splits, 10 MB out of the caches, 4.1
// us, of four 3.8, the gate of 1 x 28672 4.0 (one load after another 160 x 2048 of eight took 1.6 us more).
template <class OUT, int SPLITS>
__global__ void __launch_bounds__(256) linear_e4m3_join_kernel(const float* __restrict__ part, int64_t M, int64_t N,
                                                               uint32_t pieces, OUT out) {
  constexpr int H = OUT::GATED ? 2 : 1;   // the gate's, the others'
  const int64_t cols = N / H;
  const uint32_t unit = blockIdx.x * 256u + threadIdx.x;   // (M * pieces < 2^31)
  const int64_t row = unit / pieces, col = 8 * (int64_t)(unit % pieces);
  if (row >= M) return;   // (by groups of 16 lanes where codes are written: pieces % 16 == 0)
  const float* p = part + row * N + col;
  const bool two = col + 4 < cols;   // (else the second four are those of the first, and nobody's)
  float4_t a[SPLITS][H][2];
#pragma unroll
  for (int s = 0; s < SPLITS; ++s)
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float* q = p + (int64_t)s * M * N + h * cols;
      a[s][h][0] = *reinterpret_cast<const float4_t*>(q);
      a[s][h][1] = *reinterpret_cast<const float4_t*>(q + (two ? 4 : 0));
    }
  __builtin_amdgcn_sched_barrier(0);
  float v[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[h][e] = a[0][h][e >> 2][e & 3];
#pragma unroll
      for (int s = 1; s < SPLITS; ++s) v[h][e] += a[s][h][e >> 2][e & 3];
    }
  if (out.whole) out.template piece<true>(v[0], v[H - 1], row, col, cols);
  else out.template piece<false>(v[0], v[H - 1], row, col, cols);
}

// ------------------------------------------------------------------------------------------------
// short batches: bound by the weight's bytes
// ------------------------------------------------------------------------------------------------
// A workgroup takes `per` rows of W (of a gated product `per` columns of the results: as many rows of each half), so many
// that the grid is one round of the CUs where it can be and each draws the same share; its eight waves split K and are joined
// in order through LDS. A tile is 16 rows of W, or eight columns' gate's rows and their others', so that any number of tiles
// may share a workgroup, and x's codes. A wave streams its part of K on its own, without a barrier: pieces of 16 rows x 128
// codes, in each stage x's TM and then W's TN, pass through the wave's SLOTS places in LDS, copied there by whole lines SLOTS
// pieces ahead: 16 KB a wave, 128 KB a CU on their way. With many rows a workgroup the waves take stages in turn, so that they
// read a row's next 1 KB together (1 x 28672 x 4096 gated 26.7 -> 25.6 us), and workgroups begin at different KB of their rows,
// an XCD's at all of them: rows of 4 KB read at the same KB by every CU draw from few of the memory's channels (1 x 28672 x
// 4096 24.1 -> 22.5, 1 x 128256 x 4096 98.2 -> 91.2). With few rows, eight parts of K, whose words of four stages' scales serve
// them all (1 x 2048 x 8192 7.1 -> 6.3 us).
//
// Straight to registers, in the instruction's own shape, a load runs at a quarter of the rate, 38 GB/s a CU from L2 for 150,
// for four lanes side by side are four rows: 8 x 6144 x 4096 took 8.6 us so and takes 7.3, 32 x 4096 x 4096 9.8 and 7.1. Now
// HBM bounds it: 1 x 28672 x 4096 in 20.8 us, 2.3 of them the launch, draws 6.4 TB/s, 1 x 128256 x 4096 6.5; smaller weights
// are on their way before the CUs' 128 KB each have come (4096 x 4096 in 6.6 us).
template <class OUT, int TM, int TN>
__global__ void __launch_bounds__(512) linear_e4m3_stream_kernel(Operands P, OUT out, int per, bool once) {
  constexpr int TILES = TM * TN, CH = TILES < 8 ? TILES : 8, COLS = OUT::GATED ? 8 : 16;
  constexpr int SLOTS = 8, PIECE = 16 * GROUP, PPS = TM + TN;   // pieces a stage
  constexpr int XQ = (16 * TM + 63) / 64, WQ = (16 * TN + 63) / 64, WORDS = 64 * (XQ + WQ);   // a stage's words: x's rows, W's
  constexpr bool TURNS = TN >= 4;
  // Places for words: of the stages that SLOTS pieces reach ahead, or of fours of them, four ahead at most.
  constexpr int PLACES = TURNS && (PPS - 1 + SLOTS) / PPS > 1 ? 4 : 2;
  static_assert(PPS >= 2 && (!TURNS || (PPS - 1 + SLOTS) / PPS < PLACES), "words stay until they are used");
  __shared__ __attribute__((aligned(1024))) char ring[8][SLOTS * PIECE];
  __shared__ __attribute__((aligned(256))) uint32_t words[8][PLACES][WORDS];
  static_assert(sizeof(ring) >= 8 * CH * 64 * sizeof(float4_t), "the sums take the ring's place");
  typedef __attribute__((address_space(3))) const u32x4 LdsFrag;
  const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t cols = OUT::GATED ? P.N / 2 : P.N, c0 = (int64_t)blockIdx.x * per, c1 = min(c0 + per, cols);
  // the wave's stages: w, w + 8, ..., or the w-th eighth
  const int k0 = TURNS ? w : (int)((int64_t)w * P.nk / 8);
  const int ni = TURNS ? (P.nk - w + 7) / 8 : (int)((int64_t)(w + 1) * P.nk / 8) - k0;
  const int rot = TURNS && ni > 0 ? (int)(blockIdx.x / 8 % (unsigned)ni) : 0;   // (workgroups go round the 8 XCDs)
  auto stage_of = [&](int i) { return TURNS ? w + 8 * (i + rot < ni ? i + rot : i + rot - ni) : k0 + i; };
  auto has_words = [&](int i) { return TURNS || i == 0 || (stage_of(i) & 3) == 0; };
  auto place_of = [&](int i) { return (TURNS ? i : stage_of(i) >> 2) & (PLACES - 1); };
  const int M = (int)P.M;

  // copies: 8 rows of 128 bytes each; lane l takes row l >> 3, physical chunk l & 7 of it (swap_of)
  const uint32_t slots = (uint32_t)(uintptr_t)ring[w], words0 = (uint32_t)(uintptr_t)words[w];
  const char* xbase = reinterpret_cast<const char*>(P.x);
  const char* wbase[2];
  uint32_t xoff[TM][2], woff[TN][2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = 8 * h + (lane >> 3), c = 16 * ((lane & 7) ^ swap_of(row));
#pragma unroll
    for (int i = 0; i < TM; ++i) xoff[i][h] = (uint32_t)(min(16 * i + row, M - 1) * P.ldx + c);   // (rows past the last: nobody's)
#pragma unroll
    for (int j = 0; j < TN; ++j)
      woff[j][h] = (uint32_t)((min(c0 + COLS * j + (OUT::GATED ? row & 7 : row), c1 - 1) - c0) * P.ldw + c);
    wbase[h] = reinterpret_cast<const char*>(P.w + (c0 + (OUT::GATED && h ? cols : 0)) * P.ldw);
  }
  uint32_t wword[WQ];
#pragma unroll
  for (int q = 0; q < WQ; ++q) {
    const int r = min(64 * q + lane, 16 * TN - 1);
    const int64_t c = min(c0 + COLS * (r >> 4) + (OUT::GATED ? r & 7 : r & 15), c1 - 1);
    wword[q] = (uint32_t)(4 * (OUT::GATED && (r & 8) ? c + cols : c));
  }
  uint32_t xword[XQ];
#pragma unroll
  for (int q = 0; q < XQ; ++q) xword[q] = (uint32_t)(4 * min(64 * q + lane, M - 1));
  int slot = 0;   // of the stage's first piece
  // piece t of the wave's stage i into place (slot + at) % SLOTS; ahead of a stage's first, its words
  auto copy = [&](int i, int t, int at) {
    const int64_t k = stage_of(i);
    const uint32_t to = slots + (uint32_t)(((slot + at) & (SLOTS - 1)) * PIECE);
    if (t == 0 && has_words(i)) {
      const uint32_t wto = words0 + (uint32_t)(place_of(i) * WORDS * 4);
#pragma unroll
      for (int q = 0; q < XQ; ++q) dma4_at(P.xs + (k >> 2) * 4 * M, xword[q], wto + 256 * q);
#pragma unroll
      for (int q = 0; q < WQ; ++q) dma4_at(P.ws + (k >> 2) * 4 * P.N, wword[q], wto + 256 * (XQ + q));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (t < TM) dma16_at(xbase + k * GROUP, xoff[t < TM ? t : 0][h], to + 1024 * h);
      else if (once) dma16_once_at(wbase[h] + k * GROUP, woff[t < TM ? 0 : t - TM][h], to + 1024 * h);
      else dma16_at(wbase[h] + k * GROUP, woff[t < TM ? 0 : t - TM][h], to + 1024 * h);
    }
  };
  const uint32_t at0 = (uint32_t)(l16 * GROUP + 16 * (g ^ swap_of(l16))), at1 = (uint32_t)(l16 * GROUP + 16 * ((4 + g) ^ swap_of(l16)));
  // piece t of stage i from its place, once it has landed (SLOTS - 1 pieces may be behind it), and the next into it
  auto take = [&](int i, int t) {
    if (i + (t + SLOTS - 1) / PPS < ni) wait_vm<2 * (SLOTS - 1)>();
    else wait_vm<0>();
    const uint32_t from = slots + (uint32_t)(((slot + t) & (SLOTS - 1)) * PIECE);
    const i32x8 f = both_chunks(*(LdsFrag*)(uintptr_t)(from + at0), *(LdsFrag*)(uintptr_t)(from + at1));
    if (i + (t + SLOTS) / PPS < ni) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      copy(i + (t + SLOTS) / PPS, (t + SLOTS) % PPS, t + SLOTS);
    }
    return f;
  };
#pragma unroll
  for (int t = 0; t < SLOTS; ++t)
    if (t / PPS < ni) copy(t / PPS, t % PPS, t);
  float4_t acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
  uint32_t xs[TM], ws[TN];
  for (int i = 0; i < ni; ++i) {
    i32x8 xf[TM];
#pragma unroll
    for (int r = 0; r < TM; ++r) xf[r] = take(i, r);
    if (has_words(i)) {   // (landed before x's first piece)
      const uint32_t* p = words[w][place_of(i)];
      const int shift = 8 * (stage_of(i) & 3);
#pragma unroll
      for (int r = 0; r < TM; ++r) xs[r] = p[16 * r + l16] >> shift;
#pragma unroll
      for (int j = 0; j < TN; ++j) ws[j] = p[64 * XQ + 16 * j + l16] >> shift;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const i32x8 wf = take(i, TM + j);
#pragma unroll
      for (int r = 0; r < TM; ++r) acc[r * TN + j] = mfma_codes<0>(wf, xf[r], acc[r * TN + j], ws[j], xs[r]);
    }
    if (!TURNS) {
#pragma unroll
      for (int r = 0; r < TM; ++r) xs[r] >>= 8;
#pragma unroll
      for (int j = 0; j < TN; ++j) ws[j] >>= 8;
    }
    slot = (slot + PPS) & (SLOTS - 1);
  }
  __syncthreads();   // every wave has read its last pieces, and no copy is on its way
  float4_t(*red)[CH][64] = reinterpret_cast<float4_t(*)[CH][64]>(&ring[0][0]);
  // CH tiles at a time: wave t joins tile t's eight sums in order; lane (l16, g) has row l16, and of the tile's rows of W
  // (g = 0, 1 the gate's, 2, 3 the same columns' others) 4 g ..
#pragma unroll
  for (int first = 0; first < TILES; first += CH) {
    if (first) __syncthreads();
#pragma unroll
    for (int t = first; t < first + CH && t < TILES; ++t) red[w][t - first][lane] = acc[t];
    __syncthreads();
    const int t = first + w;
    if (w >= CH || t >= TILES) continue;
    float4_t a = red[0][w][lane], b = a;
    if (OUT::GATED) b = red[0][w][(lane + 32) & 63];
#pragma unroll
    for (int v = 1; v < 8; ++v) {
      const float4_t p = red[v][w][lane], q = OUT::GATED ? red[v][w][(lane + 32) & 63] : p;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        a[r] += p[r];
        b[r] += q[r];
      }
    }
    const int row = 16 * (t / TN) + l16;
    const int64_t col = c0 + COLS * (t % TN) + 4 * g;
    if (row >= M || col >= c1 || (OUT::GATED && g >= 2)) continue;
    if (!OUT::GATED && out.part) *reinterpret_cast<float4_t*>(out.part + row * P.N + col) = a;   // (N % 4 == 0)
    else out.four(a, b, row, col, cols);
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
struct Plan {
  int bm, bn, splits;
  bool join;     // the sums through memory
  bool stream;   // the streaming kernel: every wave its own part of K, no tile in LDS that waves share
};
int64_t weight_rows(const fs_linear& c) { return c.gated ? 2 * c.N : c.N; }

// Columns of the results that a workgroup of the streaming kernel takes, of `cols`: a multiple of eight, so many that the
// grid is one round of the 256 CUs, or the fewest rounds where that is more than seven tiles; and the tiles of its kernel.
int64_t stream_columns(int64_t cols, bool gated) {
  const int64_t most = 256 * (gated ? 56 : 112), rounds = (cols + most - 1) / most;
  return ((cols + 256 * rounds - 1) / (256 * rounds) + 7) / 8 * 8;
}
int stream_tiles(int64_t cols, bool gated) {
  const int64_t tiles = gated ? stream_columns(cols, true) / 8 : (stream_columns(cols, false) + 15) / 16;
  return tiles <= 2 ? (int)tiles : tiles <= 4 ? 4 : 7;
}

// Tiles: the cheapest of what a sweep over 26 shapes of 40 to 4000 rows fits (us; by 4 to 12 % rms, and its choice is within
// 1 % of the best one's time on average, 7 % at most): `first` for a grid, `round` for each further round of the CUs' places
// (two of the smaller tiles share a CU: stage2 for both), a stage of 128, and a MB of results or of sums in memory. Codes
// leave tiles of 128 columns by themselves, a gate's tiles of 256; other sums go through memory, as those of K splits do. Eight
// splits pay 1 us beside their bytes: of 19 shapes of 80 to 640 rows that this leaves with four, 16 are the faster for it (160 x
// 2048 x 8192 15.6 us for 17.5, 512 x 1024 x 8192 16.1 for 19.1, 129 x 1024 x 4096 9.5 for 10.2), three the slower by up to 3 % (200 x
// 6144 x 16384 43.8 for 42.6). Beyond the sweep's 4000 rows, and for many tiles below, the fit is off by up to a fifth (8005 x 28672 x
// 4096 863 us for 730, 2777 x 28672 x 4096 302 for 262, 8005 x 4096 x 4096 117 for 126, 2777 x 4096 x 14336 128 for 142); the largest
// tile is ahead of the next there by as much or more.
Plan plan_for(const fs_linear& c) {
  const int64_t M = c.M, N = weight_rows(c), nk = c.K / GROUP;
  const bool codes = c.out_scales != nullptr;
  if (M <= STREAM_ROWS) {
    const int rows = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int tiles = codes ? stream_tiles(N, false) : stream_tiles(c.N, c.gated != 0);
    if (rows <= 32 || (tiles <= 2 && rows * c.K <= STREAM_BYTES)) return Plan{rows, 16 * tiles, 1, codes, true};
  }
  struct Cand {
    int bm, bn;
    double first, round, stage, stage2, sums_mb, out_mb;   // stage2 0: one a CU
  };
  static const Cand cands[] = {{64, 64, 3.9, 0.6, 0.32, 0.46, 0.14, 0.26},   {64, 128, 3.9, 0.1, 0.46, 0.64, 0.18, 0.30},
                               {128, 128, 4.7, 2.6, 0.56, 0.0, 0.13, 0.31},  {256, 128, 5.2, 2.1, 0.85, 0.0, 0.18, 0.44},
                               {64, 256, 4.0, 2.6, 0.67, 0.0, 0.0, 0.23},    {128, 256, 5.5, 3.9, 0.86, 0.0, 0.0, 0.38},
                               {256, 256, 9.7, 16.7, 0.97, 0.0, 0.21, 0.44}};
  Plan best{64, 64, 1, codes, false};
  double least = 1e30;
  for (const Cand& t : cands) {
    if (t.bn == 256 && t.bm < 256 && !(codes && c.gated)) continue;   // (no other kernels of these)
    if (t.bm == 64 && t.bn == 128 && codes && c.gated) continue;
    const bool whole = !codes || t.bn == 256 || (t.bn == 128 && !c.gated);
    const int64_t tiles = ((M + t.bm - 1) / t.bm) * ((N + t.bn - 1) / t.bn);
    for (int s = 1; s <= 8; s *= 2) {
      // (a split starts at a whole word of scales; partials are stored four columns at a time)
      const bool join = s > 1 || !whole;
      if (s > 1 && (nk % (4 * s) != 0 || (t.bn == 256 && t.bm < 256))) break;
      if (join && (N % 4 != 0 || c.N % 4 != 0)) break;
      const int64_t wgs = tiles * s, places = t.stage2 > 0.0 ? 512 : 256, rest = wgs % places;
      const double one = t.stage2 > 0.0 ? (rest > 0 && rest <= 256) : (double)(wgs / places + (rest > 0));
      const double two = t.stage2 > 0.0 ? (double)(wgs / places + (rest > 256)) : 0.0;
      const double out_mb = (double)M * (double)N * 2e-6, sums_mb = 2.0 * s * out_mb;
      const double us = t.first + t.round * (one + two - 1.0) + (double)(nk / s) * (one * t.stage + two * t.stage2) +
                        (join ? t.sums_mb * sums_mb + (s == 8 ? 3.9 : 2.9) + 0.125 * sums_mb + 0.05 * out_mb : t.out_mb * out_mb);
      if (us < least) least = us, best = Plan{t.bm, t.bn, s, join, false};
    }
  }
  return best;
}

int64_t encoded_bytes(const fs_linear& c) { return c.x_scales ? 0 : align256(c.M * c.K) + align256(scale_bytes(c.M, c.K)); }
int64_t sums_bytes(const fs_linear& c, const Plan& p) {
  return p.join ? (int64_t)p.splits * c.M * weight_rows(c) * (int64_t)sizeof(float) : 0;
}

// The launchers: false, with nothing launched, of a plan that no kernel here takes.
template <class OUT, int TM>
bool launch_stream(const Operands& P, const OUT& out, int tn, int64_t per, hipStream_t s) {
  const int64_t cols = OUT::GATED ? P.N / 2 : P.N;
  if (P.M > 16 * TM || per > tn * (OUT::GATED ? 8 : 16)) return false;   // (rows or columns that nobody takes)
  const dim3 grid((unsigned)((cols + per - 1) / per));
  const bool once = P.N * P.nk * GROUP >= READ_ONCE;
  if (tn == 1) linear_e4m3_stream_kernel<OUT, TM, 1><<<grid, 512, 0, s>>>(P, out, (int)per, once);
  else if (tn == 2) linear_e4m3_stream_kernel<OUT, TM, 2><<<grid, 512, 0, s>>>(P, out, (int)per, once);
  else if constexpr (TM > 2) return false;
  else if (tn == 4) linear_e4m3_stream_kernel<OUT, TM, 4><<<grid, 512, 0, s>>>(P, out, (int)per, once);
  else if (tn == 7) linear_e4m3_stream_kernel<OUT, TM, 7><<<grid, 512, 0, s>>>(P, out, (int)per, once);
  else return false;
  return true;
}
template <class OUT>
bool launch_stream(const Operands& P, const OUT& out, const Plan& p, int64_t per, hipStream_t s) {
  const int tn = p.bn / 16;
  switch (p.splits == 1 ? p.bm : 0) {
    case 16: return launch_stream<OUT, 1>(P, out, tn, per, s);
    case 32: return launch_stream<OUT, 2>(P, out, tn, per, s);
    case 64: return launch_stream<OUT, 4>(P, out, tn, per, s);
    case 128: return launch_stream<OUT, 8>(P, out, tn, per, s);
    default: return false;
  }
}

// PARTS: a class of which only the sums in memory are asked for.
template <class OUT, bool PARTS>
bool launch_tiles(const Operands& P, const OUT& out, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(8 * ((P.ntiles + 7) / 8)), (unsigned)p.splits);
  const auto tile = [&](int bm, int bn) { return p.bm == bm && p.bn == bn; };
  if (p.stream || (!PARTS && p.splits != 1)) return false;
  if (tile(256, 256)) {
    gemm_e4m3_long_kernel<OUT, PARTS><<<grid, 512, 0, s>>>(P, out);
  } else if constexpr (OUT::CODES && OUT::GATED) {
    if (tile(128, 256)) gemm_e4m3_tile_kernel<OUT, 128, 256, 2, 4, 3><<<grid, 512, 0, s>>>(P, out);
    else if (tile(64, 256)) gemm_e4m3_tile_kernel<OUT, 64, 256, 1, 8, 3><<<grid, 512, 0, s>>>(P, out);
    else return false;
  } else {
    if (tile(256, 128)) gemm_e4m3_tile_kernel<OUT, 256, 128, 4, 2, 3><<<grid, 512, 0, s>>>(P, out);
    else if (tile(128, 128)) gemm_e4m3_tile_kernel<OUT, 128, 128, 2, 4, 4><<<grid, 512, 0, s>>>(P, out);
    else if (tile(64, 128)) gemm_e4m3_tile_kernel<OUT, 64, 128, 2, 2, 3><<<grid, 256, 0, s>>>(P, out);
    else if constexpr (OUT::CODES) return false;
    else if (tile(64, 64)) gemm_e4m3_tile_kernel<OUT, 64, 64, 2, 2, 4><<<grid, 256, 0, s>>>(P, out);
    else return false;
  }
  return true;
}

template <class OUT>
int run(const fs_linear& c, Operands P, const Plan& p, float* part, hipStream_t s) {
  OUT out;
  out.C = reinterpret_cast<uint16_t*>(c.out);
  out.ldc = c.ldo;
  out.R = reinterpret_cast<const uint16_t*>(c.residual);
  out.ldr = c.ldr;
  out.bias = c.bias;
  out.up = c.N;
  out.dtype = c.dtype;
  out.bias_dtype = c.bias_dtype;
  out.act = c.activation;
  out.whole = c.N % 8 == 0 && al16(c.out) && c.ldo % 8 == 0 && al16(c.residual) && c.ldr % 8 == 0 && al16(c.bias);
  out.scales = reinterpret_cast<uint8_t*>(c.out_scales);
  out.rows = c.M;
  out.part = nullptr;
  bool done = false;
  if (p.join) {
    typedef LinearOut<false, false> Sums;
    Sums sums{};
    sums.part = part;
    if (p.splits == 1 || p.splits == 2 || p.splits == 4 || p.splits == 8)   // (what the join takes)
      done = p.stream ? launch_stream(P, sums, p, stream_columns(P.N, false), s)   // (rows of W in their order, gated or not)
                      : launch_tiles<Sums, true>(P, sums, p, s);
  } else if constexpr (OUT::CODES) {
    done = launch_tiles<OUT, false>(P, out, p, s);   // (the others' codes go through memory)
  } else {
    done = p.stream ? launch_stream(P, out, p, stream_columns(c.N, c.gated != 0), s) : launch_tiles<OUT, false>(P, out, p, s);
  }
  FS_CHECK_ARG(done, "linear_e4m3: no kernel of %d x %d, %d splits, %d %d", p.bm, p.bn, p.splits, p.join, p.stream);
  if (p.join) {
    const uint32_t pieces = (uint32_t)((c.N + 7) / 8);
    const dim3 grid((unsigned)((c.M * pieces + 255) / 256));
    if (p.splits == 8) linear_e4m3_join_kernel<OUT, 8><<<grid, 256, 0, s>>>(part, P.M, P.N, pieces, out);
    else if (p.splits == 4) linear_e4m3_join_kernel<OUT, 4><<<grid, 256, 0, s>>>(part, P.M, P.N, pieces, out);
    else if (p.splits == 2) linear_e4m3_join_kernel<OUT, 2><<<grid, 256, 0, s>>>(part, P.M, P.N, pieces, out);
    else linear_e4m3_join_kernel<OUT, 1><<<grid, 256, 0, s>>>(part, P.M, P.N, pieces, out);
  }
  return fs::launch_status("linear_e4m3");
}

int linear(const fs_linear& c, const Plan& p, char* work, hipStream_t s) {
  const int64_t N = weight_rows(c);
  const uint8_t* x = reinterpret_cast<const uint8_t*>(c.x);
  const uint8_t* xs = reinterpret_cast<const uint8_t*>(c.x_scales);
  int64_t ldx = c.ldx;
  if (!xs) {
    uint8_t* codes = reinterpret_cast<uint8_t*>(work);
    uint8_t* words = codes + align256(c.M * c.K);
    fs::quantize_rows_e4m3(c.x, c.ldx, c.M, c.K, c.x_dtype, codes, c.K, reinterpret_cast<uint32_t*>(words), s);
    x = codes;
    xs = words;
    ldx = c.K;
  }
  Operands P{x, reinterpret_cast<const uint8_t*>(c.w), xs, reinterpret_cast<const uint8_t*>(c.w_scales), ldx, c.ldw, c.M, N,
             (int)(c.K / GROUP), (int)((c.M + p.bm - 1) / p.bm), 0};
  P.ntiles = P.tiles_m * (int)((N + p.bn - 1) / p.bn);
  float* part = reinterpret_cast<float*>(work + encoded_bytes(c));
  if (c.out_scales) return c.gated ? run<LinearOut<true, true>>(c, P, p, part, s) : run<LinearOut<false, true>>(c, P, p, part, s);
  return c.gated ? run<LinearOut<true, false>>(c, P, p, part, s) : run<LinearOut<false, false>>(c, P, p, part, s);
}

// What sizes are refused for; and the plan of the others.
int check(const fs_linear* c, const char* what, Plan& p) {
  FS_CHECK_ARG(c, "%s: null pointer", what);
  FS_CHECK_ARG(c->M >= 0 && c->N > 0 && c->K > 0 && c->K % GROUP == 0, "%s: M %lld N %lld K %lld (K a multiple of %d)", what,
               (long long)c->M, (long long)c->N, (long long)c->K, GROUP);
  // a copy's offset inside its tile of rows, and a row's scale word inside its group of K, are 32 bits
  FS_CHECK_ARG(c->K <= (1 << 22) && c->M < (1 << 29) && c->N < (1 << 28), "%s: M %lld N %lld K %lld", what, (long long)c->M,
               (long long)c->N, (long long)c->K);
  // below 2^32 threads a launch: 64 for a row's 512 columns that are encoded, 512 a tile, one for eight columns from memory
  FS_CHECK_ARG(c->x_scales || waves_fit(c->M * ((c->K + 511) / 512)), "%s: M %lld K %lld", what, (long long)c->M,
               (long long)c->K);
  FS_CHECK_ARG(!c->out_scales || c->N % GROUP == 0, "%s: codes of %lld columns (a multiple of %d)", what, (long long)c->N, GROUP);
  p = plan_for(*c);
  FS_CHECK_ARG((!p.join || c->M * ((c->N + 7) / 8) < 0x7fffff00LL) &&
                   (p.stream || ((c->M + p.bm - 1) / p.bm) * ((weight_rows(*c) + p.bn - 1) / p.bn) < (1 << 22)),
               "%s: M %lld N %lld", what, (long long)c->M, (long long)c->N);
  return 0;
}

}  // namespace

extern "C" int64_t fs_linear_e4m3_workspace_size(const fs_linear* c) {
  Plan p;
  return check(c, "linear_e4m3_workspace_size", p) ? 0 : encoded_bytes(*c) + sums_bytes(*c, p);
}

extern "C" int fs_linear_e4m3_plan(const fs_linear* c, int32_t* plan) {
  FS_CHECK_ARG(plan, "linear_e4m3_plan: null pointer");
  Plan p;
  if (int e = check(c, "linear_e4m3_plan", p)) return e;
  plan[0] = p.bm;
  plan[1] = p.bn;
  plan[2] = p.splits;
  plan[3] = p.join;
  return 0;
}

extern "C" int fs_linear_e4m3(const fs_linear* call, void* workspace, int64_t workspace_bytes, void* stream) {
  Plan p;
  if (int e = check(call, "linear_e4m3", p)) return e;
  const fs_linear& c = *call;
  FS_CHECK_ARG(c.x && c.w && c.w_scales && c.out, "linear_e4m3: null pointer");
  FS_CHECK_ARG(c.x_scales || c.x_dtype == FS_F32 || c.x_dtype == FS_BF16 || c.x_dtype == FS_F16, "linear_e4m3: rows of dtype %d",
               c.x_dtype);
  FS_CHECK_ARG(c.out_scales || c.dtype == FS_BF16 || c.dtype == FS_F16, "linear_e4m3: results are bf16, f16 or codes (dtype %d)",
               c.dtype);
  FS_CHECK_ARG(!c.bias || c.bias_dtype == FS_F32 || c.bias_dtype == FS_BF16 || c.bias_dtype == FS_F16,
               "linear_e4m3: bias of dtype %d", c.bias_dtype);
  FS_CHECK_ARG(c.activation >= FS_ACT_NONE && c.activation <= FS_ACT_GELU_TANH, "linear_e4m3: activation %d", c.activation);
  FS_CHECK_ARG(!c.residual || !c.out_scales, "linear_e4m3: no residual is added to codes");
  FS_CHECK_ARG(c.ldx >= c.K && c.ldw >= c.K && c.ldo >= c.N && (!c.residual || c.ldr >= c.N), "linear_e4m3: leading dimensions");
  FS_CHECK_ARG(c.ldw % 16 == 0 && al16(c.w) && (!c.x_scales || (c.ldx % 16 == 0 && al16(c.x))) &&
                   (!c.out_scales || (c.ldo % 16 == 0 && al16(c.out))),
               "linear_e4m3: codes need 16-byte aligned rows");
  FS_CHECK_ARG(((reinterpret_cast<uintptr_t>(c.w_scales) | reinterpret_cast<uintptr_t>(c.x_scales) |
                 reinterpret_cast<uintptr_t>(c.out_scales)) & 3) == 0,
               "linear_e4m3: scales need whole words");
  FS_CHECK_ARG(c.ldw < (1 << 23) && (!c.x_scales || c.ldx < (1 << 23)), "linear_e4m3: ldx %lld ldw %lld", (long long)c.ldx,
               (long long)c.ldw);
  if (c.M == 0) return 0;
  const int64_t need = encoded_bytes(c) + sums_bytes(c, p);
  FS_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0),
               "linear_e4m3: workspace %lld < %lld bytes (or not 256-byte aligned)", (long long)workspace_bytes, (long long)need);
  return linear(c, p, reinterpret_cast<char*>(workspace), fs::as_stream(stream));
}
