// Products of two matrices of e4m3 codes (rows_e4m3.h): the kernels, for whatever finishes their results (Out).
#pragma once

#include "rows_e4m3.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
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

// What finishes results, a class of which a kernel gets an instance:
//   GATED          a tile's columns are half gate's (rows 0 .. N/2 - 1 of W), half the others' (N/2 .. N - 1), and the
//                  results have N/2 columns
//   STAGED         a finished tile's sums go through LDS as floats, eight columns a thread: out.piece<WHOLE>(v, up, row,
//                  col, cols), WHOLE being out.whole; else from the registers, rounded first
//   finish(a, row, col0, cols)   four columns' sums, from col0 on, to what is rounded and stored (`cols`: how many there
//                  are), and store(a, row, col0, cols) that
//   part           not null: the f32 sums as they are, [split][M][N], instead
template <int DT_>
struct ResidualOut {   // round(a (+ R))
  static constexpr int DT = DT_;
  static constexpr bool GATED = false, STAGED = false;
  uint16_t* C;
  int64_t ldc;
  const uint16_t* R;
  int64_t ldr;
  bool vec;
  float* part;
  FS_DEVICE void finish(float4_t& a, int64_t row, int64_t col0, int64_t cols) const {
    if (!R) return;
    if (vec && col0 + 4 <= cols) {
      const u32x2_t r = *reinterpret_cast<const u32x2_t*>(R + row * ldr + col0);
#pragma unroll
      for (int e = 0; e < 4; ++e) a[e] += half_of<DT>(r[e >> 1], e & 1);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col0 + e < cols) a[e] += Elem<DT>::to_f32(R[row * ldr + col0 + e]);
    }
  }
  FS_DEVICE void store(const float4_t& a, int64_t row, int64_t col0, int64_t cols) const {
    store_row4<DT>(a, C + row * ldc, col0, cols, vec);
  }
};

// Four columns' sums finished and stored.
template <class OUT>
FS_DEVICE void put4(const OUT& out, float4_t a, int64_t row, int64_t col0, int64_t cols) {
  if (col0 >= cols) return;
  out.finish(a, row, col0, cols);
  out.store(a, row, col0, cols);
}

// A finished tile of ROWS x COLS sums in LDS, PITCH floats a row (where gated the gate's columns, then the others'):
// finished by all of the workgroup's THREADS, eight columns of the results at a time, row by row.
template <class OUT, bool WHOLE, int ROWS, int COLS, int PITCH, int THREADS>
FS_DEVICE void finish_pieces(const OUT& out, const float* sums, int tid, int64_t m0, int64_t M, int64_t c0, int64_t cols) {
  constexpr int OC = OUT::GATED ? COLS / 2 : COLS, PIECES = OC / 8;
  static_assert(ROWS * PIECES % 64 == 0 && PITCH % 4 == 0, "whole waves");
#pragma unroll 1
  for (int u = tid; u < ROWS * PIECES; u += THREADS) {
    const int r = u / PIECES, p = u % PIECES;
    float v[8], up[8];
    const float* at = sums + r * PITCH + 8 * p;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4_t a = *reinterpret_cast<const float4_t*>(at + 4 * h);
      const float4_t b = OUT::GATED ? *reinterpret_cast<const float4_t*>(at + OC + 4 * h) : a;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = a[e], up[4 * h + e] = b[e];
    }
    if (m0 + r < M && c0 + 8 * p < cols) out.template piece<WHOLE>(v, up, m0 + r, c0 + 8 * p, cols);
  }
}
template <class OUT, int ROWS, int COLS, int PITCH, int THREADS>
FS_DEVICE void finish_tile(const OUT& out, const float* sums, int tid, int64_t m0, int64_t M, int64_t c0, int64_t cols) {
  if (out.whole) finish_pieces<OUT, true, ROWS, COLS, PITCH, THREADS>(out, sums, tid, m0, M, c0, cols);
  else finish_pieces<OUT, false, ROWS, COLS, PITCH, THREADS>(out, sums, tid, m0, M, c0, cols);
}

// ------------------------------------------------------------------------------------------------
// up to 16 rows: one launch, bound by the weights' bytes
// ------------------------------------------------------------------------------------------------
// A workgroup takes 16 TN columns of C; its eight waves split K and are joined in order through LDS. Weights go straight
// from HBM to registers in the instruction's own shape (a lane's two 16-byte chunks of a row's 128; a wave's load covers
// whole lines), DEPTH stages ahead. While the first of them are on their way the workgroup encodes the rows into LDS,
// eight lanes to a group: M K bytes of codes (XB at most, which bounds the rows) and a byte per
// row and group.
template <class OUT, int TN, int DEPTH, int XB>
__global__ void __launch_bounds__(512) gemm_e4m3_short_kernel(const uint16_t* __restrict__ X, int64_t ldx,
                                                              const uint8_t* __restrict__ W, int64_t ldw,
                                                              const uint8_t* __restrict__ wsc, OUT out, int M, int64_t N,
                                                              int nk) {
  constexpr int DT = OUT::DT;
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
  if (l16 < M) put4(out, a, l16, n0 + 16 * w + 4 * g, N);
}

// ------------------------------------------------------------------------------------------------
// LDS-fed tiles
// ------------------------------------------------------------------------------------------------
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Copies straight into LDS, 16 or 4 bytes a lane at a wave-uniform base plus the lane's offset; lane l lands at
// lds + 16 l (4 l). Counted by vmcnt; the waits are explicit. once: of what no other workgroup reads, past the caches.
// (s_nop: a copy may read m0 one wait state behind its writing, and inside the asm the compiler puts none.)
FS_DEVICE void dma16_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
FS_DEVICE void dma16_once_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
FS_DEVICE void dma4_at(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
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
template <class OUT, int BM, int BN, int WGM, int WGN, int NS>
__global__ void __launch_bounds__(64 * WGM * WGN) gemm_e4m3_tile_kernel(Operands P, OUT out) {
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
    if (OUT::GATED && !in_x) {   // (a copy's eight rows are of one tile of 16, the gate's or the others')
      const int wr = 8 * q - BM;
      const int64_t at = n0 / 2 + 16 * (wr >> 5) + (wr & 8), lead = min(at, P.N / 2 - 1);
      base[i] = reinterpret_cast<const char*>(P.w + (lead + (wr & 16 ? P.N / 2 : 0)) * P.ldw);
      off[i] = (uint32_t)((min(at + cr, P.N / 2 - 1) - lead) * P.ldw + 16 * c);
      continue;
    }
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
    int64_t r = min(lead + (in_x ? 64 * wave : 64 * wave - BM) + lane, rows - 1);
    if (OUT::GATED && !in_x) {
      const int wr = 64 * wave - BM + lane;
      r = min(n0 / 2 + 16 * (wr >> 5) + (wr & 15), P.N / 2 - 1) + (wr & 16 ? P.N / 2 : 0);
    }
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
  if constexpr (OUT::STAGED) {
    if (!out.part) {
      constexpr int PITCH = BN + 4;
      static_assert(sizeof(smem) >= BM * PITCH * sizeof(float), "the sums take the ring's place");
      static_assert(!OUT::GATED || TN % 2 == 0, "a gate's tile and its other's in one wave");
      float* sums = reinterpret_cast<float*>(smem);
      __syncthreads();   // every wave has read its last operands, and no copy is on its way
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int col = OUT::GATED ? (j & 1) * (BN / 2) + wn * (BN / WGN / 2) + 16 * (j >> 1) : wn * (BN / WGN) + 16 * j;
          *reinterpret_cast<float4_t*>(sums + (wm * (BM / WGM) + 16 * i + l16) * PITCH + col + 4 * g) = acc[i][j];
        }
      __syncthreads();
      finish_tile<OUT, BM, BN, PITCH, 64 * NW>(out, sums, threadIdx.x, m0, P.M, OUT::GATED ? n0 / 2 : n0,
                                               OUT::GATED ? P.N / 2 : P.N);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = m0 + wm * (BM / WGM) + 16 * i + l16;
    if (row >= P.M) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int64_t col0 = n0 + wn * (BN / WGN) + 16 * j + 4 * g;
      if (out.part) {   // (N % 4 == 0; never of a gated class)
        if (col0 < P.N) *reinterpret_cast<float4_t*>(out.part + ((int64_t)split * P.M + row) * P.N + col0) = acc[i][j];
      } else if constexpr (!OUT::STAGED) {
        put4(out, acc[i][j], row, col0, P.N);
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
template <class OUT, bool PARTIAL>
__global__ void __launch_bounds__(512, 2) gemm_e4m3_long_kernel(Operands P, OUT to) {
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
    if (OUT::GATED)   // of a wave's 64 columns 32 are the gate's, copied by waves 0..3, 32 the others'
      wo[i] = (uint32_t)((min(n0 / 2 + 32 * i + (crow & 31) + cr, P.N / 2 - 1) - n0 / 2) * P.ldw + 16 * cc);
  }
  const int split = blockIdx.y, nk = P.nk / (int)gridDim.y, first = split * nk;   // (nk % 4 == 0 where K is split)
  const char* xb = reinterpret_cast<const char*>(P.x + m0 * P.ldx + (int64_t)first * GROUP);
  const int64_t wlead = OUT::GATED ? n0 / 2 + (wave >> 2 ? P.N / 2 : 0) : n0;
  const char* wb = reinterpret_cast<const char*>(P.w + wlead * P.ldw + (int64_t)first * GROUP);
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
  int64_t srow = min((wm ? n0 : m0) + 64 * (wave & 3) + lane, srows - 1);
  if (OUT::GATED && wm) srow = min(n0 / 2 + 32 * (wave & 3) + (lane & 31), P.N / 2 - 1) + (lane >> 5 ? P.N / 2 : 0);
  const uint32_t so = (uint32_t)(4 * srow);
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
      float* prow = to.part + ((int64_t)split * P.M + row) * P.N;
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
  if constexpr (OUT::STAGED) {   // 128 rows at a time, each wave's own 64 columns of them
    constexpr int FP = 256 + 4;
    static_assert(SMEM >= 128 * FP * (int)sizeof(float), "the sums take the ring's place");
    float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      __syncthreads();   // every wave has read its last operands (the rows before), and no copy is on its way
      if (wm == h) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t)
              *reinterpret_cast<float4_t*>(sums + (32 * i + l32) * FP + (OUT::GATED ? 128 * j + 32 * wn : 64 * wn + 32 * j) + 8 * t +
                                           4 * half) = four(i, j, t);
      }
      __syncthreads();
      finish_tile<OUT, 128, 256, FP, 512>(to, sums, threadIdx.x, m0 + 128 * h, P.M, OUT::GATED ? n0 / 2 : n0,
                                          OUT::GATED ? P.N / 2 : P.N);
    }
    return;
  }
  if constexpr (!OUT::STAGED) {
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
          if (row < P.M) to.finish(a, row, col0, P.N);
          *reinterpret_cast<u32x2_t*>(out + (32 * i + l32) * PITCH + 2 * (32 * j + 8 * t + 4 * half)) =
              u32x2_t{(uint32_t)Elem<OUT::DT>::store_bits(a[0]) | ((uint32_t)Elem<OUT::DT>::store_bits(a[1]) << 16),
                      (uint32_t)Elem<OUT::DT>::store_bits(a[2]) | ((uint32_t)Elem<OUT::DT>::store_bits(a[3]) << 16)};
        }
    }
    const int64_t col = n0 + wn * 64 + 8 * (lane & 7);
    uint16_t* C = to.C;
    const int64_t ldc = to.ldc;
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
}

}  // namespace
