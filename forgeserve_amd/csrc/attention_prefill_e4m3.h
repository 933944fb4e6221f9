// The prefill kernel over a pool of e4m3 codes (attention.hip includes this file behind its own prefill kernel, whose
// split of the work, ring order and folds it shares).

namespace {

// The four bytes of nan_codes as four bits.
FS_DEVICE uint32_t code_bits(uint32_t n) { return (n >> 7 & 1u) | (n >> 14 & 2u) | (n >> 21 & 4u) | (n >> 28 & 8u); }

// pair_step over operands without NaN (the workgroup's conversion zeroes such values and says which they were): the
// products run without a branch. nan: some value of the stage was NaN; then nans(mt) has a bit for each of the lane's
// eight values of dims 16 mt .., and a product of two indicators (which values are NaN, which keys a row sees) says
// which sums it belongs to.
template <int DT, int D, class Value, class Nans, class Scales>
FS_DEVICE void pair_step_clean(const float4_t (&sc)[2][2], Value value, bool nan, Nans nans, Scales scales, int j0,
                               const bool (&ok)[2], bool fresh, const int (&rpos)[2], int rmin, float scale,
                               float4_t (&acc)[D / 16][2], float (&m_run)[2], float (&l_run)[2]) {
  constexpr int MT = D / 16;
  typedef Operand<DT> O;
  const int g = (threadIdx.x & 63) >> 4;
  const bool full = ok[0] && ok[1] && j0 + 31 <= rmin;   // wave-uniform
  // the row sees the lane's keys e <= last_key(u, row's position)
  auto last_key = [&](int u, int pos) { return (ok[u] ? pos : -1) - j0 - 16 * u - 4 * g; };
  float s[2][2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][nt][e] = sc[u][nt][e];
  if (!full) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int last = last_key(u, rpos[nt]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] = e <= last ? s[u][nt][e] : -INFINITY;
      }
  }
  u32x4 pf[2];
  float alpha[2];
  const bool moved = pair_probs_e4m3<DT, true>(s, scales, scale, m_run, l_run, alpha, pf);
  if (moved && !fresh) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
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
  if (!full) {   // a probability is 0 where its key is hidden, whatever the scale there
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) pf[nt] &= seen_bits(rpos[nt]);
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      acc[mt + i][0] = O::mfma(now[i], pf[0], acc[mt + i][0]);
      acc[mt + i][1] = O::mfma(now[i], pf[1], acc[mt + i][1]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  if (nan) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const u32x4 seen = seen_bits(rpos[nt]) & O::ONES;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t bits = nans(mt);
        u32x4 bad;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          bad[c] = ((bits >> (2 * c) & 1u ? 0xffffu : 0u) | (bits >> (2 * c + 1) & 1u ? 0xffff0000u : 0u)) & O::ONES;
        const float4_t n = O::mfma(bad, seen, float4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[mt][nt][e] = n[e] > 0.f ? __uint_as_float(0x7fc00000u) : acc[mt][nt][e];
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// prefill kernel: attn_prefill_kernel's split, order and folds over codes
// ------------------------------------------------------------------------------------------------
// The ring carries the codes (half the bytes, PF_TILES tiles a stage), and the workgroup turns each stage into operands
// once, for its 256 query rows, where each wave doing so for itself would convert every tile eight times: a stage's
// conversion is 16 bytes of keys twice and of values twice per thread, against 240 vector instructions a pair and wave
// for the softmax. The operands lie in LDS in the order that the products read them: k-step ks of a tile's keys and the
// pair's values of dims 16 mt .. are 1 KB each, lane after lane. Two stages of codes are on their way while one is
// multiplied; the one buffer of operands costs a second barrier a stage.
//
// No unit is full: vector instructions take 58% of the SIMDs' time, products 26% of the matrix cores', and a wave waits for
// 36% of its own, at two waves per SIMD (238 registers at 128 dims). Measured (us): prompts of 4096, 2811, 2196 and 1829
// tokens, 32/8 heads of 128: 442 (610 TFLOP/s), f16 447, where the 16-bit pool's kernel, which converts nothing, takes
// 410; of 64 dims: 322, 317 and 283. Raising the waves' priority in their products, keys read a tile ahead, values read
// before the softmax: each within 1%. Stages of 4 tiles with two buffers of operands, so that one stage is converted
// beside the products of another behind one barrier: 7% more at 128 dims, 13% at 64.
template <int DT, int D, int BSZ>
__global__ void __launch_bounds__(64 * PF_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
attn_prefill_e4m3_kernel(AttnParams P) {
  constexpr int KS = D / 32, MT = D / 16;
  constexpr int TK = 16 * D;                        // bytes of a tile's key codes (and of its values')
  constexpr int TB = 2 * TK;                        // a tile's codes in LDS: keys, then values
  constexpr int CPT = TB / 1024;                    // 1 KB copies per tile
  constexpr int CPW = PF_TILES * CPT / PF_WAVES;    // copies of codes per wave per stage; one of scales comes on top
  constexpr int STAGE = PF_TILES * TB;
  constexpr int NS = 2;                             // stages of codes
  constexpr int THREADS = 64 * PF_WAVES;
  static_assert(PF_WAVES % CPT == 0 && CPW >= 1, "every wave copies the same part of its tiles");
  __shared__ __attribute__((aligned(1024))) char ring[NS * STAGE];
  __shared__ __attribute__((aligned(1024))) char kop[PF_TILES * 2 * TK];   // operands: keys by tile
  __shared__ __attribute__((aligned(1024))) char vop[PF_TILES * 2 * TK];   // values by pair
  __shared__ __attribute__((aligned(256))) uint32_t sring[NS][64];         // a stage's scale bytes: 32 per tile
  __shared__ __attribute__((aligned(16))) float vscale[PF_TILES][16];      // the values' scales of the operands' stage
  __shared__ uint32_t vnan[PF_TILES / 2][MT / 4][64];   // a bit for each value of the operands' stage that was NaN
  __shared__ int nan_stage;                         // the last stage that had one (+ 1)
  __shared__ int tbl[MAX_SPLIT / 16 + 1];           // the chunk's physical blocks (-1: unmapped)

  const int nkv = P.kv.n_kv_heads;
  const int64_t e_idx = blockIdx.x / nkv;
  const int hkv = (int)(blockIdx.x - e_idx * nkv);
  if (e_idx >= P.n_items[0]) return;   // uniform over the workgroup
  typedef __attribute__((address_space(4))) const AttnItem ConstItem;
  ConstItem* ep = (ConstItem*)(uintptr_t)(P.items + e_idx);
  const int b = ep->b, zb = ep->z, s = ep->s, qmax_item = ep->qmax;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int BS = BSZ ? BSZ : P.kv.block_size;
  const int kbeg = s * P.split;
  const int kend = min(kbeg + P.split, qmax_item + 1);
  const int ntiles = max((kend - kbeg + 15) >> 4, 0);
  const int npairs = (ntiles + 1) >> 1;
  const int nst = (2 * npairs + PF_TILES - 1) / PF_TILES;

  // this wave's query tile: the unit kernel's tile z, with its rows, positions and furthest query
  const int z = zb * PF_WAVES + w;
  const int row0 = z * QTILE;
  const int nrows = min(QTILE, P.T * P.G - row0);   // <= 0: a wave past the last tile (copies and converts only)
  const int* posb = P.pos + (int64_t)b * P.T;
  int rpos[2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int r = 16 * nt + l16;
    rpos[nt] = (r < nrows) ? posb[(row0 + r) / P.G] : -1;
  }
  const int qmax = nrows > 0 ? tile_qmax(P, b, z) : -1;
  const int rmin = rows_min_seen(rpos, nrows);
  const int ntiles_w = nrows > 0 ? min(max((min(kbeg + P.split, qmax + 1) - kbeg + 15) >> 4, 0), ntiles) : 0;

  u32x4 qf[2][KS];
  load_queries_e4m3<DT, D, 2>(P, b, hkv, row0, nrows, qf);

  // the chunk's table entries
  const int blk0 = kbeg / BS;
  const int nblk = ntiles > 0 ? (kbeg + 16 * ntiles - 1) / BS - blk0 + 1 : 0;
  int unmapped = 0;
  if (tid == 0) nan_stage = 0;
  for (int i = tid; i < nblk; i += THREADS) {
    const int blk = blk0 + i;
    int v = blk < P.max_blocks ? P.table[(int64_t)b * P.table_stride + blk] : -1;
    v = (v >= 0 && v < P.kv.num_blocks) ? v : -1;
    unmapped |= v < 0;
    tbl[i] = v;
  }
  // every load above has landed (the copies below are counted by the explicit waits only)
  __builtin_amdgcn_s_waitcnt(0);
  const bool all_mapped = !__syncthreads_or(unmapped);   // (the common case: no lookups per tile)

  // This wave copies part p = w % CPT of every tile it copies (keys for p < CPT/2, else values), 16 bytes a lane in the
  // pool's order: of the keys chunk c * 16 + slot (16 dims of a slot), of the values whole 4-key groups.
  const int p = w % CPT;
  const bool kpart = p < CPT / 2;
  const char* pool_h = reinterpret_cast<const char*>(kpart ? key_tile(P.kv, 0, hkv) : value_tile(P.kv, 0, hkv));
  const char* pool_s = reinterpret_cast<const char*>(tile_scales(P.kv, 0, hkv));
  const int64_t blk_stride = kpart ? P.kv.k_block : P.kv.v_block;
  const int slot_mul = kpart ? 16 : D;
  const uint32_t ring0 = (uint32_t)(uintptr_t)ring, sring0 = (uint32_t)(uintptr_t)sring;

  // The copies of the next stage, k: lane j finds the byte offsets of the stage's tile j / 8 (codes relative to pool_h,
  // scales to pool_s); a position behind the last pair copies some tile again. All of it comes from a thread index that
  // the compiler takes for new each time, here and in convert(): kept over the stages the addresses would need registers,
  // and spilled ones are waited for together with the copies.
  int copied = 0;   // the pair copied next
  auto issue = [&](int k) {
    int lane = threadIdx.x;
    asm volatile("" : "+v"(lane));
    lane &= 63;
    int pair = copied;
#pragma unroll
    for (int i = 1; i < PF_TILES / 2; ++i) {
      copied = pf_next_pair(copied, npairs);
      pair = lane >> 4 >= i ? copied : pair;
    }
    copied = pf_next_pair(copied, npairs);
    const int t = min(2 * pair + (lane >> 3 & 1), ntiles - 1);
    const int key0 = kbeg + 16 * t;
    const int bi = key0 / BS;
    const int ph = tbl[bi - blk0];
    const int64_t pb = ph >= 0 ? ph : 0;         // unmapped: block 0, masked in the step
    const int slot0 = key0 - bi * BS;
    const uint64_t o = (uint64_t)(pb * blk_stride + slot0 * slot_mul);
    const int ch = (kpart ? p : p - CPT / 2) * 64 + lane;
    const uint32_t coff = kpart ? (uint32_t)((ch >> 4) * 16 * BS + (ch & 15) * 16) : (uint32_t)(16 * ch);
    const uint32_t base = ring0 + (uint32_t)((k % NS) * STAGE) + (uint32_t)(p * 1024);
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      const int u = (w + PF_WAVES * i) / CPT;   // the stage's tile this copy fills
      const uint64_t ou = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(o >> 32), 8 * u) << 32) |
                          (uint32_t)__builtin_amdgcn_readlane((int)o, 8 * u);
      pf_dma16(pool_h + ou, coff, base + (uint32_t)(u * TB));
    }
    // the stage's scales, 8 words a tile (four of the keys, four of the values): every wave copies them, to the same
    // place, so that all of them count the same copies
    const int word = lane & 7;
    pf_dma4(pool_s + pb * P.kv.k_slot + slot0 + (word < 4 ? 4 * word : BS + 4 * (word - 4)), sring0 + (uint32_t)((k % NS) * 256));
  };
  static_assert(THREADS % D == 0, "");
  static_assert(PF_TILES == 8, "a stage's scales are one word a lane");

  // one stage's codes into operands
  auto convert = [&](int k) {
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const char* raw = ring + (k % NS) * STAGE;
    const uint32_t* sc = sring[k % NS];
    const uint8_t* sb = reinterpret_cast<const uint8_t*>(sc);
    if (tid < PF_TILES * 16) vscale[tid >> 4][tid & 15] = scale_value(sb[32 * (tid >> 4) + 16 + (tid & 15)]);
#pragma unroll
    for (int i = 0; i < PF_TILES * D / THREADS; ++i) {   // keys: chunk x = c * 16 + slot of tile u
      const uint32_t u = i * (THREADS / D) + tid / D, x = tid % D, c = x >> 4, slot = x & 15;
      const u32x4 q = *reinterpret_cast<const u32x4*>(raw + u * TB + 16 * x);
      const float sk = scale_value(sb[32 * u + slot]);
      char* to = kop + u * 2 * TK + (2 * (c >> 2) * 64 + (c & 3) * 16 + slot) * 16;   // k-step 2 (c / 4), then the next
      *reinterpret_cast<u32x4*>(to) = operand8<DT>(q[0], q[1], sk);
      *reinterpret_cast<u32x4*>(to + 1024) = operand8<DT>(q[2], q[3], sk);
    }
#pragma unroll
    for (int i = 0; i < (PF_TILES / 2 * D + THREADS - 1) / THREADS; ++i) {   // values: place x of both tiles of a pair
      const uint32_t pr = i * (THREADS / D) + tid / D, x = tid % D;
      if (PF_TILES / 2 * D % THREADS && pr >= PF_TILES / 2) break;
      const uint32_t gk = x / (D / 4), y = x % (D / 4), q = y >> 4, r = y & 15;   // 4-key group, 64 dims, dim % 16
      u32x4 a = *reinterpret_cast<const u32x4*>(raw + (2 * pr) * TB + TK + 16 * x);
      u32x4 c = *reinterpret_cast<const u32x4*>(raw + (2 * pr + 1) * TB + TK + 16 * x);
      uint32_t bits = 0, found = 0;
#pragma unroll
      for (int m = 0; m < 4; ++m) found |= nan_codes(a[m]) | nan_codes(c[m]);
      if (found) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const uint32_t na = nan_codes(a[m]), nc = nan_codes(c[m]);
          bits |= (code_bits(na) | code_bits(nc) << 4) << (8 * m);
          a[m] &= ~((na >> 7) * 255u);
          c[m] &= ~((nc >> 7) * 255u);
        }
        nan_stage = k + 1;   // (by any number of threads)
      }
      vnan[pr][q][gk * 16 + r] = bits;
      u32x4 vso = {};
      if (DT == FS_F16) {   // (a slot that was never written may hold any byte: what stands there must stay finite)
        float sa[4], sd[4];
        four_scales(sc[8 * (2 * pr) + 4 + gk], sa);
        four_scales(sc[8 * (2 * pr + 1) + 4 + gk], sd);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sa[e] = fminf(sa[e], scale_value(ScaleRange<FS_F16>::HI));
          sd[e] = fminf(sd[e], scale_value(ScaleRange<FS_F16>::HI));
        }
        vso = scale_operand(sa, sd);
      }
      char* to = vop + pr * 4 * TK + (4 * q * 64 + gk * 16 + r) * 16;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const u32x4 o = operand8<DT>(a[m], c[m], 1.f);
        *reinterpret_cast<u32x4*>(to + 1024 * m) = DT == FS_F16 ? times8(o, vso) : o;
      }
    }
  };

  float4_t acc[MT][2], O[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      acc[mt][nt] = float4_t{0.f, 0.f, 0.f, 0.f};
      O[mt][nt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  float Ms[2] = {-INFINITY, -INFINITY}, Ls[2] = {0.f, 0.f};
  // the finished partial of class v into the row state, then an empty partial for the next class
  auto fold = [&]() {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const float l = sum_across_groups(l_run[nt]);
      float Mn, cM, cm;
      if (fold_weights(Ms[nt], partial_reference(m_run[nt], l), Mn, cM, cm)) {
        Ls[nt] = fold_value(Ls[nt], cM, l, cm);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) O[mt][nt][c] = fold_value(O[mt][nt][c], cM, acc[mt][nt][c], cm);
        Ms[nt] = Mn;
      }
      m_run[nt] = -INFINITY;
      l_run[nt] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[mt][nt] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
  };

#pragma unroll
  for (int k = 0; k < NS; ++k)
    if (k < nst) issue(k);
  int next = 0;   // the pair consumed next
  bool fresh = true;   // acc is all zeros
  int cur_v = 0;
  const float scale = positive_scale(P.scale_log2);
  auto mapped = [&](int key0) { return all_mapped || tbl[key0 / BS - blk0] >= 0; };
  typedef __attribute__((address_space(3))) const u32x4 LdsOp;
  const uint32_t kad = (uint32_t)(uintptr_t)kop + 16 * lane, vad = (uint32_t)(uintptr_t)vop + 16 * lane;
  for (int k = 0; k < nst; ++k) {
    if (k + 1 < nst) pf_wait_vm<CPW + 1>();
    else pf_wait_vm<0>();
    __syncthreads();   // stage k has landed for every wave, and the operands of stage k-1 are no longer being read
    convert(k);
    __syncthreads();
    const bool nan = __builtin_amdgcn_readfirstlane(nan_stage) == k + 1;
    if (k + NS < nst) issue(k + NS);
#pragma unroll 1
    for (int u = 0; u < PF_TILES; u += 2) {
      if (k * (PF_TILES / 2) + u / 2 >= npairs) break;
      const int pair = next;
      next = pf_next_pair(next, npairs);
      if (nrows <= 0) continue;
      if ((pair & 7) != cur_v) {   // a new class: fold the last one into the row state
        fold();
        fresh = true;
        cur_v = pair & 7;
      }
      if (2 * pair >= ntiles_w) continue;   // wholly above every query of the wave
      auto value = [&](int mt) { return *(LdsOp*)(uintptr_t)(vad + (uint32_t)(u * 2 * TK + mt * 1024)); };
      float4_t sc[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 kf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[ks] = *(LdsOp*)(uintptr_t)(kad + (uint32_t)((u + h) * 2 * TK + ks * 1024));
        tile_scores_e4m3<DT, D, true>(kf, qf, sc[h]);
        __builtin_amdgcn_sched_barrier(0);   // (one tile's keys in registers)
      }
      auto scales = [&](int h, float (&vs)[4]) {
        const float4_t x = *reinterpret_cast<const float4_t*>(&vscale[u + h][4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) vs[e] = x[e];
      };
      const int key0 = kbeg + 32 * pair;
      const bool ok[2] = {mapped(key0), 2 * pair + 1 < ntiles && mapped(key0 + 16)};
      auto nans = [&](int mt) { return vnan[u >> 1][mt >> 2][lane] >> (8 * (mt & 3)); };
      pair_step_clean<DT, D>(sc, value, nan, nans, scales, key0, ok, fresh, rpos, rmin, scale, acc, m_run, l_run);
      fresh = false;
    }
  }
  if (nrows <= 0) return;
  fold();
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int r = 16 * nt + l16;
    if (r >= nrows) continue;
#pragma unroll
    for (int mt = 0; mt < MT; mt += 4)
      attn_emit<D, 4, DT | FS_STORE_E4M3>(P, b, s, kbeg, hkv, row0 + r, rpos[nt], mt, Ms[nt], Ls[nt],
                                          {O[mt][nt], O[mt + 1][nt], O[mt + 2][nt], O[mt + 3][nt]});
  }
}

}  // namespace
