// The prefill kernel over a pool of e4m3 codes (attention.hip includes this file behind its own prefill kernel, whose
// split of the work, ring order and folds it shares).

namespace {

// ------------------------------------------------------------------------------------------------
// prefill kernel: attn_prefill_kernel's split, order and folds over codes
// ------------------------------------------------------------------------------------------------
// The ring carries the codes (half the bytes, PF_TILES tiles a stage), and the workgroup turns each stage into operands
// once, for its 256 query rows, where each wave doing so for itself would convert every tile eight times: a stage's
// conversion is 16 bytes of keys twice and of values twice per thread, against 240 vector instructions a pair and wave
// for the softmax. The operands lie in LDS in the order that the products read them: k-step ks of a tile's keys and the
// pair's values of dims 16 mt .. are 1 KB each, lane after lane. Two stages of codes are on their way while one is
// multiplied; the one buffer of operands costs a second barrier a stage.
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
  const int rmin = rows_min_pos(rpos, nrows);
  const int ntiles_w = nrows > 0 ? min(max((min(kbeg + P.split, qmax + 1) - kbeg + 15) >> 4, 0), ntiles) : 0;

  u32x4 qf[2][KS];
  load_queries_e4m3<DT, D, 2>(P, b, hkv, row0, nrows, qf);

  // the chunk's table entries
  const int blk0 = kbeg / BS;
  const int nblk = ntiles > 0 ? (kbeg + 16 * ntiles - 1) / BS - blk0 + 1 : 0;
  int unmapped = 0;
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
  uint32_t coff;
  {
    const int ch = (kpart ? p : p - CPT / 2) * 64 + lane;
    coff = kpart ? (uint32_t)((ch >> 4) * 16 * BS + (ch & 15) * 16) : (uint32_t)(16 * ch);
  }
  const char* pool_h = reinterpret_cast<const char*>(kpart ? key_tile(P.kv, 0, hkv) : value_tile(P.kv, 0, hkv));
  const char* pool_s = reinterpret_cast<const char*>(tile_scales(P.kv, 0, hkv));
  const int64_t blk_stride = kpart ? P.kv.k_block : P.kv.v_block;
  const int slot_mul = kpart ? 16 : D;
  const uint32_t ring0 = (uint32_t)(uintptr_t)ring, sring0 = (uint32_t)(uintptr_t)sring;

  // Lane j holds the byte offsets of the tile at ring position 64 * win + j (codes relative to pool_h, scales to
  // pool_s), refreshed when a stage enters the next 64 positions; a position without a tile copies the last tile again.
  static_assert(64 % PF_TILES == 0, "a stage's positions lie in one 64-position window");
  uint32_t woff_lo = 0, woff_hi = 0, soff_lo = 0, soff_hi = 0;
  auto refresh = [&](int win) {
    const int j = min(64 * win + lane, 2 * npairs - 1);
    const int t = min(2 * pf_pair(j >> 1, npairs) + (j & 1), ntiles - 1);
    const int key0 = kbeg + 16 * t;
    const int bi = key0 / BS;
    const int ph = tbl[bi - blk0];
    const int64_t pb = ph >= 0 ? ph : 0;         // unmapped: block 0, masked in the step
    const int slot0 = key0 - bi * BS;
    const uint64_t o = (uint64_t)(pb * blk_stride + slot0 * slot_mul), os = (uint64_t)(pb * P.kv.k_slot + slot0);
    woff_lo = (uint32_t)o;
    woff_hi = (uint32_t)(o >> 32);
    soff_lo = (uint32_t)os;
    soff_hi = (uint32_t)(os >> 32);
  };
  auto issue = [&](int k) {
    if ((k & (64 / PF_TILES - 1)) == 0) refresh(k / (64 / PF_TILES));
    const uint32_t base = ring0 + (uint32_t)((k % NS) * STAGE) + (uint32_t)(p * 1024);
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      const int u = (w + PF_WAVES * i) / CPT;   // the stage's tile this copy fills
      const int j = (PF_TILES * k + u) & 63;
      const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)woff_hi, j) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)woff_lo, j);
      pf_dma16(pool_h + o, coff, base + (uint32_t)(u * TB));
    }
    // the stage's scales, 8 words a tile (four of the keys, four of the values): every wave copies them, to the same
    // place, so that all of them count the same copies
    const int j = (PF_TILES * k + (lane >> 3)) & 63, word = lane & 7;
    const uint64_t o = ((uint64_t)(uint32_t)__shfl((int)soff_hi, j, 64) << 32) | (uint32_t)__shfl((int)soff_lo, j, 64);
    pf_dma4(pool_s + o + (word < 4 ? 4 * word : BS + 4 * (word - 4)), sring0 + (uint32_t)((k % NS) * 256));
  };
  static_assert(PF_TILES == 8, "a stage's scales are one word a lane");

  // one stage's codes into operands (its addresses from a thread index that the compiler takes for new each time: kept
  // over the stages they would need registers, and spilled ones are waited for with the copies)
  auto convert = [&](int k) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const char* raw = ring + (k % NS) * STAGE;
    const uint32_t* sc = sring[k % NS];
    const uint8_t* sb = reinterpret_cast<const uint8_t*>(sc);
    if (tid < PF_TILES * 16) vscale[tid >> 4][tid & 15] = scale_value(sb[32 * (tid >> 4) + 16 + (tid & 15)]);
#pragma unroll
    for (int i = 0; i < PF_TILES * D / THREADS; ++i) {   // keys: chunk x = c * 16 + slot of tile u
      const int n = i * THREADS + tid, u = n / D, x = n % D, c = x >> 4, slot = x & 15;
      const u32x4 q = *reinterpret_cast<const u32x4*>(raw + u * TB + 16 * x);
      const float sk = scale_value(sb[32 * u + slot]);
      char* to = kop + u * 2 * TK + (2 * (c >> 2) * 64 + (c & 3) * 16 + slot) * 16;   // k-step 2 (c / 4), then the next
      *reinterpret_cast<u32x4*>(to) = operand8<DT>(q[0], q[1], sk);
      *reinterpret_cast<u32x4*>(to + 1024) = operand8<DT>(q[2], q[3], sk);
    }
#pragma unroll
    for (int i = 0; i < (PF_TILES / 2 * D + THREADS - 1) / THREADS; ++i) {   // values: place x of both tiles of a pair
      const int n = i * THREADS + tid, pr = n / D, x = n % D;
      if (PF_TILES / 2 * D % THREADS && n >= PF_TILES / 2 * D) break;
      const int gk = x / (D / 4), y = x % (D / 4), q = y >> 4, r = y & 15;   // 4-key group, 64 dims, dim % 16
      const u32x4 a = *reinterpret_cast<const u32x4*>(raw + (2 * pr) * TB + TK + 16 * x);
      const u32x4 c = *reinterpret_cast<const u32x4*>(raw + (2 * pr + 1) * TB + TK + 16 * x);
      u32x4 vso = {};
      if (DT == FS_F16) {
        float sa[4], sd[4];
        four_scales(sc[8 * (2 * pr) + 4 + gk], sa);
        four_scales(sc[8 * (2 * pr + 1) + 4 + gk], sd);
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
      pair_step_e4m3<DT, D, true>(sc, value, [] { asm volatile("" ::: "memory"); }, scales, key0, ok, fresh, qmax, rpos, rmin, scale, acc, m_run, l_run);
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
