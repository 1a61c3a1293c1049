// The decode kernel for more than 32 rows a sequence: a pair of CTAs has a tile of 64 or 128 of them (part of mla_decode.cu).
//
// One CTA alone has room for two blocks of 64 keys beside 64 queries, and a block's chain of loads, products and softmax takes three times as
// long as its products.  A pair shares a block: CTA c has the rows [R c, R c + R) of the tile's 2 R and loads keys [32 c, 32 c + 32),
//
//   S   [2 R x 64 keys]       = Q K^T     cta_group::2, M = 128 (R = 32: half of it padding), N = 64: 36 steps
//   O^T [512 dims x 2 R]     += V^T P^T   cta_group::2, M = 256 twice, N = 2 R: CTA c has the dims [256 c, 256 c + 256)
//
// so a block takes 36 KB of each CTA, and four or five of them are in flight.  CTA c's value tile is its dims of all 64 keys: of its own
// keys it has them; those of the peer's keys are loaded, once the first product has read the tile, over the half of its own keys' latent
// that is the peer's dims.  Either way keys 0-31 then lie in chunks 0-3 and keys 32-63 in chunks 4-7.  P takes the place of the rope dims.
// Both products are issued in the leader (CTA 0).  S has keys 0-31 in lanes 0-63 and keys 32-63 in lanes 64-127, a row a lane.
//
// O's columns are the rows of both CTAs, so a rescaling is the business of both: each block they tell each other whether one of
// their rows needs it, which is hidden by the blocks in flight, and it is rare: P may be 2^32 above the running maximum (mla_prefill.cu).
#pragma once

namespace lt {
namespace decode {
namespace pair {

constexpr int kOwnKeys = 32;
constexpr uint32_t kChunk = kOwnKeys * 128;                 // 32 keys x 64 bf16
constexpr uint32_t kSlot = kChunks * kChunk;
constexpr int kWarpK = 11, kWarpV = 12, kLoad0 = 12;        // kTma: two warps; else K and V have half of the warps from kLoad0 each
template <Load kLoad> constexpr int kLoaders = kLoad == kTma ? 1 : kLoad == kCopy ? 8 : 16;
template <Load kLoad> constexpr int kPairThreads = 32 * (kLoad0 + kLoaders<kLoad>);
constexpr float kMostOver = 32.f;

template <int R>
struct PairPlan {
  static constexpr int kSlots = R == 64 ? 4 : 5;
  static constexpr uint32_t kQChunk = R * 128;
  static constexpr uint32_t kOffKV = 0;
  static constexpr uint32_t kOffQ = kOffKV + kSlots * kSlot;
  static constexpr uint32_t kOffP = kOffQ + kChunks * kQChunk;              // R = 64: keys 32-63 of P, two buffers; keys 0-31 fill the rope chunk
  static constexpr uint32_t kPHalf = R * kOwnKeys * 2;
  static constexpr uint32_t kOffMisc = kOffP + (R == 64 ? 2 * kPHalf : 4096);      // (R = 32: the 64 rows of the operand end in there)
  static constexpr uint32_t kSmem = kOffMisc + 3072;
  static constexpr uint32_t kTmemS = 4 * R;                 // O^T: two blocks of 2 R columns; then S, 32 columns a slot
  static constexpr uint32_t kTmemCols = 512;
  static_assert(kOffQ % 1024 == 0 && kSlot % 1024 == 0 && kOffP % 1024 == 0, "swizzled tiles");
  static_assert(kOffQ + (kChunks - 1) * kQChunk + 64 * 128 <= kOffMisc, "the operand ends inside");
  static_assert(kTmemS + 32 * kSlots <= kTmemCols, "tensor memory");
  static_assert(kSmem <= 232448, "shared memory");
};

struct PairMisc {
  // in the leader: what the products wait for, from both CTAs
  uint64_t k_full[5], v_full[5], p_ready[5], q_ready;
  // in each CTA
  uint64_t qk_done[5], slot_free[5], q_free, drained[2], vote[2], corr_full, fin_full;
  uint32_t vote_flag[2];
  uint32_t left, tmem_base;
  int start_b, start_k, count, meta_groups;
  long long start_pos, total;
  int scan[32];
  float top[4][64];                   // of a row's four threads: maxima, sums
  float corr[128], scale[128];        // of the tile's rows
};
static_assert(sizeof(PairMisc) <= 3072, "PairMisc");

__device__ __forceinline__ void arrive_expect_cluster(uint32_t addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(addr), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
// a wait for what the other CTA has written
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, const BlockWaiter& w, int site, int iter) {
  uint32_t since = 0, ok;
  for (;;) {
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendHintNs) : "memory");
    if (ok) return true;
    if (w.gives_up(since, site, iter)) return false;
  }
}
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void commit_pair(uint32_t addr) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(addr) : "memory");
}
// Four steps of a product, the operands da and db 16-byte units apart
template <int kDa, int kDb>
__device__ __forceinline__ void mma4_pair(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate_first) {
  asm volatile(
      "{\n\t.reg .pred pf, po;\n\t.reg .b32 a, b;\n\t.reg .b64 ad, bd;\n\tsetp.ne.b32 pf, %6, 0;\n\tsetp.eq.b32 po, 0, 0;\n\t"
      "mov.b64 ad, {%1, %2};\n\tmov.b64 bd, {%3, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, pf;\n\t"
      "add.u32 a, %1, %7;\n\tadd.u32 b, %3, %8;\n\tmov.b64 ad, {a, %2};\n\tmov.b64 bd, {b, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, po;\n\t"
      "add.u32 a, %1, 2 * %7;\n\tadd.u32 b, %3, 2 * %8;\n\tmov.b64 ad, {a, %2};\n\tmov.b64 bd, {b, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, po;\n\t"
      "add.u32 a, %1, 3 * %7;\n\tadd.u32 b, %3, 3 * %8;\n\tmov.b64 ad, {a, %2};\n\tmov.b64 bd, {b, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, po;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate_first), "n"(kDa), "n"(kDb) : "memory");
}
// two steps
template <int kDa, int kDb>
__device__ __forceinline__ void mma2_pair(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate_first) {
  asm volatile(
      "{\n\t.reg .pred pf, po;\n\t.reg .b32 a, b;\n\t.reg .b64 ad, bd;\n\tsetp.ne.b32 pf, %6, 0;\n\tsetp.eq.b32 po, 0, 0;\n\t"
      "mov.b64 ad, {%1, %2};\n\tmov.b64 bd, {%3, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, pf;\n\t"
      "add.u32 a, %1, %7;\n\tadd.u32 b, %3, %8;\n\tmov.b64 ad, {a, %2};\n\tmov.b64 bd, {b, %4};\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], ad, bd, %5, po;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate_first), "n"(kDa), "n"(kDb) : "memory");
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_but_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// a running block's slot and the parity of its barriers
template <int kSlots>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == kSlots) { slot = 0; phase ^= 1u; }
  }
};

template <int R, Load kLoad>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads<kLoad>, 1)
mla_decode_pair_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_q, const Params p) {
  using PL = PairPlan<R>;
  constexpr int kSlots = PL::kSlots, kTile = 2 * R;
  using Cursor = Ring<kSlots>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  // Swizzled tiles.  There is no room for rounding; the driver has put the base on such a boundary so far, in both CTAs alike.
  if ((sbase & 1023u) != 0) {
    pdl_wait();
    if (threadIdx.x == 0) Waiter{g_status, p.epoch, 0}.fail(kSiteAlign, (int)(sbase & 1023u));
    return;
  }
  PairMisc& ms = *reinterpret_cast<PairMisc*>(smem_raw + PL::kOffMisc);
  const BlockWaiter wt{&ms.left, p.wait_limit};
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank(), peer = cta ^ 1u;
  const int cluster = (int)blockIdx.x >> 1, g = cluster / p.row_tiles, rt = cluster - g * p.row_tiles;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 5; ++i) {
      // arrivals of both CTAs: a loader warp each with its bytes; the threads' own copies; the converting warps
      mbar_init(&ms.k_full[i], kLoad == kTma ? 2 : kLoaders<kLoad>);
      mbar_init(&ms.v_full[i], kLoad == kTma ? 2 : kLoaders<kLoad>);
      mbar_init(&ms.p_ready[i], 2 * kSoftmaxWarps);
      mbar_init(&ms.qk_done[i], 1);
      mbar_init(&ms.slot_free[i], 1);
    }
    mbar_init(&ms.q_ready, 2);
    mbar_init(&ms.q_free, 1);
    mbar_init(&ms.corr_full, 1);
    mbar_init(&ms.fin_full, 1);
    for (int i = 0; i < 2; ++i) { mbar_init(&ms.drained[i], 1); mbar_init(&ms.vote[i], 1); }
    ms.left = 0;
    ms.count = 0;
    fence_mbar_init();
    if (kLoad == kTma) tma_prefetch_desc(&map_kv);
    if (p.flat_q) tma_prefetch_desc(&map_q);
  }
  __syncthreads();
  cluster_sync_all();
  if (warp == kWarpQk) {
    tmem_alloc_pair(&ms.tmem_base, PL::kTmemCols);
    tmem_relinquish_pair();
  }
  pdl_wait();
  find_share(p, ms, g, warp, lane);
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem_base, 0);
  const int row0 = rt * kTile + R * (int)cta;               // this CTA's first row of the sequence's

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax, epilogue
    // Warp: TMEM lanes 32 (warp % 4), columns 16 (warp / 4).  Thread: row r, keys 32 h + 16 c + [0, 16).
    const int quarter = warp & 3, c = warp >> 2, tl = 32 * quarter + lane, r = tl & 63, h = tl >> 6;
    const bool live = (quarter & 1) * 32 < R;
    const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
    const uint32_t a_p_ready = mapa(smem_u32(&ms.p_ready[0]), 0);
    const uint32_t a_vote = mapa(smem_u32(&ms.vote[0]), peer), a_flag = mapa(smem_u32(&ms.vote_flag[0]), peer);
    Walk w(ms);
    Cursor at, prev, prev2;                                 // of blocks kb, kb - 1, kb - 2
    int kb = 0;
    uint32_t corrs = 0;                                     // rescalings so far
    // A wait here that gives up is passed like any other: the warps meet at named barriers, so they take the same steps.
    bool more = w.next(p);
    while (more) {
      const int row = row0 + r;
      const int lim = min(w.len, w.len - p.q_len + 1 + row / p.heads), low = w.len - p.q_len + 1 + row0 / p.heads;     // low: what this CTA's first row sees
      float m = kMInit, l = 0.f;
      for (int k = w.k0; k < w.k1; ++k, ++kb) {
        mbar_wait(&ms.qk_done[at.slot], at.phase, wt, kSiteS, kb);
        __syncwarp();
        tc_fence_after();
        float v[16];
        float mx = -INFINITY;
        if (live) {
          tmem_ld16(tmem + PL::kTmemS + 32 * at.slot + 16 * c + lane_base, v);
          tmem_wait_ld();
          if ((k + 1) * kBlock > low) {
            const int seen = lim - k * kBlock - 32 * h - 16 * c;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = e < seen ? v[e] * p.scale_log2 : -INFINITY;
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] *= p.scale_log2;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, v[e]);
        }
        const bool first = k == w.k0;
        const bool mine = softmax_any(mx > m + kMostOver);
        // whether one of the pair's rows needs it
        if (threadIdx.x == 0) {
          st_cluster_u32(a_flag + 4u * (kb & 1), mine ? 1u : 0u);
          mbar_arrive_cluster_release(a_vote + 8u * (kb & 1));
        }
        wait_cluster(&ms.vote[kb & 1], (kb >> 1) & 1, wt, kSiteVote, kb);
        // (put to the vote among the threads once more: a wait that gave up must not part them)
        if (softmax_any(first || mine || *reinterpret_cast<volatile uint32_t*>(&ms.vote_flag[kb & 1]) != 0)) {
          if (live) ms.top[2 * c + h][r] = mx;
          softmax_sync();
          float f = 1.f;
          if (live) {
            const float now = fmaxf(m, fmaxf(fmaxf(ms.top[0][r], ms.top[1][r]), fmaxf(ms.top[2][r], ms.top[3][r])));
            f = fast_exp2(m - now);
            m = now;
            l *= f;
          }
          if (!first) {
            // the factors of all of the tile's rows, in both CTAs
            if (live && h == 0 && c == 0) {
              ms.corr[R * cta + r] = f;
              st_cluster_f32(mapa(smem_u32(&ms.corr[R * cta + r]), peer), f);
            }
            fence_cluster();
            softmax_sync();
            if (threadIdx.x == 0) mbar_arrive_cluster_release(mapa(smem_u32(&ms.corr_full), peer));
            wait_cluster(&ms.corr_full, corrs & 1, wt, kSiteVote, kb);
            ++corrs;
            mbar_wait(&ms.slot_free[prev.slot], prev.phase, wt, kSitePv, kb);
            __syncwarp();
            tc_fence_after();
#pragma unroll 1
            for (int x = kTile * c; x < kTile * (c + 1); x += 16) {
              float o[16];
              tmem_ld16(tmem + lane_base + x, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= ms.corr[(x & (kTile - 1)) + e];
              tmem_st16(tmem + lane_base + x, o);
            }
            tmem_wait_st();
          }
        }
        if (R == 64 && kb >= 2) {                           // this buffer's last P has been read
          mbar_wait(&ms.slot_free[prev2.slot], prev2.phase, wt, kSitePv, kb);
          __syncwarp();
        }
        if (live) {
          const uint32_t rope = sbase + PL::kOffKV + at.slot * kSlot + (kChunks - 1) * kChunk;
          const uint32_t ph = h == 0 ? rope : R == 64 ? sbase + PL::kOffP + (kb & 1) * PL::kPHalf : rope + PL::kPHalf;
          // 8 rows x 8 keys a matrix of 128 bytes: rows first, then keys
          const uint32_t to = ph + 2 * c * (R * 16) + r * 16;
          uint32_t u[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = fast_exp2(v[2 * e] - m), b = fast_exp2(v[2 * e + 1] - m);
            l += a + b;
            u[e] = bf16x2(a, b);
          }
          st_shared16(to, make_uint4(u[0], u[1], u[2], u[3]));
          st_shared16(to + R * 16, make_uint4(u[4], u[5], u[6], u[7]));
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(a_p_ready + 8u * at.slot);
        prev2 = prev; prev = at; at.advance();
      }
      // epilogue: this CTA's dims of all of the tile's rows
      softmax_sync();                                       // (the maxima have been read)
      if (live) ms.top[2 * c + h][r] = l;
      const bool whole = w.whole();
      const int slot = cluster * 2 + (w.index == 0 ? 0 : 1);
      softmax_sync();
      if (live && h == 0 && c == 0) {
        const float sum = ms.top[0][r] + ms.top[1][r] + ms.top[2][r] + ms.top[3][r], f = whole ? (sum > 0.f ? 1.f / sum : 0.f) : 1.f;
        ms.scale[R * cta + r] = f;
        st_cluster_f32(mapa(smem_u32(&ms.scale[R * cta + r]), peer), f);
        if (whole) {
          if (row < p.rows) p.lse[(long long)w.b * p.rows + row] = sum > 0.f ? (m + __log2f(sum)) * kLn2 : INFINITY;
        } else {
          p.part_ml[(long long)slot * kTile + R * cta + r] = make_float2(m, sum);
        }
      }
      fence_cluster();
      softmax_sync();
      if (threadIdx.x == 0) mbar_arrive_cluster_release(mapa(smem_u32(&ms.fin_full), peer));
      wait_cluster(&ms.fin_full, w.index & 1, wt, kSiteVote, kb);
      mbar_wait(&ms.slot_free[prev.slot], prev.phase, wt, kSitePv, kb);
      __syncwarp();
      tc_fence_after();
      const int rows = min(kTile, p.rows - rt * kTile), d = 256 * (int)cta + 128 * c + 32 * quarter + lane;
      float o[2][16];
      tmem_ld16(tmem + lane_base + kTile * c, o[0]);
#pragma unroll 1
      for (int x0 = 0; x0 < kTile; x0 += 32) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {                       // (the next columns come while these are written)
          const int x = x0 + 16 * y;
          tmem_wait_ld();
          if (x + 16 < kTile) tmem_ld16(tmem + lane_base + kTile * c + x + 16, o[y ^ 1]);
          if (whole) {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + ((long long)w.b * p.rows + rt * kTile + x) * kDV + d;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (x + e < rows) {
                const float f = ms.scale[x + e];
                dst[e * kDV] = __float2bfloat16(f > 0.f ? o[y][e] * f : 0.f);      // a row without keys: 0, whatever the values of others
              }
          } else {
            float* dst = p.part_o + ((long long)slot * kTile + x) * kDV + d;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (x + e < rows) dst[e * kDV] = o[y][e];
          }
        }
      }
      tc_fence_before();
      more = w.next(p);
    }
  } else if (warp == kWarpQk) {
    // ------------------------------------------------------------ S = Q K^T (the leader, one thread)
    // A slot's S is free with the slot: the second product of its last block was behind the softmax that read it.
    if (cta == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(1, 1, false, false, 128, kBlock);
      const uint64_t q_desc = umma_desc(sbase + PL::kOffQ, 16, 1024, kSwz128);
      const uint32_t hi = (uint32_t)(q_desc >> 32);
      const uint32_t a_done = smem_u32(&ms.qk_done[0]), a_done_peer = mapa(a_done, 1), a_q = smem_u32(&ms.q_free);
      Walk w(ms);
      Cursor at;
      int kb = 0;
      bool ok = true;
      while (ok && w.next(p)) {
        if (!(ok = mbar_wait(&ms.q_ready, w.index & 1, wt, kSiteQ, kb))) break;
        for (int k = w.k0; k < w.k1; ++k, ++kb) {
          if (!(ok = mbar_wait(&ms.k_full[at.slot], at.phase, wt, kSiteKv, kb))) break;
          if (kLoad != kTma) fence_proxy_async_smem();
          tc_fence_after();
          const uint32_t k_lo = (uint32_t)umma_desc(sbase + PL::kOffKV + at.slot * kSlot, 16, 1024, kSwz128);
#pragma unroll 1
          for (int j = 0; j < kChunks; ++j)
            mma4_pair<2, 2>(tmem + PL::kTmemS + 32 * at.slot, (uint32_t)q_desc + (PL::kQChunk >> 4) * j, hi, k_lo + (kChunk >> 4) * j, hi, idesc, (uint32_t)j);
          commit_pair(a_done + 8u * at.slot);
          commit_pair(a_done_peer + 8u * at.slot);
          at.advance();
        }
        if (ok) {
          commit_pair(a_q);
          commit_pair(mapa(a_q, 1));
        }
      }
      if (!ok) {                                            // given up: what has been issued ends before the tensor memory goes
        commit_pair(smem_u32(&ms.drained[0]));
        mbar_drain(&ms.drained[0], 0);
      }
    }
    __syncwarp();
  } else if (warp == kWarpPv) {
    // ------------------------------------------------------------ O^T += V^T P^T (the leader, one thread)
    if (cta == 0 && elect_one()) {
      constexpr uint32_t idesc = umma_idesc(1, 1, true, false, 256, kTile);
      const uint32_t a_free = smem_u32(&ms.slot_free[0]), a_free_peer = mapa(a_free, 1);
      Walk w(ms);
      Cursor at;
      int kb = 0;
      bool ok = true;
      while (ok && w.next(p))
        for (int k = w.k0; k < w.k1; ++k, ++kb) {
          if (!(ok = mbar_wait(&ms.v_full[at.slot], at.phase, wt, kSiteKv, kb) && mbar_wait(&ms.p_ready[at.slot], at.phase, wt, kSiteP, kb))) break;
          if (kLoad != kTma) fence_proxy_async_smem();
          tc_fence_after();
          const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot, rope = slot + (kChunks - 1) * kChunk;
          const uint64_t vd = umma_desc(slot, kChunk, 1024, kSwz128);               // dims along M: two chunks of 64, 8 keys 1024 bytes
          const uint64_t pd = umma_desc(rope, R * 16, 128, kSwzNone);
          const uint32_t p1 = R == 64 ? sbase + PL::kOffP + (kb & 1) * PL::kPHalf : rope + PL::kPHalf;
          const uint32_t v_lo = (uint32_t)vd, v_hi = (uint32_t)(vd >> 32), p_hi = (uint32_t)(pd >> 32), p1_lo = (uint32_t)umma_desc(p1, R * 16, 128, kSwzNone);
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            mma2_pair<128, 2 * R>(tmem + kTile * i, v_lo + (2 * kChunk >> 4) * i, v_hi, (uint32_t)pd, p_hi, idesc, k == w.k0 ? 0u : 1u);
            mma2_pair<128, 2 * R>(tmem + kTile * i, v_lo + (4 * kChunk >> 4) + (2 * kChunk >> 4) * i, v_hi, p1_lo, p_hi, idesc, 1u);
          }
          commit_pair(a_free + 8u * at.slot);
          commit_pair(a_free_peer + 8u * at.slot);
          at.advance();
        }
      if (!ok) {
        commit_pair(smem_u32(&ms.drained[1]));
        mbar_drain(&ms.drained[1], 0);
      }
    }
    __syncwarp();
  } else if (warp == kWarpQ) {
    // ------------------------------------------------------------ this CTA's queries of the next piece, when the last product with these is complete
    const uint32_t a_ready = mapa(smem_u32(&ms.q_ready), 0);
    Walk w(ms);
    const uint64_t pol = l2_policy_evict_first();
    bool ok = true;
    int asked = 0;
    while (w.next(p)) {
      if (w.index > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&ms.q_free, (w.index - 1) & 1, wt, kSiteQ, w.index)))) break;
      if (p.flat_q) {
        if (lane == 0) arrive_expect_cluster(a_ready, kChunks * PL::kQChunk);
        __syncwarp();
        if (lane < kChunks) tma_load_3d_pair_hint(sbase + PL::kOffQ + lane * PL::kQChunk, &map_q, 64 * lane, row0, w.b, a_ready, pol);
      } else {
        for (int r = 0; r < R; ++r) {
          const int row = row0 + r, j = row / p.heads, h = row - j * p.heads;
          const bool in = row < p.rows;
          const uint8_t* src = p.q + (in ? w.b * p.q_b + j * p.q_j + h * p.q_h : 0);
          for (int c = lane; c < kD / 8; c += 32)
            cp_async16_or_zero(sbase + PL::kOffQ + (uint32_t)(c >> 3) * PL::kQChunk + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (in ? 16 * c : 0), in);
        }
        cp_async_wait_all();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(a_ready);
      }
      ++asked;
    }
    if (!ok && asked > 0 && lane == 0 && cta == 0) mbar_drain(&ms.q_ready, (asked - 1) & 1);        // given up: what is in flight lands first
    __syncwarp();
  } else if (kLoad == kTma ? warp <= kWarpV : warp >= kLoad0) {
    // ------------------------------------------------------------ keys (own 32, all dims) and values (the peer's 32, own 256 dims)
    // kTma: a warp each, chunks of 32 rows of a page.  Else a warp has some adjacent rows (of a page: pages are multiples of 16 rows).
    constexpr int kHalfWarps = kLoad == kTma ? 1 : kLoaders<kLoad> / 2, kRowsOwn = kOwnKeys / kHalfWarps;
    constexpr int kRowBytes = kLoad == kPacked ? kPackedRow : 2 * kD;
    const bool is_v = kLoad == kTma ? warp == kWarpV : warp - kLoad0 >= kHalfWarps;
    const int part = kLoad == kTma ? 0 : (warp - kLoad0) % kHalfWarps, first_row = kRowsOwn * part;      // of the 32
    const int half = is_v ? (int)peer : (int)cta;                                    // whose keys
    const uint32_t a_full = mapa(smem_u32(is_v ? &ms.v_full[0] : &ms.k_full[0]), 0);
    uint64_t* const waits = is_v ? ms.qk_done : ms.slot_free;
    const uint32_t chunk0 = is_v ? (cta == 0 ? 4 : 0) : 0;                           // where its first chunk goes
    const int dim0 = is_v ? 256 * (int)cta : 0;
    struct Coming { int page, row, n; };                                             // n of the warp's rows hold keys
    Walk w(ms);
    const int count = ms.count;
    int k_at = 0, looked = 0;
    if (w.next(p)) k_at = w.k0;
    auto look = [&]() -> Coming {
      Coming x{-1, 0, 0};
      if (looked >= count) return x;
      const int key = k_at * kBlock + kOwnKeys * half + first_row;
      x.n = min(max(w.len - key, 0), kRowsOwn);
      if (x.n > 0) x.page = __ldcg(p.table + w.b * p.table_pitch + key / p.block_size);
      x.row = key % p.block_size;
      ++looked;
      if (++k_at == w.k1 && w.next(p)) k_at = w.k0;
      return x;
    };
    auto rows_of = [&](const Coming& x) -> const uint8_t* {
      return (unsigned)x.page < (unsigned)p.n_blocks ? p.cache + (long long)x.page * p.block_pitch + (long long)x.row * kRowBytes : nullptr;
    };
    auto to_l2 = [&](const Coming& x) {                     // (the other rows are the peer's to bring in)
      const uint8_t* src = rows_of(x);
      if (!is_v && src != nullptr && lane == 0) l2_prefetch_1d(src, (uint32_t)(x.n * kRowBytes));
    };
    // a slot is free (K) or its keys have been read (V)
    auto free_for = [&](const Cursor& at, int kb) -> bool {
      if (is_v) return mbar_wait(&waits[at.slot], at.phase, wt, kSiteFree, kb);
      return kb < kSlots || mbar_wait(&waits[at.slot], at.phase ^ 1u, wt, kSiteFree, kb);
    };
    // 16-byte pieces of rows first_row .. + kRowsOwn, zeros behind the keys
    auto copy_rows = [&](const Coming& x, uint32_t slot) {
      const uint8_t* src = rows_of(x);
      const int pieces = is_v ? 32 : kD / 8;
      for (int y = lane; y < kRowsOwn * pieces; y += 32) {
        const int r = y / pieces, c = y - r * pieces, row = first_row + r;
        const bool in = src != nullptr && r < x.n;
        cp_async16_or_zero(slot + (chunk0 + (c >> 3)) * kChunk + row * 128 + (((c & 7) ^ (row & 7)) << 4), in ? src + (long long)r * kRowBytes + 2 * dim0 + 16 * c : p.cache, in);
      }
    };
    Cursor at;
    bool ok = true;
    Coming c0 = look(), c1 = look(), c2 = look();
    if (kLoad != kPacked) {
      const uint64_t pol = l2_policy_evict_first();
      int asked = 0, pending = -1;                          // slot whose copies are under way (kCopy)
      auto announce = [&]() {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(a_full + 8u * pending);
        pending = -1;
      };
      if (kLoad == kCopy) { to_l2(c0); to_l2(c1); }
      for (int kb = 0; kb < count; ++kb) {
        const Coming c3 = look();
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
        if ((looked + rt) % p.row_tiles == 0) to_l2(c2);
        // a block's copies land while the next one's are issued, unless there is nothing to issue yet
        const bool idle = is_v ? !mbar_test(&waits[at.slot], at.phase) : kb >= kSlots && !mbar_test(&waits[at.slot], at.phase ^ 1u);
        if (pending >= 0 && __any_sync(0xffffffffu, idle)) { cp_async_wait_all(); announce(); }
        if (!(ok = __all_sync(0xffffffffu, free_for(at, kb)))) break;
        const int chunks = is_v ? 4 : kChunks;
        if (kLoad == kTma && c0.n == kOwnKeys) {
          if (lane == 0) arrive_expect_cluster(a_full + 8u * at.slot, chunks * kChunk);
          __syncwarp();
          if (lane < chunks)
            tma_load_3d_pair_hint(slot + (chunk0 + lane) * kChunk, &map_kv, dim0 + 64 * lane, c0.row, (unsigned)c0.page < (unsigned)p.n_blocks ? c0.page : p.n_blocks,
                                  a_full + 8u * at.slot, pol);
          asked = kb + 1;
        } else {
          copy_rows(c0, slot);                              // (kTma: the rows at a sequence's end, and none)
          cp_async_commit();
          if (pending >= 0) { cp_async_wait_but_one(); announce(); }
          pending = at.slot;
          if (kLoad == kTma) { cp_async_wait_all(); announce(); }
        }
        at.advance();
        c0 = c1; c1 = c2; c2 = c3;
      }
      cp_async_wait_all();
      if (pending >= 0) announce();
      if (!ok && asked > 0) __nanosleep(100000);            // given up: what is in flight lands first (some microseconds; its barrier is the leader's)
    } else if (!is_v) {
      // Of each 128 dims eight lanes have 16 codes of a row each, four rows at a time.  A group's registers are loaded for the next
      // block as soon as they are converted for this one, from L2, where the rows were brought a block before.
      const int sub = lane >> 3, c = lane & 7, row = first_row + sub;
      static_assert(kLoad != kPacked || kRowsOwn == 4, "a row a lane group");
      uint4 codes[4], rope;
      float4 scale;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      auto load = [&](const uint8_t* src, int n) {
        const bool in = src != nullptr && sub < n;
        const uint8_t* from = src + sub * kRowBytes;
        scale = in ? __ldcg(reinterpret_cast<const float4*>(from + 512)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) codes[j] = in ? __ldcg(reinterpret_cast<const uint4*>(from + 128 * j) + c) : zero;
        rope = in ? __ldcg(reinterpret_cast<const uint4*>(from + 528) + c) : zero;
      };
      to_l2(c0);
      to_l2(c1);
      load(rows_of(c0), c0.n);
      for (int kb = 0; ok && kb < count; ++kb) {
        const Coming c3 = look();
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
        if ((looked + rt) % p.row_tiles == 0) to_l2(c2);
        if (!(ok = __all_sync(0xffffffffu, free_for(at, kb)))) break;
        const float f[4] = {scale.x, scale.y, scale.z, scale.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 a, b;
          convert16(codes[j], f[j], a, b);
          // lanes of odd chunks write their second half first: the eight lanes of a phase then cover all banks
          const uint32_t base = slot + (2 * j + (c >> 2)) * kChunk + row * 128, u = 2 * (c & 3), odd = c >> 2;
          st_shared16(base + (((u + odd) ^ (row & 7)) << 4), odd ? b : a);
          st_shared16(base + (((u + 1 - odd) ^ (row & 7)) << 4), odd ? a : b);
        }
        st_shared16(slot + (kChunks - 1) * kChunk + row * 128 + ((c ^ (row & 7)) << 4), rope);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(a_full + 8u * at.slot);
        load(rows_of(c1), c1.n);
        at.advance();
        c0 = c1; c1 = c2; c2 = c3;
      }
    } else {
      // the peer's rows: 16 lanes a row, 16 codes each of this CTA's 256 dims
      const int sub = lane >> 4, c = lane & 15;
      uint4 codes[2];
      float scale[2];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      auto load = [&](const uint8_t* src, int n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool in = src != nullptr && sub + 2 * i < n;
          const uint8_t* from = src + (sub + 2 * i) * kRowBytes;
          codes[i] = in ? __ldcg(reinterpret_cast<const uint4*>(from + dim0) + c) : zero;
          scale[i] = in ? __ldcg(reinterpret_cast<const float*>(from + 512) + dim0 / 128 + (c >> 3)) : 0.f;
        }
      };
      load(rows_of(c0), c0.n);
      for (int kb = 0; ok && kb < count; ++kb) {
        const Coming c3 = look();
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
        if (!(ok = __all_sync(0xffffffffu, free_for(at, kb)))) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = first_row + sub + 2 * i;
          uint4 a, b;
          convert16(codes[i], scale[i], a, b);
          const uint32_t base = slot + (chunk0 + (c >> 2)) * kChunk + row * 128, u = 2 * (c & 3), odd = (c >> 2) & 1;
          st_shared16(base + (((u + odd) ^ (row & 7)) << 4), odd ? b : a);
          st_shared16(base + (((u + 1 - odd) ^ (row & 7)) << 4), odd ? a : b);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_release(a_full + 8u * at.slot);
        load(rows_of(c1), c1.n);
        at.advance();
        c0 = c1; c1 = c2; c2 = c3;
      }
    }
  }

  if (warp == kWarpQk && rt == 0 && cta == 0 && lane == 0 && p.meta) write_meta(p, ms, g);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();                                       // nothing of this CTA is in use by the other
  tc_fence_after();
  if (warp == kWarpQk) tmem_dealloc_pair(tmem, PL::kTmemCols);
  if (threadIdx.x == 0) {
    wt.report(g_status, p.epoch);
    if (blockIdx.x == 0) atomicAdd(&g_status[3], 1);
  }
}

// pairs that can run at once
template <int R, Load kLoad>
static int pairs() {
  static thread_local int cached_dev = -1, cached = 0;
  const int dev = current_device();
  if (dev == cached_dev) return cached;
  int n = sm_count() / 2, q = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sm_count()); cfg.blockDim = dim3(kPairThreads<kLoad>); cfg.dynamicSmemBytes = PairPlan<R>::kSmem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  if (ensure_smem<mla_decode_pair_kernel<R, kLoad>>(dev, PairPlan<R>::kSmem) &&
      cudaOccupancyMaxActiveClusters(&q, mla_decode_pair_kernel<R, kLoad>, &cfg) == cudaSuccess && q > 0)
    n = q;
  cudaGetLastError();
  cached_dev = dev; cached = n;
  return n;
}
template <int R, Load kLoad>
static int launch(const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  if (!ensure_smem<mla_decode_pair_kernel<R, kLoad>>(current_device(), PairPlan<R>::kSmem)) return LITEDSA_ERR_CUDA;
  return launch_pdl(mla_decode_pair_kernel<R, kLoad>, dim3((unsigned)(2 * p.groups * p.row_tiles)), kPairThreads<kLoad>, PairPlan<R>::kSmem, st, map, map_q, p);
}
template <int R>
static int launch(Load l, const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  return l == kTma ? pair::launch<R, kTma>(map, map_q, p, st) : l == kCopy ? pair::launch<R, kCopy>(map, map_q, p, st) : pair::launch<R, kPacked>(map, map_q, p, st);
}

}  // namespace pair
}  // namespace decode
}  // namespace lt
