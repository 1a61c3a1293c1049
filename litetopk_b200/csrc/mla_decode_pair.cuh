// The decode kernel for more than 64 rows a sequence: a pair of CTAs has a tile of 128 of them (part of mla_decode.cu).
//
// One CTA alone has room for two blocks of 64 keys beside 64 queries, and a block's chain of loads, products and softmax takes three times as
// long as its products.  A pair shares a block: CTA c has the rows [R c, R c + R) of the tile's 2 R and loads keys [32 c, 32 c + 32),
//
//   S   [2 R x 64 keys]       = Q K^T     cta_group::2, M = 128, N = 64: 36 steps
//   O^T [512 dims x 2 R]     += V^T P^T   cta_group::2, M = 256 twice, N = 2 R: CTA c has the dims [256 c, 256 c + 256)
//
// so a block takes 36 KB of each CTA, and four of them are in flight.  CTA c's value tile is its dims of all 64 keys: of its own
// keys it has them; those of the peer's keys are loaded, once the first product has read the tile, over the half of its own keys' latent
// that is the peer's dims.  Either way keys 0-31 then lie in chunks 0-3 and keys 32-63 in chunks 4-7.  P takes the place of the rope dims.
// Both products are issued in the leader (CTA 0).  S has keys 0-31 in lanes 0-63 and keys 32-63 in lanes 64-127, a row a lane.
//
// O's columns are the rows of both CTAs, so a rescaling is the business of both, and rare: P may be 2^32 above the running maximum
// (mla_prefill.cu).  A CTA whose rows need one has four warps of the other do their part and holds its P back until that is
// done; asking each other every block took 1600 cycles of it.
//
// Measured: 48 sequences of 1000 to 6001 keys, two tokens of 128 heads, bf16 in pages of 16, 100.5 us in a few calls (one CTA to 64 rows: 133), 120 at the
// power limit: a block a pair takes 1400 cycles, the tensor pipe is at 74 %; change of sequence 7000 cycles.  128 sequences of 2048 to 4096 packed keys, 128
// heads, 139.5 us (215), 165 at the power limit: 2600 cycles, which are the converting warps' instructions (their loads wait for nothing; the tensor pipe is at
// 57 %, the issue slots at 61 %).
#pragma once

namespace lt {
namespace decode {
namespace pair {

constexpr int kOwnKeys = 32;
constexpr uint32_t kMiscBytes = 3 * 1024;
constexpr uint32_t kChunk = kOwnKeys * 128;                 // 32 keys x 64 bf16
constexpr uint32_t kSlot = kChunks * kChunk;
// Warps 0-7: softmax; 8, 9: products; 10: queries.  kTma: 11 and 13 request keys (the issue of small boxes paces a warp), 12 values; kPacked:
// 11 brings keys into L2, 12-19 convert keys, 20-23 values.  The last four: the other CTA's rescalings.
constexpr int kWarpK0 = 11, kWarpV = 12, kWarpK1 = 13, kWarpBring = 11, kLoad0 = 12, kKeyWarps = 8, kValueWarps = 4;
template <Load kLoad> constexpr int kWarpAid = kLoad == kTma ? 16 : 24;
template <Load kLoad> constexpr int kPairThreads = 32 * (kWarpAid<kLoad> + 4);
constexpr float kMostOver = 32.f;
constexpr int R = 64;                                       // rows of a CTA

struct PL {
  static constexpr int kSlots = 4;
  static constexpr uint32_t kQChunk = R * 128;
  static constexpr uint32_t kOffKV = 0;
  static constexpr uint32_t kOffQ = kOffKV + kSlots * kSlot;
  static constexpr uint32_t kOffP = kOffQ + kChunks * kQChunk;              // keys 32-63 of P, two buffers; keys 0-31 fill the rope chunk
  static constexpr uint32_t kPHalf = R * kOwnKeys * 2;
  static constexpr uint32_t kOffMisc = kOffP + 2 * kPHalf;
  static constexpr uint32_t kSmem = kOffMisc + kMiscBytes;
  static constexpr uint32_t kTmemS = 4 * R;                 // O^T: two blocks of 2 R columns; then S, 32 columns a slot
  static constexpr uint32_t kTmemCols = 512;
  static_assert(kOffQ % 1024 == 0 && kSlot % 1024 == 0 && kOffP % 1024 == 0, "swizzled tiles");
  static_assert(kTmemS + 32 * kSlots <= kTmemCols, "tensor memory");
  static_assert(kSmem <= 232448, "shared memory");
};

struct PairMisc {
  // in the leader: what the products wait for, from both CTAs
  uint64_t k_full[4], v_full[4], p_ready[4], q_ready;
  // in each CTA
  uint64_t qk_done[4], slot_free[4], q_free, drained[2], asked, answered, fin_full;
  uint64_t decided;                   // a block's maxima are settled
  uint32_t changes, asks;             // how often they changed; how often the peer was asked to rescale
  uint32_t asked_slot, asked_phase, over;      // of the block whose products are in O; no more will be asked
  uint32_t left, tmem_base;
  int start_b, start_k, count, meta_groups;
  long long start_pos, total;
  int scan[32];
  float top[4][64];                   // of a row's threads: maxima, sums
  float most[64];                     // what the rows' exponentials are relative to
  float corr[64], corr_peer[64];      // factors of this CTA's and of the peer's rows
  alignas(8) float scale[128];        // of the tile's rows
};
static_assert(sizeof(PairMisc) <= kMiscBytes, "PairMisc");

// (relaxed: nothing that this thread has written is announced, and a release waited a thousand cycles for its prefetches)
__device__ __forceinline__ void arrive_expect_cluster(uint32_t addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(addr), "r"(bytes) : "memory");
}
// a word into the peer's shared memory, counted by the barrier there: the words that a barrier has counted are there when it says so
__device__ __forceinline__ void st_async_f32(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ uint32_t try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendHintNs) : "memory");
  return ok;
}
// a wait for what the other CTA has written
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, const BlockWaiter& w, int site, int iter) {
  uint32_t since = 0;
  while (!try_wait_cluster(bar, parity))
    if (w.gives_up(since, site, iter)) return false;
  return true;
}
// a vote among the four warps of a softmax group
__device__ __forceinline__ bool group_any(int group, bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"((uint32_t)x), "r"(3 + group) : "memory");
  return r != 0;
}
// and of the four that rescale for the peer
__device__ __forceinline__ bool aid_any(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}
// R columns of this warp's 32 lanes, column x by factor x
__device__ __forceinline__ void rescale(uint32_t taddr, const float* factors) {
  tc_fence_after();
#pragma unroll 1
  for (int x = 0; x < R; x += 16) {
    float o[16];
    tmem_ld16(taddr + x, o);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= factors[x + e];
    tmem_st16(taddr + x, o);
  }
  tmem_wait_st();
  tc_fence_before();
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

// What a group's pairs bring into L2 they bring in turn: true once in `every` calls, the first time after `left` of them
struct Turn {
  int every, left;
  __device__ __forceinline__ bool operator()() {
    if (left-- > 0) return false;
    left = every - 1;
    return true;
  }
};
// a running block's slot and the parity of its barriers
template <int kSlots>
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void advance() {
    if (++slot == kSlots) { slot = 0; phase ^= 1u; }
  }
};

// A launch that cannot be: NaN in all results, and no parts for the merge
__device__ __forceinline__ void refuse(const Params& p) {
  const long long i0 = (long long)blockIdx.x * blockDim.x + threadIdx.x, step = (long long)gridDim.x * blockDim.x, rows = (long long)p.B * p.rows;
  for (long long i = i0; i < rows * (kDV / 2); i += step) reinterpret_cast<uint32_t*>(p.out)[i] = 0x7fff7fffu;
  for (long long i = i0; i < rows; i += step) p.lse[i] = __uint_as_float(0x7fffffffu);
  if (p.meta)
    for (long long i = i0; i < p.groups; i += step) p.meta[i] = make_int4(-1, 0, 0, 0);
}

template <Load kLoad>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads<kLoad>, 1)
mla_decode_pair_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_q, const Params p) {
  constexpr int kSlots = PL::kSlots, kTile = 2 * R;
  using Cursor = Ring<kSlots>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  // Swizzled tiles.  There is no room for rounding; the driver has put the base on such a boundary so far, in both CTAs alike.
  if ((sbase & 1023u) != 0) {
    pdl_wait();
    refuse(p);
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
    for (int i = 0; i < PL::kSlots; ++i) {
      // warps of both CTAs
      mbar_init(&ms.k_full[i], 2 * (kLoad == kTma ? 2 : kKeyWarps));
      mbar_init(&ms.v_full[i], 2 * (kLoad == kTma ? 1 : kValueWarps));
      mbar_init(&ms.p_ready[i], 2);
      mbar_init(&ms.qk_done[i], 1);
      mbar_init(&ms.slot_free[i], 1);
    }
    mbar_init(&ms.q_ready, 2);
    mbar_init(&ms.q_free, 1);
    mbar_init(&ms.asked, 1);
    mbar_init(&ms.answered, 1);
    mbar_init(&ms.decided, 1);
    ms.over = ms.changes = ms.asks = 0;
    mbar_init(&ms.fin_full, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&ms.drained[i], 1);
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
    if (kLoad == kPacked) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");     // 2 x 88 + 4 x 72 + 40 = 7 x 72, as launched
    // Two groups of four warps take turns, a block each: warp (warp % 4) has TMEM lanes 32 (warp % 4), a thread row r and keys 32 h + [0, 32).
    // Blocks' maxima are settled in order (decided): whoever finds a row past its bound changes the row's for both groups, which
    // the other sees before it hands its P over.
    const int quarter = warp & 3, c = warp >> 2, tl = 32 * quarter + lane, r = tl & 63, h = tl >> 6;
    const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
    const uint32_t a_p_ready = mapa(smem_u32(&ms.p_ready[0]), 0);
    volatile uint32_t* const changes = &ms.changes;
    volatile uint32_t* const asks = &ms.asks;
    Walk w(ms);
    Cursor at, prev, prev2;                                 // of blocks kb, kb - 1, kb - 2
    int kb = 0;
    uint32_t seen = 0, wholes = 0;                          // changes; sequences ended here
    // A wait here that gives up is passed like any other: the warps meet at named barriers, so they take the same steps.
    bool more = w.next(p);
    while (more) {
      const int row = row0 + r;
      const int lim = min(w.len, w.len - p.q_len + 1 + row / p.heads), low = w.len - p.q_len + 1 + row0 / p.heads;     // low: what this CTA's first row sees
      float m = kMInit, l = 0.f;
      auto renew = [&]() {                                  // the row's maximum as the groups have settled it
        seen = *changes;
        const float now = ms.most[r];
        l *= fast_exp2(m - now);
        m = now;
      };
      for (int k = w.k0; k < w.k1; ++k, ++kb, prev2 = prev, prev = at, at.advance()) {
        if ((kb & 1) != c) continue;
        mbar_wait(&ms.qk_done[at.slot], at.phase, wt, kSiteS, kb);
        __syncwarp();
        tc_fence_after();
        float v[32];
        float mx = -INFINITY;
        tmem_ld32(tmem + PL::kTmemS + 32 * at.slot + lane_base, v);
        tmem_wait_ld();
        if ((k + 1) * kBlock > low) {
          const int keys = lim - k * kBlock - 32 * h;
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = e < keys ? v[e] * p.scale_log2 : -INFINITY;
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] *= p.scale_log2;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) mx = fmaxf(mx, v[e]);
        const bool first = k == w.k0;
        if (k == w.k0 + 1) {                                // (a piece's first block changes them)
          mbar_wait(&ms.decided, (kb - 1) & 1, wt, kSiteVote, kb);
          __syncwarp();
          if (*changes != seen) renew();
        }
        auto must = [&]() { return first || __any_sync(0xffffffffu, mx > m + kMostOver); };
        const bool need = must();
        if (kb >= 2) {                                      // this buffer's last P has been read
          mbar_wait(&ms.slot_free[prev2.slot], prev2.phase, wt, kSitePv, kb);
          __syncwarp();
        }
        auto put_p = [&]() -> float {
          float sum = 0.f;
          const uint32_t rope = sbase + PL::kOffKV + at.slot * kSlot + (kChunks - 1) * kChunk;
          const uint32_t ph = h == 0 ? rope : sbase + PL::kOffP + (kb & 1) * PL::kPHalf;
          // 8 rows x 8 keys a matrix of 128 bytes: rows first, then keys
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = fast_exp2(v[8 * j + 2 * e] - m), b = fast_exp2(v[8 * j + 2 * e + 1] - m);
              sum += a + b;
              u[e] = bf16x2(a, b);
            }
            st_shared16(ph + j * (R * 16) + r * 16, make_uint4(u[0], u[1], u[2], u[3]));
          }
          fence_proxy_async_smem();
          tc_fence_before();
          return sum;
        };
        // P is written as if no row needed a new maximum
        float sum = need ? 0.f : put_p();
        bool stale = false;
        if (!first) {
          mbar_wait(&ms.decided, (kb - 1) & 1, wt, kSiteVote, kb);
          __syncwarp();
          stale = *changes != seen;
        }
        // (what a thread finds is put to the vote before steps depend on it: where waits have given up, threads may find different things)
        bool change = group_any(c, need || stale);
        if (change && !first && group_any(c, stale)) {
          renew();
          change = group_any(c, must());
          if (!change) {
            sum = put_p();
            group_any(c, false);
          }
        }
        if (change) {
          ms.top[h][r] = mx;
          group_any(c, false);
          const float now = fmaxf(m, fmaxf(ms.top[0][r], ms.top[1][r])), f = fast_exp2(m - now);
          m = now;
          l *= f;
          if (h == 0) {
            ms.most[r] = m;
            if (!first) {
              ms.corr[r] = f;
              st_cluster_f32(mapa(smem_u32(&ms.corr_peer[r]), peer), f);
            }
          }
          if (!first) {
            // the columns of these rows: this CTA's dims here, the peer's by its four warps
            const uint32_t asked = *asks;
            fence_cluster();
            group_any(c, false);
            if ((threadIdx.x & 127) == 0) {
              st_cluster_u32(mapa(smem_u32(&ms.asked_slot), peer), (uint32_t)prev.slot);
              st_cluster_u32(mapa(smem_u32(&ms.asked_phase), peer), prev.phase);
              mbar_arrive_cluster_release(mapa(smem_u32(&ms.asked), peer));
            }
            mbar_wait(&ms.slot_free[prev.slot], prev.phase, wt, kSitePv, kb);
            __syncwarp();
            for (int i = 0; i < 2; ++i) rescale(tmem + lane_base + kTile * i + R * cta, ms.corr);
            wait_cluster(&ms.answered, asked & 1, wt, kSiteAid, kb);
            __syncwarp();
            if ((threadIdx.x & 127) == 0) *asks = asked + 1;
          }
          sum = put_p();
          ++seen;
          group_any(c, false);
          if ((threadIdx.x & 127) == 0) *changes = seen;
        }
        l += sum;
        if ((threadIdx.x & 127) == 0) {                     // (all warps have fenced what they wrote)
          mbar_arrive(&ms.decided);
          mbar_arrive_cluster(a_p_ready + 8u * at.slot);
        }
      }
      softmax_sync();                                       // (after the last block's change)
      if (*changes != seen) renew();
      // epilogue: this CTA's dims of all of the tile's rows
      ms.top[2 * c + h][r] = l;
      const bool whole = w.whole();
      const int slot = cluster * 2 + (w.index == 0 ? 0 : 1);
      softmax_sync();
      if (h == 0 && c == 0) {
        const float sum = ms.top[0][r] + ms.top[1][r] + ms.top[2][r] + ms.top[3][r];
        if (whole) {
          const float f = sum != 0.f ? 1.f / sum : 0.f;
          ms.scale[R * cta + r] = f;
          st_async_f32(mapa(smem_u32(&ms.scale[R * cta + r]), peer), f, mapa(smem_u32(&ms.fin_full), peer));
        } else {
          p.part_ml[(long long)slot * kTile + R * cta + r] = make_float2(m, sum);
        }
      }
      if (whole) {                                          // (both CTAs alike; the peer's factors are its own words on the barrier)
        if (threadIdx.x == 0) mbar_arrive_expect_tx(&ms.fin_full, 4 * R);
        softmax_sync();
        wait_cluster(&ms.fin_full, wholes++ & 1, wt, kSiteVote, kb);
        if (h == 0 && c == 0 && row < p.rows) {
          const float sum = ms.top[0][r] + ms.top[1][r] + ms.top[2][r] + ms.top[3][r];
          p.lse[(long long)w.b * p.rows + row] = sum != 0.f ? (m + __log2f(sum)) * kLn2 : INFINITY;
        }
      }
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
            // Two rows a word, one dim; then lanes 2 i and 2 i + 1 exchange, for two dims of a row each
            const int odd = lane & 1;
            const uint32_t order = odd ? 0x3276u : 0x5410u;
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out) + (((long long)w.b * p.rows + rt * kTile + x + odd) * kDV + (d & ~1)) / 2;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float2 f = *reinterpret_cast<const float2*>(&ms.scale[x + e]);
              // (a row without keys: 0, whatever the values of others)
              const uint32_t mine = bf16x2(f.x != 0.f ? o[y][e] * f.x : 0.f, f.y != 0.f ? o[y][e + 1] * f.y : 0.f);
              const uint32_t its = __shfl_xor_sync(0xffffffffu, mine, 1);
              if (x + e + odd < rows) dst[e * (kDV / 2)] = __byte_perm(mine, its, order);
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
      softmax_sync();                                       // (either group's P may start the next piece)
      more = w.next(p);
    }
    // The peer asks for nothing any more: all of its P are in O.
    if (threadIdx.x == 0) {
      *reinterpret_cast<volatile uint32_t*>(&ms.over) = 1;
      mbar_arrive(&ms.asked);
    }
  } else if (warp >= kWarpAid<kLoad>) {
    // ------------------------------------------------------------ rescalings that the peer asks for
    if (kLoad == kPacked) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    const int quarter = warp & 3;
    const uint32_t a_answered = mapa(smem_u32(&ms.answered), peer);
    for (uint32_t n = 0;; ++n) {
      // (Most launches ask for none, so this wait may last as long as the launch; it ends with the softmax warps, whose waits are bounded.)
      uint32_t ok = 0;
      for (uint32_t i = 0; !ok && !wt.aborting() && i < (1u << 24); ++i) ok = try_wait_cluster(&ms.asked, n & 1);
      if (aid_any(!ok || *reinterpret_cast<volatile uint32_t*>(&ms.over) != 0)) break;      // (all four warps or none)
      const uint32_t slot = *reinterpret_cast<volatile uint32_t*>(&ms.asked_slot), phase = *reinterpret_cast<volatile uint32_t*>(&ms.asked_phase);
      mbar_wait(&ms.slot_free[slot < kSlots ? slot : 0], phase, wt, kSiteAid, (int)n);
      __syncwarp();
      for (int c = 0; c < 2; ++c) rescale(tmem + ((uint32_t)(32 * quarter) << 16) + kTile * c + R * peer, ms.corr_peer);
      if (!aid_any(false) && warp == kWarpAid<kLoad> && lane == 0) mbar_arrive_cluster_release(a_answered);
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
          const uint32_t p1 = sbase + PL::kOffP + (kb & 1) * PL::kPHalf;
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
    while (w.next(p)) {
      if (w.index > 0 && !__all_sync(0xffffffffu, mbar_wait(&ms.q_free, (w.index - 1) & 1, wt, kSiteQ, w.index))) break;
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
        if (lane == 0) mbar_arrive_cluster(a_ready);
      }
    }
  } else if (kLoad == kPacked && warp == kWarpBring) {
    // ------------------------------------------------------------ this CTA's keys into L2, two blocks ahead of the converting warps
    const int count = ms.count;
    Ahead<true> next(ms, p, kOwnKeys * (int)cta, kOwnKeys, lane);
    Turn mine_to_bring{p.row_tiles, rt};
    Cursor at;
    for (int kb = 0; kb < count; ++kb, next.advance(p, lane)) {
      // (Nothing waits for this warp, so the barrier can be two phases ahead of it and look as if it were behind; then this waits for
      // another phase, or for the end.)
      bool go = true;
      while (kb >= kSlots && go && !mbar_try_wait(&ms.slot_free[at.slot], at.phase ^ 1u)) go = !wt.aborting() && *reinterpret_cast<volatile uint32_t*>(&ms.over) == 0;
      if (!__all_sync(0xffffffffu, go)) break;
      at.advance();
      if (!mine_to_bring()) continue;
      for (int d = kb == 0 ? 0 : 2; d < 3; ++d) {
        const int n = next.rows_in(d), row = __shfl_sync(0xffffffffu, next.row, next.i + d), one = min(n, p.block_size - row);
        const uint8_t* src = next.rows_of(p, d, kPackedRow);
        if (src != nullptr && lane == 0 && one > 0) l2_prefetch_1d(src, (uint32_t)(one * kPackedRow));
        const int page2 = __shfl_sync(0xffffffffu, next.page2, next.i + d);
        if (one < n && page2 < p.n_blocks && lane == 0) l2_prefetch_1d(p.cache + (long long)page2 * p.block_pitch, (uint32_t)((n - one) * kPackedRow));
      }
    }
  } else if (kLoad == kTma ? warp <= kWarpK1 : warp >= kLoad0) {
    // ------------------------------------------------------------ keys (own 32, all dims) and values (the peer's 32, own 256 dims)
    constexpr int kRowBytes = kLoad == kPacked ? kPackedRow : 2 * kD;
    const bool is_v = kLoad == kTma ? warp == kWarpV : warp >= kLoad0 + kKeyWarps;
    // The warp's rows of the 32.  kTma: pages of multiples of 32 rows have one box of rows a chunk, others two; keys of one box are shared out by chunks, of
    // two by box.  kPacked: 4 rows a warp of keys, 8 of values (of one page: pages are multiples of 16 rows).
    const int boxes = kLoad == kTma ? kOwnKeys / p.box_rows : 1, second = kLoad == kTma && warp == kWarpK1 ? 1 : 0;
    const int rows_own = kLoad == kTma ? (is_v || boxes == 1 ? kOwnKeys : 16) : is_v ? kOwnKeys / kValueWarps : kOwnKeys / kKeyWarps;
    const int first_row = kLoad == kTma ? (rows_own < kOwnKeys ? 16 * second : 0) : rows_own * (is_v ? warp - kLoad0 - kKeyWarps : warp - kLoad0);
    const int box = kLoad == kTma && is_v && boxes > 1 ? (lane >> 2) & 1 : 0;        // the lane's, for values
    const int half = is_v ? (int)peer : (int)cta;                                    // whose keys
    const uint32_t a_full = mapa(smem_u32(is_v ? &ms.v_full[0] : &ms.k_full[0]), 0);
    uint64_t* const waits = is_v ? ms.qk_done : ms.slot_free;
    const uint32_t chunk0 = is_v ? (cta == 0 ? 4 : 0) : 0;                           // where its first chunk goes
    const int dim0 = is_v ? 256 * (int)cta : 0;
    const int count = ms.count;
    // a slot is free (K) or its keys have been read (V)
    auto free_for = [&](const Cursor& at, int kb) -> bool {
      if (is_v) return mbar_wait(&waits[at.slot], at.phase, wt, kSiteFree, kb);
      return kb < kSlots || mbar_wait(&waits[at.slot], at.phase ^ 1u, wt, kSiteFree, kb);
    };
    Cursor at;
    bool ok = true;
    // The page, row and number of the warp's rows of a block, for the loads through registers
    struct Coming { int page, row, n; };
    Walk w(ms);
    int k_at = 0, looked = 0;
    PageAt pa(p.block_size);
    const int* table = nullptr;
    auto piece = [&]() {
      if (!w.next(p)) return;
      k_at = w.k0;
      table = p.table + w.b * p.table_pitch;
      pa.at(k_at * kBlock + kOwnKeys * half + first_row);
    };
    auto look = [&]() -> Coming {
      Coming x{-1, 0, 0};
      if (looked >= count) return x;
      x.n = min(max(w.len - k_at * kBlock - kOwnKeys * half - first_row, 0), rows_own);
      if (x.n > 0) x.page = __ldcg(table + pa.page);
      x.row = pa.row;
      ++looked;
      pa.advance();
      if (++k_at == w.k1) piece();
      return x;
    };
    auto rows_of = [&](const Coming& x) -> const uint8_t* {
      return (unsigned)x.page < (unsigned)p.n_blocks ? p.cache + (long long)x.page * p.block_pitch + (long long)x.row * kRowBytes : nullptr;
    };
    if (kLoad == kPacked) piece();
    if (kLoad != kPacked) {
      Ahead<true> next(ms, p, kOwnKeys * half + first_row, rows_own, lane);
      Turn mine_to_bring{p.row_tiles, rt};
      // (the other rows are the peer's to bring in)
      auto to_l2 = [&](int d) {
        const uint8_t* src = next.rows_of(p, d, kRowBytes);
        const int n = next.rows_in(d);
        if (!is_v && src != nullptr && lane == 0 && (rows_own < kOwnKeys || second == 0)) l2_prefetch_1d(src, (uint32_t)(n * kRowBytes));
      };
      const uint64_t pol = l2_policy_evict_first();
      // what the lane requests of a block
      const int chunk = is_v ? lane & 3 : boxes == 1 ? lane + 5 * second : lane;
      const bool mine = is_v ? lane < 4 * boxes : boxes == 1 ? (second ? lane < 4 : lane < 5) : lane < kChunks;
      const uint32_t bytes = (is_v ? 4u * kChunk : boxes == 1 ? (second ? 4u : 5u) * kChunk : kChunks * kChunk / 2);
      for (int kb = 0; kb < count; ++kb, next.advance(p, lane)) {
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
        const int n = next.rows_in(0), page1 = __shfl_sync(0xffffffffu, next.page, next.i), page2 = __shfl_sync(0xffffffffu, next.page2, next.i);
        const int row1 = __shfl_sync(0xffffffffu, next.row, next.i), row2 = row1 + 16 - (row1 + 16 >= p.block_size ? p.block_size : 0);
        if (mine_to_bring()) to_l2(2);
        if (!(ok = __all_sync(0xffffffffu, free_for(at, kb)))) break;
        if (n == rows_own || (n == 0 && p.n_blocks > 0)) {  // (of a page beyond the cache, or none: zeros; a cache without pages has no map)
          if (lane == 0) arrive_expect_cluster(a_full + 8u * at.slot, bytes);
          __syncwarp();
          if (mine)
            tma_load_3d_pair_hint(slot + (chunk0 + chunk) * kChunk + (first_row + 16 * box) * 128, &map_kv, dim0 + 64 * chunk, box ? row2 : row1,
                                  box ? page2 : page1, a_full + 8u * at.slot, pol);
        } else {
          // zeros behind a sequence's end: 0 x NaN is NaN
          for (int x = second == 0 || boxes > 1 ? 0 : rows_own; x < rows_own; x += 16) {
            const int page = x ? page2 : page1, rows = page < p.n_blocks ? n - x : 0;
            const uint8_t* from = p.cache + (page < p.n_blocks ? (long long)page * p.block_pitch + (long long)(x ? row2 : row1) * kRowBytes + 2 * dim0 + 16 * lane : 0);
            const uint32_t to = slot + (chunk0 + (lane >> 3)) * kChunk + (first_row + x) * 128;
            for (int c = 0; c < (is_v ? 1 : 3); ++c)        // 512 bytes of each row
              if (c < 2 || lane < 8)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                  cp_async16_or_zero(to + 4 * c * kChunk + r * 128 + (((lane & 7) ^ (r & 7)) << 4), r < rows ? from + 512 * c + r * kRowBytes : p.cache, r < rows);
          }
          cp_async_wait_all();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(a_full + 8u * at.slot);
        }
        at.advance();
      }
    } else if (!is_v) {
      // Of each 128 dims eight lanes have 16 codes of a row each, four rows at a time.  A group's registers are loaded for the next
      // block as soon as they are converted for this one, from L2, where the rows were brought a block before.
      const int sub = lane >> 3, c = lane & 7, row = first_row + sub;
      static_assert(kOwnKeys / kKeyWarps == 4 && kOwnKeys / kValueWarps == 8, "rows of a warp");
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
      Coming c1 = look(), c2 = look();
      load(rows_of(c1), c1.n);
      for (int kb = 0; ok && kb < count; ++kb) {
        c1 = c2; c2 = look();                               // (moved before the next is asked for: a move waits for its load)
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
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
        if (lane == 0) mbar_arrive_cluster(a_full + 8u * at.slot);
        load(rows_of(c1), c1.n);                            // (the next)
        at.advance();
      }
    } else {
      // the peer's rows: 16 lanes a row, 16 codes each of this CTA's 256 dims
      const int sub = lane >> 4, c = lane & 15;
      uint4 codes[4];
      float scale[4];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      auto load = [&](const uint8_t* src, int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = src != nullptr && sub + 2 * i < n;
          const uint8_t* from = src + (sub + 2 * i) * kRowBytes;
          codes[i] = in ? __ldcg(reinterpret_cast<const uint4*>(from + dim0) + c) : zero;
          scale[i] = in ? __ldcg(reinterpret_cast<const float*>(from + 512) + dim0 / 128 + (c >> 3)) : 0.f;
        }
      };
      Coming c1 = look(), c2 = look();
      load(rows_of(c1), c1.n);
      for (int kb = 0; ok && kb < count; ++kb) {
        c1 = c2; c2 = look();                               // (moved before the next is asked for: a move waits for its load)
        const uint32_t slot = sbase + PL::kOffKV + at.slot * kSlot;
        if (!(ok = __all_sync(0xffffffffu, free_for(at, kb)))) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = first_row + sub + 2 * i;
          uint4 a, b;
          convert16(codes[i], scale[i], a, b);
          const uint32_t base = slot + (chunk0 + (c >> 2)) * kChunk + row * 128, u = 2 * (c & 3), odd = (c >> 2) & 1;
          st_shared16(base + (((u + odd) ^ (row & 7)) << 4), odd ? b : a);
          st_shared16(base + (((u + 1 - odd) ^ (row & 7)) << 4), odd ? a : b);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(a_full + 8u * at.slot);
        load(rows_of(c1), c1.n);                            // (the next)
        at.advance();
      }
    }
  }

  if (warp == kWarpQk && rt == 0 && cta == 0 && lane == 0 && p.meta) write_meta(p, ms, g);
  tc_fence_before();
  __syncthreads();
  // Given up: what is in flight lands before either CTA's memory goes.  (Loads, factors and commits are counted by barriers of which some are the other
  // CTA's and may never complete.  A CTA that has not given up has nothing in flight: its last block's second product is complete.)
  if (threadIdx.x == 0 && wt.aborting()) drain_uncounted();
  cluster_sync_all();                                       // nothing of this CTA is in use by the other
  tc_fence_after();
  if (warp == kWarpQk) tmem_dealloc_pair(tmem, PL::kTmemCols);
  if (threadIdx.x == 0) {
    wt.report(g_status, p.epoch);
    if (blockIdx.x == 0) atomicAdd(&g_status[3], 1);
  }
}

// pairs that can run at once
template <Load kLoad>
static int pairs() {
  static thread_local int cached_dev = -1, cached = 0;
  const int dev = current_device();
  if (dev == cached_dev) return cached;
  int n = sm_count() / 2, q = 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sm_count()); cfg.blockDim = dim3(kPairThreads<kLoad>); cfg.dynamicSmemBytes = PL::kSmem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = 2; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
  cfg.attrs = &at; cfg.numAttrs = 1;
  if (ensure_smem<mla_decode_pair_kernel<kLoad>>(dev, PL::kSmem) &&
      cudaOccupancyMaxActiveClusters(&q, mla_decode_pair_kernel<kLoad>, &cfg) == cudaSuccess && q > 0)
    n = q;
  cudaGetLastError();
  cached_dev = dev; cached = n;
  return n;
}
template <Load kLoad>
static int launch(const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  if (!ensure_smem<mla_decode_pair_kernel<kLoad>>(current_device(), PL::kSmem)) return LITEDSA_ERR_CUDA;
  return launch_pdl(mla_decode_pair_kernel<kLoad>, dim3((unsigned)(2 * p.groups * p.row_tiles)), kPairThreads<kLoad>, PL::kSmem, st, map, map_q, p);
}
static int launch(Load l, const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  return l == kTma ? pair::launch<kTma>(map, map_q, p, st) : pair::launch<kPacked>(map, map_q, p, st);
}

}  // namespace pair
}  // namespace decode
}  // namespace lt
