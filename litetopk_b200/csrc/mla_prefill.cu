// Expanded latent attention (sm_100a): the dense prefill of MLA over a batch of sequences of their own lengths.
//
//   s = sm_scale (q[0:128] . k_nope + q[128:192] . k_rope), p = softmax of s over the keys a token sees, out = p v[0:128]
//
// per head; k_rope is one vector a token for all heads.  Bound by the tensor cores: 640 flops a (query, key, head).
//
// A CTA takes 256 queries of a head as two tiles of 128 rows and streams the keys in blocks of 128.  Tensor memory is full: two S
// (128 columns each; P, bf16, takes the place of its S and is the A operand of the second product from there) and two O.
// While one tile's S is turned into P by its four warps, the tensor cores have the other tile's products:
//
//   P0 V(i), Q0 K(i+1), P1 V(i), Q1 K(i+1), P0 V(i+1), ...
//
// A thread has a row: no reductions between threads, and the rare rescaling of O is its warp's own business (the maximum that P is
// relative to is taken anew only when a block's sum asks for it, kMostSum).  P of a block's first 64 keys is handed over before the others', so
// that its product begins meanwhile.  Keys and values pass through one ring of eight 16 KB granules (128 tokens x 64 dims) in the order of
// use, three of K and two of V a block: with a stage of K and of V each released as a whole the V of a block would come too late.
//
// CTAs take work dynamically (cluster launch control: a running CTA takes the place of one that has not been launched), the heavy
// tiles first, heads one after the other so that the CTAs that run share their K and V in L2.  A call of few tiles leaves
// most of its last wave idle: its last tiles are cut along the keys, and a second kernel merges the pieces in fp32.
//
// Measured: 8192 tokens x 64 heads, causal, 1221 us = 1126 TFLOP/s when the power limit has brought the clock down to 1.55 GHz, 1047 = 1312 in a few calls
// (a library's matrix product: 1391 and 1657); 4096 tokens behind 28672, 16 heads, 1107 us = 1164 TFLOP/s, 957 = 1346 in a few calls.  A block of a tile takes
// 2000 cycles of a CTA, of which the tensor cores compute 1300: the exponentials (128 a row and block) and the hand-overs fill the rest.  Works of up to 128
// queries have one tile at work and nothing beside it: 4 tokens behind 16384, 64 heads, 147 us (their bytes: 82).
#include "common.cuh"
#include "tensor_map.cuh"

namespace lt {
namespace prefill {

constexpr int kRows = 128, kPair = 256, kBlock = 128, kDV = 128;
constexpr uint32_t kGranule = 128 * 128;                    // 128 tokens x 64 bf16
constexpr int kRing = 8, kPerBlock = 5;                     // granules; of a block: K 0-2, V 3-4
constexpr uint32_t kQTile = 3 * kGranule;
constexpr uint32_t kOffQ = 0, kOffRing = 2 * kQTile, kOffMisc = kOffRing + kRing * kGranule;
constexpr uint32_t kSmem = kOffMisc + 1024 + 1024;
static_assert(kSmem <= 232448, "shared memory");
constexpr int kWarpMma = 8, kWarpLoad = 9, kThreads = 384;     // (warps 10 and 11 have nothing to do: registers are dealt out by four warps)
constexpr uint32_t kTmemO = 256;                            // S0, S1, O0, O1: 128 columns each
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMInit = -1e30f;
// P is relative to a maximum that may be stale: a block's exponentials are computed with the row's last one, and only if their sum
// shows that some were above it by more than this is the maximum taken anew, O rescaled and the block repeated.  A pass over the scores for
// their maximum cost a quarter of a row's softmax; P is as exact in bf16 above one as below, and fp32 sums hold 2^32 as well as 1.
constexpr float kMostSum = 4294967296.f;

struct Work {
  int head, q0, rows;          // queries [q0, q0 + rows) of the call's tokens
  int k0, nk;                  // keys of the sequence: [k0, k0 + nk) of the call's
  int lim0;                    // causal: row r sees keys [0, lim0 + r) of the sequence
  int b0, n[2];                // blocks [b0, b0 + n[t]) for tile t
  int part;                    // -1: the tiles as a whole; else which piece's place in the workspace
  int live;                    // 0: no more work
};
struct Misc {
  uint64_t k_full[2], v_full[2], k_free[2], v_free[2];      // by the parity of the block
  uint64_t q_full[2], q_free[2], s_ready[2], p_ready[2][2], half_done[2], o_done[2], work_full[2], work_empty[2], clc, drained;
  uint4 clc_answer;
  Work work[2];
  uint32_t left, tmem_base;
  int scan[2 * kThreads / 32];
};
static_assert(sizeof(Misc) <= 1024, "Misc");

struct Params {
  const int32_t *cu_q, *cu_k;  // [B + 1], or null: one sequence
  uint8_t* out;                // [Tq, heads, 128] bf16
  float* lse;                  // [Tq, heads]
  float* part_o;               // [piece][256][128]
  float2* part_ml;             // [piece][256]: (maximum, sum)
  int4* plan;                  // (tiles, first tile that is cut, pieces a tile, this launch) for the merge
  int B, Tq, Tk, heads, ctas, causal, max_pieces;
  float scale_log2;
  int epoch;
  uint32_t wait_limit;
};

enum { kSiteFull = 1, kSiteEmpty, kSiteQ, kSiteQFree, kSiteS, kSiteP, kSiteO, kSiteWork, kSiteWorkEmpty, kSiteClc };
static __device__ int g_status[8];

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// work stealing among the blocks of this launch: asks for one that has not started (16 bytes of answer on the barrier)
__device__ __forceinline__ void clc_ask(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ int clc_block(const uint4* answer) {      // its blockIdx.x, -1 if there is none
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .b64 a, b;\n\t.reg .pred p;\n\t"
      "ld.shared.v2.b64 {a, b}, [%2];\n\tmov.b128 h, {a, b};\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=r"(x) : "r"(smem_u32(answer)) : "memory");
  return ok ? (int)x : -1;
}

__device__ __forceinline__ int start_of(const int32_t* cu, int b, int B, int T) {
  if (cu == nullptr) return b == 0 ? 0 : T;
  return min(max(__ldcg(cu + b), 0), T);
}
__host__ __device__ __forceinline__ int blocks_seen(int keys) { return keys <= 0 ? 0 : (keys - 1) / kBlock + 1; }

// How the call's tiles (pairs of 128 rows, of all heads) are cut: tiles [0, whole) as they are, the others into `pieces` each.
// Only calls of few tiles: as many waves of whole tiles as there are, the rest cut so that its pieces fill the CTAs, at a cost of
// three blocks a piece for its set-up and its way through memory.  Evaluated by one warp.
struct Cut { int whole, pieces; };
__device__ __forceinline__ Cut cut_of(int tiles, int most_blocks, const Params& p, int lane) {
  Cut c{tiles, 1};
  if (p.max_pieces == 0 || tiles > 4 * p.ctas) return c;
  const int rest = tiles % p.ctas;
  if (rest == 0) return c;
  const int most = min(min(p.max_pieces / rest, most_blocks / 2), 1023);
  uint32_t best = 0xffffffffu;
  for (int s = lane + 1; s <= most; s += 32) {
    const uint32_t cost = (uint32_t)((rest * s + p.ctas - 1) / p.ctas) * (uint32_t)((most_blocks + s - 1) / s + (s > 1 ? 3 : 0));
    best = min(best, min(cost, 0x3fffffu) << 10 | (uint32_t)s);
  }
  best = __reduce_min_sync(0xffffffffu, best);
  if (best != 0xffffffffu && (best & 1023u) > 1) { c.whole = tiles - rest; c.pieces = (int)(best & 1023u); }
  return c;
}

// Calls of many tiles take those of more than a third of the longest one's blocks first, of all heads, then the others: what the last CTAs to
// finish are still at is then short (a batch of 11 sequences 398 -> 376 us, 8192 tokens of 64 heads 1101 -> 1047, all in a few calls; in one order / from a
// quarter / a third / half on, between two events behind a flush of L2, us: 5 prompts of 100 to 6000 tokens, 32 heads, 723 / 693 / 708 / 689, 40 of 50 to 900,
// 16 heads, 135 / 132 / 121 / 133, 3 of 4000, 24 heads, 372 / 357 / 349 / 350; but 20 of 300 to 700 behind 2000, 16 heads, 271 / 280 / 280 / 282, where all
// tiles are among the first and the order is one).  Among the first and among the others, as in calls of few: a head's tiles from its last to its first, then
// the next head's, so that CTAs that run together share keys and values in L2.
//
// A lane keeps how many tiles the sequences [0, (lane + 1) each) have among the first and among the others, and of `each` = 1 its sequence: to find a
// work's tile then takes one read of memory where there are up to 1024 sequences, none up to 32.  (Looking 32 sequences at a time through all of them, 1000
// prompts of up to 60 tokens, 16 heads, took 1069 us, now 366; 256 prompts of 20 to 150 tokens 163, now 130.)
struct Order {
  int all, first, least;      // tiles of a head, those of more than `least` blocks
  int each, upto[2];
  int q0, k0;
  int2 len;
};
// Of a sequence, the tiles of more than x blocks: its last ones
__device__ __forceinline__ int tiles_above(int x, int nq, int nk, int causal) {
  const int all = (nq + kPair - 1) / kPair;
  return x < 0 ? all : nk <= kBlock * x ? 0 : causal ? all - max(kBlock * x - (nk - nq), 0) / kPair : all;
}
__device__ __forceinline__ int2 lengths_of(const Params& p, int b, int& q0, int& k0) {
  q0 = start_of(p.cu_q, b, p.B, p.Tq);
  k0 = start_of(p.cu_k, b, p.B, p.Tk);
  return make_int2(max(start_of(p.cu_q, b + 1, p.B, p.Tq) - q0, 0), max(start_of(p.cu_k, b + 1, p.B, p.Tk) - k0, 0));
}
__device__ __forceinline__ int inclusive(int v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += u;
  }
  return v;
}
// By one warp.
__device__ __forceinline__ Order order_of(int tiles_a_head, int most, const Params& p, int lane) {
  Order o;
  o.all = tiles_a_head;
  o.least = (long long)tiles_a_head * p.heads > 4 * p.ctas ? most / 3 : -1;
  o.each = (p.B + 31) / 32;
  o.len = make_int2(0, 0);
  o.q0 = o.k0 = 0;
  int own[2] = {0, 0};
  const int b1 = min((lane + 1) * o.each, p.B);
#pragma unroll 8
  for (int b = lane * o.each; b < b1; ++b) {
    o.len = lengths_of(p, b, o.q0, o.k0);
    const int above = tiles_above(o.least, o.len.x, o.len.y, p.causal);
    own[0] += above;
    own[1] += (o.len.x + kPair - 1) / kPair - above;
  }
  o.upto[0] = inclusive(own[0], lane);
  o.upto[1] = inclusive(own[1], lane);
  o.first = __shfl_sync(0xffffffffu, o.upto[0], 31);
  return o;
}

// Work number w, by one warp.
__device__ __forceinline__ Work work_of(int w, const Order& o, const Cut& c, const Params& p, int lane) {
  Work k;
  k.live = 0;
  if (o.all <= 0) return k;                                // no sequence has a query
  const int tile = w < c.whole ? w : c.whole + (w - c.whole) / c.pieces, piece = w < c.whole ? 0 : (w - c.whole) % c.pieces;
  const int later = tile >= o.first * p.heads, n = later ? o.all - o.first : o.first, in = tile - later * o.first * p.heads;
  k.live = in < n * p.heads;
  if (!k.live) return k;
  k.head = in / n;
  int at = n - 1 - (in - k.head * n);
  int upto = later ? o.upto[1] : o.upto[0];
  uint32_t hit = __ballot_sync(0xffffffffu, at < upto);
  int l = hit ? __ffs(hit) - 1 : 31, before = __shfl_sync(0xffffffffu, upto, max(l - 1, 0));
  if (l > 0) at -= before;
  int q0 = o.q0, k0 = o.k0;
  int2 len = o.len;
  if (o.each > 1) {                                        // among the run's sequences
    const int end = min((l + 1) * o.each, p.B);
#pragma unroll 1
    for (int b0 = l * o.each;; b0 += 32) {
      const int b = b0 + lane;
      len = make_int2(0, 0);
      if (b < end) len = lengths_of(p, b, q0, k0);
      const int above = tiles_above(o.least, len.x, len.y, p.causal);
      upto = inclusive(later ? (len.x + kPair - 1) / kPair - above : above, lane);
      hit = __ballot_sync(0xffffffffu, at < upto);
      l = hit ? __ffs(hit) - 1 : 31;
      before = __shfl_sync(0xffffffffu, upto, hit ? max(l - 1, 0) : 31);
      if (l > 0 || !hit) at -= before;
      if (hit) break;
      if (b0 + 32 >= end) { k.live = 0; return k; }        // (not reached: the tiles of all sequences are n)
    }
  }
  const int q_start = __shfl_sync(0xffffffffu, q0, l), k_start = __shfl_sync(0xffffffffu, k0, l);
  const int nq = __shfl_sync(0xffffffffu, len.x, l);
  k.nk = __shfl_sync(0xffffffffu, len.y, l);
  const int first = tiles_above(o.least, nq, k.nk, p.causal);
  if (!later) at += (nq + kPair - 1) / kPair - first;
  k.q0 = q_start + at * kPair;
  k.rows = min(kPair, nq - at * kPair);
  k.k0 = k_start;
  k.lim0 = k.nk - nq + at * kPair + 1;
  int nb[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int last = min(k.rows, kRows * (t + 1)) - 1;     // last row of the tile
    nb[t] = k.rows <= kRows * t ? 0 : blocks_seen(p.causal ? min(k.nk, k.lim0 + last) : k.nk);
  }
  k.part = -1;
  int from = 0, to = max(nb[0], nb[1]);
  if (w >= c.whole && c.pieces > 1) {
    k.part = w - c.whole;
    from = (int)((long long)to * piece / c.pieces);
    to = (int)((long long)to * (piece + 1) / c.pieces);
  }
  k.b0 = from;
  k.n[0] = max(min(nb[0], to) - from, 0);
  k.n[1] = max(min(nb[1], to) - from, 0);
  return k;
}

__global__ void __launch_bounds__(kThreads, 1)
mla_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kn, const __grid_constant__ CUtensorMap map_kr,
                   const __grid_constant__ CUtensorMap map_v, const Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023u) & ~1023u;      // swizzled tiles
  uint8_t* sm = smem_raw + (sbase - raw);
  Misc& ms = *reinterpret_cast<Misc*>(sm + kOffMisc);
  const BlockWaiter wt{&ms.left, p.wait_limit};
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ms.k_full[i], 1); mbar_init(&ms.v_full[i], 1); mbar_init(&ms.k_free[i], 1); mbar_init(&ms.v_free[i], 1);
      mbar_init(&ms.q_full[i], 1); mbar_init(&ms.q_free[i], 1); mbar_init(&ms.s_ready[i], 1);
      mbar_init(&ms.p_ready[i][0], 4); mbar_init(&ms.p_ready[i][1], 4); mbar_init(&ms.half_done[i], 1);
      mbar_init(&ms.o_done[i], 1); mbar_init(&ms.work_full[i], 1); mbar_init(&ms.work_empty[i], 9);
    }
    mbar_init(&ms.clc, 1);
    mbar_init(&ms.drained, 1);
    ms.left = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_q); tma_prefetch_desc(&map_kn); tma_prefetch_desc(&map_kr); tma_prefetch_desc(&map_v);
  }
  if (warp == kWarpMma) {
    tmem_alloc_cta(&ms.tmem_base, 512);
    tmem_relinquish_cta();
  }
  pdl_wait();
  // tiles of a head and the longest tile's blocks
  int tiles = 0, most = 0;
  for (int b = (int)threadIdx.x; b < p.B; b += kThreads) {
    const int nq = max(start_of(p.cu_q, b + 1, p.B, p.Tq) - start_of(p.cu_q, b, p.B, p.Tq), 0);
    const int nk = max(start_of(p.cu_k, b + 1, p.B, p.Tk) - start_of(p.cu_k, b, p.B, p.Tk), 0);
    tiles += (nq + kPair - 1) / kPair;
    if (nq > 0) most = max(most, blocks_seen(nk));
  }
  tiles = __reduce_add_sync(0xffffffffu, tiles);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) { ms.scan[2 * warp] = tiles; ms.scan[2 * warp + 1] = most; }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  tiles = most = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) { tiles += ms.scan[2 * w]; most = max(most, ms.scan[2 * w + 1]); }
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem_base, 0);

  if (warp < 8) {
    // ------------------------------------------------------------ softmax of tile t, a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");     // 2 x 200 + 104 = 3 x 168, as launched
    const int t = warp >> 2, r = 32 * (warp & 3) + lane, rr = kRows * t + r;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_col = tmem + lane_base + 128 * t, o_col = tmem + lane_base + kTmemO + 128 * t;
    const float c = p.scale_log2;
    const uint64_t c2 = pack2(c, c);
    int ns = 0, no = 0, block0 = 0;                        // phases of s_ready and o_done; blocks of the works before this
    bool ok = true;
    for (int it = 0; ok; ++it) {
      ok = __all_sync(0xffffffffu, mbar_wait(&ms.work_full[it & 1], (it >> 1) & 1, wt, kSiteWork, it));
      if (!ok) break;
      const Work k = ms.work[it & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.work_empty[it & 1]);
      if (!k.live) break;
      const int lim = p.causal ? min(k.nk, k.lim0 + rr) : k.nk;
      const int low = p.causal ? min(k.nk, k.lim0 + kRows * t) : k.nk;       // what the tile's first row sees
      float m = kMInit, l = 0.f;
      for (int i = 0; i < k.n[t]; ++i, ++ns) {
        ok = __all_sync(0xffffffffu, mbar_wait(&ms.s_ready[t], ns & 1, wt, kSiteS, i));
        if (!ok) break;
        tc_fence_after();
        const int key0 = (k.b0 + i) * kBlock;
        const int valid = k.nk - key0;
        if (valid < kBlock) {
          // Value rows behind the sequence's end: zeros, whatever lies there.  (Both tiles write them; the block's other granules are
          // in nobody's way, and the slots are not given back before this tile's PV.)
          const int from = max(valid, 0), b = block0 + i;
          ok = __all_sync(0xffffffffu, mbar_wait(&ms.v_full[b & 1], (b >> 1) & 1, wt, kSiteFull, i)) && ok;
#pragma unroll 1
          for (int j = 3; j < kPerBlock; ++j) {
            const int g = kPerBlock * b + j;
            const uint32_t base = sbase + kOffRing + (uint32_t)(g & 7) * kGranule;
            for (int x = r; x < (kBlock - from) * 8; x += kRows)
              asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(base + from * 128 + 16 * x), "r"(0) : "memory");
          }
          fence_proxy_async_smem();
        }
        // The block's two halves one after the other: the first one's product runs while the second is computed.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int seen = lim - key0 - 64 * h;
          const bool masked = key0 + 64 * (h + 1) > low;
          uint32_t w[32];
          for (bool anew = i + h == 0;;) {
            float v[2][32];
            tmem_ld32(s_col + 64 * h, v[0]);
            tmem_ld32(s_col + 64 * h + 32, v[1]);
            tmem_wait_ld();
            if (masked)
#pragma unroll
              for (int x = 0; x < 64; ++x) v[x >> 5][x & 31] = x < seen ? v[x >> 5][x & 31] : -INFINITY;
            if (anew) {
              float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int x = 0; x < 64; x += 8)
#pragma unroll
                for (int z = 0; z < 4; ++z) mx[z] = fmaxf(mx[z], fmaxf(v[x >> 5][(x & 31) + z], v[x >> 5][(x & 31) + z + 4]));
              const float now = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))), f = fast_exp2((m - now) * c);
              m = now;
              l *= f;
              if (i + h > 0) {
                // (the PV of the block before is complete where S is there; that of this one's first half, if this is the second, has been issued)
                if (h > 0) {
                  ok = __all_sync(0xffffffffu, mbar_wait(&ms.half_done[t], ns & 1, wt, kSiteP, i)) && ok;
                  tc_fence_after();
                }
#pragma unroll 1
                for (int x = 0; x < 128; x += 32) {
                  float o[32];
                  tmem_ld32(o_col + x, o);
                  tmem_wait_ld();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] *= f;
                  tmem_st32(o_col + x, o);
                }
              }
            }
            const float mc = -m * c;
            const uint64_t m2 = pack2(mc, mc);
            uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              const float2 e = unpack2(fma2(pack2(v[y >> 4][2 * (y & 15)], v[y >> 4][2 * (y & 15) + 1]), c2, m2));
              const float2 r = make_float2(fast_exp2(e.x), fast_exp2(e.y));
              sum[y & 3] = add2(sum[y & 3], pack2(r.x, r.y));
              w[y] = bf16x2(r.x, r.y);
            }
            const float2 both = unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])));
            if (anew || !__any_sync(0xffffffffu, !(both.x + both.y <= kMostSum))) {
              l += both.x + both.y;
              break;
            }
            anew = true;
          }
          tmem_st16(s_col + 32 * h, w);
          tmem_st16(s_col + 32 * h + 16, w + 16);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ms.p_ready[t][h]);
        }
      }
      if (!ok) break;
      block0 += max(k.n[0], k.n[1]);
      // epilogue
      const bool mine = rr < k.rows;
      const long long row = (long long)(k.q0 + rr) * p.heads + k.head, prow = (long long)k.part * kPair + rr;
      if (k.n[t] > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&ms.o_done[t], no & 1, wt, kSiteO, it));
        if (!ok) break;
        ++no;
        tc_fence_after();
      }
      const float f = l != 0.f ? 1.f / l : 0.f;
      if (mine) {
        if (k.part < 0) p.lse[row] = l != 0.f ? (m * c + __log2f(l)) * kLn2 : INFINITY;     // (NaN: a score was none)
        else p.part_ml[prow] = make_float2(m * c, l);
      }
      if (k.part < 0) {
        uint4* dst = reinterpret_cast<uint4*>(p.out + row * (2 * kDV));
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          float o[32];
          if (k.n[t] > 0) {                                                 // warp-uniform
            tmem_ld32(o_col + 32 * x, o);
            tmem_wait_ld();
          }
          if (mine) {
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              uint32_t w[4];
#pragma unroll
              for (int z = 0; z < 4; ++z) w[z] = l != 0.f ? bf16x2(o[8 * y + 2 * z] * f, o[8 * y + 2 * z + 1] * f) : 0u;   // without keys: 0
              dst[4 * x + y] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      } else if (k.n[t] > 0) {
        float4* dst = reinterpret_cast<float4*>(p.part_o + prow * kDV);
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {
          float o[32];
          tmem_ld32(o_col + 32 * x, o);
          tmem_wait_ld();
          if (mine)
#pragma unroll
            for (int y = 0; y < 8; ++y) dst[8 * x + y] = make_float4(o[4 * y], o[4 * y + 1], o[4 * y + 2], o[4 * y + 3]);
        }
      }
      tc_fence_before();
    }
  } else {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
   if (warp == kWarpMma) {
    // ------------------------------------------------------------ the products (one thread: elected, so that the compiler knows the
    // descriptors to be the warp's; under a branch on the lane a product took 110 to 130 cycles to issue, of which it computes 64)
    if (elect_one()) {
      constexpr uint32_t idesc_qk = umma_idesc(1, 1, false, false, 128, 128), idesc_pv = umma_idesc(1, 1, false, true, 128, 128),
                         idesc_half = umma_idesc(1, 1, false, true, 128, 64);
      const uint64_t q_desc = umma_desc(sbase + kOffQ, 16, 1024, kSwz128), k_desc = umma_desc(sbase + kOffRing, 16, 1024, kSwz128),
                     v_desc = umma_desc(sbase + kOffRing, kGranule, 1024, kSwz128);
      // A tile's second product of a block is issued in front of its next first one, of the next work if there is no more in this: while
      // the tile with the longer reach finishes a work, the other begins the next.
      struct Due { int b, first, last, wait_v, free_v; };     // block, whether O begins and ends with it, whether V is first or last used
      Due due[2];
      int nq[2] = {0, 0}, np[2] = {0, 0}, block0 = 0;
      bool has[2] = {false, false}, ok = true;
      auto pv = [&](int t) {
        if (!has[t]) return;
        has[t] = false;
        const Due& x = due[t];
        const int b = x.b, g = kPerBlock * b + 3;
        if (x.wait_v && !(ok = mbar_wait(&ms.v_full[b & 1], (b >> 1) & 1, wt, kSiteFull, b))) return;
        const uint32_t d = tmem + kTmemO + 128 * t, a = tmem + 128 * t;
        const uint64_t v0 = v_desc + (uint32_t)(g & 7) * (kGranule >> 4);
        const bool split = (g & 7) == 7;                      // the block's two granules of V lie at the ring's two ends
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!(ok = mbar_wait(&ms.p_ready[t][h], np[t] & 1, wt, kSiteP, b))) return;
          tc_fence_after();
          if (!split) {
#pragma unroll
            for (int y = 4 * h; y < 4 * h + 4; ++y) mma_ts(d, a + 8 * y, v0 + 128 * y, idesc_pv, y == 0 && x.first ? 0u : 1u);
          } else {
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
              for (int y = 4 * h; y < 4 * h + 4; ++y) mma_ts(d + 64 * z, a + 8 * y, (z ? v_desc : v0) + 128 * y, idesc_half, y == 0 && x.first ? 0u : 1u);
          }
          if (h == 0) mma_commit_cta(&ms.half_done[t]);
        }
        ++np[t];
        if (x.free_v) mma_commit_cta(&ms.v_free[b & 1]);
        if (x.last) mma_commit_cta(&ms.o_done[t]);
      };
      for (int it = 0; ok; ++it) {
        if (!mbar_test(&ms.work_full[it & 1], (it >> 1) & 1)) {            // nothing to go on with yet
          pv(0);
          if (ok) pv(1);
        }
        if (!ok || !(ok = mbar_wait(&ms.work_full[it & 1], (it >> 1) & 1, wt, kSiteWork, it))) break;
        const Work& k = ms.work[it & 1];
        const int n0 = k.n[0], n1 = k.n[1], live = k.live, n = max(n0, n1);
        mbar_arrive(&ms.work_empty[it & 1]);
        if (!live) break;
        // Q_t K(i) writes S over the P that P_t V(i - 1) reads.  Both are issued by this thread, and a CTA's products go through its
        // tensor core in the order of issue: the reads of the earlier are behind it when the later's first results are written.
        for (int i = 0; i < n && ok; ++i)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int mine = t ? n1 : n0, others = t ? n0 : n1, b = block0 + i;
            if (ok) pv(t);
            if (!ok || i >= mine) continue;
            const bool first_user = t == 0 || i >= others, last_user = t == 1 || i >= others;
            if (i == 0) {
              if (!(ok = mbar_wait(&ms.q_full[t], nq[t] & 1, wt, kSiteQ, it))) continue;
              ++nq[t];
            }
            if (first_user && !(ok = mbar_wait(&ms.k_full[b & 1], (b >> 1) & 1, wt, kSiteFull, i))) continue;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 3; ++j) {
              const uint64_t kd = k_desc + (uint32_t)((kPerBlock * b + j) & 7) * (kGranule >> 4), qd = q_desc + ((kQTile * t + kGranule * j) >> 4);
#pragma unroll
              for (int x = 0; x < 4; ++x) mma_ss(tmem + 128 * t, qd + 2 * x, kd + 2 * x, idesc_qk, (uint32_t)(j | x));
            }
            mma_commit_cta(&ms.s_ready[t]);
            if (last_user) mma_commit_cta(&ms.k_free[b & 1]);
            if (i + 1 == mine) mma_commit_cta(&ms.q_free[t]);
            due[t] = Due{b, i == 0, i + 1 == mine, first_user, last_user};
            has[t] = true;
          }
        block0 += n;
      }
      if (ok) pv(0);
      if (ok) pv(1);
      if (!ok) {                                              // given up: what has been issued ends before the tensor memory goes
        mma_commit_cta(&ms.drained);
        mbar_drain(&ms.drained, 0);
      }
    }
    __syncwarp();
   } else if (warp == kWarpLoad) {
    // ------------------------------------------------------------ work and loads (one warp; lane 0 waits and issues)
    const int tiles_all = tiles * p.heads;
    const Cut cut = cut_of(tiles_all, most, p, lane);
    const Order order = order_of(tiles, most, p, lane);
    const uint64_t once = l2_policy_evict_first();
    uint64_t keep;
    asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(keep));
    int w = (int)blockIdx.x, block0 = 0, asked[2] = {0, 0}, nq[2] = {0, 0}, clc_asked = 0, clc_got = 0;
    bool ok = true;
    for (int it = 0; ok;) {
      if (w == 0 && lane == 0 && p.plan) *p.plan = make_int4(tiles, cut.whole, cut.pieces, p.epoch);
      Work k;
      k.live = 0;
      if (w >= 0) k = work_of(w, order, cut, p, lane);
      if (w >= 0 && lane == 0) {                              // ask for the next while this one is loaded
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(&ms.clc, 16);
        clc_ask(&ms.clc_answer, &ms.clc);
      }
      if (w >= 0) ++clc_asked;
      if (k.live || w < 0) {
        if (lane == 0) {
          ok = it < 2 || mbar_wait(&ms.work_empty[it & 1], ((it >> 1) & 1) ^ 1, wt, kSiteWorkEmpty, it);
          if (ok) {
            ms.work[it & 1] = k;
            mbar_arrive(&ms.work_full[it & 1]);
          }
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        if (!ok || w < 0) break;
        if (lane == 0) {
          auto load_q = [&](int t) {
            if (k.n[t] == 0 || (nq[t] > 0 && !(ok = mbar_wait(&ms.q_free[t], (nq[t] - 1) & 1, wt, kSiteQFree, it)))) return;
            mbar_arrive_expect_tx(&ms.q_full[t], kQTile);
            for (int j = 0; j < 3; ++j)
              tma_load_3d_hint(sbase + kOffQ + kQTile * t + kGranule * j, &map_q, 64 * j, k.head, k.q0 + kRows * t, &ms.q_full[t], once);
            ++nq[t];
          };
          load_q(0);
          const int n = max(k.n[0], k.n[1]);
          for (int i = 0; i < n && ok; ++i) {
            const int at = k.k0 + (k.b0 + i) * kBlock;
            // Granule g takes the place of g - 8: of K's last of two blocks before, V's two, and K's first two of the block before.
            const int b = block0 + i;
            for (int j = 0; j < kPerBlock; ++j) {
              uint64_t* bar = j < 3 ? &ms.k_full[b & 1] : &ms.v_full[b & 1];
              const uint32_t dst = sbase + kOffRing + (uint32_t)((kPerBlock * b + j) & 7) * kGranule;
              const int old = j < 3 ? b - 2 : b - 1;
              if (i == 0 && j == 3) load_q(1);                // (the other tile can still be at work with its Q)
              if (!ok) break;
              if (old >= 0 && j != 2 && j != 4) {
                uint64_t* freed = j == 1 ? &ms.v_free[old & 1] : &ms.k_free[old & 1];
                if (!(ok = mbar_wait(freed, (old >> 1) & 1, wt, kSiteEmpty, i))) break;
              }
              if (j == 0 || j == 3) {
                mbar_arrive_expect_tx(bar, (j == 0 ? 3 : 2) * kGranule);
                ++asked[j == 3];
              }
              if (j < 2) tma_load_3d_hint(dst, &map_kn, 64 * j, k.head, at, bar, keep);
              else if (j == 2) tma_load_2d_hint(dst, &map_kr, 0, at, bar, keep);
              else tma_load_3d_hint(dst, &map_v, 64 * (j - 3), k.head, at, bar, keep);
            }
          }
          block0 += n;
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
        ++it;
      }
      if (!ok) break;
      int next = -1;
      if (lane == 0) {
        ok = mbar_wait(&ms.clc, clc_got & 1, wt, kSiteClc, it);
        if (ok) next = clc_block(&ms.clc_answer);
      }
      ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
      if (ok) ++clc_got;
      w = __shfl_sync(0xffffffffu, next, 0);
    }
    if (!ok && lane == 0) {                                   // given up: what is in flight lands first
      // (K's last granules may not have been requested: then the barrier's phase does not end, and the limit does)
      for (int b = max(asked[0] - 2, 0); b < asked[0]; ++b) mbar_drain(&ms.k_full[b & 1], (b >> 1) & 1);
      for (int b = max(asked[1] - 2, 0); b < asked[1]; ++b) mbar_drain(&ms.v_full[b & 1], (b >> 1) & 1);
      for (int t = 0; t < 2; ++t)
        if (nq[t] > 0) mbar_drain(&ms.q_full[t], (nq[t] - 1) & 1);
      if (clc_asked > clc_got) mbar_drain(&ms.clc, clc_got & 1);
    }
    __syncwarp();
   }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpMma) tmem_dealloc_cta(tmem, 512);
  if (threadIdx.x == 0) {
    wt.report(g_status, p.epoch);
    if (blockIdx.x == 0) atomicAdd(&g_status[3], 1);
  }
}

// out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over the pieces of cut tile blockIdx.y; a warp has a row, eight pieces' loads under way
constexpr int kMergeWarps = 8;
__global__ void __launch_bounds__(32 * kMergeWarps) mla_prefill_merge_kernel(const Params p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  const int4 plan = __ldcg(p.plan);
  const Cut cut{plan.y, plan.z};
  const int w0 = cut.whole + (int)blockIdx.y * cut.pieces, rr = (int)blockIdx.x * kMergeWarps + warp;
  if (plan.w != p.epoch) return;                              // a launch that gave up before it had a plan: whatever lies there is none
  if (cut.pieces < 2 || cut.whole + (int)blockIdx.y >= plan.x * p.heads) return;
  const Work k = work_of(w0, order_of(plan.x, 0, p, lane), cut, p, lane);
  if (!k.live || rr >= k.rows) return;
  const long long base = (long long)k.part * kPair + rr;
  float m = kMInit;
  for (int i = lane; i < cut.pieces; i += 32) {
    const float2 ml = __ldcg(p.part_ml + base + (long long)i * kPair);
    if (ml.y != 0.f) m = fmaxf(m, ml.x);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i0 = 0; i0 < cut.pieces; i0 += 8) {
    float4 v[8];
    float2 ml[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      ml[u] = make_float2(0.f, 0.f);
      if (i0 + u < cut.pieces) {
        const long long at = base + (long long)(i0 + u) * kPair;
        ml[u] = __ldcg(p.part_ml + at);
        v[u] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * kDV) + lane);
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (ml[u].y == 0.f) continue;                           // beyond the list, or a piece without keys for this row
      const float f = fast_exp2(ml[u].x - m);
      l += f * ml[u].y;
      a.x += f * v[u].x; a.y += f * v[u].y; a.z += f * v[u].z; a.w += f * v[u].w;
    }
  }
  const float f = l != 0.f ? 1.f / l : 0.f;
  const long long row = (long long)(k.q0 + rr) * p.heads + k.head;
  reinterpret_cast<uint2*>(p.out + row * (2 * kDV))[lane] = make_uint2(bf16x2(a.x * f, a.y * f), bf16x2(a.z * f, a.w * f));
  if (lane == 0) p.lse[row] = l != 0.f ? (m + __log2f(l)) * kLn2 : INFINITY;
}

// Pieces that a call's workspace holds: none where its tiles are known to be many, or its sequences too short to be cut; else what cut_of can
// come to: pieces of two blocks, of at most a tile a query and head and of fewer tiles than CTAs.
static int pieces_of(int Tq, int Tk, int heads) {
  const int ctas = sm_count(), blocks = blocks_seen(Tk);
  const int64_t tiles = (int64_t)((Tq + kPair - 1) / kPair) * heads;
  if (tiles > 4 * ctas || blocks < 4) return 0;
  return (int)min((int64_t)4 * ctas, min((int64_t)Tq * heads, (int64_t)max(ctas - 1, 1)) * (blocks / 2));
}

}  // namespace prefill
}  // namespace lt

extern "C" int64_t litedsa_mla_prefill_workspace(int Tq, int Tk, int heads) {
  if (Tq <= 0 || Tk <= 0 || heads <= 0) return 0;
  const int64_t n = lt::prefill::pieces_of(Tq, Tk, heads);
  return n == 0 ? 0 : 16 + n * lt::prefill::kPair * (lt::prefill::kDV * 4 + 8);
}

extern "C" int litedsa_mla_prefill(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k_nope, int64_t k_token_stride,
                                   int64_t k_head_stride, const void* k_rope, int64_t k_rope_stride, const void* v, int64_t v_token_stride,
                                   int64_t v_head_stride, const int32_t* cu_q, const int32_t* cu_k, int B, float sm_scale, int causal, void* out,
                                   float* lse, int Tq, int Tk, int heads, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace lt;
  using namespace lt::prefill;
  if (!q || !out || !lse || (Tk > 0 && (!k_nope || !k_rope || !v)) || (cu_q == nullptr) != (cu_k == nullptr)) {
    if (Tq != 0) return LITEDSA_ERR_ARG;
  }
  if (Tq < 0 || Tk < 0 || heads <= 0 || B < 0 || (!cu_q && B != 1)) return LITEDSA_ERR_SHAPE;
  if (!(sm_scale >= 0.f)) return LITEDSA_ERR_UNSUPPORTED;
  if (((uintptr_t)q | (uintptr_t)k_nope | (uintptr_t)k_rope | (uintptr_t)v | (uintptr_t)out | (uintptr_t)workspace) & 15 || ((uintptr_t)lse & 3) ||
      (q_token_stride | q_head_stride | k_token_stride | k_head_stride | k_rope_stride | v_token_stride | v_head_stride) % 8)
    return LITEDSA_ERR_UNSUPPORTED;
  // (a tensor map has no stride of 0)
  if ((Tq > 1 && q_token_stride <= 0) || (heads > 1 && q_head_stride <= 0) || (Tk > 1 && (k_token_stride <= 0 || k_rope_stride <= 0 || v_token_stride <= 0)) ||
      (Tk > 0 && heads > 1 && (k_head_stride <= 0 || v_head_stride <= 0)))
    return LITEDSA_ERR_UNSUPPORTED;
  if (Tq == 0 || B == 0) return LITEDSA_OK;
  const int64_t tiles = cu_q ? min((int64_t)Tq, Tq / kPair + (int64_t)B) : (Tq + kPair - 1) / kPair;
  Params p = {};
  p.max_pieces = pieces_of(Tq, Tk, heads);
  if (tiles * heads + p.max_pieces >= (1ll << 31) - 1) return LITEDSA_ERR_UNSUPPORTED;
  const int64_t need = litedsa_mla_prefill_workspace(Tq, Tk, heads);
  if (need > 0 && (!workspace || workspace_bytes < need)) return workspace ? LITEDSA_ERR_SHAPE : LITEDSA_ERR_ARG;
  p.cu_q = cu_q; p.cu_k = cu_k;
  p.out = reinterpret_cast<uint8_t*>(out); p.lse = lse;
  if (p.max_pieces) {
    p.plan = reinterpret_cast<int4*>(workspace);
    p.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + 16);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)p.max_pieces * kPair * kDV);
  }
  p.B = B; p.Tq = Tq; p.Tk = Tk; p.heads = heads; p.ctas = sm_count(); p.causal = causal != 0;
  p.scale_log2 = fmaxf(sm_scale * kLog2e, 1e-30f);           // not 0: masked scores are -inf before they are scaled
  p.epoch = next_launch_epoch(); p.wait_limit = wait_limit_ticks();
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto bf16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap mq, mn, mr, mv;
  // strides of dimensions of one are never used, but have to be such as a map can hold
  auto pitch = [](int64_t elements, int64_t n, int64_t least) -> uint64_t { return (uint64_t)(2 * (n > 1 ? elements : least)); };
  if (!make_map_3d(&mq, q, bf16, 192, heads, Tq, pitch(q_head_stride, heads, 192), pitch(q_token_stride, Tq, 192), 64, 1, kRows)) return LITEDSA_ERR_CUDA;
  mn = mr = mv = mq;
  if (Tk > 0 && (!make_map_3d(&mn, k_nope, bf16, 128, heads, Tk, pitch(k_head_stride, heads, 128), pitch(k_token_stride, Tk, 128), 64, 1, kBlock) ||
                 !make_map_2d(&mr, k_rope, bf16, 64, Tk, pitch(k_rope_stride, Tk, 64), 64, kBlock) ||
                 !make_map_3d(&mv, v, bf16, 128, heads, Tk, pitch(v_head_stride, heads, 128), pitch(v_token_stride, Tk, 128), 64, 1, kBlock)))
    return LITEDSA_ERR_CUDA;
  if (!ensure_smem<mla_prefill_kernel>(current_device(), kSmem)) return LITEDSA_ERR_CUDA;
  const int rc = launch_pdl(mla_prefill_kernel, dim3((unsigned)(tiles * heads + p.max_pieces)), kThreads, kSmem, st, mq, mn, mr, mv, p);
  if (rc != LITEDSA_OK || p.max_pieces == 0) return rc;
  return launch_pdl(mla_prefill_merge_kernel, dim3(kPair / kMergeWarps, (unsigned)min(tiles * heads, (int64_t)p.ctas)), 32 * kMergeWarps, 0, st, p);
}

// Status block of the kernel; layout and return rule as litedsa_attn_status.
extern "C" int litedsa_mla_prefill_status(int* out4_host, int reset) {
  using namespace lt::prefill;
  if (out4_host && cudaMemcpyFromSymbol(out4_host, g_status, sizeof(int) * 4) != cudaSuccess) return LITEDSA_ERR_CUDA;
  if (reset) {
    const int z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (cudaMemcpyToSymbol(g_status, z, sizeof(z)) != cudaSuccess) return LITEDSA_ERR_CUDA;
  }
  return (out4_host && out4_host[0] != 0) ? LITEDSA_ERR_TIMEOUT : LITEDSA_OK;
}
