// Absorbed latent attention over a paged cache (sm_100a): the decode step of MLA, dense.
//
//   s = sm_scale q . k[0:576], p = softmax of s over the keys a row sees, out = p k[0:512]
//
// for the rows (token j, head h) of every sequence; token j of q_len sees keys [0, len - q_len + 1 + j).
// One cache row serves all heads, so a CTA takes up to 64 rows of one sequence (a pair of CTAs more: mla_decode_pair.cuh) and streams
// its keys once, in blocks of 64:
//
//   S   [64 rows x 64 keys]    = Q K^T        (M = 64, N = 64: 36 steps of 16 dims, both operands in shared memory)
//   O^T [512 dims x R rows]   += V^T P^T      (M = 128 four times, N = R = 16, 32 or 64: A = the K tile itself, read along dims)
//
// The second product is taken transposed because O needs 512 columns of tensor memory for 128 lanes of rows, which leaves no
// room for S, but R columns for each of four times 128 lanes of dims; and because its cost then follows the rows that exist.  The row
// statistics stay per thread (S has rows on lanes), and only the rare rescaling of O wants them by column, from shared memory.
//
// Work is cut along the keys: the blocks of all sequences in a row are dealt to groups in equal shares (a group: a CTA; of more than 64 rows
// as many pairs of CTAs as a sequence has tiles of 128, which read the same keys at about the same time, once from memory and again from L2).  A share's
// pieces of sequences that other groups have parts of go to a workspace in fp32 and are merged by a second kernel.  Every size but those of the
// tensors is read on the device, so captured calls follow new lengths.
//
// Packed rows (512 e4m3 codes, four fp32 scales, 64 bf16) pass through registers: sixteen warps load a block ahead, convert it to
// bf16 (exact where the scales are powers of two) and write the same tile that TMA writes for bf16 rows.
//
// Bound by memory up to 16 rows, by the tensor cores from 64 on.  Measured: 5 sequences of 65 to 131 thousand keys, 16 heads, bf16, 113 us = 5.0 TB/s
// with the merge (a copy: 6.5), 103 in the first calls; 64 heads 127, 113 in the first calls; 32 sequences of up to 8191 packed keys, 64 heads, 51 us,
// where fifteen blocks a CTA take 3800 cycles each, the latency of loads, conversion, products and softmax over two slots, and start, pieces' ends and
// merge 20 us.
//
// A key beyond the sequence's end is in no product: its S is replaced, and its value row is zeroed before the second product, whatever its page holds.
// A row's sum of exponentials is 0 where it sees no key, and NaN where a score is NaN or +infinity: maxima pass NaN over, sums and products keep it, and the
// ends and the merge ask for a sum of 0, not for a positive one.
#include "common.cuh"
#include "tensor_map.cuh"

namespace lt {
namespace decode {

constexpr int kD = 576, kDV = 512;
constexpr int kBlock = 64;                                  // keys
constexpr int kChunks = kD / 64;
constexpr uint32_t kChunkBytes = kBlock * 128;              // 64 keys x 64 bf16
constexpr uint32_t kSlotBytes = kChunks * kChunkBytes;
constexpr int kSlots = 2;
constexpr int kMostStartCost = 5;                           // blocks
constexpr int kGroups = 5;                                  // a tile's chunks are loaded and given back in groups: four of 128 dims, the rope dims
// Warps 0-7: softmax.  Who loads: one warp by TMA (bf16 rows in pages of multiples of 64), 8 by cp.async (bf16 rows in other pages:
// a box is 16 rows then, and 36 boxes a block take a warp 3400 cycles to issue), 16 through registers (packed rows).  TMA / cp.async with pages of 64, us:
// 5 sequences of 65 to 131 thousand keys, 64 heads 127 / 132, 16 heads 113 / 116; 32 of up to 8191, 64 heads, 47 / 52; 64 of 1000 to 4000, 32 heads, 48 / 52.
// cp.async takes as long with pages of 16.
enum Load { kTma, kCopy, kPacked };
constexpr int kSoftmaxWarps = 8, kWarpQk = 8, kWarpPv = 9, kWarpQ = 10, kWarpTma = 11, kWarpLoad0 = 12;
template <Load kLoad> constexpr int kLoadWarps = kLoad == kTma ? 0 : kLoad == kCopy ? 8 : 16;
template <Load kLoad> constexpr int kThreads = 32 * (kWarpLoad0 + kLoadWarps<kLoad>);
constexpr int kPackedRow = 656;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kMInit = -1e30f;
// The running maximum that P is relative to moves only when a row overshoots it by this much (in powers of two): P is at most 2^8,
// as exact in bf16 as below one, and O is rarely rescaled.
constexpr float kOvershoot = 8.f;

template <int kRows>
struct Plan {
  static constexpr uint32_t kQChunk = kRows * 128;
  static constexpr uint32_t kOffQ = 0;                      // rows behind kRows that the M = 64 operand covers are whatever lies there
  static constexpr uint32_t kOffKV = (kChunks * kQChunk + 1023) / 1024 * 1024;
  static constexpr uint32_t kOffMisc = kOffKV + kSlots * kSlotBytes;
  static constexpr uint32_t kSmem = kOffMisc + 2048 + 1024;
  static constexpr uint32_t kTmemS = 4 * kRows;             // columns: O^T, then two S
  static constexpr uint32_t kTmemCols = 4 * kRows + 128 <= 256 ? 256 : 512;
  static_assert(kQChunk % 1024 == 0 && (kChunks - 1) * kQChunk + 64 * 128 <= kOffMisc, "the operand ends inside");
  static_assert(kSmem <= 232448, "shared memory");
};

struct Misc {
  uint64_t kv_full[kSlots][kGroups], kv_free[kSlots][kGroups], s_ready[2], p_ready[2], q_ready, q_free, drained[2];
  uint32_t left, tmem_base;
  int start_b, start_k, count, meta_groups;
  long long start_pos, total;
  int scan[32];
  float corr[64], top[2][64], sum[2][64];
};
static_assert(sizeof(Misc) <= 2048, "Misc");

struct Params {
  const uint8_t* q;               // [B, q_len, heads, 576] bf16, byte pitches
  long long q_b, q_j, q_h;
  const uint8_t* cache;           // packed rows
  long long block_pitch;
  const int32_t* table;           // [B, cols]
  long long table_pitch;
  const int32_t* lens;
  uint8_t* out;                   // [B, rows, 512] bf16
  float* lse;                     // [B, rows]
  float* part_o;                  // [CTA or pair][2][rows of its tile][512]
  float2* part_ml;                // [CTA or pair][2][rows of its tile]: (maximum, sum)
  int4* meta;                     // [groups]: (sequence, slot, parts, 0) of a sequence that begins here and ends in another group, or (-1, ..)
  int flat_q;                     // a sequence's rows are evenly spaced: they come by TMA
  int B, q_len, heads, rows, row_tiles, groups, cols, block_size, n_blocks, box_rows, start_cost;      // row_tiles: pairs to a group; box_rows: of a pair's loads
  float scale_log2;
  int epoch;
  uint32_t wait_limit;
};

enum { kSiteKv = 1, kSiteS, kSiteP, kSitePv, kSiteQ, kSiteFree, kSiteVote, kSiteAid, kSiteAlign };
static __device__ int g_status[8];

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// The page and the row in it of a key that moves on by a block at a time: a division took a loading warp 200 cycles, five a block.
struct PageAt {
  int size, add_page, add_row, page, row;
  __device__ __forceinline__ explicit PageAt(int block_size) : size(block_size), add_page(kBlock / block_size), page(0), row(0) { add_row = kBlock - add_page * size; }
  __device__ __forceinline__ void at(int key) {
    page = key / size;
    row = key - page * size;
  }
  __device__ __forceinline__ void advance() {
    page += add_page;
    row += add_row;
    if (row >= size) { row -= size; ++page; }
  }
};
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool softmax_any(bool x) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"((uint32_t)x) : "memory");
  return r != 0;
}

__device__ __forceinline__ int len_of(const Params& p, int b) {
  return (int)min((long long)max(__ldcg(p.lens + b), 0), (long long)p.cols * p.block_size);
}
__device__ __forceinline__ int blocks_of(int len) { return max((len + kBlock - 1) / kBlock, 1); }      // an empty sequence: one masked block

// Walks a CTA's share: blocks [k0, k1) of sequence b, piece by piece.
struct Walk {
  int b, k0, k1, nb, len, left, index;
  template <class M>
  __device__ __forceinline__ Walk(const M& ms) : b(ms.start_b - 1), k0(0), k1(ms.start_k), nb(0), len(0), left(ms.count), index(-1) {}
  __device__ __forceinline__ bool next(const Params& p) {
    if (left <= 0) return false;
    k0 = index < 0 ? k1 : 0;
    ++b; ++index;
    len = len_of(p, b);
    nb = blocks_of(len);
    k1 = min(nb, k0 + left);
    left -= k1 - k0;
    return true;
  }
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == nb; }
};

// Where a loading warp's rows of a block lie, for the blocks that it comes to: lane i has those of the i-th from the last look on.  Looked up thirty
// at a time: a look and its divisions a block took such a warp 400 to 1000 cycles, a third of what a block takes.
template <bool kTwo>
struct Ahead {
  Walk w;
  int at, i, offset, own;                                   // rows [offset, offset + own) of each block
  bool more;
  int page, row, n, page2;                                  // n of them hold keys; n_blocks: a page beyond the cache, or none; page2: of rows from 16 on
  template <class M>
  __device__ __forceinline__ Ahead(const M& ms, const Params& p, int first, int rows, int lane) : w(ms), i(0), offset(first), own(rows), page(0), row(0), n(0), page2(0) {
    more = w.next(p);
    at = w.k0;
    fill(p, 0, lane);
  }
  __device__ __forceinline__ void fill(const Params& p, int filled, int lane) {
    if (lane >= filled) { page = page2 = p.n_blocks; row = n = 0; }
    while (more && filled < 32) {
      const int take = min(32 - filled, w.k1 - at);
      if (lane >= filled && lane < filled + take) {
        const int key = (at + lane - filled) * kBlock + offset;
        n = min(max(w.len - key, 0), own);
        if (n > 0) {
          const int c = key / p.block_size;
          const int* from = p.table + w.b * p.table_pitch + c;
          row = key - c * p.block_size;
          page = __ldcg(from);
          if ((unsigned)page >= (unsigned)p.n_blocks) page = p.n_blocks;
          if (kTwo) {
            page2 = n > 16 && row + 16 >= p.block_size ? __ldcg(from + 1) : page;
            if ((unsigned)page2 >= (unsigned)p.n_blocks) page2 = p.n_blocks;
          }
        }
      }
      filled += take;
      at += take;
      if (at == w.k1) { more = w.next(p); at = w.k0; }
    }
  }
  __device__ __forceinline__ void advance(const Params& p, int lane) {
    if (++i < 30) return;
    page = __shfl_down_sync(0xffffffffu, page, 30);
    row = __shfl_down_sync(0xffffffffu, row, 30);
    n = __shfl_down_sync(0xffffffffu, n, 30);
    if (kTwo) page2 = __shfl_down_sync(0xffffffffu, page2, 30);
    i = 0;
    fill(p, 2, lane);
  }
  // of the block d = 0, 1, 2 from the current one
  __device__ __forceinline__ int rows_in(int d) const { return __shfl_sync(0xffffffffu, n, i + d); }
  __device__ __forceinline__ const uint8_t* rows_of(const Params& p, int d, int row_bytes) const {           // none: nullptr
    const int x = __shfl_sync(0xffffffffu, page, i + d), r = __shfl_sync(0xffffffffu, row, i + d);
    return x < p.n_blocks ? p.cache + (long long)x * p.block_pitch + (long long)r * row_bytes : nullptr;
  }
};

// Group g's share: [g total / groups, (g + 1) total / groups) of all sequences' blocks in a row, a sequence preceded by p.start_cost blocks that nobody
// has: what its beginning, another piece for somebody, costs.  All threads of a block; ms.count is 0 before.
template <class M>
__device__ __forceinline__ void find_share(const Params& p, M& ms, int g, int warp, int lane) {
  const int nt = (int)blockDim.x, per = (p.B + nt - 1) / nt;
  const int b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) mine += blocks_of(len_of(p, b)) + p.start_cost;
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) ms.scan[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  int before = incl - mine, total = 0;
  for (int w = 0; w < nt / 32; ++w) {
    if (w < warp) before += ms.scan[w];
    total += ms.scan[w];
  }
  const int used = min(p.groups, total);
  if (g < used) {
#pragma unroll
    for (int end = 0; end < 2; ++end) {
      const int x = (int)((long long)(g + end) * total / used);
      if (x == total) {
        if (threadIdx.x == 0) atomicAdd(&ms.count, total - p.B * p.start_cost);
      } else if (x >= before && x < before + mine) {
        int at = before, b = b0;
        for (;; ++b) {
          const int n = blocks_of(len_of(p, b)) + p.start_cost;
          if (x < at + n) break;
          at += n;
        }
        const int k = max(x - at - p.start_cost, 0), blocks = at - b * p.start_cost + k;      // before x
        atomicAdd(&ms.count, end ? blocks : -blocks);
        if (end == 0) {
          ms.start_b = b; ms.start_k = k;
          ms.start_pos = at; ms.total = total; ms.meta_groups = used;
        }
      }
    }
  }
  __syncthreads();
}

// which sequence of group g others have the rest of
template <class M>
__device__ __forceinline__ void write_meta(const Params& p, const M& ms, int g) {
  int4 e = make_int4(-1, 0, 0, 0);
  Walk w(ms);
  long long end = ms.start_pos;
  while (w.next(p)) {
    end += p.start_cost + w.nb;                                           // behind the sequence's last block
    if (w.k0 == 0 && w.k1 < w.nb) e = make_int4(w.b, w.index == 0 ? 0 : 1, (int)((end * ms.meta_groups - 1) / ms.total) - g + 1, 0);
  }
  p.meta[g] = e;
}

// 16 e4m3 codes x scale -> 16 bf16
__device__ __forceinline__ void convert16(const uint4& c, float scale, uint4& a, uint4& b) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i] >> (16 * k)), __NV_E4M3);
      float2 f = __half22float2(__half2(h));
      asm("{\n\t.reg .b64 x, s;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 s, {%2, %2};\n\tmul.rn.f32x2 x, x, s;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(f.x), "+f"(f.y) : "f"(scale));
      o[2 * i + k] = bf16x2(f.x, f.y);
    }
  }
  a = make_uint4(o[0], o[1], o[2], o[3]);
  b = make_uint4(o[4], o[5], o[6], o[7]);
}

__device__ __forceinline__ void st_shared16(uint32_t a, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void st_shared4(uint32_t a, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }

template <int kRows, Load kLoad>
__global__ void __launch_bounds__(kThreads<kLoad>, 1)
mla_decode_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_q, const Params p) {
  using PL = Plan<kRows>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), sbase = (raw + 1023u) & ~1023u;      // swizzled tiles
  uint8_t* sm = smem_raw + (sbase - raw);
  Misc& ms = *reinterpret_cast<Misc*>(sm + PL::kOffMisc);
  const BlockWaiter wt{&ms.left, p.wait_limit};
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const int g = (int)blockIdx.x;
  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i)
      for (int j = 0; j < kGroups; ++j) { mbar_init(&ms.kv_full[i][j], kLoad == kTma ? 1 : kLoad == kCopy ? 32 * kLoadWarps<kCopy> : kLoadWarps<kPacked>); mbar_init(&ms.kv_free[i][j], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&ms.s_ready[i], 1); mbar_init(&ms.p_ready[i], kSoftmaxWarps); }
    mbar_init(&ms.q_ready, 1);
    mbar_init(&ms.q_free, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&ms.drained[i], 1);
    ms.left = 0;
    ms.count = 0;
    fence_mbar_init();
    if (kLoad == kTma) tma_prefetch_desc(&map_kv);
    if (p.flat_q) tma_prefetch_desc(&map_q);
  }
  if (warp == kWarpQk) {
    tmem_alloc_cta(&ms.tmem_base, PL::kTmemCols);
    tmem_relinquish_cta();
  }
  pdl_wait();
  find_share(p, ms, g, warp, lane);
  const uint32_t tmem = __shfl_sync(0xffffffffu, ms.tmem_base, 0);

  if (warp < kSoftmaxWarps) {
    // ------------------------------------------------------------ softmax, epilogue
    // A warp has 16 rows and half of a block's keys: lane l rows l / 4 and l / 4 + 8, of every 8 keys the pair 2 (l % 4).
    const int quarter = warp & 3, half = warp >> 2, r0 = 16 * quarter + (lane >> 2), qd = lane & 3;
    const bool live = 16 * quarter < kRows;
    const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
    Walk w(ms);
    int kb = 0;
    // A wait here that gives up is passed like any other: the warps meet at named barriers, so they take the same steps.  (A warp's lanes may give up at
    // different times: they meet again before the warp reads tensor memory.)
    bool more = w.next(p);
    while (more) {
      // rows' limits
      int lim[2], low;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lim[i] = min(w.len, w.len - p.q_len + 1 + (r0 + 8 * i) / p.heads);
      }
      low = w.len - p.q_len + 1;                                          // what the first row sees
      float m[2] = {kMInit, kMInit}, l[2] = {0.f, 0.f};
      for (int k = w.k0; k < w.k1; ++k, ++kb) {
        mbar_wait(&ms.s_ready[kb & 1], (kb >> 1) & 1, wt, kSiteS, kb);
        __syncwarp();
        tc_fence_after();
        float v[16];
        float mx[2] = {-INFINITY, -INFINITY};
        if (live) {
          tmem_ld_16x256b_x4(tmem + PL::kTmemS + 64 * (kb & 1) + 32 * half + lane_base, v);
          tmem_wait_ld();
          if ((k + 1) * kBlock > low) {
            const int key0 = k * kBlock + 32 * half + 2 * qd;
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = key0 + 8 * (e >> 2) + (e & 1) < lim[(e >> 1) & 1] ? v[e] * p.scale_log2 : -INFINITY;
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] *= p.scale_log2;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) mx[(e >> 1) & 1] = fmaxf(mx[(e >> 1) & 1], v[e]);
        }
        const bool first = k == w.k0;
        if (softmax_any(first || mx[0] > m[0] + kOvershoot || mx[1] > m[1] + kOvershoot)) {
          // the rows' maxima over the block, and O relative to them
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            if (live && qd == 0) ms.top[half][r0 + 8 * i] = mx[i];
          }
          softmax_sync();
          if (live) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float now = fmaxf(m[i], fmaxf(ms.top[0][r0 + 8 * i], ms.top[1][r0 + 8 * i])), f = fast_exp2(m[i] - now);
              m[i] = now;
              l[i] *= f;
              if (half == 0 && qd == 0) ms.corr[r0 + 8 * i] = f;
            }
          }
          if (!first) {
            softmax_sync();
            mbar_wait(&ms.kv_free[(kb - 1) & 1][kGroups - 1], ((kb - 1) >> 1) & 1, wt, kSitePv, kb);
            __syncwarp();
            tc_fence_after();
#pragma unroll 1
            for (int c = 2 * kRows * half; c < 2 * kRows * (half + 1); c += 16) {
              float o[16];
              tmem_ld16(tmem + lane_base + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= ms.corr[(c & (kRows - 1)) + e];
              tmem_st16(tmem + lane_base + c, o);
            }
            tmem_wait_st();
          }
        }
        const uint32_t slot = sbase + PL::kOffKV + (kb & 1) * kSlotBytes;
        if (live) {
          // P takes the place of the block's rope dims, which the first product was the last to read
          const uint32_t prow = slot + (kChunks - 1) * kChunkBytes + r0 * 128 + 4 * qd;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              e[x] = fast_exp2(v[4 * i + x] - m[x >> 1]);
              l[x >> 1] += e[x];
            }
            const uint32_t at = prow + (((4 * half + i) ^ (r0 & 7)) << 4);
            st_shared4(at, bf16x2(e[0], e[1]));
            st_shared4(at + 8 * 128, bf16x2(e[2], e[3]));
          }
        }
        const int valid = w.len - k * kBlock;
        if (valid < kBlock) {                                             // value rows behind the end: nothing, whatever the page holds
          const int from = max(valid, 0);
          for (int i = (int)threadIdx.x; i < (kBlock - from) * 64; i += 32 * kSoftmaxWarps)
            st_shared16(slot + (uint32_t)((i >> 3) & 7) * kChunkBytes + (from + (i >> 6)) * 128 + (i & 7) * 16, make_uint4(0, 0, 0, 0));
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ms.p_ready[kb & 1]);
      }
      // epilogue: O^T has dims on lanes; a warp writes 32 dims of a row at a time, half of the columns
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (live && qd == 0) ms.sum[half][r0 + 8 * i] = l[i];
      }
      const bool whole = w.whole();
      const int slot = g * 2 + (w.index == 0 ? 0 : 1);
      softmax_sync();
      if (live && half == 0 && qd == 0)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 8 * i;
          const float sum = ms.sum[0][r] + ms.sum[1][r];
          ms.corr[r] = whole ? (sum != 0.f ? 1.f / sum : 0.f) : 1.f;
          if (whole) {
            if (r < p.rows) p.lse[(long long)w.b * p.rows + r] = sum != 0.f ? (m[i] + __log2f(sum)) * kLn2 : INFINITY;
          } else {
            p.part_ml[(long long)slot * kRows + r] = make_float2(m[i], sum);
          }
        }
      softmax_sync();
      mbar_wait(&ms.kv_free[(kb - 1) & 1][kGroups - 1], ((kb - 1) >> 1) & 1, wt, kSitePv, kb);
      __syncwarp();
      tc_fence_after();
      float o[2][16];
      tmem_ld16(tmem + lane_base + 2 * kRows * half, o[0]);
#pragma unroll 1
      for (int c0 = 2 * kRows * half; c0 < 2 * kRows * (half + 1); c0 += 32) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {                                     // (the next columns come while these are written)
          const int c = c0 + 16 * u, r = c & (kRows - 1), d = c / kRows * 128 + 32 * quarter + lane;
          tmem_wait_ld();
          if (c + 16 < 2 * kRows * (half + 1)) tmem_ld16(tmem + lane_base + c + 16, o[u ^ 1]);
          if (whole) {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.out) + ((long long)w.b * p.rows + r) * kDV + d;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (r + e < p.rows) {
                const float f = ms.corr[r + e];
                dst[e * kDV] = __float2bfloat16(f != 0.f ? o[u][e] * f : 0.f);     // a row without keys: 0, whatever the values of others
              }
          } else {
            float* dst = p.part_o + ((long long)slot * kRows + r) * kDV + d;
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (r + e < p.rows) dst[e * kDV] = o[u][e];
          }
        }
      }
      tc_fence_before();
      more = w.next(p);
    }
  } else if (warp == kWarpQk) {
    // ------------------------------------------------------------ S = Q K^T (one thread)
    // Two threads issue the products: with one, the second product of a block would wait behind the keys of the next.  S is free
    // when a block's keys are there: its slot was given back by the second product of the block that had it, and the S, before.
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc(1, 1, false, false, 64, kBlock);
      const uint64_t q_desc = umma_desc(sbase + PL::kOffQ, 16, 1024, kSwz128);
      Walk w(ms);
      int kb = 0;
      bool ok = true;
      while (ok && w.next(p)) {
        if (!(ok = mbar_wait(&ms.q_ready, w.index & 1, wt, kSiteQ, kb))) break;
        for (int k = w.k0; ok && k < w.k1; ++k, ++kb) {
          const uint64_t kd = umma_desc(sbase + PL::kOffKV + (kb & 1) * kSlotBytes, 16, 1024, kSwz128);
          const uint32_t d = tmem + PL::kTmemS + 64 * (kb & 1);
#pragma unroll 1
          for (int j = 0; j < kChunks; ++j) {
            if ((j & 1) == 0) {
              if (!(ok = mbar_wait(&ms.kv_full[kb & 1][j >> 1], (kb >> 1) & 1, wt, kSiteKv, kb))) break;
              if (kLoad == kCopy) fence_proxy_async_smem();               // what cp.async wrote, for the tensor core
              tc_fence_after();
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
              mma_f16(d, q_desc + (PL::kQChunk >> 4) * j + 2 * s, kd + (kChunkBytes >> 4) * j + 2 * s, idesc, (uint32_t)(j | s));
          }
          if (ok) mma_commit_cta(&ms.s_ready[kb & 1]);
        }
        if (ok) mma_commit_cta(&ms.q_free);
      }
      if (!ok) {                                                          // given up: what has been issued ends before the tensor memory goes
        mma_commit_cta(&ms.drained[0]);
        mbar_drain(&ms.drained[0], 0);
      }
    }
    __syncwarp();
  } else if (warp == kWarpPv) {
    // ------------------------------------------------------------ O^T += V^T P^T (one thread)
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc(1, 1, true, false, 128, kRows);
      Walk w(ms);
      int kb = 0;
      bool ok = true;
      while (ok && w.next(p))
        for (int k = w.k0; k < w.k1; ++k, ++kb) {
          if (!(ok = mbar_wait(&ms.p_ready[kb & 1], (kb >> 1) & 1, wt, kSiteP, kb))) break;
          if (kLoad == kCopy) fence_proxy_async_smem();
          tc_fence_after();
          const uint32_t slot = sbase + PL::kOffKV + (kb & 1) * kSlotBytes;
          const uint64_t vd = umma_desc(slot, kChunkBytes, 1024, kSwz128);                          // dims along M: two chunks of 64, 8 keys 1024 bytes
          const uint64_t pd = umma_desc(slot + (kChunks - 1) * kChunkBytes, 16, 1024, kSwz128);
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
              mma_f16(tmem + kRows * i, vd + (2 * kChunkBytes >> 4) * i + 128 * s, pd + 2 * s, idesc, k == w.k0 && s == 0 ? 0u : 1u);
            mma_commit_cta(&ms.kv_free[kb & 1][i]);
          }
          mma_commit_cta(&ms.kv_free[kb & 1][kGroups - 1]);
        }
      if (!ok) {
        mma_commit_cta(&ms.drained[1]);
        mbar_drain(&ms.drained[1], 0);
      }
    }
    __syncwarp();
  } else if (warp == kWarpQ) {
    // ------------------------------------------------------------ queries of the next piece, when the last product with these is complete
    Walk w(ms);
    const uint64_t pol = l2_policy_evict_first();
    bool ok = true;
    int asked = 0;
    while (w.next(p)) {
      if (w.index > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(&ms.q_free, (w.index - 1) & 1, wt, kSiteQ, w.index)))) break;
      if (p.flat_q) {
        if (lane == 0) mbar_arrive_expect_tx(&ms.q_ready, kChunks * PL::kQChunk);
        __syncwarp();
        if (lane < kChunks) tma_load_3d_hint(sbase + PL::kOffQ + lane * PL::kQChunk, &map_q, 64 * lane, 0, w.b, &ms.q_ready, pol);
      } else {
        for (int r = 0; r < kRows; ++r) {
          const int j = r / p.heads, h = r - j * p.heads;
          const bool in = r < p.rows;
          const uint8_t* src = p.q + (in ? w.b * p.q_b + j * p.q_j + h * p.q_h : 0);
          for (int c = lane; c < kD / 8; c += 32)
            cp_async16_or_zero(sbase + PL::kOffQ + (uint32_t)(c >> 3) * PL::kQChunk + r * 128 + (((c & 7) ^ (r & 7)) << 4), src + (in ? 16 * c : 0), in);
        }
        cp_async_wait_all();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ms.q_ready);
      }
      ++asked;
    }
    if (!ok && asked > 0 && lane == 0) mbar_drain(&ms.q_ready, (asked - 1) & 1);        // given up: what is in flight lands first
    __syncwarp();
  } else if (kLoad == kTma) {
   if (warp == kWarpTma) {
    // ------------------------------------------------------------ bf16 rows by TMA: a block is of one page, nine boxes of 64 dims
    // The block two ahead of the one requested is brought into L2: the load that follows a freed slot then takes L2's latency.
    const int count = ms.count;
    Ahead<false> next(ms, p, 0, kBlock, lane);
    const uint64_t pol = l2_policy_evict_first();
    const uint32_t mine = sbase + PL::kOffKV + lane * kChunkBytes;
    int asked = 0;
    bool ok = true;
    for (int kb = 0; ok && kb < count; ++kb, next.advance(p, lane)) {
      const int page = __shfl_sync(0xffffffffu, next.page, next.i), row = __shfl_sync(0xffffffffu, next.row, next.i);
      const bool some = next.rows_in(0) > 0;
#pragma unroll 1
      for (int j = 0; j < kGroups; ++j) {
        if (kb >= kSlots && !(ok = __all_sync(0xffffffffu, mbar_wait(&ms.kv_free[kb & 1][j], ((kb >> 1) & 1) ^ 1, wt, kSiteFree, kb)))) break;
        if (lane == 0) mbar_arrive_expect_tx(&ms.kv_full[kb & 1][j], some ? (j < kGroups - 1 ? 2 : 1) * kChunkBytes : 0u);
        __syncwarp();
        if (some && (lane >> 1) == j && lane < kChunks)
          tma_load_3d_hint(mine + (kb & 1) * kSlotBytes, &map_kv, 64 * lane, row, page, &ms.kv_full[kb & 1][j], pol);
        asked = kGroups * kb + j + 1;
      }
      const uint8_t* src = next.rows_of(p, 2, 2 * kD);
      if (src != nullptr && lane == 0) l2_prefetch_1d(src, kBlock * 2 * kD);
    }
    if (!ok)                                                              // given up: what is in flight lands first
      for (int i = max(asked - kSlots * kGroups, 0); i < asked; ++i) {
        const int kb = i / kGroups;
        mbar_drain(&ms.kv_full[kb & 1][i - kb * kGroups], (kb >> 1) & 1);
      }
   }
  } else if (warp >= kWarpLoad0) {
    // ------------------------------------------------------------ rows by cp.async, or packed rows through registers
    // Warp v has kOwn adjacent rows of a block (of one page: pages are multiples of 16 rows).
    constexpr int kOwn = kBlock / (kLoad == kTma ? 16 : kLoadWarps<kLoad>);
    constexpr int kRowBytes = kLoad == kCopy ? 2 * kD : kPackedRow;
    struct Coming { int page, row, n; };                                  // n of the warp's rows hold keys
    const int v = warp - kWarpLoad0;
    Walk w(ms);
    const int count = ms.count;
    int at = 0, looked = 0;
    PageAt pa(p.block_size);
    auto piece = [&]() {
      if (!w.next(p)) return;
      at = w.k0;
      pa.at(at * kBlock + kOwn * v);
    };
    piece();
    auto look = [&]() -> Coming {
      Coming x{-1, 0, 0};
      if (looked >= count) return x;
      x.n = min(max(w.len - at * kBlock - kOwn * v, 0), kOwn);
      if (x.n > 0) x.page = __ldcg(p.table + w.b * p.table_pitch + pa.page);
      x.row = pa.row;
      ++looked;
      pa.advance();
      if (++at == w.k1) piece();
      return x;
    };
    auto rows_of = [&](const Coming& x) -> const uint8_t* {
      return (unsigned)x.page < (unsigned)p.n_blocks ? p.cache + (long long)x.page * p.block_pitch + (long long)x.row * kRowBytes : nullptr;
    };
    auto to_l2 = [&](const Coming& x) {
      const uint8_t* src = rows_of(x);
      if (src != nullptr && lane == 0) l2_prefetch_1d(src, (uint32_t)(x.n * kRowBytes));
    };
    bool ok = true;
    Coming c0, c1 = look(), c2 = look(), c3 = look();
    to_l2(c1);
    to_l2(c2);
    if (kLoad == kCopy) {
      for (int kb = 0; ok && kb < count; ++kb) {
        c0 = c1; c1 = c2; c2 = c3; c3 = look();
        const uint32_t slot = sbase + PL::kOffKV + (kb & 1) * kSlotBytes;
        const uint8_t* src = rows_of(c0);
        to_l2(c2);
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          if (kb >= kSlots && !(ok = __all_sync(0xffffffffu, mbar_wait(&ms.kv_free[kb & 1][j], ((kb >> 1) & 1) ^ 1, wt, kSiteFree, kb)))) break;
          constexpr int kWide = 16;                                       // 16-byte pieces of a row in a group of two chunks
#pragma unroll
          for (int i = 0; i < (j < kGroups - 1 ? kOwn * kWide / 32 : kOwn * kWide / 64); ++i) {
            const int x = lane + 32 * i, r = j < kGroups - 1 ? x / kWide : x / 8, c = j < kGroups - 1 ? x % kWide : x % 8;
            const bool in = src != nullptr && r < c0.n;
            const int row = kOwn * v + r;
            cp_async16_or_zero(slot + (2 * j + (c >> 3)) * kChunkBytes + row * 128 + (((c & 7) ^ (row & 7)) << 4),
                               in ? src + r * kRowBytes + 256 * j + 16 * c : p.cache, in);
          }
          cp_async_mbar_arrive_noinc(&ms.kv_full[kb & 1][j]);
        }
      }
      cp_async_wait_all();
    } else {
      // Of each 128 dims eight lanes have 16 codes of a row each, four rows at a time.  A group's registers are loaded for the next
      // block as soon as they are converted for this one, from L2, where the rows were brought a block before.
      constexpr int kSets = kOwn / 4;
      const int sub = lane >> 3, c = lane & 7;
      uint4 codes[kGroups - 1][kSets], rope[kSets];
      float4 scale[kSets];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      auto load = [&](const uint8_t* src, int n, int j) {                  // group j's registers
#pragma unroll
        for (int i = 0; i < kSets; ++i) {
          const int r = sub + 4 * i;
          const bool in = src != nullptr && r < n;
          const uint8_t* row = src + r * kRowBytes;
          if (j == 0) scale[i] = in ? __ldcg(reinterpret_cast<const float4*>(row + 512)) : make_float4(0.f, 0.f, 0.f, 0.f);
          if (j < kGroups - 1) codes[j % (kGroups - 1)][i] = in ? __ldcg(reinterpret_cast<const uint4*>(row + 128 * j) + c) : zero;
          else rope[i] = in ? __ldcg(reinterpret_cast<const uint4*>(row + 528) + c) : zero;
        }
      };
      {
        const uint8_t* src = rows_of(c1);
#pragma unroll
        for (int j = 0; j < kGroups; ++j) load(src, c1.n, j);
      }
      for (int kb = 0; ok && kb < count; ++kb) {
        c0 = c1; c1 = c2; c2 = c3; c3 = look();
        const uint32_t slot = sbase + PL::kOffKV + (kb & 1) * kSlotBytes;
        const uint8_t* next = rows_of(c1);
        to_l2(c2);
        float4 mult[kSets];
#pragma unroll
        for (int i = 0; i < kSets; ++i) mult[i] = scale[i];
        // (groups 0 and 1, then the others: what is written for the tensor core has to be fenced before it is announced, and five fences
        // a block took a quarter of the conversion's time)
#pragma unroll
        for (int two = 0; two < 2; ++two) {
#pragma unroll
          for (int j = 2 * two; j < (two ? kGroups : 2); ++j) {
            if (kb >= kSlots) ok = __all_sync(0xffffffffu, mbar_wait(&ms.kv_free[kb & 1][j], ((kb >> 1) & 1) ^ 1, wt, kSiteFree, kb)) && ok;
#pragma unroll
            for (int i = 0; i < kSets; ++i) {
              const int r = kOwn * v + sub + 4 * i;
              if (j < kGroups - 1) {
                uint4 a, b;
                convert16(codes[j % (kGroups - 1)][i], j == 0 ? mult[i].x : j == 1 ? mult[i].y : j == 2 ? mult[i].z : mult[i].w, a, b);
                // lanes of odd chunks write their second half first: the eight lanes of a phase then cover all banks
                const uint32_t base = slot + (2 * j + (c >> 2)) * kChunkBytes + r * 128, u = 2 * (c & 3), odd = c >> 2;
                st_shared16(base + (((u + odd) ^ (r & 7)) << 4), odd ? b : a);
                st_shared16(base + (((u + 1 - odd) ^ (r & 7)) << 4), odd ? a : b);
              } else {
                st_shared16(slot + (kChunks - 1) * kChunkBytes + r * 128 + ((c ^ (r & 7)) << 4), rope[i]);
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (ok && lane < (two ? kGroups - 2 : 2)) mbar_arrive(&ms.kv_full[kb & 1][2 * two + lane]);
#pragma unroll
          for (int j = 2 * two; j < (two ? kGroups : 2); ++j) load(next, c1.n, j);
        }
      }
    }
  }

  if (warp == kWarpQk && lane == 0 && p.meta) write_meta(p, ms, g);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kWarpQk) tmem_dealloc_cta(tmem, PL::kTmemCols);
  if (threadIdx.x == 0) {
    wt.report(g_status, p.epoch);
    if (blockIdx.x == 0) atomicAdd(&g_status[3], 1);
  }
}

// The rows of sequences that several groups have parts of: out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.  Blocks deal out the
// rows among themselves: of a sequence of up to 8 parts a warp has a row, of one of more a block has: each warp sums every eighth
// part and the eight sums meet in shared memory.  (With a block per row and listed sequence, mostly idle, 36 sequences of 256 rows in
// two or three parts took 76 us.)
constexpr int kMergeWarps = 8, kMaxGroups = 1024;      // (at most one a CTA)
__device__ __forceinline__ void add_parts(const Params& p, int kRows, int g, const int4& e, int row, float m, int from, int step, float4 (&a)[4], float& l,
                                          int lane) {
  const int rt = row / kRows, r = row - rt * kRows;
  for (int i0 = from; i0 < e.z; i0 += 2 * step) {
    float4 v[2][4];
    float2 ml[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int i = i0 + u * step;
      ml[u] = make_float2(kMInit, 0.f);
      if (i < e.z) {
        const long long s = ((long long)((g + i) * p.row_tiles + rt) * 2 + (i == 0 ? e.y : 0)) * kRows + r;
        ml[u] = __ldcg(&p.part_ml[s]);
        const float4* src = reinterpret_cast<const float4*>(p.part_o + s * kDV);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[u][c] = __ldcg(src + 32 * c + lane);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (ml[u].y == 0.f) continue;                    // beyond the list, or a part without keys
      const float f = fast_exp2(ml[u].x - m);
      l += f * ml[u].y;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        a[c].x += f * v[u][c].x; a[c].y += f * v[u][c].y; a[c].z += f * v[u][c].z; a[c].w += f * v[u][c].w;
      }
    }
  }
}
// Up to 8 parts: the first three are asked for before their weights are known.
__device__ __forceinline__ void add_few(const Params& p, int kRows, int g, const int4& e, int row, float4 (&a)[4], float& l, float& m, int lane) {
  const int rt = row / kRows, r = row - rt * kRows;
  const long long s0 = ((long long)(g * p.row_tiles + rt) * 2 + e.y) * kRows + r, ds = 2LL * p.row_tiles * kRows, s1 = s0 - (long long)e.y * kRows;
  auto slot = [&](int i) { return i == 0 ? s0 : s1 + i * ds; };
  float4 v[3][4];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < 3; ++u)
      if (i0 + u < e.z) {
        const float4* src = reinterpret_cast<const float4*>(p.part_o + slot(i0 + u) * kDV);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[u][c] = __ldcg(src + 32 * c + lane);
      }
  };
  float2 ml = make_float2(kMInit, 0.f);
  if (lane < e.z) ml = __ldcg(&p.part_ml[slot(lane)]);
  load(0);
  m = ml.x;
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
  m = __shfl_sync(0xffffffffu, m, 0);
  const float w = fast_exp2(ml.x - m);
#pragma unroll
  for (int i0 = 0; i0 < 8; i0 += 3) {
    if (i0 >= e.z) break;
    if (i0) load(i0);
#pragma unroll
    for (int u = 0; u < 3; ++u) {
      const float f = __shfl_sync(0xffffffffu, w, i0 + u), y = __shfl_sync(0xffffffffu, ml.y, i0 + u);
      if (y == 0.f) continue;                          // beyond the list, or a part without keys
      l += f * y;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        a[c].x += f * v[u][c].x; a[c].y += f * v[u][c].y; a[c].z += f * v[u][c].z; a[c].w += f * v[u][c].w;
      }
    }
  }
}
__global__ void __launch_bounds__(32 * kMergeWarps, 2) mla_decode_merge_kernel(const Params p, int kRows) {
  __shared__ float4 acc[kMergeWarps][kDV / 4];
  __shared__ float sum_l[kMergeWarps];
  __shared__ int4 list[kMaxGroups];                    // {sequence, slot of its first part, parts, group of the first}
  __shared__ int units[kMaxGroups + 1], found[2][kMergeWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_trigger();
  pdl_wait();
  // The cut sequences, and where each one's units of work begin
  int n = 0, all = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32 * kMergeWarps) {
    const int g = g0 + (int)threadIdx.x;
    int4 e = make_int4(-1, 0, 0, 0);
    if (g < p.groups) e = __ldcg(p.meta + g);
    const bool cut = e.x >= 0 && e.z > 0;
    const int mine = !cut ? 0 : e.z <= 8 ? (p.rows + kMergeWarps - 1) / kMergeWarps : p.rows;
    const uint32_t mask = __ballot_sync(0xffffffffu, cut);
    int incl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31) { found[0][warp] = __popc(mask); found[1][warp] = incl; }
    __syncthreads();
    int at = n + __popc(mask & ((1u << lane) - 1u)), before = all + incl - mine;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
      if (w < warp) { at += found[0][w]; before += found[1][w]; }
      n += found[0][w];
      all += found[1][w];
    }
    if (cut) {
      list[at] = make_int4(e.x, e.y, e.z, g);
      units[at] = before;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) units[n] = all;
  __syncthreads();
  int at = 0;
  for (int u = (int)blockIdx.x; u < all; u += (int)gridDim.x) {
    while (units[at + 1] <= u) ++at;
    const int4 e = list[at];
    const int g = e.w;
    const bool alone = e.z <= 8;                       // a warp a row
    const int row = alone ? (u - units[at]) * kMergeWarps + warp : u - units[at];
    if (row < p.rows) {                                // (the same for all of a block that shares a row)
      float4 a[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) a[c] = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f, m = kMInit;
      if (alone) {
        add_few(p, kRows, g, e, row, a, l, m, lane);
      } else {
        const int rt = row / kRows, r = row - rt * kRows;
        for (int i = lane; i < e.z; i += 32)
          m = fmaxf(m, __ldcg(&p.part_ml[((long long)((g + i) * p.row_tiles + rt) * 2 + (i == 0 ? e.y : 0)) * kRows + r].x));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        add_parts(p, kRows, g, e, row, m, warp, kMergeWarps, a, l, lane);
      }
      const long long to = (long long)e.x * p.rows + row;
      if (alone) {
        const float f = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          reinterpret_cast<uint2*>(p.out)[to * (kDV / 4) + 32 * c + lane] = make_uint2(bf16x2(a[c].x * f, a[c].y * f), bf16x2(a[c].z * f, a[c].w * f));
        if (lane == 0) p.lse[to] = l != 0.f ? (m + __log2f(l)) * kLn2 : INFINITY;
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[warp][32 * c + lane] = a[c];
        if (lane == 0) sum_l[warp] = l;
        __syncthreads();
        if (threadIdx.x < kDV / 4) {
          float4 o = acc[0][threadIdx.x];
          l = sum_l[0];
#pragma unroll
          for (int w = 1; w < kMergeWarps; ++w) {
            const float4 x = acc[w][threadIdx.x];
            o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
            l += sum_l[w];
          }
          const float f = l != 0.f ? 1.f / l : 0.f;
          reinterpret_cast<uint2*>(p.out)[to * (kDV / 4) + threadIdx.x] = make_uint2(bf16x2(o.x * f, o.y * f), bf16x2(o.z * f, o.w * f));
          if (threadIdx.x == 0) p.lse[to] = l != 0.f ? (m + __log2f(l)) * kLn2 : INFINITY;
        }
        __syncthreads();
      }
    }
  }
}

template <int kRows, Load kLoad>
static int launch(const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  if (!ensure_smem<mla_decode_kernel<kRows, kLoad>>(current_device(), Plan<kRows>::kSmem)) return LITEDSA_ERR_CUDA;
  return launch_pdl(mla_decode_kernel<kRows, kLoad>, dim3((unsigned)p.groups), kThreads<kLoad>, Plan<kRows>::kSmem, st, map, map_q, p);
}
template <int kRows>
static int launch(Load l, const CUtensorMap& map, const CUtensorMap& map_q, const Params& p, cudaStream_t st) {
  return l == kTma ? launch<kRows, kTma>(map, map_q, p, st) : l == kCopy ? launch<kRows, kCopy>(map, map_q, p, st)
                                                                         : launch<kRows, kPacked>(map, map_q, p, st);
}

}  // namespace decode
}  // namespace lt

#include "mla_decode_pair.cuh"

namespace lt {
namespace decode {

// Up to 64 rows a CTA has a tile, more have pairs of CTAs, 128 rows a pair.  (32 sequences of up to 8191 packed rows, 64 heads: 61 us against 67 with pairs of
// 32 rows a CTA; 256 rows, bf16: 112 against 133 with four CTAs of 64; 128 sequences of 128 heads, packed: 160 against 215.  All with equal shares of blocks.)
struct Shape {
  int per, tiles, groups;
  bool pair;
  Shape(int rows, Load l) : pair(rows > 64) {
    per = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
    tiles = (rows + per - 1) / per;
    const int units = !pair ? sm_count() : l == kPacked ? decode::pair::pairs<kPacked>() : decode::pair::pairs<kTma>();
    groups = min(max(1, units / tiles), kMaxGroups);
  }
  int64_t part_bytes() const { return (int64_t)groups * tiles * 2 * per * (kDV * 4 + 8); }
  int64_t bytes() const { return groups == 1 ? 0 : part_bytes() + (int64_t)groups * 16; }
};
// What a workspace has to hold does not depend on how rows are loaded, as a caller does not know that.
static int64_t workspace(int rows) { return max(Shape(rows, kTma).bytes(), Shape(rows, kPacked).bytes()); }

}  // namespace decode
}  // namespace lt

extern "C" int64_t litedsa_mla_decode_workspace(int q_len, int heads) {
  if (q_len <= 0 || heads <= 0 || heads > 128 || (int64_t)q_len * heads > (1 << 20)) return 0;
  return lt::decode::workspace(q_len * heads);
}

extern "C" int litedsa_mla_decode(const void* q, int64_t q_batch_stride, int64_t q_token_stride, int64_t q_head_stride,
                                  const void* cache, int packed, int64_t n_blocks, int block_size, int64_t block_stride_bytes,
                                  const int32_t* block_table, int64_t table_stride, int table_cols, const int32_t* seq_lens,
                                  float sm_scale, void* out, float* lse, int B, int q_len, int heads, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace lt;
  using namespace lt::decode;
  if (!q || (!cache && n_blocks > 0) || (!block_table && table_cols > 0) || !seq_lens || !out || !lse) return LITEDSA_ERR_ARG;
  if (B < 0 || q_len <= 0 || heads <= 0 || heads > 128 || (int64_t)q_len * heads > (1 << 20) || table_cols < 0 || n_blocks < 0 || block_size <= 0)
    return LITEDSA_ERR_SHAPE;
  if (block_size % 16 || n_blocks >= (1ll << 31) || (int64_t)table_cols * block_size >= (1ll << 31) - kBlock) return LITEDSA_ERR_UNSUPPORTED;
  // (the blocks of all sequences are counted in 32 bits)
  if (B * ((int64_t)table_cols * block_size / kBlock + 1 + kMostStartCost) >= (1ll << 31)) return LITEDSA_ERR_UNSUPPORTED;
  const int row = packed ? kPackedRow : 2 * kD;
  if (n_blocks > 1 && block_stride_bytes < (int64_t)block_size * row) return LITEDSA_ERR_SHAPE;
  if (((uintptr_t)q | (uintptr_t)cache | (uintptr_t)out | (uintptr_t)workspace) & 15 || block_stride_bytes % 16 ||
      (q_batch_stride | q_token_stride | q_head_stride) % 8 || ((uintptr_t)lse & 3))
    return LITEDSA_ERR_UNSUPPORTED;
  if (B == 0) return LITEDSA_OK;
  const Load load = packed ? kPacked : q_len * heads > 64 || block_size % kBlock == 0 ? kTma : kCopy;
  const Shape s(q_len * heads, load);
  const int64_t need = decode::workspace(q_len * heads);
  if (need > 0 && (!workspace || workspace_bytes < need)) return workspace ? LITEDSA_ERR_SHAPE : LITEDSA_ERR_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  Params p = {};
  p.q = reinterpret_cast<const uint8_t*>(q);
  p.q_b = 2 * q_batch_stride; p.q_j = 2 * q_token_stride; p.q_h = 2 * q_head_stride;
  p.cache = reinterpret_cast<const uint8_t*>(cache); p.block_pitch = block_stride_bytes;
  p.table = block_table; p.table_pitch = table_stride; p.lens = seq_lens;
  p.out = reinterpret_cast<uint8_t*>(out); p.lse = lse;
  if (s.groups > 1) {
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)s.groups * s.tiles * 2 * s.per * kDV);
    p.meta = reinterpret_cast<int4*>(reinterpret_cast<char*>(workspace) + s.part_bytes());
  }
  p.B = B; p.q_len = q_len; p.heads = heads; p.rows = q_len * heads; p.row_tiles = s.tiles; p.groups = s.groups;
  p.cols = n_blocks == 0 ? 0 : table_cols; p.block_size = block_size; p.n_blocks = (int)n_blocks;
  // 7000 cycles at 1400 to 2600 a block of a pair, 5500 at 3000 to 3800 of a CTA (0 / 2 / 4 / 6: 256 rows, bf16 109 / 106 / 103 / 102 us; 128 rows, packed 147 /
  // 142 / 144 / 146; 64 rows, packed 57.7 / 52.0 / 51.9 / 53.4; 16 rows, packed 44.9 / 44.4 / 46.4 / 48.9).  Elsewhere, 0 / 2 / 5 / 8, between two events behind a
  // flush of L2: 16 heads, 20 x 500-3000 keys, bf16 30 / 28 / 28 / 28; 64 heads, 10 x 5000-30000, bf16 64 / 62 / 62 / 62; 32 heads, 64 x 100-3000, packed
  // 50 / 46 / 48 / 50; 64 heads, 300 x 64-600, packed 67 / 62 / 62 / 62; 128 heads, bf16, 20 x 2000-20000 87 / 86 / 85 / 85, 200 x 100-900 75 / 69 / 65 / 67;
  // 128 heads, 300 x 100-900, packed 99 / 95 / 91 / 93; three tokens of 128 heads, 40 x 500-3000, packed 101 / 97 / 95 / 99
  p.start_cost = s.pair && !packed ? kMostStartCost : 2;
  p.box_rows = block_size % pair::kOwnKeys == 0 ? pair::kOwnKeys : 16;
  p.scale_log2 = sm_scale * kLog2e;
  p.epoch = next_launch_epoch(); p.wait_limit = wait_limit_ticks();
  CUtensorMap map = {};
  if (load == kTma && n_blocks > 0 &&
      !make_map_3d(&map, cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kD, (uint64_t)block_size, (uint64_t)n_blocks, 2 * kD,
                   (uint64_t)(n_blocks > 1 ? block_stride_bytes : (int64_t)block_size * row), 64, s.pair ? (uint32_t)p.box_rows : (uint32_t)kBlock, 1))
    return LITEDSA_ERR_CUDA;
  // Rows (token, head) of a sequence that are evenly spaced (one token, or no gap behind a token's heads) are a matrix.
  CUtensorMap map_q = {};
  p.flat_q = q_len == 1 || q_token_stride == heads * q_head_stride;
  const int64_t row_stride = heads > 1 ? q_head_stride : q_len > 1 ? q_token_stride : kD;
  if (p.flat_q && !make_map_3d(&map_q, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kD, (uint64_t)p.rows, (uint64_t)B, (uint64_t)(2 * row_stride),
                               (uint64_t)(2 * (B > 1 ? q_batch_stride : kD)), 64, (uint32_t)(s.pair ? s.per / 2 : s.per), 1))
    p.flat_q = 0;                                                          // (a stride of 0, for one, is no map's)
  const int rc = s.per == 16 ? launch<16>(load, map, map_q, p, st) : s.per == 32 ? launch<32>(load, map, map_q, p, st)
                 : s.per == 64 ? launch<64>(load, map, map_q, p, st) : pair::launch(load, map, map_q, p, st);
  if (rc != LITEDSA_OK || s.groups == 1) return rc;
  const int64_t most = (int64_t)min(B, s.groups) * p.rows;                 // rows that can need it
  return launch_pdl(mla_decode_merge_kernel, dim3((unsigned)min(most, (int64_t)2 * sm_count())), 32 * kMergeWarps, 0, st, p, s.per);
}

// Status block of the kernel; layout and return rule as litedsa_attn_status.
extern "C" int litedsa_mla_decode_status(int* out4_host, int reset) {
  using namespace lt::decode;
  if (out4_host && cudaMemcpyFromSymbol(out4_host, g_status, sizeof(int) * 4) != cudaSuccess) return LITEDSA_ERR_CUDA;
  if (reset) {
    const int z[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (cudaMemcpyToSymbol(g_status, z, sizeof(z)) != cudaSuccess) return LITEDSA_ERR_CUDA;
  }
  return (out4_host && out4_host[0] != 0) ? LITEDSA_ERR_TIMEOUT : LITEDSA_OK;
}
