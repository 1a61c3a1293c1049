// Appending tokens to a paged latent cache (sm_100a): the rotation of the rope dims by the token's position, the packed row's
// quantisation and the scatter into pages in one pass, together with the rotation of the queries' rope dims.
//
//   rotation  pair i of the 64 dims, (x, y) = dims (2i, 2i + 1) interleaved, (i, i + 32) else:
//             (x cos_i - y sin_i, y cos_i + x sin_i), computed in fp32 and rounded to bf16 once
//   packed    512 e4m3 codes | 4 fp32 scales | 64 bf16: scale = the smallest power of two that brings a group's 128 dims into
//             +-448, so that code x scale is exact in bf16 and attention over the row rounds nothing again
//
// Compiled without flushing to zero: numbers below 2^-126 are turned and packed like any others.
//
// Element-wise and bound by memory; a few tokens by latency, so a token is a block of its own: up to eight warps of it rotate heads
// (eight lanes a head, eight heads a warp), the last one has the cache row, sixteen latent dims a lane, so that a group's
// maximum is three shuffles.  Everything is read and written once, 16 bytes an access, neighbouring lanes neighbouring bytes.
//
// Measured: 8192 tokens of 64 heads into packed rows 32.6 us = 4.7 TB/s (a copy: 6.5), into bf16 rows 33.2; one token of 128 heads 1.8 us in a
// replayed graph of fifty.
#include "common.cuh"

namespace lt {
namespace append {

constexpr int kMaxHeadWarps = 8;

struct Params {
  const uint8_t *kv_c, *k_rope, *q_in;
  const void *positions, *slots;
  const float* cos_sin;
  uint8_t *cache, *q_out, *k_out;
  // pitches in bytes
  long long kv_c_pitch, k_rope_pitch, cs_pitch, q_in_token, q_in_head, q_out_token, q_out_head, k_out_pitch, block_pitch;
  long long n_rows, n_pos;
  int block_size, heads;
  int pos64, slot64;
};

__device__ __forceinline__ long long index_at(const void* p, int wide, int i) {
  return wide ? __ldcg(reinterpret_cast<const long long*>(p) + i) : (long long)__ldcg(reinterpret_cast<const int*>(p) + i);
}
__device__ __forceinline__ uint4 load16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ float lo_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// A vector of 64 dims has eight lanes, 16 bytes each: four pairs of neighbours, or eight dims whose partners lane j ^ 4 has.
template <bool kInterleaved>
struct Turn {
  static constexpr int kPairs = kInterleaved ? 4 : 8;
  float c[kPairs], s[kPairs];
  __device__ __forceinline__ void load(const float* row, int j) {
    const int first = kInterleaved ? 4 * j : 8 * (j & 3);
#pragma unroll
    for (int i = 0; i < kPairs; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + first + i), b = *reinterpret_cast<const float4*>(row + 32 + first + i);
      c[i] = a.x; c[i + 1] = a.y; c[i + 2] = a.z; c[i + 3] = a.w;
      s[i] = b.x; s[i + 1] = b.y; s[i + 2] = b.z; s[i + 3] = b.w;
    }
    if (!kInterleaved && j < 4)                        // x c - y s of the first half, y c + x s of the second
#pragma unroll
      for (int i = 0; i < kPairs; ++i) s[i] = -s[i];
  }
  // all 32 lanes
  __device__ __forceinline__ uint4 operator()(const uint4& v) const {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = lo_of(u[i]), y = hi_of(u[i]);
      if (kInterleaved) {
        o[i] = bf16x2(x * c[i] - y * s[i], y * c[i] + x * s[i]);
      } else {
        const uint32_t w = __shfl_xor_sync(0xffffffffu, u[i], 4);
        o[i] = bf16x2(x * c[(2 * i) % kPairs] + lo_of(w) * s[(2 * i) % kPairs], y * c[(2 * i + 1) % kPairs] + hi_of(w) * s[(2 * i + 1) % kPairs]);
      }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
  }
};

template <bool kInterleaved, bool kPacked>
__global__ void __launch_bounds__(32 * (kMaxHeadWarps + 1)) append_kv_kernel(const Params p) {
  const int t = (int)blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, head_warps = (blockDim.x >> 5) - 1;
  const int j = lane & 7;
  pdl_trigger();
  pdl_wait();
  const long long pos = index_at(p.positions, p.pos64, t);
  const bool known = pos >= 0 && pos < p.n_pos;        // not in the table: the token is left out
  const float* angles = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(p.cos_sin) + pos * p.cs_pitch);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  Turn<kInterleaved> turn;
  if (warp < head_warps) {
    // (the first heads are on their way while the position and its angles are looked up)
    const uint8_t* src = p.q_in + t * p.q_in_token + 16 * j;
    uint8_t* dst = p.q_out + t * p.q_out_token + 16 * j;
    int h = 8 * warp + (lane >> 3);
    uint4 a = h < p.heads ? load16(src + h * p.q_in_head) : zero, b = h + 4 < p.heads ? load16(src + (h + 4) * p.q_in_head) : zero;
    if (!known) return;
    turn.load(angles, j);
    for (;;) {
      a = turn(a);
      b = turn(b);
      if (h < p.heads) *reinterpret_cast<uint4*>(dst + h * p.q_out_head) = a;
      if (h + 4 < p.heads) *reinterpret_cast<uint4*>(dst + (h + 4) * p.q_out_head) = b;
      h += 8 * head_warps;
      if (h - (lane >> 3) >= p.heads) return;
      a = h < p.heads ? load16(src + h * p.q_in_head) : zero;
      b = h + 4 < p.heads ? load16(src + (h + 4) * p.q_in_head) : zero;
    }
  }
  if (!known) return;
  turn.load(angles, j);
  const long long slot = index_at(p.slots, p.slot64, t);
  uint8_t* row = nullptr;
  if (slot >= 0 && slot < p.n_rows)
    row = p.cache + (slot / p.block_size) * p.block_pitch + (slot % p.block_size) * (kPacked ? 656 : 1152);
  const uint4 k = turn(lane < 8 ? load16(p.k_rope + t * p.k_rope_pitch + 16 * j) : zero);
  if (lane < 8) {
    if (row) *reinterpret_cast<uint4*>(row + (kPacked ? 528 : 1024) + 16 * j) = k;
    if (p.k_out) *reinterpret_cast<uint4*>(p.k_out + t * p.k_out_pitch + 16 * j) = k;
  }
  if (!row) return;                                    // padding, or no row of this cache (warp-uniform)
  const uint8_t* src = p.kv_c + t * p.kv_c_pitch;
  if (!kPacked) {
    const uint4 a = load16(src + 16 * lane), b = load16(src + 512 + 16 * lane);
    *reinterpret_cast<uint4*>(row + 16 * lane) = a;
    *reinterpret_cast<uint4*>(row + 512 + 16 * lane) = b;
    return;
  }
  const uint4 a = load16(src + 32 * lane), b = load16(src + 32 * lane + 16);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t amax = 0;                                   // of the magnitudes' bits: bf16 in the upper half of a float
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, max((w[i] << 16) & 0x7fff0000u, w[i] & 0x7fff0000u));
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  // amax = m 2^e with 1 <= m < 2, 448 = 1.75 2^8: exponent e - 8, one more if m > 1.75; not below that of the smallest
  // normal number (groups of zeros, too).  Infinities and NaN have e = 128: a finite scale, codes of 448 and NaN.
  const int e = max((int)(amax >> 23) - 127 - 8 + ((amax & 0x007fffffu) > 0x00600000u ? 1 : 0), -126);
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = make_float2(lo_of(w[2 * i]) * inv, hi_of(w[2 * i]) * inv), y = make_float2(lo_of(w[2 * i + 1]) * inv, hi_of(w[2 * i + 1]) * inv);
    o[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3) << 16);
  }
  *reinterpret_cast<uint4*>(row + 16 * lane) = make_uint4(o[0], o[1], o[2], o[3]);
  if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(row + 512 + (lane >> 1)) = (uint32_t)(e + 127) << 23;
}

// whether vectors of 64 elements in two dimensions lie apart
static bool apart(int64_t n0, int64_t stride0, int64_t n1, int64_t stride1) {
  if (n0 <= 1) return n1 <= 1 || stride1 >= 64;
  if (n1 <= 1) return stride0 >= 64;
  const bool inner1 = stride1 <= stride0;
  const int64_t in = inner1 ? stride1 : stride0, out = inner1 ? stride0 : stride1, n = inner1 ? n1 : n0;
  return in >= 64 && (out - 64) / in >= n - 1;
}

}  // namespace append
}  // namespace lt

extern "C" int litedsa_append_kv(const void* kv_c, int64_t kv_c_stride, const void* k_rope, int64_t k_rope_stride,
                                 const void* positions, int positions_64, const float* cos_sin, int64_t n_positions,
                                 int64_t cos_sin_stride, const void* slots, int slots_64, void* cache, int packed,
                                 int64_t n_blocks, int block_size, int64_t block_stride_bytes, int interleaved,
                                 const void* q_rope, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                                 int64_t q_out_token_stride, int64_t q_out_head_stride, int heads, void* k_out,
                                 int64_t k_out_stride, int T, void* stream) {
  using namespace lt;
  if (!kv_c || !k_rope || !positions || (!cos_sin && n_positions > 0) || !slots || (!cache && n_blocks > 0)) return LITEDSA_ERR_ARG;
  if ((q_rope == nullptr) != (q_out == nullptr)) return LITEDSA_ERR_ARG;
  if (T < 0 || n_positions < 0 || n_blocks < 0 || block_size <= 0 || (q_rope && heads <= 0)) return LITEDSA_ERR_SHAPE;
  if (n_blocks > 1 && block_stride_bytes < (int64_t)block_size * (packed ? 656 : 1152)) return LITEDSA_ERR_SHAPE;
  if (((uintptr_t)kv_c | (uintptr_t)k_rope | (uintptr_t)cos_sin | (uintptr_t)cache | (uintptr_t)q_rope | (uintptr_t)q_out |
       (uintptr_t)k_out) & 15)
    return LITEDSA_ERR_UNSUPPORTED;
  if ((kv_c_stride | k_rope_stride | (q_rope ? q_token_stride | q_head_stride | q_out_token_stride | q_out_head_stride : 0) |
       (k_out ? k_out_stride : 0)) % 8 || cos_sin_stride % 4 || block_stride_bytes % 16)
    return LITEDSA_ERR_UNSUPPORTED;
  // (several threads would write the same words)
  if ((q_rope && !append::apart(T, q_out_token_stride, heads, q_out_head_stride)) || (k_out && !append::apart(T, k_out_stride, 1, 0)))
    return LITEDSA_ERR_UNSUPPORTED;
  if (T == 0) return LITEDSA_OK;
  append::Params p = {};
  p.kv_c = reinterpret_cast<const uint8_t*>(kv_c); p.k_rope = reinterpret_cast<const uint8_t*>(k_rope);
  p.q_in = reinterpret_cast<const uint8_t*>(q_rope);
  p.positions = positions; p.slots = slots; p.cos_sin = cos_sin;
  p.cache = reinterpret_cast<uint8_t*>(cache); p.q_out = reinterpret_cast<uint8_t*>(q_out); p.k_out = reinterpret_cast<uint8_t*>(k_out);
  p.kv_c_pitch = 2 * kv_c_stride; p.k_rope_pitch = 2 * k_rope_stride; p.cs_pitch = 4 * cos_sin_stride;
  p.q_in_token = 2 * q_token_stride; p.q_in_head = 2 * q_head_stride;
  p.q_out_token = 2 * q_out_token_stride; p.q_out_head = 2 * q_out_head_stride;
  p.k_out_pitch = 2 * k_out_stride; p.block_pitch = block_stride_bytes;
  p.n_rows = n_blocks * block_size; p.n_pos = n_positions;
  p.block_size = block_size; p.heads = q_rope ? heads : 0;
  p.pos64 = positions_64; p.slot64 = slots_64;
  const int warps = min(append::kMaxHeadWarps, (p.heads + 7) / 8) + 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)T);
  if (interleaved) return packed ? launch_pdl(append::append_kv_kernel<true, true>, grid, 32 * warps, 0, st, p)
                                 : launch_pdl(append::append_kv_kernel<true, false>, grid, 32 * warps, 0, st, p);
  return packed ? launch_pdl(append::append_kv_kernel<false, true>, grid, 32 * warps, 0, st, p)
                : launch_pdl(append::append_kv_kernel<false, false>, grid, 32 * warps, 0, st, p);
}
