// Appending K/V rows to a cache of E4M3 bytes with one scale per (block, kv
// head), for K and for V (gfx950), and the launch plan of the attention over it.
//
// The scale of a block is the smallest power of two s with amax <= 448 s over
// the finite elements written to it so far (at least 2^-100). A power of two
// costs E4M3 nothing: its values keep three mantissa bits at any exponent, so
// x / s is exact before the one rounding, and a scale that grows later moves the
// bytes already there by a whole number of exponents, exact but for values that
// leave E4M3's normal range at its lower end (there: rounded once more).
//
//   a token at offset 0 opens its block: s = what the call's tokens need
//   else s' = max(s, what they need); where s' > s, b' = E4M3(b * s / s')
//   byte = E4M3(x / s'), rounded to nearest even, infinities to +-448
//
// One workgroup owns a (block, kv head) of the call: the first of the
// neighbouring tokens that share a block leads, and its workgroup takes them all,
// K in one half of the lanes and V in the other. Rows are staged in LDS, where V
// is read across tokens. V's bytes of one token lie in every 16-byte vector of
// its tile, so a partly filled tile is read and written whole: contiguous
// vectors instead of single bytes in every 32-byte sector.

#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kLeastScale = -100;  // exponent

// The smallest power of two s with amax <= 448 s; amax finite, as f32 bits.
__device__ __forceinline__ float needed_scale(uint32_t amax_bits) {
  // 448 = 1.75 * 2^8
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float((uint32_t)(max(e, kLeastScale) + 127) << 23);
}

// Two f32 -> E4M3 bytes in half `kHi` of a word (round to nearest even;
// |x| <= 448 or NaN).
template <bool kHi>
__device__ __forceinline__ uint32_t fp8_pair(float a, float b, uint32_t old) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, kHi);
}

// A 16-byte vector of T as f32 (8 or 4 values).
template <typename T>
__device__ __forceinline__ void widen(const uint4& v, float (&f)[16 / sizeof(T)]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = low_half_f32<T>(w[e]);
      f[2 * e + 1] = high_half_f32<T>(w[e]);
    }
  }
}

// One byte scaled by `ratio` (a scale over a larger one).
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return fp8_pair<true>(hi[0] * ratio, hi[1] * ratio,
                        fp8_pair<false>(lo[0] * ratio, lo[1] * ratio, 0u));
}

template <typename T, int D, int BS, int W>
__global__ __launch_bounds__(W == 1 ? 128 : 256) void scaled_append_kernel(
    const T* __restrict__ key, const T* __restrict__ value, int64_t key_token_stride,
    int64_t value_token_stride, float* __restrict__ key_scales, float* __restrict__ value_scales,
    int64_t scale_block_stride, uint8_t* __restrict__ key_cache, uint8_t* __restrict__ value_cache,
    const int64_t* __restrict__ slot_mapping, int64_t num_tokens, int64_t num_blocks,
    int64_t block_stride, int64_t head_stride, int32_t num_kv_heads) {
  constexpr int NT = W == 1 ? 128 : 256;
  constexpr int H = NT / 2;                   // lanes of K, and of V
  constexpr int VR = D * (int)sizeof(T) / 16;  // 16-byte vectors of a row
  constexpr int E = 16 / (int)sizeof(T);       // elements of one
  constexpr int NU = D * BS / 16;              // 16-byte units of a tile
  __shared__ __align__(16) uint4 s_rows[2][BS * VR];
  __shared__ int64_t s_tok[BS];  // last token of the run at each offset, -1: none
  __shared__ uint32_t s_max[2][2][NT / 64];
  __shared__ float s_old[2];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int which = __builtin_amdgcn_readfirstlane(tid / H);  // 0: K, 1: V
  const int h = tid % H;
  // kv heads fastest: neighbouring workgroups read neighbouring slices of a row
  const int head = (int)(blockIdx.x % (uint32_t)num_kv_heads);
  const int64_t t0 = (int64_t)(blockIdx.x / (uint32_t)num_kv_heads) * W;

  // the block of token t, -1: padding or past the pool
  auto block_of = [&](int64_t slot) {
    const int64_t b = slot < 0 ? -1 : slot / BS;
    return b < num_blocks ? b : (int64_t)-1;
  };
  uint64_t leaders;
  {
    const int64_t t = t0 + lane;
    bool lead = false;
    if (lane < W && t < num_tokens) {
      const int64_t b = block_of(slot_mapping[t]);
      lead = b >= 0 && (t == 0 || block_of(slot_mapping[t - 1]) != b);
    }
    leaders = __ballot(lead);
  }
  for (; leaders != 0; leaders &= leaders - 1) {
    const int64_t first = t0 + __builtin_ctzll(leaders);
    const int64_t blk = block_of(slot_mapping[first]);
    // ---- the run's tokens by offset ----
    if (tid < BS) s_tok[tid] = -1;
    __syncthreads();
    for (int64_t base = first; wave == 0; base += 64) {
      const int64_t t = base + lane;
      const int64_t slot = t < num_tokens ? slot_mapping[t] : (int64_t)-1;
      const uint64_t other = __ballot(block_of(slot) != blk);
      const int n = other != 0 ? __builtin_ctzll(other) : 64;
      if (lane < n)
        atomicMax(reinterpret_cast<long long*>(&s_tok[slot % BS]), (long long)t);
      if (n < 64) break;
    }
    __syncthreads();
    const uint64_t have = __ballot(lane < BS && s_tok[lane % BS] >= 0);
    const bool fresh = (have & 1u) != 0;
    constexpr uint64_t kAll = BS == 64 ? ~0ull : (1ull << BS) - 1;

    // ---- rows to LDS, their largest element ----
    const T* src = which == 0 ? key : value;
    const int64_t stride = which == 0 ? key_token_stride : value_token_stride;
    uint32_t amax = 0, inf = 0;
    for (int i = h; i < BS * VR; i += H) {
      const int off = i / VR;
      const int64_t t = s_tok[off];
      if (t < 0) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(src + t * stride + (int64_t)head * D +
                                                      (i % VR) * E);
      s_rows[which][i] = v;
      float f[E];
      widen<T>(v, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
        amax = max(amax, a < 0x7f800000u ? a : 0u);
        inf |= a == 0x7f800000u ? 1u : 0u;
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      amax = max(amax, (uint32_t)__shfl_xor((int)amax, m, 64));
      inf |= (uint32_t)__shfl_xor((int)inf, m, 64);
    }
    if (lane == 0) {
      s_max[which][0][h / 64] = amax;
      s_max[which][1][h / 64] = inf;
    }
    float* scales = (which == 0 ? key_scales : value_scales) + blk * scale_block_stride + head;
    // (one lane reads the scale that one lane replaces below)
    if (h == 0) s_old[which] = fresh ? 0.f : *scales;
    __syncthreads();
    const float old = s_old[which];
#pragma unroll
    for (int i = 0; i < H / 64; ++i) {
      amax = max(amax, s_max[which][0][i]);
      inf |= s_max[which][1][i];
    }
    const float scale = fmaxf(needed_scale(amax), old);
    const float inv = 1.f / scale;  // (exact for powers of two)
    const bool grown = !fresh && scale > old;
    const float ratio = old / scale;
    if (h == 0) *scales = scale;
    const bool any_inf = inf != 0;

    auto quantised = [&](float x) {
      x *= inv;
      if (any_inf) x = x > 448.f ? 448.f : x < -448.f ? -448.f : x;  // (NaN stays)
      return x;
    };
    uint8_t* tile = (which == 0 ? key_cache : value_cache) + blk * block_stride +
                    (int64_t)head * head_stride;
    uint4* units = reinterpret_cast<uint4*>(tile);
    const T* rows = reinterpret_cast<const T*>(s_rows[which]);
    if (which == 0) {
      // unit (chunk c, offset): 16 dims of a token
      for (int i = h; i < NU; i += H) {
        const int off = i % BS, c = i / BS;
        if ((have >> off) & 1u) {
          uint32_t w[4];
          float f[16];
          const uint4* r = reinterpret_cast<const uint4*>(rows + off * D + c * 16);
#pragma unroll
          for (int q = 0; q < 16 / E; ++q)
            widen<T>(r[q], *reinterpret_cast<float(*)[E]>(f + q * E));
#pragma unroll
          for (int q = 0; q < 4; ++q)
            w[q] = fp8_pair<true>(quantised(f[4 * q + 2]), quantised(f[4 * q + 3]),
                                  fp8_pair<false>(quantised(f[4 * q]), quantised(f[4 * q + 1]), 0u));
          units[i] = make_uint4(w[0], w[1], w[2], w[3]);
        } else if (grown) {
          const uint4 v = units[i];
          units[i] = make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio),
                                rescale4(v.w, ratio));
        }
      }
    } else {
      // unit: 16 tokens of a dim (8-token blocks: 8 of two dims)
      for (int i = h; i < NU; i += H) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (have != kAll) {
          const uint4 v = units[i];
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
          if (grown) {
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = rescale4(w[q], ratio);
          }
        }
        const int off0 = BS >= 16 ? (i % (BS >= 16 ? BS / 16 : 1)) * 16 : 0;
        const uint32_t mine = (uint32_t)(have >> off0);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          // four bytes, of tokens off .. off + 3 of a dim
          const int off = off0 + (BS >= 16 ? 4 * q : (4 * q) % 8);
          const int d = BS >= 16 ? i / (BS >= 16 ? BS / 16 : 1) : 2 * i + q / 2;
          const uint32_t m = (mine >> (off - off0)) & 15u;
          if (m == 0) continue;
          uint32_t b = 0, put = 0;
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool in = (m >> e) & 1u;
            x[e] = in ? quantised(load_as_f32(rows + (off + e) * D + d)) : 0.f;
            put |= in ? 0xffu << (8 * e) : 0u;
          }
          b = fp8_pair<true>(x[2], x[3], fp8_pair<false>(x[0], x[1], 0u));
          w[q] = (w[q] & ~put) | (b & put);
        }
        units[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncthreads();  // (s_tok and s_rows are taken again)
  }
}

// Few tokens have a workgroup each, which makes the most of them when each is in
// a block of its own; from kAppendWide tokens on a workgroup looks through a
// block's worth of tokens for those that lead one.
constexpr int64_t kAppendWide = 2048;

template <typename T, int D, int BS>
hipError_t launch_append(const ScaledAppendArgs& a, const CacheGeom& g, hipStream_t stream) {
  auto go = [&](auto w) {
    constexpr int W = decltype(w)::value;
    const int64_t grid = (a.num_tokens + W - 1) / W * g.num_kv_heads;
    hipLaunchKernelGGL((scaled_append_kernel<T, D, BS, W>), dim3((unsigned)grid),
                       dim3(W == 1 ? 128 : 256), 0, stream, static_cast<const T*>(a.key),
                       static_cast<const T*>(a.value), a.key_token_stride, a.value_token_stride,
                       a.key_scales, a.value_scales, a.scale_block_stride,
                       static_cast<uint8_t*>(a.key_cache), static_cast<uint8_t*>(a.value_cache),
                       a.slot_mapping, a.num_tokens, g.num_blocks, g.block_stride, g.head_stride,
                       g.num_kv_heads);
    return hipGetLastError();
  };
  if (a.num_tokens < kAppendWide) return go(std::integral_constant<int, 1>{});
  return go(std::integral_constant<int, BS>{});
}

template <typename T>
hipError_t launch_append_t(const ScaledAppendArgs& a, const CacheGeom& g, hipStream_t stream) {
#define VPA_SCALED(DV, BV) \
  if (g.head_dim == DV && g.block_size == BV) return launch_append<T, DV, BV>(a, g, stream);
#define VPA_SCALED_D(DV) VPA_SCALED(DV, 8) VPA_SCALED(DV, 16) VPA_SCALED(DV, 32)
  VPA_SCALED_D(64) VPA_SCALED_D(96) VPA_SCALED_D(128) VPA_SCALED_D(192) VPA_SCALED_D(256)
#undef VPA_SCALED_D
#undef VPA_SCALED
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_scaled_append(int dtype, const ScaledAppendArgs& a, const CacheGeom& g,
                                hipStream_t stream) {
  switch (dtype) {
    case VPA_DTYPE_BF16:
      return launch_append_t<bf16_t>(a, g, stream);
    case VPA_DTYPE_F16:
      return launch_append_t<f16_t>(a, g, stream);
    default:
      return launch_append_t<float>(a, g, stream);
  }
}

// Rows: up to 64 of a (sequence, kv head) split the keys over the waves, more
// have a wave per 16 or 32 of them. Keys: chunks over workgroups until there are
// two workgroups per compute unit of an MI355X (256), of at least 256 keys and,
// where there are enough workgroups, at most 2048, so that a batch's long
// contexts do not run on alone. The numbers are constants, not the device's:
// results and workspace do not depend on a partition's size.
ScaledPlan scaled_plan(int dtype, int32_t num_seqs, int32_t max_query_len, int32_t max_ctx,
                       int64_t total_rows, int32_t num_heads, int32_t num_kv_heads,
                       int32_t head_dim) {
  constexpr int64_t kWorkgroups = 512, kLeast = 256, kMost = 2048;
  ScaledPlan p{};
  const int64_t rows = (int64_t)max_query_len * (num_heads / num_kv_heads);
  const bool two = dtype != VPA_DTYPE_F32 && head_dim <= 128;
  p.nq = two && rows > 16 ? 2 : 1;
  p.split_keys = rows <= 64 ? 1 : 0;
  p.lds_rows = p.split_keys ? (int32_t)(rows < 16 * p.nq ? rows : 16 * p.nq) : 0;
  const int64_t per = p.split_keys ? 16 * p.nq : 64 * p.nq;
  const int64_t tiles = (rows + per - 1) / per;
  p.tiles = (int32_t)tiles;
  const int64_t units = (int64_t)num_seqs * num_kv_heads * tiles;
  const int64_t chunks = units >= kWorkgroups ? 1 : (kWorkgroups + units - 1) / units;
  int64_t tokens = ((max_ctx + chunks - 1) / chunks + kLeast - 1) / kLeast * kLeast;
  if (p.split_keys && tokens > kMost) tokens = kMost;
  if (tokens < kLeast) tokens = kLeast;
  p.chunk_tokens = (int32_t)tokens;
  p.max_chunks = (int32_t)((max_ctx + tokens - 1) / tokens);
  if (p.max_chunks < 1) p.max_chunks = 1;
  p.grid = units * p.max_chunks;
  p.workspace_bytes =
      p.max_chunks > 1 ? (size_t)total_rows * num_heads * p.max_chunks * (head_dim + 2) * 4 : 0;
  return p;
}

}  // namespace vpa
