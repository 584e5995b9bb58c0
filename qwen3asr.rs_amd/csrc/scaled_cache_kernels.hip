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
// One wave owns K or V of a (block, kv head) of the call: the first of the
// neighbouring tokens that share a block leads, and its wave takes them all, without
// a barrier. Rows are staged in LDS, where V is read across tokens. V's bytes of one
// token lie in every 16-byte vector of its tile, so a partly filled tile is read and
// written whole: contiguous vectors instead of single bytes in every 32-byte sector;
// the tile's loads are under way before the rows' largest element is known.
// A prompt's append is bound by HBM (8 kv heads of 128 dims, bf16: 32768 tokens 39 us
// for 202 MB, 5.2 TB/s read and written), a decode step's by the chain of its loads and
// the tiles read and written around single tokens (256 tokens 7.4 us for 17 MB; with a
// workgroup of 256 lanes for K and V of a block, and its barriers, 9.4 and 69 us).

#include <algorithm>
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

// Four bytes scaled by `ratio` (a scale over a larger one).
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return fp8_pair<true>(hi[0] * ratio, hi[1] * ratio,
                        fp8_pair<false>(lo[0] * ratio, lo[1] * ratio, 0u));
}

template <typename T, int D, int BS, int W>
__global__ __launch_bounds__(64) void scaled_append_kernel(
    const T* __restrict__ key, const T* __restrict__ value, int64_t key_token_stride,
    int64_t value_token_stride, float* __restrict__ key_scales, float* __restrict__ value_scales,
    int64_t scale_block_stride, uint8_t* __restrict__ key_cache, uint8_t* __restrict__ value_cache,
    const int64_t* __restrict__ slot_mapping, int64_t num_tokens, int64_t num_blocks,
    int64_t block_stride, int64_t head_stride, int32_t num_kv_heads) {
  constexpr int VR = D * (int)sizeof(T) / 16;  // 16-byte vectors of a row
  constexpr int E = 16 / (int)sizeof(T);       // elements of one
  constexpr int NV = BS * VR;                  // vectors of all rows
  constexpr int NR = (NV + 63) / 64;           // of a lane
  constexpr int NU = D * BS / 16;              // 16-byte units of a tile
  constexpr int NL = (NU + 63) / 64;           // units of a lane
  // a partly filled tile is loaded before its rows are looked at where the registers
  // allow it
  static constexpr bool kAhead = NL <= 4;
  static constexpr int kUnroll = kAhead ? NL : 1;
  static_assert(W <= 32, "a window and the end of its last run fit 64 tokens");
  __shared__ __align__(16) uint4 s_rows[BS * VR];
  __shared__ int s_tok[BS];  // last token of the run at each offset, from t0 on; -1: none

  const int lane = threadIdx.x;
  // kv heads fastest: neighbouring workgroups read neighbouring slices of a row
  uint32_t w = blockIdx.x;
  const int head = (int)(w % (uint32_t)num_kv_heads);
  w /= (uint32_t)num_kv_heads;
  const bool is_k = (w & 1u) == 0;
  const int64_t t0 = (int64_t)(w >> 1) * W;

  // the block of a slot, -1: padding or past the pool
  auto block_of = [&](int64_t slot) {
    const int64_t b = slot < 0 ? -1 : slot / BS;
    return b < num_blocks ? b : (int64_t)-1;
  };
  auto slot_at = [&](int64_t t) {
    return t >= 0 && t < num_tokens ? slot_mapping[t] : (int64_t)-1;
  };
  // lane l: token t0 - 1 + l; a run that starts at lane 1 .. W ends before lane 63
  // where its slots are distinct
  const int64_t my_slot = slot_at(t0 - 1 + lane);
  const int64_t my_blk = block_of(my_slot);
  const int64_t before = __shfl_up(my_blk, 1, 64);
  uint64_t leaders = __ballot(lane >= 1 && lane <= W && my_blk >= 0 && my_blk != before);

  const T* src = is_k ? key : value;
  const int64_t stride = is_k ? key_token_stride : value_token_stride;
  for (; leaders != 0; leaders &= leaders - 1) {
    const int l = __builtin_ctzll(leaders);
    const int64_t blk = __shfl(my_blk, l, 64);
    // ---- the run's tokens by offset ----
    if (lane < BS) s_tok[lane] = -1;
    lds_wave_sync();
    {
      const uint64_t other = __ballot(lane >= l && my_blk != blk);
      const int end = other != 0 ? __builtin_ctzll(other) : 64;
      if (lane >= l && lane < end) atomicMax(&s_tok[my_slot % BS], lane - 1);
      for (int64_t base = t0 + 63; end == 64; base += 64) {  // (repeated slots)
        const int64_t slot = slot_at(base + lane);
        const uint64_t out = __ballot(block_of(slot) != blk);
        const int n = out != 0 ? __builtin_ctzll(out) : 64;
        if (lane < n) atomicMax(&s_tok[slot % BS], (int)(base + lane - t0));
        if (n < 64) break;
      }
    }
    lds_wave_sync();
    const uint64_t have = __ballot(lane < BS && s_tok[lane % BS] >= 0);
    const bool fresh = (have & 1u) != 0;
    constexpr uint64_t kAll = (1ull << BS) - 1;

    float* scales = (is_k ? key_scales : value_scales) + blk * scale_block_stride + head;
    const float old = fresh ? 0.f : *scales;
    uint8_t* tile = (is_k ? key_cache : value_cache) + blk * block_stride +
                    (int64_t)head * head_stride;
    uint4* units = reinterpret_cast<uint4*>(tile);
    uint4 ahead[kUnroll];
    if (kAhead && have != kAll) {
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (NU % 64 == 0 || 64 * k + lane < NU) ahead[k] = units[64 * k + lane];
    }
    auto held = [&](int k) { return kAhead ? ahead[k % kUnroll] : units[64 * k + lane]; };
    auto rescaled = [&](const uint4& v, float ratio) {
      return make_uint4(rescale4(v.x, ratio), rescale4(v.y, ratio), rescale4(v.z, ratio),
                        rescale4(v.w, ratio));
    };

    // ---- rows to LDS, their largest element ----
    const T* rows0 = src + t0 * stride + (int64_t)head * D;
    uint32_t amax = 0, special = 0;
    // vectors under way together
    constexpr int U = NR <= 8 ? NR : NR % 8 == 0 ? 8 : 6;
    static_assert(NR % U == 0, "whole groups of vectors");
    for (int r = 0; r < NR; r += U) {
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = 64 * (r + u) + lane, t = NV % 64 == 0 || i < NV ? s_tok[i / VR] : -1;
        v[u] = t >= 0 ? *reinterpret_cast<const uint4*>(rows0 + t * stride + (i % VR) * E)
                      : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (NV % 64 == 0 || 64 * (r + u) + lane < NV) s_rows[64 * (r + u) + lane] = v[u];
        float f[E];
        widen<T>(v[u], f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t a = __float_as_uint(f[e]) & 0x7fffffffu;
          const uint32_t over = 0x7f7fffffu - a;  // (its sign: infinite or NaN)
          amax = max(amax, a & ~(uint32_t)((int32_t)over >> 31));
          special |= over;
        }
      }
    }
    // (as f32: numbers without a sign are ordered as their bits)
    amax = __float_as_uint(wave_max_dpp(__uint_as_float(amax)));
    const bool any_special = __ballot((special >> 31) != 0) != 0;
    const float scale = fmaxf(needed_scale(amax), old);
    const float inv = 1.f / scale;  // (exact for powers of two)
    const bool grown = !fresh && scale > old;
    const float ratio = old / scale;
    if (lane == 0) *scales = scale;
    lds_wave_sync();

    auto quantised = [&](auto clamped, float x) {
      x *= inv;
      if constexpr (decltype(clamped)::value) x = x > 448.f ? 448.f : x < -448.f ? -448.f : x;
      return x;  // (NaN stays)
    };
    const T* rows = reinterpret_cast<const T*>(s_rows);
    auto write = [&](auto clamped) {
      if (is_k) {
        // unit (chunk c, offset): 16 dims of a token
#pragma unroll kUnroll
        for (int k = 0; k < NL; ++k) {
          const int i = 64 * k + lane;
          if (NU % 64 != 0 && i >= NU) break;
          const int off = i % BS, c = i / BS;
          if ((have >> off) & 1u) {
            uint32_t q4[4];
            float f[16];
            const uint4* r = reinterpret_cast<const uint4*>(rows + off * D + c * 16);
#pragma unroll
            for (int q = 0; q < 16 / E; ++q)
              widen<T>(r[q], *reinterpret_cast<float(*)[E]>(f + q * E));
#pragma unroll
            for (int q = 0; q < 4; ++q)
              q4[q] = fp8_pair<true>(quantised(clamped, f[4 * q + 2]), quantised(clamped, f[4 * q + 3]),
                                     fp8_pair<false>(quantised(clamped, f[4 * q]), quantised(clamped, f[4 * q + 1]), 0u));
            units[i] = make_uint4(q4[0], q4[1], q4[2], q4[3]);
          } else {
            const uint4 v = held(k);
            units[i] = grown ? rescaled(v, ratio) : v;
          }
        }
      } else {
        // unit: 16 tokens of a dim (8-token blocks: 8 of two dims)
#pragma unroll kUnroll
        for (int k = 0; k < NL; ++k) {
          const int i = 64 * k + lane;
          if (NU % 64 != 0 && i >= NU) break;
          uint32_t q4[4] = {0u, 0u, 0u, 0u};
          if (have != kAll) {
            const uint4 v = grown ? rescaled(held(k), ratio) : held(k);
            q4[0] = v.x, q4[1] = v.y, q4[2] = v.z, q4[3] = v.w;
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
            uint32_t put = 0;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool in = (m >> e) & 1u;
              x[e] = in ? quantised(clamped, load_as_f32(rows + (off + e) * D + d)) : 0.f;
              put |= in ? 0xffu << (8 * e) : 0u;
            }
            const uint32_t b = fp8_pair<true>(x[2], x[3], fp8_pair<false>(x[0], x[1], 0u));
            q4[q] = (q4[q] & ~put) | (b & put);
          }
          units[i] = make_uint4(q4[0], q4[1], q4[2], q4[3]);
        }
      }
    };
    if (any_special) write(std::true_type{});  // (uniform)
    else write(std::false_type{});
    lds_wave_sync();  // (s_tok and s_rows are taken again)
  }
}

// Few tokens have two waves each (and head), which makes the most of them when each
// is in a block of its own; from kAppendWide tokens on a wave looks through a block's
// worth of tokens for those that lead one.
constexpr int64_t kAppendWide = 2048;

template <typename T, int D, int BS>
hipError_t launch_append(const ScaledAppendArgs& a, const CacheGeom& g, hipStream_t stream) {
  auto go = [&](auto w) {
    constexpr int W = decltype(w)::value;
    const int64_t grid = 2 * ((a.num_tokens + W - 1) / W) * g.num_kv_heads;
    hipLaunchKernelGGL((scaled_append_kernel<T, D, BS, W>), dim3((unsigned)grid),
                       dim3(64), 0, stream, static_cast<const T*>(a.key),
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

// Rows: a wave takes 16 or 32 of a (sequence, kv head). Of up to 256 rows the waves of a
// workgroup share each such tile and split the keys, unless there are enough tiles for
// waves of their own: 1024 for contexts of up to 512 keys (32 times 200 rows over 100
// keys: 33 us split, 14 not; 128 decode steps of 60 to 128 keys 10.8, 7.6), 2048 beyond
// (64 times 200 rows over 2000 keys: 184, 173; 40 rows each, 1024 tiles: 61, 66), where
// one tile alone is always split (a decode). Contexts of one step of 64 keys have nothing
// to split (256 of them: 17 us, 8), and more than 256 rows go without (8000 keys, 128
// rows: 19 us split, 24 not; a batch of 64 with 1024 rows each keeps its waves busy). That
// border is the batch's: one to four prompts of 1024 rows (512 positions) would gain by the
// split over shorter contexts (one over 2000 keys 38 us, 23 split; over 6500 56, 54; four
// over 4000 102, 89) and lose over long ones (four over 8000 177, 183; two over 6000 80, 81).
// Waves with rows of their own are a workgroup each: four to one end at different keys
// and leave the last one's without rows (64 times 400 rows: 68 us for 53; 512 rows each
// of 32 prompts, head dim 256: 548, 496, both of a build of their own; never more than 2 %
// faster).
// Keys: chunks over workgroups until an MI355X has one of four waves (split keys) per
// compute unit or two waves (with rows of their own, which finish at different times) per
// SIMD, of at least 256 keys; where the waves split the keys and there are enough
// workgroups at most 4096, so that a batch's long contexts do not run on alone. Contexts
// of up to 512 keys stay whole, as the second launch costs what it saves or more (a
// prompt of 512 rows: 19.4 us in two chunks, 15.8 whole). (Twice as many chunks of a
// prompt's rows pay where contexts differ, 3 of 2000 to 8000: 146 us for 197, and cost as
// much where they do not, 129 for 109; the lengths are the device's.)
// The numbers are constants, not the device's: results and workspace do not depend on a
// partition's size.
ScaledPlan scaled_plan(int dtype, int32_t num_seqs, int32_t max_query_len, int32_t max_ctx,
                       int64_t total_rows, int32_t num_heads, int32_t num_kv_heads,
                       int32_t head_dim) {
  constexpr int64_t kLeast = 256, kWhole = 512, kMost = 4096;
  ScaledPlan p{};
  const int64_t rows = (int64_t)max_query_len * (num_heads / num_kv_heads);
  p.nq = dtype != VPA_DTYPE_F32 && rows > 16 ? 2 : 1;
  const int64_t row_tiles = (rows + 16 * p.nq - 1) / (16 * p.nq);
  const int64_t units = row_tiles * num_seqs * num_kv_heads;
  const bool few = units < (max_ctx <= kWhole ? 1024 : 2048) ||
                   (row_tiles == 1 && max_ctx > kWhole);
  p.split_keys = rows <= 256 && max_ctx > 64 && few ? 1 : 0;
  p.lds_rows = p.split_keys ? (int32_t)(rows < 16 * p.nq ? rows : 16 * p.nq) : 0;
  p.tiles = (int32_t)row_tiles;
  int64_t tokens = max_ctx;
  if (max_ctx > kWhole) {
    const int64_t wanted = p.split_keys ? 256 : 2048;
    const int64_t chunks = units >= wanted ? 1
                           : p.split_keys  ? (wanted + units - 1) / units
                                           : wanted / units;
    tokens = (max_ctx + chunks - 1) / chunks;
    if (p.split_keys && tokens > kMost) tokens = kMost;
  }
  const int64_t step = p.split_keys ? kLeast : 64;
  tokens = std::max((tokens + step - 1) / step * step, kLeast);
  p.chunk_tokens = (int32_t)tokens;
  p.max_chunks = (int32_t)((max_ctx + tokens - 1) / tokens);
  if (p.max_chunks < 1) p.max_chunks = 1;
  p.grid = units * p.max_chunks;
  p.workspace_bytes =
      p.max_chunks > 1 ? (size_t)total_rows * num_heads * p.max_chunks * (head_dim + 2) * 4 : 0;
  return p;
}

}  // namespace vpa
