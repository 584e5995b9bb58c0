// Eviction of cached tokens by their accumulated attention weight for gfx950.
//
// For each sequence s of L > budget tokens and each kv head j, `budget` tokens
// are kept: the first keep_first, the last keep_last, and of the rest the ones
// with the highest scores[s, j, t] (equal scores: the lower index; a NaN below
// every number). The kept tokens move to the front in their order, in the key
// cache, the value cache and the scores, so the sequence goes on as one of
// `budget` tokens in the blocks it has; the scores behind them become 0. The
// tiles of a (block, kv head) pair are a head's own, so every head keeps its own
// tokens under one shared block table. Sequences of at most `budget` tokens stay
// as they are.
//
// select: one workgroup per (sequence, kv head) finds the threshold score by
//   counting digits from the top of the scores' order-preserving bit patterns (11,
//   11 and 10 bits), then walks the tokens once, in order, to write the kept
//   indices and the moved scores. Bound by its few dependent passes over a row.
// move: in place. Kept index i is at or past i, so whoever moves the kept tokens
//   of one stretch after another never overwrites one that is still to be
//   read, as long as a stretch is read whole before it is written. K units of
//   different dims and V rows of different dims never meet, so the work splits
//   over the dims without any order between workgroups: one short sequence still
//   fills the chip. Bound by the bytes it moves.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr uint32_t kNone = 0xffffffffu;

// Order-preserving pattern of a score: NaN 0, then -inf .. +inf; -0 is +0.
__device__ __forceinline__ uint32_t score_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int context_of(const EvictArgs& a, int s, int bs) {
  return (int)min((uint64_t)min(a.context_lens[s], (uint32_t)a.max_ctx),
                  (uint64_t)a.block_table_stride * (uint64_t)bs);
}

// Inclusive sum over the workgroup's threads before and with this one, and the
// total. Every thread calls it; s_w is free again after the next barrier.
__device__ __forceinline__ int group_scan(int v, int* s_w, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int in = wave_scan_i32(v);
  if (lane == 63) s_w[wave] = in;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const int n = s_w[w];
    before += w < wave ? n : 0;
    total += n;
  }
  return before + in;
}

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a,
                                                                   int32_t num_kv_heads, int32_t bs) {
  __shared__ int s_hist[kBins];
  __shared__ int s_w[2][kSelWaves];
  __shared__ int s_digit, s_rank;
  const int j = (int)(blockIdx.x % (uint32_t)num_kv_heads);
  const int s = (int)(blockIdx.x / (uint32_t)num_kv_heads);
  const int tid = threadIdx.x;
  const int L = context_of(a, s, bs);
  uint32_t* kept = a.kept + ((int64_t)s * num_kv_heads + j) * a.budget;
  if (j == 0 && tid == 0) a.new_lens[s] = (uint32_t)min(L, a.budget);
  if (L <= a.budget) {  // nothing to evict
    for (int i = tid; i < a.budget; i += kSelThreads) kept[i] = i < L ? (uint32_t)i : kNone;
    return;
  }
  float* score = a.scores + s * a.score_seq_stride + j * a.score_head_stride;
  const int lo = a.keep_first, hi = L - a.keep_last;  // lo < hi: budget >= first + last
  const int want = a.budget - a.keep_first - a.keep_last;

  // threshold: `prefix` is the pattern of the want-th highest score of the
  // middle, `rank` how many scores equal to it are kept
  uint32_t prefix = 0;
  int rank = want;
  if (want > 0) {
    int shift = 32;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t seen = pass == 0 ? 0u : 0xffffffffu << shift;
      shift -= bits;
      for (int i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0;
      __syncthreads();
      for (int t = lo + tid; t < hi; t += kSelThreads) {
        const uint32_t key = score_key(score[t]);
        if ((key & seen) == prefix) atomicAdd(&s_hist[(key >> shift) & ((1u << bits) - 1)], 1);
      }
      __syncthreads();
      // bins from the highest down, two per thread; the one where the count
      // reaches `rank`
      const int b = kBins - 1 - 2 * tid;
      const int n0 = s_hist[b], n1 = s_hist[b - 1];
      int total;
      const int upto = group_scan(n0 + n1, s_w[0], total);
      const int before = upto - n0 - n1;
      if (before < rank && rank <= upto) {
        const bool second = rank > before + n0;
        s_digit = second ? b - 1 : b;
        s_rank = rank - before - (second ? n0 : 0);
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      rank = s_rank;
      __syncthreads();
    }
  }
  // one walk in order: kept indices and scores, a stretch of 1024 tokens read
  // before its part is written (at or before it)
  int done = 0, equal = 0;
  for (int t0 = 0; t0 < L; t0 += kSelThreads) {
    const int t = t0 + tid;
    const float f = t < L ? score[t] : 0.f;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // read before the barriers below
    const bool middle = t >= lo && t < hi;
    const uint32_t key = score_key(f);
    const bool eq = want > 0 && middle && key == prefix;
    int eq_total, total;
    const int eq_rank = equal + group_scan(eq ? 1 : 0, s_w[0], eq_total);  // 1-based
    const bool keep = t < L && (!middle || (want > 0 && (key > prefix || (eq && eq_rank <= rank))));
    const int pos = done + group_scan(keep ? 1 : 0, s_w[1], total) - 1;
    // (the wait above and group_scan's barriers stand between every thread's
    // read of its score and the writes below)
    if (keep && pos < a.budget) {
      kept[pos] = (uint32_t)t;
      score[pos] = f;
    }
    equal += eq_total;
    done += total;
    __syncthreads();
  }
  for (int t = a.budget + tid; t < L; t += kSelThreads) score[t] = 0.f;
}

constexpr int kMoveThreads = 256;

// Waits until this wave's loads have arrived, then for the workgroup's other
// waves: no store after it can overtake a load before it.
__device__ __forceinline__ void loads_done_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One workgroup per (sequence, kv head, K or V, group of `dims` dims): moves
// those dims of every kept token, kStretch tokens at a time.
// E: cache element (moved as it is).
template <typename E, int BS>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(
    EvictArgs a, int32_t num_kv_heads, int32_t head_dim, int32_t dims, int64_t num_blocks,
    int64_t block_stride, int64_t head_stride) {
  constexpr int X = 16 / (int)sizeof(E);
  constexpr int kStretch = 256;
  const int groups = head_dim / dims;
  uint32_t w = blockIdx.x;
  const int dg = (int)(w % (uint32_t)groups);
  w /= (uint32_t)groups;
  const bool value = w & 1;
  w >>= 1;
  const int j = (int)(w % (uint32_t)num_kv_heads);
  const int s = (int)(w / (uint32_t)num_kv_heads);
  const int L = context_of(a, s, BS);
  if (L <= a.budget) return;
  const uint32_t* kept = a.kept + ((int64_t)s * num_kv_heads + j) * a.budget;
  const uint32_t* table = a.block_tables + (int64_t)s * a.block_table_stride;
  E* cache = static_cast<E*>(value ? a.value_cache : a.key_cache) + j * head_stride;
  const int d0 = dg * dims;
  const int i_thr = threadIdx.x;  // token of the stretch
  for (int i0 = 0; i0 < a.budget; i0 += kStretch) {
    const int n = min(kStretch, a.budget - i0);
    if (kept[i0 + n - 1] == (uint32_t)(i0 + n - 1)) continue;  // all in place
    const int i = i0 + i_thr;
    const uint32_t src = i_thr < n ? kept[i] : kNone;
    // a token whose block is not one of the pool's (a table entry past it) is
    // neither read nor written
    const bool live = i_thr < n && src < (uint32_t)L;
    const uint32_t sb = live ? table[src / BS] : kNone, db = live ? table[i / BS] : kNone;
    const bool from = (int64_t)sb < num_blocks && live, to = from && (int64_t)db < num_blocks;
    const E* ps = cache + (from ? (int64_t)sb : 0) * block_stride;
    E* pd = cache + (to ? (int64_t)db : 0) * block_stride;
    if (!value) {
      for (int d = 0; d < dims; d += 4 * X) {
        uint4 u[4] = {};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (to && d + q * X < dims)
            u[q] = *reinterpret_cast<const uint4*>(ps + (d0 + d + q * X) * BS + (src % BS) * X);
        loads_done_barrier();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (to && d + q * X < dims)
            *reinterpret_cast<uint4*>(pd + (d0 + d + q * X) * BS + (i % BS) * X) = u[q];
      }
    } else {
      for (int d = 0; d < dims; d += 16) {
        E u[16] = {};
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (to && d + q < dims) u[q] = ps[(d0 + d + q) * BS + src % BS];
        loads_done_barrier();
#pragma unroll
        for (int q = 0; q < 16; ++q)
          if (to && d + q < dims) pd[(d0 + d + q) * BS + i % BS] = u[q];
      }
    }
  }
}

template <typename E>
hipError_t move_typed(const EvictArgs& a, const CacheGeom& g, hipStream_t stream) {
  constexpr int X = 16 / (int)sizeof(E);
  const int dims = g.head_dim % 32 == 0 ? 32 : std::max(16, X);
  const int64_t grid =
      (int64_t)a.num_seqs * g.num_kv_heads * 2 * (g.head_dim / dims);
  const auto k = g.block_size == 8    ? evict_move_kernel<E, 8>
                 : g.block_size == 16 ? evict_move_kernel<E, 16>
                                      : evict_move_kernel<E, 32>;
  hipLaunchKernelGGL(k, dim3((uint32_t)grid), dim3(kMoveThreads), 0, stream, a, g.num_kv_heads,
                     g.head_dim, dims, g.num_blocks, g.block_stride, g.head_stride);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_evict(int cache_dtype, const EvictArgs& a, const CacheGeom& g,
                        hipStream_t stream) {
  hipLaunchKernelGGL(evict_select_kernel, dim3((uint32_t)((int64_t)a.num_seqs * g.num_kv_heads)),
                     dim3(kSelThreads), 0, stream, a, g.num_kv_heads, g.block_size);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (cache_dtype == VPA_DTYPE_F32) return move_typed<uint32_t>(a, g, stream);
  if (cache_dtype == VPA_DTYPE_FP8_E4M3) return move_typed<uint8_t>(a, g, stream);
  return move_typed<uint16_t>(a, g, stream);
}

}  // namespace vpa
