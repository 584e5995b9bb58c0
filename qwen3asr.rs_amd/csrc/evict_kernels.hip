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
//   fills the chip. Bound by the bytes it moves, whole columns read.
//
// Measured, 8 heads of 128 dims in 16 bits: 64 sequences of 600 to 4096 tokens cut to
// 1024 take 15 + 198 us (666 MB of columns read, 250 MB written: 4.6 TB/s, 0.97 of a
// large copy); the same of 1088 tokens each 11 + 118 us; one of 8192 cut to 4096 takes
// 13 + 18 us.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

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
template <int kWaves>
__device__ __forceinline__ int group_scan(int v, int* s_w, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int in = wave_scan_i32(v);
  if (lane == 63) s_w[wave] = in;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int n = s_w[w];
    before += w < wave ? n : 0;
    total += n;
  }
  return before + in;
}

// Items of a chunk held by a thread: wave w has tokens w * 64 * R + 64 i + lane of
// the chunk's kThreads * R, so a wave's tokens are one run.
constexpr int kItems = 16;

// One workgroup per (sequence, kv head). A row of up to 16 tokens per thread is
// read once and stays in registers for the three digits and the final walk; a
// longer one is read chunk by chunk in each of the four passes.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictArgs a, int32_t num_kv_heads,
                                                                int32_t bs_log2) {
  const int bs = 1 << bs_log2;
  constexpr int kWaves = kThreads / 64;
  constexpr int kChunk = kThreads * kItems;
  constexpr int kPer = kBins / kThreads;  // bins per thread
  __shared__ int s_hist[3][kBins];  // (a digit's each: cleared at once)
  __shared__ int s_w[2][kWaves];
  __shared__ int s_digit, s_rank, s_count;
  const int j = (int)(blockIdx.x % (uint32_t)num_kv_heads);
  const int s = (int)(blockIdx.x / (uint32_t)num_kv_heads);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int L = context_of(a, s, bs);
  const int64_t pair = (int64_t)s * num_kv_heads + j;
  uint32_t* kept = a.kept + pair * a.budget;
  if (j == 0 && tid == 0) a.new_lens[s] = (uint32_t)min(L, a.budget);
  if (L <= a.budget) {  // nothing to evict
    for (int i = tid; i < a.budget; i += kThreads) kept[i] = i < L ? (uint32_t)i : kNone;
    return;
  }
  float* score = a.scores + s * a.score_seq_stride + j * a.score_head_stride;
  uint2* columns = a.columns + pair * a.max_columns;
  const int lo = a.keep_first, hi = L - a.keep_last;  // lo < hi: budget >= first + last
  const int want = a.budget - a.keep_first - a.keep_last;
  const int chunks = (L + kChunk - 1) / kChunk;
  // items per thread of a chunk
  auto items_of = [&](int c) { return (min(L - c * kChunk, kChunk) + kThreads - 1) / kThreads; };
  float f[kItems];
  uint32_t inside, middle;  // bit i: item i is one of the sequence's tokens; of its middle
  auto load_chunk = [&](int c) {
    const int R = items_of(c), t0 = c * kChunk + wave * 64 * R + lane;
    inside = middle = 0u;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int t = t0 + 64 * i;
      const bool in = i < R && t < L;
      f[i] = 0.f;
      if (in) f[i] = score[t];
      inside |= (uint32_t)in << i;
      middle |= (uint32_t)(in && t >= lo && t < hi) << i;
    }
    // (opaque, so that the bits stay bits: as comparisons kept from pass to pass
    // they would not fit the scalar registers)
    asm volatile("" : "+v"(inside), "+v"(middle));
  };
  load_chunk(0);
#pragma unroll
  for (int i = tid; i < 3 * kBins; i += kThreads) s_hist[i / kBins][i % kBins] = 0;
  __syncthreads();

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
      for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load_chunk(c);
        const int R = items_of(c);
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
          if (i >= R) continue;  // (uniform)
          const uint32_t key = score_key(f[i]);
          if (((middle >> i) & 1u) && (key & seen) == prefix)
            atomicAdd(&s_hist[pass][(key >> shift) & ((1u << bits) - 1)], 1);
        }
      }
      __syncthreads();
      // bins from the highest down, kPer per thread; the one where the count
      // reaches `rank`
      const int b = kBins - 1 - kPer * tid;
      int n[kPer], mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        n[i] = s_hist[pass][b - i];
        mine += n[i];
      }
      int total;
      const int upto = group_scan<kWaves>(mine, s_w[0], total);
      int before = upto - mine;
      if (before < rank && rank <= upto) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          if (before < rank && rank <= before + n[i]) {
            s_digit = b - i;
            s_rank = rank - before;
            s_count = n[i];
          }
          before += n[i];
        }
      }
      __syncthreads();
      prefix |= (uint32_t)s_digit << shift;
      rank = s_rank;
      // all scores of the digit stay (often one, after two digits): they are above the
      // pattern before its first
      if (pass == 1 && rank == s_count && prefix != 0) {
        --prefix;
        rank = 0;
        break;
      }
    }
  }
  // in token order: kept indices, moved scores, and each table column's kept
  // tokens for the move. Every score of a chunk is read (waited for) before the
  // barrier, every write lies at or before the chunk's tokens.
  int done = 0, equal = 0;
  for (int c = 0; c < chunks; ++c) {
    if (chunks > 1) {
      __syncthreads();  // (the previous chunk's counts are read)
      load_chunk(c);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int R = items_of(c), t0 = c * kChunk + wave * 64 * R + lane;
    // bit i: token i of the thread is kept whatever its place among equals; is
    // one of the equals
    uint32_t above = 0, ties = 0;
    int n_above = 0, n_ties = 0;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const uint32_t key = score_key(f[i]);
      above |= (uint32_t)(want > 0 && key > prefix) << i;
      ties |= (uint32_t)(want > 0 && key == prefix) << i;
    }
    above = (above & middle) | (inside & ~middle);
    ties &= middle;
    asm volatile("" : "+v"(above), "+v"(ties));
    n_above = wave_sum_i32(__builtin_popcount(above));
    n_ties = wave_sum_i32(__builtin_popcount(ties));
    if (lane == 0) {
      s_w[0][wave] = n_above;
      s_w[1][wave] = n_ties;
    }
    __syncthreads();
    int eq = equal, kept_before = done;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int na = s_w[0][w], nt = s_w[1][w];
      // of a wave's ties those that are among the first `rank` stay
      const int take = min(max(rank - equal, 0), nt);
      if (w < wave) {
        eq += nt;
        kept_before += na + take;
      }
      equal += nt;
      done += na + take;
    }
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (i >= R) continue;  // (uniform)
      const int t = t0 + 64 * i;
      const uint64_t tie = __ballot((ties >> i) & 1u);
      const bool tie_kept = ((ties >> i) & 1u) && eq + __builtin_popcountll(tie & below) < rank;
      const bool mine = ((above >> i) & 1u) || tie_kept;
      const uint64_t keep = __ballot(mine);
      const int pos = kept_before + __builtin_popcountll(keep & below);
      if (mine && pos < a.budget) {
        kept[pos] = (uint32_t)t;
        score[pos] = f[i];
      }
      if ((lane & (bs - 1)) == 0 && t < L) {
        const uint32_t full = 0xffffffffu >> (32 - bs), mask = (uint32_t)(keep >> lane) & full;
        columns[t >> bs_log2] = make_uint2(mask, (uint32_t)pos);
        // the first column that loses a token: what lies before it stays in place
        if (mask != full && pos == t) a.first_column[pair] = (uint32_t)(t >> bs_log2);
      }
      eq += __builtin_popcountll(tie);
      kept_before += __builtin_popcountll(keep);
      __builtin_amdgcn_sched_barrier(0);  // (one item's lane masks at a time fit the scalar registers)
    }
  }
  __syncthreads();
  for (int t = a.budget + tid; t < L; t += kThreads) score[t] = 0.f;
}

// One workgroup per (sequence, kv head, K or V, group of DG dims): DG dims of a
// cache block are one run of DG * BS elements in the key tile (whole chunks) and
// in the value tile (whole rows) alike. The workgroup walks the table's columns in
// batches: it reads the runs of a batch's columns that have kept tokens, 16
// bytes per lane, into LDS as they lie, then gathers from there, 16 bytes at a
// time, what goes to each destination block, and writes runs of whole vectors
// (single elements of a value row only where a batch ends inside a vector). A
// column's kept tokens come from the selection as a bit mask and the place of the
// first; from them the batch makes a list of where each place's token lies in
// LDS, common to all its dims, so a gathered element costs one LDS read. (Putting
// each token's elements from registers to their places instead takes a
// predicated LDS write for every element that is read, kept or not: 330 us for 64
// sequences of 600 to 4096 tokens, 8 heads of 128 dims in 16 bits, cut to 1024
// tokens; 197 us so.) Reading whole columns costs nothing: a value row's 32-byte
// sector holds 16 tokens. The next two batches' runs are in flight while one is
// written: they lie behind everything that is written (a place is at or before
// the token that moves to it). Columns before the first evicted token stay, and
// columns without kept tokens are left out of the batches.
// E: cache element, moved as it is; BS tokens per block; NV vectors per thread and
// batch.
template <typename E, int BS, int DG, int kThreads, int NV>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(
    EvictArgs a, int32_t num_kv_heads, int32_t head_dim, int64_t num_blocks, int64_t block_stride,
    int64_t head_stride) {
  constexpr int EB = (int)sizeof(E);
  constexpr int X = 16 / EB;
  constexpr int VPB = DG * BS / X;            // 16-byte vectors of a block's run
  constexpr int kCols = kThreads * NV / VPB;  // columns of a batch
  constexpr int kTok = kCols * BS;            // tokens of a batch
  // a wave's vectors lie in one column (and its units in one block): its index,
  // and the addresses made from it, stay in scalar registers
  constexpr bool kUniform = VPB % 64 == 0;
  // A run in LDS. Value rows are read at one token by lanes of different rows, so
  // 8 bytes of padding follow every 256: rows that would share a bank do not.
  constexpr int kRunBytes = VPB * 16 + (VPB + 15) / 16 * 8;
  constexpr int RUN = (kRunBytes + 15) / 16 * 16 / EB;
  constexpr int U = BS < X ? BS : X;          // tokens of a value unit
  constexpr int kInfo = 512;  // columns whose masks, places and blocks wait in LDS
  static_assert(DG % X == 0 && kThreads * NV % VPB == 0 && kCols >= 1 && kInfo % (2 * kCols) == 0,
                "whole chunks, columns and pairs of batches");
  static_assert(kThreads == kInfo, "a column per thread");
  __shared__ __align__(16) E s_run[kCols * RUN];
  __shared__ __align__(16) uint32_t s_src[kTok + 2 * U];  // of each place: its token's byte in s_run
  __shared__ uint2 s_col[kInfo];                          // {mask, place of the first kept token}
  // offsets (elements) of the blocks of the columns and of the places, -1: absent
  __shared__ int64_t s_from[kInfo], s_to[kInfo + 1];
  __shared__ uint16_t s_list[kInfo];  // the columns with kept tokens
  __shared__ int s_p1, s_absent[2], s_listed[kThreads / 64];
  const int groups = head_dim / DG;
  uint32_t w = blockIdx.x;
  const int dg = (int)(w % (uint32_t)groups);
  w /= (uint32_t)groups;
  const bool value = w & 1;
  w >>= 1;
  const int j = (int)(w % (uint32_t)num_kv_heads);
  const int s = (int)(w / (uint32_t)num_kv_heads);
  const int64_t pair = (int64_t)s * num_kv_heads + j;
  const uint2* columns = a.columns + pair * a.max_columns;
  const uint32_t* table = a.block_tables + (int64_t)s * a.block_table_stride;
  auto offset_of = [&](int c) {
    const uint32_t b = table[c];
    return (int64_t)b < num_blocks ? (int64_t)b * block_stride : (int64_t)-1;
  };
  const int L = context_of(a, s, BS);
  if (L <= a.budget) return;  // (and the selection wrote no columns)
  // Where all columns fit, they are read at once (what lies past the context is
  // not used); else window by window.
  const bool whole = a.max_columns <= kInfo;
  if (whole)
    for (int i = threadIdx.x; i < a.max_columns; i += kThreads) {
      s_col[i] = columns[i];
      s_from[i] = offset_of(i);
    }
  const int c_begin = (int)a.first_column[pair];
  E* cache = static_cast<E*>(value ? a.value_cache : a.key_cache) + j * head_stride +
             (int64_t)dg * DG * BS;
  const int tid = threadIdx.x;
  const int c_end = (L + BS - 1) / BS;

  auto row_at = [](int row) { return row * BS + row * BS * EB / 256 * (8 / EB); };  // in a run
  auto uniform64 = [](int64_t v) {
    if constexpr (kUniform)
      return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                       (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
    else return v;
  };
  auto uniform = [](int v) {
    if constexpr (kUniform) return __builtin_amdgcn_readfirstlane(v);
    else return v;
  };
  if (tid < 2) s_absent[tid] = 0;
  int flip = 0, p0 = c_begin * BS;  // (nothing before c_begin moves)
  for (int sc = whole ? 0 : c_begin; sc < c_end; sc += kInfo) {
    const int n = min(kInfo, c_end - sc), to0 = whole ? 0 : p0 / BS;
    const int64_t* places = whole ? s_from : s_to;  // blocks from place to0 * BS on
    if (!whole) {
      __syncthreads();
      for (int i = tid; i <= n; i += kThreads) {
        if (i < n) {
          s_col[i] = columns[sc + i];
          s_from[i] = offset_of(sc + i);
        }
        s_to[i] = to0 + i < c_end ? offset_of(to0 + i) : -1;
      }
    }
    __syncthreads();
    // the columns that move, in order
    const bool moves = tid < n && (!whole || tid >= c_begin) && s_col[tid].x != 0;
    const uint64_t mask = __ballot(moves);
    if ((tid & 63) == 0) s_listed[tid >> 6] = __builtin_popcountll(mask);
    __syncthreads();
    int before = 0, listed = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) {
      before += i < tid >> 6 ? s_listed[i] : 0;
      listed += s_listed[i];
    }
    if (moves) s_list[before + __builtin_popcountll(mask & ((1ull << (tid & 63)) - 1))] = (uint16_t)tid;
    __syncthreads();
    // (a column whose block is not one of the pool's is neither read nor moved)
    auto load_data = [&](uint4(&u)[NV], int c0) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = uniform(c0 + (k * kThreads + tid) / VPB);
        u[k] = make_uint4(0u, 0u, 0u, 0u);
        if (c < listed) {
          const int64_t at = uniform64(s_from[s_list[c]]);
          if (at >= 0)
            u[k] = load_stream(reinterpret_cast<const uint4*>(cache + at) + (k * kThreads + tid) % VPB);
        }
      }
    };
    auto batch = [&](uint4(&u)[NV], int c0) {
      const int c_last = min(c0 + kCols, listed) - 1;
      const int aligned = p0 / U * U;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int q = k * kThreads + tid, v = q % VPB;
        if (!value) {
          *reinterpret_cast<uint4*>(s_run + q / VPB * RUN + v * X) = u[k];
        } else {
          uint2* to = reinterpret_cast<uint2*>(reinterpret_cast<char*>(s_run + q / VPB * RUN) +
                                               v * 16 + v / 16 * 8);
          to[0] = make_uint2(u[k].x, u[k].y);
          to[1] = make_uint2(u[k].z, u[k].w);
        }
      }
      for (int i = tid; i < kTok; i += kThreads) {
        const int off = i % BS, c = c0 + i / BS;
        if (c > c_last) break;
        const int at = s_list[c];
        const uint2 col = s_col[at];
        if ((col.x >> off) & 1u) {
          const bool there = s_from[at] >= 0;
          s_src[(int)col.y + __builtin_popcount(col.x & ((1u << off) - 1u)) - aligned] =
              there ? (uint32_t)(i / BS * RUN + (value ? off : off * X)) * EB : kNone;
          if (!there) s_absent[flip] = 1;
        }
        if (c == c_last && off == 0) s_p1 = (int)col.y + __builtin_popcount(col.x);
      }
      lds_group_barrier();  // the batch is read and lies in LDS
      const int p1 = s_p1;
      const bool all_there = s_absent[flip] == 0;
      load_data(u, c0 + 2 * kCols);
      if (tid == 0) s_absent[flip ^ 1] = 0;
      const int b0 = p0 / BS, nb = p1 > p0 ? (p1 - 1) / BS - b0 + 1 : 0;
      if (!value) {
        for (int q = tid; q < nb * VPB; q += kThreads) {
          const int i = uniform(q / VPB), v = q % VPB, p = (b0 + i) * BS + v % BS;
          const int64_t to = uniform64(places[b0 + i - to0]);
          if (to < 0 || p < p0 || p >= p1) continue;
          const uint32_t src = s_src[p - aligned];
          if (src == kNone) continue;
          *(reinterpret_cast<uint4*>(cache + to) + v) = *reinterpret_cast<const uint4*>(
              reinterpret_cast<const char*>(s_run) + src + v / BS * (BS * 16));
        }
      } else {
        constexpr int SEG = BS / U, UPB = DG * SEG;  // units of a row and of a block
        for (int q = tid; q < nb * UPB; q += kThreads) {
          const int i = uniform(q / UPB), v = q % UPB, row = v / SEG;
          const int p = (b0 + i) * BS + v % SEG * U;
          const int64_t at = uniform64(places[b0 + i - to0]);
          if (at < 0 || p + U <= p0 || p >= p1) continue;
          E* to = cache + at + v * U;
          const char* from = reinterpret_cast<const char*>(s_run + row_at(row));
          const uint32_t* src = s_src + (p - aligned);
          if (p >= p0 && p + U <= p1 && all_there) {
            union {
              uint4 v4;
              uint2 v2;
              E e[X];
            } out;
#pragma unroll
            for (int e = 0; e < U; ++e) out.e[e] = *reinterpret_cast<const E*>(from + src[e]);
            if constexpr (U == X) *reinterpret_cast<uint4*>(to) = out.v4;
            else *reinterpret_cast<uint2*>(to) = out.v2;
          } else {
            for (int e = 0; e < U; ++e)
              if (p + e >= p0 && p + e < p1 && src[e] != kNone)
                to[e] = *reinterpret_cast<const E*>(from + src[e]);
          }
        }
      }
      p0 = p1;
      flip ^= 1;
      lds_group_barrier();  // (LDS is read)
    };
    uint4 even[NV], odd[NV];
    load_data(even, 0);
    load_data(odd, kCols);
    for (int c0 = 0; c0 < listed; c0 += 2 * kCols) {
      batch(even, c0);
      if (c0 + kCols < listed) batch(odd, c0 + kCols);
    }
  }
}

template <typename E, int BS, int DG, int kThreads, int NV>
hipError_t move_launch(const EvictArgs& a, const CacheGeom& g, hipStream_t stream) {
  const int64_t grid = (int64_t)a.num_seqs * g.num_kv_heads * 2 * (g.head_dim / DG);
  hipLaunchKernelGGL((evict_move_kernel<E, BS, DG, kThreads, NV>), dim3((uint32_t)grid),
                     dim3(kThreads), 0, stream, a, g.num_kv_heads, g.head_dim, g.num_blocks,
                     g.block_stride, g.head_stride);
  return hipGetLastError();
}

template <typename E, int BS>
hipError_t move_bs(const EvictArgs& a, const CacheGeom& g, hipStream_t stream) {
  constexpr int kThin = 16 / (int)sizeof(E) > 8 ? 16 : 8;
  // groups of 32 dims unless they leave compute units idle: one sequence of 8192
  // tokens cut to 4096 takes 18 us in groups of 8 (256 workgroups), 64 sequences
  // of 600 to 4096 cut to 1024 take 197 us in groups of 32, 214 in groups of 8
  const int64_t wide = (int64_t)a.num_seqs * g.num_kv_heads * 2 * (g.head_dim / 32);
  return wide >= 1024 ? move_launch<E, BS, 32, 512, 4>(a, g, stream)
                      : move_launch<E, BS, kThin, 512, 4>(a, g, stream);
}

template <typename E>
hipError_t move_typed(const EvictArgs& a, const CacheGeom& g, hipStream_t stream) {
  switch (g.block_size) {
    case 8: return move_bs<E, 8>(a, g, stream);
    case 16: return move_bs<E, 16>(a, g, stream);
    case 32: return move_bs<E, 32>(a, g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

size_t evict_workspace_bytes(int32_t num_seqs, int32_t num_kv_heads, int32_t max_ctx,
                             int32_t block_size) {
  const size_t pairs = (size_t)num_seqs * num_kv_heads;
  return pairs * ((max_ctx + block_size - 1) / block_size) * sizeof(uint2) +
         pairs * sizeof(uint32_t);
}

hipError_t launch_evict(int cache_dtype, const EvictArgs& args, void* workspace,
                        const CacheGeom& g, hipStream_t stream) {
  EvictArgs a = args;
  const int64_t pairs = (int64_t)a.num_seqs * g.num_kv_heads;
  a.max_columns = (a.max_ctx + g.block_size - 1) / g.block_size;
  a.columns = static_cast<uint2*>(workspace);
  a.first_column = reinterpret_cast<uint32_t*>(a.columns + pairs * a.max_columns);
  const int bs_log2 = __builtin_ctz((unsigned)g.block_size);
  // 16 scores per thread in registers
  if (a.max_ctx <= 256 * kItems)
    hipLaunchKernelGGL(evict_select_kernel<256>, dim3((uint32_t)pairs), dim3(256), 0, stream, a,
                       g.num_kv_heads, bs_log2);
  else
    hipLaunchKernelGGL(evict_select_kernel<1024>, dim3((uint32_t)pairs), dim3(1024), 0, stream, a,
                       g.num_kv_heads, bs_log2);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // no sequence is cut; of contexts without tokens there is no workspace either
  if (a.max_ctx <= a.budget) return e;
  if (cache_dtype == VPA_DTYPE_F32) return move_typed<uint32_t>(a, g, stream);
  if (cache_dtype == VPA_DTYPE_FP8_E4M3) return move_typed<uint8_t>(a, g, stream);
  return move_typed<uint16_t>(a, g, stream);
}

}  // namespace vpa
