// Verification of drafted tokens against the target's logits, from given
// random numbers, for gfx950.
//
// Sequence b drafted x_0 .. x_{n-1}; row i of its target logits is the
// model's answer after x_{i-1} (row n: after the last draft). With
// p_i = softmax(target_i / T) and q_i = softmax(draft_i / T) (a drafter without
// logits: q_i is 1 at x_i), draft i is accepted while
//   accept_u[i] * q_i(x_i) < p_i(x_i),
// and the first one that is not is replaced by a token of max(p_i - q_i, 0),
// scaled to sum 1; if all are accepted, one more token of p_n follows. So every
// emitted token is distributed as the target's own. A token is drawn as the
// first v with cumsum(r)[v] > sample_u * sum(r). T <= 0: a draft is accepted if it
// is the row's first maximum, and the first maximum replaces it.
// This is the sampling counterpart of the greedy next token (token_kernels.hip)
// and takes n = 0 as plain sampling. NaN logits and -inf have probability 0.
//
// The answers are whole numbers next to a border of a sum over the vocabulary: in f32
// the cumulative sum is off by 2^-24 of the total, more than many of its 150 000 steps,
// so weights and sums are f64 throughout, exponentials included (within 4e-14). The
// f64 instructions of the exponentials are most of the calls with draft logits: 17 of
// them, 93 cycles of a SIMD at the rates measured alone, per 64 logits, which is 52 of
// the 71 to 75 us that the 87.5 million of 64 sequences with four drafts take at 2.4 GHz
// (151 936 tokens, bf16; 175 MB, 27 us at the streaming rate); what the other 20 us are
// has not been taken apart. f32 first and f64 for the drawn row alone needs that row
// read once more by a launch of its own and took 148 us in all against 121 then.
//
// Launches, over segments of 4096 logits: stats (every row's segment maxima and sums,
// or first maxima: each logit is read once), rest (max(p - q, 0) needs both rows'
// totals first; only where drafts have logits), draw (the segment, then the place in
// it). Rest and draw merge the stats and test the drafts themselves (pick_row: cheaper
// than a launch between them). Measured: 64 sequences as above 73 + 24 + 11 us; one
// sequence of four drafts without logits 4.3 + 9.6; 128 of up to three, greedy (156
// MB), 20 + 4; one token of each of 64 sequences sampled 14 + 8. Rows that do not all
// begin at 16 bytes are read by element: 64 sequences of 151 935 tokens 173 + 34 + 12.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "verify_weight.h"
#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kThreads = 256;
constexpr int kSeg = 4096;  // logits of a segment: 16 per thread
constexpr int kPer = kSeg / kThreads;
constexpr int kMaxDrafts = kVerifyMaxDrafts;
constexpr int kMaxRows = 2 * kMaxDrafts + 1;
constexpr uint32_t kNone = 0xffffffffu;

struct Buffers {
  // [target rows then draft rows][segments]: maximum, and the sum of weights
  // against it (greedy: the first maximum's index, as bits)
  float* max;
  double* sum;
  double* rest;  // [num_seqs][segments] of max(p - q, 0)
  int32_t segs;
};

__device__ __forceinline__ float seq_temperature(const VerifyArgs& a, int b) {
  return a.temperature == nullptr ? 1.f : a.temperature[b];
}
__device__ __forceinline__ int seq_drafts(const VerifyArgs& a, int b) {
  return a.num_drafts == nullptr ? a.max_drafts
                                 : (int)min(a.num_drafts[b], (uint32_t)a.max_drafts);
}
template <typename T>
__device__ __forceinline__ const T* target_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.target) + b * a.target_seq_stride + i * a.target_row_stride;
}
template <typename T>
__device__ __forceinline__ const T* draft_row(const VerifyArgs& a, int b, int i) {
  return static_cast<const T*>(a.draft) + b * a.draft_seq_stride + i * a.draft_row_stride;
}

// One of N threads' logits of a segment, -inf past the row: vector q = t + N i of the
// segment, so element e of it is logit seg * 4096 + q * X + e.
template <typename T, int N>
__device__ __forceinline__ void load_segment(const T* row, int t, int seg, int vocab, bool vec_ok,
                                             float (&f)[kSeg / N]) {
  constexpr int X = pack_x<T>(), kPer = kSeg / N;
  uint4 u[kPer / X];
#pragma unroll
  for (int i = 0; i < kPer / X; ++i) {
    const int at = seg * kSeg + (t + N * i) * X;
    u[i] = make_uint4(0u, 0u, 0u, 0u);
    if (vec_ok && at + X <= vocab) u[i] = load_stream(reinterpret_cast<const uint4*>(row + at));
  }
#pragma unroll
  for (int i = 0; i < kPer / X; ++i) {
    const int at = seg * kSeg + (t + N * i) * X;
    if (vec_ok && at + X <= vocab) {
      const T* e = reinterpret_cast<const T*>(&u[i]);
#pragma unroll
      for (int k = 0; k < X; ++k) f[i * X + k] = load_as_f32(e + k);
    } else {
#pragma unroll
      for (int k = 0; k < X; ++k)
        f[i * X + k] = at + k < vocab ? load_as_f32(row + at + k) : -INFINITY;
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ int segment_index(int t, int seg, int k) {  // logit of f[k]
  constexpr int X = pack_x<T>();
  return seg * kSeg + (t + N * (k / X)) * X + k % X;
}

template <int kCtrl>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)(uint32_t)u, kCtrl, 0xf, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), kCtrl, 0xf, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Sum over each row of 16 lanes, in every lane of it.
__device__ __forceinline__ double row16_sum_f64(double v) {
  v += dpp_f64<kDppQuadXor1>(v);
  v += dpp_f64<kDppQuadXor2>(v);
  v += dpp_f64<kDppRowHalfMirror>(v);
  return v + dpp_f64<kDppRowMirror>(v);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v = row16_sum_f64(v);
  return (readlane_f64(v, 0) + readlane_f64(v, 16)) + (readlane_f64(v, 32) + readlane_f64(v, 48));
}
// Sum over the workgroup's first four waves, in every thread; s4 is free again
// after the next barrier.
__device__ __forceinline__ double group_sum_f64(double v, double* s4) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) s4[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s4[0] + s4[1]) + (s4[2] + s4[3]);
}

// (greater value, lower index) over the workgroup
struct Best {
  float v;
  uint32_t i;
};
__device__ __forceinline__ void take_best(Best& a, float v, uint32_t i) {
  if (v > a.v || (v == a.v && i < a.i)) a = {v, i};
}

// Statistics of each segment of each row, by kWaves waves: four where there are few
// segments; else one, whose reductions and addresses serve 64 logits of a thread
// instead of 16.
template <typename T, int kWaves>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a, Buffers w,
                                                                bool vec_ok) {
  constexpr int N = 64 * kWaves, kPer = kSeg / N;
  __shared__ float s_m[4];
  __shared__ uint32_t s_i[4];
  __shared__ double s_s[4];
  const int rows_t = a.num_seqs * (a.max_drafts + 1);
  const int rows = rows_t + (a.draft == nullptr ? 0 : a.num_seqs * a.max_drafts);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const uint32_t unit = kWaves == 4 ? blockIdx.x : blockIdx.x * 4 + (uint32_t)wave;
  const int r = (int)(unit / (uint32_t)w.segs);
  if (r >= rows) return;  // (whole units; of four waves, whole workgroups)
  const int seg = (int)(unit - (uint32_t)r * (uint32_t)w.segs);
  const int t = kWaves == 4 ? (int)threadIdx.x : lane;
  const bool is_target = r < rows_t;
  const int per = is_target ? a.max_drafts + 1 : a.max_drafts;
  const int rr = is_target ? r : r - rows_t;
  const int b = rr / per, i = rr - b * per;
  const float temp = seq_temperature(a, b);
  const bool greedy = !(temp > 0.f);
  if (i >= seq_drafts(a, b) + (is_target ? 1 : 0) || (greedy && !is_target)) return;
  float f[kPer];
  load_segment<T, N>(is_target ? target_row<T>(a, b, i) : draft_row<T>(a, b, i), t, seg, a.vocab,
                     vec_ok, f);
  const int64_t at = (int64_t)r * w.segs + seg;
  if (greedy) {
    Best best{-INFINITY, kNone};
#pragma unroll
    for (int k = 0; k < kPer; ++k)  // (indices ascend with k; a NaN is never greater)
      if (f[k] > best.v) best = {f[k], (uint32_t)segment_index<T, N>(t, seg, k)};
#pragma unroll
    for (int m = 1; m < 64; m <<= 1)
      take_best(best, __shfl_xor(best.v, m, 64), __shfl_xor(best.i, m, 64));
    if constexpr (kWaves == 4) {
      if (lane == 0) {
        s_m[wave] = best.v;
        s_i[wave] = best.i;
      }
      __syncthreads();
      if (threadIdx.x == 0)
        for (int v = 1; v < 4; ++v) take_best(best, s_m[v], s_i[v]);
    }
    if (t == 0) {
      w.max[at] = best.v;
      w.sum[at] = __builtin_bit_cast(double, (uint64_t)best.i);
    }
    return;
  }
  float mx = f[0];
#pragma unroll
  for (int k = 1; k < kPer; ++k) mx = fmaxf(mx, f[k]);  // (a NaN loses)
  mx = fmaxf(mx, -INFINITY);
  mx = wave_max_dpp(mx);
  if constexpr (kWaves == 4) {
    if (lane == 0) s_m[wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  }
  const Scale sc(mx, temp);
  double s0 = 0.0, s1 = 0.0;
  if (sc.odd) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) s0 += sc.weight(f[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; k += 2) {
      s0 += sc.plain(f[k]);
      s1 += sc.plain(f[k + 1]);
    }
  }
  double sum;
  if constexpr (kWaves == 4) sum = group_sum_f64(s0 + s1, s_s);
  else sum = wave_sum_f64(s0 + s1);
  if (t == 0) {
    w.max[at] = mx;
    w.sum[at] = sum;
  }
}

// What became of a sequence's drafts.
struct Pick {
  int took;          // accepted drafts, and the target row that is drawn from
  bool greedy;       // the last token is `best`, nothing is drawn
  bool rejected;     // the row's draft was: drawn from what is left of the row without it
  uint32_t drafted;  // that draft
  uint32_t best;
  float max_p, max_q;
  double sum_p, sum_q;  // totals of the row's weights, and of its draft row's
};
struct PickShared {
  float max[kMaxRows];
  double sum[kMaxRows];
  uint32_t best[kMaxDrafts + 1];
  uint64_t good;
};

// Merges the segments of the sequence's rows, LPR lanes (16 or 64) a row, and tests
// its drafts; called by the whole workgroup of kGroup threads, the result in
// every thread.
template <typename T, int kGroup, int LPR>
__device__ __forceinline__ Pick pick_row(const VerifyArgs& a, const Buffers& w, int b,
                                         PickShared& sh) {
  constexpr int kHeld = 64 / LPR;  // segments a lane holds: the first 64 are read once
  const int K = a.max_drafts, n = seq_drafts(a, b);
  const float temp = seq_temperature(a, b);
  const bool greedy = !(temp > 0.f);
  const bool have_q = !greedy && a.draft != nullptr;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the drafts' own logits, read ahead of the merge
  uint32_t x = kNone;
  float lx = -INFINITY, lq = -INFINITY, au = 0.f;
  if (wave == 0 && lane < n) {
    x = a.draft_ids[(int64_t)b * K + lane];
    if (!greedy && x < (uint32_t)a.vocab) {
      lx = load_as_f32(target_row<T>(a, b, lane) + x);
      if (have_q) lq = load_as_f32(draft_row<T>(a, b, lane) + x);
      au = a.accept_u[(int64_t)b * K + lane];
    }
  }
  const int rows = n + 1 + (have_q ? n : 0);
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += kGroup / LPR) {
    const int q = r0 + (int)threadIdx.x / LPR, part = (int)threadIdx.x % LPR;
    const bool is_target = q <= n;
    const int64_t at = ((is_target ? (int64_t)b * (K + 1) + q
                                   : (int64_t)a.num_seqs * (K + 1) + (int64_t)b * K + (q - n - 1))) *
                       w.segs;
    const int segs = q < rows ? w.segs : 0;
    float v[kHeld], mx = -INFINITY;
    double held[kHeld], sum = 0.0;
    uint32_t best = kNone;
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int g = part + LPR * u;
      v[u] = -INFINITY;
      held[u] = 0.0;
      if (g < segs) {
        v[u] = w.max[at + g];
        held[u] = w.sum[at + g];
      }
    }
    auto take = [&](float value, double stat) {
      if (greedy) {
        const uint32_t i = (uint32_t)__builtin_bit_cast(uint64_t, stat);
        if (value > mx || (value == mx && i < best)) {
          mx = value;
          best = i;
        }
      } else {
        mx = fmaxf(mx, value);
      }
    };
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (part + LPR * u < segs) take(v[u], held[u]);
    for (int g = part + 64; g < segs; g += LPR) take(w.max[at + g], greedy ? w.sum[at + g] : 0.0);
    if (greedy) {
#pragma unroll
      for (int m = 1; m < LPR; m <<= 1) {
        const float om = __shfl_xor(mx, m, 64);
        const uint32_t oi = __shfl_xor(best, m, 64);
        if (om > mx || (om == mx && oi < best)) {
          mx = om;
          best = oi;
        }
      }
    } else {
      mx = fmaxf(mx, dpp<kDppQuadXor1>(mx));
      mx = fmaxf(mx, dpp<kDppQuadXor2>(mx));
      mx = fmaxf(mx, dpp<kDppRowHalfMirror>(mx));
      mx = fmaxf(mx, dpp<kDppRowMirror>(mx));
      if constexpr (LPR == 64)
        mx = fmaxf(fmaxf(readlane_f(mx, 0), readlane_f(mx, 16)),
                   fmaxf(readlane_f(mx, 32), readlane_f(mx, 48)));
      const Scale sc(mx, temp);
#pragma unroll
      for (int u = 0; u < kHeld; ++u)
        if (v[u] != -INFINITY) sum += held[u] * sc.weight(v[u]);
      for (int g = part + 64; g < segs; g += LPR) {
        const float value = w.max[at + g];
        if (value != -INFINITY) sum += w.sum[at + g] * sc.weight(value);
      }
      sum = row16_sum_f64(sum);
      if constexpr (LPR == 64)
        sum = (readlane_f64(sum, 0) + readlane_f64(sum, 16)) +
              (readlane_f64(sum, 32) + readlane_f64(sum, 48));
    }
    if (q < rows && part == 0) {
      sh.max[q] = mx;
      sh.sum[q] = sum;
      // (a greedy row without a number: 0, as the argmax gives)
      if (is_target) sh.best[q] = best == kNone ? 0u : best;
    }
  }
  __syncthreads();
  if (wave == 0) {  // lane i tests draft i
    bool good = false;
    if (lane < n && x < (uint32_t)a.vocab) {
      if (greedy) {
        good = sh.best[lane] == x;
      } else {
        const double px = Scale(sh.max[lane], temp).weight(lx) / sh.sum[lane];
        double qx = 1.0;
        if (have_q) {
          const double sum = sh.sum[n + 1 + lane];  // 0: no logit with any weight
          qx = sum > 0.0 ? Scale(sh.max[n + 1 + lane], temp).weight(lq) / sum : 0.0;
        }
        good = (double)au * qx < px;
      }
    }
    const uint64_t mask = __ballot(good);
    if (lane == 0) sh.good = mask;
  }
  __syncthreads();
  Pick p;
  p.took = ~sh.good == 0 ? 64 : __builtin_ctzll(~sh.good);  // at most n
  p.greedy = greedy;
  p.rejected = p.took < n;
  p.drafted = p.rejected ? a.draft_ids[(int64_t)b * K + p.took] : kNone;
  p.best = sh.best[p.took];
  p.max_p = sh.max[p.took];
  p.sum_p = sh.sum[p.took];
  const int q = p.rejected && have_q ? n + 1 + p.took : p.took;
  p.max_q = sh.max[q];
  p.sum_q = sh.sum[q];
  return p;
}

// What a logit (l of the target, d of the draft) weighs in max(p - q, 0). Both
// products are rounded (not fused into the difference), so that equal
// probabilities leave exactly 0.
__device__ __forceinline__ double residual(double wp, double wq, double inv_p, double inv_q) {
#pragma clang fp contract(off)
  const double r = wp * inv_p - wq * inv_q;
  return r > 0.0 ? r : 0.0;
}
__device__ __forceinline__ double inverse(double sum) { return sum > 0.0 ? 1.0 / sum : 0.0; }

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a, Buffers w,
                                                               bool vec_ok) {
  __shared__ PickShared sh;
  __shared__ double s4[4];
  const int b = blockIdx.y;
  const Pick p = pick_row<T, kThreads, 16>(a, w, b, sh);
  if (p.greedy || !p.rejected) return;
  const float temp = seq_temperature(a, b);
  const Scale sp(p.max_p, temp), sq(p.max_q, temp);
  const double inv_p = inverse(p.sum_p), inv_q = inverse(p.sum_q);
  const T* rt = target_row<T>(a, b, p.took);
  const T* rd = draft_row<T>(a, b, p.took);
#pragma unroll 1
  for (int seg = blockIdx.x; seg < w.segs; seg += gridDim.x) {
    float f[kPer], d[kPer];
    load_segment<T, kThreads>(rt, threadIdx.x, seg, a.vocab, vec_ok, f);
    load_segment<T, kThreads>(rd, threadIdx.x, seg, a.vocab, vec_ok, d);
    double r = 0.0;
    if (sp.odd || sq.odd) {
#pragma unroll 1
      for (int k = 0; k < kPer; ++k)
        r += residual(sp.weight(f[k]), sq.weight(d[k]), inv_p, inv_q);
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        r += residual(sp.plain(f[k]), sq.plain(d[k]), inv_p, inv_q);
    }
    r = group_sum_f64(r, s4);
    if (threadIdx.x == 0) w.rest[(int64_t)b * w.segs + seg] = r;
    __syncthreads();  // (s4 is read)
  }
}

constexpr int kDrawThreads = 1024;
constexpr int kDrawWaves = kDrawThreads / 64;

template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp_add_f64(double v) {  // 0 from lanes that are not there
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, kRows, 0xf, kRows == 0xf);
  const uint32_t hi =
      __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, kRows, 0xf, kRows == 0xf);
  return v + __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// Inclusive prefix sum over the workgroup's threads in their order.
__device__ __forceinline__ double group_scan_f64(double v, double* s_w, double& total) {
  const int wave = threadIdx.x >> 6;
  v = dpp_add_f64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
  v = dpp_add_f64<0x112, 0xf>(v);
  v = dpp_add_f64<0x114, 0xf>(v);
  v = dpp_add_f64<0x118, 0xf>(v);
  v = dpp_add_f64<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3, :31 into 2 and 3
  v = dpp_add_f64<0x143, 0xc>(v);
  if ((threadIdx.x & 63) == 63) s_w[wave] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int i = 0; i < kDrawWaves; ++i) {
    before += i < wave ? s_w[i] : 0.0;
    total += s_w[i];
  }
  return before + v;
}
// The lowest `first` and the highest `last` (kNone: none; last counted from 1) of
// the workgroup.
__device__ __forceinline__ void group_first_last(uint32_t& first, uint32_t& last, uint2* s_w) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    first = min(first, (uint32_t)__shfl_xor(first, m, 64));
    last = max(last, (uint32_t)__shfl_xor(last, m, 64));
  }
  if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = make_uint2(first, last);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kDrawWaves; ++i) {
    first = min(first, s_w[i].x);
    last = max(last, s_w[i].y);
  }
}

// Four logits from `at` on, -inf past the row.
template <typename T>
__device__ __forceinline__ void load4(const T* row, int at, int vocab, bool vec_ok, float (&f)[4]) {
  if (vec_ok && at + 4 <= vocab) {
    uint32_t u[4];
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(row + at);
    else *reinterpret_cast<uint2*>(u) = *reinterpret_cast<const uint2*>(row + at);
    const T* e = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = load_as_f32(e + k);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = at + k < vocab ? load_as_f32(row + at + k) : -INFINITY;
  }
}

template <typename T>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyArgs a, Buffers w,
                                                                   bool vec_ok) {
  static_assert(kSeg == 4 * kDrawThreads, "four logits a thread");
  __shared__ PickShared sh;
  __shared__ double s_w[4][kDrawWaves];
  __shared__ uint2 s_u[2][kDrawWaves];
  __shared__ double s_before;
  __shared__ int s_seg;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int K = a.max_drafts;
  const Pick p = pick_row<T, kDrawThreads, 64>(a, w, b, sh);
  uint32_t* out = a.out_ids + (int64_t)b * (K + 1);
  for (int i = tid; i <= K; i += kDrawThreads)
    if (i != p.took) out[i] = i < p.took ? a.draft_ids[(int64_t)b * K + i] : kNone;
  if (tid == 0) a.out_count[b] = (uint32_t)p.took + 1u;
  out += p.took;
  if (p.greedy) {
    if (tid == 0) *out = p.best;
    return;
  }
  const float temp = seq_temperature(a, b);
  const Scale sp(p.max_p, temp), sq(p.max_q, temp);
  const double inv_p = inverse(p.sum_p), inv_q = inverse(p.sum_q);
  const T* rt = target_row<T>(a, b, p.took);
  // drawn from the residual; or, of a drafter without logits, from the row without
  // the draft; or from the whole row
  bool residuals = p.rejected && a.draft != nullptr;
  const int without = p.rejected && a.draft == nullptr && p.drafted < (uint32_t)a.vocab
                          ? (int)p.drafted
                          : -1;
  const T* rd = residuals ? draft_row<T>(a, b, p.took) : rt;
  float f[4], d[4] = {};
  double r[4];
  // the weights drawn from of the thread's four logits of segment seg, their sum
  auto weigh = [&](int seg) {
    const int at = seg * kSeg + tid * 4;
    load4<T>(rt, at, a.vocab, vec_ok, f);
    if (residuals) load4<T>(rd, at, a.vocab, vec_ok, d);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      r[k] = at + k == without ? 0.0 : sp.weight(f[k]);
      if (residuals) r[k] = residual(r[k], sq.weight(d[k]), inv_p, inv_q);
      sum += r[k];
    }
    return sum;
  };
  // the drafted token's segment without it (summed again: a difference would keep
  // the rounding of its sum)
  double rest_of_draft = 0.0;
  if (without >= 0) {
    double all;
    group_scan_f64(weigh(without / kSeg), s_w[0], all);
    rest_of_draft = all;
  }
  const int per = (w.segs + kDrawThreads - 1) / kDrawThreads;
  const int g0 = min(tid * per, w.segs), g1 = min(g0 + per, w.segs);
  const int64_t row_at = ((int64_t)b * (K + 1) + p.took) * w.segs;
  auto segment_sum = [&](int g) {
    if (residuals) return w.rest[(int64_t)b * w.segs + g];
    if (without >= 0 && g == without / kSeg) return rest_of_draft;
    const float m = w.max[row_at + g];
    return m == -INFINITY ? 0.0 : w.sum[row_at + g] * sp.weight(m);
  };
  double mine, upto, total;
#pragma unroll 1
  for (int round = 1;; ++round) {
    mine = 0.0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) mine += segment_sum(g);
    upto = group_scan_f64(mine, s_w[round], total);
    if (!residuals || total > 0.0) break;
    residuals = false;  // p equals q: drawn from p
  }
  if (!(total > 0.0)) {  // no logit with any weight, or only the drafted one
    if (tid == 0)
      *out = without >= 0 && sp.weight(load_as_f32(rt + without)) > 0.0 ? (uint32_t)without : 0u;
    return;
  }
  // the segment: the first whose running sum passes the target
  const double target = (double)a.sample_u[b] * total;
  uint32_t first = mine > 0.0 && upto > target ? (uint32_t)tid : kNone;
  uint32_t last = mine > 0.0 ? (uint32_t)tid + 1u : 0u;
  group_first_last(first, last, s_u[0]);
  if ((uint32_t)tid == (first != kNone ? first : last - 1u)) {  // (rounding: the last with any weight)
    double run = upto - mine, start = run;
    int found = g0;
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      const double v = per == 1 ? mine : segment_sum(g);
      if (v > 0.0) {
        found = g;
        start = run;
      }
      run += v;
      if (run > target) break;
    }
    s_seg = found;
    s_before = start;
  }
  __syncthreads();
  // the place in it
  const int at = s_seg * kSeg + tid * 4;
  const double sum = weigh(s_seg);
  upto = group_scan_f64(sum, s_w[3], total) - sum + s_before;
  first = kNone;
  last = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    upto += r[k];
    if (first == kNone && r[k] > 0.0 && upto > target) first = (uint32_t)(at + k);
    if (r[k] > 0.0) last = (uint32_t)(at + k) + 1u;  // 0: none
  }
  group_first_last(first, last, s_u[1]);
  if (tid == 0) *out = first != kNone ? first : last - 1u;
}

struct Sizes {
  int32_t segs;
  size_t max_at, rest_at, bytes;
};
Sizes sizes(int32_t num_seqs, int32_t max_drafts, int32_t vocab) {
  Sizes z;
  z.segs = (vocab + kSeg - 1) / kSeg;
  const size_t rows = (size_t)num_seqs * (2 * max_drafts + 1);
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  z.rest_at = up(rows * z.segs * sizeof(double));
  z.max_at = z.rest_at + up((size_t)num_seqs * z.segs * sizeof(double));
  z.bytes = z.max_at + up(rows * z.segs * sizeof(float));
  return z;
}

template <typename T>
hipError_t verify_typed(const VerifyArgs& a, hipStream_t stream) {
  const Sizes z = sizes(a.num_seqs, a.max_drafts, a.vocab);
  char* base = static_cast<char*>(a.workspace);
  Buffers w;
  w.sum = reinterpret_cast<double*>(base);
  w.rest = reinterpret_cast<double*>(base + z.rest_at);
  w.max = reinterpret_cast<float*>(base + z.max_at);
  w.segs = z.segs;
  auto whole = [](const void* p, int64_t s, int64_t r) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 &&
                            (s * (int64_t)sizeof(T)) % 16 == 0 && (r * (int64_t)sizeof(T)) % 16 == 0);
  };
  const bool vec_ok = whole(a.target, a.target_seq_stride, a.target_row_stride) &&
                      whole(a.draft, a.draft_seq_stride, a.draft_row_stride);
  const int rows = a.num_seqs * (a.max_drafts + 1) + (a.draft == nullptr ? 0 : a.num_seqs * a.max_drafts);
  const uint32_t units = (uint32_t)z.segs * (uint32_t)rows;
  // (9728 segments of one sequence's row each take 43 us in all, 45 by four waves; 190
  // take 16, 13 by four)
  if (units >= 4096)
    hipLaunchKernelGGL((verify_stats_kernel<T, 1>), dim3((units + 3) / 4), dim3(kThreads), 0, stream,
                       a, w, vec_ok);
  else
    hipLaunchKernelGGL((verify_stats_kernel<T, 4>), dim3(units), dim3(kThreads), 0, stream, a, w,
                       vec_ok);
  // (two segments to a workgroup share its merge of the stats where every compute unit
  // has eight: 24 us for 64 sequences of 151 936 tokens, 27 one by one, 27 by three)
  const int per_group = z.segs * a.num_seqs >= 2048 ? 2 : 1;
  if (a.draft != nullptr)
    hipLaunchKernelGGL(verify_rest_kernel<T>,
                       dim3((uint32_t)((z.segs + per_group - 1) / per_group), (uint32_t)a.num_seqs),
                       dim3(kThreads), 0, stream, a, w, vec_ok);
  hipLaunchKernelGGL(verify_draw_kernel<T>, dim3((uint32_t)a.num_seqs), dim3(kDrawThreads), 0,
                     stream, a, w, vec_ok);
  return hipGetLastError();
}

}  // namespace

size_t verify_workspace_bytes(int32_t num_seqs, int32_t max_drafts, int32_t vocab) {
  return sizes(num_seqs, max_drafts, vocab).bytes;
}

hipError_t launch_verify(int dtype, const VerifyArgs& a, hipStream_t stream) {
  switch (dtype) {
    case VPA_DTYPE_F32: return verify_typed<float>(a, stream);
    case VPA_DTYPE_F16: return verify_typed<f16_t>(a, stream);
    case VPA_DTYPE_BF16: return verify_typed<bf16_t>(a, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vpa
