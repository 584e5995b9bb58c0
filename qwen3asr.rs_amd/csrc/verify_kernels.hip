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
// The draw's answer is a whole number next to a border of a sum over the
// vocabulary: in f32 the cumulative sum is off by 2^-24 of the total, more than
// many of its 150 000 steps, so the one row that is drawn from is summed in f64
// (exponentials included); the acceptance tests, one comparison per draft, take
// f32 exponentials summed per segment and merged in f64.
//
// Launches, over segments of 4096 logits: stats (every row's segment maxima,
// sums and first maxima: each logit is read once, the bound of the whole), pick
// (one workgroup per sequence merges them and tests the drafts), sums (f64 sums
// of the drawn row's segments), rest (max(p - q, 0) needs both rows' totals
// first; only where drafts have logits), draw (the segment, then the place in
// it).

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kThreads = 256;
constexpr int kSeg = 4096;  // logits of a segment: 16 per thread
constexpr int kPer = kSeg / kThreads;
constexpr int kMaxDrafts = kVerifyMaxDrafts;

enum Mode : int32_t {
  kDone = 0,      // the last token is known (greedy)
  kPlain = 1,     // drawn from the target row
  kResidual = 2,  // from max(p - q, 0)
  kExcluded = 3,  // from the target row without the drafted token
};
struct Pick {
  int32_t row;   // accepted drafts, and the target row that is drawn from
  int32_t mode;
  float max_p, max_q;
  uint32_t drafted;  // the rejected draft
};

struct Buffers {
  float2* stats;     // [target rows then draft rows][segments] {max, sum}
  uint32_t* best;    // [target rows][segments] first maximum
  Pick* picks;       // [num_seqs]
  double2* sums;     // [num_seqs][segments] of the target row and the draft row
  double* rest;      // [num_seqs][segments] of what is drawn from
  int32_t segs;
};

// e^x for x <= 0 in f64 (0 below -708 and for NaN): x = n ln 2 + r, Taylor sum
// of e^r to r^13 (|r| <= 0.35: 0.35^14 / 14! < 2^-57).
__device__ __forceinline__ double exp_nonpos(double x) {
  if (!(x > -708.0)) return 0.0;
  const double n = __builtin_rint(x * 1.44269504088896340736);
  double r = __builtin_fma(n, -0.69314718055994530942, x);
  r = __builtin_fma(n, -2.3190468138462995584e-17, r);
  double p = 1.0 / 6227020800.0;
  p = __builtin_fma(p, r, 1.0 / 479001600.0);
  p = __builtin_fma(p, r, 1.0 / 39916800.0);
  p = __builtin_fma(p, r, 1.0 / 3628800.0);
  p = __builtin_fma(p, r, 1.0 / 362880.0);
  p = __builtin_fma(p, r, 1.0 / 40320.0);
  p = __builtin_fma(p, r, 1.0 / 5040.0);
  p = __builtin_fma(p, r, 1.0 / 720.0);
  p = __builtin_fma(p, r, 1.0 / 120.0);
  p = __builtin_fma(p, r, 1.0 / 24.0);
  p = __builtin_fma(p, r, 1.0 / 6.0);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  return __builtin_bit_cast(double, __builtin_bit_cast(int64_t, p) + ((int64_t)n << 52));
}
// Weight of a logit l against the maximum m: e^((l - m) / T), 1 at the maximum
// (also an infinite one), 0 for -inf and NaN.
__device__ __forceinline__ double weight64(float l, float m, double inv_t) {
  if (l == m) return l == -INFINITY ? 0.0 : 1.0;
  return exp_nonpos(((double)l - (double)m) * inv_t);
}

__device__ __forceinline__ float seq_temperature(const VerifyArgs& a, int b) {
  return a.temperature == nullptr ? 1.f : a.temperature[b];
}
__device__ __forceinline__ int seq_drafts(const VerifyArgs& a, int b) {
  return a.num_drafts == nullptr ? a.max_drafts
                                 : (int)min(a.num_drafts[b], (uint32_t)a.max_drafts);
}

// The thread's 16 logits of a segment, -inf past the row: vector q = tid + 256 i
// of the segment, so element e of it is logit seg * 4096 + q * X + e.
template <typename T>
__device__ __forceinline__ void load_segment(const T* row, int seg, int vocab, bool vec_ok,
                                             float (&f)[kPer]) {
  constexpr int X = pack_x<T>();
#pragma unroll
  for (int i = 0; i < kPer / X; ++i) {
    const int at = seg * kSeg + ((int)threadIdx.x + kThreads * i) * X;
    if (vec_ok && at + X <= vocab) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + at);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int k = 0; k < X; ++k) f[i * X + k] = load_as_f32(e + k);
    } else {
#pragma unroll
      for (int k = 0; k < X; ++k)
        f[i * X + k] = at + k < vocab ? load_as_f32(row + at + k) : -INFINITY;
    }
  }
}
template <typename T>
__device__ __forceinline__ int segment_index(int seg, int k) {  // logit of f[k]
  constexpr int X = pack_x<T>();
  return seg * kSeg + ((int)threadIdx.x + kThreads * (k / X)) * X + k % X;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
// Sum over the workgroup, in every thread; s4 is free again after the next
// barrier.
__device__ __forceinline__ double group_sum_f64(double v, double* s4) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) s4[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s4[0] + s4[1]) + (s4[2] + s4[3]);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a, Buffers w,
                                                                bool vec_ok) {
  __shared__ float s_m[4];
  __shared__ uint32_t s_i[4];
  __shared__ float s_s[4];
  const int rows_t = a.num_seqs * (a.max_drafts + 1);
  const int r = (int)(blockIdx.x / (uint32_t)w.segs);
  const int seg = (int)(blockIdx.x - (uint32_t)r * (uint32_t)w.segs);
  const bool is_target = r < rows_t;
  const int per = is_target ? a.max_drafts + 1 : a.max_drafts;
  const int rr = is_target ? r : r - rows_t;
  const int b = rr / per, i = rr - b * per;
  if (i >= seq_drafts(a, b) + (is_target ? 1 : 0)) return;
  const float temp = seq_temperature(a, b);
  const bool greedy = !(temp > 0.f);
  if (greedy && !is_target) return;
  const T* row = is_target ? static_cast<const T*>(a.target) + b * a.target_seq_stride +
                                 i * a.target_row_stride
                           : static_cast<const T*>(a.draft) + b * a.draft_seq_stride +
                                 i * a.draft_row_stride;
  float f[kPer];
  load_segment<T>(row, seg, a.vocab, vec_ok, f);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float mx = -INFINITY;
  uint32_t at = 0xffffffffu;
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (f[k] > mx) {  // (indices ascend with k; a NaN is never greater)
      mx = f[k];
      at = (uint32_t)segment_index<T>(seg, k);
    }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const float om = __shfl_xor(mx, m, 64);
    const uint32_t oi = __shfl_xor(at, m, 64);
    if (om > mx || (om == mx && oi < at)) {
      mx = om;
      at = oi;
    }
  }
  if (lane == 0) {
    s_m[wave] = mx;
    s_i[wave] = at;
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < 4; ++v)
    if (s_m[v] > mx || (s_m[v] == mx && s_i[v] < at)) {
      mx = s_m[v];
      at = s_i[v];
    }
  float sum = 0.f;
  if (!greedy) {
    const float c = fminf(1.44269504f / temp, 3.0e38f);  // (finite: 0 * c is 0 at the maximum)
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const float x = (f[k] - mx) * c;
      const float e = mx == INFINITY ? (f[k] == mx ? 1.f : 0.f) : __builtin_amdgcn_exp2f(x);
      sum += x == x || mx == INFINITY ? e : 0.f;
    }
    sum = wave_sum_dpp(sum);
    if (lane == 0) s_s[wave] = sum;
    __syncthreads();
    sum = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
  }
  if (threadIdx.x == 0) {
    w.stats[(int64_t)r * w.segs + seg] = make_float2(mx, sum);
    if (is_target) w.best[(int64_t)r * w.segs + seg] = at;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_pick_kernel(VerifyArgs a, Buffers w) {
  __shared__ float s_max[2 * kMaxDrafts + 1];
  __shared__ double s_sum[2 * kMaxDrafts + 1];
  __shared__ uint32_t s_best[kMaxDrafts + 1];
  const int b = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int K = a.max_drafts, n = seq_drafts(a, b);
  const float temp = seq_temperature(a, b);
  const bool greedy = !(temp > 0.f);
  const double inv_t = 1.0 / (double)temp;
  const int rows = n + 1 + (greedy || a.draft == nullptr ? 0 : n);
  for (int q = wave; q < rows; q += 4) {  // a wave merges a row's segments
    const bool is_target = q <= n;
    const int64_t r = is_target ? (int64_t)b * (K + 1) + q
                                : (int64_t)a.num_seqs * (K + 1) + (int64_t)b * K + (q - n - 1);
    const float2* st = w.stats + r * w.segs;
    float mx = -INFINITY;
    uint32_t at = 0xffffffffu;
    for (int g = lane; g < w.segs; g += 64) {
      const float v = st[g].x;
      const uint32_t i = is_target ? w.best[r * w.segs + g] : 0u;
      if (v > mx || (v == mx && i < at)) {
        mx = v;
        at = i;
      }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const float om = __shfl_xor(mx, m, 64);
      const uint32_t oi = __shfl_xor(at, m, 64);
      if (om > mx || (om == mx && oi < at)) {
        mx = om;
        at = oi;
      }
    }
    double sum = 0.0;
    if (!greedy)
      for (int g = lane; g < w.segs; g += 64) sum += (double)st[g].y * weight64(st[g].x, mx, inv_t);
    sum = wave_sum_f64(sum);
    if (lane == 0) {
      s_max[is_target ? q : K + q - n] = mx;
      s_sum[is_target ? q : K + q - n] = sum;
      if (is_target) s_best[q] = at;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // lane i tests draft i
  bool good = false;
  uint32_t x = 0xffffffffu;
  if (lane < n) {
    x = a.draft_ids[(int64_t)b * K + lane];
    if (greedy) {
      good = s_best[lane] == x;
    } else if (x < (uint32_t)a.vocab) {
      const T* tr = static_cast<const T*>(a.target) + b * a.target_seq_stride +
                    lane * a.target_row_stride;
      const double px = weight64(load_as_f32(tr + x), s_max[lane], inv_t) / s_sum[lane];
      double qx = 1.0;
      if (a.draft != nullptr) {
        const T* dr = static_cast<const T*>(a.draft) + b * a.draft_seq_stride +
                      lane * a.draft_row_stride;
        const double sum = s_sum[K + 1 + lane];  // 0: no logit with any weight
        qx = sum > 0.0 ? weight64(load_as_f32(dr + x), s_max[K + 1 + lane], inv_t) / sum : 0.0;
      }
      good = (double)a.accept_u[(int64_t)b * K + lane] * qx < px;
    }
  }
  const uint64_t mask = __ballot(good);
  const int took = ~mask == 0 ? 64 : __builtin_ctzll(~mask);  // at most n
  uint32_t* out = a.out_ids + (int64_t)b * (K + 1);
  for (int i = lane; i <= K; i += 64) {
    const uint32_t id = i < took ? a.draft_ids[(int64_t)b * K + i] : 0xffffffffu;
    if (i != took) out[i] = id;
  }
  if (lane != 0) return;
  a.out_count[b] = (uint32_t)took + 1u;
  Pick p;
  p.row = took;
  p.max_p = s_max[took];
  p.max_q = 0.f;
  p.drafted = 0xffffffffu;
  p.mode = kPlain;
  if (greedy) {
    p.mode = kDone;
    const uint32_t id = s_best[took];
    out[took] = id == 0xffffffffu ? 0u : id;  // a row with no number: 0, as the argmax gives
  } else if (took < n) {
    p.drafted = a.draft_ids[(int64_t)b * K + took];
    p.mode = a.draft == nullptr ? kExcluded : kResidual;
    if (a.draft != nullptr) p.max_q = s_max[K + 1 + took];
  }
  w.picks[b] = p;
}

// The row a sequence draws from, and its draft row.
template <typename T>
__device__ __forceinline__ const T* picked_target(const VerifyArgs& a, int b, const Pick& p) {
  return static_cast<const T*>(a.target) + b * a.target_seq_stride + p.row * a.target_row_stride;
}
template <typename T>
__device__ __forceinline__ const T* picked_draft(const VerifyArgs& a, int b, const Pick& p) {
  return static_cast<const T*>(a.draft) + b * a.draft_seq_stride + p.row * a.draft_row_stride;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(VerifyArgs a, Buffers w,
                                                               bool vec_ok) {
  __shared__ double s4[2][4];
  const int seg = blockIdx.x, b = blockIdx.y;
  const Pick p = w.picks[b];
  if (p.mode == kDone) return;
  const double inv_t = 1.0 / (double)seq_temperature(a, b);
  float f[kPer];
  load_segment<T>(picked_target<T>(a, b, p), seg, a.vocab, vec_ok, f);
  double sp = 0.0, sq = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (p.mode != kExcluded || (uint32_t)segment_index<T>(seg, k) != p.drafted)
      sp += weight64(f[k], p.max_p, inv_t);
  sp = group_sum_f64(sp, s4[0]);
  if (p.mode == kResidual) {
    load_segment<T>(picked_draft<T>(a, b, p), seg, a.vocab, vec_ok, f);
#pragma unroll
    for (int k = 0; k < kPer; ++k) sq += weight64(f[k], p.max_q, inv_t);
    sq = group_sum_f64(sq, s4[1]);
  }
  if (threadIdx.x == 0) {
    w.sums[(int64_t)b * w.segs + seg] = make_double2(sp, sq);
    w.rest[(int64_t)b * w.segs + seg] = sp;  // what is drawn from, but for kResidual
  }
}

// Totals over the segments of a sequence, in a fixed order, in every thread.
__device__ __forceinline__ double2 total_sums(const Buffers& w, int b, double (*s4)[4]) {
  double sp = 0.0, sq = 0.0;
  for (int g = threadIdx.x; g < w.segs; g += kThreads) {
    const double2 v = w.sums[(int64_t)b * w.segs + g];
    sp += v.x;
    sq += v.y;
  }
  const double tp = group_sum_f64(sp, s4[0]);
  return make_double2(tp, group_sum_f64(sq, s4[1]));
}

// What logit (l of the target, d of the draft) weighs in max(p - q, 0). Both
// products are rounded (not fused into the difference), so that equal
// probabilities leave exactly 0.
__device__ __forceinline__ double residual(float l, float d, const Pick& p, double inv_t,
                                           double inv_p, double inv_q) {
#pragma clang fp contract(off)
  const double r = weight64(l, p.max_p, inv_t) * inv_p - weight64(d, p.max_q, inv_t) * inv_q;
  return r > 0.0 ? r : 0.0;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a, Buffers w,
                                                               bool vec_ok) {
  __shared__ double s4[3][4];
  const int seg = blockIdx.x, b = blockIdx.y;
  const Pick p = w.picks[b];
  if (p.mode != kResidual) return;
  const double inv_t = 1.0 / (double)seq_temperature(a, b);
  float f[kPer], d[kPer];
  load_segment<T>(picked_target<T>(a, b, p), seg, a.vocab, vec_ok, f);
  load_segment<T>(picked_draft<T>(a, b, p), seg, a.vocab, vec_ok, d);
  const double2 t = total_sums(w, b, s4);
  const double inv_p = t.x > 0.0 ? 1.0 / t.x : 0.0, inv_q = t.y > 0.0 ? 1.0 / t.y : 0.0;
  double r = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) r += residual(f[k], d[k], p, inv_t, inv_p, inv_q);
  r = group_sum_f64(r, s4[2]);
  if (threadIdx.x == 0) w.rest[(int64_t)b * w.segs + seg] = r;
}

// Inclusive prefix sum over the workgroup's threads in their order.
__device__ __forceinline__ double group_scan_f64(double v, double* s4, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const double o = __shfl_up(v, m, 64);
    if (lane >= m) v += o;
  }
  if (lane == 63) s4[wave] = v;
  __syncthreads();
  double before = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) before += i < wave ? s4[i] : 0.0;
  total = ((s4[0] + s4[1]) + s4[2]) + s4[3];
  return before + v;
}

// First thread-ordered place of the workgroup where a value in `mine` is set
// (kNone where no thread has one): minimum over threads.
__device__ __forceinline__ uint32_t group_min(uint32_t v, uint32_t* s) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = min(v, (uint32_t)__shfl_xor(v, m, 64));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return min(min(s[0], s[1]), min(s[2], s[3]));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a, Buffers w) {
  __shared__ double s4[6][4];
  __shared__ uint32_t s_u[4][4];
  __shared__ double s_target, s_before;
  __shared__ int s_seg;
  constexpr uint32_t kNone = 0xffffffffu;
  const int b = blockIdx.x, tid = threadIdx.x;
  Pick p = w.picks[b];
  if (p.mode == kDone) return;
  uint32_t* out = a.out_ids + (int64_t)b * (a.max_drafts + 1) + p.row;
  const double inv_t = 1.0 / (double)seq_temperature(a, b);
  const double2 t = total_sums(w, b, s4);
  // the segments' sums, scanned in order by chunks of 256 of them
  double rest_total = 0.0;
  for (int g = tid; g < w.segs; g += kThreads) rest_total += w.rest[(int64_t)b * w.segs + g];
  rest_total = group_sum_f64(rest_total, s4[2]);
  const bool fall_back = p.mode == kResidual && !(rest_total > 0.0);
  // p equals q (every difference rounds to nothing): draw from p
  if (fall_back) p.mode = kPlain;
  const double total = fall_back ? t.x : rest_total;
  if (!(total > 0.0)) {  // no logit with any weight, or only the drafted one
    if (tid == 0)
      *out = p.mode == kExcluded && p.drafted < (uint32_t)a.vocab &&
                     weight64(load_as_f32(picked_target<T>(a, b, p) + p.drafted), p.max_p, inv_t) > 0.0
                 ? p.drafted
                 : 0u;
    return;
  }
  const double target = (double)a.sample_u[b] * total;
  // the segment: the first whose running sum passes the target; each thread
  // has a run of segments
  {
    const int per = (w.segs + kThreads - 1) / kThreads;
    const int g0 = min(tid * per, w.segs), g1 = min(g0 + per, w.segs);
    auto seg_sum = [&](int g) {
      const int64_t at = (int64_t)b * w.segs + g;
      return fall_back ? w.sums[at].x : w.rest[at];
    };
    double mine = 0.0;
    for (int g = g0; g < g1; ++g) mine += seg_sum(g);
    double all;
    const double upto = group_scan_f64(mine, s4[4], all);
    const uint32_t first = group_min(mine > 0.0 && upto > target ? (uint32_t)tid : kNone, s_u[2]);
    const uint32_t last = kNone - group_min(mine > 0.0 ? kNone - (uint32_t)tid : kNone, s_u[3]);
    if ((uint32_t)tid == (first != kNone ? first : last)) {  // (rounding: the last with any weight)
      double run = upto - mine, start = run;
      int found = g0;
      for (int g = g0; g < g1; ++g) {
        const double v = seg_sum(g);
        if (v > 0.0) {
          found = g;
          start = run;
        }
        run += v;
        if (run > target) break;
      }
      s_seg = found;
      s_before = start;
      s_target = target;
    }
  }
  __syncthreads();
  const int seg = s_seg;
  const double inv_p = t.x > 0.0 ? 1.0 / t.x : 0.0, inv_q = t.y > 0.0 ? 1.0 / t.y : 0.0;
  const T* rt = picked_target<T>(a, b, p);
  const T* rd = p.mode == kResidual ? picked_draft<T>(a, b, p) : nullptr;
  // 16 consecutive logits per thread
  const int at = seg * kSeg + tid * kPer;
  double r[kPer], sum = 0.0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    r[k] = 0.0;
    if (at + k < a.vocab) {
      const float l = load_as_f32(rt + at + k);
      if (p.mode == kResidual)
        r[k] = residual(l, load_as_f32(rd + at + k), p, inv_t, inv_p, inv_q);
      else if (p.mode == kPlain || (uint32_t)(at + k) != p.drafted)
        r[k] = weight64(l, p.max_p, inv_t);
    }
    sum += r[k];
  }
  double seg_total;
  double upto = group_scan_f64(sum, s4[3], seg_total) - sum + s_before;
  uint32_t first = kNone, last = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    upto += r[k];
    if (first == kNone && r[k] > 0.0 && upto > s_target) first = (uint32_t)(at + k);
    if (r[k] > 0.0) last = (uint32_t)(at + k) + 1u;  // 0: none
  }
  first = group_min(first, s_u[0]);
  last = kNone - group_min(kNone - last, s_u[1]);
  if (tid == 0) *out = first != kNone ? first : last - 1u;
}

struct Sizes {
  int32_t segs;
  size_t best_at, picks_at, sums_at, rest_at, bytes;
};
Sizes sizes(int32_t num_seqs, int32_t max_drafts, int32_t vocab) {
  Sizes z;
  z.segs = (vocab + kSeg - 1) / kSeg;
  const size_t t = (size_t)num_seqs * (max_drafts + 1), d = (size_t)num_seqs * max_drafts;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  size_t at = up((t + d) * z.segs * sizeof(float2));
  z.best_at = at;
  at += up(t * z.segs * sizeof(uint32_t));
  z.picks_at = at;
  at += up((size_t)num_seqs * sizeof(Pick));
  z.sums_at = at;
  at += up((size_t)num_seqs * z.segs * sizeof(double2));
  z.rest_at = at;
  at += up((size_t)num_seqs * z.segs * sizeof(double));
  z.bytes = at;
  return z;
}

template <typename T>
hipError_t verify_typed(const VerifyArgs& a, hipStream_t stream) {
  const Sizes z = sizes(a.num_seqs, a.max_drafts, a.vocab);
  char* base = static_cast<char*>(a.workspace);
  Buffers w;
  w.stats = reinterpret_cast<float2*>(base);
  w.best = reinterpret_cast<uint32_t*>(base + z.best_at);
  w.picks = reinterpret_cast<Pick*>(base + z.picks_at);
  w.sums = reinterpret_cast<double2*>(base + z.sums_at);
  w.rest = reinterpret_cast<double*>(base + z.rest_at);
  w.segs = z.segs;
  auto whole = [](const void* p, int64_t s, int64_t r) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 &&
                            (s * (int64_t)sizeof(T)) % 16 == 0 && (r * (int64_t)sizeof(T)) % 16 == 0);
  };
  const bool vec_ok = whole(a.target, a.target_seq_stride, a.target_row_stride) &&
                      whole(a.draft, a.draft_seq_stride, a.draft_row_stride);
  const int rows = a.num_seqs * (a.max_drafts + 1) + (a.draft == nullptr ? 0 : a.num_seqs * a.max_drafts);
  const dim3 per_seg((uint32_t)z.segs, (uint32_t)a.num_seqs);
  hipLaunchKernelGGL(verify_stats_kernel<T>, dim3((uint32_t)z.segs * (uint32_t)rows),
                     dim3(kThreads), 0, stream, a, w, vec_ok);
  hipLaunchKernelGGL(verify_pick_kernel<T>, dim3((uint32_t)a.num_seqs), dim3(kThreads), 0, stream, a,
                     w);
  hipLaunchKernelGGL(verify_sums_kernel<T>, per_seg, dim3(kThreads), 0, stream, a, w, vec_ok);
  if (a.draft != nullptr)
    hipLaunchKernelGGL(verify_rest_kernel<T>, per_seg, dim3(kThreads), 0, stream, a, w, vec_ok);
  hipLaunchKernelGGL(verify_draw_kernel<T>, dim3((uint32_t)a.num_seqs), dim3(kThreads), 0, stream, a,
                     w);
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
