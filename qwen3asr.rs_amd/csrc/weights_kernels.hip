// Attention weights of the cached tokens for gfx950: for each sequence s and
// kv head j,
//   scores[s, j, t] += sum over the call's query rows r and the query heads
//                      h of kv head j of softmax_t(scale * q[r, h] . K[s, j, t])
// over the tokens a row sees (all of the context, or with `causal` the tokens
// up to its own place at the context's end). A cache is cut by these sums
// (evict_kernels.hip).
//
// A weight needs its row's maximum and sum over the whole context, so every logit is
// needed twice. Three forms, by the rows a (sequence, kv head) has at most (a row
// being one query head of one new token) and the number of these pairs:
//   * up to 16 rows, contexts whose logits fit 64 KiB of LDS and are short or many: one
//     launch, a workgroup per pair, the logits kept in LDS (weight_logits_kernel, whole);
//   * up to 16 rows otherwise: a pass over the keys writes the logits (f32, log2 units)
//     and per chunk the row's maximum and sum, a pass over the logits joins the chunks'
//     pairs and adds the weights up. A logit costs 8 bytes of traffic per row against
//     the token's key row, read once: 6 % at two rows and D = 128 in 16 bits;
//   * more rows: both passes read the keys (mostly from the last-level cache the second
//     time) and form the logits, 16 rows at a time from registers (weight_rows_kernel).
// Each score is added to by one thread in a fixed order.
//
// The key tile [D/x][block][x] of 16 tokens is, vector for vector, the B operand
// of the 16-row matrix instructions: lane l holds token l % 16 and the x dims of
// chunk l / 16 (+ 4 per instruction). So the keys go from memory to the matrix
// cores with no shuffle and no LDS; the query rows (a row being one query head of
// one new token, 16 of one kv head per workgroup) are the A operand, loaded in
// the same order of dims. f32 keys take v_mfma_f32_16x16x4_f32 in the same way.
// Bound by the bytes of the keys, with many rows also by the vector instructions of
// their exponentials and reductions. Measured in 16 bits at 16 query and 8 kv heads of
// 128: 256 sequences of 16 to 4096 tokens (424 MB of keys), one row each, 76 us = 5.6
// TB/s (f32 142 us, fp8 keys 49); 8 sequences of 1000 to 6000 tokens (57 MB), 32 rows
// each, 38 us (19 per pass; 78 with stored logits); one sequence of 1500 tokens, 5.6 +
// 4.3 us; all rows of one prompt of 512 tokens 110 us, of 2048 432, of 8192 2360.

#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kThreads = 256;

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 wbf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 wf16x8_t __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x4_t mma16(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (std::is_same_v<T, bf16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(wbf16x8_t, a),
                                                   __builtin_bit_cast(wbf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(wf16x8_t, a),
                                                  __builtin_bit_cast(wf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma16_f32(const uint4& a, const uint4& b, f32x4_t c) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0,
                                              0);
}

// E4M3FN byte pairs -> f32 (exact, through bf16).
__device__ __forceinline__ void fp8x4_f32(uint32_t w, uint4& out) {
  const uint32_t lo = fp8x2_to_pk<bf16_t>(w, false), hi = fp8x2_to_pk<bf16_t>(w, true);
  out = make_uint4(lo << 16, lo & 0xffff0000u, hi << 16, hi & 0xffff0000u);
}

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp<kDppQuadXor1>(v));
  v = fmaxf(v, dpp<kDppQuadXor2>(v));
  v = fmaxf(v, dpp<kDppRowHalfMirror>(v));
  return fmaxf(v, dpp<kDppRowMirror>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp<kDppQuadXor1>(v);
  v += dpp<kDppQuadXor2>(v);
  v += dpp<kDppRowHalfMirror>(v);
  return v + dpp<kDppRowMirror>(v);
}

// The rows of sequence s: first query row and number of them, in bounds.
struct SeqRows {
  int64_t first;
  int n;
};
__device__ __forceinline__ SeqRows seq_rows(const WeightsArgs& a, int s) {
  if (a.cu_seqlens_q == nullptr) return {s, s < a.total_rows ? 1 : 0};
  const int64_t lo = a.cu_seqlens_q[s], hi = a.cu_seqlens_q[s + 1];
  const int64_t n = min(min(hi, a.total_rows) - lo, (int64_t)a.max_query_len);
  return {lo, (int)max(n, (int64_t)0)};
}
__device__ __forceinline__ int seq_len(const WeightsArgs& a, int s, int bs) {
  return (int)min((uint64_t)min(a.context_lens[s], (uint32_t)a.max_ctx),
                  (uint64_t)a.block_table_stride * (uint64_t)bs);
}

// A workgroup's kv head, sequence and part of the sequence: consecutive workgroups
// take the pairs, so the parts that only long sequences have come last.
struct Place {
  int j, s, part;
};
__device__ __forceinline__ Place place(const WeightsArgs& a, int num_kv_heads) {
  const uint32_t pairs = (uint32_t)a.num_seqs * (uint32_t)num_kv_heads;
  const uint32_t pair = blockIdx.x % pairs;
  return {(int)(pair % (uint32_t)num_kv_heads), (int)(pair / (uint32_t)num_kv_heads),
          (int)(blockIdx.x / pairs)};
}

// The sequence at place r of the lengths in descending order (equal 32nds of max_ctx
// in the order of their indexes), for at most kOrdered sequences: a wave holds the
// lengths and counts by ballots. The 256 sequences of the head of this file took 85 us in
// the order of the indexes, 76 in this one.
constexpr int kOrdered = 512;
__device__ __forceinline__ int longest(const WeightsArgs& a, int r) {
  const int lane = threadIdx.x & 63;
  const int shift = max(27 - (int)__clz(a.max_ctx), 0);
  int bin[kOrdered / 64];
#pragma unroll
  for (int i = 0; i < kOrdered / 64; ++i) {
    const int s = i * 64 + lane;
    bin[i] = s < a.num_seqs ? (int)(min(a.context_lens[s], (uint32_t)a.max_ctx) >> shift) : -1;
  }
  auto at_least = [&](int t) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kOrdered / 64; ++i) n += __popcll(__ballot(bin[i] >= t));
    return n;
  };
  int t = 0;
#pragma unroll
  for (int b = 32; b > 0; b /= 2)
    if (at_least(t + b) > r) t += b;
  r -= at_least(t + 1);
  int s = 0;
#pragma unroll
  for (int i = 0; i < kOrdered / 64; ++i) {
    const uint64_t m = __ballot(bin[i] == t);
    const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                                 __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
    const uint64_t hit = __ballot(bin[i] == t && before == r);
    if (hit != 0) s = i * 64 + __builtin_ctzll(hit);
    r -= __popcll(m);
  }
  return s;
}

// Tiles of 16 tokens whose keys a wave holds, by the 16-byte chunks of a key row: at
// most 64 registers.
constexpr int wave_tiles(int chunks) { return chunks <= 16 ? 4 : chunks <= 32 ? 2 : 1; }

// Shapes of the operands, by query type T, cache element C (T itself, or any with
// fp8 keys) and head dim.
template <typename T, typename C, int D>
struct Frag {
  static constexpr bool kF8 = std::is_same_v<C, fp8_t>;
  static constexpr bool kF32 = std::is_same_v<T, float>;
  static constexpr int X = pack_x<C>();
  static constexpr int CH = D / X;              // chunks of a key row
  static constexpr int KV = (CH + 3) / 4;       // vectors of a lane per 16 tokens
  static constexpr bool kRagged = CH % 4 != 0;  // (head dim 96 in fp8: the last is half there)
  static constexpr int QV = X * (int)ElemTraits<T>::kBytes / 16;  // query vectors per chunk
  static constexpr int TW = wave_tiles(CH);
  static_assert(D % X == 0, "whole chunks");

  uint4 v[KV];
};

// The 16 query rows from m0 on as the A operand, zeros past the last.
template <typename T, typename C, int D>
__device__ __forceinline__ void load_rows(const WeightsArgs& a, const SeqRows& rows, int j, int group,
                                          int m0, int m_count,
                                          uint4 (&qv)[Frag<T, C, D>::KV][Frag<T, C, D>::QV]) {
  using F = Frag<T, C, D>;
  const int lane = threadIdx.x & 63;
  const int m = m0 + (lane & 15), r = m / group;
  const T* q = static_cast<const T*>(a.query) +
               ((rows.first + min(r, rows.n - 1)) * a.num_heads + j * group + (m - r * group)) * D;
#pragma unroll
  for (int v = 0; v < F::KV; ++v)
#pragma unroll
    for (int h = 0; h < F::QV; ++h) {
      const int c = (lane >> 4) + 4 * v;
      qv[v][h] = make_uint4(0u, 0u, 0u, 0u);
      if (m < m_count && (!F::kRagged || c < F::CH))
        qv[v][h] =
            *reinterpret_cast<const uint4*>(q + c * F::X + h * (16 / ElemTraits<T>::kBytes));
    }
}

// The keys of 16 tokens: this lane's token lies at `off` of block `phys`.
template <typename T, typename C, int D, bool kOnce>
__device__ __forceinline__ void load_keys(const C* keys, int64_t block_stride, int64_t phys, int off,
                                          int bs_log2, Frag<T, C, D>& f) {
  using F = Frag<T, C, D>;
  const int c0 = (threadIdx.x & 63) >> 4;
  const uint4* tile = reinterpret_cast<const uint4*>(keys + phys * block_stride) + off;
#pragma unroll
  for (int v = 0; v < F::KV; ++v) {
    const int c = c0 + 4 * v;
    f.v[v] = make_uint4(0u, 0u, 0u, 0u);
    if (!F::kRagged || c < F::CH) {
      const uint4* src = tile + (c << bs_log2);
      if constexpr (kOnce) f.v[v] = load_stream(src);
      else f.v[v] = *src;
    }
  }
}

// Products of 16 rows and 16 tokens: lane l gets rows (l / 16) * 4 + i of token l % 16.
template <typename T, typename C, int D>
__device__ __forceinline__ f32x4_t products(
    const uint4 (&qv)[Frag<T, C, D>::KV][Frag<T, C, D>::QV], const Frag<T, C, D>& f) {
  using F = Frag<T, C, D>;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < F::KV; ++v) {
    if constexpr (F::kF8 && F::kF32) {
      const uint32_t w[4] = {f.v[v].x, f.v[v].y, f.v[v].z, f.v[v].w};
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        uint4 k;
        fp8x4_f32(w[h], k);
        acc = mma16_f32(qv[v][h], k, acc);
      }
    } else if constexpr (F::kF8) {
      uint4 lo, hi;
      fp8x16_to_pk<T>(f.v[v], lo, hi);
      acc = mma16<T>(qv[v][0], lo, acc);
      acc = mma16<T>(qv[v][1], hi, acc);
    } else if constexpr (F::kF32) {
      acc = mma16_f32(qv[v][0], f.v[v], acc);
    } else {
      acc = mma16<T>(qv[v][0], f.v[v], acc);
    }
  }
  return acc;
}

// Running maximum and sum of one row over the tokens a lane has seen. They begin at
// the lowest value, so that a masked logit (-inf) adds exp2(-inf) = 0.
struct RowStat {
  float m = -FLT_MAX, s = 0.f;
  __device__ __forceinline__ void add(float l) {
    const float n = fmaxf(m, l);
    s = fmaf(s, __builtin_amdgcn_exp2f(m - n), __builtin_amdgcn_exp2f(l - n));
    m = n;
  }
  __device__ __forceinline__ void join(float om, float os) {
    const float n = fmaxf(m, om);
    s = s * __builtin_amdgcn_exp2f(m - n) + os * __builtin_amdgcn_exp2f(om - n);
    m = n;
  }
  // over the 16 lanes of a row
  __device__ __forceinline__ void join16() {
    const float n = row16_max(m);
    s = row16_sum(s * __builtin_amdgcn_exp2f(m - n));
    m = n;
  }
};

// Few rows (one tile of 16 per kv head), first pass or both. One workgroup per (kv
// head, sequence, chunk): its waves share the chunk's tiles of 16 tokens evenly, each
// a run of them, with the next TW tiles' keys in flight. kWhole: the chunk is the
// whole context; its logits stay in LDS and the weights are added here.
template <typename T, typename C, int D, bool kWhole, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void weight_logits_kernel(
    WeightsArgs a, int32_t num_kv_heads, int32_t bs_log2, int64_t num_blocks, int64_t block_stride,
    int64_t head_stride, float* __restrict__ logits, float2* __restrict__ stats, int32_t ctx_pad,
    int32_t max_chunks, int32_t chunk_tokens) {
  using F = Frag<T, C, D>;
  constexpr int TW = F::TW;
  __shared__ float s_m[kWaves][16], s_s[kWaves][16];
  extern __shared__ uint32_t s_dyn[];  // the chunk's block ids, then its logits (kWhole)
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place(a, num_kv_heads);
  const int j = at.j, chunk = at.part;
  // the longest first, so that none is left to run alone at the end
  const int s = kWhole && a.num_seqs <= kOrdered ? longest(a, at.s) : at.s;
  const int group = a.num_heads / num_kv_heads;
  const int L = seq_len(a, s, 1 << bs_log2);
  const SeqRows rows = seq_rows(a, s);
  const int m_count = min(rows.n * group, 16);  // rows of this kv head
  const int64_t begin = (int64_t)chunk * chunk_tokens;
  if (begin >= L || m_count == 0) return;

  const int tiles = ((int)min((int64_t)chunk_tokens, L - begin) + 15) / 16;
  const int per = (tiles + kWaves - 1) / kWaves;
  const int nt = min(per, tiles - wave * per);  // tiles of this wave, none if negative
  const int t_wave = (int)begin + wave * per * 16;
  const int b_first = (int)begin >> bs_log2;  // (chunks are whole blocks)
  {
    const int n = (((int)begin + tiles * 16 - 1) >> bs_log2) - b_first + 1;
    const int last = (L - 1) >> bs_log2;
    const uint32_t* table = a.block_tables + (int64_t)s * a.block_table_stride;
    for (int i = threadIdx.x; i < n; i += 64 * kWaves) s_dyn[i] = table[min(b_first + i, last)];
  }
  uint4 qv[F::KV][F::QV];
  load_rows<T, C, D>(a, rows, j, group, 0, m_count, qv);
  float scale = a.scale * 1.4426950408889634f;
  if constexpr (F::kF8) scale *= *a.k_scale;
  const C* keys = static_cast<const C*>(a.key_cache) + j * head_stride;

  // per row of the lane: last token it sees, plus one, and where its logits go
  float* s_logits = reinterpret_cast<float*>(s_dyn + (chunk_tokens >> bs_log2));
  int see[4];
  float* dst[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = (lane >> 4) * 4 + i, r = m / group;
    see[i] = m >= m_count ? 0 : a.causal ? min(L, r + 1 + L - rows.n) : L;
    dst[i] = (kWhole ? s_logits + m * chunk_tokens
                     : logits + ((rows.first + r) * a.num_heads + j * group + (m - r * group)) *
                                    ctx_pad) +
             t_wave + (lane & 15);
  }
  lds_group_barrier();
  Frag<T, C, D> f[TW];
  bool ok[TW];
  auto load = [&](int u, int i) {
    const int tok = min(t_wave + i * 16 + (lane & 15), L - 1);  // past the end: masked below
    const uint32_t phys = s_dyn[(tok >> bs_log2) - b_first];
    ok[u] = (int64_t)phys < num_blocks;
    load_keys<T, C, D, true>(keys, block_stride, ok[u] ? (int64_t)phys : 0,
                             tok & ((1 << bs_log2) - 1), bs_log2, f[u]);
  };
  RowStat st[4];
  auto use = [&](int u, int i, const f32x4_t& acc, bool there) {
    const int tok = t_wave + i * 16 + (lane & 15);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k >= m_count) break;  // (uniform: rows 0 .. 3 are in the first lanes)
      const float l = there && tok < see[k] ? acc[k] * scale : -INFINITY;
      st[k].add(l);
      if ((lane >> 4) * 4 + k < m_count) dst[k][i * 16] = l;
    }
  };
#pragma unroll
  for (int u = 0; u < TW; ++u)
    if (u < nt) load(u, u);
  int i0 = 0;
#pragma unroll 1
  for (; i0 + 2 * TW <= nt; i0 += TW) {
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      const f32x4_t acc = products<T, C, D>(qv, f[u]);
      const bool there = ok[u];
      load(u, i0 + u + TW);
      use(u, i0 + u, acc, there);
    }
  }
#pragma unroll 1
  for (; i0 < nt; i0 += TW) {  // at most two rounds
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      if (i0 + u < nt) {
        const f32x4_t acc = products<T, C, D>(qv, f[u]);
        const bool there = ok[u];
        if (i0 + u + TW < nt) load(u, i0 + u + TW);
        use(u, i0 + u, acc, there);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    st[k].join16();
    if ((lane & 15) == 0) {
      s_m[wave][(lane >> 4) * 4 + k] = st[k].m;
      s_s[wave][(lane >> 4) * 4 + k] = st[k].s;
    }
  }
  lds_group_barrier();
  const int m = threadIdx.x;
  if constexpr (kWhole) {
    if (m < m_count) {
      RowStat all;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all.join(s_m[w][m], s_s[w][m]);
      s_m[0][m] = all.m;
      s_s[0][m] = all.s == 0.f ? 0.f : 1.f / all.s;  // (a row that sees no token adds nothing)
    }
    lds_group_barrier();
    float* out = a.scores + s * a.score_seq_stride + j * a.score_head_stride;
    for (int t = threadIdx.x; t < L; t += 64 * kWaves) {
      float sum = 0.f;
      for (int i = 0; i < m_count; ++i) {
        const float l = s_logits[i * chunk_tokens + t];
        sum += l == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l - s_m[0][i]) * s_s[0][i];
      }
      out[t] += sum;
    }
  } else if (m < m_count) {
    RowStat all;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all.join(s_m[w][m], s_s[w][m]);
    const int r = m / group;
    stats[((rows.first + r) * a.num_heads + j * group + (m - r * group)) * max_chunks + chunk] =
        make_float2(all.m, all.s);
  }
}

// Maximum and reciprocal sum of a row, from its chunks' pairs, by kLanes lanes (four
// pairs each in flight); a row that sees no token gets a reciprocal of 0.
template <int kLanes>
__device__ __forceinline__ float2 merge_row(const float2* st, int chunks, int part) {
  RowStat all;
  for (int c = part; c < chunks; c += 4 * kLanes) {
    float2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = st[min(c + i * kLanes, chunks - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i * kLanes < chunks) all.join(v[i].x, v[i].y);
  }
#pragma unroll
  for (int x = 1; x < kLanes; x *= 2)
    all.join(__shfl_xor(all.m, x, 64), __shfl_xor(all.s, x, 64));
  return make_float2(all.m, all.s == 0.f ? 0.f : 1.f / all.s);
}

// Second pass of few rows: one workgroup per (kv head, sequence, 1024 tokens), four tokens
// 256 apart per thread (single words: score rows have any alignment).
__global__ __launch_bounds__(kThreads) void weight_sum_kernel(WeightsArgs a, int32_t num_kv_heads,
                                                              int32_t bs,
                                                              const float* __restrict__ logits,
                                                              const float2* __restrict__ stats,
                                                              int32_t ctx_pad, int32_t max_chunks,
                                                              int32_t chunk_tokens) {
  __shared__ float2 s_row[16];
  const Place at = place(a, num_kv_heads);
  const int j = at.j, s = at.s;
  const int64_t begin = (int64_t)at.part * 1024;
  const int group = a.num_heads / num_kv_heads;
  const int L = seq_len(a, s, bs);
  const SeqRows rows = seq_rows(a, s);
  const int m_count = min(rows.n * group, 16);
  if (begin >= L || m_count == 0) return;
  const int t = (int)begin + threadIdx.x;
  auto row_of = [&](int m) {
    const int r = m / group;
    return (rows.first + r) * a.num_heads + j * group + (m - r * group);
  };
  float* out = a.scores + s * a.score_seq_stride + j * a.score_head_stride + t;
  float l[4], acc[4];
  auto load = [&](int m) {
    const float* src = logits + row_of(m) * ctx_pad + t;
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = t + i * 256 < L ? src[i * 256] : -INFINITY;
  };
  load(0);  // in flight while the rows' sums are joined
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = t + i * 256 < L ? out[i * 256] : 0.f;
  {
    const int m = threadIdx.x >> 4, part = threadIdx.x & 15;
    const int chunks = (L + chunk_tokens - 1) / chunk_tokens;
    const float2 row = merge_row<16>(stats + row_of(min(m, m_count - 1)) * max_chunks, chunks, part);
    if (part == 0) s_row[m] = row;
  }
  lds_group_barrier();
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m = 0; m < m_count; ++m) {
    const float2 row = s_row[m];
    float w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = l[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l[i] - row.x) * row.y;
    if (m + 1 < m_count) load(m + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += w[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t + i * 256 < L) out[i * 256] = acc[i] + sum[i];
}

// Sizes of the passes of many rows, by the 16-byte vectors of a query row: the keys of a
// wave's tiles take 64 registers (in the query's type), the queries of a block of rows
// 16 KiB of LDS.
constexpr int row_tiles(int vectors) { return vectors <= 16 ? 4 : vectors <= 32 ? 2 : 1; }
constexpr int row_block(int vectors) { return 16 * row_tiles(vectors); }

// Waves per SIMD of these passes: four (128 registers), or three where 32-bit queries
// meet fp8 keys, which would spill. The first pass over 8 sequences of 1000 to 6000
// tokens with 64 rows each took 18.6 us, with three 21.6.
template <typename T, typename C>
constexpr int kRowWaves = std::is_same_v<T, float> && !std::is_same_v<T, C> ? 3 : 4;

// Both passes of many rows; the logits are formed anew in the second (kSum). A workgroup
// holds the keys of a piece of 4 * TW tiles in registers, converted to the query's type,
// while a block of rows passes by in LDS, 16 at a time. First pass: one workgroup per (kv
// head, sequence, chunk of `subs` pieces, block of rows), writing the rows' pairs;
// second: per (kv head, sequence, piece), all rows.
template <typename T, typename C, int D, bool kSum>
__global__ __launch_bounds__(kThreads, (kRowWaves<T, C>)) void weight_rows_kernel(
    WeightsArgs a, int32_t num_kv_heads, int32_t bs_log2, int64_t num_blocks, int64_t block_stride,
    int64_t head_stride, float2* __restrict__ stats, int32_t max_chunks, int32_t subs) {
  using F = Frag<T, C, D>;
  constexpr int RV = D * (int)ElemTraits<T>::kBytes / 16;  // vectors of a query row
  constexpr int TW = row_tiles(RV), RB = row_block(RV);
  constexpr int kPiece = 64 * TW;
  __shared__ uint4 s_q[RB][RV + 1];  // (padded: 16 rows in different banks)
  __shared__ float2 s_row[kSum ? 1 : 4][RB];
  __shared__ int s_see[RB];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Place at = place(a, num_kv_heads);
  const int j = at.j, s = at.s;
  const int group = a.num_heads / num_kv_heads;
  const int L = seq_len(a, s, 1 << bs_log2);
  const SeqRows rows = seq_rows(a, s);
  const int m_count = rows.n * group;
  const int chunk = kSum ? 0 : at.part % max_chunks;
  const int mb = kSum ? 0 : at.part / max_chunks * RB;
  const int chunks = (L + kPiece * subs - 1) / (kPiece * subs);
  const int64_t begin = kSum ? (int64_t)at.part * kPiece : (int64_t)chunk * subs * kPiece;
  if (begin >= L || mb >= m_count) return;
  float scale = a.scale * 1.4426950408889634f;
  if constexpr (F::kF8) scale *= *a.k_scale;
  const C* keys = static_cast<const C*>(a.key_cache) + j * head_stride;
  const uint32_t* table = a.block_tables + (int64_t)s * a.block_table_stride;
  auto row_of = [&](int m) {
    const int r = m / group;
    return (rows.first + r) * a.num_heads + j * group + (m - r * group);
  };
  uint4 kv[TW][F::KV][F::QV];
  bool ok[TW];
  auto load = [&](int t_wave) {
    uint32_t phys[TW];
#pragma unroll
    for (int u = 0; u < TW; ++u)
      phys[u] = table[min(t_wave + u * 16 + (lane & 15), L - 1) >> bs_log2];
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      const int tok = min(t_wave + u * 16 + (lane & 15), L - 1);
      ok[u] = (int64_t)phys[u] < num_blocks;
      Frag<T, C, D> f;
      load_keys<T, C, D, false>(keys, block_stride, ok[u] ? (int64_t)phys[u] : 0,
                                tok & ((1 << bs_log2) - 1), bs_log2, f);
#pragma unroll
      for (int v = 0; v < F::KV; ++v) {
        if constexpr (F::kF8 && F::kF32) {
          fp8x4_f32(f.v[v].x, kv[u][v][0]);
          fp8x4_f32(f.v[v].y, kv[u][v][1]);
          fp8x4_f32(f.v[v].z, kv[u][v][2]);
          fp8x4_f32(f.v[v].w, kv[u][v][3]);
        } else if constexpr (F::kF8) {
          fp8x16_to_pk<T>(f.v[v], kv[u][v][0], kv[u][v][1]);
        } else {
          kv[u][v][0] = f.v[v];
        }
      }
    }
  };
  // the queries of a block of rows (zeros past the last) and the last token each sees,
  // plus one
  auto stage = [&](int m_at) {
    for (int i = threadIdx.x; i < RB * RV; i += kThreads) {
      const int mi = i / RV, m = m_at + mi;
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (m < m_count)
        q = reinterpret_cast<const uint4*>(static_cast<const T*>(a.query) + row_of(m) * D)[i - mi * RV];
      s_q[mi][i - mi * RV] = q;
    }
    const int m = m_at + threadIdx.x;
    if (threadIdx.x < RB)
      s_see[threadIdx.x] = m >= m_count ? 0 : a.causal ? min(L, m / group + 1 + L - rows.n) : L;
  };
  // the products of rows from .. to of the block: visit(first of the lane's four rows, acc)
  auto block_rows = [&](int from, int to, auto visit) {
#pragma unroll 1
    for (int m0 = from; m0 < to; m0 += 16) {
      asm volatile("" ::: "memory");  // (no later read of LDS moves up: registers)
      f32x4_t acc[TW];
#pragma unroll
      for (int u = 0; u < TW; ++u) acc[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < F::KV; ++v) {
        const int c = (lane >> 4) + 4 * v;
#pragma unroll
        for (int h = 0; h < F::QV; ++h) {
          uint4 q = make_uint4(0u, 0u, 0u, 0u);
          if (!F::kRagged || c < F::CH) q = s_q[m0 + (lane & 15)][c * F::QV + h];
#pragma unroll
          for (int u = 0; u < TW; ++u) {
            if constexpr (F::kF32) acc[u] = mma16_f32(q, kv[u][v][h], acc[u]);
            else acc[u] = mma16<T>(q, kv[u][v][h], acc[u]);
          }
        }
      }
      visit(m0 + (lane >> 4) * 4, acc);
    }
  };
  // whether every row sees every token of the wave's tiles (uniform)
  auto all_seen = [&](int t_wave) {
    bool there = true;
#pragma unroll
    for (int u = 0; u < TW; ++u) there &= ok[u];
    return t_wave + 16 * TW <= (a.causal ? L - rows.n + 1 : L) && __all(there);
  };
  auto logit = [&](float acc, int u, int t_wave, int see) {
    return ok[u] && t_wave + u * 16 + (lane & 15) < see ? acc * scale : -INFINITY;
  };
  if constexpr (!kSum) {
    const int n = min(RB, m_count - mb);
    stage(mb);
    for (int sub = 0; sub < subs; ++sub) {
      const int64_t piece = begin + sub * kPiece;
      if (piece >= L) break;
      const int t_wave = (int)piece + wave * 16 * TW;
      load(t_wave);
      if (sub == 0) lds_group_barrier();
      auto stat = [&](int mi, const float(&l)[TW]) {
        RowStat st;
#pragma unroll
        for (int u = 0; u < TW; ++u) st.m = fmaxf(st.m, l[u]);
        st.m = row16_max(st.m);
#pragma unroll
        for (int u = 0; u < TW; ++u) st.s += __builtin_amdgcn_exp2f(l[u] - st.m);
        st.s = row16_sum(st.s);
        float2& mine = s_row[wave][mi];
        if ((lane & 15) == 0) {
          if (sub > 0) st.join(mine.x, mine.y);
          mine = make_float2(st.m, st.s);
        }
      };
      if (all_seen(t_wave)) {
        block_rows(0, n, [&](int mi, const f32x4_t(&acc)[TW]) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float l[TW];
#pragma unroll
            for (int u = 0; u < TW; ++u) l[u] = acc[u][k] * scale;
            stat(mi + k, l);
          }
        });
      } else {
        block_rows(0, n, [&](int mi, const f32x4_t(&acc)[TW]) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float l[TW];
#pragma unroll
            for (int u = 0; u < TW; ++u) l[u] = logit(acc[u][k], u, t_wave, s_see[mi + k]);
            stat(mi + k, l);
          }
        });
      }
    }
    lds_group_barrier();
    const int m = mb + threadIdx.x;
    if (threadIdx.x < n) {
      RowStat all;
#pragma unroll
      for (int w = 0; w < 4; ++w) all.join(s_row[w][threadIdx.x].x, s_row[w][threadIdx.x].y);
      stats[row_of(m) * max_chunks + chunk] = make_float2(all.m, all.s);
    }
  } else {
    const int t_wave = (int)begin + wave * 16 * TW;
    constexpr int kLanes = kThreads / RB;  // lanes that merge a row's pairs
    float sum[TW];
#pragma unroll
    for (int u = 0; u < TW; ++u) sum[u] = 0.f;
    load(t_wave);
#pragma unroll 1
    for (int m_at = 0; m_at < m_count; m_at += RB) {
      const int n = min(RB, m_count - m_at);
      if (m_at > 0) lds_group_barrier();  // (the rows before are used)
      stage(m_at);
      const int m = threadIdx.x / kLanes, part = threadIdx.x % kLanes;
      const float2 row =
          merge_row<kLanes>(stats + row_of(min(m_at + m, m_count - 1)) * max_chunks, chunks, part);
      if (part == 0) s_row[0][m] = row;
      lds_group_barrier();
      // (tiles with rows past the last take the masked form: an infinite key has no
      // product with a query of zeros)
      const int plain = all_seen(t_wave) ? n & ~15 : 0;
      if (plain > 0) {
        block_rows(0, plain, [&](int mi, const f32x4_t(&acc)[TW]) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 row = s_row[0][mi + k];
#pragma unroll
            for (int u = 0; u < TW; ++u)
              sum[u] = fmaf(__builtin_amdgcn_exp2f(fmaf(acc[u][k], scale, -row.x)), row.y, sum[u]);
          }
        });
      }
      if (plain < n) {
        block_rows(plain, n, [&](int mi, const f32x4_t(&acc)[TW]) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 row = s_row[0][mi + k];
#pragma unroll
            for (int u = 0; u < TW; ++u) {
              const float l = logit(acc[u][k], u, t_wave, s_see[mi + k]);
              sum[u] += l == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l - row.x) * row.y;
            }
          }
        });
      }
    }
    float* out = a.scores + s * a.score_seq_stride + j * a.score_head_stride;
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      sum[u] += __shfl_xor(sum[u], 16, 64);
      sum[u] += __shfl_xor(sum[u], 32, 64);
      const int tok = t_wave + u * 16 + lane;
      if (lane < 16 && tok < L) out[tok] += sum[u];
    }
  }
}

template <typename T, typename C, int D>
hipError_t weights_launch(const WeightsArgs& a, const WeightsPlan& p, const CacheGeom& g,
                          hipStream_t stream) {
  const int bs_log2 = __builtin_ctz((unsigned)g.block_size);
  float2* stats = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + p.stats_at);
  if (p.few) {
    float* logits = static_cast<float*>(a.workspace);
    const uint32_t lds = (uint32_t)(p.chunk_tokens >> bs_log2) * 4;
    if (p.whole && p.wide) {
      hipLaunchKernelGGL((weight_logits_kernel<T, C, D, true, 8>), dim3((uint32_t)p.first_grid),
                         dim3(512), lds + (uint32_t)p.lds_logits, stream, a, g.num_kv_heads,
                         bs_log2, g.num_blocks, g.block_stride, g.head_stride, logits, stats,
                         p.ctx_pad, p.max_chunks, p.chunk_tokens);
      return hipGetLastError();
    }
    if (p.whole) {
      hipLaunchKernelGGL((weight_logits_kernel<T, C, D, true, 4>), dim3((uint32_t)p.first_grid),
                         dim3(kThreads), lds + (uint32_t)p.lds_logits, stream, a, g.num_kv_heads,
                         bs_log2, g.num_blocks, g.block_stride, g.head_stride, logits, stats,
                         p.ctx_pad, p.max_chunks, p.chunk_tokens);
      return hipGetLastError();
    }
    hipLaunchKernelGGL((weight_logits_kernel<T, C, D, false, 4>), dim3((uint32_t)p.first_grid),
                       dim3(kThreads), lds, stream, a, g.num_kv_heads, bs_log2, g.num_blocks,
                       g.block_stride, g.head_stride, logits, stats, p.ctx_pad, p.max_chunks,
                       p.chunk_tokens);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(weight_sum_kernel, dim3((uint32_t)p.second_grid), dim3(kThreads), 0, stream,
                       a, g.num_kv_heads, g.block_size, logits, stats, p.ctx_pad, p.max_chunks,
                       p.chunk_tokens);
    return hipGetLastError();
  }
  const int subs = p.chunk_tokens / (64 * row_tiles(D * (int)ElemTraits<T>::kBytes / 16));
  hipLaunchKernelGGL((weight_rows_kernel<T, C, D, false>), dim3((uint32_t)p.first_grid),
                     dim3(kThreads), 0, stream, a, g.num_kv_heads, bs_log2, g.num_blocks,
                     g.block_stride, g.head_stride, stats, p.max_chunks, subs);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((weight_rows_kernel<T, C, D, true>), dim3((uint32_t)p.second_grid),
                     dim3(kThreads), 0, stream, a, g.num_kv_heads, bs_log2, g.num_blocks,
                     g.block_stride, g.head_stride, stats, p.max_chunks, subs);
  return hipGetLastError();
}

template <typename T, typename C>
hipError_t weights_typed(const WeightsArgs& a, const WeightsPlan& p, const CacheGeom& g,
                         hipStream_t stream) {
  switch (g.head_dim) {
    case 64: return weights_launch<T, C, 64>(a, p, g, stream);
    case 96: return weights_launch<T, C, 96>(a, p, g, stream);
    case 128: return weights_launch<T, C, 128>(a, p, g, stream);
    case 192: return weights_launch<T, C, 192>(a, p, g, stream);
    case 256: return weights_launch<T, C, 256>(a, p, g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// A pair per row and chunk (of kWeightsChunk tokens or a multiple), and of few rows the
// logits.
size_t weights_workspace_bytes(int64_t total_rows, int32_t num_heads, int32_t max_ctx, bool few) {
  const int64_t chunks = ((int64_t)max_ctx + kWeightsChunk - 1) / kWeightsChunk;
  return (size_t)(total_rows * num_heads * chunks) *
         ((few ? kWeightsChunk * sizeof(float) : 0) + sizeof(float2));
}

WeightsPlan weights_plan(int dtype, const WeightsArgs& a, const CacheGeom& g) {
  WeightsPlan p;
  const int64_t pairs = (int64_t)g.num_kv_heads * a.num_seqs;
  const int64_t m_max = (int64_t)a.max_query_len * (a.num_heads / g.num_kv_heads);
  auto parts = [&](int tokens) { return ((int64_t)a.max_ctx + tokens - 1) / tokens; };
  // (at 16 rows the stored logits took 26 us for 8 sequences of 4000 tokens and 76 for
  // 64 of 2000, the second reading of the keys 28 and 86)
  p.few = weights_few(a.max_query_len, a.num_heads, g.num_kv_heads);
  p.whole = p.wide = false;
  p.lds_logits = 0;
  p.ctx_pad = (int32_t)(parts(kWeightsChunk) * kWeightsChunk);
  p.chunk_tokens = kWeightsChunk;
  if (p.few) {
    // Whole contexts per workgroup where none is left alone for long: eight waves take 2.8
    // us per 1000 tokens, two launches of many workgroups 8.7 us at the least. Short
    // contexts (one sequence of 300 tokens, 8 kv heads: 7.0 us; 8.6 in two launches; 1000
    // tokens 9.2 and 8.7), contexts short for the number of pairs (32 sequences of 1000
    // 13.9 and 17.1, 48 of 2000 38 and 40; 32 of up to 4096 30 and 28), and 512 pairs or
    // more (64 of up to 4096 36 and 40, 512 of them 207 and 246). By four waves from 2048
    // pairs on (256 sequences of up to 4096: 104 us, 110 by eight; 128 of them 62 and 53;
    // nothing between was measured). All at 128 dims in 16 bits; the other types and dims
    // follow the same borders.
    const int64_t lds = m_max * p.ctx_pad * (int64_t)sizeof(float);
    p.whole = lds <= 65536 && (pairs >= 512 || a.max_ctx <= std::max<int64_t>(768, 4 * pairs));
    p.wide = pairs < 2048;
    if (p.whole) {
      p.chunk_tokens = p.ctx_pad;
      p.lds_logits = (int32_t)lds;
    }
    // chunks of 256 to 1024 tokens (64 to 256 per wave) while each compute unit has four
    while (!p.whole && p.chunk_tokens < 1024 && pairs * parts(2 * p.chunk_tokens) >= 1024)
      p.chunk_tokens *= 2;
    p.first_grid = pairs * parts(p.chunk_tokens);
    p.second_grid = pairs * parts(1024);
  } else {
    const int vectors = g.head_dim * (dtype == VPA_DTYPE_F32 ? 4 : 2) / 16;
    const int64_t blocks = (m_max + row_block(vectors) - 1) / row_block(vectors);
    while (p.chunk_tokens < 1024 && pairs * blocks * parts(2 * p.chunk_tokens) >= 1024)
      p.chunk_tokens *= 2;
    p.first_grid = pairs * blocks * parts(p.chunk_tokens);
    p.second_grid = pairs * parts(64 * row_tiles(vectors));
  }
  p.max_chunks = (int32_t)parts(p.chunk_tokens);
  p.stats_at = p.few ? (size_t)(a.total_rows * a.num_heads) * p.ctx_pad * sizeof(float) : 0;
  return p;
}

hipError_t launch_attention_weights(int dtype, int cache_dtype, const WeightsArgs& a,
                                    const CacheGeom& g, hipStream_t stream) {
  const bool fp8 = cache_dtype == VPA_DTYPE_FP8_E4M3;
  const WeightsPlan p = weights_plan(dtype, a, g);
  switch (dtype) {
    case VPA_DTYPE_F32:
      return fp8 ? weights_typed<float, fp8_t>(a, p, g, stream)
                 : weights_typed<float, float>(a, p, g, stream);
    case VPA_DTYPE_F16:
      return fp8 ? weights_typed<f16_t, fp8_t>(a, p, g, stream)
                 : weights_typed<f16_t, f16_t>(a, p, g, stream);
    case VPA_DTYPE_BF16:
      return fp8 ? weights_typed<bf16_t, fp8_t>(a, p, g, stream)
                 : weights_typed<bf16_t, bf16_t>(a, p, g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vpa
