// Attention weights of the cached tokens for gfx950: for each sequence s and
// kv head j,
//   scores[s, j, t] += sum over the call's query rows r and the query heads
//                      h of kv head j of softmax_t(scale * q[r, h] . K[s, j, t])
// over the tokens a row sees (all of the context, or with `causal` the tokens
// up to its own place at the context's end). A cache is cut by these sums
// (evict_kernels.hip).
//
// A weight needs its row's maximum and sum over the whole context, so the
// keys' logits are formed once and kept: a pass over the keys writes the
// logits (f32, log2 units) and per chunk of 256 tokens the row's maximum and
// sum, then a pass over the logits merges the chunks' pairs and adds the
// weights up, each score by one thread in a fixed order. A logit costs 8 bytes
// of traffic per query head against the token's D-element key row, read once:
// 6 % at two query heads per kv head and D = 128 in 16 bits. Reading the keys a
// second time instead would cost 100 %.
//
// The key tile [D/x][block][x] of 16 tokens is, vector for vector, the B operand
// of the 16-row matrix instructions: lane l holds token l % 16 and the x dims of
// chunk l / 16 (+ 4 per instruction). So the keys go from memory to the matrix
// cores with no shuffle and no LDS; the query rows (a row being one query head of
// one new token, 16 of one kv head per workgroup) are the A operand, loaded in
// the same order of dims. f32 keys take v_mfma_f32_16x16x4_f32 in the same way.
// Bound by the bytes of the keys.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kChunk = kWeightsChunk;  // tokens of a workgroup, 64 per wave
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

// C: cache element; T: query element (C, or any with fp8 keys).
template <typename T, typename C, int D>
__global__ __launch_bounds__(kThreads) void weight_logits_kernel(WeightsArgs a, int32_t num_kv_heads,
                                                                 int32_t bs_log2, int64_t num_blocks,
                                                                 int64_t block_stride,
                                                                 int64_t head_stride,
                                                                 float* __restrict__ logits,
                                                                 float2* __restrict__ stats,
                                                                 int32_t ctx_pad, int32_t max_chunks) {
  constexpr bool kF8 = std::is_same_v<C, fp8_t>;
  constexpr bool kF32 = std::is_same_v<T, float>;
  constexpr int X = pack_x<C>();
  constexpr int CH = D / X;               // chunks of a key row
  constexpr int KV = (CH + 3) / 4;        // vectors of a lane per 16 tokens
  constexpr bool kRagged = CH % 4 != 0;   // (head dim 96 in fp8: the last vector is half there)
  constexpr int QV = X * (int)ElemTraits<T>::kBytes / 16;  // query vectors per chunk
  // tiles of 16 tokens whose keys are in flight together: at most 64 registers
  constexpr int TW = KV * 4 <= 64 / 4 ? 4 : KV * 2 <= 64 / 4 ? 2 : 1;
  static_assert(D % X == 0, "whole chunks");

  __shared__ float s_m[4][16], s_s[4][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bs = 1 << bs_log2;
  const int s = blockIdx.y;
  const int j = (int)(blockIdx.x % (uint32_t)num_kv_heads);
  const int rest = (int)(blockIdx.x / (uint32_t)num_kv_heads);
  const int chunk = rest % max_chunks, rg = rest / max_chunks;
  const int group = a.num_heads / num_kv_heads;
  const int L = seq_len(a, s, bs);
  const SeqRows rows = seq_rows(a, s);
  const int m_count = rows.n * group;  // rows of this kv head
  if (chunk * kChunk >= L || rg * 16 >= m_count) return;

  // query row of this lane in the A operand, zeros past the last
  const int c0 = lane >> 4;
  uint4 qv[KV][QV];
  {
    const int m = rg * 16 + (lane & 15);
    const int r = m / group;
    const T* q = static_cast<const T*>(a.query) +
                 ((rows.first + min(r, rows.n - 1)) * a.num_heads + j * group + (m - r * group)) * D;
#pragma unroll
    for (int v = 0; v < KV; ++v)
#pragma unroll
      for (int h = 0; h < QV; ++h) {
        const int c = c0 + 4 * v;
        qv[v][h] = make_uint4(0u, 0u, 0u, 0u);
        if (m < m_count && (!kRagged || c < CH))
          qv[v][h] = *reinterpret_cast<const uint4*>(q + c * X + h * (16 / ElemTraits<T>::kBytes));
      }
  }
  float scale = a.scale * 1.4426950408889634f;
  if constexpr (kF8) scale *= *a.k_scale;

  const uint32_t* table = a.block_tables + (int64_t)s * a.block_table_stride;
  const C* keys = static_cast<const C*>(a.key_cache) + j * head_stride;
  const int t_wave = chunk * kChunk + wave * 64;
  // last token each of the lane's four rows sees, plus one
  int see[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = rg * 16 + (lane >> 4) * 4 + i;
    const int r = m / group;
    see[i] = m >= m_count ? 0 : a.causal ? min(L, r + 1 + L - rows.n) : L;
  }
  float lg[4][4];  // [tile][row]
#pragma unroll
  for (int t4 = 0; t4 < 4; t4 += TW) {
    uint4 kv[TW][KV];
    bool ok[TW];
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      const int tok = t_wave + (t4 + u) * 16 + (lane & 15);
      const int tc = min(tok, L - 1);  // past the context: its last token, masked below
      const uint32_t phys = table[tc >> bs_log2];
      ok[u] = (int64_t)phys < num_blocks;
      const uint4* tile = reinterpret_cast<const uint4*>(
          keys + (ok[u] ? (int64_t)phys : 0) * block_stride) + (tc & (bs - 1));
#pragma unroll
      for (int v = 0; v < KV; ++v) {
        const int c = c0 + 4 * v;
        kv[u][v] = make_uint4(0u, 0u, 0u, 0u);
        if (!kRagged || c < CH) kv[u][v] = load_stream(tile + (c << bs_log2));
      }
    }
#pragma unroll
    for (int u = 0; u < TW; ++u) {
      f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < KV; ++v) {
        if constexpr (kF8 && kF32) {
          const uint32_t w[4] = {kv[u][v].x, kv[u][v].y, kv[u][v].z, kv[u][v].w};
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint4 f;
            fp8x4_f32(w[h], f);
            acc = mma16_f32(qv[v][h], f, acc);
          }
        } else if constexpr (kF8) {
          uint4 lo, hi;
          fp8x16_to_pk<T>(kv[u][v], lo, hi);
          acc = mma16<T>(qv[v][0], lo, acc);
          acc = mma16<T>(qv[v][1], hi, acc);
        } else if constexpr (kF32) {
          acc = mma16_f32(qv[v][0], kv[u][v], acc);
        } else {
          acc = mma16<T>(qv[v][0], kv[u][v], acc);
        }
      }
      const int tok = t_wave + (t4 + u) * 16 + (lane & 15);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        lg[t4 + u][i] = ok[u] && tok < see[i] ? acc[i] * scale : -INFINITY;
    }
  }
  // the logits, and the row's maximum and sum over the wave's tokens
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int mi = (lane >> 4) * 4 + i, m = rg * 16 + mi;
    const float mx = row16_max(fmaxf(fmaxf(lg[0][i], lg[1][i]), fmaxf(lg[2][i], lg[3][i])));
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      sum += lg[u][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lg[u][i] - mx);
    sum = row16_sum(sum);
    if ((lane & 15) == 0) {
      s_m[wave][mi] = mx;
      s_s[wave][mi] = sum;
    }
    if (m < m_count) {
      const int r = m / group;
      float* dst = logits + ((rows.first + r) * a.num_heads + j * group + (m - r * group)) * ctx_pad +
                   t_wave + (lane & 15);
#pragma unroll
      for (int u = 0; u < 4; ++u) dst[16 * u] = lg[u][i];
    }
  }
  __syncthreads();
  const int m = rg * 16 + threadIdx.x;
  if (threadIdx.x < 16 && m < m_count) {
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mx = fmaxf(mx, s_m[w][threadIdx.x]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float sw = s_s[w][threadIdx.x];
      if (sw != 0.f) sum += sw * __builtin_amdgcn_exp2f(s_m[w][threadIdx.x] - mx);
    }
    const int r = m / group;
    stats[((rows.first + r) * a.num_heads + j * group + (m - r * group)) * max_chunks + chunk] =
        make_float2(mx, sum);
  }
}

// Rows merged at once in the second pass.
constexpr int kRowTile = 64;

// One workgroup per (1024 tokens, kv head, sequence), four tokens per thread.
__global__ __launch_bounds__(kThreads) void weight_sum_kernel(WeightsArgs a, int32_t num_kv_heads,
                                                              int32_t bs,
                                                              const float* __restrict__ logits,
                                                              const float2* __restrict__ stats,
                                                              int32_t ctx_pad, int32_t max_chunks) {
  __shared__ float s_max[kRowTile], s_inv[kRowTile];
  const int s = blockIdx.z, j = blockIdx.y;
  const int t = blockIdx.x * 1024 + threadIdx.x * 4;
  const int group = a.num_heads / num_kv_heads;
  const int L = seq_len(a, s, bs);
  if (blockIdx.x * 1024 >= (uint32_t)L) return;
  const SeqRows rows = seq_rows(a, s);
  const int m_count = rows.n * group;
  const int chunks = (L + kChunk - 1) / kChunk;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int m0 = 0; m0 < m_count; m0 += kRowTile) {
    const int n = min(kRowTile, m_count - m0);
    __syncthreads();
    {  // four lanes per row merge the chunks' pairs
      const int mi = threadIdx.x >> 2, part = threadIdx.x & 3;
      float mx = -INFINITY, sum = 0.f;
      if (mi < n) {
        const int m = m0 + mi, r = m / group;
        const float2* st =
            stats + ((rows.first + r) * a.num_heads + j * group + (m - r * group)) * max_chunks;
        for (int c = part; c < chunks; c += 4) mx = fmaxf(mx, st[c].x);
        mx = wave_max_range<1, 2>(mx);
        for (int c = part; c < chunks; c += 4)
          if (st[c].y != 0.f) sum += st[c].y * __builtin_amdgcn_exp2f(st[c].x - mx);
        sum = wave_sum_range<1, 2>(sum);
      }
      if (mi < n && part == 0) {
        // a row that sees no token adds nothing
        s_max[mi] = mx == -INFINITY ? 0.f : mx;
        s_inv[mi] = sum == 0.f ? 0.f : 1.f / sum;
      }
    }
    __syncthreads();
    if (t < L) {
      for (int mi = 0; mi < n; ++mi) {
        const int m = m0 + mi, r = m / group;
        const float4 l = *reinterpret_cast<const float4*>(
            logits + ((rows.first + r) * a.num_heads + j * group + (m - r * group)) * ctx_pad + t);
        const float mx = s_max[mi], inv = s_inv[mi];
        acc[0] += l.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l.x - mx) * inv;
        acc[1] += l.y == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l.y - mx) * inv;
        acc[2] += l.z == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l.z - mx) * inv;
        acc[3] += l.w == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(l.w - mx) * inv;
      }
    }
  }
  float* out = a.scores + s * a.score_seq_stride + j * a.score_head_stride + t;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t + i < L) out[i] += acc[i];
}

struct Layout {
  int64_t rows;  // (query row, head) pairs
  int32_t ctx_pad, max_chunks;
  size_t stats_at, bytes;
};
Layout layout(int64_t total_rows, int32_t num_heads, int32_t max_ctx) {
  Layout l;
  l.rows = total_rows * num_heads;
  l.max_chunks = std::max(1, (max_ctx + kChunk - 1) / kChunk);
  l.ctx_pad = l.max_chunks * kChunk;
  l.stats_at = (size_t)l.rows * l.ctx_pad * sizeof(float);
  l.bytes = l.stats_at + (size_t)l.rows * l.max_chunks * sizeof(float2);
  return l;
}

template <typename T, typename C, int D>
void logits_launch(const WeightsArgs& a, const CacheGeom& g, const Layout& l, hipStream_t stream) {
  const int group = a.num_heads / g.num_kv_heads;
  const int64_t rgs = ((int64_t)a.max_query_len * group + 15) / 16;
  const dim3 grid((uint32_t)(g.num_kv_heads * l.max_chunks * rgs), (uint32_t)a.num_seqs);
  float* logits = static_cast<float*>(a.workspace);
  float2* stats = reinterpret_cast<float2*>(static_cast<char*>(a.workspace) + l.stats_at);
  hipLaunchKernelGGL((weight_logits_kernel<T, C, D>), grid, dim3(kThreads), 0, stream, a,
                     g.num_kv_heads, __builtin_ctz((unsigned)g.block_size), g.num_blocks,
                     g.block_stride, g.head_stride, logits, stats, l.ctx_pad, l.max_chunks);
}

template <typename T, typename C>
hipError_t logits_typed(const WeightsArgs& a, const CacheGeom& g, const Layout& l,
                        hipStream_t stream) {
  switch (g.head_dim) {
    case 64: logits_launch<T, C, 64>(a, g, l, stream); break;
    case 96: logits_launch<T, C, 96>(a, g, l, stream); break;
    case 128: logits_launch<T, C, 128>(a, g, l, stream); break;
    case 192: logits_launch<T, C, 192>(a, g, l, stream); break;
    case 256: logits_launch<T, C, 256>(a, g, l, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace

size_t weights_workspace_bytes(int64_t total_rows, int32_t num_heads, int32_t max_ctx) {
  return layout(total_rows, num_heads, max_ctx).bytes;
}

hipError_t launch_attention_weights(int dtype, int cache_dtype, const WeightsArgs& a,
                                    const CacheGeom& g, hipStream_t stream) {
  const Layout l = layout(a.total_rows, a.num_heads, a.max_ctx);
  const bool fp8 = cache_dtype == VPA_DTYPE_FP8_E4M3;
  hipError_t e = hipErrorInvalidValue;
  switch (dtype) {
    case VPA_DTYPE_F32:
      e = fp8 ? logits_typed<float, fp8_t>(a, g, l, stream)
              : logits_typed<float, float>(a, g, l, stream);
      break;
    case VPA_DTYPE_F16:
      e = fp8 ? logits_typed<f16_t, fp8_t>(a, g, l, stream)
              : logits_typed<f16_t, f16_t>(a, g, l, stream);
      break;
    case VPA_DTYPE_BF16:
      e = fp8 ? logits_typed<bf16_t, fp8_t>(a, g, l, stream)
              : logits_typed<bf16_t, bf16_t>(a, g, l, stream);
      break;
  }
  if (e != hipSuccess) return e;
  const float* logits = static_cast<const float*>(a.workspace);
  const float2* stats =
      reinterpret_cast<const float2*>(static_cast<const char*>(a.workspace) + l.stats_at);
  hipLaunchKernelGGL(weight_sum_kernel,
                     dim3((uint32_t)((l.ctx_pad + 1023) / 1024), (uint32_t)g.num_kv_heads,
                          (uint32_t)a.num_seqs),
                     dim3(kThreads), 0, stream, a, g.num_kv_heads, g.block_size, logits, stats,
                     l.ctx_pad, l.max_chunks);
  return hipGetLastError();
}

}  // namespace vpa
