// Logits made ready for the choice of a token, in place (gfx950): penalties for
// tokens that occurred, biases, and the tokens that a grammar allows.
//
// Row r of sequence b (draft i's rows see drafts 0 .. i - 1 besides the generated
// tokens). For a token v with c occurrences among those:
//   x = c > 0 or v in the prompt: x > 0 ? x / repetition : x * repetition
//   x -= frequency * c;  x -= presence where c > 0;  x += bias(v)
//   x = -inf where the row's mask does not allow v
// in f32, rounded once. Everything but the mask touches few of a row's logits, and
// eight masked neighbours are written without being read, so the floor is the
// token lists, the touched logits and the masked ones written (a mask that changes
// from token to token has all of the row read and written); without a mask nothing
// sweeps the vocabulary.
//
// A workgroup owns a range of a row's tokens: it counts the listed tokens of its
// range in LDS, sweeps the range with the mask, 16 bytes of logits at a time, and
// then settles the listed tokens that the mask allows, after its own sweep's stores.
// Few rows are cut into several ranges. The counts are kept in a hash table where the
// lists fit one (kHash; their capacity bounds its load to 3/4), else in an array over
// a range of the vocabulary, of which only the listed entries are cleared. A word per
// token holds its count, whether it is in the prompt and which bias it has; integers,
// so the order of atomics does not show.
//
// 256 rows of 151936 bf16 logits, masks that leave every other token out: 29 us, 155 MB
// read and written (5.3 TB/s; 33 us with workgroups of 512; 47 with workgroups for the
// sweep and others for the lists of a row). Masked elements stored one by one, without
// reading their neighbours: 43 us. The sweep's first loads issued before the lists are
// counted: no difference. One row without a mask: 6 us, the chain of its lists' loads.

#include <algorithm>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kAdjustThreads = 1024;
constexpr uint32_t kCountMask = (1u << 20) - 1;  // occurrences
constexpr uint32_t kInPrompt = 1u << 20;
constexpr int kBiasShift = 21;      // entry + 1, at most kAdjustMaxBias
constexpr int kDirectTokens = 32768;  // vocabulary part of a workgroup without a hash table
constexpr uint32_t kEmpty = 0xffffffffu;
constexpr int kRangeTokens = 4096;  // least range of a workgroup that sweeps

template <typename T>
struct AdjustRow {
  T* x;
  const uint32_t* mask;  // or null
};
template <typename T>
__device__ __forceinline__ AdjustRow<T> adjust_row(const AdjustArgs& a, int b, int i) {
  const uint32_t row = (uint32_t)b * (uint32_t)a.rows_per_seq + (uint32_t)i;
  const uint32_t* mask = nullptr;
  if (a.allowed != nullptr) {
    const uint32_t k = a.allowed_rows != nullptr ? a.allowed_rows[row] : row;
    if (k < (uint32_t)a.num_masks) mask = a.allowed + (int64_t)k * a.allowed_stride;
  }
  return {static_cast<T*>(a.logits) + b * a.seq_stride + i * a.row_stride, mask};
}

// -inf to the tokens lo .. hi - 1 of a row that its mask leaves out, 8 tokens at a
// time; lo is 0 or a 16-byte boundary of the row.
template <typename T>
__device__ void sweep_mask(const AdjustRow<T>& r, int vocab, int lo, int hi) {
  constexpr int kVec = 8 * sizeof(T) / 16;  // 16-byte vectors of 8 tokens
  T low;
  store_from_f32<T>(&low, -INFINITY);
  uint32_t pair;  // 4 bytes of -inf
  if constexpr (sizeof(T) == 4) pair = 0xff800000u;
  else pair = pack2<T>(-INFINITY, -INFINITY);
  auto bits_at = [&](int t) -> uint32_t {  // of tokens t .. t + 7; past the vocabulary: allowed
    const int w = t >> 5, sh = t & 31;
    const uint32_t a = r.mask[w], b = sh > 24 && 32 * (w + 1) < vocab ? r.mask[w + 1] : 0u;
    const uint32_t v = (uint32_t)((((uint64_t)b << 32) | a) >> sh) & 0xffu;
    const int left = hi - t;
    return left < 8 ? (v | (0xffu << left)) & 0xffu : v;
  };
  int first = lo;
  if (lo == 0) {  // up to the row's first boundary, token by token
    first = min((int)(((16 - ((uintptr_t)r.x & 15)) & 15) / sizeof(T)), hi);
    const int t = threadIdx.x;
    if (t < first && !((r.mask[t >> 5] >> (t & 31)) & 1u)) r.x[t] = low;
  }
  constexpr int U = 4;  // of 8 tokens, under way together
  for (int t0 = first + 8 * (int)threadIdx.x; t0 < hi; t0 += 8 * U * kAdjustThreads) {
    uint32_t bits[U];
    uint4 v[U][kVec];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 8 * u * kAdjustThreads;
      bits[u] = t < hi ? bits_at(t) : 0xffu;
      const uint4* src = reinterpret_cast<const uint4*>(r.x + t);
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        v[u][k] = bits[u] != 0u && bits[u] != 0xffu && t + 8 <= hi
                      ? src[k]
                      : make_uint4(pair, pair, pair, pair);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + 8 * u * kAdjustThreads;
      if (bits[u] == 0xffu) continue;
      if (t + 8 > hi) {
        for (int e = 0; e < hi - t; ++e)
          if (!((bits[u] >> e) & 1u)) r.x[t + e] = low;
        continue;
      }
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        uint32_t w[4] = {v[u][k].x, v[u][k].y, v[u][k].z, v[u][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            w[e] = (bits[u] >> (4 * k + e)) & 1u ? w[e] : pair;
          } else {
            const uint32_t two = bits[u] >> (2 * e);
            const uint32_t keep = (two & 1u ? 0xffffu : 0u) | (two & 2u ? 0xffff0000u : 0u);
            w[e] = (w[e] & keep) | (pair & ~keep);
          }
        }
        reinterpret_cast<uint4*>(r.x + t)[k] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <typename T, bool kHash>
__global__ __launch_bounds__(kAdjustThreads) void adjust_logits_kernel(const AdjustArgs a,
                                                                       int32_t range,
                                                                       int32_t table) {
  extern __shared__ uint32_t s_words[];  // [table] (kHash: and [table] tokens)
  uint32_t* const s_keys = s_words + table;
  const int tid = threadIdx.x;
  // rows vary fastest: a row's ranges lie rows apart
  const uint32_t rows = (uint32_t)a.num_seqs * (uint32_t)a.rows_per_seq;
  const uint32_t row = blockIdx.x % rows;
  const int part = (int)(blockIdx.x / rows);
  const int b = (int)(row / (uint32_t)a.rows_per_seq), i = (int)(row % (uint32_t)a.rows_per_seq);
  const AdjustRow<T> r = adjust_row<T>(a, b, i);
  // tokens v0 .. v1 - 1: ranges begin at 16-byte boundaries of the row
  const uint32_t shift = (uint32_t)(((16 - ((uintptr_t)r.x & 15)) & 15) / sizeof(T));
  const uint32_t v0 = part == 0 ? 0u : min((uint32_t)a.vocab, (uint32_t)part * range + shift);
  const uint32_t v1 = min((uint32_t)a.vocab, (uint32_t)(part + 1) * range + shift);
  const bool penal = a.repetition != nullptr || a.presence != nullptr || a.frequency != nullptr;
  const int n_gen =
      penal && a.generated != nullptr
          ? (int)min(a.gen_len != nullptr ? a.gen_len[b] : (uint32_t)a.generated_stride,
                     (uint32_t)a.generated_stride)
          : 0;
  const int n_draft = penal && a.draft_ids != nullptr ? i : 0;
  const int n_prompt =
      a.repetition != nullptr && a.prompt != nullptr
          ? (int)min(a.prompt_len != nullptr ? a.prompt_len[b] : (uint32_t)a.prompt_stride,
                     (uint32_t)a.prompt_stride)
          : 0;
  const int n_bias =
      a.bias_ids == nullptr
          ? 0
          : (int)min(a.bias_len != nullptr ? a.bias_len[b] : (uint32_t)a.bias_stride,
                     (uint32_t)a.bias_stride);
  const uint32_t* gen = a.generated + (int64_t)b * a.generated_stride;
  const uint32_t* draft = a.draft_ids + (int64_t)b * (a.rows_per_seq - 1);
  const uint32_t* prompt = a.prompt + (int64_t)b * a.prompt_stride;
  const uint32_t* bias_ids = a.bias_ids + (int64_t)b * a.bias_stride;
  // the word of token t; the table has room for every listed token
  auto find = [&](uint32_t t) -> uint32_t* {
    if constexpr (kHash) {
      uint32_t at = (t * 2654435761u) >> 7;
      for (;; ++at) {
        at &= (uint32_t)table - 1u;
        // (read first: many lanes may look for one token)
        uint32_t key = s_keys[at];
        if (key == kEmpty) key = atomicCAS(&s_keys[at], kEmpty, t);
        if (key == kEmpty || key == t) return &s_words[at];
      }
    } else {
      return &s_words[t - v0];
    }
  };
  auto each = [&](const uint32_t* list, int n, auto&& body) {
    for (int k = tid; k < n; k += kAdjustThreads) {
      const uint32_t t = list[k];
      if (t >= v0 && t < v1) body(t, k);
    }
  };
  if constexpr (kHash) {
    for (int k = tid; k < table; k += kAdjustThreads) {
      s_words[k] = 0u;
      s_keys[k] = kEmpty;
    }
  } else {
    auto clear = [&](uint32_t t, int) { s_words[t - v0] = 0u; };
    each(gen, n_gen, clear);
    each(draft, n_draft, clear);
    each(prompt, n_prompt, clear);
    each(bias_ids, n_bias, clear);
  }
  __syncthreads();
  auto count = [&](uint32_t t, int) { atomicAdd(find(t), 1u); };
  each(gen, n_gen, count);
  each(draft, n_draft, count);
  each(prompt, n_prompt, [&](uint32_t t, int) {
    uint32_t* w = find(t);
    if (!(*w & kInPrompt)) atomicOr(w, kInPrompt);  // (a placeholder fills most of a prompt)
  });
  __syncthreads();
  if (n_bias > 0) {
    // (the lower bits stand still here: the last entry of a token is the maximum)
    each(bias_ids, n_bias, [&](uint32_t t, int k) {
      uint32_t* w = find(t);
      const uint32_t low = *w & ((1u << kBiasShift) - 1u);
      atomicMax(w, ((uint32_t)(k + 1) << kBiasShift) | low);
    });
    __syncthreads();
  }
  if (r.mask != nullptr) {
    sweep_mask<T>(r, a.vocab, (int)v0, (int)v1);
    // the sweep's stores are done before a listed token of the same vector is stored
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  }
  const float rep = a.repetition != nullptr ? a.repetition[b] : 1.f;
  const float pres = a.presence != nullptr ? a.presence[b] : 0.f;
  const float freq = a.frequency != nullptr ? a.frequency[b] : 0.f;
  auto settle = [&](uint32_t t, uint32_t w) {
    if (r.mask != nullptr && !((r.mask[t >> 5] >> (t & 31)) & 1u)) return;
    float x = load_as_f32(r.x + t);
    const uint32_t c = w & kCountMask;
    if (a.repetition != nullptr && (c > 0 || (w & kInPrompt))) x = x > 0.f ? x / rep : x * rep;
    if (c > 0) {
      x -= freq * (float)c;
      x -= pres;
    }
    const uint32_t e = w >> kBiasShift;
    if (e > 0) x += a.bias[(int64_t)b * a.bias_stride + (e - 1)];
    store_from_f32<T>(r.x + t, x);
  };
  if constexpr (kHash) {
    for (int k = tid; k < table; k += kAdjustThreads) {
      const uint32_t t = s_keys[k];
      if (t != kEmpty) settle(t, s_words[k]);
    }
  } else {
    // the first lane that takes a token's word settles it
    auto take = [&](uint32_t t, int) {
      const uint32_t w = atomicExch(&s_words[t - v0], 0u);
      if (w != 0u) settle(t, w);
    };
    each(gen, n_gen, take);
    each(draft, n_draft, take);
    each(prompt, n_prompt, take);
    each(bias_ids, n_bias, take);
  }
}

template <typename T>
hipError_t launch_adjust(const AdjustArgs& a, hipStream_t stream) {
  const bool penal = a.repetition != nullptr || a.presence != nullptr || a.frequency != nullptr;
  int64_t listed = 0;
  if (penal && a.generated != nullptr) listed += a.generated_stride;
  if (penal && a.draft_ids != nullptr) listed += a.rows_per_seq - 1;
  if (a.repetition != nullptr && a.prompt != nullptr) listed += a.prompt_stride;
  if (a.bias_ids != nullptr) listed += a.bias_stride;
  const int64_t rows = (int64_t)a.num_seqs * a.rows_per_seq;
  if (listed == 0 && a.allowed == nullptr) return hipSuccess;
  // a table of 8 bytes per place, at most 128 KiB of the compute unit's 160
  int table = 256;
  while (table < 32768 && (int64_t)table * 3 / 4 < listed) table *= 2;
  const bool hash = table <= 16384;
  // one range per row, or where there is something to sweep about 512 workgroups; an
  // array holds a range's words and those before its first boundary
  int64_t parts = 1;
  if (a.allowed != nullptr) {
    parts = (512 + rows - 1) / rows;
    parts = std::max<int64_t>(
        1, std::min<int64_t>(parts, (a.vocab + kRangeTokens - 1) / kRangeTokens));
  }
  const int64_t most = hash ? ((int64_t)1 << 30) : kDirectTokens - 8;
  parts = std::max(parts, (a.vocab + most - 1) / most);
  const int range = (int)(((a.vocab + parts - 1) / parts + 7) / 8 * 8);
  const dim3 grid((unsigned)(rows * parts));
  if (hash)
    hipLaunchKernelGGL((adjust_logits_kernel<T, true>), grid, dim3(kAdjustThreads),
                       (size_t)table * 8, stream, a, range, table);
  else
    hipLaunchKernelGGL((adjust_logits_kernel<T, false>), grid, dim3(kAdjustThreads),
                       (size_t)kDirectTokens * 4, stream, a, range, kDirectTokens);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_adjust_logits(int dtype, const AdjustArgs& a, hipStream_t stream) {
  switch (dtype) {
    case VPA_DTYPE_BF16:
      return launch_adjust<bf16_t>(a, stream);
    case VPA_DTYPE_F16:
      return launch_adjust<f16_t>(a, stream);
    default:
      return launch_adjust<float>(a, stream);
  }
}

}  // namespace vpa
