// Attention over a paged cache of E4M3 bytes with one scale per (block, kv
// head), for K and for V (gfx950 MFMA). One kernel serves a decode step, drafted
// tokens and the rows of a prompt; the files that include it hold its instances
// for one query type each.
//
// For query row r, its sequence's cached tokens t and their block b(t):
//   s_t = softmax_scale * ks[b(t)] * (q_r . K_t)       K_t, V_t: the bytes' values
//   out = sum_t p_t vs[b(t)] V_t / (sum_t p_t + eps),  p_t = exp(s_t - max_t s_t)
// over the tokens the row sees. Scales that are powers of two, as the append
// makes them, cost nothing: the conversion of the bytes for the matrix
// instructions takes a power of two along, here a block's scale over the largest
// of the step's (K) or of those met so far (V: `vrow`), so that no operand passes
// 448; that largest one is part of the softmax scale and of the output. Every
// product is exact as long as the ratio is at least 2^-5 (E4M3's least number,
// 2^-9, stays normal in f16). Steps with smaller ratios or other scales multiply
// the f32 scores and probabilities instead. V's reference is then the largest scale that
// the row itself sees: blocks that it does not see, louder by any factor, do not push its
// weights p_t vs_t / vrow out of f16's range.
//
// Work of a wave: 16 NQ rows (a row is a position and a query head of the kv
// head; heads fastest, so any group size fills the rows) over 64 keys at a time
// = 4 tiles of 16 keys. S^T = K Q^T with v_mfma_f32_16x16x32: lane l gives token
// l % 16 of a tile and, as K's 16-byte vectors hold 16 dims of a token, the dims
// 16 (l / 16) + 64 i .. + 15, one load for two k-steps; Q is loaded in the same
// order. The result holds, per lane, column (row of Q) l % 16 and tokens
// 4 (l / 16) .. + 3 of each tile. O^T += V^T P^T takes V's rows as they lie:
// lane l holds dim l % 16 and the 16 tokens of tile l / 16, which are two
// k-steps of 8. P^T has to follow: lane row g needs tile g's 16 tokens where it
// has 4 tokens of each tile, a transposition of 4 x 4 registers by lane rows,
// eight v_permlane swaps for 64 keys. So no value of K, V or P goes through LDS
// and the waves run without barriers; LDS only joins the waves' results at the end.
//
// Precision: scores, softmax and sums are f32. P goes through the matrix
// instructions as f16 (V's bytes are exact in f16 whatever the query's type):
// rounded to 11 bits, off by at most 2^-11 of itself; f32 queries use two f16
// values (22 bits), and three bf16 values for Q, which hold an f32 exactly. The
// probabilities stay below 2^kSlack (the reference maximum moves only when it is
// exceeded by more) and are scaled by 2^kProbLog2, which keeps f16's smallest
// step at 2^-31 of a probability of 1. Like the maximum, vrow moving rescales the
// sums.
//
// Few rows (decode): the waves of a workgroup split a chunk's keys, 64 at a time,
// and are joined in LDS; long contexts are split in chunks over workgroups and
// joined by a second launch (scaled_merge_kernel). Many rows: a workgroup is one
// wave with its own rows, and all of them read the same keys, through L1 and L2.
//
// Bounds, with 16 query and 8 kv heads of 128 dims: a decode of 256 sequences of 800 to
// 4096 tokens by HBM (77 us, 5.3 TB/s; a read-only kernel reaches as much); one of 1500
// tokens by its two launches and their dependent loads (8.0 us, 6.0 + 2.4 on their own);
// rows of prompts by the issue of vector instructions, about 470 beside 64 matrix
// instructions for 32 rows and 64 keys (512 rows each of 64 prompts of 560 to 1600 tokens:
// 347 us, 691 TFLOP/s; matrix units busy 31 % of the time, vector issue 71 %). There the
// next operands' bytes are converted between the matrix instructions (1 to 5 % of a
// prompt's time); without any conversion the same call takes 12 % less, without
// exponentials 7 %, without loads 5 %. A reference of V's scales per row costs such calls
// 1 to 4 %, a decode nothing. Not kept: 8 waves that split the keys (97 us for the
// 256 sequences).
#pragma once

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

typedef __bf16 sa_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 sa_f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <typename K>
__device__ __forceinline__ f32x4_t mfma16x16x32(const uint4& a, const uint4& b, const f32x4_t& c) {
  if constexpr (std::is_same_v<K, f16_t>)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sa_f16x8, a),
                                                  __builtin_bit_cast(sa_f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sa_bf16x8, a),
                                                   __builtin_bit_cast(sa_bf16x8, b), c, 0, 0, 0);
}

// Sixteen E4M3 bytes times a power of two (f32; the two halves' own) -> sixteen
// values of K in two operands.
template <typename K>
__device__ __forceinline__ void fp8x16_times(const uint4& v, float slo, float shi, uint4& lo,
                                             uint4& hi) {
  auto cvt = [](uint32_t w, float s, auto half) -> uint32_t {
    constexpr bool h = decltype(half)::value;
    if constexpr (std::is_same_v<K, f16_t>)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, h));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, h));
  };
  constexpr std::false_type l{};
  constexpr std::true_type h{};
  lo = make_uint4(cvt(v.x, slo, l), cvt(v.x, slo, h), cvt(v.y, slo, l), cvt(v.y, slo, h));
  hi = make_uint4(cvt(v.z, shi, l), cvt(v.z, shi, h), cvt(v.w, shi, l), cvt(v.w, shi, h));
}

// Four times: a matrix instruction, then two vector instructions in its shadow.
__device__ __forceinline__ void alternate() {
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
  }
}

constexpr int kScaledWaves = 4;  // of a workgroup that splits the keys
constexpr int kScaledKeys = 64;  // keys of a step
constexpr float kScaledSlack = 8.f;
constexpr int kScaledProbLog2 = 7;
// How far above a row's own the wave's reference of V's scales is taken for it where the
// conversion takes the ratios along, exactly.
constexpr float kScaledReach = 32.f;

// Maximum / sum over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float max_rows(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_rows(float v) { return sum_xor32(sum_xor16(v)); }

// w[b] of lane row g -> w[g] of lane row b (4 x 4, by lane rows).
__device__ __forceinline__ void transpose_rows(uint32_t (&w)[4]) {
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[b], w[b + 2], false, false);
    w[b] = r[0];
    w[b + 2] = r[1];
  }
#pragma unroll
  for (int b = 0; b < 4; b += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[b], w[b + 1], false, false);
    w[b] = r[0];
    w[b + 1] = r[1];
  }
}

struct ScaledDev {
  const void* query;
  const uint8_t* key_cache;
  const uint8_t* value_cache;
  const float* key_scales;
  const float* value_scales;
  int64_t scale_block_stride;
  const uint32_t* block_tables;
  const uint32_t* cu_seqlens_q;
  const uint32_t* context_lens;
  void* out;
  float* part_out;   // [total rows * heads][max_chunks][D]
  float* part_stat;  // [total rows * heads][max_chunks][2]: maximum, sum
  int64_t block_stride, head_stride;  // bytes
  int64_t num_blocks, total_rows;
  int32_t block_table_stride, num_seqs, max_query_len, max_ctx;
  int32_t num_heads, num_kv_heads, group, causal;
  int32_t tiles, chunk_tokens, max_chunks;
  int32_t split_keys;  // the waves share 16 NQ rows and split the keys
  int32_t lds_rows;    // rows kept in LDS then
  float scale_log2, denom_eps;
};

// Query types whose waves may take two tiles of 16 rows. (f32 queries' parts leave no
// registers for a second one: 1000 rows of 8 prompts 200 us with one tile, 222 with two.)
template <typename T>
constexpr bool scaled_two_tiles() {
  return !std::is_same_v<T, float>;
}

// Waves per SIMD: O, Q and two tiles' bytes are what a wave holds. Two row tiles of head
// dims 192 and 256 fill it alone, and share each conversion: 512 rows each of 32 prompts
// of 1000 to 2000 tokens, calls of 192 / 256 dims, 450 / 512 us, 620 / 717 with one tile.
// (Four row tiles of head dim 128, alone too, are slower than two waves of two: 450 us
// for 340.) Head dim 64's two tiles fit three waves, in 168 registers.
template <typename T, int D, int BS, int NQ>
constexpr int scaled_waves_per_eu() {
  if (D == 64 && NQ == 2 && BS > 8) return 3;
  return D <= 128 || (D == 192 && NQ == 1 && !std::is_same_v<T, float>) ? 2 : 1;
}

template <typename T, int D, int BS, int NQ>
__global__ __launch_bounds__(64 * kScaledWaves)
__attribute__((amdgpu_waves_per_eu(scaled_waves_per_eu<T, D, BS, NQ>()))) void scaled_attention_kernel(
    const ScaledDev a) {
  constexpr bool kF32 = std::is_same_v<T, float>;
  using K = std::conditional_t<std::is_same_v<T, f16_t>, f16_t, bf16_t>;  // of S's operands
  constexpr int QP = kF32 ? 3 : 1;   // parts of Q
  constexpr int PP = kF32 ? 2 : 1;   // parts of P
  constexpr int NC = (D + 63) / 64;  // loads of a lane per 16-key tile of K
  constexpr int DT = D / 16;
  constexpr int CH = D / 16;  // 16-byte chunks of a key
  // Where a wave's registers hold two tiles' bytes besides its sums, V is under
  // way while S is computed and the next K during the softmax; otherwise V
  // during the softmax and the next K during P.V.
  constexpr bool kEarly = NQ == 1 && D <= 128;
  constexpr bool kLate = NQ == 2 && D == 256;  // where half of V's have been used

  extern __shared__ float s_join[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, kg = lane >> 4;
  // kv heads vary fastest, then a sequence's row tiles (the last, which see most
  // keys, first): workgroups that read the same keys are close and, at 8 kv heads,
  // on one XCD
  uint32_t w = blockIdx.x;
  const int j = (int)(w % (uint32_t)a.num_kv_heads);
  w /= (uint32_t)a.num_kv_heads;
  const int qt = a.tiles - 1 - (int)(w % (uint32_t)a.tiles);
  w /= (uint32_t)a.tiles;
  const int s = (int)(w % (uint32_t)a.num_seqs);
  const int chunk = (int)(w / (uint32_t)a.num_seqs);

  uint32_t qa = (uint32_t)s, qb = (uint32_t)s + 1u;
  if (a.cu_seqlens_q != nullptr) {
    qa = a.cu_seqlens_q[s];
    qb = a.cu_seqlens_q[s + 1];
  }
  int n = qb > qa ? (int)min(qb - qa, (uint32_t)a.max_query_len) : 0;
  n = (int64_t)qa >= a.total_rows ? 0 : (int)min((int64_t)n, a.total_rows - (int64_t)qa);
  const int L = (int)min(a.context_lens[s], (uint32_t)a.max_ctx);
  const int rows = n * a.group;
  const int r0 = qt * 16 * NQ;
  if (r0 >= rows) return;  // (uniform over the workgroup)
  const int nchunks = max(1, (L + a.chunk_tokens - 1) / a.chunk_tokens);
  if (chunk >= nchunks) return;

  // keys that some row of the wave sees, and the part of them here
  const int shift = L - n;
  const int last_pos = (min(r0 + 16 * NQ, rows) - 1) / a.group;
  int n_keys = a.causal ? min(L, last_pos + shift + 1) : L;
  n_keys = max(n_keys, 0);
  const int k_end = min(n_keys, (chunk + 1) * a.chunk_tokens);
  const int k_step = a.split_keys ? kScaledKeys * kScaledWaves : kScaledKeys;
  const int k_first = chunk * a.chunk_tokens + (a.split_keys ? wave * kScaledKeys : 0);
  // the last key that every row of the wave sees
  const int all_see = a.causal ? r0 / a.group + shift : L - 1;

  int limit[NQ];  // last key of this lane's rows (the lane's column of S^T)
  int64_t orow[NQ];  // their row of `out`
  uint4 qop[NQ][QP][2 * NC];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r = r0 + 16 * q + c16;
    const bool ok = r < rows;
    const int pos = ok ? r / a.group : 0;
    const int64_t row = ((int64_t)qa + pos) * a.num_heads + (int64_t)j * a.group + (ok ? r % a.group : 0);
    orow[q] = row;
    limit[q] = !ok ? -1 : a.causal ? pos + shift : L - 1;
    const T* src = static_cast<const T*>(a.query) + row * D;
#pragma unroll
    for (int st = 0; st < 2 * NC; ++st) {
      const int dim = 16 * (kg + 4 * (st / 2)) + 8 * (st % 2);
      const bool in = dim < D;  // (head dim 96 ends inside a step: zeros)
      if constexpr (kF32) {
        uint32_t part[3][4];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 v = in ? *reinterpret_cast<const float4*>(src + dim + e)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
          float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int p = 0; p < 3; ++p) {
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
              const uint32_t pk = pack2_hw<bf16_t>(x[h], x[h + 1]);
              part[p][(e + h) / 2] = pk;
              x[h] -= low_half_f32<bf16_t>(pk);
              x[h + 1] -= high_half_f32<bf16_t>(pk);
            }
          }
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
          qop[q][p][st] = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
      } else {
        qop[q][0][st] = in ? *reinterpret_cast<const uint4*>(src + dim) : make_uint4(0, 0, 0, 0);
      }
    }
  }

  f32x4_t o[NQ][DT];
  float kref = 1.f;
  float m[NQ], mt[NQ], lsum[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    m[q] = mt[q] = -INFINITY;
    lsum[q] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[q][dt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // V's reference: the largest scale that a row has seen or, where the conversion takes the
  // ratio along, the largest of all that the wave's steps held. Rows of a wave differ in it
  // only where the wave is `apart`.
  float vrow[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) vrow[q] = 1.50463277e-36f;  // 2^-119 (over 2^kScaledProbLog2 normal)
  constexpr int kApart = 1, kNan = 2;
  int state = 0;  // (uniform)

  if (k_first < k_end) {
    const uint32_t* bt = a.block_tables + (int64_t)s * a.block_table_stride;
    const int last_blk = (L - 1) / BS;
    const uint8_t* kbase = a.key_cache + (int64_t)j * a.head_stride;
    const uint8_t* vbase = a.value_cache + (int64_t)j * a.head_stride;
    constexpr int NI = BS == 8 ? 2 : 1;  // blocks of a 16-key tile

    // Ids of this lane row's tile (tile kg of the step; clamped to the last block).
    struct Ids {
      uint32_t id[NI];
    };
    auto load_ids = [&](int k0) {
      Ids r;
#pragma unroll
      for (int i = 0; i < NI; ++i) r.id[i] = bt[min((k0 + 16 * kg + 8 * i) / BS, last_blk)];
      return r;
    };
    // Scales of that tile; 0 for an absent block's.
    struct Scales {
      float k[NI], v[NI];
    };
    const uint32_t max_id = (uint32_t)min(a.num_blocks - 1, (int64_t)0xffffffff);
    auto present = [&](uint32_t id) { return id <= max_id; };
    auto load_scales = [&](const Ids& d) {
      Scales r;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const bool ok = present(d.id[i]);
        const int64_t at = (int64_t)(ok ? d.id[i] : 0u) * a.scale_block_stride + j;
        const float ks = a.key_scales[at], vs = a.value_scales[at];
        r.k[i] = ok ? ks : 0.f;
        r.v[i] = ok ? vs : 0.f;
      }
      return r;
    };
    auto load16 = [](const uint8_t* p) {
      if constexpr (NQ == 1) return load_stream(reinterpret_cast<const uint4*>(p));
      else return *reinterpret_cast<const uint4*>(p);
    };
    // absent blocks read block 0 (in bounds) and are masked
    auto load_k = [&](const Ids& d, uint4 (&buf)[4][NC]) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t id0 = (uint32_t)__builtin_amdgcn_readlane((int)d.id[0], 16 * b);
        int64_t at = (int64_t)(present(id0) ? id0 : 0u) * a.block_stride;
        if constexpr (NI == 2) {
          const uint32_t id1 = (uint32_t)__builtin_amdgcn_readlane((int)d.id[1], 16 * b);
          const int64_t at1 = (int64_t)(present(id1) ? id1 : 0u) * a.block_stride;
          at = c16 < 8 ? at : at1;
        }
        const int off = BS == 8 ? (c16 & 7) : BS == 16 ? c16 : 16 * (b & 1) + c16;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int c = kg + 4 * i;
          buf[b][i] = load16(kbase + at + ((c < CH ? c : kg) * BS + off) * 16);
        }
      }
    };
    auto load_v = [&](const Ids& d, uint4 (&buf)[DT]) {
      const uint8_t* p[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i)
        p[i] = vbase + (int64_t)(present(d.id[i]) ? d.id[i] : 0u) * a.block_stride + c16 * BS +
               (BS == 32 ? 16 * (kg & 1) : 0);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if constexpr (NI == 2) {
          const uint2 lo = *reinterpret_cast<const uint2*>(p[0] + dt * 16 * BS);
          const uint2 hi = *reinterpret_cast<const uint2*>(p[1] + dt * 16 * BS);
          buf[dt] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          buf[dt] = load16(p[0] + dt * 16 * BS);
        }
      }
    };

    // x of tile b's tokens, the second of its blocks where `second`. (Both lanes are read by
    // the whole wave: under a branch of some lanes the one read might not be written.)
    auto of_tile = [](const float(&x)[NI], int b, bool second) {
      const float lo = readlane_f(x[0], 16 * b);
      if constexpr (NI == 2) {
        const float hi = readlane_f(x[1], 16 * b);
        return second ? hi : lo;
      }
      return lo;
    };

    // Bytes of tokens past the context or in an absent block are stale, NaN among
    // them, and 0 * NaN is NaN: zeros.
    struct Keep {
      uint32_t x[4];
    };
    auto keep_of = [&](const Ids& d, int k0) {
      Keep r;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int left = present(d.id[NI == 2 ? x / 2 : 0]) ? L - (k0 + 16 * kg + 4 * x) : 0;
        r.x[x] = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
      }
      return r;
    };
    auto kept = [](const uint4& v, const Keep& k) {
      return make_uint4(v.x & k.x[0], v.y & k.x[1], v.z & k.x[2], v.w & k.x[3]);
    };
    // 1 in each byte that is NaN
    auto nan_bytes = [](uint32_t x) {
      return (((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
    };
    uint4 kraw[4][NC], vraw[DT];
    Ids ids = load_ids(k_first), ids1 = load_ids(k_first + k_step);
    Scales sc = load_scales(ids);
    load_k(ids, kraw);

    for (int k0 = k_first; k0 < k_end; k0 += k_step) {
      if constexpr (kEarly) load_v(ids, vraw);
      const Ids ids2 = load_ids(k0 + 2 * k_step);
      const Scales sc1 = load_scales(ids1);

      // ---- scales ----
      // x over a power of two `ref`; both are powers of two, 2^-5 ref <= x <= ref
      auto ratio = [](float x, float ref) {
        return __uint_as_float(__float_as_uint(x) - __float_as_uint(ref) + 0x3f800000u);
      };
      auto plain = [](float x, float ref) {
        return ((__float_as_uint(x) | __float_as_uint(ref)) & 0x7fffffu) == 0 &&
               x >= ref * 0.03125f && x <= ref;
      };
      auto all_plain = [&](const float(&x)[NI], float ref) {
        bool odd = !plain(x[0], ref);
        if constexpr (NI == 2) odd = odd || !plain(x[1], ref);
        return __ballot(odd) == 0;  // (uniform)
      };
      auto largest = [&](const float(&x)[NI]) {
        float v = fabsf(x[0]);
        if constexpr (NI == 2) v = fmaxf(v, fabsf(x[1]));
        return max_rows(v);
      };
      bool kfast = all_plain(sc.k, kref);
      if (!kfast) {  // (rare where scales are powers of two of one size)
        kref = largest(sc.k);
        kfast = all_plain(sc.k, kref);
      }
      kfast = kfast && kref * a.scale_log2 > 0.f;  // (a maximum goes through the scale)
      const float fs = kfast ? kref * a.scale_log2 : 1.f;
      float kr[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) kr[i] = kfast ? ratio(sc.k[i], kref) : 1.f;

      // ---- S^T, 64 dims of a tile at a time, the next ones' bytes converted meanwhile ----
      f32x4_t sv[NQ][4];
      auto tile_ratio = [&](int b) { return of_tile(kr, b, c16 >= 8); };
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int q = 0; q < NQ; ++q) sv[q][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      uint4 kop[2][2];
      {
        const float krb = tile_ratio(0);
        fp8x16_times<K>(kraw[0][0], krb, krb, kop[0][0], kop[0][1]);
      }
#pragma unroll
      for (int t = 0; t < 4 * NC; ++t) {
        if constexpr (!kEarly) __builtin_amdgcn_sched_barrier(0);
        if (t + 1 < 4 * NC) {
          const float krb = tile_ratio((t + 1) / NC);
          fp8x16_times<K>(kraw[(t + 1) / NC][(t + 1) % NC], krb, krb, kop[(t + 1) % 2][0],
                          kop[(t + 1) % 2][1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int p = QP - 1; p >= 0; --p)
              sv[q][t / NC] =
                  mfma16x16x32<K>(kop[t % 2][h], qop[q][p][2 * (t % NC) + h], sv[q][t / NC]);
        if constexpr (NQ == 2) alternate();
      }
      if constexpr (kEarly) {
        if (k0 + k_step < k_end) load_k(ids1, kraw);
      } else {
        __builtin_amdgcn_sched_barrier(0);
        load_v(ids, vraw);
      }

      // ---- other scales, masks ----
      if (!kfast) {
        asm volatile("" ::: "memory");  // (a branch, not selects)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const float ksb = of_tile(sc.k, b, kg >= 2) * a.scale_log2;
#pragma unroll
          for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[q][b][r] *= ksb;
        }
      }
      // every key inside the context, in a present block, seen by every row
      bool mine = present(ids.id[0]);
      if constexpr (NI == 2) mine = mine && present(ids.id[1]);
      const bool full = __ballot(!mine) == 0 && k0 + kScaledKeys <= min(L, all_see + 1);
      if (!full) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          bool here = present((uint32_t)__builtin_amdgcn_readlane((int)ids.id[0], 16 * b));
          if constexpr (NI == 2) {
            const bool h1 = present((uint32_t)__builtin_amdgcn_readlane((int)ids.id[1], 16 * b));
            here = kg < 2 ? here : h1;
          }
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            const int last = here ? limit[q] - (k0 + 16 * b + 4 * kg) : -1;
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[q][b][r] = r <= last ? sv[q][b][r] : -INFINITY;
          }
        }
      }

      // ---- online softmax ----
      // Each lane looks at its own 16 keys of a row; only where one passes the
      // reference maximum by more than the slack are the row's four lanes compared.
      float mx[NQ];
      bool move = false;
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        mx[q] = sv[q][0][0];
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx[q] = fmaxf(mx[q], sv[q][b][r]);
        mx[q] *= fs;
        mt[q] = fmaxf(mt[q], mx[q]);
        move = move || mx[q] > m[q] + kScaledSlack;  // (m is -inf before the first key)
      }
      // (a row that is apart sees nothing of the steps to come: it may look in vain)
      bool vmore = fabsf(sc.v[0]) > vrow[0];
      if constexpr (NI == 2) vmore = vmore || fabsf(sc.v[1]) > vrow[0];
      if (__ballot(move || vmore) != 0) {
        float fix[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float mn = fmaxf(m[q], max_rows(mx[q]));
          fix[q] = m[q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[q] - mn);
          m[q] = mn;
          lsum[q] *= fix[q];
        }
        if (__ballot(vmore) != 0) {
          float vref = fmaxf(fabsf(sc.v[0]), fabsf(sc.v[NI - 1]));
#pragma unroll
          for (int q = 0; q < NQ; ++q) vref = fmaxf(vref, vrow[q]);
          vref = wave_max_dpp(vref);
          const float reach = all_plain(sc.v, vref) ? kScaledReach : 1.f;
          bool off = false;
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            float seen = k0 + 16 * kg <= limit[q] ? fabsf(sc.v[0]) : 0.f;
            if constexpr (NI == 2)
              seen = fmaxf(seen, k0 + 16 * kg + 8 <= limit[q] ? fabsf(sc.v[1]) : 0.f);
            seen = fmaxf(vrow[q], max_rows(seen));
            // (a row that sees nothing at all takes any)
            const float to = limit[q] < k_first || seen * reach >= vref ? vref : seen;
            fix[q] *= vrow[q] / to;
            vrow[q] = to;
            off = off || to != vref;
          }
          state = (state & kNan) | (__ballot(off) != 0 ? kApart : 0);
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[q][dt][r] *= fix[q];
      }
      const bool vfast = all_plain(sc.v, vrow[0]) && (state & kApart) == 0;
      float vr[NI];
#pragma unroll
      for (int i = 0; i < NI; ++i) vr[i] = vfast ? ratio(sc.v[i], vrow[0]) : 1.f;

      // ---- probabilities, as operands of P.V ----
      uint32_t pw[NQ][PP][2][4];  // [two tokens of a tile's four][tile]
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const float mu = (m[q] == -INFINITY ? 0.f : m[q]) - (float)kScaledProbLog2;
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            sv[q][b][r] = __builtin_amdgcn_exp2f(fmaf(sv[q][b][r], fs, -mu));
            lsum[q] += sv[q][b][r];
          }
      }
      if (!vfast) {
        asm volatile("" ::: "memory");  // (a branch, and nothing of it before)
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          const float over = 1.f / vrow[q];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            // (of a block that the row does not see: perhaps infinite, times 0)
            const int t0 = k0 + 16 * b + (NI == 2 ? 8 * (kg / 2) : 0);
            const float vs = of_tile(sc.v, b, kg >= 2);
            const float f = t0 <= limit[q] ? vs * over : 0.f;
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[q][b][r] *= f;
          }
        }
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f32x4_t p = sv[q][b];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            pw[q][0][h][b] = pack2_hw<f16_t>(p[2 * h], p[2 * h + 1]);
            if constexpr (PP == 2)
              pw[q][1][h][b] = pack2_hw<f16_t>(p[2 * h] - low_half_f32<f16_t>(pw[q][0][h][b]),
                                               p[2 * h + 1] - high_half_f32<f16_t>(pw[q][0][h][b]));
          }
        }
#pragma unroll
        for (int p = 0; p < PP; ++p)
#pragma unroll
          for (int h = 0; h < 2; ++h) transpose_rows(pw[q][p][h]);
      }

      // ---- O^T += V^T P^T, the next dims' bytes converted meanwhile ----
      if (!full) {
        // A NaN value of a token that only later rows see would reach every row
        // of the tile through 0 * NaN: such bytes count as 0 here and are gone
        // through once more after the loop.
        const Keep keep = keep_of(ids, k0);
        uint32_t any = 0;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          __builtin_amdgcn_sched_barrier(0);
          vraw[dt] = kept(vraw[dt], keep);
          any |= nan_bytes(vraw[dt].x) | nan_bytes(vraw[dt].y) | nan_bytes(vraw[dt].z) |
                 nan_bytes(vraw[dt].w);
        }
        if (a.causal && __ballot(any != 0) != 0) {
          state |= kNan;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            __builtin_amdgcn_sched_barrier(0);
            vraw[dt].x &= ~(nan_bytes(vraw[dt].x) * 0xffu);
            vraw[dt].y &= ~(nan_bytes(vraw[dt].y) * 0xffu);
            vraw[dt].z &= ~(nan_bytes(vraw[dt].z) * 0xffu);
            vraw[dt].w &= ~(nan_bytes(vraw[dt].w) * 0xffu);
          }
        }
      }
      // (past the end too, where the clamped ids read one block once more: a branch here
      // costs the registers of a second copy of the bytes)
      if constexpr (!kEarly && !kLate) {
        __builtin_amdgcn_sched_barrier(0);
        load_k(ids1, kraw);
      }
      uint4 vop[2][2];
      fp8x16_times<f16_t>(vraw[0], vr[0], vr[NI - 1], vop[0][0], vop[0][1]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        if constexpr (!kEarly) __builtin_amdgcn_sched_barrier(0);
        if constexpr (kLate)
          if (dt == DT / 2) load_k(ids1, kraw);
        if (dt + 1 < DT)
          fp8x16_times<f16_t>(vraw[dt + 1], vr[0], vr[NI - 1], vop[(dt + 1) % 2][0],
                              vop[(dt + 1) % 2][1]);
#pragma unroll
        for (int p = PP - 1; p >= 0; --p)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < NQ; ++q)
              o[q][dt] = mfma16x16x32<f16_t>(
                  vop[dt % 2][h],
                  make_uint4(pw[q][p][0][2 * h], pw[q][p][1][2 * h], pw[q][p][0][2 * h + 1],
                             pw[q][p][1][2 * h + 1]),
                  o[q][dt]);
        if constexpr (NQ == 2) alternate();
      }
      ids = ids1;
      ids1 = ids2;
      sc = sc1;
    }

    // NaN values, which the steps that were not full left out (masked rows, the context's
    // end, an absent block; the other steps' come out the same): a row gets a NaN in each
    // dim where a token it sees has one, by a product of flags.
    if ((state & kNan) != 0) {
      for (int k0 = k_first; k0 < k_end; k0 += k_step) {
        ids = load_ids(k0);
        load_v(ids, vraw);
        const Keep keep = keep_of(ids, k0);
        uint32_t vis[NQ][2][4];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const int t = k0 + 16 * b + 4 * kg + 2 * h;
              vis[q][h][b] = (t <= limit[q] ? 0x3c00u : 0u) | (t < limit[q] ? 0x3c000000u : 0u);
            }
            transpose_rows(vis[q][h]);
          }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          __builtin_amdgcn_sched_barrier(0);
          const uint4 x = kept(vraw[dt], keep);
          uint4 op[2];
          fp8x16_to_pk<f16_t>(make_uint4(nan_bytes(x.x) * 0x38u, nan_bytes(x.y) * 0x38u,
                                         nan_bytes(x.z) * 0x38u, nan_bytes(x.w) * 0x38u),
                              op[0], op[1]);  // 0x38: 1.0
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            f32x4_t c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < 2; ++h)
              c = mfma16x16x32<f16_t>(op[h],
                                      make_uint4(vis[q][0][2 * h], vis[q][1][2 * h],
                                                 vis[q][0][2 * h + 1], vis[q][1][2 * h + 1]),
                                      c);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[q][dt][r] = c[r] > 0.f ? NAN : o[q][dt][r];
          }
        }
      }
    }
  }

  // ---- to the true maximum, then out: whole rows, a chunk's part, or joined ----
  float fo[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    mt[q] = max_rows(mt[q]);
    const float f = m[q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[q] - mt[q]);
    const float f1 = f * (1.f / (1 << kScaledProbLog2));
    lsum[q] = sum_rows(lsum[q]) * f1;
    fo[q] = f1 * vrow[q];
  }
  const bool single = nchunks == 1;
  T* out = static_cast<T*>(a.out);
  auto store4 = [&](int64_t row, int d, const float (&v)[4], float mx, float sum) {
    if (single) {
      const float inv = sum > 0.f || sum != sum ? 1.f / (sum + a.denom_eps) : 0.f;
      if constexpr (kF32) {
        *reinterpret_cast<float4*>(out + row * D + d) =
            make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      } else {
        *reinterpret_cast<uint2*>(out + row * D + d) =
            make_uint2(pack2_hw<T>(v[0] * inv, v[1] * inv), pack2_hw<T>(v[2] * inv, v[3] * inv));
      }
    } else {
      const int64_t at = row * a.max_chunks + chunk;
      *reinterpret_cast<float4*>(a.part_out + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) *reinterpret_cast<float2*>(a.part_stat + 2 * at) = make_float2(mx, sum);
    }
  };
  // (compared here: kept from above, each would hold a pair of registers over the loop)
  int split = a.split_keys, end = rows;
  asm volatile("" : "+s"(split), "+s"(end));
  if (split == 0) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      if (r0 + 16 * q + c16 >= end) continue;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const float v[4] = {o[q][dt][0] * fo[q], o[q][dt][1] * fo[q], o[q][dt][2] * fo[q],
                            o[q][dt][3] * fo[q]};
        store4(orow[q], 16 * dt + 4 * kg, v, mt[q], lsum[q]);
      }
    }
    return;
  }
  // [wave][row][D] sums, then [wave][row][2] maxima and sums
  const int nr = a.lds_rows;
  float* s_stat = s_join + kScaledWaves * nr * D;
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int r = 16 * q + c16;
    if (r >= nr) continue;
    float* dst = s_join + (wave * nr + r) * D + 4 * kg;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<float4*>(dst + 16 * dt) =
          make_float4(o[q][dt][0] * fo[q], o[q][dt][1] * fo[q], o[q][dt][2] * fo[q],
                      o[q][dt][3] * fo[q]);
    if (kg == 0) {
      s_stat[2 * (wave * nr + r)] = mt[q];
      s_stat[2 * (wave * nr + r) + 1] = lsum[q];
    }
  }
  __syncthreads();
  const int live = min(nr, rows - r0);
  for (int e = threadIdx.x; e < live * (D / 4); e += 64 * kScaledWaves) {
    const int r = e / (D / 4), d = 4 * (e % (D / 4));
    float mx = -INFINITY;
#pragma unroll
    for (int x = 0; x < kScaledWaves; ++x) mx = fmaxf(mx, s_stat[2 * (x * nr + r)]);
    float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < kScaledWaves; ++x) {
      // (a wave without a maximum has seen no key: zeros; or nothing but NaN, which stays)
      const float mw = s_stat[2 * (x * nr + r)];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mx);
      const float4 y = *reinterpret_cast<const float4*>(s_join + (x * nr + r) * D + d);
      sum = fmaf(f, s_stat[2 * (x * nr + r) + 1], sum);
      v[0] = fmaf(f, y.x, v[0]);
      v[1] = fmaf(f, y.y, v[1]);
      v[2] = fmaf(f, y.z, v[2]);
      v[3] = fmaf(f, y.w, v[3]);
    }
    const int rr = r0 + r;
    const int64_t row =
        ((int64_t)qa + rr / a.group) * a.num_heads + (int64_t)j * a.group + rr % a.group;
    store4(row, d, v, mx, sum);
  }
}

// Joins the chunks of the rows whose context has more than one: a wave per row
// (of a position, heads fastest).
template <typename T, int D>
__global__ __launch_bounds__(256) void scaled_merge_kernel(const ScaledDev a, int32_t row_tiles) {
  const int lane = threadIdx.x & 63;
  const int s = (int)(blockIdx.x / (uint32_t)row_tiles);
  const int r = (int)(blockIdx.x % (uint32_t)row_tiles) * 4 + (int)(threadIdx.x >> 6);
  uint32_t qa = (uint32_t)s, qb = (uint32_t)s + 1u;
  if (a.cu_seqlens_q != nullptr) {
    qa = a.cu_seqlens_q[s];
    qb = a.cu_seqlens_q[s + 1];
  }
  int n = qb > qa ? (int)min(qb - qa, (uint32_t)a.max_query_len) : 0;
  n = (int64_t)qa >= a.total_rows ? 0 : (int)min((int64_t)n, a.total_rows - (int64_t)qa);
  const int L = (int)min(a.context_lens[s], (uint32_t)a.max_ctx);
  const int nchunks = (L + a.chunk_tokens - 1) / a.chunk_tokens;
  if (nchunks <= 1 || r >= n * a.num_heads) return;
  const int64_t row = (int64_t)qa * a.num_heads + r;
  // eight chunks' parts at a time, all of them under way before one is used
  const float2* stat = reinterpret_cast<const float2*>(a.part_stat) + row * a.max_chunks;
  const float* part = a.part_out + row * a.max_chunks * D;
  constexpr int NV = (D + 63) / 64, U = 8;
  float mx = -INFINITY, sum = 0.f, v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) v[k] = 0.f;
  for (int c0 = 0; c0 < nchunks; c0 += U) {
    float2 st[U];
    float x[U][NV];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + u, nchunks - 1);
      st[u] = stat[c];
#pragma unroll
      for (int k = 0; k < NV; ++k) x[u][k] = part[(int64_t)c * D + min(lane + 64 * k, D - 1)];
    }
    float top = mx;
#pragma unroll
    for (int u = 0; u < U; ++u) top = fmaxf(top, c0 + u < nchunks ? st[u].x : -INFINITY);
    // (a part without a maximum has seen no key: zeros; or nothing but NaN, which stays)
    const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - top);
    mx = top;
    sum *= f;
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] *= f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool have = c0 + u < nchunks;
      const float g = st[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st[u].x - mx);
      sum = fmaf(g, have ? st[u].y : 0.f, sum);
#pragma unroll
      for (int k = 0; k < NV; ++k) v[k] = have ? fmaf(g, x[u][k], v[k]) : v[k];
    }
  }
  const float inv = sum > 0.f || sum != sum ? 1.f / (sum + a.denom_eps) : 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (lane + 64 * k < D)
      store_from_f32<T>(static_cast<T*>(a.out) + row * D + lane + 64 * k, v[k] * inv);
}

template <typename T, int D, int BS, int NQ>
hipError_t launch_scaled_t(const ScaledDev& d, int64_t grid, hipStream_t stream) {
  const size_t lds = d.split_keys ? (size_t)kScaledWaves * d.lds_rows * (D + 2) * 4 : 0;
  hipLaunchKernelGGL((scaled_attention_kernel<T, D, BS, NQ>), dim3((unsigned)grid),
                     dim3(d.split_keys ? 64 * kScaledWaves : 64), lds, stream, d);
  if (d.max_chunks > 1) {
    const int tiles = (int)(((int64_t)d.max_query_len * d.num_heads + 3) / 4);
    hipLaunchKernelGGL((scaled_merge_kernel<T, D>), dim3((unsigned)tiles * d.num_seqs), dim3(256),
                       0, stream, d, tiles);
  }
  return hipGetLastError();
}

template <typename T, int D, int BS>
hipError_t launch_scaled_q(const ScaledDev& d, int64_t grid, int nq, hipStream_t stream) {
  if constexpr (scaled_two_tiles<T>())
    if (nq == 2) return launch_scaled_t<T, D, BS, 2>(d, grid, stream);
  return launch_scaled_t<T, D, BS, 1>(d, grid, stream);
}

template <typename T>
hipError_t launch_scaled(const ScaledArgs& a, const CacheGeom& g, const ScaledPlan& p,
                         hipStream_t stream) {
  const int64_t rows = a.total_rows * a.num_heads;
  float* part = static_cast<float*>(a.workspace);
  const ScaledDev d{a.query,
                    static_cast<const uint8_t*>(a.key_cache),
                    static_cast<const uint8_t*>(a.value_cache),
                    a.key_scales,
                    a.value_scales,
                    a.scale_block_stride,
                    a.block_tables,
                    a.cu_seqlens_q,
                    a.context_lens,
                    a.out,
                    part,
                    part == nullptr ? nullptr : part + rows * p.max_chunks * g.head_dim,
                    g.block_stride,
                    g.head_stride,
                    g.num_blocks,
                    a.total_rows,
                    a.block_table_stride,
                    a.num_seqs,
                    a.max_query_len,
                    a.max_ctx,
                    a.num_heads,
                    g.num_kv_heads,
                    a.num_heads / g.num_kv_heads,
                    a.causal,
                    p.tiles,
                    p.chunk_tokens,
                    p.max_chunks,
                    p.split_keys,
                    p.lds_rows,
                    a.scale * 1.4426950408889634f,
                    a.denom_eps};
#define VPA_SCALED(DV, BV)                           \
  if (g.head_dim == DV && g.block_size == BV)        \
    return launch_scaled_q<T, DV, BV>(d, p.grid, p.nq, stream);
#define VPA_SCALED_D(DV) VPA_SCALED(DV, 8) VPA_SCALED(DV, 16) VPA_SCALED(DV, 32)
  VPA_SCALED_D(64) VPA_SCALED_D(96) VPA_SCALED_D(128) VPA_SCALED_D(192) VPA_SCALED_D(256)
#undef VPA_SCALED_D
#undef VPA_SCALED
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace vpa
