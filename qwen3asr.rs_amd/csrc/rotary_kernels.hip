// Rotary positions of several axes for gfx950, with the rows' RMS norm in
// front, in two forms: q and k rows rotated into row buffers (rotary_qk), and
// q rotated while k and v go straight into the paged cache
// (rotary_reshape_and_cache).
//
// The decoder normalises each head row of q and k, rotates it by its token's
// position and appends k and v to the cache right after
// (vasr-models/src/model/thinker_text.rs:1041-1068, 1101-1109). For a row x of
// D values:
//   n = x * w / sqrt(mean(x^2) + eps)                    (where a weight is given)
//   a_i = positions[axis(i)] * inv_freq[i],  i < R / 2   (R rotated dims)
//   y_p = n_p cos a_i - n_s sin a_i,  y_s = n_s cos a_i + n_p sin a_i
// over the pairs (p, s) = (i, i + R/2), or (2i, 2i + 1) for `adjacent`; dims
// from R on are copied. Norm, angles and products are computed once in f32
// (the angle's turns in f64) and rounded once, at the store: the steps of a
// row have no reason to round in between.
//
// Angles: a position of a million times a frequency of 1 needs 20 bits before
// the point, so the turns a / 2 pi are formed and reduced to an eighth of a
// turn in f64 (4 instructions) and only the remainder goes to f32.
//
// A lane holds two 16-byte vectors of a row that contain whole pairs
// (vectors c and R/2 + c of split pairs; 2c and 2c + 1 of adjacent ones and of
// the copied rest), so nothing crosses lanes but the norm's sum, and the X
// angles of a lane serve every head of its token.
//
// Both kernels are bound by the bytes of the rows. Measured at 16 + 8 heads of 128
// in 16 bits: rotary_qk 14.3 us for 4500 tokens with 64 rotated dims (55 MB, 3.9
// TB/s; 4.2 us for one token); into the cache 135 us for 32768 tokens in runs of
// 512 that start inside a block (538 MB, 4.0 TB/s, against 4.8 TB/s of a large
// copy), 9.5 us for 256 tokens of a decode step.

#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "vpa_device.h"
#include "vpa_internal.h"

namespace vpa {
namespace {

constexpr int kThreads = 256;

// cos and sin of 2 pi * t (t: turns, f64). t is reduced to r, |r| <= 1/8,
// around a quarter turn q; the Taylor sums of sin and cos at |2 pi r| <= pi/4
// end below 2^-28 (x^11 / 11!, x^12 / 12!).
__device__ __forceinline__ void turn_sincos(double t, float& s, float& c) {
  const double q4 = __builtin_rint(t * 4.0);
  const float x = (float)((t - q4 * 0.25) * 6.283185307179586476925);
  const int q = (int)(int64_t)q4 & 3;
  const float x2 = x * x;
  float sp = fmaf(x2, 2.75573192e-6f, -1.98412698e-4f);
  sp = fmaf(sp, x2, 8.33333333e-3f);
  sp = fmaf(sp, x2, -1.66666667e-1f);
  sp = fmaf(sp * x2, x, x);
  float cp = fmaf(x2, -2.75573192e-7f, 2.48015873e-5f);
  cp = fmaf(cp, x2, -1.38888889e-3f);
  cp = fmaf(cp, x2, 4.16666667e-2f);
  cp = fmaf(cp, x2, -0.5f);
  cp = fmaf(cp, x2, 1.f);
  const float s0 = (q & 1) ? cp : sp, c0 = (q & 1) ? sp : cp;
  s = (q & 2) ? -s0 : s0;
  c = ((q + 1) & 2) ? -c0 : c0;
}

// One 16-byte vector of T <-> f32 values.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[pack_x<T>()]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = low_half_f32<T>(w[i]);
      f[2 * i + 1] = high_half_f32<T>(w[i]);
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&f)[pack_x<T>()]) {
  if constexpr (std::is_same_v<T, float>)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  else
    return make_uint4(pack2_hw<T>(f[0], f[1]), pack2_hw<T>(f[2], f[3]), pack2_hw<T>(f[4], f[5]),
                      pack2_hw<T>(f[6], f[7]));
}

__device__ __forceinline__ void store_nt(uint4* dst, const uint4& v) {
  typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(u32x4{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4*>(dst));
}
template <typename E>
__device__ __forceinline__ void store_nt(E* dst, E v) {  // one cache element
  if constexpr (sizeof(E) == 1)
    __builtin_nontemporal_store(__builtin_bit_cast(unsigned char, v),
                                reinterpret_cast<unsigned char*>(dst));
  else if constexpr (sizeof(E) == 2)
    __builtin_nontemporal_store(__builtin_bit_cast(unsigned short, v),
                                reinterpret_cast<unsigned short*>(dst));
  else
    __builtin_nontemporal_store(__builtin_bit_cast(unsigned int, v),
                                reinterpret_cast<unsigned int*>(dst));
}

// Where a lane's two vectors lie in a row, and its first frequency.
template <typename T>
struct LaneChunk {
  static constexpr int X = pack_x<T>();
  int a, b;      // first elements of the two vectors
  bool rotated;  // false: copied (past the rotated dims)
  bool adjacent;
  __device__ __forceinline__ LaneChunk(int c, int rotary_dim, bool adj) {
    const int pairs = rotary_dim / (2 * X);
    rotated = c < pairs;
    adjacent = adj || !rotated;
    a = adjacent ? 2 * c * X : c * X;
    b = adjacent ? a + X : rotary_dim / 2 + c * X;
  }
};

// The X angles of a lane (chunk c) for the token `tok`.
template <typename T>
__device__ __forceinline__ void lane_angles(const RotaryArgs& r, int64_t tok, int c, bool rotated,
                                            float (&sn)[pack_x<T>()], float (&cs)[pack_x<T>()]) {
  constexpr int X = pack_x<T>();
#pragma unroll
  for (int e = 0; e < X; ++e) {
    sn[e] = 0.f;
    cs[e] = 1.f;
  }
  if (!rotated) return;
  // positions of the token on every axis, and the axes of the X frequencies
  // (one byte each); an axis past the last reads as the last
  double pos[kRotaryMaxAxes];
#pragma unroll
  for (int x = 0; x < kRotaryMaxAxes; ++x) {
    const int64_t at = min(x, r.num_axes - 1) * r.axis_stride + tok;
    pos[x] = r.positions_i64 ? (double)static_cast<const int64_t*>(r.positions)[at]
                             : (double)static_cast<const uint32_t*>(r.positions)[at];
  }
  uint32_t ax[X / 4] = {};
  if (r.axes != nullptr) {
#pragma unroll
    for (int w = 0; w < X / 4; ++w)
      ax[w] = *reinterpret_cast<const uint32_t*>(r.axes + c * X + 4 * w);
  }
  const double2* freq = reinterpret_cast<const double2*>(r.inv_freq + c * X);
#pragma unroll
  for (int e = 0; e < X; ++e) {
    const uint32_t axis = (ax[e / 4] >> (8 * (e % 4))) & 0xffu;
    const double p = axis == 0 ? pos[0] : axis == 1 ? pos[1] : axis == 2 ? pos[2] : pos[3];
    const double f = e % 2 ? freq[e / 2].y : freq[e / 2].x;
    turn_sincos(p * (f * 0.15915494309189533576888), sn[e], cs[e]);
  }
}

// Sum over the `lg` lanes (a power of two, at most 32) of a row, in each of them.
__device__ __forceinline__ float row_sum(float v, int lg) {
  if (lg > 1) v += dpp<kDppQuadXor1>(v);
  if (lg > 2) v += dpp<kDppQuadXor2>(v);
  if (lg > 4) v += dpp<kDppRowHalfMirror>(v);
  if (lg > 8) v += dpp<kDppRowMirror>(v);
  if (lg > 16) v = sum_xor16(v);
  return v;
}

// A lane's two vectors of a norm's weights, packed. They are loaded before the
// rows: loads return in order, so weights loaded with a row would hold it up until
// the row prefetched before them has come.
struct NormLane {
  uint4 a, b;
  bool on;  // (uniform)
};
template <typename T>
__device__ __forceinline__ NormLane norm_lane(const T* w, const LaneChunk<T>& lc, bool active) {
  NormLane n{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u), w != nullptr};
  if (n.on && active) {
    n.a = *reinterpret_cast<const uint4*>(w + lc.a);
    n.b = *reinterpret_cast<const uint4*>(w + lc.b);
  }
  return n;
}
__device__ __forceinline__ uint4 pick(bool first, const uint4& a, const uint4& b) {
  return make_uint4(first ? a.x : b.x, first ? a.y : b.y, first ? a.z : b.z, first ? a.w : b.w);
}

// Norm and rotation of a lane's two vectors of a q row (is_q) or k row, in place.
// Lanes past the row hold zeros; every lane of the row's lg calls it.
template <typename T>
__device__ __forceinline__ void turn_row(float (&fa)[pack_x<T>()], float (&fb)[pack_x<T>()],
                                         bool rotated, bool adjacent, int lg, int head_dim,
                                         float eps, bool is_q, const NormLane& qn,
                                         const NormLane& kn, const float (&sn)[pack_x<T>()],
                                         const float (&cs)[pack_x<T>()]) {
  constexpr int X = pack_x<T>();
  if (qn.on || kn.on) {  // (uniform)
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < X; ++e) ss = fmaf(fa[e], fa[e], fmaf(fb[e], fb[e], ss));
    ss = row_sum(ss, lg);
    if (is_q ? qn.on : kn.on) {
      // 1 / sqrt: the hardware's, within an ulp, and one Newton step
      const float x = ss * (1.f / (float)head_dim) + eps;
      float inv = __builtin_amdgcn_rsqf(x);
      if (x >= FLT_MIN && x < INFINITY) inv *= fmaf(-0.5f * x * inv, inv, 1.5f);
      float wa[X], wb[X];
      unpack<T>(pick(is_q, qn.a, kn.a), wa);
      unpack<T>(pick(is_q, qn.b, kn.b), wb);
#pragma unroll
      for (int e = 0; e < X; ++e) {
        fa[e] *= inv * wa[e];
        fb[e] *= inv * wb[e];
      }
    }
  }
  if (!rotated) return;
  if (adjacent) {  // (uniform)
#pragma unroll
    for (int e = 0; e < X; e += 2) {
      const float p = fa[e], q = fa[e + 1], r = fb[e], s = fb[e + 1];
      fa[e] = fmaf(p, cs[e / 2], -(q * sn[e / 2]));
      fa[e + 1] = fmaf(q, cs[e / 2], p * sn[e / 2]);
      fb[e] = fmaf(r, cs[X / 2 + e / 2], -(s * sn[X / 2 + e / 2]));
      fb[e + 1] = fmaf(s, cs[X / 2 + e / 2], r * sn[X / 2 + e / 2]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < X; ++e) {
      const float p = fa[e], s = fb[e];
      fa[e] = fmaf(p, cs[e], -(s * sn[e]));
      fb[e] = fmaf(s, cs[e], p * sn[e]);
    }
  }
}

// q and k rows rotated into row buffers. A group of lg lanes serves one token
// and every nhb-th head row of it (the q heads, then the k heads); the groups
// of a token lie side by side, so each pass over them reads and writes whole
// stretches of the token's row. The outputs may be the inputs (each row is
// read and written by the same lanes, which read it first).
template <typename T>
__global__ __launch_bounds__(kThreads) void rotary_qk_kernel(
    const T* q, const T* k, int64_t q_stride, int64_t k_stride, T* out_q, T* out_k,
    int64_t out_q_stride, int64_t out_k_stride, const T* __restrict__ q_norm,
    const T* __restrict__ k_norm, float eps, RotaryArgs r, int64_t num_tokens, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t lg_log2, int32_t nhb) {
  constexpr int X = pack_x<T>();
  const int lg = 1 << lg_log2;
  const int64_t unit = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> lg_log2;
  const int64_t tok = unit / nhb;
  const int h0 = (int)(unit - tok * nhb);
  const int c = threadIdx.x & (lg - 1);
  if (tok >= num_tokens) return;  // (whole lane groups)
  const bool active = c < head_dim / (2 * X);
  const LaneChunk<T> lc(c, r.rotary_dim, r.adjacent);
  const int rows = num_heads + num_kv_heads;
  float sn[X], cs[X];
  uint4 na, nb;
  auto load_row = [&](int h) {
    na = nb = make_uint4(0u, 0u, 0u, 0u);
    if (active && h < rows) {
      const T* src = h < num_heads ? q + tok * q_stride + (int64_t)h * head_dim
                                   : k + tok * k_stride + (int64_t)(h - num_heads) * head_dim;
      na = *reinterpret_cast<const uint4*>(src + lc.a);
      nb = *reinterpret_cast<const uint4*>(src + lc.b);
    }
  };
  const NormLane qn = norm_lane(q_norm, lc, active), kn = norm_lane(k_norm, lc, active);
  load_row(h0);
  lane_angles<T>(r, tok, c, active && lc.rotated, sn, cs);
#pragma unroll 1
  for (int h = h0; h < rows; h += nhb) {  // the next row in flight while one is turned
    float fa[X], fb[X];
    unpack<T>(na, fa);
    unpack<T>(nb, fb);
    load_row(h + nhb);
    const bool is_q = h < num_heads;
    turn_row<T>(fa, fb, active && lc.rotated, r.adjacent, lg, head_dim, eps, is_q, qn, kn, sn, cs);
    if (active) {
      T* dst = is_q ? out_q + tok * out_q_stride + (int64_t)h * head_dim
                    : out_k + tok * out_k_stride + (int64_t)(h - num_heads) * head_dim;
      *reinterpret_cast<uint4*>(dst + lc.a) = pack<T>(fa);
      *reinterpret_cast<uint4*>(dst + lc.b) = pack<T>(fb);
    }
  }
}

// Lanes of a head row and lane groups of a workgroup, of the second form.
template <typename T, int D>
struct RowLanes {
  static constexpr int NC = D / (2 * pack_x<T>());  // lanes with work
  static constexpr int LG = NC <= 4 ? 4 : NC <= 8 ? 8 : NC <= 16 ? 16 : 32;
  static constexpr int NG = kThreads / LG;
};

// One workgroup per (group of tg tokens, `heads` kv heads), tg at most the lane
// groups: a lane group serves one token throughout, so its angles are made once for
// all the heads (at one head per workgroup they were a quarter of the time of a
// long prompt). NG / tg heads at a time: their q rows are rotated into out, the k
// rows rotated and the v rows copied (or quantised) into LDS as [head][token][D]
// rows of the cache type, and these written out along the token axis as the cache
// tiles lie: key units of 16 bytes, value elements (whole vectors where the
// group's tokens are an aligned run of a block). Tokens alone in their blocks (a
// decode step) leave with non-temporal stores, as in reshape_and_cache.
template <typename T, typename C, int D, int BS>
__global__ __launch_bounds__(kThreads) void rotary_cache_kernel(
    const T* q, const T* __restrict__ k, const T* __restrict__ v, int64_t q_stride,
    int64_t k_stride, int64_t v_stride, T* out, int64_t out_stride,
    const T* __restrict__ q_norm, const T* __restrict__ k_norm, float eps, RotaryArgs r,
    C* __restrict__ key_cache, C* __restrict__ value_cache,
    const int64_t* __restrict__ slot_mapping, int64_t num_tokens, int64_t num_slots,
    int64_t block_stride, int64_t head_stride, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, int32_t num_kv_heads, int32_t group, int32_t tg_log2,
    int32_t heads) {
  constexpr bool kQuant = !std::is_same_v<T, C>;
  constexpr int X = pack_x<T>();   // row elements per vector
  constexpr int XC = pack_x<C>();  // cache elements per vector
  constexpr int CHC = D / XC;      // vectors of a cache row
  constexpr int CHT = D / X;       // vectors of an input row
  constexpr int NC = RowLanes<T, D>::NC, LG = RowLanes<T, D>::LG, NG = RowLanes<T, D>::NG;
  constexpr int VPT = (NG * CHT + kThreads - 1) / kThreads;  // value vectors per thread
  // (one vector of padding per row: tokens of one dim lie in different banks;
  // without it the tile writes waited 32 us for banks in a prompt of 32768 tokens)
  constexpr int DP = D + XC;
  __shared__ __align__(16) C s_k[NG * DP];
  __shared__ __align__(16) C s_v[NG * DP];
  __shared__ int64_t slots[BS];
  __shared__ bool s_run, s_alone;

  const int tid = threadIdx.x;
  const int tg = 1 << tg_log2;
  const int hb = NG >> tg_log2;  // heads at a time
  const int parts = (num_kv_heads + heads - 1) / heads;
  // Consecutive workgroups go to the eight XCDs in turn; this gives each XCD one run
  // of the groups, so that the two groups which share a cache block (runs that do
  // not start at a block's first token) complete its sectors in one L2.
  const uint32_t bid = (blockIdx.x & 7u) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  const int j_begin = (int)(bid % (uint32_t)parts) * heads;
  const int j_end = min(j_begin + heads, num_kv_heads);
  const int64_t t0 = (int64_t)(bid / (uint32_t)parts) << tg_log2;
  if (t0 >= num_tokens) return;  // (the grid is a multiple of 8)
  // the tokens' slots, and whether they are an aligned run of a block or have no
  // neighbour in their block (the first wave; tg is at most 32)
  if (tid < 64) {
    int64_t s = tid < tg && t0 + tid < num_tokens ? slot_mapping[t0 + tid] : -1;
    s = s < num_slots ? s : -1;  // out of range: skipped like padding
    if (tid < tg) slots[tid] = s;
    const int64_t before = __shfl_up(s, 1, 64);
    const bool inner = tid > 0 && tid < tg;
    const uint64_t broken = __ballot(inner && (s < 0 || s != before + 1));
    const uint64_t shared = __ballot(inner && s >= 0 && before >= 0 && s / BS == before / BS);
    if (tid == 0) {
      s_run = broken == 0 && s >= 0 && (s & (tg - 1)) == 0;
      s_alone = shared == 0;
    }
  }
  float ks = 1.f, vs = 1.f;
  if constexpr (kQuant) {
    ks = *k_scale;
    vs = *v_scale;
  }
  const int c = tid & (LG - 1), t = (tid / LG) & (tg - 1), sub = (tid / LG) >> tg_log2;
  const int64_t tok = t0 + t;
  const bool live = tok < num_tokens, active = live && c < NC;
  const LaneChunk<T> lc(c, r.rotary_dim, r.adjacent);
  // the token's rows from this lane's first vector on; its second is `step` on
  const T* q_tok = q + (live ? tok : t0) * q_stride + lc.a;
  const T* k_tok = k + (live ? tok : t0) * k_stride + lc.a;
  T* out_tok = out + (live ? tok : t0) * out_stride + lc.a;
  const int step = lc.b - lc.a;
  const NormLane qn = norm_lane(q_norm, lc, c < NC), kn = norm_lane(k_norm, lc, c < NC);
  // what the next heads begin with, in flight while these are written out: the
  // value rows (head, then token), and the first of the token's rows (of each
  // head its q heads, then k)
  uint4 vv[VPT], na, nb;
  int h, kind;
  auto load_row = [&](int j0, int nh) {
    na = nb = make_uint4(0u, 0u, 0u, 0u);
    if (active && h < nh) {
      const T* src = kind < group ? q_tok + ((j0 + h) * group + kind) * D : k_tok + (j0 + h) * D;
      na = *reinterpret_cast<const uint4*>(src);
      nb = *reinterpret_cast<const uint4*>(src + step);
    }
  };
  auto begin = [&](int j0) {
    const int nh = min(hb, j_end - j0);
    h = sub / (group + 1);
    kind = sub - h * (group + 1);
    load_row(j0, nh);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = tid + i * kThreads, row = e / CHT;
      vv[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < nh << tg_log2 && t0 + (row & (tg - 1)) < num_tokens)
        vv[i] = *reinterpret_cast<const uint4*>(v + (t0 + (row & (tg - 1))) * v_stride +
                                                (j0 + (row >> tg_log2)) * D + (e - row * CHT) * X);
    }
  };
  begin(j_begin);
  float sn[X], cs[X];
  lane_angles<T>(r, live ? tok : t0, c, c < NC && lc.rotated, sn, cs);

  for (int j0 = j_begin; j0 < j_end; j0 += hb) {
    const int nh = min(hb, j_end - j0);
#pragma unroll 1
    while (h < nh) {
      float fa[X], fb[X];
      unpack<T>(na, fa);
      unpack<T>(nb, fb);
      const bool is_q = kind < group;
      const int head = j0 + h;
      T* dst_q = out_tok + (head * group + kind) * D;
      C* dst_k = &s_k[((h << tg_log2) + t) * DP + lc.a];
      for (kind += hb; kind > group; kind -= group + 1) ++h;
      load_row(j0, nh);
      turn_row<T>(fa, fb, c < NC && lc.rotated, r.adjacent, LG, D, eps, is_q, qn, kn, sn, cs);
      if (!active) continue;
      if (is_q) {
        *reinterpret_cast<uint4*>(dst_q) = pack<T>(fa);
        *reinterpret_cast<uint4*>(dst_q + step) = pack<T>(fb);
      } else if constexpr (kQuant) {
#pragma unroll
        for (int e = 0; e < X; ++e) {
          dst_k[e].x = (uint8_t)fp8_from_f32(fa[e] / ks);
          dst_k[step + e].x = (uint8_t)fp8_from_f32(fb[e] / ks);
        }
      } else {
        *reinterpret_cast<uint4*>(dst_k) = pack<T>(fa);
        *reinterpret_cast<uint4*>(dst_k + step) = pack<T>(fb);
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int e = tid + i * kThreads, row = e / CHT;
      if (row >= nh << tg_log2) continue;
      C* dst = &s_v[row * DP + (e - row * CHT) * X];
      if constexpr (kQuant) {
        float f[X];
        unpack<T>(vv[i], f);
#pragma unroll
        for (int x = 0; x < X; ++x) dst[x].x = (uint8_t)fp8_from_f32(f[x] / vs);
      } else {
        *reinterpret_cast<uint4*>(dst) = vv[i];
      }
    }
    lds_group_barrier();
    if (j0 + hb < j_end) begin(j0 + hb);

    const int64_t s0 = slots[0];
    const bool run = s_run, alone = s_alone;
    const int units = CHC << tg_log2;
    if (run && tg >= XC) {
      const int64_t blk = s0 / BS;
      const int off = (int)(s0 - blk * BS);
      C* kt = key_cache + blk * block_stride + off * XC;
      C* vt = value_cache + blk * block_stride + off;
      const int vr_log2 = tg_log2 - __builtin_ctz(XC);  // vectors of a value row's run
      for (int i = tid; i < nh * units; i += kThreads) {
        const int hh = i / units, e = i - hh * units;
        const int64_t at = (int64_t)(j0 + hh) * head_stride;
        const int ch = e >> tg_log2, tt = e & (tg - 1);
        *reinterpret_cast<uint4*>(kt + at + (ch * BS + tt) * XC) =
            *reinterpret_cast<const uint4*>(&s_k[((hh << tg_log2) + tt) * DP + ch * XC]);
        const int d = e >> vr_log2, sg = e & ((1 << vr_log2) - 1);
        union {
          uint4 v4;
          C e[XC];
        } u;
#pragma unroll
        for (int x = 0; x < XC; ++x) u.e[x] = s_v[((hh << tg_log2) + sg * XC + x) * DP + d];
        *reinterpret_cast<uint4*>(vt + at + d * BS + sg * XC) = u.v4;
      }
    } else {
      // a thread writes one token's units throughout
      const int tt = tid & (tg - 1), i0 = tid >> tg_log2, di = kThreads >> tg_log2;
      const int64_t s = slots[tt];
      if (s >= 0) {
        const int64_t blk = s / BS;
        const int off = (int)(s - blk * BS);
        for (int hh = 0; hh < nh; ++hh) {
          const int64_t at = blk * block_stride + (int64_t)(j0 + hh) * head_stride;
          C* kt = key_cache + at + off * XC;
          C* vt = value_cache + at + off;
          const C* k_row = &s_k[((hh << tg_log2) + tt) * DP];
          const C* v_row = &s_v[((hh << tg_log2) + tt) * DP];
          for (int ch = i0; ch < CHC; ch += di) {
            uint4* dst = reinterpret_cast<uint4*>(kt + ch * (BS * XC));
            const uint4 u = *reinterpret_cast<const uint4*>(k_row + ch * XC);
            if (alone) store_nt(dst, u);  // (uniform)
            else *dst = u;
          }
          for (int d = i0; d < D; d += di) {
            if (alone) store_nt(vt + d * BS, v_row[d]);
            else vt[d * BS] = v_row[d];
          }
        }
      }
    }
    if (j0 + hb < j_end) lds_group_barrier();  // (LDS is read)
  }
}

template <typename T>
hipError_t rotary_qk_typed(const RotaryRows& a, const RotaryArgs& r, hipStream_t stream) {
  constexpr int X = pack_x<T>();
  int lg_log2 = 0;
  while ((1 << lg_log2) < a.head_dim / (2 * X)) ++lg_log2;
  const int rows = a.num_heads + a.num_kv_heads;
  // rows per lane group: as many as share one set of angles without leaving the
  // chip idle
  int per = 1;
  while (per < 16 && per < rows && (a.num_tokens * rows / (2 * per) << lg_log2) >= 131072) per *= 2;
  const int nhb = (rows + per - 1) / per;
  const int64_t threads = a.num_tokens * nhb << lg_log2;
  const int64_t grid = (threads + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(rotary_qk_kernel<T>, dim3((uint32_t)grid), dim3(kThreads), 0, stream,
                     static_cast<const T*>(a.q), static_cast<const T*>(a.k), a.q_stride,
                     a.k_stride, static_cast<T*>(a.out_q), static_cast<T*>(a.out_k),
                     a.out_q_stride, a.out_k_stride, static_cast<const T*>(a.q_norm),
                     static_cast<const T*>(a.k_norm), a.eps, r, a.num_tokens, a.num_heads,
                     a.num_kv_heads, a.head_dim, lg_log2, nhb);
  return hipGetLastError();
}

template <typename T, typename C, int D, int BS>
hipError_t rotary_cache_launch(const RotaryRows& a, const RotaryArgs& r, const RotaryCache& k,
                               const CacheGeom& g, hipStream_t stream) {
  // tokens of a workgroup: a block's, at most one per lane group; fewer in small
  // calls (decode steps), down to 4, until every compute unit has a workgroup
  constexpr int NG = RowLanes<T, D>::NG;
  int tg_log2 = __builtin_ctz((unsigned)std::min(BS, NG));
  auto groups = [&] { return (a.num_tokens + (1 << tg_log2) - 1) >> tg_log2; };
  while (tg_log2 > 2 && groups() * g.num_kv_heads < 256) --tg_log2;
  // kv heads of a workgroup: those it serves at a time, or more to share the angles
  int heads = NG >> tg_log2;
  if (groups() * ((g.num_kv_heads + heads - 1) / heads) < 256) heads = 1;
  while (heads < g.num_kv_heads &&
         groups() * ((g.num_kv_heads + 2 * heads - 1) / (2 * heads)) >= 1024)
    heads *= 2;
  const int64_t grid = (groups() * ((g.num_kv_heads + heads - 1) / heads) + 7) / 8 * 8;
  hipLaunchKernelGGL((rotary_cache_kernel<T, C, D, BS>), dim3((uint32_t)grid), dim3(kThreads), 0,
                     stream, static_cast<const T*>(a.q), static_cast<const T*>(a.k),
                     static_cast<const T*>(k.v), a.q_stride, a.k_stride, k.v_stride,
                     static_cast<T*>(a.out_q), a.out_q_stride, static_cast<const T*>(a.q_norm),
                     static_cast<const T*>(a.k_norm), a.eps, r, static_cast<C*>(k.key_cache),
                     static_cast<C*>(k.value_cache), k.slot_mapping, a.num_tokens,
                     g.num_blocks * BS, g.block_stride, g.head_stride, k.k_scale, k.v_scale,
                     g.num_kv_heads, a.num_heads / g.num_kv_heads, tg_log2, heads);
  return hipGetLastError();
}

template <typename T, typename C, int D>
hipError_t rotary_cache_bs(const RotaryRows& a, const RotaryArgs& r, const RotaryCache& k,
                           const CacheGeom& g, hipStream_t stream) {
  switch (g.block_size) {
    case 8: return rotary_cache_launch<T, C, D, 8>(a, r, k, g, stream);
    case 16: return rotary_cache_launch<T, C, D, 16>(a, r, k, g, stream);
    case 32: return rotary_cache_launch<T, C, D, 32>(a, r, k, g, stream);
  }
  return hipErrorInvalidValue;
}

template <typename T, typename C>
hipError_t rotary_cache_typed(const RotaryRows& a, const RotaryArgs& r, const RotaryCache& k,
                              const CacheGeom& g, hipStream_t stream) {
  switch (g.head_dim) {
    case 64: return rotary_cache_bs<T, C, 64>(a, r, k, g, stream);
    case 96: return rotary_cache_bs<T, C, 96>(a, r, k, g, stream);
    case 128: return rotary_cache_bs<T, C, 128>(a, r, k, g, stream);
    case 192: return rotary_cache_bs<T, C, 192>(a, r, k, g, stream);
    case 256: return rotary_cache_bs<T, C, 256>(a, r, k, g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_rotary_qk(int dtype, const RotaryRows& a, const RotaryArgs& r,
                            hipStream_t stream) {
  switch (dtype) {
    case VPA_DTYPE_F32: return rotary_qk_typed<float>(a, r, stream);
    case VPA_DTYPE_F16: return rotary_qk_typed<f16_t>(a, r, stream);
    case VPA_DTYPE_BF16: return rotary_qk_typed<bf16_t>(a, r, stream);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_rotary_cache(int dtype, int cache_dtype, const RotaryRows& a,
                               const RotaryArgs& r, const RotaryCache& k, const CacheGeom& g,
                               hipStream_t stream) {
  const bool fp8 = cache_dtype == VPA_DTYPE_FP8_E4M3;
  switch (dtype) {
    case VPA_DTYPE_F32:
      return fp8 ? rotary_cache_typed<float, fp8_t>(a, r, k, g, stream)
                 : rotary_cache_typed<float, float>(a, r, k, g, stream);
    case VPA_DTYPE_F16:
      return fp8 ? rotary_cache_typed<f16_t, fp8_t>(a, r, k, g, stream)
                 : rotary_cache_typed<f16_t, f16_t>(a, r, k, g, stream);
    case VPA_DTYPE_BF16:
      return fp8 ? rotary_cache_typed<bf16_t, fp8_t>(a, r, k, g, stream)
                 : rotary_cache_typed<bf16_t, bf16_t>(a, r, k, g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace vpa
