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
// Both kernels are bound by the bytes of the rows.

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

// Sum over the `lg` lanes (a power of two) of a row.
__device__ __forceinline__ float row_sum(float v, int lg) {
  for (int m = 1; m < lg; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Norm and rotation of a lane's two vectors, in place. Lanes past the row
// (active false) hold zeros; every lane of the row's lg calls it.
template <typename T>
__device__ __forceinline__ void turn_row(float (&fa)[pack_x<T>()], float (&fb)[pack_x<T>()],
                                         const LaneChunk<T>& lc, bool active, int lg, int head_dim,
                                         float eps, const T* w, const float (&sn)[pack_x<T>()],
                                         const float (&cs)[pack_x<T>()]) {
  constexpr int X = pack_x<T>();
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < X; ++e) ss = fmaf(fa[e], fa[e], fmaf(fb[e], fb[e], ss));
    ss = row_sum(ss, lg);
    const float inv = 1.f / sqrtf(ss / (float)head_dim + eps);
    float wa[X], wb[X];
    unpack<T>(*reinterpret_cast<const uint4*>(w + (active ? lc.a : 0)), wa);
    unpack<T>(*reinterpret_cast<const uint4*>(w + (active ? lc.b : 0)), wb);
#pragma unroll
    for (int e = 0; e < X; ++e) {
      fa[e] *= inv * wa[e];
      fb[e] *= inv * wb[e];
    }
  }
  if (!lc.rotated) return;
  if (lc.adjacent) {
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
    const T* q, const T* k, int64_t q_stride, int64_t k_stride, T* out_q, T* out_k, int64_t out_q_stride, int64_t out_k_stride, const T* __restrict__ q_norm,
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
  float sn[X], cs[X];
  lane_angles<T>(r, tok, c, active && lc.rotated, sn, cs);
  for (int h = h0; h < num_heads + num_kv_heads; h += nhb) {
    const bool is_q = h < num_heads;
    const int64_t in = is_q ? tok * q_stride + (int64_t)h * head_dim
                            : tok * k_stride + (int64_t)(h - num_heads) * head_dim;
    const T* src = (is_q ? q : k) + in;
    float fa[X] = {}, fb[X] = {};
    if (active) {
      unpack<T>(*reinterpret_cast<const uint4*>(src + lc.a), fa);
      unpack<T>(*reinterpret_cast<const uint4*>(src + lc.b), fb);
    }
    turn_row<T>(fa, fb, lc, active, lg, head_dim, eps, is_q ? q_norm : k_norm, sn, cs);
    if (active) {
      T* dst = is_q ? out_q + tok * out_q_stride + (int64_t)h * head_dim
                    : out_k + tok * out_k_stride + (int64_t)(h - num_heads) * head_dim;
      *reinterpret_cast<uint4*>(dst + lc.a) = pack<T>(fa);
      *reinterpret_cast<uint4*>(dst + lc.b) = pack<T>(fb);
    }
  }
}

// One workgroup per (group of tg tokens, kv head): the q heads of that kv head
// rotated into out, k rotated and v copied (or quantised) into LDS as
// [token][D] rows of the cache type, then written out along the token axis as
// the cache tiles lie: key units of 16 bytes, value elements (whole vectors
// where the group's tokens fill a block).
template <typename T, typename C, int D, int BS>
__global__ __launch_bounds__(kThreads) void rotary_cache_kernel(
    const T* q, const T* __restrict__ k, const T* __restrict__ v, int64_t q_stride,
    int64_t k_stride, int64_t v_stride, T* out, int64_t out_stride,
    const T* __restrict__ q_norm, const T* __restrict__ k_norm, float eps, RotaryArgs r,
    C* __restrict__ key_cache, C* __restrict__ value_cache,
    const int64_t* __restrict__ slot_mapping, int64_t num_tokens, int64_t num_slots,
    int64_t block_stride, int64_t head_stride, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, int32_t num_kv_heads, int32_t group, int32_t tg_log2) {
  constexpr bool kQuant = !std::is_same_v<T, C>;
  constexpr int X = pack_x<T>();   // row elements per vector
  constexpr int XC = pack_x<C>();  // cache elements per vector
  constexpr int CHC = D / XC;      // vectors of a cache row
  constexpr int NC = D / (2 * X);  // lanes with work in a row
  constexpr int LG = NC <= 4 ? 4 : NC <= 8 ? 8 : NC <= 16 ? 16 : 32;
  constexpr int NG = kThreads / LG;
  __shared__ __align__(16) C s_k[BS * D];
  __shared__ __align__(16) C s_v[BS * D];
  __shared__ int64_t slots[BS];

  const int tid = threadIdx.x;
  const int tg = 1 << tg_log2;
  const int j = (int)(blockIdx.x % (uint32_t)num_kv_heads);
  const int64_t t0 = (int64_t)(blockIdx.x / (uint32_t)num_kv_heads) * tg;
  if (tid < BS) {
    int64_t s = -1;
    if (tid < tg && t0 + tid < num_tokens) s = slot_mapping[t0 + tid];
    slots[tid] = s < num_slots ? s : -1;  // out of range: skipped like padding
  }
  float ks = 1.f, vs = 1.f;
  if constexpr (kQuant) {
    ks = *k_scale;
    vs = *v_scale;
  }
  const int c = tid & (LG - 1), grp = tid / LG;
  const bool active = c < NC;
  const LaneChunk<T> lc(c, r.rotary_dim, r.adjacent);
  // rows of a token: its q heads of kv head j, then k. Groups beyond the
  // tokens take every step-th row of a token.
  const int step = NG > tg ? NG >> tg_log2 : 1;
  for (int t = NG > tg ? grp & (tg - 1) : grp; t < tg; t += NG) {
    const int64_t tok = t0 + t;
    if (tok >= num_tokens) continue;
    float sn[X], cs[X];
    lane_angles<T>(r, tok, c, active && lc.rotated, sn, cs);
    for (int h = NG > tg ? grp >> tg_log2 : 0; h <= group; h += step) {
      const bool is_q = h < group;
      const T* src = is_q ? q + tok * q_stride + (int64_t)(j * group + h) * D
                          : k + tok * k_stride + (int64_t)j * D;
      float fa[X] = {}, fb[X] = {};
      if (active) {
        unpack<T>(*reinterpret_cast<const uint4*>(src + lc.a), fa);
        unpack<T>(*reinterpret_cast<const uint4*>(src + lc.b), fb);
      }
      turn_row<T>(fa, fb, lc, active, LG, D, eps, is_q ? q_norm : k_norm, sn, cs);
      if (!active) continue;
      if (is_q) {
        T* dst = out + tok * out_stride + (int64_t)(j * group + h) * D;
        *reinterpret_cast<uint4*>(dst + lc.a) = pack<T>(fa);
        *reinterpret_cast<uint4*>(dst + lc.b) = pack<T>(fb);
      } else if constexpr (kQuant) {
#pragma unroll
        for (int e = 0; e < X; ++e) {
          s_k[t * D + lc.a + e].x = (uint8_t)fp8_from_f32(fa[e] / ks);
          s_k[t * D + lc.b + e].x = (uint8_t)fp8_from_f32(fb[e] / ks);
        }
      } else {
        *reinterpret_cast<uint4*>(&s_k[t * D + lc.a]) = pack<T>(fa);
        *reinterpret_cast<uint4*>(&s_k[t * D + lc.b]) = pack<T>(fb);
      }
    }
  }
  for (int i = tid; i < tg * (D / X); i += kThreads) {
    const int t = i / (D / X), d = (i - t * (D / X)) * X;
    if (t0 + t >= num_tokens) continue;
    const uint4 u = *reinterpret_cast<const uint4*>(v + (t0 + t) * v_stride + (int64_t)j * D + d);
    if constexpr (kQuant) {
      float f[X];
      unpack<T>(u, f);
#pragma unroll
      for (int e = 0; e < X; ++e) s_v[t * D + d + e].x = (uint8_t)fp8_from_f32(f[e] / vs);
    } else {
      *reinterpret_cast<uint4*>(&s_v[t * D + d]) = u;
    }
  }
  __syncthreads();

  const int64_t s0 = slots[0];
  if (tg == BS && BS >= XC) {
    bool whole = s0 >= 0 && s0 % BS == 0;
#pragma unroll
    for (int i = 1; i < BS; ++i) whole = whole && slots[i] == s0 + i;
    if (whole) {
      const int64_t at = s0 / BS * block_stride + j * head_stride;
      uint4* kt = reinterpret_cast<uint4*>(key_cache + at);
      uint4* vt = reinterpret_cast<uint4*>(value_cache + at);
      constexpr int VR = BS >= XC ? BS / XC : 1;  // vectors of a value-tile row
      for (int i = tid; i < CHC * BS; i += kThreads) {
        const int ch = i / BS, t = i - ch * BS;
        kt[i] = *reinterpret_cast<const uint4*>(&s_k[t * D + ch * XC]);
        const int d = i / VR, sg = i - d * VR;
        union {
          uint4 v;
          C e[XC];
        } u;
#pragma unroll
        for (int e = 0; e < XC; ++e) u.e[e] = s_v[(sg * XC + e) * D + d];
        vt[i] = u.v;
      }
      return;
    }
  }
  for (int i = tid; i < CHC << tg_log2; i += kThreads) {
    const int t = i & (tg - 1), ch = i >> tg_log2;
    const int64_t s = slots[t];
    if (s < 0) continue;
    const int64_t blk = s / BS;
    const int off = (int)(s - blk * BS);
    *reinterpret_cast<uint4*>(key_cache + blk * block_stride + j * head_stride +
                              (int64_t)(ch * BS + off) * XC) =
        *reinterpret_cast<const uint4*>(&s_k[t * D + ch * XC]);
  }
  for (int i = tid; i < D << tg_log2; i += kThreads) {
    const int t = i & (tg - 1), d = i >> tg_log2;
    const int64_t s = slots[t];
    if (s < 0) continue;
    const int64_t blk = s / BS;
    const int off = (int)(s - blk * BS);
    value_cache[blk * block_stride + j * head_stride + (int64_t)d * BS + off] = s_v[t * D + d];
  }
}

template <typename T>
hipError_t rotary_qk_typed(const RotaryRows& a, const RotaryArgs& r, hipStream_t stream) {
  constexpr int X = pack_x<T>();
  int lg_log2 = 0;
  while ((1 << lg_log2) < a.head_dim / (2 * X)) ++lg_log2;
  const int rows = a.num_heads + a.num_kv_heads;
  const int nhb = rows;
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
  int tg_log2 = 0;
  while ((1 << tg_log2) < BS) ++tg_log2;
  const int64_t grid =
      ((a.num_tokens + (1 << tg_log2) - 1) >> tg_log2) * (int64_t)g.num_kv_heads;
  hipLaunchKernelGGL((rotary_cache_kernel<T, C, D, BS>), dim3((uint32_t)grid), dim3(kThreads), 0,
                     stream, static_cast<const T*>(a.q), static_cast<const T*>(a.k),
                     static_cast<const T*>(k.v), a.q_stride, a.k_stride, k.v_stride,
                     static_cast<T*>(a.out_q), a.out_q_stride, static_cast<const T*>(a.q_norm),
                     static_cast<const T*>(a.k_norm), a.eps, r, static_cast<C*>(k.key_cache),
                     static_cast<C*>(k.value_cache), k.slot_mapping, a.num_tokens,
                     g.num_blocks * BS, g.block_stride, g.head_stride, k.k_scale, k.v_scale,
                     g.num_kv_heads, a.num_heads / g.num_kv_heads, tg_log2);
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
