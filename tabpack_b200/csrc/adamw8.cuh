// AdamW with both moments held in 8 bits.
//
// Storage.  A member's elements are cut into blocks of 128; each block has one fp32 scale per
// moment.  The first moment m is an e4m3 code (sign, 4-bit exponent, 3-bit mantissa, subnormals)
// times max|m| / 448.  The second moment is kept as its root u = sqrt(v), whose logarithm spans
// half as many decades: an unsigned code of 4 exponent and 4 mantissa bits, value
// 2^(e - 15) (1 + f / 16) for code 16 e + f > 0 and 0 for code 0, times max u / 1.9375.  A nonzero
// u never becomes 0 (the lowest code instead): a vanished denominator would blow the step up.
//
// Rounding.  Both are rounded up or down at random, in proportion to the distance, with 16 bits
// each.  Round to nearest would freeze v: one step moves it by (1 - beta2) (g^2 / v - 1), about
// 0.1 %, far inside half a code step (3 %), while the random rounding follows it in the mean.
// The bits come from Philox4x32-10, one call per 4 elements, counter (element / 4, tensor, member,
// step): they depend on neither the launch nor the sharding of the members.
//
// Everything a code depends on is computed in fp32 with one rounding per operation (no fused
// multiply-add), so a stored state does not depend on how the compiler contracts.  The parameter
// update uses the unrounded moments and the approximate reciprocal and division (2 ulp), below the
// rounding of p itself.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tp {

constexpr int ADAMW8_BLOCK = 128;        // elements per scale: one warp, four consecutive elements a lane
constexpr int ADAMW8_WARPS = 8;
constexpr int ADAMW8_TILE = 32;          // blocks of one CTA
constexpr float ADAMW8_TINY = 7.8886090522101181e-31f;  // 2^-100: a block below it is stored as zeros

struct AdamW8Scalars {
  const float* lr;
  const float* beta1;
  const float* beta2;
  const float* eps;
  const float* wd;
  float lr_s, beta1_s, beta2_s, eps_s;
  float one_m_b1_s, one_m_b2_s;  // host double precision, rounded once
  float wd_s, wd_mult_s;         // 1 - lr * wd (all scalar)
  float step_size_s;             // lr / (1 - beta1^step) when lr, beta1 and step are scalar
  float bc1_s, inv_sqrt_bc2_s;   // scalar beta and step
  int64_t step;
  uint32_t ks[20];               // Philox key schedule
  uint32_t member_base;
};

struct AdamW8Tensors {
  tp_opt8_tensor t[TP_MAX_OPT_TENSORS];
  uint32_t tile0[TP_MAX_OPT_TENSORS + 1];        // first tile of each tensor; one tile = one CTA's blocks
  uint32_t member_tiles[TP_MAX_OPT_TENSORS];     // tiles of one member
  int n;
};

struct AdamW8Member {
  float mult, b1, one_m_b1, b2, one_m_b2, step_size, inv_sqrt_bc2, eps;
};

// 1 - b^t from 1 - b, without the cancellation of a power next to 1 (and, for a scalar b, without
// the rounding of b itself: 1 - (float)0.999 is off by 1e-5 relative).
__device__ __forceinline__ float bias_correction(float one_m_b, float t) { return -expm1f(t * log1pf(-one_m_b)); }

__device__ __forceinline__ AdamW8Member adamw8_member(const AdamW8Scalars& s, int m, const int64_t* steps) {
  AdamW8Member c;
  const float lr = s.lr ? s.lr[m] : s.lr_s;
  c.b1 = s.beta1 ? s.beta1[m] : s.beta1_s;
  c.b2 = s.beta2 ? s.beta2[m] : s.beta2_s;
  c.one_m_b1 = s.beta1 ? __fsub_rn(1.0f, c.b1) : s.one_m_b1_s;
  c.one_m_b2 = s.beta2 ? __fsub_rn(1.0f, c.b2) : s.one_m_b2_s;
  c.eps = s.eps ? s.eps[m] : s.eps_s;
  c.mult = (s.lr || s.wd) ? 1.0f - lr * (s.wd ? s.wd[m] : s.wd_s) : s.wd_mult_s;
  const float t = (float)(steps ? steps[m] : s.step);
  const float bc1 = (s.beta1 || steps) ? bias_correction(c.one_m_b1, t) : s.bc1_s;
  c.step_size = (s.lr || s.beta1 || steps) ? lr / bc1 : s.step_size_s;
  c.inv_sqrt_bc2 = (s.beta2 || steps) ? rsqrtf(bias_correction(c.one_m_b2, t)) : s.inv_sqrt_bc2_s;
  return c;
}

__device__ __forceinline__ float4 adamw8_load_first(uint32_t c, float scale) {
  const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), __NV_E4M3));
  const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3));
  const float2 x = __half22float2(a), y = __half22float2(b);
  return make_float4(__fmul_rn(x.x, scale), __fmul_rn(x.y, scale), __fmul_rn(y.x, scale), __fmul_rn(y.y, scale));
}

__device__ __forceinline__ float adamw8_load_root(uint32_t code, float scale) {
  const float v = code ? __uint_as_float((code + (112u << 4)) << 19) : 0.0f;
  return __fmul_rn(v, scale);
}

// e4m3 code of x / scale (inv = 1 / scale), rounded with the 16 random bits r.
__device__ __forceinline__ uint32_t adamw8_store_first(float x, float inv, uint32_t r) {
  const float y = fminf(__fmul_rn(fabsf(x), inv), 448.0f);
  const uint32_t normal = ((__float_as_uint(y) + (r << 4)) >> 20) - (120u << 3);
  const uint32_t small = (uint32_t)__fadd_rn(__fmul_rn(y, 512.0f), __fmul_rn((float)r, 1.0f / 65536.0f));
  return (y >= 0.015625f ? normal : small) | (x < 0.0f ? 128u : 0u);
}

// e4m4 code of u / scale.
__device__ __forceinline__ uint32_t adamw8_store_root(float u, float inv, uint32_t r) {
  const float y = fminf(__fmul_rn(u, inv), 1.9375f);
  const int code = (int)((__float_as_uint(y) + (r << 3)) >> 19) - (112 << 4);
  return u > 0.0f ? (uint32_t)min(max(code, 1), 255) : 0u;
}

// Scale and reciprocal of a block whose largest magnitude has the bits `big`.  A block that is
// next to nothing is stored as zeros (its reciprocal would overflow); one with an infinity or a NaN
// gets a NaN scale and zero codes, so that every moment of the block reads as NaN.
__device__ __forceinline__ void adamw8_scale(uint32_t big, float top, float& scale, float& inv) {
  const float b = __uint_as_float(big);
  scale = 0.0f;
  inv = 0.0f;
  if (big >= 0x7F800000u) {
    scale = __uint_as_float(0x7FC00000u);
  } else if (b >= ADAMW8_TINY) {
    scale = __fmul_rn(b, 1.0f / top);
    inv = __fdiv_rn(1.0f, scale);
  }
}

// The tensor, member and first block of tile `tile`.
__device__ __forceinline__ int adamw8_tensor_of(const AdamW8Tensors& ts, uint32_t tile) {
  int i = 0;
  while (i + 1 < ts.n && tile >= ts.tile0[i + 1]) ++i;
  return i;
}

// One warp takes one block of 128 elements at a time: lane l holds elements 4 l .. 4 l + 3, the two
// block maxima are warp reductions.
__global__ void __launch_bounds__(32 * ADAMW8_WARPS) adamw8_kernel(const __grid_constant__ AdamW8Tensors ts,
                                                                   const __grid_constant__ AdamW8Scalars s) {
  const int ti = adamw8_tensor_of(ts, blockIdx.x);
  const tp_opt8_tensor& T = ts.t[ti];
  const uint32_t local = blockIdx.x - ts.tile0[ti];
  const int m = (int)(local / ts.member_tiles[ti]);
  const int64_t inner = T.inner;
  const int64_t nb = (inner + ADAMW8_BLOCK - 1) / ADAMW8_BLOCK;
  const int64_t first = (int64_t)(local % ts.member_tiles[ti]) * ADAMW8_TILE;
  const int lane = lane_id();
  const AdamW8Member c = adamw8_member(s, m, T.step);
  const uint32_t step = (uint32_t)(T.step ? T.step[m] : s.step);
  float* P = T.p + m * inner;
  const float* G = T.grad + m * inner;
  uint8_t* M = T.exp_avg + m * inner;
  uint8_t* V = T.exp_avg_sq + m * inner;
  float* MS = T.exp_avg_scale + m * nb;
  float* VS = T.exp_avg_sq_scale + m * nb;
  const bool vec = (inner & 3) == 0 &&
                   ((reinterpret_cast<uintptr_t>(T.p) | reinterpret_cast<uintptr_t>(T.grad)) & 15u) == 0 &&
                   ((reinterpret_cast<uintptr_t>(T.exp_avg) | reinterpret_cast<uintptr_t>(T.exp_avg_sq)) & 3u) == 0;
  const int64_t last = min(nb, first + ADAMW8_TILE);
  for (int64_t b = first + warp_id(); b < last; b += ADAMW8_WARPS) {
    const int64_t e = b * ADAMW8_BLOCK + 4 * lane;
    const int have = (int)max((int64_t)0, min((int64_t)4, inner - e));
    float p[4] = {0, 0, 0, 0}, g[4] = {0, 0, 0, 0};
    uint32_t mc = 0, vc = 0;
    if (vec && have == 4) {
      const float4 p4 = *reinterpret_cast<const float4*>(P + e);
      const float4 g4 = __ldcs(reinterpret_cast<const float4*>(G + e));
      p[0] = p4.x, p[1] = p4.y, p[2] = p4.z, p[3] = p4.w;
      g[0] = g4.x, g[1] = g4.y, g[2] = g4.z, g[3] = g4.w;
      mc = *reinterpret_cast<const uint32_t*>(M + e);
      vc = *reinterpret_cast<const uint32_t*>(V + e);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < have) {
          p[j] = P[e + j];
          g[j] = G[e + j];
          mc |= (uint32_t)M[e + j] << (8 * j);
          vc |= (uint32_t)V[e + j] << (8 * j);
        }
    }
    const float4 m4 = adamw8_load_first(mc, MS[b]);
    const float us = VS[b];
    float mm[4] = {m4.x, m4.y, m4.z, m4.w}, u[4];
    uint32_t mbig = 0, ubig = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float u0 = adamw8_load_root((vc >> (8 * j)) & 0xFFu, us);
      mm[j] = __fadd_rn(__fmul_rn(mm[j], c.b1), __fmul_rn(g[j], c.one_m_b1));
      u[j] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(u0, u0), c.b2), __fmul_rn(__fmul_rn(g[j], g[j]), c.one_m_b2)));
      if (j >= have) mm[j] = u[j] = 0.0f;
      mbig = max(mbig, __float_as_uint(fabsf(mm[j])));
      ubig = max(ubig, __float_as_uint(u[j]) & 0x7FFFFFFFu);
      p[j] = p[j] * c.mult - c.step_size * __fdividef(mm[j], u[j] * c.inv_sqrt_bc2 + c.eps);
    }
    mbig = __reduce_max_sync(0xFFFFFFFFu, mbig);
    ubig = __reduce_max_sync(0xFFFFFFFFu, ubig);
    float ms, minv, vs, vinv;
    adamw8_scale(mbig, 448.0f, ms, minv);
    adamw8_scale(ubig, 1.9375f, vs, vinv);
    const uint4 r = philox4x32_10_ks(make_uint4((uint32_t)(e >> 2), T.id, s.member_base + (uint32_t)m, step), s.ks);
    const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
    uint32_t mo = 0, vo = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (minv > 0.0f) mo |= adamw8_store_first(mm[j], minv, rw[j] & 0xFFFFu) << (8 * j);
      if (vinv > 0.0f) vo |= adamw8_store_root(u[j], vinv, rw[j] >> 16) << (8 * j);
    }
    if (vec && have == 4) {
      *reinterpret_cast<float4*>(P + e) = make_float4(p[0], p[1], p[2], p[3]);
      *reinterpret_cast<uint32_t*>(M + e) = mo;
      *reinterpret_cast<uint32_t*>(V + e) = vo;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < have) {
          P[e + j] = p[j];
          M[e + j] = (uint8_t)(mo >> (8 * j));
          V[e + j] = (uint8_t)(vo >> (8 * j));
        }
    }
    __syncwarp();  // every lane has read the block's scales
    if (lane == 0) {
      MS[b] = ms;
      VS[b] = vs;
    }
  }
}

struct AdamW8Moments {
  tp_opt8_values t[TP_MAX_OPT_TENSORS];
  uint32_t tile0[TP_MAX_OPT_TENSORS + 1];
  uint32_t member_tiles[TP_MAX_OPT_TENSORS];
  int n;
};

// The moments that the codes stand for: m and v = u^2, in fp32 or bf16.
template <typename T>
__global__ void __launch_bounds__(32 * ADAMW8_WARPS) adamw8_moments_kernel(const __grid_constant__ AdamW8Moments ts) {
  int ti = 0;
  while (ti + 1 < ts.n && blockIdx.x >= ts.tile0[ti + 1]) ++ti;
  const tp_opt8_values& A = ts.t[ti];
  const uint32_t local = blockIdx.x - ts.tile0[ti];
  const int64_t m = local / ts.member_tiles[ti];
  const int64_t inner = A.inner;
  const int64_t nb = (inner + ADAMW8_BLOCK - 1) / ADAMW8_BLOCK;
  const int64_t first = (int64_t)(local % ts.member_tiles[ti]) * ADAMW8_TILE;
  const int64_t last = min(nb, first + ADAMW8_TILE);
  for (int64_t b = first + warp_id(); b < last; b += ADAMW8_WARPS) {
    const float ms = A.exp_avg_scale[m * nb + b], us = A.exp_avg_sq_scale[m * nb + b];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t e = b * ADAMW8_BLOCK + 32 * j + lane_id();
      if (e < inner) {
        const float x = adamw8_load_first(A.exp_avg[m * inner + e], ms).x;
        const float u = adamw8_load_root(A.exp_avg_sq[m * inner + e], us);
        reinterpret_cast<T*>(A.m)[m * inner + e] = from_f32<T>(x);
        reinterpret_cast<T*>(A.v)[m * inner + e] = from_f32<T>(__fmul_rn(u, u));
      }
    }
  }
}

}  // namespace tp
