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
// update uses the unrounded moments and an approximate reciprocal (1 ulp), below the rounding of p.
//
// Bound: 16.1 bytes an element against some 90 instructions (a fifth of them the random bits), near
// the point where the SM's issue slots and the memory take equally long.  So the fp32 arithmetic is
// done in pairs (f32x2), the codes of a block are formed without the rules for subnormals, zeros and
// empty blocks where a vote says that none is there, and the next blocks are on their way to shared
// memory meanwhile.  209 M elements: 610 to 617 us, 5.5 TB/s, 86 % of a copy's rate.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace tp {

constexpr int ADAMW8_BLOCK = 128;        // elements per scale: one warp, four consecutive elements a lane
constexpr int ADAMW8_WARPS = 4;
constexpr int ADAMW8_STAGES = 4;         // blocks of a warp on the way or in use, a power of two
constexpr int ADAMW8_STAGE = 32 * 40;    // bytes: p, g (16 a lane), both codes (4 a lane)
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
  int tile_blocks;                               // blocks of one tile, 4 to 64
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
  c.eps = fmaxf(s.eps ? s.eps[m] : s.eps_s, 1.17549435e-38f);  // the denominator's reciprocal stays finite
  c.mult = (s.lr || s.wd) ? 1.0f - lr * (s.wd ? s.wd[m] : s.wd_s) : s.wd_mult_s;
  const float t = (float)(steps ? steps[m] : s.step);
  const float bc1 = (s.beta1 || steps) ? bias_correction(c.one_m_b1, t) : s.bc1_s;
  c.step_size = (s.lr || s.beta1 || steps) ? lr / bc1 : s.step_size_s;
  c.inv_sqrt_bc2 = (s.beta2 || steps) ? rsqrtf(bias_correction(c.one_m_b2, t)) : s.inv_sqrt_bc2_s;
  return c;
}

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Correctly rounded square roots of two numbers from 2^-94 up (others: something within an ulp, or
// NaN for 0, infinities and NaN).  Goldschmidt's iteration on s ~ sqrt(v) and h ~ 1 / (2 sqrt(v)) from
// the approximate reciprocal root, then Markstein's correction s + h (v - s^2) with the residual exact in
// a fused multiply-add (P. Markstein, IA-64 and Elementary Functions, 2000).  In pairs it takes half
// the instructions of two calls; tp_root_check compares it with CUDA's over every mantissa.
__device__ __forceinline__ f32x2 sqrt2(f32x2 v) {
  const float2 f = halves(v);
  float r0, r1;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(f.x));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(f.y));
  // h with its sign changed, so that no product needs one: s + (-h) (s^2 - v)
  const f32x2 r = pair(r0, r1);
  f32x2 s = mul2(v, r), h = mul2(r, pair(-0.5f, -0.5f));
  const f32x2 e = fma2(s, h, pair(0.5f, 0.5f));
  s = fma2(s, e, s);
  h = fma2(h, e, h);
  return fma2(fma2(s, s, pair(-f.x, -f.y)), h, s);
}

__global__ void root_check_kernel(uint32_t first, uint32_t count, unsigned long long* differ) {
  unsigned long long n = 0;
  // 64 bits: next to the largest count a 32-bit number would start again from 0
  for (uint64_t i = blockIdx.x * blockDim.x + threadIdx.x; i < count; i += gridDim.x * blockDim.x) {
    const float v = __uint_as_float(first + (uint32_t)i);
    const float2 s = halves(sqrt2(pair(v, v)));
    n += __float_as_uint(s.x) != __float_as_uint(__fsqrt_rn(v));
    n += __float_as_uint(s.y) != __float_as_uint(__fsqrt_rn(v));
  }
  if (n) atomicAdd(differ, n);
}

// Four e4m3 codes -> their values times `scale`, as pairs.
__device__ __forceinline__ void adamw8_load_first(uint32_t c, f32x2 scale, f32x2 (&m)[2]) {
  const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xFFFFu), __NV_E4M3));
  const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3));
  const float2 x = __half22float2(a), y = __half22float2(b);
  m[0] = mul2(pair(x.x, x.y), scale);
  m[1] = mul2(pair(y.x, y.y), scale);
}

// Four e4m4 codes: code c > 0 is the fp32 number with the bits (c + 112 * 16) << 19.
__device__ __forceinline__ void adamw8_load_root(uint32_t c, f32x2 scale, f32x2 (&u)[2]) {
  constexpr uint32_t bias = (112u << 4) << 19;
  float v[4] = {__uint_as_float((c & 0xFFu) * (1u << 19) + bias), __uint_as_float((c & 0xFF00u) * (1u << 11) + bias),
                __uint_as_float((c & 0xFF0000u) * (1u << 3) + bias), __uint_as_float((c >> 24) * (1u << 19) + bias)};
  if (((c - 0x01010101u) & ~c & 0x80808080u) != 0) {  // a zero byte
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((c >> (8 * j)) & 0xFFu) == 0) v[j] = 0.0f;
  }
  u[0] = mul2(pair(v[0], v[1]), scale);
  u[1] = mul2(pair(v[2], v[3]), scale);
}

// Subnormal e4m3 codes, y < 2^-6: floor(512 y + r / 2^16), left in the number's low byte by adding
// 2^23 towards minus infinity.  `r8`: the 16 random bits r times 2^8; half of it is the fraction of
// 1 + r / 2^16.
__device__ __forceinline__ uint32_t adamw8_small_first(float y, uint32_t r8) {
  const float r = __fsub_rn(__uint_as_float(0x3F800000u | r8 >> 1), 1.0f);
  return __float_as_uint(__fadd_rd(__fmaf_rn(y, 512.0f, r), 8388608.0f));
}

// e4m4 code of u / scale = y.
__device__ __forceinline__ uint32_t adamw8_code_root(float u, float y, uint32_t r) {
  const int code = (int)((__float_as_uint(y) + (r << 3)) >> 19) - (112 << 4);
  return u > 0.0f ? (uint32_t)min(max(code, 1), 255) : 0u;
}

__device__ __forceinline__ uint32_t bytes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// The top bytes of four words.
__device__ __forceinline__ uint32_t top4(const uint32_t (&w)[4]) {
  return __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
}

// Philox4x32-10 over the first counter word with the other three fixed: the products of the first
// round's third word and the second round's first do not depend on it.
struct PhiloxGroup {
  uint32_t a, b, y, w;  // w ^ key of the first round; second round: lo ^ key, hi ^ key, lo
  const uint32_t* ks;
  __device__ PhiloxGroup(uint32_t c1, uint32_t c2, uint32_t c3, const uint32_t* keys) : ks(keys) {
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * c2;
    a = c3 ^ ks[1];
    y = (uint32_t)p1 ^ ks[2];
    const uint64_t p0 = (uint64_t)0xD2511F53u * ((uint32_t)(p1 >> 32) ^ c1 ^ ks[0]);
    b = (uint32_t)(p0 >> 32) ^ ks[3];
    w = (uint32_t)p0;
  }
  __device__ uint4 at(uint32_t c0) const {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0;
    const uint64_t p1 = (uint64_t)0xCD9E8D57u * ((uint32_t)(p0 >> 32) ^ a);
    uint4 c = make_uint4((uint32_t)(p1 >> 32) ^ y, (uint32_t)p1, (uint32_t)p0 ^ b, w);
#pragma unroll
    for (int i = 2; i < 10; ++i) {
      const uint64_t q0 = (uint64_t)0xD2511F53u * c.x, q1 = (uint64_t)0xCD9E8D57u * c.z;
      c = make_uint4((uint32_t)(q1 >> 32) ^ c.y ^ ks[2 * i], (uint32_t)q1, (uint32_t)(q0 >> 32) ^ c.w ^ ks[2 * i + 1],
                     (uint32_t)q0);
    }
    return c;
  }
};

// One lane's share of a block.
struct AdamW8Lane {
  float p[4], g[4];
  uint32_t m, v;  // codes
  float ms, vs;   // the block's scales
};

// Element j of lane `lane`: consecutive elements with vector access, else 32 apart, so that both
// ways neighbouring lanes touch neighbouring memory.
template <bool VEC>
__device__ __forceinline__ int adamw8_at(int lane, int j) {
  return VEC ? 4 * lane + j : lane + 32 * j;
}

// A lane's place in the warp's current block.
struct AdamW8Ptr {
  float* p;
  const float* g;
  uint8_t* m;
  uint8_t* v;
  __device__ void next() {
    p += ADAMW8_BLOCK;
    g += ADAMW8_BLOCK;
    m += ADAMW8_BLOCK;
    v += ADAMW8_BLOCK;
  }
};

// Vector access: block `ahead` blocks on, copied to `stage` (each lane reads back what it
// copied); `left`: elements of the member from that block's first on.
__device__ __forceinline__ void adamw8_issue(char* stage, const AdamW8Ptr& a, int ahead, int left, int lane) {
  const int o = ahead * ADAMW8_BLOCK;
  char* s16 = stage + 16 * lane;
  char* s4 = stage + 1024 + 4 * lane;
  if (4 * lane < left) {
    cp_async16(smem_u32(s16), a.p + o);
    cp_async16(smem_u32(s16) + 512, a.g + o);
    cp_async4(smem_u32(s4), a.m + o);
    cp_async4(smem_u32(s4) + 128, a.v + o);
  } else if (left > 0) {  // behind the member's end
    *reinterpret_cast<uint4*>(s16) = *reinterpret_cast<uint4*>(s16 + 512) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint32_t*>(s4) = *reinterpret_cast<uint32_t*>(s4 + 128) = 0;
  }
  cp_async_commit();
}

__device__ __forceinline__ void adamw8_take(AdamW8Lane& x, const char* stage, int lane) {
  const float4 p4 = *reinterpret_cast<const float4*>(stage + 16 * lane);
  const float4 g4 = *reinterpret_cast<const float4*>(stage + 512 + 16 * lane);
  x.p[0] = p4.x, x.p[1] = p4.y, x.p[2] = p4.z, x.p[3] = p4.w;
  x.g[0] = g4.x, x.g[1] = g4.y, x.g[2] = g4.z, x.g[3] = g4.w;
  x.m = *reinterpret_cast<const uint32_t*>(stage + 1024 + 4 * lane);
  x.v = *reinterpret_cast<const uint32_t*>(stage + 1152 + 4 * lane);
}

// Any alignment, the block `AHEAD` blocks on into registers.
template <int AHEAD>
__device__ __forceinline__ void adamw8_fetch(AdamW8Lane& x, const AdamW8Ptr& a, int left, int lane) {
  constexpr int o = AHEAD * ADAMW8_BLOCK;
  uint32_t mb[4], vb[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = lane + 32 * j < left;
    x.p[j] = in ? a.p[o + 32 * j] : 0.0f;
    x.g[j] = in ? __ldcs(a.g + o + 32 * j) : 0.0f;
    mb[j] = in ? a.m[o + 32 * j] : 0u;
    vb[j] = in ? a.v[o + 32 * j] : 0u;
  }
  x.m = bytes4(mb[0], mb[1], mb[2], mb[3]);
  x.v = bytes4(vb[0], vb[1], vb[2], vb[3]);
}

// One block; returns its new scales.
template <bool VEC>
__device__ __forceinline__ float2 adamw8_block(const AdamW8Lane& x, const AdamW8Member& c, const AdamW8Ptr& a, int left,
                                             int lane, const PhiloxGroup& philox, uint32_t group, uint32_t* words) {
  f32x2 m[2], u[2];
  adamw8_load_first(x.m, pair(x.ms, x.ms), m);
  adamw8_load_root(x.v, pair(x.vs, x.vs), u);
  float mm[4], uu[4], p[4];
  f32x2 v[2];
  const f32x2 b1 = pair(c.b1, c.b1), o1 = pair(c.one_m_b1, c.one_m_b1), b2 = pair(c.b2, c.b2),
              o2 = pair(c.one_m_b2, c.one_m_b2);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 g = pair(x.g[2 * h], x.g[2 * h + 1]);
    // the sums one by one: the assembler would contract a paired product and sum
    const float2 ma = halves(mul2(m[h], b1)), mb = halves(mul2(g, o1));
    const float2 va = halves(mul2(mul2(u[h], u[h]), b2)), vb = halves(mul2(mul2(g, g), o2));
    mm[2 * h] = __fadd_rn(ma.x, mb.x), mm[2 * h + 1] = __fadd_rn(ma.y, mb.y);
    m[h] = pair(mm[2 * h], mm[2 * h + 1]);
    v[h] = pair(__fadd_rn(va.x, vb.x), __fadd_rn(va.y, vb.y));
    u[h] = sqrt2(v[h]);
    const float2 uf = halves(u[h]);
    uu[2 * h] = uf.x, uu[2 * h + 1] = uf.y;
  }
  // the block's largest magnitudes (as integers: a NaN is above everything) and the smallest root
  float umin = fminf(fminf(uu[0], uu[1]), fminf(uu[2], uu[3]));
  float umax = max_nan(max_nan(uu[0], uu[1]), max_nan(uu[2], uu[3]));
  if (__any_sync(0xFFFFFFFFu, !(umin >= 7.1e-15f && umax < INFINITY))) {
    // outside sqrt2's range (2^-94 up): zeros, next to zeros, infinities, NaN
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float2 vf = halves(v[h]);
      uu[2 * h] = __fsqrt_rn(vf.x), uu[2 * h + 1] = __fsqrt_rn(vf.y);
      u[h] = pair(uu[2 * h], uu[2 * h + 1]);
    }
    if (left < ADAMW8_BLOCK) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (adamw8_at<VEC>(lane, j) >= left) mm[j] = uu[j] = 0.0f;
    }
    umin = fminf(fminf(uu[0], uu[1]), fminf(uu[2], uu[3]));
    umax = max_nan(max_nan(uu[0], uu[1]), max_nan(uu[2], uu[3]));
  }
  uint32_t mbig = __float_as_uint(max_nan(max_nan(fabsf(mm[0]), fabsf(mm[1])), max_nan(fabsf(mm[2]), fabsf(mm[3]))));
  mbig = __reduce_max_sync(0xFFFFFFFFu, mbig);
  const uint32_t ubig = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(umax));
  // p (1 - lr wd) - step m / (u / sqrt(bc2) + eps)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 den = halves(fma2(u[h], pair(c.inv_sqrt_bc2, c.inv_sqrt_bc2), pair(c.eps, c.eps)));
    const f32x2 up = mul2(mul2(m[h], pair(-c.step_size, -c.step_size)), pair(reciprocal(den.x), reciprocal(den.y)));
    const float2 pf = halves(fma2(pair(x.p[2 * h], x.p[2 * h + 1]), pair(c.mult, c.mult), up));
    p[2 * h] = pf.x, p[2 * h + 1] = pf.y;
  }
  // even lanes form the first moment's scale, odd ones the root's
  float scale = 0.0f, inv = 0.0f;
  {
    const uint32_t big = lane & 1 ? ubig : mbig;
    if (big >= 0x7F800000u) {
      scale = __uint_as_float(0x7FC00000u);  // every moment of the block reads as NaN
    } else if (__uint_as_float(big) >= ADAMW8_TINY) {
      scale = __fmul_rn(__uint_as_float(big), lane & 1 ? 1.0f / 1.9375f : 1.0f / 448.0f);
      inv = __frcp_rn(scale);
    }
  }
  const float minv = __shfl_sync(0xFFFFFFFFu, inv, 0), vinv = __shfl_sync(0xFFFFFFFFu, inv, 1);
  const uint4 rnd = philox.at(group);
  uint32_t rw[4] = {rnd.x, rnd.y, rnd.z, rnd.w};
  if (!VEC) {  // the words of elements 4 l .. 4 l + 3 to the lanes that hold those elements
    reinterpret_cast<uint4*>(words)[lane] = rnd;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) rw[j] = words[lane + 32 * j];
    __syncwarp();
  }
  float ym[4], yu[4];  // signed and not: the first codes drop the sign bit
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const float2 y = halves(mul2(pair(mm[2 * h], mm[2 * h + 1]), pair(minv, minv)));
    const float2 z = halves(mul2(pair(uu[2 * h], uu[2 * h + 1]), pair(vinv, vinv)));
    ym[2 * h] = y.x, ym[2 * h + 1] = y.y;
    yu[2 * h] = z.x, yu[2 * h + 1] = z.y;
  }
  // Codes of normal values: the number's bits plus the random ones below the code's last place, then
  // the code's 8 bits, shifted into the top byte (e4m3: exponent offset 120, whose 0xC0 in that byte
  // the packed word takes off; e4m4: offset 112, 0).  A value scaled by the rounded reciprocal
  // exceeds the code's largest by 3 ulp at most, which the 16 random bits (16 and 8 ulp short of a
  // carry) do not carry over.
  uint32_t mc[4], vc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mc[j] = __float_as_uint(ym[j]) * 16u + __byte_perm(rw[j], 0, 0x4104);
    vc[j] = __float_as_uint(yu[j]) * 32u + __byte_perm(rw[j], 0, 0x4324);
  }
  uint32_t mo = (top4(mc) & 0x7F7F7F7Fu) ^ 0x40404040u, vo = top4(vc);
  const bool msmall =
      !(fminf(fminf(fabsf(ym[0]), fabsf(ym[1])), fminf(fabsf(ym[2]), fabsf(ym[3]))) >= 0.015625f);  // 2^-6
  const bool usmall = !(__fmul_rn(umin, vinv) >= 3.2424927e-05f);                       // 2^-15 (1 + 1 / 16)
  if (__any_sync(0xFFFFFFFFu, msmall)) {
    uint32_t pick = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      mc[j] = adamw8_small_first(fabsf(ym[j]), __byte_perm(rw[j], 0, 0x4104));
      if (!(fabsf(ym[j]) >= 0.015625f)) pick |= 0xFFu << (8 * j);
    }
    mo = (mo & ~pick) | (bytes4(mc[0], mc[1], mc[2], mc[3]) & pick);
    if (!(minv > 0.0f)) mo = 0;
  }
  if (__any_sync(0xFFFFFFFFu, usmall)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) vc[j] = vinv > 0.0f ? adamw8_code_root(uu[j], yu[j], rw[j] >> 16) : 0u;
    vo = bytes4(vc[0], vc[1], vc[2], vc[3]);
  }
  // the signs are the top bits of the values
  const uint32_t mb[4] = {__float_as_uint(mm[0]), __float_as_uint(mm[1]), __float_as_uint(mm[2]), __float_as_uint(mm[3])};
  if (minv > 0.0f) mo |= top4(mb) & 0x80808080u;
  if (VEC) {
    if (4 * lane < left) {
      *reinterpret_cast<float4*>(a.p) = make_float4(p[0], p[1], p[2], p[3]);
      *reinterpret_cast<uint32_t*>(a.m) = mo;
      *reinterpret_cast<uint32_t*>(a.v) = vo;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (lane + 32 * j < left) {
        a.p[32 * j] = p[j];
        a.m[32 * j] = (uint8_t)(mo >> (8 * j));
        a.v[32 * j] = (uint8_t)(vo >> (8 * j));
      }
    }
  }
  return make_float2(__shfl_sync(0xFFFFFFFFu, scale, 0), __shfl_sync(0xFFFFFFFFu, scale, 1));
}

// The warp's share of a tile, `run` blocks from `run` times its number on (`blocks` in all).  `a`
// points to the tile's first element, `left` are the elements of the member from there on.  Lane i
// holds the scales of the warp's i-th block from first to last: one load and one store for the run.
// (Scales stored block by block, 4 bytes into sectors that other warps read, cost half the time:
// 850 us against 511 us for the same traffic without them, 209 M elements.)
template <bool VEC>
__device__ __forceinline__ void adamw8_tile(const AdamW8Member& c, AdamW8Ptr a, float* ms, float* vs, int run, int blocks,
                                            int left, const PhiloxGroup& philox, uint32_t group, char* stages) {
  const int lane = lane_id(), first = warp_id() * run, at = first * ADAMW8_BLOCK + (VEC ? 4 * lane : lane);
  const int n = min(run, blocks - first);
  if (n <= 0) return;
  a.p += at;
  a.g += at;
  a.m += at;
  a.v += at;
  left -= first * ADAMW8_BLOCK;
  group += first * (ADAMW8_BLOCK / 4) + lane;
  float sm = 0.0f, sv = 0.0f;
  if (lane < n) sm = ms[first + lane], sv = vs[first + lane];
  AdamW8Lane next;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < ADAMW8_STAGES - 1; ++i)
      adamw8_issue(stages + i * ADAMW8_STAGE, a, i, i < n ? left - i * ADAMW8_BLOCK : 0, lane);
  } else {
    adamw8_fetch<0>(next, a, left, lane);
  }
  for (int i = 0; i < n; ++i) {
    AdamW8Lane x;
    if constexpr (VEC) {
      cp_async_wait<ADAMW8_STAGES - 2>();
      adamw8_take(x, stages + i % ADAMW8_STAGES * ADAMW8_STAGE, lane);
      constexpr int ahead = ADAMW8_STAGES - 1;  // into the stage of the block before: read, and free
      adamw8_issue(stages + (i + ahead) % ADAMW8_STAGES * ADAMW8_STAGE, a, ahead,
                   i + ahead < n ? left - ahead * ADAMW8_BLOCK : 0, lane);
    } else {
      x = next;
      if (i + 1 < n) adamw8_fetch<1>(next, a, left - ADAMW8_BLOCK, lane);
    }
    x.ms = __shfl_sync(0xFFFFFFFFu, sm, i);
    x.vs = __shfl_sync(0xFFFFFFFFu, sv, i);
    const float2 scale = adamw8_block<VEC>(x, c, a, left, lane, philox, group, reinterpret_cast<uint32_t*>(stages));
    if (lane == i) sm = scale.x, sv = scale.y;
    a.next();
    left -= ADAMW8_BLOCK;
    group += ADAMW8_BLOCK / 4;
  }
  if (lane < n) ms[first + lane] = sm, vs[first + lane] = sv;
}

// One warp takes one block of 128 elements at a time, four a lane; the block's maxima are warp
// reductions.  The grid is one CTA per tile of a member's blocks, over all members and tensors.
// Six CTAs of four warps an SM, 78 registers a thread and no spills: 610 to 617 us for 209 M elements.  Seven
// CTAs (72 registers, no spills) take 627 to 632, eight (64, with spills) 624 to 635, three of eight warps 644
// to 651.
__global__ void __launch_bounds__(32 * ADAMW8_WARPS, 6) adamw8_kernel(const __grid_constant__ AdamW8Tensors ts,
                                                                      const __grid_constant__ AdamW8Scalars s) {
  __shared__ AdamW8Member shared;
  __shared__ __align__(16) char stages[ADAMW8_WARPS][ADAMW8_STAGES * ADAMW8_STAGE];
  int ti = 0;
  while (ti + 1 < ts.n && blockIdx.x >= ts.tile0[ti + 1]) ++ti;
  const tp_opt8_tensor& T = ts.t[ti];
  const uint32_t local = blockIdx.x - ts.tile0[ti];
  const uint32_t m = local / ts.member_tiles[ti];
  // the coefficients take a logarithm and an exponential each: one warp forms them
  if (warp_id() == 0) {
    const AdamW8Member c = adamw8_member(s, (int)m, T.step);
    if (lane_id() == 0) shared = c;
  }
  __syncthreads();
  const AdamW8Member c = shared;
  const int64_t inner = T.inner;
  const int64_t nb = (inner + ADAMW8_BLOCK - 1) / ADAMW8_BLOCK;
  const int64_t first = (int64_t)(local - m * ts.member_tiles[ti]) * ts.tile_blocks;
  const int blocks = (int)min((int64_t)ts.tile_blocks, nb - first);
  const int64_t e = m * inner + first * ADAMW8_BLOCK;
  const int left = (int)min((int64_t)ts.tile_blocks * ADAMW8_BLOCK, inner - first * ADAMW8_BLOCK);
  const AdamW8Ptr a = {T.p + e, T.grad + e, T.exp_avg + e, T.exp_avg_sq + e};
  float* ms = T.exp_avg_scale + m * nb + first;
  float* vs = T.exp_avg_sq_scale + m * nb + first;
  const int run = ts.tile_blocks / ADAMW8_WARPS;
  const PhiloxGroup philox(T.id, s.member_base + m, (uint32_t)(T.step ? T.step[m] : s.step), s.ks);
  const uint32_t group = (uint32_t)(first * (ADAMW8_BLOCK / 4));
  const bool vec = (inner & 3) == 0 &&
                   ((reinterpret_cast<uintptr_t>(T.p) | reinterpret_cast<uintptr_t>(T.grad)) & 15u) == 0 &&
                   ((reinterpret_cast<uintptr_t>(T.exp_avg) | reinterpret_cast<uintptr_t>(T.exp_avg_sq)) & 3u) == 0;
  if (vec)
    adamw8_tile<true>(c, a, ms, vs, run, blocks, left, philox, group, stages[warp_id()]);
  else
    adamw8_tile<false>(c, a, ms, vs, run, blocks, left, philox, group, stages[warp_id()]);
}

struct AdamW8Moments {
  tp_opt8_values t[TP_MAX_OPT_TENSORS];
  uint32_t tile0[TP_MAX_OPT_TENSORS + 1];
  uint32_t member_tiles[TP_MAX_OPT_TENSORS];
  int n;
  int tile_blocks;
};

// The moments that the codes stand for: m and v = u^2, in fp32 or bf16.
template <typename T>
__global__ void __launch_bounds__(32 * ADAMW8_WARPS) adamw8_moments_kernel(const __grid_constant__ AdamW8Moments ts) {
  int ti = 0;
  while (ti + 1 < ts.n && blockIdx.x >= ts.tile0[ti + 1]) ++ti;
  const tp_opt8_values& A = ts.t[ti];
  const uint32_t local = blockIdx.x - ts.tile0[ti];
  const uint32_t m = local / ts.member_tiles[ti];
  const int64_t inner = A.inner;
  const int64_t nb = (inner + ADAMW8_BLOCK - 1) / ADAMW8_BLOCK;
  const int64_t first = (int64_t)(local - m * ts.member_tiles[ti]) * ts.tile_blocks;
  const int64_t last = min(nb, first + ts.tile_blocks);
  const uint8_t* mc = A.exp_avg + m * inner;
  const uint8_t* vc = A.exp_avg_sq + m * inner;
  const float* ms = A.exp_avg_scale + m * nb;
  const float* vs = A.exp_avg_sq_scale + m * nb;
  T* mo = reinterpret_cast<T*>(A.m) + m * inner;
  T* vo = reinterpret_cast<T*>(A.v) + m * inner;
  const bool vec = (inner & 3) == 0 &&
                   ((reinterpret_cast<uintptr_t>(A.exp_avg) | reinterpret_cast<uintptr_t>(A.exp_avg_sq)) & 3u) == 0 &&
                   ((reinterpret_cast<uintptr_t>(A.m) | reinterpret_cast<uintptr_t>(A.v)) & (4 * sizeof(T) - 1)) == 0;
  // a run of blocks per warp, lane i with the scales of its i-th; four blocks' codes loaded ahead of use
  const int run = ts.tile_blocks / ADAMW8_WARPS, lane = lane_id();
  const int64_t b0 = first + warp_id() * run;
  const int n = (int)min((int64_t)run, last - b0);
  float sm = 0.0f, sv = 0.0f;
  if (lane < n) sm = ms[b0 + lane], sv = vs[b0 + lane];
  for (int i0 = 0; i0 < n; i0 += 4) {
    uint32_t cm[4], cv[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      cm[k] = cv[k] = 0;
      if (i0 + k >= n) continue;
      const int64_t e = (b0 + i0 + k) * ADAMW8_BLOCK;
      const int left = (int)min((int64_t)ADAMW8_BLOCK, inner - e);
      if (vec) {
        if (4 * lane < left) {
          cm[k] = __ldcs(reinterpret_cast<const uint32_t*>(mc + e) + lane);
          cv[k] = __ldcs(reinterpret_cast<const uint32_t*>(vc + e) + lane);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (lane + 32 * j < left) {
            cm[k] |= (uint32_t)mc[e + lane + 32 * j] << (8 * j);
            cv[k] |= (uint32_t)vc[e + lane + 32 * j] << (8 * j);
          }
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i0 + k >= n) break;
      const int64_t e = (b0 + i0 + k) * ADAMW8_BLOCK;
      const int left = (int)min((int64_t)ADAMW8_BLOCK, inner - e);
      const float bm = __shfl_sync(0xFFFFFFFFu, sm, i0 + k), bv = __shfl_sync(0xFFFFFFFFu, sv, i0 + k);
      f32x2 x[2], u[2];
      adamw8_load_first(cm[k], pair(bm, bm), x);
      adamw8_load_root(cv[k], pair(bv, bv), u);
      const float2 x0 = halves(x[0]), x1 = halves(x[1]), u0 = halves(mul2(u[0], u[0])), u1 = halves(mul2(u[1], u[1]));
      if (vec) {
        if (4 * lane >= left) continue;
        if constexpr (sizeof(T) == 2) {
          reinterpret_cast<uint2*>(mo + e)[lane] = make_uint2(pack_bf16x2(x0.x, x0.y), pack_bf16x2(x1.x, x1.y));
          reinterpret_cast<uint2*>(vo + e)[lane] = make_uint2(pack_bf16x2(u0.x, u0.y), pack_bf16x2(u1.x, u1.y));
        } else {
          reinterpret_cast<float4*>(mo + e)[lane] = make_float4(x0.x, x0.y, x1.x, x1.y);
          reinterpret_cast<float4*>(vo + e)[lane] = make_float4(u0.x, u0.y, u1.x, u1.y);
        }
      } else {
        const float xs[4] = {x0.x, x0.y, x1.x, x1.y}, us[4] = {u0.x, u0.y, u1.x, u1.y};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (lane + 32 * j < left) {
            mo[e + lane + 32 * j] = from_f32<T>(xs[j]);
            vo[e + lane + 32 * j] = from_f32<T>(us[j]);
          }
      }
    }
  }
}

}  // namespace tp
