// Layer norm of a pack: member m's rows are normalised over its first n_m columns, then scaled
// and shifted per member and column.  Columns at or beyond n_m are written as zeros and never read.
//
//   xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps), y = xhat w + b
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) with g = dy w;  dw = sum_r dy xhat;  db = sum_r dy
//
// Memory bounds all of it: 4 bytes per element forward and 6 backward in bf16, 10 to 20
// instructions.  Rows of up to NORM_HELD columns stay in the registers of a group of G lanes (4 to
// 512, 16 elements each), so x and dy are read once and the variance is summed around the mean.
// A group walks over rows of one member: the member's w and b, and in the backward the columns' sums,
// stay in registers, while the next rows are on their way to shared memory (asynchronous copies: one
// row ahead in registers left the memory waiting, 192 us instead of 114 for the forward of 16384 rows
// of 8192 in bf16).  The forward takes two rows at a time, which share each reduction's latency.
// Arithmetic is in pairs (f32x2).  Ragged rows need few tests per element: the copies fill x and dy with
// zeros from column n on, forward a factor of 0 there takes the mean off nothing, and backward only
// the written padding is cleared.  Wider rows take the plain kernels at the end.
#pragma once

#include "gemm_simt.cuh"

namespace tp {

struct LayerNormArgs {
  int P, B, W;
  int64_t xm, xr, dym, dyr;  // member and row strides of x and dy, in elements
  const int32_t* n;
  const void* x;
  const float* w;
  const float* b;
  float eps;
  void* y;
  float* mean;
  float* rstd;
  const void* dy;
  void* dx;
  int dx_f32;
  float* dw;
  float* db;
  float* partial;  // (2, P, S, W) when the rows are split
  int S;           // splits of a member's rows
};

constexpr int NORM_E = 16;             // elements of a row in one lane
constexpr int NORM_HELD = 512 * NORM_E;

__device__ __forceinline__ int norm_width(const LayerNormArgs& a, int m) {
  return a.n ? min(max(a.n[m], 0), a.W) : a.W;
}

constexpr int NORM_H = NORM_E / 2;  // pairs

// V neighbouring elements are one vector: 16 bytes, 8 or 4 where all rows start on such boundaries only,
// or one element where nothing is aligned.
template <int BYTES>
struct NormWord {
  typedef uint4 type;
};
template <>
struct NormWord<8> {
  typedef uint2 type;
};
template <>
struct NormWord<4> {
  typedef uint32_t type;
};

template <typename T, int V>
__device__ __forceinline__ void norm_unpack(const char* from, f32x2* f) {
  typedef typename NormWord<V * sizeof(T)>::type Word;
  const Word u = *reinterpret_cast<const Word*>(from);
  uint32_t w[sizeof(Word) / 4];
  memcpy(w, &u, sizeof(Word));
#pragma unroll
  for (int e = 0; e < V / 2; ++e)
    f[e] = sizeof(T) == 2 ? pair(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u))
                          : pair(__uint_as_float(w[(2 * e) % (sizeof(Word) / 4)]),
                                 __uint_as_float(w[(2 * e + 1) % (sizeof(Word) / 4)]));
}

template <typename T, int V>
__device__ __forceinline__ void norm_store(T* p, const float* f) {
  if constexpr (V == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    typedef typename NormWord<V * sizeof(T)>::type Word;
    uint32_t w[sizeof(Word) / 4];
#pragma unroll
    for (int e = 0; e < (int)sizeof(Word) / 4; ++e)
      w[e] = sizeof(T) == 2 ? pack_bf16x2(f[(2 * e) % V], f[(2 * e + 1) % V]) : __float_as_uint(f[e % V]);
    Word u;
    memcpy(&u, w, sizeof(Word));
    *reinterpret_cast<Word*>(p) = u;
  }
}

// A group of G lanes of a block and its sums.
template <int G>
struct NormGroup {
  static constexpr int THREADS = G > 256 ? G : 256, GROUPS = THREADS / G, WARPS = G > 32 ? G / 32 : 1;
  int lane, group;
  float2* red;  // two halves of WARPS pairs per group, used in turn: one barrier per sum is enough
  int half = 0;
  __device__ NormGroup(float2* shared) : lane(threadIdx.x % G), group(threadIdx.x / G) {
    red = shared + group * 2 * WARPS;
  }
  // Sums of u and v over the group, in every lane.
  __device__ float2 sum(float u, float v) {
    if constexpr (G < 32) {
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
        v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
      }
      return make_float2(u, v);
    }
    // the lower half of the warp adds up u, the upper one v: 7 exchanges instead of 10
    const bool upper = lane & 16;
    float t = upper ? v : u;
    t += __shfl_xor_sync(0xFFFFFFFFu, upper ? u : v, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    if constexpr (G > 32) {
      float* r = reinterpret_cast<float*>(red + half * WARPS);
      half ^= 1;
      if (lane % 16 == 0) r[lane / 32 + (upper ? WARPS : 0)] = t;
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(G) : "memory");
      t = r[lane % WARPS + (upper ? WARPS : 0)];
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    }
    return make_float2(__shfl_sync(0xFFFFFFFFu, t, 0), __shfl_sync(0xFFFFFFFFu, t, 16));
  }
};

// Rows of one operand on their way to a lane: its share of a row, K vectors c0(k) .. c0(k) + V - 1,
// is copied to the lane's own part of a ring in shared memory (no barrier: a lane reads only what it
// copied), with zeros from column n on; unaligned rows go through registers, one row ahead.
template <typename T, int V, int G>
struct NormRows {
  static constexpr int K = NORM_E / V, THREADS = NormGroup<G>::THREADS;
  static constexpr int VB = V * sizeof(T);                    // bytes of a vector
  static constexpr int STAGE = V > 1 ? K * THREADS * VB : 0;  // of one row of every group
  const T* p;     // the lane's first element of the next row to come
  int64_t step;   // elements to the row after
  int left;       // columns below n from the lane's first on
  char* ring;
  T next[V > 1 ? 1 : NORM_E];
  __device__ static int c0(int k, int lane) { return (k * G + lane) * V; }
  // Rows first, first + by, ... of a member's `rows`.
  __device__ NormRows(const T* rows, int64_t stride, int first, int by, int lane, int n, char* shared, int stages)
      : p(rows + first * stride + lane * V), step(by * stride), left(n - lane * V), ring(shared + threadIdx.x * VB) {
    if constexpr (V > 1) {  // vectors without a column are never copied
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (left - k * G * V <= 0)
          for (int i = 0; i < stages; ++i)
            *reinterpret_cast<typename NormWord<VB>::type*>(ring + i * STAGE + k * THREADS * VB) = {};
    }
  }
  // The next row, if there is one, into stage `slot`.
  __device__ void issue(int slot, bool valid) {
    if (valid) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int have = left - k * G * V;
        if constexpr (V > 1) {
          const uint32_t to = smem_u32(ring) + slot * STAGE + k * THREADS * VB, bytes = min(have, V) * sizeof(T);
          if constexpr (VB == 16) {
            if (have > 0)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p + k * G * V), "r"(bytes)
                           : "memory");
          } else {
            if (have > 0)
              asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(p + k * G * V), "n"(VB), "r"(bytes)
                           : "memory");
          }
        } else {
          next[k] = have > 0 ? p[k * G] : from_f32<T>(0.f);
        }
      }
    }
    p += step;
    if (V > 1) cp_async_commit();
  }
  __device__ void take(int slot, f32x2 (&f)[NORM_H]) const {
    if constexpr (V > 1) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        norm_unpack<T, V>(ring + slot * STAGE + k * THREADS * VB, f + k * V / 2);
    } else {
#pragma unroll
      for (int k = 0; k < NORM_H; ++k) f[k] = pair(to_f32<T>(next[2 * k]), to_f32<T>(next[2 * k + 1]));
    }
  }
};

// 1 for the lane's columns below n, 0 for the others.
template <int V, int G>
__device__ __forceinline__ void norm_mask(int lane, int n, f32x2 (&f)[NORM_H]) {
#pragma unroll
  for (int h = 0; h < NORM_H; ++h) {
    const int c = (2 * h / V * G + lane) * V + 2 * h % V, d = V == 1 ? c + G : c + 1;
    f[h] = pair(c < n ? 1.f : 0.f, d < n ? 1.f : 0.f);
  }
}

__device__ __forceinline__ float norm_add(const f32x2 (&f)[NORM_H]) {
  f32x2 s = f[0];
#pragma unroll
  for (int h = 1; h < NORM_H; ++h) s = add2(s, f[h]);
  const float2 t = halves(s);
  return t.x + t.y;
}

// Writes a lane's share of a row; `clear`: the padding is not zero by itself (a NaN in the row, say).
template <typename T, int V, int G>
__device__ __forceinline__ void norm_write(T* row, const f32x2 (&f)[NORM_H], int lane, int n, int W, bool clear) {
#pragma unroll
  for (int k = 0; k < NORM_E / V; ++k) {
    const int c = (k * G + lane) * V;
    float v[V];
    if constexpr (V == 1) {
      const float2 t = halves(f[k / 2]);
      v[0] = k % 2 ? t.y : t.x;
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 t = halves(f[(k * V + e) / 2]);
        v[e] = t.x, v[e + 1] = t.y;
      }
    }
    if (clear && (k + 1) * G * V > n) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e >= n) v[e] = 0.f;
    }
    if (c < W) {
      if constexpr (V == 8 && sizeof(T) == 4) {
        norm_store<float, 4>(row + c, v);
        norm_store<float, 4>(row + c + 4, v + 4);
      } else {
        norm_store<T, V>(row + c, v);
      }
    }
  }
}

// Lane's columns of a (W,) fp32 parameter, `other` where there is none and from column n on (the
// padding may hold anything).
template <int V, int G>
__device__ __forceinline__ void norm_param(const float* p, int lane, int n, float other, f32x2 (&f)[NORM_H]) {
  float v[NORM_E];
#pragma unroll
  for (int k = 0; k < NORM_E / V; ++k) {
    const int c = (k * G + lane) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) v[k * V + e] = other;
    if (V >= 4 && p && c + V <= n) {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + c + e));
        v[k * V + e] = q.x;
        v[k * V + (e + 1) % V] = q.y;
        v[k * V + (e + 2) % V] = q.z;
        v[k * V + (e + 3) % V] = q.w;
      }
    } else if (p) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e < n) v[k * V + e] = __ldg(p + c + e);
    }
  }
#pragma unroll
  for (int h = 0; h < NORM_H; ++h) f[h] = pair(v[2 * h], v[2 * h + 1]);
}

// Stages of the ring, the current one included: two rows each forward, one of x and dy backward.
template <typename T, int V>
struct NormDepth {
  static constexpr int FORWARD = V == 1 ? 1 : sizeof(T) == 2 ? 3 : 2;
  static constexpr int BACKWARD = V == 1 ? 1 : sizeof(T) == 2 ? 4 : 2;
};

template <typename T, int V, int G>
__global__ void __launch_bounds__(NormGroup<G>::THREADS, NormGroup<G>::THREADS > 256 ? 1 : 2)
    layer_norm_held_forward_kernel(const LayerNormArgs a) {
  using Grp = NormGroup<G>;
  using Rows = NormRows<T, V, G>;
  constexpr int D = NormDepth<T, V>::FORWARD, AHEAD = V == 1 ? 1 : D - 1;
  __shared__ float2 red[Grp::GROUPS * 2 * Grp::WARPS];
  extern __shared__ __align__(16) char ring[];
  Grp grp(red);
  const int m = blockIdx.x / a.S, split = blockIdx.x % a.S;
  const int n = norm_width(a, m), lane = grp.lane, step = a.S * Grp::GROUPS;
  const float inv_n = 1.0f / (float)max(n, 1);
  // groups of one warp step together (their sums are warp-wide shuffles): rows beyond the last are
  // computed from what the ring holds and not written
  const int first = split * Grp::GROUPS + grp.group;
  const int rounds = (a.B - split * Grp::GROUPS + 2 * step - 1) / (2 * step);
  const T* x0 = static_cast<const T*>(a.x) + m * a.xm;
  Rows xa(x0, a.xr, first, 2 * step, lane, n, ring, D);
  Rows xb(x0, a.xr, first + step, 2 * step, lane, n, ring + D * Rows::STAGE, D);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    xa.issue(i, first + 2 * i * step < a.B);
    xb.issue(i, first + (2 * i + 1) * step < a.B);
  }
  f32x2 w[NORM_H], b[NORM_H], mask[NORM_H];
  norm_param<V, G>(a.w ? a.w + (size_t)m * a.W : nullptr, lane, n, 1.f, w);
  norm_param<V, G>(a.b ? a.b + (size_t)m * a.W : nullptr, lane, n, 0.f, b);
  norm_mask<V, G>(lane, n, mask);
  T* y = static_cast<T*>(a.y) + ((int64_t)m * a.B + first) * a.W;
  for (int i = 0, r = first; i < rounds; ++i, r += 2 * step) {
    f32x2 f[2][NORM_H];
    if (V > 1) cp_async_wait<(D > 1 ? 2 * (D - 2) : 0)>();
    xa.take(i % D, f[0]);
    xb.take(i % D, f[1]);
    xa.issue((i + AHEAD) % D, r + 2 * AHEAD * step < a.B);
    xb.issue((i + AHEAD) % D, r + (2 * AHEAD + 1) * step < a.B);
    const float2 sum = grp.sum(norm_add(f[0]), norm_add(f[1]));
    const float mean[2] = {sum.x * inv_n, sum.y * inv_n};
    float sq[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const f32x2 minus = pair(-mean[q], -mean[q]);
      f32x2 s = pair(0.f, 0.f);
#pragma unroll
      for (int h = 0; h < NORM_H; ++h) {
        f[q][h] = fma2(mask[h], minus, f[q][h]);
        s = fma2(f[q][h], f[q][h], s);
      }
      const float2 t = halves(s);
      sq[q] = t.x + t.y;
    }
    const float2 var = grp.sum(sq[0], sq[1]);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int row = r + q * step;
      if (row < a.B) {
        const float rstd = rsqrtf((q ? var.y : var.x) * inv_n + a.eps);
        const f32x2 rs = pair(rstd, rstd);
#pragma unroll
        for (int h = 0; h < NORM_H; ++h) f[q][h] = fma2(mul2(f[q][h], rs), w[h], b[h]);
        norm_write<T, V, G>(y, f[q], lane, n, a.W, !(rstd < INFINITY));
        if (lane == 0) {
          a.mean[(int64_t)m * a.B + row] = mean[q];
          a.rstd[(int64_t)m * a.B + row] = rstd;
        }
      }
      y += (int64_t)step * a.W;
    }
  }
}

// dx of the group's rows, and the columns' sums of dy xhat and dy over the block's rows.
template <typename T, int V, int G>
__global__ void __launch_bounds__(NormGroup<G>::THREADS, NormGroup<G>::THREADS > 256 ? 1 : 2)
    layer_norm_held_backward_kernel(const LayerNormArgs a) {
  using Grp = NormGroup<G>;
  using Rows = NormRows<T, V, G>;
  constexpr int D = NormDepth<T, V>::BACKWARD, AHEAD = V == 1 ? 1 : D - 1;
  __shared__ float2 red[Grp::GROUPS * 2 * Grp::WARPS];
  extern __shared__ __align__(16) char ring[];  // x, then dy; at the end the groups' column sums
  Grp grp(red);
  const int m = blockIdx.x / a.S, split = blockIdx.x % a.S;
  const int n = norm_width(a, m), lane = grp.lane, step = a.S * Grp::GROUPS;
  const float inv_n = 1.0f / (float)max(n, 1);
  const int first = split * Grp::GROUPS + grp.group;
  const int rounds = (a.B - split * Grp::GROUPS + step - 1) / step;
  Rows x(static_cast<const T*>(a.x) + m * a.xm, a.xr, first, step, lane, n, ring, D);
  Rows dy(static_cast<const T*>(a.dy) + m * a.dym, a.dyr, first, step, lane, n, ring + D * Rows::STAGE, D);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    x.issue(i, first + i * step < a.B);
    dy.issue(i, first + i * step < a.B);
  }
  const float* mean = a.mean + (int64_t)m * a.B + first;
  const float* rstd = a.rstd + (int64_t)m * a.B + first;
  float nmean = 0.f, nrstd = 0.f;
  if (first < a.B) nmean = *mean, nrstd = *rstd;
  f32x2 w[NORM_H], sw[NORM_H], sb[NORM_H];
  norm_param<V, G>(a.w ? a.w + (size_t)m * a.W : nullptr, lane, n, 1.f, w);
#pragma unroll
  for (int h = 0; h < NORM_H; ++h) sw[h] = sb[h] = pair(0.f, 0.f);
  const bool dx_f32 = sizeof(T) == 2 && a.dx_f32;
  char* dx = static_cast<char*>(a.dx) + ((int64_t)m * a.B + first) * a.W * (dx_f32 ? 4 : sizeof(T));
  const int64_t dx_step = (int64_t)step * a.W * (dx_f32 ? 4 : sizeof(T));
  for (int i = 0, r = first; i < rounds; ++i, r += step, dx += dx_step) {
    f32x2 xh[NORM_H], g[NORM_H];
    if (V > 1) cp_async_wait<(D > 1 ? 2 * (D - 2) : 0)>();
    x.take(i % D, xh);
    dy.take(i % D, g);
    const float mu = nmean, rs = nrstd;
    mean += step;
    rstd += step;
    nmean = nrstd = 0.f;  // beyond the last row: xhat = 0, times dy = 0
    if (r + step < a.B) nmean = *mean, nrstd = *rstd;
    x.issue((i + AHEAD) % D, r + AHEAD * step < a.B);
    dy.issue((i + AHEAD) % D, r + AHEAD * step < a.B);
    const bool live = r < a.B;
    if (!live) {
#pragma unroll
      for (int h = 0; h < NORM_H; ++h) g[h] = xh[h] = pair(0.f, 0.f);
    }
    // columns from n on hold x = 0: where -mean rstd is no number of fp32 they take x = mean, since an infinite
    // xhat times dy = 0 would make the row's sum a NaN
    if (!(fabsf(mu * rs) < INFINITY)) {
#pragma unroll
      for (int h = 0; h < NORM_H; ++h) {
        const int c = Rows::c0(2 * h / V, lane) + 2 * h % V, d = V == 1 ? c + G : c + 1;
        const float2 t = halves(xh[h]);
        xh[h] = pair(c < n ? t.x : mu, d < n ? t.y : mu);
      }
    }
    const f32x2 minus = pair(-mu, -mu), scale = pair(rs, rs);
    f32x2 s1 = pair(0.f, 0.f), s2 = s1;
#pragma unroll
    for (int h = 0; h < NORM_H; ++h) {  // dy is 0 from column n on
      xh[h] = mul2(add2(xh[h], minus), scale);
      sw[h] = fma2(g[h], xh[h], sw[h]);
      sb[h] = add2(sb[h], g[h]);
      g[h] = mul2(g[h], w[h]);
      s1 = add2(s1, g[h]);
      s2 = fma2(g[h], xh[h], s2);
    }
    if (a.dx == nullptr) continue;
    const float2 u = halves(s1), v = halves(s2);
    const float2 t = grp.sum(u.x + u.y, v.x + v.y);
    if (!live) continue;
    const f32x2 c1 = pair(-t.x * inv_n, -t.x * inv_n), c2 = pair(-t.y * inv_n, -t.y * inv_n);
#pragma unroll
    for (int h = 0; h < NORM_H; ++h) g[h] = mul2(fma2(xh[h], c2, add2(g[h], c1)), scale);
    const bool ragged = n < a.W;
    if (dx_f32)
      norm_write<float, V, G>(reinterpret_cast<float*>(dx), g, lane, n, a.W, ragged);
    else
      norm_write<T, V, G>(reinterpret_cast<T*>(dx), g, lane, n, a.W, ragged);
  }
  if (!a.dw && !a.db) return;
  // the block's groups in ascending order, then (with several splits) the finishing kernel
  const size_t row = ((size_t)m * a.S + split) * a.W;
  float* ow = a.S > 1 ? a.partial + row : a.dw ? a.dw + row : nullptr;
  float* ob = a.S > 1 ? a.partial + (size_t)a.P * a.S * a.W + row : a.db ? a.db + row : nullptr;
  if constexpr (Grp::GROUPS > 1) {
    float* cols = reinterpret_cast<float*>(ring);  // dw of every group's columns, then db
    constexpr int HALF = Grp::THREADS * NORM_E;
    if (V > 1) cp_async_wait<0>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NORM_E / V; ++k) {
      float* to = cols + grp.group * G * NORM_E + Rows::c0(k, lane);
      if constexpr (V == 1) {
        const float2 u = halves(sw[k / 2]), v = halves(sb[k / 2]);
        to[0] = k % 2 ? u.y : u.x;
        to[HALF] = k % 2 ? v.y : v.x;
      } else if constexpr (V == 2) {
        const float2 u = halves(sw[k]), v = halves(sb[k]);
        *reinterpret_cast<float2*>(to) = u;
        *reinterpret_cast<float2*>(to + HALF) = v;
      } else {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const int h = (k * V + e) / 2;
          const float2 u = halves(sw[h]), u2 = halves(sw[h + 1]), v = halves(sb[h]), v2 = halves(sb[h + 1]);
          *reinterpret_cast<float4*>(to + e) = make_float4(u.x, u.y, u2.x, u2.y);
          *reinterpret_cast<float4*>(to + HALF + e) = make_float4(v.x, v.y, v2.x, v2.y);
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < min(G * NORM_E, a.W); c += Grp::THREADS) {
      float u = 0.f, v = 0.f;
#pragma unroll 8
      for (int i = 0; i < Grp::GROUPS; ++i) {
        u += cols[i * G * NORM_E + c];
        v += cols[HALF + i * G * NORM_E + c];
      }
      if (ow) ow[c] = c < n ? u : 0.f;
      if (ob) ob[c] = c < n ? v : 0.f;
    }
  } else {
#pragma unroll
    for (int h = 0; h < NORM_H; ++h) {
      const int c = Rows::c0(2 * h / V, lane) + 2 * h % V, d = V == 1 ? c + G : c + 1;
      const float2 u = halves(sw[h]), v = halves(sb[h]);
      if (ow && c < a.W) ow[c] = c < n ? u.x : 0.f;
      if (ow && d < a.W) ow[d] = d < n ? u.y : 0.f;
      if (ob && c < a.W) ob[c] = c < n ? v.x : 0.f;
      if (ob && d < a.W) ob[d] = d < n ? v.y : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows wider than NORM_HELD columns.
// ---------------------------------------------------------------------------
// Sum over the block of (u, v), in every thread.
__device__ __forceinline__ float2 block_sum2(float u, float v, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
    v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  }
  __syncthreads();
  if (lane_id() == 0) red[warp_id()] = make_float2(u, v);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
    s.x += red[i].x;
    s.y += red[i].y;
  }
  return s;
}

// One block per row.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_forward_kernel(const LayerNormArgs a) {
  __shared__ float2 red[8];
  const int64_t row = blockIdx.x;
  const int m = (int)(row / a.B), r = (int)(row % a.B);
  const int n = norm_width(a, m);
  const T* x = static_cast<const T*>(a.x) + m * a.xm + r * a.xr;
  T* y = static_cast<T*>(a.y) + row * a.W;
  const float* w = a.w ? a.w + (size_t)m * a.W : nullptr;
  const float* b = a.b ? a.b + (size_t)m * a.W : nullptr;
  float s = 0.f;
  for (int c = threadIdx.x; c < n; c += 256) s += to_f32<T>(x[c]);
  const float mean = block_sum2(s, 0.f, red).x / n;
  s = 0.f;
  for (int c = threadIdx.x; c < n; c += 256) {
    const float d = to_f32<T>(x[c]) - mean;
    s += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_sum2(s, 0.f, red).x / n + a.eps);
  for (int c = threadIdx.x; c < a.W; c += 256) {
    float v = 0.f;
    if (c < n) {
      v = (to_f32<T>(x[c]) - mean) * rstd;
      if (w) v *= w[c];
      if (b) v += b[c];
    }
    y[c] = from_f32<T>(v);
  }
  if (threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// One block per row: dx.
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dx_kernel(const LayerNormArgs a) {
  __shared__ float2 red[8];
  const int64_t row = blockIdx.x;
  const int m = (int)(row / a.B), r = (int)(row % a.B);
  const int n = norm_width(a, m);
  const T* x = static_cast<const T*>(a.x) + m * a.xm + r * a.xr;
  const T* dy = static_cast<const T*>(a.dy) + m * a.dym + r * a.dyr;
  const float* w = a.w ? a.w + (size_t)m * a.W : nullptr;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < n; c += 256) {
    const float g = to_f32<T>(dy[c]) * (w ? w[c] : 1.f);
    s1 += g;
    s2 += g * ((to_f32<T>(x[c]) - mean) * rstd);
  }
  float2 t = block_sum2(s1, s2, red);
  t.x /= n;
  t.y /= n;
  for (int c = threadIdx.x; c < a.W; c += 256) {
    float v = 0.f;
    if (c < n) {
      const float g = to_f32<T>(dy[c]) * (w ? w[c] : 1.f);
      v = rstd * (g - t.x - (to_f32<T>(x[c]) - mean) * rstd * t.y);
    }
    if (a.dx_f32)
      static_cast<float*>(a.dx)[row * a.W + c] = v;
    else
      static_cast<T*>(a.dx)[row * a.W + c] = from_f32<T>(v);
  }
}

// One thread per column over a split's rows: dw and db (or their partial sums).
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_dw_kernel(const LayerNormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y, split = blockIdx.z;
  if (c >= a.W) return;
  float sw = 0.f, sb = 0.f;
  if (c < norm_width(a, m)) {
    for (int r = split; r < a.B; r += a.S) {
      const float dy = to_f32<T>(static_cast<const T*>(a.dy)[m * a.dym + r * a.dyr + c]);
      const float x = to_f32<T>(static_cast<const T*>(a.x)[m * a.xm + r * a.xr + c]);
      sw += dy * ((x - a.mean[(int64_t)m * a.B + r]) * a.rstd[(int64_t)m * a.B + r]);
      sb += dy;
    }
  }
  if (a.S > 1) {
    const size_t at = ((size_t)m * a.S + split) * a.W + c;
    a.partial[at] = sw;
    a.partial[(size_t)a.P * a.S * a.W + at] = sb;
  } else {
    if (a.dw) a.dw[(size_t)m * a.W + c] = sw;
    if (a.db) a.db[(size_t)m * a.W + c] = sb;
  }
}

// The splits' partial sums: 32 columns a block, SLICES threads over the splits of each in turn.
template <int SLICES>
__global__ void __launch_bounds__(32 * SLICES) layer_norm_finish_kernel(const LayerNormArgs a, int col_blocks) {
  __shared__ float2 part[SLICES][32];
  const int m = blockIdx.x / col_blocks, lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = (blockIdx.x % col_blocks) * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < a.W) {
    const float* p = a.partial + (size_t)m * a.S * a.W + c;
    const size_t second = (size_t)a.P * a.S * a.W;
#pragma unroll 4
    for (int i = slice; i < a.S; i += SLICES) {
      s.x += p[(size_t)i * a.W];
      s.y += p[second + (size_t)i * a.W];
    }
  }
  part[slice][lane] = s;
  __syncthreads();
  if (slice != 0 || c >= a.W) return;
#pragma unroll
  for (int i = 1; i < SLICES; ++i) {
    s.x += part[i][lane].x;
    s.y += part[i][lane].y;
  }
  if (a.dw) a.dw[(size_t)m * a.W + c] = s.x;
  if (a.db) a.db[(size_t)m * a.W + c] = s.y;
}

// The members' terms of a shared input's gradient, in member order in fp32 and rounded once, V at a time.
// Memory bounds it, or the launch: every term is read once (7 x 333 x 771, odd and so element by element:
// 6.2 us under the profiler with cold caches; a library reduction and its dispatch took 6 us more of the call).
template <typename T, int V>
__global__ void __launch_bounds__(256) layer_norm_member_sum_kernel(const float* terms, T* out, int P, int64_t n) {
  const int64_t step = (int64_t)gridDim.x * 256 * V;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; i < n; i += step) {
    float s[V] = {};
#pragma unroll 4
    for (int m = 0; m < P; ++m) {
      const float* p = terms + m * n + i;
      if constexpr (V == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        s[0] += f.x, s[1] += f.y, s[2] += f.z, s[3] += f.w;
      } else {
        s[0] += *p;
      }
    }
    if constexpr (V == 4 && sizeof(T) == 2)
      *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
    else if constexpr (V == 4)
      *reinterpret_cast<float4*>(out + i) = make_float4(s[0], s[1], s[2], s[3]);
    else
      out[i] = from_f32<T>(s[0]);
  }
}

}  // namespace tp
