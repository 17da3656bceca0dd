// Layer norm of a pack: member m's rows are normalised over its first n_m columns, then scaled
// and shifted per member and column.  Columns at or beyond n_m are written as zeros and never read.
//
//   xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps), y = xhat w + b
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) with g = dy w;  dw = sum_r dy xhat;  db = sum_r dy
//
// Memory bounds all of it: 4 bytes per element forward and 6 backward in bf16, 10 to 20
// instructions.  Rows of up to NORM_HELD columns stay in the registers of a group of G lanes (8 to
// 512, 16 elements each), so x and dy are read once and the variance is summed around the mean.
// A group walks over rows of one member: the member's w and b, and in the backward the columns' sums,
// stay in registers, and the next row is on its way while the current one is reduced.  Wider rows
// take the plain kernels at the end.
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

// V neighbouring elements in their own type: 16 bytes, or one element where nothing is aligned.
template <typename T, int V>
struct NormVec {
  uint4 u;
  __device__ void load(const T* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ void get(float (&f)[V]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 2) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
      } else {
        f[e] = __uint_as_float(w[e]);
      }
    }
  }
  __device__ static void store(T* p, const float (&f)[V]) {
    uint4 w;
    if constexpr (sizeof(T) == 2)
      w = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                     pack_bf16x2(f[6], f[7]));
    else
      w = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    *reinterpret_cast<uint4*>(p) = w;
  }
};

template <typename T>
struct NormVec<T, 1> {
  T u;
  __device__ void load(const T* p) { u = *p; }
  __device__ void zero() { u = from_f32<T>(0.f); }
  __device__ void get(float (&f)[1]) const { f[0] = to_f32<T>(u); }
  __device__ static void store(T* p, const float (&f)[1]) { *p = from_f32<T>(f[0]); }
};

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
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
      u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
      v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    }
    if constexpr (G > 32) {
      float2* r = red + half * WARPS;
      half ^= 1;
      if (lane % 32 == 0) r[lane / 32] = make_float2(u, v);
      asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(G) : "memory");
      u = v = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        u += r[i].x;
        v += r[i].y;
      }
    }
    return make_float2(u, v);
  }
};

// A row's elements c0(k) .. c0(k) + V - 1 of one lane, k < E / V, as far as they are below n.
template <typename T, int V, int G>
struct NormRow {
  static constexpr int K = NORM_E / V;
  NormVec<T, V> raw[K];
  __device__ static int c0(int k, int lane) { return (k * G + lane) * V; }
  __device__ void load(const T* row, int lane, int n) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (c0(k, lane) < n)
        raw[k].load(row + c0(k, lane));
      else
        raw[k].zero();
    }
  }
  __device__ void get(float (&f)[NORM_E]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float v[V];
      raw[k].get(v);
#pragma unroll
      for (int e = 0; e < V; ++e) f[k * V + e] = v[e];
    }
  }
};

// Lane's columns of a (W,) fp32 parameter, `other` where there is none.
template <int V, int G>
__device__ __forceinline__ void norm_param(const float* p, int lane, int n, float other, float (&f)[NORM_E]) {
#pragma unroll
  for (int k = 0; k < NORM_E / V; ++k) {
    const int c = (k * G + lane) * V;
    if (V >= 4 && p && c < n) {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p + c + e));
        f[k * V + e] = q.x;
        f[k * V + (e + 1) % V] = q.y;
        f[k * V + (e + 2) % V] = q.z;
        f[k * V + (e + 3) % V] = q.w;
      }
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c + e >= n) f[k * V + e] = other;  // the padding may hold anything
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) f[k * V + e] = p && c + e < n ? __ldg(p + c + e) : other;
    }
  }
}

template <typename T, int V, int G>
__global__ void __launch_bounds__(NormGroup<G>::THREADS) layer_norm_held_forward_kernel(const LayerNormArgs a) {
  using Grp = NormGroup<G>;
  __shared__ float2 red[Grp::GROUPS * 2 * Grp::WARPS];
  Grp grp(red);
  const int m = blockIdx.x / a.S, split = blockIdx.x % a.S;
  const int n = norm_width(a, m), lane = grp.lane, step = a.S * Grp::GROUPS;
  const float inv_n = 1.0f / (float)max(n, 1);
  const T* x = static_cast<const T*>(a.x) + m * a.xm;
  float w[NORM_E], b[NORM_E];
  norm_param<V, G>(a.w ? a.w + (size_t)m * a.W : nullptr, lane, n, 1.f, w);
  norm_param<V, G>(a.b ? a.b + (size_t)m * a.W : nullptr, lane, n, 0.f, b);
  // groups of one warp step together (their sums are warp-wide shuffles): rows beyond the last
  // are computed again from the last and not written
  const int first = split * Grp::GROUPS + grp.group;
  const int rounds = (a.B - split * Grp::GROUPS + step - 1) / step;
  NormRow<T, V, G> next;
  next.load(x + min(first, a.B - 1) * a.xr, lane, n);
  for (int i = 0; i < rounds; ++i) {
    const int r = first + i * step;
    float f[NORM_E];
    next.get(f);
    if (i + 1 < rounds) next.load(x + min(r + step, a.B - 1) * a.xr, lane, n);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NORM_E; ++j) {
      if (NormRow<T, V, G>::c0(j / V, lane) + j % V >= n) f[j] = 0.f;
      s += f[j];
    }
    const float mean = grp.sum(s, 0.f).x * inv_n;
    s = 0.f;
#pragma unroll
    for (int j = 0; j < NORM_E; ++j) {
      f[j] = NormRow<T, V, G>::c0(j / V, lane) + j % V < n ? f[j] - mean : 0.f;
      s += f[j] * f[j];
    }
    const float rstd = 1.0f / sqrtf(grp.sum(s, 0.f).x * inv_n + a.eps);
    if (r >= a.B) continue;
    T* y = static_cast<T*>(a.y) + ((int64_t)m * a.B + r) * a.W;
#pragma unroll
    for (int k = 0; k < NORM_E / V; ++k) {
      const int c = NormRow<T, V, G>::c0(k, lane);
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = c + e < n ? f[k * V + e] * rstd * w[k * V + e] + b[k * V + e] : 0.f;
      if (c < a.W) NormVec<T, V>::store(y + c, v);
    }
    if (lane == 0) {
      a.mean[(int64_t)m * a.B + r] = mean;
      a.rstd[(int64_t)m * a.B + r] = rstd;
    }
  }
}

// dx of the group's rows, and the columns' sums of dy xhat and dy over the block's rows.
template <typename T, int V, int G>
__global__ void __launch_bounds__(NormGroup<G>::THREADS, NormGroup<G>::THREADS > 256 ? 1 : 2)
    layer_norm_held_backward_kernel(const LayerNormArgs a) {
  using Grp = NormGroup<G>;
  __shared__ float2 red[Grp::GROUPS * 2 * Grp::WARPS];
  __shared__ __align__(16) float cols[Grp::GROUPS > 1 ? Grp::THREADS * NORM_E : 1];
  Grp grp(red);
  const int m = blockIdx.x / a.S, split = blockIdx.x % a.S;
  const int n = norm_width(a, m), lane = grp.lane, step = a.S * Grp::GROUPS;
  const float inv_n = 1.0f / (float)max(n, 1);
  const T* x = static_cast<const T*>(a.x) + m * a.xm;
  const T* dy = static_cast<const T*>(a.dy) + m * a.dym;
  const float* mean = a.mean + (int64_t)m * a.B;
  const float* rstd = a.rstd + (int64_t)m * a.B;
  float w[NORM_E], sw[NORM_E], sb[NORM_E];
  norm_param<V, G>(a.w ? a.w + (size_t)m * a.W : nullptr, lane, n, 1.f, w);
#pragma unroll
  for (int j = 0; j < NORM_E; ++j) sw[j] = sb[j] = 0.f;
  const int first = split * Grp::GROUPS + grp.group;
  const int rounds = (a.B - split * Grp::GROUPS + step - 1) / step;
  NormRow<T, V, G> nx, ndy;
  float nmean = 0.f, nrstd = 0.f;
  const auto fetch = [&](int r) {
    r = min(r, a.B - 1);
    nx.load(x + r * a.xr, lane, n);
    ndy.load(dy + r * a.dyr, lane, n);
    nmean = mean[r];
    nrstd = rstd[r];
  };
  fetch(first);
  for (int i = 0; i < rounds; ++i) {
    const int r = first + i * step;
    float h[NORM_E], g[NORM_E];
    nx.get(h);
    ndy.get(g);
    const float mu = nmean, rs = nrstd;
    if (i + 1 < rounds) fetch(r + step);
    const bool live = r < a.B;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NORM_E; ++j) {
      const bool in = live && NormRow<T, V, G>::c0(j / V, lane) + j % V < n;
      h[j] = in ? (h[j] - mu) * rs : 0.f;
      g[j] = in ? g[j] : 0.f;
      sw[j] += g[j] * h[j];
      sb[j] += g[j];
      g[j] *= w[j];
      s1 += g[j];
      s2 += g[j] * h[j];
    }
    if (a.dx == nullptr) continue;
    const float2 t = grp.sum(s1, s2);
    if (!live) continue;
    const float c1 = t.x * inv_n, c2 = t.y * inv_n;
    const int64_t at = ((int64_t)m * a.B + r) * a.W;
#pragma unroll
    for (int k = 0; k < NORM_E / V; ++k) {
      const int c = NormRow<T, V, G>::c0(k, lane);
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e)
        v[e] = c + e < n ? rs * (g[k * V + e] - c1 - h[k * V + e] * c2) : 0.f;
      if (c >= a.W) continue;
      if (sizeof(T) == 2 && a.dx_f32) {
        float* d = static_cast<float*>(a.dx) + at + c;
        if constexpr (V >= 4) {
#pragma unroll
          for (int e = 0; e < V; e += 4)
            *reinterpret_cast<float4*>(d + e) = make_float4(v[e], v[(e + 1) % V], v[(e + 2) % V], v[(e + 3) % V]);
        } else {
          d[0] = v[0];
        }
      } else {
        NormVec<T, V>::store(static_cast<T*>(a.dx) + at + c, v);
      }
    }
  }
  if (!a.dw && !a.db) return;
  // the block's groups in ascending order, then (with several splits) the finishing kernel
  const size_t row = ((size_t)m * a.S + split) * a.W;
  float* ow = a.S > 1 ? a.partial + row : a.dw ? a.dw + row : nullptr;
  float* ob = a.S > 1 ? a.partial + (size_t)a.P * a.S * a.W + row : a.db ? a.db + row : nullptr;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const float(&s)[NORM_E] = which ? sb : sw;
    float* o = which ? ob : ow;
    if constexpr (Grp::GROUPS > 1) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NORM_E; ++j)
        cols[grp.group * G * NORM_E + NormRow<T, V, G>::c0(j / V, lane) + j % V] = s[j];
      __syncthreads();
      for (int c = threadIdx.x; c < min(G * NORM_E, a.W); c += Grp::THREADS) {
        float t = 0.f;
#pragma unroll 8
        for (int i = 0; i < Grp::GROUPS; ++i) t += cols[i * G * NORM_E + c];
        if (o) o[c] = t;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NORM_E; ++j) {
        const int c = NormRow<T, V, G>::c0(j / V, lane) + j % V;
        if (o && c < a.W) o[c] = s[j];
      }
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

// The splits' partial sums: 32 columns a block, eight threads over the splits of each in turn.
__global__ void __launch_bounds__(256) layer_norm_finish_kernel(const LayerNormArgs a, int col_blocks) {
  __shared__ float2 part[8][32];
  const int m = blockIdx.x / col_blocks, lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int c = (blockIdx.x % col_blocks) * 32 + lane;
  float2 s = make_float2(0.f, 0.f);
  if (c < a.W) {
    const float* p = a.partial + (size_t)m * a.S * a.W + c;
    const size_t second = (size_t)a.P * a.S * a.W;
#pragma unroll 4
    for (int i = slice; i < a.S; i += 8) {
      s.x += p[(size_t)i * a.W];
      s.y += p[second + (size_t)i * a.W];
    }
  }
  part[slice][lane] = s;
  __syncthreads();
  if (slice != 0 || c >= a.W) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    s.x += part[i][lane].x;
    s.y += part[i][lane].y;
  }
  if (a.dw) a.dw[(size_t)m * a.W + c] = s.x;
  if (a.db) a.db[(size_t)m * a.W + c] = s.y;
}

}  // namespace tp
