// Layer norm of a pack: member m's rows are normalised over its first n_m columns, then scaled
// and shifted per member and column.  Columns at or beyond n_m are written as zeros and never read.
//
//   xhat = (x - mean) rstd, rstd = 1 / sqrt(var + eps), y = xhat w + b
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) with g = dy w;  dw = sum_r dy xhat;  db = sum_r dy
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
  int S, rows_per_split;
};

__device__ __forceinline__ int norm_width(const LayerNormArgs& a, int m) {
  return a.n ? min(max(a.n[m], 0), a.W) : a.W;
}

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
    const int r1 = min(a.B, (split + 1) * a.rows_per_split);
    for (int r = split * a.rows_per_split; r < r1; ++r) {
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

// The splits' partial sums, in ascending order.
__global__ void __launch_bounds__(256) layer_norm_finish_kernel(const LayerNormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x, m = blockIdx.y;
  if (c >= a.W) return;
  const float* p = a.partial + (size_t)m * a.S * a.W + c;
  float sw = 0.f, sb = 0.f;
  for (int i = 0; i < a.S; ++i) {
    sw += p[(size_t)i * a.W];
    sb += p[((size_t)a.P * a.S + i) * a.W];
  }
  if (a.dw) a.dw[(size_t)m * a.W + c] = sw;
  if (a.db) a.db[(size_t)m * a.W + c] = sb;
}

}  // namespace tp
