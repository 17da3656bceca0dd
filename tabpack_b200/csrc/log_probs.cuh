// Log probabilities of given labels from raw scores (logits), with the entropy, the best
// classes and the gradient.
//
//   z' = z - max z,  L = log sum exp z',  log p_c = z'_c - L,  H = -sum_c p_c log p_c
//   dz_c = g_l ([c = label] - p_c) - g_H p_c (log p_c + H)
//
// The maximum and L stay apart: max z + L would lose L where the scores are large (a row of the
// type's lowest value still has log p = -log C).  p = 0 contributes nothing to H, so masked classes
// (-inf) are allowed; a row with nothing but -inf has log p = -inf, H = 0 and no gradient.
#pragma once

#include "gemm_simt.cuh"

namespace tp {

struct LogProbsArgs {
  int64_t rows;
  int C;
  int64_t ld;              // row stride of the logits
  const void* logits;
  const int64_t* labels;
  int64_t label_rows;      // row r has label r % label_rows
  int64_t ignore_index;
  int k;
  float* log_prob;
  float* entropy;
  float* top;              // (rows, k)
  int64_t* which;          // (rows, k)
  float* stats;            // (rows, 3): max, L, H
  const float* g_l;        // (rows,) or one value (stride 0), or nullptr
  const float* g_h;
  int g_l_stride, g_h_stride;
  void* dlogits;           // (rows, C)
};

// Ascending integer order of floats (NaN above everything, -0 equal to +0), then descending
// position: the largest key is the best class, ties to the lowest index.
__device__ __forceinline__ unsigned long long class_key(float v, uint32_t c) {
  uint32_t u = __float_as_uint(v + 0.0f);
  if (v != v) u = 0x7FFFFFFFu;
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (uint32_t)~c;
}

__device__ __forceinline__ float class_value(unsigned long long key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}

// One block per row.
template <typename T>
__global__ void __launch_bounds__(256) log_probs_forward_kernel(const LogProbsArgs a) {
  __shared__ float red[3][8];
  __shared__ unsigned long long best[8];
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  float mx = -INFINITY;
  bool nan = false;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float v = to_f32<T>(z[c]);
    mx = fmaxf(mx, v);
    nan |= v != v;
  }
  nan = __syncthreads_or(nan);
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
  if (lane_id() == 0) red[0][warp_id()] = mx;
  __syncthreads();
  for (int i = 0; i < 8; ++i) mx = fmaxf(mx, red[0][i]);
  if (nan || mx == INFINITY) mx = __uint_as_float(0x7FC00000u);
  float s = 0.f, t = 0.f;
  if (mx != -INFINITY)
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const float d = to_f32<T>(z[c]) - mx, e = expf(d);
      s += e;
      if (e != 0.f) t += e * d;
    }
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
  }
  if (lane_id() == 0) red[1][warp_id()] = s, red[2][warp_id()] = t;
  __syncthreads();
  s = t = 0.f;
  for (int i = 0; i < 8; ++i) s += red[1][i], t += red[2][i];
  const bool empty = mx == -INFINITY;
  const float L = empty ? 0.f : logf(s);
  const float H = empty ? 0.f : L - t / s;
  if (threadIdx.x == 0) {
    const int64_t y = a.labels[row % a.label_rows];
    float lp = 0.f;
    if (y != a.ignore_index) {
      if (y < 0 || y >= a.C)
        lp = __uint_as_float(0x7FC00000u);
      else
        lp = empty ? -INFINITY : to_f32<T>(z[y]) - mx - L;
    }
    a.log_prob[row] = lp;
    a.entropy[row] = H;
    a.stats[3 * row] = mx;
    a.stats[3 * row + 1] = L;
    a.stats[3 * row + 2] = H;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.k; ++j) {
    unsigned long long b = 0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const unsigned long long key = class_key(to_f32<T>(z[c]), c);
      if (key < last && key > b) b = key;
    }
    for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, (unsigned long long)b, o));
    __syncthreads();
    if (lane_id() == 0) best[warp_id()] = b;
    __syncthreads();
    for (int i = 0; i < 8; ++i) b = max(b, best[i]);
    last = b;
    if (threadIdx.x == 0) {
      a.top[row * a.k + j] = empty ? -INFINITY : class_value(b) - mx - L;
      a.which[row * a.k + j] = (int64_t)(uint32_t)~(uint32_t)b;
    }
  }
}

// One block per row.
template <typename T>
__global__ void __launch_bounds__(256) log_probs_backward_kernel(const LogProbsArgs a) {
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  T* dz = static_cast<T*>(a.dlogits) + row * a.C;
  const float mx = a.stats[3 * row], L = a.stats[3 * row + 1], H = a.stats[3 * row + 2];
  int64_t y = a.labels[row % a.label_rows];
  float gl = a.g_l ? a.g_l[row * a.g_l_stride] : 0.f;
  const float gh = a.g_h ? a.g_h[row * a.g_h_stride] : 0.f;
  if (!a.g_l || y == a.ignore_index) {
    gl = 0.f;
    y = -1;
  } else if (y < 0 || y >= a.C) {
    gl = __uint_as_float(0x7FC00000u);
  }
  const bool empty = mx == -INFINITY;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    float g = 0.f;
    if (!empty) {
      const float lp = to_f32<T>(z[c]) - mx - L, p = expf(lp);
      g = -gl * p;
      if (p != 0.f) g -= gh * p * (lp + H);
    }
    if (c == y && !empty) g += gl;
    dz[c] = from_f32<T>(g);
  }
}

}  // namespace tp
