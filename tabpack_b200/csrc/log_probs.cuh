// Log probabilities of given labels from raw scores (logits), with the entropy, the best
// classes and the gradient.
//
//   z' = z - max z,  S = sum exp z',  L = log S,  log p_c = z'_c - L
//   H = -sum_c p_c log p_c = L - sum_c exp(z'_c) z'_c / S
//   dz_c = g_l ([c = label] - p_c) - g_H p_c (log p_c + H)
//
// The maximum and L stay apart: max z + L would lose L where the scores are large (a row of the
// type's lowest value still has log p = -log C).  z' is bounded below by LP_FAR, far under the last
// nonzero exponential, so that masked classes (-inf) contribute exp(z') z' = 0 and not NaN; a
// row with nothing but -inf has S = 0 and is told by that: log p = -inf, H = 0, no gradient.
//
// Memory bounds these kernels: 2 or 4 bytes a class against 8 to 12 instructions.  Rows of up
// to 1024 classes are held in registers by a thread (16), 8 lanes (64) or a warp (256, 1024), so the
// row is read once and the softmax takes its maximum first; longer rows take one block and one pass
// with a running maximum.  Rows start anywhere: whole 16-byte vectors are loaded between the
// first and last boundary inside the row, single elements before and after.
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
  float* stats;            // (rows, 3): max, L, H; C > LP_REREAD only
  const float* g_l;        // (rows,) or one value (stride 0), or nullptr
  const float* g_h;
  int g_l_stride, g_h_stride;
  void* dlogits;           // (rows, C)
};

constexpr float LP_FAR = -200.0f;
constexpr int LP_REREAD = TP_LABEL_STATS_CLASSES;  // rows up to here: the backward takes the statistics anew
constexpr int LP_CHUNK = 2048;       // classes of one warp in the streaming backward

__device__ __forceinline__ float lp_nan() { return __uint_as_float(0x7FC00000u); }

// exp(x) for x <= 0 from the base-2 exponential (2^-22 relative, and x's rounding times |x|).
__device__ __forceinline__ float exp_neg(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

// Ascending integer order of floats, at least 1: NaN above everything, -0 equal to +0.
__device__ __forceinline__ uint32_t class_order(float v) {
  uint32_t u = __float_as_uint(v + 0.0f);
  if (v != v) u = 0x7FFFFFFFu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ float class_value(uint32_t order) {
  return __uint_as_float((order & 0x80000000u) ? (order & 0x7FFFFFFFu) : ~order);
}

template <typename T>
struct Row {
  static constexpr int V = 16 / sizeof(T);
  const T* base;  // the 16-byte boundary at or before the row's first element
  int phase;      // elements between it and the row
  int C;
  __device__ Row(const T* z, int C_) : C(C_) {
    phase = (int)((reinterpret_cast<uintptr_t>(z) & 15u) / sizeof(T));
    base = z - phase;
  }
  __device__ int vectors() const { return (phase + C + V - 1) / V; }
  __device__ int first(int i) const { return i * V - phase; }  // class of vector i's first element
  // Vector i; elements outside the row read as -inf.
  __device__ void load(int i, float (&v)[V]) const {
    const int c0 = first(i);
    if (c0 >= 0 && c0 + V <= C) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(base) + i);
      unpack(u, v);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        v[e] = (c0 + e >= 0 && c0 + e < C) ? to_f32<T>(base[(int64_t)i * V + e]) : -INFINITY;
    }
  }
  __device__ static void unpack(const uint4& u, float (&v)[V]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = __uint_as_float(w[e]);
    }
  }
};

struct RowStats {
  float m, L, H;  // m = -inf and L = 0: no classes
  __device__ bool empty() const { return m == -INFINITY && L == 0.f; }
};

__device__ __forceinline__ RowStats row_stats(float m, float s, float t) {
  RowStats r;
  r.m = m;
  r.L = s == 0.f ? 0.f : logf(s);
  r.H = s == 0.f ? 0.f : r.L - t / s;
  return r;
}

// What the row's leader writes.
template <typename T>
__device__ __forceinline__ void write_row(const LogProbsArgs& a, int64_t row, const T* z, const RowStats& st) {
  const int64_t y = a.labels[row % a.label_rows];
  float lp = 0.f;
  if (y != a.ignore_index)
    lp = (y < 0 || y >= a.C) ? lp_nan() : st.empty() ? -INFINITY : to_f32<T>(z[y]) - st.m - st.L;
  a.log_prob[row] = lp;
  a.entropy[row] = st.H;
  if (a.C > LP_REREAD) {
    a.stats[3 * row] = st.m;
    a.stats[3 * row + 1] = st.L;
    a.stats[3 * row + 2] = st.H;
  }
}

__device__ __forceinline__ void write_best(const LogProbsArgs& a, int64_t row, int j, uint32_t order, uint32_t c,
                                           const RowStats& st) {
  a.top[row * a.k + j] = st.empty() ? -INFINITY : class_value(order) - st.m - st.L;
  a.which[row * a.k + j] = c;
}

// Gradient of one score, before the label's own term.
struct RowGrad {
  float a, b;  // dz = p (a + b log p): a = -(g_l + g_H H), b = -g_H
  float gl;    // at the label
  int y;       // -1: no label's term
  bool empty;
};

__device__ __forceinline__ RowGrad row_grad(const LogProbsArgs& a, int64_t row, const RowStats& st) {
  RowGrad g;
  const int64_t y = a.labels[row % a.label_rows];
  g.gl = a.g_l ? a.g_l[row * a.g_l_stride] : 0.f;
  const float gh = a.g_h ? a.g_h[row * a.g_h_stride] : 0.f;
  g.y = -1;
  if (!a.g_l || y == a.ignore_index)
    g.gl = 0.f;
  else if (y < 0 || y >= a.C)
    g.gl = lp_nan();
  else
    g.y = (int)y;
  g.a = -(g.gl + gh * st.H);
  g.b = -gh;
  g.empty = st.empty();
  return g;
}

__device__ __forceinline__ float score_grad(const RowGrad& g, const RowStats& st, float z, int c) {
  // a masked class: p = 0 and a finite log p, so that its product is 0
  const float lp = max_nan(z - st.m - st.L, LP_FAR);
  float d = exp_neg(lp) * (g.a + g.b * lp);
  if (c == g.y) d += g.gl;
  return g.empty ? 0.f : d;
}

// ---------------------------------------------------------------------------
// Rows in registers: G lanes (1, 8 or 32) hold E scores each, vectors of the row in turn.
// ---------------------------------------------------------------------------
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  return v;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

template <typename T, int G, int E>
struct HeldRow {
  static constexpr int V = Row<T>::V;
  float z[E];
  __device__ void load(const Row<T>& r, int lane) {
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      float v[V];
      r.load(j * G + lane, v);
#pragma unroll
      for (int e = 0; e < V; ++e) z[j * V + e] = v[e];
    }
  }
  __device__ RowStats stats() const {
    float m = z[0];
#pragma unroll
    for (int j = 1; j < E; ++j) m = fmaxf(m, z[j]);
    m = group_max<G>(fmaxf(m, -INFINITY));
    const float m0 = m == -INFINITY ? 0.f : m;
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float d = max_nan(z[j] - m0, LP_FAR), e = exp_neg(d);
      s += e;
      t += e * d;
    }
    return row_stats(m, group_sum<G>(s), group_sum<G>(t));
  }
  __device__ static int at(const Row<T>& r, int lane, int j) { return r.first((j / V) * G + lane) + j % V; }
};

// blockDim 256; a row beyond the last is computed again from the last and not written.
template <typename T, int G, int E, bool TOP>
__global__ void __launch_bounds__(256) log_probs_held_forward_kernel(const LogProbsArgs a) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  const int64_t row = min(at, a.rows - 1);
  const int lane = threadIdx.x & (G - 1);
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const Row<T> r(z, a.C);
  HeldRow<T, G, E> h;
  h.load(r, lane);
  const RowStats st = h.stats();
  const bool mine = lane == 0 && at < a.rows;
  if (mine) write_row<T>(a, row, z, st);
  if constexpr (TOP) {
    // k rounds: the lanes' best unused classes, then the group's; its lane looks for its next best
    uint32_t order[E];
    uint32_t best = 0, where = 0xFFFFFFFFu;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = h.at(r, lane, j);
      order[j] = (c >= 0 && c < a.C) ? class_order(h.z[j]) : 0u;
      if (order[j] > best) best = order[j], where = (uint32_t)c;
    }
    for (int i = 0; i < a.k; ++i) {
      uint32_t b = best, w = where;
      if constexpr (G == 32) {
        b = __reduce_max_sync(0xFFFFFFFFu, best);
        w = __reduce_min_sync(0xFFFFFFFFu, best == b ? where : 0xFFFFFFFFu);
      } else {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) {
          const uint32_t bo = __shfl_xor_sync(0xFFFFFFFFu, b, o), wo = __shfl_xor_sync(0xFFFFFFFFu, w, o);
          if (bo > b || (bo == b && wo < w)) b = bo, w = wo;
        }
      }
      if (mine) write_best(a, row, i, b, w, st);
      if (w == where) {
        best = 0;
        where = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const uint32_t c = (uint32_t)h.at(r, lane, j);
          if (c == w) order[j] = 0;
          if (order[j] > best) best = order[j], where = c;
        }
      }
    }
  }
}

template <typename T, int G, int E>
__global__ void __launch_bounds__(256) log_probs_held_backward_kernel(const LogProbsArgs a) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  const int64_t row = min(at, a.rows - 1);
  const int lane = threadIdx.x & (G - 1);
  const Row<T> r(static_cast<const T*>(a.logits) + row * a.ld, a.C);
  HeldRow<T, G, E> h;
  h.load(r, lane);
  const RowStats st = h.stats();
  const RowGrad g = row_grad(a, row, st);
  if constexpr (G == 1) {
    // the warp's 32 rows are one piece of dlogits: gather them in shared memory and write it in words
    __shared__ __align__(16) T stage[8][32 * E];
    T* mine = stage[warp_id()];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = h.at(r, lane, j);
      if (c >= 0 && c < a.C) mine[lane_id() * a.C + c] = from_f32<T>(score_grad(g, st, h.z[j], c));
    }
    __syncwarp();
    const int64_t row0 = at - lane_id();
    const int n = (int)min((int64_t)32, a.rows - row0) * a.C;
    if (n <= 0) return;
    T* out = static_cast<T*>(a.dlogits) + row0 * a.C;  // 32 rows: whole 4-byte words from an aligned dlogits
    constexpr int PER = 4 / sizeof(T);
    if ((reinterpret_cast<uintptr_t>(out) & 3u) == 0) {
      for (int i = lane_id(); i < n / PER; i += 32)
        reinterpret_cast<uint32_t*>(out)[i] = reinterpret_cast<const uint32_t*>(mine)[i];
      for (int i = n / PER * PER + lane_id(); i < n; i += 32) out[i] = mine[i];
    } else {
      for (int i = lane_id(); i < n; i += 32) out[i] = mine[i];
    }
  } else {
    if (at >= a.rows) return;
    T* out = static_cast<T*>(a.dlogits) + row * a.C;
    constexpr int V = Row<T>::V;
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      const int c0 = r.first(j * G + lane);
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = score_grad(g, st, h.z[j * V + e], c0 + e);
      if (c0 >= 0 && c0 + V <= a.C && (reinterpret_cast<uintptr_t>(out + c0) & 15u) == 0) {
        uint4 u;
        if constexpr (sizeof(T) == 2)
          u = make_uint4(pack_bf16x2(d[0], d[1]), pack_bf16x2(d[2], d[3]), pack_bf16x2(d[4], d[5]),
                         pack_bf16x2(d[6], d[7]));
        else
          u = make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
        *reinterpret_cast<uint4*>(out + c0) = u;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (c0 + e >= 0 && c0 + e < a.C) out[c0 + e] = from_f32<T>(d[e]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Long rows: one block per row, one pass.
// ---------------------------------------------------------------------------

// The warp's 32 best classes so far, lane i the i-th: order and the class's complement (ties to
// the lowest class), 0 where there is none yet.
struct BestList {
  unsigned long long key = 0;
  __device__ static unsigned long long make(uint32_t order, uint32_t c) {
    return ((unsigned long long)order << 32) | (uint32_t)~c;
  }
  __device__ unsigned long long threshold(int k) const { return __shfl_sync(0xFFFFFFFFu, key, k - 1); }
  // Every lane of the warp with the same `k`.
  __device__ void insert(unsigned long long k) {
    const unsigned above = __ballot_sync(0xFFFFFFFFu, key > k);
    const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, key, 1);
    const int pos = __popc(above);
    if (lane_id() == pos) key = k;
    if (lane_id() > pos) key = up;
  }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(1024) log_probs_long_forward_kernel(const LogProbsArgs a) {
  constexpr int V = Row<T>::V, U = 32 / V;  // vectors in flight: 32 scores a thread
  __shared__ float red[3][32];
  __shared__ unsigned long long keys[TOP ? 32 * TP_MAX_TOP_K : 1];
  const int64_t row = blockIdx.x;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const Row<T> r(z, a.C);
  const int nv = r.vectors(), threads = blockDim.x, warps = threads >> 5;
  float m = -INFINITY, s = 0.f, t = 0.f;
  BestList best;
  unsigned long long limit = 0;
  for (int i0 = 0; i0 < nv; i0 += U * threads) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * threads + threadIdx.x;
      if (i < nv) {
        r.load(i, v[u]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = -INFINITY;
      }
    }
    float cm = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        cm = fmaxf(cm, v[u][e]);
        if (TOP) nan |= v[u][e] != v[u][e];
      }
    if (cm > m) {
      if (m != -INFINITY) {
        const float d = fmaxf(m - cm, LP_FAR), c = exp_neg(d);
        t = c * (t + s * d);
        s *= c;
      }
      m = cm;
    }
    const float m0 = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = max_nan(v[u][e] - m0, LP_FAR), x = exp_neg(d);
        s += x;
        t += x * d;
      }
    if constexpr (TOP) {
      // most pieces hold nothing above the k-th best: one comparison for 32 scores
      const bool any = nan || class_order(cm) >= (uint32_t)(limit >> 32);
      if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int c0 = r.first(i0 + u * threads + threadIdx.x);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const int c = c0 + e;
            const bool in = c >= 0 && c < a.C;
            const unsigned long long k = in ? BestList::make(class_order(v[u][e]), (uint32_t)c) : 0ull;
            unsigned todo = __ballot_sync(0xFFFFFFFFu, k > limit);
            while (todo) {
              const unsigned long long kk = __shfl_sync(0xFFFFFFFFu, k, __ffs(todo) - 1);
              todo &= todo - 1;
              if (kk > limit) {
                best.insert(kk);
                limit = best.threshold(a.k);
              }
            }
          }
        }
      }
    }
  }
  // join the threads' sums at the block's maximum
  const float wm = group_max<32>(m);
  if (lane_id() == 0) red[0][warp_id()] = wm;
  if (TOP && lane_id() < a.k) keys[warp_id() * a.k + lane_id()] = best.key;
  __syncthreads();
  const float bm = group_max<32>(lane_id() < warps ? red[0][lane_id()] : -INFINITY);
  if (m != -INFINITY) {
    const float d = fmaxf(m - bm, LP_FAR), c = m == bm ? 1.f : exp_neg(d);
    t = m == bm ? t : c * (t + s * d);
    s *= c;
  }
  s = group_sum<32>(s);
  t = group_sum<32>(t);
  if (lane_id() == 0) {
    red[1][warp_id()] = s;
    red[2][warp_id()] = t;
  }
  __syncthreads();
  if (warp_id() != 0) return;
  s = group_sum<32>(lane_id() < warps ? red[1][lane_id()] : 0.f);
  t = group_sum<32>(lane_id() < warps ? red[2][lane_id()] : 0.f);
  const RowStats st = row_stats(bm, s, t);
  if (lane_id() == 0) write_row<T>(a, row, z, st);
  if constexpr (TOP) {
    for (int i = a.k; i < warps * a.k; ++i) {
      const unsigned long long k = keys[i];
      if (k > limit) {
        best.insert(k);
        limit = best.threshold(a.k);
      }
    }
    if (lane_id() < a.k) write_best(a, row, lane_id(), (uint32_t)(best.key >> 32), (uint32_t)~(uint32_t)best.key, st);
  }
}

// One warp per LP_CHUNK scores of a row.
template <typename T>
__global__ void __launch_bounds__(256) log_probs_stream_backward_kernel(const LogProbsArgs a, int chunks) {
  constexpr int V = Row<T>::V, U = LP_CHUNK / (32 * V);
  const int64_t task = (int64_t)blockIdx.x * 8 + warp_id();
  const int64_t row = task / chunks;
  if (row >= a.rows) return;
  const int i0 = (int)(task % chunks) * (LP_CHUNK / V) + lane_id();
  const Row<T> r(static_cast<const T*>(a.logits) + row * a.ld, a.C);
  T* out = static_cast<T*>(a.dlogits) + row * a.C;
  const int nv = r.vectors();
  RowStats st;
  st.m = a.stats[3 * row];
  st.L = a.stats[3 * row + 1];
  st.H = a.stats[3 * row + 2];
  const RowGrad g = row_grad(a, row, st);
  const bool same = ((reinterpret_cast<uintptr_t>(out) / sizeof(T)) & (V - 1)) == (uintptr_t)r.phase;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + 32 * u;
    if (i >= nv) break;
    float v[V];
    r.load(i, v);
    const int c0 = r.first(i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = score_grad(g, st, v[e], c0 + e);
    if (same && c0 >= 0 && c0 + V <= a.C) {
      uint4 w;
      if constexpr (sizeof(T) == 2)
        w = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                       pack_bf16x2(v[6], v[7]));
      else
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      *reinterpret_cast<uint4*>(out + c0) = w;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c0 + e >= 0 && c0 + e < a.C) out[c0 + e] = from_f32<T>(v[e]);
    }
  }
}

}  // namespace tp
