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
// to 1024 classes are held in registers, 16 scores a lane (32 from 512 classes on) of a thread, 4, 8,
// 16 or 32 lanes, so the row is read once and the softmax takes its maximum first (a row's fixed cost,
// reductions and label, is paid once per group: 8 scores a lane took half again as long on 50 and 200
// classes); longer rows take one block (few of them a cluster of up to eight) and one pass with a running
// maximum, the next vectors of each thread on their way meanwhile.  Rows start anywhere: whole 16-byte
// vectors are loaded between the first and last boundary inside the row, single elements before and after.
//
// The best classes take nothing from the pass: the k-th largest of the threads' maxima is a bound that
// at least k scores reach and few others do.  Only the threads whose maximum reaches it have
// their scores looked at again (a long row's from the cache, spread over the block); what reaches the
// bound goes through shared memory into a sort of 32 keys and a sorted list of 32.
#pragma once

#include "gemm_simt.cuh"

namespace tp {

struct LogProbsArgs {
  int64_t rows;
  int C;
  int64_t ld;              // row stride of the logits
  const void* logits;
  const int64_t* labels;
  uint32_t label_rows;     // row r has label r % label_rows; 0: its own
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
constexpr int LP_WARPS = 8;          // of a block on long rows, at most
constexpr int LP_CHUNK = 2048;       // classes of one warp in the streaming backward

__device__ __forceinline__ float lp_nan() { return __uint_as_float(0x7FC00000u); }

// exp(x) for x <= 0 from the base-2 exponential (2^-22 relative, and x's rounding times |x|).
__device__ __forceinline__ float exp_neg(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}

__device__ __forceinline__ f32x2 exp_neg2(f32x2 x) {
  const float2 y = halves(mul2(x, pair(1.4426950408889634f, 1.4426950408889634f)));
  float2 r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(y.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(y.y));
  return pair(r.x, r.y);
}

// z - max, bounded below, of two scores.
__device__ __forceinline__ f32x2 bounded2(f32x2 d) {
  const float2 t = halves(d);
  return pair(max_nan(t.x, LP_FAR), max_nan(t.y, LP_FAR));
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
  // Vector i as it is stored; elements outside the row read as -inf.
  __device__ uint4 raw(int i) const {
    const int c0 = first(i);
    if (c0 >= 0 && c0 + V <= C) return __ldg(reinterpret_cast<const uint4*>(base) + i);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const bool in = c0 + e >= 0 && c0 + e < C;
      const T* p = base + (int64_t)i * V + e;
      if constexpr (sizeof(T) == 2) {
        const uint32_t h = in ? *reinterpret_cast<const uint16_t*>(p) : 0xFF80u;
        w[e / 2] = e % 2 ? w[e / 2] | h << 16 : h;
      } else {
        w[e] = in ? *reinterpret_cast<const uint32_t*>(p) : 0xFF800000u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static uint4 nothing() {
    const uint32_t w = sizeof(T) == 2 ? 0xFF80FF80u : 0xFF800000u;
    return make_uint4(w, w, w, w);
  }
  __device__ static void unpack(const uint4& u, float* v) {
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
  // Writes vector i of a row that begins at `out` (C elements), by 16 bytes where it can.
  __device__ void store(T* out, int i, const float (&d)[V]) const {
    const int c0 = first(i);
    if (c0 >= 0 && c0 + V <= C && (reinterpret_cast<uintptr_t>(out + c0) & 15u) == 0) {
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
        if (c0 + e >= 0 && c0 + e < C) out[c0 + e] = from_f32<T>(d[e]);
    }
  }
};

// A row's label, loaded before the row is reduced.
__device__ __forceinline__ int64_t row_label(const LogProbsArgs& a, int64_t row) {
  return a.labels[a.label_rows ? (uint32_t)row % a.label_rows : (uint32_t)row];
}

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
struct RowLabel {
  float z;        // the label's score
  bool in, skip;  // a class of the row; equal to ignore_index
  template <typename T>
  __device__ RowLabel(const LogProbsArgs& a, int64_t row, const T* scores) {
    const int64_t y = row_label(a, row);
    skip = y == a.ignore_index;
    in = y >= 0 && y < a.C;
    z = in ? to_f32<T>(scores[y]) : 0.f;
  }
};

__device__ __forceinline__ void write_row(const LogProbsArgs& a, int64_t row, const RowLabel& y, const RowStats& st) {
  a.log_prob[row] = y.skip ? 0.f : !y.in ? lp_nan() : st.empty() ? -INFINITY : y.z - st.m - st.L;
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

// dz = p (a + b log p) with a = -(g_l + g_H H), b = -g_H, and g_l at the label.
struct RowGrad {
  f32x2 m, L, a, b;  // the first two negated
  float gl;
  int y;             // -1: no label's term
};

// What a row's gradient takes besides its scores, loaded before the row is reduced.
struct RowUpstream {
  int64_t y;
  float gl, gh;
  __device__ RowUpstream(const LogProbsArgs& a, int64_t row) {
    y = row_label(a, row);
    gl = a.g_l ? a.g_l[row * a.g_l_stride] : 0.f;
    gh = a.g_h ? a.g_h[row * a.g_h_stride] : 0.f;
  }
};

__device__ __forceinline__ RowGrad row_grad(const LogProbsArgs& a, const RowUpstream& up, const RowStats& st) {
  RowGrad g;
  const int64_t y = up.y;
  const float gh = up.gh;
  g.gl = up.gl;
  g.y = -1;
  if (!a.g_l || y == a.ignore_index)
    g.gl = 0.f;
  else if (y < 0 || y >= a.C)
    g.gl = lp_nan();
  else if (!st.empty())
    g.y = (int)y;
  const float u = st.empty() ? 0.f : -(g.gl + gh * st.H), m = st.empty() ? 0.f : -st.m;
  g.a = pair(u, u);
  g.b = pair(-gh, -gh);
  g.m = pair(m, m);  // a row without classes: every p is 0
  g.L = pair(-st.L, -st.L);
  return g;
}

// In place, V scores from class c0 on; `known`: their probabilities, where they are at hand.
template <int V, bool KNOWN>
__device__ __forceinline__ void score_grad(const RowGrad& g, float (&z)[V], int c0, const float* known) {
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    // a masked class: p = 0 and a finite log p, so that its product is 0
    const f32x2 lp = bounded2(add2(add2(pair(z[e], z[e + 1]), g.m), g.L));
    const float2 d = halves(mul2(KNOWN ? pair(known[e], known[e + 1]) : exp_neg2(lp), fma2(g.b, lp, g.a)));
    z[e] = d.x, z[e + 1] = d.y;
  }
  if ((unsigned)(g.y - c0) < (unsigned)V && g.y >= 0) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c0 + e == g.y) z[e] += g.gl;
  }
}

// ---------------------------------------------------------------------------
// Rows in registers: G lanes (1 to 32) hold E scores each, vectors of the row in turn.
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
    uint4 u[E / V];
#pragma unroll
    for (int j = 0; j < E / V; ++j) u[j] = r.raw(j * G + lane);
#pragma unroll
    for (int j = 0; j < E / V; ++j) Row<T>::unpack(u[j], z + j * V);
  }
  __device__ float own_max() const {  // of the lane's scores, -inf without any (a NaN is passed over)
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) m = fmaxf(m, z[j]);
    return m;
  }
  // KEEP: leaves exp(z - max) / S in `p`.
  template <bool KEEP = false>
  __device__ RowStats stats(float own, float* p = nullptr) const {
    const float m = group_max<G>(own);
    const float m0 = m == -INFINITY ? 0.f : -m;
    f32x2 s = pair(0.f, 0.f), t = s;
#pragma unroll
    for (int j = 0; j < E; j += 2) {
      const f32x2 d = bounded2(add2(pair(z[j], z[j + 1]), pair(m0, m0))), e = exp_neg2(d);
      s = add2(s, e);
      t = fma2(e, d, t);
      if constexpr (KEEP) {
        const float2 f = halves(e);
        p[j] = f.x, p[j + 1] = f.y;
      }
    }
    const float2 a = halves(s), b = halves(t);
    const float sum = group_sum<G>(a.x + a.y);
    if constexpr (KEEP) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
      for (int j = 0; j < E; ++j) p[j] *= inv;
    }
    return row_stats(m, sum, group_sum<G>(b.x + b.y));
  }
  __device__ static int at(const Row<T>& r, int lane, int j) { return r.first((j / V) * G + lane) + j % V; }
};

// ---------------------------------------------------------------------------
// Best classes of a warp.  A key is a score's order and the class's complement (ties to the lowest
// class), 0 where there is none.
// ---------------------------------------------------------------------------
typedef unsigned long long class_key;
constexpr int LP_CANDIDATES = 128;  // keys of one piece in shared memory

__device__ __forceinline__ class_key make_key(uint32_t order, uint32_t c) {
  return ((class_key)order << 32) | (uint32_t)~c;
}

// Bitonic networks over the lanes, descending (Batcher, 1968): all stages, or the last only, which
// sorts a bitonic sequence.
template <typename K>
__device__ __forceinline__ K lanes_exchange(K v, int stride, bool keep_max) {
  const K o = __shfl_xor_sync(0xFFFFFFFFu, v, stride);
  return (v < o) == keep_max ? o : v;
}
template <typename K>
__device__ __forceinline__ K lanes_merge(K v) {
#pragma unroll
  for (int stride = 16; stride > 0; stride >>= 1) v = lanes_exchange(v, stride, (lane_id() & stride) == 0);
  return v;
}
template <typename K>
__device__ __forceinline__ K lanes_sort(K v) {
#pragma unroll
  for (int size = 2; size < 32; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1)
      v = lanes_exchange(v, stride, ((lane_id() & stride) == 0) == ((lane_id() & size) == 0));
  return lanes_merge(v);
}

// The warp's 32 best classes so far, lane i the i-th.
struct BestList {
  class_key key = 0;
  __device__ class_key limit(int k) const { return __shfl_sync(0xFFFFFFFFu, key, k - 1); }
  // Takes in the lanes' keys, descending.
  __device__ void join(class_key sorted) {
    const class_key o = __shfl_sync(0xFFFFFFFFu, sorted, 31 - lane_id());
    key = lanes_merge(max(key, o));
  }
  // Every lane of the warp with the same `k`.
  __device__ void insert(class_key k) {
    const unsigned above = __ballot_sync(0xFFFFFFFFu, key > k);
    const class_key up = __shfl_up_sync(0xFFFFFFFFu, key, 1);
    const int pos = __popc(above);
    if (lane_id() == pos) key = k;
    if (lane_id() > pos) key = up;
  }
};

// Takes the lanes' N scores into the list.  `cls(j)`: the class of a lane's j-th score, -1 for none;
// `bound`: a value that the k best scores reach (a NaN does too).  What reaches it, usually little
// more than k keys, is gathered in `buf` (LP_CANDIDATES keys and a counter of this warp, 0 on entry
// and on exit); where it does not fit (many equal scores) the keys are inserted one by one.
template <int N, typename F>
__device__ __forceinline__ void best_take(BestList& best, int k, const float (&z)[N], F cls, float bound, class_key* buf,
                                          int* count) {
  class_key limit = best.limit(k);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (z[j] < bound) continue;
    const int c = cls(j);
    const class_key key = make_key(class_order(z[j]), (uint32_t)c);
    if (c >= 0 && key > limit) {
      const int at = atomicAdd(count, 1);
      if (at < LP_CANDIDATES) buf[at] = key;
    }
  }
  __syncwarp();
  const int n = *count;
  __syncwarp();
  if (lane_id() == 0) *count = 0;
  if (n <= LP_CANDIDATES) {
    for (int i = 0; i < n; i += 32) best.join(lanes_sort(i + lane_id() < n ? buf[i + lane_id()] : (class_key)0));
  } else {
#pragma unroll 1
    for (int j = 0; j < N; ++j) {
      const int c = cls(j);
      float v = z[0];  // z[j] without an index into registers
#pragma unroll
      for (int i = 1; i < N; ++i)
        if (i == j) v = z[i];
      const class_key key = c >= 0 ? make_key(class_order(v), (uint32_t)c) : (class_key)0;
      unsigned todo = __ballot_sync(0xFFFFFFFFu, key > limit);
      while (todo) {
        const class_key one = __shfl_sync(0xFFFFFFFFu, key, __ffs(todo) - 1);
        todo &= todo - 1;
        if (one > limit) {
          best.insert(one);
          limit = best.limit(k);
        }
      }
    }
  }
  __syncwarp();
}

// A key of a held row's class: 32 bits are enough for bf16, whose scores have 16.
template <typename T>
struct HeldKey {
  typedef class_key type;
  __device__ static type make(float z, int c) { return make_key(class_order(z), (uint32_t)c); }
  __device__ static uint32_t order(type k) { return (uint32_t)(k >> 32); }
  __device__ static uint32_t class_of(type k) { return ~(uint32_t)k; }
};
template <>
struct HeldKey<__nv_bfloat16> {
  typedef uint32_t type;
  // of an order's low half, all zeros or (below zero, and a NaN) all ones, nothing is lost
  __device__ static type make(float z, int c) { return (class_order(z) & 0xFFFF0000u) | (uint32_t)(0xFFFF - c); }
  __device__ static uint32_t order(type k) { return (k & 0x80000000u) ? (k & 0xFFFF0000u) : (k | 0xFFFFu); }
  __device__ static uint32_t class_of(type k) { return 0xFFFFu - (k & 0xFFFFu); }
};

// blockDim 256; a row beyond the last is computed again from the last and not written.
template <typename T, int G, int E, bool TOP>
__global__ void __launch_bounds__(256) log_probs_held_forward_kernel(const LogProbsArgs a) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  const int64_t row = min(at, a.rows - 1);
  const int lane = threadIdx.x & (G - 1);
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const Row<T> r(z, a.C);
  const RowLabel label(a, row, z);
  HeldRow<T, G, E> h;
  h.load(r, lane);
  const float own = h.own_max();
  const RowStats st = h.stats(own);
  const bool mine = lane == 0 && at < a.rows;
  if (mine) write_row(a, row, label, st);
  if constexpr (TOP) {
    if constexpr (G < 32) {
      // k rounds: the lanes' best classes below the last one taken, then the group's; its lane looks for
      // its next best
      typedef HeldKey<T> Key;
      typename Key::type key[E], best = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = h.at(r, lane, j);
        key[j] = (c >= 0 && c < a.C) ? Key::make(h.z[j], c) : 0;
        best = max(best, key[j]);
      }
      for (int i = 0; i < a.k; ++i) {
        typename Key::type b = best;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xFFFFFFFFu, b, o));
        if (mine) write_best(a, row, i, Key::order(b), Key::class_of(b), st);
        if (b == best) {
          best = 0;
#pragma unroll
          for (int j = 0; j < E; ++j) best = max(best, key[j] < b ? key[j] : 0);
        }
      }
    } else {
      __shared__ class_key buf[8][LP_CANDIDATES];
      __shared__ int count[8];
      if (lane == 0) count[warp_id()] = 0;
      __syncwarp();
      const auto cls = [&](int j) {
        const int c = h.at(r, lane, j);
        return c < a.C ? c : -1;
      };
      const float bound = class_value(__shfl_sync(0xFFFFFFFFu, lanes_sort(class_order(own)), a.k - 1));
      BestList best;
      best_take<E>(best, a.k, h.z, cls, bound, buf[warp_id()], &count[warp_id()]);
      if (lane < a.k && at < a.rows)
        write_best(a, row, lane, (uint32_t)(best.key >> 32), (uint32_t)~(uint32_t)best.key, st);
    }
  }
}

template <typename T, int G, int E>
__global__ void __launch_bounds__(256) log_probs_held_backward_kernel(const LogProbsArgs a) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
  const int64_t row = min(at, a.rows - 1);
  const int lane = threadIdx.x & (G - 1);
  const Row<T> r(static_cast<const T*>(a.logits) + row * a.ld, a.C);
  const RowUpstream up(a, row);
  HeldRow<T, G, E> h;
  h.load(r, lane);
  float p[E];
  const RowStats st = h.template stats<true>(h.own_max(), p);
  const RowGrad g = row_grad(a, up, st);
  constexpr int V = Row<T>::V;
  T* out = static_cast<T*>(a.dlogits) + row * a.C;
  // the same for every row: a warp's groups stay together
  const bool aligned = a.C % V == 0 && a.ld % V == 0 &&
                       ((reinterpret_cast<uintptr_t>(a.dlogits) | reinterpret_cast<uintptr_t>(a.logits)) & 15u) == 0;
  if (G == 32 || (G > 1 && aligned)) {
    if (at >= a.rows) return;
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = h.z[j * V + e];
      score_grad<V, true>(g, d, r.first(j * G + lane), p + j * V);
      r.store(out, j * G + lane, d);
    }
  } else if constexpr (G < 32) {
    // short rows that begin anywhere: the warp's rows are one piece of dlogits, gathered in shared
    // memory and written 16 bytes at a time
    __shared__ __align__(16) T stage[8][32 * E];
    T* mine = stage[warp_id()];
    const int slot = lane_id() / G;
#pragma unroll
    for (int j = 0; j < E / V; ++j) {
      float d[V];
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = h.z[j * V + e];
      const int c0 = r.first(j * G + lane);
      score_grad<V, true>(g, d, c0, p + j * V);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (c0 + e >= 0 && c0 + e < a.C) mine[slot * a.C + c0 + e] = from_f32<T>(d[e]);
    }
    __syncwarp();
    const int64_t row0 = at - slot;
    const int n = (int)max((int64_t)0, min((int64_t)(32 / G), a.rows - row0)) * a.C;
    out = static_cast<T*>(a.dlogits) + row0 * a.C;
    int i = 0;
    if ((reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
      for (; i + V <= n; i += V * 32)
        if (i + V * (lane_id() + 1) <= n)
          reinterpret_cast<uint4*>(out + i)[lane_id()] = reinterpret_cast<const uint4*>(mine + i)[lane_id()];
      i = n / V * V;
    }
    for (i += lane_id(); i < n; i += 32) out[i] = mine[i];
  }
}

// ---------------------------------------------------------------------------
// Long rows: one block per row (or a cluster, where the rows are few), one pass.
// ---------------------------------------------------------------------------

// Sums of exp(z - m) and exp(z - m) (z - m) taken over to a maximum `to` >= m.
__device__ __forceinline__ void rescale(float m, float to, float& s, float& t) {
  if (m == -INFINITY || m == to) return;
  const float d = fmaxf(m - to, LP_FAR), c = exp_neg(d);
  t = c * (t + s * d);
  s *= c;
}

// n sorted lists of a block's warps, this warp's `list` also in lists[its number], two by two into
// lists[0].  Every thread, after a __syncthreads; ends with one.
__device__ __forceinline__ void merge_lists(uint32_t list, uint32_t (*lists)[32], int n) {
  const int wid = warp_id();
  for (int half = LP_WARPS / 2; half > 0; half >>= 1) {
    if (wid < half && wid + half < n) {
      list = lanes_merge(max(list, lists[wid + half][31 - lane_id()]));
      lists[wid][lane_id()] = list;
    }
    __syncthreads();
  }
}

// The same for best classes; warp 0 ends with the result in `best` and in lists[0].
__device__ __forceinline__ void join_lists(BestList& best, class_key (*lists)[LP_CANDIDATES], int n) {
  const int wid = warp_id();
  for (int half = LP_WARPS / 2; half > 0; half >>= 1) {
    if (wid < half && wid + half < n) {
      best.join(lists[wid + half][lane_id()]);
      lists[wid][lane_id()] = best.key;
    }
    if (half < n) __syncthreads();
  }
}

// SPLIT: the row is spread over the `cluster` CTAs of a thread-block cluster, which read each other's
// sums and lists through distributed shared memory; the first one writes.
// A thread keeps 3 (bf16) or 4 (fp32) vectors on their way, which leaves room for four blocks an SM without
// spills (8192 rows of 65536 in bf16: 190 us; 4 vectors with spills 221, with three blocks an SM 198; in
// fp32, 4096 rows of 40000: 104 us with 4, 110 with 3).
// Pieces inside the row are loaded without a check per vector: 177 us instead of 190 for those rows, 95 % of a
// copy's rate (with the best classes the same change took 60 us instead of 57 for 2048 rows of 50000: not there).
template <typename T, bool TOP, bool SPLIT>
__global__ void __launch_bounds__(32 * LP_WARPS, SPLIT ? 1 : 4)
    log_probs_long_forward_kernel(const LogProbsArgs a, int cluster) {
  constexpr int V = Row<T>::V, U = V == 8 ? 3 : 4;  // vectors of a thread in one piece
  __shared__ float red[3][LP_WARPS];
  __shared__ class_key buf[TOP ? LP_WARPS : 1][TOP ? LP_CANDIDATES : 1];
  __shared__ uint32_t maxima[TOP ? LP_WARPS : 1][32];
  __shared__ uint16_t again[TOP ? 32 * LP_WARPS : 1];  // threads whose scores are looked at again
  __shared__ int count[LP_WARPS + 1];                  // of each warp's buf; last: of `again`
  __shared__ float sums[3];                            // SPLIT: this CTA's maximum and sums
  __shared__ uint32_t all[TOP && SPLIT ? LP_WARPS : 1][32];
  const int rank = SPLIT ? (int)cluster_ctarank() : 0, parts = SPLIT ? cluster : 1;
  const int64_t row = blockIdx.x / (unsigned)parts;
  const T* z = static_cast<const T*>(a.logits) + row * a.ld;
  const Row<T> r(z, a.C);
  const int nv = r.vectors(), threads = blockDim.x, warps = threads >> 5, wid = warp_id();
  const int stride = threads * parts, mine = rank * threads + threadIdx.x;  // vectors mine, mine + stride, ...
  if (TOP && lane_id() == 0) count[wid] = count[LP_WARPS] = 0;
  const int whole = (r.phase + a.C) / V;  // vectors before the last one that the row cuts
  float m = -INFINITY;
  f32x2 s = pair(0.f, 0.f), t = s;
  uint4 next[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * stride + mine;
    next[u] = i < nv ? r.raw(i) : Row<T>::nothing();
  }
  for (int i0 = 0; i0 < nv; i0 += U * stride) {
    float v[U * V];
#pragma unroll
    for (int u = 0; u < U; ++u) Row<T>::unpack(next[u], v + u * V);
    if (!TOP && i0 + 2 * U * stride <= whole) {
      const uint4* p = reinterpret_cast<const uint4*>(r.base) + (i0 + U * stride + mine);
#pragma unroll
      for (int u = 0; u < U; ++u) next[u] = __ldg(p + u * stride);
    } else if (i0 + U * stride < nv) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + (U + u) * stride + mine;
        next[u] = i < nv ? r.raw(i) : Row<T>::nothing();
      }
    }
    float cm = -INFINITY;
#pragma unroll
    for (int e = 0; e < U * V; ++e) cm = fmaxf(cm, v[e]);
    if (cm > m) {
      if (m != -INFINITY) {
        const float d = fmaxf(m - cm, LP_FAR), c = exp_neg(d);
        t = mul2(pair(c, c), fma2(s, pair(d, d), t));
        s = mul2(s, pair(c, c));
      }
      m = cm;
    }
    const float m0 = m == -INFINITY ? 0.f : -m;
#pragma unroll
    for (int e = 0; e < U * V; e += 2) {
      const f32x2 d = bounded2(add2(pair(v[e], v[e + 1]), pair(m0, m0))), x = exp_neg2(d);
      s = add2(s, x);
      t = fma2(x, d, t);
    }
  }
  // join the threads' sums at the block's maximum
  const float wm = group_max<32>(m);
  if (lane_id() == 0) red[0][wid] = wm;
  const float2 sh = halves(s), th = halves(t);
  float s1 = sh.x + sh.y, t1 = th.x + th.y;
  uint32_t order = 0, list = 0;  // the thread's maximum; the warp's, sorted
  if constexpr (TOP) {
    // a thread with a NaN, which its sum then holds, is above all; one without scores counts as -inf
    order = s1 != s1 ? 0xFFFFFFFFu : class_order(m);
    list = lanes_sort(order);
    maxima[wid][lane_id()] = list;
  }
  __syncthreads();
  float bm = group_max<32>(lane_id() < warps ? red[0][lane_id()] : -INFINITY);
  rescale(m, bm, s1, t1);
  s1 = group_sum<32>(s1);
  t1 = group_sum<32>(t1);
  if (lane_id() == 0) {
    red[1][wid] = s1;
    red[2][wid] = t1;
  }
  if constexpr (TOP) {
    // the k-th largest of all threads' maxima: the warps' sorted lists, two by two
    merge_lists(list, maxima, warps);
  } else {
    __syncthreads();
  }
  if constexpr (SPLIT) {
    s1 = group_sum<32>(lane_id() < warps ? red[1][lane_id()] : 0.f);
    t1 = group_sum<32>(lane_id() < warps ? red[2][lane_id()] : 0.f);
    if (threadIdx.x == 0) sums[0] = bm, sums[1] = s1, sums[2] = t1;
    __syncwarp();
    cluster_sync();
    // lane i holds CTA i's maximum and sums
    const bool other = lane_id() < parts;
    const uint32_t at = mapa_shared(smem_u32(sums), other ? lane_id() : 0);
    const float om = other ? __uint_as_float(ld_shared_cluster_u32(at)) : -INFINITY;
    s1 = other ? __uint_as_float(ld_shared_cluster_u32(at + 4)) : 0.f;
    t1 = other ? __uint_as_float(ld_shared_cluster_u32(at + 8)) : 0.f;
    bm = group_max<32>(om);
    rescale(om, bm, s1, t1);
    s1 = group_sum<32>(s1);
    t1 = group_sum<32>(t1);
  }
  BestList best;
  if constexpr (TOP) {
    uint32_t bound = maxima[0][a.k - 1];
    if constexpr (SPLIT) {
      // the CTAs' lists, one a warp, and again two by two
      list = wid < parts ? ld_shared_cluster_u32(mapa_shared(smem_u32(&maxima[0][lane_id()]), wid)) : 0u;
      all[wid][lane_id()] = list;
      __syncthreads();
      merge_lists(list, all, parts);
      bound = all[0][a.k - 1];
    }
    if (order >= bound) again[atomicAdd(&count[LP_WARPS], 1)] = (uint16_t)threadIdx.x;
    __syncthreads();
    // those threads' vectors, spread over the block
    const int per = (nv + stride - 1) / stride;
    const int64_t tasks = (int64_t)count[LP_WARPS] * per;
    for (int64_t p0 = wid * 32; p0 < tasks; p0 += threads) {
      const int64_t p = p0 + lane_id();
      const int64_t i64 = p < tasks ? rank * threads + again[p / per] + (p % per) * stride : nv;
      const int i = (int)min(i64, (int64_t)nv);
      float v[V];
      Row<T>::unpack(i < nv ? r.raw(i) : Row<T>::nothing(), v);
      const auto cls = [&](int j) {
        const int c = r.first(i) + j;
        return i < nv && c < a.C ? c : -1;
      };
      best_take<V>(best, a.k, v, cls, class_value(bound), buf[wid], &count[wid]);
    }
    const int lists = (int)min((int64_t)warps, (tasks + 31) / 32);
    buf[wid][lane_id()] = best.key;
    __syncthreads();
    join_lists(best, buf, lists);
    if constexpr (SPLIT) {
      __syncwarp();
      cluster_sync();
      if (rank == 0) {
        if (wid > 0) best.key = wid < parts ? ld_shared_cluster_u64(mapa_shared(smem_u32(&buf[0][lane_id()]), wid)) : 0ull;
        if (wid > 0) buf[wid][lane_id()] = best.key;
        __syncthreads();
        join_lists(best, buf, parts);
      }
      __syncwarp();
    }
  }
  if constexpr (SPLIT) {
    cluster_sync();  // no CTA leaves while the first one reads its lists
    if (rank != 0) return;
  }
  if (wid != 0) return;
  if constexpr (!SPLIT) {
    s1 = group_sum<32>(lane_id() < warps ? red[1][lane_id()] : 0.f);
    t1 = group_sum<32>(lane_id() < warps ? red[2][lane_id()] : 0.f);
  }
  const RowStats st = row_stats(bm, s1, t1);
  if (lane_id() == 0) write_row(a, row, RowLabel(a, row, z), st);
  if (TOP && lane_id() < a.k)
    write_best(a, row, lane_id(), (uint32_t)(best.key >> 32), (uint32_t)~(uint32_t)best.key, st);
}

// One warp per LP_CHUNK scores of a row.  Five blocks an SM, 48 registers (50 registers, four
// blocks: 348 us instead of 324 for 8192 rows of 65536 in bf16).
template <typename T>
__global__ void __launch_bounds__(256, 5) log_probs_stream_backward_kernel(const LogProbsArgs a, int chunks) {
  constexpr int V = Row<T>::V, U = LP_CHUNK / (32 * V);
  const uint32_t task = blockIdx.x * 8 + warp_id();
  const uint32_t row = task / (uint32_t)chunks;
  if (row >= a.rows) return;
  const int i0 = (int)(task % (uint32_t)chunks) * (LP_CHUNK / V) + lane_id();
  const Row<T> r(static_cast<const T*>(a.logits) + (int64_t)row * a.ld, a.C);
  T* out = static_cast<T*>(a.dlogits) + (int64_t)row * a.C;
  const int nv = r.vectors();
  RowStats st;
  st.m = a.stats[3 * (int64_t)row];
  st.L = a.stats[3 * (int64_t)row + 1];
  st.H = a.stats[3 * (int64_t)row + 2];
  const RowGrad g = row_grad(a, RowUpstream(a, row), st);
  for (int u0 = 0; u0 < U; u0 += 4) {
    uint4 raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * (u0 + u);
      raw[u] = i < nv ? r.raw(i) : Row<T>::nothing();
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * (u0 + u);
      if (i >= nv) return;
      float d[V];
      Row<T>::unpack(raw[u], d);
      score_grad<V, false>(g, d, r.first(i), nullptr);
      r.store(out, i, d);
    }
  }
}

}  // namespace tp
