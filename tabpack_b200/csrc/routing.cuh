// Routing of rows to the members of a pack, and the moves of rows that it asks for.
//
// Per row of scores z over E members: p = softmax(z), the k best finite z (ties: lowest member), their
// weights w = p / sum of the chosen p, or p.  The (row, slot) pairs are sorted by member with a stable
// counting sort: `position` is a pair's place, `offsets` where a member's rows begin; pairs without a member
// (a row with fewer than k finite scores) come after the last member's.
//
// The gate reads each score once and holds a row in one warp's registers; the sort adds a count per block and
// member, which the second launch sums up itself instead of in a launch of its own.
#pragma once

#include "common.cuh"

namespace tp {

constexpr int ROUTE_MAX_EXPERTS = 1024;
constexpr int ROUTE_MAX_K = 32;
constexpr int ROUTE_WARPS = 16;

struct RouteArgs {
  int rows, E, k, renorm;
  long long ld;           // elements between rows of the scores
  const void* logits;
  float* weight;          // (rows, k)
  int32_t* expert;        // (rows, k), -1 where there is none
  int32_t* position;      // (rows, k)
  int32_t* offsets;       // (E + 1)
  float* importance;      // (E)
  int32_t* counts;        // workspace (blocks, E + 1)
  float* partial;         // workspace (blocks, E): sums of p over a block's rows
  int rows_per_block;
  const float* g_weight;      // backward, (rows, k) or null
  const float* g_importance;  // (E) or null
  void* dlogits;              // (rows, E)
};

// fp32 as an unsigned number of the same order; every NaN above +inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xFFFFFFFFu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
constexpr uint32_t KEY_NEG_INF = 0x007FFFFFu;  // the key of -inf; smaller ones are of no score

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// A row's scores as keys, lane l holding members l, l + 32, ...; 0 past the last member.
template <typename T, int V>
__device__ __forceinline__ void route_load(const T* z, int E, int lane, uint32_t (&key)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    key[v] = e < E ? order_key((float)z[e]) : 0u;
  }
}

// Shared memory of both phases: counts[ROUTE_WARPS][E + 1], then base[E + 1], then sums[ROUTE_WARPS][E].
__host__ __device__ inline size_t route_shared_bytes(int E) {
  return sizeof(int) * ((size_t)(ROUTE_WARPS + 1) * (E + 1) + (size_t)ROUTE_WARPS * E);
}

// Weights and members of the block's rows, their counts per member, and the sums of p.
template <typename T, int V>
__device__ __forceinline__ void route_gate(const RouteArgs& a, int block, int* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = a.E, k = a.k;
  int* hist = smem + ROUTE_WARPS * (E + 1);
  float* sums = reinterpret_cast<float*>(hist + E + 1);
  for (int e = threadIdx.x; e <= E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int r0 = block * a.rows_per_block, r1 = min(a.rows, r0 + a.rows_per_block);
  float imp[V];
#pragma unroll
  for (int v = 0; v < V; ++v) imp[v] = 0.f;
  for (int r = r0 + warp; r < r1; r += ROUTE_WARPS) {
    uint32_t key[V];
    route_load<T, V>(static_cast<const T*>(a.logits) + (long long)r * a.ld, E, lane, key);
    // this lane's best and its member: the lowest of equal ones
    uint32_t best = 0;
    int which = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) {
        best = key[v];
        which = lane + 32 * v;
      }
    const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
    const bool some = top > KEY_NEG_INF;
    const float zmax = some ? key_value(top) : 0.f;
    float e[V], total = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      e[v] = key[v] > KEY_NEG_INF ? expf(key_value(key[v]) - zmax) : 0.f;
      total += e[v];
    }
    total = warp_sum(total);
    const float inv = some ? 1.f / total : 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) imp[v] = fmaf(e[v], inv, imp[v]);
    // the k best: lane j keeps slot j
    uint32_t my_key = 0;
    int my_expert = -1;
    for (int j = 0; j < k; ++j) {
      const uint32_t b = j == 0 ? top : __reduce_max_sync(0xFFFFFFFFu, best);
      if (b <= KEY_NEG_INF) break;
      const int who = (int)__reduce_min_sync(0xFFFFFFFFu, best == b ? (unsigned)which : 0xFFFFFFFFu);
      if (lane == j) {
        my_key = b;
        my_expert = who;
      }
      if (which == who && best == b) {  // this lane's next best
        best = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (lane + 32 * v == who) key[v] = 0;
          if (key[v] > best) {
            best = key[v];
            which = lane + 32 * v;
          }
        }
      }
    }
    float w = my_expert >= 0 ? expf(key_value(my_key) - zmax) : 0.f;
    if (a.renorm) {
      const float s = warp_sum(w);
      w = my_expert >= 0 ? w / s : 0.f;
    } else {
      w = my_expert >= 0 ? w / total : 0.f;
    }
    if (lane < k) {
      a.weight[(long long)r * k + lane] = w;
      a.expert[(long long)r * k + lane] = my_expert;
      atomicAdd(&hist[my_expert < 0 ? E : my_expert], 1);  // whole numbers: any order gives the same count
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane + 32 * v < E) sums[warp * E + lane + 32 * v] = imp[v];
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    a.counts[(long long)block * (E + 1) + e] = hist[e];
    if (e < E) {
      float s = 0.f;
      for (int w = 0; w < ROUTE_WARPS; ++w) s += sums[w * E + e];
      a.partial[(long long)block * E + e] = s;
    }
  }
}

// Places of the block's pairs, and the block's share of the offsets and sums.
__device__ __forceinline__ void route_place(const RouteArgs& a, int block, int blocks, int* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = a.E;
  int* cnt = smem;                             // [warp][E + 1]
  int* base = smem + ROUTE_WARPS * (E + 1);    // [E + 1]
  __shared__ int carry[33];
  // counts of earlier blocks and of all of them, per member; then where the member's rows begin
  if (threadIdx.x < 33) carry[threadIdx.x] = 0;
  __syncthreads();
  for (int e0 = 0; e0 <= E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    int before = 0, all = 0;
    if (e <= E) {
#pragma unroll 8
      for (int b = 0; b < blocks; ++b) {
        const int c = a.counts[(long long)b * (E + 1) + e];
        before += b < block ? c : 0;
        all += c;
      }
    }
    int inc = all;  // inclusive sums over the block's threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) carry[warp] = inc;
    __syncthreads();
    int first = carry[32];
    for (int w = 0; w < warp; ++w) first += carry[w];
    first += inc - all;
    __syncthreads();
    if (threadIdx.x == blockDim.x - 1) carry[32] = first + all;
    if (e <= E) {
      base[e] = first + before;
      if (block == 0) a.offsets[e] = first;
    }
    __syncthreads();
  }
  // each warp's pairs are consecutive; its counts per member come before its places
  for (int i = threadIdx.x; i < ROUTE_WARPS * (E + 1); i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int r0 = block * a.rows_per_block, r1 = min(a.rows, r0 + a.rows_per_block);
  const int pairs = max(0, r1 - r0) * a.k, first_pair = r0 * a.k;
  const int per = ((pairs + ROUTE_WARPS - 1) / ROUTE_WARPS + 31) & ~31;
  const int p0 = min(pairs, warp * per), p1 = min(pairs, p0 + per);
  int* mine = cnt + warp * (E + 1);
  for (int pass = 0; pass < 2; ++pass) {
    for (int p = p0; p < p1; p += 32) {
      const bool in = p + lane < p1;
      const unsigned active = __ballot_sync(0xFFFFFFFFu, in);
      if (in) {
        int e = a.expert[first_pair + p + lane];
        if (e < 0) e = E;
        const unsigned same = __match_any_sync(active, e);
        const unsigned lower = same & ((1u << lane) - 1u);
        if (pass) a.position[first_pair + p + lane] = mine[e] + __popc(lower);
        __syncwarp(active);
        if (!lower) mine[e] += __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();
    if (pass == 0) {
      for (int e = threadIdx.x; e <= E; e += blockDim.x) {
        int run = base[e];
        for (int w = 0; w < ROUTE_WARPS; ++w) {
          const int c = cnt[w * (E + 1) + e];
          cnt[w * (E + 1) + e] = run;
          run += c;
        }
      }
      __syncthreads();
    }
  }
  // the sums of p: members block, block + blocks, ..., a warp each
  for (int e = block + blocks * warp; e < E; e += blocks * ROUTE_WARPS) {
    float s = 0.f;
    for (int b = lane; b < blocks; b += 32) s += a.partial[(long long)b * E + e];
    s = warp_sum(s);
    if (lane == 0) a.importance[e] = s;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_gate_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_gate<T, V>(a, blockIdx.x, route_smem);
}

__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_place_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_place(a, blockIdx.x, gridDim.x, route_smem);
}

// Few rows: both phases in one block.
template <typename T, int V>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_small_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_gate<T, V>(a, 0, route_smem);
  __syncthreads();
  route_place(a, 0, 1, route_smem);
}

// dz of a row by one warp: p is formed again from the scores (reading it would cost more than the sums).
template <typename T, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs a) {
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const int E = a.E, k = a.k;
  const T* z = static_cast<const T*>(a.logits) + (long long)r * a.ld;
  float p[V], best = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    p[v] = e < E ? (float)z[e] : -INFINITY;
    best = max_nan(best, p[v]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
  const bool some = best != -INFINITY;
  float total = 0.f, ph = 0.f;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int e = lane + 32 * v;
    p[v] = p[v] == -INFINITY ? 0.f : expf(p[v] - best);
    total += p[v];
    h[v] = (a.g_importance != nullptr && e < E) ? a.g_importance[e] : 0.f;
  }
  total = warp_sum(total);
  const float inv = some ? 1.f / total : 0.f;
  // slot j on lane j
  float w = 0.f, g = 0.f;
  int who = -1;
  if (lane < k && a.g_weight != nullptr) {
    who = a.expert[(long long)r * k + lane];
    w = a.weight[(long long)r * k + lane];
    g = who >= 0 ? a.g_weight[(long long)r * k + lane] : 0.f;
    if (who < 0) w = 0.f;
  }
  const float wg = warp_sum(w * g);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    p[v] *= inv;
    ph = fmaf(p[v], h[v], ph);
  }
  ph = warp_sum(ph);
  const float through = ph + (a.renorm ? 0.f : wg);
  const float own = a.renorm ? w * (g - wg) : w * g;
  T* out = static_cast<T*>(a.dlogits) + (long long)r * E;
  float d[V];
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = p[v] * (h[v] - through);
  for (int j = 0; j < k; ++j) {
    const int e = __shfl_sync(0xFFFFFFFFu, who, j);
    const float t = __shfl_sync(0xFFFFFFFFu, own, j);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (lane + 32 * v == e) d[v] += t;
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (lane + 32 * v < E) out[lane + 32 * v] = (T)d[v];
}

// ---------------------------------------------------------------------------
// Moves of rows by a plan: xs[position[t, j]] = x[t], out[t] = sum_j w[t, j] y[position[t, j]] and the
// latter's gradients.  Places at or behind offsets[E] belong to pairs without a member: their rows are zero
// in what is written and not read.  Memory is the bound: each row is read and written once, in vectors of
// BYTES (the widest that all rows are aligned to).
// ---------------------------------------------------------------------------
struct RowsArgs {
  int T, k, W, E;
  const int32_t* position;  // (T, k)
  const int32_t* offsets;   // (E + 1)
  const float* weight;      // (T, k), or null: ones
  const void* x;            // dispatch: (T, W); combine: y (T k, W)
  long long x_ld;
  void* out;                // dispatch: (T k, W); combine: (T, W)
  const void* dout;         // backward of combine: (T, W)
  long long dout_ld;
  void* dy;                 // (T k, W), or null
  float* dw;                // (T, k), or null
  int vecs;                 // vectors of a row
  FastDiv div_vecs;
};

template <typename T, int BYTES>
struct RowVec {
  static constexpr int N = BYTES / (int)sizeof(T);
  T v[N];
};
template <typename T, int BYTES>
__device__ __forceinline__ RowVec<T, BYTES> row_load(const void* p, long long elem) {
  RowVec<T, BYTES> r;
  const char* s = static_cast<const char*>(p) + elem * (long long)sizeof(T);
  if constexpr (BYTES == 16)
    *reinterpret_cast<uint4*>(r.v) = __ldg(reinterpret_cast<const uint4*>(s));
  else if constexpr (BYTES == 8)
    *reinterpret_cast<uint2*>(r.v) = __ldg(reinterpret_cast<const uint2*>(s));
  else if constexpr (BYTES == 4)
    *reinterpret_cast<uint32_t*>(r.v) = __ldg(reinterpret_cast<const uint32_t*>(s));
  else
    *reinterpret_cast<uint16_t*>(r.v) = __ldg(reinterpret_cast<const uint16_t*>(s));
  return r;
}
template <typename T, int BYTES>
__device__ __forceinline__ void row_store(void* p, long long elem, const RowVec<T, BYTES>& r) {
  char* s = static_cast<char*>(p) + elem * (long long)sizeof(T);
  if constexpr (BYTES == 16)
    *reinterpret_cast<uint4*>(s) = *reinterpret_cast<const uint4*>(r.v);
  else if constexpr (BYTES == 8)
    *reinterpret_cast<uint2*>(s) = *reinterpret_cast<const uint2*>(r.v);
  else if constexpr (BYTES == 4)
    *reinterpret_cast<uint32_t*>(s) = *reinterpret_cast<const uint32_t*>(r.v);
  else
    *reinterpret_cast<uint16_t*>(s) = *reinterpret_cast<const uint16_t*>(r.v);
}

// (row, vector) of each thread: 256 consecutive vectors of the whole table per block.
__device__ __forceinline__ bool rows_place(const RowsArgs& a, int& t, int& c) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.T * a.vecs) return false;
  if (i < 0x7FFFFFFFLL) {
    t = (int)fastdiv((uint32_t)i, a.div_vecs);
    c = (int)((uint32_t)i - (uint32_t)t * (uint32_t)a.vecs);
  } else {
    t = (int)(i / a.vecs);
    c = (int)(i - (long long)t * a.vecs);
  }
  return true;
}

template <typename T, int BYTES>
__global__ void __launch_bounds__(256) rows_dispatch_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  int t, c;
  if (!rows_place(a, t, c)) return;
  const int used = max(0, min(__ldg(a.offsets + a.E), a.T * a.k));
  const V x = row_load<T, BYTES>(a.x, (long long)t * a.x_ld + c * V::N);
  V zero;
#pragma unroll
  for (int i = 0; i < V::N; ++i) zero.v[i] = (T)0.f;
  for (int j = 0; j < a.k; ++j) {
    const int p = __ldg(a.position + (long long)t * a.k + j);
    if ((unsigned)p < (unsigned)(a.T * a.k)) row_store<T, BYTES>(a.out, (long long)p * a.W + c * V::N, p < used ? x : zero);
  }
}

template <typename T, int BYTES>
__global__ void __launch_bounds__(256) rows_combine_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  int t, c;
  if (!rows_place(a, t, c)) return;
  const int used = max(0, min(__ldg(a.offsets + a.E), a.T * a.k));
  float s[V::N];
#pragma unroll
  for (int i = 0; i < V::N; ++i) s[i] = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int p = __ldg(a.position + (long long)t * a.k + j);
    if ((unsigned)p >= (unsigned)used) continue;
    const float w = a.weight ? __ldg(a.weight + (long long)t * a.k + j) : 1.f;
    const V y = row_load<T, BYTES>(a.x, (long long)p * a.x_ld + c * V::N);
#pragma unroll
    for (int i = 0; i < V::N; ++i) s[i] = fmaf(w, (float)y.v[i], s[i]);
  }
  V out;
#pragma unroll
  for (int i = 0; i < V::N; ++i) out.v[i] = (T)s[i];
  row_store<T, BYTES>(a.out, (long long)t * a.W + c * V::N, out);
}

// G threads a row: dy's rows and the dot products <dout[t], y[position[t, j]]>.
template <typename T, int BYTES, int G>
__global__ void __launch_bounds__(256) rows_combine_backward_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  constexpr int WARPS = G > 32 ? G / 32 : 1;
  __shared__ float red[256 / G][ROUTE_MAX_K][WARPS];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int t = blockIdx.x * (256 / G) + group;
  const bool live = t < a.T;
  const int used = max(0, min(__ldg(a.offsets + a.E), a.T * a.k));
  if (G > 32 || live) {
    for (int j = 0; j < a.k; ++j) {
      float dot = 0.f;
      int p = -1;
      if (live) {
        p = __ldg(a.position + (long long)t * a.k + j);
        const bool there = (unsigned)p < (unsigned)used, inside = (unsigned)p < (unsigned)(a.T * a.k);
        const float w = there ? (a.weight ? __ldg(a.weight + (long long)t * a.k + j) : 1.f) : 0.f;
        for (int c = lane; c < a.vecs; c += G) {
          const V d = row_load<T, BYTES>(a.dout, (long long)t * a.dout_ld + c * V::N);
          if (there && a.dw) {
            const V y = row_load<T, BYTES>(a.x, (long long)p * a.x_ld + c * V::N);
#pragma unroll
            for (int i = 0; i < V::N; ++i) dot = fmaf((float)d.v[i], (float)y.v[i], dot);
          }
          if (a.dy && inside) {
            V o;
#pragma unroll
            for (int i = 0; i < V::N; ++i) o.v[i] = there ? (T)(w * (float)d.v[i]) : (T)0.f;
            row_store<T, BYTES>(a.dy, (long long)p * a.W + c * V::N, o);
          }
        }
      }
      if (a.dw) {
        const unsigned mask = G >= 32 ? 0xFFFFFFFFu : (((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G));
#pragma unroll
        for (int o = (G > 32 ? 32 : G) / 2; o; o >>= 1) dot += __shfl_xor_sync(mask, dot, o);
        if (G <= 32) {
          if (lane == 0) a.dw[(long long)t * a.k + j] = dot;
        } else if ((lane & 31) == 0) {
          red[group][j][lane >> 5] = dot;
        }
      }
    }
  }
  if (G > 32 && a.dw) {
    __syncthreads();
    if (live && lane < a.k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) s += red[group][lane][w];
      a.dw[(long long)t * a.k + lane] = s;
    }
  }
}

}  // namespace tp
