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
  int32_t* counts;        // workspace (E + 1, blocks): pairs of a gate block with each member
  float* partial;         // workspace (E, blocks): sums of p over a block's rows
  int32_t* totals;        // workspace (E + 1)
  int rows_per_block;     // of a gate block
  int blocks, gates;      // gate blocks, and how many of them a place block takes
  const float* g_weight;      // backward, (rows, k) or null
  const float* g_importance;  // (E) or null
  void* dlogits;              // (rows, E)
};

// Sums and largest values over G neighbouring lanes, for every lane of them.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {  // (no NaN among them)
  if constexpr (G == 32) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  } else {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
  }
}
template <int G>
__device__ __forceinline__ int lanes_min(unsigned v) {
  if constexpr (G == 32) {
    return (int)__reduce_min_sync(0xFFFFFFFFu, v);
  } else {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = min(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return (int)v;
  }
}

// A row's scores, lane l of its G holding members l, l + G, ...; -inf past the last member.  The first F are there for sure.
template <typename T, int G, int F, int V>
__device__ __forceinline__ void route_load(const T* z, int E, int l, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = i < F || l + G * i < E ? (float)z[l + G * i] : -INFINITY;
}

constexpr float LOG2E = 1.4426950408889634f;
// exp(z - m), m the row's largest score: the difference first, so that it is 0 for the largest whatever its size, and at most
// -inf for the others (the type's lowest number beside ordinary ones: a term of 0).
__device__ __forceinline__ float exp_of(float z, float m) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"((z - m) * LOG2E));
  return r;
}

// Shared memory of the gate: hist[E + 1], sums[ROUTE_WARPS][E]; of the places: base[E + 1], counts[ROUTE_WARPS][E + 1].
__host__ __device__ inline size_t route_shared_bytes(int E) { return sizeof(int) * ((size_t)(ROUTE_WARPS + 1) * (E + 1)); }

// Weights and members of the block's rows, their counts per member, and the sums of p; G lanes a row.  Instructions bound
// it (some 500 a row for 257 members and 6 slots with a warp a row, 40 us for 65521 of them): each lane finds its two best at once, so that a slot costs two
// reductions and a search through the lane's scores only where one lane has three of a row's best.
template <typename T, int G, int F, int V>
__device__ __forceinline__ void route_gate(const RouteArgs& a, int block, int* smem) {
  constexpr int RPW = 32 / G;  // rows of a warp at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % G;
  const int E = a.E, k = a.k;
  int* hist = smem;
  float* sums = reinterpret_cast<float*>(hist + E + 1);
  for (int e = threadIdx.x; e <= E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int r0 = block * a.rows_per_block, r1 = min(a.rows, r0 + a.rows_per_block);
  const T* logits = static_cast<const T*>(a.logits);
  float imp[V], next[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    imp[v] = 0.f;
    next[v] = -INFINITY;
  }
  int r = r0 + warp * RPW + lane / G;
  if (r < r1) route_load<T, G, F, V>(logits + (long long)r * a.ld, E, l, next);
  for (int first = r0 + warp * RPW; first < r1; first += ROUTE_WARPS * RPW, r += ROUTE_WARPS * RPW) {
    const bool live = r < r1;  // (rows past the last one hold what the lanes had before; nothing of them is kept)
    float z[V];
#pragma unroll
    for (int v = 0; v < V; ++v) z[v] = next[v];
    if (r + ROUTE_WARPS * RPW < r1) route_load<T, G, F, V>(logits + (long long)(r + ROUTE_WARPS * RPW) * a.ld, E, l, next);
    // this lane's two best, b1 and b2, and which they are (equal ones: the lower first; a NaN is never greater)
    float b1, b2;
    int w1, w2;
    auto two_best = [&]() {
      b1 = b2 = -INFINITY;
      w1 = w2 = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool first = z[v] > b1, second = z[v] > b2;
        b2 = first ? b1 : second ? z[v] : b2;
        w2 = first ? w1 : second ? v : w2;
        b1 = first ? z[v] : b1;
        w1 = first ? v : w1;
      }
    };
    two_best();
    float top = lanes_max<G>(b1);
    const float m = top > -INFINITY ? top : 0.f;
    float e[V], total = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      e[v] = exp_of(z[v], m);  // 0 for -inf
      total += e[v];
    }
    total = lanes_sum<G>(total);
    if (__any_sync(0xFFFFFFFFu, total != total)) {
      // a NaN or +inf: all weights are NaN, and a NaN ranks as +inf
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (z[v] != z[v]) z[v] = INFINITY;
      two_best();
      top = lanes_max<G>(b1);
    }
    const float inv = !live || !(top > -INFINITY) ? 0.f : 1.f / total;
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v) imp[v] = fmaf(e[v], inv, imp[v]);
    }
    // the k best: lane j keeps slot j
    float mine = 0.f, best = b1;
    int my_expert = -1, which = l + G * w1;
    bool spare = true;  // b2 is the next one
    for (int j = 0; j < k; ++j) {
      const float b = j == 0 ? top : lanes_max<G>(best);
      if (G == 32 && b == -INFINITY) break;
      const int who = lanes_min<G>(best == b ? (unsigned)which : 0xFFFFFFFFu);
      if (b == -INFINITY) continue;  // (of a row that shares the warp with others)
      if (l == j) {
        mine = b;
        my_expert = who;
      }
      if (which == who && best == b) {
        if (spare) {
          best = b2;
          which = l + G * w2;
          spare = false;
        } else {
          // the best one behind (b, who)
          best = -INFINITY;
          int w = 0;
#pragma unroll
          for (int v = 0; v < V; ++v)
            if ((z[v] < b || (z[v] == b && l + G * v > who)) && z[v] > best) {
              best = z[v];
              w = v;
            }
          which = l + G * w;
        }
      }
    }
    __syncwarp();
    float w = my_expert >= 0 ? exp_of(mine, m) : 0.f;
    const float of = a.renorm ? lanes_sum<G>(w) : total;
    if (my_expert >= 0) w = total == total ? w / of : total;
    if (live && l < k) {
      a.weight[(long long)r * k + l] = w;
      a.expert[(long long)r * k + l] = my_expert;
      atomicAdd(&hist[my_expert < 0 ? E : my_expert], 1);  // whole numbers: any order gives the same count
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int o = G; o < 32; o <<= 1) imp[v] += __shfl_xor_sync(0xFFFFFFFFu, imp[v], o);
    if (lane < G && l + G * v < E) sums[warp * E + l + G * v] = imp[v];
  }
  __syncthreads();
  // (a single block's sums are the result; its counts stay in shared memory)
  for (int e = threadIdx.x; e <= E; e += blockDim.x) {
    if (a.blocks > 1) a.counts[(long long)e * a.blocks + block] = hist[e];
    if (e < E) {
      float s = 0.f;
      for (int w = 0; w < ROUTE_WARPS; ++w) s += sums[w * E + e];
      if (a.blocks > 1)
        a.partial[(long long)e * a.blocks + block] = s;
      else
        a.importance[e] = s;
    }
  }
}

// Per member, by one block: how many pairs earlier gate blocks have (in place of each one's count), how many there are,
// and the sum of p.
__global__ void __launch_bounds__(256) route_scan_kernel(const RouteArgs a) {
  __shared__ int counts[8];
  __shared__ float sums[8];
  const int e = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int32_t* c = a.counts + (long long)e * a.blocks;
  const int per = (a.blocks + 255) / 256, b0 = threadIdx.x * per, b1 = min(a.blocks, b0 + per);
  int n = 0;
  float s = 0.f;
  for (int b = b0; b < b1; ++b) {
    n += c[b];
    if (e < a.E) s += a.partial[(long long)e * a.blocks + b];
  }
  int inc = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += t;
  }
  s = lanes_sum<32>(s);
  if (lane == 31) {
    counts[warp] = inc;
    sums[warp] = s;
  }
  __syncthreads();
  int run = inc - n;
  for (int w = 0; w < warp; ++w) run += counts[w];
  for (int b = b0; b < b1; ++b) {
    const int t = c[b];
    c[b] = run;
    run += t;
  }
  if (threadIdx.x == 255) {
    a.totals[e] = run;
    float all = 0.f;
    for (int w = 0; w < 8; ++w) all += sums[w];
    if (e < a.E) a.importance[e] = all;
  }
}

// Places of the pairs of a.gates gate blocks from the first one, `gate`, on.  ONE: there is one block, whose counts the
// gate left where `base` will be.
template <bool ONE>
__device__ __forceinline__ void route_place(const RouteArgs& a, int gate, int* smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = a.E;
  int* base = smem;         // [E + 1]
  int* cnt = smem + E + 1;  // [warp][E + 1]
  __shared__ int carry[ROUTE_WARPS + 1];
  // where the members' rows begin: sums of the totals
  if (threadIdx.x == 0) carry[ROUTE_WARPS] = 0;
  for (int e0 = 0; e0 <= E; e0 += blockDim.x) {
    const int e = e0 + threadIdx.x;
    const int all = e <= E ? (ONE ? base[e] : a.totals[e]) : 0;
    int inc = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += t;
    }
    if (lane == 31) carry[warp] = inc;
    __syncthreads();
    int first = carry[ROUTE_WARPS] + inc - all;
    for (int w = 0; w < warp; ++w) first += carry[w];
    __syncthreads();
    if (threadIdx.x == blockDim.x - 1) carry[ROUTE_WARPS] = first + all;
    if (e <= E) {
      base[e] = first + (ONE ? 0 : a.counts[(long long)e * a.blocks + gate]);
      if (gate == 0) a.offsets[e] = first;
    }
  }
  // each warp's pairs are consecutive; its counts per member come before its places
  for (int i = threadIdx.x; i < ROUTE_WARPS * (E + 1); i += blockDim.x) cnt[i] = 0;
  __syncthreads();
  const int r0 = (int)min((long long)a.rows, (long long)gate * a.rows_per_block);
  const int r1 = (int)min((long long)a.rows, (long long)r0 + (long long)a.gates * a.rows_per_block);
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
}

template <typename T, int G, int F, int V>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, V <= 16 ? 2 : 1) route_gate_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_gate<T, G, F, V>(a, blockIdx.x, route_smem);
}

__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_place_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_place<false>(a, blockIdx.x * a.gates, route_smem);
}

// Few rows: all of it in one block.
template <typename T, int G, int F, int V>
__global__ void __launch_bounds__(32 * ROUTE_WARPS) route_small_kernel(const RouteArgs a) {
  extern __shared__ int route_smem[];
  route_gate<T, G, F, V>(a, 0, route_smem);
  __syncthreads();
  route_place<true>(a, 0, route_smem);
}

// dz of a row by G lanes: p is formed again from the scores (reading it would cost more than the sums).  Lane j then
// writes the chosen member of slot j over what the row's formula without the slots' gradients gave.
template <typename T, int G, int F, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs a) {
  const int l = threadIdx.x % G;
  const int E = a.E, k = a.k, stride = gridDim.x * (256 / G);
  const T* logits = static_cast<const T*>(a.logits);
  T* dlogits = static_cast<T*>(a.dlogits);
  float h[V], next[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    h[v] = (a.g_importance != nullptr && l + G * v < E) ? a.g_importance[l + G * v] : 0.f;
    next[v] = -INFINITY;
  }
  int r = blockIdx.x * (256 / G) + (int)threadIdx.x / G;
  if (r < a.rows) route_load<T, G, F, V>(logits + (long long)r * a.ld, E, l, next);
  for (int first = blockIdx.x * (256 / G) + (int)(threadIdx.x & ~31u) / G; first < a.rows; first += stride, r += stride) {
    const bool live = r < a.rows;
    float p[V], best = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = next[v];
      best = max_nan(best, p[v]);
    }
    if (r + stride < a.rows) route_load<T, G, F, V>(logits + (long long)(r + stride) * a.ld, E, l, next);
    // slot j on lane j
    float w = 0.f, g = 0.f, z_mine = 0.f, h_mine = 0.f;
    int who = -1;
    if (live && l < k && a.g_weight != nullptr) {
      who = a.expert[(long long)r * k + l];
      if ((unsigned)who < (unsigned)E) {
        w = a.weight[(long long)r * k + l];
        g = a.g_weight[(long long)r * k + l];
        z_mine = (float)logits[(long long)r * a.ld + who];
        if (a.g_importance != nullptr) h_mine = a.g_importance[who];
      } else {
        who = -1;
      }
    }
#pragma unroll
    for (int o = G / 2; o; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    const bool some = best != -INFINITY;
    const float m = some ? best : 0.f;
    float total = 0.f, ph = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = exp_of(p[v], m);
      total += p[v];
      ph = fmaf(p[v], h[v], ph);
    }
    float wg = w * g;
#pragma unroll
    for (int o = G / 2; o; o >>= 1) {
      total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
      ph += __shfl_xor_sync(0xFFFFFFFFu, ph, o);
      wg += __shfl_xor_sync(0xFFFFFFFFu, wg, o);
    }
    const float inv = some ? 1.f / total : 0.f;
    const float through = fmaf(ph, inv, a.renorm ? 0.f : wg);
    T* out = dlogits + (long long)r * E;
    if (live) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (v < F || l + G * v < E) out[l + G * v] = (T)(p[v] * inv * (h[v] - through));
    }
    __syncwarp();
    if (who >= 0) {
      const float p_mine = exp_of(z_mine, m) * inv;
      out[who] = (T)fmaf(w, a.renorm ? g - wg : g, p_mine * (h_mine - through));
    }
  }
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
  int span;                 // rows of a grid row
  int turns;                // vectors of a thread (combine)
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

// (row, vector) of this thread: number i of a.span rows, which have fewer than 2^31 vectors.
__device__ __forceinline__ bool rows_place(const RowsArgs& a, uint32_t i, int& t, int& c) {
  const uint32_t r = fastdiv(i, a.div_vecs);
  t = (int)(blockIdx.y * (uint32_t)a.span + r);
  c = (int)(i - r * (uint32_t)a.vecs);
  return r < (uint32_t)a.span && t < a.T;
}

template <typename T, int BYTES>
__global__ void __launch_bounds__(256) rows_dispatch_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  int t, c;
  if (!rows_place(a, blockIdx.x * 256 + threadIdx.x, t, c)) return;
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

// U rows of a vector on their way at a time (k of them where there are up to four); a.turns vectors a thread, 256 apart.
// (32768 rows of two of 4096 bf16 each: 152 us while a 64-bit index was taken apart on a branch, 134 without it, 119 with
// four vectors a thread one after the other, 6.8 TB/s; four at once take more registers and 131 us.)
template <typename T, int BYTES, int U>
__global__ void __launch_bounds__(256) rows_combine_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  const int used = max(0, min(__ldg(a.offsets + a.E), a.T * a.k));
#pragma unroll 1
  for (int h = 0; h < a.turns; ++h) {
    int t, c;
    if (!rows_place(a, (blockIdx.x * a.turns + h) * 256 + threadIdx.x, t, c)) return;
    float s[V::N];
#pragma unroll
    for (int i = 0; i < V::N; ++i) s[i] = 0.f;
    for (int j0 = 0; j0 < (U < 4 ? 1 : a.k); j0 += U) {
      int p[U];
      float w[U];
      V y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = U < 4 || j0 + u < a.k;
        p[u] = in ? __ldg(a.position + (long long)t * a.k + j0 + u) : -1;
        w[u] = in && a.weight ? __ldg(a.weight + (long long)t * a.k + j0 + u) : 1.f;
      }
      // (a row that takes no part is replaced by row 0, so that the loads need not wait for one another's conditions)
#pragma unroll
      for (int u = 0; u < U; ++u)
        y[u] = row_load<T, BYTES>(a.x, ((unsigned)p[u] < (unsigned)used ? (long long)p[u] : 0ll) * a.x_ld + c * V::N);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool there = (unsigned)p[u] < (unsigned)used;
#pragma unroll
        for (int i = 0; i < V::N; ++i) s[i] = there ? fmaf(w[u], (float)y[u].v[i], s[i]) : s[i];
      }
    }
    V out;
#pragma unroll
    for (int i = 0; i < V::N; ++i) out.v[i] = (T)s[i];
    row_store<T, BYTES>(a.out, (long long)t * a.W + c * V::N, out);
  }
}

// G threads a row: dy's rows and the dot products <dout[t], y[position[t, j]]>, of U slots at a time (all of them where there
// are up to three), so that dout is loaded once for them.  (32768 rows of two of 4096 bf16: 234 -> 227 us, 5.9 TB/s; 1003 rows of
// three of 771 fp32: 7.4 -> 6.6, and 9.5 with two slots at a time, one of them row 0 in vain.)
template <typename T, int BYTES, int G, int U>
__global__ void __launch_bounds__(256) rows_combine_backward_kernel(const RowsArgs a) {
  using V = RowVec<T, BYTES>;
  constexpr int WARPS = G > 32 ? G / 32 : 1;
  __shared__ float red[256 / G][ROUTE_MAX_K][WARPS];
  const int group = threadIdx.x / G, lane = threadIdx.x % G;
  const int t = blockIdx.x * (256 / G) + group;
  const bool live = t < a.T;
  const int used = max(0, min(__ldg(a.offsets + a.E), a.T * a.k));
  if (G > 32 || live) {  // (with G > 32 there is a row for every block)
    for (int j0 = 0; j0 < (U < 4 ? 1 : a.k); j0 += U) {
      float dot[U], w[U];
      int p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool in = U < 4 || j0 + u < a.k;
        dot[u] = 0.f;
        p[u] = in ? __ldg(a.position + (long long)t * a.k + j0 + u) : -1;
        w[u] = in && a.weight ? __ldg(a.weight + (long long)t * a.k + j0 + u) : 1.f;
      }
      for (int c = lane; c < a.vecs; c += G) {
        const V d = row_load<T, BYTES>(a.dout, (long long)t * a.dout_ld + c * V::N);
        V y[U];
        if (a.dw) {
#pragma unroll
          for (int u = 0; u < U; ++u)
            y[u] = row_load<T, BYTES>(a.x, ((unsigned)p[u] < (unsigned)used ? (long long)p[u] : 0ll) * a.x_ld + c * V::N);
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V::N; ++i) dot[u] = fmaf((float)d.v[i], (float)y[u].v[i], dot[u]);
        }
        if (a.dy) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if ((unsigned)p[u] >= (unsigned)(a.T * a.k)) continue;
            V o;
#pragma unroll
            for (int i = 0; i < V::N; ++i) o.v[i] = p[u] < used ? (T)(w[u] * (float)d.v[i]) : (T)0.f;
            row_store<T, BYTES>(a.dy, (long long)p[u] * a.W + c * V::N, o);
          }
        }
      }
      if (a.dw) {
        const unsigned mask = G >= 32 ? 0xFFFFFFFFu : (((1u << (G & 31)) - 1u) << ((threadIdx.x & 31) / G * G));
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (U == 4 && j0 + u >= a.k) break;
          if ((unsigned)p[u] >= (unsigned)used) dot[u] = 0.f;  // (row 0 was in its place)
#pragma unroll
          for (int o = (G > 32 ? 32 : G) / 2; o; o >>= 1) dot[u] += __shfl_xor_sync(mask, dot[u], o);
          if (G <= 32) {
            if (lane == 0) a.dw[(long long)t * a.k + j0 + u] = dot[u];
          } else if ((lane & 31) == 0) {
            red[group][j0 + u][lane >> 5] = dot[u];
          }
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
