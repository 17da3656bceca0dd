// Rows in 4-bit floating point with a scale per block of columns, and products of such rows.
//
// A value is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times its block's scale:
//   nvfp4: blocks of 16 columns, scale s 2^r.  2^r is the row's: the power of two with max|row| <= 2688 2^r <
//          2 max|row| (at least 2^-100), 2688 = 6 * 448; s = e4m3(max|block| / (6 2^r)), at most 448.
//   mxfp4: blocks of 32 columns, scale 2^(floor(log2 max|block|) - 2), at least 2^-100; larger values than 6 scales
//          become 6 scales.
// Codes are rounded to nearest, ties to the even code.  Every scale of the nvfp4 form has four significant bits, so
// x / scale is a tie only where it is one exactly, and a correctly rounded quotient decides as the exact one would.
// A row with a NaN or an infinity is NaN as a whole (its row scale).
//
// Layout.  Codes: two a byte, the even column's in the low half, rows of 16 ceil(K / 32) bytes, zeros at the end.
// Scales: as the tensor core takes them, tiles of 128 rows by 4 blocks, byte 16 (row % 32) + 4 (row / 32) + block % 4
// of the tile's 512; a row of tiles covers K rounded up to 256 columns.  Groups of rows begin in a tile of their own:
// group g of equal groups of B rows in tile g ceil(B / 128), ragged group g in tile floor(first row / 128) + g (which
// leaves every group the tiles that it needs, since floor(b / 128) - floor(a / 128) + 1 >= ceil((b - a) / 128)).
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace tp {

enum : int { FP4_NV = 0, FP4_MX = 1 };

struct Fp4Rows {
  uint8_t* codes;    // (rows, pitch)
  uint8_t* scales;   // (tiles, atoms, 512)
  float* row_scale;  // (rows): 2^r (nvfp4) or 1 (mxfp4); NaN for a row that is not finite
  int pitch, atoms;
};

// Groups of rows: P equal ones of B rows, or ragged ones by their offsets.
struct Fp4Groups {
  int P;
  long long rows;          // of the matrix
  int B;                   // equal groups
  const int32_t* offsets;  // (P + 1) device, or null
};

__device__ __forceinline__ long long fp4_first_row(const Fp4Groups& g, int m) {
  if (g.offsets == nullptr) return (long long)m * g.B;
  return min(max((long long)__ldg(g.offsets + m), 0ll), g.rows);
}
__device__ __forceinline__ long long fp4_end_row(const Fp4Groups& g, int m) {
  if (g.offsets == nullptr) return (long long)(m + 1) * g.B;
  const long long first = fp4_first_row(g, m);
  return max(first, min((long long)__ldg(g.offsets + m + 1), g.rows));
}
__device__ __forceinline__ long long fp4_first_tile(const Fp4Groups& g, int m) {
  if (g.offsets == nullptr) return (long long)m * ((g.B + 127) / 128);
  return fp4_first_row(g, m) / 128 + m;
}
// Group and first row of a tile; false where no row lies in it.
__device__ __forceinline__ bool fp4_tile(const Fp4Groups& g, long long tile, int& m, long long& row0, int& rows) {
  if (g.offsets == nullptr) {
    const int per = (g.B + 127) / 128;
    m = (int)(tile / per);
  } else {
    int lo = 0, hi = g.P - 1;  // the last group whose first tile is not behind this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (fp4_first_tile(g, mid) <= tile)
        lo = mid;
      else
        hi = mid - 1;
    }
    m = lo;
  }
  if (m >= g.P) return false;
  row0 = fp4_first_row(g, m) + (tile - fp4_first_tile(g, m)) * 128;
  const long long end = fp4_end_row(g, m);
  if (row0 >= end || tile < fp4_first_tile(g, m)) return false;
  rows = (int)min(128ll, end - row0);
  return true;
}

__device__ __forceinline__ float pow2f(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }

// 2^r of a row with largest magnitude `big`: its significand against that of 2688 = 1.3125 * 2^11.
__device__ __forceinline__ float nvfp4_row_scale(float big) {
  const uint32_t u = __float_as_uint(big);
  const int e = (int)(u >> 23) - 127;
  const int r = e - ((u & 0x7FFFFFu) > 0x280000u ? 10 : 11);
  return pow2f(max(r, -100));
}

struct Fp4QuantArgs {
  Fp4Groups groups;
  int K;
  const void* x;
  long long ld;
  const int32_t* n_features;  // (P) or null: columns of a group's rows that count
  Fp4Rows out;
};

// Eight values as four bytes of codes, the first in the lowest half byte.
__device__ __forceinline__ uint32_t fp4_pack8(const float (&q)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(r)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return r;
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {  // (of a byte without a sign)
  const uint32_t e = byte >> 3, f = byte & 7u;
  return e ? __uint_as_float(((e + 120u) << 23) | (f << 20)) : (float)f * 0.001953125f;
}

// e4m3(big / (6 row)): the quotient correctly rounded first (Markstein: one correction by the exact remainder).
__device__ __forceinline__ uint8_t nvfp4_scale_byte(float big, float row_inverse) {
  const float t = big * row_inverse, sixth = 0.16666667f;
  const float q = t * sixth;
  return (uint8_t)__nv_cvt_float_to_fp8(fmaf(fmaf(-q, 6.f, t), sixth, q), __NV_SATFINITE, __NV_E4M3);
}

// mxfp4: a block's scale byte from its largest magnitude, its scale s and that one's reciprocal.
__device__ __forceinline__ uint8_t mxfp4_scale(float big, float& s, float& inv) {
  const int e = max((int)(__float_as_uint(big) >> 23) - 129, -100);
  s = pow2f(e);
  inv = pow2f(-e);
  return (uint8_t)(e + 127);
}

// Two values over s: the correctly rounded quotients, by the reciprocal and one correction (exact for a power of two).
template <int FORMAT>
__device__ __forceinline__ void fp4_quotients(float& x, float& y, float s, float inv) {
  const f32x2 v = pair(x, y), i = pair(inv, inv);
  f32x2 t = mul2(v, i);
  if constexpr (FORMAT == FP4_NV) t = fma2(fma2(pair(-s, -s), t, v), i, t);
  const float2 h = halves(t);
  x = h.x;
  y = h.y;
}

// Rows go by vectors of 16 bytes, consecutive threads of a row's G consecutive ones; the 2 to 8 lanes
// of a block of columns find its scale together.  The scales' values and reciprocals come from a table by their byte.
struct Fp4Row {
  long long row;
  int n;              // columns that count
  bool live;
  uint8_t* scales;    // of this row in its tile
};
// Row r of a tile; false where the tile has none.
__device__ __forceinline__ bool fp4_row(const Fp4QuantArgs& a, long long tile, int r, Fp4Row& q) {
  int m, rows;
  long long row0;
  if (!fp4_tile(a.groups, tile, m, row0, rows)) return false;
  q.live = r < rows;
  q.row = row0 + r;
  q.n = q.live ? (a.n_features ? min(__ldg(a.n_features + m), a.K) : a.K) : 0;
  q.scales = a.out.scales + tile * a.out.atoms * 512 + (r & 31) * 16 + (r >> 5) * 4;
  return true;
}

// The largest magnitude of a vector, NaN if it holds one.
template <typename T>
__device__ __forceinline__ float fp4_largest(const uint4& q) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 2) {
    // magnitudes of bf16 are in the order of their bits, NaN above infinity
    uint32_t k = w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int j = 1; j < 4; ++j) k = __vmaxu2(k, w[j] & 0x7FFF7FFFu);
    return max_nan(__uint_as_float(k << 16), __uint_as_float(k & 0xFFFF0000u));
  } else {
    return max_nan(max_nan(fabsf(__uint_as_float(w[0])), fabsf(__uint_as_float(w[1]))),
                   max_nan(fabsf(__uint_as_float(w[2])), fabsf(__uint_as_float(w[3]))));
  }
}

// A vector's codes and, by the first lane of a block of columns, its scale byte.  `most`: the vector's largest magnitude;
// zero: a row that is not finite.
template <typename T, int FORMAT>
__device__ __forceinline__ void fp4_vector(const Fp4QuantArgs& a, const Fp4Row& row, const float2* table, int v, const uint4& u,
                                           float most, float scale, float scale_inverse, bool zero) {
  constexpr int N = FORMAT == FP4_NV ? 16 : 32, E = 16 / (int)sizeof(T), L = N / E;
  const int b = v / L;
#pragma unroll
  for (int o = 1; o < L; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
  float s, inv;
  uint8_t byte;
  if constexpr (FORMAT == FP4_NV) {
    byte = zero ? (uint8_t)0 : nvfp4_scale_byte(most, scale_inverse);
    const float2 e = table[byte];
    s = e.x * scale;
    inv = e.y * scale_inverse;
  } else {
    byte = mxfp4_scale(most, s, inv);
  }
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  float q[8] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 2) {
      q[2 * j] = __uint_as_float(w[j] << 16);
      q[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      q[j] = __uint_as_float(w[j]);
    }
  }
#pragma unroll
  for (int i = 0; i < E; i += 2) fp4_quotients<FORMAT>(q[i], q[i + 1], s, inv);
  const uint32_t c = zero ? 0u : fp4_pack8(q);
  if (b < a.out.atoms * 4) {  // (the padding's blocks too: zero)
    if (v % L == 0) row.scales[(b >> 2) * 512 + (b & 3)] = row.live && b * N < a.K ? byte : (uint8_t)0;
    if (row.live && v * (E / 2) < a.out.pitch) {
      uint8_t* codes = a.out.codes + row.row * a.out.pitch;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint32_t*>(codes + v * 4) = c;
      else
        *reinterpret_cast<uint16_t*>(codes + v * 2) = (uint16_t)c;
    }
  }
}

__device__ __forceinline__ void fp4_table(float2* table) {  // value and reciprocal of an e4m3 byte (0 of 0)
  for (int i = threadIdx.x; i < 128; i += blockDim.x) {
    const float v = e4m3_value(i);
    table[i] = make_float2(v, v > 0.f ? __frcp_rn(v) : 0.f);
  }
}

// Columns c on of a row, zeros from column n on.  Rows off 16-byte boundaries (ALIGNED false): the two 16-byte blocks of memory
// that the vector lies in, neither without an element of the row, moved into place (16384 rows of 8191 bf16: mxfp4 264 us element by
// element, 115 like this; nvfp4 194, 135).
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 fp4_load(const T* x, int c, int n) {
  constexpr int E = 16 / (int)sizeof(T);
  if constexpr (ALIGNED) {
    if (c + E <= n) return __ldg(reinterpret_cast<const uint4*>(x + c));
    T e[E];
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = c + i < n ? x[c + i] : (T)0.f;
    return *reinterpret_cast<const uint4*>(e);
  } else {
    if (c >= n) return make_uint4(0, 0, 0, 0);
    const uintptr_t p = reinterpret_cast<uintptr_t>(x + c);
    const uint32_t off = (uint32_t)p & 15u;
    const uint4* block = reinterpret_cast<const uint4*>(p - off);
    const uint4 lo = __ldg(block);
    uint4 hi = make_uint4(0, 0, 0, 0);
    if (off && reinterpret_cast<uintptr_t>(block + 1) < reinterpret_cast<uintptr_t>(x + n)) hi = __ldg(block + 1);
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (off & 8u) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4u) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2u) * 8u);
    }
    const int keep = n - c;
    if (keep < E) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2)
          w[i] = 2 * i + 1 < keep ? w[i] : 2 * i < keep ? w[i] & 0xFFFFu : 0u;
        else
          w[i] = i < keep ? w[i] : 0u;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Rows onto 16-byte boundaries, a vector a thread; `vecs` of a row of the result.
__global__ void __launch_bounds__(256) align_rows_kernel(const __nv_bfloat16* x, long long ld, int rows, int cols, uint4* out, int vecs,
                                                        const FastDiv div, int span) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, r = fastdiv(i, div);
  const long long row = (long long)blockIdx.y * span + r;
  if (r >= (uint32_t)span || row >= rows) return;
  const int v = (int)(i - r * (uint32_t)vecs);
  out[row * vecs + v] = fp4_load<__nv_bfloat16, false>(x + row * ld, 8 * v, cols);
}

// The largest magnitude of a row among the vectors of this thread (of G), NaN if one is.
template <typename T, int G, bool ALIGNED>
__device__ __forceinline__ float fp4_row_max(const T* x, int n, int at) {
  constexpr int E = 16 / (int)sizeof(T), U = 4;
  float big = 0.f;
  for (int v = at; v * E < n; v += U * G) {
    uint4 u[U];
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = fp4_load<T, ALIGNED>(x, (v + j * G) * E, n);
#pragma unroll
    for (int j = 0; j < U; ++j) big = max_nan(big, fp4_largest<T>(u[j]));
  }
  return big;
}

// G threads a row, H vectors at a time; a block of the grid takes four rows (i, i + 32, i + 64, i + 96 of a tile), or one with
// G = 256.  nvfp4 reads a row twice (for its largest magnitude first), mxfp4 once
// (16384 rows of 8192 fp32: 113 us, 5.4 TB/s; 140 with a thread's own block by strided vectors, 171 by way of shared memory).
template <typename T, int FORMAT, int G, int H, bool ALIGNED>
__global__ void __launch_bounds__(G == 256 ? 256 : 4 * G) fp4_quantize_rows_kernel(const Fp4QuantArgs a) {
  constexpr int N = FORMAT == FP4_NV ? 16 : 32, E = 16 / (int)sizeof(T), L = N / E;
  constexpr int ROWS = G == 256 ? 1 : 4, PER = 128 / ROWS;
  __shared__ float2 table[128];
  __shared__ float warp_max[ROWS * G / 32];
  const int tile = blockIdx.x / PER, part = blockIdx.x % PER;
  const int at = threadIdx.x % G, lane = threadIdx.x & 31;
  Fp4Row q;
  if (!fp4_row(a, tile, ROWS == 1 ? part : part + 32 * (int)(threadIdx.x / G), q)) return;
  if (FORMAT == FP4_NV) fp4_table(table);
  const T* x = static_cast<const T*>(a.x) + q.row * a.ld;
  float big = 0.f;
  auto row_max = [&]() {
#pragma unroll
    for (int o = 16; o; o >>= 1) big = max_nan(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
    if constexpr (G > 32) {
      if (lane == 0) warp_max[threadIdx.x >> 5] = big;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < G / 32; ++w) big = max_nan(big, warp_max[threadIdx.x / G * (G / 32) + w]);
    }
  };
  float scale = 1.f;
  if constexpr (FORMAT == FP4_NV) {
    if (q.live) big = fp4_row_max<T, G, ALIGNED>(x, q.n, at);
    row_max();
    if constexpr (G == 32) __syncthreads();  // (the table)
    scale = nvfp4_row_scale(big);
  }
  const bool zero = FORMAT == FP4_NV && !(big < INFINITY);
  const float scale_inverse = __uint_as_float((254u << 23) - __float_as_uint(scale));  // (of a power of two)
  const int vecs = a.out.atoms * 4 * L;
  for (int v0 = 0; v0 < vecs; v0 += G * H) {
    uint4 u[H];
#pragma unroll
    for (int h = 0; h < H; ++h) u[h] = fp4_load<T, ALIGNED>(x, (v0 + h * G + at) * E, q.n);
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (v0 + h * G >= vecs) break;  // (the same for all of the block's threads)
      const float most = fp4_largest<T>(u[h]);
      if constexpr (FORMAT == FP4_MX) big = max_nan(big, most);
      fp4_vector<T, FORMAT>(a, q, table, v0 + h * G + at, u[h], most, scale, scale_inverse, zero);
    }
  }
  if constexpr (FORMAT == FP4_MX) row_max();
  if (q.live && at == 0) a.out.row_scale[q.row] = big < INFINITY ? scale : __uint_as_float(0x7FC00000u);
}

// nvfp4 of rows that G threads hold at once (G H vectors), read once: a block goes through groups of four rows, the next one's
// vectors on their way to shared memory meanwhile, since a row's scale needs its largest magnitude before the first code.  A
// warp's vectors come in as they lie in memory and are dealt out again so that a lane has whole blocks of columns.
// (16384 rows of 8192 bf16: 98 us in two passes, of which the second misses L2 by half; 88 us with a vector a lane, the block's
// scale found by two of them with shuffles, 150 instructions a vector; 80 us like this, 4.3 TB/s.  The instructions still bound it.)
template <typename T, int G, int H, bool ALIGNED>
__global__ void __launch_bounds__(4 * G, 256 / G) fp4_quantize_stream_kernel(const Fp4QuantArgs a, const long long groups) {
  constexpr int N = 16, E = 16 / (int)sizeof(T), L = N / E;  // columns of a block, of a vector; vectors of a block
  static_assert(H % L == 0, "whole blocks");
  extern __shared__ uint4 slots[];  // [2][H][threads]
  __shared__ float2 table[128];
  __shared__ float warp_max[2][G / 8];
  const int at = threadIdx.x % G, lane = threadIdx.x & 31, sub = threadIdx.x / G;
  const int blocks = a.out.atoms * 4;  // with those of the padding, which are zero
  fp4_table(table);
  __syncthreads();
  auto slot = [&](int stage, int h) -> uint4* { return slots + (stage * H + h) * (4 * G) + threadIdx.x; };
  auto fetch = [&](long long group, int stage, Fp4Row& q) -> bool {
    bool ok = false;
    if (group < groups) {
      ok = fp4_row(a, group / 32, (int)(group % 32) + 32 * sub, q);
      if (ok) {
        const T* x = static_cast<const T*>(a.x) + q.row * a.ld;
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const int c = (h * G + at) * E;
          if (ALIGNED && c + E <= q.n)
            cp_async16(smem_u32(slot(stage, h)), x + c);
          else
            *slot(stage, h) = fp4_load<T, ALIGNED>(x, c, q.n);
        }
      }
    }
    cp_async_commit();
    return ok;
  };
  Fp4Row now, then;
  now.row = then.row = 0;
  now.live = then.live = false;
  int stage = 0;
  bool here = fetch(blockIdx.x, 0, now);
  for (long long group = blockIdx.x; group < groups; group += gridDim.x, stage ^= 1) {
    const bool there = fetch(group + gridDim.x, stage ^ 1, then);
    cp_async_wait<1>();
    __syncwarp();
    if (here) {  // (of all threads of the block or none)
      // of the L vectors h = p L.. of all lanes: this lane's block is number lane % (32 / L) of vector p L + lane / (32 / L)
      uint4 u[H];
      float most[H / L], big = 0.f;
#pragma unroll
      for (int p = 0; p < H / L; ++p) {
        const uint4* from = slot(stage, p * L + lane / (32 / L)) - lane + L * (lane % (32 / L));
        most[p] = 0.f;
#pragma unroll
        for (int i = 0; i < L; ++i) {
          u[p * L + i] = from[i];
          most[p] = max_nan(most[p], fp4_largest<T>(u[p * L + i]));
        }
        big = max_nan(big, most[p]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) big = max_nan(big, __shfl_xor_sync(0xFFFFFFFFu, big, o));
      if constexpr (G > 32) {
        if (lane == 0) warp_max[stage][threadIdx.x >> 5] = big;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + sub), "n"(G) : "memory");  // the row's threads
#pragma unroll
        for (int w = 0; w < G / 32; ++w) big = max_nan(big, warp_max[stage][sub * (G / 32) + w]);
      }
      const float scale = nvfp4_row_scale(big);
      const float scale_inverse = __uint_as_float((254u << 23) - __float_as_uint(scale));  // (of a power of two)
      const bool zero = !(big < INFINITY);
      if (now.live && at == 0) a.out.row_scale[now.row] = zero ? __uint_as_float(0x7FC00000u) : scale;
#pragma unroll
      for (int p = 0; p < H / L; ++p) {
        const int v = (p * L + lane / (32 / L)) * G + (at - lane) + L * (lane % (32 / L)), b = v / L;
        if (b >= blocks) continue;
        const uint8_t byte = zero ? (uint8_t)0 : nvfp4_scale_byte(most[p], scale_inverse);
        const float2 e = table[byte];
        const float s = e.x * scale, inv = e.y * scale_inverse;
        now.scales[(b >> 2) * 512 + (b & 3)] = now.live && b * N < a.K ? byte : (uint8_t)0;
        if (now.live && b * (N / 2) < a.out.pitch) {
          uint32_t c[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float q[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (sizeof(T) == 2) {
                const uint4& w4 = u[p * L + j];
                const uint32_t w = i == 0 ? w4.x : i == 1 ? w4.y : i == 2 ? w4.z : w4.w;
                q[2 * i] = __uint_as_float(w << 16);
                q[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
              } else {
                const uint4& w4 = u[p * L + 2 * j + i / 2];
                q[2 * i] = __uint_as_float(i & 1 ? w4.z : w4.x);
                q[2 * i + 1] = __uint_as_float(i & 1 ? w4.w : w4.y);
              }
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2) fp4_quotients<FP4_NV>(q[i], q[i + 1], s, inv);
            c[j] = zero ? 0u : fp4_pack8(q);
          }
          *reinterpret_cast<uint2*>(a.out.codes + now.row * a.out.pitch + b * (N / 2)) = make_uint2(c[0], c[1]);
        }
      }
    } else if constexpr (G > 32) {
      // (a turn without rows too: the maxima of the turn before have been read before the turn after it writes over them)
      asm volatile("bar.sync %0, %1;" ::"r"(1 + sub), "n"(G) : "memory");
    }
    __syncwarp();  // (the slots are filled again by the next turn's copies)
    now = then;
    here = there;
  }
}

struct Fp4ValuesArgs {
  Fp4Groups groups;
  int K;
  Fp4Rows in;
  __nv_bfloat16* out;  // (rows, K)
};

// Four codes' values times s, which bf16 holds exactly, as two words of two.
__device__ __forceinline__ uint2 fp4_decode4(uint32_t codes, float s) {
  uint32_t lo, hi;
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %2;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
  const float2 x = __half22float2(*reinterpret_cast<__half2*>(&lo)), y = __half22float2(*reinterpret_cast<__half2*>(&hi));
  return make_uint2(pack_bf16x2(x.x * s, x.y * s), pack_bf16x2(y.x * s, y.y * s));
}

// A thread takes eight columns (four bytes of codes), consecutive threads consecutive ones.  Rows off 16-byte boundaries are
// written by way of shared memory, in pairs of a warp's 256 consecutive columns (16384 x 8191: 389 -> 92 us).
template <int FORMAT, int G, bool VEC>
__global__ void __launch_bounds__(256) fp4_values_kernel(const Fp4ValuesArgs a) {
  constexpr int N = FORMAT == FP4_NV ? 16 : 32;
  constexpr int PER = 128 * G / 256;
  __shared__ uint4 staged[VEC ? 1 : 8][32];
  const int tile = blockIdx.x / PER, part = blockIdx.x % PER;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int at = G == 32 ? lane : (int)threadIdx.x;
  const int r = G == 32 ? 2 * part + (warp & 1) + 32 * (warp >> 1) : part;
  int m, rows;
  long long row0;
  if (!fp4_tile(a.groups, tile, m, row0, rows) || r >= rows) return;  // (of a warp all threads)
  const long long row = row0 + r;
  const float rs = __ldg(a.in.row_scale + row);
  const uint8_t* from = a.in.scales + (long long)tile * a.in.atoms * 512 + (r & 31) * 16 + (r >> 5) * 4;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.in.codes + row * a.in.pitch);
  __nv_bfloat16* out = a.out + row * a.K;
  auto decode = [&](int i) -> uint4 {
    const int b = 8 * i / N;
    const uint32_t byte = __ldg(from + (b >> 2) * 512 + (b & 3)), c = __ldg(codes + i);
    float s;
    if (FORMAT == FP4_NV) {
      const uint32_t e = byte >> 3, f = byte & 7u;
      s = (e ? __uint_as_float(((e + 120u) << 23) | (f << 20)) : (float)f * 0.001953125f) * rs;
    } else {
      s = pow2f((int)byte - 127) * rs;
    }
    const uint2 lo = fp4_decode4(c, s), hi = fp4_decode4(c >> 16, s);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  if constexpr (VEC) {  // (K is a multiple of 8)
#pragma unroll 4
    for (int i = at; 8 * i < a.K; i += G) *reinterpret_cast<uint4*>(out + 8 * i) = decode(i);
  } else {
#pragma unroll 2
    for (int i0 = at - lane; 8 * i0 < a.K; i0 += G) {
      staged[warp][lane] = 8 * (i0 + lane) < a.K ? decode(i0 + lane) : make_uint4(0, 0, 0, 0);
      __syncwarp();
      const uint16_t* s = reinterpret_cast<const uint16_t*>(staged[warp]);
      uint16_t* to = reinterpret_cast<uint16_t*>(out + 8 * i0);
      const int count = min(256, a.K - 8 * i0), odd = (int)(reinterpret_cast<uintptr_t>(to) >> 1) & 1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = odd + 2 * (lane + 32 * k);
        if (j + 1 < count)
          *reinterpret_cast<uint32_t*>(to + j) = (uint32_t)s[j] | (uint32_t)s[j + 1] << 16;
        else if (j < count)
          to[j] = s[j];
      }
      if (odd && lane == 0) to[0] = s[0];
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------------------
// y = relu(q(x) q(w_m)^T + b_m): both operands in 4 bits, block scales applied by the tensor core, sums in fp32, row
// scales in the epilogue.  A = rows of x (128 a tile), B = rows of w; both K-major, 256 columns (128 bytes) a stage.
// The scales of a stage are copied from shared to tensor memory by tcgen05.cp, which the tensor core runs in order
// with the products of the same thread.
// ---------------------------------------------------------------------------
struct Fp4Problem {
  Fp4Groups groups;  // rows of x; groups.P members
  int x_shared;      // equal groups that all read the same rows of x
  int K, N;
  const int32_t* in_f;   // (P) or null
  const int32_t* out_f;  // (P) or null
  const float* x_row;
  const float* w_row;  // (P, N)
  const float* bias;   // (P, N) or null
  int relu;
  void* y;  // (rows of y, N)
  int y_f32, y_vec;
  int n_tiles;
};

// sum * x's row scale * w's row scale + bias, the scales being powers of two of at most 2^117.  A sum (below 2^47: 2^24 products of
// at most 2688^2) times 2^80 is within fp32; what a larger scale has beyond goes to the other one, so that nothing in between
// overflows where the result does not.  (Cut at 2^127: then the result is infinite all the same, and a sum of 0 is no NaN.)
constexpr float FP4_SCALE_STEP = 1208925819614629174706176.f;
__device__ __forceinline__ float fp4_result(float sum, float x_scale, float w_scale, float bias) {
  const bool large = x_scale > FP4_SCALE_STEP;
  const float first = large ? FP4_SCALE_STEP : x_scale, rest = large ? x_scale * (1.f / FP4_SCALE_STEP) : 1.f;
  const float second = rest * w_scale, most = 1.70141183e38f;
  return fmaf(sum * first, second > most ? most : second, bias);  // (a NaN stays one)
}

enum : int { FT_MMA = 0, FT_ZERO = 1, FT_END = 2 };
struct Fp4Tile {
  int kind, member, x_row, y_row, rows, nt, x_tile, n_valid;
};

template <int BN_, int FORMAT, bool PAIR_ = false>
struct Fp4Cfg {
  static constexpr bool PAIR = PAIR_;
  static_assert(!PAIR || BN_ == 256, "pairs take tiles of 256 columns");
  static constexpr int BM = 128, BN = BN_, BK = 256;
  static constexpr int TILE_M = PAIR ? 256 : 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // rows of w that a CTA stages (of their scales, all of the tile's)
  static constexpr int ATOMS = FORMAT == FP4_NV ? 4 : 2;  // scale tiles of 128 rows a stage
  static constexpr int A_BYTES = BM * 128, B_BYTES = B_ROWS * 128;
  static constexpr int SB_TILES = BN > 128 ? BN / 128 : 1;
  static constexpr int SA_BYTES = ATOMS * 512, SB_BYTES = SB_TILES * ATOMS * 512;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SA_BYTES + SB_BYTES;
  // (pairs, 9472 x 8192 x 8192: five stages 260 us in mxfp4 and 300 in nvfp4, four 273 and 303)
  static constexpr int STAGES = PAIR ? 5 : BN == 256 ? 3 : BN == 128 ? 5 : 6;
  static constexpr int ACCS = BN == 256 ? 1 : 2;
  // tensor memory columns: accumulators, then buffers of a stage's scales (of x, of w)
  static constexpr int SA_COLS = 4 * ATOMS, SB_COLS = 4 * ATOMS * SB_TILES, S_COL = ACCS * BN, S_COLS = SA_COLS + SB_COLS;
  static constexpr int TMEM_COLS = BN == 64 ? 256 : 512;
  static constexpr int SBUFS = 4;
  static_assert(S_COL + SBUFS * S_COLS <= TMEM_COLS, "tensor memory");
  static constexpr int EPI_WARP0 = 4, EPI_WARPS = 8, SCALE_WARP0 = EPI_WARP0 + EPI_WARPS, SCALE_WARPS = 2;
  static constexpr int THREADS = 32 * (SCALE_WARP0 + SCALE_WARPS);
  static constexpr int TRING = 4;
  static constexpr int CTRL_BYTES = 512;  // barriers (384 bytes), tiles
  static constexpr int ROW_BYTES = 144;  // a warp's staged row of 128 bytes, padded; 16 rows at a time
  static constexpr int WCOLS = BN / 2;   // columns of an epilogue warp
  static constexpr int EPI_BYTES = 16 * ROW_BYTES + WCOLS * 8;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + CTRL_BYTES + EPI_WARPS * EPI_BYTES;
  static_assert(SMEM_BYTES <= 227 * 1024, "fits an SM");
};

// Descriptor of 128 rows' scales in shared memory: 32 x 16 bytes, 8-row groups 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// They go into four columns of tensor memory, the same in each quarter of the lanes.
// PAIR: in both CTAs, each from its own shared memory.
template <bool PAIR = false>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (PAIR)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

#define TP_UMMA_FP4(group, kind)                                                                                      \
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n tcgen05.mma.cta_group::" group ".kind::" kind                \
               " [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d_tmem),                                                 \
               "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                \
               : "memory")
// A pair's products: 128 rows of A and half of B's from each CTA, A's scales of its own rows and B's of all columns in
// each CTA's tensor memory.
template <int FORMAT, bool PAIR = false>
__device__ __forceinline__ void umma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sa,
                                         uint32_t sb, uint32_t accumulate) {
  if constexpr (PAIR && FORMAT == FP4_NV)
    TP_UMMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
  else if constexpr (PAIR)
    TP_UMMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
  else if constexpr (FORMAT == FP4_NV)
    TP_UMMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  else
    TP_UMMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
}
#undef TP_UMMA_FP4

// Instruction descriptor: A and B e2m1; scales e4m3 (nvfp4) or powers of two (mxfp4), `id` the half of a scale word
// that this product takes (mxfp4: 0 or 2).
template <int FORMAT>
__device__ __forceinline__ uint32_t idesc_fp4(int n, uint32_t id, int m = 128) {
  return (id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((FORMAT == FP4_MX ? 1u : 0u) << 23) |
         ((uint32_t)(m >> 7) << 27) | (id << 29);
}

template <int BN, int FORMAT, bool PAIR>
__global__ void __launch_bounds__(Fp4Cfg<BN, FORMAT, PAIR>::THREADS, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB, const Fp4Problem pr) {
  using Cfg = Fp4Cfg<BN, FORMAT, PAIR>;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smA + Cfg::STAGES * Cfg::A_BYTES;
  uint8_t* smSA = smB + Cfg::STAGES * Cfg::B_BYTES;
  uint8_t* smSB = smSA + Cfg::STAGES * Cfg::SA_BYTES;
  uint8_t* ctrl = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* tfull = empty + Cfg::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done_bar = tempty + 2;
  constexpr int TRING = Cfg::TRING;
  uint64_t* tr_full = done_bar + 1;
  uint64_t* tr_empty = tr_full + TRING;
  uint64_t* s_ready = tr_empty + TRING;          // a buffer of scales is in tensor memory
  uint64_t* s_free = s_ready + Cfg::SBUFS;       // the products that read it have completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + Cfg::SBUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ring = reinterpret_cast<volatile int*>(ctrl + 384);
  static_assert(8 * (2 * Cfg::STAGES + 5 + 2 * TRING + 2 * Cfg::SBUFS) + 8 <= 384 && 384 + 32 * TRING <= Cfg::CTRL_BYTES,
                "control block");
  const int warp = warp_id(), lane = lane_id();
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const int worker = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x, workers = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int n_sb_tiles = (pr.N + 127) / 128;  // scale tiles of a member's rows of w

  // (`whole`: all lanes of the warp read, and lane 0 frees the slot once they have)
  auto ring_read = [&](int k, bool whole) -> Fp4Tile {
    Fp4Tile t;
    const int s = k & (TRING - 1);
    if (!mbar_wait(&tr_full[s], (uint32_t)(k / TRING) & 1u, abort_flag)) {
      t.kind = FT_END;
      return t;
    }
    const volatile int* e = ring + 8 * s;
    t.kind = e[0];
    t.member = e[1];
    t.x_row = e[2];
    t.y_row = e[3];
    t.rows = e[4];
    t.nt = e[5];
    t.x_tile = e[6];
    t.n_valid = e[7];
    if (whole) __syncwarp();
    if (!whole || lane == 0) mbar_arrive(&tr_empty[s]);
    return t;
  };
  // columns that a tile multiplies (16 a CTA at least)
  auto columns = [&](const Fp4Tile& t) {
    const int left = t.n_valid - t.nt * BN;
    return min(BN, PAIR ? (left + 31) & ~31 : (left + 15) & ~15);
  };
  auto k_blocks = [&](int member) {
    const int k = pr.in_f ? min(__ldg(pr.in_f + member), pr.K) : pr.K;
    return (k + Cfg::BK - 1) / Cfg::BK;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < Cfg::SBUFS; ++i) {
      mbar_init(&s_ready[i], Cfg::SCALE_WARPS);
      mbar_init(&s_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], PAIR ? 2 * Cfg::EPI_WARPS : Cfg::EPI_WARPS);  // the leader's counts both CTAs
    }
    mbar_init(done_bar, 1);
    for (int i = 0; i < TRING; ++i) {
      mbar_init(&tr_full[i], 1);
      mbar_init(&tr_empty[i], (rank == 0 ? 3 + Cfg::SCALE_WARPS : 2) + Cfg::EPI_WARPS);  // producers, MMA, scales, epilogue
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSA);
    prefetch_tmap(&tmSB);
  }
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_alloc_pair(tmem_slot, Cfg::TMEM_COLS);
    else
      tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the peer's barriers are initialised before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------------ producers: x by warp 0, w by warp 3, each with
    // its scales (a copy takes one thread about 190 cycles, a stage's products 512)
    if (lane == 0) {
      const bool is_a = warp == 0;
      const CUtensorMap* map = is_a ? &tmA : &tmB;
      const CUtensorMap* scale_map = is_a ? &tmSA : &tmSB;
      uint8_t* const to = is_a ? smA : smB;
      uint8_t* const scale_to = is_a ? smSA : smSB;
      const uint32_t leader0 = PAIR ? mapa_shared(smem_u32(full), 0) : 0;
      const int bytes = is_a ? Cfg::A_BYTES : Cfg::B_BYTES, scale_bytes = is_a ? Cfg::SA_BYTES : Cfg::SB_BYTES;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const Fp4Tile t = ring_read(k, false);
        if (t.kind == FT_END) break;
        if (t.kind != FT_MMA) continue;
        const int kblocks = k_blocks(t.member);
        const int row = is_a ? t.x_row + rank * Cfg::BM : t.nt * BN + (PAIR ? rank * (columns(t) / 2) : 0);
        const int plane = is_a ? 0 : t.member;
        const int tile = is_a ? t.x_tile + rank : t.member * n_sb_tiles + t.nt * BN / 128;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          // (the bytes of both are announced by the first; the others' may arrive before)
          if constexpr (PAIR) {  // both CTAs' bytes complete on the leader's barrier
            if (is_a && rank == 0) mbar_arrive_expect_tx(&full[stage], 2 * Cfg::STAGE_BYTES);
            tma_load_3d_pair(to + stage * bytes, map, leader0 + 8u * stage, kb * 128, row, plane);
            tma_load_3d_pair(scale_to + stage * scale_bytes, scale_map, leader0 + 8u * stage, 0, kb * 2 * Cfg::ATOMS, tile);
          } else {
            if (is_a) mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
            tma_load_3d(to + stage * bytes, map, &full[stage], kb * 128, row, plane);
            tma_load_3d(scale_to + stage * scale_bytes, scale_map, &full[stage], 0, kb * 2 * Cfg::ATOMS, tile);
          }
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA (a pair's leader fills both CTAs' TMEM)
    if (lane == 0 && rank == 0) {
      int stage = 0, acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      // descriptors of the first stage; the address field counts 16 bytes
      const uint64_t adesc0 = smem_desc_sw128(smem_u32(smA), 16, 1024), bdesc0 = smem_desc_sw128(smem_u32(smB), 16, 1024);
      uint32_t buf = 0, buf_phase = 0;
      for (int k = 0; ok; ++k) {
        const Fp4Tile t = ring_read(k, false);
        if (t.kind == FT_END) break;
        if (t.kind != FT_MMA) continue;
        const int n_mma = columns(t);
        const uint32_t idesc[2] = {idesc_fp4<FORMAT>(n_mma, 0, Cfg::TILE_M),
                                   idesc_fp4<FORMAT>(n_mma, FORMAT == FP4_NV ? 0 : 2, Cfg::TILE_M)};
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
        // tiles of 64 columns take one half of a scale tile of 128
        const uint32_t sb_shift = BN == 64 ? (uint32_t)(t.nt & 1) * 2u : 0u;
        const int kblocks = k_blocks(t.member);
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag)) break;
        tc_fence_after();
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&s_ready[buf], buf_phase, abort_flag)) {  // (the stage has landed before)
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t ad = adesc0 + (uint64_t)(stage * (Cfg::A_BYTES / 16)), bd = bdesc0 + (uint64_t)(stage * (Cfg::B_BYTES / 16));
          const uint32_t sa_at = tmem_base + Cfg::S_COL + buf * Cfg::S_COLS, sb_at = sa_at + Cfg::SA_COLS + sb_shift;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int i = FORMAT == FP4_NV ? s : s >> 1;
            umma_fp4<FORMAT, PAIR>(d_tmem, ad + 2 * s, bd + 2 * s, idesc[s & 1], sa_at + 4 * i, sb_at + 4 * i * Cfg::SB_TILES,
                                   (kb | s) != 0 ? 1u : 0u);
          }
          if constexpr (PAIR)
            umma_commit_pair(smem_u32(&s_free[buf]));
          else
            umma_commit(&s_free[buf]);
          buf = (buf + 1) % Cfg::SBUFS;
          if (buf == 0) buf_phase ^= 1u;
          if constexpr (PAIR)
            umma_commit_both(&empty[stage]);
          else
            umma_commit(&empty[stage]);
          if (++stage == Cfg::STAGES) stage = 0;
        }
        if (!ok) break;
        if constexpr (PAIR)
          umma_commit_both(&tfull[acc]);
        else
          umma_commit(&tfull[acc]);
        if (++acc == Cfg::ACCS) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if constexpr (PAIR)
        umma_commit_pair(smem_u32(done_bar));
      else
        umma_commit(done_bar);
      volatile int no_abort = 0;
      mbar_wait(done_bar, 0, &no_abort);
    }
  } else if (warp >= Cfg::SCALE_WARP0) {
    // ------------------------------------------------------------------ scales to tensor memory, half of a stage a warp
    // (a thread takes some 36 cycles to issue each of these instructions: with the copies on the thread of the products
    // a stage took 1400 cycles instead of the products' 512, the copies one stage ahead 1300, on one thread of their own 1090)
    if (lane == 0 && rank == 0) {
      const uint64_t sadesc0 = scale_desc(smem_u32(smSA)), sbdesc0 = scale_desc(smem_u32(smSB));
      int stage = 0;
      uint32_t phase = 0, buf = 0, buf_phase = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const Fp4Tile t = ring_read(k, false);
        if (t.kind == FT_END) break;
        if (t.kind != FT_MMA) continue;
        const int kblocks = k_blocks(t.member);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag) || !mbar_wait(&s_free[buf], buf_phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t sad = sadesc0 + (uint64_t)(stage * (Cfg::SA_BYTES / 16)), sbd = sbdesc0 + (uint64_t)(stage * (Cfg::SB_BYTES / 16));
          const uint32_t sa_tmem = tmem_base + Cfg::S_COL + buf * Cfg::S_COLS, sb_tmem = sa_tmem + Cfg::SA_COLS;
          // a product's columns of w take consecutive columns of scales: tile c of step i at (i * tiles + c) * 4
#pragma unroll
          for (int h = 0; h < Cfg::ATOMS / 2; ++h) {
            const int i = h + (warp - Cfg::SCALE_WARP0) * (Cfg::ATOMS / 2);
            tmem_copy_scales<PAIR>(sa_tmem + 4 * i, sad + 32 * i);
#pragma unroll
            for (int c = 0; c < Cfg::SB_TILES; ++c)
              tmem_copy_scales<PAIR>(sb_tmem + 4 * (i * Cfg::SB_TILES + c), sbd + 32 * (c * Cfg::ATOMS + i));
          }
          if constexpr (PAIR)
            umma_commit_pair(smem_u32(&s_ready[buf]));
          else
            umma_commit(&s_ready[buf]);
          buf = (buf + 1) % Cfg::SBUFS;
          if (buf == 0) buf_phase ^= 1u;
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scheduler
    int pub = 0;
    auto publish = [&](const Fp4Tile& t) -> bool {
      const int s = pub & (TRING - 1);
      if (!mbar_wait(&tr_empty[s], ((uint32_t)(pub / TRING) & 1u) ^ 1u, abort_flag)) return false;
      __syncwarp();
      if (lane == 0) {
        volatile int* e = ring + 8 * s;
        e[0] = t.kind;
        e[1] = t.member;
        e[2] = t.x_row;
        e[3] = t.y_row;
        e[4] = t.rows;
        e[5] = t.nt;
        e[6] = t.x_tile;
        e[7] = t.n_valid;
        mbar_arrive(&tr_full[s]);
      }
      ++pub;
      return true;
    };
    const Fp4Groups& g = pr.groups;
    // rows of group i: members, then (ragged) the rows before the first and behind the last member's
    const int n_groups = g.offsets ? g.P + 2 : g.P;
    auto group = [&](int i, int& first, int& end) {
      if (i < g.P) {
        first = (int)fp4_first_row(g, i);
        end = (int)fp4_end_row(g, i);
      } else if (i == g.P) {
        first = 0;
        end = (int)fp4_first_row(g, 0);
      } else {
        first = (int)fp4_first_row(g, g.P);
        end = (int)g.rows;
      }
    };
    Fp4Tile t;
    bool ok = true;
    int g0 = 0, first = 0, end = 0, tiles = 0, inc = 0;
    long long before = 0;
    auto load_groups = [&]() {
      first = end = 0;
      if (g0 + lane < n_groups) group(g0 + lane, first, end);
      tiles = (end - first + Cfg::TILE_M - 1) / Cfg::TILE_M * pr.n_tiles;
      inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
    };
    load_groups();
    for (long long i = worker; ok; i += workers) {
      int sum = __shfl_sync(0xFFFFFFFFu, inc, 31);
      while (i >= before + sum && g0 + 32 < n_groups) {
        before += sum;
        g0 += 32;
        load_groups();
        sum = __shfl_sync(0xFFFFFFFFu, inc, 31);
      }
      if (i >= before + sum) break;
      const int local = (int)(i - before);
      const int who = __ffs(__ballot_sync(0xFFFFFFFFu, local < inc)) - 1;
      const int r = local - __shfl_sync(0xFFFFFFFFu, inc - tiles, who);
      const int f = __shfl_sync(0xFFFFFFFFu, first, who), e = __shfl_sync(0xFFFFFFFFu, end, who);
      const int mts = (e - f + Cfg::TILE_M - 1) / Cfg::TILE_M;
      t.member = g0 + who;
      t.nt = r / mts;
      const int mt = r - t.nt * mts;
      t.y_row = f + mt * Cfg::TILE_M;
      t.x_row = pr.x_shared ? mt * Cfg::TILE_M : t.y_row;
      t.rows = min(Cfg::TILE_M, e - t.y_row);
      t.kind = FT_ZERO;
      t.n_valid = t.x_tile = 0;
      if (t.member < g.P) {
        t.x_tile = (int)(pr.x_shared ? 0 : fp4_first_tile(g, t.member)) + mt * (Cfg::TILE_M / 128);
        t.n_valid = pr.out_f ? min(__ldg(pr.out_f + t.member), pr.N) : pr.N;
        if (t.nt * BN < t.n_valid && k_blocks(t.member) > 0) t.kind = FT_MMA;
      }
      ok = publish(t);
    }
    if (ok) {
      t.kind = FT_END;
      publish(t);
    }
  } else if (warp >= Cfg::EPI_WARP0) {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - Cfg::EPI_WARP0;
    const int q = warp & 3, half = ew >> 2;
    constexpr int WCOLS = Cfg::WCOLS;
    constexpr int NCH = WCOLS / 32;
    uint8_t* stage_warp = ctrl + Cfg::CTRL_BYTES + ew * Cfg::EPI_BYTES;
    float* sbias = reinterpret_cast<float*>(stage_warp + 16 * Cfg::ROW_BYTES);
    float* sscale = sbias + WCOLS;
    uint8_t* stage_row = stage_warp + (lane & 15) * Cfg::ROW_BYTES;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int k = 0;; ++k) {
      const Fp4Tile t = ring_read(k, true);
      if (t.kind == FT_END) break;
      const int cbase = t.nt * BN + half * WCOLS;
      const int nch = min(NCH, max(0, (pr.N - cbase + 31) / 32));
      const int rows = t.rows - rank * Cfg::BM - q * 32;
      const long long row0 = (long long)t.y_row + rank * Cfg::BM + q * 32;
      const bool mma = t.kind == FT_MMA;
      const bool biased = mma || t.nt * BN < t.n_valid;  // (without input features: the bias alone)
      float rs = 0.f;
      if (biased) {
        __syncwarp();
        for (int j = lane; j < WCOLS; j += 32) {
          const bool in = cbase + j < t.n_valid;
          sbias[j] = (in && pr.bias) ? __ldg(pr.bias + (long long)t.member * pr.N + cbase + j) : 0.f;
          sscale[j] = in && mma ? __ldg(pr.w_row + (long long)t.member * pr.N + cbase + j) : 0.f;
        }
        if (mma && lane < rows) rs = __ldg(pr.x_row + (long long)t.x_row + rank * Cfg::BM + q * 32 + lane);
        __syncwarp();
      }
      if (mma) {
        if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
        tc_fence_after();
      }
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * WCOLS);
      auto release = [&]() {  // the accumulator has been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR)
            mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));  // the leader's MMA thread waits on it
          else
            mbar_arrive(&tempty[acc]);
        }
        if (++acc == Cfg::ACCS) {
          acc = 0;
          acc_phase ^= 1u;
        }
      };
      if (mma && !pr.y_f32 && pr.y_vec && !__any_sync(0xFFFFFFFFu, rs > FP4_SCALE_STEP)) {
        // bf16: the whole slice goes to registers, rounded, before the accumulator is given back (there is one)
        uint32_t y[WCOLS / 2], v[2][16];
        tmem_ld_32x32b_x16(t_row, v[0]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < WCOLS; c += 16) {
          if (c + 16 < WCOLS) tmem_ld_32x32b_x16(t_row + (uint32_t)(c + 16), v[(c / 16 + 1) & 1]);
          const uint32_t(&u)[16] = v[(c / 16) & 1];
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 sc = *reinterpret_cast<const float4*>(sscale + c + j), bi = *reinterpret_cast<const float4*>(sbias + c + j);
            float x0 = fmaf(__uint_as_float(u[j]) * rs, sc.x, bi.x), x1 = fmaf(__uint_as_float(u[j + 1]) * rs, sc.y, bi.y);
            float x2 = fmaf(__uint_as_float(u[j + 2]) * rs, sc.z, bi.z), x3 = fmaf(__uint_as_float(u[j + 3]) * rs, sc.w, bi.w);
            if (pr.relu) x0 = max_nan(x0, 0.f), x1 = max_nan(x1, 0.f), x2 = max_nan(x2, 0.f), x3 = max_nan(x3, 0.f);
            y[(c + j) / 2] = pack_bf16x2(x0, x1);
            y[(c + j) / 2 + 1] = pack_bf16x2(x2, x3);
          }
          tmem_wait_ld();
        }
        release();
        if (rows > 0) {
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(pr.y);
          const int nv = t.n_valid - cbase;  // (columns behind the member's: zeros, whatever was multiplied there)
          constexpr int PIECES = WCOLS < 64 ? WCOLS / 8 : 8;  // of 16 bytes, of a staged row
#pragma unroll
          for (int c = 0; c < WCOLS; c += 8 * PIECES) {
            if (cbase + c < pr.N) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                __syncwarp();
                if ((lane >> 4) == h) {
#pragma unroll
                  for (int p = 0; p < PIECES; ++p) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                      const int j = c / 2 + 4 * p + e;
                      w[e] = 2 * j + 1 < nv ? y[j] : 2 * j < nv ? y[j] & 0xFFFFu : 0u;
                    }
                    *reinterpret_cast<uint4*>(stage_row + 16 * p) = make_uint4(w[0], w[1], w[2], w[3]);
                  }
                }
                __syncwarp();
                const int p = lane % PIECES, col0 = cbase + c + 8 * p;
#pragma unroll
                for (int i = 0; i < PIECES / 2; ++i) {
                  const int r = lane / PIECES + i * (32 / PIECES);
                  if (16 * h + r < rows && col0 < pr.N)
                    *reinterpret_cast<uint4*>(out + (row0 + 16 * h + r) * pr.N + col0) =
                        *reinterpret_cast<const uint4*>(stage_warp + r * Cfg::ROW_BYTES + 16 * p);
                }
              }
            }
          }
        }
        continue;
      }
      if (rows > 0) {
#pragma unroll 1
        for (int c = 0; c < nch; ++c) {
          uint32_t v[32];
          if (mma) {
            tmem_ld_32x32b_x32(t_row + (uint32_t)(32 * c), v);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0u;
          }
          const int nv = t.n_valid - (cbase + 32 * c), col0 = cbase + 32 * c;
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            __syncwarp();
            if ((lane >> 4) == h) {
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  const int o = 32 * c + j + e;
                  x[e] = 0.f;
                  if (biased) {
                    x[e] = fp4_result(__uint_as_float(v[j + e]), rs, sscale[o], sbias[o]);
                    if (pr.relu) x[e] = max_nan(x[e], 0.f);
                    if (j + e >= nv) x[e] = 0.f;
                  }
                }
                if (pr.y_f32) {
                  *reinterpret_cast<float4*>(stage_row + j * 4) = make_float4(x[0], x[1], x[2], x[3]);
                  *reinterpret_cast<float4*>(stage_row + j * 4 + 16) = make_float4(x[4], x[5], x[6], x[7]);
                } else {
                  *reinterpret_cast<uint4*>(stage_row + j * 2) =
                      make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
                }
              }
            }
            __syncwarp();
            const int some = min(rows - 16 * h, 16);
            if (pr.y_vec) {
              // 16-byte pieces: 8 (fp32) or 4 (bf16) of a row
              const int per = pr.y_f32 ? 8 : 4, size = pr.y_f32 ? 4 : 2;
              for (int i = lane; i < 16 * per; i += 32) {
                const int r = i / per, p = i - r * per;
                if (r < some && (col0 * size + 16 * p) < pr.N * size)
                  *reinterpret_cast<uint4*>(static_cast<uint8_t*>(pr.y) + ((row0 + 16 * h + r) * pr.N + col0) * size + 16 * p) =
                      *reinterpret_cast<const uint4*>(stage_warp + r * Cfg::ROW_BYTES + 16 * p);
              }
            } else if (col0 + lane < pr.N) {
              for (int r = 0; r < some; ++r) {
                const long long at = (row0 + 16 * h + r) * pr.N + col0 + lane;
                if (pr.y_f32)
                  static_cast<float*>(pr.y)[at] = *reinterpret_cast<const float*>(stage_warp + r * Cfg::ROW_BYTES + 4 * lane);
                else
                  static_cast<__nv_bfloat16*>(pr.y)[at] =
                      *reinterpret_cast<const __nv_bfloat16*>(stage_warp + r * Cfg::ROW_BYTES + 2 * lane);
              }
            }
          }
        }
      }
      if (mma) release();
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // neither CTA leaves while the other may still signal it
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    else
      tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace tp
