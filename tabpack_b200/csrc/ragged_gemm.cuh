// Products over ragged groups of rows: member m of a pack multiplies rows offsets[m] .. offsets[m + 1] - 1 of one
// (rows, width) matrix.
//
//   RAGGED_FWD  : Y[r, o] = relu(sum_i X[r, i] W_m[o, i] + b_m[o])   A = X, B = W, both K-major
//   RAGGED_DGRAD: dX[r, i] = sum_o G[r, o] W_m[o, i]                  A = G K-major, B = W MN-major
//   RAGGED_WGRAD: dW_m[o, i] = sum_r G[r, o] X[r, i]                  A = X^T, B = G^T, both MN-major; K = the member's rows
//
// in_features / out_features cut a member's columns; what lies beyond takes no part, whatever it holds, and is zero
// in the result.  Rows that belong to no member are zero in Y and dX.
//
// The group sizes are known on the device only: each CTA's scheduler warp walks the groups, 32 at a time, and finds
// its tiles by sums over the warp.  A group's last tile reads rows of the next group (they are not stored), and the
// last block of a cut K loop holds elements beyond the cut: the MMA warp writes zeros over those in shared memory
// before it multiplies, since a zero factor on one side alone would let a NaN of another member through.
#pragma once

#include "common.cuh"

namespace tp {

enum : int { RAGGED_FWD = 0, RAGGED_DGRAD = 1, RAGGED_WGRAD = 2 };
enum : int { RT_MMA = 0, RT_ZERO = 1, RT_END = 2 };

struct RaggedProblem {
  int P, R;                // members, rows of the matrix
  int in, out;             // widths: columns of x / w, rows of w
  const int32_t* offsets;  // (P + 1)
  const int32_t* in_f;     // (P) or null
  const int32_t* out_f;    // (P) or null
  const float* bias;       // forward: (P, out) or null
  int relu;
  void* c;                 // forward: y (R, out), dgrad: dx (R, in), wgrad: dw (P, out, in) fp32
  int c_vec;               // rows of y / dx lie on 16-byte boundaries
  int m_tiles;             // wgrad: tiles of a member along `in`
  int n_tiles;             // tiles along the columns of the result (forward: out, dgrad: in, wgrad: out)
};

// Rows of group g: members 0 .. P - 1, then the rows before the first and behind the last member's.
__device__ __forceinline__ void ragged_group(const RaggedProblem& p, int g, int& first, int& end) {
  const int i = g < p.P ? g : p.P;
  const int o = min(max(__ldg(p.offsets + (g == p.P ? 0 : i)), 0), p.R);
  if (g == p.P) {
    first = 0;
    end = o;
  } else {
    first = o;
    end = g == p.P + 1 ? p.R : max(o, min(max(__ldg(p.offsets + i + 1), 0), p.R));
  }
}

struct RaggedTile {
  int kind, member, row0, rows, nt, k_len, n_valid, m_valid;
};

template <int BN_, int MODE>
struct RaggedCfg {
  static constexpr int BM = 128, BN = BN_, BK = 64;
  static constexpr bool A_MN = MODE == RAGGED_WGRAD;
  static constexpr bool B_MN = MODE != RAGGED_FWD;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 6 : 7;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int EPI_WARP0 = 4, EPI_WARPS = 8;
  static constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
  static constexpr int TRING = 4;
  static constexpr int CTRL_BYTES = 512;
  static constexpr int ROW_BYTES = 80;  // a warp's staged row of 32 bf16, padded against bank conflicts
  static constexpr int WCOLS = BN / 2;  // columns of an epilogue warp
  static constexpr int SMEM_BYTES =
      1024 + STAGES * STAGE_BYTES + CTRL_BYTES + EPI_WARPS * (32 * ROW_BYTES + WCOLS * 4);
  static_assert(SMEM_BYTES <= 227 * 1024, "fits an SM");
};

// Zeros over elements k_first .. k_end - 1 (along K, within a stage) of a K-major operand of `rows` rows.
__device__ __forceinline__ void zero_k_major(uint8_t* s, int rows, int k_first, int k_end, int lane) {
  for (int r = lane; r < rows; r += 32)
    for (int k = k_first; k < k_end;) {
      uint8_t* piece = s + r * 128 + (((k >> 3) ^ (r & 7)) << 4);
      if ((k & 7) == 0 && k + 8 <= k_end) {
        *reinterpret_cast<uint4*>(piece) = make_uint4(0, 0, 0, 0);
        k += 8;
      } else {
        *reinterpret_cast<uint16_t*>(piece + (k & 7) * 2) = 0;
        ++k;
      }
    }
}
// The same of an MN-major operand: K rows of 128 bytes in `chunks` pieces of 64 columns.
__device__ __forceinline__ void zero_mn_major(uint8_t* s, int chunks, int k_first, int k_end, int lane) {
  const int n = (k_end - k_first) * 8;
  for (int i = lane; i < chunks * n; i += 32) {
    const int c = i / n, r = i - c * n;
    *reinterpret_cast<uint4*>(s + c * 8192 + (k_first + (r >> 3)) * 128 + (r & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
}

// A warp's staged 32 x 32 bf16 values, rows row0 .. , columns col0 .. , into the result: 16-byte pieces, or a
// column a lane where rows have no such alignment.
__device__ __forceinline__ void ragged_flush(__nv_bfloat16* c, int ld, int vec, long long row0, int rows, int col0,
                                             const uint8_t* stage, int row_bytes, int lane) {
  if (vec) {
    const int q = lane & 3;
    if (col0 + 8 * q >= ld) return;
    __nv_bfloat16* to = c + row0 * ld + col0 + 8 * q;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = (lane >> 2) + 8 * k;
      if (r < rows)
        *reinterpret_cast<uint4*>(to + (long long)r * ld) = *reinterpret_cast<const uint4*>(stage + r * row_bytes + q * 16);
    }
  } else if (col0 + lane < ld) {
    __nv_bfloat16* to = c + row0 * ld + col0 + lane;
    for (int r = 0; r < min(rows, 32); ++r)
      to[(long long)r * ld] = *reinterpret_cast<const __nv_bfloat16*>(stage + r * row_bytes + 2 * lane);
  }
}

template <int BN, int MODE>
__global__ void __launch_bounds__(RaggedCfg<BN, MODE>::THREADS, 1)
    ragged_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const RaggedProblem pr) {
  using Cfg = RaggedCfg<BN, MODE>;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smem + Cfg::STAGES * Cfg::A_BYTES;
  uint8_t* ctrl = smem + Cfg::STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + Cfg::STAGES;
  uint64_t* tfull = empty + Cfg::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done_bar = tempty + 2;
  constexpr int TRING = Cfg::TRING;
  uint64_t* tr_full = done_bar + 1;
  uint64_t* tr_empty = tr_full + TRING;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tr_empty + TRING);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ring = reinterpret_cast<volatile int*>(ctrl + 256);  // 8 ints a slot
  static_assert(8 * (2 * Cfg::STAGES + 5 + 2 * TRING) + 8 <= 256 && 256 + 32 * TRING <= Cfg::CTRL_BYTES, "control block");

  const int warp = warp_id(), lane = lane_id();

  // (`whole`: all lanes of the warp read, and lane 0 frees the slot once they have)
  auto ring_read = [&](int k, bool whole) -> RaggedTile {
    RaggedTile t;
    const int s = k & (TRING - 1);
    if (!mbar_wait(&tr_full[s], (uint32_t)(k / TRING) & 1u, abort_flag)) {
      t.kind = RT_END;
      return t;
    }
    const volatile int* e = ring + 8 * s;
    t.kind = e[0];
    t.member = e[1];
    t.row0 = e[2];
    t.rows = e[3];
    t.nt = e[4];
    t.k_len = e[5];
    t.n_valid = e[6];
    t.m_valid = e[7];
    if (whole) __syncwarp();
    if (!whole || lane == 0) mbar_arrive(&tr_empty[s]);
    return t;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], Cfg::EPI_WARPS);
    }
    mbar_init(done_bar, 1);
    for (int i = 0; i < TRING; ++i) {
      mbar_init(&tr_full[i], 1);
      mbar_init(&tr_empty[i], 2 + Cfg::EPI_WARPS);  // producer, MMA warp, epilogue warps
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const RaggedTile t = ring_read(k, false);
        if (t.kind == RT_END) break;
        if (t.kind != RT_MMA) continue;
        const int kblocks = (t.k_len + Cfg::BK - 1) / Cfg::BK;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* a = smA + stage * Cfg::A_BYTES;
          uint8_t* b = smB + stage * Cfg::B_BYTES;
          const int k0 = kb * Cfg::BK;
          mbar_arrive_expect_tx(&full[stage], Cfg::STAGE_BYTES);
          if constexpr (MODE == RAGGED_WGRAD) {
            // row0: the tile's first input feature; `rows`: the member's first row
#pragma unroll
            for (int c = 0; c < Cfg::BM / 64; ++c) tma_load_3d(a + c * 8192, &tmA, &full[stage], t.row0 + c * 64, t.rows + k0, 0);
#pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_3d(b + c * 8192, &tmB, &full[stage], t.nt * BN + c * 64, t.rows + k0, 0);
          } else {
            tma_load_3d(a, &tmA, &full[stage], k0, t.row0, 0);
            if constexpr (MODE == RAGGED_FWD) {
              tma_load_3d(b, &tmB, &full[stage], k0, t.nt * BN, t.member);
            } else {
#pragma unroll
              for (int c = 0; c < BN / 64; ++c) tma_load_3d(b + c * 8192, &tmB, &full[stage], t.nt * BN + c * 64, k0, t.member);
            }
          }
          if (++stage == Cfg::STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    const int k_full = MODE == RAGGED_FWD ? pr.in : MODE == RAGGED_DGRAD ? pr.out : -1;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const RaggedTile t = ring_read(k, true);
      if (t.kind == RT_END) break;
      if (t.kind != RT_MMA) continue;
      const int n_mma = min(BN, (t.n_valid - t.nt * BN + 15) & ~15);
      const uint32_t idesc = idesc_bf16_f32(n_mma, Cfg::A_MN, Cfg::B_MN);
      const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
      if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag)) break;
      tc_fence_after();
      const int kblocks = (t.k_len + Cfg::BK - 1) / Cfg::BK;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag)) {
          ok = false;
          break;
        }
        uint8_t* a = smA + stage * Cfg::A_BYTES;
        uint8_t* b = smB + stage * Cfg::B_BYTES;
        const int left = min(Cfg::BK, t.k_len - kb * Cfg::BK);
        const int steps = (left + 15) >> 4;
        // (a K loop over the whole width ends where the copies fill with zeros by themselves)
        if ((left & 15) && t.k_len != k_full) {
          if constexpr (Cfg::A_MN)
            zero_mn_major(a, Cfg::BM / 64, left, 16 * steps, lane);
          else
            zero_k_major(a, Cfg::BM, left, 16 * steps, lane);
          if constexpr (Cfg::B_MN)
            zero_mn_major(b, BN / 64, left, 16 * steps, lane);
          else
            zero_k_major(b, BN, left, 16 * steps, lane);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        tc_fence_after();
        if (lane == 0) {
          const uint32_t a_base = smem_u32(a), b_base = smem_u32(b);
          for (int s = 0; s < steps; ++s) {
            const uint64_t adesc = Cfg::A_MN ? smem_desc_sw128(a_base + s * 2048, 8192, 1024)
                                             : smem_desc_sw128(a_base + s * 32, 16, 1024);
            const uint64_t bdesc = Cfg::B_MN ? smem_desc_sw128(b_base + s * 2048, 8192, 1024)
                                             : smem_desc_sw128(b_base + s * 32, 16, 1024);
            umma_f16(d_tmem, adesc, bdesc, idesc, (kb | s) != 0 ? 1u : 0u);
          }
          umma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == Cfg::STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok) break;
      if (lane == 0) umma_commit(&tfull[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) umma_commit(done_bar);  // every MMA of this CTA has completed once it flips
    volatile int no_abort = 0;
    mbar_wait(done_bar, 0, &no_abort);
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scheduler
    int pub = 0;
    auto publish = [&](const RaggedTile& t) -> bool {
      const int s = pub & (TRING - 1);
      if (!mbar_wait(&tr_empty[s], ((uint32_t)(pub / TRING) & 1u) ^ 1u, abort_flag)) return false;
      __syncwarp();
      if (lane == 0) {
        volatile int* e = ring + 8 * s;
        e[0] = t.kind;
        e[1] = t.member;
        e[2] = t.row0;
        e[3] = t.rows;
        e[4] = t.nt;
        e[5] = t.k_len;
        e[6] = t.n_valid;
        e[7] = t.m_valid;
        mbar_arrive(&tr_full[s]);
      }
      ++pub;
      return true;
    };
    RaggedTile t;
    bool ok = true;
    if constexpr (MODE == RAGGED_WGRAD) {
      const int per = pr.m_tiles * pr.n_tiles;
      const long long total = (long long)pr.P * per;
      for (long long i = blockIdx.x; ok && i < total; i += gridDim.x) {
        t.member = (int)(i / per);
        const int r = (int)(i - (long long)t.member * per);
        t.nt = r / pr.m_tiles;
        t.row0 = (r - t.nt * pr.m_tiles) * Cfg::BM;
        int end;
        ragged_group(pr, t.member, t.rows, end);
        t.k_len = end - t.rows;
        t.m_valid = pr.in_f ? min(__ldg(pr.in_f + t.member), pr.in) : pr.in;
        t.n_valid = pr.out_f ? min(__ldg(pr.out_f + t.member), pr.out) : pr.out;
        t.kind = (t.k_len > 0 && t.row0 < t.m_valid && t.nt * BN < t.n_valid) ? RT_MMA : RT_ZERO;
        ok = publish(t);
      }
    } else {
      int g0 = 0;          // first group of the 32 that the lanes hold
      long long before = 0;  // tiles of the groups before them
      int first = 0, end = 0, tiles = 0, inc = 0;
      auto load_groups = [&]() {
        first = end = 0;
        if (g0 + lane < pr.P + 2) ragged_group(pr, g0 + lane, first, end);
        tiles = (end - first + Cfg::BM - 1) / Cfg::BM * pr.n_tiles;
        inc = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
          if (lane >= o) inc += v;
        }
      };
      load_groups();
      for (long long i = blockIdx.x; ok; i += gridDim.x) {
        int sum = __shfl_sync(0xFFFFFFFFu, inc, 31);
        while (i >= before + sum && g0 + 32 < pr.P + 2) {
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
        const int mt = (e - f + Cfg::BM - 1) / Cfg::BM;
        t.member = g0 + who;
        t.nt = r / mt;
        t.row0 = f + (r - t.nt * mt) * Cfg::BM;
        t.rows = min(Cfg::BM, e - t.row0);
        t.m_valid = t.rows;
        t.kind = RT_ZERO;
        t.k_len = t.n_valid = 0;
        if (t.member < pr.P) {
          const int in_m = pr.in_f ? min(__ldg(pr.in_f + t.member), pr.in) : pr.in;
          const int out_m = pr.out_f ? min(__ldg(pr.out_f + t.member), pr.out) : pr.out;
          t.k_len = MODE == RAGGED_FWD ? in_m : out_m;
          t.n_valid = MODE == RAGGED_FWD ? out_m : in_m;
          if (t.nt * BN < t.n_valid && t.k_len > 0) t.kind = RT_MMA;
        }
        ok = publish(t);
      }
    }
    if (ok) {
      t.kind = RT_END;
      publish(t);
    }
  } else if (warp >= Cfg::EPI_WARP0) {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - Cfg::EPI_WARP0;
    const int q = warp & 3, half = ew >> 2;
    constexpr int WCOLS = Cfg::WCOLS;
    constexpr int NCH = (WCOLS + 31) / 32;
    uint8_t* stage_warp = ctrl + Cfg::CTRL_BYTES + ew * (32 * Cfg::ROW_BYTES + WCOLS * 4);
    float* sbias = reinterpret_cast<float*>(stage_warp + 32 * Cfg::ROW_BYTES);
    uint8_t* stage_row = stage_warp + lane * Cfg::ROW_BYTES;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int k = 0;; ++k) {
      const RaggedTile t = ring_read(k, true);
      if (t.kind == RT_END) break;
      const int cbase = t.nt * BN + half * WCOLS;
      if constexpr (MODE == RAGGED_WGRAD) {
        // lane = input feature, register = output feature: 32 consecutive floats of a row of dw per store
        const int col = t.row0 + q * 32 + lane;
        float* base = static_cast<float*>(pr.c) + (long long)t.member * pr.out * pr.in + col;
        const int nch = min(NCH, max(0, (pr.out - cbase + 31) / 32));
        const bool store = col < pr.in, valid = col < t.m_valid;
        if (t.kind == RT_MMA) {
          if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
          tc_fence_after();
          const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * WCOLS);
#pragma unroll 1
          for (int c = 0; c < nch; ++c) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(t_row + (uint32_t)(32 * c), v);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              const int o = cbase + 32 * c + j;
              if (store && o < pr.out)
                base[(long long)o * pr.in] = (valid && o < t.n_valid) ? __uint_as_float(v[j]) : 0.f;
            }
          }
        } else if (store) {
          const int o1 = min(cbase + WCOLS, pr.out);
          for (int o = cbase; o < o1; ++o) base[(long long)o * pr.in] = 0.f;
        }
      } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(pr.c);
        const int ld = MODE == RAGGED_FWD ? pr.out : pr.in;
        const int nch = min(NCH, max(0, (ld - cbase + 31) / 32));
        const int rows = t.rows - q * 32;  // of this warp, may be below 1 or above 32
        const long long row0 = (long long)t.row0 + q * 32;
        if (t.kind == RT_MMA) {
          const bool biased = MODE == RAGGED_FWD && pr.bias != nullptr;
          if constexpr (MODE == RAGGED_FWD) {
            __syncwarp();
            for (int j = lane; j < WCOLS; j += 32)
              sbias[j] = (biased && cbase + j < t.n_valid) ? __ldg(pr.bias + (long long)t.member * pr.out + cbase + j) : 0.f;
            __syncwarp();
          }
          if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
          tc_fence_after();
          const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + half * WCOLS);
          if (rows > 0) {
#pragma unroll 1
            for (int c = 0; c < nch; ++c) {
              uint32_t v[32];
              tmem_ld_32x32b_x32(t_row + (uint32_t)(32 * c), v);
              tmem_wait_ld();
              const int nv = t.n_valid - (cbase + 32 * c);
#pragma unroll
              for (int j = 0; j < 32; j += 8) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  x[e] = __uint_as_float(v[j + e]);
                  if constexpr (MODE == RAGGED_FWD) {
                    x[e] += sbias[32 * c + j + e];
                    if (pr.relu) x[e] = max_nan(x[e], 0.f);
                  }
                  if (j + e >= nv) x[e] = 0.f;
                }
                *reinterpret_cast<uint4*>(stage_row + j * 2) =
                    make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
              }
              __syncwarp();
              ragged_flush(out, ld, pr.c_vec, row0, rows, cbase + 32 * c, stage_warp, Cfg::ROW_BYTES, lane);
              __syncwarp();
            }
          }
        } else if (rows > 0) {
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(stage_row + 16 * j) = make_uint4(0, 0, 0, 0);
          __syncwarp();
          for (int c = 0; c < nch; ++c)
            ragged_flush(out, ld, pr.c_vec, row0, rows, cbase + 32 * c, stage_warp, Cfg::ROW_BYTES, lane);
        }
      }
      if (t.kind == RT_MMA) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&tempty[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
}

// ---------------------------------------------------------------------------
// The same products on the CUDA cores in fp32: 64 x 64 tiles, 4 x 4 results a thread.
// ---------------------------------------------------------------------------
struct RaggedSimt {
  RaggedProblem p;
  const float* a;  // forward: x, dgrad: g, wgrad: x
  long long a_ld;
  const float* b;  // forward, dgrad: w (rows at w_ld, members at out * w_ld), wgrad: g
  long long b_ld;
};

template <int MODE>
__global__ void __launch_bounds__(256) ragged_simt_kernel(const RaggedSimt s) {
  constexpr int TB = 64, TK = 16;
  __shared__ float As[TK][TB + 4];
  __shared__ float Bs[TK][TB + 4];
  const RaggedProblem& p = s.p;
  const int tid = threadIdx.x, lane = tid & 31;
  // this block's tile: along M the rows of the member (or its input features), along N the result's columns
  int member = 0, m0 = 0, m_end = 0, first = 0, k_len = 0, n_valid = 0, m_valid = 0;
  const int nt = blockIdx.x % p.n_tiles;
  const int i = blockIdx.x / p.n_tiles;
  if (MODE == RAGGED_WGRAD) {
    member = i / p.m_tiles;
    m0 = (i - member * p.m_tiles) * TB;
    m_end = p.in;
    int end;
    ragged_group(p, member, first, end);
    k_len = end - first;
    m_valid = p.in_f ? min(p.in_f[member], p.in) : p.in;
    n_valid = p.out_f ? min(p.out_f[member], p.out) : p.out;
  } else {
    int before = 0, g0 = 0;
    for (;; g0 += 32) {
      if (g0 >= p.P + 2) return;
      int f = 0, e = 0;
      if (g0 + lane < p.P + 2) ragged_group(p, g0 + lane, f, e);
      const int tiles = (e - f + TB - 1) / TB;
      int inc = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      const int sum = __shfl_sync(0xFFFFFFFFu, inc, 31);
      if (i < before + sum) {
        const int who = __ffs(__ballot_sync(0xFFFFFFFFu, i - before < inc)) - 1;
        member = g0 + who;
        m0 = __shfl_sync(0xFFFFFFFFu, f, who) + (i - before - __shfl_sync(0xFFFFFFFFu, inc - tiles, who)) * TB;
        m_end = __shfl_sync(0xFFFFFFFFu, e, who);
        break;
      }
      before += sum;
    }
    if (member < p.P) {
      const int in_m = p.in_f ? min(p.in_f[member], p.in) : p.in;
      const int out_m = p.out_f ? min(p.out_f[member], p.out) : p.out;
      k_len = MODE == RAGGED_FWD ? in_m : out_m;
      n_valid = MODE == RAGGED_FWD ? out_m : in_m;
    }
    m_valid = m_end;
  }
  const int n0 = nt * TB;
  const int n_end = MODE == RAGGED_DGRAD ? p.in : p.out;
  const int tx = tid & 15, ty = tid >> 4;
  float acc[4][4] = {};
  if (n0 < n_valid && m0 < m_valid) {
    const float* w = s.b + (MODE == RAGGED_WGRAD ? 0 : (long long)member * p.out * s.b_ld);
    for (int k0 = 0; k0 < k_len; k0 += TK) {
      for (int j = tid; j < TB * TK; j += 256) {
        const int m = MODE == RAGGED_WGRAD ? j % TB : j / TK, k = MODE == RAGGED_WGRAD ? j / TB : j % TK;
        float v = 0.f;
        if (k0 + k < k_len && m0 + m < m_valid)
          v = MODE == RAGGED_WGRAD ? s.a[(long long)(first + k0 + k) * s.a_ld + m0 + m]
                                   : s.a[(long long)(m0 + m) * s.a_ld + k0 + k];
        As[k][m] = v;
      }
      for (int j = tid; j < TB * TK; j += 256) {
        const int n = MODE == RAGGED_FWD ? j / TK : j % TB, k = MODE == RAGGED_FWD ? j % TK : j / TB;
        float v = 0.f;
        if (k0 + k < k_len && n0 + n < n_valid)
          v = MODE == RAGGED_FWD     ? w[(long long)(n0 + n) * s.b_ld + k0 + k]
              : MODE == RAGGED_DGRAD ? w[(long long)(k0 + k) * s.b_ld + n0 + n]
                                     : w[(long long)(first + k0 + k) * s.b_ld + n0 + n];
        Bs[k][n] = v;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < TK; ++k) {
        const float4 a = *reinterpret_cast<const float4*>(&As[k][ty * 4]);
        const float4 b = *reinterpret_cast<const float4*>(&Bs[k][tx * 4]);
        const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(av[x], bv[y], acc[x][y]);
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int m = m0 + ty * 4 + x;
    if (m >= m_end) continue;
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int n = n0 + tx * 4 + y;
      if (n >= n_end) continue;
      float v = acc[x][y];
      if (MODE == RAGGED_FWD) {
        if (p.bias != nullptr && n < n_valid) v += p.bias[(long long)member * p.out + n];
        if (p.relu) v = max_nan(v, 0.f);
      }
      if (n >= n_valid || m >= m_valid) v = 0.f;
      if (MODE == RAGGED_WGRAD)
        static_cast<float*>(p.c)[((long long)member * p.out + n) * p.in + m] = v;
      else
        static_cast<float*>(p.c)[(long long)m * (MODE == RAGGED_FWD ? p.out : p.in) + n] = v;
    }
  }
}

// ---------------------------------------------------------------------------
// g = dy [y > 0] with rows at g_ld (a multiple of 8 columns: an operand of the products), and the members' sums of
// g over their rows.  A block takes 64 columns of a member's share of rows; the shares' sums are added up in order
// by a second launch.  Memory: dy and y are read once, g is written once.
// ---------------------------------------------------------------------------
struct RaggedAct {
  int P, R, N, S;  // S: shares of a member's rows
  const int32_t* offsets;
  const int32_t* out_f;
  const void* dy;
  long long dy_ld;
  const void* y;  // (R, N), or null: no ReLU
  void* g;        // or null
  long long g_ld;
  float* db;       // (P, N), or null
  float* partial;  // (S, P, N) where S > 1
};

template <typename T>
__global__ void __launch_bounds__(256) ragged_act_kernel(const RaggedAct a) {
  __shared__ float red[32][65];
  const int m = blockIdx.y, cg = threadIdx.x & 7, rl = threadIdx.x >> 3;
  const int c0 = blockIdx.x * 64 + cg * 8;
  RaggedProblem p{};
  p.P = a.P;
  p.R = a.R;
  p.offsets = a.offsets;
  int first, end;
  ragged_group(p, m, first, end);
  const int per = (end - first + a.S - 1) / a.S;
  const int r0 = first + min(end - first, (int)blockIdx.z * per), r1 = min(end, r0 + per);
  const int out_m = a.out_f ? min(a.out_f[m], a.N) : a.N;
  const T* dy = static_cast<const T*>(a.dy);
  const T* y = static_cast<const T*>(a.y);
  T* g = static_cast<T*>(a.g);
  float sum[8] = {};
  for (int r = r0 + rl; r < r1; r += 32) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = c0 + j;
      if (c < a.N) {
        T v = dy[(long long)r * a.dy_ld + c];
        if (y != nullptr && !((float)y[(long long)r * a.N + c] > 0.f)) v = (T)0.f;
        if (c >= out_m) v = (T)0.f;
        if (g != nullptr) g[(long long)r * a.g_ld + c] = v;
        sum[j] += (float)v;
      } else if (g != nullptr && c < a.g_ld) {
        g[(long long)r * a.g_ld + c] = (T)0.f;
      }
    }
  }
  if (a.db == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[rl][cg * 8 + j] = sum[j];
  __syncthreads();
  if (threadIdx.x < 64) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c < a.N) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 32; ++r) s += red[r][threadIdx.x];
      (a.S > 1 ? a.partial + (long long)blockIdx.z * a.P * a.N : a.db)[(long long)m * a.N + c] = s;
    }
  }
}

__global__ void __launch_bounds__(256) ragged_bias_kernel(const RaggedAct a) {
  const long long n = (long long)a.P * a.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int k = 0; k < a.S; ++k) s += a.partial[k * n + i];
  a.db[i] = s;
}

}  // namespace tp
