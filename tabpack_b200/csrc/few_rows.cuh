// Linear layers over groups of a few rows: the weights are the bound, each read once from memory.
//
// Here the weights' rows are the 128 lanes of the accumulator and 32 rows of x (64 in 4 bits, where a product's scales begin at
// an even column of a tile's four) its columns: Y^T = W X^T.  A stage is then mostly weights, where 128-row tiles of x would be
// nearly empty, and the tiles are small enough that every SM gets some; where there are few all the same, the K loop is split
// over a cluster of up to eight CTAs, which add their parts up in order through distributed shared memory.  Two CTAs share an
// SM, so that one's start and end lie under the other's copies.
#pragma once

#include "fp4.cuh"
#include "ragged_gemm.cuh"

namespace tp {

enum : int { FEW_BF16 = 0, FEW_NV = 1, FEW_MX = 2 };

struct FewArgs {
  Fp4Groups groups;  // rows of y: ragged, or P equal groups
  int x_shared;      // equal groups that all read the same rows of x
  int K, N;
  const int32_t* in_f;   // (P) or null
  const int32_t* out_f;  // (P) or null
  const float* bias;     // (P, N) or null
  int relu;
  void* y;  // (rows of y, N)
  int y_f32;
  // 4-bit operands
  const uint8_t* x_scales;
  const float* x_row;
  const uint8_t* w_scales;  // (P, ceil(N / 128), atoms, 512)
  const float* w_row;       // (P, N)
  int atoms;
};

// Contiguous bytes (a multiple of 16, on 16-byte boundaries) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

template <int KIND>
struct FewCfg {
  static constexpr bool FP4 = KIND != FEW_BF16;
  static constexpr int BM = 128, BN = FP4 ? 64 : 32;
  static constexpr int BK = FP4 ? 256 : 64;  // 128 bytes of a row
  static constexpr int ATOMS = KIND == FEW_NV ? 4 : KIND == FEW_MX ? 2 : 0;
  static constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, S_BYTES = ATOMS * 512;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + 2 * S_BYTES;
  static constexpr int STAGES = FP4 ? 3 : 5;
  static constexpr int TMEM_COLS = FP4 ? 128 : 32;  // accumulator, then both operands' scales
  static constexpr int SA_COL = 64, SB_COL = 80;
  static constexpr int CTRL_BYTES = 256;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + CTRL_BYTES;
  static_assert(SMEM_BYTES <= 113 * 1024, "two CTAs an SM");
};

template <int KIND>
__global__ void __launch_bounds__(128, 2)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const FewArgs pr,
                    const int split) {
  using Cfg = FewCfg<KIND>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smA + STAGES * Cfg::A_BYTES;
  uint8_t* smSA = smB + STAGES * Cfg::B_BYTES;
  uint8_t* smSB = smSA + STAGES * Cfg::S_BYTES;
  uint8_t* ctrl = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_id(), lane = lane_id();
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int m0 = (int)(blockIdx.x / (unsigned)split) * Cfg::BM;  // first output

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) tmem_alloc(tmem_slot, Cfg::TMEM_COLS);

  // this CTA's rows: the y-th piece of BN among the groups' (every warp finds it for itself)
  constexpr int BN = Cfg::BN;
  const Fp4Groups& g = pr.groups;
  const int n_groups = g.offsets ? g.P + 2 : g.P;
  int member = -1, row0 = 0, rows = 0, local = 0;
  if (g.offsets == nullptr) {
    const int per = (g.B + BN - 1) / BN;
    member = blockIdx.y / per;
    local = ((int)blockIdx.y - member * per) * BN;
    row0 = member * g.B + local;
    rows = min(BN, g.B - local);
  } else {
    int before = 0, lowest = (int)g.rows;
    for (int g0 = 0; g0 < n_groups; g0 += 32) {
      const int i = g0 + lane;
      int first = 0, end = 0;
      if (i < g.P) {
        first = (int)fp4_first_row(g, i);
        end = (int)fp4_end_row(g, i);
      } else if (i == g.P) {
        end = (int)fp4_first_row(g, 0);
      } else if (i == g.P + 1) {
        first = (int)fp4_first_row(g, g.P);
        end = (int)g.rows;
      }
      // (the rows before the first member's end where any member's begin, should the offsets decrease)
      lowest = min(lowest, __reduce_min_sync(0xFFFFFFFFu, i < g.P ? first : (int)g.rows));
      if (i == g.P) end = min(end, lowest);
      const int n = (end - first + BN - 1) / BN;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
        if (lane >= o) inc += v;
      }
      const int y = (int)blockIdx.y - before;
      const unsigned hit = __ballot_sync(0xFFFFFFFFu, y < inc);
      if (hit) {
        const int who = __ffs(hit) - 1;
        member = g0 + who;
        local = (y - __shfl_sync(0xFFFFFFFFu, inc - n, who)) * BN;
        row0 = __shfl_sync(0xFFFFFFFFu, first, who) + local;
        rows = min(BN, __shfl_sync(0xFFFFFFFFu, end, who) - row0);
        break;
      }
      before += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
  }
  const bool work = member >= 0, real = work && member < g.P;
  const int k_len = real ? (pr.in_f ? min(__ldg(pr.in_f + member), pr.K) : pr.K) : 0;
  const int n_valid = real ? (pr.out_f ? min(__ldg(pr.out_f + member), pr.N) : pr.N) : 0;
  const int all_blocks = m0 < n_valid ? (k_len + Cfg::BK - 1) / Cfg::BK : 0;
  // this CTA's share of the K loop
  const int share = (all_blocks + split - 1) / split;
  const int kb0 = min(all_blocks, rank * share), kb1 = min(all_blocks, kb0 + share);
  // bf16: the last block may hold elements beyond the member's width
  const bool cut = !Cfg::FP4 && (k_len & 15) != 0 && k_len != pr.K && kb1 == all_blocks && kb1 > kb0;
  const int o = m0 + warp * 32 + lane;  // this thread's output
  const float bias = (pr.bias && real && o < n_valid) ? __ldg(pr.bias + (long long)member * pr.N + o) : 0.f;
  const float ws = (Cfg::FP4 && real && o < n_valid) ? __ldg(pr.w_row + (long long)member * pr.N + o) : 1.f;

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (kb1 > kb0) {
    const int x_row = pr.x_shared ? local : row0;
    if (warp == 0 && lane == 0) {
      const uint8_t* sa = nullptr;
      const uint8_t* sb = nullptr;
      if constexpr (Cfg::FP4) {
        sa = pr.w_scales + ((long long)member * ((pr.N + 127) / 128) + m0 / 128) * pr.atoms * 512;
        sb = pr.x_scales + ((pr.x_shared ? 0ll : fp4_first_tile(g, member)) + local / 128) * pr.atoms * 512;
      }
      for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
        const int s = i % STAGES;
        if (!mbar_wait(&empty[s], ((uint32_t)(i / STAGES) & 1u) ^ 1u, abort_flag)) break;
        mbar_arrive_expect_tx(&full[s], Cfg::STAGE_BYTES);
        const int k0 = Cfg::FP4 ? kb * 128 : kb * Cfg::BK;
        tma_load_3d(smA + s * Cfg::A_BYTES, &tmA, &full[s], k0, m0, member);
        tma_load_3d(smB + s * Cfg::B_BYTES, &tmB, &full[s], k0, x_row, 0);
        if constexpr (Cfg::FP4) {
          bulk_load(smSA + s * Cfg::S_BYTES, sa + kb * Cfg::S_BYTES, Cfg::S_BYTES, &full[s]);
          bulk_load(smSB + s * Cfg::S_BYTES, sb + kb * Cfg::S_BYTES, Cfg::S_BYTES, &full[s]);
        }
      }
    } else if (warp == 1) {
      bool ok = true;
      auto multiply = [&](int i, int steps) {
        const int s = i % STAGES;
        const uint32_t a_base = smem_u32(smA + s * Cfg::A_BYTES), b_base = smem_u32(smB + s * Cfg::B_BYTES);
        if constexpr (Cfg::FP4) {
          constexpr int FORMAT = KIND == FEW_NV ? FP4_NV : FP4_MX;
          const uint64_t sa = scale_desc(smem_u32(smSA + s * Cfg::S_BYTES)), sb = scale_desc(smem_u32(smSB + s * Cfg::S_BYTES));
#pragma unroll
          for (int j = 0; j < Cfg::ATOMS; ++j) {
            tmem_copy_scales(tmem_base + Cfg::SA_COL + 4 * j, sa + 32 * j);
            tmem_copy_scales(tmem_base + Cfg::SB_COL + 4 * j, sb + 32 * j);
          }
          // 64 rows are two of a scale tile's four columns
          const uint32_t shift = (uint32_t)(local / 64 & 1) * 2u;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = FORMAT == FP4_NV ? j : j >> 1;
            const uint32_t id = FORMAT == FP4_NV ? 0u : (uint32_t)(j & 1) * 2u;
            umma_fp4<FORMAT>(tmem_base, smem_desc_sw128(a_base + j * 32, 16, 1024), smem_desc_sw128(b_base + j * 32, 16, 1024),
                             idesc_fp4<FORMAT>(Cfg::BN, id), tmem_base + Cfg::SA_COL + 4 * at,
                             tmem_base + Cfg::SB_COL + 4 * at + shift, (i | j) != 0 ? 1u : 0u);
          }
        } else {
          const uint32_t idesc = idesc_bf16_f32(Cfg::BN, false, false);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < steps)
              umma_f16(tmem_base, smem_desc_sw128(a_base + j * 32, 16, 1024), smem_desc_sw128(b_base + j * 32, 16, 1024),
                       idesc, (i | j) != 0 ? 1u : 0u);
        }
        umma_commit(&empty[s]);
      };
      const int n = kb1 - kb0, last = min(Cfg::BK, k_len - (kb1 - 1) * Cfg::BK);
      const int plain = cut ? n - 1 : n;
      if (lane == 0) {
        for (int i = 0; i < plain; ++i) {
          if (!mbar_wait(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          multiply(i, i < n - 1 ? 4 : (last + 15) >> 4);
        }
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if constexpr (!Cfg::FP4) {
        if (ok && cut) {
          const int s = plain % STAGES;
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(&full[s], (uint32_t)(plain / STAGES) & 1u, abort_flag));
          if (ok) {
            const int end = (last + 15) & ~15;
            zero_k_major(smA + s * Cfg::A_BYTES, Cfg::BM, last, end, lane);
            zero_k_major(smB + s * Cfg::B_BYTES, Cfg::BN, last, end, lane);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            tc_fence_after();
            if (lane == 0) multiply(plain, (last + 15) >> 4);
          }
        }
      }
      if (lane == 0) umma_commit(done);
    }
    __syncwarp();
    // every product has completed (so have the copies it waited for)
    volatile int no_abort = 0;
    mbar_wait(done, 0, &no_abort);
  }
  __syncwarp();
  tc_fence_after();
  // rows j0 .. j0 + 31 of the sums, zeros where this CTA has none
  auto sums = [&](int j0, float (&v)[32]) {
    if (kb1 > kb0) {
      uint32_t u[32];
      tmem_ld_32x32b_x32(tmem_base + ((uint32_t)(warp * 32) << 16) + (uint32_t)j0, u);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(u[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = 0.f;
    }
  };
  auto store = [&](int j, float x) {
    if (all_blocks == 0)
      x = bias;  // (without input features)
    else if constexpr (Cfg::FP4)
      x = fp4_result(x, __ldg(pr.x_row + (pr.x_shared ? local : row0) + j), ws, bias);
    else
      x += bias;
    if (pr.relu) x = max_nan(x, 0.f);
    if (o >= n_valid) x = 0.f;
    if (o < pr.N) {
      const long long at = (long long)(row0 + j) * pr.N + o;
      if (pr.y_f32)
        static_cast<float*>(pr.y)[at] = x;
      else
        static_cast<__nv_bfloat16*>(pr.y)[at] = __float2bfloat16_rn(x);
    }
  };
  if (split == 1) {
    if (work) {
      for (int j0 = 0; j0 < rows; j0 += 32) {
        float v[32];
        sums(j0, v);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (j0 + j < rows) store(j0 + j, v[j]);
      }
    }
  } else {
    // parts to shared memory (the stages are free: every copy has landed), then each CTA adds up some of the rows
    float* part = reinterpret_cast<float*>(smem);
    for (int j0 = 0; j0 < BN; j0 += 32) {
      float v[32];
      sums(j0, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) part[(j0 + j) * 128 + warp * 32 + lane] = v[j];
    }
    cluster_sync();
    if (work) {
      for (int j = rank; j < rows; j += split) {
        float x = 0.f;
        const uint32_t at = smem_u32(part + j * 128 + warp * 32 + lane);
        for (int r = 0; r < split; ++r) x += __uint_as_float(ld_shared_cluster_u32(mapa_shared(at, r)));
        store(j, x);
      }
    }
    cluster_sync();  // no CTA leaves while another reads its part
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
}

}  // namespace tp
