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
//
// Large groups run on CTA pairs (cta_group::2): 256 x 256 tiles of which each CTA stages 128 rows of A and half of B,
// two thirds of the operand bytes per product.  A stage that needs zeros then completes on a barrier of its own CTA;
// the peer reports its zeros to the leader, which issues the products.
//
// Results in fp32 are summed over at most RAGGED_SEGMENT elements of K in one accumulator, the pieces in the epilogue's
// registers with the rounding of fp32: the tensor core's own sums do not round to nearest, and over 23054 rows came out 2.6e-5 off
// (5e-7 with the cut, which costs 5 % of the time: 8 x 4096 x 4096 over 4096 rows each 863 us, 816 with pieces of 8192).
// Few tiles over many rows are split over CTAs, into parts that a second launch adds up in order.
//
// fp32 operands come as three bf16 parts each (ragged_split_kernel), and the six products of parts whose terms exceed 2^-24
// of the result are summed: a sixth of the bf16 rate, where the CUDA cores give a twenty-fifth.  Single CTAs hold all parts of a
// block in a stage; tiles of 256 columns on pairs, which leave no tensor memory for two accumulators a tile, go through the K loop
// once for each product.  Either way the product of the first parts has an accumulator of its own, on pairs the one before the
// others': so the others round at their own size, and are left out where it is not finite.  An infinite number is its first
// part, the other parts are 0, so its large product is infinite or NaN as the definition has it, while the small ones would
// add inf * 0 or an infinity of the other sign.  (Both gradients of 12 members, 4099 rows, 100 -> 512: 32 us by six loops, 22 by
// one; forward of 8 members of 512 rows, 512 -> 512, 29 by six loops, 17 by one; 8 x 2048 rows, 1024 -> 1024, 185 by one and 177
// on pairs, of which 6 are the second accumulator.)
#pragma once

#include <type_traits>

#include "common.cuh"

namespace tp {

enum : int { RAGGED_FWD = 0, RAGGED_DGRAD = 1, RAGGED_WGRAD = 2 };
enum : int { RT_MMA = 0, RT_ZERO = 1, RT_END = 2 };
constexpr int RAGGED_SEGMENT = 1024, RAGGED_SEGMENT_F32 = 512;

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
  int splits;              // wgrad: parts of a member's rows; c holds a (P, out, in) result for each
  int a_part, b_part;      // fp32: columns between the parts of A and B
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

// forward, dgrad: `rows` rows from row0 on, sums from element `part` on; wgrad: input features from row0 on, `rows` is the
// first row of the sum, `part` its part.  add, bit 0: on top of the piece before; bit 1: more is to come.
struct RaggedTile {
  int kind, member, row0, rows, nt, k_len, n_valid, m_valid, part, add;
};

template <int BN_, int MODE, bool PAIR_, bool F32 = false>
struct RaggedCfg {
  static constexpr bool PAIR = PAIR_;
  // fp32 on single CTAs: a stage holds all three parts of its operands, whose six products go to two accumulators, that of
  // the first parts and that of the others
  static constexpr bool ALL = F32 && !PAIR;
  static_assert(!ALL || BN_ == 128, "two accumulators of two buffers");
  static constexpr int PARTS = ALL ? 3 : 1, PASSES = F32 && !ALL ? 6 : 1, PRODUCTS = ALL ? 6 : 1;
  static constexpr bool TWICE = F32 && !ALL;  // a tile fills two accumulators one after the other
  static constexpr int SEGMENT = F32 ? RAGGED_SEGMENT_F32 : RAGGED_SEGMENT;
  static_assert(!PAIR || BN_ == 256, "pairs take tiles of 256 columns");
  static constexpr int BM = 128, BN = BN_, BK = 64;
  static constexpr int TILE_M = PAIR ? 256 : 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;  // columns of B that a CTA stages
  static constexpr bool A_MN = MODE == RAGGED_WGRAD;
  static constexpr bool B_MN = MODE != RAGGED_FWD;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = B_ROWS * BK * 2, STAGE_BYTES = PARTS * (A_BYTES + B_BYTES);
  // fp32 results are summed up over the pieces of the K loop in the epilogue's registers, 64 columns a thread at most
  static constexpr bool SUMS = F32 || MODE == RAGGED_WGRAD;
  static constexpr int STAGES = ALL ? 2 : PAIR ? (F32 && MODE != RAGGED_WGRAD ? 5 : 6) : BN == 256 ? 4 : BN == 128 ? 6 : 7;
  static constexpr int ACC_COLS = ALL ? 2 * BN : BN, TMEM_COLS = 2 * ACC_COLS;
  static constexpr int EPI_WARP0 = 4, EPI_WARPS = SUMS && BN == 256 ? 16 : 8;
  static constexpr int THREADS = 32 * (EPI_WARP0 + EPI_WARPS);
  static constexpr int TRING = 4;
  static constexpr int RING_INTS = 10;
  static constexpr int CTRL_BYTES = 640;
  static constexpr int ROW_BYTES = 80;  // a warp's staged row of 32 bf16, padded against bank conflicts
  static constexpr int WCOLS = BN / (EPI_WARPS / 4);  // columns of an epilogue warp
  static constexpr int EPI_BYTES = MODE == RAGGED_WGRAD ? 0 : 32 * ROW_BYTES + WCOLS * 4;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + CTRL_BYTES + EPI_WARPS * EPI_BYTES;
  static_assert(SMEM_BYTES <= 227 * 1024, "fits an SM");
};

// Zeros over elements k_first .. k_end - 1 (along K, within a stage; k_end the next multiple of 16) of a K-major operand
// of `rows` rows (a multiple of 32): a mask over the 16-byte piece that k_first lies in, zeros in the one behind it.
// (An element at a time took 6 us a tile.)
__device__ __forceinline__ void zero_k_major(uint8_t* s, int rows, int k_first, int k_end, int lane) {
  const int p = k_first >> 3, keep = k_first & 7;
  // elements 2 i and 2 i + 1 of the piece
  uint32_t mask[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mask[i] = keep >= 2 * i + 2 ? 0xFFFFFFFFu : keep == 2 * i + 1 ? 0x0000FFFFu : 0u;
  const bool second = p + 1 < (k_end >> 3);
#pragma unroll 4
  for (int r = lane; r < rows; r += 32) {
    uint8_t* row = s + r * 128;
    uint4* at = reinterpret_cast<uint4*>(row + ((p ^ (r & 7)) << 4));
    uint4 v = *at;
    v = make_uint4(v.x & mask[0], v.y & mask[1], v.z & mask[2], v.w & mask[3]);
    *at = v;
    if (second) *reinterpret_cast<uint4*>(row + (((p + 1) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
  }
}
// The same of an MN-major operand: K rows of 128 bytes in pieces of 64 columns.
template <int CHUNKS>
__device__ __forceinline__ void zero_mn_major(uint8_t* s, int k_first, int k_end, int lane) {
  const int n = (k_end - k_first) * 8;
  uint4* at = reinterpret_cast<uint4*>(s + k_first * 128) + lane;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
    for (int i = lane; i < n; i += 32) at[c * 512 + i - lane] = make_uint4(0, 0, 0, 0);
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

// A warp's staged 32 x 16 fp32 values into the result.
__device__ __forceinline__ void ragged_flush_f32(float* c, int ld, int vec, long long row0, int rows, int col0,
                                                 const uint8_t* stage, int row_bytes, int lane) {
  if (vec) {
    const int q = lane & 3;
    if (col0 + 4 * q >= ld) return;
    float* to = c + row0 * ld + col0 + 4 * q;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = (lane >> 2) + 8 * k;
      if (r < rows) *reinterpret_cast<float4*>(to + (long long)r * ld) = *reinterpret_cast<const float4*>(stage + r * row_bytes + q * 16);
    }
  } else {
    const int q = lane & 15;
    if (col0 + q >= ld) return;
    float* to = c + row0 * ld + col0 + q;
    for (int r = lane >> 4; r < min(rows, 32); r += 2)
      to[(long long)r * ld] = *reinterpret_cast<const float*>(stage + r * row_bytes + 4 * q);
  }
}

// Columns that a pair multiplies in a tile: the rest of the member's, rounded up to 32 (16 a CTA).
__device__ __forceinline__ int ragged_n(bool pair, int bn, const RaggedTile& t) {
  const int left = t.n_valid - t.nt * bn;
  return min(bn, pair ? (left + 31) & ~31 : (left + 15) & ~15);
}

// One of the products by this CTA (pair), number `worker` of `workers`.
template <int BN, int MODE, bool PAIR, bool F32>
__device__ __forceinline__ void ragged_gemm(const CUtensorMap& tmA, const CUtensorMap& tmB, const RaggedProblem& pr,
                                            const int worker, const int workers) {
  using Cfg = RaggedCfg<BN, MODE, PAIR, F32>;
  constexpr int STAGES = Cfg::STAGES, TRING = Cfg::TRING;
  extern __shared__ uint8_t dyn_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smem + STAGES * Cfg::PARTS * Cfg::A_BYTES;
  uint8_t* ctrl = smem + STAGES * Cfg::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ctrl);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* done_bar = tempty + 2;
  uint64_t* tr_full = done_bar + 1;
  uint64_t* tr_empty = tr_full + TRING;
  uint64_t* cut_full = tr_empty + TRING;    // pairs: a stage that needs zeros has landed in this CTA
  uint64_t* cut_peer = cut_full + STAGES;   // pairs: the peer has put in its zeros
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(cut_peer + STAGES);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* ring = reinterpret_cast<volatile int*>(ctrl + 384);
  static_assert(8 * (4 * STAGES + 5 + 2 * TRING) + 8 <= 384 && 384 + 4 * Cfg::RING_INTS * TRING <= Cfg::CTRL_BYTES,
                "control block");

  const int warp = warp_id(), lane = lane_id();
  const int rank = PAIR ? (int)cluster_ctarank() : 0;

  // (`whole`: all lanes of the warp read, and lane 0 frees the slot once they have)
  auto ring_read = [&](int k, bool whole) -> RaggedTile {
    RaggedTile t;
    const int s = k & (TRING - 1);
    if (!mbar_wait(&tr_full[s], (uint32_t)(k / TRING) & 1u, abort_flag)) {
      t.kind = RT_END;
      return t;
    }
    const volatile int* e = ring + Cfg::RING_INTS * s;
    t.kind = e[0];
    t.member = e[1];
    t.row0 = e[2];
    t.rows = e[3];
    t.nt = e[4];
    t.k_len = e[5];
    t.n_valid = e[6];
    t.m_valid = e[7];
    t.part = e[8];
    t.add = e[9];
    if (whole) __syncwarp();
    if (!whole || lane == 0) mbar_arrive(&tr_empty[s]);
    return t;
  };
  // a K loop over the whole width ends where the copies fill with zeros by themselves
  const int k_full = MODE == RAGGED_FWD ? pr.in : MODE == RAGGED_DGRAD ? pr.out : -1;
  auto is_cut = [&](const RaggedTile& t) {
    return (t.k_len & 15) != 0 && (MODE == RAGGED_WGRAD || t.part + t.k_len != k_full);
  };
  // fp32: which parts of A and B a pass multiplies, two bits each: hh, then lh, hl, mm, mh, hm
  auto a_of = [&](int pass) { return F32 ? (0x148 >> (2 * pass)) & 3 : 0; };
  auto b_of = [&](int pass) { return F32 ? (0x460 >> (2 * pass)) & 3 : 0; };
  // zeros from element `left` of a stage's K on, up to the next step of 16; by a whole warp
  auto zero_tail = [&](int stage, int left) {
    const int end = (left + 15) & ~15;
#pragma unroll
    for (int part = 0; part < Cfg::PARTS; ++part) {
      uint8_t* a = smA + (stage * Cfg::PARTS + part) * Cfg::A_BYTES;
      uint8_t* b = smB + (stage * Cfg::PARTS + part) * Cfg::B_BYTES;
      if constexpr (Cfg::A_MN)
        zero_mn_major<Cfg::BM / 64>(a, left, end, lane);
      else
        zero_k_major(a, Cfg::BM, left, end, lane);
      if constexpr (Cfg::B_MN)
        zero_mn_major<Cfg::B_ROWS / 64>(b, left, end, lane);
      else
        zero_k_major(b, Cfg::B_ROWS, left, end, lane);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&cut_full[s], 1);
      mbar_init(&cut_peer[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], PAIR ? 2 * Cfg::EPI_WARPS : Cfg::EPI_WARPS);  // the leader's counts both CTAs
    }
    mbar_init(done_bar, 1);
    for (int i = 0; i < TRING; ++i) {
      mbar_init(&tr_full[i], 1);
      mbar_init(&tr_empty[i], 3 + Cfg::EPI_WARPS);  // producers, MMA warp, epilogue warps
    }
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
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
    // ------------------------------------------------------------------ producers: A by warp 0, B by warp 3
    // (one thread takes about 190 cycles a copy, a stage's products 512: with both operands on one thread the issue of
    // copies bound the gradients, whose operands take two each)
    if (lane == 0) {
      const bool is_a = warp == 0;
      const CUtensorMap* map = is_a ? &tmA : &tmB;
      constexpr bool WG = MODE == RAGGED_WGRAD;
      const int boxes = is_a ? (Cfg::A_MN ? Cfg::BM / 64 : 1) : (Cfg::B_MN ? Cfg::B_ROWS / 64 : 1);
      const bool mn = is_a ? Cfg::A_MN : Cfg::B_MN;
      uint8_t* const ring0 = is_a ? smA : smB;
      const int bytes = is_a ? Cfg::A_BYTES : Cfg::B_BYTES;
      const uint32_t leader0 = PAIR ? mapa_shared(smem_u32(full), 0) : 0;
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      // One stage: a pair's bytes complete on the leader's barrier, those of a stage that needs zeros (OWN) on this
      // CTA's own.  The A producer announces the bytes of both (B's may arrive first: the phase waits for its arrival).
      auto produce = [&](auto own, int x, int y, int z) -> bool {
        constexpr bool OWN = decltype(own)::value;
        if (!mbar_wait(&empty[stage], phase ^ 1u, abort_flag)) return false;
        uint64_t* bar = PAIR && OWN ? &cut_full[stage] : &full[stage];
        if (is_a) {
          if (OWN)
            mbar_arrive_expect_tx(bar, Cfg::STAGE_BYTES);
          else if (rank == 0)
            mbar_arrive_expect_tx(bar, 2 * Cfg::STAGE_BYTES);
        }
#pragma unroll
        for (int part = 0; part < Cfg::PARTS; ++part) {
          uint8_t* dst = ring0 + (stage * Cfg::PARTS + part) * bytes;
          const int at = x + part * (is_a ? pr.a_part : pr.b_part);
          for (int c = 0; c < boxes; ++c) {
            if constexpr (OWN)
              tma_load_3d(dst + c * 8192, map, bar, at + (mn ? c * 64 : 0), y, z);
            else
              tma_load_3d_pair(dst + c * 8192, map, leader0 + 8u * stage, at + (mn ? c * 64 : 0), y, z);
          }
        }
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
        return true;
      };
      for (int k = 0; ok; ++k) {
        const RaggedTile t = ring_read(k, false);
        if (t.kind == RT_END) break;
        if (t.kind != RT_MMA) continue;
        const int kblocks = (t.k_len + Cfg::BK - 1) / Cfg::BK;
        // the copies' coordinates: along K and along the other side
        const int b_col = t.nt * BN + (PAIR ? rank * (ragged_n(true, BN, t) / 2) : 0);
        const int other = is_a ? t.row0 + rank * Cfg::BM : b_col;
        const int k_first = WG ? t.rows : t.part, z = (is_a || WG) ? 0 : t.member;
        const int common = !PAIR ? 0 : is_cut(t) ? kblocks - 1 : kblocks;  // stages on the common barrier
        for (int pass = 0; ok && pass < Cfg::PASSES; ++pass) {
          const int shift = Cfg::PASSES == 1 ? 0 : is_a ? a_of(pass) * pr.a_part : b_of(pass) * pr.b_part;
          int kb = 0;
          for (; ok && kb < common; ++kb) {
            const int at = k_first + kb * Cfg::BK;
            ok = produce(std::bool_constant<!PAIR>(), (mn ? other : at) + shift, mn ? at : other, z);
          }
          for (; ok && kb < kblocks; ++kb) {
            const int at = k_first + kb * Cfg::BK;
            ok = produce(std::bool_constant<true>(), (mn ? other : at) + shift, mn ? at : other, z);
          }
        }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------------ MMA (a pair's leader fills both CTAs' TMEM)
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0, cut_phase = 0;  // cut_phase: a bit per stage
    bool ok = true;
    // descriptors of the first stage; the address field counts 16 bytes
    const uint64_t adesc0 = Cfg::A_MN ? smem_desc_sw128(smem_u32(smA), 8192, 1024) : smem_desc_sw128(smem_u32(smA), 16, 1024);
    const uint64_t bdesc0 = Cfg::B_MN ? smem_desc_sw128(smem_u32(smB), 8192, 1024) : smem_desc_sw128(smem_u32(smB), 16, 1024);
    for (int k = 0; ok; ++k) {
      const RaggedTile t = ring_read(k, true);
      if (t.kind == RT_END) break;
      if (t.kind != RT_MMA) continue;
      const uint32_t idesc = idesc_bf16_f32(ragged_n(PAIR, BN, t), Cfg::A_MN, Cfg::B_MN, Cfg::TILE_M);
      uint32_t d_tmem = tmem_base + (uint32_t)(acc * Cfg::ACC_COLS);
      if (!mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag)) break;
      tc_fence_after();
      // an accumulator is complete once this thread's products so far are
      auto hand_over = [&]() {
        if (lane == 0) {
          if constexpr (PAIR) {
            umma_commit_both(&tfull[acc]);
          } else {
            umma_commit(&tfull[acc]);
          }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      };
      const int kblocks = (t.k_len + Cfg::BK - 1) / Cfg::BK;
      const int last = t.k_len - (kblocks - 1) * Cfg::BK;  // elements of the last block
      const bool cut = is_cut(t);
      // a stage's products and its release, by one thread
      auto multiply = [&](int stage, int steps, bool first) {
#pragma unroll
        for (int product = 0; product < Cfg::PRODUCTS; ++product) {
          const int a_part = Cfg::ALL ? a_of(product) : 0, b_part = Cfg::ALL ? b_of(product) : 0;
          const uint64_t adesc = adesc0 + (uint64_t)((stage * Cfg::PARTS + a_part) * (Cfg::A_BYTES / 16));
          const uint64_t bdesc = bdesc0 + (uint64_t)((stage * Cfg::PARTS + b_part) * (Cfg::B_BYTES / 16));
          const uint32_t d = Cfg::ALL && product > 0 ? d_tmem + BN : d_tmem;
#pragma unroll
          for (int s = 0; s < Cfg::BK / 16; ++s) {
            // 16 elements further along K: 32 bytes of a K-major row, 16 rows of an MN-major block (in units of 16 bytes)
            const uint64_t ad = adesc + (uint64_t)(s * (Cfg::A_MN ? 128 : 2)), bd = bdesc + (uint64_t)(s * (Cfg::B_MN ? 128 : 2));
            const uint32_t on = (first && s == 0 && product < 2) ? 0u : 1u;
            if (s < steps) {
              if constexpr (PAIR)
                umma_f16_pair(d, ad, bd, idesc, on);
              else
                umma_f16(d, ad, bd, idesc, on);
            }
          }
        }
        if constexpr (PAIR) {  // frees the stage in both CTAs
          umma_commit_both(&empty[stage]);
        } else {
          umma_commit(&empty[stage]);
        }
      };
      // one thread goes through the blocks; the whole warp comes together for one that needs zeros
      const int plain = cut ? kblocks - 1 : kblocks;
      for (int pass = 0; ok && pass < Cfg::PASSES; ++pass) {
        const bool opens = pass == 0 || (Cfg::TWICE && pass == 1);  // the first products of an accumulator
        if (Cfg::TWICE && pass == 1) {
          hand_over();
          d_tmem = tmem_base + (uint32_t)(acc * Cfg::ACC_COLS);
          ok = __all_sync(0xFFFFFFFFu, mbar_wait(&tempty[acc], acc_phase ^ 1u, abort_flag));
          if (!ok) break;
          tc_fence_after();
        }
        if (lane == 0) {
          int st = stage;
          uint32_t ph = phase;
          for (int kb = 0; kb < plain; ++kb) {
            if (!mbar_wait(&full[st], ph, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (kb < kblocks - 1)
              multiply(st, Cfg::BK / 16, opens && kb == 0);
            else
              multiply(st, (last + 15) >> 4, opens && kb == 0);
            if (++st == STAGES) {
              st = 0;
              ph ^= 1u;
            }
          }
        }
        phase ^= (uint32_t)((stage + plain) / STAGES) & 1u;
        stage = (stage + plain) % STAGES;
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (ok && cut) {
          if constexpr (PAIR) {
            const uint32_t ph = (cut_phase >> stage) & 1u;
            ok = mbar_wait(&cut_full[stage], ph, abort_flag);
            if (__all_sync(0xFFFFFFFFu, ok)) {
              zero_tail(stage, last);
              ok = mbar_wait<true>(&cut_peer[stage], ph, abort_flag);
            }
            if (lane == 0) mbar_arrive(&full[stage]);  // the stage's phase goes on without the common barrier
            cut_phase ^= 1u << stage;
          } else {
            ok = mbar_wait(&full[stage], phase, abort_flag);
            if (__all_sync(0xFFFFFFFFu, ok)) zero_tail(stage, last);
          }
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (ok) {
            tc_fence_after();
            if (lane == 0) multiply(stage, (last + 15) >> 4, opens && kblocks == 1);
            __syncwarp();
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) break;
      hand_over();
    }
    if (lane == 0) {  // every MMA of this CTA has completed once it flips
      if constexpr (PAIR)
        umma_commit_pair(smem_u32(done_bar));
      else
        umma_commit(done_bar);
    }
    volatile int no_abort = 0;
    mbar_wait(done_bar, 0, &no_abort);
  } else if (warp == 1) {
    // ------------------------------------------------------------------ zeros of a pair's second CTA
    int stage = 0;
    uint32_t cut_phase = 0;
    for (int k = 0;; ++k) {
      const RaggedTile t = ring_read(k, true);
      if (t.kind == RT_END) break;
      if (t.kind != RT_MMA) continue;
      const int kblocks = (t.k_len + Cfg::BK - 1) / Cfg::BK;
      bool ok = true;
      for (int pass = 0; ok && pass < Cfg::PASSES; ++pass) {
        const int last = (stage + kblocks - 1) % STAGES;
        stage = (stage + kblocks) % STAGES;
        if (!is_cut(t)) continue;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&cut_full[last], (cut_phase >> last) & 1u, abort_flag));
        cut_phase ^= 1u << last;
        if (!ok) break;
        zero_tail(last, t.k_len - (kblocks - 1) * Cfg::BK);
        if (lane == 0) mbar_arrive_release_cluster(mapa_shared(smem_u32(&cut_peer[last]), 0));
      }
      if (!ok) break;
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------------ scheduler (a pair's CTAs find the same tiles)
    int pub = 0;
    auto publish = [&](const RaggedTile& t) -> bool {
      const int s = pub & (TRING - 1);
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(&tr_empty[s], ((uint32_t)(pub / TRING) & 1u) ^ 1u, abort_flag))) return false;
      if (lane == 0) {
        volatile int* e = ring + Cfg::RING_INTS * s;
        e[0] = t.kind;
        e[1] = t.member;
        e[2] = t.row0;
        e[3] = t.rows;
        e[4] = t.nt;
        e[5] = t.k_len;
        e[6] = t.n_valid;
        e[7] = t.m_valid;
        e[8] = t.part;
        e[9] = t.add;
        mbar_arrive(&tr_full[s]);
      }
      ++pub;
      return true;
    };
    RaggedTile t;
    t.part = t.add = 0;
    bool ok = true;
    if constexpr (MODE == RAGGED_WGRAD) {
      const int tiles = pr.m_tiles * pr.n_tiles, per = tiles * pr.splits;
      const long long total = (long long)pr.P * per;
      for (long long i = worker; ok && i < total; i += workers) {
        t.member = (int)(i / per);
        const int r = (int)(i - (long long)t.member * per);
        t.part = r / tiles;
        const int tile = r - t.part * tiles;
        t.nt = tile / pr.m_tiles;
        t.row0 = (tile - t.nt * pr.m_tiles) * Cfg::TILE_M;
        int first, end;
        ragged_group(pr, t.member, first, end);
        const int share = ((end - first + pr.splits - 1) / pr.splits + 63) & ~63;
        first = (int)min((long long)end, (long long)first + (long long)t.part * share);
        end = min(end, first + share);
        t.m_valid = pr.in_f ? min(__ldg(pr.in_f + t.member), pr.in) : pr.in;
        t.n_valid = pr.out_f ? min(__ldg(pr.out_f + t.member), pr.out) : pr.out;
        if (end > first && t.row0 < t.m_valid && t.nt * BN < t.n_valid) {
          t.kind = RT_MMA;
          // pieces of about the same length
          const int pieces = (end - first + Cfg::SEGMENT - 1) / Cfg::SEGMENT;
          const int piece = ((end - first + pieces - 1) / pieces + 63) & ~63;
          for (int k = first; ok && k < end; k += piece) {
            t.rows = k;
            t.k_len = min(piece, end - k);
            t.add = (k > first ? 1 : 0) | (k + piece < end ? 2 : 0);
            ok = publish(t);
          }
        } else {
          t.kind = RT_ZERO;
          t.k_len = t.add = 0;
          ok = publish(t);
        }
      }
    } else {
      int g0 = 0;          // first group of the 32 that the lanes hold
      long long before = 0;  // tiles of the groups before them
      int first = 0, end = 0, tiles = 0, inc = 0, lowest = pr.R;
      auto load_groups = [&]() {
        first = end = 0;
        if (g0 + lane < pr.P + 2) ragged_group(pr, g0 + lane, first, end);
        // (the rows before the first member's end where any member's begin, should the offsets decrease)
        lowest = min(lowest, __reduce_min_sync(0xFFFFFFFFu, g0 + lane < pr.P ? first : pr.R));
        if (g0 + lane == pr.P) end = min(end, lowest);
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
        const int mt = (e - f + Cfg::TILE_M - 1) / Cfg::TILE_M;
        t.member = g0 + who;
        t.nt = r / mt;
        t.row0 = f + (r - t.nt * mt) * Cfg::TILE_M;
        t.rows = min(Cfg::TILE_M, e - t.row0);
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
        if (F32 && t.kind == RT_MMA) {
          // pieces of the K loop, added up in the result
          const int whole = t.k_len, pieces = (whole + Cfg::SEGMENT - 1) / Cfg::SEGMENT;
          const int piece = ((whole + pieces - 1) / pieces + 63) & ~63;
          for (int k = 0; ok && k < whole; k += piece) {
            t.part = k;
            t.k_len = min(piece, whole - k);
            t.add = (k > 0 ? 1 : 0) | (k + piece < whole ? 2 : 0);
            ok = publish(t);
          }
          t.part = t.add = 0;
        } else {
          ok = publish(t);
        }
      }
    }
    if (ok) {
      t.kind = RT_END;
      publish(t);
    }
  } else if (warp >= Cfg::EPI_WARP0) {
    // ------------------------------------------------------------------ epilogue
    const int ew = warp - Cfg::EPI_WARP0;
    const int q = warp & 3, slice = ew >> 2;  // lanes and columns of the accumulator
    constexpr int WCOLS = Cfg::WCOLS;
    constexpr int NCH = (WCOLS + 31) / 32;
    uint8_t* stage_warp = ctrl + Cfg::CTRL_BYTES + ew * Cfg::EPI_BYTES;
    float* sbias = reinterpret_cast<float*>(stage_warp + 32 * Cfg::ROW_BYTES);
    uint8_t* stage_row = stage_warp + lane * Cfg::ROW_BYTES;
    int acc = 0;
    uint32_t acc_phase = 0;
    float sum[Cfg::SUMS ? WCOLS : 1];
    auto release = [&]() {  // the accumulator has been read
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));  // the leader's MMA warp waits on it
        else
          mbar_arrive(&tempty[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    };
    for (int k = 0;; ++k) {
      const RaggedTile t = ring_read(k, true);
      if (t.kind == RT_END) break;
      const int cbase = t.nt * BN + slice * WCOLS;
      const bool mma = t.kind == RT_MMA;
      const bool biased = MODE == RAGGED_FWD && (mma || t.nt * BN < t.n_valid);  // (without input features: the bias alone)
      if (biased && !(t.add & 1)) {
        __syncwarp();
        for (int j = lane; j < WCOLS; j += 32)
          sbias[j] = (pr.bias != nullptr && cbase + j < t.n_valid) ? __ldg(pr.bias + (long long)t.member * pr.out + cbase + j) : 0.f;
        __syncwarp();
      }
      if (mma) {
        if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
        tc_fence_after();
      }
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * Cfg::ACC_COLS + slice * WCOLS);
      if constexpr (Cfg::SUMS) {
        if (!(t.add & 1)) {
#pragma unroll
          for (int c = 0; c < WCOLS; ++c) sum[c] = 0.f;
        }
        if (mma) {
#pragma unroll
          for (int c = 0; c < WCOLS; c += 8) {
            uint32_t v[8];
            tmem_ld_32x32b_x8(t_row + (uint32_t)c, v);
            if constexpr (Cfg::ALL) {
              uint32_t u[8];
              tmem_ld_32x32b_x8(t_row + (uint32_t)(BN + c), u);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float large = __uint_as_float(v[j]);
                sum[c + j] += fabsf(large) < INFINITY ? large + __uint_as_float(u[j]) : large;
              }
            } else {
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 8; ++j) sum[c + j] += __uint_as_float(v[j]);
            }
          }
          release();
          if constexpr (Cfg::TWICE) {
            if (!mbar_wait(&tfull[acc], acc_phase, abort_flag)) break;
            tc_fence_after();
            const uint32_t t_small = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * Cfg::ACC_COLS + slice * WCOLS);
#pragma unroll
            for (int c = 0; c < WCOLS; c += 8) {
              uint32_t v[8];
              tmem_ld_32x32b_x8(t_small + (uint32_t)c, v);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (fabsf(sum[c + j]) < INFINITY) sum[c + j] += __uint_as_float(v[j]);
            }
            release();
          }
          if (t.add & 2) continue;
        }
        if constexpr (MODE == RAGGED_WGRAD) {
          // lane = input feature, register = output feature: 32 consecutive floats of a row of dw per store
          const int col = t.row0 + rank * Cfg::BM + q * 32 + lane;
          if (col < pr.in) {
            float* to = static_cast<float*>(pr.c) + (((long long)t.part * pr.P + t.member) * pr.out + cbase) * pr.in + col;
            const int n_out = pr.out - cbase, n_valid = col < t.m_valid ? t.n_valid - cbase : 0;
#pragma unroll
            for (int j = 0; j < WCOLS; ++j) {
              if (j < n_out) *to = j < n_valid ? sum[j] : 0.f;
              to += pr.in;
            }
          }
        } else {
          const int ld = MODE == RAGGED_FWD ? pr.out : pr.in;
          const int rows = t.rows - rank * Cfg::BM - q * 32;  // of this warp, may be below 1 or above 32
          const long long row0 = (long long)t.row0 + rank * Cfg::BM + q * 32;
          if (rows > 0) {
#pragma unroll
            for (int c = 0; c < WCOLS; c += 16) {
              const int col0 = cbase + c;
              if (col0 < ld) {
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  float x[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    x[e] = sum[c + j + e];
                    if (biased) {
                      x[e] += sbias[c + j + e];
                      if (pr.relu) x[e] = max_nan(x[e], 0.f);
                    }
                    if (col0 + j + e >= t.n_valid) x[e] = 0.f;
                  }
                  *reinterpret_cast<float4*>(stage_row + j * 4) = make_float4(x[0], x[1], x[2], x[3]);
                }
                __syncwarp();
                ragged_flush_f32(static_cast<float*>(pr.c), ld, pr.c_vec, row0, rows, col0, stage_warp, Cfg::ROW_BYTES, lane);
                __syncwarp();
              }
            }
          }
        }
      } else {
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(pr.c);
        const int ld = MODE == RAGGED_FWD ? pr.out : pr.in;
        const int nch = min(NCH, max(0, (ld - cbase + 31) / 32));
        const int rows = t.rows - rank * Cfg::BM - q * 32;  // of this warp, may be below 1 or above 32
        const long long row0 = (long long)t.row0 + rank * Cfg::BM + q * 32;
        if (rows > 0 && mma) {
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
        } else if (rows > 0) {
#pragma unroll 1
          for (int c = 0; c < nch; ++c) {
            if (c == 0 || biased) {
              __syncwarp();
#pragma unroll 1
              for (int j = 0; j < 32; j += 2) {
                float x[2] = {0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  if (biased && cbase + 32 * c + j + e < t.n_valid) x[e] = sbias[32 * c + j + e];
                  if (pr.relu) x[e] = max_nan(x[e], 0.f);
                }
                *reinterpret_cast<uint32_t*>(stage_row + j * 2) = pack_bf16x2(x[0], x[1]);
              }
              __syncwarp();
            }
            ragged_flush(out, ld, pr.c_vec, row0, rows, cbase + 32 * c, stage_warp, Cfg::ROW_BYTES, lane);
          }
        }
        if (mma) release();
      }
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

template <int BN, int MODE, bool PAIR, bool F32>
__global__ void __launch_bounds__(RaggedCfg<BN, MODE, PAIR, F32>::THREADS, 1)
    ragged_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                       const __grid_constant__ RaggedProblem pr) {
  constexpr int shift = PAIR ? 1 : 0;
  ragged_gemm<BN, MODE, PAIR, F32>(tmA, tmB, pr, (int)(blockIdx.x >> shift), (int)(gridDim.x >> shift));
}

// Both gradients in one launch, dx by the first n CTAs: where all tiles fit the SMs at once, neither waits for the other.
template <int BN, bool F32>
__global__ void __launch_bounds__(RaggedCfg<BN, RAGGED_WGRAD, false, F32>::THREADS, 1)
    ragged_gradients_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                            const __grid_constant__ RaggedProblem pr, const __grid_constant__ CUtensorMap tmA2,
                            const __grid_constant__ CUtensorMap tmB2, const __grid_constant__ RaggedProblem pr2, const int n) {
  static_assert(RaggedCfg<BN, RAGGED_WGRAD, false, F32>::THREADS == RaggedCfg<BN, RAGGED_DGRAD, false, F32>::THREADS, "one block size");
  if ((int)blockIdx.x < n)
    ragged_gemm<BN, RAGGED_DGRAD, false, F32>(tmA, tmB, pr, (int)blockIdx.x, n);
  else
    ragged_gemm<BN, RAGGED_WGRAD, false, F32>(tmA2, tmB2, pr2, (int)blockIdx.x - n, (int)gridDim.x - n);
}

// dw = the sum of its parts, in their order.
__global__ void __launch_bounds__(256) ragged_parts_kernel(const float* parts, float* dw, long long n, int count) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 4
  for (int k = 0; k < count; ++k) s += __ldcs(parts + k * n + i);
  dw[i] = s;
}

// ---------------------------------------------------------------------------
// fp32 operands as three bf16 parts, x = h + m + l with h = bf16(x), m = bf16(x - h), l = bf16(x - h - m): 24 bits in
// all, each difference exact (of numbers below 2^-102 l falls below bf16's smallest normal number).  A row's parts lie side by
// side, `cols` columns (a multiple of 64) each, zeros at the end.
// Of a number that is not finite h is the whole; of one that would round to infinity h is bf16's largest, and m has the rest.
// ---------------------------------------------------------------------------
constexpr float BF16_MAX = 3.3895313892515355e38f;

struct SplitArgs {
  const float* x[3];  // up to three matrices in a launch
  long long ld[3], rows[3];
  int width[3], cols[3], vec[3];  // vec: rows on 16-byte boundaries
  FastDiv div[3];                 // by the pieces of 8 columns of a row
  __nv_bfloat16* out[3];
};

__global__ void __launch_bounds__(256) ragged_split_kernel(const SplitArgs a) {
  const int k = blockIdx.y;
  const int pieces = a.cols[k] / 8;
  const long long total = a.rows[k] * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i < 0x7FFFFFFFLL ? (long long)fastdiv((uint32_t)i, a.div[k]) : i / pieces;
    const int c = 8 * (int)(i - r * pieces);
    const float* x = a.x[k] + r * a.ld[k] + c;
    float v[8];
    if (a.vec[k] && c + 8 <= a.width[k]) {
      const float4 lo = __ldg(reinterpret_cast<const float4*>(x)), hi = __ldg(reinterpret_cast<const float4*>(x) + 1);
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < a.width[k] ? __ldg(x + e) : 0.f;
    }
    __nv_bfloat16* out = a.out[k] + 3 * r * a.cols[k] + c;
    bool odd = false;  // a first part is infinite or NaN: of eight numbers hardly ever one
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      uint32_t w[4];
      float h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[e] = __bfloat162float(__float2bfloat16_rn(v[e]));
        if (p == 0) odd |= !(fabsf(h[e]) < INFINITY);
      }
      if (p == 0 && odd) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool finite = fabsf(v[e]) < INFINITY;
          if (finite) h[e] = fminf(fmaxf(h[e], -BF16_MAX), BF16_MAX);
          v[e] = finite ? v[e] - h[e] : 0.f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] -= h[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(h[2 * e], h[2 * e + 1]);
      *reinterpret_cast<uint4*>(out + p * a.cols[k]) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// ---------------------------------------------------------------------------
// g = dy [y > 0] with rows at g_ld (a multiple of 8 columns: an operand of the products), and the members' sums of
// g over their rows.  A block takes 64 or 256 columns of a member's share of rows; the shares' sums are added up in order
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

// Eight columns of a row as they lie in memory, zeros from column n on.
template <typename T, bool VEC>
struct Act8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, int c0, int n) {
    if (VEC) {  // (rows on 16-byte boundaries, n a multiple of 8)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = __ldcs(reinterpret_cast<const uint4*>(p + c0) + i);
    } else {
      T v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c0 + j < n ? p[c0 + j] : (T)0.f;
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = reinterpret_cast<const uint4*>(v)[i];
    }
  }
  __device__ __forceinline__ float get(int j) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(u);
    if (sizeof(T) == 4) return __uint_as_float(w[j]);
    return __uint_as_float((j & 1) ? (w[j >> 1] & 0xFFFF0000u) : (w[j >> 1] << 16));
  }
};

// VEC: dy and y have rows on 16-byte boundaries and N is a multiple of 8.  C threads side by side take 8 C columns.
template <typename T, bool VEC, int C, bool RELU>
__global__ void __launch_bounds__(256) ragged_act_kernel(const RaggedAct a) {
  constexpr int U = (RELU ? 4 : 8) * 2 / (int)sizeof(T);  // rows of a thread on their way
  constexpr int ROWS = 256 / C;                           // rows side by side
  __shared__ float red[ROWS][8 * C + 1];
  const int m = blockIdx.y, cg = threadIdx.x % C, rl = threadIdx.x / C;
  const int c0 = blockIdx.x * 8 * C + cg * 8;
  RaggedProblem p{};
  p.P = a.P;
  p.R = a.R;
  p.offsets = a.offsets;
  int first, end;
  ragged_group(p, m, first, end);
  const int per = (end - first + a.S - 1) / a.S;
  const int r0 = (int)min((long long)end, first + (long long)blockIdx.z * per), r1 = min(end, r0 + per);
  const int out_m = a.out_f ? min(a.out_f[m], a.N) : a.N;
  const T* dy = static_cast<const T*>(a.dy);
  const T* y = static_cast<const T*>(a.y);
  T* g = static_cast<T*>(a.g);
  float sum[8] = {};
  if (c0 < a.N || (g != nullptr && c0 < a.g_ld)) {
    for (int r = r0 + rl; r < r1; r += ROWS * U) {
      Act8<T, VEC> d[U], s[RELU ? U : 1];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + ROWS * u < r1) {
          d[u].load(dy + (long long)(r + ROWS * u) * a.dy_ld, c0, a.N);
          if constexpr (RELU) s[u].load(y + (long long)(r + ROWS * u) * a.N, c0, a.N);
        }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r + ROWS * u < r1) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = d[u].get(j);
            if constexpr (RELU) v[j] = s[u].get(j) > 0.f ? v[j] : 0.f;
            if (c0 + j >= out_m) v[j] = 0.f;
            sum[j] += v[j];
          }
          if (g != nullptr) {
            T* to = g + (long long)(r + ROWS * u) * a.g_ld + c0;
            if (sizeof(T) == 2) {  // (rows of g are multiples of 8)
              *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]),
                                                         pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
            } else {
              reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
              reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
            }
          }
        }
      }
    }
  }
  if (a.db == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[rl][cg * 8 + j] = sum[j];
  __syncthreads();
  if (threadIdx.x < 8 * C) {
    const int c = blockIdx.x * 8 * C + threadIdx.x;
    if (c < a.N) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) s += red[r][threadIdx.x];
      (a.S > 1 ? a.partial + (long long)blockIdx.z * a.P * a.N : a.db)[(long long)m * a.N + c] = s;
    }
  }
}

__global__ void __launch_bounds__(256) ragged_bias_kernel(const RaggedAct a) {
  const long long n = (long long)a.P * a.N, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
#pragma unroll 8
  for (int k = 0; k < a.S; ++k) s += a.partial[k * n + i];
  a.db[i] = s;
}

}  // namespace tp
