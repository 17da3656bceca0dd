// C ABI of routing, row moves, ragged linear layers, and 4-bit rows and products (declared in
// include/tabpack_b200.h): host-side validation, tensor maps and kernel dispatch.
#include <algorithm>

#include "few_rows.cuh"
#include "fp4.cuh"
#include "host.cuh"
#include "ragged_gemm.cuh"
#include "routing.cuh"

namespace tp {

// This translation unit's share of the device-side error flag (read and cleared).
int take_routed_error(int* v) {
  TP_CUDA_TRY(cudaMemcpyFromSymbol(v, g_device_error, sizeof(int)));
  const int zero = 0;
  TP_CUDA_TRY(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)));
  return TP_OK;
}

namespace {

// More than 48 KB of shared memory for a kernel: once per device and kernel.
template <auto* KERNEL>
int allow_smem(size_t bytes) {
  static std::atomic<size_t> have[64] = {};
  static std::mutex mu;  // (another thread's smaller size must not come after a larger one)
  int dev = 0;
  TP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(TP_EUNSUPPORTED, "device index %d out of range", dev);
  if (have[dev].load(std::memory_order_acquire) >= bytes) return TP_OK;
  std::lock_guard<std::mutex> lock(mu);
  if (have[dev].load(std::memory_order_relaxed) >= bytes) return TP_OK;
  TP_CUDA_TRY(cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  have[dev].store(bytes, std::memory_order_release);
  return TP_OK;
}

// ------------------------------------------------------------------ routing

// Gate blocks: one where there are few rows, else up to four an SM (two run at a time; a warp's rows are a chain of
// reductions).  A place block takes the rows of `gates` of them: two blocks an SM (65521 rows, 6 of 257: 9.8 us, one block 12.1, four 9.9).
struct RoutePlan {
  int rows, blocks, gates;
};
RoutePlan route_plan(int64_t rows, int32_t k) {
  RoutePlan p{};
  p.rows = rows * k <= 1024 ? (int)std::max<int64_t>(rows, 1) : (int)std::max<int64_t>(16, (rows + 4 * 148 - 1) / (4 * 148));
  p.blocks = (int)((rows + p.rows - 1) / p.rows);
  p.gates = std::max(1, p.blocks / 296);
  return p;
}

constexpr long long ROUTE_MAX_PAIRS = (1ll << 31) - (1ll << 20);  // (the kernels look some rows ahead, in 32 bits)

int check_route(const tp_route_args* a) {
  if (!a) return fail(TP_EINVAL, "null routing arguments");
  if (a->rows <= 0 || a->E <= 0 || a->E > ROUTE_MAX_EXPERTS || a->top_k <= 0 ||
      a->top_k > std::min(ROUTE_MAX_K, a->E) || a->rows > ROUTE_MAX_PAIRS || a->rows * a->top_k > ROUTE_MAX_PAIRS)
    return fail(TP_EINVAL, "routing needs rows > 0, 1 to %d members, top_k up to %d and the members, rows top_k <= 2^31 - 2^20 "
                "(got %lld, %d, %d)", ROUTE_MAX_EXPERTS, ROUTE_MAX_K, (long long)a->rows, a->E, a->top_k);
  if (a->dtype != TP_DTYPE_F32 && a->dtype != TP_DTYPE_BF16) return fail(TP_EINVAL, "bad logits dtype");
  if (!a->logits || !a->weight || !a->expert) return fail(TP_EINVAL, "null logits, weights or members");
  if (a->logits_stride < a->E && a->rows > 1) return fail(TP_EINVAL, "rows of logits overlap");
  if (!aligned_to(dtype_size(a->dtype), {a->logits, a->dlogits}) ||
      !aligned_to(4, {a->weight, a->expert, a->position, a->offsets, a->importance, a->workspace, a->g_weight, a->g_importance}))
    return fail(TP_EALIGN, "routing data not aligned to its type");
  return TP_OK;
}

RouteArgs route_args(const tp_route_args* a) {
  RouteArgs k{};
  k.rows = (int)a->rows;
  k.E = a->E;
  k.k = a->top_k;
  k.renorm = a->renormalize;
  k.ld = a->logits_stride;
  k.logits = a->logits;
  k.weight = a->weight;
  k.expert = a->expert;
  k.position = a->position;
  k.offsets = a->offsets;
  k.importance = a->importance;
  const RoutePlan plan = route_plan(a->rows, a->top_k);
  k.rows_per_block = plan.rows;
  k.blocks = plan.blocks;
  k.gates = plan.gates;
  k.g_weight = a->g_weight;
  k.g_importance = a->g_importance;
  k.dlogits = a->dlogits;
  return k;
}

template <typename T, int G, int F, int V>
int launch_route(const RouteArgs& k, cudaStream_t st) {
  const int blocks = k.blocks;
  const size_t smem = route_shared_bytes(k.E);
  if (blocks == 1) {
    int rc = allow_smem<route_small_kernel<T, G, F, V>>(smem);
    if (rc) return rc;
    route_small_kernel<T, G, F, V><<<1, 32 * ROUTE_WARPS, smem, st>>>(k);
  } else {
    int rc = allow_smem<route_gate_kernel<T, G, F, V>>(smem);
    if (!rc) rc = allow_smem<route_place_kernel>(smem);
    if (rc) return rc;
    route_gate_kernel<T, G, F, V><<<blocks, 32 * ROUTE_WARPS, smem, st>>>(k);
    route_scan_kernel<<<k.E + 1, 256, 0, st>>>(k);
    route_place_kernel<<<(blocks + k.gates - 1) / k.gates, 32 * ROUTE_WARPS, smem, st>>>(k);
  }
  return TP_OK;
}

template <typename T, int G, int F, int V>
int launch_route_backward(const RouteArgs& k, cudaStream_t st) {
  constexpr int ROWS = 256 / G;
  route_backward_kernel<T, G, F, V><<<std::min((k.rows + ROWS - 1) / ROWS, 8 * device_info().sms), 256, 0, st>>>(k);
  return TP_OK;
}

// Lanes a row and registers a lane for its scores: few lanes where a row's scores fit eight registers of them (and the slots
// their lanes), since a row's reductions and ends then share their instructions with other rows'.  Gate and backward of 65536
// rows: 24 members, 2 slots, 7.4 and 5.2 us with 4 lanes, 17.6 and 15.9 with 32; 64 members, 4 slots, 15.9 and 8.7 with 8
// lanes, 23.6 and 17.0 with 32.  The backward holds less else and takes 16 lanes up to 18 registers: 32768 rows of 160 8.7
// against 11.5; the gate does not: 20.3 against 19, and 65521 rows of 257 69 against 39.
template <typename T>
int dispatch_route(const RouteArgs& k, bool backward, cudaStream_t st) {
  const int E = k.E, slots = k.k;
#define TP_ROUTE(g, f, v) \
  if (E <= g * v && slots <= g) return backward ? launch_route_backward<T, g, f, v>(k, st) : launch_route<T, g, f, v>(k, st);
#define TP_ROUTE_G(g) TP_ROUTE(g, 0, 2) TP_ROUTE(g, 2, 4) TP_ROUTE(g, 4, 6) TP_ROUTE(g, 6, 8)
#define TP_ROUTE_BACK(f, v) \
  if (backward && E <= 16 * v && slots <= 16) return launch_route_backward<T, 16, f, v>(k, st);
  TP_ROUTE_G(4)
  TP_ROUTE_G(8)
  TP_ROUTE_G(16)
  TP_ROUTE_BACK(8, 10) TP_ROUTE_BACK(10, 12) TP_ROUTE_BACK(12, 14) TP_ROUTE_BACK(14, 16) TP_ROUTE_BACK(16, 18)
  TP_ROUTE(32, 0, 4)
  TP_ROUTE(32, 4, 5) TP_ROUTE(32, 5, 6) TP_ROUTE(32, 6, 7) TP_ROUTE(32, 7, 8) TP_ROUTE(32, 8, 9) TP_ROUTE(32, 9, 10)
  TP_ROUTE(32, 10, 12) TP_ROUTE(32, 12, 14) TP_ROUTE(32, 14, 16) TP_ROUTE(32, 16, 20) TP_ROUTE(32, 20, 24) TP_ROUTE(32, 24, 32)
#undef TP_ROUTE_BACK
#undef TP_ROUTE_G
#undef TP_ROUTE
  return fail(TP_EINVAL, "too many members");
}

// ------------------------------------------------------------------ row moves

int check_rows(const tp_rows_args* a) {
  if (!a) return fail(TP_EINVAL, "null row move arguments");
  if (a->rows <= 0 || a->k <= 0 || a->k > ROUTE_MAX_K || a->W <= 0 || a->E <= 0 || a->rows > ROUTE_MAX_PAIRS ||
      a->rows * a->k > ROUTE_MAX_PAIRS)
    return fail(TP_EINVAL, "row moves need rows, W, E > 0, 1 <= k <= %d, rows k <= 2^31 - 2^20 (got %lld, %d, %d, %d)", ROUTE_MAX_K,
                (long long)a->rows, a->W, a->E, a->k);
  if (a->dtype != TP_DTYPE_F32 && a->dtype != TP_DTYPE_BF16) return fail(TP_EINVAL, "bad row dtype");
  if (!a->position || !a->offsets) return fail(TP_EINVAL, "null plan");
  if (!aligned_to(dtype_size(a->dtype), {a->x, a->out, a->dout, a->dy}) ||
      !aligned_to(4, {a->position, a->offsets, a->weight, a->dweight}))
    return fail(TP_EALIGN, "rows not aligned to their type");
  return TP_OK;
}

RowsArgs rows_args(const tp_rows_args* a) {
  RowsArgs k{};
  k.T = (int)a->rows;
  k.k = a->k;
  k.W = a->W;
  k.E = a->E;
  k.position = a->position;
  k.offsets = a->offsets;
  k.weight = a->weight;
  k.x = a->x;
  k.x_ld = a->x_stride;
  k.out = a->out;
  k.dout = a->dout;
  k.dout_ld = a->dout_stride;
  k.dy = a->dy;
  k.dw = a->dweight;
  return k;
}

// The widest vectors (bytes) on which every row of the given tables begins.
int rows_vector(const tp_rows_args* a) {
  const int size = (int)dtype_size(a->dtype);
  long long all = (long long)a->W * size | 16;
  if (a->x) all |= reinterpret_cast<intptr_t>(a->x) | a->x_stride * size;
  if (a->out) all |= reinterpret_cast<intptr_t>(a->out);
  if (a->dout) all |= reinterpret_cast<intptr_t>(a->dout) | a->dout_stride * size;
  if (a->dy) all |= reinterpret_cast<intptr_t>(a->dy);
  return (int)(all & -all);
}

enum { ROWS_DISPATCH, ROWS_COMBINE, ROWS_BACKWARD };

template <typename T, int BYTES, int U>
void launch_rows_backward(const RowsArgs& k, cudaStream_t st) {
  if (k.vecs <= 16)
    rows_combine_backward_kernel<T, BYTES, 8, U><<<(k.T + 31) / 32, 256, 0, st>>>(k);
  else if (k.vecs <= 128)
    rows_combine_backward_kernel<T, BYTES, 32, U><<<(k.T + 7) / 8, 256, 0, st>>>(k);
  else
    rows_combine_backward_kernel<T, BYTES, 256, U><<<k.T, 256, 0, st>>>(k);
}

template <typename T, int BYTES>
int launch_rows(RowsArgs k, int what, cudaStream_t st) {
  k.vecs = k.W / (BYTES / (int)sizeof(T));
  k.div_vecs = make_fastdiv((uint32_t)k.vecs);
  k.span = std::min(k.T, (0x7FFFFFFF - 1024) / k.vecs);
  if (k.span < 1) return fail(TP_EINVAL, "rows too long for a row move");
  // (four vectors a thread once the blocks, eight an SM, come in four rounds all the same)
  const long long vecs = (long long)k.span * k.vecs;
  k.turns = what == ROWS_COMBINE && vecs >= 4ll * 8 * 256 * device_info().sms ? 4 : 1;
  const dim3 blocks((unsigned)((vecs + 256 * k.turns - 1) / (256 * k.turns)), (unsigned)(((long long)k.T + k.span - 1) / k.span));
  if (blocks.y > 65535) return fail(TP_EINVAL, "too many elements for one row move");
  if (what == ROWS_DISPATCH)
    rows_dispatch_kernel<T, BYTES><<<blocks, 256, 0, st>>>(k);
  else if (what == ROWS_COMBINE)
    (k.k == 1   ? rows_combine_kernel<T, BYTES, 1>
     : k.k == 2 ? rows_combine_kernel<T, BYTES, 2>
     : k.k == 3 ? rows_combine_kernel<T, BYTES, 3>
                : rows_combine_kernel<T, BYTES, 4>)<<<blocks, 256, 0, st>>>(k);
  else
    (k.k == 1   ? launch_rows_backward<T, BYTES, 1>
     : k.k == 2 ? launch_rows_backward<T, BYTES, 2>
     : k.k == 3 ? launch_rows_backward<T, BYTES, 3>
                : launch_rows_backward<T, BYTES, 4>)(k, st);
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

int dispatch_rows(const tp_rows_args* a, int what, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  const RowsArgs k = rows_args(a);
  const int v = rows_vector(a);
  if (a->dtype == TP_DTYPE_BF16) {
    switch (v) {
      case 2: return launch_rows<__nv_bfloat16, 2>(k, what, st);
      case 4: return launch_rows<__nv_bfloat16, 4>(k, what, st);
      case 8: return launch_rows<__nv_bfloat16, 8>(k, what, st);
      default: return launch_rows<__nv_bfloat16, 16>(k, what, st);
    }
  }
  switch (v) {
    case 4: return launch_rows<float, 4>(k, what, st);
    case 8: return launch_rows<float, 8>(k, what, st);
    default: return launch_rows<float, 16>(k, what, st);
  }
}

// ------------------------------------------------------------------ ragged linear layers

// A (planes, rows, inner) tensor with rows at `ld` elements, in 128-byte swizzled boxes of box_inner x box_rows.
int make_map_ld(CUtensorMap* map, CUtensorMapDataType type, int size, const void* ptr, uint64_t inner, uint64_t rows,
                uint64_t planes, uint64_t ld, uint32_t box_inner, uint32_t box_rows) {
  auto enc = encode_fn();
  if (!enc) return fail(TP_EUNSUPPORTED, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {inner, rows, planes};
  cuuint64_t strides[2] = {ld * size, ld * size * rows};
  cuuint32_t box[3] = {box_inner, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, type, 3, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TP_EINVAL, "cuTensorMapEncodeTiled failed (%d) for dims %llu x %llu x %llu", (int)r,
                (unsigned long long)planes, (unsigned long long)rows, (unsigned long long)inner);
  return TP_OK;
}

// Scale tiles (atoms of 512 bytes, row tile by row tile) as rows of 256 bytes, in boxes of `rows` rows of `tiles` tiles.
int make_scale_map(CUtensorMap* map, const void* ptr, int atoms, long long row_tiles, int rows, int tiles) {
  auto enc = encode_fn();
  if (!enc) return fail(TP_EUNSUPPORTED, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {64, (cuuint64_t)atoms * 2, (cuuint64_t)row_tiles};
  cuuint64_t strides[2] = {256, (cuuint64_t)atoms * 512};
  cuuint32_t box[3] = {64, (cuuint32_t)rows, (cuuint32_t)tiles};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TP_EINVAL, "cuTensorMapEncodeTiled failed (%d) for scales", (int)r);
  return TP_OK;
}

constexpr int32_t MAX_WIDTH = 1 << 24;

// Columns of a tile: narrower ones while they still fit the SMs at once.  Two rounds of narrow tiles take longer than one of
// wide ones, which read less (bf16, tiles of 64 / 128 / 256 columns: 7 x 367 rows, 200 -> 531, 10.0 / 9.4 / 12.1 us;
// 4 x 512 rows, 2048 -> 1024, 28 / 18.6 / 21; 2048 -> 4096 85 / 55 / 40).
int tile_columns(long long row_tiles, int cols) {
  int bn = 256;
  while (bn > 64 && row_tiles * ((cols + bn / 2 - 1) / (bn / 2)) <= device_info().sms) bn /= 2;
  return bn;
}

int check_ragged(const tp_ragged_linear_args* a) {
  if (!a) return fail(TP_EINVAL, "null ragged linear arguments");
  if (a->P <= 0 || a->P > 65535 || a->max_in <= 0 || a->max_out <= 0 || a->max_in > MAX_WIDTH || a->max_out > MAX_WIDTH ||
      a->rows <= 0 || a->rows > ROUTE_MAX_PAIRS)
    return fail(TP_EINVAL, "a ragged linear layer needs 1 <= P <= 65535, widths > 0, 0 < rows <= 2^31 - 2^20 (got %d, %d, %d, %lld)",
                a->P, a->max_in, a->max_out, (long long)a->rows);
  if (a->dtype != TP_DTYPE_F32 && a->dtype != TP_DTYPE_BF16) return fail(TP_EINVAL, "bad ragged linear dtype");
  if (!a->offsets || !a->x || !a->w) return fail(TP_EINVAL, "null offsets, x or w");
  if (a->x_stride < a->max_in || a->w_stride < a->max_in) return fail(TP_EINVAL, "rows of x or w overlap");
  if (!aligned_to(4, {a->offsets, a->in_features, a->out_features, a->bias, a->dw, a->dbias}) ||
      !aligned_to(dtype_size(a->dtype), {a->x, a->w, a->y, a->dy, a->dx}))
    return fail(TP_EALIGN, "ragged linear data not aligned to its type");
  if (a->dtype == TP_DTYPE_BF16 && (!aligned16(a->x) || !aligned16(a->w) || a->x_stride % 8 || a->w_stride % 8))
    return fail(TP_EALIGN, "bf16 x and w need 16-byte aligned rows");
  return TP_OK;
}

RaggedProblem ragged_problem(const tp_ragged_linear_args* a) {
  RaggedProblem p{};
  p.P = a->P;
  p.R = (int)a->rows;
  p.in = a->max_in;
  p.out = a->max_out;
  p.offsets = a->offsets;
  p.in_f = a->in_features;
  p.out_f = a->out_features;
  return p;
}

// Launch of a kernel whose CTAs (or CTA pairs) go through tiles: as many as run at once.
template <auto* KERNEL, bool PAIR>
int persistent_launch(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, int threads, size_t smem, long long tiles,
                      cudaStream_t st) {
  int rc = allow_smem<KERNEL>(smem);
  if (rc) return rc;
  cfg->blockDim = dim3(threads);
  cfg->dynamicSmemBytes = smem;
  cfg->stream = st;
  int workers = device_info().sms;
  if constexpr (PAIR) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
    static std::atomic<int> pairs[64] = {};
    int dev = 0;
    TP_CUDA_TRY(cudaGetDevice(&dev));
    int n = pairs[dev].load(std::memory_order_relaxed);
    if (n == 0) {
      cfg->gridDim = dim3(2 * (workers / 2));
      TP_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, KERNEL, cfg));
      if (n <= 0) return fail(TP_EUNSUPPORTED, "no CTA pair of this kernel fits on the device");
      pairs[dev].store(n, std::memory_order_relaxed);
    }
    workers = n;
  }
  const int grid = (int)std::min<long long>(std::max<long long>(tiles, 1), workers);
  cfg->gridDim = dim3(PAIR ? 2 * grid : grid);
  return TP_OK;
}

template <int BN, int MODE, bool PAIR, bool F32>
int launch_ragged(const RaggedProblem& p, const CUtensorMap& ma, const CUtensorMap& mb, long long tiles, cudaStream_t st) {
  using Cfg = RaggedCfg<BN, MODE, PAIR, F32>;
  constexpr auto kern = ragged_gemm_kernel<BN, MODE, PAIR, F32>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  int rc = persistent_launch<kern, PAIR>(&cfg, attr, Cfg::THREADS, Cfg::SMEM_BYTES, tiles, st);
  if (rc) return rc;
  TP_PROF(MODE == RAGGED_FWD ? TP_PROF_FWD : MODE == RAGGED_DGRAD ? TP_PROF_DGRAD : TP_PROF_WGRAD, st);
  TP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ma, mb, p));
  return TP_OK;
}

// How a product is cut into tiles, from its sizes alone.
// (fp32: 128 columns, or pairs; with all of a block's parts in a stage 64 or 256 columns were never faster: 8 x 512 rows,
// 512 -> 512, 24 / 17 / 29 us, 12 x 340 rows, 100 -> 512, 11.5 / 10.4 / 14.8.)
struct RaggedPlan {
  bool pair;
  int bn, tile_m, splits;
};

RaggedPlan ragged_plan(int mode, bool f32, int P, int64_t R, int in, int out) {
  RaggedPlan plan{false, 256, 128, 1};
  const int cols = mode == RAGGED_DGRAD ? in : out;
  const long long used = std::min<long long>(P, R);
  const int sms = 148;
  // Pairs where their 256-row tiles are mostly full and there is at least one for each pair of SMs: members of 1024
  // rows on average (wgrad: input widths), since a member's last tile is half empty on average.  (8 members of 4096 x 4096:
  // 1024 rows each 191 us against 198, backward 428 against 467; 512 full ones 114 against 124; but 64 members of 1100 rows,
  // 1024 x 1024, 142 against 136.)
  const long long rows = mode == RAGGED_WGRAD ? in : R / P;
  const long long pair_tiles = (mode == RAGGED_WGRAD ? (long long)P * ((in + 255) / 256) : R / 256) * ((cols + 255) / 256);
  if (rows >= 1024 && pair_tiles >= sms / 2) {
    plan.pair = true;
    plan.tile_m = 256;
    return plan;
  }
  // tiles along the rows: every member that has rows ends in a partial one
  const long long m_tiles = mode == RAGGED_WGRAD ? (long long)P * ((in + 127) / 128) : std::max(used, R / 128 + used / 2);
  plan.bn = f32 ? 128 : tile_columns(m_tiles, cols);
  if (mode == RAGGED_WGRAD) {
    // parts of 512 rows at least, as many as the SMs take at once, 256 MB of results at most
    const long long tiles = m_tiles * ((cols + plan.bn - 1) / plan.bn);
    const long long most = std::max(1ll, (256ll << 20) / std::max(1ll, 4ll * P * in * out));
    plan.splits = (int)std::max(1ll, std::min({sms / tiles, (long long)R / P / 512, most, 64ll}));
  }
  return plan;
}

// One of the products: A and B with their row strides; fp32 operands as their parts, at a_part and b_part columns.
struct RaggedCall {
  RaggedProblem p;
  RaggedPlan plan;
  CUtensorMap ma, mb;
  long long most;  // tiles at most
  void* result;
};
long long ragged_tiles(int mode, const RaggedPlan& plan, int P, int64_t R, int in, int out) {
  const int cols = mode == RAGGED_DGRAD ? in : out;
  const long long n = (cols + plan.bn - 1) / plan.bn, m = (in + plan.tile_m - 1) / plan.tile_m;
  return mode == RAGGED_WGRAD ? (long long)P * m * n * plan.splits : ((long long)R / plan.tile_m + P + 2) * n;
}

template <int MODE, bool F32>
int ragged_call(RaggedCall& c, const RaggedProblem& problem, const RaggedPlan& plan, const void* a_ptr, long long a_ld,
                const void* b_ptr, long long b_ld, float* parts) {
  RaggedProblem& p = c.p;
  p = problem;
  c.plan = plan;
  const int cols = MODE == RAGGED_DGRAD ? p.in : p.out;  // columns of the result
  const int bn = plan.bn;
  p.n_tiles = (cols + bn - 1) / bn;
  p.m_tiles = (p.in + plan.tile_m - 1) / plan.tile_m;
  p.splits = plan.splits;
  p.c_vec = aligned16(p.c) && cols % (F32 ? 4 : 8) == 0;
  c.result = p.c;
  if (MODE == RAGGED_WGRAD && plan.splits > 1) p.c = parts;
  c.most = ragged_tiles(MODE, plan, p.P, p.R, p.in, p.out);
  if (c.most > 0x7FFFFFFFLL) return fail(TP_EINVAL, "too many tiles");
  const auto T = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // fp32: all three parts of a row are the map's columns
  const uint64_t in = F32 ? (uint64_t)(MODE == RAGGED_WGRAD ? a_ld : b_ld) : p.in, out = F32 ? (uint64_t)(MODE == RAGGED_DGRAD ? a_ld : b_ld) : p.out;
  int rc;
  if (MODE == RAGGED_FWD) {
    rc = make_map_ld(&c.ma, T, 2, a_ptr, F32 ? (uint64_t)a_ld : p.in, p.R, 1, a_ld, 64, 128);
    if (!rc) rc = make_map_ld(&c.mb, T, 2, b_ptr, in, p.out, p.P, b_ld, 64, plan.pair ? bn / 2 : bn);
  } else if (MODE == RAGGED_DGRAD) {
    rc = make_map_ld(&c.ma, T, 2, a_ptr, out, p.R, 1, a_ld, 64, 128);
    if (!rc) rc = make_map_ld(&c.mb, T, 2, b_ptr, in, p.out, p.P, b_ld, 64, 64);
  } else {
    rc = make_map_ld(&c.ma, T, 2, a_ptr, in, p.R, 1, a_ld, 64, 64);
    if (!rc) rc = make_map_ld(&c.mb, T, 2, b_ptr, out, p.R, 1, b_ld, 64, 64);
  }
  return rc;
}
int ragged_add_parts(const RaggedCall& c, cudaStream_t st) {
  if (c.plan.splits == 1) return TP_OK;
  const long long n = (long long)c.p.P * c.p.out * c.p.in;
  ragged_parts_kernel<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(static_cast<const float*>(c.p.c), static_cast<float*>(c.result),
                                                                  n, c.plan.splits);
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}
template <int MODE, bool F32>
int ragged_product(const RaggedProblem& p, const void* a_ptr, long long a_ld, const void* b_ptr, long long b_ld, float* parts,
                   cudaStream_t st) {
  RaggedCall c;
  int rc = ragged_call<MODE, F32>(c, p, ragged_plan(MODE, F32, p.P, p.R, p.in, p.out), a_ptr, a_ld, b_ptr, b_ld, parts);
  if (rc) return rc;
  if (c.plan.pair)
    rc = launch_ragged<256, MODE, true, F32>(c.p, c.ma, c.mb, c.most, st);
  else if (F32 || c.plan.bn == 128)
    rc = launch_ragged<128, MODE, false, F32>(c.p, c.ma, c.mb, c.most, st);
  else if constexpr (!F32)
    rc = c.plan.bn == 256 ? launch_ragged<256, MODE, false, false>(c.p, c.ma, c.mb, c.most, st)
                          : launch_ragged<64, MODE, false, false>(c.p, c.ma, c.mb, c.most, st);
  return rc || MODE != RAGGED_WGRAD ? rc : ragged_add_parts(c, st);
}

template <int BN, bool F32>
int launch_gradients(const RaggedCall& x, const RaggedCall& w, cudaStream_t st) {
  constexpr auto kern = ragged_gradients_kernel<BN, F32>;
  using W = RaggedCfg<BN, RAGGED_WGRAD, false, F32>;
  constexpr int smem = std::max(W::SMEM_BYTES, RaggedCfg<BN, RAGGED_DGRAD, false, F32>::SMEM_BYTES);
  int rc = allow_smem<kern>(smem);
  if (rc) return rc;
  TP_PROF(TP_PROF_WGRAD, st);
  kern<<<(unsigned)(x.most + w.most), W::THREADS, smem, st>>>(x.ma, x.mb, x.p, w.ma, w.mb, w.p, (int)x.most);
  TP_CUDA_TRY(cudaGetLastError());
  return ragged_add_parts(w, st);
}

// Both gradients, g (rows, out) and x (rows, in) with their row strides: in one launch where the tiles of both, of 64 or else
// 128 columns, fit the SMs at once (7 members, 2571 rows, 200 -> 531 bf16: 19 us one after the other, 12.2 together; 12 members, 4099 rows,
// 100 -> 512 fp32: 43, 22).
template <bool F32>
int ragged_gradients(const RaggedProblem& px, const void* g, long long g_ld, const void* w, long long w_ld, const RaggedProblem& pw,
                     const void* x, long long x_ld, float* parts, cudaStream_t st) {
  for (int bn = F32 ? 128 : 64; bn <= 128; bn *= 2) {
    RaggedPlan plan_x{false, bn, 128, 1}, plan_w = plan_x;
    const long long tiles_x = ragged_tiles(RAGGED_DGRAD, plan_x, px.P, px.R, px.in, px.out);
    const long long tiles_w = ragged_tiles(RAGGED_WGRAD, plan_w, px.P, px.R, px.in, px.out), sms = device_info().sms;
    if (tiles_x + tiles_w > sms) continue;
    // (the workspace holds the parts that the product alone would be split into)
    plan_w.splits = (int)std::min<long long>(ragged_plan(RAGGED_WGRAD, F32, px.P, px.R, px.in, px.out).splits, (sms - tiles_x) / tiles_w);
    RaggedCall cx, cw;
    int rc = ragged_call<RAGGED_DGRAD, F32>(cx, px, plan_x, g, g_ld, w, w_ld, nullptr);
    if (!rc) rc = ragged_call<RAGGED_WGRAD, F32>(cw, pw, plan_w, x, x_ld, g, g_ld, parts);
    if (rc) return rc;
    if constexpr (!F32)
      if (bn == 64) return launch_gradients<64, false>(cx, cw, st);
    return launch_gradients<128, F32>(cx, cw, st);
  }
  const int rc = ragged_product<RAGGED_DGRAD, F32>(px, g, g_ld, w, w_ld, nullptr, st);
  return rc ? rc : ragged_product<RAGGED_WGRAD, F32>(pw, x, x_ld, g, g_ld, parts, st);
}

int split_cols(int width) { return (width + 63) / 64 * 64; }
// Bytes of a matrix's three parts.
size_t split_bytes(long long rows, int width) { return (size_t)rows * split_cols(width) * 6; }

// The parts of up to three fp32 matrices.
struct Splits {
  SplitArgs k{};
  int count = 0;
  long long blocks = 1;
  __nv_bfloat16* add(const void* x, long long ld, long long rows, int width, void* out) {
    const int i = count++, cols = split_cols(width);
    k.x[i] = static_cast<const float*>(x);
    k.ld[i] = ld;
    k.rows[i] = rows;
    k.width[i] = width;
    k.cols[i] = cols;
    k.vec[i] = aligned16(x) && ld % 4 == 0;
    k.div[i] = make_fastdiv((uint32_t)(cols / 8));
    k.out[i] = static_cast<__nv_bfloat16*>(out);
    blocks = std::max(blocks, (rows * (cols / 8) + 255) / 256);
    return k.out[i];
  }
  int launch(cudaStream_t st) const {
    ragged_split_kernel<<<dim3((unsigned)std::min<long long>(blocks, 16 * 148), count), 256, 0, st>>>(k);
    TP_CUDA_TRY(cudaGetLastError());
    return TP_OK;
  }
};

// Columns of a block of the activation gradient: long pieces of each row where that leaves blocks enough (256 / 64 columns:
// 4080 rows of 512 4.9 / 5.4 us, 8192 of 512 5.6 / 8.5; 2569 of 531 10.7 / 6.3, 9001 of 190 14 / 6.7).
int ragged_strip(const tp_ragged_linear_args* a) { return a->rows * a->max_out >= (2ll << 20) && a->max_out >= 256 ? 256 : 64; }
// Shares of a member's rows in the bias gradient: about eight blocks an SM, 64 rows each at least (32768 rows of 4096: 9 shares
// 55 us with their sum, 4 65, one 91; 9001 rows of 190 to one member: 64 shares 11.4, 32 12, 16 17).
int ragged_shares(const tp_ragged_linear_args* a) {
  const long long strips = (a->max_out + ragged_strip(a) - 1) / ragged_strip(a);
  const long long want = 8ll * 148 / std::max(1ll, strips * a->P), most = a->rows / ((long long)a->P * 64);
  return (int)std::max(1ll, std::min({want, most, 64ll}));
}
// Columns between rows of the copy of g; 0: dy is taken as it is.
long long ragged_g_stride(const tp_ragged_linear_args* a) {
  if (a->dx == nullptr && a->dw == nullptr) return 0;
  if (a->relu) return (a->max_out + 7ll) / 8 * 8;
  if (a->dtype == TP_DTYPE_BF16 && (a->dy_stride % 8 || !aligned16(a->dy))) return (a->max_out + 7ll) / 8 * 8;
  return 0;
}
template <typename T, bool VEC, int C>
void launch_act_relu(const RaggedAct& k, dim3 grid, cudaStream_t st) {
  if (k.y)
    ragged_act_kernel<T, VEC, C, true><<<grid, 256, 0, st>>>(k);
  else
    ragged_act_kernel<T, VEC, C, false><<<grid, 256, 0, st>>>(k);
}
template <typename T>
void launch_act(const RaggedAct& k, bool vec, bool wide, dim3 grid, cudaStream_t st) {
  if (vec)
    wide ? launch_act_relu<T, true, 32>(k, grid, st) : launch_act_relu<T, true, 8>(k, grid, st);
  else
    wide ? launch_act_relu<T, false, 32>(k, grid, st) : launch_act_relu<T, false, 8>(k, grid, st);
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// The workspace.  Forward: the parts of fp32 x and w.  Backward: g, the shares' sums of g, the partial results of dw,
// the parts of fp32 g, x and w.
struct RaggedSpace {
  size_t shares, parts, g3, x3, w3, bytes;
};
RaggedSpace ragged_space(const tp_ragged_linear_args* a) {
  RaggedSpace s{};
  const bool f32 = a->dtype == TP_DTYPE_F32;
  if (a->dy) {
    s.shares = round256((size_t)a->rows * (size_t)ragged_g_stride(a) * dtype_size(a->dtype));
    s.parts = s.shares;
    if (a->dbias && ragged_shares(a) > 1) s.parts += round256((size_t)ragged_shares(a) * a->P * a->max_out * sizeof(float));
    s.g3 = s.parts;
    if (a->dw) {
      const int splits = ragged_plan(RAGGED_WGRAD, a->dtype == TP_DTYPE_F32, a->P, a->rows, a->max_in, a->max_out).splits;
      if (splits > 1) s.g3 += round256((size_t)splits * a->P * a->max_out * a->max_in * sizeof(float));
    }
  }
  s.x3 = s.g3 + (f32 && (a->dx || a->dw) ? round256(split_bytes(a->rows, a->max_out)) : 0);
  s.w3 = s.x3 + (f32 && (!a->dy || a->dw) ? round256(split_bytes(a->rows, a->max_in)) : 0);
  s.bytes = s.w3 + (f32 && (!a->dy || a->dx) ? split_bytes((long long)a->P * a->max_out, a->max_in) : 0);
  return s;
}

// ------------------------------------------------------------------ 4-bit rows

int check_fp4_groups(int32_t P, int32_t K, int32_t format, int64_t rows, const int32_t* offsets, bool shared) {
  if (P <= 0 || P > (1 << 20) || K <= 0 || K > MAX_WIDTH || rows <= 0 || rows >= (1ll << 31) - 256)
    return fail(TP_EINVAL, "4-bit rows need P, K > 0, 0 < rows < 2^31 - 256 (got %d, %d, %lld)", P, K, (long long)rows);
  if (format != TP_FP4_NV && format != TP_FP4_MX) return fail(TP_EINVAL, "bad 4-bit format %d", format);
  if (!offsets && !shared && rows % P) return fail(TP_EINVAL, "%lld rows are not %d equal groups", (long long)rows, P);
  if (!aligned_to(4, {offsets})) return fail(TP_EALIGN, "offsets not aligned to their type");
  return TP_OK;
}

long long fp4_row_tiles(const Fp4Groups& g) {
  return g.offsets ? g.rows / 128 + g.P : (long long)g.P * ((g.B + 127) / 128);
}

int check_fp4(const tp_fp4_args* a) {
  if (!a) return fail(TP_EINVAL, "null 4-bit row arguments");
  int rc = check_fp4_groups(a->P, a->K, a->format, a->rows, a->offsets, false);
  if (rc) return rc;
  if (!a->codes || !a->scales || !a->row_scale) return fail(TP_EINVAL, "null codes or scales");
  if (!aligned_to(16, {a->codes, a->scales}) || !aligned_to(4, {a->row_scale, a->n_features}) || !aligned_to(2, {a->values}))
    return fail(TP_EALIGN, "codes and scales need 16-byte boundaries");
  return TP_OK;
}

Fp4Groups fp4_groups(int32_t P, int64_t rows, const int32_t* offsets) {
  Fp4Groups g{};
  g.P = P;
  g.rows = rows;
  g.B = offsets ? 0 : (int)(rows / P);
  g.offsets = offsets;
  return g;
}

// The workspace of a 4-bit linear layer that quantises its rows: codes, scales, row scales.
struct Fp4Space {
  size_t scales, row_scale, bytes;
};
Fp4Space fp4_space(const tp_fp4_linear_args* a) {
  Fp4Space s{};
  s.scales = round256((size_t)a->rows * tp_fp4_pitch(a->K));
  const Fp4Groups g = fp4_groups(a->x_shared ? 1 : a->P, a->rows, a->offsets);
  s.row_scale = s.scales + (size_t)fp4_row_tiles(g) * tp_fp4_scale_tiles(a->K, a->format) * 512;
  s.bytes = s.row_scale + (size_t)a->rows * sizeof(float);
  return s;
}

Fp4Rows fp4_rows(const tp_fp4_args* a) {
  Fp4Rows r{};
  r.codes = a->codes;
  r.scales = a->scales;
  r.row_scale = a->row_scale;
  r.pitch = tp_fp4_pitch(a->K);
  r.atoms = tp_fp4_scale_tiles(a->K, a->format);
  return r;
}

// Few long rows go to a block each instead of a warp each, which takes a row's pieces one after the other and leaves most
// of the GPU idle: up to this many columns for each tile of 128 rows.
// mxfp4, a block / a warp a row: 1024 rows of 8192 bf16 8.6 / 12.9 us, 4096 of them 24.5 / 20.8; 128 rows of 2048 2.8 / 4.3,
// 1024 of them 6.1 / 5.2.  nvfp4 against the rows through shared memory: 128 rows of 8192 4.3 / 5.3, 512 of them 6.8 / 6.3.
// Values: 4096 rows of 8192 16.9 / 22.7, 1024 of 2048 3.9 / 6.1, 4096 of 1024 7.6 / 5.2.
constexpr long long FP4_COLUMNS_MX = 512, FP4_COLUMNS_NV = 4096, FP4_COLUMNS_VALUES = 256;

// nvfp4 of rows of at most 4 G vectors: groups of four rows through shared memory, 1024 threads an SM.
template <typename T, int G, bool ALIGNED>
int launch_stream(const Fp4QuantArgs& k, long long tiles, cudaStream_t st) {
  constexpr auto kern = fp4_quantize_stream_kernel<T, G, 4, ALIGNED>;
  constexpr size_t smem = (size_t)2 * 4 * 4 * G * 16;
  int rc = allow_smem<kern>(smem);
  if (rc) return rc;
  const long long groups = tiles * 32, most = (long long)device_info().sms * (256 / G);
  kern<<<(unsigned)std::min(groups, most), 4 * G, smem, st>>>(k, groups);
  return TP_OK;
}

template <typename T, int FORMAT, bool ALIGNED>
int launch_quantize(const Fp4QuantArgs& k, cudaStream_t st) {
  const long long tiles = fp4_row_tiles(k.groups);
  constexpr int E = 16 / (int)sizeof(T);
  const bool stream = FORMAT == FP4_NV && k.K <= 256 * 4 * E;
  const bool few = tiles * (stream ? FP4_COLUMNS_NV : FP4_COLUMNS_MX) <= k.K;
  if (tiles * 128 > 0x7FFFFFFFLL) return fail(TP_EINVAL, "too many rows");
  if (few) {
    fp4_quantize_rows_kernel<T, FORMAT, 256, 4, ALIGNED><<<(unsigned)(tiles * 128), 256, 0, st>>>(k);
    return TP_OK;
  }
  if constexpr (FORMAT == FP4_NV) {
    if (k.K <= 32 * 4 * E) return launch_stream<T, 32, ALIGNED>(k, tiles, st);
    if (k.K <= 64 * 4 * E) return launch_stream<T, 64, ALIGNED>(k, tiles, st);
    if (k.K <= 128 * 4 * E) return launch_stream<T, 128, ALIGNED>(k, tiles, st);
    if (stream) return launch_stream<T, 256, ALIGNED>(k, tiles, st);
  }
  fp4_quantize_rows_kernel<T, FORMAT, 32, 4, ALIGNED><<<(unsigned)(tiles * 32), 128, 0, st>>>(k);
  return TP_OK;
}
template <typename T>
int dispatch_quantize(const Fp4QuantArgs& k, bool nv, bool aligned, cudaStream_t st) {
  if (nv) return aligned ? launch_quantize<T, FP4_NV, true>(k, st) : launch_quantize<T, FP4_NV, false>(k, st);
  return aligned ? launch_quantize<T, FP4_MX, true>(k, st) : launch_quantize<T, FP4_MX, false>(k, st);
}

template <int FORMAT>
int launch_values(const Fp4ValuesArgs& k, bool vec, cudaStream_t st) {
  const long long tiles = fp4_row_tiles(k.groups);
  const bool few = tiles * FP4_COLUMNS_VALUES <= k.K;
  const long long blocks = tiles * (few ? 128 : 16);
  if (blocks > 0x7FFFFFFFLL) return fail(TP_EINVAL, "too many rows");
  auto kern = few ? (vec ? fp4_values_kernel<FORMAT, 256, true> : fp4_values_kernel<FORMAT, 256, false>)
                  : (vec ? fp4_values_kernel<FORMAT, 32, true> : fp4_values_kernel<FORMAT, 32, false>);
  kern<<<(unsigned)blocks, 256, 0, st>>>(k);
  return TP_OK;
}

template <int BN, int FORMAT, bool PAIR>
int launch_fp4(const Fp4Problem& p, const CUtensorMap (&m)[4], long long tiles, cudaStream_t st) {
  using Cfg = Fp4Cfg<BN, FORMAT, PAIR>;
  constexpr auto kern = fp4_gemm_kernel<BN, FORMAT, PAIR>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  int rc = persistent_launch<kern, PAIR>(&cfg, attr, Cfg::THREADS, Cfg::SMEM_BYTES, tiles, st);
  if (rc) return rc;
  TP_PROF(TP_PROF_FWD, st);
  TP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, m[0], m[1], m[2], m[3], p));
  return TP_OK;
}

template <int FORMAT>
int dispatch_fp4(const Fp4Problem& p, const CUtensorMap (&m)[4], bool pair, int bn, long long tiles, cudaStream_t st) {
  if (pair) return launch_fp4<256, FORMAT, true>(p, m, tiles, st);
  if (bn == 256) return launch_fp4<256, FORMAT, false>(p, m, tiles, st);
  if (bn == 128) return launch_fp4<128, FORMAT, false>(p, m, tiles, st);
  return launch_fp4<64, FORMAT, false>(p, m, tiles, st);
}

// ------------------------------------------------------------------ a few rows a group

// The kernel for few rows a member: up to 16, or 32 where the K loop is long, and up to 512 tiles of 128 outputs (each a CTA of
// its own, which finds its rows by looking through the groups).  It / the kernel for many rows, in bf16: one row through
// 8192 x 8192 37 / 61 us, 32 of them 42 / 49, 64 of them 44 / 49; 8 members of one row, 4096 x 4096, 60 / 63; 32 of one row,
// 1024 x 1024, 20 / 22; but 32 rows through 512 x 512 11 / 7.6, 64 members of one row, 1024 x 4096, 106 / 101, of 32 rows
// 122 / 104.  In 4 bits: 15 / 22.5, 17.9 / 18.6, 21 / 18.8; 23 / 26; 10.8 / 13.7; 8.6 / 5.9, 57 / 48.
bool few_rows(int32_t P, int64_t rows, int32_t K, int32_t N) {
  const int64_t used = std::min<int64_t>(P, rows);
  return P <= 1024 && rows <= (K >= 4096 ? 32 : 16) * used && used * ((N + 127) / 128) <= 512;
}

template <int KIND>
int launch_few(const FewArgs& f, const CUtensorMap& ma, const CUtensorMap& mb, cudaStream_t st) {
  using Cfg = FewCfg<KIND>;
  constexpr auto kern = few_rows_kernel<KIND>;
  int rc = allow_smem<kern>(Cfg::SMEM_BYTES);
  if (rc) return rc;
  const long long m_tiles = (f.N + 127) / 128, rows = f.groups.rows, used = std::min<long long>(f.groups.P, rows);
  // pieces of the rows: at most, and as many as are likely to hold rows
  constexpr int BN = Cfg::BN;
  const long long most = f.groups.offsets ? rows / BN + used + 2 : (long long)f.groups.P * ((f.groups.B + BN - 1) / BN);
  const long long likely = f.groups.offsets ? std::max(used, rows / BN) : most;
  // the K loop over a cluster while the SMs (two CTAs each) are not full and each part has four blocks (in 4 bits, clusters of
  // 1 / 2 / 4 / 8: one row, 8192 x 8192, 23.7 / 16.7 / 14.8 / 20.2 us; 2048 x 2048 9.6 / 8.0 / 7.1 / 6.7; 8 members of one row,
  // 1024 x 1024, 8.2 / 7.5 / 7.2 / 12.6)
  int split = 1;
  while (split < 8 && 2 * split * m_tiles * likely <= 2ll * device_info().sms && f.K >= 2 * split * 4 * Cfg::BK) split *= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)(m_tiles * split), (unsigned)most);
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  TP_PROF(TP_PROF_FWD, st);
  TP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, ma, mb, f, split));
  return TP_OK;
}

}  // namespace
}  // namespace tp

using namespace tp;

extern "C" {

size_t tp_route_workspace_size(int64_t rows, int32_t E, int32_t top_k) {
  if (rows <= 0 || E <= 0 || top_k <= 0 || route_plan(rows, top_k).blocks == 1) return 0;
  return ((size_t)route_plan(rows, top_k).blocks * (2 * (size_t)E + 1) + E + 1) * 4;
}

int tp_route_forward(const tp_route_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  int rc = check_route(a);
  if (rc) return rc;
  if (!a->position || !a->offsets || !a->importance) return fail(TP_EINVAL, "null routing output");
  const size_t need = tp_route_workspace_size(a->rows, a->E, a->top_k);
  if (need > 0 && (!a->workspace || a->workspace_bytes < need))
    return fail(TP_EINVAL, "routing workspace of %zu bytes is smaller than the %zu needed", a->workspace_bytes, need);
  RouteArgs k = route_args(a);
  k.counts = static_cast<int32_t*>(a->workspace);  // (unused with one block)
  if (need > 0) k.partial = reinterpret_cast<float*>(k.counts + (size_t)k.blocks * (a->E + 1));
  if (need > 0) k.totals = k.counts + (size_t)k.blocks * (2 * (size_t)a->E + 1);
  rc = a->dtype == TP_DTYPE_BF16 ? dispatch_route<__nv_bfloat16>(k, false, st) : dispatch_route<float>(k, false, st);
  if (rc) return rc;
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

int tp_route_backward(const tp_route_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  int rc = check_route(a);
  if (rc) return rc;
  if (!a->dlogits) return fail(TP_EINVAL, "null routing gradient");
  const RouteArgs k = route_args(a);
  rc = a->dtype == TP_DTYPE_BF16 ? dispatch_route<__nv_bfloat16>(k, true, st) : dispatch_route<float>(k, true, st);
  if (rc) return rc;
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

int tp_dispatch_rows(const tp_rows_args* a, void* stream) {
  int rc = check_rows(a);
  if (rc) return rc;
  if (!a->x || !a->out) return fail(TP_EINVAL, "null rows");
  tp_rows_args b = *a;
  b.dout = nullptr;
  b.dy = nullptr;
  return dispatch_rows(&b, ROWS_DISPATCH, stream);
}

int tp_combine_rows(const tp_rows_args* a, void* stream) {
  int rc = check_rows(a);
  if (rc) return rc;
  if (!a->x || !a->out) return fail(TP_EINVAL, "null rows");
  tp_rows_args b = *a;
  b.dout = nullptr;
  b.dy = nullptr;
  return dispatch_rows(&b, ROWS_COMBINE, stream);
}

int tp_combine_rows_backward(const tp_rows_args* a, void* stream) {
  int rc = check_rows(a);
  if (rc) return rc;
  if (!a->dout || (a->dweight && !a->x)) return fail(TP_EINVAL, "null rows");
  if (!a->dy && !a->dweight) return TP_OK;
  tp_rows_args b = *a;
  b.out = nullptr;
  if (!b.dweight) b.x = nullptr;
  return dispatch_rows(&b, ROWS_BACKWARD, stream);
}

int tp_align_rows(const void* x, int64_t x_stride, int64_t rows, int32_t cols, void* out, int64_t out_stride, void* stream) {
  if (!x || !out || rows <= 0 || rows >= (1ll << 31) || cols <= 0 || cols > MAX_WIDTH || (x_stride < cols && rows > 1) ||
      out_stride < cols || out_stride % 8 || out_stride > MAX_WIDTH)
    return fail(TP_EINVAL, "rows to align need 0 < rows < 2^31, 0 < cols <= the strides, out's a multiple of 8");
  if (!aligned_to(2, {x}) || !aligned16(out)) return fail(TP_EALIGN, "rows to align are not aligned to their type, or out not to 16 bytes");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  const int vecs = (int)(out_stride / 8), span = (int)std::min<int64_t>(rows, (0x7FFFFFFF - 1024) / vecs);
  const dim3 grid((unsigned)(((long long)span * vecs + 255) / 256), (unsigned)((rows + span - 1) / span));
  if (grid.y > 65535) return fail(TP_EINVAL, "too many elements to align");
  align_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), x_stride, (int)rows, cols, static_cast<uint4*>(out), vecs,
                                          make_fastdiv((uint32_t)vecs), span);
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

static int check_ragged_workspace(const tp_ragged_linear_args* a, size_t need) {
  if (need > 0 && (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace)))
    return fail(TP_EINVAL, "ragged linear workspace of %zu bytes is smaller than the %zu needed, or not aligned",
                a->workspace_bytes, need);
  return TP_OK;
}

size_t tp_ragged_linear_workspace_size(const tp_ragged_linear_args* a) {
  if (!a || a->P <= 0 || a->max_out <= 0 || a->rows <= 0) return 0;
  return ragged_space(a).bytes;
}

int tp_ragged_linear_forward(const tp_ragged_linear_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = check_ragged(a);
  if (rc) return rc;
  if (!a->y) return fail(TP_EINVAL, "null ragged linear output");
  RaggedProblem p = ragged_problem(a);
  p.bias = a->bias;
  p.relu = a->relu;
  p.c = a->y;
  if (a->dtype == TP_DTYPE_BF16 && few_rows(a->P, a->rows, a->max_in, a->max_out)) {
    FewArgs f{};
    f.groups = fp4_groups(a->P, a->rows, a->offsets);
    f.K = a->max_in;
    f.N = a->max_out;
    f.in_f = a->in_features;
    f.out_f = a->out_features;
    f.bias = a->bias;
    f.relu = a->relu;
    f.y = a->y;
    const auto T = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    CUtensorMap ma, mb;
    rc = make_map_ld(&ma, T, 2, a->w, a->max_in, a->max_out, a->P, a->w_stride, 64, 128);
    if (!rc) rc = make_map_ld(&mb, T, 2, a->x, a->max_in, a->rows, 1, a->x_stride, 64, FewCfg<FEW_BF16>::BN);
    return rc ? rc : launch_few<FEW_BF16>(f, ma, mb, st);
  }
  if (a->dtype == TP_DTYPE_BF16)
    return ragged_product<RAGGED_FWD, false>(p, a->x, a->x_stride, a->w, a->w_stride, nullptr, st);
  tp_ragged_linear_args fwd = *a;
  fwd.dy = nullptr;
  fwd.dx = nullptr;
  fwd.dw = nullptr;
  const RaggedSpace space = ragged_space(&fwd);
  rc = check_ragged_workspace(a, space.bytes);
  if (rc) return rc;
  char* ws = static_cast<char*>(a->workspace);
  Splits k;
  const void* x = k.add(a->x, a->x_stride, a->rows, a->max_in, ws + space.x3);
  const void* w = k.add(a->w, a->w_stride, (long long)a->P * a->max_out, a->max_in, ws + space.w3);
  rc = k.launch(st);
  if (rc) return rc;
  const int cols = split_cols(a->max_in);
  p.a_part = p.b_part = cols;
  return ragged_product<RAGGED_FWD, true>(p, x, 3 * cols, w, 3 * cols, nullptr, st);
}

int tp_ragged_linear_backward(const tp_ragged_linear_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = check_ragged(a);
  if (rc) return rc;
  if (!a->dy || (a->relu && !a->y)) return fail(TP_EINVAL, "null ragged linear gradient or output");
  if (a->dy_stride < a->max_out) return fail(TP_EINVAL, "rows of dy overlap");
  const RaggedSpace space = ragged_space(a);
  rc = check_ragged_workspace(a, space.bytes);
  if (rc) return rc;
  const bool bf16 = a->dtype == TP_DTYPE_BF16;
  float* parts = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + space.parts);
  const long long g_ld = ragged_g_stride(a);
  const void* g = g_ld ? a->workspace : a->dy;
  const long long ld = g_ld ? g_ld : a->dy_stride;
  if (g_ld || a->dbias) {
    RaggedAct k{};
    k.P = a->P;
    k.R = (int)a->rows;
    k.N = a->max_out;
    k.S = ragged_shares(a);
    k.offsets = a->offsets;
    k.out_f = a->out_features;
    k.dy = a->dy;
    k.dy_ld = a->dy_stride;
    k.y = a->relu ? a->y : nullptr;
    k.g = g_ld ? a->workspace : nullptr;
    k.g_ld = g_ld;
    k.db = a->dbias;
    k.partial = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + space.shares);
    TP_PROF(TP_PROF_ACT_BACKWARD, st);
    const bool wide = ragged_strip(a) == 256;
    const dim3 grid((a->max_out + ragged_strip(a) - 1) / ragged_strip(a), a->P, k.S);
    const size_t size = dtype_size(a->dtype);
    const bool vec = a->max_out % 8 == 0 && aligned16(a->dy) && aligned16(k.y) && a->dy_stride * size % 16 == 0;
    if (bf16)
      launch_act<__nv_bfloat16>(k, vec, wide, grid, st);
    else
      launch_act<float>(k, vec, wide, grid, st);
    if (a->dbias && k.S > 1)
      ragged_bias_kernel<<<(unsigned)(((long long)a->P * a->max_out + 255) / 256), 256, 0, st>>>(k);
    TP_CUDA_TRY(cudaGetLastError());
  }
  RaggedProblem p = ragged_problem(a), q = p;
  p.c = a->dx;
  q.c = a->dw;
  if (!a->dx && !a->dw) return TP_OK;
  if (bf16) {
    if (a->dx && a->dw) return ragged_gradients<false>(p, g, ld, a->w, a->w_stride, q, a->x, a->x_stride, parts, st);
    return a->dx ? ragged_product<RAGGED_DGRAD, false>(p, g, ld, a->w, a->w_stride, nullptr, st)
                 : ragged_product<RAGGED_WGRAD, false>(q, a->x, a->x_stride, g, ld, parts, st);
  }
  char* ws = static_cast<char*>(a->workspace);
  const int gc = split_cols(a->max_out), xc = split_cols(a->max_in);
  Splits k;
  const void* g3 = k.add(g, ld, a->rows, a->max_out, ws + space.g3);
  const void* x3 = a->dw ? k.add(a->x, a->x_stride, a->rows, a->max_in, ws + space.x3) : nullptr;
  const void* w3 = a->dx ? k.add(a->w, a->w_stride, (long long)a->P * a->max_out, a->max_in, ws + space.w3) : nullptr;
  rc = k.launch(st);
  if (rc) return rc;
  p.a_part = q.b_part = gc;
  p.b_part = q.a_part = xc;
  if (a->dx && a->dw) return ragged_gradients<true>(p, g3, 3 * gc, w3, 3 * xc, q, x3, 3 * xc, parts, st);
  return a->dx ? ragged_product<RAGGED_DGRAD, true>(p, g3, 3 * gc, w3, 3 * xc, nullptr, st)
               : ragged_product<RAGGED_WGRAD, true>(q, x3, 3 * xc, g3, 3 * gc, parts, st);
}

int32_t tp_fp4_pitch(int32_t K) { return (K + 31) / 32 * 16; }
int32_t tp_fp4_scale_tiles(int32_t K, int32_t format) { return (K + 255) / 256 * (format == TP_FP4_MX ? 2 : 4); }

int tp_fp4_quantize(const tp_fp4_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  int rc = check_fp4(a);
  if (rc) return rc;
  if (!a->x || (a->dtype != TP_DTYPE_F32 && a->dtype != TP_DTYPE_BF16)) return fail(TP_EINVAL, "null x or bad dtype");
  if (a->x_stride < a->K && a->rows > 1) return fail(TP_EINVAL, "rows of x overlap");
  if (!aligned_to(dtype_size(a->dtype), {a->x})) return fail(TP_EALIGN, "x not aligned to its type");
  Fp4QuantArgs k{};
  k.groups = fp4_groups(a->P, a->rows, a->offsets);
  k.K = a->K;
  k.x = a->x;
  k.ld = a->x_stride;
  k.n_features = a->n_features;
  k.out = fp4_rows(a);
  const size_t size = dtype_size(a->dtype);
  const bool vec = aligned16(a->x) && a->x_stride * size % 16 == 0, nv = a->format == TP_FP4_NV;
  rc = a->dtype == TP_DTYPE_BF16 ? dispatch_quantize<__nv_bfloat16>(k, nv, vec, st) : dispatch_quantize<float>(k, nv, vec, st);
  if (rc) return rc;
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

int tp_fp4_values(const tp_fp4_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  TP_PROF(TP_PROF_OTHER, st);
  int rc = check_fp4(a);
  if (rc) return rc;
  if (!a->values) return fail(TP_EINVAL, "null values");
  Fp4ValuesArgs k{};
  k.groups = fp4_groups(a->P, a->rows, a->offsets);
  k.K = a->K;
  k.in = fp4_rows(a);
  k.out = static_cast<__nv_bfloat16*>(a->values);
  const bool vec = aligned16(a->values) && a->K % 8 == 0;
  rc = a->format == TP_FP4_NV ? launch_values<FP4_NV>(k, vec, st) : launch_values<FP4_MX>(k, vec, st);
  if (rc) return rc;
  TP_CUDA_TRY(cudaGetLastError());
  return TP_OK;
}

size_t tp_fp4_linear_workspace_size(const tp_fp4_linear_args* a) {
  if (!a || !a->x || a->P <= 0 || a->K <= 0 || a->rows <= 0) return 0;
  return fp4_space(a).bytes;
}

int tp_fp4_linear_forward(const tp_fp4_linear_args* a, void* stream) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!a) return fail(TP_EINVAL, "null 4-bit linear arguments");
  int rc = check_fp4_groups(a->P, a->K, a->format, a->rows, a->offsets, a->x_shared != 0);
  if (rc) return rc;
  if (a->N <= 0 || a->N > MAX_WIDTH) return fail(TP_EINVAL, "a 4-bit linear layer needs N > 0 (got %d)", a->N);
  if (a->x_shared && a->offsets) return fail(TP_EINVAL, "shared rows have no offsets");
  if (a->x_shared && a->rows * a->P >= (1ll << 31) - 256) return fail(TP_EINVAL, "too many rows of y");
  if (a->dtype != TP_DTYPE_F32 && a->dtype != TP_DTYPE_BF16) return fail(TP_EINVAL, "bad 4-bit linear dtype");
  tp_fp4_linear_args q = *a;
  if (a->x) {
    const Fp4Space space = fp4_space(a);
    if (!a->workspace || a->workspace_bytes < space.bytes || !aligned16(a->workspace))
      return fail(TP_EINVAL, "4-bit linear workspace of %zu bytes is smaller than the %zu needed, or not aligned",
                  a->workspace_bytes, space.bytes);
    uint8_t* ws = static_cast<uint8_t*>(a->workspace);
    q.x_codes = ws;
    q.x_scales = ws + space.scales;
    q.x_row_scale = reinterpret_cast<const float*>(ws + space.row_scale);
    a = &q;
  }
  if (!a->x_codes || !a->x_scales || !a->x_row_scale || !a->w_codes || !a->w_scales || !a->w_row_scale || !a->y)
    return fail(TP_EINVAL, "null 4-bit linear operand or output");
  if (!aligned_to(16, {a->x_codes, a->x_scales, a->w_codes, a->w_scales}) ||
      !aligned_to(4, {a->x_row_scale, a->w_row_scale, a->bias, a->in_features, a->out_features}) ||
      !aligned_to(dtype_size(a->dtype), {a->y}))
    return fail(TP_EALIGN, "codes and scales need 16-byte boundaries");
  if (a->x) {
    tp_fp4_args x{};
    x.P = a->x_shared ? 1 : a->P;
    x.K = a->K;
    x.format = a->format;
    x.dtype = a->dtype;
    x.rows = a->rows;
    x.offsets = a->offsets;
    x.n_features = a->in_features;
    x.x = a->x;
    x.x_stride = a->x_stride;
    x.codes = const_cast<uint8_t*>(a->x_codes);
    x.scales = const_cast<uint8_t*>(a->x_scales);
    x.row_scale = const_cast<float*>(a->x_row_scale);
    rc = tp_fp4_quantize(&x, stream);
    if (rc) return rc;
  }
  Fp4Problem p{};
  p.groups = fp4_groups(a->P, a->x_shared ? a->rows * a->P : a->rows, a->offsets);
  p.x_shared = a->x_shared;
  p.K = a->K;
  p.N = a->N;
  p.in_f = a->in_features;
  p.out_f = a->out_features;
  p.x_row = a->x_row_scale;
  p.w_row = a->w_row_scale;
  const int atoms = tp_fp4_scale_tiles(a->K, a->format);
  p.bias = a->bias;
  p.relu = a->relu;
  p.y = a->y;
  p.y_f32 = a->dtype == TP_DTYPE_F32;
  p.y_vec = aligned16(a->y) && (long long)a->N * dtype_size(a->dtype) % 16 == 0;
  const long long rows = p.groups.rows;
  const int pitch = tp_fp4_pitch(a->K);
  const auto T = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  CUtensorMap ma, mb;
  if (few_rows(a->P, rows, a->K, a->N)) {
    FewArgs f{};
    f.groups = p.groups;
    f.x_shared = a->x_shared;
    f.K = a->K;
    f.N = a->N;
    f.in_f = a->in_features;
    f.out_f = a->out_features;
    f.bias = a->bias;
    f.relu = a->relu;
    f.y = a->y;
    f.y_f32 = p.y_f32;
    f.x_scales = a->x_scales;
    f.x_row = a->x_row_scale;
    f.w_scales = a->w_scales;
    f.w_row = a->w_row_scale;
    f.atoms = atoms;
    rc = make_map_ld(&ma, T, 1, a->w_codes, pitch, a->N, a->P, pitch, 128, 128);
    if (!rc) rc = make_map_ld(&mb, T, 1, a->x_codes, pitch, a->rows, 1, pitch, 128, FewCfg<FEW_NV>::BN);
    if (rc) return rc;
    return a->format == TP_FP4_NV ? launch_few<FEW_NV>(f, ma, mb, st) : launch_few<FEW_MX>(f, ma, mb, st);
  }
  const long long m_tiles = p.groups.offsets ? std::max<long long>(std::min<long long>(a->P, rows), rows / 128 + std::min<long long>(a->P, rows) / 2)
                                             : (long long)a->P * ((p.groups.B + 127) / 128);
  // Pairs where their 256-row tiles are mostly full (half a tile of a ragged member is not) and every pair of SMs has one:
  // 4 x 512 rows, 8192 x 8192, 84 us against 102; 16 x 700, 2048 x 2048, 47 against 50; 16 x 256 of them 24.5 against 24.9.
  const bool pair = rows / a->P >= 512 && rows / 256 * ((a->N + 255) / 256) >= device_info().sms / 2;
  const int bn = pair ? 256 : tile_columns(m_tiles, a->N);
  p.n_tiles = (a->N + bn - 1) / bn;
  const long long most = (p.groups.offsets ? rows / 128 + a->P + 2 : m_tiles) * p.n_tiles;
  if (most > 0x7FFFFFFFLL) return fail(TP_EINVAL, "too many tiles");
  CUtensorMap m[4];
  rc = make_map_ld(&m[0], T, 1, a->x_codes, pitch, a->rows, 1, pitch, 128, 128);
  if (!rc) rc = make_map_ld(&m[1], T, 1, a->w_codes, pitch, a->N, a->P, pitch, 128, pair ? 128 : bn);
  // a stage's scales: two or four tiles of 512 bytes as rows of 256, of one or two tiles of 128 rows
  const long long x_tiles = a->x_shared ? (a->rows + 127) / 128 : fp4_row_tiles(p.groups);
  const int step = a->format == TP_FP4_NV ? 8 : 4;
  if (!rc) rc = make_scale_map(&m[2], a->x_scales, atoms, x_tiles, step, 1);
  if (!rc) rc = make_scale_map(&m[3], a->w_scales, atoms, (long long)a->P * ((a->N + 127) / 128), step, bn == 256 ? 2 : 1);
  if (rc) return rc;
  return a->format == TP_FP4_NV ? dispatch_fp4<FP4_NV>(p, m, pair, bn, most, st) : dispatch_fp4<FP4_MX>(p, m, pair, bn, most, st);
}

}  // extern "C"
