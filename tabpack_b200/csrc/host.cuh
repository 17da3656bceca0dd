// Host-side helpers that the library's translation units share: errors, optional launch timing, device
// properties, tensor maps, alignment checks.
#pragma once

#include <cudaTypedefs.h>

#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <mutex>
#include <string>
#include <vector>

#include "common.cuh"

namespace tp {

inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

inline int cuda_fail(cudaError_t e, const char* what) {
  return fail(TP_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}

#define TP_CUDA_TRY(expr)                           \
  do {                                              \
    cudaError_t e_ = (expr);                        \
    if (e_ != cudaSuccess) return cuda_fail(e_, #expr); \
  } while (0)

// ---- optional per-launch timing (tp_profile_start / tp_profile_stop) -----------------
// Off by default (one relaxed atomic load per launch).  When on, each kernel launch (or, for
// entry points without a GEMM inside, each call) is bracketed by two CUDA events taken from a
// pool that tp_profile_start creates on the current device; tp_profile_stop waits for them and
// adds up the elapsed time per kernel family.
inline std::atomic<int> g_prof_on{0};
inline std::mutex g_prof_mu;
inline std::vector<cudaEvent_t> g_prof_events;  // two per slot
inline std::vector<int> g_prof_kind;            // family of each slot
inline int g_prof_used = 0;
inline int g_prof_dropped = 0;

struct ProfScope {
  cudaStream_t st;
  int slot = -1;
  ProfScope(int kind, cudaStream_t s) : st(s) {
    if (!g_prof_on.load(std::memory_order_relaxed)) return;
    std::lock_guard<std::mutex> lk(g_prof_mu);
    if (g_prof_used >= (int)g_prof_kind.size()) {
      ++g_prof_dropped;
      return;
    }
    slot = g_prof_used++;
    g_prof_kind[slot] = kind;
    cudaEventRecord(g_prof_events[2 * slot], st);
  }
  ~ProfScope() {
    if (slot >= 0) cudaEventRecord(g_prof_events[2 * slot + 1], st);
  }
  ProfScope(const ProfScope&) = delete;
  ProfScope& operator=(const ProfScope&) = delete;
};

#define TP_PROF_CAT2(a, b) a##b
#define TP_PROF_CAT(a, b) TP_PROF_CAT2(a, b)
#define TP_PROF(kind, stream) ProfScope TP_PROF_CAT(prof_scope_, __LINE__)((kind), (stream))

struct DeviceInfo {
  int sms = 0;
  int major = 0, minor = 0;
};

inline DeviceInfo device_info() {
  static std::mutex mu;
  static DeviceInfo cache[64];
  static bool have[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  if (dev >= 0 && dev < 64 && !have[dev]) {
    cudaDeviceGetAttribute(&cache[dev].sms, cudaDevAttrMultiProcessorCount, dev);
    cudaDeviceGetAttribute(&cache[dev].major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&cache[dev].minor, cudaDevAttrComputeCapabilityMinor, dev);
    have[dev] = true;
  }
  return (dev >= 0 && dev < 64) ? cache[dev] : DeviceInfo{};
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// bf16 tensor (planes, rows, inner) with 128-byte swizzled boxes (box_inner x box_rows x 1).
inline int make_map(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t rows, uint64_t planes, uint32_t box_inner,
             uint32_t box_rows) {
  auto enc = encode_fn();
  if (!enc) return fail(TP_EUNSUPPORTED, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[3] = {inner, rows, planes};
  cuuint64_t strides[2] = {inner * 2, inner * rows * 2};
  cuuint32_t box[3] = {box_inner, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TP_EINVAL, "cuTensorMapEncodeTiled failed (%d) for dims %llu x %llu x %llu", (int)r,
                (unsigned long long)planes, (unsigned long long)rows, (unsigned long long)inner);
  return TP_OK;
}

// 2-D map over a (rows, inner) bf16 table for TMA gather4: a box of 64 columns x 1 row (gather4
// loads take one-row boxes), 128-byte swizzle like the tiled operand maps.
inline int make_gather_map(CUtensorMap* map, const void* ptr, uint64_t inner, uint64_t rows) {
  auto enc = encode_fn();
  if (!enc) return fail(TP_EUNSUPPORTED, "cuTensorMapEncodeTiled is unavailable");
  cuuint64_t dims[2] = {inner, rows};
  cuuint64_t strides[1] = {inner * 2};
  cuuint32_t box[2] = {64, 1};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(TP_EINVAL, "cuTensorMapEncodeTiled failed (%d) for a %llu x %llu gather table", (int)r,
                (unsigned long long)rows, (unsigned long long)inner);
  return TP_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// All of them (or null) on boundaries of `size` bytes, a power of two.
inline bool aligned_to(size_t size, std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & (size - 1)) == 0;
}
inline size_t dtype_size(int dtype) { return dtype == TP_DTYPE_BF16 ? 2 : 4; }

}  // namespace tp
