// mr_host.h — what the host sides of the entry points share.
#pragma once

#include "mr_common.cuh"

#include <new>

namespace mr {

// No C++ exception leaves the C ABI: what building a message may throw is an
// allocation failure.
template <typename F>
inline mr_status guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return MR_ERR_OUT_OF_MEMORY;
  } catch (...) {
    return MR_ERR_INVALID_ARGUMENT;
  }
}

// The context's device is current while this lives; the caller's is afterwards.
struct DeviceScope {
  int prev = -1;
  cudaError_t err;
  explicit DeviceScope(const mr_ctx* ctx) {
    int cur = -1;
    err = cudaGetDevice(&cur);
    if (err == cudaSuccess && cur != ctx->device) {
      err = cudaSetDevice(ctx->device);
      prev = cur;
    }
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

// Sets a kernel's attributes the first time a context launches it.
enum KernelAttr : unsigned {
  kAttrSort = 1u,
  kAttrProduct = 2u  // and the next three bits: mxmm_kernel's instances
};
template <typename F>
inline cudaError_t attrs_once(mr_ctx* ctx, unsigned bit, F&& set) {
  if (ctx->kernel_attrs & bit) return cudaSuccess;
  const cudaError_t e = set();
  if (e == cudaSuccess) ctx->kernel_attrs |= bit;
  return e;
}

// The shape and pointers of sorted tokens (mr_sort.cu).
mr_status check_plan(mr_ctx* ctx, const mr_sorted* s);

inline uint64_t addr(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace mr
