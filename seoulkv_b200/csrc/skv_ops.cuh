// skv_ops.cuh -- host side shared by the stand-alone operators (rotary, tree
// attention, accumulated weights, eviction): errors, the current device and
// kernel launches that may start before the kernel ahead of them has ended.
#pragma once
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "../../include/seoulkv_b200.h"

namespace skv {

void set_last_error(const std::string &msg);

// Sets skv_last_error() and returns `code`; nothing is thrown through the C
// entries (a message that cannot be stored is dropped).
inline int op_fail(int code, const char *fmt, ...) noexcept {
  char buf[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  try {
    set_last_error(buf);
  } catch (...) {
  }
  return code;
}

inline int op_cuda(cudaError_t e, const char *what) noexcept {
  return e == cudaSuccess ? SKV_OK : op_fail(SKV_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Makes `device` current for one call and restores the caller's afterwards.
class DeviceScope {
 public:
  explicit DeviceScope(int device) noexcept {
    err_ = cudaGetDevice(&old_);
    if (err_ == cudaSuccess && device != old_) {
      err_ = cudaSetDevice(device);
      changed_ = err_ == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(old_);
  }
  DeviceScope(const DeviceScope &) = delete;
  DeviceScope &operator=(const DeviceScope &) = delete;
  cudaError_t error() const { return err_; }

 private:
  int old_ = 0;
  bool changed_ = false;
  cudaError_t err_;
};

// Strides as the kernels take them: 0 for a dimension of one element (its own
// stride means nothing).
inline void op_strides(int64_t *to, const int64_t *from, const int64_t *size, int n) noexcept {
  for (int i = 0; i < n; ++i) to[i] = size[i] == 1 ? 0 : from[i];
}

// SMs of a device, asked once.
inline int sm_count(int64_t device, int *sms) noexcept {
  static int known[64];
  if (device < 0 || device >= 64) return op_fail(SKV_E_INVALID, "device ordinal out of range");
  int n = __atomic_load_n(&known[device], __ATOMIC_RELAXED);
  if (!n) {
    if (int rc = op_cuda(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, (int)device), "device attribute")) return rc;
    __atomic_store_n(&known[device], n, __ATOMIC_RELAXED);
  }
  *sms = n;
  return SKV_OK;
}

// Dynamic shared memory of a kernel (`set`: one flag per device and kernel), raised once.
inline int op_shared_memory(const void *kernel, int bytes, int device, bool *set) noexcept {
  if (__atomic_load_n(&set[device], __ATOMIC_RELAXED)) return SKV_OK;
  if (int rc = op_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "shared memory size"))
    return rc;
  __atomic_store_n(&set[device], true, __ATOMIC_RELAXED);
  return SKV_OK;
}

// Launch; the kernel's blocks may be placed while the kernel before it on the
// stream still runs, which hides its launch and its prologue.
// That holds once every block of the kernel before has called
// grid_dependency_release() or ended; a kernel that never does (any that is
// not of these operators) ends first.  Such a kernel's threads call
// grid_dependency_wait() before they read or write global memory: it returns
// when the kernel before has ended, and with it all that were before that.
template <typename... P, typename... A>
inline cudaError_t op_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, unsigned cluster,
                             A &&...args) noexcept {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n++].val.programmaticStreamSerializationAllowed = 1;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_release() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace skv
