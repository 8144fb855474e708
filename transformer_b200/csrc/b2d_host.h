// b2d_host.h — host helpers shared by the library's translation units.
#pragma once

#include <cuda_runtime.h>

#include <utility>

#include "../../include/b2d.h"

namespace b2d {

// Keeps the text of a failing CUDA call for b2d_cuda_error (this thread) and
// returns the status it maps to.
b2d_status cuda_failed(cudaError_t e, const char* what);

// Makes `device` current for a call and restores the caller's device after it.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    err_ = cudaGetDevice(&prev_);
    if (err_ == cudaSuccess && prev_ != device) {
      err_ = cudaSetDevice(device);
      changed_ = err_ == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t error() const { return err_; }

 private:
  int prev_ = 0;
  bool changed_ = false;
  cudaError_t err_ = cudaSuccess;
};

// Launch with an optional programmatic dependency on the stream's previous
// kernel (the kernel calls griddepcontrol.wait before it reads that one's output).
template <class... KArgs, class... Args>
cudaError_t launch(void (*k)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl,
                   Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, std::forward<Args>(args)...);
}

}  // namespace b2d
