// What the TorchScript bindings (torch_ops.cpp, feature_ops.cpp) share: checks of
// tensors, the current device, status codes as exceptions.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include "../../include/pca_neighbors.h"

namespace {

#define PCA_CHECK_GPU(x)                                                       \
  TORCH_CHECK((x).device().is_cuda(), #x " must be CUDA tensor")
#define PCA_CHECK_CONTIGUOUS(x)                                                \
  TORCH_CHECK((x).is_contiguous(), #x " must be contiguous")
#define PCA_CHECK_INPUT(cond) TORCH_CHECK(cond, "Input mismatch")

inline int dtype_code(const at::Tensor &x) {
  switch (x.scalar_type()) {
  case at::kFloat:
    return PCA_F32;
  case at::kDouble:
    return PCA_F64;
  case at::kHalf:
    return PCA_F16;
  case at::kBFloat16:
    return PCA_BF16;
  default:
    TORCH_CHECK(false, "unsupported element type ", x.scalar_type());
  }
}

// Restores the previously current device when it goes out of scope
// (the reference calls c10::cuda::MaybeSetDevice, knn_cuda.cu:116).
struct DeviceScope {
  int previous = -1;
  explicit DeviceScope(int device) {
    TORCH_CHECK(hipGetDevice(&previous) == hipSuccess, "hipGetDevice failed");
    if (previous != device) {
      TORCH_CHECK(hipSetDevice(device) == hipSuccess, "hipSetDevice failed");
    } else {
      previous = -1;
    }
  }
  ~DeviceScope() {
    if (previous >= 0)
      (void)hipSetDevice(previous);
  }
};

inline void check_status(int status) {
  if (status == PCA_OK)
    return;
  const char *detail = pca_last_error();
  TORCH_CHECK(false, (detail && detail[0]) ? detail
                                           : pca_status_string(status));
}

} // namespace
