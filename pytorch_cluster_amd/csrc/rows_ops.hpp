// norm_rotate and lookup: what their kernels (norm_rotate.hip, lookup.hip) and the C
// ABI (features_capi.hip) share.
#pragma once

#include "attention.hpp"

namespace pca {

// Leaves the text that pca_last_error() returns; returns `status` (capi.hip).
int fail(int status, const char *fmt, ...);

struct NormRotateSide {
  HeadRows x, dout;              // dout: backward
  const void *weight = nullptr;  // [d] or NULL
  void *out = nullptr;           // [rows, heads, d], dense; backward: dx
  void *dweight = nullptr;       // [d] or NULL
  int heads = 0;
};

struct NormRotateCall {
  NormRotateSide side[2];        // queries, keys (heads 0: none)
  const float *pos = nullptr;    // [rows, axes]
  const float *freq = nullptr;   // [axes, rotated]
  int rows = 0, d = 0, axes = 0, rotated = 0;
  float eps = 0.f;
  int weight_dtype = 0;
  float *part = nullptr;         // backward: [blocks, 2, d]
};

hipError_t norm_rotate_forward(const NormRotateCall &c, int dtype,
                               hipStream_t stream);
size_t norm_rotate_workspace_bytes(int64_t rows, int d);
hipError_t norm_rotate_backward(NormRotateCall c, int dtype, void *workspace,
                                hipStream_t stream);

struct LookupCall {
  const void *rows = nullptr;  // forward: the table; backward: the gradient rows
  const void *index = nullptr; // int32 or int64
  bool wide_index = true;
  int64_t table = 0, entries = 0, width = 0;
  float scale = 1.f;
  void *out = nullptr;
};

hipError_t lookup_forward(const LookupCall &c, int dtype, hipStream_t stream);
size_t lookup_workspace_bytes(int64_t table, int64_t entries, int64_t width);
hipError_t lookup_backward(const LookupCall &c, int dtype, void *workspace,
                           hipStream_t stream);

} // namespace pca
