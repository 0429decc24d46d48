// What the attention kernels (attention_impl.hpp), their dispatch (attention.hip) and
// the C ABI (features_capi.hip) share.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace pca {

// One side of an attention: [rows, heads, d] elements, the last dimension dense.
struct HeadRows {
  const void *data = nullptr;
  int64_t row = 0, head = 0; // strides in elements
  bool vec = false; // every row starts on 16 bytes and is a multiple of 16 long
};

struct AttentionCall {
  HeadRows q, k, v;
  const int2 *spans_q = nullptr; // rows of k that belong to a row of q: [begin,
                                 // end) ([nq]; NULL: all of them)
  const int2 *spans_k = nullptr; // the same for a row of k ([nk])
  const float *pos_q = nullptr, *pos_k = nullptr; // [nq, axes], [nk, axes]
  const float *slope = nullptr;                   // [hq]; NULL: no bias
  int axes = 0;
  int nq = 0, nk = 0, hq = 0, hk = 0, d = 0;
  float scale = 1.f, cap = 0.f;
  float under_tanh = 0.f; // with a cap: what a product is multiplied by for exp2 in
                          // tanh, 2 log2 e scale / cap (set_cap)

  void *out = nullptr;  // [nq, hq, d], dense
  void *rest = nullptr; // the same: what rounding took off out; or NULL (backward:
                        // read)
  float *lse = nullptr; // [hq, nq]: log2 of the sum of exp2 of the scores (in
                        // units of log 2); +inf for a row without keys

  // backward
  const void *out_in = nullptr;
  HeadRows dout;
  void *dq = nullptr, *dk = nullptr, *dv = nullptr; // dense
  // from the kernel of dq to that of dk and dv: -delta and what the scores are
  // relative to ([hq, nq]), -slope log2 e ([hq])
  float *minus_delta = nullptr, *base = nullptr, *minus_slope = nullptr;

  // the looped side cut into up to `splits` pieces that meet in a kernel of their own
  int splits = 1;
  int rows = 0;             // owned rows of a workgroup
  int *pieces = nullptr;    // [hk, tiles of owned rows]: in use; 1: the result is
                            // written already
  float *part = nullptr;    // forward, dq: [splits, nq, hq, d]; dk, dv:
                            // [splits, 2, nk, hk, d]
  float *part_ml = nullptr; // forward: [splits, nq, hq, 2]
};

// Which of the kernels of a pass runs (owned rows of a workgroup), and in how many
// pieces.
struct AttentionPlan {
  int rows = 128;
  int splits = 1;
};

// One per element type (0 fp32, 2 fp16, 3 bf16: pca_dtype) and width of a head:
// attention_<type>_d<width>.hip.  `pass`: 0 forward, 1 dq, 2 dk and dv.
typedef hipError_t (*AttentionLauncher)(const AttentionCall &, int pass,
                                        int rows, hipStream_t);
#define PCA_ATTENTION_DECLARE(type)                                            \
  hipError_t attention_##type##_d32(const AttentionCall &, int, int,           \
                                    hipStream_t);                              \
  hipError_t attention_##type##_d48(const AttentionCall &, int, int,           \
                                    hipStream_t);                              \
  hipError_t attention_##type##_d64(const AttentionCall &, int, int,           \
                                    hipStream_t);                              \
  hipError_t attention_##type##_d96(const AttentionCall &, int, int,           \
                                    hipStream_t);                              \
  hipError_t attention_##type##_d128(const AttentionCall &, int, int,          \
                                     hipStream_t)
PCA_ATTENTION_DECLARE(f32);
PCA_ATTENTION_DECLARE(f16);
PCA_ATTENTION_DECLARE(bf16);
#undef PCA_ATTENTION_DECLARE

// Owned rows of a workgroup: 16 (its waves divide the looped rows), 64 or at most this
// many.  Two blocks of 16 columns per wave share every left operand; where the sums of
// both do not fit the registers of two waves per SIMD it is one.  Heads of 128, 128 rows
// against 64: bf16 forward 291 us against 404 (with bias and cap 488, 549), dq 680 - 1,036
// against 632 - 646; fp32 forward 726 against 587.  Narrow heads have few sums, and four
// waves per SIMD of one block cover more (attention_plan has what was measured).
constexpr int kFewRows = 16;
constexpr int most_rows(int pass, int size, int width) {
  return width <= 32 || (width <= 64 && pass != 2 && size == 2) ||
                 (width > 64 && (pass > 0 || size == 4))
             ? 64
             : 128;
}

// Looped rows of a piece, at least: four tiles of fp32 rows, eight of 16-bit ones.  With
// four, eight and sixteen of the fp32 tiles 12 examples of up to 1,300 rows, 4 heads of
// 48, train in 461, 520 and 944 us.
constexpr int least_rows(int size) {
  return size == 4 ? 128 : 512;
}

AttentionPlan attention_plan(int pass, int64_t nq, int64_t nk, int hq, int hk,
                             int size, int d);
size_t attention_workspace_bytes(int backward, int64_t nq, int64_t nk, int hq,
                                 int hk, int d);
// workspace: of attention_workspace_bytes(0, ...) / (1, ...)
hipError_t attention_forward(AttentionCall c, int dtype, void *workspace,
                             hipStream_t stream);
hipError_t attention_backward(AttentionCall c, int dtype, void *workspace,
                              hipStream_t stream);
hipError_t attention_spans(const int64_t *ids_a, int na, const int64_t *ids_b,
                           int nb, int2 *spans, hipStream_t stream);

} // namespace pca
