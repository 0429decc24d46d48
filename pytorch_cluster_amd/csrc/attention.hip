// Attention inside examples: which kernel runs, the spans of the rows, and the kernels
// that put the pieces of a cut side together (attention_impl.hpp has the others).
#include "attention.hpp"
#include "attention_impl.hpp"

#include <algorithm>

namespace pca {

namespace {

size_t attn_align(size_t v) { return (v + 255) & ~(size_t)255; }

// First entry of the sorted `ids` at [lo, hi) that is not below `id` (`above`: that is
// above it).
__device__ __forceinline__ int bound_of(const int64_t *ids, int lo, int hi,
                                        int64_t id, bool above) {
  while (lo < hi) {
    const int mid = lo + ((hi - lo) >> 1);
    const int64_t v = ids[mid];
    if (v < id || (above && v == id))
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo;
}

// The same by the lanes of a wave, 64 places at a time.
__device__ __forceinline__ int wave_bound_of(const int64_t *ids, int n,
                                             int64_t id, bool above) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 64) {
    // places lo + step, lo + 2 step, ...: the last one that is still below
    const int step = (hi - lo + 63) / 64;
    const int at = lo + lane * step;
    bool below = false;
    if (at < hi) {
      const int64_t v = ids[at];
      below = v < id || (above && v == id);
    }
    const int many = __popcll(__ballot(below));
    if (many == 0)
      return lo;
    hi = min(lo + many * step, hi);
    lo = lo + (many - 1) * step + 1;
  }
  const int at = lo + lane;
  bool below = false;
  if (at < hi) {
    const int64_t v = ids[at];
    below = v < id || (above && v == id);
  }
  return lo + __popcll(__ballot(below));
}

// spans[i] = [first row of b with row i's id, first one with a larger id).  The waves
// of a workgroup find where its first and its last id lie, three dependent reads for
// 200,000 rows; only workgroups with rows of several examples search further, between
// the two.
__global__ __launch_bounds__(256) void spans_kernel(const int64_t *ids_a, int na,
                                                    const int64_t *ids_b,
                                                    int nb, int2 *spans) {
  __shared__ int edge[2];
  const int first = blockIdx.x * 256;
  const int last = min(first + 256, na) - 1;
  const int wave = threadIdx.x >> 6;
  const int64_t id_first = ids_a[first], id_last = ids_a[last];
  if (wave < 2) {
    const int e = wave == 0 ? wave_bound_of(ids_b, nb, id_first, false)
                            : wave_bound_of(ids_b, nb, id_last, true);
    if ((threadIdx.x & 63) == 0)
      edge[wave] = e;
  }
  __syncthreads();
  const int i = first + threadIdx.x;
  if (i > last)
    return;
  const int lo = edge[0], hi = max(edge[0], edge[1]);
  int2 v = make_int2(lo, hi);
  if (id_first != id_last) {
    const int64_t id = ids_a[i];
    v.x = bound_of(ids_b, lo, hi, id, false);
    v.y = bound_of(ids_b, v.x, hi, id, true);
  }
  spans[i] = v;
}

template <typename T>
__device__ __forceinline__ void put(void *out, int64_t at, float v) {
  static_cast<T *>(out)[at] = (T)v;
}
__device__ __forceinline__ void put_as(int dtype, void *out, int64_t at,
                                       float v) {
  if (dtype == 0)
    put<float>(out, at, v);
  else if (dtype == 2)
    put<_Float16>(out, at, v);
  else
    put<__bf16>(out, at, v);
}

// Output rows from the pieces' sums, maxima and sums of weights: 32 lanes a row, four
// elements each.
__global__ __launch_bounds__(256) void join_forward_kernel(AttentionCall c,
                                                           int dtype) {
  const int64_t rows = (int64_t)c.nq * c.hq;
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= rows)
    return;
  float top = -__builtin_inff(), sum = 0.f;
  for (int s = 0; s < c.splits; ++s)
    top = fmaxf(top, c.part_ml[(s * rows + row) * 2]);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int e0 = (threadIdx.x & 31) * 4;
  for (int s = 0; s < c.splits; ++s) {
    const float m = c.part_ml[(s * rows + row) * 2];
    const float l = c.part_ml[(s * rows + row) * 2 + 1];
    if (m == -__builtin_inff() && l == 0.f)
      continue; // nothing in this piece
    const float w = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
    sum += l * w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e0 + e < c.d)
        acc[e] = fmaf(c.part[(s * rows + row) * c.d + e0 + e], w, acc[e]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e0 + e < c.d)
      put_as(dtype, c.out, row * c.d + e0 + e, acc[e] * inv);
  if (e0 == 0 && c.lse) {
    const int64_t query = row / c.hq, head = row % c.hq;
    c.lse[head * c.nq + query] =
        sum == 0.f ? __builtin_inff() : top + __builtin_amdgcn_logf(sum);
  }
}

// out[i] = sum over the pieces, in their order.
__global__ __launch_bounds__(256) void join_sum_kernel(const float *part,
                                                       int pieces,
                                                       int64_t stride,
                                                       int64_t count, int dtype,
                                                       void *out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count)
    return;
  float v = 0.f;
  for (int s = 0; s < pieces; ++s)
    v += part[s * stride + i];
  put_as(dtype, out, i, v);
}

AttentionLauncher launcher(int dtype, int d) {
#define PCA_BY_WIDTH(type)                                                     \
  (d <= 32 ? attention_##type##_d32                                            \
           : d <= 64 ? attention_##type##_d64 : attention_##type##_d128)
  return dtype == 0 ? PCA_BY_WIDTH(f32)
                    : dtype == 2 ? PCA_BY_WIDTH(f16) : PCA_BY_WIDTH(bf16);
#undef PCA_BY_WIDTH
}

hipError_t join_sum(const AttentionCall &c, const float *part, int64_t stride,
                    int64_t count, int dtype, void *out, hipStream_t stream) {
  const int64_t blocks = (count + 255) / 256;
  if (blocks > INT32_MAX)
    return hipErrorInvalidValue;
  join_sum_kernel<<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(
      part, c.splits, stride, count, dtype, out);
  return hipGetLastError();
}

} // namespace

AttentionPlan attention_plan(int pass, int64_t nq, int64_t nk, int hq, int hk,
                             int dtype, int d) {
  const int64_t rows_q = nq * (hq / hk);
  const int64_t owned = pass == 2 ? nk : rows_q;
  const int64_t looped = pass == 2 ? rows_q : nk;
  AttentionPlan p;
  const int rows = wide_rows(pass, dtype == 0 ? 4 : 2, d);
  const int64_t wide = (owned + rows - 1) / rows * hk;
  p.wide = wide >= 256;
  if (!p.wide) {
    const int64_t few =
        std::max<int64_t>(1, (owned + kFewRows - 1) / kFewRows * hk);
    const int64_t most = (looped + 255) / 256;
    p.splits = (int)std::clamp<int64_t>(1024 / few, 1,
                                        std::clamp<int64_t>(most, 1, 256));
  }
  return p;
}

static size_t part_bytes(int pass, int64_t nq, int64_t nk, int hq, int hk,
                         int dtype, int d) {
  const int splits = attention_plan(pass, nq, nk, hq, hk, dtype, d).splits;
  if (splits <= 1)
    return 0;
  const int64_t one = pass == 2 ? 2 * nk * hk * d : nq * hq * d;
  size_t bytes = attn_align(sizeof(float) * (size_t)(splits * one));
  if (pass == 0)
    bytes += attn_align(sizeof(float) * 2 * (size_t)(splits * nq * hq));
  return bytes;
}

size_t attention_workspace_bytes(int pass, int64_t nq, int64_t nk, int hq,
                                 int hk, int dtype, int d) {
  if (pass == 0)
    return 256 + part_bytes(0, nq, nk, hq, hk, dtype, d);
  return attn_align(sizeof(float) * (size_t)(nq * hq)) + 256 +
         std::max(part_bytes(1, nq, nk, hq, hk, dtype, d),
                  part_bytes(2, nq, nk, hq, hk, dtype, d));
}

hipError_t attention_forward(AttentionCall c, int dtype, void *workspace,
                             hipStream_t stream) {
  const AttentionPlan p = attention_plan(0, c.nq, c.nk, c.hq, c.hk, dtype, c.d);
  c.splits = p.splits;
  c.part = static_cast<float *>(workspace);
  c.part_ml = c.part + attn_align(sizeof(float) * (size_t)p.splits * c.nq *
                                  c.hq * c.d) /
                           sizeof(float);
  hipError_t e = launcher(dtype, c.d)(c, 0, p.wide, stream);
  if (e != hipSuccess || p.splits == 1 || c.nq == 0)
    return e;
  const int64_t blocks = ((int64_t)c.nq * c.hq + 7) / 8;
  join_forward_kernel<<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(c,
                                                                        dtype);
  return hipGetLastError();
}

hipError_t attention_backward(AttentionCall c, int dtype, void *workspace,
                              hipStream_t stream) {
  c.delta = static_cast<float *>(workspace);
  c.part = c.delta +
           attn_align(sizeof(float) * (size_t)c.nq * c.hq) / sizeof(float);
  const AttentionPlan pq = attention_plan(1, c.nq, c.nk, c.hq, c.hk, dtype, c.d);
  c.splits = pq.splits;
  hipError_t e = launcher(dtype, c.d)(c, 1, pq.wide, stream);
  if (e == hipSuccess && c.splits > 1 && c.nq > 0) {
    const int64_t count = (int64_t)c.nq * c.hq * c.d;
    e = join_sum(c, c.part, count, count, dtype, c.dq, stream);
  }
  if (e != hipSuccess)
    return e;
  const AttentionPlan pk = attention_plan(2, c.nq, c.nk, c.hq, c.hk, dtype, c.d);
  c.splits = pk.splits;
  e = launcher(dtype, c.d)(c, 2, pk.wide, stream);
  if (e == hipSuccess && c.splits > 1 && c.nk > 0) {
    const int64_t count = (int64_t)c.nk * c.hk * c.d;
    e = join_sum(c, c.part, 2 * count, count, dtype, c.dk, stream);
    if (e == hipSuccess)
      e = join_sum(c, c.part + count, 2 * count, count, dtype, c.dv, stream);
  }
  return e;
}

hipError_t attention_spans(const int64_t *ids_a, int na, const int64_t *ids_b,
                           int nb, int2 *spans, hipStream_t stream) {
  if (na <= 0)
    return hipSuccess;
  spans_kernel<<<dim3((unsigned)((na + 255) / 256)), dim3(256), 0, stream>>>(
      ids_a, na, ids_b, nb, spans);
  return hipGetLastError();
}

} // namespace pca
