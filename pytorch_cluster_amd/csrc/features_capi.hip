// C ABI of the operators on the features of the rows (declared in
// include/pca_features.h): checks on the host, then the launches of attention.hip,
// norm_rotate.hip and lookup.hip on the caller's stream.
#include "../../include/pca_features.h"

#include "attention.hpp"
#include "launchers.hpp"
#include "rows_ops.hpp"

#include <cmath>

namespace {

constexpr int64_t kMost = 2147483646; // rows, entries
// Rows of attention's sides (times heads of a group): with room for a tile behind them.
constexpr int64_t kMostOwned = kMost - 1024;
constexpr int64_t kMostGroups = UINT32_MAX / 256;

bool type_ok(int dtype) {
  return dtype == PCA_F32 || dtype == PCA_F16 || dtype == PCA_BF16;
}
size_t type_size(int dtype) { return dtype == PCA_F32 ? 4 : 2; }

bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int launched(hipError_t e, const char *what) {
  if (e == hipSuccess)
    return PCA_OK;
  return pca::fail(PCA_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

int no_workspace(const char *what, size_t want, const void *workspace,
                 size_t bytes) {
  if (want == 0)
    return PCA_OK;
  if (workspace == nullptr || bytes < want ||
      (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return pca::fail(PCA_ERR_WORKSPACE,
                     "%s needs %zu bytes of workspace, aligned to 256", what,
                     want);
  return PCA_OK;
}

pca::HeadRows head_rows(const void *data, int64_t row, int64_t head, int64_t d,
                        int dtype) {
  pca::HeadRows r;
  r.data = data;
  r.row = row;
  r.head = head;
  const int64_t size = (int64_t)type_size(dtype);
  // (rows of a tile, at most 128, are addressed by 32 bits)
  r.vec = on16(data) && row * size % 16 == 0 && head * size % 16 == 0 &&
          d * size % 16 == 0 && row >= 0 && row * size < (1 << 24);
  return r;
}

bool attention_sizes_ok(int64_t nq, int64_t nk, int64_t hq, int64_t hk,
                        int64_t d) {
  return nq >= 0 && nk >= 0 && nk <= kMostOwned && hk >= 1 && hq >= hk &&
         hq % hk == 0 && hq <= 65535 && nq <= kMostOwned / (hq / hk) &&
         d >= 1 &&
         d <= PCA_ATTENTION_MAX_D &&
         // (workgroups of 64 owned rows or more, 256 threads, that one launch numbers;
         // of 16 rows where they are at most 256)
         (nq * (hq / hk) + 63) / 64 * hk <= kMostGroups &&
         (nk + 63) / 64 * hk <= kMostGroups;
}

int attention_call(const pca_attention_args *a, pca::AttentionCall &c) {
  if (a == nullptr)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "attention: no arguments");
  if (!type_ok(a->dtype))
    return pca::fail(PCA_ERR_UNSUPPORTED,
                     "attention takes float32, float16 and bfloat16");
  if (a->d > PCA_ATTENTION_MAX_D)
    return pca::fail(PCA_ERR_UNSUPPORTED, "attention: heads of up to %d, got %d",
                     PCA_ATTENTION_MAX_D, (int)a->d);
  if (!attention_sizes_ok(a->nq, a->nk, a->hq, a->hk, a->d))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention: sizes out of range (%lld x %d and %lld x %d "
                     "rows and heads of %d)",
                     (long long)a->nq, (int)a->hq, (long long)a->nk, (int)a->hk,
                     (int)a->d);
  if ((a->nq > 0 && a->q == nullptr) ||
      (a->nk > 0 && (a->k == nullptr || a->v == nullptr)))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "attention: a tensor is NULL");
  if (a->slope != nullptr &&
      (a->axes < 1 || a->axes > 3 || (a->nq > 0 && a->pos_q == nullptr) ||
       (a->nk > 0 && a->pos_k == nullptr)))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention: a slope needs positions of 1 to 3 axes");
  if (((reinterpret_cast<uintptr_t>(a->spans_q) |
        reinterpret_cast<uintptr_t>(a->spans_k)) &
       7) != 0)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention: spans have to start on 8 bytes");
  if (!std::isfinite(a->scale) || !std::isfinite(a->cap) || a->cap < 0.f)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention: scale and cap have to be finite, cap not "
                     "negative");
  c.q = head_rows(a->q, a->q_row, a->q_head, a->d, a->dtype);
  c.k = head_rows(a->k, a->k_row, a->k_head, a->d, a->dtype);
  c.v = head_rows(a->v, a->v_row, a->v_head, a->d, a->dtype);
  c.spans_q = reinterpret_cast<const int2 *>(a->spans_q);
  c.spans_k = reinterpret_cast<const int2 *>(a->spans_k);
  c.slope = a->slope;
  c.pos_q = a->pos_q;
  c.pos_k = a->pos_k;
  c.axes = a->slope ? a->axes : 0;
  c.nq = (int)a->nq;
  c.nk = (int)a->nk;
  c.hq = a->hq;
  c.hk = a->hk;
  c.d = a->d;
  c.scale = a->scale;
  c.cap = a->cap;
  return PCA_OK;
}

int norm_rotate_call(const pca_norm_rotate_args *a, pca::NormRotateCall &c) {
  if (a == nullptr)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "norm_rotate: no arguments");
  if (!type_ok(a->dtype) || !type_ok(a->weight_dtype))
    return pca::fail(PCA_ERR_UNSUPPORTED,
                     "norm_rotate takes float32, float16 and bfloat16");
  if (a->rows < 0 || a->rows > kMost || a->hq < 1 || a->hk < 0 ||
      a->hq > 65535 || a->hk > 65535 || a->d < 1 ||
      a->d > PCA_NORM_ROTATE_MAX_D || a->axes < 1 || a->axes > 3 ||
      a->rotated < 0 || a->rotated > a->d / 2)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "norm_rotate: sizes out of range (%lld rows, %d + %d heads "
                     "of %d, %d axes, %d pairs)",
                     (long long)a->rows, (int)a->hq, (int)a->hk, (int)a->d,
                     (int)a->axes, (int)a->rotated);
  if (a->rows > 0 &&
      (a->q == nullptr || (a->hk > 0 && a->k == nullptr) ||
       (a->rotated > 0 && (a->pos == nullptr || a->freq == nullptr))))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "norm_rotate: a tensor is NULL");
  if (!std::isfinite(a->eps) || a->eps < 0.f)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "norm_rotate: eps has to be finite and not negative");
  c.side[0].x = head_rows(a->q, a->q_row, a->q_head, a->d, a->dtype);
  c.side[1].x = head_rows(a->k, a->k_row, a->k_head, a->d, a->dtype);
  c.side[0].weight = a->weight_q;
  c.side[1].weight = a->weight_k;
  c.side[0].heads = a->hq;
  c.side[1].heads = a->hk;
  c.pos = a->pos;
  c.freq = a->freq;
  c.rows = (int)a->rows;
  c.d = a->d;
  c.axes = a->axes;
  c.rotated = a->rotated;
  c.eps = a->eps;
  c.weight_dtype = a->weight_dtype;
  return PCA_OK;
}

int lookup_call(const void *rows, const void *index, int32_t index_bytes,
                int64_t table_rows, int64_t entries, int64_t width, float scale,
                int32_t dtype, const void *out, bool rows_by_entry,
                pca::LookupCall &c) {
  if (!type_ok(dtype))
    return pca::fail(PCA_ERR_UNSUPPORTED,
                     "lookup takes float32, float16 and bfloat16");
  if (table_rows < 0 || table_rows > kMost || entries < 0 || entries > kMost ||
      width < 0 || width > (1 << 20) || (index_bytes != 4 && index_bytes != 8))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "lookup: sizes out of range (%lld rows of %lld, %lld "
                     "entries)",
                     (long long)table_rows, (long long)width,
                     (long long)entries);
  const int64_t read = rows_by_entry ? entries : table_rows;
  const int64_t written = rows_by_entry ? table_rows : entries;
  if ((entries > 0 && index == nullptr) ||
      (read > 0 && width > 0 && rows == nullptr) ||
      (written > 0 && width > 0 && out == nullptr))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "lookup: a tensor is NULL");
  if (!on16(rows) || !on16(out))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "lookup: tensors have to start on 16 bytes");
  if (!std::isfinite(scale))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "lookup: scale has to be finite");
  c.rows = rows;
  c.index = index;
  c.wide_index = index_bytes == 8;
  c.table = table_rows;
  c.entries = entries;
  c.width = width;
  c.scale = scale;
  return PCA_OK;
}

} // namespace

extern "C" {

int pca_spans(const int64_t *ids_a, int64_t na, const int64_t *ids_b,
              int64_t nb, int32_t *spans, void *stream) {
  if (na < 0 || nb < 0 || na > kMostOwned || nb > kMostOwned ||
      (na > 0 && (ids_a == nullptr || spans == nullptr)) ||
      (nb > 0 && ids_b == nullptr) ||
      (reinterpret_cast<uintptr_t>(spans) & 7) != 0)
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "spans: NULL pointer or size out of range");
  return launched(pca::attention_spans(ids_a, (int)na, ids_b, (int)nb,
                                       reinterpret_cast<int2 *>(spans),
                                       static_cast<hipStream_t>(stream)),
                  "spans");
}

size_t pca_attention_workspace_bytes(int64_t nq, int64_t nk, int32_t hq,
                                     int32_t hk, int32_t d, int backward) {
  if (!attention_sizes_ok(nq, nk, hq, hk, d))
    return 0;
  return pca::attention_workspace_bytes(backward ? 1 : 0, nq, nk, hq, hk, d);
}

int pca_attention_forward(const pca_attention_args *args, void *out, void *rest,
                          float *lse, void *workspace, size_t workspace_bytes,
                          void *stream) {
  pca::AttentionCall c;
  int rc = attention_call(args, c);
  if (rc != PCA_OK)
    return rc;
  if (args->nq > 0 && (out == nullptr || !on16(out) || !on16(rest)))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention: out and rest have to start on 16 bytes");
  rc = no_workspace("attention",
                    pca::attention_workspace_bytes(0, c.nq, c.nk, c.hq, c.hk,
                                                   c.d),
                    workspace, workspace_bytes);
  if (rc != PCA_OK)
    return rc;
  c.out = out;
  c.rest = rest;
  c.lse = lse;
  return launched(pca::attention_forward(c, args->dtype, workspace,
                                         static_cast<hipStream_t>(stream)),
                  "attention");
}

int pca_attention_backward(const pca_attention_args *args, const void *out,
                           const void *rest, const float *lse, const void *dout,
                           int64_t dout_row, int64_t dout_head, void *dq,
                           void *dk, void *dv, void *workspace,
                           size_t workspace_bytes, void *stream) {
  pca::AttentionCall c;
  int rc = attention_call(args, c);
  if (rc != PCA_OK)
    return rc;
  if ((c.nq > 0 && (out == nullptr || lse == nullptr || dout == nullptr ||
                    dq == nullptr)) ||
      (c.nk > 0 && (dk == nullptr || dv == nullptr)))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention backward: a tensor is NULL");
  if (!on16(out) || !on16(rest) || !on16(dq) || !on16(dk) || !on16(dv))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention backward: dense tensors have to start on 16 "
                     "bytes");
  if (c.nq > 0 && c.nk > 0 &&
      (c.spans_q == nullptr) != (c.spans_k == nullptr))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "attention backward: spans of one side only");
  rc = no_workspace("attention backward",
                    pca::attention_workspace_bytes(1, c.nq, c.nk, c.hq, c.hk,
                                                   c.d),
                    workspace, workspace_bytes);
  if (rc != PCA_OK)
    return rc;
  c.out_in = out;
  c.rest = const_cast<void *>(rest);
  c.lse = const_cast<float *>(lse);
  c.dout = head_rows(dout, dout_row, dout_head, c.d, args->dtype);
  c.dq = dq;
  c.dk = dk;
  c.dv = dv;
  return launched(pca::attention_backward(c, args->dtype, workspace,
                                          static_cast<hipStream_t>(stream)),
                  "attention backward");
}

int pca_norm_rotate_forward(const pca_norm_rotate_args *args, void *out_q,
                            void *out_k, void *stream) {
  pca::NormRotateCall c;
  const int rc = norm_rotate_call(args, c);
  if (rc != PCA_OK)
    return rc;
  if (args->rows > 0 && (out_q == nullptr || (args->hk > 0 && out_k == nullptr)))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT, "norm_rotate: a tensor is NULL");
  if (!on16(out_q) || !on16(out_k))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "norm_rotate: outputs have to start on 16 bytes");
  c.side[0].out = out_q;
  c.side[1].out = out_k;
  return launched(pca::norm_rotate_forward(c, args->dtype,
                                           static_cast<hipStream_t>(stream)),
                  "norm_rotate");
}

size_t pca_norm_rotate_workspace_bytes(int64_t rows, int32_t d) {
  if (rows < 0 || rows > kMost || d < 1 || d > PCA_NORM_ROTATE_MAX_D)
    return 0;
  return pca::norm_rotate_workspace_bytes(rows, d);
}

int pca_norm_rotate_backward(const pca_norm_rotate_args *args,
                             const void *dout_q, int64_t dout_q_row,
                             int64_t dout_q_head, const void *dout_k,
                             int64_t dout_k_row, int64_t dout_k_head, void *dq,
                             void *dk, void *dweight_q, void *dweight_k,
                             void *workspace, size_t workspace_bytes,
                             void *stream) {
  pca::NormRotateCall c;
  int rc = norm_rotate_call(args, c);
  if (rc != PCA_OK)
    return rc;
  if (args->rows > 0 &&
      (dq == nullptr || dout_q == nullptr ||
       (args->hk > 0 && (dk == nullptr || dout_k == nullptr))))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "norm_rotate backward: a tensor is NULL");
  if (!on16(dq) || !on16(dk))
    return pca::fail(PCA_ERR_INVALID_ARGUMENT,
                     "norm_rotate backward: dq and dk have to start on 16 bytes");
  rc = no_workspace("norm_rotate backward",
                    pca::norm_rotate_workspace_bytes(args->rows, args->d),
                    workspace, workspace_bytes);
  if (rc != PCA_OK)
    return rc;
  c.side[0].dout =
      head_rows(dout_q, dout_q_row, dout_q_head, args->d, args->dtype);
  c.side[1].dout =
      head_rows(dout_k, dout_k_row, dout_k_head, args->d, args->dtype);
  c.side[0].out = dq;
  c.side[1].out = dk;
  c.side[0].dweight = dweight_q;
  c.side[1].dweight = dweight_k;
  return launched(pca::norm_rotate_backward(c, args->dtype, workspace,
                                            static_cast<hipStream_t>(stream)),
                  "norm_rotate backward");
}

int pca_lookup(const void *table, const void *index, int32_t index_bytes,
               int64_t table_rows, int64_t entries, int64_t width, float scale,
               int32_t dtype, void *out, void *stream) {
  pca::LookupCall c;
  const int rc = lookup_call(table, index, index_bytes, table_rows, entries,
                             width, scale, dtype, out, false, c);
  if (rc != PCA_OK)
    return rc;
  c.out = out;
  return launched(
      pca::lookup_forward(c, dtype, static_cast<hipStream_t>(stream)),
      "lookup");
}

size_t pca_lookup_grad_workspace_bytes(int64_t table_rows, int64_t entries,
                                       int64_t width) {
  if (table_rows < 0 || table_rows > kMost || entries < 0 || entries > kMost ||
      width < 0 || width > (1 << 20))
    return 0;
  return pca::lookup_workspace_bytes(table_rows, entries, width);
}

int pca_lookup_grad(const void *dout, const void *index, int32_t index_bytes,
                    int64_t table_rows, int64_t entries, int64_t width,
                    float scale, int32_t dtype, void *dtable, void *workspace,
                    size_t workspace_bytes, void *stream) {
  pca::LookupCall c;
  int rc = lookup_call(dout, index, index_bytes, table_rows, entries, width,
                       scale, dtype, dtable, true, c);
  if (rc != PCA_OK)
    return rc;
  rc = no_workspace("lookup gradient",
                    pca::lookup_workspace_bytes(table_rows, entries, width),
                    workspace, workspace_bytes);
  if (rc != PCA_OK)
    return rc;
  c.out = dtable;
  return launched(pca::lookup_backward(c, dtype, workspace,
                                       static_cast<hipStream_t>(stream)),
                  "lookup gradient");
}

} // extern "C"
