/*
 * pca_features.h -- C ABI of the operators on the features of the rows:
 * attention inside examples, norm with rotation, lookup.  In the same library
 * (libpca_neighbors.so) and by the same rules as pca_neighbors.h: plain device
 * pointers and sizes, asynchronous on `stream`, a status code, no allocation,
 * no synchronisation; pca_last_error() has the text of the last failure on the
 * calling thread.  All entry points record kernels only and may be captured
 * into a graph.  The same call gives the same bits.
 *
 * Element types: PCA_F32, PCA_F16, PCA_BF16.  Sums, softmax statistics and
 * norms are held in 32 bits, angles in 64.
 *
 * "dense" tensors have no strides: [a, b, c] is row-major and starts on 16
 * bytes.  Others give strides in elements for all but the last dimension,
 * which is dense; any alignment to the element type is taken, and rows that
 * start on 16 bytes and are a multiple of 16 bytes long are read faster.
 */
#ifndef PCA_FEATURES_H
#define PCA_FEATURES_H

#include "pca_neighbors.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Widest head of pca_attention_* and of pca_norm_rotate_*. */
#define PCA_ATTENTION_MAX_D 128
#define PCA_NORM_ROTATE_MAX_D 256

/*
 * spans[2 i], spans[2 i + 1] = first row of b whose example id is that of row
 * i of a, first row behind them (ids sorted; equal if b has none): which rows
 * of b belong to row i.  spans: [2 na] int32, on 8 bytes.
 */
int pca_spans(const int64_t *ids_a, int64_t na, const int64_t *ids_b,
              int64_t nb, int32_t *spans, void *stream);

/*
 * Softmax attention of every row of q over the rows of k that its span names:
 *
 *   t_ij = scale q_i . k_j
 *   s_ij = (cap > 0 ? cap tanh(t_ij / cap) : t_ij) - slope_h |pos_q_i - pos_k_j|
 *   out_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij)        (no such j: zeros)
 *
 * per head h of hq; head h reads head h / (hq / hk) of k and v.
 */
typedef struct pca_attention_args {
  const void *q, *k, *v;            /* [nq, hq, d], [nk, hk, d], [nk, hk, d]  */
  int64_t q_row, q_head;            /* strides in elements                    */
  int64_t k_row, k_head;
  int64_t v_row, v_head;
  const int32_t *spans_q;           /* [nq, 2] rows of k per row of q, by     */
                                    /* pca_spans; NULL: all rows              */
  const int32_t *spans_k;           /* [nk, 2] rows of q per row of k; used   */
                                    /* by the backward pass                   */
  const float *pos_q, *pos_k;       /* [nq, axes], [nk, axes]; with slope     */
  const float *slope;               /* [hq], or NULL: no bias                 */
  int32_t axes;                     /* 1 .. 3                                 */
  int32_t dtype;
  int64_t nq, nk;                   /* nq * hq / hk and nk, each rounded up   */
                                    /* to 64, times hk: below 2^30            */
  int32_t hq, hk, d;                /* hq a multiple of hk, d <= 128          */
  float scale;
  float cap;                        /* 0: none; above 2^127: 2^127            */
} pca_attention_args;

/* Scratch of the forward (backward = 0) or the backward call (1); 0: sizes not
 * supported. */
size_t pca_attention_workspace_bytes(int64_t nq, int64_t nk, int32_t hq,
                                     int32_t hk, int32_t d, int backward);

/* out: [nq, hq, d] dense.  For the backward pass: lse, [hq, nq] fp32, and, with
 * 16-bit types, rest: what rounding took off out, [nq, hq, d]; or NULL. */
int pca_attention_forward(const pca_attention_args *args, void *out, void *rest,
                          float *lse, void *workspace, size_t workspace_bytes,
                          void *stream);

/* Gradients of q, k, v (dense, all three are written) from that of out.  rest
 * may be NULL: dq and dk are then less exact (16-bit types). */
int pca_attention_backward(const pca_attention_args *args, const void *out,
                           const void *rest, const float *lse, const void *dout,
                           int64_t dout_row, int64_t dout_head, void *dq,
                           void *dk, void *dv, void *workspace,
                           size_t workspace_bytes, void *stream);

/*
 * Norm of every head of q and k and rotation by the row's position:
 *
 *   y = weight x / sqrt(mean(x^2) + eps)
 *   a_c = sum_p pos_p freq_pc                                 c < rotated
 *   out_c = y_c cos a_c - y_{c + rotated} sin a_c
 *   out_{c + rotated} = y_{c + rotated} cos a_c + y_c sin a_c
 *
 * and y itself from element 2 rotated on.  The mean is formed in 32 bits: x^2
 * has to stay in their range.
 */
typedef struct pca_norm_rotate_args {
  const void *q, *k;                /* [rows, hq, d], [rows, hk, d]           */
  int64_t q_row, q_head;
  int64_t k_row, k_head;
  const void *weight_q, *weight_k;  /* [d] of weight_dtype, or NULL: ones     */
  const float *pos;                 /* [rows, axes]                           */
  const float *freq;                /* [axes, rotated]                        */
  int64_t rows;
  int32_t hq, hk;                   /* hk may be 0: no k                      */
  int32_t d, axes, rotated;         /* d <= 256, axes 1 .. 3, 2 rotated <= d  */
  int32_t dtype, weight_dtype;
  float eps;
} pca_norm_rotate_args;

/* out_q, out_k: dense. */
int pca_norm_rotate_forward(const pca_norm_rotate_args *args, void *out_q,
                            void *out_k, void *stream);

size_t pca_norm_rotate_workspace_bytes(int64_t rows, int32_t d);

/* dq, dk: dense; dweight_q, dweight_k: [d] of weight_dtype, or NULL. */
int pca_norm_rotate_backward(const pca_norm_rotate_args *args,
                             const void *dout_q, int64_t dout_q_row,
                             int64_t dout_q_head, const void *dout_k,
                             int64_t dout_k_row, int64_t dout_k_head, void *dq,
                             void *dk, void *dweight_q, void *dweight_k,
                             void *workspace, size_t workspace_bytes,
                             void *stream);

/*
 * out[e] = scale table[index[e]]; zeros where the index lies outside
 * [0, table_rows).  index: int32 or int64 (index_bytes 4 or 8).  table:
 * [table_rows, width] dense, out: [entries, width] dense.  scale is finite;
 * rows and entries are below 2^31 - 1, width at most 2^20.
 */
int pca_lookup(const void *table, const void *index, int32_t index_bytes,
               int64_t table_rows, int64_t entries, int64_t width, float scale,
               int32_t dtype, void *out, void *stream);

size_t pca_lookup_grad_workspace_bytes(int64_t table_rows, int64_t entries,
                                       int64_t width);

/* dtable[n] = scale * sum of dout[e] over the entries with index[e] = n (zeros
 * where there are none); dense. */
int pca_lookup_grad(const void *dout, const void *index, int32_t index_bytes,
                    int64_t table_rows, int64_t entries, int64_t width,
                    float scale, int32_t dtype, void *dtable, void *workspace,
                    size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
