// Attention inside examples: which kernel runs, the spans of the rows, and the kernels
// that put the pieces of a cut side together (attention_impl.hpp has the others).
#include "attention.hpp"
#include "attention_impl.hpp"

#include <algorithm>
#include <cfloat>

namespace pca {

namespace {

size_t attn_align(size_t v) { return (v + 255) & ~(size_t)255; }

// One step of a search in the sorted `ids`: [lo, hi] holds the first entry that is not
// below `id` (`above`: that is above it); eight places are looked at at once.
__device__ __forceinline__ void search_step(const int64_t *ids, int &lo, int &hi,
                                            int64_t id, bool above) {
  const int n = hi - lo, step = n / 8 + 1;
  int64_t v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    v[k] = ids[min(lo + k * step, hi - 1)];
  int below = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    below += lo + k * step < hi && (v[k] < id || (above && v[k] == id));
  hi = below == 0 ? lo : min(lo + below * step, hi);
  lo = below == 0 ? lo : lo + (below - 1) * step + 1;
}

// First entry of the sorted `ids` that is not below `id` (`above`: that is above it), by
// the lanes of a wave, 64 places at a time.
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
// the two.  Latency alone: 2.4 us for one example of 1,024 rows, 5.4 us for a thousand
// examples in 35,000 rows, 7.5 us for 32 queries among 143,000 rows.
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
    int lo_end = lo, hi_end = hi, hi_begin = hi;
    v.x = lo;
    while (v.x < hi_begin || lo_end < hi_end) {
      if (v.x < hi_begin)
        search_step(ids_b, v.x, hi_begin, id, false);
      if (lo_end < hi_end)
        search_step(ids_b, lo_end, hi_end, id, true);
    }
    v.y = max(v.x, lo_end);
  }
  spans[i] = v;
}

// Writes v rounded to T; returns what that takes off.
template <typename T>
__device__ __forceinline__ float put(void *out, int64_t at, float v) {
  const T r = (T)v;
  static_cast<T *>(out)[at] = r;
  return v - (float)r;
}
__device__ __forceinline__ float put_as(int dtype, void *out, int64_t at,
                                        float v) {
  return dtype == 0   ? put<float>(out, at, v)
         : dtype == 2 ? put<_Float16>(out, at, v)
                      : put<__bf16>(out, at, v);
}

// Pieces in use for row (query, head) of q.  (Sides are cut into pieces where there are
// few workgroups: rows, and their products with heads, are far below 2^31 here.)
__device__ __forceinline__ int pieces_of(const AttentionCall &c, int row) {
  const int query = row / c.hq, head = row - query * c.hq;
  const int group = c.hq / c.hk, kv = head / group;
  const int tiles = (c.nq * group + c.rows - 1) / c.rows;
  return c.pieces[kv * tiles + (query * group + head - kv * group) / c.rows];
}

// Output rows from the pieces' sums, maxima and sums of weights,
//
//   o = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s,   m = max_s m_s:
//
// 32 lanes take four elements each; where there are many pieces, `shares` groups of lanes
// divide them and meet in LDS, in their order.  Four ragged
// scans, up to 1,024 queries each of 8 heads of 64, up to 8 pieces: 13 us; 256 rows of 128
// in up to 64 pieces: 7 us, latency.
__global__ __launch_bounds__(256) void
join_forward_kernel(AttentionCall c, int dtype, int shares) {
  __shared__ float lds_acc[8][128], lds_ml[8][2];
  const int rows = c.nq * c.hq;
  const int grp = threadIdx.x / 32, share = grp % shares;
  const int row = blockIdx.x * (8 / shares) + grp / shares;
  const int e0 = (threadIdx.x & 31) * 4;
  const int pieces = row < rows ? pieces_of(c, row) : 1;
  const bool there = pieces > 1;
  float top = -__builtin_inff(), sum = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (there) {
#pragma unroll 8
    for (int s = share; s < pieces; s += shares)
      top = fmaxf(top, c.part_ml[((int64_t)s * rows + row) * 2]);
#pragma unroll 4
    for (int s = share; s < pieces; s += shares) {
      const float m = c.part_ml[((int64_t)s * rows + row) * 2];
      const float l = c.part_ml[((int64_t)s * rows + row) * 2 + 1];
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      const float *from = c.part + ((int64_t)s * rows + row) * c.d + e0;
      if (c.d % 4 == 0) {
        if (e0 < c.d)
          __builtin_memcpy(v, __builtin_assume_aligned(from, 16), 16);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = e0 + e < c.d ? from[e] : 0.f;
      }
      // (-inf: nothing in this piece)
      const float w = m == -__builtin_inff() ? 0.f
                      : m == top             ? 1.f
                                 : __builtin_amdgcn_exp2f(m - top);
      sum = fmaf(l, w, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[e] = fmaf(v[e], w, acc[e]);
    }
  }
  if (shares > 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      lds_acc[grp][e0 + e] = acc[e];
    if (e0 == 0) {
      lds_ml[grp][0] = top;
      lds_ml[grp][1] = sum;
    }
    __syncthreads();
    if (share != 0)
      return;
    for (int k = 1; k < shares; ++k)
      top = fmaxf(top, lds_ml[grp + k][0]);
    sum = acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
    for (int k = 0; k < shares; ++k) {
      const float m = lds_ml[grp + k][0];
      const float w = m == -__builtin_inff() ? 0.f
                      : m == top             ? 1.f
                                 : __builtin_amdgcn_exp2f(m - top);
      sum = fmaf(lds_ml[grp + k][1], w, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        acc[e] = fmaf(lds_acc[grp + k][e0 + e], w, acc[e]);
    }
  }
  if (!there)
    return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e0 + e < c.d) {
      const int64_t at = (int64_t)row * c.d + e0 + e;
      const float left = put_as(dtype, c.out, at, acc[e] * inv);
      if (c.rest)
        put_as(dtype, c.rest, at, left);
    }
  if (e0 == 0 && c.lse) {
    const int query = row / c.hq, head = row % c.hq;
    c.lse[(int64_t)head * c.nq + query] =
        sum == 0.f ? __builtin_inff() : top + __builtin_amdgcn_logf(sum);
  }
}

// Rows of dq (SECOND: of dk, then of dv) as sums over the pieces, in their order: 32
// lanes a row.
template <bool SECOND>
__global__ __launch_bounds__(256) void join_sum_kernel(AttentionCall c,
                                                       int dtype) {
  const int keys = c.nk * c.hk;
  const int rows = SECOND ? 2 * keys : c.nq * c.hq;
  const int row = blockIdx.x * 8 + threadIdx.x / 32;
  const int e0 = (threadIdx.x & 31) * 4;
  if (row >= rows || e0 >= c.d)
    return;
  const int at = SECOND && row >= keys ? row - keys : row;
  int pieces;
  if (SECOND) {
    const int key = at / c.hk, tiles = (c.nk + c.rows - 1) / c.rows;
    pieces = c.pieces[(at - key * c.hk) * tiles + key / c.rows];
  } else {
    pieces = pieces_of(c, at);
  }
  if (pieces <= 1)
    return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < pieces; ++s) {
    const float *from = c.part + ((int64_t)s * rows + row) * c.d + e0;
    if (c.d % 4 == 0) {
      float x[4];
      __builtin_memcpy(x, __builtin_assume_aligned(from, 16), 16);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] += x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] += e0 + e < c.d ? from[e] : 0.f;
    }
  }
  void *out = !SECOND ? c.dq : row < keys ? c.dk : c.dv;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e0 + e < c.d)
      put_as(dtype, out, (int64_t)at * c.d + e0 + e, v[e]);
}

// Numbers that go with the cap, in fp32's range: a cap of 2^127 or more is one of 2^127
// (cap log2 e is formed, and bends nothing that is not as large), and behind a tiny one
// products of zero stay zero (and not zero times infinity).
void set_cap(AttentionCall &c) {
  if (c.cap <= 0.f)
    return;
  c.cap = std::min(c.cap, 0x1p127f);
  const double in = 2.0 * 1.44269504088896340736 * c.scale / c.cap;
  c.under_tanh = (float)std::clamp(in, -(double)FLT_MAX, (double)FLT_MAX);
}

AttentionLauncher launcher(int dtype, int d) {
#define PCA_BY_WIDTH(type)                                                     \
  (d <= 32   ? attention_##type##_d32                                          \
   : d <= 48 ? attention_##type##_d48                                          \
   : d <= 64 ? attention_##type##_d64                                          \
   : d <= 96 ? attention_##type##_d96                                          \
             : attention_##type##_d128)
  return dtype == 0 ? PCA_BY_WIDTH(f32)
                    : dtype == 2 ? PCA_BY_WIDTH(f16) : PCA_BY_WIDTH(bf16);
#undef PCA_BY_WIDTH
}

unsigned join_blocks(int64_t rows, int per) {
  return (unsigned)((rows + per - 1) / per);
}

int element_size(int dtype) { return dtype == 0 ? 4 : 2; }

} // namespace

// Rows of a workgroup (both sides measured, us; bf16 where nothing else is said).  128 or
// 64 rows: heads of 64 with a bias, forward, 16 x 1,024 rows of 8 heads 118 / 106, 4 x 4,096
// rows 365 / 317 (four waves per SIMD cover the distances), forward and backward with
// dk / dv at 128 and 64 rows 235 / 260, fp32 306 / 337; heads of 32, a thousand graphs of 35
// rows on average, all three kernels 183 / 120.  64 rows as well if 128 leave a CU less
// than two workgroups.  16 rows, whose waves divide the keys, or 64, with their joins: 32
// single queries 43 / 54, one cloud of 1,024 rows 24 / 25, four ragged scans with 1,024
// queries each at most 131 / 85.
//
// Pieces of the looped side where workgroups are few (about three to a CU; those of 128
// rows never are): 2,048 workgroups' worth.  12 ragged examples in fp32, one to eight
// pieces: 756, 640, 589, 623; four ragged scans, one, four, eight: 269, 100, 92; from
// 1,024 workgroups on pieces lose (clouds, one and two: 384, 497).  With 16 rows a
// workgroup 512 workgroups' worth (32 queries, 16 to 128 pieces: 58, 60, 71, 97).  How many
// of the pieces a tile of rows uses goes by the length of its own examples
// (pieces_in_use).  Rows are counted, which is right for long examples; many short ones
// are a longer chain of tiles than their rows say.
AttentionPlan attention_plan(int pass, int64_t nq, int64_t nk, int hq, int hk,
                             int size, int d) {
  const int64_t rows_q = nq * (hq / hk);
  const int64_t owned = pass == 2 ? nk : rows_q;
  const int64_t looped = pass == 2 ? rows_q : nk;
  auto groups = [&](int rows) { return (owned + rows - 1) / rows * hk; };
  AttentionPlan p;
  p.rows = most_rows(pass, size, d);
  if (groups(p.rows) < 512)
    p.rows = 64;
  if (owned <= 256)
    p.rows = kFewRows;
  const int64_t n = std::max<int64_t>(1, groups(p.rows));
  const int64_t want = p.rows == kFewRows             ? 512
                       : p.rows == 64 && n < 800 ? 2048
                                                      : 0;
  const int64_t most = looped / least_rows(size);
  p.splits = (int)std::clamp<int64_t>((want + n / 2) / n, 1,
                                      std::clamp<int64_t>(most, 1, 64));
  return p;
}

// Where the pieces' results lie behind `base` (pass as in the plan); returns the bytes.
static size_t lay_out(AttentionCall &c, int pass, const AttentionPlan &p,
                      char *base) {
  c.rows = p.rows;
  c.splits = p.splits;
  if (p.splits <= 1)
    return 0;
  const int64_t owned = pass == 2 ? c.nk : (int64_t)c.nq * (c.hq / c.hk);
  const int64_t tiles = (owned + p.rows - 1) / p.rows;
  const int64_t rows =
      pass == 2 ? 2 * (int64_t)c.nk * c.hk : (int64_t)c.nq * c.hq;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char *q = base + at;
    at += attn_align(bytes);
    return q;
  };
  c.part = reinterpret_cast<float *>(
      take(sizeof(float) * (size_t)(p.splits * rows * c.d)));
  c.pieces = reinterpret_cast<int *>(take(sizeof(int) * (size_t)(tiles * c.hk)));
  if (pass == 0)
    c.part_ml =
        reinterpret_cast<float *>(take(sizeof(float) * 2 * p.splits * rows));
  return at;
}

size_t attention_workspace_bytes(int backward, int64_t nq, int64_t nk, int hq,
                                 int hk, int d) {
  AttentionCall c;
  c.nq = (int)nq;
  c.nk = (int)nk;
  c.hq = hq;
  c.hk = hk;
  c.d = d;
  size_t most = 0;
  for (int pass = backward ? 1 : 0; pass <= (backward ? 2 : 0); ++pass)
    for (int size : {2, 4}) // (the same for all element types)
      most = std::max(
          most, lay_out(c, pass, attention_plan(pass, nq, nk, hq, hk, size, d),
                        nullptr));
  if (backward)
    most += 2 * attn_align(sizeof(float) * (size_t)(nq * hq)) +
            attn_align(sizeof(float) * (size_t)hq);
  return most + 256;
}

hipError_t attention_forward(AttentionCall c, int dtype, void *workspace,
                             hipStream_t stream) {
  set_cap(c);
  const AttentionPlan p = attention_plan(0, c.nq, c.nk, c.hq, c.hk,
                                         element_size(dtype), c.d);
  lay_out(c, 0, p, static_cast<char *>(workspace));
  const hipError_t e = launcher(dtype, c.d)(c, 0, p.rows, stream);
  if (e != hipSuccess || p.splits == 1 || c.nq == 0)
    return e;
  // (rows alone fill the chip: a group a row)
  const int64_t rows = (int64_t)c.nq * c.hq;
  const int shares = rows >= 8192       ? 1
                     : p.splits >= 32   ? 8
                     : p.splits >= 4    ? 4
                                        : 1;
  join_forward_kernel<<<dim3(join_blocks(rows, 8 / shares)), dim3(256), 0,
                        stream>>>(c, dtype, shares);
  return hipGetLastError();
}

hipError_t attention_backward(AttentionCall c, int dtype, void *workspace,
                              hipStream_t stream) {
  set_cap(c);
  const size_t one = attn_align(sizeof(float) * (size_t)c.nq * c.hq);
  char *base = static_cast<char *>(workspace);
  c.minus_delta = reinterpret_cast<float *>(base);
  c.base = reinterpret_cast<float *>(base + one);
  c.minus_slope = reinterpret_cast<float *>(base + 2 * one);
  base += 2 * one + attn_align(sizeof(float) * (size_t)c.hq);
  const int size = element_size(dtype);
  const AttentionPlan pq = attention_plan(1, c.nq, c.nk, c.hq, c.hk, size, c.d);
  lay_out(c, 1, pq, base);
  hipError_t e = launcher(dtype, c.d)(c, 1, pq.rows, stream);
  if (e == hipSuccess && pq.splits > 1 && c.nq > 0) {
    join_sum_kernel<false>
        <<<dim3(join_blocks((int64_t)c.nq * c.hq, 8)), dim3(256), 0, stream>>>(
            c, dtype);
    e = hipGetLastError();
  }
  if (e != hipSuccess)
    return e;
  const AttentionPlan pk = attention_plan(2, c.nq, c.nk, c.hq, c.hk, size, c.d);
  lay_out(c, 2, pk, base);
  e = launcher(dtype, c.d)(c, 2, pk.rows, stream);
  if (e == hipSuccess && pk.splits > 1 && c.nk > 0) {
    join_sum_kernel<true><<<dim3(join_blocks(2 * (int64_t)c.nk * c.hk, 8)),
                            dim3(256), 0, stream>>>(c, dtype);
    e = hipGetLastError();
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
