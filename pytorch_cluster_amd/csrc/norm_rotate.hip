// Norms of queries and keys per head, with the rotation by the rows' positions in the
// same pass:
//
//   y = w x / sqrt(mean(x^2) + eps)              over the d elements of a head
//   a_c = sum_p pos_p freq_pc                    c < rotated
//   out_c = y_c cos a_c - y_{c+rotated} sin a_c
//   out_{c+rotated} = y_{c+rotated} cos a_c + y_c sin a_c;  the rest as y
//
// A group of lanes takes a row (all heads of it) with 16 bytes of a head per lane.  The
// angles are the same for every head: the group forms them once, in 64 bits -- a
// position of 50 m at 100 rad / m is known to 3e-4 rad in fp32 --, reduced to a
// fraction of a turn before they become fp32.  Partners of a pair lie in different
// lanes and meet in LDS, an element of padding to every eight against bank conflicts.
//
// Backward, with g the gradient turned back, r = sqrt(mean(x^2) + eps) and xhat = x / r:
// dw = sum g xhat, dx = (g w - xhat mean(g w xhat)) / r.  Every workgroup adds up dw of its
// rows and a second kernel adds up the workgroups, in a fixed order.
//
// Bound by memory, forwards more than backwards.  131,072 rows of 8 + 2 heads of 128, bf16,
// three axes, 63 pairs: forward 161 us = 4.2 TB/s (a large copy: 5.0), backward, which reads
// x and the gradient, 297 us = 3.4 TB/s; there the chain of a head -- sum across lanes,
// exchange, second sum -- at three waves per SIMD is not covered throughout (vector unit
// busy 47 % of the cycles).  With the head's tensors picked by every lane and one head at
// a time 308 and 555 us.  1,024 rows of 4 + 4 heads of 32, fp32: 5.2 us, latency.
#include "rows_ops.hpp"

#include "attention_impl.hpp"

#include <algorithm>

namespace pca {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowBlocks = 1024; // workgroups, at most: four to a CU, each with rows enough
                                 // that its share of dw costs little

// Elements e0, e0 + 1, ... of a weight, ones if there is none (behind d: something).  One
// branch on the type for all of them, so that their loads are under way together.
template <int PER>
__device__ __forceinline__ void load_weight(float (&w)[PER], const void *p,
                                            int dtype, int e0, int d) {
#pragma unroll
  for (int i = 0; i < PER; ++i)
    w[i] = 1.f;
  if (p == nullptr)
    return;
  int at[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    at[i] = min(e0 + i, d - 1);
  if (dtype == 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      w[i] = static_cast<const float *>(p)[at[i]];
  } else {
    uint16_t v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      v[i] = static_cast<const uint16_t *>(p)[at[i]];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      w[i] = dtype == 2 ? (float)__builtin_bit_cast(_Float16, v[i])
                        : __uint_as_float((uint32_t)v[i] << 16);
  }
}

__device__ __forceinline__ int padded(int e) { return e + (e >> 3); }

// cos and sin of the angles of row `row` into cs / sn (by the lanes of its group).
__device__ __forceinline__ void row_angles(const NormRotateCall &c, int64_t row,
                                           int lane, int lanes, float *cs,
                                           float *sn) {
  for (int r = lane; r < c.rotated; r += lanes) {
    double a = 0.0;
    for (int p = 0; p < c.axes; ++p)
      a += (double)c.pos[row * c.axes + p] * (double)c.freq[p * c.rotated + r];
    // half turns: sin and cos of pi times what is left of whole turns
    const double t = a * 0.15915494309189533577;
    const float f = (float)(2.0 * (t - __builtin_rint(t)));
    float s, o;
    sincospif(f, &s, &o);
    cs[padded(r)] = o;
    sn[padded(r)] = s;
  }
}

// A wave's LDS accesses in order, without a barrier of the workgroup.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// LANES lanes a row.  A workgroup takes heads [blockIdx.y heads_each, ...) (side 0's, then
// side 1's) of its rows, HEADS at a time, whose chains of dependent steps -- sums across
// lanes, the exchange in LDS -- overlap; the next ones' loads are under way meanwhile.
// Which head it is is the same in every lane: bases, strides and weights are picked by
// the scalar unit.
template <typename T, int LANES, bool BACKWARD>
__global__ __launch_bounds__(kRowThreads, BACKWARD ? 3 : 4) void
norm_rotate_kernel(NormRotateCall c, int heads_each) {
  constexpr int PER = 16 / (int)sizeof(T), DP = PER * LANES;
  constexpr int HEADS = BACKWARD && PER == 8 ? 1 : 2; // (as many as the registers hold)
  constexpr int LINE = DP + DP / 8 + 1;
  constexpr int GROUPS = kRowThreads / LANES;
  __shared__ float line[GROUPS][HEADS][LINE];
  __shared__ float angle[GROUPS][2][DP / 2 + DP / 16 + 1];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int e0 = lane * PER;
  const int head0 = blockIdx.y * heads_each;
  const int stop = min(head0 + heads_each, c.side[0].heads + c.side[1].heads);
  const float per_d = 1.f / (float)c.d;
  float w[2][PER], dw[2][PER];
  int other[PER]; // where an element's partner lies; its own place if it has none
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = e0 + i;
    other[i] = padded(e < c.rotated       ? e + c.rotated
                      : e < 2 * c.rotated ? e - c.rotated
                                          : e);
    dw[0][i] = dw[1][i] = 0.f;
  }
#pragma unroll
  for (int s = 0; s < 2; ++s)
    load_weight<PER>(w[s], c.side[s].weight, c.weight_dtype, e0, c.d);

  for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < c.rows;
       first += (int64_t)gridDim.x * GROUPS) {
    // (groups behind the last row repeat it and write nothing)
    const bool there = first + grp < c.rows;
    const int64_t row = there ? first + grp : c.rows - 1;
    float cs[PER], sn[PER];
    row_angles(c, row, lane, LANES, angle[grp][0], angle[grp][1]);
    wave_fence();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = e0 + i;
      cs[i] = 1.f;
      sn[i] = 0.f;
      if (e < 2 * c.rotated) {
        const int r = e < c.rotated ? e : e - c.rotated;
        cs[i] = angle[grp][0][padded(r)];
        sn[i] = angle[grp][1][padded(r)];
        // forward: the first of a pair loses, the second gains; back: reversed
        if ((e < c.rotated) != BACKWARD)
          sn[i] = -sn[i];
      }
    }
    wave_fence();

#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const NormRotateSide &side = c.side[s];
      const int before = s == 0 ? 0 : c.side[0].heads;
      const int begin = max(head0 - before, 0);
      const int end = min(stop - before, side.heads);
      const T *const x_row =
          static_cast<const T *>(side.x.data) + row * side.x.row + e0;
      const T *const g_row =
          static_cast<const T *>(side.dout.data) + row * side.dout.row + e0;
      T *const out_row =
          static_cast<T *>(side.out) + row * side.heads * c.d + e0;
      auto load = [&](const T *p, bool vec) {
        attn::u32x4 r = {0, 0, 0, 0};
        if (vec) {
          if (e0 < c.d)
            r = *reinterpret_cast<const attn::u32x4 *>(p);
        } else {
          T e[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i)
            e[i] = e0 + i < c.d ? p[i] : (T)0.f;
          __builtin_memcpy(&r, e, 16);
        }
        return r;
      };
      attn::u32x4 next_x[HEADS], next_g[HEADS];
      auto fetch = [&](int h0) {
#pragma unroll
        for (int k = 0; k < HEADS; ++k)
          if (h0 + k < end) {
            next_x[k] = load(x_row + (h0 + k) * side.x.head, side.x.vec);
            if constexpr (BACKWARD)
              next_g[k] =
                  load(g_row + (h0 + k) * side.dout.head, side.dout.vec);
          }
      };
      fetch(begin);
      for (int h0 = begin; h0 < end; h0 += HEADS) {
        T raw[PER];
        float x[HEADS][PER], y[HEADS][PER], sum[HEADS], inv[HEADS];
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
          __builtin_memcpy(raw, &next_x[k], 16);
          sum[k] = 0.f;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            x[k][i] = (float)raw[i];
            sum[k] = fmaf(x[k][i], x[k][i], sum[k]);
          }
          if constexpr (BACKWARD) {
            __builtin_memcpy(raw, &next_g[k], 16);
#pragma unroll
            for (int i = 0; i < PER; ++i)
              y[k][i] = (float)raw[i];
          }
        }
        fetch(h0 + HEADS);
#pragma unroll
        for (int sh = 1; sh < LANES; sh <<= 1)
#pragma unroll
          for (int k = 0; k < HEADS; ++k)
            sum[k] += __shfl_xor(sum[k], sh);
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
          inv[k] = __builtin_amdgcn_rsqf(fmaf(sum[k], per_d, c.eps));
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            x[k][i] *= inv[k];
            if constexpr (!BACKWARD)
              y[k][i] = x[k][i] * w[s][i];
            line[grp][k][padded(e0 + i)] = y[k][i];
          }
        }
        wave_fence();
#pragma unroll
        for (int k = 0; k < HEADS; ++k)
#pragma unroll
          for (int i = 0; i < PER; ++i)
            y[k][i] = fmaf(line[grp][k][other[i]], sn[i], y[k][i] * cs[i]);
        wave_fence();
        if constexpr (BACKWARD) {
          float dot[HEADS];
#pragma unroll
          for (int k = 0; k < HEADS; ++k) {
            dot[k] = 0.f;
            const bool adds = there && h0 + k < end;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const float a = y[k][i] * x[k][i];
              dw[s][i] += adds ? a : 0.f;
              y[k][i] *= w[s][i];
              dot[k] = fmaf(y[k][i], x[k][i], dot[k]);
            }
          }
#pragma unroll
          for (int sh = 1; sh < LANES; sh <<= 1)
#pragma unroll
            for (int k = 0; k < HEADS; ++k)
              dot[k] += __shfl_xor(dot[k], sh);
#pragma unroll
          for (int k = 0; k < HEADS; ++k) {
            dot[k] *= per_d;
#pragma unroll
            for (int i = 0; i < PER; ++i)
              y[k][i] = inv[k] * fmaf(-x[k][i], dot[k], y[k][i]);
          }
        }
#pragma unroll
        for (int k = 0; k < HEADS; ++k) {
          if (h0 + k >= end || !there)
            break;
          T *out = out_row + (int64_t)(h0 + k) * c.d;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            raw[i] = (T)y[k][i];
          if (c.d % PER == 0) {
            if (e0 < c.d) {
              attn::u32x4 o;
              __builtin_memcpy(&o, raw, 16);
              __builtin_nontemporal_store(
                  o, reinterpret_cast<attn::u32x4 *>(out));
            }
          } else {
#pragma unroll
            for (int i = 0; i < PER; ++i)
              if (e0 + i < c.d)
                out[i] = raw[i];
          }
        }
      }
    }
  }

  if constexpr (BACKWARD) {
    // the workgroup's share of dw: group after group
    const int64_t at = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        line[grp][0][padded(e0 + i)] = dw[s][i];
      __syncthreads();
      for (int e = threadIdx.x; e < c.d; e += kRowThreads) {
        float sum = 0.f;
        for (int k = 0; k < GROUPS; ++k)
          sum += line[k][0][padded(e)];
        c.part[(at * 2 + s) * c.d + e] = sum;
      }
    }
  }
}

// dw[s][e] = sum over the workgroups: 16 columns a workgroup, 16 threads each.  1,024
// workgroups' 2 x 128 columns: 6 us, latency of 64 reads in steps of eight.
__global__ __launch_bounds__(256) void
sum_weights_kernel(NormRotateCall c, int blocks) {
  __shared__ float part[16][17];
  const int col = threadIdx.x % 16, stripe = threadIdx.x / 16;
  const int at = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (at < 2 * c.d)
#pragma unroll 8
    for (int b = stripe; b < blocks; b += 16)
      sum += c.part[(int64_t)b * 2 * c.d + at];
  part[stripe][col] = sum;
  __syncthreads();
  if (stripe == 0 && at < 2 * c.d) {
    sum = 0.f;
#pragma unroll
    for (int s = 0; s < 16; ++s)
      sum += part[s][col];
    void *out = c.side[at / c.d].dweight;
    const int e = at % c.d;
    if (out == nullptr)
      return;
    if (c.weight_dtype == 0)
      static_cast<float *>(out)[e] = sum;
    else if (c.weight_dtype == 2)
      static_cast<_Float16 *>(out)[e] = (_Float16)sum;
    else
      static_cast<__bf16 *>(out)[e] = (__bf16)sum;
  }
}

template <typename T, int LANES>
hipError_t launch_rows(const NormRotateCall &c, bool backward, int &blocks,
                       hipStream_t stream) {
  constexpr int GROUPS = kRowThreads / LANES;
  const int heads = c.side[0].heads + c.side[1].heads;
  // A workgroup takes all heads of its rows, whose angles it then forms once, where the
  // rows alone give every CU two workgroups, else a part of them.  (1,024 rows of 4 + 4
  // heads are 32 workgroups with 8 lanes a row, and 256 this way.)
  const int64_t want = (c.rows + GROUPS - 1) / GROUPS;
  int each = heads;
  while (each > 1 && want * ((heads + each - 1) / each) < 512)
    each = (each + 1) / 2;
  const int parts = (heads + each - 1) / each;
  const int most = std::max(1, kRowBlocks / parts);
  const dim3 grid((unsigned)std::min<int64_t>(want, most), (unsigned)parts);
  blocks = (int)(grid.x * grid.y);
  if (backward)
    norm_rotate_kernel<T, LANES, true>
        <<<grid, dim3(kRowThreads), 0, stream>>>(c, each);
  else
    norm_rotate_kernel<T, LANES, false>
        <<<grid, dim3(kRowThreads), 0, stream>>>(c, each);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const NormRotateCall &c, bool backward, int &blocks,
                       hipStream_t stream) {
  constexpr int PER = 16 / (int)sizeof(T);
  const int pieces = (c.d + PER - 1) / PER;
  return pieces <= 4    ? launch_rows<T, 4>(c, backward, blocks, stream)
         : pieces <= 8  ? launch_rows<T, 8>(c, backward, blocks, stream)
         : pieces <= 16 ? launch_rows<T, 16>(c, backward, blocks, stream)
         : pieces <= 32 ? launch_rows<T, 32>(c, backward, blocks, stream)
                        : launch_rows<T, 64>(c, backward, blocks, stream);
}

hipError_t launch_norm_rotate(const NormRotateCall &c, int dtype, bool backward,
                              int &blocks, hipStream_t stream) {
  return dtype == 0   ? launch_type<float>(c, backward, blocks, stream)
         : dtype == 2 ? launch_type<_Float16>(c, backward, blocks, stream)
                      : launch_type<__bf16>(c, backward, blocks, stream);
}

} // namespace

hipError_t norm_rotate_forward(const NormRotateCall &c, int dtype,
                               hipStream_t stream) {
  if (c.rows == 0)
    return hipSuccess;
  int blocks = 0;
  return launch_norm_rotate(c, dtype, false, blocks, stream);
}

size_t norm_rotate_workspace_bytes(int64_t, int d) {
  return sizeof(float) * 2 * (size_t)kRowBlocks * (size_t)d;
}

hipError_t norm_rotate_backward(NormRotateCall c, int dtype, void *workspace,
                                hipStream_t stream) {
  c.part = static_cast<float *>(workspace);
  int blocks = 0;
  if (c.rows > 0) {
    const hipError_t e = launch_norm_rotate(c, dtype, true, blocks, stream);
    if (e != hipSuccess)
      return e;
  }
  if (c.side[0].dweight || c.side[1].dweight)
    sum_weights_kernel<<<dim3((2 * c.d + 15) / 16), dim3(256), 0, stream>>>(
        c, blocks);
  return hipGetLastError();
}

} // namespace pca
