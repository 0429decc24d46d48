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
// Backward, with g the gradient turned back: dw = sum g x / r, dx = (g w - xhat mean(g
// w xhat)) / r.  Every workgroup adds up dw of its rows and a second kernel adds up the
// workgroups, in a fixed order.
#include "rows_ops.hpp"

#include "attention_impl.hpp"

#include <algorithm>

namespace pca {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowBlocks = 1024; // workgroups of the backward pass, at most

__device__ __forceinline__ float weight_at(const void *w, int dtype, int e) {
  return dtype == 0   ? static_cast<const float *>(w)[e]
         : dtype == 2 ? (float)static_cast<const _Float16 *>(w)[e]
                      : (float)static_cast<const __bf16 *>(w)[e];
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

// Rotates the PER elements from e0 that the lane holds (of a row in `line`).
template <int PER>
__device__ __forceinline__ void turn(float (&y)[PER], float *line, int e0,
                                     int d, int rotated, const float (&cs)[PER],
                                     const float (&sn)[PER]) {
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (e0 + i < d)
      line[padded(e0 + i)] = y[i];
  wave_fence();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = e0 + i;
    if (e < 2 * rotated) {
      const int other = e < rotated ? e + rotated : e - rotated;
      y[i] = fmaf(line[padded(other)], sn[i], y[i] * cs[i]);
    }
  }
  wave_fence();
}

// LANES lanes a row.  `heads_each`: heads that a group takes (side 0's, then side 1's).
template <typename T, int LANES, bool BACKWARD>
__global__ __launch_bounds__(kRowThreads) void
norm_rotate_kernel(NormRotateCall c, int heads_each) {
  constexpr int PER = 16 / (int)sizeof(T), DP = PER * LANES;
  constexpr int LINE = DP + DP / 8 + 1;
  constexpr int GROUPS = kRowThreads / LANES;
  __shared__ float line[GROUPS][LINE];
  __shared__ float angle[GROUPS][2][DP / 2 + DP / 16 + 1];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int e0 = lane * PER;
  const int heads = c.side[0].heads + c.side[1].heads;
  const int parts = (heads + heads_each - 1) / heads_each;
  float w[2][PER], dw[2][PER];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      w[s][i] = 1.f;
      dw[s][i] = 0.f;
      if (c.side[s].weight && e0 + i < c.d)
        w[s][i] = weight_at(c.side[s].weight, c.weight_dtype, e0 + i);
    }

  const int64_t items = (int64_t)c.rows * parts;
  for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < items;
       first += (int64_t)gridDim.x * GROUPS) {
    const int64_t item = first + grp;
    const bool there = item < items; // (lanes of a group agree)
    const int64_t row = there ? item / parts : 0;
    const int head0 = there ? (int)(item % parts) * heads_each : 0;
    float cs[PER], sn[PER];
    if (there)
      row_angles(c, row, lane, LANES, angle[grp][0], angle[grp][1]);
    wave_fence();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = e0 + i;
      cs[i] = 1.f;
      sn[i] = 0.f;
      if (there && e < 2 * c.rotated) {
        const int r = e < c.rotated ? e : e - c.rotated;
        cs[i] = angle[grp][0][padded(r)];
        sn[i] = angle[grp][1][padded(r)];
        // forward: the first of a pair loses, the second gains; back: reversed
        if ((e < c.rotated) != BACKWARD)
          sn[i] = -sn[i];
      }
    }
    wave_fence();
    const int stop = there ? min(head0 + heads_each, heads) : 0;
    for (int h = head0; h < stop; ++h) {
      const int s = h < c.side[0].heads ? 0 : 1;
      const NormRotateSide &side = c.side[s];
      const int head = s == 0 ? h : h - c.side[0].heads;
      T raw[PER];
      float x[PER], sum = 0.f;
      const attn::u32x4 v =
          attn::load_piece<T, DP>(side.x, row, head, lane, c.d);
      __builtin_memcpy(raw, &v, 16);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        x[i] = (float)raw[i];
        sum = fmaf(x[i], x[i], sum);
      }
#pragma unroll
      for (int sh = 1; sh < LANES; sh <<= 1)
        sum += __shfl_xor(sum, sh);
      const float inv = 1.f / __builtin_sqrtf(sum / (float)c.d + c.eps);
      float y[PER];
      if constexpr (!BACKWARD) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          y[i] = x[i] * inv * w[s][i];
        turn<PER>(y, line[grp], e0, c.d, c.rotated, cs, sn);
      } else {
        const attn::u32x4 gv =
            attn::load_piece<T, DP>(side.dout, row, head, lane, c.d);
        __builtin_memcpy(raw, &gv, 16);
#pragma unroll
        for (int i = 0; i < PER; ++i)
          y[i] = (float)raw[i];
        turn<PER>(y, line[grp], e0, c.d, c.rotated, cs, sn);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          x[i] *= inv;
          dw[s][i] = fmaf(y[i], x[i], dw[s][i]);
          y[i] *= w[s][i];
          dot = fmaf(y[i], x[i], dot);
        }
#pragma unroll
        for (int sh = 1; sh < LANES; sh <<= 1)
          dot += __shfl_xor(dot, sh);
        dot /= (float)c.d;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          y[i] = inv * (y[i] - x[i] * dot);
      }
      T *out = static_cast<T *>(side.out) +
               (row * side.heads + head) * (int64_t)c.d + e0;
      if (c.d % PER == 0) {
        if (e0 < c.d) {
#pragma unroll
          for (int i = 0; i < PER; ++i)
            raw[i] = (T)y[i];
          attn::u32x4 o;
          __builtin_memcpy(&o, raw, 16);
          *reinterpret_cast<attn::u32x4 *>(out) = o;
        }
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (e0 + i < c.d)
            out[i] = (T)y[i];
      }
    }
  }

  if constexpr (BACKWARD) {
    // the workgroup's share of dw: group after group
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        line[grp][padded(e0 + i)] = dw[s][i];
      __syncthreads();
      for (int e = threadIdx.x; e < c.d; e += kRowThreads) {
        float sum = 0.f;
        for (int k = 0; k < GROUPS; ++k)
          sum += line[k][padded(e)];
        c.part[((int64_t)blockIdx.x * 2 + s) * c.d + e] = sum;
      }
    }
  }
}

// dw[s][e] = sum over the workgroups: 16 columns a workgroup, 16 threads each.
__global__ __launch_bounds__(256) void
sum_weights_kernel(NormRotateCall c, int blocks) {
  __shared__ float part[16][17];
  const int col = threadIdx.x % 16, stripe = threadIdx.x / 16;
  const int at = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (at < 2 * c.d)
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
  // a group takes all heads of a row where the rows alone fill the chip
  int each = heads;
  while (each > 1 && (int64_t)c.rows * ((heads + each - 1) / each) / GROUPS < 512)
    each = (each + 1) / 2;
  const int64_t items = (int64_t)c.rows * ((heads + each - 1) / each);
  const int64_t want = (items + GROUPS - 1) / GROUPS;
  blocks = (int)std::min<int64_t>(want, backward ? kRowBlocks : 16384);
  if (backward)
    norm_rotate_kernel<T, LANES, true>
        <<<dim3(blocks), dim3(kRowThreads), 0, stream>>>(c, each);
  else
    norm_rotate_kernel<T, LANES, false>
        <<<dim3(blocks), dim3(kRowThreads), 0, stream>>>(c, each);
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
