// Attention inside the examples of a batch: forward and backward kernels.
//
//   t_ij = scale q_i . k_j          u = cap tanh(t / cap)   (cap > 0; else u = t)
//   s_ij = u - slope_h |p_i - p_j|  over the rows j of row i's example
//   o_i  = sum_j exp(s_ij) v_j / sum_j exp(s_ij)
//
// and backwards, with P = exp(s - log sum exp s), delta_i = do_i . o_i:
//
//   dS = P (do_i . v_j - delta_i)   dT = dS (1 - (u / cap)^2)
//   dq = scale sum_j dT k_j   dk = scale sum_i dT q_i   dv = sum_i P do_i
//
// With 16-bit rows the forward pass also leaves what rounding took off o_i (`rest`):
// an error of delta_i would be the same for all j and add up, where those of P and dT,
// rounded for the matrix cores, do not.  dq and dk are 1.5 times as far from the exact
// ones as their own rounding without it (one in two rows with few near keys).
//
// Everything a kernel sums over lies along the matrix instruction's contraction and
// everything it owns along its columns: scores are formed transposed, S^T = K Q^T, so
// that a lane holds scores of ONE owned row (its column, lane % 16) and four
// neighbouring looped rows per 16 x 16 block.  The row's maximum and sum are then
// registers plus two exchanges between lanes, and the block's registers are already the
// right operand of the next product (O^T += V^T P^T): the order of the contraction is
// free as long as both operands use the same, so slot 8 g + j of a 32-wide step stands
// for row 16 (j / 4) + 4 g + j % 4 of the step, which is what the lane holds.  The left
// operand V^T comes transposed out of LDS (ds_read_tr16_b64) from rows stored as they
// are in memory.  In fp32 the matrix instruction takes one element per lane and the
// same layouts hold with steps of 16.
//
// Owned rows of the forward and of dq are (query, head of the group) pairs, so that the
// heads that share a key head share its tiles as well; the kernel of dk and dv owns
// keys and loops over those pairs.  No atomics: the same call gives the same bits.
//
// A tile of owned rows may touch several examples.  Its spans (begin and end of each
// row's partner rows) are collected first; every span is walked in tiles of its own
// that hold nothing of another example (rows beyond it are zeros), and where a wave's
// columns belong to several examples the products are kept only in the columns that
// the span belongs to: values of other examples, infinities and NaN among them, reach
// nothing.  A tile costs 2.0 - 2.5 us of latency in a workgroup however few rows of it
// a span fills, so examples of a few rows pay for tiles of 64: 303 graphs of 6 rows take
// 91 us.  Neighbouring short spans in one tile, masked lane by lane, took 31 us there,
// but the masks' registers cost the long examples 10 - 24 % and were taken back.
//
// What bounds them (one MI355X; 16 clouds of 1,024 rows, 8 heads of 64, bf16, positions
// on three axes): the vector unit.  64 pairs of rows cost 17 - 19 vector instructions
// (exponential and square root at a quarter of the rate); 7 of them and the square root are
// the distance, which is the same for all heads and formed again for each of them, in each
// of the three kernels.  Forward 104 us, the vector unit busy for 81 % of the cycles and the
// matrix cores for 16; dq 120 us, 69 and 21 %; dk and dv 156 us, 53 and 21 %, with two
// waves per SIMD, which no longer cover each other's products, exchanges and barriers.
// Without bias and cap a forward call reaches 912 TFLOP/s with heads of 128 (4 examples
// of 4,096 rows, 8 heads, bf16: 301 us) and 687 with heads of 64, forward and backward 694
// and 639 (a product of 8,192^3: 1,261); fp32, where the matrix cores are busy for half of
// the cycles, 117 - 122 of 153, and 95 with the backward pass.
//
// Tiles come by loads that bypass the registers (request16), one tile ahead: with loads
// into registers and stores to LDS 4 examples of 4,096 rows with everything on took 1,312
// / 1,375 / 1,833 us instead of 576 / 680 / 964 (now 493 / 643 / 858).
//
// Exponentials, reciprocals, square roots and logarithms are the vector unit's own, off by
// a step of fp32; results below 2^-126 are zeros.
#pragma once

#include "attention.hpp"
#include "device_utils.hpp"

#include <type_traits>

namespace pca {
namespace attn {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kThreads = 256, kWaves = 4;

template <typename T> __device__ __forceinline__ float to_float(T v) {
  return (float)v;
}

// acc += a b: both operands 16 bytes of a lane, element 0 of the contraction first.
template <typename T>
__device__ __forceinline__ void mma(f32x4 &acc, u32x4 a, u32x4 b) {
  if constexpr (std::is_same<T, float>::value) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a);
    const f32x4 fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[c], fb[c], acc, 0, 0, 0);
  } else if constexpr (std::is_same<T, _Float16>::value) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc, 0, 0,
        0);
  } else {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0,
        0, 0);
  }
}

// Sizes that follow from the element type and the width of a head that a kernel is built
// for: what is computed goes by it, what lies in LDS by the next power of two.
template <typename T, int DP> struct Shape {
  static constexpr int SZ = sizeof(T);
  static constexpr int PER = 16 / SZ;          // elements of 16 bytes
  static constexpr int LDS = DP <= 32 ? 32 : DP <= 64 ? 64 : 128;
  static constexpr int CH = LDS / PER;         // 16-byte pieces of a row
  static constexpr int KS = (DP * SZ + 63) / 64; // steps of a product over d
  static constexpr int DB = DP / 16;           // 16-wide blocks over d
  static constexpr int BYTES = LDS * SZ;       // of a row in LDS
  static constexpr int KF = SZ == 2 ? 32 : 16; // rows of a step over rows
  static constexpr int FB = KF / 16;           // ... in blocks
  // A tile's rows lie in LDS one after the other, as the loads that bypass the
  // registers leave them.  Piece p of row r is kept at place p ^ turn(r).  The 16 lanes
  // that read 16 bytes each at a time are not neighbours: rows 0 - 3 and 12 - 15 of one
  // piece, 4 - 11 of the next (rows_operand).  With 16-bit elements pairs of pieces of 8
  // neighbouring rows are read as well (turned_operand).  Both then lie on 64 different
  // banks; rows r and r + 8 of 16 have to be turned alike for that (told apart they cost
  // twice the cycles, a third of the LDS's in dq of heads of 128).
  __device__ __forceinline__ static int turn(int row) {
    constexpr int ROWS = CH >= 16 ? 1 : 16 / CH; // that fill the banks
    if (SZ == 4)
      return row / ROWS & (CH >= 16 ? 15 : CH - 1);
    return (row / ROWS & (CH >= 16 ? 7 : CH / 2 - 1)) << 1;
  }
};

// 16 bytes of row `row` at piece `piece`; zeros beyond d.
template <typename T, int DP>
__device__ __forceinline__ u32x4 load_piece(const HeadRows &x, int64_t row,
                                            int head, int piece, int d) {
  constexpr int PER = Shape<T, DP>::PER;
  const T *p = static_cast<const T *>(x.data) + row * x.row +
               (int64_t)head * x.head + piece * PER;
  u32x4 r = {0, 0, 0, 0};
  if (x.vec) {
    if (piece * PER < d)
      r = *reinterpret_cast<const u32x4 *>(p);
  } else {
    T e[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      e[i] = piece * PER + i < d ? p[i] : (T)0.f;
    __builtin_memcpy(&r, e, 16);
  }
  return r;
}

// What rows behind the end of a span are read from.
static __device__ const uint32_t kZeros[4] = {0, 0, 0, 0};

// Loads that go from memory to LDS without registers: lane l's 16 (4) bytes to `lds` +
// 16 l (4 l).  Nothing waits for them but arrive().  (m0 is written and used inside one
// statement: the compiler keeps nothing in it between statements, and has it reserved, so
// that it cannot be named as clobbered.)
__device__ __forceinline__ void request16(const void *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\t"
               "s_nop 0\n\t"
               "global_load_lds_dwordx4 %0, off"
               :
               : "v"(from), "s"(lds)
               : "memory");
}
__device__ __forceinline__ void request16(const void *base, uint32_t offset,
                                          uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\t"
               "s_nop 0\n\t"
               "global_load_lds_dwordx4 %0, %1"
               :
               : "v"(offset), "s"(base), "s"(lds)
               : "memory");
}
__device__ __forceinline__ void request4(const void *from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\t"
               "s_nop 0\n\t"
               "global_load_lds_dword %0, off"
               :
               : "v"(from), "s"(lds)
               : "memory");
}
__device__ __forceinline__ void request4(const void *base, uint32_t offset,
                                         uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\t"
               "s_nop 0\n\t"
               "global_load_lds_dword %0, %1"
               :
               : "v"(offset), "s"(base), "s"(lds)
               : "memory");
}
// Everything this wave has requested is in LDS; then everything the others have.
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return (uint32_t)(uintptr_t)p; // (the low half of a generic address)
}

// Rows of looped tiles of one head of a tensor on their way to LDS: ROWS rows of [begin,
// end), zeros behind the end.  Pieces beyond d are left alone: the caller has cleared
// them.  A whole tile costs a thread nothing but the loads: its offset in a tile never
// changes, the tile's address is formed by the scalar unit.
template <typename T, int DP, int ROWS> struct Requests {
  using S = Shape<T, DP>;
  static constexpr int N = ROWS * S::CH / kThreads;      // per thread
  static constexpr int STEP = kThreads / S::CH;          // rows between them
  static constexpr int LANES = STEP % 16 == 0 ? 1 : 2;   // places turned alike
  static_assert(ROWS * S::CH % kThreads == 0, "tile does not fill the threads");
  const HeadRows &x;
  int d, wave;
  uint32_t row_bytes;     // of the vector path
  uint32_t offset[LANES]; // bytes of this thread's first pieces from a tile's row
  bool on[LANES];         // they lie in d

  __device__ __forceinline__ Requests(const HeadRows &rows, int width)
      : x(rows), d(width), row_bytes((uint32_t)(rows.row * S::SZ)) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int l = 0; l < LANES; ++l) {
      const int p = piece(threadIdx.x / S::CH + l * STEP);
      offset[l] = (uint32_t)(threadIdx.x / S::CH) * row_bytes + p * 16;
      on[l] = p * S::PER < d;
    }
  }
  __device__ __forceinline__ static int piece(int row) {
    return threadIdx.x % S::CH ^ S::turn(row);
  }
  __device__ __forceinline__ void operator()(int begin, int end, int head,
                                             char *tile) const {
    const char *const first =
        static_cast<const char *>(x.data) + (int64_t)head * x.head * S::SZ;
    uint32_t lds = lds_address(tile) + wave * 1024;
    if (x.vec && begin + ROWS <= end) {
      const char *from = first + (uint64_t)(uint32_t)begin * row_bytes;
      if (LANES == 1) {
        if (on[0])
#pragma unroll
          for (int e = 0; e < N; ++e)
            request16(from + (uint64_t)(e * STEP * row_bytes), offset[0],
                      lds + kWaves * e * 1024);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (on[e % LANES])
            request16(from + (uint64_t)(e * STEP * row_bytes),
                      offset[e % LANES], lds + kWaves * e * 1024);
      }
      return;
    }
#pragma unroll 1
    for (int e = 0; e < N; ++e) {
      const int row = threadIdx.x / S::CH + e * STEP;
      const int p = piece(row);
      if (x.vec) {
        const char *from =
            first + (int64_t)(begin + row) * row_bytes + p * 16;
        if (p * S::PER < d)
          request16(begin + row < end ? (const void *)from
                                      : (const void *)kZeros,
                    lds + kWaves * e * 1024);
      } else {
        u32x4 v = {0, 0, 0, 0};
        if (begin + row < end)
          v = load_piece<T, DP>(x, begin + row, head, p, d);
        *reinterpret_cast<u32x4 *>(tile + (threadIdx.x + e * kThreads) * 16) =
            v;
      }
    }
  }
};

// Clears what requests leave alone.
template <int BYTES> __device__ __forceinline__ void clear_lds(char *p) {
  for (int i = threadIdx.x * 16; i < BYTES; i += kThreads * 16)
    *reinterpret_cast<u32x4 *>(p + i) = u32x4{0, 0, 0, 0};
  __syncthreads();
}

// Left operand with the tile's rows as its rows: row block `block`, step `ks` of d.
template <typename T, int DP>
__device__ __forceinline__ u32x4 rows_operand(const char *tile, int block,
                                              int ks) {
  using S = Shape<T, DP>;
  const int lane = threadIdx.x & 63, i = lane & 15;
  return *reinterpret_cast<const u32x4 *>(
      tile + (block * 16 + i) * S::BYTES +
      ((lane >> 4 ^ S::turn(i)) ^ ks * 4) * 16);
}

// Left operand with d as its rows (16 of block `db`) and the tile's rows from `row0` (a
// multiple of 16) as the contraction, in the order described above.
template <typename T, int DP>
__device__ __forceinline__ u32x4 turned_operand(const char *tile, int row0,
                                                int db) {
  using S = Shape<T, DP>;
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  if constexpr (S::SZ == 4) {
    u32x4 r;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int row = g * 4 + c;
      r[c] = *reinterpret_cast<const uint32_t *>(
          tile + (row0 + row) * S::BYTES +
          ((i >> 2 ^ S::turn(row)) ^ db * 4) * 16 + (i & 3) * 4);
    }
    return r;
  } else {
    // lane i of a group of 16 names 4 elements of row i / 4 and gets column i of
    // the 4 x 16 elements that the group names
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int row = g * 4 + (i >> 2);
    const char *p = tile + (row0 + row) * S::BYTES +
                    (((i & 3) >> 1 ^ S::turn(row)) ^ db * 2) * 16 + (i & 1) * 8;
    const s16x4 lo =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4 *)(p + 16 * S::BYTES));
    const u32x2 a = __builtin_bit_cast(u32x2, lo);
    const u32x2 b = __builtin_bit_cast(u32x2, hi);
    return u32x4{a[0], a[1], b[0], b[1]};
  }
}

// Right operand of a step over the looped rows from the blocks that a lane holds.
// Rounded to the element type: the matrix cores take nothing wider with 16-bit rows.
// Their sums stay in 32 bits.
template <typename T>
__device__ __forceinline__ u32x4 block_operand(const f32x4 *blocks) {
  if constexpr (std::is_same<T, float>::value) {
    return __builtin_bit_cast(u32x4, blocks[0]);
  } else {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[i] = (T)blocks[i >> 2][i & 3];
    u32x4 r;
    __builtin_memcpy(&r, e, 16);
    return r;
  }
}

// Four neighbouring elements of an output row.
template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v, int left, bool vec) {
  T e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    e[i] = (T)v[i];
  if (vec && left >= 4) {
    __builtin_memcpy(__builtin_assume_aligned(p, 4 * sizeof(T)), e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left)
        p[i] = e[i];
  }
}

// What rounding the elements of a row to T takes off.
template <typename T> __device__ __forceinline__ f32x4 rest4(f32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] -= (float)(T)v[i];
  return v;
}

// Over the four groups of 16 lanes, by exchanges in the vector unit: the two results of
// a swap of v with itself hold both partners' values.
template <typename Op>
__device__ __forceinline__ float across_groups(float v, Op op) {
  const uint32_t a = __float_as_uint(v);
  const auto x = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const uint32_t b =
      __float_as_uint(op(__uint_as_float(x[0]), __uint_as_float(x[1])));
  const auto y = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return op(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float across_groups_max(float v) {
  return across_groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float across_groups_sum(float v) {
  return across_groups(v, [](float a, float b) { return a + b; });
}

// tanh y, x = 2 y log2 e: (exp2(x) - 1) / (exp2(x) + 1), and near 0, where that difference
// would lose digits, the series (error 2e-8 relative below 0.35).
__device__ __forceinline__ float tanh_of(float x) {
  const float e = __builtin_amdgcn_exp2f(x);
  const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
  const float y = x * 0.34657359027997264f, z = y * y;
  const float near =
      y + y * z *
              (-0.33333333333f +
               z * (0.13333333333f +
                    z * (-0.05396825397f +
                         z * (0.02186948854f + z * -0.00886323553f))));
  return fabsf(y) < 0.35f ? near : far;
}

// Spans of the rows that a workgroup owns, in order, each cut into tiles.
template <int ROWS> struct Spans {
  int begin[ROWS], end[ROWS];
  int first[ROWS + 1]; // tiles before a span
  int count;
};

// Collects the spans of owned rows [row0, row0 + ROWS) (row / group is the row that has
// a span; no spans: all of the looped rows), whole workgroup; `tile`: rows of a tile.
template <int ROWS>
__device__ __forceinline__ void
collect_spans(Spans<ROWS> &s, const int2 *spans, int row0, int rows, int group,
              int all, int tile) {
  if (spans == nullptr) {
    if (threadIdx.x == 0) {
      s.begin[0] = 0;
      s.end[0] = all;
      s.first[0] = 0;
      s.first[1] = (all + tile - 1) / tile;
      s.count = 1;
    }
    __syncthreads();
    return;
  }
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int count = 0;
    int2 last = make_int2(-1, -1);
#pragma unroll
    for (int base = 0; base < ROWS; base += 64) {
      const int row = row0 + base + lane;
      const bool there = base + lane < ROWS && row < rows;
      int2 v = make_int2(-1, -1);
      if (there)
        v = spans[row / group];
      int2 before;
      before.x = __shfl_up(v.x, 1);
      before.y = __shfl_up(v.y, 1);
      if (lane == 0)
        before = last;
      const bool head = there && v.x < v.y &&
                        (v.x != before.x || v.y != before.y);
      const unsigned long long heads = __ballot(head);
      if (head) {
        const int at = count + __popcll(heads & ((1ull << lane) - 1));
        s.begin[at] = v.x;
        s.end[at] = v.y;
      }
      count += __popcll(heads);
      last.x = __shfl(v.x, 63);
      last.y = __shfl(v.y, 63);
    }
    if (lane == 0) {
      s.count = count;
      s.first[0] = 0;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int sum = 0;
    for (int i = 0; i < s.count; ++i) {
      sum += (s.end[i] - s.begin[i] + tile - 1) / tile;
      s.first[i + 1] = sum;
    }
  }
  __syncthreads();
}

// The tiles of this workgroup's piece, in order: rows [begin, end of the tile or of its
// span), the whole list once for each of `rounds` heads.  All of it is the same in every
// lane and kept in scalar registers.
template <int ROWS> struct Walk {
  const Spans<ROWS> &s;
  int left, round, count, span, first, begin, end, tile;
  __device__ __forceinline__ Walk(const Spans<ROWS> &spans, int rounds,
                                  int piece, int pieces, int tile_rows)
      : s(spans), left(0), round(0), span(0), first(0), begin(0), end(0),
        tile(tile_rows) {
    count = __builtin_amdgcn_readfirstlane(s.count);
    const int once =
        count > 0 ? __builtin_amdgcn_readfirstlane(s.first[count]) : 0;
    const int total = once * rounds;
    // (the first total % pieces pieces have one tile more)
    const int share = pieces == 1 ? total : total / pieces;
    const int more = total - share * pieces;
    int at = share * piece + min(piece, more);
    left = share + (piece < more);
    if (left > 0) {
      if (rounds > 1) {
        round = at / once;
        at -= round * once;
      }
      while (__builtin_amdgcn_readfirstlane(s.first[span + 1]) <= at)
        ++span;
      enter();
      begin += (at - __builtin_amdgcn_readfirstlane(s.first[span])) * tile;
    }
  }
  __device__ __forceinline__ void enter() {
    first = begin = __builtin_amdgcn_readfirstlane(s.begin[span]);
    end = __builtin_amdgcn_readfirstlane(s.end[span]);
  }
  __device__ __forceinline__ bool there() const { return left > 0; }
  __device__ __forceinline__ void next() {
    --left;
    begin += tile;
    if (begin >= end && left > 0) { // (no span is empty)
      if (++span == count) {
        span = 0;
        ++round;
      }
      enter();
    }
  }
};

// The work of workgroup `block`: which tile of owned rows, which key head, which piece
// of the looped rows.  Workgroups of an XCD (every eighth) take neighbouring tiles of
// the same key head: they read the same rows, through one L2.  (Runs of 8 to 32
// workgroups dealt to the XCDs by turns: 79 us instead of 71 where long and short
// examples follow each other.)
struct Place {
  int tile, head, piece, tiles;
  __device__ __forceinline__ Place(int number, int heads, int pieces)
      : tiles(number) {
    // (blocks of an XCD: a grid that is no multiple of 8 leaves the first ones one
    // more)
    const int grid = tiles * heads * pieces, x = blockIdx.x & 7;
    const int b = x * (grid >> 3) + min(x, grid & 7) + (blockIdx.x >> 3);
    piece = b % pieces;
    tile = b / pieces % tiles;
    head = b / pieces / tiles;
  }
};

// Waves per SIMD that the registers are cut to: four where the sums of one block of
// columns leave room for them (five or six for heads of 32 were no faster), else two; the
// waves that divide tiles of wide heads among them come one to a SIMD, and LDS holds no
// more of them anyway.
template <typename T, int DP, int RB, int WK> constexpr int waves_wanted() {
  if (WK > 1)
    return DP > 64 ? 1 : 2;
  return sizeof(T) == 2 && DP <= 64 && RB == 1 ? 4 : 2;
}

// Rows of looped tiles per wave and step: the tile's 16-byte pieces fill the threads.
// (Tiles of 32 rows for 16-bit heads of 128, so that two workgroups share a CU's LDS, were
// slower: forward 609 us against 575, dk and dv 1,110 against 908.)
template <typename T, int WK> struct Looped {
  static constexpr int wave = WK == 1 ? (sizeof(T) == 2 ? 64 : 32)
                                      : (sizeof(T) == 2 ? 32 : 16);
  static constexpr int tile = wave * WK;
};

// Pieces that the looped rows of a tile of owned rows [first, last] are cut into, up to
// c.splits: as many as leave each some tiles (least_rows), so that short examples stay
// whole and long ones are shared, whatever is next to them.  Known from two spans; the
// workgroups of the others end at once.
template <typename T>
__device__ __forceinline__ int
pieces_in_use(const AttentionCall &c, const int2 *spans, int first, int last,
              int all, int rounds, const Place &place) {
  if (c.splits == 1)
    return 1;
  int rows = all;
  if (spans)
    rows = __builtin_amdgcn_readfirstlane(spans[last].y - spans[first].x);
  const int n = min(
      max((int)((int64_t)rows * rounds / least_rows(sizeof(T))), 1),
      c.splits);
  if (place.piece == 0 && threadIdx.x == 0)
    c.pieces[place.head * place.tiles + place.tile] = n;
  return n;
}

// A lane's owned column.
struct Column {
  bool valid = false;
  int row = 0, head = 0; // of the query or key tensor
  int2 span = {0, 0};
  float slope = 0.f; // times log2 e
  float p[3] = {0.f, 0.f, 0.f};
};

__device__ __forceinline__ void load_position(float (&p)[3], const float *pos,
                                              int64_t row, int axes) {
#pragma unroll
  for (int a = 0; a < 3; ++a)
    p[a] = a < axes ? pos[row * axes + a] : 0.f;
}

__device__ __forceinline__ Column query_column(const AttentionCall &c, int row,
                                               int group, int head0) {
  Column r;
  r.valid = row < c.nq * group;
  if (r.valid) {
    r.row = row / group;
    r.head = head0 + row % group;
    r.span = c.spans_q ? c.spans_q[r.row] : make_int2(0, c.nk);
    if (c.slope) {
      r.slope = c.slope[r.head] * kLog2e;
      load_position(r.p, c.pos_q, r.row, c.axes);
    }
  }
  return r;
}

// Which of a wave's columns a span belongs to.
template <int RB> struct Members {
  int span = -1;
  bool in[RB];
  bool some = false, mixed = false; // any column; some and not all
  __device__ __forceinline__ void of(int number, int begin, int end,
                                     const Column (&col)[RB]) {
    if (number == span)
      return;
    span = number;
    bool any = false, all = true;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      in[rb] = col[rb].span.x == begin && col[rb].span.y == end;
      any |= in[rb] && col[rb].valid;
      all &= in[rb] || !col[rb].valid;
    }
    some = __ballot(any) != 0;
    mixed = __ballot(!all) != 0;
  }
};

// Sums of a wave's columns: blocks of d, blocks of columns.
template <typename T, int DP, int RB> using Sums = f32x4[Shape<T, DP>::DB][RB];

// acc += (rows of the tile from row0, turned) p.  Where the columns belong to several
// examples, only those that the tile belongs to: the others' sums stay as they are,
// whatever the tile holds.
template <typename T, int DP, int RB>
__device__ __forceinline__ void add_product(Sums<T, DP, RB> &acc,
                                            const char *tile, int row0,
                                            const u32x4 (&p)[RB],
                                            const Members<RB> &members) {
  using S = Shape<T, DP>;
  if (members.mixed) {
#pragma unroll
    for (int db = 0; db < S::DB; ++db) {
      const u32x4 a = turned_operand<T, DP>(tile, row0, db);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        f32x4 t = acc[db][rb];
        mma<T>(t, a, p[rb]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[db][rb][r] = members.in[rb] ? t[r] : acc[db][rb][r];
      }
    }
  } else {
#pragma unroll
    for (int db = 0; db < S::DB; ++db) {
      const u32x4 a = turned_operand<T, DP>(tile, row0, db);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        mma<T>(acc[db][rb], a, p[rb]);
    }
  }
}

// Scores in units of log 2 less `base` (per block and row of it), from products.  With
// a cap, `flat` gets 1 - tanh^2 (in fp32) or a quarter of it: kFlatUp.
template <typename T>
constexpr float kFlatUp = std::is_same<T, float>::value ? 1.f : 4.f;

// Up to which cap 16-bit rows take the short form, cap (1 - 2 w) with the cap itself in
// `base`: an exponential and a reciprocal, but what it rounds is as large as the cap, so
// a score is off by 1.7e-7 cap: 2e-5 here, a 24th of what rounding a weight to fp16 takes
// off.  Beyond, and in fp32, a score is as exact as its own size (tanh_of): 16,384 rows of
// 8 heads of 128 in four examples, bf16, forward 509 us instead of 361, with the backward
// pass 1,999 instead of 1,595.
constexpr float kShortCap = 128.f;
template <typename T>
__device__ __forceinline__ bool short_cap(const AttentionCall &c) {
  return !std::is_same<T, float>::value && c.cap <= kShortCap;
}

// What cap_scores adds to every score: it wants `base` less this.
template <typename T>
__device__ __forceinline__ float under_cap(const AttentionCall &c) {
  return c.cap > 0.f && short_cap<T>(c) ? c.cap * kLog2e : 0.f;
}

template <typename T, bool SHORT, bool FLAT>
__device__ __forceinline__ void cap_scores(f32x4 &s, const AttentionCall &c,
                                           f32x4 base, f32x4 *flat) {
  const float in = c.under_tanh, out = c.cap * kLog2e;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if constexpr (SHORT) {
      // tanh = 1 - 2 w (the 1 is in base: under_cap), 1 - tanh^2 = 4 (w - w^2)
      const float w =
          __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[r] * in) + 1.f);
      s[r] = fmaf(w, -2.f * out, -base[r]);
      if constexpr (FLAT)
        (*flat)[r] = fmaf(-w, w, w);
    } else {
      const float t = tanh_of(s[r] * in);
      s[r] = fmaf(t, out, -base[r]);
      if constexpr (FLAT)
        (*flat)[r] = fmaf(-t, t, 1.f) * (1.f / kFlatUp<T>);
    }
  }
}
__device__ __forceinline__ f32x4 all4(float v) { return f32x4{v, v, v, v}; }

// Takes slope times distance off: p of the columns, `pos` of the looped rows.
__device__ __forceinline__ float far_by(const float (&p)[3], float x) {
  return fabsf(p[0] - x);
}
__device__ __forceinline__ float far_by(const float (&p)[3], float x, float y,
                                        float z) {
  const float a = p[0] - x, b = p[1] - y, e = p[2] - z;
  return __builtin_amdgcn_sqrtf(fmaf(e, e, fmaf(b, b, a * a)));
}

// Numbers of rows [begin, end) to LDS, `stride` apart in memory.
template <int KT>
__device__ __forceinline__ void request_numbers(const float *from, int stride,
                                                int begin, int end,
                                                float (&lds)[KT]) {
  const int lane = threadIdx.x & 63;
  const int row0 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64;
  if (row0 >= KT || (KT < 64 && lane >= KT))
    return;
  const float *base = from + (int64_t)(begin + row0) * stride;
  const uint32_t to = lds_address(&lds[row0]);
  if (begin + KT <= end)
    request4(base, (uint32_t)(lane * stride) * 4u, to);
  else
    request4(begin + row0 + lane < end ? (const void *)(base + lane * stride)
                                       : (const void *)kZeros,
             to);
}
// Positions, axis by axis (the third of two stays as it is: cleared).
template <int KT>
__device__ __forceinline__ void request_positions(const float *pos, int begin,
                                                  int end, int axes,
                                                  float (*lds)[KT]) {
  request_numbers<KT>(pos, axes, begin, end, lds[0]);
  if (axes > 1)
    request_numbers<KT>(pos + 1, axes, begin, end, lds[1]);
  if (axes > 2)
    request_numbers<KT>(pos + 2, axes, begin, end, lds[2]);
}

// The four looped rows of a block that a lane has scores of: `at`, at + 1, ...
template <int RB, int NB, int KT>
__device__ __forceinline__ void take_distance(f32x4 (&s)[RB][NB],
                                              const AttentionCall &c,
                                              const Column (&col)[RB],
                                              const float (&pos)[3][KT],
                                              int part) {
  const int g = (threadIdx.x & 63) >> 4;
  if (c.axes == 1) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int at = part + b * 16 + g * 4;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(&pos[0][at]);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[rb][b][r] =
              fmaf(-col[rb].slope, far_by(col[rb].p, x[r]), s[rb][b][r]);
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int at = part + b * 16 + g * 4;
      const f32x4 x = *reinterpret_cast<const f32x4 *>(&pos[0][at]);
      const f32x4 y = *reinterpret_cast<const f32x4 *>(&pos[1][at]);
      const f32x4 z = *reinterpret_cast<const f32x4 *>(&pos[2][at]);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[rb][b][r] = fmaf(-col[rb].slope,
                             far_by(col[rb].p, x[r], y[r], z[r]), s[rb][b][r]);
    }
  }
}

// ---- forward ------------------------------------------------------------------

// A row's largest weight is 2^this when what is subtracted is set.  Rounded for the matrix
// cores, fp16 weights end at 2^-25: with 7 bits above 1 what is lost of a row is below
// 2^-32 of its largest weight each, with none (2^-25 each) 20,000 keys that far below one
// other vanish from the products and stay in the sum, 0.06 % of it.  Up to 2^15 fits.
template <typename T>
constexpr float kWeightBits = std::is_same<T, _Float16>::value ? 7.f : 0.f;

// Rows of a wave's columns: RB blocks of 16.  WK waves share the same columns and
// divide every tile among them (few rows); the others own columns of their own.
//
// One pass over the keys: with m what is subtracted so far, l the weights' sum,
//
//   l' = l 2^(m - m') + sum_j 2^(s_j - m')     o' = o 2^(m - m') + sum_j 2^(s_j - m') v_j
//
// where m' differs from m only if a weight would be above 2^8 (fp16 2^15, see kWeightBits),
// in 32-bit sums, and nearly all tiles skip the scaling.
//
// Bound by the vector unit (see above) where rows are many; by latency where they are
// few: one cloud of 1,024 rows, 4 heads of 32, fp32, in pieces, 17 us; 32 single queries
// over 8,192 rows at most, 2 key heads of 128, bf16, 35 us = 4.2 TB/s of keys and values.
template <typename T, int DP, int RB, int WK>
__global__ __launch_bounds__(kThreads, (waves_wanted<T, DP, RB, WK>())) void
attention_forward_kernel(AttentionCall c) {
  using S = Shape<T, DP>;
  constexpr int WQ = kWaves / WK, ROWS = RB * 16 * WQ;
  constexpr int KW = Looped<T, WK>::wave, KT = Looped<T, WK>::tile;
  constexpr int KB = KW / 16;
  constexpr int TILE = KT * S::BYTES;
  __shared__ __attribute__((aligned(16))) char lds_tiles[4 * TILE];
  __shared__ __attribute__((aligned(16))) float lds_pos[2][3][KT];
  __shared__ float lds_ml[kWaves][16][2];
  __shared__ Spans<ROWS> spans;

  const int group = c.hq / c.hk, rows = c.nq * group;
  const Place place((rows + ROWS - 1) / ROWS, c.hk, c.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int wq = wave / WK;
  const int part = __builtin_amdgcn_readfirstlane(wave % WK * KW);
  const int row0 = place.tile * ROWS;
  const int pieces =
      pieces_in_use<T>(c, c.spans_q, row0 / group,
                           (min(row0 + ROWS, rows) - 1) / group, c.nk, 1, place);
  if (place.piece >= pieces)
    return; // (the whole workgroup)

  Column col[RB];
  u32x4 q[RB][S::KS];
  f32x4 acc[S::DB][RB];
  // what is subtracted from the scores, the weights' sum (of this lane's rows), and
  // whether there has been a row
  float m[RB], l[RB];
  bool seen[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    col[rb] = query_column(c, row0 + (wq * RB + rb) * 16 + i, group,
                           place.head * group);
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
      q[rb][ks] = u32x4{0, 0, 0, 0};
      if (col[rb].valid)
        q[rb][ks] = load_piece<T, DP>(c.q, col[rb].row, col[rb].head,
                                      ks * 4 + g, c.d);
    }
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      acc[db][rb] = f32x4{0, 0, 0, 0};
    m[rb] = l[rb] = 0.f;
    seen[rb] = false;
  }

  const Requests<T, DP, KT> request_k(c.k, c.d), request_v(c.v, c.d);
  collect_spans<ROWS>(spans, c.spans_q, row0, rows, group, c.nk, KT);
  // Two buffers: while a tile is worked on, the next one is on its way.
  auto request = [&](int begin, int end, int buffer) {
    char *tile = lds_tiles + buffer * 2 * TILE;
    request_k(begin, end, place.head, tile);
    request_v(begin, end, place.head, tile + TILE);
    if (c.slope)
      request_positions<KT>(c.pos_k, begin, end, c.axes, lds_pos[buffer]);
  };
  if (c.axes == 2)
    clear_lds<sizeof(lds_pos)>(reinterpret_cast<char *>(lds_pos));
  if (c.d < S::LDS)
    clear_lds<4 * TILE>(lds_tiles);

  Walk<ROWS> walk(spans, 1, place.piece, pieces, KT);
  int buffer = 0;
  Members<RB> members;
  if (walk.there())
    request(walk.begin, walk.end, 0);
  for (; walk.there(); buffer ^= 1) {
    const int begin = walk.begin, end = walk.end;
    members.of(walk.span, walk.first, end, col);
    arrive();
    walk.next();
    if (walk.there())
      request(walk.begin, walk.end, buffer ^ 1);
    const char *lds_k = lds_tiles + buffer * 2 * TILE + part * S::BYTES;
    const char *lds_v = lds_k + TILE;

    if (!members.some || begin + part >= end)
      continue;
    const bool(&in)[RB] = members.in;
    const bool mixed = members.mixed;
    const bool cut = begin + part + KW > end;

    f32x4 s[RB][KB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        s[rb][kb] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int ks = 0; ks < S::KS; ++ks) {
        const u32x4 a = rows_operand<T, DP>(lds_k, kb, ks);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          mma<T>(s[rb][kb], a, q[rb][ks]);
      }

    auto capped = [&](auto is_short) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          cap_scores<T, decltype(is_short)::value, false>(
              s[rb][kb], c, all4(m[rb] - under_cap<T>(c)), nullptr);
    };
    if (c.cap > 0.f) {
      if (__builtin_expect(short_cap<T>(c), 1))
        capped(std::true_type());
      else
        capped(std::false_type());
    } else {
      const float in = c.scale * kLog2e;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[rb][kb][r] = fmaf(s[rb][kb][r], in, -m[rb]);
    }
    if (c.slope)
      take_distance<RB, KB>(s, c, col, lds_pos[buffer], part);
    if (cut || mixed) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!in[rb] || begin + part + kb * 16 + g * 4 + r >= end)
              s[rb][kb][r] = -__builtin_inff();
    }
    float top[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      top[rb] = s[rb][0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          top[rb] = fmaxf(top[rb], s[rb][kb][r]);
    }

    // What is subtracted moves only when a weight would be more than 256 times what
    // the largest was when it was set, far from any limit: most tiles leave the sums
    // as they are.
    bool move[RB], moves = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      top[rb] = across_groups_max(top[rb]);
      move[rb] = top[rb] > kWeightBits<T> + 8.f ||
                 (!seen[rb] && top[rb] > -__builtin_inff());
      moves |= move[rb];
    }
    if (__ballot(moves) != 0) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const float by = move[rb] ? top[rb] - kWeightBits<T> : 0.f;
        const float keep =
            move[rb] && seen[rb] ? __builtin_amdgcn_exp2f(-by) : 1.f;
        seen[rb] |= move[rb];
        m[rb] += by;
        l[rb] *= keep;
#pragma unroll
        for (int db = 0; db < S::DB; ++db)
          acc[db][rb] *= keep;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[rb][kb][r] -= by;
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(s[rb][kb][r]);
          s[rb][kb][r] = e;
          l[rb] += e;
        }

#pragma unroll
    for (int f = 0; f < KB / S::FB; ++f) {
      u32x4 p[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        p[rb] = block_operand<T>(&s[rb][f * S::FB]);
      add_product<T, DP, RB>(acc, lds_v, f * S::KF, p, members);
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    l[rb] = across_groups_sum(l[rb]);
    if (!seen[rb] && l[rb] == 0.f) // (not: scores that were all NaN)
      m[rb] = -__builtin_inff();   // nothing to be put together with others
  }

  if constexpr (WK > 1) {
    // the waves' shares of the same 16 columns: one maximum, then sums in the order
    // of the waves
    static_assert(RB == 1 && WQ == 1, "one block of columns");
    static_assert(kWaves * 16 * (DP + 4) * 4 <= 4 * TILE, "sums do not fit");
    auto lds_acc = reinterpret_cast<float(*)[16][DP + 4]>(lds_tiles);
    if (g == 0) {
      lds_ml[wave][i][0] = m[0];
      lds_ml[wave][i][1] = l[0];
    }
    __syncthreads();
    float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
    for (int w = 0; w < WK; ++w)
      top = fmaxf(top, lds_ml[w][i][0]);
#pragma unroll
    for (int w = 0; w < WK; ++w)
      if (lds_ml[w][i][0] != -__builtin_inff())
        sum += lds_ml[w][i][1] * __builtin_amdgcn_exp2f(lds_ml[w][i][0] - top);
    const float keep = m[0] == -__builtin_inff()
                           ? 1.f
                           : __builtin_amdgcn_exp2f(m[0] - top);
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      *reinterpret_cast<f32x4 *>(&lds_acc[wave][i][db * 16 + g * 4]) =
          acc[db][0] * keep;
    __syncthreads();
    m[0] = top;
    l[0] = sum;
    // wave w finishes blocks w, w + 4, ... of d
#pragma unroll
    for (int db = 0; db < S::DB; ++db) {
      f32x4 t = {0, 0, 0, 0};
      if (db % kWaves == wave) {
#pragma unroll
        for (int w = 0; w < WK; ++w)
          t += *reinterpret_cast<const f32x4 *>(&lds_acc[w][i][db * 16 + g * 4]);
      }
      acc[db][0] = t;
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    if (!col[rb].valid)
      continue;
    const int64_t at = (int64_t)col[rb].row * c.hq + col[rb].head;
    const bool vec = c.d % 4 == 0;
    const bool first = g == 0 && (WK == 1 || wave == 0);
    if (pieces > 1) {
      const int64_t o = (int64_t)place.piece * c.nq * c.hq + at;
#pragma unroll
      for (int db = 0; db < S::DB; ++db) {
        if (WK > 1 && db % kWaves != wave)
          continue;
        const int e = db * 16 + g * 4;
        store4<float>(c.part + o * c.d + e, acc[db][rb], c.d - e, vec);
      }
      if (first) {
        c.part_ml[o * 2] = m[rb];
        c.part_ml[o * 2 + 1] = l[rb];
      }
    } else {
      const float inv = l[rb] == 0.f ? 0.f : 1.f / l[rb];
#pragma unroll
      for (int db = 0; db < S::DB; ++db) {
        if (WK > 1 && db % kWaves != wave)
          continue;
        const int e = db * 16 + g * 4;
        const f32x4 v = acc[db][rb] * inv;
        store4<T>(static_cast<T *>(c.out) + at * c.d + e, v, c.d - e, vec);
        if (c.rest)
          store4<T>(static_cast<T *>(c.rest) + at * c.d + e, rest4<T>(v),
                    c.d - e, vec);
      }
      if (first && c.lse)
        c.lse[(int64_t)col[rb].head * c.nq + col[rb].row] =
            l[rb] == 0.f ? __builtin_inff()
                         : m[rb] + __builtin_amdgcn_logf(l[rb]);
    }
  }
}

// ---- backward -----------------------------------------------------------------

// Factors that keep dS inside fp16's range, one per column: a power of two that grows
// or shrinks with the largest value met (bf16 and fp32 have the range of the sums and
// need none).  Sums are kept times the factor.
template <typename T> struct Range {
  static constexpr bool on = std::is_same<T, _Float16>::value;
  float factor = on ? 0x1p96f : 1.f;

  // Before a step with values up to `top` (of the lane): what the sums so far have to
  // be multiplied by.
  __device__ __forceinline__ bool moves(float top) const {
    return on && top * factor > 0x1p15f;
  }
  __device__ __forceinline__ float move(float top) {
    top = across_groups_max(top);
    if (!(top * factor > 0x1p15f))
      return 1.f;
    // (a finite top: exponents of values stay between those of fp32)
    const int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
    const float next = __uint_as_float((uint32_t)(min(127 + 12 - e, 250)) << 23);
    const float by = next / factor;
    if (e == 128)
      return 1.f; // an infinity or NaN stays what it is
    factor = next;
    return by;
  }
};

// Probabilities go to fp16 products times 2^14 (at most 1, and as small as one in the
// number of rows).
template <typename T>
constexpr float kWeightUp = std::is_same<T, _Float16>::value ? 0x1p14f : 1.f;

// WK waves' sums of the same 16 columns, in the order of the waves: afterwards wave w
// holds blocks w, w + 4, ... of d.
template <typename T, int DP, int RB, int WK>
__device__ __forceinline__ void
join_waves(Sums<T, DP, RB> &acc, float (*lds)[16][DP + 4]) {
  if constexpr (WK > 1) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    __syncthreads();
#pragma unroll
    for (int db = 0; db < Shape<T, DP>::DB; ++db)
      *reinterpret_cast<f32x4 *>(&lds[wave][i][db * 16 + g * 4]) = acc[db][0];
    __syncthreads();
#pragma unroll
    for (int db = 0; db < Shape<T, DP>::DB; ++db) {
      f32x4 t = {0, 0, 0, 0};
      if (db % kWaves == wave) {
#pragma unroll
        for (int w = 0; w < WK; ++w)
          t += *reinterpret_cast<const f32x4 *>(&lds[w][i][db * 16 + g * 4]);
      }
      acc[db][0] = t;
    }
  }
}

// A column's sums to memory: to the gradient, or to the piece's place.
template <typename T, int DP, int RB, int WK>
__device__ __forceinline__ void
store_columns(const Sums<T, DP, RB> &acc, int rb, void *out, float *part,
              int64_t at, int d, float factor) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const bool vec = d % 4 == 0;
#pragma unroll
  for (int db = 0; db < Shape<T, DP>::DB; ++db) {
    if (WK > 1 && db % kWaves != wave)
      continue;
    const int e = db * 16 + g * 4;
    const f32x4 v = acc[db][rb] * factor;
    if (part)
      store4<float>(part + at * d + e, v, d - e, vec);
    else
      store4<T>(static_cast<T *>(out) + at * d + e, v, d - e, vec);
  }
}

// dq of the rows that a workgroup owns, looping over keys; writes what the kernel of dk
// and dv takes of a row.
//
// Scores are formed again (P = 2^(s - lse): no memory for them), three products a pair.
// -delta is what the product with v starts from.  A step is as many rows as the matrix
// instruction's contraction, so that scores and dP of a step alone hold registers.  4 x
// 4,096 rows, 8 heads of 128, bf16, bias and cap: 643 us, 641 TFLOP/s of its three
// products; vector unit 50 %, matrix cores 28 %, LDS 31 % of the cycles at two waves per
// SIMD.  One block of columns per wave, since two spill (680 -
// 1,036 us).
template <typename T, int DP, int RB, int WK>
__global__ __launch_bounds__(kThreads, (waves_wanted<T, DP, RB, WK>())) void
attention_dq_kernel(AttentionCall c) {
  using S = Shape<T, DP>;
  constexpr int WQ = kWaves / WK, ROWS = RB * 16 * WQ;
  constexpr int KW = Looped<T, WK>::wave, KT = Looped<T, WK>::tile;
  constexpr int KB = KW / 16;
  constexpr int TILE = KT * S::BYTES;
  __shared__ __attribute__((aligned(16))) char lds_tiles[4 * TILE];
  __shared__ __attribute__((aligned(16))) float lds_pos[2][3][KT];
  __shared__ Spans<ROWS> spans;

  const int group = c.hq / c.hk, rows = c.nq * group;
  const Place place((rows + ROWS - 1) / ROWS, c.hk, c.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int wq = wave / WK;
  const int part = __builtin_amdgcn_readfirstlane(wave % WK * KW);
  const int row0 = place.tile * ROWS;
  const int pieces =
      pieces_in_use<T>(c, c.spans_q, row0 / group,
                           (min(row0 + ROWS, rows) - 1) / group, c.nk, 1, place);
  if (place.piece >= pieces)
    return; // (the whole workgroup)

  Column col[RB];
  u32x4 q[RB][S::KS], dout[RB][S::KS];
  f32x4 acc[S::DB][RB];
  float lse[RB], delta[RB];
  Range<T> range[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    col[rb] = query_column(c, row0 + (wq * RB + rb) * 16 + i, group,
                           place.head * group);
    HeadRows out, rest;
    out.data = c.out_in;
    out.row = (int64_t)c.hq * c.d;
    out.head = c.d;
    out.vec = c.d * S::SZ % 16 == 0;
    rest = out;
    rest.data = c.rest;
    float sum = 0.f;
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
      q[rb][ks] = dout[rb][ks] = u32x4{0, 0, 0, 0};
      if (col[rb].valid) {
        const int piece = ks * 4 + g;
        q[rb][ks] =
            load_piece<T, DP>(c.q, col[rb].row, col[rb].head, piece, c.d);
        dout[rb][ks] =
            load_piece<T, DP>(c.dout, col[rb].row, col[rb].head, piece, c.d);
        const u32x4 o =
            load_piece<T, DP>(out, col[rb].row, col[rb].head, piece, c.d);
        T a[S::PER], b[S::PER];
        __builtin_memcpy(a, &o, 16);
        __builtin_memcpy(b, &dout[rb][ks], 16);
#pragma unroll
        for (int e = 0; e < S::PER; ++e)
          sum = fmaf(to_float(a[e]), to_float(b[e]), sum);
        if (c.rest) {
          const u32x4 l =
              load_piece<T, DP>(rest, col[rb].row, col[rb].head, piece, c.d);
          __builtin_memcpy(a, &l, 16);
#pragma unroll
          for (int e = 0; e < S::PER; ++e)
            sum = fmaf(to_float(a[e]), to_float(b[e]), sum);
        }
      }
    }
    delta[rb] = across_groups_sum(sum);
    lse[rb] = __builtin_inff();
    if (col[rb].valid) {
      const int64_t at = (int64_t)col[rb].head * c.nq + col[rb].row;
      lse[rb] = c.lse[at];
      if (place.piece == 0 && g == 0 && (WK == 1 || wave == 0)) {
        // as the kernel of dk and dv adds them
        c.minus_delta[at] = -delta[rb];
        c.base[at] = lse[rb] - under_cap<T>(c);
      }
    }
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      acc[db][rb] = f32x4{0, 0, 0, 0};
  }

  const Requests<T, DP, KT> request_k(c.k, c.d), request_v(c.v, c.d);
  if (c.slope && blockIdx.x == 0)
    for (int h = threadIdx.x; h < c.hq; h += kThreads)
      c.minus_slope[h] = c.slope[h] * -kLog2e;
  collect_spans<ROWS>(spans, c.spans_q, row0, rows, group, c.nk, KT);
  // Two buffers: while a tile is worked on, the next one is on its way.
  auto request = [&](int begin, int end, int buffer) {
    char *tile = lds_tiles + buffer * 2 * TILE;
    request_k(begin, end, place.head, tile);
    request_v(begin, end, place.head, tile + TILE);
    if (c.slope)
      request_positions<KT>(c.pos_k, begin, end, c.axes, lds_pos[buffer]);
  };
  if (c.axes == 2)
    clear_lds<sizeof(lds_pos)>(reinterpret_cast<char *>(lds_pos));
  if (c.d < S::LDS)
    clear_lds<4 * TILE>(lds_tiles);

  Walk<ROWS> walk(spans, 1, place.piece, pieces, KT);
  int buffer = 0;
  Members<RB> members;
  if (walk.there())
    request(walk.begin, walk.end, 0);
  for (; walk.there(); buffer ^= 1) {
    const int begin = walk.begin, end = walk.end;
    members.of(walk.span, walk.first, end, col);
    arrive();
    walk.next();
    if (walk.there())
      request(walk.begin, walk.end, buffer ^ 1);
    const char *lds_k = lds_tiles + buffer * 2 * TILE + part * S::BYTES;
    const char *lds_v = lds_k + TILE;

    if (!members.some || begin + part >= end)
      continue;
    const bool(&in)[RB] = members.in;
    const bool mixed = members.mixed;
    const bool cut = begin + part + KW > end;

#pragma unroll
    for (int f = 0; f < KB / S::FB; ++f) {
      f32x4 s[RB][S::FB], ds[RB][S::FB], flat[RB][S::FB];
#pragma unroll
      for (int b = 0; b < S::FB; ++b) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          s[rb][b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          ds[rb][b] = all4(-delta[rb]);
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks) {
          const u32x4 ak = rows_operand<T, DP>(lds_k, f * S::FB + b, ks);
          const u32x4 av = rows_operand<T, DP>(lds_v, f * S::FB + b, ks);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            mma<T>(s[rb][b], ak, q[rb][ks]);
            mma<T>(ds[rb][b], av, dout[rb][ks]);
          }
        }
      }
      auto capped = [&](auto is_short) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            cap_scores<T, decltype(is_short)::value, true>(
                s[rb][b], c, all4(lse[rb] - under_cap<T>(c)), &flat[rb][b]);
      };
      if (c.cap > 0.f) {
        if (__builtin_expect(short_cap<T>(c), 1))
          capped(std::true_type());
        else
          capped(std::false_type());
      } else {
        const float in = c.scale * kLog2e;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[rb][b][r] = fmaf(s[rb][b][r], in, -lse[rb]);
      }
      if (c.slope)
        take_distance<RB, S::FB>(s, c, col, lds_pos[buffer], part + f * S::KF);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int b = 0; b < S::FB; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            ds[rb][b][r] *= __builtin_amdgcn_exp2f(s[rb][b][r]);
      if (c.cap > 0.f) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            ds[rb][b] *= flat[rb][b];
      }
      if (cut || mixed) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!in[rb] ||
                  begin + part + f * S::KF + b * 16 + g * 4 + r >= end)
                ds[rb][b][r] = 0.f;
      }
      if constexpr (Range<T>::on) {
        float top[RB];
        bool moves = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          top[rb] = 0.f;
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              top[rb] = fmaxf(top[rb], fabsf(ds[rb][b][r]));
          moves |= range[rb].moves(top[rb]);
        }
        if (__ballot(moves) != 0) {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const float by = range[rb].move(top[rb]);
#pragma unroll
            for (int db = 0; db < S::DB; ++db)
              acc[db][rb] *= by;
          }
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            ds[rb][b] *= range[rb].factor;
      }
      u32x4 p[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        p[rb] = block_operand<T>(ds[rb]);
      add_product<T, DP, RB>(acc, lds_k, f * S::KF, p, members);
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      acc[db][rb] *= 1.f / range[rb].factor;
  if constexpr (WK > 1) {
    static_assert(kWaves * 16 * (DP + 4) * 4 <= 4 * TILE, "sums do not fit");
    auto lds_acc = reinterpret_cast<float(*)[16][DP + 4]>(lds_tiles);
    join_waves<T, DP, RB, WK>(acc, lds_acc);
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
    if (col[rb].valid) {
      const int64_t at = (int64_t)col[rb].row * c.hq + col[rb].head;
      float *piece =
          pieces > 1
              ? c.part + (int64_t)place.piece * c.nq * c.hq * c.d
              : nullptr;
      store_columns<T, DP, RB, WK>(acc, rb, c.dq, piece, at, c.d,
                                   c.cap > 0.f ? c.scale * kFlatUp<T> : c.scale);
    }
}

// dk and dv of the keys that a workgroup owns, looping over (query, head) rows, head
// after head of the group: their gradients add up in the registers, in that order.
//
// Four products a pair.  A row's numbers (position, slope, lse, delta) come with its
// tile.  P goes to dv's product, dT to dk's, both rounded for the matrix cores.  The
// call above: 858 us, 641 TFLOP/s of its four products; vector unit 42 %, matrix cores
// 28 %, LDS 35 %.
template <typename T, int DP, int RB, int WK>
__global__ __launch_bounds__(kThreads, (waves_wanted<T, DP, RB, WK>())) void
attention_dkv_kernel(AttentionCall c) {
  using S = Shape<T, DP>;
  constexpr int WQ = kWaves / WK, ROWS = RB * 16 * WQ;
  constexpr int KW = Looped<T, WK>::wave, KT = Looped<T, WK>::tile;
  constexpr int KB = KW / 16;
  constexpr int TILE = KT * S::BYTES;
  __shared__ __attribute__((aligned(16))) char lds_tiles[4 * TILE];
  // per looped row: position, -slope (times log2 e), what its scores are relative to
  // (cap_scores), -delta
  __shared__ __attribute__((aligned(16))) float lds_row[2][6][KT];
  __shared__ Spans<ROWS> spans;

  const int group = c.hq / c.hk;
  const Place place((c.nk + ROWS - 1) / ROWS, c.hk, c.splits);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i = lane & 15, g = lane >> 4;
  const int wq = wave / WK;
  const int part = __builtin_amdgcn_readfirstlane(wave % WK * KW);
  const int row0 = place.tile * ROWS, head0 = place.head * group;
  const int pieces =
      pieces_in_use<T>(c, c.spans_k, row0, min(row0 + ROWS, c.nk) - 1, c.nq,
                           group, place);
  if (place.piece >= pieces)
    return; // (the whole workgroup)

  Column col[RB];
  u32x4 k[RB][S::KS], v[RB][S::KS];
  f32x4 acc_k[S::DB][RB], acc_v[S::DB][RB];
  Range<T> range[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int row = row0 + (wq * RB + rb) * 16 + i;
    col[rb].valid = row < c.nk;
    if (col[rb].valid) {
      col[rb].row = row;
      col[rb].span = c.spans_k ? c.spans_k[row] : make_int2(0, c.nq);
      if (c.slope)
        load_position(col[rb].p, c.pos_k, row, c.axes);
    }
#pragma unroll
    for (int ks = 0; ks < S::KS; ++ks) {
      k[rb][ks] = v[rb][ks] = u32x4{0, 0, 0, 0};
      if (col[rb].valid) {
        k[rb][ks] = load_piece<T, DP>(c.k, row, place.head, ks * 4 + g, c.d);
        v[rb][ks] = load_piece<T, DP>(c.v, row, place.head, ks * 4 + g, c.d);
      }
    }
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      acc_k[db][rb] = acc_v[db][rb] = f32x4{0, 0, 0, 0};
  }

  const Requests<T, DP, KT> request_q(c.q, c.d), request_do(c.dout, c.d);
  collect_spans<ROWS>(spans, c.spans_k, row0, c.nk, 1, c.nq, KT);
  // Two buffers: while a tile is worked on, the next one is on its way.
  auto request = [&](int begin, int end, int round, int buffer) {
    char *tile = lds_tiles + buffer * 2 * TILE;
    const int head = head0 + round;
    request_q(begin, end, head, tile);
    request_do(begin, end, head, tile + TILE);
    auto &rows = lds_row[buffer];
    request_numbers<KT>(c.base + (int64_t)head * c.nq, 1, begin, end, rows[4]);
    request_numbers<KT>(c.minus_delta + (int64_t)head * c.nq, 1, begin, end,
                        rows[5]);
    if (c.slope) {
      request_positions<KT>(c.pos_q, begin, end, c.axes, rows);
      request_numbers<KT>(c.minus_slope + head, 0, begin, end, rows[3]);
    }
  };
  if (c.axes == 2)
    clear_lds<sizeof(lds_row)>(reinterpret_cast<char *>(lds_row));
  if (c.d < S::LDS)
    clear_lds<4 * TILE>(lds_tiles);

  Walk<ROWS> walk(spans, group, place.piece, pieces, KT);
  int buffer = 0;
  Members<RB> members;
  if (walk.there())
    request(walk.begin, walk.end, walk.round, 0);
  for (; walk.there(); buffer ^= 1) {
    const int begin = walk.begin, end = walk.end;
    members.of(walk.span, walk.first, end, col);
    arrive();
    walk.next();
    if (walk.there())
      request(walk.begin, walk.end, walk.round, buffer ^ 1);
    const char *lds_q = lds_tiles + buffer * 2 * TILE + part * S::BYTES;
    const char *lds_do = lds_q + TILE;

    if (!members.some || begin + part >= end)
      continue;
    const bool(&in)[RB] = members.in;
    const bool mixed = members.mixed;
    const bool cut = begin + part + KW > end;

#pragma unroll
    for (int f = 0; f < KB / S::FB; ++f) {
      f32x4 pr[RB][S::FB], ds[RB][S::FB], flat[RB][S::FB], lse[S::FB];
      const auto &rows = lds_row[buffer];
      const int at = part + f * S::KF + g * 4;
#pragma unroll
      for (int b = 0; b < S::FB; ++b) {
        lse[b] = *reinterpret_cast<const f32x4 *>(&rows[4][at + b * 16]);
        const f32x4 minus_delta =
            *reinterpret_cast<const f32x4 *>(&rows[5][at + b * 16]);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          pr[rb][b] = f32x4{0, 0, 0, 0};
          ds[rb][b] = minus_delta;
        }
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks) {
          const u32x4 aq = rows_operand<T, DP>(lds_q, f * S::FB + b, ks);
          const u32x4 ao = rows_operand<T, DP>(lds_do, f * S::FB + b, ks);
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            mma<T>(pr[rb][b], aq, k[rb][ks]);
            mma<T>(ds[rb][b], ao, v[rb][ks]);
          }
        }
      }
      auto capped = [&](auto is_short) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            cap_scores<T, decltype(is_short)::value, true>(
                pr[rb][b], c, lse[b], &flat[rb][b]);
      };
      if (c.cap > 0.f) {
        if (__builtin_expect(short_cap<T>(c), 1))
          capped(std::true_type());
        else
          capped(std::false_type());
      } else {
        const float in = c.scale * kLog2e;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              pr[rb][b][r] = fmaf(pr[rb][b][r], in, -lse[b][r]);
      }
      if (c.slope) {
#pragma unroll
        for (int b = 0; b < S::FB; ++b) {
          const f32x4 slope =
              *reinterpret_cast<const f32x4 *>(&rows[3][at + b * 16]);
          const f32x4 x =
              *reinterpret_cast<const f32x4 *>(&rows[0][at + b * 16]);
          if (c.axes == 1) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                pr[rb][b][r] = fmaf(slope[r], far_by(col[rb].p, x[r]),
                                    pr[rb][b][r]);
          } else {
            const f32x4 y =
                *reinterpret_cast<const f32x4 *>(&rows[1][at + b * 16]);
            const f32x4 z =
                *reinterpret_cast<const f32x4 *>(&rows[2][at + b * 16]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
              for (int r = 0; r < 4; ++r)
                pr[rb][b][r] = fmaf(slope[r],
                                    far_by(col[rb].p, x[r], y[r], z[r]),
                                    pr[rb][b][r]);
          }
        }
      }
#pragma unroll
      for (int b = 0; b < S::FB; ++b)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            pr[rb][b][r] = __builtin_amdgcn_exp2f(pr[rb][b][r]);
            ds[rb][b][r] *= pr[rb][b][r];
          }
      if (c.cap > 0.f) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            ds[rb][b] *= flat[rb][b];
      }
      if (cut || mixed) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!in[rb] || begin + at + b * 16 + r >= end)
                pr[rb][b][r] = ds[rb][b][r] = 0.f;
      }
      if constexpr (kWeightUp<T> != 1.f) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            pr[rb][b] *= kWeightUp<T>;
      }
      if constexpr (Range<T>::on) {
        float top[RB];
        bool moves = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          top[rb] = 0.f;
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              top[rb] = fmaxf(top[rb], fabsf(ds[rb][b][r]));
          moves |= range[rb].moves(top[rb]);
        }
        if (__ballot(moves) != 0) {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) {
            const float by = range[rb].move(top[rb]);
#pragma unroll
            for (int db = 0; db < S::DB; ++db)
              acc_k[db][rb] *= by;
          }
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int b = 0; b < S::FB; ++b)
            ds[rb][b] *= range[rb].factor;
      }
      u32x4 p[RB], x[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        p[rb] = block_operand<T>(pr[rb]);
        x[rb] = block_operand<T>(ds[rb]);
      }
      add_product<T, DP, RB>(acc_v, lds_do, f * S::KF, p, members);
      add_product<T, DP, RB>(acc_k, lds_q, f * S::KF, x, members);
    }
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int db = 0; db < S::DB; ++db)
      acc_k[db][rb] *= 1.f / range[rb].factor;
  if constexpr (WK > 1) {
    static_assert(kWaves * 16 * (DP + 4) * 4 <= 4 * TILE, "sums do not fit");
    auto lds_acc = reinterpret_cast<float(*)[16][DP + 4]>(lds_tiles);
    join_waves<T, DP, RB, WK>(acc_k, lds_acc);
    join_waves<T, DP, RB, WK>(acc_v, lds_acc);
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
    if (col[rb].valid) {
      const int64_t at = (int64_t)col[rb].row * c.hk + place.head;
      const int64_t one = (int64_t)c.nk * c.hk * c.d;
      float *piece = pieces > 1 ? c.part + place.piece * 2 * one : nullptr;
      store_columns<T, DP, RB, WK>(acc_k, rb, c.dk, piece, at, c.d,
                                   c.cap > 0.f ? c.scale * kFlatUp<T> : c.scale);
      store_columns<T, DP, RB, WK>(acc_v, rb, c.dv, piece ? piece + one : nullptr,
                                   at, c.d, 1.f / kWeightUp<T>);
    }
}

// ---- launch -------------------------------------------------------------------

template <typename T, int DP>
hipError_t launch(const AttentionCall &c, int pass, int rows,
                  hipStream_t stream) {
  const int64_t owned =
      pass == 2 ? c.nk : (int64_t)c.nq * (c.hq / c.hk);
  const int64_t grid = (owned + rows - 1) / rows * c.hk * c.splits;
  if (grid <= 0)
    return hipSuccess;
  if (grid * kThreads > UINT32_MAX) // (what a launch can number; checked before)
    return hipErrorInvalidValue;
  const dim3 g((unsigned)grid), b(kThreads);
#define PCA_LAUNCH(kernel, most)                                               \
  if (rows == kFewRows)                                                        \
    kernel<T, DP, 1, 4><<<g, b, 0, stream>>>(c);                               \
  else if (rows == 64)                                                         \
    kernel<T, DP, 1, 1><<<g, b, 0, stream>>>(c);                               \
  else                                                                         \
    kernel<T, DP, most / 64, 1><<<g, b, 0, stream>>>(c)
  if (pass == 0) {
    PCA_LAUNCH(attention_forward_kernel, most_rows(0, sizeof(T), DP));
  } else if (pass == 1) {
    PCA_LAUNCH(attention_dq_kernel, most_rows(1, sizeof(T), DP));
  } else {
    PCA_LAUNCH(attention_dkv_kernel, most_rows(2, sizeof(T), DP));
  }
#undef PCA_LAUNCH
  return hipGetLastError();
}

} // namespace attn
} // namespace pca
