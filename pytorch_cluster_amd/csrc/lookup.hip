// Rows of a table by index, out_e = scale table[index_e], and the gradient of the
// table:
//
//   dtable_n = scale sum over e with index_e = n of dout_e
//
// An index outside the table names no row: its output row is zeros and it adds to no
// gradient (places that a search left empty hold -1).
//
// The gradient is summed in 32 bits without atomics: the entries are sorted by index,
// stable and by digits of up to 10 bits (entries of no row come last), and the sorted
// list is cut into chunks of equal length whatever the rows are -- one row may have most
// entries.  A group of lanes adds up a chunk, run after run; a run that lies in one
// chunk goes straight to the gradient, the others leave their first and last sums in
// the workspace, and the chunk where a run starts adds up its parts.  The same call
// gives the same bits.
//
// The forward pass is bound by memory; of the gradient 40 % is the sort, mostly ranks in
// LDS and six launches, and the sums are memory's.  1,310,720 entries of 64 fp32 components in a table of 65,536 rows:
// forward 96 us = 3.6 TB/s of output and indices (the table comes from the caches, whose
// reads of single rows are what keeps it from the copy's 5.0); gradient: digits 16 + 9
// + 39 us (count, scan, scatter of two passes), sums 81 us = 4.1 TB/s, joins 9.5 us.
// 1,048,576 entries of 64 bf16 components, 4,096 rows, a few of which have most entries:
// forward 23.5 us = 6.0 TB/s (written past the caches), digits 37, sums 38, joins 15 us.
#include "rows_ops.hpp"

#include "attention_impl.hpp"

#include <algorithm>

namespace pca {

namespace {

constexpr int kSortThreads = 1024, kPer = 4;
constexpr int kTile = kSortThreads * kPer; // entries of a sorting workgroup
// (1,024 digits, a thread each: two passes for tables of up to a million rows.  A pass of
// 1.3 million entries takes 32 us, most of it the ranks in LDS; with 8-bit digits a table
// of 65,536 rows is two passes as well, one of 200,000 three.)
constexpr int kBits = 10, kDigits = 1 << kBits;
static_assert(kDigits == kSortThreads, "a thread for each digit");

size_t lk_align(size_t v) { return (v + 255) & ~(size_t)255; }

__device__ __forceinline__ int64_t index_at(const LookupCall &c, int64_t e) {
  return c.wide_index ? static_cast<const int64_t *>(c.index)[e]
                      : (int64_t) static_cast<const int32_t *>(c.index)[e];
}
// Sorting key of an entry: its row, `table` for none.
__device__ __forceinline__ uint32_t key_at(const LookupCall &c, int64_t e) {
  const int64_t i = index_at(c, e);
  return (uint32_t)(i >= 0 && i < c.table ? i : c.table);
}

// ---- forward ------------------------------------------------------------------

// A thread takes kAhead pieces of 16 bytes of output rows, kAhead reads of indices and
// then of rows in flight.
constexpr int kAhead = 4;

// I: what counts pieces (32 bits where they suffice: the division by the pieces of a row
// is most of the arithmetic).
template <typename T, typename I>
__global__ __launch_bounds__(256) void lookup_kernel(LookupCall c, I pieces,
                                                     I total) {
  constexpr int PER = 16 / (int)sizeof(T);
  const I first = (I)blockIdx.x * (256 * kAhead) + threadIdx.x;
  I e[kAhead], e0[kAhead];
  int64_t row[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const I at = min(first + k * 256, total - 1);
    e[k] = at / pieces;
    e0[k] = (at - e[k] * pieces) * PER;
    row[k] = index_at(c, (int64_t)e[k]);
  }
  T v[kAhead][PER];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      v[k][i] = (T)0.f;
    if (row[k] >= 0 && row[k] < c.table) {
      const T *from = static_cast<const T *>(c.rows) + row[k] * c.width + e0[k];
      if (c.width % PER == 0) {
        __builtin_memcpy(v[k], __builtin_assume_aligned(from, 16), 16);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if ((int64_t)e0[k] + i < c.width)
            v[k][i] = from[i];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    if (first + k * 256 >= total)
      break;
    T *to = static_cast<T *>(c.out) + (int64_t)e[k] * c.width + e0[k];
    const bool there = row[k] >= 0 && row[k] < c.table;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      v[k][i] = there ? (T)((float)v[k][i] * c.scale) : (T)0.f;
    if (c.width % PER == 0) {
      // (written once and read by nobody here: the caches stay with the table)
      attn::u32x4 o;
      __builtin_memcpy(&o, v[k], 16);
      __builtin_nontemporal_store(o, reinterpret_cast<attn::u32x4 *>(to));
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if ((int64_t)e0[k] + i < c.width)
          to[i] = v[k][i];
    }
  }
}

// ---- the entries in the order of their rows -------------------------------------

struct Sorted {
  uint64_t *a, *b;    // [entries] (key, entry), by turns
  uint32_t *digits;   // [kDigits][tiles], then [kDigits] totals
  uint32_t *keys, *perm; // [entries]: the result
  int tiles;
};

struct Pass {
  int number, shift, bits;
  bool last;
};

__device__ __forceinline__ uint64_t pair_at(const LookupCall &c,
                                            const Sorted &s, const Pass &p,
                                            int e) {
  if (p.number == 0)
    return (uint64_t)key_at(c, e) << 32 | (uint32_t)e;
  return (p.number & 1 ? s.a : s.b)[e];
}

// Zeros to the gradient, by workgroups `block` of `blocks`: `clear` bytes from 16-byte
// bounds on.
__device__ __forceinline__ void clear_rows(void *out, int64_t clear, int block,
                                           int blocks) {
  const int64_t whole = clear / 16;
  for (int64_t i = (int64_t)block * kSortThreads + threadIdx.x; i < whole;
       i += (int64_t)blocks * kSortThreads)
    static_cast<uint4 *>(out)[i] = make_uint4(0, 0, 0, 0);
  if (block == 0 && threadIdx.x < (clear % 16) / 2)
    static_cast<uint16_t *>(out)[whole * 8 + threadIdx.x] = 0;
}

// Entries of a tile by digit; in the first pass the whole grid also clears the
// gradient (rows without entries keep the zeros).
__global__ __launch_bounds__(kSortThreads) void
lookup_count_kernel(LookupCall c, Sorted s, Pass p, int64_t clear) {
  __shared__ uint32_t count[kDigits];
  const int tid = threadIdx.x;
  if (clear > 0)
    clear_rows(c.out, clear, blockIdx.x, gridDim.x);
  const int tile = blockIdx.x;
  if (tile >= s.tiles)
    return;
  count[tid] = 0u;
  __syncthreads();
  const uint32_t mask = (1u << p.bits) - 1;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t e = (int64_t)tile * kTile + i * kSortThreads + tid;
    if (e < c.entries)
      atomicAdd(&count[(uint32_t)(pair_at(c, s, p, (int)e) >> 32) >> p.shift &
                       mask],
                1u);
  }
  __syncthreads();
  if (tid < 1 << p.bits)
    s.digits[(size_t)tid * s.tiles + tile] = count[tid];
}

// Exclusive prefix of one value per thread of a workgroup; part: a word per wave.
__device__ __forceinline__ uint32_t prefix(uint32_t v, uint32_t *part,
                                           uint32_t &total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t up = v;
#pragma unroll
  for (int sh = 1; sh < 64; sh <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)up, sh);
    up += lane >= sh ? o : 0u;
  }
  __syncthreads(); // (part may be in use)
  if (lane == 63)
    part[wave] = up;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSortThreads / 64; ++w) {
    before += w < wave ? part[w] : 0u;
    total += part[w];
  }
  return before + up - v;
}

// A workgroup per digit: entries of the digit in the tiles before each.
__global__ __launch_bounds__(kSortThreads) void lookup_scan_kernel(Sorted s) {
  __shared__ uint32_t part[kSortThreads / 64];
  uint32_t *column = s.digits + (size_t)blockIdx.x * s.tiles;
  uint32_t before = 0;
  for (int first = 0; first < s.tiles; first += kSortThreads) {
    const int at = first + (int)threadIdx.x;
    const uint32_t v = at < s.tiles ? column[at] : 0u;
    uint32_t total;
    const uint32_t run = before + prefix(v, part, total);
    if (at < s.tiles)
      column[at] = run;
    before += total;
  }
  if (threadIdx.x == 0)
    s.digits[(size_t)kDigits * s.tiles + blockIdx.x] = before;
}

// Ranks of this thread's entries (kPer, 64 apart, the wave's are neighbours) among the
// entries of the same digit in the tile, and in `local` where a digit's entries begin.
// place: [waves][kDigits]; afterwards a wave's first place per digit.
__device__ __forceinline__ void
rank_tile(const uint64_t (&v)[kPer], int mine, int some, int shift, int bits,
          uint32_t (*place)[kDigits], uint32_t *part, uint32_t (&rank)[kPer],
          uint32_t &local) {
  constexpr int WAVES = kSortThreads / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t mask = (1u << bits) - 1;
  for (int i = tid; i < WAVES * kDigits; i += kSortThreads)
    (&place[0][0])[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t digit = (uint32_t)(v[i] >> 32) >> shift & mask;
    const bool is = mine + i * 64 < some;
    uint64_t same = __ballot(is);
    for (int b = 0; b < bits; ++b) {
      const bool set = (digit >> b & 1u) != 0u;
      const uint64_t lanes = __ballot(set);
      same &= set ? lanes : ~lanes;
    }
    // (the first of them counts for all; a wave's atomics come in order)
    const int leader =
        same != 0 ? __ffsll((unsigned long long)same) - 1 : lane;
    uint32_t before = 0;
    if (is && lane == leader)
      before = atomicAdd(&place[wave][digit], (uint32_t)__popcll(same));
    before = (uint32_t)__shfl((int)before, leader);
    rank[i] = before + (uint32_t)__popcll(same & ((1ull << lane) - 1));
  }
  __syncthreads();
  uint32_t count = 0, total;
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
    count += place[w][tid];
  local = prefix(count, part, total);
  uint32_t run = local;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const uint32_t n = place[w][tid];
    place[w][tid] = run;
    run += n;
  }
  __syncthreads();
}

// A tile's entries by digit, those of a digit in the order they came in: put together in
// LDS first, so that neighbouring threads write neighbouring places.
__global__ __launch_bounds__(kSortThreads) void
lookup_scatter_kernel(LookupCall c, Sorted s, Pass p) {
  __shared__ uint64_t lds[kTile];
  __shared__ uint32_t place[kSortThreads / 64][kDigits];
  __shared__ uint32_t part[kSortThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = (int)blockIdx.x * kTile;
  const int some = (int)min((int64_t)kTile, c.entries - first);
  const int mine = wave * (64 * kPer) + lane;
  const uint32_t mask = (1u << p.bits) - 1;
  uint64_t v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    v[i] = pair_at(c, s, p, first + min(mine + i * 64, some - 1));
  // what is before the digit's entries: of smaller digits, in the tiles before
  uint32_t offset = 0, all = 0, total;
  if (tid < 1 << p.bits) {
    offset = s.digits[(size_t)tid * s.tiles + blockIdx.x];
    all = s.digits[(size_t)kDigits * s.tiles + tid];
  }
  uint32_t rank[kPer], local;
  rank_tile(v, mine, some, p.shift, p.bits, place, part, rank, local);
  offset += prefix(all, part, total);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t digit = (uint32_t)(v[i] >> 32) >> p.shift & mask;
    if (mine + i * 64 < some)
      lds[place[wave][digit] + rank[i]] = v[i];
  }
  __syncthreads();
  place[0][tid] = offset - local; // (modulo 2^32)
  __syncthreads();
  uint64_t *out = p.number & 1 ? s.b : s.a;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = i * kSortThreads + tid;
    if (at < some) {
      const uint64_t pair = lds[at];
      const uint32_t to =
          place[0][(uint32_t)(pair >> 32) >> p.shift & mask] + (uint32_t)at;
      if (to < (uint64_t)c.entries) {
        if (p.last) {
          s.keys[to] = (uint32_t)(pair >> 32);
          s.perm[to] = (uint32_t)pair;
        } else {
          out[to] = pair;
        }
      }
    }
  }
}

// All passes of at most a tile's entries, by one workgroup; the others clear the
// gradient.
__global__ __launch_bounds__(kSortThreads) void
lookup_small_sort_kernel(LookupCall c, Sorted s, int bits, int64_t clear) {
  __shared__ uint64_t lds[kTile];
  __shared__ uint32_t place[kSortThreads / 64][kDigits];
  __shared__ uint32_t part[kSortThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x > 0) {
    clear_rows(c.out, clear, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int some = (int)c.entries;
  if (some == 0)
    return;
  const int mine = wave * (64 * kPer) + lane;
  uint64_t v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = min(mine + i * 64, some - 1);
    v[i] = (uint64_t)key_at(c, e) << 32 | (uint32_t)e;
  }
  for (int shift = 0; shift < bits; shift += kBits) {
    const int now = min(kBits, bits - shift);
    const uint32_t mask = (1u << now) - 1;
    uint32_t rank[kPer], local;
    rank_tile(v, mine, some, shift, now, place, part, rank, local);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (mine + i * 64 < some)
        lds[place[wave][(uint32_t)(v[i] >> 32) >> shift & mask] + rank[i]] =
            v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      v[i] = lds[min(mine + i * 64, some - 1)];
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (mine + i * 64 < some) {
      s.keys[mine + i * 64] = (uint32_t)(v[i] >> 32);
      s.perm[mine + i * 64] = (uint32_t)v[i];
    }
}

// ---- sums of runs ---------------------------------------------------------------

struct Chunks {
  int64_t length;  // entries of a chunk
  int64_t count;   // chunks
  float *ends;     // [count, 2, width]: sums of a chunk's first and last run where
                   // they do not lie in it
};

// Lanes that take an entry's row, 16 bytes each (wide rows: in columns of LANES pieces,
// blockIdx.y).  Eight rows are under way per group.  A workgroup whose chunks lie inside
// one run with an entry to spare on both sides leaves one sum for all of them, in the
// place of its first chunk: a row with 131,000 entries is 4,096 chunks, a megabyte of sums
// that one workgroup would read for the join (53 us; 15 this way).
template <typename T, int LANES>
__global__ __launch_bounds__(256) void
lookup_sum_kernel(LookupCall c, Sorted s, Chunks k) {
  constexpr int PER = 16 / (int)sizeof(T), GROUPS = 256 / LANES, AHEAD = 8;
  __shared__ float part[GROUPS][LANES * PER + 1];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int64_t chunk = (int64_t)blockIdx.x * GROUPS + grp;
  const uint32_t none = (uint32_t)c.table;
  // (the same in the whole workgroup; sorted keys: all between the two are alike)
  const int64_t before = (int64_t)blockIdx.x * GROUPS * k.length - 1;
  const int64_t behind = before + 1 + GROUPS * k.length;
  const bool inside = before >= 0 && behind < c.entries &&
                      s.keys[before] == s.keys[behind] &&
                      s.keys[behind] != none;
  int64_t e0 = ((int64_t)blockIdx.y * LANES + lane) * PER;
  if (e0 >= c.width) {
    if (!inside)
      return;
    e0 = 0; // (read, and not written)
  }
  if (chunk >= k.count)
    return; // (not inside)
  const int64_t begin = chunk * k.length;
  const int64_t end = min(begin + k.length, c.entries);
  const bool vec = c.width % PER == 0;
  uint32_t now = s.keys[begin];
  if (now == none)
    return;
  bool open = begin > 0 && s.keys[begin - 1] == now; // the run started before
  float sum[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    sum[i] = 0.f;
  auto put = [&](bool last) {
    if (open || last) {
      float *to = k.ends + (chunk * 2 + (open ? 0 : 1)) * c.width + e0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (vec || e0 + i < c.width)
          to[i] = sum[i];
    } else {
      T *to = static_cast<T *>(c.out) + (int64_t)now * c.width + e0;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (vec || e0 + i < c.width)
          to[i] = (T)(sum[i] * c.scale);
    }
  };
  // the next entries' keys and numbers are read while their predecessors' rows are
  // under way
  uint32_t key[AHEAD], perm[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int64_t e = min(begin + j, end - 1);
    key[j] = s.keys[e];
    perm[j] = s.perm[e];
  }
  for (int64_t at = begin; at < end; at += AHEAD) {
    T v[AHEAD][PER];
    uint32_t next_key[AHEAD], next_perm[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const T *from =
          static_cast<const T *>(c.rows) + (int64_t)perm[j] * c.width + e0;
      if (vec) {
        __builtin_memcpy(v[j], __builtin_assume_aligned(from, 16), 16);
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          v[j][i] = e0 + i < c.width ? from[i] : (T)0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int64_t e = min(at + AHEAD + j, end - 1);
      next_key[j] = s.keys[e];
      next_perm[j] = s.perm[e];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (at + j >= end)
        break;
      if (key[j] != now) {
        put(false);
        now = key[j];
        open = false;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          sum[i] = 0.f;
        if (now == none)
          return;
      }
#pragma unroll
      for (int i = 0; i < PER; ++i)
        sum[i] += (float)v[j][i];
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      key[j] = next_key[j];
      perm[j] = next_perm[j];
    }
  }
  if (!inside) {
    put(end < c.entries && s.keys[end] == now);
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    part[grp][lane * PER + i] = sum[i];
  __syncthreads();
  for (int col = threadIdx.x; col < LANES * PER; col += 256) {
    const int64_t e = (int64_t)blockIdx.y * LANES * PER + col;
    if (e >= c.width)
      continue;
    float all = 0.f;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j)
      all += part[j][col];
    k.ends[(int64_t)blockIdx.x * GROUPS * 2 * c.width + e] = all;
  }
}

// The parts of a run that starts in chunk `chunk` and goes on behind it; chunk `stop` is the
// first that does not begin with its row.  Chunks up to a workgroup's first, workgroups
// that lie inside the run, chunks behind them.
template <int GROUPS> struct Parts {
  int chunk, head, whole, count; // (chunks are far below 2^31)
  __device__ __forceinline__ Parts(int from, int stop) : chunk(from) {
    const int next = (int)((unsigned)from / GROUPS + 1) * GROUPS;
    head = min(next, stop) - from;
    whole = (int)((unsigned)max(stop - 1 - next, 0) / GROUPS);
    count = stop - from - whole * (GROUPS - 1);
  }
  __device__ __forceinline__ int operator[](int n) const {
    return chunk + n + (GROUPS - 1) * min(max(n - head, 0), whole);
  }
};

// A group of lanes per chunk: where a run starts in it that goes on behind it, the run's
// parts are added up.  Runs of many parts (kLong or more) are added up by the whole
// workgroup, one after the other: parts dealt to the groups, put together in the order
// of the groups.
constexpr int kLong = 16;

template <typename T, int LANES>
__global__ __launch_bounds__(256) void
lookup_join_kernel(LookupCall c, Sorted s, Chunks k) {
  constexpr int PER = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  __shared__ float part[GROUPS][LANES * PER + 1];
  __shared__ int64_t long_stop[GROUPS];
  const int lane = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int64_t e0 = ((int64_t)blockIdx.y * LANES + lane) * PER;
  auto row_of = [&](int64_t chunk) {
    return s.keys[min((chunk + 1) * k.length, c.entries) - 1];
  };
  const bool vec = c.width % PER == 0 && e0 < c.width;
  auto add = [&](float (&sum)[PER], int64_t chunk, int64_t at) {
    const float *from = k.ends + (at * 2 + (at == chunk ? 1 : 0)) * c.width + e0;
    if (vec) {
      float v[PER];
      __builtin_memcpy(v, __builtin_assume_aligned(from, 16), sizeof(v));
#pragma unroll
      for (int i = 0; i < PER; ++i)
        sum[i] += v[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i < c.width)
        sum[i] += from[i];
  };
  {
    const int64_t chunk = (int64_t)blockIdx.x * GROUPS + grp;
    const int64_t begin = chunk * k.length, end = begin + k.length;
    int64_t stop = 0;
    bool many = false;
    if (end < c.entries) {
      const uint32_t now = s.keys[end - 1];
      if (now != (uint32_t)c.table && s.keys[end] == now &&
          !(s.keys[begin] == now && begin > 0 && s.keys[begin - 1] == now)) {
        // chunks behind this one that begin with the run's row
        int64_t lo = chunk + 1, hi = k.count;
        for (int64_t step = 1; lo + step < hi; step *= 2) {
          if (s.keys[(lo + step) * k.length] != now) {
            hi = lo + step;
            break;
          }
          lo += step;
        }
        while (hi - lo > 1) {
          const int64_t mid = (lo + hi) >> 1;
          if (s.keys[mid * k.length] == now)
            lo = mid;
          else
            hi = mid;
        }
        stop = hi;
        const Parts<GROUPS> parts((int)chunk, (int)stop);
        many = parts.count >= kLong;
        if (!many && e0 < c.width) {
          float sum[PER];
#pragma unroll
          for (int i = 0; i < PER; ++i)
            sum[i] = 0.f;
          if (parts.whole == 0) {
            for (int64_t at = chunk; at < stop; ++at)
              add(sum, chunk, at);
          } else {
            for (int n = 0; n < parts.count; ++n)
              add(sum, chunk, parts[n]);
          }
          T *to = static_cast<T *>(c.out) + (int64_t)now * c.width + e0;
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (e0 + i < c.width)
              to[i] = (T)(sum[i] * c.scale);
        }
      }
    }
    if (lane == 0)
      long_stop[grp] = many ? stop : 0;
  }
  __syncthreads();
  for (int g = 0; g < GROUPS; ++g) {
    const int64_t stop = long_stop[g];
    if (stop == 0)
      continue; // (the whole workgroup)
    const int64_t chunk = (int64_t)blockIdx.x * GROUPS + g;
    float sum[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      sum[i] = 0.f;
    const Parts<GROUPS> parts((int)chunk, (int)stop);
#pragma unroll 8
    for (int n = grp; n < parts.count; n += GROUPS)
      add(sum, chunk, parts[n]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i)
      part[grp][lane * PER + i] = sum[i];
    __syncthreads();
    for (int col = threadIdx.x; col < LANES * PER; col += 256) {
      const int64_t e = (int64_t)blockIdx.y * LANES * PER + col;
      if (e >= c.width)
        continue;
      float all = 0.f;
      for (int j = 0; j < GROUPS; ++j)
        all += part[j][col];
      static_cast<T *>(c.out)[(int64_t)row_of(chunk) * c.width + e] =
          (T)(all * c.scale);
    }
  }
}

int bit_length(uint64_t v) {
  int n = 0;
  while (v >> n)
    ++n;
  return n;
}

Chunks chunks_of(int64_t entries) {
  Chunks k;
  // (32,768 chunks are 128 a CU: groups of lanes enough for rows in flight, and each of
  // them leaves two rows to join at most)
  k.length = std::clamp<int64_t>((entries + 32767) / 32768, 16, 1 << 20);
  k.count = (entries + k.length - 1) / k.length;
  k.ends = nullptr;
  return k;
}

template <typename T, int LANES>
void launch_sums(const LookupCall &c, const Sorted &s, const Chunks &k,
                 hipStream_t stream) {
  constexpr int PER = 16 / (int)sizeof(T), GROUPS = 256 / LANES;
  const unsigned columns =
      (unsigned)((c.width + LANES * PER - 1) / (LANES * PER));
  lookup_sum_kernel<T, LANES>
      <<<dim3((unsigned)((k.count + GROUPS - 1) / GROUPS), columns), dim3(256),
         0, stream>>>(c, s, k);
  lookup_join_kernel<T, LANES>
      <<<dim3((unsigned)((k.count + GROUPS - 1) / GROUPS), columns), dim3(256),
         0, stream>>>(c, s, k);
}

template <typename T>
hipError_t launch_type(const LookupCall &c, const Sorted &s, const Chunks &k,
                       hipStream_t stream) {
  const int64_t pieces = (c.width * (int64_t)sizeof(T) + 15) / 16;
  if (pieces <= 4)
    launch_sums<T, 4>(c, s, k, stream);
  else if (pieces <= 8)
    launch_sums<T, 8>(c, s, k, stream);
  else if (pieces <= 16)
    launch_sums<T, 16>(c, s, k, stream);
  else if (pieces <= 32)
    launch_sums<T, 32>(c, s, k, stream);
  else
    launch_sums<T, 64>(c, s, k, stream);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_forward(const LookupCall &c, hipStream_t stream) {
  const int64_t pieces = (c.width * (int64_t)sizeof(T) + 15) / 16;
  const int64_t total = pieces * c.entries;
  const int64_t blocks = (total + 256 * kAhead - 1) / (256 * kAhead);
  if (blocks > INT32_MAX)
    return hipErrorInvalidValue;
  if (total < (1ll << 31))
    lookup_kernel<T, uint32_t><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(
        c, (uint32_t)pieces, (uint32_t)total);
  else
    lookup_kernel<T, int64_t><<<dim3((unsigned)blocks), dim3(256), 0, stream>>>(
        c, pieces, total);
  return hipGetLastError();
}

size_t element_size(int dtype) { return dtype == 0 ? 4 : 2; }

} // namespace

hipError_t lookup_forward(const LookupCall &c, int dtype, hipStream_t stream) {
  if (c.entries == 0 || c.width == 0)
    return hipSuccess;
  return dtype == 0   ? launch_forward<float>(c, stream)
         : dtype == 2 ? launch_forward<_Float16>(c, stream)
                      : launch_forward<__bf16>(c, stream);
}

size_t lookup_workspace_bytes(int64_t, int64_t entries, int64_t width) {
  const Chunks k = chunks_of(entries);
  const int64_t tiles = (entries + kTile - 1) / kTile;
  return 2 * lk_align(8 * (size_t)entries) + 2 * lk_align(4 * (size_t)entries) +
         lk_align(4 * (size_t)kDigits * (size_t)(tiles + 1)) +
         lk_align(8 * (size_t)k.count * (size_t)width) + 256;
}

hipError_t lookup_backward(const LookupCall &c, int dtype, void *workspace,
                           hipStream_t stream) {
  if (c.table == 0 || c.width == 0)
    return hipSuccess;
  char *base = static_cast<char *>(workspace);
  auto take = [&](size_t bytes) {
    char *p = base;
    base += lk_align(bytes);
    return p;
  };
  Sorted s;
  Chunks k = chunks_of(c.entries);
  const int64_t tiles = (c.entries + kTile - 1) / kTile;
  s.tiles = (int)tiles;
  s.a = reinterpret_cast<uint64_t *>(take(8 * (size_t)c.entries));
  s.b = reinterpret_cast<uint64_t *>(take(8 * (size_t)c.entries));
  s.keys = reinterpret_cast<uint32_t *>(take(4 * (size_t)c.entries));
  s.perm = reinterpret_cast<uint32_t *>(take(4 * (size_t)c.entries));
  s.digits =
      reinterpret_cast<uint32_t *>(take(4 * (size_t)kDigits * (tiles + 1)));
  k.ends = reinterpret_cast<float *>(take(8 * (size_t)k.count * c.width));
  const int64_t clear =
      c.table * c.width * (int64_t)element_size(dtype); // bytes
  const int bits = bit_length((uint64_t)c.table);
  if (c.entries <= kTile) {
    const int64_t fill = std::min<int64_t>(
        (clear + kSortThreads * 64 - 1) / (kSortThreads * 64), 2048);
    Sorted one = s;
    LookupCall some = c;
    lookup_small_sort_kernel<<<dim3((unsigned)(1 + fill)), dim3(kSortThreads),
                               0, stream>>>(some, one, bits, clear);
    if (c.entries == 0)
      return hipGetLastError();
  } else {
    const int passes = (bits + kBits - 1) / kBits;
    const int each = (bits + passes - 1) / passes;
    for (int n = 0; n < passes; ++n) {
      Pass p;
      p.number = n;
      p.shift = n * each;
      p.bits = std::min(each, bits - p.shift);
      p.last = n == passes - 1;
      const int64_t fill =
          n == 0 ? std::min<int64_t>(
                       (clear + kSortThreads * 64 - 1) / (kSortThreads * 64), 2048)
                 : 0;
      lookup_count_kernel<<<dim3((unsigned)std::max<int64_t>(tiles, fill)),
                            dim3(kSortThreads), 0, stream>>>(
          c, s, p, n == 0 ? clear : 0);
      lookup_scan_kernel<<<dim3(1u << p.bits), dim3(kSortThreads), 0, stream>>>(
          s);
      lookup_scatter_kernel<<<dim3((unsigned)tiles), dim3(kSortThreads), 0,
                              stream>>>(c, s, p);
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return e;
  return dtype == 0   ? launch_type<float>(c, s, k, stream)
         : dtype == 2 ? launch_type<_Float16>(c, s, k, stream)
                      : launch_type<__bf16>(c, s, k, stream);
}

} // namespace pca
