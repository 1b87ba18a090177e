// pages.hip -- operations on the pages of a paged cache: copying pages, forking
// sequences, freeing them and compacting the pool.
//
// All of it moves bytes and whole numbers, so what bounds it is HBM where pages
// are copied and launch latency everywhere else.
//   copy     page dst[i] := page src[i] of every plane (K, V, their 8-bit copy,
//            the scales)
//   fork     the parent's table row, and a copy of its partly filled last page
//   free     U[id] = 1 if a row's used columns name page id; the ids with U = 0,
//            ascending
//   compact  n = sum U; the i-th id >= n with U = 1 goes to the i-th id < n with
//            U = 0.  Sources and destinations are disjoint, so the copies need
//            no order, and as many ids < n are unused as ids >= n are used.
#include <algorithm>

#include "fat_common.h"

namespace fat {

// One tensor of a pool: `outer` x `inner` rows of `row` bytes per page, which
// the host has merged where they lie behind each other.
struct Plane {
  uint8_t* base;
  int64_t page;             // bytes between pages
  int64_t outer_stride, inner_stride;
  uint32_t inner;           // rows per outer step
  uint32_t vpr;             // vectors per row
  uint32_t vpp;             // vectors per page
  uint32_t inv;             // floor(2^32 / vpp) (vpp > 1)
  uint32_t cpp;             // chunks of 1 KiB per page; 0: its pages aren't runs of whole ones
  int32_t log2v;            // log2 of the vector's bytes
};

constexpr int kMaxPlanes = 6;
constexpr int kCopyThreads = 256;
constexpr int kChunk = 1024;     // bytes: 16 per lane of a wave
constexpr int kWaveChunks = 8;   // per wave and step
constexpr int kStepChunks = kCopyThreads / 64 * kWaveChunks;
constexpr int kVectors = 2;      // per thread and step
constexpr int kStepVectors = kVectors * kCopyThreads;

struct Planes {
  Plane p[kMaxPlanes];
  int32_t n;
  int32_t num_pages;
};

__device__ __forceinline__ int64_t plane_steps(const Plane& pl, int64_t count) {
  return pl.cpp ? (count * pl.cpp + kStepChunks - 1) / kStepChunks : (count * pl.vpp + kStepVectors - 1) / kStepVectors;
}

// Quotient and remainder of uniform numbers.
__device__ __forceinline__ int64_t divide(int64_t x, uint32_t by, uint32_t& rest) {
  const int64_t q = x <= 0xffffffffll ? (int64_t)((uint32_t)x / by) : x / by;
  rest = (uint32_t)(x - q * by);
  return q;
}

// Pages that are runs of 1 KiB chunks (all but slices of a pool, and scales):
// 32 chunks of them, 8 per wave.  A chunk has one pair of ids, so its addresses
// are scalar, and a lane holds nothing but its 16 bytes of each chunk: all of a
// wave's loads are in flight before its first store, at full occupancy.  Copying
// 12000 scattered pages of 32 KiB reaches 4.9 TB/s (read and written), pages in a
// row 5.5, torch's copy of such a tensor 5.1; with an address per lane and 128
// registers a thread it was 3.6.  Plain stores: past the caches they gain 2 % where
// the pool is larger than those and lose 20 % where it isn't.
template <typename Pair>
__device__ __forceinline__ void copy_chunks(const Plane& pl, int64_t step, int64_t count, Pair pair) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lane = (threadIdx.x & 63) * 16;
  uint32_t c;
  int64_t i = divide(step * kStepChunks + wave * kWaveChunks, pl.cpp, c);
  u32x4 x[kWaveChunks];
  uint8_t* to[kWaveChunks];
  int s = 0, d = 0;
  bool on = i < count && pair(i, s, d);
#pragma unroll
  for (int u = 0; u < kWaveChunks; ++u) {
    to[u] = nullptr;
    if (on) {
      const uint8_t* from = pl.base + (int64_t)s * pl.page + (int64_t)c * kChunk;
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + lane));
      to[u] = pl.base + (int64_t)d * pl.page + (int64_t)c * kChunk;
    }
    if (++c == pl.cpp) {
      c = 0;
      ++i;
      on = i < count && pair(i, s, d);
    }
  }
#pragma unroll
  for (int u = 0; u < kWaveChunks; ++u)
    if (to[u]) *reinterpret_cast<u32x4*>(to[u] + lane) = x[u];
}

// Any other plane: 512 vectors of its pages (more per thread spilled).
template <typename V, typename Pair>
__device__ __forceinline__ void copy_vectors(const Plane& pl, int64_t step, int64_t count, Pair pair) {
  uint32_t rest;
  const int64_t i0 = divide(step * kStepVectors, pl.vpp, rest);
  V x[kVectors];
  uint8_t* to[kVectors];
#pragma unroll
  for (int u = 0; u < kVectors; ++u) {
    uint32_t v = rest + threadIdx.x + u * kCopyThreads;
    uint32_t k = pl.vpp > 1 ? __umulhi(v, pl.inv) : v;  // v / vpp, or one less
    v -= k * pl.vpp;
    if (v >= pl.vpp) {
      v -= pl.vpp;
      ++k;
    }
    int s, d;
    to[u] = nullptr;
    if (i0 + k < count && pair(i0 + k, s, d)) {
      const uint32_t r = v / pl.vpr;
      const uint32_t o = r / pl.inner;
      const int64_t off = (int64_t)o * pl.outer_stride + (int64_t)(r - o * pl.inner) * pl.inner_stride +
                          (int64_t)(v - r * pl.vpr) * (int64_t)sizeof(V);
      x[u] = *reinterpret_cast<const V*>(pl.base + (int64_t)s * pl.page + off);
      to[u] = pl.base + (int64_t)d * pl.page + off;
    }
  }
#pragma unroll
  for (int u = 0; u < kVectors; ++u)
    if (to[u]) *reinterpret_cast<V*>(to[u]) = x[u];
}

// pair(i, src, dst) gives the ids of pair i and whether it is to be copied.
template <typename Pair>
__device__ __forceinline__ void copy_step(const Plane& pl, int64_t step, int64_t count, Pair pair) {
  if (pl.cpp) {
    copy_chunks(pl, step, count, pair);
    return;
  }
  switch (pl.log2v) {
    case 4: copy_vectors<u32x4>(pl, step, count, pair); break;
    case 3: copy_vectors<u32x2>(pl, step, count, pair); break;
    case 2: copy_vectors<u32>(pl, step, count, pair); break;
    case 1: copy_vectors<uint16_t>(pl, step, count, pair); break;
    default: copy_vectors<uint8_t>(pl, step, count, pair); break;
  }
}

// blockIdx.y: plane; blockIdx.x: steps of it, the grid's width apart.
__global__ __launch_bounds__(kCopyThreads, 8) void copy_pages_kernel(const Planes planes,
                                                                     const int32_t* __restrict__ src,
                                                                     const int32_t* __restrict__ dst, int64_t count) {
  const Plane pl = planes.p[blockIdx.y];
  const int64_t steps = plane_steps(pl, count);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x)
    copy_step(pl, step, count, [&](int64_t i, int& s, int& d) {
      s = src[i];
      d = dst[i];
      return (unsigned)s < (unsigned)planes.num_pages && (unsigned)d < (unsigned)planes.num_pages;
    });
}

// ---------------------------------------------------------------------------
// Fork
// ---------------------------------------------------------------------------
struct ForkParams {
  Planes planes;
  const int32_t* parents;
  const int32_t* children;
  const int32_t* pages;
  int32_t* pt;
  int32_t* lens;
  int64_t pt_sb;
  int32_t B, max_pages, P;
};

// 240 forks of pages of 384 KiB (with their 8-bit copy) take 39 us: 92 MB written,
// 2.4 TB/s.  A fill of as much takes 15 us and torch's copy of 16 such pages to 240
// places 34, so its writes alone don't bound it.
// blockIdx.y: the fork; blockIdx.z: a plane of its last page, or (the last) its
// table row; blockIdx.x: steps.  Every workgroup of a fork reads only its
// parent's row, which no fork of the call writes, and decides alike.
__global__ __launch_bounds__(kCopyThreads, 8) void fork_kernel(const ForkParams p) {
  if ((int)blockIdx.z < p.planes.n && (int64_t)blockIdx.x >= plane_steps(p.planes.p[blockIdx.z], 1)) return;
  const int i = blockIdx.y;
  const int parent = p.parents[i], child = p.children[i];
  if ((unsigned)parent >= (unsigned)p.B || (unsigned)child >= (unsigned)p.B || parent == child) return;
  const int len = p.lens[parent];
  if (len < 0 || len > (int64_t)p.max_pages * p.P) return;
  const int full = len / p.P;
  const bool tail = len != full * p.P;
  const int32_t* from = p.pt + (int64_t)parent * p.pt_sb;
  int src = 0, dst = 0;
  if (tail) {
    src = from[full];
    dst = p.pages[i];
    if ((unsigned)src >= (unsigned)p.planes.num_pages || (unsigned)dst >= (unsigned)p.planes.num_pages) return;
  }
  if ((int)blockIdx.z == p.planes.n) {
    int32_t* to = p.pt + (int64_t)child * p.pt_sb;
    const int step = gridDim.x * kCopyThreads;
    for (int c = blockIdx.x * kCopyThreads + threadIdx.x; c < full; c += step) to[c] = from[c];
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      if (tail) to[full] = dst;
      p.lens[child] = len;
    }
    return;
  }
  if (!tail) return;
  const Plane pl = p.planes.p[blockIdx.z];
  const int64_t steps = plane_steps(pl, 1);
  for (int64_t step = blockIdx.x; step < steps; step += gridDim.x)
    copy_step(pl, step, 1, [&](int64_t, int& s, int& d) {
      s = src;
      d = dst;
      return true;
    });
}

// ---------------------------------------------------------------------------
// Which pages are in use, and lists of them
// ---------------------------------------------------------------------------
// A byte per page, not a bit: bytes are plain stores that all write the same
// value (whatever the order, and each XCD's L2 writes back the bytes it has),
// where bits would be atomics at the level all XCDs share.
struct UseParams {
  int32_t* lens;  // (written for freed rows only)
  int32_t* held;
  int32_t* pt;    // (written when compacting only)
  const int32_t* rows;
  int64_t pt_sb;
  int32_t B, max_pages, P, num_pages, nrows;
  uint8_t* used;     // [groups * kUseGroup]
  int32_t* counts;   // [groups]: used pages of each kUseGroup ids
  int32_t* list;     // free: the free pages [num_pages]; compact: destinations
  int32_t* src;      // compact: sources
  int32_t* rank;     // compact: a moved page's place in src
  int32_t* remap;    // compact
  int32_t* total;    // free: free pages; compact: used pages
};

constexpr int kUseGroup = 4096;  // ids that one workgroup counts and lists
constexpr int kUseThreads = 256;

__device__ __forceinline__ int used_columns(const UseParams& p, int b) {
  const int64_t len = max(p.lens[b], 0);
  int64_t n = (len + p.P - 1) / p.P;
  if (p.held) n = max(n, (int64_t)p.held[b]);
  return (int)min(n, (int64_t)p.max_pages);
}

// Clears the flags and empties the freed rows.
__global__ __launch_bounds__(kUseThreads) void use_clear_kernel(const UseParams p, int64_t words) {
  const int64_t step = (int64_t)gridDim.x * kUseThreads;
  const int64_t t = (int64_t)blockIdx.x * kUseThreads + threadIdx.x;
  for (int64_t i = t; i < words; i += step) reinterpret_cast<u32x4*>(p.used)[i] = u32x4{0u, 0u, 0u, 0u};
  for (int64_t i = t; i < p.nrows; i += step) {
    const int b = p.rows[i];
    if ((unsigned)b >= (unsigned)p.B) continue;
    p.lens[b] = 0;
    if (p.held) p.held[b] = 0;
  }
}

// blockIdx.y: rows, the grid's height apart; blockIdx.x: 4096 columns.  Bound by
// the scattered byte stores, whose lines every XCD's L2 writes back: 14 us for 1.1
// million ids, 4 of them for reading those (17 at 1024 columns; 27 and 35 with
// stores that go past the L2).
constexpr int kMarkEach = 16;  // columns per thread
__global__ __launch_bounds__(kUseThreads) void use_mark_kernel(const UseParams p) {
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const int n = used_columns(p, b);
    const int32_t* row = p.pt + (int64_t)b * p.pt_sb;
    const int c0 = blockIdx.x * (kMarkEach * kUseThreads) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < kMarkEach; ++u) {
      const int c = c0 + u * kUseThreads;
      if (c < n) {
        const int id = row[c];
        if ((unsigned)id < (unsigned)p.num_pages) p.used[id] = 1;
      }
    }
  }
}

// Sum over the workgroup (all threads get it) and the sum over the threads before.
template <int THREADS = kUseThreads>
__device__ __forceinline__ int use_scan(int x, int& before) {
  __shared__ int s[THREADS / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int y = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int z = __shfl_up(y, off);
    y += lane >= off ? z : 0;
  }
  __syncthreads();
  if (lane == 63) s[w] = y;
  __syncthreads();
  int total = 0;
  before = y - x;
#pragma unroll
  for (int k = 0; k < THREADS / 64; ++k) {
    before += k < w ? s[k] : 0;
    total += s[k];
  }
  return total;
}

__global__ __launch_bounds__(kUseThreads) void use_count_kernel(const UseParams p) {
  const u32x4 f = reinterpret_cast<const u32x4*>(p.used)[(int64_t)blockIdx.x * kUseThreads + threadIdx.x];
  int before;
  const int n = use_scan(__popc(f[0]) + __popc(f[1]) + __popc(f[2]) + __popc(f[3]), before);
  if (threadIdx.x == 0) p.counts[blockIdx.x] = n;
}

// Writes the lists.  COMPACT: sources and destinations of the moves and the new
// ids of the pages that stay, else the free pages.  A wave has 64 ids at a time,
// whose flags are a ballot, so that its stores lie next to each other (a thread
// with 16 ids in a row took 9.7 instead of 5 us for 1.4 million ids).
template <bool COMPACT>
__global__ __launch_bounds__(kUseThreads) void use_list_kernel(const UseParams p) {
  constexpr int kWaves = kUseThreads / 64, kEach = kUseGroup / kUseThreads;
  __shared__ int s_before[kEach * kWaves];
  const int groups = gridDim.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int mine = 0, all = 0, dummy;
  for (int i = threadIdx.x; i < groups; i += kUseThreads) {
    const int c = p.counts[i];
    all += c;
    mine += i < (int)blockIdx.x ? c : 0;
  }
  unsigned long long flags[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    flags[j] = __ballot(p.used[(int64_t)blockIdx.x * kUseGroup + j * kUseThreads + threadIdx.x] != 0);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (lane == 0) s_before[j * kWaves + wave] = __popcll(flags[j]);
  }
  const int n = use_scan(all, dummy);  // (synchronises)
  const int first = use_scan(mine, dummy);
  int before = 0, x = wave == 0 ? s_before[lane] : 0;
  static_assert(kEach * kWaves == 64, "a wave scans the counts of a group's 64 ids each");
  use_scan(x, before);
  if (wave == 0) s_before[lane] = first + before;
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.total = COMPACT ? n : p.num_pages - n;
  // COMPACT: used ids below n, from whom the moved ones' ranks count.  They are
  // the used ids of the whole groups below n and those of its own group.
  int below = 0;
  if constexpr (COMPACT) {
    const int gn = n / kUseGroup;
    int w = 0;
    for (int i = threadIdx.x; i < min(gn, groups); i += kUseThreads) w += p.counts[i];
    if (gn < groups) {
      const u32x4 h = reinterpret_cast<const u32x4*>(p.used)[(int64_t)gn * kUseThreads + threadIdx.x];
      const int k0 = gn * kUseGroup + threadIdx.x * 16;
#pragma unroll
      for (int j = 0; j < 16; ++j) w += k0 + j < n ? (int)((h[j / 4] >> (8 * (j % 4))) & 1) : 0;
    }
    below = use_scan(w, dummy);
  }
  const int nfree = p.num_pages - n;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int id = blockIdx.x * kUseGroup + j * kUseThreads + threadIdx.x;
    const bool used = (flags[j] >> lane) & 1;
    const int rank = s_before[j * kWaves + wave] + __popcll(flags[j] & ((1ull << lane) - 1));
    if (id < p.num_pages) {
      if constexpr (COMPACT) {
        if (!used && id < n) p.list[id - rank] = id;
        if (used && id >= n) {
          p.src[rank - below] = id;
          p.rank[id] = rank - below;
        } else {
          p.remap[id] = used ? id : -1;
        }
      } else {
        if (!used) p.list[id - rank] = id;
        else p.list[nfree + rank] = -1;
      }
    }
  }
  if constexpr (COMPACT) {
    if (blockIdx.x == 0 && threadIdx.x == 0) p.counts[groups] = n - below;  // moves
  }
}

// The four launches above in one workgroup, for small pools and tables: the
// flags are bits in LDS, whose popcounts are scanned; id i's rank is that of its
// word and of the bits below it.
constexpr int kSmallThreads = 1024;
constexpr int kSmallPages = 1 << 16;    // ids
constexpr int kSmallEntries = 1 << 15;  // table entries

template <bool COMPACT>
__global__ __launch_bounds__(kSmallThreads) void use_small_kernel(const UseParams p) {
  constexpr int kWords = kSmallPages / 32, kEach = kWords / kSmallThreads;
  __shared__ uint32_t bits[kWords];
  __shared__ int before[kWords];
  const int tid = threadIdx.x;
#pragma unroll
  for (int k = 0; k < kEach; ++k) bits[tid * kEach + k] = 0;
  for (int i = tid; i < p.nrows; i += kSmallThreads) {
    const int b = p.rows[i];
    if ((unsigned)b >= (unsigned)p.B) continue;
    p.lens[b] = 0;
    if (p.held) p.held[b] = 0;
  }
  __syncthreads();  // the rows' lengths too: one workgroup shares its L1
  constexpr int kWaves = kSmallThreads / 64;
  const int wave = tid >> 6, lane = tid & 63;
  const int per_row = max(1, kWaves / max(p.B, 1));
  for (int u = wave; u < p.B * per_row; u += kWaves) {
    const int b = u / per_row;
    const int cols = used_columns(p, b);
    const int32_t* row = p.pt + (int64_t)b * p.pt_sb;
#pragma unroll 4
    for (int c = (u - b * per_row) * 64 + lane; c < cols; c += per_row * 64) {
      const int id = row[c];
      if ((unsigned)id < (unsigned)p.num_pages) atomicOr(bits + (id >> 5), 1u << (id & 31));
    }
  }
  __syncthreads();
  int x = 0, at;
#pragma unroll
  for (int k = 0; k < kEach; ++k) x += __popc(bits[tid * kEach + k]);
  const int n = use_scan<kSmallThreads>(x, at);
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    before[tid * kEach + k] = at;
    at += __popc(bits[tid * kEach + k]);
  }
  __syncthreads();
  auto rank = [&](int id) { return before[id >> 5] + __popc(bits[id >> 5] & ((1u << (id & 31)) - 1)); };
  const int below = COMPACT && n < p.num_pages ? rank(n) : n;  // used ids below n
  if (tid == 0) {
    *p.total = COMPACT ? n : p.num_pages - n;
    if constexpr (COMPACT) p.counts[(p.num_pages + kUseGroup - 1) / kUseGroup] = n - below;  // moves
  }
  for (int id = tid; id < p.num_pages; id += kSmallThreads) {
    const bool used = (bits[id >> 5] >> (id & 31)) & 1;
    const int r = rank(id);
    if constexpr (COMPACT) {
      if (!used && id < n) p.list[id - r] = id;
      if (used && id >= n) {
        p.src[r - below] = id;
        p.rank[id] = r - below;
      } else {
        p.remap[id] = used ? id : -1;
      }
    } else {
      if (!used) p.list[id - r] = id;
      else p.list[p.num_pages - n + r] = -1;
    }
  }
}

// The moves: blockIdx.y < n planes: copies of that plane; the last: new ids.
__global__ __launch_bounds__(kCopyThreads, 8) void compact_apply_kernel(const Planes planes, const UseParams p,
                                                                        int groups) {
  const int moves = p.counts[groups];
  if ((int)blockIdx.y < planes.n) {
    const Plane pl = planes.p[blockIdx.y];
    const int64_t steps = plane_steps(pl, moves);
    for (int64_t step = blockIdx.x; step < steps; step += gridDim.x)
      copy_step(pl, step, moves, [&](int64_t i, int& s, int& d) {
        s = p.src[i];
        d = p.list[i];
        return true;
      });
    return;
  }
  const int n = *p.total;
  const int64_t stride = (int64_t)gridDim.x * kCopyThreads;
  for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < moves; i += stride)
    p.remap[p.src[i]] = p.list[i];
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    const int cols = used_columns(p, b);
    int32_t* row = p.pt + (int64_t)b * p.pt_sb;
    for (int c = threadIdx.x; c < cols; c += kCopyThreads) {
      const int id = row[c];
      if (id >= n && id < p.num_pages) row[c] = p.list[p.rank[id]];
    }
  }
}

}  // namespace fat

// ===========================================================================
// Host side
// ===========================================================================
namespace {

int dtype_bytes(int32_t dtype) {
  switch (dtype) {
    case FAT_DTYPE_F16:
    case FAT_DTYPE_BF16: return 2;
    case FAT_DTYPE_I8:
    case FAT_DTYPE_FP8E4M3: return 1;
    case FAT_DTYPE_F32: return 4;
    default: return 0;
  }
}

// A plane of `slots` x `heads` rows of `row` bytes (byte strides).
fat::Plane make_plane(void* base, int64_t page, int64_t slots, int64_t slot_stride, int64_t heads, int64_t head_stride,
                      int64_t row) {
  // The dimension with the smaller stride inside; a dimension of one element
  // has no stride of its own.
  if (heads == 1) head_stride = row;
  if (slots == 1) slot_stride = heads == 1 ? row : head_stride * heads;
  int64_t outer = slots, os = slot_stride, inner = heads, is = head_stride;
  if (os < is) {
    std::swap(outer, inner);
    std::swap(os, is);
  }
  if (is == row) {  // rows of the inner dimension lie behind each other
    row *= inner;
    inner = outer;
    is = os;
    outer = 1;
    os = 0;
    if (is == row) {
      row *= inner;
      inner = 1;
      is = 0;
    }
  }
  int log2v = 4;
  const uint64_t bits = (uint64_t)(uintptr_t)base | (uint64_t)page | (uint64_t)(outer > 1 ? os : 0) |
                        (uint64_t)(inner > 1 ? is : 0) | (uint64_t)row;
  while (log2v > 0 && (bits & ((1u << log2v) - 1))) --log2v;
  fat::Plane p{};
  p.base = static_cast<uint8_t*>(base);
  p.page = page;
  p.outer_stride = os;
  p.inner_stride = is;
  p.inner = (uint32_t)inner;
  p.vpr = (uint32_t)(row >> log2v);
  p.vpp = (uint32_t)(outer * inner * (row >> log2v));
  p.inv = p.vpp > 1 ? (uint32_t)((uint64_t(1) << 32) / p.vpp) : 0;
  const uint64_t run = (uint64_t)p.vpp << log2v;
  p.cpp = log2v == 4 && p.vpr == p.vpp && run % fat::kChunk == 0 ? (uint32_t)(run / fat::kChunk) : 0;
  p.log2v = log2v;
  return p;
}

int make_planes(const fat_pool& a, fat::Planes* out, const char* who) {
  if (!a.k_cache || !a.v_cache || !a.quant_k_cache != !a.quant_v_cache || !a.k_scale != !a.v_scale) {
    fat_host::set_error("%s: k_cache and v_cache are required, the 8-bit copy and the scales come in pairs", who);
    return FAT_E_INVALID;
  }
  if (a.num_pages <= 0 || a.page_size <= 0 || a.num_kv_heads <= 0 || a.head_dim <= 0) {
    fat_host::set_error("%s: num_pages, page_size, num_kv_heads and head_dim must be positive", who);
    return FAT_E_INVALID;
  }
  const int64_t eb = dtype_bytes(a.dtype);
  if (!eb) {
    fat_host::set_error("%s: unknown dtype %d", who, a.dtype);
    return FAT_E_UNSUPPORTED;
  }
  const int64_t P = a.page_size, H = a.num_kv_heads, D = a.head_dim;
  if (P > (1 << 30) / D / H || P * H * D * eb > (1 << 30)) {
    fat_host::set_error("%s: pages of more than 1 GiB", who);
    return FAT_E_UNSUPPORTED;
  }
  auto ok = [&](int64_t sp, int64_t ss, int64_t sh) {
    return (a.num_pages == 1 || sp > 0) && (P == 1 || ss > 0) && (H == 1 || sh > 0);
  };
  if (!ok(a.k_stride_page, a.k_stride_slot, a.k_stride_head) || !ok(a.v_stride_page, a.v_stride_slot, a.v_stride_head) ||
      (a.quant_k_cache && (!ok(a.qk_stride_page, a.qk_stride_slot, a.qk_stride_head) ||
                           !ok(a.qv_stride_page, a.qv_stride_slot, a.qv_stride_head))) ||
      (a.k_scale && ((a.num_pages > 1 && a.scale_stride_page <= 0) || (H > 1 && a.scale_stride_head <= 0)))) {
    fat_host::set_error("%s: the strides of pages, slots, heads and scales must be positive", who);
    return FAT_E_INVALID;
  }
  out->n = 0;
  out->num_pages = a.num_pages;
  auto add = [&](void* base, int64_t b, int64_t sp, int64_t ss, int64_t sh) {
    out->p[out->n++] = make_plane(base, b * sp, P, b * ss, H, b * sh, b * D);
  };
  add(a.k_cache, eb, a.k_stride_page, a.k_stride_slot, a.k_stride_head);
  add(a.v_cache, eb, a.v_stride_page, a.v_stride_slot, a.v_stride_head);
  if (a.quant_k_cache) {
    add(a.quant_k_cache, 1, a.qk_stride_page, a.qk_stride_slot, a.qk_stride_head);
    add(a.quant_v_cache, 1, a.qv_stride_page, a.qv_stride_slot, a.qv_stride_head);
  }
  if (a.k_scale) {
    out->p[out->n++] = make_plane(a.k_scale, 4 * a.scale_stride_page, 1, 0, H, 4 * a.scale_stride_head, 4);
    out->p[out->n++] = make_plane(a.v_scale, 4 * a.scale_stride_page, 1, 0, H, 4 * a.scale_stride_head, 4);
  }
  return FAT_OK;
}

int64_t host_steps(const fat::Plane& p, int64_t count) {
  return p.cpp ? (count * p.cpp + fat::kStepChunks - 1) / fat::kStepChunks
               : (count * p.vpp + fat::kStepVectors - 1) / fat::kStepVectors;
}

// Workgroups (of 256 threads) that fill the chip: 8 per CU.
constexpr int64_t kFullGrid = 8 * 256;
// A workgroup per step where the number of steps is known (2 % over kFullGrid's
// loops), within a launch's limit of 2^32 threads.
constexpr int64_t kWideGrid = 1 << 22;

unsigned copy_grid(const fat::Planes& pl, int64_t count, int64_t limit = kFullGrid) {
  int64_t most = 1;
  for (int i = 0; i < pl.n; ++i) most = std::max(most, host_steps(pl.p[i], count));
  return (unsigned)std::min(most, limit);
}

int64_t use_groups(int64_t num_pages) { return (num_pages + fat::kUseGroup - 1) / fat::kUseGroup; }

// Workspace: flags, three id lists, counts (one more: the number of moves).
void use_workspace(fat::UseParams* p, void* ws) {
  const int64_t groups = use_groups(p->num_pages);
  uint8_t* at = static_cast<uint8_t*>(ws);
  p->used = at;
  at += groups * fat::kUseGroup;
  auto ints = [&](int64_t n) {
    int32_t* r = reinterpret_cast<int32_t*>(at);
    at += 4 * n;
    return r;
  };
  p->src = ints(groups * fat::kUseGroup);
  p->rank = ints(groups * fat::kUseGroup);
  p->list = ints(groups * fat::kUseGroup);
  p->counts = ints(groups + 1);
}

bool use_args_ok(const void* lens, const void* pt, int64_t pt_sb, int batch, int max_pages, int num_pages, int P,
                 const void* ws, const char* who) {
  if (!lens || !pt || !ws) {
    fat_host::set_error("%s: a required pointer is NULL", who);
    return false;
  }
  if (batch < 0 || max_pages <= 0 || num_pages <= 0 || num_pages > (1 << 30) || P <= 0 || pt_sb < 0 ||
      (batch > 1 && pt_sb < max_pages) || (uintptr_t)ws % 16) {
    fat_host::set_error("%s: batch %d, max_pages %d, num_pages %d, page_size %d, page_table_stride %lld or the "
                        "workspace's alignment invalid", who, batch, max_pages, num_pages, P, (long long)pt_sb);
    return false;
  }
  return true;
}

// The pages in use, and the lists of them.  One workgroup where it has at most
// 32 table entries and 64 ids per thread, else four launches (each some 2 us).
template <bool COMPACT>
int launch_use(const fat::UseParams& p, hipStream_t stream) {
  if (p.num_pages <= fat::kSmallPages && (int64_t)p.B * p.max_pages <= fat::kSmallEntries) {
    hipLaunchKernelGGL((fat::use_small_kernel<COMPACT>), dim3(1), dim3(fat::kSmallThreads), 0, stream, p);
    return fat_host::launch_status("use_small_kernel");
  }
  const int64_t groups = use_groups(p.num_pages);
  const int64_t words = groups * fat::kUseGroup / 16;
  const int64_t most = std::max<int64_t>(words, p.nrows);
  const unsigned clear = (unsigned)std::min<int64_t>((most + fat::kUseThreads - 1) / fat::kUseThreads, kFullGrid);
  hipLaunchKernelGGL(fat::use_clear_kernel, dim3(clear), dim3(fat::kUseThreads), 0, stream, p, words);
  int rc = fat_host::launch_status("use_clear_kernel");
  if (rc != FAT_OK) return rc;
  if (p.B > 0) {
    constexpr int kColumns = fat::kMarkEach * fat::kUseThreads;
    const dim3 grid((unsigned)((p.max_pages + kColumns - 1) / kColumns), (unsigned)std::min(p.B, 32768));
    hipLaunchKernelGGL(fat::use_mark_kernel, grid, dim3(fat::kUseThreads), 0, stream, p);
    if ((rc = fat_host::launch_status("use_mark_kernel")) != FAT_OK) return rc;
  }
  hipLaunchKernelGGL(fat::use_count_kernel, dim3((unsigned)groups), dim3(fat::kUseThreads), 0, stream, p);
  if ((rc = fat_host::launch_status("use_count_kernel")) != FAT_OK) return rc;
  hipLaunchKernelGGL((fat::use_list_kernel<COMPACT>), dim3((unsigned)groups), dim3(fat::kUseThreads), 0, stream, p);
  return fat_host::launch_status("use_list_kernel");
}

}  // namespace

extern "C" size_t fat_pages_workspace_bytes(int32_t num_pages) {
  if (num_pages <= 0) return 0;
  const int64_t groups = use_groups(num_pages);
  return (size_t)(groups * fat::kUseGroup * 13 + 4 * (groups + 1));
}

extern "C" int fat_copy_pages(const fat_copy_pages_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || (a->count > 0 && (!a->src || !a->dst))) {
    fat_host::set_error("fat_copy_pages: src and dst are required");
    return FAT_E_INVALID;
  }
  fat::Planes planes{};
  int rc = make_planes(a->pool, &planes, "fat_copy_pages");
  if (rc != FAT_OK) return rc;
  if (a->count < 0 || a->count > 0x7fffffff) {
    fat_host::set_error("fat_copy_pages: count must be in [0, 2^31), got %lld", (long long)a->count);
    return FAT_E_INVALID;
  }
  if (a->count == 0) return FAT_OK;
  const dim3 grid(copy_grid(planes, a->count, kWideGrid), planes.n), block(fat::kCopyThreads);
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  hipLaunchKernelGGL(fat::copy_pages_kernel, grid, block, 0, stream, planes, a->src, a->dst, a->count);
  return fat_host::launch_status("copy_pages_kernel");
}

extern "C" int fat_fork_sequences(const fat_fork_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || !a->page_table || !a->seq_lens || (a->count > 0 && (!a->parents || !a->children || !a->pages))) {
    fat_host::set_error("fat_fork_sequences: parents, children, pages, page_table and seq_lens are required");
    return FAT_E_INVALID;
  }
  fat::ForkParams prm{};
  int rc = make_planes(a->pool, &prm.planes, "fat_fork_sequences");
  if (rc != FAT_OK) return rc;
  if (a->count < 0 || a->batch <= 0 || a->max_pages <= 0 || (a->batch > 1 && a->page_table_stride < a->max_pages)) {
    fat_host::set_error("fat_fork_sequences: count %d, batch %d, max_pages %d or page_table_stride %lld invalid",
                        a->count, a->batch, a->max_pages, (long long)a->page_table_stride);
    return FAT_E_INVALID;
  }
  if (a->count > a->batch) {  // some row would be given twice
    fat_host::set_error("fat_fork_sequences: at most batch = %d forks in a call, got %d", a->batch, a->count);
    return FAT_E_INVALID;
  }
  if (a->count == 0) return FAT_OK;
  prm.pt = a->page_table;
  prm.lens = a->seq_lens;
  prm.pt_sb = a->page_table_stride;
  prm.B = a->batch;
  prm.max_pages = a->max_pages;
  prm.P = a->pool.page_size;
  const unsigned table = (unsigned)std::min<int64_t>((a->max_pages + 1023) / 1024, 64);
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  constexpr int kHeight = 65535;  // of a grid; the forks of a call are independent
  for (int64_t i = 0; i < a->count && rc == FAT_OK; i += kHeight) {
    prm.parents = a->parents + i;
    prm.children = a->children + i;
    prm.pages = a->pages + i;
    const dim3 grid(std::max(copy_grid(prm.planes, 1), table), (unsigned)std::min<int64_t>(a->count - i, kHeight),
                    prm.planes.n + 1);
    hipLaunchKernelGGL(fat::fork_kernel, grid, dim3(fat::kCopyThreads), 0, stream, prm);
    rc = fat_host::launch_status("fork_kernel");
  }
  return rc;
}

extern "C" int fat_free_sequences(const fat_free_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || !a->pages || !a->num_free || (a->count > 0 && !a->rows)) {
    fat_host::set_error("fat_free_sequences: rows, pages and num_free are required");
    return FAT_E_INVALID;
  }
  if (!use_args_ok(a->seq_lens, a->page_table, a->page_table_stride, a->batch, a->max_pages, a->num_pages,
                   a->page_size, a->workspace, "fat_free_sequences"))
    return FAT_E_INVALID;
  if (a->count < 0) {
    fat_host::set_error("fat_free_sequences: count must be >= 0, got %d", a->count);
    return FAT_E_INVALID;
  }
  fat::UseParams prm{};
  prm.lens = a->seq_lens;
  prm.held = a->held;
  prm.pt = const_cast<int32_t*>(a->page_table);
  prm.rows = a->rows;
  prm.pt_sb = a->page_table_stride;
  prm.B = a->batch;
  prm.max_pages = a->max_pages;
  prm.P = a->page_size;
  prm.num_pages = a->num_pages;
  prm.nrows = a->count;
  use_workspace(&prm, a->workspace);
  prm.list = a->pages;
  prm.total = a->num_free;
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  return launch_use<false>(prm, stream);
}

extern "C" int fat_compact_pages(const fat_compact_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || !a->remap || !a->num_used) {
    fat_host::set_error("fat_compact_pages: remap and num_used are required");
    return FAT_E_INVALID;
  }
  fat::Planes planes{};
  int rc = make_planes(a->pool, &planes, "fat_compact_pages");
  if (rc != FAT_OK) return rc;
  if (!use_args_ok(a->seq_lens, a->page_table, a->page_table_stride, a->batch, a->max_pages, a->pool.num_pages,
                   a->pool.page_size, a->workspace, "fat_compact_pages"))
    return FAT_E_INVALID;
  fat::UseParams prm{};
  prm.lens = const_cast<int32_t*>(a->seq_lens);
  prm.held = const_cast<int32_t*>(a->held);
  prm.pt = a->page_table;
  prm.pt_sb = a->page_table_stride;
  prm.B = a->batch;
  prm.max_pages = a->max_pages;
  prm.P = a->pool.page_size;
  prm.num_pages = a->pool.num_pages;
  use_workspace(&prm, a->workspace);
  prm.remap = a->remap;
  prm.total = a->num_used;
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  if ((rc = launch_use<true>(prm, stream)) != FAT_OK) return rc;
  const int groups = (int)use_groups(prm.num_pages);
  // At most half of the pages move; the number is known on the device only.
  const unsigned wide = std::max(copy_grid(planes, prm.num_pages / 2 + 1),
                                 (unsigned)std::min<int64_t>(std::max(prm.B, 1), kFullGrid));
  const dim3 grid(wide, planes.n + 1), block(fat::kCopyThreads);
  hipLaunchKernelGGL(fat::compact_apply_kernel, grid, block, 0, stream, planes, prm, groups);
  return fat_host::launch_status("compact_apply_kernel");
}
