// validate.hip -- the device half of the validation: one launch reduces the
// lengths, offsets and used page-table entries that a call is to check
// (flashattn_tile/paging.py:84-130 validate_cache, as called by
// flashattn_tile/kernels/decode.py:503-522, and kernels/prefill.py:194-233)
// to a few numbers, instead of a dozen framework reductions.
//
// fat_check_begin / fat_check_wait: what the Python package runs.  The kernel
// writes its numbers into page-locked host memory and the host polls them, so
// a validated call neither copies nor synchronises.
//
// fat_cache_stats: the same numbers of a paged cache in device memory, for
// callers of the C library that have no page-locked words or copy them with
// other results.
#include <limits.h>

#include <algorithm>
#include <atomic>
#include <chrono>

#include "fat_common.h"

namespace fat {

constexpr int kStatsThreads = 1024;

// out[0..4] = min(seq_lens), max(seq_lens), min and max of page_table[b, c]
// over every row b and column c < min(ceil(max_len / P), max_pages) (INT_MAX
// and INT_MIN when no entry is used), sum_b ceil(max(seq_lens[b], 0) / P).
__global__ __launch_bounds__(kStatsThreads) void cache_stats_kernel(const int32_t* __restrict__ lens,
                                                                    const int32_t* __restrict__ pt, int B,
                                                                    int max_pages, int64_t pt_sb, int P,
                                                                    int64_t* __restrict__ out) {
  __shared__ int s_min[kStatsThreads / 64], s_max[kStatsThreads / 64];
  __shared__ long long s_sum[kStatsThreads / 64];
  __shared__ int s_need;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = tid >> 6;
  int mn = INT_MAX, mx = INT_MIN;
  long long pages = 0;
  for (int b = tid; b < B; b += kStatsThreads) {
    const int l = lens[b];
    mn = min(mn, l);
    mx = max(mx, l);
    pages += (max(l, 0) + (long long)P - 1) / P;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    mn = min(mn, __shfl_xor(mn, off));
    mx = max(mx, __shfl_xor(mx, off));
    pages += __shfl_xor(pages, off);
  }
  if (lane == 0) {
    s_min[w] = mn;
    s_max[w] = mx;
    s_sum[w] = pages;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kStatsThreads / 64; ++i) {
      mn = min(mn, s_min[i]);
      mx = max(mx, s_max[i]);
      pages += s_sum[i];
    }
    out[0] = mn;
    out[1] = mx;
    out[4] = pages;
    // Columns the longest sequence uses (as the torch restatement: floor((max + P - 1) / P)).
    const long long need = mx > 0 ? ((long long)mx + P - 1) / P : 0;
    s_need = (int)min(need, (long long)max_pages);
  }
  __syncthreads();
  const int need = s_need;
  int pmn = INT_MAX, pmx = INT_MIN;
  const long long n = (long long)B * need;
  for (long long i = tid; i < n; i += kStatsThreads) {
    const int b = (int)(i / need);
    const int c = (int)(i - (long long)b * need);
    const int v = pt[b * pt_sb + c];
    pmn = min(pmn, v);
    pmx = max(pmx, v);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    pmn = min(pmn, __shfl_xor(pmn, off));
    pmx = max(pmx, __shfl_xor(pmx, off));
  }
  __syncthreads();  // s_min / s_max are reused
  if (lane == 0) {
    s_min[w] = pmn;
    s_max[w] = pmx;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kStatsThreads / 64; ++i) {
      pmn = min(pmn, s_min[i]);
      pmx = max(pmx, s_max[i]);
    }
    out[2] = pmn;
    out[3] = pmx;
  }
}

constexpr int kCheckThreads = 256;
// Table entries per workgroup.  One workgroup of 1024 threads took 27.8 us
// for a table of 64 sequences of up to 1000 pages; 16 workgroups of 256 take
// 8.5 us, of which the lengths, the launch and the writes to the host are 4.3.
constexpr int64_t kCheckEntries = 4096;

struct CheckParams {
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* lens;
  const int32_t* pt;
  int64_t pt_sb;
  int64_t* host;
  int64_t ticket;
  int32_t B, max_pages, P;
  const float* values;
  int64_t count;
  const int32_t* ids[3];
  int32_t num_pages;
  int32_t tokens;
  const int32_t* held;
};

struct RMin { template <typename T> static __device__ __forceinline__ T f(T a, T b) { return a < b ? a : b; } };
struct RMax { template <typename T> static __device__ __forceinline__ T f(T a, T b) { return a > b ? a : b; } };
struct RSum { template <typename T> static __device__ __forceinline__ T f(T a, T b) { return a + b; } };
struct ROr { template <typename T> static __device__ __forceinline__ T f(T a, T b) { return a | b; } };

// Reduction over the workgroup; every thread gets the result.
template <typename Op>
__device__ __forceinline__ long long check_reduce(long long x) {
  __shared__ long long s[kCheckThreads / 64];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x = Op::f(x, __shfl_xor(x, off));
  __syncthreads();  // the previous reduction's reads are done
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  x = s[0];
#pragma unroll
  for (int i = 1; i < kCheckThreads / 64; ++i) x = Op::f(x, s[i]);
  return x;
}

// Latency-bound: a few dependent loads, then a PCIe write per workgroup.  The
// stores are system-scope (written through to host memory) and each
// workgroup's ticket follows its results once they are complete (vmcnt(0)),
// so no cache is written back and the host needs no synchronisation.
template <int KIND>
__global__ __launch_bounds__(kCheckThreads) void check_kernel(const CheckParams p) {
  constexpr bool TABLE = KIND == FAT_CHECK_CACHE || KIND == FAT_CHECK_PAGED;
  constexpr bool LENS = TABLE || KIND == FAT_CHECK_APPEND;
  constexpr bool CU = KIND == FAT_CHECK_VARLEN || KIND == FAT_CHECK_PAGED;
  const int tid = threadIdx.x;
  auto put = [&](int word, long long v) {
    __hip_atomic_store(p.host + word, (int64_t)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  };
  long long mn = INT_MAX, mx = INT_MIN, pages = 0, flags = 0, mq = INT_MIN, mk = INT_MIN, keyless = INT_MAX;
  int pmn = INT_MAX, pmx = INT_MIN;
  for (int b = tid; b < p.B; b += kCheckThreads) {
    long long len = 0, lq = 0, lk = 0;
    if constexpr (LENS) {
      len = p.lens[b];
      mn = min(mn, len);
      mx = max(mx, len);
      pages += (max(len, 0ll) + p.P - 1) / p.P;
      lk = len;
    }
    if constexpr (CU) {
      lq = (long long)p.cu_q[b + 1] - p.cu_q[b];
      if constexpr (KIND == FAT_CHECK_VARLEN) lk = (long long)p.cu_k[b + 1] - p.cu_k[b];
      flags |= (lq < 0 ? 1 : 0) | (KIND == FAT_CHECK_VARLEN && lk < 0 ? 2 : 0) | (lk < lq ? 4 : 0);
      mq = max(mq, lq);
      mk = max(mk, lk);
      // a packed sequence without keys, a cached one without tokens
      if (lq > 0 && (KIND == FAT_CHECK_VARLEN ? lk == 0 : lk <= 0)) keyless = min(keyless, (long long)b);
    }
    if constexpr (KIND == FAT_CHECK_APPEND) {
      const int block = len < 0 ? 0 : (int)min(len / p.P, (long long)p.max_pages - 1);
      const int id = p.pt[b * p.pt_sb + block];
      pmn = min(pmn, id);
      pmx = max(pmx, id);
    }
  }
  if constexpr (KIND == FAT_CHECK_RANGE) {
    // Order-preserving integers, so that the reductions below apply; a NaN is
    // tracked apart (bit 0 of flags).
    const int64_t step = (int64_t)gridDim.x * kCheckThreads;
#pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * kCheckThreads + tid; i < p.count; i += step) {
      const float v = p.values[i];
      const int bits = __builtin_bit_cast(int, v);
      const int key = bits ^ ((bits >> 31) & 0x7fffffff);
      pmn = min(pmn, key);
      pmx = max(pmx, key);
      flags |= v != v ? 1 : 0;
    }
    pmn = (int)check_reduce<RMin>(pmn);
    pmx = (int)check_reduce<RMax>(pmx);
    const bool nan = check_reduce<ROr>(flags) != 0;
    pmn = nan ? INT_MIN : pmn;  // no float's key: the host sees a NaN
    pmx = nan ? INT_MAX : pmx;
  }
  if constexpr (LENS) mx = check_reduce<RMax>(mx);
  if constexpr (TABLE) {
    const long long need = mx > 0 ? min((mx + p.P - 1) / p.P, (long long)p.max_pages) : 0;
    const long long n = (long long)p.B * need;
    const uint32_t cols = (uint32_t)need;
    const long long step = (long long)gridDim.x * kCheckThreads;
#pragma unroll 4
    for (long long i = (long long)blockIdx.x * kCheckThreads + tid; i < n; i += step) {
      const long long b = n <= 0xffffffffll ? (long long)((uint32_t)i / cols) : i / need;
      const int id = p.pt[b * p.pt_sb + (i - b * need)];
      pmn = min(pmn, id);
      pmx = max(pmx, id);
    }
  }
  if constexpr (TABLE || KIND == FAT_CHECK_APPEND) {
    pmn = (int)check_reduce<RMin>(pmn);
    pmx = (int)check_reduce<RMax>(pmx);
  }
  if (blockIdx.x == 0) {  // uniform
    if constexpr (LENS) {
      mn = check_reduce<RMin>(mn);
      pages = check_reduce<RSum>(pages);
    }
    if constexpr (CU) {
      flags = check_reduce<ROr>(flags);
      mq = check_reduce<RMax>(mq);
      mk = check_reduce<RMax>(mk);
      keyless = check_reduce<RMin>(keyless);
    }
    if (tid == 0) {
      put(0, mn);
      put(1, mx);
      put(2, pages);
      if constexpr (CU) {
        put(3, p.cu_q[0]);
        put(4, p.cu_q[p.B]);
        if constexpr (KIND == FAT_CHECK_VARLEN) {
          put(5, p.cu_k[0]);
          put(6, p.cu_k[p.B]);
        }
        put(7, flags);
        put(8, mq);
        put(9, mk);
        const bool any = keyless != INT_MAX;
        put(10, any ? keyless : -1);
        put(11, any ? (long long)p.cu_q[keyless + 1] - p.cu_q[keyless] : 0);
      }
    }
  }
  if (tid == 0) {
    const int at = FAT_CHECK_RESULTS + 2 * blockIdx.x;
    put(at, (long long)(((unsigned long long)(uint32_t)pmx << 32) | (uint32_t)pmn));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the results are complete
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    put(at + 1, p.ticket);
  }
}

// FREE and SHARED: workgroup 0 reduces the lengths (and the rows to free, the
// groups, their prefixes), the others' waves take the used columns of the table,
// SHARED with a comparison of those that a prefix fills with the group's first row
// (a difference makes the smallest id INT_MIN, which stands for nothing else).  A
// row's columns go to `per_row` waves in turn, so no entry costs a division and few
// long rows spread as well as many short ones: 512 rows of up to 8000 ids take 8 us,
// 4 rows 5.
constexpr int kRowsThreads = 1024;
constexpr int kRowsWaves = kRowsThreads / 64;
constexpr int64_t kRowsEntries = 4096;  // table entries per workgroup

// Reduces the first `waves` waves' x[0 .. N - 1] (x[i] by op[i]): all of a wave's
// shuffles overlap, and the workgroup synchronises once.  Threads i < N return
// the i-th.  (Waves without an element shuffle nothing: sixteen waves' took 4 us
// of a check's 11.)
enum RowOp : int { kMin, kMax, kSum, kOr };
template <int N>
__device__ __forceinline__ long long rows_reduce(long long (&x)[N], const RowOp (&op)[N], int waves) {
  __shared__ long long s[kRowsWaves][N];
  auto f = [](RowOp o, long long a, long long b) {
    return o == kMin ? (a < b ? a : b) : o == kMax ? (a > b ? a : b) : o == kSum ? a + b : (a | b);
  };
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < waves) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = f(op[i], x[i], __shfl_xor(x[i], off));
    }
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[wave][i] = x[i];
    }
  }
  __syncthreads();
  long long r = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if ((int)threadIdx.x == i) {
      r = s[0][i];
      for (int w = 1; w < waves; ++w) r = f(op[i], r, s[w][i]);
    }
  }
  return r;
}

template <int KIND>
__global__ __launch_bounds__(kRowsThreads) void check_rows_kernel(const CheckParams p) {
  constexpr bool SHARED = KIND == FAT_CHECK_SHARED;
  const int tid = threadIdx.x;
  const int G = (int)p.count;
  const int32_t* prefix = p.ids[0];
  auto put = [&](int word, long long v) {
    __hip_atomic_store(p.host + word, (int64_t)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
  };
  auto pages_of = [&](int len) { return (int)(((unsigned)max(len, 0) + (unsigned)p.P - 1) / (unsigned)p.P); };
  long long range[2] = {INT_MAX, INT_MIN};
  const RowOp range_op[2] = {kMin, kMax};
  const int workers = ((int)gridDim.x - 1) * kRowsWaves;
  if (blockIdx.x == 0) {  // uniform
    if constexpr (SHARED) {
      // min and max length, pages, flags, sequences of a group, prefix, keys behind it, and three sums
      long long x[10] = {INT_MAX, INT_MIN, 0, 0, 0, 0, 0, 0, 0, 0};
      const RowOp op[10] = {kMin, kMax, kSum, kOr, kMax, kMax, kMax, kSum, kSum, kSum};
      for (int b = tid; b < p.B; b += kRowsThreads) {
        const long long len = p.lens[b];
        int g = -1, hi = G;  // the largest g with cu_q[g] <= b, if any
        while (hi - g > 1) {
          const int mid = (g + hi) >> 1;
          if (p.cu_q[mid] <= b) g = mid;
          else hi = mid;
        }
        const long long n = g < 0 ? 0 : prefix[g];
        x[0] = min(x[0], len);
        x[1] = max(x[1], len);
        x[2] += pages_of((int)len);
        x[3] |= n > len - p.tokens + 1 ? 4 : 0;
        x[6] = max(x[6], len - n);
        x[8] += len - n;
      }
      for (int g = tid; g < G; g += kRowsThreads) {
        const long long seqs = (long long)p.cu_q[g + 1] - p.cu_q[g], n = prefix[g];
        x[3] |= (seqs < 0 ? 1 : 0) | (n < 0 ? 2 : 0);
        x[4] = max(x[4], seqs);
        if (seqs > 0) {
          x[5] = max(x[5], n);
          x[7] += n;
          x[9] += n * seqs;
        }
      }
      const long long r = rows_reduce(x, op, (int)min((max((int64_t)p.B, p.count) + 63) / 64, (int64_t)kRowsWaves));
      const int word[10] = {0, 1, 2, 7, 5, 6, 8, 9, 10, 11};
#pragma unroll
      for (int i = 0; i < 10; ++i) {
        if (tid == i) put(word[i], r);
      }
      if (tid == 0) {
        put(3, p.cu_q[0]);
        put(4, p.cu_q[G]);
      }
    } else {
      long long x[4] = {INT_MAX, INT_MIN, 0, 0};
      const RowOp op[4] = {kMin, kMax, kSum, kOr};
      for (int b = tid; b < p.B; b += kRowsThreads) {
        const long long len = p.lens[b];
        x[0] = min(x[0], len);
        x[1] = max(x[1], len);
        x[2] += pages_of((int)len);
      }
      if (p.held) {
        for (int b = tid; b < p.B; b += kRowsThreads) x[3] |= p.held[b] > p.max_pages ? 2 : 0;
      }
      for (int64_t i = tid; i < p.count; i += kRowsThreads) x[3] |= (unsigned)p.ids[0][i] >= (unsigned)p.B ? 1 : 0;
      const long long r = rows_reduce(x, op, (int)min((max((int64_t)p.B, p.count) + 63) / 64, (int64_t)kRowsWaves));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (tid == i) put(i < 3 ? i : 7, r);
      }
    }
  } else {
    const int lane = tid & 63;
    const int worker = ((int)blockIdx.x - 1) * kRowsWaves + __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per_row = max(1, workers / p.B);
    int pmn = INT_MAX, pmx = INT_MIN;
    bool differs = false;
    for (long long u = worker; u < (long long)p.B * per_row; u += workers) {
      const int b = (int)(u / per_row);
      const int32_t* row = p.pt + b * p.pt_sb;
      const int32_t* first = row;
      int cols = min(pages_of(p.lens[b]), p.max_pages);
      int same = 0;
      if constexpr (SHARED) {
        // The largest g with cu_q[g] <= b, if any: 64 samples at a time.
        int g = -1;
        for (long long lo = 0, n = G; n > 0;) {
          const long long step = (n + 63) / 64;
          const long long at = lo + lane * step;
          const unsigned long long below = __ballot(at < lo + n && p.cu_q[at < lo + n ? at : lo] <= b);
          if (!below) break;
          g = (int)(lo + (63 - __clzll(below)) * step);
          n = min(step, lo + n - g) - 1;
          lo = g + 1;
        }
        const int lead = g < 0 ? b : max(p.cu_q[g], 0);
        same = lead == b ? 0 : min(max(prefix[g], 0) / p.P, cols);
        first = p.pt + lead * p.pt_sb;
      }
      if constexpr (!SHARED) {
        if (p.held) cols = min(max(cols, p.held[b]), p.max_pages);
      }
      const int stride = per_row * 64;
#pragma unroll 8
      for (long long c = (u - (long long)b * per_row) * 64 + lane; c < cols; c += stride) {
        const int id = row[c];
        pmn = min(pmn, id);
        pmx = max(pmx, id);
        if constexpr (SHARED) {
          if (c < same) differs |= first[c] != id;
        }
      }
    }
    range[0] = differs ? INT_MIN : SHARED ? max(pmn, INT_MIN + 1) : pmn;
    range[1] = pmx;
    const long long r = rows_reduce(range, range_op, kRowsWaves);
    range[0] = r;
    range[1] = __shfl(r, 1);
  }
  if (tid < 64) {  // the wave whose results the tickets follow
    const int at = FAT_CHECK_RESULTS + 2 * blockIdx.x;
    if (tid == 0) put(at, (long long)(((unsigned long long)(uint32_t)range[1] << 32) | (uint32_t)range[0]));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the results are complete
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (tid == 0) put(at + 1, p.ticket);
  }
}

// COPY and FORK: ranges, and ids that are given twice or on both sides.  One
// workgroup marks a list's ids in a bitmap in LDS, 2^19 ids at a time (a pool of
// more takes several turns over the list): the bit that was there before is a
// repetition, and the other list's ids are looked up in it.  8192 pairs take 7.6
// us (30 with the owners of the ids in device memory), 16 pairs 2.5.  FORK: the
// other workgroups mark the pages that the forks take, and look the used columns
// of all rows up among them (one that is makes the smallest id INT_MIN).
constexpr int kListThreads = 1024;
constexpr int kListIds = 1 << 19;

template <int KIND>
__global__ __launch_bounds__(kListThreads) void check_lists_kernel(const CheckParams p) {
  constexpr bool FORK = KIND == FAT_CHECK_FORK;
  __shared__ uint32_t bits[kListIds / 32];
  __shared__ int s_flags;
  const int tid = threadIdx.x;
  const int n = (int)p.count;
  const int32_t* a = p.ids[0];
  const int32_t* b = p.ids[1];
  const int32_t* pages = p.ids[2];
  const int limit = FORK ? p.B : p.num_pages;
  int flags = 0;
  if (tid == 0) s_flags = 0;
  auto clear = [&](int ids) {
    __syncthreads();
    for (int i = tid; i < (ids + 31) / 32; i += kListThreads) bits[i] = 0;
    __syncthreads();
  };
  auto mark = [&](unsigned x) { return (atomicOr(bits + (x >> 5), 1u << (x & 31)) >> (x & 31)) & 1; };
  // FORK: whether fork i's parent ends inside a page (its pages[i] is used).
  auto tail = [&](int i, int& len) {
    const int parent = a[i];
    len = (unsigned)parent < (unsigned)limit ? p.lens[parent] : 0;
    return len > 0 && len <= (int64_t)p.max_pages * p.P && len % p.P != 0;
  };
  auto finish = [&](int word, long long v) {
    auto put = [&](int at, long long x) {
      __hip_atomic_store(p.host + at, (int64_t)x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    };
    put(word, v);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the result is complete
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    put(FAT_CHECK_RESULTS + 2 * blockIdx.x + 1, p.ticket);
  };
  if constexpr (FORK) {
    if (blockIdx.x > 0) {  // uniform
      const int lane = tid & 63;
      const int workers = ((int)gridDim.x - 1) * (kListThreads / 64);
      const int worker = ((int)blockIdx.x - 1) * (kListThreads / 64) + __builtin_amdgcn_readfirstlane(tid >> 6);
      const int per_row = max(1, workers / p.B);
      bool found = false;
      for (int base = 0; base < p.num_pages; base += min(kListIds, p.num_pages - base)) {
        const unsigned ids = min(kListIds, p.num_pages - base);
        clear(ids);
        for (int i = tid; i < n; i += kListThreads) {
          int len;
          if (tail(i, len) && pages[i] >= base && (unsigned)(pages[i] - base) < ids) mark(pages[i] - base);
        }
        __syncthreads();
        for (long long u = worker; u < (long long)p.B * per_row; u += workers) {
          const int r = (int)(u / per_row);
          const int32_t* row = p.pt + r * p.pt_sb;
          const int64_t used = ((int64_t)max(p.lens[r], 0) + p.P - 1) / p.P;
          const int cols = (int)min(used, (int64_t)p.max_pages);
#pragma unroll 8
          for (long long c = (u - (long long)r * per_row) * 64 + lane; c < cols; c += per_row * 64) {
            const int id = row[c];
            if (id >= base && (unsigned)(id - base) < ids) found |= (bits[(id - base) >> 5] >> ((id - base) & 31)) & 1;
          }
        }
      }
      if (found) s_flags = 1;
      __syncthreads();
      if (tid == 0) finish(FAT_CHECK_RESULTS + 2 * blockIdx.x, s_flags ? (long long)(uint32_t)INT_MIN : (long long)INT_MAX);
      return;
    }
  }
  for (int base = 0; base < limit; base += min(kListIds, limit - base)) {
    const unsigned ids = min(kListIds, limit - base);
    clear(ids);
#pragma unroll 8
    for (int i = tid; i < n; i += kListThreads) {
      const int y = b[i];
      if ((unsigned)y >= (unsigned)limit) flags |= 2;
      else if ((unsigned)(y - base) < ids && mark(y - base)) flags |= 4;
    }
    __syncthreads();
#pragma unroll 8
    for (int i = tid; i < n; i += kListThreads) {
      const int x = a[i];
      if ((unsigned)x >= (unsigned)limit) flags |= 1;
      else if ((unsigned)(x - base) < ids && ((bits[(x - base) >> 5] >> ((x - base) & 31)) & 1)) flags |= 8;
    }
  }
  if constexpr (FORK) {
    for (int i = tid; i < n; i += kListThreads) {
      const int x = a[i], y = b[i];
      int len;
      if ((unsigned)y < (unsigned)limit && p.lens[y] != 0) flags |= 16;
      if (tail(i, len)) {
        if ((unsigned)p.pt[x * p.pt_sb + len / p.P] >= (unsigned)p.num_pages) flags |= 64;
        if ((unsigned)pages[i] >= (unsigned)p.num_pages) flags |= 128;
      }
      if (len < 0 || len > (int64_t)p.max_pages * p.P) flags |= 32;
    }
    for (int base = 0; base < p.num_pages; base += min(kListIds, p.num_pages - base)) {
      const unsigned ids = min(kListIds, p.num_pages - base);
      clear(ids);
      for (int i = tid; i < n; i += kListThreads) {
        int len;
        if (tail(i, len) && (unsigned)(pages[i] - base) < ids && mark(pages[i] - base)) flags |= 256;
      }
    }
  }
  __syncthreads();
  if (flags) atomicOr(&s_flags, flags);
  __syncthreads();
  if (tid == 0) {
    __hip_atomic_store(p.host + FAT_CHECK_RESULTS, (int64_t)INT_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    finish(7, s_flags);
  }
}

}  // namespace fat

namespace {

int check_groups(const fat_check_args* a) {
  if (a->kind == FAT_CHECK_VARLEN || a->kind == FAT_CHECK_APPEND || a->kind == FAT_CHECK_COPY) return 1;
  if (a->kind == FAT_CHECK_SHARED || a->kind == FAT_CHECK_FREE || a->kind == FAT_CHECK_FORK) {
    const int64_t n = ((int64_t)a->batch * a->max_pages + fat::kRowsEntries - 1) / fat::kRowsEntries;
    return (int)std::min<int64_t>(1 + std::max<int64_t>(n, 1), FAT_CHECK_MAX_GROUPS);
  }
  const int64_t entries = a->kind == FAT_CHECK_RANGE ? a->count : (int64_t)a->batch * a->max_pages;
  const int64_t n = (entries + fat::kCheckEntries - 1) / fat::kCheckEntries;
  return (int)std::min<int64_t>(std::max<int64_t>(n, 1), FAT_CHECK_MAX_GROUPS);
}

bool check_args_ok(const fat_check_args* a, const char* who) {
  const bool shared = a && a->kind == FAT_CHECK_SHARED;
  const bool cu = a && (a->kind == FAT_CHECK_VARLEN || a->kind == FAT_CHECK_PAGED || shared);
  const bool range = a && a->kind == FAT_CHECK_RANGE;
  const bool copy = a && a->kind == FAT_CHECK_COPY, fork = a && a->kind == FAT_CHECK_FORK;
  const bool lens = a && a->kind != FAT_CHECK_VARLEN && !range && !copy;
  const bool ids = copy || fork || shared || (a && a->kind == FAT_CHECK_FREE && a->count > 0);
  if (!a || !a->host || (ids && !a->ids[0]) || ((copy || fork) && !a->ids[1]) ||
      (fork && !a->ids[2]) || (cu && !a->cu_q) || (a->kind == FAT_CHECK_VARLEN && !a->cu_k) || (lens && !a->seq_lens) ||
      (lens && !a->page_table) || (range && !a->values)) {
    fat_host::set_error("%s: a required pointer is NULL", who);
    return false;
  }
  if (a->kind < FAT_CHECK_CACHE || a->kind > FAT_CHECK_SHARED || (!range && !copy && a->batch <= 0) ||
      a->ticket <= 0 || (range && a->count <= 0) || (a->kind == FAT_CHECK_FREE && a->count < 0) ||
      (shared && (a->count <= 0 || a->count > INT_MAX || a->tokens <= 0)) ||
      ((copy || fork) && (a->count <= 0 || a->count > INT_MAX || a->num_pages <= 0)) ||
      (lens && (a->max_pages <= 0 || a->page_size <= 0 || a->page_table_stride < 0)) ||
      (a->kind == FAT_CHECK_CACHE && a->page_table_stride < a->max_pages)) {
    fat_host::set_error("%s: kind %d, batch %d, ticket %lld, max_pages %d, page_size %d or page_table_stride %lld "
                        "invalid", who, a->kind, a->batch, (long long)a->ticket, a->max_pages, a->page_size,
                        (long long)a->page_table_stride);
    return false;
  }
  return true;
}

}  // namespace

extern "C" int fat_check_begin(const fat_check_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!check_args_ok(a, "fat_check_begin")) return FAT_E_INVALID;
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
  const hipError_t e = hipStreamIsCapturing(stream, &cap);
  if (e != hipSuccess || cap != hipStreamCaptureStatusNone) {
    if (e != hipSuccess) (void)hipGetLastError();
    fat_host::set_error("fat_check_begin: the stream is capturing: a validated call waits for the GPU (use the "
                        "launch functions below the validation under capture)");
    return FAT_E_LAUNCH;
  }
  const fat::CheckParams prm{a->cu_q, a->cu_k, a->seq_lens, a->page_table, a->page_table_stride, a->host,
                             a->ticket, a->batch, a->max_pages, a->page_size, a->values, a->count,
                             {a->ids[0], a->ids[1], a->ids[2]}, a->num_pages, a->tokens, a->held};
  const dim3 grid((unsigned)check_groups(a)), block(fat::kCheckThreads);
  switch (a->kind) {
    case FAT_CHECK_CACHE: hipLaunchKernelGGL((fat::check_kernel<FAT_CHECK_CACHE>), grid, block, 0, stream, prm); break;
    case FAT_CHECK_VARLEN: hipLaunchKernelGGL((fat::check_kernel<FAT_CHECK_VARLEN>), grid, block, 0, stream, prm); break;
    case FAT_CHECK_PAGED: hipLaunchKernelGGL((fat::check_kernel<FAT_CHECK_PAGED>), grid, block, 0, stream, prm); break;
    case FAT_CHECK_RANGE: hipLaunchKernelGGL((fat::check_kernel<FAT_CHECK_RANGE>), grid, block, 0, stream, prm); break;
    case FAT_CHECK_FREE:
      hipLaunchKernelGGL((fat::check_rows_kernel<FAT_CHECK_FREE>), grid, dim3(fat::kRowsThreads), 0, stream, prm);
      break;
    case FAT_CHECK_SHARED:
      hipLaunchKernelGGL((fat::check_rows_kernel<FAT_CHECK_SHARED>), grid, dim3(fat::kRowsThreads), 0, stream, prm);
      break;
    case FAT_CHECK_COPY:
      hipLaunchKernelGGL((fat::check_lists_kernel<FAT_CHECK_COPY>), grid, dim3(fat::kListThreads), 0, stream, prm);
      break;
    case FAT_CHECK_FORK:
      hipLaunchKernelGGL((fat::check_lists_kernel<FAT_CHECK_FORK>), grid, dim3(fat::kListThreads), 0, stream, prm);
      break;
    default: hipLaunchKernelGGL((fat::check_kernel<FAT_CHECK_APPEND>), grid, block, 0, stream, prm); break;
  }
  return fat_host::launch_status("check_kernel");
}

extern "C" int fat_check_wait(const fat_check_args* a, void* stream_ptr, int64_t* result) {
  fat_host::clear_error();
  if (!check_args_ok(a, "fat_check_wait")) return FAT_E_INVALID;
  if (!result) {
    fat_host::set_error("fat_check_wait: result is NULL");
    return FAT_E_INVALID;
  }
  const int n = check_groups(a);
  // Tickets arrive in any order; `done` are known to be here.
  int done = 0;
  auto arrived = [&] {
    while (done < n && __atomic_load_n(a->host + FAT_CHECK_RESULTS + 2 * done + 1, __ATOMIC_ACQUIRE) == a->ticket)
      ++done;
    return done == n;
  };
  const auto limit = std::chrono::steady_clock::now() + std::chrono::milliseconds(2);
  bool here = arrived();
  for (int spin = 1; !here; ++spin) {
    __builtin_ia32_pause();
    here = arrived();
    if (!here && (spin & 255) == 0 && std::chrono::steady_clock::now() > limit) break;
  }
  if (!here) {
    const hipError_t e = hipStreamSynchronize(static_cast<hipStream_t>(stream_ptr));
    if (e != hipSuccess) {
      (void)hipGetLastError();
      fat_host::set_error("fat_check_wait: the stream failed: %s", hipGetErrorString(e));
      return FAT_E_LAUNCH;
    }
    if (!arrived()) {
      fat_host::set_error("fat_check_wait: no result for ticket %lld (was it begun on this stream?)",
                          (long long)a->ticket);
      return FAT_E_INVALID;
    }
  }
  for (int i = 0; i < 12; ++i) result[i] = a->host[i];
  int32_t lo = INT_MAX, hi = INT_MIN;
  for (int i = 0; i < n; ++i) {
    const uint64_t w = (uint64_t)a->host[FAT_CHECK_RESULTS + 2 * i];
    lo = std::min(lo, (int32_t)(uint32_t)w);
    hi = std::max(hi, (int32_t)(uint32_t)(w >> 32));
  }
  if (a->kind == FAT_CHECK_RANGE) {
    const bool nan = lo == INT_MIN && hi == INT_MAX;
    lo = nan ? 0x7fc00000 : lo ^ ((lo >> 31) & 0x7fffffff);
    hi = nan ? 0x7fc00000 : hi ^ ((hi >> 31) & 0x7fffffff);
  }
  if (a->kind == FAT_CHECK_SHARED && lo == INT_MIN) {
    result[7] |= 8;
    lo = 0;
  }
  if (a->kind == FAT_CHECK_FORK && lo == INT_MIN) result[7] |= 512;
  result[12] = lo;
  result[13] = hi;
  result[14] = result[15] = 0;
  return FAT_OK;
}

extern "C" int fat_cache_stats(const fat_cache_stats_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || !a->seq_lens || !a->out || (a->batch > 0 && a->max_pages > 0 && !a->page_table)) {
    fat_host::set_error("fat_cache_stats: a required pointer is NULL");
    return FAT_E_INVALID;
  }
  if (a->batch < 0 || a->max_pages < 0 || a->page_size <= 0 || (a->max_pages > 0 && a->page_table_stride < a->max_pages)) {
    fat_host::set_error("fat_cache_stats: batch %d, max_pages %d, page_size %d or page_table_stride %lld invalid",
                        a->batch, a->max_pages, a->page_size, (long long)a->page_table_stride);
    return FAT_E_INVALID;
  }
  hipLaunchKernelGGL(fat::cache_stats_kernel, dim3(1), dim3(fat::kStatsThreads), 0,
                     static_cast<hipStream_t>(stream_ptr), a->seq_lens, a->page_table, a->batch, a->max_pages,
                     a->page_table_stride, a->page_size, a->out);
  return fat_host::launch_status("cache_stats_kernel");
}
