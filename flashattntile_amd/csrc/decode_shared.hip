// decode_shared.hip -- decode of sequences that share a prefix: the keys that a
// group shares are read once for the queries of all of its sequences.
//
// A group's sequences hold the same first N keys.  With the rows r = (sequence,
// token, query head) of one KV head and
//   m = max_j s_rj,  l = sum_j 2^(s_rj - m),  acc = sum_j 2^(s_rj - m) v_j
// over any set of keys (s in log2 units), two disjoint sets join to M = max(m,
// m'), l 2^(m - M) + l' 2^(m' - M) and likewise acc; the output is acc / l.  So
// the launch computes (m, l, acc) of
//   prefix items  up to 32 RB rows of a group x a chunk of its N shared keys,
//                 read through the table row of the group's first sequence;
//   own items     the rows of one sequence x a chunk of the keys behind N, read
//                 through its own table row;
// and a second kernel joins them, a row's partials in the order of its keys.
// On 8-bit caches N is the prefix's whole pages: the page that it ends in has one
// scale for the shared keys and those behind them, so every sequence has other
// codes of them there.
//
// What bounds it: own items stream K and V once (HBM: 128 sequences x 630 bf16
// keys, 8 KV heads, D 128 take 63 us, 5.2 TB/s); a prefix item does 4 x 32 RB x D
// FLOPs per key, so long prefixes under many sequences are bound by the two products
// and the softmax between them, which wait for each other (128 sequences x 32
// heads x 32768 keys: 104 us in fp16, 0.66 PFLOP/s; 132 with bf16 queries, whose P
// has two parts, on fp8; without a single load 94).
//
// Both kinds run the same tile: 32 keys x 32 rows per wave on
// v_mfma_f32_32x32x16, S^T = K Q^T with K as the A operand (its rows staged in
// LDS) and O^T += V^T P^T with P^T straight from S^T's registers and V^T by
// transposed LDS reads.  RB = 4: a workgroup's four waves are four blocks of 32 rows
// and share every tile.  RB = 1: they have the same 32 rows, take tiles in turn (KG =
// 4 key groups) and join at the end.
#include <algorithm>

#include "decode_params.h"

namespace fat {

struct SharedParams {
  const uint8_t* q;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* pt;
  const int32_t* lens;
  const int32_t* cu;      // [G + 1]
  const int32_t* prefix;  // [G]
  uint8_t* out;
  float* ws_acc;  // [B * T * H, S, D]
  float* ws_ml;   // [B * T * H, S, 2]
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh;
  int64_t k_sh, v_sh;               // bytes
  uint32_t k_sp, k_ss, v_sp, v_ss;  // bytes; a page is below 4 GiB
  int64_t sc_sh;
  uint32_t sc_sp;
  int64_t pt_sb;
  int32_t B, G, T, H, Hkv, group;
  int32_t P, num_pages, max_pages;
  uint32_t invP;  // floor(2^32 / P), 2^32 - 1 for P = 1: floor(t / P) is the high product of t, or one more
  // Columns and slots that a key group's next tile lies behind its last one
  // (32 KG tokens), for prefix items and own items.
  uint32_t step_col[2], step_slot[2];
  float scale_log2;  // > 0 (or NaN)
  // Applied to every Q dword as it is loaded, (q & q_and) ^ q_xor: a negative
  // softmax scale runs as its absolute value with Q's signs flipped (exact), a
  // zero one with Q zeroed.  Identity: ~0u, 0.
  uint32_t q_and, q_xor;
  int32_t tiles;                     // row tiles of the largest group
  int32_t prefix_split, prefix_chunk;  // partials and keys of each
  int32_t split, chunk;
  int32_t prefix_blocks;  // workgroups of prefix items, before those of own items
  int32_t own_tiles;      // row tiles of a sequence
};

constexpr int kSharedWaves = 4;
// m moves only when a tile's maximum exceeds it by more than this (log2 units):
// p stays below 2^8, exact in the fp32 sums, and most tiles rescale nothing.
constexpr float kSharedLazy = 8.0f;

// The group of sequence b: the largest g with cu[g] <= b (-1: none).
__device__ __forceinline__ int group_of(const int32_t* cu, int G, int b) {
  int lo = -1, hi = G;  // cu[lo] <= b < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// (Not as inline asm: it would read the MFMA's results without the wait states
// that the compiler puts in front of an instruction it knows.)
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// 16 int8 or e4m3 codes as their exact values in QT (8 packed pairs).
template <typename QT, int KV>
__device__ __forceinline__ void codes_exact(const u32x4& raw, u32 (&o)[8]) {
  if constexpr (std::is_same<QT, F16>::value) {
    k8_exact_f16<KV>(raw, o);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (KV == KV_FP8) {
        o[2 * j] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[j], 1.0f, false));
        o[2 * j + 1] = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[j], 1.0f, true));
      } else {
        float f[4];
        i8x4_biased(raw[j], f);
        o[2 * j] = Pair<QT>::pack(f[0] - 128.0f, f[1] - 128.0f);
        o[2 * j + 1] = Pair<QT>::pack(f[2] - 128.0f, f[3] - 128.0f);
      }
    }
  }
}

template <typename QT, int KV, int D, int RB>
struct SharedTile {
  static_assert(RB == 1 || RB == kSharedWaves, "one row block, or one per wave");
  static constexpr int KG = kSharedWaves / RB;  // key groups
  static constexpr int kBufs = RB == 1 ? 1 : 2;  // LDS tiles per key group
  static constexpr int KS = D / 16;              // MFMA k-steps
  static constexpr int DB = D / 32;              // 32-dim blocks of O^T
  static constexpr int K_RS = D + 8;             // LDS row strides (elements), spreading reads over the banks
  static constexpr int V_RS = D + 32;
  static constexpr int EB = KV == KV_SAME ? 2 : 1;
  static constexpr int EPC = 16 / EB;            // elements per 16-byte chunk
  static constexpr int CPR = D / EPC;            // chunks per row
  static constexpr int NT = 64 * RB;             // lanes that stage a tile
  static constexpr int NCH = 32 * CPR;           // its chunks
  static constexpr int NLD = NCH > NT ? NCH / NT : 1;  // per lane
  static constexpr int OS = D + 4;               // row stride (floats) of the key groups' join
  static constexpr int kTile = 32 * (K_RS + V_RS);  // elements
  // 8-bit caches: the codes are staged as they are, exact in fp16 and bf16.
  // k_scale multiplies the fp32 scores and v_scale P, whose product with the codes
  // of V then runs in bf16 for fp16 queries too: its exponents hold any scale,
  // where in fp16 the P of a page with a small scale would lose its bits beside one
  // with a large scale, and V times its scale would be rounded once more.
  static constexpr bool FOLD = KV != KV_SAME;
  using VT = typename std::conditional<FOLD, BF16, QT>::type;  // of the second product
  static constexpr int kScaleFloats = FOLD ? 64 : 0;  // of a tile's keys: K's, V's
  static constexpr int kTileBytes = KG * kBufs * (kTile * 2 + kScaleFloats * 4);
  static constexpr int kJoinBytes = KG > 1 ? (kSharedWaves * 32 * OS + kSharedWaves * 32 * 2) * 4 : 0;
  static constexpr int kBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
};

// Rows [row0, row0 + 32 RB) of the R = n_seq T group rows of sequences b0 .. and
// KV head kvh, against keys [t_begin, t_end) of table row `ptrow`; partials to
// slot `slot` of S.
template <typename QT, int KV, int D, int RB>
__device__ __forceinline__ void shared_segment(const SharedParams& p, uint8_t* smem, int b0, int n_seq, int kvh, int row0,
                                               const int32_t* ptrow, int t_begin, int t_end, int slot, int S) {
  using Tl = SharedTile<QT, KV, D, RB>;
  constexpr int KG = Tl::KG, KS = Tl::KS, DB = Tl::DB, K_RS = Tl::K_RS, V_RS = Tl::V_RS, EPC = Tl::EPC, CPR = Tl::CPR,
                NT = Tl::NT, NCH = Tl::NCH, NLD = Tl::NLD, OS = Tl::OS;
  constexpr bool FOLD = Tl::FOLD;
  using VT = typename Tl::VT;
  // P enters the second product as bf16 hi + lo parts: one bf16 alone (2^-9) would
  // show beside the output's own rounding where a row sees few keys.  fp16 P is one
  // part: its half step, 2^-11, is the output's own (relative error 2.6e-4 to 2.9e-4,
  // with P in 32 bits 2.1e-4), and a second part would double the second product.
  constexpr bool SPLIT_P = std::is_same<VT, BF16>::value;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, kg = w / RB;
  const int li = lane & 31;  // key row (A operand) / row column (B, S^T)
  const int g = lane >> 5;   // k-group: head dims 16 ks + 8 g .. + 7 of k-step ks
  const int per_seq = p.T * p.group;
  const int R = n_seq * per_seq;
  const int n_tiles = t_end > t_begin ? (t_end - t_begin + 31) >> 5 : 0;

  auto row_of = [&](int r) {  // global row of row r of the item
    const int s = r / per_seq;
    const int in = r - s * per_seq;
    const int t = in / p.group;
    return ((int64_t)(b0 + s) * p.T + t) * p.H + kvh * p.group + (in - t * p.group);
  };
  if (n_tiles == 0) {  // uniform: partials of weight 0, whose acc the join leaves alone
    for (int r = row0 + threadIdx.x; r < min(row0 + 32 * RB, R); r += kSharedWaves * 64) {
      const int64_t at = row_of(r) * S + slot;
      p.ws_ml[2 * at] = -INFINITY;
      p.ws_ml[2 * at + 1] = 0.f;
    }
    return;
  }

  // This lane's row, and the end of its visible keys: token t of a sequence of
  // len keys sees those before len - T + 1 + t.
  const int my_row = min(row0 + 32 * rb + li, R - 1);
  const int seq = my_row / per_seq;
  const int in_seq = my_row - seq * per_seq;
  const int my_t = in_seq / p.group;
  const int my_h = kvh * p.group + (in_seq - my_t * p.group);
  const int my_b = b0 + seq;
  const int my_end = min(t_end, min(p.lens[my_b], p.max_pages * p.P) - p.T + 1 + my_t);
  // Tiles that end before all of the wave's rows do need no mask.
  int all_end = my_end;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) all_end = min(all_end, __shfl_xor(all_end, off));
  all_end = __builtin_amdgcn_readfirstlane(all_end);

  u32x4 qf[KS];
  {
    const uint8_t* qp = p.q + 2 * ((int64_t)my_b * p.q_sb + (int64_t)my_t * p.q_st + (int64_t)my_h * p.q_sh + 8 * g);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = (*reinterpret_cast<const u32x4*>(qp + 32 * ks) & p.q_and) ^ p.q_xor;
  }

  // Staging: chunk i NT + st of a tile is this lane's, st its place in the key group.
  // (Where a tile has fewer chunks than lanes, the others load what lane st loads.)
  const int st = (rb * 64 + lane) % NCH;
  const bool stages = NCH >= NT || rb * 64 + lane < NCH;
  const int srow = st / CPR;  // row of chunk 0; chunk i's is srow + i NT / CPR
  const int scol = st % CPR;
  const uint8_t* const kh = p.k + (int64_t)kvh * p.k_sh + 16 * scol;
  const uint8_t* const vh = p.v + (int64_t)kvh * p.v_sh + 16 * scol;
  const float* const ksh = KV != KV_SAME ? p.ks + (int64_t)kvh * p.sc_sh : nullptr;
  const float* const vsh = KV != KV_SAME ? p.vs + (int64_t)kvh * p.sc_sh : nullptr;
  struct Raw {
    u32x4 k[NLD], v[NLD];
    float ksc[NLD], vsc[NLD];
  };
  // Page ids of this lane's rows of the tile that the next fetch loads, and their
  // slots; col: their table columns.  Rows behind the end look up its last key
  // (a row that the sequence uses); ids are clamped, so every address lies in the
  // pool.  Tokens, columns and slots move on by additions: a division per row
  // and tile took as long as a quarter of the softmax.
  int pid[NLD];
  uint32_t slot_of[NLD], col[NLD], in_page[NLD];
  const uint32_t P = p.P;
  auto place = [&](uint32_t tok, uint32_t& c, uint32_t& s) __attribute__((always_inline)) {
    c = __umulhi(tok, p.invP);
    s = tok - c * P;
    if (s >= P) {
      s -= P;
      ++c;
    }
  };
  uint32_t last_col, last_slot;
  place((uint32_t)t_end - 1, last_col, last_slot);
  last_col = __builtin_amdgcn_readfirstlane(last_col);
  last_slot = __builtin_amdgcn_readfirstlane(last_slot);
#pragma unroll
  for (int i = 0; i < NLD; ++i) place((uint32_t)(t_begin + 32 * kg + srow + i * (NT / CPR)), col[i], in_page[i]);
  const uint32_t step_col = p.step_col[RB == 1], step_slot = p.step_slot[RB == 1];
  auto lookup = [&](int t) __attribute__((always_inline)) {
    const bool tail = t_begin + 32 * t + 32 > t_end;  // uniform
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      uint32_t c = col[i];
      slot_of[i] = in_page[i];
      if (tail) {
        asm volatile("");  // a branch that is seldom taken, and not selects in every tile
        const bool in = t_begin + 32 * t + srow + i * (NT / CPR) < t_end;
        c = in ? c : last_col;
        slot_of[i] = in ? slot_of[i] : last_slot;
      }
      pid[i] = ptrow[c];
      col[i] += step_col;
      in_page[i] += step_slot;
      if (in_page[i] >= P) {
        in_page[i] -= P;
        ++col[i];
      }
    }
  };
  // The tile that fetch_k loads next becomes the one whose ids are here, the one it
  // loaded last that of fetch_v; tile t's ids are asked for.  They go out ahead
  // of the rows that a caller then loads: loads return in order, so waiting for
  // them leaves those rows in flight.
  uint32_t k_page[NLD], k_slot[NLD], v_page[NLD], v_slot[NLD];
  auto advance = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      v_page[i] = k_page[i];
      v_slot[i] = k_slot[i];
      k_page[i] = (uint32_t)min(max(pid[i], 0), p.num_pages - 1);
      k_slot[i] = slot_of[i];
    }
    lookup(t);
  };
  auto fetch_k = [&](Raw& R) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      R.k[i] = *reinterpret_cast<const u32x4*>(kh + (uint64_t)k_page[i] * p.k_sp + (uint32_t)__umul24(k_slot[i], p.k_ss));
      if constexpr (FOLD) R.ksc[i] = ksh[(uint64_t)k_page[i] * p.sc_sp];
    }
  };
  auto fetch_v = [&](Raw& R, const uint32_t* page, const uint32_t* slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      R.v[i] = *reinterpret_cast<const u32x4*>(vh + (uint64_t)page[i] * p.v_sp + (uint32_t)__umul24(slot[i], p.v_ss));
      if constexpr (FOLD) R.vsc[i] = vsh[(uint64_t)page[i] * p.sc_sp];
    }
  };
  // A chunk as ET elements: a copy, or the exact values of 8-bit codes.
  auto put = [&](auto et, uint16_t* dst, const u32x4& raw) __attribute__((always_inline)) {
    if constexpr (KV == KV_SAME) {
      *reinterpret_cast<u32x4*>(dst) = raw;
    } else {
      u32 o[8];
      codes_exact<decltype(et), KV>(raw, o);
      *reinterpret_cast<u32x4*>(dst) = u32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<u32x4*>(dst + 8) = u32x4{o[4], o[5], o[6], o[7]};
    }
  };
  uint16_t* const tile0 = reinterpret_cast<uint16_t*>(smem) + kg * Tl::kBufs * Tl::kTile;
  float* const sc0 = reinterpret_cast<float*>(smem + KG * Tl::kBufs * Tl::kTile * 2) + kg * Tl::kBufs * Tl::kScaleFloats;
  auto store_k = [&](const Raw& R, int buf) __attribute__((always_inline)) {
    if (!stages) return;
    uint16_t* const Kt = tile0 + buf * Tl::kTile;
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int row = srow + i * (NT / CPR);
      put(QT{}, &Kt[row * K_RS + scol * EPC], R.k[i]);
      if constexpr (FOLD) {
        if (scol == 0) sc0[buf * Tl::kScaleFloats + row] = R.ksc[i] * p.scale_log2;
      }
    }
  };
  auto store_v = [&](const Raw& R, int t, int buf) __attribute__((always_inline)) {
    if (!stages) return;
    const bool last = t_begin + 32 * t + 32 > t_end;  // uniform
    uint16_t* const Vt = tile0 + buf * Tl::kTile + 32 * K_RS;
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int row = srow + i * (NT / CPR);
      u32x4 vv = R.v[i];
      if constexpr (FOLD) {
        // behind the end: a scale of 0, which the codes' finite values keep at 0
        const float sc = !last || t_begin + 32 * t + row < t_end ? R.vsc[i] : 0.f;
        put(VT{}, &Vt[row * V_RS + scol * EPC], vv);
        if (scol == 0) sc0[buf * Tl::kScaleFloats + 32 + row] = sc;
      } else {
        if (last) {
          asm volatile("");  // a branch
          // behind the end: zeros; the scores there are masked, and 0 * v stays 0
          // whatever the last key's v holds
          const bool in = t_begin + 32 * t + row < t_end;
          vv = u32x4{in ? vv[0] : 0u, in ? vv[1] : 0u, in ? vv[2] : 0u, in ? vv[3] : 0u};
        }
        put(VT{}, &Vt[row * V_RS + scol * EPC], vv);
      }
    }
  };

  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
  float m_run = -INFINITY;  // log2 units
  float l_run = 0.f;
  const int tr_c = (lane & 15) >> 2, tr_j = lane & 3, tr_G = lane >> 4;
  const int tr_row = 4 * (tr_G >> 1) + tr_c;
  const int tr_col = 16 * (tr_G & 1) + 4 * tr_j;

  // S^T of the keys in K buffer `buf` (in log2 units for 8-bit caches, whose
  // scales it applies): row li over keys (r & 3) + 4 g + 8 (r >> 2).
  auto qk = [&](f32x16& s, int buf) __attribute__((always_inline)) {
    const uint16_t* const Kt = tile0 + buf * Tl::kTile;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(&Kt[li * K_RS + 16 * ks + 8 * g]);
      s = Mfma<QT>::mma(a, qf[ks], s);
    }
  };
  auto scale_s = [&](f32x16& s, int buf) __attribute__((always_inline)) {
    if constexpr (FOLD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 ck = *reinterpret_cast<const f32x4*>(&sc0[buf * Tl::kScaleFloats + 4 * g + 8 * j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * j + e] *= ck[e];
      }
    }
  };
  const float c = FOLD ? 1.f : p.scale_log2;
  auto mask = [&](f32x16& s, int t) __attribute__((always_inline)) {
    const int kb = t_begin + 32 * t;
    if (kb + 32 > all_end) {  // uniform
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = kb + (r & 3) + 4 * g + 8 * (r >> 2) < my_end ? s[r] : -INFINITY;
    }
  };
  // Moves the running maximum to one of mx, a lane's largest score.
  auto raise = [&](float mx) __attribute__((always_inline)) {
    mx = xor32<OpMax>(mx) * c;
    if (__any(mx > m_run + kSharedLazy)) {
      const bool grow = mx > m_run + kSharedLazy;
      const float alpha = grow ? fast_exp2(m_run - mx) : 1.f;
      m_run = grow ? mx : m_run;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
    }
  };
  auto largest = [&](const f32x16& s) __attribute__((always_inline)) {
    float mx = max3(s[0], s[1], s[2]);
#pragma unroll
    for (int r = 3; r < 15; r += 2) mx = max3(mx, s[r], s[r + 1]);
    return fmaxf(mx, s[15]);
  };
  u32x4 pf[2], pl[2];
  // Scores 2 j and 2 j + 1 as P = 2^(s - m), times v_scale where V is staged as
  // codes.  m_use: a row that has seen no key yet keeps m = -inf; its scores are
  // -inf too, and 2^(-inf - 0) = 0.
  float m_use = 0.f;
  f32x4 cv[4];
  auto load_cv = [&](int buf) __attribute__((always_inline)) {
    m_use = m_run == -INFINITY ? 0.f : m_run;
    if constexpr (FOLD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) cv[j] = *reinterpret_cast<const f32x4*>(&sc0[buf * Tl::kScaleFloats + 32 + 4 * g + 8 * j]);
    }
  };
  auto piece = [&](const f32x16& s, int j) __attribute__((always_inline)) {
    float x0 = fast_exp2(FOLD ? s[2 * j] - m_use : __builtin_fmaf(s[2 * j], c, -m_use));
    float x1 = fast_exp2(FOLD ? s[2 * j + 1] - m_use : __builtin_fmaf(s[2 * j + 1], c, -m_use));
    l_run += x0 + x1;
    if constexpr (FOLD) {
      x0 *= cv[j >> 1][2 * (j & 1)];
      x1 *= cv[j >> 1][2 * (j & 1) + 1];
    }
    const u32 hp = Pair<VT>::pack(x0, x1);
    pf[j >> 2][j & 3] = hp;
    if constexpr (SPLIT_P) pl[j >> 2][j & 3] = Pair<VT>::pack(x0 - Pair<VT>::lo(hp), x1 - Pair<VT>::hi(hp));
  };
  // O^T += V^T P^T: entry e is keys 16 u .. + 15 of the tile (u = e / DB), dims 32 db ..
  // + 31 (db = e % DB).
  auto read_v = [&](int buf, int e) __attribute__((always_inline)) {
    const uint16_t* vp = tile0 + buf * Tl::kTile + 32 * K_RS + (16 * (e / DB) + tr_row) * V_RS + 32 * (e % DB) + tr_col;
    const u32x2 lo = lds_read_tr16(vp);
    const u32x2 hi = lds_read_tr16(vp + 8 * V_RS);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
  };
  auto pv = [&](const u32x4& a, int e) __attribute__((always_inline)) {
    acc[e % DB] = Mfma<VT>::mma(a, pf[e / DB], acc[e % DB]);
    if constexpr (SPLIT_P) acc[e % DB] = Mfma<VT>::mma(a, pl[e / DB], acc[e % DB]);
  };

  if constexpr (RB == 1) {
    // Each wave has its own tiles: no workgroup barrier.
    Raw R;
    f32x16 s;
    if (kg < n_tiles) {
      lookup(kg);
      advance(kg + KG);
      fetch_k(R);
      fetch_v(R, k_page, k_slot);
    }
    for (int t = kg; t < n_tiles; t += KG) {
      store_k(R, 0);
      store_v(R, t, 0);
      if (t + KG < n_tiles) {
        advance(t + 2 * KG);
        fetch_k(R);
        fetch_v(R, k_page, k_slot);
      }
      wave_lds_fence();
      qk(s, 0);
      scale_s(s, 0);
      mask(s, t);
      raise(largest(s));
      load_cv(0);
#pragma unroll
      for (int j = 0; j < 8; ++j) piece(s, j);
#pragma unroll
      for (int e = 0; e < 2 * DB; ++e) pv(read_v(0, e), e);
      wave_lds_fence();
    }
  } else {
    // Round i: S = K Q^T of tile i + 1 beside the exponentials of tile i, then O += V P
    // of tile i beside the maximum of tile i + 1.  K(i + 1) and V(i) lie in LDS, K(i +
    // 2) and V(i + 1) in registers (loaded a round ago, stored at this one's end),
    // and K(i + 3) and V(i + 2) are loaded.  One barrier a round: behind it every wave is
    // done with round i - 1, whose buffers the round's stores take.  Tiles behind the
    // end stage the last key, and their scores are masked.
    Raw Ra, Rb;
    f32x16 sa, sb;
    lookup(0);
    advance(1);
    fetch_k(Ra);
    fetch_v(Ra, k_page, k_slot);
    advance(2);
    fetch_k(Rb);
    fetch_v(Rb, k_page, k_slot);
    advance(3);
    store_k(Ra, 0);
    store_v(Ra, 0, 0);
    store_k(Rb, 1);
    fetch_k(Rb);
    __syncthreads();
    qk(sa, 0);
    scale_s(sa, 0);
    mask(sa, 0);
    raise(largest(sa));
    auto round = [&](int i, f32x16& s, f32x16& s2, const Raw& X, Raw& Y) __attribute__((always_inline)) {
      const int now = i & 1, next = now ^ 1;
      advance(i + 4);
      fetch_v(Y, v_page, v_slot);
      fetch_k(Y);
      __syncthreads();
      load_cv(now);
      // A part of the softmax in the shadow of each MFMA; LDS reads run LOOK entries
      // ahead of theirs.  sched_barrier keeps the steps apart: left to itself the
      // compiler lines the MFMAs up behind the exponentials.
      constexpr int LOOK = 3;
      const uint16_t* const Kn = tile0 + next * Tl::kTile + li * K_RS + 8 * g;
      u32x4 ka[KS], va[2 * DB];
#pragma unroll
      for (int r = 0; r < 16; ++r) s2[r] = 0.f;
#pragma unroll
      for (int k = 0; k < LOOK; ++k) ka[k] = *reinterpret_cast<const u32x4*>(Kn + 16 * k);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        s2 = Mfma<QT>::mma(ka[k], qf[k], s2);
        if (k + LOOK < KS) ka[k + LOOK] = *reinterpret_cast<const u32x4*>(Kn + 16 * (k + LOOK));
        else va[k + LOOK - KS] = read_v(now, k + LOOK - KS);
#pragma unroll
        for (int j = 8 * k / KS; j < 8 * (k + 1) / KS; ++j) piece(s, j);
        __builtin_amdgcn_sched_barrier(0);
      }
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 2 * DB; ++e) {
        pv(va[e], e);
        if (e + LOOK < 2 * DB) va[e + LOOK] = read_v(now, e + LOOK);
        if (e == DB / 2 - 1) {
          scale_s(s2, next);
          mask(s2, i + 1);
        }
        if (e == DB) mx = largest(s2);
        __builtin_amdgcn_sched_barrier(0);
      }
      raise(mx);
      store_k(X, now);
      store_v(X, i + 1, next);
    };
    for (int i = 0; i < n_tiles; i += 2) {
      round(i, sa, sb, Rb, Ra);
      if (i + 1 < n_tiles) round(i + 1, sb, sa, Ra, Rb);  // uniform
    }
  }

  const float l_tot = xor32<OpAdd>(l_run);
  if constexpr (KG == 1) {
    if (row0 + 32 * rb + li < R) {
      const int64_t at = row_of(row0 + 32 * rb + li) * S + slot;
      float* o = p.ws_acc + at * D + 4 * g;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4*>(o + 32 * db + 8 * r4) =
              f32x4{acc[db][4 * r4], acc[db][4 * r4 + 1], acc[db][4 * r4 + 2], acc[db][4 * r4 + 3]};
      if (g == 0) {
        p.ws_ml[2 * at] = m_run;
        p.ws_ml[2 * at + 1] = l_tot;
      }
    }
  } else {
    // Join the key groups: sum over kg of acc 2^(m - M).
    __syncthreads();  // every wave is done with its tiles
    float* so = reinterpret_cast<float*>(smem);       // [waves][32][OS]
    float* sml = so + kSharedWaves * 32 * OS;         // [waves][32][2]
    const int nvalid = min(32, R - row0);
    if (li < nvalid) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4*>(&so[(w * 32 + li) * OS + 32 * db + 4 * g + 8 * r4]) =
              f32x4{acc[db][4 * r4], acc[db][4 * r4 + 1], acc[db][4 * r4 + 2], acc[db][4 * r4 + 3]};
    }
    if (g == 0) {
      sml[(w * 32 + li) * 2] = m_run;
      sml[(w * 32 + li) * 2 + 1] = l_tot;
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < nvalid * (D / 4); idx += kSharedWaves * 64) {
      const int r = idx / (D / 4);
      const int d = 4 * (idx - r * (D / 4));
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; ++k) M = fmaxf(M, sml[(k * 32 + r) * 2]);
      f32x4 A = {0.f, 0.f, 0.f, 0.f};
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const int at = k * 32 + r;
        const float m = sml[at * 2];
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - M);  // a NaN in l or acc stays one
        A += *reinterpret_cast<const f32x4*>(&so[at * OS + d]) * f;
        L = __builtin_fmaf(sml[at * 2 + 1], f, L);
      }
      const int64_t at = row_of(row0 + r) * S + slot;
      *reinterpret_cast<f32x4*>(p.ws_acc + at * D + d) = A;
      if (d == 0) {
        p.ws_ml[2 * at] = M;
        p.ws_ml[2 * at + 1] = L;
      }
    }
  }
}

// The keys of a prefix of n that are read once for its group.
template <int KV>
__device__ __forceinline__ int shared_keys(const SharedParams& p, int n) {
  return KV == KV_SAME ? n : n - n % p.P;
}

template <typename QT, int KV, int D, int RB>
__global__ __launch_bounds__(kSharedWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void decode_shared_kernel(const SharedParams p) {
  constexpr int kBytes = SharedTile<QT, KV, D, RB>::kBytes > SharedTile<QT, KV, D, 1>::kBytes
                             ? SharedTile<QT, KV, D, RB>::kBytes
                             : SharedTile<QT, KV, D, 1>::kBytes;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBytes];
  const int S = p.prefix_split + p.split;
  const int cap = p.max_pages * p.P;  // all token places are below it: columns below max_pages
  if ((int)blockIdx.x < p.prefix_blocks) {
    // Row tiles of the same keys run 8 ids apart, on one XCD, and meet in its L2.
    const int step = 8 * p.tiles;
    const int k = blockIdx.x / step;
    const int rem = blockIdx.x - k * step;
    const int tile = rem >> 3;
    const int unit = k * 8 + (rem & 7);
    if (unit >= p.G * p.prefix_split * p.Hkv) return;
    const int gs = unit / p.Hkv;
    const int kvh = unit - gs * p.Hkv;
    const int grp = gs / p.prefix_split;
    const int slot = gs - grp * p.prefix_split;
    const int b0 = min(max(p.cu[grp], 0), p.B);
    const int b1 = min(max(p.cu[grp + 1], b0), p.B);
    const int row0 = tile * 32 * RB;
    if (row0 >= (b1 - b0) * p.T * p.group) return;
    const int n = shared_keys<KV>(p, min(max(p.prefix[grp], 0), cap));
    const int t_begin = min(slot * p.prefix_chunk, n);
    const int t_end = slot == p.prefix_split - 1 ? n : min(t_begin + p.prefix_chunk, n);
    shared_segment<QT, KV, D, RB>(p, smem, b0, b1 - b0, kvh, row0, p.pt + (int64_t)b0 * p.pt_sb, t_begin, t_end, slot, S);
    return;
  }
  const int id = blockIdx.x - p.prefix_blocks;
  // The slots of a sequence lie far apart: workgroups go to the XCDs and to their
  // shader engines in turn, and where many sequences have no keys in their second
  // half, slots side by side would leave every other engine idle (128 sequences of 100
  // to 2000 bf16 keys in four chunks: 111 us so, 77 apart).
  const int per_b = p.Hkv * p.own_tiles;
  const int slot = id / (p.B * per_b);
  const int r = id - slot * (p.B * per_b);
  const int b = r / per_b;
  const int y = r - b * per_b;
  const int kvh = y / p.own_tiles;
  const int tile = y - kvh * p.own_tiles;
  const int grp = group_of(p.cu, p.G, b);
  const int len = min(max(p.lens[b], 0), cap);
  const int n = grp < 0 ? 0 : min(shared_keys<KV>(p, min(max(p.prefix[grp], 0), cap)), len);
  const int t_begin = min((int64_t)n + (int64_t)slot * p.chunk, (int64_t)len);
  const int t_end = slot == p.split - 1 ? len : min((int64_t)t_begin + p.chunk, (int64_t)len);
  shared_segment<QT, KV, D, 1>(p, smem, b, 1, kvh, tile * 32, p.pt + (int64_t)b * p.pt_sb, t_begin, t_end,
                               p.prefix_split + slot, S);
}

// Joins a row's S partials, one wave per row: lane s has those of slots s and s +
// 64.  Slots of weight 0 (no keys) do not count.
constexpr int kJoinRows = 4;
template <typename QT, int D>
__global__ __launch_bounds__(64 * kJoinRows) void shared_join_kernel(const SharedParams p) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kJoinRows + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= (int64_t)p.B * p.T * p.H) return;
  const int S = p.prefix_split + p.split;
  float m[2], l[2], f[2];
  float M = -INFINITY;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = lane + 64 * j;
    m[j] = -INFINITY;
    l[j] = 0.f;
    if (s < S) {
      m[j] = p.ws_ml[2 * (row * S + s)];
      l[j] = p.ws_ml[2 * (row * S + s) + 1];
    }
    M = fmaxf(M, m[j]);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
  float L = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    f[j] = m[j] == -INFINITY ? 0.f : fast_exp2(m[j] - M);
    L += l[j] * f[j];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off);
  constexpr int E = D / 64;
  float a[E];
#pragma unroll
  for (int e = 0; e < E; ++e) a[e] = 0.f;
  const float* acc = p.ws_acc + row * S * D + E * lane;
  // Eight slots' loads in flight.  Those of weight 0 are left out: they may never have
  // been written, and few of a batch's sequences have keys in all of their slots.
  unsigned long long left[2] = {__ballot(f[0] != 0.f), __ballot(f[1] != 0.f)};
  while (left[0] | left[1]) {  // uniform
    float x[8][E], w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool low = left[0] != 0;
      const unsigned long long some = low ? left[0] : left[1];
      const int at = some ? __builtin_ctzll(some) : 0;
      // None left: slot 0 or 64 once more, with a weight of 0.
      w[i] = some ? __shfl(low ? f[0] : f[1], at) : 0.f;
      const int s = min(at + (low ? 0 : 64), S - 1);
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = acc[(int64_t)s * D + e];
      if (low) left[0] &= left[0] - 1;
      else left[1] &= left[1] - 1;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int e = 0; e < E; ++e) a[e] = __builtin_fmaf(w[i] != 0.f ? x[i][e] : 0.f, w[i], a[e]);
    }
  }
  const int64_t bt = row / p.H;
  const int h = (int)(row - bt * p.H);
  const int b = (int)(bt / p.T);
  const int t = (int)(bt - (int64_t)b * p.T);
  const int64_t o = (int64_t)b * p.o_sb + (int64_t)t * p.o_st + (int64_t)h * p.o_sh + E * lane;
#pragma unroll
  for (int e = 0; e < E; ++e) store_elem<QT>(p.out, o + e, L == 0.f ? 0.f : a[e] / L);
}

}  // namespace fat

// ===========================================================================
// Host side
// ===========================================================================
namespace {

template <typename QT, int KV, int D>
void launch_shared_d(const fat::SharedParams& prm, int rb, unsigned blocks, hipStream_t stream) {
  const dim3 block(64 * fat::kSharedWaves);
  switch (rb) {
    case 4: hipLaunchKernelGGL((fat::decode_shared_kernel<QT, KV, D, 4>), dim3(blocks), block, 0, stream, prm); break;
    default: hipLaunchKernelGGL((fat::decode_shared_kernel<QT, KV, D, 1>), dim3(blocks), block, 0, stream, prm); break;
  }
}

template <typename QT, int KV>
void launch_shared_kv(const fat::SharedParams& prm, int D, int rb, unsigned blocks, hipStream_t stream) {
  if (D == 128) launch_shared_d<QT, KV, 128>(prm, rb, blocks, stream);
  else launch_shared_d<QT, KV, 64>(prm, rb, blocks, stream);
}

template <typename QT>
void launch_shared(const fat::SharedParams& prm, int kv, int D, int rb, unsigned blocks, hipStream_t stream) {
  switch (kv) {
    case fat::KV_SAME: launch_shared_kv<QT, fat::KV_SAME>(prm, D, rb, blocks, stream); break;
    case fat::KV_I8: launch_shared_kv<QT, fat::KV_I8>(prm, D, rb, blocks, stream); break;
    default: launch_shared_kv<QT, fat::KV_FP8>(prm, D, rb, blocks, stream); break;
  }
}

template <typename QT>
void launch_join(const fat::SharedParams& prm, int D, hipStream_t stream) {
  const int64_t rows = (int64_t)prm.B * prm.T * prm.H;
  const dim3 grid((unsigned)((rows + fat::kJoinRows - 1) / fat::kJoinRows)), block(64 * fat::kJoinRows);
  if (D == 128) hipLaunchKernelGGL((fat::shared_join_kernel<QT, 128>), grid, block, 0, stream, prm);
  else hipLaunchKernelGGL((fat::shared_join_kernel<QT, 64>), grid, block, 0, stream, prm);
}

}  // namespace

extern "C" size_t fat_paged_decode_shared_workspace_bytes(int32_t rows, int32_t num_heads, int32_t head_dim,
                                                          int32_t splits) {
  if (rows <= 0 || num_heads <= 0 || head_dim <= 0 || splits <= 0) return 0;
  return (size_t)rows * num_heads * splits * (head_dim + 2) * sizeof(float);
}

extern "C" int fat_paged_decode_shared(const fat_shared_args* a, void* stream_ptr) {
  fat_host::clear_error();
  if (!a || !a->q || !a->k_cache || !a->v_cache || !a->page_table || !a->seq_lens || !a->cu_groups ||
      !a->prefix_lens || !a->out || !a->workspace) {
    fat_host::set_error("fat_paged_decode_shared: a required pointer is NULL");
    return FAT_E_INVALID;
  }
  if (a->batch <= 0 || a->groups <= 0 || a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_pages <= 0 ||
      a->max_pages <= 0 || a->page_size <= 0 || a->max_group <= 0) {
    fat_host::set_error("fat_paged_decode_shared: batch, groups, max_group, heads, page_size, num_pages and max_pages "
                        "must be positive");
    return FAT_E_INVALID;
  }
  if (a->num_heads % a->num_kv_heads != 0) {
    fat_host::set_error("fat_paged_decode_shared: num_heads %d must be divisible by num_kv_heads %d", a->num_heads,
                        a->num_kv_heads);
    return FAT_E_INVALID;
  }
  if ((int64_t)a->max_pages * a->page_size > 0x7fffffffLL - 4096) {
    fat_host::set_error("fat_paged_decode_shared: max_pages * page_size overflows int32 positions");
    return FAT_E_INVALID;
  }
  if (a->prefix_split < 1 || a->prefix_split > 64 || a->split < 1 || a->split > 64 || a->prefix_chunk < 32 ||
      a->chunk < 32 || a->prefix_chunk % 32 || a->chunk % 32 || a->q_len < 0 || a->q_len > 64) {
    fat_host::set_error("fat_paged_decode_shared: prefix_split %d and split %d must be in [1, 64], prefix_chunk %d and "
                        "chunk %d positive multiples of 32, q_len %d in [0, 64]", a->prefix_split, a->split,
                        a->prefix_chunk, a->chunk, a->q_len);
    return FAT_E_INVALID;
  }
  if (a->row_blocks != 0 && a->row_blocks != 1 && a->row_blocks != 4) {
    fat_host::set_error("fat_paged_decode_shared: row_blocks must be 0 (by the rows), 1 or 4, got %d", a->row_blocks);
    return FAT_E_INVALID;
  }
  if ((int64_t)a->prefix_split * a->prefix_chunk > 0x7fffffffLL || (int64_t)a->split * a->chunk > 0x7fffffffLL) {
    fat_host::set_error("fat_paged_decode_shared: splits times chunk overflow int32 positions");
    return FAT_E_INVALID;
  }
  int kv = -1;
  if (a->q_dtype == FAT_DTYPE_F16 || a->q_dtype == FAT_DTYPE_BF16) {
    if (a->kv_dtype == a->q_dtype) kv = fat::KV_SAME;
    else if (a->kv_dtype == FAT_DTYPE_I8) kv = fat::KV_I8;
    else if (a->kv_dtype == FAT_DTYPE_FP8E4M3) kv = fat::KV_FP8;
  }
  if (kv < 0 || (a->head_dim != 64 && a->head_dim != 128)) {
    fat_host::set_error("fat_paged_decode_shared: takes fp16/bf16 queries on a cache of their type, int8 or fp8e4m3, "
                        "head_dim 64 or 128");
    return FAT_E_UNSUPPORTED;
  }
  if (kv != fat::KV_SAME && (!a->k_scale || !a->v_scale)) {
    fat_host::set_error("fat_paged_decode_shared: int8/fp8 K/V need k_scale and v_scale");
    return FAT_E_INVALID;
  }
  const int T = a->q_len > 1 ? a->q_len : 1;
  const int eb = kv == fat::KV_SAME ? 2 : 1;
  // Rows of a KV head are numbered in 32 bits, 128 a tile.
  if ((int64_t)a->batch * T > (0x7fffffffLL - 128) / (a->num_heads / a->num_kv_heads)) {
    fat_host::set_error("fat_paged_decode_shared: batch %d x q_len %d x %d heads per KV head are too many query rows",
                        a->batch, T, a->num_heads / a->num_kv_heads);
    return FAT_E_UNSUPPORTED;
  }
  const uintptr_t align = (uintptr_t)a->q | (uintptr_t)(2 * a->q_stride_b) | (uintptr_t)(2 * a->q_stride_h) |
                          (uintptr_t)(T > 1 ? 2 * a->q_stride_t : 0) | (uintptr_t)a->workspace | (uintptr_t)a->k_cache |
                          (uintptr_t)a->v_cache | (uintptr_t)(eb * a->k_stride_page) |
                          (uintptr_t)(eb * a->k_stride_slot) | (uintptr_t)(eb * a->k_stride_head) |
                          (uintptr_t)(eb * a->v_stride_page) | (uintptr_t)(eb * a->v_stride_slot) |
                          (uintptr_t)(eb * a->v_stride_head);
  if (align & 15) {
    fat_host::set_error("fat_paged_decode_shared: q, K, V and workspace pointers and row strides must be 16-byte aligned");
    return FAT_E_INVALID;
  }
  // K/V offsets are products of 32-bit (page) and 24-bit (slot) factors; a page's
  // rows lie within 4 GiB of its start.
  auto fits = [&](int64_t sp, int64_t ss) {
    return sp >= 0 && ss >= 0 && eb * sp < (1LL << 32) && eb * ss < (1LL << 24) && a->page_size < (1 << 24) &&
           eb * ss * (int64_t)a->page_size < (1LL << 32);
  };
  if (!fits(a->k_stride_page, a->k_stride_slot) || !fits(a->v_stride_page, a->v_stride_slot) ||
      a->scale_stride_page < 0 || a->scale_stride_page >= (1LL << 32)) {
    fat_host::set_error("fat_paged_decode_shared: K/V strides must be non-negative, pages below 4 GiB "
                        "and slots below 16 MiB apart");
    return FAT_E_UNSUPPORTED;
  }
  const int S = a->prefix_split + a->split;
  const size_t need = fat_paged_decode_shared_workspace_bytes(a->batch * T, a->num_heads, a->head_dim, S);
  if (a->workspace_bytes < (int64_t)need) {
    fat_host::set_error("fat_paged_decode_shared: this launch needs %zu bytes of workspace, the caller's holds %lld",
                        need, (long long)a->workspace_bytes);
    return FAT_E_INVALID;
  }
  // Partials are written while the launch's other buffers are read.
  const uintptr_t ws = (uintptr_t)a->workspace;
  for (const void* p : {a->q, a->k_cache, a->v_cache, (const void*)a->k_scale, (const void*)a->v_scale,
                        (const void*)a->page_table, (const void*)a->seq_lens, (const void*)a->cu_groups,
                        (const void*)a->prefix_lens, (const void*)a->out}) {
    if ((uintptr_t)p >= ws && (uintptr_t)p < ws + need) {
      fat_host::set_error("fat_paged_decode_shared: the workspace overlaps another buffer of the launch");
      return FAT_E_INVALID;
    }
  }
  fat::SharedParams prm{};
  prm.q = static_cast<const uint8_t*>(a->q);
  prm.k = static_cast<const uint8_t*>(a->k_cache);
  prm.v = static_cast<const uint8_t*>(a->v_cache);
  prm.ks = a->k_scale;
  prm.vs = a->v_scale;
  prm.pt = a->page_table;
  prm.lens = a->seq_lens;
  prm.cu = a->cu_groups;
  prm.prefix = a->prefix_lens;
  prm.out = static_cast<uint8_t*>(a->out);
  prm.ws_acc = static_cast<float*>(a->workspace);
  prm.ws_ml = prm.ws_acc + (size_t)a->batch * T * a->num_heads * S * a->head_dim;
  prm.q_sb = a->q_stride_b;
  prm.q_st = T > 1 ? a->q_stride_t : 0;
  prm.q_sh = a->q_stride_h;
  prm.o_sb = a->out_stride_b;
  prm.o_st = T > 1 ? a->out_stride_t : 0;
  prm.o_sh = a->out_stride_h;
  prm.k_sp = (uint32_t)(eb * a->k_stride_page);
  prm.k_ss = (uint32_t)(eb * a->k_stride_slot);
  prm.k_sh = eb * a->k_stride_head;
  prm.v_sp = (uint32_t)(eb * a->v_stride_page);
  prm.v_ss = (uint32_t)(eb * a->v_stride_slot);
  prm.v_sh = eb * a->v_stride_head;
  prm.sc_sp = (uint32_t)a->scale_stride_page;
  prm.sc_sh = a->scale_stride_head;
  prm.pt_sb = a->page_table_stride;
  prm.B = a->batch;
  prm.G = a->groups;
  prm.T = T;
  prm.H = a->num_heads;
  prm.Hkv = a->num_kv_heads;
  prm.group = a->num_heads / a->num_kv_heads;
  prm.P = a->page_size;
  prm.invP = a->page_size > 1 ? (uint32_t)((uint64_t(1) << 32) / (uint32_t)a->page_size) : 0xffffffffu;
  prm.num_pages = a->num_pages;
  prm.max_pages = a->max_pages;
  const float scale = a->softmax_scale;
  prm.scale_log2 = (scale == 0.f ? 1.f : scale < 0.f ? -scale : scale) * fat::kLog2e;
  prm.q_and = scale == 0.f ? 0u : ~0u;
  prm.q_xor = scale < 0.f ? 0x80008000u : 0u;
  prm.prefix_split = a->prefix_split;
  prm.prefix_chunk = a->prefix_chunk;
  prm.split = a->split;
  prm.chunk = a->chunk;
  const int64_t rows = (int64_t)std::min(a->max_group, a->batch) * T * prm.group;
  const int rb = a->row_blocks ? a->row_blocks : rows > 32 ? 4 : 1;
  for (int own = 0; own < 2; ++own) {
    const uint32_t step = 32 * (own ? fat::kSharedWaves : fat::kSharedWaves / rb);
    prm.step_col[own] = step / (uint32_t)a->page_size;
    prm.step_slot[own] = step % (uint32_t)a->page_size;
  }
  const int64_t tiles = (rows + 32 * rb - 1) / (32 * rb);
  const int64_t units = (int64_t)a->groups * a->prefix_split * a->num_kv_heads;
  const int64_t own_tiles = (T * prm.group + 31) / 32;
  const int64_t prefix_blocks = (units + 7) / 8 * 8 * tiles;
  const int64_t own_blocks = (int64_t)a->batch * a->split * a->num_kv_heads * own_tiles;
  if (prefix_blocks + own_blocks > 0x7fffffffLL) {
    fat_host::set_error("fat_paged_decode_shared: %lld workgroups exceed one launch",
                        (long long)(prefix_blocks + own_blocks));
    return FAT_E_UNSUPPORTED;
  }
  prm.tiles = (int)tiles;
  prm.prefix_blocks = (int)prefix_blocks;
  prm.own_tiles = (int)own_tiles;
  hipStream_t stream = static_cast<hipStream_t>(stream_ptr);
  const unsigned blocks = (unsigned)(prefix_blocks + own_blocks);
  if (a->q_dtype == FAT_DTYPE_F16) launch_shared<fat::F16>(prm, kv, a->head_dim, rb, blocks, stream);
  else launch_shared<fat::BF16>(prm, kv, a->head_dim, rb, blocks, stream);
  const int rc = fat_host::launch_status("decode_shared_kernel");
  if (rc != FAT_OK) return rc;
  if (a->q_dtype == FAT_DTYPE_F16) launch_join<fat::F16>(prm, a->head_dim, stream);
  else launch_join<fat::BF16>(prm, a->head_dim, stream);
  return fat_host::launch_status("shared_join_kernel");
}
