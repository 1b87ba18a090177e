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
//
// What bounds it: own items stream K and V once (HBM); a prefix item does 4 x 32
// RB x D FLOPs per key, so long prefixes under many sequences are bound by the
// matrix cores and the softmax between the two products.
//
// Both kinds run the same tile: 32 keys x 32 rows per wave on
// v_mfma_f32_32x32x16, S^T = K Q^T with K as the A operand (its rows staged in
// LDS) and O^T += V^T P^T with P^T straight from S^T's registers and V^T by
// transposed LDS reads.  A workgroup's four waves are RB row blocks x KG = 4 / RB
// key groups: the RB waves of a key group share its tiles, the key groups take
// tiles in turn and join at the end.
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
  int64_t k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;  // bytes
  int64_t sc_sp, sc_sh;
  int64_t pt_sb;
  int32_t B, G, T, H, Hkv, group;
  int32_t P, log2P, num_pages, max_pages;
  uint32_t invP;
  float scale_log2;
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

template <typename QT, int KV, int D, int RB>
struct SharedTile {
  static constexpr int KG = kSharedWaves / RB;
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
  static constexpr bool FOLD = KV != KV_SAME && std::is_same<QT, F16>::value;  // k_scale on the scores
  static constexpr int kTileBytes = KG * kBufs * kTile * 2 + (FOLD ? KG * kBufs * 32 * 4 : 0);
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
  // P enters the second product as bf16 hi + lo parts: one bf16 alone (2^-9) would
  // show beside the output's own rounding where a row sees few keys.
  constexpr bool SPLIT_P = std::is_same<QT, BF16>::value;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = w % RB, kg = w / RB;
  const int li = lane & 31;  // key row (A operand) / row column (B, S^T)
  const int g = lane >> 5;   // k-group: head dims 16 ks + 8 g .. + 7 of k-step ks
  const int per_seq = p.T * p.group;
  const int R = n_seq * per_seq;
  const int n_tiles = t_end > t_begin ? (t_end - t_begin + 31) >> 5 : 0;

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
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + 32 * ks);
  }

  // Staging: chunk i NT + st of a tile is this lane's, st its place in the key group.
  const int st = rb * 64 + lane;
  const bool stages = NCH >= NT || st < NCH;
  const int srow = st / CPR;  // row of chunk 0; chunk i's is srow + i NT / CPR
  const int scol = st % CPR;
  const uint8_t* const kh = p.k + (int64_t)kvh * p.k_sh + 16 * scol;
  const uint8_t* const vh = p.v + (int64_t)kvh * p.v_sh + 16 * scol;
  const float* const ksh = KV != KV_SAME ? p.ks + (int64_t)kvh * p.sc_sh : nullptr;
  const float* const vsh = KV != KV_SAME ? p.vs + (int64_t)kvh * p.sc_sh : nullptr;
  struct Raw {
    u32x4 k[NLD], v[NLD];
    float ksc[NLD], vsc[NLD];
  } R0;
  int pid[NLD], pslot[NLD];
  // Page id and slot of this lane's rows of tile t; rows behind the end look up
  // its last key (a row that the sequence uses), columns and ids are clamped.
  auto lookup = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const uint32_t tok = (uint32_t)min(t_begin + 32 * t + srow + i * (NT / CPR), t_end - 1);
      uint32_t col;
      if (p.log2P >= 0) {
        col = tok >> p.log2P;
      } else {  // floor(tok / P): the high product is it or one less
        col = __umulhi(tok, p.invP);
        col += tok - col * (uint32_t)p.P >= (uint32_t)p.P ? 1u : 0u;
      }
      pslot[i] = (int)(tok - col * (uint32_t)p.P);
      pid[i] = ptrow[min((int)col, p.max_pages - 1)];
    }
  };
  // Loads tile t (whose ids are here), and the ids of tile t + KG behind it.
  auto fetch = [&](int t) __attribute__((always_inline)) {
    int phys[NLD], sl[NLD];
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      phys[i] = min(max(pid[i], 0), p.num_pages - 1);
      sl[i] = pslot[i];
    }
    lookup(t + KG);
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      R0.k[i] = *reinterpret_cast<const u32x4*>(kh + (int64_t)phys[i] * p.k_sp + (int64_t)sl[i] * p.k_ss);
      R0.v[i] = *reinterpret_cast<const u32x4*>(vh + (int64_t)phys[i] * p.v_sp + (int64_t)sl[i] * p.v_ss);
      if constexpr (KV != KV_SAME) {
        R0.ksc[i] = ksh[(int64_t)phys[i] * p.sc_sp];
        R0.vsc[i] = vsh[(int64_t)phys[i] * p.sc_sp];
      }
    }
  };
  // A chunk as QT elements: a copy, or round_to_QT(float(x) * scale) of 8-bit
  // codes (sc = 1 with FOLD's K: exact).
  auto put = [&](uint16_t* dst, const u32x4& raw, float sc) __attribute__((always_inline)) {
    if constexpr (KV == KV_SAME) {
      *reinterpret_cast<u32x4*>(dst) = raw;
    } else {
      const float nb = -128.0f * sc;
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float f[4];
          if constexpr (KV == KV_I8) {
            i8x4_biased(raw[2 * h2 + j], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = __builtin_fmaf(f[e], sc, nb);
          } else {
            fp8x4(raw[2 * h2 + j], f);
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = f[e] * sc;
          }
          o[2 * j] = Pair<QT>::pack(f[0], f[1]);
          o[2 * j + 1] = Pair<QT>::pack(f[2], f[3]);
        }
        *reinterpret_cast<u32x4*>(dst + 8 * h2) = o;
      }
    }
  };
  uint16_t* const tile0 = reinterpret_cast<uint16_t*>(smem) + kg * Tl::kBufs * Tl::kTile;
  float* const ksc0 = reinterpret_cast<float*>(smem + KG * Tl::kBufs * Tl::kTile * 2) + kg * Tl::kBufs * 32;
  auto store = [&](int t, int buf) __attribute__((always_inline)) {
    if (!stages) return;
    uint16_t* const Kt = tile0 + buf * Tl::kTile;
    uint16_t* const Vt = Kt + 32 * K_RS;
#pragma unroll
    for (int i = 0; i < NLD; ++i) {
      const int row = srow + i * (NT / CPR);
      // V behind the end is zero: the scores there are masked, and 0 * v stays 0
      // whatever the last key's v holds.
      const bool in = t_begin + 32 * t + row < t_end;
      const u32x4 vv = {in ? R0.v[i][0] : 0u, in ? R0.v[i][1] : 0u, in ? R0.v[i][2] : 0u, in ? R0.v[i][3] : 0u};
      put(&Kt[row * K_RS + scol * EPC], R0.k[i], FOLD ? 1.0f : R0.ksc[i]);
      put(&Vt[row * V_RS + scol * EPC], vv, KV != KV_SAME && !in ? 0.0f : R0.vsc[i]);
      if constexpr (FOLD) {
        if (scol == 0) ksc0[buf * 32 + row] = R0.ksc[i];
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
  const float c = p.scale_log2;
  const int tr_c = (lane & 15) >> 2, tr_j = lane & 3, tr_G = lane >> 4;
  const int tr_row = 4 * (tr_G >> 1) + tr_c;
  const int tr_col = 16 * (tr_G & 1) + 4 * tr_j;

  auto compute = [&](int t, int buf) __attribute__((always_inline)) {
    const uint16_t* const Kt = tile0 + buf * Tl::kTile;
    const uint16_t* const Vt = Kt + 32 * K_RS;
    f32x16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(&Kt[li * K_RS + 16 * ks + 8 * g]);
      s = Mfma<QT>::mma(a, qf[ks], s);
    }
    // Row li over keys kb + (r & 3) + 4 g + 8 (r >> 2).
    const int kb = t_begin + 32 * t;
    f32x4 ck[4];
    if constexpr (FOLD) {
#pragma unroll
      for (int j = 0; j < 4; ++j) ck[j] = *reinterpret_cast<const f32x4*>(&ksc0[buf * 32 + 4 * g + 8 * j]) * c;
    }
    float mx = -INFINITY;
    const bool masked = kb + 32 > all_end;  // uniform
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = s[r] * (FOLD ? ck[r >> 2][r & 3] : c);
      if (masked) x = kb + (r & 3) + 4 * g + 8 * (r >> 2) < my_end ? x : -INFINITY;
      s[r] = x;
      mx = fmaxf(mx, x);
    }
    mx = xor32<OpMax>(mx);
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
    // A row that has seen no key yet keeps m = -inf; its scores are -inf too,
    // and 2^(-inf - 0) = 0.
    const float m_use = m_run == -INFINITY ? 0.f : m_run;
    u32x4 pf[2], pl[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int e2 = 0; e2 < 4; ++e2) {
        const float x0 = fast_exp2(s[8 * u + 2 * e2] - m_use);
        const float x1 = fast_exp2(s[8 * u + 2 * e2 + 1] - m_use);
        l_run += x0 + x1;
        const u32 hp = Pair<QT>::pack(x0, x1);
        pf[u][e2] = hp;
        if constexpr (SPLIT_P) pl[u][e2] = Pair<QT>::pack(x0 - Pair<QT>::lo(hp), x1 - Pair<QT>::hi(hp));
      }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int vrow = 16 * u + tr_row;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint16_t* vp = &Vt[vrow * V_RS + 32 * db + tr_col];
        const u32x2 lo = lds_read_tr16(vp);
        const u32x2 hi = lds_read_tr16(vp + 8 * V_RS);
        const u32x4 a = {lo[0], lo[1], hi[0], hi[1]};
        acc[db] = Mfma<QT>::mma(a, pf[u], acc[db]);
        if constexpr (SPLIT_P) acc[db] = Mfma<QT>::mma(a, pl[u], acc[db]);
      }
    }
  };

  if constexpr (RB == 1) {
    // Each wave has its own tiles: no workgroup barrier.
    if (kg < n_tiles) {
      lookup(kg);
      fetch(kg);
    }
    for (int t = kg; t < n_tiles; t += KG) {
      store(t, 0);
      if (t + KG < n_tiles) fetch(t + KG);
      wave_lds_fence();
      compute(t, 0);
      wave_lds_fence();
    }
  } else {
    // The same number of rounds for all key groups (the barriers): a round behind
    // the end stages zeros of the last key's page and masks them all.
    const int rounds = (n_tiles + KG - 1) / KG;
    if (rounds > 0) {
      lookup(kg);
      fetch(kg);
      store(kg, 0);
    }
    for (int i = 0; i < rounds; ++i) {
      const int t = kg + i * KG;
      if (i + 1 < rounds) fetch(t + KG);
      // Tile i is here, and every wave is done with tile i - 1, whose buffer the
      // next store takes.
      __syncthreads();
      compute(t, i & 1);
      if (i + 1 < rounds) store(t + KG, (i + 1) & 1);
    }
  }

  const float l_tot = xor32<OpAdd>(l_run);
  auto row_of = [&](int r) {  // global row of row r of the item
    const int s = r / per_seq;
    const int in = r - s * per_seq;
    const int t = in / p.group;
    return ((int64_t)(b0 + s) * p.T + t) * p.H + kvh * p.group + (in - t * p.group);
  };
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
    const int nvalid = min(32 * RB, R - row0);
    if (32 * rb + li < nvalid) {
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
      const int at0 = (r >> 5) * 32 + (r & 31);  // key group 0's; the next ones' lie RB waves on
      float M = -INFINITY;
#pragma unroll
      for (int k = 0; k < KG; ++k) M = fmaxf(M, sml[(k * RB * 32 + at0) * 2]);
      f32x4 A = {0.f, 0.f, 0.f, 0.f};
      float L = 0.f;
#pragma unroll
      for (int k = 0; k < KG; ++k) {
        const int at = k * RB * 32 + at0;
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

template <typename QT, int KV, int D, int RB>
__global__ __launch_bounds__(kSharedWaves * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void decode_shared_kernel(const SharedParams p) {
  constexpr int kBytes = SharedTile<QT, KV, D, RB>::kBytes > SharedTile<QT, KV, D, 1>::kBytes
                             ? SharedTile<QT, KV, D, RB>::kBytes
                             : SharedTile<QT, KV, D, 1>::kBytes;
  __shared__ __attribute__((aligned(16))) uint8_t smem[kBytes];
  const int S = p.prefix_split + p.split;
  const int cap = p.max_pages * p.P;
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
    const int n = min(max(p.prefix[grp], 0), cap);
    const int t_begin = min(slot * p.prefix_chunk, n);
    const int t_end = slot == p.prefix_split - 1 ? n : min(t_begin + p.prefix_chunk, n);
    shared_segment<QT, KV, D, RB>(p, smem, b0, b1 - b0, kvh, row0, p.pt + (int64_t)b0 * p.pt_sb, t_begin, t_end, slot, S);
    return;
  }
  const int id = blockIdx.x - p.prefix_blocks;
  const int per_b = p.split * p.Hkv * p.own_tiles;
  const int b = id / per_b;
  const int r = id - b * per_b;
  const int slot = r / (p.Hkv * p.own_tiles);
  const int y = r - slot * (p.Hkv * p.own_tiles);
  const int kvh = y / p.own_tiles;
  const int tile = y - kvh * p.own_tiles;
  const int grp = group_of(p.cu, p.G, b);
  const int len = min(max(p.lens[b], 0), cap);
  const int n = grp < 0 ? 0 : min(max(p.prefix[grp], 0), len);
  const int t_begin = min((int64_t)n + (int64_t)slot * p.chunk, (int64_t)len);
  const int t_end = slot == p.split - 1 ? len : min((int64_t)t_begin + p.chunk, (int64_t)len);
  shared_segment<QT, KV, D, 1>(p, smem, b, 1, kvh, tile * 32, p.pt + (int64_t)b * p.pt_sb, t_begin, t_end,
                               p.prefix_split + slot, S);
}

// Joins a row's S partials, one wave per row: lane s has those of slots s and s +
// 64.  Slots of weight 0 (no keys) are not read.
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
  for (int s = 0; s < S; ++s) {
    const float w = __shfl(s < 64 ? f[0] : f[1], s & 63);
    if (w != 0.f) {  // uniform
#pragma unroll
      for (int e = 0; e < E; ++e) a[e] = __builtin_fmaf(acc[(int64_t)s * D + e], w, a[e]);
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
    case 2: hipLaunchKernelGGL((fat::decode_shared_kernel<QT, KV, D, 2>), dim3(blocks), block, 0, stream, prm); break;
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
  const int S = a->prefix_split + a->split;
  const size_t need = fat_paged_decode_shared_workspace_bytes(a->batch * T, a->num_heads, a->head_dim, S);
  if (a->workspace_bytes < (int64_t)need) {
    fat_host::set_error("fat_paged_decode_shared: this launch needs %zu bytes of workspace, the caller's holds %lld",
                        need, (long long)a->workspace_bytes);
    return FAT_E_INVALID;
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
  prm.k_sp = eb * a->k_stride_page;
  prm.k_ss = eb * a->k_stride_slot;
  prm.k_sh = eb * a->k_stride_head;
  prm.v_sp = eb * a->v_stride_page;
  prm.v_ss = eb * a->v_stride_slot;
  prm.v_sh = eb * a->v_stride_head;
  prm.sc_sp = a->scale_stride_page;
  prm.sc_sh = a->scale_stride_head;
  prm.pt_sb = a->page_table_stride;
  prm.B = a->batch;
  prm.G = a->groups;
  prm.T = T;
  prm.H = a->num_heads;
  prm.Hkv = a->num_kv_heads;
  prm.group = a->num_heads / a->num_kv_heads;
  prm.P = a->page_size;
  prm.log2P = -1;
  for (int l = 0; l < 31; ++l)
    if (a->page_size == (1 << l)) prm.log2P = l;
  prm.invP = a->page_size > 1 ? (uint32_t)((uint64_t(1) << 32) / (uint32_t)a->page_size) : 0;
  prm.num_pages = a->num_pages;
  prm.max_pages = a->max_pages;
  prm.scale_log2 = a->softmax_scale * fat::kLog2e;
  prm.prefix_split = a->prefix_split;
  prm.prefix_chunk = a->prefix_chunk;
  prm.split = a->split;
  prm.chunk = a->chunk;
  const int64_t rows = (int64_t)std::min(a->max_group, a->batch) * T * prm.group;
  const int rb = 1;
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
