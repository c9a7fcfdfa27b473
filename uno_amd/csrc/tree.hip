// Attention of a tree of drafted tokens over a KV cache.
//
// Node t of sequence b (parents[b, t] an earlier node, or -1 for a root, or less for padding) attends to the
// sequence's n = lengths[b] committed cache rows, its ancestors and itself; node a's K and V are cache row n + a.
// The queries of one (sequence, K/V head) pair, rep q heads x T nodes, are the rows of one product, so each
// cache row is read once per row tile.
//
// A workgroup takes one row tile and one range of the keys (see tree_range); ranges of one sequence are merged by a second
// kernel. Two walks, by the number of rows (see tree_plan):
// * few rows (16; fp32 32), bound by HBM: tree_attn_kernel, K and V straight into the MFMAs' registers;
// * more rows, bf16, bound by LDS, MFMA and VALU alike: tree_attn_lds_kernel, K and V tiles shared through LDS.
// In both S^T = K Q^T and O^T = V^T P^T, so that a query is a column: its maximum and sum are one number in a lane, and S^T's
// accumulators are P^T's operand as they stand.
// The maximum that a row's weights refer to moves only when a score exceeds it by 2^8 (the weights stay
// within fp32 and bf16 range), so that most tiles pass without rescaling. Scores, statistics and outputs are fp32.
//
// The weights of bf16 products are rounded to bf16 (half a step, 2^-8 of each; their sum is not), as in the framework's other bf16
// attention: the output's error against 64 bits is 2.3e-3 of its size, where its own rounding to bf16 makes 1.7e-3. A second
// product with what the rounding leaves makes it 1.7e-3, for a quarter more time where the matrix cores bind: 8 sequences of 4096
// rows, 16 nodes 33.4 -> 34.6 us, 32 nodes 38.2 -> 42.8, 16 sequences of 16384 rows, 64 nodes 330 -> 416. And what is left of a
// weight may be 0 or negative, so that an infinite committed value would give NaN. fp32 products have fp32 weights.
#include "tree.h"
#include "../../include/unok.h"

namespace {

template <typename T, int D> struct TileOps;

// bf16: tiles of 32 keys. Slot j of lane group g is key 4 g + j (j < 4) or 16 + 4 g + j - 4, in P and in V.
template <int D> struct TileOps<bf16_t, D> {
  static constexpr int KT = 32, NS = 2, NDT = D / 16;   // keys per tile, 16-key subtiles, 16-dim output tiles
  static constexpr int KS = D / 32, VW = D / 32;        // k-steps of S; dwords of a lane's V row part
  struct Q { bf16x8_t f[KS]; };
  struct K { bf16x8_t f[NS][KS]; };
  struct V { uint32_t w[8][VW]; };
  typedef f32x4_t Acc;

  static __device__ __forceinline__ int slot_key(int j, int g) { return j < 4 ? 4 * g + j : 12 + 4 * g + j; }
  // The dim of accumulator element e of output tile c
  static __device__ __forceinline__ int dim(int c, int e, int g) { return (4 * g + e) * NDT + c; }

  static __device__ __forceinline__ void load_q(Q& q, const bf16_t* row, int g) {
#pragma unroll
    for (int s = 0; s < KS; ++s) q.f[s] = *(const bf16x8_t*)(row + 32 * s + 8 * g);
  }
  template <bool PAST, typename F> static __device__ __forceinline__ void load_k(K& k, F row, int m, int g) {
#pragma unroll
    for (int a = 0; a < NS; ++a) {
      const bf16_t* r = row(16 * a + m);
#pragma unroll
      for (int s = 0; s < KS; ++s) k.f[a][s] = tree_load<PAST>((const bf16x8_t*)(r + 32 * s + 8 * g));
    }
  }
  template <bool PAST, typename F> static __device__ __forceinline__ void load_v(V& v, F row, int m, int g) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bf16_t* r = row(slot_key(j, g)) + NDT * m;
      if constexpr (VW == 4) { const u32x4_t u = tree_load<PAST>((const u32x4_t*)r); v.w[j][0] = u[0]; v.w[j][1] = u[1]; v.w[j][2] = u[2]; v.w[j][3] = u[3]; }
      else { const u32x2_t u = tree_load<PAST>((const u32x2_t*)r); v.w[j][0] = u[0]; v.w[j][1] = u[1]; }
    }
  }
  static __device__ __forceinline__ Acc score(const K& k, const Q& q, int a) {
    Acc s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KS; ++i) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k.f[a][i], q.f[i], s, 0, 0, 0);
    return s;
  }
  template <int QT> static __device__ __forceinline__ void add_pv(const V& v, const float (&p)[QT][8], Acc (&o)[QT][NDT]) {
    bf16x8_t pf[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i)
      pf[i] = __builtin_bit_cast(bf16x8_t, u32x4_t{pack2_bf16(p[i][0], p[i][1]), pack2_bf16(p[i][2], p[i][3]),
                                                   pack2_bf16(p[i][4], p[i][5]), pack2_bf16(p[i][6], p[i][7])});
#pragma unroll
    for (int c = 0; c < NDT; ++c) {
      u32x4_t a;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        a[j] = __builtin_amdgcn_perm(v.w[2 * j + 1][c / 2], v.w[2 * j][c / 2], c % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
      for (int i = 0; i < QT; ++i)
        o[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), pf[i], o[i][c], 0, 0, 0);
    }
  }
  // Whether v holds an infinity or NaN; clean() makes those 0.
  static __device__ __forceinline__ bool odd(const V& v) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < VW; ++i)
        bad |= (v.w[j][i] & 0x7f80u) == 0x7f80u || (v.w[j][i] & 0x7f800000u) == 0x7f800000u;
    return bad;
  }
  static __device__ __forceinline__ void clean(V& v) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        if ((v.w[j][i] & 0x7f80u) == 0x7f80u) v.w[j][i] &= 0xffff0000u;
        if ((v.w[j][i] & 0x7f800000u) == 0x7f800000u) v.w[j][i] &= 0x0000ffffu;
      }
  }
};

// fp32: tiles of 16 keys, 16x16x4 MFMAs. MFMA e of a 16-byte load uses element e: k slot g is dim 16 s + 4 g + e in S
// and key 4 g + e in O.
template <int D> struct TileOps<float, D> {
  static constexpr int KT = 16, NS = 1, NDT = D / 16;
  static constexpr int KS = D / 16, NJ = D / 64;
  struct Q { f32x4_t f[KS]; };
  struct K { f32x4_t f[1][KS]; };
  struct V { f32x4_t w[4][NJ]; };
  typedef f32x4_t Acc;

  static __device__ __forceinline__ int slot_key(int j, int g) { return 4 * g + j; }
  // output tile c = 4 jj + x holds dims 64 jj + 4 m + x
  static __device__ __forceinline__ int dim(int c, int e, int g) { return 64 * (c / 4) + 4 * (4 * g + e) + c % 4; }

  static __device__ __forceinline__ void load_q(Q& q, const float* row, int g) {
#pragma unroll
    for (int s = 0; s < KS; ++s) q.f[s] = *(const f32x4_t*)(row + 16 * s + 4 * g);
  }
  template <bool PAST, typename F> static __device__ __forceinline__ void load_k(K& k, F row, int m, int g) {
    const float* r = row(m);
#pragma unroll
    for (int s = 0; s < KS; ++s) k.f[0][s] = tree_load<PAST>((const f32x4_t*)(r + 16 * s + 4 * g));
  }
  template <bool PAST, typename F> static __device__ __forceinline__ void load_v(V& v, F row, int m, int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* r = row(slot_key(j, g)) + 4 * m;
#pragma unroll
      for (int jj = 0; jj < NJ; ++jj) v.w[j][jj] = tree_load<PAST>((const f32x4_t*)(r + 64 * jj));
    }
  }
  static __device__ __forceinline__ Acc score(const K& k, const Q& q, int a) {
    Acc s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k.f[0][i][e], q.f[i][e], s, 0, 0, 0);
    return s;
  }
  template <int QT> static __device__ __forceinline__ void add_pv(const V& v, const float (&p)[QT][4], Acc (&o)[QT][NDT]) {
#pragma unroll
    for (int c = 0; c < NDT; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < QT; ++i)
          o[i][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.w[j][c / 4][c % 4], p[i][j], o[i][c], 0, 0, 0);
  }
  static __device__ __forceinline__ bool odd(const V& v) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4 * NJ; ++i) bad |= (__float_as_uint(v.w[j][i / 4][i % 4]) & 0x7f800000u) == 0x7f800000u;
    return bad;
  }
  static __device__ __forceinline__ void clean(V& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4 * NJ; ++i)
        if ((__float_as_uint(v.w[j][i / 4][i % 4]) & 0x7f800000u) == 0x7f800000u) v.w[j][i / 4][i % 4] = 0.f;
  }
};

// Few query rows (16 QT): the four waves take key tiles in turn, each with its own running maximum and sum, and merge at the end: no
// barrier in the walk, and no LDS either. K and V go from memory into the registers that the MFMAs read:
//   S^T = K Q^T   the first operand wants 16 keys x 8 (fp32: 4) consecutive dims per lane: 16-byte loads of K;
//   O^T = V^T P^T the second operand is P^T as S^T's accumulators hold it (lane: query l % 16, four keys), and the first
//                 wants, per lane, one dim of eight (four) keys. With the accumulators' dims numbered so that lane
//                 m = l % 16 owns dims 8 m .. 8 m + 7 (4 m .. + 3 of each 64), those are 16-byte loads of V rows, and a
//                 bf16 pair of keys is one byte permute.
// One tile ahead in a second register set. Bound by HBM: 8 sequences, 32 / 8 heads of 128 bf16, one node over 16384 rows 96 us (5.6
// TB/s), over 4096 rows 28 us with the merge; a single sequence of 130 rows 8 us, which is launch and latency. fp32, 32 rows, bound
// by its 16x16x4 MFMAs: 16 nodes over 4096 rows 108 us (64 rows a workgroup, which spills: 209).
template <typename E, int D, int QT>
__global__ __launch_bounds__(256, 1) void tree_attn_kernel(const TreeAttn a) {
  using Ops = TileOps<E, D>;
  constexpr int KT = Ops::KT, NS = Ops::NS, NDT = Ops::NDT, NP = 4 * NS, ROWS = 16 * QT, LDO = D + 4;
  extern __shared__ __attribute__((aligned(16))) float merge_o[];     // [4][ROWS][LDO]
  __shared__ float merge_ml[4][ROWS][2];
  __shared__ bool merge_pad[ROWS];
  __shared__ uint32_t anc[TREE_MAX * TREE_WORDS];
  __shared__ int next[TREE_MAX];

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int rep = a.nq / a.nk, T = a.T, NR = rep * T;
  int tile, h, id;
  tree_place(a, tile, h, id);
  const Range range = tree_range(a, id, D * (int)sizeof(E));
  if (range.b < 0 || range.lo >= range.hi) return;
  const int b = range.b, n = range.n, end = range.end, lo = range.lo, hi = range.hi;
  tree_note(a, range, id, h, tile);

  if (hi > n) tree_ancestors(a.parents + b * a.ldp, T, anc, next);
  const int W = (T + 31) / 32;

  // this lane's query of each 16-row subtile (rows past the pair's last repeat it; their results are dropped)
  typename Ops::Q q[QT];
  int node[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = tile * ROWS + 16 * i + m, rc = r < NR ? r : NR - 1;
    node[i] = rc % T;
    Ops::load_q(q[i], (const E*)a.q + ((int64_t)b * T + node[i]) * a.ldq + ((int64_t)h * rep + rc / T) * D, g);
    if (threadIdx.x < 16) merge_pad[16 * i + m] = a.parents[b * a.ldp + node[i]] < -1;
  }

  const E* kbase = (const E*)a.k + b * a.kb + h * a.kh;
  const E* vbase = (const E*)a.v + b * a.vb + h * a.vh;
  typename Ops::Acc o[QT][NDT];
  float mref[QT], l[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    mref[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < NDT; ++c) o[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // scores in units of log2; the weights of a tile and their sums from them
  auto scores = [&](const typename Ops::K& k, float (&p)[QT][NP]) {
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const typename Ops::Acc z = Ops::score(k, q[i], s);
#pragma unroll
        for (int e = 0; e < 4; ++e) p[i][4 * s + e] = z[e] * a.scale_log2;
      }
  };
  auto weights = [&](float (&p)[QT][NP]) {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float mx = p[i][0];
#pragma unroll
      for (int j = 1; j < NP; ++j) mx = fmaxf(mx, p[i][j]);
      if (__ballot(mx > mref[i] + 8.f)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        // (for the queries that need it alone: a row's result does not depend on the rows beside it)
        const float to = mx > mref[i] + 8.f ? mx : mref[i];
        const float f = to == mref[i] ? 1.f : mref[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref[i] - to);
        mref[i] = to;
        l[i] *= f;
#pragma unroll
        for (int c = 0; c < NDT; ++c) o[i][c] *= f;
      }
      const float ref = mref[i] == -INFINITY ? 0.f : mref[i];
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        p[i][j] = __builtin_amdgcn_exp2f(p[i][j] - ref);
        l[i] += p[i][j];
      }
    }
  };

  // Tiles of committed rows, which every query sees: one tile ahead, in two register sets.
  const int full = hi < n ? hi : n;
  int key = lo + wid * KT;
  auto walk = [&](auto past) {
    constexpr bool PAST = decltype(past)::value;
    auto load = [&](typename Ops::K& k, typename Ops::V& v, int key0) {
      Ops::template load_k<PAST>(k, [&](int j) { return kbase + (int64_t)(key0 + j) * a.kr; }, m, g);
      Ops::template load_v<PAST>(v, [&](int j) { return vbase + (int64_t)(key0 + j) * a.vr; }, m, g);
    };
    auto step = [&](const typename Ops::K& k, const typename Ops::V& v) {
      float p[QT][NP];
      scores(k, p);
      weights(p);
      Ops::template add_pv<QT>(v, p, o);
    };
    typename Ops::K k0, k1;
    typename Ops::V v0, v1;
    if (key + KT <= full) load(k0, v0, key);
    while (key + KT <= full) {
      if (key + 5 * KT <= full) load(k1, v1, key + 4 * KT);
      step(k0, v0);
      key += 4 * KT;
      if (key + KT > full) break;
      if (key + 5 * KT <= full) load(k0, v0, key + 4 * KT);
      step(k1, v1);
      key += 4 * KT;
    }
  };
  if (range.past) walk(std::true_type{});
  else walk(std::false_type{});
  // Tiles with tree rows. Keys at or past the end read the last row, at weight 0.
#pragma unroll 1
  for (; key < hi; key += 4 * KT) {
    typename Ops::K k;
    typename Ops::V v;
    Ops::template load_k<false>(k, [&](int j) { const int r = key + j; return kbase + (int64_t)(r < end ? r : end - 1) * a.kr; }, m, g);
    Ops::template load_v<false>(v, [&](int j) { const int r = key + j; return vbase + (int64_t)(r < end ? r : end - 1) * a.vr; }, m, g);
    float p[QT][NP];
    scores(k, p);
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int r = key + Ops::slot_key(j, g), t = r - n;
        p[i][j] = r < hi && (t < 0 | tree_sees(anc, node[i], W, t)) ? p[i][j] : -INFINITY;
      }
    weights(p);
    const bool odd = __ballot(Ops::odd(v)) != 0;
    if (odd) Ops::clean(v);
    Ops::template add_pv<QT>(v, p, o);
    if (odd) {
      // An infinity or NaN among rows that some queries do not see: it was 0 in the product and is added where
      // it is seen. The weights go through this wave's part of the merge buffer.
      float* ps = merge_o + wid * ROWS * LDO;
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int j = 0; j < NP; ++j) ps[(16 * i + m) * (KT + 1) + Ops::slot_key(j, g)] = p[i][j];
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int j = 0; j < KT && key + j < hi; ++j) {
        const int t = key + j - n;
        const E* row = vbase + (int64_t)(key + j) * a.vr;
#pragma unroll
        for (int c = 0; c < NDT; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = Elem<E>::load(row + Ops::dim(c, e, g));
            if (!__ballot(!(fabsf(x) < INFINITY))) continue;
#pragma unroll
            for (int i = 0; i < QT; ++i) {
              const bool seen = t < 0 | tree_sees(anc, node[i], W, t);
              if (seen && !(fabsf(x) < INFINITY)) o[i][c][e] += ps[(16 * i + m) * (KT + 1) + j] * x;
            }
          }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  tree_merge<E, D, QT>(a, range, tile, h, id, o, mref, l, merge_o, merge_ml, merge_pad,
                       [](int c, int e, int g) { return Ops::dim(c, e, g); });
}

// max over lanes l and l ^ 32
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// bf16, more than 16 query rows: K and V tiles in LDS, filled by direct-to-LDS loads ahead of their use, 32x32x16 MFMAs, 32 rows
// to a wave, RG groups of 32 rows to a workgroup. V's columns come by LDS transpose loads (see lds_tile.h).
//   RG = 2: 4 waves, tiles of 64 keys in two stages, two workgroups to a CU; a row group's two waves take half of every tile's keys
//           each. 8 sequences, 32 / 8 heads of 128, 16 nodes over 4096 rows: 25 us and 5.3 for the merge (the 134 MB are
//           in the memory-side cache; four stages and one workgroup to a CU: 52 us in place of 45 at the time; 8 waves: 64
//           sequences of 1000 rows 66 us in place of 55); over 16384 rows 103 us, 5.2 TB/s.
//   RG = 4: 8 waves, tiles of 128 keys in two stages, key halves as above: 32 nodes over 4096 rows 39 us (4 waves, all keys
//           each: 43).
//   RG = 8: 8 waves, all keys each, tiles of 64 keys in four stages: 16 sequences, 64 nodes over 16384 rows 265-320 us, 0.85
//           PFLOP/s (RG = 4 in twice the row tiles: 350). A wave's 64 keys x 32 rows take 1024 cycles of MFMA, as many of LDS
//           reads and 900 of VALU (the exponentials are half of those), two waves to a SIMD, and the clock falls under the
//           load: the shorter time is of single calls, the longer of calls back to back. (64 rows a wave in four waves read LDS half
//           as often, but nothing runs beside a wave's own exponentials: 359 us.)
template <int D, int RG>
__global__ __launch_bounds__(RG == 2 ? 256 : 512, 2) void tree_attn_lds_kernel(const TreeAttn a) {
  constexpr int NKS = D / 16, NDT = D / 32, ROWS = 32 * RG, NW = RG == 2 ? 4 : 8;
  constexpr int KG = NW / RG, NKK = RG == 2 ? 1 : 2;    // key groups; a wave's 32-key parts of a tile
  constexpr int TK = 32 * NKK * KG, TILE = TK * D;      // keys of a tile
  constexpr int NST = RG == 8 ? 4 : 2;                  // stages
  constexpr int LPT = TK * D * 2 * 2 / (1024 * NW);     // direct-to-LDS loads per wave and tile
  constexpr int STAGE = 2 * TILE;                       // a stage: the K tile, then the V tile
  extern __shared__ __attribute__((aligned(16))) bf16_t smem[];
  __shared__ uint32_t anc[TREE_MAX * TREE_WORDS];
  __shared__ int next[TREE_MAX];

  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 5, lq = lane & 31;
  const int wid = __builtin_amdgcn_readfirstlane(w);
  const int rep = a.nq / a.nk, T = a.T, NR = rep * T, W = (T + 31) / 32;
  int tile0, h, id;
  tree_place(a, tile0, h, id);
  const Range range = tree_range(a, id, D * 2);
  if (range.b < 0 || range.lo >= range.hi) return;
  const int b = range.b, n = range.n, lo = range.lo, hi = range.hi;
  tree_note(a, range, id, h, tile0);
  const bf16_t* kbase = (const bf16_t*)a.k + b * a.kb + h * a.kh;
  const bf16_t* vbase = (const bf16_t*)a.v + b * a.vb + h * a.vh;
  const uint32_t ko = dma_lane_off<D, NW>(a.kr, 0, wid, lane), vo = dma_lane_off<D, NW>(a.vr, 0, wid, lane);
  auto fetch = [&](int key, int stage) {               // rows at or past hi read as zeros
    auto go = [&](auto past) {
#pragma unroll
      for (int i = 0; i < TK / 64; ++i) {
        dma_tile<D, NW, decltype(past)::value>(kbase, a.kr, ko, key + 64 * i, hi, smem + stage * STAGE + 64 * i * D, wid);
        dma_tile<D, NW, decltype(past)::value>(vbase, a.vr, vo, key + 64 * i, hi, smem + stage * STAGE + TILE + 64 * i * D, wid);
      }
    };
    if (range.past) go(std::true_type{});
    else go(std::false_type{});
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (lo + i * TK < hi) fetch(lo + i * TK, i);
  if (hi > n) tree_ancestors(a.parents + b * a.ldp, T, anc, next);

  // this lane's query (rows past the pair's last repeat it; their results are dropped)
  const int row = tile0 * ROWS + (wid % RG) * 32 + lq, rc = row < NR ? row : NR - 1, node = rc % T;
  const int part = wid / RG * NKK;                       // this wave's first 32-key part of a tile
  const bool pad = a.parents[b * a.ldp + node] < -1;
  bf16x8_t q[NKS];
  {
    const bf16_t* qp = (const bf16_t*)a.q + ((int64_t)b * T + node) * a.ldq + ((int64_t)h * rep + rc / T) * D;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) q[ks] = *(const bf16x8_t*)(qp + ks * 16 + g * 8);
  }
  if (a.q_factor != 1.f) {
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) q[ks] *= (__bf16)a.q_factor;
  }
  float m = -INFINITY, l = 0.f;
  f32x16_t o[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[t][j] = 0.f;

  int koff[NKS];
#pragma unroll
  for (int ks = 0; ks < NKS; ++ks) koff[ks] = lq * D + (((ks * 2 + g) ^ kswz<D>(lq)) << 3) + part * 32 * D;
  uint2 vaddr[NDT];
  const uint32_t vbase0 = lds_addr(smem + TILE) + part * 32 * D * 2;
#pragma unroll
  for (int t = 0; t < NDT; ++t) {
    const int2 off = tr_frag_off<D>(t, lane);
    vaddr[t] = make_uint2(vbase0 + 2 * off.x, vbase0 + 2 * off.y);
  }

  // One tile: of committed rows, which every query sees, in stage ST; or (MASKED) with tree rows, in stage `stage`.
  auto tile = [&](const int key, const int stage, auto stc, auto maskc) {
    constexpr bool MASKED = decltype(maskc)::value;
    constexpr int ST = decltype(stc)::value;
    constexpr bool DYN = MASKED || NST > 2;             // the stage is no constant
    const int at = DYN ? stage * STAGE : ST * STAGE;
    // the tile is in LDS (the NST - 2 after it may still be on their way), and every wave is done with the one
    // before, whose stage the next load overwrites
    if (NST > 2 && key + (NST - 2) * TK < hi) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((NST - 2) * LPT) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    bool odd = false;
    if constexpr (MASKED) {
      // An infinity or NaN in a V row that some queries do not see: 0 in the product, added afterwards where seen.
      uint32_t* vt = (uint32_t*)(smem + at + TILE);
      for (int i = tid; i < TILE / 2; i += 64 * NW) odd |= (vt[i] & 0x7f80u) == 0x7f80u || (vt[i] & 0x7f800000u) == 0x7f800000u;
      odd = __syncthreads_or(odd);
      if (odd) {
        for (int i = tid; i < TILE / 2; i += 64 * NW) {
          uint32_t u = vt[i];
          if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
          if ((u & 0x7f800000u) == 0x7f800000u) u &= 0x0000ffffu;
          vt[i] = u;
        }
        __syncthreads();
      }
    }
    const int ahead = DYN ? (stage + NST - 1) % NST : ST ^ 1, next_key = key + (NST - 1) * TK;
    if (next_key < hi && !odd) fetch(next_key, ahead);
    const bf16_t* Kc = smem + at;
    f32x16_t s[NKK];
    {
      bf16x8_t kf[NKK][NKS];
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) kf[kk][ks] = *(const bf16x8_t*)(Kc + kk * 32 * D + koff[ks]);
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk) {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[kk][j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s[kk] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk][ks], q[ks], s[kk], 0, 0, 0);
      }
      // every K fragment is read before the first product
#pragma unroll
      for (int i = 0; i < NKK * NKS; ++i) __builtin_amdgcn_sched_group_barrier(SG_DS_READ, 1, 0);
#pragma unroll
      for (int i = 0; i < NKK * NKS; ++i) __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    // V operands of the 16-key steps of half kk
    u32x2_t vlo[NKK][2][NDT], vhi[NKK][2][NDT];
    auto issue_v = [&](int kk) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int t = 0; t < NDT; ++t) {
          const uint32_t dyn = at * 2;
          tr_issue_p<D>(make_uint2(vaddr[t].x + dyn, vaddr[t].y + dyn), kk * 2 + hh, vlo[kk][hh][t],
                                                     vhi[kk][hh][t]);
        }
    };
    issue_v(0);
    if constexpr (MASKED) {
#pragma unroll
      for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int r = key + (part + kk) * 32 + 8 * (j >> 2) + 4 * g + (j & 3), t = r - n;
          s[kk][j] = r < hi && (t < 0 | tree_sees(anc, node, W, t)) ? s[kk][j] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int kk = 0; kk < NKK; ++kk)
#pragma unroll
      for (int j = 0; j < 16; ++j) top = fmaxf(top, s[kk][j]);
    top = half_max(top) * a.walk_scale;
    const bool grow = top > m + 8.f;
    if (__ballot(grow)) {
      // (for the queries that need it alone: a row's result does not depend on the rows beside it)
      const float to = grow ? top : m, f = !grow ? 1.f : m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= f;
#pragma unroll
      for (int t = 0; t < NDT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] *= f;
    }
    const float ref = m == -INFINITY ? 0.f : -m;
    bf16x8_t p[NKK][2];
    auto weights = [&](int kk) {
      float e[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        e[j] = __builtin_amdgcn_exp2f(fmaf(s[kk][j], a.walk_scale, ref));
        l += e[j];
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
        p[kk][hh] = __builtin_bit_cast(bf16x8_t, u32x4_t{pack2_bf16(e[8 * hh], e[8 * hh + 1]), pack2_bf16(e[8 * hh + 2], e[8 * hh + 3]),
                                                         pack2_bf16(e[8 * hh + 4], e[8 * hh + 5]), pack2_bf16(e[8 * hh + 6], e[8 * hh + 7])});
      if (MASKED && odd) {
        // this half's weights (-1: not seen) through the free stage, its V rows from memory
        float* ws = (float*)(smem + ahead * STAGE) + wid * 1024;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          ws[(8 * (j >> 2) + 4 * g + (j & 3)) * 32 + lq] = s[kk][j] == -INFINITY ? -1.f : e[j];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int j = 0; j < 32; ++j) {
          const int r = key + (part + kk) * 32 + j;
          if (r >= hi) break;
          const float x = ws[j * 32 + lq];          // (a NaN weight is seen)
          const bf16_t* vr = vbase + (int64_t)r * a.vr + 4 * g;
#pragma unroll
          for (int t = 0; t < NDT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float y = bf16_to_f32(vr[32 * t + 8 * (i >> 2) + (i & 3)]);
              if (!(x < 0.f) && !(fabsf(y) < INFINITY)) o[t][i] += x * y;
            }
        }
        __builtin_amdgcn_wave_barrier();
      }
    };
    auto pv = [&](int kk) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int t = 0; t < NDT; ++t)
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_join(vlo[kk][hh][t], vhi[kk][hh][t]), p[kk][hh], o[t], 0, 0, 0);
    };
    weights(0);
    tr_wait_all<NDT>(vlo[0], vhi[0]);
    if constexpr (NKK == 2) {
      issue_v(1);
      // the first half's products run while the VALU forms the second half's weights
      pv(0);
      weights(1);
      if constexpr (!MASKED) {
#pragma unroll
        for (int i = 0; i < 2 * NDT; ++i) {
          __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
          __builtin_amdgcn_sched_group_barrier(SG_VALU, 56 / (2 * NDT), 0);
        }
      }
      tr_wait_all<NDT>(vlo[1], vhi[1]);
      pv(1);
    } else {
      pv(0);
    }
    if (odd && next_key < hi) {
      __syncthreads();                                  // every wave has read its weights from the stage ahead
      fetch(next_key, ahead);
    }
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  const int full = lo + max(min(hi, n) - lo, 0) / TK * TK;
  int key = lo, stage = 0;
  if constexpr (NST == 2) {
#pragma unroll 1
    for (; key + TK < full; key += 2 * TK) {
      tile(key, 0, I0{}, std::false_type{});
      tile(key + TK, 1, I1{}, std::false_type{});
    }
    if (key < full) {
      tile(key, 0, I0{}, std::false_type{});
      key += TK;
      stage = 1;
    }
  } else {
#pragma unroll 1
    for (; key < full; key += TK, stage = (stage + 1) % NST) tile(key, stage, I0{}, std::false_type{});
  }
#pragma unroll 1
  for (; key < hi; key += TK, stage = (stage + 1) % NST) tile(key, stage, I0{}, std::true_type{});
  l += __shfl_xor(l, 32, 64);

  if constexpr (KG > 1) {
    // the other key groups' waves hand their outputs over, relative to the common maximum
    float* mo = (float*)smem;                            // [KG - 1][RG][NDT 16][64]
    float* ml = mo + (KG - 1) * RG * NDT * 16 * 64;      // [NW][64]
    const int rg = wid % RG;
    __syncthreads();
    if (g == 0) { ml[wid * 64 + lq] = m; ml[wid * 64 + 32 + lq] = l; }
    __syncthreads();
    float top = ml[rg * 64 + lq];
#pragma unroll
    for (int i = 1; i < KG; ++i) top = fmaxf(top, ml[(i * RG + rg) * 64 + lq]);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < KG; ++i) {
      const float mi = ml[(i * RG + rg) * 64 + lq], li = ml[(i * RG + rg) * 64 + 32 + lq];
      l += mi == -INFINITY ? li : li * __builtin_amdgcn_exp2f(mi - top);   // no maximum: 0, or NaN from NaN scores alone
    }
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    m = top;
#pragma unroll
    for (int t = 0; t < NDT; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[t][j] *= f;
        if (wid >= RG) mo[((wid - RG) * NDT * 16 + t * 16 + j) * 64 + lane] = o[t][j];
      }
    __syncthreads();
    if (wid >= RG) return;
#pragma unroll
    for (int i = 0; i < KG - 1; ++i)
#pragma unroll
      for (int t = 0; t < NDT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] += mo[((i * RG + wid) * NDT * 16 + t * 16 + j) * 64 + lane];
  }
  if (row >= NR) return;
  if (range.count == 1) {
    const bool none = l == 0.f || pad;
    bf16_t* dst = (bf16_t*)a.o + ((int64_t)b * T + node) * a.ldo + ((int64_t)h * rep + row / T) * D + 4 * g;
#pragma unroll
    for (int t = 0; t < NDT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : o[t][4 * j + e] / l;
        *(u32x2_t*)(dst + 32 * t + 8 * j) = u32x2_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
      }
  } else {
    const int64_t at = ((int64_t)id * a.nk + h) * NR + row;
    float* dst = a.po + at * D + 4 * g;
#pragma unroll
    for (int t = 0; t < NDT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *(f32x4_t*)(dst + 32 * t + 8 * j) = f32x4_t{o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]};
    if (g == 0) { a.pm[2 * at] = m; a.pm[2 * at + 1] = l; }
  }
}

// Depth of every node: the number of its ancestors (0 for roots and padding). One workgroup per tree.
__global__ __launch_bounds__(256) void tree_depths_kernel(const int32_t* __restrict__ parents, int T, int32_t* depths) {
  __shared__ uint32_t anc[TREE_MAX * TREE_WORDS];
  __shared__ int next[TREE_MAX];
  tree_ancestors(parents + (int64_t)blockIdx.x * T, T, anc, next);
  const int t = threadIdx.x, W = (T + 31) / 32;
  if (t >= T) return;
  int n = 0;
  for (int i = 0; i < W; ++i) n += __popc(anc[t * W + i]);
  depths[(int64_t)blockIdx.x * T + t] = n > 0 ? n - 1 : 0;
}

// The row tile is the least that holds a pair's rows, up to what a workgroup can; K and V are read once per tile.
// 16: the register walk (one sequence of 1000 rows, one node 9.8 us, with the LDS walk 13.1; 4 sequences of 2000, 32 K/V heads, 16
// nodes 28.3 and 32.4; 8 sequences of 4096, 4 nodes of 4 heads 28.0 and 29.1; over 16384 rows, where both are at HBM, 95 and 93).
// With 32 rows the register walk took 40 us where the LDS walk took 32. Head dimension 64 has half the work to a key, and 128 rows are
// enough. `share` is one round of workgroups, two to a CU for up to 64 rows and one above: with 1.5 to 4 rounds every case was
// slower.
TreePlan tree_plan(int dtype, int B, int T, int nq, int nk, int D, int max_len) {
  const int NR = nq / nk * T;
  TreePlan p;
  p.rows = NR <= 16 ? 16 : dtype == UNOK_F32 ? 32 : NR <= 64 ? 64 : NR <= 128 || D == 64 ? 128 : 256;
  p.rt = (NR + p.rows - 1) / p.rows;
  const int64_t share = (p.rows > 64 ? 256 : 512) / ((int64_t)nk * p.rt);   // one round of the workgroups that fit
  p.share = share > 1 ? (int)share : 1;
  p.ranges = max_len <= TREE_LEAST * TB ? B : B + p.share;
  return p;
}

template <typename E, int D> void launch_tree(const TreeAttn& a, const TreePlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)tree_blocks(a, plan));
  auto registers = [&](auto t) {
    constexpr int QT = decltype(t)::value;
    constexpr size_t lds = 4ull * 16 * QT * (D + 4) * sizeof(float);
    UNOK_SET_LDS_ONCE((tree_attn_kernel<E, D, QT>), lds);
    hipLaunchKernelGGL((tree_attn_kernel<E, D, QT>), grid, dim3(256), lds, st, a);
  };
  if (plan.rows == 16) {
    registers(std::integral_constant<int, 1>{});
  } else if constexpr (sizeof(E) == 4) {
    registers(std::integral_constant<int, 2>{});
  } else {
    auto tiles = [&](auto g) {
      constexpr int RG = decltype(g)::value;
      constexpr size_t lds = (RG == 2 ? 128ull : 256ull) * 2 * D * sizeof(bf16_t);   // all stages' keys
      UNOK_SET_LDS_ONCE((tree_attn_lds_kernel<D, RG>), lds);
      hipLaunchKernelGGL((tree_attn_lds_kernel<D, RG>), grid, dim3(RG == 2 ? 256 : 512), lds, st, a);
    };
    if (plan.rows == 64) tiles(std::integral_constant<int, 2>{});
    else if (plan.rows == 128) tiles(std::integral_constant<int, 4>{});
    else if constexpr (D == 128) tiles(std::integral_constant<int, 8>{});
  }
  launch_combine<E, D>(a, plan, st);
}

}  // namespace

UNOK_EXPORT int64_t unok_tree_attn_workspace(int dtype, int B, int T, int nq, int nk, int D, int max_len) {
  if (tree_sizes_ok("tree_attn", B, T, nq, nk, D, max_len)) return -1;
  if (B == 0 || T == 0) return 0;
  return plan_workspace(tree_plan(dtype, B, T, nq, nk, D, max_len), B, T, nq, D);
}

UNOK_EXPORT int unok_tree_attn(int dtype, int B, int T, int nq, int nk, int D, const void* q, int64_t ldq, const void* k,
                               int64_t k_batch, int64_t k_head, int64_t k_row, const void* v, int64_t v_batch, int64_t v_head,
                               int64_t v_row, int max_len, const int64_t* lengths, const int32_t* parents, int64_t ldp,
                               float scale, void* o, int64_t ldo, void* workspace, int64_t ws_bytes, void* stream) {
  int rc = tree_sizes_ok("tree_attn", B, T, nq, nk, D, max_len);
  if (rc) return rc;
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "tree_attn: bad dtype %d", dtype);
  if (B == 0 || T == 0) return 0;
  UNOK_REQUIRE(k && v, UNOK_EINVAL, "tree_attn: null operand");
  UNOK_REQUIRE(k_row >= D && v_row >= D && k_row < (1 << 23) && v_row < (1 << 23), UNOK_EINVAL,
               "tree_attn: row strides %lld and %lld must lie in [D, 2^23)", (long long)k_row, (long long)v_row);
  const int per16 = dtype == UNOK_BF16 ? 8 : 4;
  int64_t bits = ((uintptr_t)k | (uintptr_t)v) & 15;
  for (int64_t s : {k_batch, k_head, k_row, v_batch, v_head, v_row}) bits |= s % per16;
  UNOK_REQUIRE(bits == 0, UNOK_EALIGN, "tree_attn: operands and their strides must be multiples of 16 bytes");
  const TreePlan plan = tree_plan(dtype, B, T, nq, nk, D, max_len);
  TreeAttn a{};
  a.k = k; a.v = v;
  a.kb = k_batch; a.kh = k_head; a.kr = k_row; a.vb = v_batch; a.vh = v_head; a.vr = v_row;
  rc = tree_setup(a, "tree_attn", plan, dtype, B, T, nq, nk, D, q, ldq, max_len, lengths, parents, ldp, scale, o, ldo, workspace,
                  ws_bytes);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == UNOK_BF16) D == 128 ? launch_tree<bf16_t, 128>(a, plan, st) : launch_tree<bf16_t, 64>(a, plan, st);
  else D == 128 ? launch_tree<float, 128>(a, plan, st) : launch_tree<float, 64>(a, plan, st);
  return unok::check_launch("tree_attn");
}

UNOK_EXPORT int unok_tree_depths(int B, int T, const int32_t* parents, int32_t* depths, void* stream) {
  UNOK_REQUIRE(B >= 0 && T >= 0, UNOK_EINVAL, "tree_depths: B=%d T=%d", B, T);
  UNOK_REQUIRE(T <= TREE_MAX, UNOK_EUNSUPPORTED, "tree_depths: trees hold at most %d nodes (got %d)", TREE_MAX, T);
  if (B == 0 || T == 0) return 0;
  UNOK_REQUIRE(parents && depths, UNOK_EINVAL, "tree_depths: null operand");
  hipLaunchKernelGGL(tree_depths_kernel, dim3((unsigned)B), dim3(256), 0, (hipStream_t)stream, parents, T, depths);
  return unok::check_launch("tree_depths");
}
