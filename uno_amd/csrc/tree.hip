// Attention of a tree of drafted tokens over a KV cache.
//
// Node t of sequence b (parents[b, t] an earlier node, or -1 for a root, or less for padding) attends to the
// sequence's n = lengths[b] committed cache rows, its ancestors and itself; node a's K and V are cache row n + a.
// The queries of one (sequence, K/V head) pair, rep q heads x T nodes, are the rows of one product, so each
// cache row is read once per row tile.
//
// A workgroup takes one row tile of up to 64 query rows and one range of the keys; its four waves take
// key tiles in turn, each with its own running maximum and sum, and merge at the end: no barrier in the
// walk, and no LDS either. K and V go from memory into the registers that the MFMAs read:
//   S^T = K Q^T   the first operand wants 16 keys x 8 (fp32: 4) consecutive dims per lane: 16-byte loads of K;
//   O^T = V^T P^T the second operand is P^T as S^T's accumulators hold it (lane: query l % 16, four keys), and the first
//                 wants, per lane, one dim of eight (four) keys. With the accumulators' dims numbered so that lane
//                 m = l % 16 owns dims 8 m .. 8 m + 7 (4 m .. + 3 of each 64), those are 16-byte loads of V rows, and a
//                 bf16 pair of keys is one byte permute.
// The maximum that a wave's weights refer to moves only when a score exceeds it by 2^8 (the weights stay
// within fp32 and bf16 range), so that most tiles pass without a reduction across lanes. Scores,
// statistics and outputs are fp32; the weights of bf16 products are rounded to bf16, as their V is.
#include "common.h"
#include "../../include/unok.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr int TREE_MAX = 256, TREE_WORDS = TREE_MAX / 32;

struct TreeAttn {
  const void* q; int64_t ldq;                        // [B T, nq D]
  const void *k, *v;                                 // row (b, h, j) at b * s_b + h * s_h + j * s_r
  int64_t kb, kh, kr, vb, vh, vr;
  const int64_t* lengths;
  const int32_t* parents; int64_t ldp;               // row stride 0: one tree for all sequences
  int B, T, nq, nk, max_len, S, rt;
  void* o; int64_t ldo;
  float *po, *pm;                                    // S > 1: partial outputs [pair][S][rep T][D] and (max, sum) pairs
  float scale_log2;
};

// Keys [lo, hi) of range s of S ranges over `end` keys: ranges are whole steps of four waves' tiles of KT keys, at
// least two steps long, so a short sequence leaves the later ranges empty.
__device__ __forceinline__ int tree_step(int end, int S, int kt) {
  const int step = 4 * kt, steps = (end + step - 1) / step, per = (steps + S - 1) / S;
  return (per < 2 ? 2 : per) * step;
}

// Each node's ancestors (itself among them) as bits, by pointer doubling: thread t holds node t's set and how far
// its chain is followed. A padding node's set is empty; a parent that is no earlier node ends the chain. All
// threads of the workgroup call it.
__device__ __forceinline__ void tree_ancestors(const int32_t* parents, int T, uint32_t* anc, int* next) {
  const int t = threadIdx.x, W = (T + 31) / 32;
  bool real = false;
  int p = -1;
  uint32_t w[TREE_WORDS];
#pragma unroll
  for (int i = 0; i < TREE_WORDS; ++i) w[i] = 0;
  if (t < T) {
    p = parents[t];
    real = p >= -1;
    if (p >= t || p < 0 || parents[p] < -1) p = -1;
#pragma unroll
    for (int i = 0; i < TREE_WORDS; ++i) w[i] = real && t / 32 == i ? 1u << (t % 32) : 0u;
    for (int i = 0; i < W; ++i) anc[t * W + i] = real && t / 32 == i ? 1u << (t % 32) : 0u;
    next[t] = p;
  }
  __syncthreads();
  for (int hops = 1; hops < T; hops *= 2) {
    int far = -1;
    if (p >= 0) {
#pragma unroll
      for (int i = 0; i < TREE_WORDS; ++i)
        if (i < W) w[i] |= anc[p * W + i];
      far = next[p];
    }
    __syncthreads();
    if (p >= 0) {
#pragma unroll
      for (int i = 0; i < TREE_WORDS; ++i)
        if (i < W) anc[t * W + i] = w[i];
      next[t] = far;
      p = far;
    }
    __syncthreads();
  }
}

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
  template <typename F> static __device__ __forceinline__ void load_k(K& k, F row, int m, int g) {
#pragma unroll
    for (int a = 0; a < NS; ++a) {
      const bf16_t* r = row(16 * a + m);
#pragma unroll
      for (int s = 0; s < KS; ++s) k.f[a][s] = *(const bf16x8_t*)(r + 32 * s + 8 * g);
    }
  }
  template <typename F> static __device__ __forceinline__ void load_v(V& v, F row, int m, int g) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bf16_t* r = row(slot_key(j, g)) + NDT * m;
      if constexpr (VW == 4) { const u32x4_t u = *(const u32x4_t*)r; v.w[j][0] = u[0]; v.w[j][1] = u[1]; v.w[j][2] = u[2]; v.w[j][3] = u[3]; }
      else { const u32x2_t u = *(const u32x2_t*)r; v.w[j][0] = u[0]; v.w[j][1] = u[1]; }
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
  template <typename F> static __device__ __forceinline__ void load_k(K& k, F row, int m, int g) {
    const float* r = row(m);
#pragma unroll
    for (int s = 0; s < KS; ++s) k.f[0][s] = *(const f32x4_t*)(r + 16 * s + 4 * g);
  }
  template <typename F> static __device__ __forceinline__ void load_v(V& v, F row, int m, int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* r = row(slot_key(j, g)) + 4 * m;
#pragma unroll
      for (int jj = 0; jj < NJ; ++jj) v.w[j][jj] = *(const f32x4_t*)(r + 64 * jj);
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

template <typename E, int D, int QT>
__global__ __launch_bounds__(256, 1) void tree_attn_kernel(const TreeAttn a) {
  using Ops = TileOps<E, D>;
  constexpr int KT = Ops::KT, NS = Ops::NS, NDT = Ops::NDT, NP = 4 * NS, ROWS = 16 * QT, LDO = D + 4;
  extern __shared__ __attribute__((aligned(16))) float merge_o[];     // [4][ROWS][LDO]
  __shared__ float merge_ml[4][ROWS][2];
  __shared__ uint32_t anc[TREE_MAX * TREE_WORDS];
  __shared__ int next[TREE_MAX];

  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int pairs = a.B * a.nk, rep = a.nq / a.nk, T = a.T, NR = rep * T;
  const int lin = xcd_remap(blockIdx.x, pairs * a.S * a.rt);
  const int tile = lin % a.rt, pair = lin / a.rt % pairs, split = lin / (a.rt * pairs);
  const int b = pair / a.nk, h = pair % a.nk;
  const int64_t len = a.lengths[b];
  const int n = (int)(len < 0 ? 0 : len < a.max_len ? len : a.max_len);
  const int end = n + T < a.max_len ? n + T : a.max_len;
  const int per = tree_step(end, a.S, KT);
  const int lo = split * per, hi = lo + per < end ? lo + per : end;
  if (lo >= end) return;

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
  {
    auto load = [&](typename Ops::K& k, typename Ops::V& v, int key0) {
      Ops::load_k(k, [&](int j) { return kbase + (int64_t)(key0 + j) * a.kr; }, m, g);
      Ops::load_v(v, [&](int j) { return vbase + (int64_t)(key0 + j) * a.vr; }, m, g);
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
  }
  // Tiles with tree rows. Keys at or past the end read the last row, at weight 0.
#pragma unroll 1
  for (; key < hi; key += 4 * KT) {
    typename Ops::K k;
    typename Ops::V v;
    Ops::load_k(k, [&](int j) { const int r = key + j; return kbase + (int64_t)(r < end ? r : end - 1) * a.kr; }, m, g);
    Ops::load_v(v, [&](int j) { const int r = key + j; return vbase + (int64_t)(r < end ? r : end - 1) * a.vr; }, m, g);
    float p[QT][NP];
    scores(k, p);
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const int r = key + Ops::slot_key(j, g), t = r - n;
        if (t >= 0 && (r >= hi || !(anc[node[i] * W + t / 32] >> (t % 32) & 1))) p[i][j] = -INFINITY;
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
              const bool seen = t < 0 || (anc[node[i] * W + t / 32] >> (t % 32) & 1);
              if (seen && !(fabsf(x) < INFINITY)) o[i][c][e] += ps[(16 * i + m) * (KT + 1) + j] * x;
            }
          }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }

  // merge: every wave's outputs relative to the common maximum, summed in wave order
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] += __shfl_xor(l[i], 16, 64);
    l[i] += __shfl_xor(l[i], 32, 64);
    if (g == 0) { merge_ml[wid][16 * i + m][0] = mref[i]; merge_ml[wid][16 * i + m][1] = l[i]; }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = 16 * i + m;
    float top = merge_ml[0][r][0];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, merge_ml[w][r][0]);
    const float f = mref[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref[i] - top);
    float* dst = merge_o + (wid * ROWS + r) * LDO;
#pragma unroll
    for (int c = 0; c < NDT; c += 4)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(f32x4_t*)(dst + Ops::dim(c, e, g)) = f32x4_t{o[i][c][e] * f, o[i][c + 1][e] * f, o[i][c + 2][e] * f, o[i][c + 3][e] * f};
  }
  __syncthreads();
  const bool whole = per >= end;                         // this range is the only one
  for (int it = threadIdx.x; it < ROWS * (D / 4); it += 256) {
    const int rl = it / (D / 4), d = it % (D / 4) * 4, r = tile * ROWS + rl;
    if (r >= NR) continue;
    float top = merge_ml[0][rl][0], sum = 0.f;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, merge_ml[w][rl][0]);
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = merge_ml[w][rl][0];
      sum += mw == -INFINITY ? 0.f : merge_ml[w][rl][1] * __builtin_amdgcn_exp2f(mw - top);
      x += *(const f32x4_t*)(merge_o + (w * ROWS + rl) * LDO + d);
    }
    if (whole) {
      const int t = r % T;
      const bool none = sum == 0.f || a.parents[b * a.ldp + t] < -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : x[e] / sum;
      E* dst = (E*)a.o + ((int64_t)b * T + t) * a.ldo + ((int64_t)h * rep + r / T) * D + d;
      if constexpr (sizeof(E) == 2) *(u32x2_t*)dst = u32x2_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
      else *(f32x4_t*)dst = x;
    } else {
      const int64_t at = ((int64_t)pair * a.S + split) * NR + r;
      *(f32x4_t*)(a.po + at * D + d) = x;
      if (d == 0) { a.pm[2 * at] = top; a.pm[2 * at + 1] = sum; }
    }
  }
}

// The ranges of each query row merged: one thread per four dims. Sequences short enough for one range were written by
// the kernel above.
template <typename E, int D>
__global__ __launch_bounds__(256) void tree_combine_kernel(const TreeAttn a, int kt) {
  const int rep = a.nq / a.nk, NR = rep * a.T;
  const int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = it / (D / 4);
  const int d = (int)(it % (D / 4)) * 4;
  if (row >= (int64_t)a.B * a.nk * NR) return;
  const int pair = (int)(row / NR), r = (int)(row % NR), b = pair / a.nk, h = pair % a.nk, t = r % a.T;
  const int64_t len = a.lengths[b];
  const int n = (int)(len < 0 ? 0 : len < a.max_len ? len : a.max_len);
  const int end = n + a.T < a.max_len ? n + a.T : a.max_len;
  const int per = tree_step(end, a.S, kt), ranges = (end + per - 1) / per;
  if (ranges == 1) return;
  float top = -INFINITY, sum = 0.f;
  for (int s = 0; s < ranges; ++s) top = fmaxf(top, a.pm[2 * (((int64_t)pair * a.S + s) * NR + r)]);
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < ranges; ++s) {
    const int64_t at = ((int64_t)pair * a.S + s) * NR + r;
    const float ms = a.pm[2 * at], f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - top);
    sum += a.pm[2 * at + 1] * f;
    x += *(const f32x4_t*)(a.po + at * D + d) * f;
  }
  const bool none = sum == 0.f || a.parents[b * a.ldp + t] < -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : x[e] / sum;
  E* dst = (E*)a.o + ((int64_t)b * a.T + t) * a.ldo + ((int64_t)h * rep + r / a.T) * D + d;
  if constexpr (sizeof(E) == 2) *(u32x2_t*)dst = u32x2_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(f32x4_t*)dst = x;
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

int tree_qt(int NR) { return NR <= 16 ? 1 : NR <= 32 ? 2 : 4; }

int tree_splits(int B, int T, int nq, int nk, int max_len) {
  const int NR = nq / nk * T, rows = 16 * tree_qt(NR);
  const int64_t wgs = (int64_t)B * nk * ((NR + rows - 1) / rows);
  const int64_t want = (512 + wgs - 1) / wgs, most = (max_len + 255) / 256;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

int tree_sizes_ok(int B, int T, int nq, int nk, int D, int max_len) {
  UNOK_REQUIRE(B >= 0 && T >= 0 && nq > 0 && nk > 0 && nq % nk == 0 && max_len >= 1, UNOK_EINVAL,
               "tree_attn: B=%d T=%d nq=%d nk=%d max_len=%d", B, T, nq, nk, max_len);
  UNOK_REQUIRE(T <= TREE_MAX, UNOK_EUNSUPPORTED, "tree_attn: trees hold at most %d nodes (got %d)", TREE_MAX, T);
  UNOK_REQUIRE(D == 64 || D == 128, UNOK_EINVAL, "tree_attn: head dim %d not in {64,128}", D);
  UNOK_REQUIRE((int64_t)B * nq * (T > 0 ? T : 1) < (1ll << 24) && max_len < (1 << 30), UNOK_EINVAL,
               "tree_attn: B=%d T=%d nq=%d max_len=%d exceed the row layout", B, T, nq, max_len);
  return 0;
}

}  // namespace

UNOK_EXPORT int64_t unok_tree_attn_workspace(int B, int T, int nq, int nk, int D, int max_len) {
  if (tree_sizes_ok(B, T, nq, nk, D, max_len)) return -1;
  if (B == 0 || T == 0) return 0;
  const int64_t S = tree_splits(B, T, nq, nk, max_len);
  return S == 1 ? 0 : S * B * nq * T * (D + 2) * (int64_t)sizeof(float);
}

UNOK_EXPORT int unok_tree_attn(int dtype, int B, int T, int nq, int nk, int D, const void* q, int64_t ldq, const void* k,
                               int64_t k_batch, int64_t k_head, int64_t k_row, const void* v, int64_t v_batch, int64_t v_head,
                               int64_t v_row, int max_len, const int64_t* lengths, const int32_t* parents, int64_t ldp,
                               float scale, void* o, int64_t ldo, void* workspace, int64_t ws_bytes, void* stream) {
  int rc = tree_sizes_ok(B, T, nq, nk, D, max_len);
  if (rc) return rc;
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "tree_attn: bad dtype %d", dtype);
  if (B == 0 || T == 0) return 0;
  UNOK_REQUIRE(q && k && v && lengths && parents && o, UNOK_EINVAL, "tree_attn: null operand");
  UNOK_REQUIRE(ldp == 0 || ldp >= T, UNOK_EINVAL, "tree_attn: parents' row stride %lld for %d nodes", (long long)ldp, T);
  const int per16 = dtype == UNOK_BF16 ? 8 : 4;
  int64_t bits = ((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) & 15;
  for (int64_t s : {ldq, k_batch, k_head, k_row, v_batch, v_head, v_row, ldo}) bits |= s % per16;
  UNOK_REQUIRE(bits == 0, UNOK_EALIGN, "tree_attn: operands and their strides must be multiples of 16 bytes");
  const int64_t need = unok_tree_attn_workspace(B, T, nq, nk, D, max_len);
  UNOK_REQUIRE(need == 0 || (workspace && ws_bytes >= need && ((uintptr_t)workspace & 15) == 0), UNOK_EINVAL,
               "tree_attn: workspace of %lld bytes (16-byte aligned) required, got %lld", (long long)need, (long long)ws_bytes);
  const int NR = nq / nk * T, qt = tree_qt(NR);
  TreeAttn a{};
  a.q = q; a.ldq = ldq; a.k = k; a.v = v;
  a.kb = k_batch; a.kh = k_head; a.kr = k_row; a.vb = v_batch; a.vh = v_head; a.vr = v_row;
  a.lengths = lengths; a.parents = parents; a.ldp = ldp;
  a.B = B; a.T = T; a.nq = nq; a.nk = nk; a.max_len = max_len;
  a.S = tree_splits(B, T, nq, nk, max_len);
  a.rt = (NR + 16 * qt - 1) / (16 * qt);
  a.o = o; a.ldo = ldo;
  a.po = (float*)workspace;
  a.pm = a.po + (int64_t)a.S * B * nq * T * D;
  a.scale_log2 = scale * 1.4426950408889634f;
  const int64_t nb = (int64_t)B * nk * a.S * a.rt;
  UNOK_REQUIRE(nb < (1ll << 31), UNOK_EINVAL, "tree_attn: grid too large");
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto e, auto d, auto t) {
    using E = decltype(e);
    constexpr int DD = decltype(d)::value, QT = decltype(t)::value;
    constexpr size_t lds = 4ull * 16 * QT * (DD + 4) * sizeof(float);
    UNOK_SET_LDS_ONCE((tree_attn_kernel<E, DD, QT>), lds);
    hipLaunchKernelGGL((tree_attn_kernel<E, DD, QT>), dim3((unsigned)nb), dim3(256), lds, st, a);
    if (a.S > 1) {
      const int64_t items = (int64_t)B * nq * T * (DD / 4);
      hipLaunchKernelGGL((tree_combine_kernel<E, DD>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, st, a,
                         TileOps<E, DD>::KT);
    }
  };
  auto by_rows = [&](auto e, auto d) {
    if (qt == 1) go(e, d, std::integral_constant<int, 1>{});
    else if (qt == 2) go(e, d, std::integral_constant<int, 2>{});
    else go(e, d, std::integral_constant<int, 4>{});
  };
  auto by_dim = [&](auto e) {
    if (D == 128) by_rows(e, std::integral_constant<int, 128>{});
    else by_rows(e, std::integral_constant<int, 64>{});
  };
  if (dtype == UNOK_BF16) by_dim(bf16_t{});
  else by_dim(float{});
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
