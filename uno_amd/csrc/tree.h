// What the tree attentions over 16/32-bit and 4-bit caches share: how the keys are divided among workgroups, the trees' masks, the merge
// of a workgroup's waves and of a sequence's ranges, and the host's checks.
#pragma once
#include "common.h"
#include "lds_tile.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int TREE_MAX = 256, TREE_WORDS = TREE_MAX / 32;

struct TreeAttn {
  const void* q; int64_t ldq;                        // [B T, nq D]
  const void *k, *v;                                 // row (b, h, j) at b * s_b + h * s_h + j * s_r
  int64_t kb, kh, kr, vb, vh, vr;
  const uint8_t *ks, *vs;                            // 4-bit caches: their scales (k and v then hold the codes)
  const int64_t* lengths;
  const int32_t* parents; int64_t ldp;               // row stride 0: one tree for all sequences
  int B, T, nq, nk, max_len, rt, share;              // row tiles per (sequence, K/V head); ranges to make of all keys
  void* o; int64_t ldo;
  int2* table;                                       // each sequence's (first range, ranges); null: never more than one
  float *po, *pm;                                    // partial outputs [range][nk][rep T][D], (max, sum) pairs
  float scale_log2;
  // The LDS walk masks and compares scores before it scales them, so its scale has to be positive: another one's sign, or its
  // 0, goes into the queries (exact in bf16).
  float walk_scale, q_factor;
};

// How the keys are divided: in ranges of equal size, whatever the sequences' lengths, so that workgroups end
// together. A range is at most c blocks of TB keys, c the least from TREE_LEAST on for which all sequences' keys make about
// `share` ranges; a sequence's ranges are evened out, and numbered after those of the sequences before it. Sequences of three
// to eight blocks on average are cut into single ones while these are no more than half a round of workgroups: one sequence of
// 1000 rows, one node 10.1 us (in ranges of 256 keys 11.1), fp32 37 nodes of three of 901 rows 13.7 (16.7). Longer ones would pay
// for it in the merge (one of 1150 rows 11.4 and 10.6, of 4096 15.7 and 13.1), shorter ones need none at all (130 rows 9.0 and
// 8.0), and so would more of them (16 nodes, 8 sequences of 1000 rows 23.9 and 21.5, of 500 rows 23.1 and 19.9; of four of 500
// rows, a third of a round, 18.0 and 18.2).
constexpr int TB = 128, TREE_LEAST = 2;

struct Range { int b, n, end, first, count, lo, hi; bool past; };   // sequence, its lengths, its ranges, this range's keys

// Keys and values well above the memory-side cache's 256 MB are read past the caches (8 sequences, 8 heads of 128 bf16 over
// 16384 rows, 537 MB: 16 nodes 115 -> 103 us, one node 101 -> 94). Below, a part is found there: over 4096 rows (134 MB) 16
// nodes take 33 us, 39 with such loads, and 4 nodes in fp32 (269 MB) 53 and 63.
constexpr int64_t TREE_PAST = 384ll << 20;

__device__ __forceinline__ int tree_end(const TreeAttn& a, int b, int& n) {
  const int64_t len = a.lengths[b];
  n = (int)(len < 0 ? 0 : len < a.max_len ? len : a.max_len);
  return n + a.T < a.max_len ? n + a.T : a.max_len;
}

// A workgroup's row tile, K/V head and range. Workgroups go round the 8 XCDs: eight in a row take different (range,
// head) pairs, and the row tiles of a pair follow on the same XCD, where they share its L2. (With neighbouring pairs on
// one XCD instead, streams that are whole cache slots apart meet in the same memory channels: with the walk of
// that time, 8 sequences of 4096 rows 46 us, this way 37; 16384 rows 141 and 117.)
__device__ __forceinline__ void tree_place(const TreeAttn& a, int& tile, int& h, int& id) {
  const int x = blockIdx.x, unit = x / (8 * a.rt) * 8 + x % 8;
  tile = x / 8 % a.rt;
  h = unit % a.nk;
  id = unit / a.nk;
}

// Notes a sequence's ranges for the kernel that merges them.
__device__ __forceinline__ void tree_note(const TreeAttn& a, const Range& r, int id, int h, int tile) {
  if (a.table && id == r.first && h == 0 && tile == 0 && threadIdx.x == 0) a.table[r.b] = make_int2(r.first, r.count);
}

// Sum over lanes 0 .. l in lane l, by data-parallel moves within the wave.
__device__ __forceinline__ int wave_scan(int v) {
#define TREE_ADD(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xf, false)
  TREE_ADD(0x111, 0xf);                                  // row_shr 1, 2, 4, 8
  TREE_ADD(0x112, 0xf);
  TREE_ADD(0x114, 0xf);
  TREE_ADD(0x118, 0xf);
  TREE_ADD(0x142, 0xa);                                  // row_bcast 15 into rows 1 and 3
  TREE_ADD(0x143, 0xc);                                  // row_bcast 31 into rows 2 and 3
#undef TREE_ADD
  return v;
}

// Finds range `id`. Every wave of the workgroup does it for itself.
__device__ __forceinline__ Range tree_range(const TreeAttn& a, int id, int row_bytes) {
  const int lane = threadIdx.x & 63;
  int total = 0, n = 0, end = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    end = b0 + lane < a.B ? tree_end(a, b0 + lane, n) : 0;
    total += __builtin_amdgcn_readlane(wave_scan((end + TB - 1) / TB), 63);
  }
  const bool single = total > 2 * a.B && total <= min(8 * a.B, a.share / 2);
  int c = max((int)(((uint32_t)total + a.share - 1) / (uint32_t)a.share), single ? 1 : TREE_LEAST);
  // sequences end inside ranges: larger ones until no more than `share` are left (one round of workgroups)
  if (a.B <= 64)
    for (int i = 0; i < 12; ++i) {
      const int count = (int)((uint32_t)((end + TB - 1) / TB + c - 1) / (uint32_t)c);
      if (__builtin_amdgcn_readlane(wave_scan(count), 63) <= max(a.share, a.B)) break;
      c += (c + 15) / 16;
    }
  Range r{-1, 0, 0, 0, 0, 0, 0, (int64_t)total * TB * a.nk * row_bytes * 2 > TREE_PAST};
  int first = 0;
  for (int b0 = 0; b0 < a.B && r.b < 0; b0 += 64) {
    if (a.B > 64) end = b0 + lane < a.B ? tree_end(a, b0 + lane, n) : 0;
    const int count = (int)((uint32_t)((end + TB - 1) / TB + c - 1) / (uint32_t)c);
    const int upto = wave_scan(count);                   // ranges of the sequences up to this lane's
    const uint64_t hit = __ballot(id < first + upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      r.b = b0 + l;
      r.n = __builtin_amdgcn_readlane(n, l);
      r.end = __builtin_amdgcn_readlane(end, l);
      r.count = __builtin_amdgcn_readlane(count, l);
      r.first = first + __builtin_amdgcn_readlane(upto, l) - r.count;
    }
    first += __builtin_amdgcn_readlane(upto, 63);
  }
  if (r.b >= 0) {
    const int blocks = (r.end + TB - 1) / TB, per = (int)((uint32_t)(blocks + r.count - 1) / (uint32_t)r.count);
    r.lo = (id - r.first) * per * TB;
    r.hi = min(r.lo + per * TB, r.end);
  }
  return r;
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
    next[t] = p;
  }
  __syncthreads();
  const bool cut = t < T && (p >= t || p < 0 || next[p] < -1);
  __syncthreads();
  if (t < T) {
    if (cut) p = -1;
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

// Whether node t is among the ancestors of `node` (t outside the tree: some bit or other; no branch, so that it can stand in a
// select).
__device__ __forceinline__ bool tree_sees(const uint32_t* anc, int node, int W, int t) {
  const int i = min(max(t >> 5, 0), W - 1);
  return anc[node * W + i] >> (t & 31) & 1;
}

template <bool PAST, typename T> __device__ __forceinline__ T tree_load(const T* p) {
  if constexpr (PAST) return __builtin_nontemporal_load(p);
  else return *p;
}

// A workgroup's end, walks in which a query is a column of the wave: every wave's outputs relative to the common maximum, summed in
// wave order, and written as a range's part or, where it is the only one, as the result. o[i][c][e] is dim dim(c, e, g) of query row 16 i
// + m, four consecutive c four consecutive dims. LDS: [4][16 QT][D + 4] floats, [4][16 QT][2], and whether each row is padding.
template <typename E, int D, int QT, typename F>
__device__ __forceinline__ void tree_merge(const TreeAttn& a, const Range& range, int tile, int h, int id, const f32x4_t (&o)[QT][D / 16],
                                           const float (&mref)[QT], float (&l)[QT], float* merge_o, float (*merge_ml)[16 * QT][2],
                                           const bool* merge_pad, F dim) {
  constexpr int NDT = D / 16, ROWS = 16 * QT, LDO = D + 4;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, m = lane & 15, g = lane >> 4;
  const int rep = a.nq / a.nk, T = a.T, NR = rep * T, b = range.b;
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
        *(f32x4_t*)(dst + dim(c, e, g)) = f32x4_t{o[i][c][e] * f, o[i][c + 1][e] * f, o[i][c + 2][e] * f, o[i][c + 3][e] * f};
  }
  __syncthreads();
  const bool whole = range.count == 1;
  for (int it = threadIdx.x; it < ROWS * (D / 4); it += 256) {
    const int rl = it / (D / 4), d = it % (D / 4) * 4, r = tile * ROWS + rl;
    if (r >= NR) continue;
    float top = merge_ml[0][rl][0], sum = 0.f;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, merge_ml[w][rl][0]);
    f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = merge_ml[w][rl][0], lw = merge_ml[w][rl][1];
      sum += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - top);   // no maximum: 0, or NaN from NaN scores alone
      x += *(const f32x4_t*)(merge_o + (w * ROWS + rl) * LDO + d);
    }
    if (whole) {
      const int t = r % T;
      const bool none = sum == 0.f || merge_pad[rl];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : x[e] / sum;
      E* dst = (E*)a.o + ((int64_t)b * T + t) * a.ldo + ((int64_t)h * rep + r / T) * D + d;
      if constexpr (sizeof(E) == 2) *(u32x2_t*)dst = u32x2_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
      else *(f32x4_t*)dst = x;
    } else {
      const int64_t at = ((int64_t)id * a.nk + h) * NR + r;
      *(f32x4_t*)(a.po + at * D + d) = x;
      if (d == 0) { a.pm[2 * at] = top; a.pm[2 * at + 1] = sum; }
    }
  }
}

// The ranges of each query row merged: one thread per four dims, grid (.., sequences). Sequences of one range were
// written by the kernels above. Bound by latency when ranges are many, so eight are read at a time (one at a time: one sequence of
// 32768 rows 58 us in place of 34, 8 of 4096 rows with 16 nodes 35 in place of 33), and three where that is all there are.
template <typename E, int D>
__global__ __launch_bounds__(256) void tree_combine_kernel(const TreeAttn a) {
  const int b = blockIdx.y, rep = a.nq / a.nk, NR = rep * a.T;
  const int2 range = a.table[b];                       // first, count
  if (range.y <= 1) return;
  const int it = blockIdx.x * 256 + threadIdx.x, row = it / (D / 4), d = it % (D / 4) * 4;
  if (row >= a.nk * NR) return;
  const int h = row / NR, r = row % NR, t = r % a.T;
  const int64_t at0 = (int64_t)range.x * a.nk * NR + row, step = (int64_t)a.nk * NR;
  float top = -INFINITY, sum = 0.f;
  f32x4_t x = {0.f, 0.f, 0.f, 0.f};
  auto merge = [&](int s0, auto n) {                     // the next n ranges, in flight together
    constexpr int N = decltype(n)::value;
    f32x4_t v[N];
    float2 ml[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t at = at0 + min(s0 + i, range.y - 1) * step;
      v[i] = *(const f32x4_t*)(a.po + at * D + d);
      ml[i] = *(const float2*)(a.pm + 2 * at);
    }
    float to = top;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (s0 + i >= range.y) ml[i] = make_float2(-INFINITY, 0.f);
      to = fmaxf(to, ml[i].x);
    }
    const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - to);   // (without a maximum x is 0, sum 0 or NaN)
    top = to;
    sum *= f;
    x *= f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (ml[i].x == -INFINITY) { sum += ml[i].y; continue; }   // 0, or NaN from NaN scores alone
      const float w = __builtin_amdgcn_exp2f(ml[i].x - top);
      sum += ml[i].y * w;
      x += v[i] * w;
    }
  };
  if (range.y <= 3) merge(0, std::integral_constant<int, 3>{});
  else
    for (int s0 = 0; s0 < range.y; s0 += 8) merge(s0, std::integral_constant<int, 8>{});
  const bool none = sum == 0.f || a.parents[b * a.ldp + t] < -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = none ? 0.f : x[e] / sum;
  E* dst = (E*)a.o + ((int64_t)b * a.T + t) * a.ldo + ((int64_t)h * rep + r / a.T) * D + d;
  if constexpr (sizeof(E) == 2) *(u32x2_t*)dst = u32x2_t{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(f32x4_t*)dst = x;
}

struct TreePlan { int rows, rt, share; int64_t ranges; };   // rows per row tile; most ranges of all sequences

int tree_sizes_ok(const char* what, int B, int T, int nq, int nk, int D, int max_len) {
  UNOK_REQUIRE(B >= 0 && T >= 0 && nq > 0 && nk > 0 && nq % nk == 0 && max_len >= 1, UNOK_EINVAL,
               "%s: B=%d T=%d nq=%d nk=%d max_len=%d", what, B, T, nq, nk, max_len);
  UNOK_REQUIRE(T <= TREE_MAX, UNOK_EUNSUPPORTED, "%s: trees hold at most %d nodes (got %d)", what, TREE_MAX, T);
  UNOK_REQUIRE(D == 64 || D == 128, UNOK_EINVAL, "%s: head dim %d not in {64,128}", what, D);
  UNOK_REQUIRE((int64_t)B * nq * (T > 0 ? T : 1) < (1ll << 24) && max_len < (1 << 30) && B * (max_len / TB + 1ll) < (1ll << 30),
               UNOK_EINVAL, "%s: B=%d T=%d nq=%d max_len=%d exceed the row layout", what, B, T, nq, max_len);
  return 0;
}

// Workgroups of a walk: (range, head) units in eights, times the row tiles (see tree_place).
int64_t tree_blocks(const TreeAttn& a, const TreePlan& p) { return (p.ranges * a.nk + 7) / 8 * 8 * p.rt; }

template <typename E, int D> void launch_combine(const TreeAttn& a, const TreePlan& plan, hipStream_t st) {
  if (plan.ranges > a.B)
    hipLaunchKernelGGL((tree_combine_kernel<E, D>), dim3((unsigned)(((int64_t)a.nq * a.T * (D / 4) + 255) / 256), (unsigned)a.B),
                       dim3(256), 0, st, a);
}

int64_t plan_workspace(const TreePlan& p, int B, int T, int nq, int D) {
  return p.ranges == B ? 0 : p.ranges * nq * T * (D + 2) * (int64_t)sizeof(float) + B * (int64_t)sizeof(int2);
}

// What both cache formats check and fill in: queries, trees, outputs, workspace. `what` names the entry point.
int tree_setup(TreeAttn& a, const char* what, const TreePlan& plan, int dtype, int B, int T, int nq, int nk, int D, const void* q,
               int64_t ldq, int max_len, const int64_t* lengths, const int32_t* parents, int64_t ldp, float scale, void* o,
               int64_t ldo, void* workspace, int64_t ws_bytes) {
  UNOK_REQUIRE(q && lengths && parents && o, UNOK_EINVAL, "%s: null operand", what);
  UNOK_REQUIRE(ldp == 0 || ldp >= T, UNOK_EINVAL, "%s: parents' row stride %lld for %d nodes", what, (long long)ldp, T);
  const int64_t es = dtype == UNOK_BF16 ? 2 : 4, width = (int64_t)nq * D, rows = (int64_t)B * T;
  UNOK_REQUIRE(rows == 1 || (ldq >= width && ldo >= width), UNOK_EINVAL, "%s: rows of %lld elements, ldq=%lld ldo=%lld", what,
               (long long)width, (long long)ldq, (long long)ldo);
  UNOK_REQUIRE(!unok::rows_overlap(q, ldq * es, o, ldo * es, rows, width * es), UNOK_EINVAL,
               "%s: the output overlaps the queries", what);
  const float scale_log2 = scale * 1.4426950408889634f;
  UNOK_REQUIRE(scale_log2 - scale_log2 == 0.f, UNOK_EINVAL, "%s: scale %g must be finite", what, (double)scale);
  const int per16 = dtype == UNOK_BF16 ? 8 : 4;
  UNOK_REQUIRE((((uintptr_t)q | (uintptr_t)o) & 15) == 0 && ldq % per16 == 0 && ldo % per16 == 0, UNOK_EALIGN,
               "%s: queries and outputs and their strides must be multiples of 16 bytes", what);
  const int64_t need = plan_workspace(plan, B, T, nq, D);
  UNOK_REQUIRE(need == 0 || (workspace && ws_bytes >= need && ((uintptr_t)workspace & 15) == 0), UNOK_EINVAL,
               "%s: workspace of %lld bytes (16-byte aligned) required, got %lld", what, (long long)need, (long long)ws_bytes);
  a.q = q; a.ldq = ldq;
  a.lengths = lengths; a.parents = parents; a.ldp = ldp;
  a.B = B; a.T = T; a.nq = nq; a.nk = nk; a.max_len = max_len;
  a.rt = plan.rt;
  a.share = plan.share;
  a.o = o; a.ldo = ldo;
  a.po = (float*)workspace;
  a.pm = a.po + plan.ranges * nq * T * D;
  a.table = plan.ranges > B ? (int2*)(a.pm + plan.ranges * nq * T * 2) : nullptr;
  a.scale_log2 = scale_log2;
  a.walk_scale = scale_log2 > 0.f ? scale_log2 : scale_log2 < 0.f ? -scale_log2 : 1.f;
  a.q_factor = scale_log2 > 0.f ? 1.f : scale_log2 < 0.f ? -1.f : 0.f;
  UNOK_REQUIRE(tree_blocks(a, plan) < (1ll << 31) && B < 65536, UNOK_EINVAL, "%s: grid too large", what);
  return 0;
}

}  // namespace
