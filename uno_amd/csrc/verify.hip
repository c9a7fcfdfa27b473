// Verification of drafted tokens against the target's logits from given random numbers.
//
// A token is drawn by the inverse distribution function: the lowest index at which the running sum of the weights
// exp((z - max z) / T) exceeds u times their sum. Of a vocabulary's 150 thousand borders between tokens some lie within an fp32
// exponential's error (1e-7) of any u: with such weights about one token in 300 would be another one than the logits say, and
// depend on the order of the sums. The weights and all sums are therefore fp64, with errors around 1e-15, and the vector units form
// them about as fast as HBM delivers the logits (64 fused multiply-adds per clock and CU, some 20 to a weight).
//
// The logits are read once, in chunks of CHUNK columns, one wave each: a chunk's largest logit, the sum of its weights relative to
// that, and the column of the largest. Everything else works on these parts, and on one chunk to a drawn token.
#include "common.h"
#include "../../include/unok.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int CHUNK = 2048, VERIFY_NODES = 256;
constexpr double LOG2E = 1.4426950408889634, LOWEST = -700.0 * LOG2E;   // weights below e^-700 are 0
constexpr double LEAST = 0x1p-40;                                       // of max(p - q, 0) in all; below, p itself is drawn from

// One chunk of a row: its largest logit (NaN: the row has a NaN or +inf here), its column, the sum of the weights relative to it.
struct Part { float m; int arg; double s; };

struct Verify {
  const void *z, *y; int64_t ldz, ldy;                // target rows; the drafter's rows (null: none)
  const int64_t* tokens;
  const int32_t* parents; int64_t ldp;
  const int64_t* counts;
  const float* u;
  const float* temps; float temp;                     // per sequence, or one
  int B, T, V, nch;                                   // T: nodes of a tree, or drafted tokens
  Part* parts;                                        // [target rows, then the drafter's][nch]
  uint32_t* arrived;                                  // of a tree's rows, drawn; 0 before
  int64_t *nodes, *out_counts, *out_token;
};

// 2^x at x = d c, -1022 <= x <= 0, of N numbers side by side: 2^n (1 + r q(r)), r = x - n in [-1/2, 1/2], q the polynomial through
// (2^r - 1) / r at eight Chebyshev points. Relative error 2.1e-12, of both signs in turn (at 150 thousand columns it moves less than
// one token in 10^6; another degree, 3.7e-14, takes 5% more time); exactly 1 at 0. n is the low half of x + 1.5 2^52.
template <int N> __device__ __forceinline__ void exp2_64(double (&d)[N], double c) {
  constexpr double ROUND = 0x1.8p52;
  constexpr double Q[8] = {0x1.62e42fef9cc69p-1, 0x1.ebfbdff82a734p-3, 0x1.c6b08da70cce3p-5, 0x1.3b2ab70ad2565p-7,
                           0x1.5d877598350dep-10, 0x1.4308c7183d6a2p-13, 0x1.00c0e4e15189cp-16, 0x1.63b2d7971923fp-20};
  double t[N], r[N], q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = fma(d[i], c, ROUND);
    r[i] = fma(d[i], c, ROUND - t[i]);
    q[i] = Q[7];
  }
#pragma unroll
  for (int k = 6; k >= 0; --k)
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = fma(q[i], r[i], Q[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double p = fma(q[i], r[i], 1.0);
    d[i] = __hiloint2double(__double2hiint(p) + __double2loint(t[i]) * (1 << 20), __double2loint(p));
  }
}
// The weights of z relative to m, c = log2(e) / T.
template <int N> __device__ __forceinline__ void weights(const float (&z)[N], double m, double c, double (&w)[N]) {
  bool some[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = (double)z[i] - m;
    some[i] = w[i] * c >= LOWEST;
    w[i] = some[i] ? w[i] : 0.0;
  }
  exp2_64<N>(w, c);
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = some[i] ? w[i] : 0.0;
}
__device__ __forceinline__ double weight(float z, double m, double c) {
  const float a[1] = {z};
  double w[1];
  weights<1>(a, m, c, w);
  return w[0];
}

__device__ __forceinline__ double rate(const Verify& a, int b) {        // log2(e) / T; 0: the largest logit is taken
  const float t = a.temps ? a.temps[b] : a.temp;
  return t > 0.f ? fmax(LOG2E / (double)t, 1e-300) : 0.0;   // (an infinite T: all finite logits alike)
}
// The random number at i; below 0 it counts as 0 (and from 1 on takes the last token with a weight).
__device__ __forceinline__ double random_at(const Verify& a, int64_t i) {
  const float u = a.u[i];
  return u < 0.f ? 0.0 : (double)u;
}
__device__ __forceinline__ int drafted(const Verify& a, int b) {
  if (!a.counts) return a.T;
  const int64_t n = a.counts[b];
  return (int)(n < 0 ? 0 : n < a.T ? n : a.T);
}

template <typename T> __device__ __forceinline__ float at(const T* row, int j) { return Elem<T>::load(row + j); }

// A row of V elements as `head` elements up to the first 16-byte boundary, vectors, and the rest. Chunk c holds vectors
// [c VPC, (c + 1) VPC), the first chunk the head too, the last one the rest.
template <typename T> struct Chunks {
  static constexpr int VN = 16 / (int)sizeof(T), VPC = CHUNK / VN;
  int head, nv, V, nch;
  __device__ __forceinline__ Chunks(const T* row, int V_, int nch_) : V(V_), nch(nch_) {
    head = (int)(((16 - ((uintptr_t)row & 15)) & 15) / sizeof(T));
    head = head < V ? head : V;
    nv = (V - head) / VN;
  }
  __device__ __forceinline__ int tail() const { return head + nv * VN; }
  __device__ __forceinline__ int lo(int c) const { return c == 0 ? 0 : min(head + c * CHUNK, tail()); }
  __device__ __forceinline__ int hi(int c) const { return c == nch - 1 ? V : min(head + (c + 1) * CHUNK, tail()); }
};

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return v;
}
// The parts of one chunk of a row, by one wave.
template <typename T> __device__ __forceinline__ Part chunk_part(const T* row, int V, int nch, int chunk, double c) {
  using C = Chunks<T>;
  constexpr int NL = C::VPC / 64;
  const C ch(row, V, nch);
  const int lane = threadIdx.x & 63, v0 = chunk * C::VPC;
  const u32x4_t* vec = (const u32x4_t*)(row + ch.head);
  constexpr int N = NL * C::VN;
  float z[N];
  const bool edge = chunk == 0 ? ch.head > 0 : false, last = chunk == nch - 1 && ch.tail() < V;
  const float zh = edge && lane < ch.head ? at(row, lane) : -INFINITY;
  const float zt = last && ch.tail() + lane < V ? at(row, ch.tail() + lane) : -INFINITY;
  auto unpack = [&](auto whole) {
    u32x4_t raw[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int v = v0 + 64 * i + lane;
      raw[i] = decltype(whole)::value || v < ch.nv ? vec[v] : u32x4_t{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const bool in = decltype(whole)::value || v0 + 64 * i + lane < ch.nv;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (C::VN == 4) z[4 * i + k] = in ? __uint_as_float(raw[i][k]) : -INFINITY;
        else {
          z[8 * i + 2 * k] = in ? __uint_as_float(raw[i][k] << 16) : -INFINITY;
          z[8 * i + 2 * k + 1] = in ? __uint_as_float(raw[i][k] & 0xffff0000u) : -INFINITY;
        }
      }
    }
  };
  if (v0 + C::VPC <= ch.nv) unpack(std::true_type{});
  else unpack(std::false_type{});
  float m = -INFINITY;                                   // (NaN passes through this maximum)
#pragma unroll
  for (int i = 0; i < N; ++i) m = __builtin_elementwise_maximum(m, z[i]);
  m = __builtin_elementwise_maximum(m, __builtin_elementwise_maximum(zh, zt));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, o, 64));
  Part p{m, 0, 0.0};
  if (!(m < INFINITY)) p.m = __uint_as_float(0x7fc00000u);
  else if (m > -INFINITY) {
    if (c == 0.0) {
      int first = INT32_MAX;                             // the lowest column of the largest logit
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (z[i] == m) first = ch.head + (v0 + 64 * (i / C::VN) + lane) * C::VN + i % C::VN;
      if (zh == m) first = lane;
      if (first == INT32_MAX && zt == m) first = ch.tail() + lane;
      p.arg = wave_min(first);
    } else {
      // (beside the chunk's largest, whose weight is 1, what lies below the lowest weight need not be exactly 0)
      const double least = LOWEST / c;
      double s = 0.0;
      constexpr int G = 4;
#pragma unroll
      for (int i = 0; i < N; i += G) {
        double w[G];
#pragma unroll
        for (int k = 0; k < G; ++k) w[k] = fmax((double)z[i + k] - (double)m, least);
        exp2_64<G>(w, c);
        s += (w[0] + w[1]) + (w[2] + w[3]);
      }
      if (edge || last) {
        double w[2] = {fmax((double)zh - (double)m, least), fmax((double)zt - (double)m, least)};
        exp2_64<2>(w, c);
        s += w[0] + w[1];
      }
      p.s = wave_sum64(s);
    }
  }
  return p;
}

// One wave to a chunk; workgroups go through a row's chunks first.
template <typename T, bool TREE> __global__ __launch_bounds__(256) void verify_parts_kernel(const Verify a) {
  const int groups = (a.nch + 3) / 4, row = blockIdx.x / groups;
  const int chunk = blockIdx.x % groups * 4 + (threadIdx.x >> 6);
  if (chunk >= a.nch) return;
  const T* z;
  int b;
  if constexpr (TREE) {
    b = row / a.T;
    if (row % a.T == 0 && chunk == 0 && (threadIdx.x & 63) == 0) a.arrived[b] = 0;
    if (a.parents[b * a.ldp + row % a.T] < -1) return;   // padding
    z = (const T*)a.z + (int64_t)row * a.ldz;
  } else {
    const int targets = a.B * (a.T + 1);
    if (row < targets) {
      b = row / (a.T + 1);
      if (row % (a.T + 1) > drafted(a, b)) return;
      z = (const T*)a.z + (int64_t)row * a.ldz;
    } else {
      b = (row - targets) / a.T;
      if ((row - targets) % a.T >= drafted(a, b) || rate(a, b) == 0.0) return;
      z = (const T*)a.y + (int64_t)(row - targets) * a.ldy;
    }
  }
  const Part p = chunk_part(z, a.V, a.nch, chunk, rate(a, b));
  if ((threadIdx.x & 63) == 0) a.parts[(int64_t)row * a.nch + chunk] = p;
}

// ---- one wave's steps ------------------------------------------------------------------------------
__device__ __forceinline__ double wave_scan64(double v) {                // sum over lanes 0 .. this one
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double below = __shfl_up(v, o, 64);
    if (lane >= o) v += below;
  }
  return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// A number that a workgroup on another XCD reads in the same launch: stored past this one's caches, and read past its own.
template <typename V> __device__ __forceinline__ void hand_over(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ V taken(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A list of n values that the wave goes through in order: lane l holds values [l per, (l + 1) per), the first K of them in registers.
__device__ __forceinline__ Part listed(const Part* p) { return *p; }
__device__ __forceinline__ double2 listed(const double2* p) { return make_double2(taken(&p->x), taken(&p->y)); }
template <typename P, int K> struct Listed {
  const P* p;
  P v[K];
  int first, end;
  __device__ __forceinline__ Listed(const P* p_, int n) : p(p_) {
    const int per = (n + 63) / 64;
    first = min(n, (int)(threadIdx.x & 63) * per);
    end = min(n, first + per);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = listed(p + min(first + k, n - 1));
  }
  template <typename F> __device__ __forceinline__ void each(F f) const {   // f(index, value), in order
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (first + k < end) f(first + k, v[k]);
    for (int i = first + K; i < end; ++i) f(i, listed(p + i));
  }
};

// Of values in order across the lanes (each lane's `sum`, and `each` to go through them: f(index, weight)), the lowest index at
// which base plus the sum so far exceeds t; where none does, the last with a weight; -1: there is none. All lanes get the index,
// and in base the sum before it.
template <typename F> __device__ __forceinline__ int pick(double& base, double t, double sum, int last, F each) {
  const int lane = threadIdx.x & 63;
  const double upto = base + wave_scan64(sum);
  const uint64_t any = __ballot(last >= 0), over = __ballot(last >= 0 && upto > t);
  if (any == 0) return -1;
  const int win = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(any);
  int found = -1;
  double before = 0.0;
  if (lane == win) {
    double run = upto - sum;
    bool done = false;
    each([&](int j, double w) {
      if (!done && w > 0.0) {
        found = j;
        before = run;
        done = over && run + w > t;
      }
      run += w;
    });
  }
  base = lane_value(before, win);
  return __builtin_amdgcn_readlane(found, win);
}

// The same over columns [lo, hi), at most 64 K of them: get(j) loads what weigh(j, values, weights) makes the weights of G columns
// from j on from.
template <int K, int G, typename F, typename W> __device__ __forceinline__ int pick_column(int lo, int hi, double base, double t, F get, W weigh) {
  constexpr int KG = (K + G - 1) / G;
  const int per = (hi - lo + 63) / 64, first = lo + min(hi - lo, (int)(threadIdx.x & 63) * per), end = min(hi, first + per);
  decltype(get(0)) raw[KG][G];
#pragma unroll
  for (int k = 0; k < KG * G; ++k) raw[k / G][k % G] = get(min(first + k, hi - 1));
  double sum = 0.0, w[KG][G];
  int last = -1;
#pragma unroll
  for (int g = 0; g < KG; ++g) {
    weigh(first + g * G, raw[g], w[g]);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const int j = first + g * G + k;
      w[g][k] = j < end ? w[g][k] : 0.0;
      sum += w[g][k];
      last = w[g][k] > 0.0 ? j : last;
    }
  }
  return pick(base, t, sum, last, [&](auto f) {
#pragma unroll
    for (int k = 0; k < KG * G; ++k)
      if (first + k < end) f(first + k, w[k / G][k % G]);
  });
}

__device__ __forceinline__ double part_sum(const Part& p, double m, double c) { return p.s > 0.0 ? p.s * weight(p.m, m, c) : 0.0; }

// A row's largest logit, its lowest column, and the sum of its weights, from its parts. bad: the row has no distribution.
struct Row { float m; int arg; double s; bool bad; };
template <int K> __device__ __forceinline__ Row row_of(const Listed<Part, K>& parts, double c) {
  Row r{-INFINITY, INT32_MAX, 0.0, false};
  parts.each([&](int, const Part& p) { r.m = __builtin_elementwise_maximum(r.m, p.m); });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) r.m = __builtin_elementwise_maximum(r.m, __shfl_xor(r.m, o, 64));
  r.bad = !(r.m < INFINITY && r.m > -INFINITY);
  if (r.bad) return r;
  if (c == 0.0) {
    parts.each([&](int, const Part& p) { if (p.m == r.m) r.arg = min(r.arg, p.arg); });
    r.arg = wave_min(r.arg);
  } else {
    parts.each([&](int, const Part& p) { r.s += part_sum(p, r.m, c); });
  }
  return r;
}

// Counts one arrival of `all`; whether it is the last. What the others handed over before theirs is then there: each waited for its
// stores before it counted. (Release and acquire fences write back and drop whole L2s: 1024 of them took 30 us.) Called by one wave.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t all) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  uint32_t n = 0;
  if ((threadIdx.x & 63) == 0) n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_amdgcn_readfirstlane(n) + 1 == all;
}

// From node 0 on: the token drawn at a node leads to its first child that holds it. One wave; lane l has nodes l, l + 64, ..
__device__ void walk(const Verify& a, int b, const int32_t* drawn) {
  constexpr int NK = VERIFY_NODES / 64;
  const int lane = threadIdx.x & 63, T = a.T;
  int parent[NK], got[NK];
  int64_t token[NK];
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int t = min(64 * k + lane, T - 1);
    parent[k] = 64 * k + lane < T ? a.parents[b * a.ldp + t] : -2;
    token[k] = a.tokens[(int64_t)b * T + t];
    got[k] = taken(drawn + (int64_t)b * T + t);
  }
  int64_t path[NK];
  int at = 0, n = 0, next = -1;
#pragma unroll
  for (int k = 0; k < NK; ++k) path[k] = -1;
  if (__builtin_amdgcn_readfirstlane(parent[0]) >= -1) {
    while (true) {                                       // (ends: a child's index is larger than its parent's)
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        if (n / 64 == k && n % 64 == lane) path[k] = at;
        if (at / 64 == k) next = __builtin_amdgcn_readlane(got[k], at % 64);
      }
      ++n;
      if (next < 0) break;
      int child = T;
#pragma unroll
      for (int k = NK - 1; k >= 0; --k) {
        const uint64_t hit = __ballot(parent[k] == at && 64 * k + lane > at && token[k] == next);
        if (hit) child = 64 * k + __builtin_ctzll(hit);
      }
      if (child == T) break;
      at = child;
    }
  }
#pragma unroll
  for (int k = 0; k < NK; ++k)
    if (64 * k + lane < T) a.nodes[(int64_t)b * T + 64 * k + lane] = path[k];
  if (lane == 0) { a.out_counts[b] = n; a.out_token[b] = next; }
}

// The token of each node, one wave per row (-1: padding, or no distribution); the last of a sequence's rows follows the tree.
template <typename T> __global__ __launch_bounds__(64) void verify_draw_kernel(const Verify a, int32_t* drawn, uint32_t* arrived) {
  const int row = blockIdx.x, b = row / a.T;
  int token = -1;
  if (a.parents[b * a.ldp + row % a.T] >= -1) {
    const double c = rate(a, b), u = random_at(a, row);
    const Listed<Part, 4> parts(a.parts + (int64_t)row * a.nch, a.nch);
    const Row r = row_of(parts, c);
    if (!r.bad && c == 0.0) token = r.arg;
    else if (!r.bad) {
      const double m = r.m, t = u * lane_value(wave_scan64(r.s), 63);
      double base = 0.0;
      int last = -1;
      parts.each([&](int i, const Part& p) { if (part_sum(p, m, c) > 0.0) last = i; });
      const int ch = pick(base, t, r.s, last, [&](auto f) { parts.each([&](int i, const Part& p) { f(i, part_sum(p, m, c)); }); });
      const T* z = (const T*)a.z + (int64_t)row * a.ldz;
      const Chunks<T> cs(z, a.V, a.nch);
      if (ch >= 0)
        token = pick_column<(CHUNK + 14 + 63) / 64, 6>(cs.lo(ch), cs.hi(ch), base, t, [&](int j) { return at(z, j); },
                                                       [&](int, const float (&x)[6], double (&w)[6]) { weights<6>(x, m, c, w); });
    }
  }
  if (threadIdx.x == 0) hand_over(drawn + row, token);
  if (last_to_arrive(arrived + b, a.T)) walk(a, b, drawn);
}

// ---- drafted blocks ------------------------------------------------------------------------------
// Where a block's verification ended: row n of the target, and what the next token is drawn from (with the rows' largest logits
// and one over their sums).
struct Ended { int n, mode, token, rest; double c, mp, ip, mq, iq; };
enum : int { ENDED_KNOWN = 0, ENDED_P = 1, ENDED_ROW = 2, ENDED_POINT = 3 };   // token known; p; max(p - q, 0), q a row or one token

// Accepts drafted tokens in order: one workgroup of 16 waves per sequence, a wave to a row at a time. Bound by latency: every load
// of a row is issued before the first is waited for.
template <typename T> __global__ __launch_bounds__(1024) void verify_accept_kernel(const Verify a, Ended* ended, uint32_t* arrived) {
  __shared__ Ended rows[VERIFY_NODES + 1];
  __shared__ bool stop[VERIFY_NODES + 1];
  const int b = blockIdx.x, wid = threadIdx.x >> 6, lane = threadIdx.x & 63, L = a.T, n = drafted(a, b);
  const double c = rate(a, b);
  const Part* targets = a.parts + (int64_t)b * (L + 1) * a.nch;
  const Part* drafts = a.parts + ((int64_t)a.B * (L + 1) + (int64_t)b * L) * a.nch;
  for (int i = wid; i <= n; i += 16) {
    const bool row = a.y && i < n && c != 0.0;           // the drafter's row is read
    const int64_t x = i < n ? a.tokens[(int64_t)b * L + i] : -1;
    const bool in = x >= 0 && x < a.V;
    const double u = random_at(a, (int64_t)b * (L + 1) + i);
    const Listed<Part, 2> tp(targets + (int64_t)i * a.nch, a.nch), dp(row ? drafts + (int64_t)i * a.nch : targets, a.nch);
    const float zx = at((const T*)a.z + ((int64_t)b * (L + 1) + i) * a.ldz, in ? (int)x : 0);
    const float yx = row ? at((const T*)a.y + ((int64_t)b * L + i) * a.ldy, in ? (int)x : 0) : 0.f;
    Ended e{i, ENDED_P, -1, 0, c, 0.0, 1.0, 0.0, 1.0};
    const Row p = row_of(tp, c);
    bool stops = true;
    if (p.bad) e.mode = ENDED_KNOWN;
    else if (c == 0.0) {
      e.mode = ENDED_KNOWN;
      e.token = p.arg;
      stops = !(i < n && x == p.arg);
    } else {
      e.mp = p.m;
      e.ip = 1.0 / wave_sum64(p.s);
      if (i < n) {
        e.mode = ENDED_POINT;
        e.token = in ? (int)x : -1;
        double px = in ? weight(zx, e.mp, c) * e.ip : 0.0, qx = in ? 1.0 : 0.0;
        bool bad = false;
        if (row) {
          const Row q = row_of(dp, c);
          bad = q.bad;
          e.mode = bad ? ENDED_KNOWN : ENDED_ROW;
          if (bad) e.token = -1;
          else {
            e.mq = q.m;
            e.iq = 1.0 / wave_sum64(q.s);
            qx = in ? weight(yx, e.mq, c) * e.iq : 0.0;
          }
        }
        stops = bad || !(u * qx < px);
      }
    }
    if (lane == 0) { rows[i] = e; stop[i] = stops; }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int i = 0;
    while (i < n && !stop[i]) ++i;
    ended[b] = rows[i];
    arrived[b] = 0;
    a.out_counts[b] = i;
    if (rows[i].mode == ENDED_KNOWN) a.out_token[b] = rows[i].token;
  }
}

// p and what is left of it at column j.
template <typename T> struct Left {
  const T *z, *y;
  Ended e;
  struct Raw { float z, y; };
  __device__ __forceinline__ Left(const Verify& a, const Ended& e_, int b) : e(e_) {
    z = (const T*)a.z + ((int64_t)b * (a.T + 1) + e.n) * a.ldz;
    y = e.mode == ENDED_ROW ? (const T*)a.y + ((int64_t)b * a.T + e.n) * a.ldy : z;
  }
  __device__ __forceinline__ Raw get(int j) const { return {at(z, j), at(y, j)}; }
  // Of columns j, j + step, ..
  template <int N> __device__ __forceinline__ void of(int j, int step, const Raw (&v)[N], double (&p)[N], double (&left)[N]) const {
    float x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v[i].z;
    weights<N>(x, e.mp, e.c, p);
#pragma unroll
    for (int i = 0; i < N; ++i) left[i] = p[i] *= e.ip;
    if (e.mode == ENDED_POINT) {
#pragma unroll
      for (int i = 0; i < N; ++i) left[i] = j + i * step == e.token ? 0.0 : p[i];
    } else if (e.mode == ENDED_ROW) {
      double q[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = v[i].y;
      weights<N>(x, e.mq, e.c, q);
#pragma unroll
      for (int i = 0; i < N; ++i) left[i] = fmax(p[i] - q[i] * e.iq, 0.0);
    }
  }
};

// Sums of p and of what is left of it, a wave to PIECE columns, grid (pieces / 4, sequences); the last workgroup of a sequence
// draws its next token. Pieces are short, as one row of each sequence has to fill the chip.
constexpr int PIECE = 512;
template <typename T> __global__ __launch_bounds__(256) void verify_next_kernel(const Verify a, const Ended* ended, double2* sums,
                                                                                uint32_t* arrived) {
  const int b = blockIdx.y, wid = threadIdx.x >> 6, lane = threadIdx.x & 63, pieces = (a.V + PIECE - 1) / PIECE;
  const Ended e = ended[b];
  if (e.mode == ENDED_KNOWN) return;
  __shared__ bool last;
  const Left<T> row(a, e, b);
  double2* mine = sums + (int64_t)b * pieces;
  const int piece = blockIdx.x * 4 + wid;
  if (piece < pieces) {
    const int lo = piece * PIECE, hi = min(lo + PIECE, a.V);
    constexpr int G = 4;
    typename Left<T>::Raw raw[PIECE / 64 / G][G];
#pragma unroll
    for (int k = 0; k < PIECE / 64; ++k) raw[k / G][k % G] = row.get(min(lo + 64 * k + lane, hi - 1));
    double p = 0.0, left = 0.0;
#pragma unroll
    for (int k = 0; k < PIECE / 64; k += G) {
      double x[G], l[G];
      row.template of<G>(lo + 64 * k + lane, 64, raw[k / G], x, l);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const bool in = lo + 64 * (k + i) + lane < hi;
        p += in ? x[i] : 0.0;
        left += in ? l[i] : 0.0;
      }
    }
    p = wave_sum64(p);
    left = wave_sum64(left);
    if (lane == 0) {
      hand_over(&mine[piece].x, left);
      hand_over(&mine[piece].y, p);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (wid == 0) {
    const bool mylast = last_to_arrive(arrived + b, gridDim.x);
    if (lane == 0) last = mylast;
  }
  __syncthreads();
  if (!last || wid != 0) return;
  const Listed<double2, 5> list(mine, pieces);
  double l = 0.0, p = 0.0;
  list.each([&](int, const double2& s) { l += s.x; p += s.y; });
  const double left = wave_sum64(l), whole = wave_sum64(p);
  const bool all = e.mode == ENDED_P || left < LEAST;
  const double t = random_at(a, (int64_t)b * (a.T + 1) + a.T) * (all ? whole : left);
  int some = -1;
  list.each([&](int i, const double2& s) { if ((all ? s.y : s.x) > 0.0) some = i; });
  double base = 0.0;
  const int at = pick(base, t, all ? p : l, some, [&](auto f) { list.each([&](int i, const double2& s) { f(i, all ? s.y : s.x); }); });
  int token = -1;
  if (at >= 0)
    token = pick_column<PIECE / 64, 4>(at * PIECE, min(at * PIECE + PIECE, a.V), base, t, [&](int j) { return row.get(j); },
                                       [&](int j, const typename Left<T>::Raw (&v)[4], double (&w)[4]) {
                                         double x[4];
                                         row.template of<4>(j, 1, v, x, w);
                                         if (all) for (int i = 0; i < 4; ++i) w[i] = x[i];
                                       });
  if (lane == 0) a.out_token[b] = token;
}

int64_t pieces_of(int V) { return ((int64_t)V + PIECE - 1) / PIECE; }
int64_t chunks_of(int V) { return ((int64_t)V + CHUNK - 1) / CHUNK; }

int verify_sizes_ok(const char* what, int dtype, int B, int T, int V, int64_t rows) {
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "%s: bad dtype %d", what, dtype);
  UNOK_REQUIRE(B >= 0 && T >= 0 && V > 0 && V <= (1 << 30), UNOK_EINVAL, "%s: B=%d T=%d V=%d", what, B, T, V);
  UNOK_REQUIRE(T <= VERIFY_NODES, UNOK_EUNSUPPORTED, "%s: at most %d drafted tokens to a sequence (got %d)", what, VERIFY_NODES, T);
  UNOK_REQUIRE(B < 65536 && rows * ((chunks_of(V) + 3) / 4) < (1ll << 31), UNOK_EINVAL, "%s: B=%d T=%d V=%d: grid too large", what, B,
               T, V);
  return 0;
}

int verify_setup(Verify& a, const char* what, int dtype, int B, int T, int V, const void* z, int64_t ldz, int64_t rows,
                 const int64_t* tokens, const float* u, float temperature, const float* temperatures, int64_t* counts,
                 int64_t* token, void* workspace, int64_t ws_bytes, int64_t need) {
  UNOK_REQUIRE(z && u && counts && token && (tokens || T == 0), UNOK_EINVAL, "%s: null operand", what);
  UNOK_REQUIRE(rows == 1 || ldz >= V, UNOK_EINVAL, "%s: rows of %d logits, %lld apart", what, V, (long long)ldz);
  UNOK_REQUIRE(((uintptr_t)z & (dtype == UNOK_BF16 ? 1 : 3)) == 0, UNOK_EALIGN, "%s: logits at a fraction of an element", what);
  UNOK_REQUIRE(temperatures || (temperature >= 0.f && temperature < INFINITY), UNOK_EINVAL,
               "%s: temperature %g must be finite and not negative", what, (double)temperature);
  UNOK_REQUIRE(workspace && ws_bytes >= need && ((uintptr_t)workspace & 15) == 0, UNOK_EINVAL,
               "%s: workspace of %lld bytes (16-byte aligned) required, got %lld", what, (long long)need, (long long)ws_bytes);
  a.z = z; a.ldz = ldz;
  a.tokens = tokens;
  a.u = u; a.temp = temperature; a.temps = temperatures;
  a.B = B; a.T = T; a.V = V; a.nch = (int)chunks_of(V);
  a.parts = (Part*)workspace;
  a.out_counts = counts; a.out_token = token;
  return 0;
}

}  // namespace

UNOK_EXPORT int64_t unok_verify_tree_workspace(int dtype, int B, int T, int V) {
  if (verify_sizes_ok("verify_tree", dtype, B, T, V, (int64_t)B * T)) return -1;
  return ((int64_t)B * T * (chunks_of(V) * (int64_t)sizeof(Part) + (int64_t)sizeof(int32_t)) + B * 4ll + 15) / 16 * 16;
}

UNOK_EXPORT int unok_verify_tree(int dtype, int B, int T, int V, const void* z, int64_t ldz, const int64_t* tokens,
                                 const int32_t* parents, int64_t ldp, const float* u, float temperature,
                                 const float* temperatures, int64_t* nodes, int64_t* counts, int64_t* token, void* workspace,
                                 int64_t ws_bytes, void* stream) {
  const int64_t rows = (int64_t)B * T;
  int rc = verify_sizes_ok("verify_tree", dtype, B, T, V, rows);
  if (rc) return rc;
  UNOK_REQUIRE(T >= 1 || B == 0, UNOK_EINVAL, "verify_tree: trees of no nodes");
  if (B == 0) return 0;
  UNOK_REQUIRE(parents && nodes, UNOK_EINVAL, "verify_tree: null operand");
  UNOK_REQUIRE(ldp == 0 || ldp >= T, UNOK_EINVAL, "verify_tree: parents' row stride %lld for %d nodes", (long long)ldp, T);
  Verify a{};
  rc = verify_setup(a, "verify_tree", dtype, B, T, V, z, ldz, rows, tokens, u, temperature, temperatures, counts, token, workspace,
                    ws_bytes, unok_verify_tree_workspace(dtype, B, T, V));
  if (rc) return rc;
  a.parents = parents; a.ldp = ldp;
  a.nodes = nodes;
  int32_t* drawn = (int32_t*)(a.parts + rows * a.nch);
  a.arrived = (uint32_t*)(drawn + rows);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * ((a.nch + 3) / 4))), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, true>), grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_draw_kernel<E>, dim3((unsigned)rows), dim3(64), 0, st, a, drawn, a.arrived);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  return unok::check_launch("verify_tree");
}

UNOK_EXPORT int64_t unok_verify_draft_workspace(int dtype, int B, int L, int V) {
  if (verify_sizes_ok("verify_draft", dtype, B, L, V, (int64_t)B * (2 * L + 1))) return -1;
  return ((int64_t)B * ((2 * L + 1) * chunks_of(V) * (int64_t)sizeof(Part) + pieces_of(V) * (int64_t)sizeof(double2) +
                        (int64_t)sizeof(Ended) + 4) + 15) / 16 * 16;
}

UNOK_EXPORT int unok_verify_draft(int dtype, int B, int L, int V, const void* z, int64_t ldz, const void* y, int64_t ldy,
                                  const int64_t* tokens, const int64_t* counts, const float* u, float temperature,
                                  const float* temperatures, int64_t* accepted, int64_t* token, void* workspace,
                                  int64_t ws_bytes, void* stream) {
  const int64_t targets = (int64_t)B * (L + 1), drafts = (int64_t)B * L;
  int rc = verify_sizes_ok("verify_draft", dtype, B, L, V, targets + drafts);
  if (rc) return rc;
  if (B == 0) return 0;
  Verify a{};
  rc = verify_setup(a, "verify_draft", dtype, B, L, V, z, ldz, targets, tokens, u, temperature, temperatures, accepted, token,
                    workspace, ws_bytes, unok_verify_draft_workspace(dtype, B, L, V));
  if (rc) return rc;
  UNOK_REQUIRE(!y || drafts <= 1 || ldy >= V, UNOK_EINVAL, "verify_draft: draft rows of %d logits, %lld apart", V, (long long)ldy);
  UNOK_REQUIRE(((uintptr_t)y & (dtype == UNOK_BF16 ? 1 : 3)) == 0, UNOK_EALIGN, "verify_draft: logits at a fraction of an element");
  a.y = y; a.ldy = ldy;
  a.counts = counts;
  double2* sums = (double2*)(a.parts + (targets + drafts) * a.nch);
  Ended* ended = (Ended*)(sums + (int64_t)B * pieces_of(V));
  uint32_t* arrived = (uint32_t*)(ended + B);
  hipStream_t st = (hipStream_t)stream;
  const int groups = (a.nch + 3) / 4;
  const dim3 grid((unsigned)((targets + (y ? drafts : 0)) * groups)), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, false>), grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_accept_kernel<E>, dim3((unsigned)B), dim3(1024), 0, st, a, ended, arrived);
    hipLaunchKernelGGL(verify_next_kernel<E>, dim3((unsigned)((pieces_of(V) + 3) / 4), (unsigned)B), block, 0, st, a, ended, sums,
                       arrived);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  return unok::check_launch("verify_draft");
}
