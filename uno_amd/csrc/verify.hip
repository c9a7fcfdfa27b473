// Verification of drafted tokens against the target's logits from given random numbers.
//
// A token is drawn by the inverse distribution function: the lowest index at which the running sum of the weights
// exp((z - max z) / T) exceeds u times their sum. Of a vocabulary's 150 thousand borders between tokens some lie within an fp32
// exponential's error (1e-7) of any u: with such weights about one token in 300 would be another one than the logits say, and
// depend on the order of the sums. The weights and all sums are therefore fp64. A weight relative to its row's largest logit is a column's
// relative to its chunk's times the chunk's, with polynomials of 3.6e-14 and 3.9e-14 (roundings included); the exponent's own roundings, of
// log2(e) / T and of z - max z where that is not exact, add 2.4e-16 |z - max z| / T. So 8e-14 where weights matter, 2.5e-13 at e^-700.
//
// The logits are read once, in chunks of CHUNK columns, one wave each, of which little is kept: largest logits and sums of weights.
// Everything else works on these parts, and on a fourth of a chunk to a drawn token. 16 trees of 64 nodes, 151936 bf16 columns: the
// parts 101 us (59 at a large copy's rate; 12 fp64 and 3 other vector instructions to a weight bound it, issued in 89% of the cycles of
// busy CUs), the tokens and the paths 10. One row of 32000: 4.3 and 3.6 us, latency of loads and reductions.
#include "common.h"
#include "../../include/unok.h"

#include <initializer_list>
#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int CHUNK = 2048, VERIFY_NODES = 256;
constexpr double LOG2E = 1.4426950408889634, LOWEST = -700.0 * LOG2E;   // weights below e^-700 are 0
constexpr double LEAST = 0x1p-40;                                       // of max(p - q, 0) in all; below, p itself is drawn from

// One chunk of a row: its largest logit (NaN passes through), the column of that, and the sum of the weights relative to it. For rows
// that a token may be drawn from, the same of its fourths (the sums relative to the chunk's largest).
struct alignas(16) Part { double s; float m; int arg; };
struct alignas(16) Fourths { double s[4]; float m[4]; int arg; };

struct Verify {
  const void *z, *y; int64_t ldz, ldy;                // target rows; the drafter's rows (null: none)
  const int64_t* tokens;
  const int32_t* parents; int64_t ldp;
  const int64_t* counts;
  const float* u;
  const float* temps; float temp;                     // per sequence, or one
  int B, T, V, nch;                                   // T: nodes of a tree, or drafted tokens
  Part* parts;                                        // drafted blocks: [target rows, then the drafter's][nch]
  Fourths* fourths;                                   // [target rows][nch]
  uint32_t* arrived;                                  // [B], 0 after the parts
  int64_t *nodes, *out_counts, *out_token;
};

// 2^x at x = d c, -1022 <= x <= 0, of N numbers side by side: 2^n (1 + r q(r)), r = x - n in [-1/2, 1/2], q the polynomial through
// (2^r - 1) / r at nine Chebyshev points. Relative error 3.7e-14 before roundings; exactly 1 at 0. n is the low half of x + 1.5 2^52.
template <int N> __device__ __forceinline__ void exp2_64(double (&d)[N], double c) {
  constexpr double ROUND = 0x1.8p52;
  constexpr double Q[9] = {0x1.62e42fefa39efp-1, 0x1.ebfbdff823cedp-3, 0x1.c6b08d7047e52p-5,
                           0x1.3b2ab7181b743p-7, 0x1.5d87fe86fe95bp-10, 0x1.4308ac85ad0bbp-13,
                           0x1.ffcb9515726b1p-17, 0x1.63d13633755aap-20, 0x1.b63880e235143p-24};
  double t[N], r[N], q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = fma(d[i], c, ROUND);
    r[i] = fma(d[i], c, ROUND - t[i]);
    q[i] = Q[8];
  }
#pragma unroll
  for (int k = 7; k >= 0; --k)
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = fma(q[i], r[i], Q[k]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double p = fma(q[i], r[i], 1.0);
    d[i] = __hiloint2double(__double2hiint(p) + __double2loint(t[i]) * (1 << 20), __double2loint(p));
  }
}
// The weights of z relative to m, c = log2(e) / T.
__device__ __forceinline__ bool counts(float z, double m, double c) { return ((double)z - m) * c >= LOWEST; }
template <int N> __device__ __forceinline__ void weights(const float (&z)[N], double m, double c, double (&w)[N]) {
  bool some[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    some[i] = counts(z[i], m, c);
    w[i] = some[i] ? (double)z[i] - m : 0.0;
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
};

// A value moved between lanes by data-parallel moves; lanes that nothing reaches get 0.
template <int CTRL, int ROWS = 0xf, typename V> __device__ __forceinline__ V moved(V v) {
  auto one = [](int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); };
  if constexpr (sizeof(V) == 8) return __hiloint2double(one(__double2hiint(v)), one(__double2loint(v)));
  else return __builtin_bit_cast(V, one(__builtin_bit_cast(int, v)));
}
// Over each 16 lanes, and over the wave: all of them get the result.
template <typename V, typename F> __device__ __forceinline__ V row_all(V v, F f) {
  v = f(v, moved<0xb1>(v));                              // quads 1 0 3 2, then 2 3 0 1, mirrored eights, mirrored rows
  v = f(v, moved<0x4e>(v));
  v = f(v, moved<0x141>(v));
  return f(v, moved<0x140>(v));
}
template <typename V, typename F> __device__ __forceinline__ V wave_all(V v, F f) {
  v = row_all(v, f);
  v = f(v, __shfl_xor(v, 16, 64));
  return f(v, __shfl_xor(v, 32, 64));
}
constexpr auto add64 = [](double x, double y) { return x + y; };
__device__ __forceinline__ double wave_sum64(double v) { return wave_all(v, add64); }
__device__ __forceinline__ int wave_min(int v) { return wave_all(v, [](int x, int y) { return min(x, y); }); }
constexpr auto larger = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };   // (NaN passes through this maximum)
// Four values over the wave at once: the 16 lanes of row j get that of v[j].
template <typename V, typename F> __device__ __forceinline__ V four_all(const V (&v)[4], F f) {
  const bool upper = threadIdx.x & 32, odd = threadIdx.x & 16;
  const V a = f(upper ? v[2] : v[0], __shfl_xor(upper ? v[0] : v[2], 32, 64));
  const V b = f(upper ? v[3] : v[1], __shfl_xor(upper ? v[1] : v[3], 32, 64));
  return row_all(f(odd ? b : a, __shfl_xor(odd ? a : b, 16, 64)), f);
}
__device__ __forceinline__ double wave_scan64(double v) {                // sum over lanes 0 .. this one
  v += moved<0x111>(v);                                  // row_shr 1, 2, 4, 8
  v += moved<0x112>(v);
  v += moved<0x114>(v);
  v += moved<0x118>(v);
  v += moved<0x142, 0xa>(v);                             // row_bcast 15 into rows 1 and 3, 31 into 2 and 3
  v += moved<0x143, 0xc>(v);
  return v;
}

// Sums of weights by a table: 2^x = 2^(N / STEPS) (1 + r q(r)), N + r = STEPS x, r in [-1/2, 1/2], q the polynomial through
// (2^(r / STEPS) - 1) / r at three Chebyshev points (relative error 3.5e-14). The table holds 2^(j / STEPS) with
// j / STEPS taken from the exponent, so that N joins it there whole.
constexpr int STEP_BITS = 8, STEPS = 1 << STEP_BITS;
struct Steps {
  uint64_t v[STEPS];
  constexpr Steps() : v{} {
    for (int j = 0; j < STEPS; ++j) {
      const double y = 0.6931471805599453 * j / STEPS;
      double p = 1.0;
      for (int k = 20; k > 0; --k) p = 1.0 + p * y / k;
      v[j] = __builtin_bit_cast(uint64_t, p) - ((uint64_t)j << (52 - STEP_BITS));
    }
  }
};
__device__ const Steps steps_of_two{};

// s plus the weights of N logits (`least` in place of those below it); c in steps, k = 1.5 2^52 less the reference's whole step.
template <int N> __device__ __forceinline__ double add_weights(const float* z, float least, double c, double k, const double* table,
                                                           double s) {
  constexpr double Q[3] = {0x1.62e42fefa39efp-9, 0x1.ebfbe3a9ac80cp-19, 0x1.c6b08f7c96000p-29};
  double t[N], r[N], w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double x = (double)__builtin_elementwise_maximum(z[i], least);
    t[i] = fma(x, c, k);
    r[i] = fma(x, c, k - t[i]);
    w[i] = table[__double2loint(t[i]) & (STEPS - 1)];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const double p = fma(fma(fma(Q[2], r[i], Q[1]), r[i], Q[0]), r[i], 1.0);
    s = fma(__hiloint2double(__double2hiint(w[i]) + (__double2loint(t[i]) << (20 - STEP_BITS)), __double2loint(w[i])), p, s);
  }
  return s;
}

// The part of one chunk of a row, by one wave.
template <typename T> __device__ __forceinline__ void chunk_part(const T* row, int V, int nch, int chunk, double c, const double* table,
                                                                 Part* to, Fourths* four) {
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
  float top[4] = {zh, -INFINITY, -INFINITY, zt};
#pragma unroll
  for (int i = 0; i < N; ++i) top[i * 4 / N] = larger(top[i * 4 / N], z[i]);
  const float fourth = four_all(top, larger);
  float m = larger(fourth, __shfl_xor(fourth, 16, 64));
  m = larger(m, __shfl_xor(m, 32, 64));
  int arg = 0;
  double sum = 0.0;
  if (m < INFINITY && m > -INFINITY) {
    if (c == 0.0) {
      int first = INT32_MAX;                             // the lowest column of the largest logit
#pragma unroll
      for (int i = N - 1; i >= 0; --i)
        if (z[i] == m) first = ch.head + (v0 + 64 * (i / C::VN) + lane) * C::VN + i % C::VN;
      if (zh == m) first = lane;
      if (first == INT32_MAX && zt == m) first = ch.tail() + lane;
      arg = wave_min(first);
    } else {
      // (beside the chunk's largest, whose weight is 1, what lies below the lowest weight need not be exactly 0)
      const double cs = c * STEPS, whole = rint((double)m * cs);
      const float least = (float)((double)m + LOWEST / c);
      const double x = ((double)least - (double)m) * c;  // (LOWEST, unless its logit is no fp32 number's neighbour)
      double s[4] = {0.0, 0.0, 0.0, 0.0};
      if (fabs(whole) < 0x1p50 && x >= LOWEST - 10.0 && x <= LOWEST + 10.0) {
        const double k = 0x1.8p52 - whole;
#pragma unroll
        for (int i = 0; i < N; i += 4) s[i * 4 / N] = add_weights<4>(z + i, least, cs, k, table, s[i * 4 / N]);
        if (edge) s[0] = add_weights<1>(&zh, least, cs, k, table, s[0]);
        if (last) s[3] = add_weights<1>(&zt, least, cs, k, table, s[3]);
        double f[1] = {-fma((double)m, cs, -whole)};     // (these are relative to the whole step next to m)
        exp2_64<1>(f, 1.0 / STEPS);
        sum = four_all(s, add64) * f[0];
      } else {                                           // logits far from 0 by the temperature's measure, or temperatures far off
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float x[4] = {z[i], z[i + 1], z[i + 2], z[i + 3]};
          double w[4];
          weights<4>(x, m, c, w);
          s[i * 4 / N] += (w[0] + w[1]) + (w[2] + w[3]);
        }
        s[0] += weight(zh, m, c);
        s[3] += weight(zt, m, c);
        sum = four_all(s, add64);
      }
    }
  }
  if (four) {
    if ((lane & 15) == 0) { four->s[lane >> 4] = sum; four->m[lane >> 4] = fourth; }
    if (lane == 0) four->arg = arg;
  }
  if (to) {
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane == 0) *to = Part{sum, m, arg};
  }
}

// One wave to a chunk; workgroups go through a row's chunks first.
template <typename T, bool TREE> __global__ __launch_bounds__(256) void verify_parts_kernel(const Verify a) {
  const int groups = (a.nch + 3) / 4, row = blockIdx.x / groups;
  const int chunk = blockIdx.x % groups * 4 + (threadIdx.x >> 6);
  __shared__ double table[STEPS];
  if (threadIdx.x < STEPS) table[threadIdx.x] = __builtin_bit_cast(double, steps_of_two.v[threadIdx.x]);
  __syncthreads();
  if (chunk >= a.nch) return;
  const T* z;
  int b;
  bool target = true;
  if constexpr (TREE) {
    b = row / a.T;
    if (row % a.T == 0 && chunk == 0 && (threadIdx.x & 63) == 0) a.arrived[b] = 0;
    if (a.parents[b * a.ldp + row % a.T] < -1) return;   // padding
    z = (const T*)a.z + (int64_t)row * a.ldz;
  } else {
    const int targets = a.B * (a.T + 1);
    if (row < targets) {
      b = row / (a.T + 1);
      if (row % (a.T + 1) == 0 && chunk == 0 && (threadIdx.x & 63) == 0) a.arrived[b] = 0;
      if (row % (a.T + 1) > drafted(a, b)) return;
      z = (const T*)a.z + (int64_t)row * a.ldz;
    } else {
      target = false;
      b = (row - targets) / a.T;
      if ((row - targets) % a.T >= drafted(a, b) || rate(a, b) == 0.0) return;
      z = (const T*)a.y + (int64_t)(row - targets) * a.ldy;
    }
  }
  chunk_part(z, a.V, a.nch, chunk, rate(a, b), table, TREE ? nullptr : a.parts + (int64_t)row * a.nch + chunk,
             target ? a.fourths + (int64_t)row * a.nch + chunk : nullptr);
}

// ---- one wave's steps ------------------------------------------------------------------------------
__device__ __forceinline__ double lane_value(double v, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane), __builtin_amdgcn_readlane(__double2loint(v), lane));
}

// A number that a workgroup on another XCD reads in the same launch: stored past this one's caches, and read past its own.
template <typename V> __device__ __forceinline__ void hand_over(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ V taken(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A list of n values that the wave goes through in order: lane l holds values [l per, (l + 1) per), the first K of them in registers;
// get(i) loads one.
template <typename G, int K> struct Listed {
  G get;
  decltype(get(0)) v[K];
  int first, end;
  __device__ __forceinline__ Listed(G get_, int n) : get(get_) {
    const int per = (n + 63) / 64;
    first = min(n, (int)(threadIdx.x & 63) * per);
    end = min(n, first + per);
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = get(min(first + k, n - 1));
  }
  template <typename F> __device__ __forceinline__ void each(F f) const {   // f(index, value), in order
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (first + k < end) f(first + k, v[k]);
    for (int i = first + K; i < end; ++i) f(i, get(i));
  }
};
struct Parts {
  const Part* p;
  __device__ __forceinline__ Part operator()(int i) const { return p[i]; }
};
struct FourthParts {
  const Fourths* p;
  __device__ __forceinline__ Fourths operator()(int i) const { return p[i]; }
};
__device__ __forceinline__ const Part& whole(const Part& p) { return p; }
__device__ __forceinline__ Part whole(const Fourths& p) {
  return {(p.s[0] + p.s[1]) + (p.s[2] + p.s[3]), larger(larger(p.m[0], p.m[1]), larger(p.m[2], p.m[3])), p.arg};
}
struct Pairs {                                           // sums that other workgroups of this launch handed over
  const double2* p;
  __device__ __forceinline__ double2 operator()(int i) const { return make_double2(taken(&p[i].x), taken(&p[i].y)); }
};

// Of values in order across the lanes (`upto` the sum up to each lane's end, `sum` its own, `last` its last index with a weight, and
// `each` to go through them: f(index, weight)), the lowest index at which base plus the sum so far exceeds t; where none does, the last
// with a weight, and `over` is false; -1: there is none. All lanes get the index, and in base the sum before it.
template <typename F> __device__ __forceinline__ int pick(double& base, bool& over, double t, double upto, double sum, int last, F each) {
  const int lane = threadIdx.x & 63;
  const uint64_t any = __ballot(last >= 0), past = __ballot(last >= 0 && base + upto > t);
  over = past != 0;
  if (any == 0) return -1;
  const int win = over ? __builtin_ctzll(past) : 63 - __builtin_clzll(any);
  int found = -1;
  double before = 0.0;
  if (lane == win) {
    double run = base + (upto - sum);
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
  bool over;
  return pick(base, over, t, wave_scan64(sum), sum, last, [&](auto f) {
#pragma unroll
    for (int k = 0; k < KG * G; ++k)
      if (first + k < end) f(first + k, w[k / G][k % G]);
  });
}

// A row's largest logit, its lowest column, and the sum of its weights, from its parts. bad: the row has no distribution.
struct Row { float m; int arg; double s; bool bad; };
template <typename G, int K> __device__ __forceinline__ Row row_of(const Listed<G, K>& parts, double c) {
  Row r{-INFINITY, INT32_MAX, 0.0, false};
  parts.each([&](int, const auto& p) { r.m = larger(r.m, whole(p).m); });
  r.m = wave_all(r.m, larger);
  r.bad = !(r.m < INFINITY && r.m > -INFINITY);
  if (r.bad) return r;
  if (c == 0.0) {
    parts.each([&](int, const auto& p) { if (whole(p).m == r.m) r.arg = min(r.arg, whole(p).arg); });
    r.arg = wave_min(r.arg);
  } else {
    parts.each([&](int, const auto& p) { r.s += whole(p).s * weight(whole(p).m, r.m, c); });
  }
  return r;
}

// Counts one arrival of `all`; whether it is the last. What the others handed over before theirs is then there: each waited for its
// stores, which go past its caches, before it counted. The last one needs no acquire: what it reads of the others are loads past its own
// caches (`taken`) alone, issued after the count has come back, since they stand behind a branch on it, and the compiler moves nothing
// above the empty statement. (Release and acquire fences write back and drop whole L2s: 1024 of them took 30 us.) Called by one wave.
__device__ __forceinline__ bool last_to_arrive(uint32_t* counter, uint32_t all) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  uint32_t n = 0;
  if ((threadIdx.x & 63) == 0) n = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const bool last = __builtin_amdgcn_readfirstlane(n) + 1 == all;
  asm volatile("" ::: "memory");
  return last;
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

// The token drawn from a row, by one wave: the fourth of a chunk in which the running sum exceeds t, then its columns, a vector or two
// to a lane (before the first one those up to the first boundary, after the last one the rest).
template <typename T> __device__ __forceinline__ int draw(const T* z, const Verify& a, const Listed<FourthParts, 2>& parts, double c, double u) {
  const Row r = row_of(parts, c);
  if (r.bad || c == 0.0) return r.bad ? -1 : r.arg;
  const int lane = threadIdx.x & 63;
  const double m = r.m, upto = wave_scan64(r.s), t = u * lane_value(upto, 63);
  auto fourths = [&](auto f) {
    parts.each([&](int i, const Fourths& p) {
      const double w = weight(whole(p).m, m, c);
      // (of a fourth in which no column counts, some columns' lowest weights may have been added)
#pragma unroll
      for (int k = 0; k < 4; ++k) f(4 * i + k, counts(p.m[k], m, c) ? p.s[k] * w : 0.0);
    });
  };
  int last = -1;
  fourths([&](int i, double w) { last = w > 0.0 ? i : last; });
  double base = 0.0;
  bool over;
  const int at4 = pick(base, over, t, upto, r.s, last, fourths);
  if (at4 < 0) return -1;
  using C = Chunks<T>;
  constexpr int COLS = CHUNK / 4 / 64;                   // to a lane
  const C ch(z, a.V, a.nch);
  const int body = ch.head + at4 * (CHUNK / 4);
  int token = -1;
  double start = base;
  for (int step = at4 == 0 && ch.head > 0 ? 0 : 1; step < 3; ++step) {   // head, vectors, rest
    if (step == 2 && (at4 != 4 * ch.nch - 1 || ch.tail() == ch.V)) break;
    const int j = step == 0 ? lane : step == 1 ? body + COLS * lane : ch.tail() + lane;
    const int n = step == 0 ? lane < ch.head : step == 1 ? max(0, min(COLS, ch.tail() - j)) : j < ch.V;
    float x[COLS];
#pragma unroll
    for (int k = 0; k < COLS; ++k) x[k] = -INFINITY;
    if (step != 1) {
      if (n) x[0] = at(z, j);
    } else {
#pragma unroll
      for (int v = 0; v < COLS / C::VN; ++v)
        if (n >= (v + 1) * C::VN) {
          const u32x4_t raw = *(const u32x4_t*)(z + j + v * C::VN);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (C::VN == 4) x[4 * v + k] = __uint_as_float(raw[k]);
            else { x[2 * k] = __uint_as_float(raw[k] << 16); x[2 * k + 1] = __uint_as_float(raw[k] & 0xffff0000u); }
          }
        }
    }
    double w[COLS], sum = 0.0;
    int some = -1;
    weights<COLS>(x, m, c, w);
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      sum += w[k];
      some = w[k] > 0.0 ? j + k : some;
    }
    const double all = wave_scan64(sum);
    double before = start;
    const int got = pick(before, over, t, all, sum, some, [&](auto f) {
#pragma unroll
      for (int k = 0; k < COLS; ++k) f(j + k, w[k]);
    });
    if (got >= 0) token = got;
    if (over) break;
    start += lane_value(all, 63);
  }
  return token;
}

// The token of each node, a wave to a row (-1: padding, or no distribution), ROWS rows of a sequence to a workgroup; the last workgroup
// of a sequence follows the tree. Workgroups that count their arrival in one place wait for each other: 16 sequences of 64 nodes 18 us
// where each row has its own, in eights 9.3; 8 sequences of 16 nodes 6.8 and 8.0, since there waves of one CU wait for each other more.
// Both forms with the parts (us, alone / in eights): 151936 columns, one sequence of 17 nodes 11.4 / 13.0, of 63 15.5 / 17.1, 4 of 16 15.5
// / 17.3, 4 of 63 35.6 / 34.8, 8 of 16 23.0 / 24.0, 8 of 32 34.9 / 34.8, 8 of 63 59.8 / 57.7, 16 of 16 33.9 / 34.7, 16 of 24 46.7 / 46.0, 16 of 63 120
// / 114; 32000 columns, 1 of 63 10.8 / 10.9, 4 of 32 12.7 / 12.6, 8 of 16 12.3 / 12.3, 16 of 8 12.1 / 12.2, 16 of 16 16.7 / 15.5. So a rule on
// the nodes alone is off by up to 2 us for one to four sequences of 17 to 48 nodes, and by 1 for 16 sequences of 16 over small vocabularies.
constexpr int DRAW_ALONE = 16, DRAW_ROWS = 8;            // up to DRAW_ALONE nodes each has a workgroup
template <typename T, int ROWS> __global__ __launch_bounds__(64 * ROWS) void verify_draw_kernel(const Verify a, int32_t* drawn) {
  __shared__ int tokens[ROWS];
  const int b = blockIdx.y, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int node0 = blockIdx.x * ROWS, node = min(node0 + wid, a.T - 1);
  const int64_t row = (int64_t)b * a.T + node;
  const Listed<FourthParts, 2> parts({a.fourths + row * a.nch}, a.nch);
  const double c = rate(a, b), u = random_at(a, row);
  const int parent = a.parents[b * a.ldp + node];
  int token = -1;
  if (node0 + wid < a.T && parent >= -1) token = draw((const T*)a.z + row * a.ldz, a, parts, c, u);
  if (ROWS == 1 && a.T == 1) {                           // (no one to wait for)
    if (lane == 0) { a.nodes[b] = parent >= -1 ? 0 : -1; a.out_counts[b] = parent >= -1; a.out_token[b] = token; }
    return;
  }
  if (lane == 0) tokens[wid] = token;
  __syncthreads();
  if (wid != 0) return;
  if (lane < ROWS && node0 + lane < a.T) hand_over(drawn + (int64_t)b * a.T + node0 + lane, tokens[lane]);
  if (last_to_arrive(a.arrived + b, gridDim.x)) walk(a, b, drawn);
}

// ---- drafted blocks ------------------------------------------------------------------------------
// Where a block's verification ended: row n of the target, and what the next token is drawn from (with the rows' largest logits
// and one over their sums).
struct Ended { int n, mode, token, rest; double c, mp, ip, mq, iq; };
constexpr int WAVES = 16;
enum : int { ENDED_KNOWN = 0, ENDED_P = 1, ENDED_ROW = 2, ENDED_POINT = 3 };   // token known; p; max(p - q, 0), q a row or one token

// Accepts drafted tokens in order: a wave of the workgroup to a row at a time. Bound by latency: every load of a row is issued before the
// first is waited for. All of them get where it ended.
template <typename T> __device__ __forceinline__ Ended accept(const Verify& a, int b, Ended* rows, bool* stop) {
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, L = a.T, n = drafted(a, b);
  const double c = rate(a, b);
  const Part* targets = a.parts + (int64_t)b * (L + 1) * a.nch;
  const Part* drafts = a.parts + ((int64_t)a.B * (L + 1) + (int64_t)b * L) * a.nch;
  for (int i = wid; i <= n; i += WAVES) {
    const bool row = a.y && i < n && c != 0.0;           // the drafter's row is read
    const int64_t x = i < n ? a.tokens[(int64_t)b * L + i] : -1;
    const bool in = x >= 0 && x < a.V;
    const double u = random_at(a, (int64_t)b * (L + 1) + i);
    const Listed<Parts, 2> tp(Parts{targets + (int64_t)i * a.nch}, a.nch), dp(Parts{row ? drafts + (int64_t)i * a.nch : targets}, a.nch);
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
  int first = 0;
  for (int i = 0; i < n; i += 64) {
    const uint64_t here = __ballot(i + lane < n && stop[i + lane]);
    first = here ? i + __builtin_ctzll(here) : n;
    if (here) break;
  }
  return rows[first];
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

// Finds where a sequence ended (every workgroup for itself: 8 sequences of 15 tokens of 151936 15.3 us, with a kernel before it for that
// 5.8 + 10.6 and a launch), then sums p and what is left of it, a wave to PIECE columns, grid (pieces / WAVES, sequences); the last
// workgroup of a sequence draws its next token. Pieces are short, as one row of each sequence has to fill the chip.
constexpr int PIECE = 512;
template <typename T> __global__ __launch_bounds__(64 * WAVES) void verify_next_kernel(const Verify a, double2* sums) {
  __shared__ Ended rows[VERIFY_NODES + 1];
  __shared__ bool stop[VERIFY_NODES + 1];
  const int b = blockIdx.y, wid = threadIdx.x >> 6, lane = threadIdx.x & 63, pieces = (a.V + PIECE - 1) / PIECE;
  const Ended e = accept<T>(a, b, rows, stop);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.out_counts[b] = e.n;
    if (e.mode == ENDED_KNOWN) a.out_token[b] = e.token;
  }
  if (e.mode == ENDED_KNOWN) return;
  if (e.mode == ENDED_P) {                               // p's sums are there already
    if (blockIdx.x || wid) return;
    const int64_t at = (int64_t)b * (a.T + 1) + e.n;
    const Listed<FourthParts, 2> parts({a.fourths + at * a.nch}, a.nch);
    const int token = draw((const T*)a.z + at * a.ldz, a, parts, e.c, random_at(a, (int64_t)b * (a.T + 1) + a.T));
    if (lane == 0) a.out_token[b] = token;
    return;
  }
  __shared__ bool last;
  const Left<T> row(a, e, b);
  double2* mine = sums + (int64_t)b * pieces;
  const int piece = blockIdx.x * WAVES + wid;
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
    const bool mylast = last_to_arrive(a.arrived + b, gridDim.x);
    if (lane == 0) last = mylast;
  }
  __syncthreads();
  if (!last || wid != 0) return;
  const Listed<Pairs, 5> list(Pairs{mine}, pieces);
  double l = 0.0, p = 0.0;
  list.each([&](int, const double2& s) { l += s.x; p += s.y; });
  const double left = wave_sum64(l), whole = wave_sum64(p);
  const bool all = left < LEAST;
  const double t = random_at(a, (int64_t)b * (a.T + 1) + a.T) * (all ? whole : left);
  int some = -1;
  list.each([&](int i, const double2& s) { if ((all ? s.y : s.x) > 0.0) some = i; });
  double base = 0.0;
  bool over;
  const int at = pick(base, over, t, wave_scan64(all ? p : l), all ? p : l, some,
                      [&](auto f) { list.each([&](int i, const double2& s) { f(i, all ? s.y : s.x); }); });
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

struct Span { const void* p; int64_t bytes; };

// What is written, the workspace among it, shares no memory with anything else: workgroups end at different times.
int verify_apart(const char* what, std::initializer_list<Span> read, std::initializer_list<Span> written) {
  auto meet = [](const Span& a, const Span& b) {
    return a.p && b.p && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
  };
  for (const Span* w = written.begin(); w != written.end(); ++w) {
    for (const Span& r : read) UNOK_REQUIRE(!meet(*w, r), UNOK_EINVAL, "%s: an output or the workspace overlaps an operand", what);
    for (const Span* v = written.begin(); v != w; ++v) UNOK_REQUIRE(!meet(*w, *v), UNOK_EINVAL, "%s: outputs or the workspace overlap", what);
  }
  return 0;
}

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
  a.out_counts = counts; a.out_token = token;
  return 0;
}

}  // namespace

UNOK_EXPORT int64_t unok_verify_tree_workspace(int dtype, int B, int T, int V) {
  if (verify_sizes_ok("verify_tree", dtype, B, T, V, (int64_t)B * T)) return -1;
  return ((int64_t)B * T * (chunks_of(V) * (int64_t)sizeof(Fourths) + (int64_t)sizeof(int32_t)) + B * 4ll + 15) / 16 * 16;
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
  const int64_t es = dtype == UNOK_BF16 ? 2 : 4, ids = rows * (int64_t)sizeof(int64_t), each = B * (int64_t)sizeof(int64_t);
  rc = verify_apart("verify_tree",
                    {{z, ((rows - 1) * ldz + V) * es}, {tokens, ids}, {parents, ((B - 1) * ldp + T) * 4}, {u, rows * 4}, {temperatures, B * 4ll}},
                    {{nodes, ids}, {counts, each}, {token, each}, {workspace, unok_verify_tree_workspace(dtype, B, T, V)}});
  if (rc) return rc;
  a.parents = parents; a.ldp = ldp;
  a.nodes = nodes;
  a.fourths = (Fourths*)workspace;
  int32_t* drawn = (int32_t*)(a.fourths + rows * a.nch);
  a.arrived = (uint32_t*)(drawn + rows);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * ((a.nch + 3) / 4))), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, true>), grid, block, 0, st, a);
    if (T <= DRAW_ALONE)
      hipLaunchKernelGGL((verify_draw_kernel<E, 1>), dim3((unsigned)T, (unsigned)B), dim3(64), 0, st, a, drawn);
    else
      hipLaunchKernelGGL((verify_draw_kernel<E, DRAW_ROWS>), dim3((unsigned)((T + DRAW_ROWS - 1) / DRAW_ROWS), (unsigned)B),
                         dim3(64 * DRAW_ROWS), 0, st, a, drawn);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  return unok::check_launch("verify_tree");
}

UNOK_EXPORT int64_t unok_verify_draft_workspace(int dtype, int B, int L, int V) {
  if (verify_sizes_ok("verify_draft", dtype, B, L, V, (int64_t)B * (2 * L + 1))) return -1;
  const int64_t chunks = chunks_of(V) * ((2 * L + 1) * (int64_t)sizeof(Part) + (L + 1) * (int64_t)sizeof(Fourths));
  return (B * (chunks + pieces_of(V) * (int64_t)sizeof(double2) + 4) + 15) / 16 * 16;
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
  const int64_t es = dtype == UNOK_BF16 ? 2 : 4, each = B * (int64_t)sizeof(int64_t);
  rc = verify_apart("verify_draft",
                    {{z, ((targets - 1) * ldz + V) * es}, {y, drafts ? ((drafts - 1) * ldy + V) * es : 0}, {tokens, drafts * 8}, {counts, each},
                     {u, targets * 4}, {temperatures, B * 4ll}},
                    {{accepted, each}, {token, each}, {workspace, unok_verify_draft_workspace(dtype, B, L, V)}});
  if (rc) return rc;
  a.y = y; a.ldy = ldy;
  a.counts = counts;
  a.parts = (Part*)workspace;
  a.fourths = (Fourths*)(a.parts + (targets + drafts) * a.nch);
  double2* sums = (double2*)(a.fourths + targets * a.nch);
  a.arrived = (uint32_t*)(sums + (int64_t)B * pieces_of(V));
  hipStream_t st = (hipStream_t)stream;
  const int groups = (a.nch + 3) / 4;
  const dim3 grid((unsigned)((targets + (y ? drafts : 0)) * groups)), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, false>), grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_next_kernel<E>, dim3((unsigned)((pieces_of(V) + WAVES - 1) / WAVES), (unsigned)B), dim3(64 * WAVES), 0,
                       st, a, sums);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  return unok::check_launch("verify_draft");
}
