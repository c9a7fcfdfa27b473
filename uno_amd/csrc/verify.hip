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
  int64_t *nodes, *out_counts, *out_token;
};

// 2^x for -1022 <= x <= 0: 2^n (1 + r q(r)), r = x - n in [-1/2, 1/2], q the polynomial through (2^r - 1) / r at ten Chebyshev
// points. Relative error 6.4e-16; exactly 1 at 0.
__device__ __forceinline__ double exp2_64(double x) {
  const double n = __builtin_rint(x), r = x - n;
  double q = 0x1.e5e9f548e5725p-28;
  q = fma(q, r, 0x1.b6571de2f2351p-24);
  q = fma(q, r, 0x1.62bfe46117445p-20);
  q = fma(q, r, 0x1.ffcb76789860fp-17);
  q = fma(q, r, 0x1.4309130378460p-13);
  q = fma(q, r, 0x1.5d87fe908f88ap-10);
  q = fma(q, r, 0x1.3b2ab6fba385fp-7);
  q = fma(q, r, 0x1.c6b08d7044119p-5);
  q = fma(q, r, 0x1.ebfbdff82c590p-3);
  q = fma(q, r, 0x1.62e42fefa39f7p-1);
  const double p = fma(q, r, 1.0);
  return __hiloint2double(__double2hiint(p) + (int)n * (1 << 20), __double2loint(p));
}
// The weight of z relative to m, c = log2(e) / T.
__device__ __forceinline__ double weight(float z, double m, double c) {
  const double x = ((double)z - m) * c;
  const bool some = x >= LOWEST;
  const double w = exp2_64(some ? x : 0.0);
  return some ? w : 0.0;
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
__device__ __forceinline__ int wave_or(bool v) { return __ballot(v) != 0; }

// The parts of one chunk of a row, by one wave.
template <typename T> __device__ __forceinline__ Part chunk_part(const T* row, int V, int nch, int chunk, double c) {
  using C = Chunks<T>;
  constexpr int NL = C::VPC / 64;
  const C ch(row, V, nch);
  const int lane = threadIdx.x & 63, v0 = chunk * C::VPC;
  const u32x4_t* vec = (const u32x4_t*)(row + ch.head);
  u32x4_t raw[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int v = v0 + 64 * i + lane;
    raw[i] = v < ch.nv ? vec[v] : u32x4_t{0, 0, 0, 0};
  }
  float z[NL * C::VN + 2];
  z[NL * C::VN] = chunk == 0 && lane < ch.head ? at(row, lane) : -INFINITY;
  z[NL * C::VN + 1] = chunk == nch - 1 && ch.tail() + lane < V ? at(row, ch.tail() + lane) : -INFINITY;
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const bool in = v0 + 64 * i + lane < ch.nv;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (C::VN == 4) z[4 * i + k] = in ? __uint_as_float(raw[i][k]) : -INFINITY;
      else {
        z[8 * i + 2 * k] = in ? __uint_as_float(raw[i][k] << 16) : -INFINITY;
        z[8 * i + 2 * k + 1] = in ? __uint_as_float(raw[i][k] & 0xffff0000u) : -INFINITY;
      }
    }
  }
  float m = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < NL * C::VN + 2; ++i) {
    m = fmaxf(m, z[i]);
    bad |= !(z[i] < INFINITY);
  }
  m = wave_max(m);
  Part p{m, 0, 0.0};
  if (wave_or(bad)) p.m = __uint_as_float(0x7fc00000u);
  else if (m > -INFINITY) {
    if (c == 0.0) {
      int first = INT32_MAX;                             // the lowest column of the largest logit
#pragma unroll
      for (int i = NL * C::VN - 1; i >= 0; --i)
        if (z[i] == m) first = ch.head + (v0 + 64 * (i / C::VN) + lane) * C::VN + i % C::VN;
      if (z[NL * C::VN] == m) first = lane;
      if (first == INT32_MAX && z[NL * C::VN + 1] == m) first = ch.tail() + lane;
      p.arg = wave_min(first);
    } else {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < NL * C::VN + 2; ++i) s += weight(z[i], (double)m, c);
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

// ---- workgroup-wide steps (256 threads) ---------------------------------------------------------
struct Shared { double wave[4]; float fmax[4]; int flag[4], win, last; };

__device__ __forceinline__ double scan64(double v, Shared& sh, double& total) {   // sum over threads 0 .. this one
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double below = __shfl_up(v, o, 64);
    if (lane >= o) v += below;
  }
  __syncthreads();
  if (lane == 63) sh.wave[w] = v;
  __syncthreads();
  double before = 0.0;
  total = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) before += sh.wave[i];
    total += sh.wave[i];
  }
  return before + v;
}

// The lowest index j of [lo, hi) at which base plus the weights up to j exceeds t, or where none does, the last with a weight
// (-1: no weight at all). `of` gives an index's weight. `start` becomes base plus the weights before j.
template <typename F> __device__ int pick(int lo, int hi, double base, double t, Shared& sh, F of, double& start) {
  const int n = hi - lo, per = (n + 255) / 256;
  const int first = lo + min(n, (int)threadIdx.x * per), end = min(hi, first + per);
  double sum = 0.0, total;
  int some = -1;
  for (int j = first; j < end; ++j) {
    const double w = of(j);
    sum += w;
    some = w > 0.0 ? j : some;
  }
  const double upto = base + scan64(sum, sh, total);
  if (threadIdx.x == 0) { sh.win = INT32_MAX; sh.last = -1; }
  __syncthreads();
  if (some >= 0) {
    atomicMax(&sh.last, some);
    if (upto > t) atomicMin(&sh.win, (int)threadIdx.x);
  }
  __syncthreads();
  const int win = sh.win, last = sh.last;
  // the thread that holds the index goes through its weights again
  __syncthreads();
  if (win == INT32_MAX ? (last >= first && last < end) : win == (int)threadIdx.x) {
    double run = upto - sum;
    int j = first, found = some;
    double before = run;
    for (; j < end; ++j) {
      const double w = of(j);
      if (w > 0.0) {
        before = run;
        if (win != INT32_MAX && run + w > t) { found = j; break; }
      }
      run += w;
    }
    sh.last = found;
    sh.wave[0] = before;
  }
  __syncthreads();
  const int found = sh.last;
  start = sh.wave[0];
  __syncthreads();
  return found;
}

// A row's largest logit over its parts (NaN: no distribution).
__device__ __forceinline__ float row_max(const Part* parts, int nch, Shared& sh) {
  float m = -INFINITY;
  bool bad = false;
  for (int c = threadIdx.x; c < nch; c += 256) {
    const float x = parts[c].m;
    bad |= x != x;
    m = fmaxf(m, x);
  }
  m = wave_max(m);
  const int any = wave_or(bad);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { sh.fmax[threadIdx.x >> 6] = m; sh.flag[threadIdx.x >> 6] = any; }
  __syncthreads();
  m = fmaxf(fmaxf(sh.fmax[0], sh.fmax[1]), fmaxf(sh.fmax[2], sh.fmax[3]));
  return sh.flag[0] | sh.flag[1] | sh.flag[2] | sh.flag[3] || m == -INFINITY ? __uint_as_float(0x7fc00000u) : m;
}
__device__ __forceinline__ double part_sum(const Part& p, double m, double c) { return p.s > 0.0 ? p.s * weight(p.m, m, c) : 0.0; }

// The token of each node: one workgroup per row. (-1: padding, or no distribution.)
template <typename T> __global__ __launch_bounds__(256) void verify_draw_kernel(const Verify a, int32_t* drawn) {
  __shared__ Shared sh;
  const int row = blockIdx.x, b = row / a.T;
  if (a.parents[b * a.ldp + row % a.T] < -1) {
    if (threadIdx.x == 0) drawn[row] = -1;
    return;
  }
  const Part* parts = a.parts + (int64_t)row * a.nch;
  const double c = rate(a, b);
  const float m = row_max(parts, a.nch, sh);
  int token = -1;
  if (m == m) {
    if (c == 0.0) {
      int first = INT32_MAX;
      for (int i = threadIdx.x; i < a.nch; i += 256)
        if (parts[i].m == m) first = min(first, parts[i].arg);
      first = wave_min(first);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) sh.flag[threadIdx.x >> 6] = first;
      __syncthreads();
      token = min(min(sh.flag[0], sh.flag[1]), min(sh.flag[2], sh.flag[3]));
    } else {
      double sum = 0.0, total, start;
      for (int i = threadIdx.x; i < a.nch; i += 256) sum += part_sum(parts[i], m, c);
      (void)scan64(sum, sh, total);
      const double t = random_at(a, row) * total;
      const int ch = pick(0, a.nch, 0.0, t, sh, [&](int i) { return part_sum(parts[i], m, c); }, start);
      const T* z = (const T*)a.z + (int64_t)row * a.ldz;
      const Chunks<T> cs(z, a.V, a.nch);
      if (ch >= 0) token = pick(cs.lo(ch), cs.hi(ch), start, t, sh, [&](int j) { return weight(at(z, j), m, c); }, start);
    }
  }
  if (threadIdx.x == 0) drawn[row] = token;
}

// From node 0 on: the token drawn at a node leads to its first child that holds it. One workgroup per sequence, a thread to a node.
__global__ __launch_bounds__(256) void verify_walk_kernel(const Verify a, const int32_t* drawn) {
  __shared__ int next;
  const int b = blockIdx.x, t = threadIdx.x, T = a.T;
  const bool node = t < T;
  const int parent = node ? a.parents[b * a.ldp + t] : -2;
  const int64_t token = node ? a.tokens[(int64_t)b * T + t] : -1;
  if (node) a.nodes[(int64_t)b * T + t] = -1;
  __syncthreads();
  const bool none = a.parents[b * a.ldp] < -1;           // no root
  int at = 0, n = none ? 0 : 1, got = none ? -1 : drawn[(int64_t)b * T];
  if (!none && t == 0) a.nodes[(int64_t)b * T] = 0;
  while (n > 0 && got >= 0) {                            // (ends: a child's index is larger than its parent's)
    __syncthreads();
    if (t == 0) next = T;
    __syncthreads();
    if (node && t > at && parent == at && token == got) atomicMin(&next, t);
    __syncthreads();
    if (next == T) break;
    at = next;
    got = drawn[(int64_t)b * T + at];
    if (t == 0) a.nodes[(int64_t)b * T + n] = at;
    ++n;
  }
  if (t == 0) { a.out_counts[b] = n; a.out_token[b] = got; }
}

// ---- drafted blocks ------------------------------------------------------------------------------
// Where a block's verification ended: row n of the target, and what the next token is drawn from.
struct Ended { int n, mode, token, rest; double c, mp, sp, mq, sq; };
enum : int { ENDED_KNOWN = 0, ENDED_P = 1, ENDED_ROW = 2, ENDED_POINT = 3 };   // token known; p; max(p - q, 0), q a row or one token

// The largest logit and the sum of a row by one wave.
__device__ __forceinline__ void wave_row(const Part* parts, int nch, double c, double& m, double& s, int& arg, bool& bad) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  bool odd = false;
  for (int i = lane; i < nch; i += 64) {
    const float x = parts[i].m;
    odd |= x != x;
    top = fmaxf(top, x);
  }
  top = wave_max(top);
  bad = wave_or(odd) || top == -INFINITY;
  m = top;
  s = 0.0;
  arg = -1;
  if (bad) return;
  if (c == 0.0) {
    int first = INT32_MAX;
    for (int i = lane; i < nch; i += 64)
      if (parts[i].m == top) first = min(first, parts[i].arg);
    arg = wave_min(first);
  } else {
    for (int i = lane; i < nch; i += 64) s += part_sum(parts[i], m, c);
    s = wave_sum64(s);
  }
}

// Accepts drafted tokens in order: one workgroup of 16 waves per sequence, a wave to a row at a time.
template <typename T> __global__ __launch_bounds__(1024) void verify_accept_kernel(const Verify a, Ended* ended) {
  __shared__ Ended rows[VERIFY_NODES + 1];
  __shared__ bool stop[VERIFY_NODES + 1];
  const int b = blockIdx.x, wid = threadIdx.x >> 6, lane = threadIdx.x & 63, L = a.T, n = drafted(a, b);
  const double c = rate(a, b);
  const Part* targets = a.parts + (int64_t)b * (L + 1) * a.nch;
  const Part* drafts = a.parts + ((int64_t)a.B * (L + 1) + (int64_t)b * L) * a.nch;
  for (int i = wid; i <= n; i += 16) {
    Ended e{i, ENDED_P, -1, 0, c, 0.0, 1.0, 0.0, 1.0};
    bool bad, stops = true;
    int arg;
    wave_row(targets + (int64_t)i * a.nch, a.nch, c, e.mp, e.sp, arg, bad);
    const int64_t x = i < n ? a.tokens[(int64_t)b * L + i] : -1;
    const bool in = x >= 0 && x < a.V;
    if (bad) e.mode = ENDED_KNOWN;
    else if (c == 0.0) {
      e.mode = ENDED_KNOWN;
      e.token = arg;
      stops = !(i < n && x == arg);
    } else if (i < n) {
      const T* z = (const T*)a.z + ((int64_t)b * (L + 1) + i) * a.ldz;
      const double p = in ? weight(at(z, (int)x), e.mp, c) / e.sp : 0.0;
      double q = in ? 1.0 : 0.0;
      e.mode = ENDED_POINT;
      e.token = in ? (int)x : -1;
      if (a.y) {
        wave_row(drafts + (int64_t)i * a.nch, a.nch, c, e.mq, e.sq, arg, bad);
        e.mode = ENDED_ROW;
        if (bad) { e.mode = ENDED_KNOWN; e.token = -1; }
        else q = in ? weight(at((const T*)a.y + ((int64_t)b * L + i) * a.ldy, (int)x), e.mq, c) / e.sq : 0.0;
      }
      stops = bad || !(random_at(a, (int64_t)b * (L + 1) + i) * q < p);
    }
    if (lane == 0) { rows[i] = e; stop[i] = stops; }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int i = 0;
    while (i < n && !stop[i]) ++i;
    ended[b] = rows[i];
    a.out_counts[b] = i;
    a.out_token[b] = rows[i].mode == ENDED_KNOWN ? rows[i].token : -1;
  }
}

// p and what is left of it at column j.
template <typename T> struct Left {
  const T *z, *y;
  Ended e;
  __device__ __forceinline__ Left(const Verify& a, const Ended& e_, int b) : e(e_) {
    z = (const T*)a.z + ((int64_t)b * (a.T + 1) + e.n) * a.ldz;
    y = e.mode == ENDED_ROW ? (const T*)a.y + ((int64_t)b * a.T + e.n) * a.ldy : nullptr;
  }
  __device__ __forceinline__ double p(int j) const { return weight(at(z, j), e.mp, e.c) / e.sp; }
  __device__ __forceinline__ double left(int j) const {
    const double x = p(j);
    if (e.mode == ENDED_P) return x;
    if (e.mode == ENDED_POINT) return j == e.token ? 0.0 : x;
    const double d = x - weight(at(y, j), e.mq, e.c) / e.sq;
    return d > 0.0 ? d : 0.0;
  }
};

// Sums of p and of what is left of it, a wave to a chunk: grid (chunks / 4, sequences).
template <typename T> __global__ __launch_bounds__(256) void verify_left_kernel(const Verify a, const Ended* ended, double2* sums) {
  const int b = blockIdx.y, chunk = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (chunk >= a.nch || ended[b].mode == ENDED_KNOWN) return;
  const Left<T> row(a, ended[b], b);
  const Chunks<T> cs(row.z, a.V, a.nch);
  const int lo = cs.lo(chunk), hi = cs.hi(chunk);
  double p = 0.0, left = 0.0;
  for (int j = lo + lane; j < hi; j += 64) {
    p += row.p(j);
    left += row.left(j);
  }
  p = wave_sum64(p);
  left = wave_sum64(left);
  if (lane == 0) sums[(int64_t)b * a.nch + chunk] = make_double2(left, p);
}

// The next token: one workgroup per sequence.
template <typename T> __global__ __launch_bounds__(256) void verify_next_kernel(const Verify a, const Ended* ended, const double2* sums) {
  __shared__ Shared sh;
  const int b = blockIdx.x;
  if (ended[b].mode == ENDED_KNOWN) return;
  Left<T> row(a, ended[b], b);
  const double2* mine = sums + (int64_t)b * a.nch;
  double l = 0.0, p = 0.0, left, whole, start;
  for (int i = threadIdx.x; i < a.nch; i += 256) { l += mine[i].x; p += mine[i].y; }
  (void)scan64(l, sh, left);
  (void)scan64(p, sh, whole);
  if (left < LEAST) row.e.mode = ENDED_P;
  const bool all = row.e.mode == ENDED_P;
  const double t = random_at(a, (int64_t)b * (a.T + 1) + a.T) * (all ? whole : left);
  const int ch = pick(0, a.nch, 0.0, t, sh, [&](int i) { return all ? mine[i].y : mine[i].x; }, start);
  const Chunks<T> cs(row.z, a.V, a.nch);
  const int token = ch < 0 ? -1 : pick(cs.lo(ch), cs.hi(ch), start, t, sh, [&](int j) { return row.left(j); }, start);
  if (threadIdx.x == 0) a.out_token[b] = token;
}

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
  return ((int64_t)B * T * (chunks_of(V) * (int64_t)sizeof(Part) + (int64_t)sizeof(int32_t)) + 15) / 16 * 16;
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
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(rows * ((a.nch + 3) / 4))), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, true>), grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_draw_kernel<E>, dim3((unsigned)rows), block, 0, st, a, drawn);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  hipLaunchKernelGGL(verify_walk_kernel, dim3((unsigned)B), block, 0, st, a, drawn);
  return unok::check_launch("verify_tree");
}

UNOK_EXPORT int64_t unok_verify_draft_workspace(int dtype, int B, int L, int V) {
  if (verify_sizes_ok("verify_draft", dtype, B, L, V, (int64_t)B * (2 * L + 1))) return -1;
  return (int64_t)B * ((2 * L + 1) * chunks_of(V) * (int64_t)sizeof(Part) + chunks_of(V) * (int64_t)sizeof(double2) +
                       (int64_t)sizeof(Ended));
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
  Ended* ended = (Ended*)(sums + (int64_t)B * a.nch);
  hipStream_t st = (hipStream_t)stream;
  const int groups = (a.nch + 3) / 4;
  const dim3 grid((unsigned)((targets + (y ? drafts : 0)) * groups)), block(256);
  auto run = [&](auto e) {
    using E = decltype(e);
    hipLaunchKernelGGL((verify_parts_kernel<E, false>), grid, block, 0, st, a);
    hipLaunchKernelGGL(verify_accept_kernel<E>, dim3((unsigned)B), dim3(1024), 0, st, a, ended);
    hipLaunchKernelGGL(verify_left_kernel<E>, dim3((unsigned)groups, (unsigned)B), block, 0, st, a, ended, sums);
    hipLaunchKernelGGL(verify_next_kernel<E>, dim3((unsigned)B), block, 0, st, a, ended, sums);
  };
  if (dtype == UNOK_BF16) run(bf16_t{});
  else run(float{});
  return unok::check_launch("verify_draft");
}
