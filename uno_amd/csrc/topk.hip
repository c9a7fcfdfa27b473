// The top logits of a row, and the distillation loss from a teacher's top logits.
#include "common.h"
#include "../../include/unok.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// 16 bytes of a row as floats: 8 bf16 or 4 fp32 values.
template <typename T> constexpr int VN = 16 / (int)sizeof(T);
template <typename T> __device__ __forceinline__ void unpack16(const u32x4_t u, float (&v)[VN<T>]) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
  }
}
template <typename T> __device__ __forceinline__ u32x4_t pack16(const float (&v)[VN<T>]) {
  if constexpr (std::is_same<T, float>::value)
    return u32x4_t{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
  else
    return u32x4_t{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7])};
}

// A span of n elements at p as: head elements up to the first 16-byte boundary, nv vectors of 16 bytes, the rest.
template <typename T> struct Span {
  int head, nv;
  __device__ __forceinline__ Span(const T* p, int n) {
    head = (int)(((16 - ((uintptr_t)p & 15)) & 15) / sizeof(T));
    head = head < n ? head : n;
    nv = (n - head) / VN<T>;
  }
  __device__ __forceinline__ int tail() const { return head + nv * VN<T>; }
};

// Values as unsigned keys in torch.topk's order: NaN above +inf, -0 equal to 0. No value has key 0.
__device__ __forceinline__ uint32_t value_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// Maximum over the wave, by data-parallel moves; the same value in every lane.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#define TK_MAX_STEP(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xf, false))
  TK_MAX_STEP(0x111, 0xf);                               // row_shr 1, 2, 4, 8
  TK_MAX_STEP(0x112, 0xf);
  TK_MAX_STEP(0x114, 0xf);
  TK_MAX_STEP(0x118, 0xf);
  TK_MAX_STEP(0x142, 0xa);                               // row_bcast 15 into rows 1 and 3
  TK_MAX_STEP(0x143, 0xc);                               // row_bcast 31 into rows 2 and 3
#undef TK_MAX_STEP
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// The greatest t with at least k of the wave's N x 64 values v >= t, where `on` (0: a value that does not count, which no t
// may reach); 0 if fewer than k count. SH low bits of t are not looked for: they are those of every value.
template <int N, int SH>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&v)[N], int used, int k) {
  uint32_t top = 0, low = 0;                             // low: ~ of the least value that counts
#pragma unroll
  for (int j = 0; j < N; ++j) {
    top = max(top, v[j]);
    low = max(low, v[j] == 0 ? 0u : ~v[j]);
  }
  uint32_t hi = wave_umax(top) >> SH, lo = (~wave_umax(low)) >> SH;
  if (hi == 0) return 0;
  // invariant: at least k values >= lo, or lo is the least value
  while (lo < hi) {
    const uint32_t mid = lo + (hi - lo + 1) / 2;
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < used) n += __popcll(__ballot((v[j] >> SH) >= mid));
    if (n >= k) lo = mid;
    else hi = mid - 1;
  }
  return lo << SH;
}

// Candidates of one wave: (value key, ~column) pairs in CAP entries of LDS, of which the wave's k largest are
// always among the first `cnt`. Nothing with a value key <= `floor` can still enter the k largest.
constexpr int TK_CAP = 512, TK_KEEP = 384, TK_MAX = 256;

// SH: value keys differ in their upper 32 - SH bits only (bf16: 16).
template <int SH> struct Candidates {
  uint64_t* buf;
  int lane, k, cnt;
  uint32_t floor, next_floor;

  __device__ __forceinline__ Candidates(uint64_t* b, int l, int kk) : buf(b), lane(l), k(kk), cnt(0), floor(0), next_floor(0) {}

  // Appends the lanes' candidates with `on`; drops what cannot be among the k largest when the room ends.
  __device__ __forceinline__ void push(bool on, uint32_t key, uint32_t col) {
    on = on && key > floor;
    const uint64_t mask = __ballot(on);
    if (mask == 0) return;
    if (on) buf[cnt + lanes_below(mask)] = ((uint64_t)key << 32) | (uint32_t)~col;
    cnt += __popcll(mask);
    if (cnt > TK_CAP - 64) cut(false);
  }

  // Between two steps all candidates lie left of what follows, so of equal values only the old ones count.
  __device__ __forceinline__ void step_end() { floor = next_floor > floor ? next_floor : floor; }

  // Keeps the entries whose value is among the k largest, ties included; with `exact`, or when ties leave more than
  // TK_KEEP, the k largest entries and no more.
  __device__ __forceinline__ void cut(bool exact) {
    if (cnt <= k) return;
    constexpr int NE = TK_CAP / 64;
    const int used = (cnt + 63) / 64;
    uint32_t hi[NE], lo[NE];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      const int i = j * 64 + lane;
      const uint64_t e = i < cnt ? buf[i] : 0;
      hi[j] = (uint32_t)(e >> 32);
      lo[j] = (uint32_t)e;
    }
    uint32_t t = kth_largest<NE, SH>(hi, used, k);
    if (SH > 0) {                                        // the low bits: ones for negative values (and NaN), zeros for others
      uint32_t low = 0;
#pragma unroll
      for (int j = 0; j < NE; ++j) low = max(low, (hi[j] >> SH) == (t >> SH) ? hi[j] : 0u);
      t = wave_umax(low);
    }
    int above = 0, tied = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      if (j >= used) continue;
      above += __popcll(__ballot(hi[j] > t));
      tied += __popcll(__ballot(hi[j] == t));
    }
    uint32_t u = 0;                                    // least ~column of the kept ties
    if (above + tied > k && (exact || above + tied > TK_KEEP)) {
      uint32_t tie[NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) tie[j] = hi[j] == t ? lo[j] : 0u;
      u = kth_largest<NE, 0>(tie, used, k - above);
    }
    __builtin_amdgcn_wave_barrier();
    int at = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) {
      if (j >= used) continue;
      const bool keep = hi[j] > t || (hi[j] == t && lo[j] >= u);
      const uint64_t mask = __ballot(keep);
      if (keep) buf[at + lanes_below(mask)] = ((uint64_t)hi[j] << 32) | lo[j];
      at += __popcll(mask);
    }
    __builtin_amdgcn_wave_barrier();
    cnt = at;
    floor = t - 1 > floor ? t - 1 : floor;
    next_floor = t;
  }
};

// The least float that may pass `floor` (a value equal to the result passes the first test, and push decides).
__device__ __forceinline__ float floor_value(uint32_t floor) {
  if (floor == 0) return __uint_as_float(0xff800000u);            // -inf: everything passes
  return key_value(floor);
}

// Merges the waves' candidates of a row: every wave leaves its at most k largest, and an entry's rank is the number
// of larger entries.
template <int SH, typename F>
__device__ __forceinline__ void rank_entries(uint64_t* all, int* wave_cnt, Candidates<SH>& c, int k, int wid, F emit) {
  c.cut(true);
  if (c.lane == 0) wave_cnt[wid] = c.cnt;
  __syncthreads();
  const int n0 = wave_cnt[0], n1 = n0 + wave_cnt[1], n2 = n1 + wave_cnt[2], n3 = n2 + wave_cnt[3];
  for (int i = threadIdx.x; i < n3; i += 256) {
    const int w = (i >= n0) + (i >= n1) + (i >= n2);
    const uint64_t e = all[w * TK_CAP + i - (w == 0 ? 0 : w == 1 ? n0 : w == 2 ? n1 : n2)];
    int rank = 0;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int n = wave_cnt[v];
#pragma unroll 8
      for (int q = 0; q < n; ++q) rank += all[v * TK_CAP + q] > e;
    }
    if (rank < k) emit(rank, e);
  }
}

// The k largest of a row's columns [c0, c0 + width) and the part's softmax statistics, one workgroup per (row, part).
// parts == 1 writes values, columns and log-sum-exp; otherwise the part's sorted entries (missing ones 0) and
// (max, sum of e^(z - max)) go to the workspace for topk_merge_kernel.
//
// One pass: a wave takes every fourth step of 4 x 64 16-byte loads. A group of 16 bytes is looked into only
// if its largest value can pass the wave's floor; the first step sets the floor to the k-th largest of its
// 256 groups' maxima (each is one element, so k elements reach it).
template <typename T>
__global__ __launch_bounds__(256) void row_topk_kernel(const T* __restrict__ z, int64_t ldz, int V, int k, int parts,
                                                       int width, float* __restrict__ values, int64_t* __restrict__ cols,
                                                       float* __restrict__ lse, uint64_t* __restrict__ ws_key,
                                                       float2* __restrict__ ws_stat) {
  constexpr int U = 4, N = VN<T>, STEP = 64 * U;       // vectors per step
  __shared__ uint64_t buf[4 * TK_CAP];
  __shared__ float red[32];
  __shared__ int wave_cnt[4];
  __shared__ uint32_t bound_[4];                         // per wave: a value key that k of its elements reach
  volatile uint32_t* bound = bound_;
  if (threadIdx.x < 4) bound[threadIdx.x] = 0;
  __syncthreads();
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int c0 = part * width, n = min(width, V - c0);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const T* p = z + row * ldz + c0;
  const Span<T> sp(p, n);
  constexpr int SH = sizeof(T) == 2 ? 16 : 0;
  Candidates<SH> cand(buf + wid * TK_CAP, lane, k);
  float m = -INFINITY, s = 0.f;

  constexpr uint32_t NOTHING = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;   // -inf
  // elements outside the vectors: the head by wave 0 before its steps, the tail by wave 3 after its steps
  auto single = [&](int first, int cnt) {
    for (int i = 0; i < cnt; i += 64) {
      const bool in = i + lane < cnt;
      const float v = in ? Elem<T>::load(p + first + i + lane) : -INFINITY;
      cand.push(in, value_key(v), (uint32_t)(c0 + first + i + lane));
      if (v > m) { s *= fast_expf(m - v); m = v; }
      s += fast_expf(v - (m == -INFINITY ? 0.f : m));
      cand.step_end();
    }
  };
  if (wid == 0) single(0, sp.head);
  const u32x4_t* pv = (const u32x4_t*)(p + sp.head);
  bool fresh = true;
  for (int q0 = wid * STEP; q0 < sp.nv; q0 += 4 * STEP) {
    u32x4_t raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int q = q0 + i * 64 + lane;
      raw[i] = q < sp.nv ? pv[q] : u32x4_t{NOTHING, NOTHING, NOTHING, NOTHING};
    }
    float gm[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float v[N];
      unpack16<T>(raw[i], v);
      gm[i] = v[0];
#pragma unroll
      for (int e = 1; e < N; ++e) gm[i] = fmaxf(gm[i], v[e]);
      if (gm[i] > m) { s *= fast_expf(m - gm[i]); m = gm[i]; }
      const float ref = m == -INFINITY ? 0.f : m;      // -inf then adds 0, and a NaN is seen
#pragma unroll
      for (int e = 0; e < N; ++e) s += fast_expf(v[e] - ref);
    }
    // what the other waves have found by now spares this one candidates (whenever it is seen: the k largest are
    // the same)
    const uint32_t others = max(max(bound[0], bound[1]), max(bound[2], bound[3]));
    if (others > 0 && others - 1 > cand.floor) cand.floor = others - 1;
    if (fresh) {
      fresh = false;
      uint32_t key[U];
      int cnt = 0;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        key[i] = q0 + i * 64 + lane < sp.nv ? value_key(gm[i]) : 0u;
        cnt += __popcll(__ballot(key[i] != 0));
      }
      if (cnt >= k) {
        const uint32_t t = kth_largest<U, SH>(key, U, k);  // (its low bits zero: a bound all the same)
        if (t > 0 && t - 1 > cand.floor) cand.floor = t - 1;
        if (lane == 0) bound[wid] = t;
      }
    }
    // bit 8 i + e (fp32: 4 i + e): element e of vector i may enter. (A lane that has met a NaN, which fmaxf
    // drops, looks into every vector from then on.)
    const float least = floor_value(cand.floor);
    uint32_t may = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool look = q0 + i * 64 + lane < sp.nv && (!(gm[i] < least) || s != s);
      if (__ballot(look) == 0) continue;
      float v[N];
      unpack16<T>(raw[i], v);
#pragma unroll
      for (int e = 0; e < N; ++e) may |= look && !(v[e] < least) ? 1u << (i * N + e) : 0u;
    }
    while (__ballot(may != 0)) {
      const int at = may ? __builtin_ctz(may) : 0;
      uint32_t w = raw[0][0];
      const int word = at * (int)sizeof(T) / 4;
#pragma unroll
      for (int i = 0; i < 4 * U; ++i) w = word == i ? raw[i / 4][i % 4] : w;
      if constexpr (sizeof(T) == 2) w = at & 1 ? w & 0xffff0000u : w << 16;
      cand.push(may != 0, value_key(__uint_as_float(w)), (uint32_t)(c0 + sp.head + (q0 + (at / N) * 64 + lane) * N + at % N));
      may &= may - 1;
    }
    cand.step_end();
    if (lane == 0 && cand.next_floor > bound[wid]) bound[wid] = cand.next_floor;
  }
  if (wid == 3) single(sp.tail(), n - sp.tail());

  const float mb = block_max(m, red);
  s = block_sum(m == -INFINITY ? s : s * fast_expf(m - mb), red);
  if (parts == 1) {
    rank_entries(buf, wave_cnt, cand, k, wid, [&](int rank, uint64_t e) {
      const float v = key_value((uint32_t)(e >> 32));
      values[row * k + rank] = v;
      cols[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)e;
      // a NaN, +inf or nothing but -inf decides the sum
      if (rank == 0) lse[row] = v - v == 0.f ? mb + logf(s) : v;
    });
  } else {
    uint64_t* o = ws_key + ((int64_t)row * parts + part) * k;
    if (threadIdx.x == 0) ws_stat[row * parts + part] = make_float2(mb, s);
    for (int i = threadIdx.x; i < k; i += 256)
      if (i >= n) o[i] = 0;
    rank_entries(buf, wave_cnt, cand, k, wid, [&](int rank, uint64_t e) { o[rank] = e; });
  }
}

// The parts' entries and statistics of a row, merged; one workgroup per row.
__global__ __launch_bounds__(256) void topk_merge_kernel(const uint64_t* __restrict__ ws_key,
                                                         const float2* __restrict__ ws_stat, int k, int parts,
                                                         float* __restrict__ values, int64_t* __restrict__ cols,
                                                         float* __restrict__ lse) {
  __shared__ uint64_t buf[4 * TK_CAP];
  __shared__ float red[32];
  __shared__ int wave_cnt[4];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const uint64_t* src = ws_key + row * parts * k;
  const int n = parts * k;
  Candidates<0> cand(buf + wid * TK_CAP, lane, k);
  for (int i = wid * 64; i < n; i += 256) {
    const uint64_t e = i + lane < n ? src[i + lane] : 0;
    cand.push(e != 0, (uint32_t)(e >> 32), ~(uint32_t)e);
  }
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x; i < parts; i += 256) {
    const float2 st = ws_stat[row * parts + i];
    if (st.x > m) { s = s * fast_expf(m - st.x) + st.y; m = st.x; }
    else if (st.x > -INFINITY) s += st.y * fast_expf(st.x - m);
  }
  const float mb = block_max(m, red);
  s = block_sum(m == -INFINITY ? s : s * fast_expf(m - mb), red);
  rank_entries(buf, wave_cnt, cand, k, wid, [&](int rank, uint64_t e) {
    const float v = key_value((uint32_t)(e >> 32));
    values[row * k + rank] = v;
    cols[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)e;
    if (rank == 0) lse[row] = v - v == 0.f ? mb + logf(s) : v;
  });
}

// Parts of a row: with fewer rows than fill the chip (two workgroups per CU), as many as do, of at least 4096 columns.
int topk_parts(int R, int V) {
  const int want = (512 + R - 1) / (R > 0 ? R : 1), most = V / 4096;
  const int p = want < most ? want : most;
  return p < 1 ? 1 : p;
}

// ---------------------------------------------------------------------------------------
// Distillation from a teacher's top logits. Row r: teacher logits t_i at columns idx_i (entries with t_i = -inf or
// a column outside the vocabulary do not count), p = softmax(t / tau) over them, q = softmax(z / tau) over all
// columns:
//   L = tau^2 inv_n sum_r sum_i p_i (log p_i - log q_idx_i)
//   dL/dz_j = tau inv_n (q_j - sum_{i: idx_i = j} p_i), zero in a row without an entry.
// ---------------------------------------------------------------------------------------
constexpr int DK_MAX = 256;

// The entries of a row as a wave sees them, entry lane + 64 i in step i: columns (-1: does not count) and the
// logarithms of their probabilities; returns whether there is any.
template <typename F>
__device__ __forceinline__ bool teacher_row(const float* __restrict__ t, const int64_t* __restrict__ idx, int k, int V,
                                            float inv_tau, int lane, F use) {
  float x[DK_MAX / 64];
  int col[DK_MAX / 64];
  float m = -INFINITY;
  bool any = false;
#pragma unroll
  for (int i = 0; i < DK_MAX / 64; ++i) {
    const int e = lane + 64 * i;
    col[i] = -1;
    x[i] = -INFINITY;
    if (e < k) {
      const int64_t c = idx[e];
      const float v = t[e] * inv_tau;
      if (c >= 0 && c < V && !(v == -INFINITY)) { col[i] = (int)c; x[i] = v; m = fmaxf(m, v); any = true; }
    }
  }
  if (__ballot(any) == 0) return false;
  m = wave_max(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < DK_MAX / 64; ++i)
    if (col[i] >= 0) s += expf(x[i] - m);
  s = wave_sum(s);
  const float l = m + logf(s);
#pragma unroll
  for (int i = 0; i < DK_MAX / 64; ++i) use(lane + 64 * i, col[i], x[i] - l);
  return true;
}

// sum_i p_i (log p_i - log q_i) of a row, in one wave, from the row's (max, sum of e^(z / tau - max)).
template <typename T>
__device__ __forceinline__ float distill_row(const T* __restrict__ z, const float* __restrict__ t,
                                             const int64_t* __restrict__ idx, int k, int V, float inv_tau, int lane, float m,
                                             float s) {
  const float l = logf(s);
  float acc = 0.f;
  teacher_row(t, idx, k, V, inv_tau, lane, [&](int, int col, float logp) {
    if (col < 0) return;
    const float pr = expf(logp);
    if (!(pr == 0.f)) acc += pr * (logp - (Elem<T>::load(z + col) * inv_tau - m) + l);
  });
  return wave_sum(acc);
}

// (max, sum of e^(x - max)) of x = z / tau over a part of a row; one workgroup per (row, part). A row in one part also gets
// its loss. Bound by HBM.
template <typename T>
__global__ __launch_bounds__(256) void distill_stats_kernel(const T* __restrict__ z, int64_t ldz, int V, int parts,
                                                            int width, int k, const float* __restrict__ t,
                                                            const int64_t* __restrict__ idx, float inv_tau,
                                                            float2* __restrict__ stat, float* __restrict__ row_loss) {
  constexpr int N = VN<T>;
  __shared__ float red[32];
  const int64_t row = blockIdx.x / parts;
  const int c0 = (int)(blockIdx.x % parts) * width, n = min(width, V - c0);
  const T* p = z + row * ldz + c0;
  const Span<T> sp(p, n);
  float m = -INFINITY, s = 0.f;
  const u32x4_t* pv = (const u32x4_t*)(p + sp.head);
  for (int q = threadIdx.x; q < sp.nv; q += 256) {
    float v[N];
    unpack16<T>(pv[q], v);
    float g = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) { v[e] *= inv_tau; g = fmaxf(g, v[e]); }
    if (g > m) { s *= fast_expf(m - g); m = g; }
    const float ref = m == -INFINITY ? 0.f : m;        // -inf then adds 0, and a NaN is seen
#pragma unroll
    for (int e = 0; e < N; ++e) s += fast_expf(v[e] - ref);
  }
  auto single = [&](float v) {
    if (v > m) { s *= fast_expf(m - v); m = v; }
    s += fast_expf(v - (m == -INFINITY ? 0.f : m));
  };
  for (int j = threadIdx.x; j < sp.head; j += 256) single(Elem<T>::load(p + j) * inv_tau);
  for (int j = sp.tail() + threadIdx.x; j < n; j += 256) single(Elem<T>::load(p + j) * inv_tau);
  const float mb = block_max(m, red);
  s = block_sum(m == -INFINITY ? s : s * fast_expf(m - mb), red);
  if (threadIdx.x == 0) stat[blockIdx.x] = make_float2(mb, s);
  if (parts == 1 && threadIdx.x < 64) {
    const float loss = distill_row(p, t + row * k, idx + row * k, k, V, inv_tau, threadIdx.x, mb, s);
    if (threadIdx.x == 0) row_loss[row] = loss;
  }
}

// The same for rows in several parts. One wave per row.
template <typename T>
__global__ __launch_bounds__(256) void distill_rows_kernel(const T* __restrict__ z, int64_t ldz, int R, int V, int parts,
                                                           int k, const float2* __restrict__ stat,
                                                           const float* __restrict__ t, const int64_t* __restrict__ idx,
                                                           float inv_tau, float2* __restrict__ row_stat,
                                                           float* __restrict__ row_loss) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (row >= R) return;
  float m = -INFINITY, s = 0.f;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, stat[row * parts + i].x);
  m = wave_max(m);
  for (int i = lane; i < parts; i += 64) {
    const float2 st = stat[row * parts + i];
    s += st.x == -INFINITY ? st.y : st.y * fast_expf(st.x - m);
  }
  s = wave_sum(s);
  const float loss = distill_row(z + row * ldz, t + row * k, idx + row * k, k, V, inv_tau, lane, m, s);
  if (lane == 0) { row_stat[row] = make_float2(m, s); row_loss[row] = loss; }
}

// loss = scale inv_n sum of the rows' losses, in a fixed order (one workgroup).
__global__ __launch_bounds__(1024) void distill_sum_kernel(int R, const float* __restrict__ row_loss,
                                                           const float* __restrict__ inv_n, float scale, float* loss) {
  __shared__ float red[32];
  float acc = 0.f;
  for (int r = threadIdx.x; r < R; r += 1024) acc += row_loss[r];
  acc = block_sum(acc, red);
  if (threadIdx.x == 0) loss[0] = acc * scale * (inv_n ? inv_n[0] : 1.f);
}

// grad = g inv_n scale (q - p) of a part of a row; grad may be z itself. The entries' columns are written after the
// barrier, once more, from the logits read before it: entries that name the same column each write the sum of
// all their probabilities.
template <typename T>
__global__ __launch_bounds__(256) void distill_bwd_kernel(const T* z, int64_t ldz, int V, int parts, int width, int k,
                                                          const float2* __restrict__ row_stat, const float* __restrict__ t,
                                                          const int64_t* __restrict__ idx, float inv_tau,
                                                          const float* __restrict__ gscale, const float* __restrict__ inv_n,
                                                          float scale,
                                                          T* grad, int64_t ldg) {
  constexpr int N = VN<T>;
  __shared__ int cols[DK_MAX];
  __shared__ float prob[DK_MAX];
  __shared__ int live;
  const int64_t row = blockIdx.x / parts;
  const int c0 = (int)(blockIdx.x % parts) * width, n = min(width, V - c0);
  const T* p = z + row * ldz + c0;
  T* g = grad + row * ldg + c0;
  if (threadIdx.x < 64) {
    const bool any = teacher_row(t + row * k, idx + row * k, k, V, inv_tau, threadIdx.x, [&](int e, int col, float logp) {
      cols[e] = col;
      prob[e] = col < 0 ? 0.f : expf(logp);
    });
    if (threadIdx.x == 0) live = any;
  }
  __syncthreads();
  const Span<T> sp(p, n);
  const bool aligned = (((uintptr_t)p ^ (uintptr_t)g) & 15) == 0;   // both reach 16-byte boundaries together
  if (!live) {
    for (int j = threadIdx.x; j < n; j += 256) Elem<T>::store(g + j, 0.f);
    return;
  }
  const float2 rs = row_stat[row];
  const float c = gscale[0] * scale * (inv_n ? inv_n[0] : 1.f), m = rs.x, cq = c / rs.y;
  // the entry of this thread in this part: its logit, and the sum of the probabilities at its column
  const int col = threadIdx.x < (unsigned)k ? cols[threadIdx.x] - c0 : -1;
  const bool mine = col >= 0 && col < n;
  float zc = 0.f, psum = 0.f;
  if (mine) {
    zc = Elem<T>::load(p + col);
    for (int e = 0; e < k; ++e) psum += cols[e] == col + c0 ? prob[e] : 0.f;
  }
  __syncthreads();
  auto one = [&](float v) { return cq * fast_expf(v * inv_tau - m); };
  if (aligned) {
    const u32x4_t* pv = (const u32x4_t*)(p + sp.head);
    u32x4_t* gv = (u32x4_t*)(g + sp.head);
    for (int q = threadIdx.x; q < sp.nv; q += 256) {
      float v[N];
      unpack16<T>(pv[q], v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = one(v[e]);
      gv[q] = pack16<T>(v);
    }
    for (int j = threadIdx.x; j < sp.head; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
    for (int j = sp.tail() + threadIdx.x; j < n; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
  } else {
    for (int j = threadIdx.x; j < n; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the columns' first values are stored before the second ones
  __syncthreads();
  if (mine) Elem<T>::store(g + col, fast_expf(zc * inv_tau - m) / rs.y * c - psum * c);
}

// Parts of a row of the statistics and the gradient, as topk_parts, of at least 8192 columns.
int distill_parts(int R, int V) {
  const int want = (1024 + R - 1) / (R > 0 ? R : 1), most = V / 8192;
  const int p = want < most ? want : most;
  return p < 1 ? 1 : p;
}

void distill_split(int R, int V, int& parts, int& width) {
  parts = distill_parts(R, V);
  width = ((V + parts - 1) / parts + 7) / 8 * 8;
  parts = (V + width - 1) / width;                     // a last part may fall away by the rounding
}

int distill_check(const char* what, int dtype, int R, int V, int k, int64_t ldz, float tau) {
  UNOK_REQUIRE(R >= 0 && V >= 1 && (R <= 1 || ldz >= V), UNOK_EINVAL, "%s: R=%d V=%d ldz=%lld", what, R, V, (long long)ldz);
  UNOK_REQUIRE(k >= 1 && k <= DK_MAX, UNOK_EINVAL, "%s: k=%d must lie in [1, %d]", what, k, DK_MAX);
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "%s: bad dtype %d", what, dtype);
  UNOK_REQUIRE(tau > 0.f && tau < INFINITY, UNOK_EINVAL, "%s: temperature %g must be positive", what, (double)tau);
  return 0;
}

}  // namespace

UNOK_EXPORT int64_t unok_row_topk_workspace(int R, int V, int k) {
  if (R <= 0 || V <= 0 || k <= 0) return 0;
  const int64_t parts = topk_parts(R, V);
  return parts == 1 ? 0 : R * parts * (8ll * k + 8);
}

UNOK_EXPORT int unok_row_topk(int dtype, int R, int V, int k, const void* z, int64_t ldz, float* values, int64_t* cols,
                              float* lse, void* workspace, int64_t ws_bytes, void* stream) {
  UNOK_REQUIRE(R >= 0 && V >= 0 && (R <= 1 || ldz >= V), UNOK_EINVAL, "row_topk: R=%d V=%d ldz=%lld", R, V, (long long)ldz);
  UNOK_REQUIRE(k >= 1 && k <= TK_MAX && k <= V, UNOK_EINVAL, "row_topk: k=%d must lie in [1, min(%d, V=%d)]", k, TK_MAX, V);
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "row_topk: bad dtype %d", dtype);
  if (R == 0) return 0;
  UNOK_REQUIRE(z && values && cols && lse, UNOK_EINVAL, "row_topk: null operand");
  const int parts = topk_parts(R, V);
  const int64_t need = unok_row_topk_workspace(R, V, k);
  UNOK_REQUIRE(need == 0 || (workspace && ws_bytes >= need && ((uintptr_t)workspace & 7) == 0), UNOK_EINVAL,
               "row_topk: workspace of %lld bytes (8-byte aligned) required, got %lld", (long long)need, (long long)ws_bytes);
  UNOK_REQUIRE((int64_t)R * parts < (1ll << 31), UNOK_EINVAL, "row_topk: R=%d", R);
  const int width = ((V + parts - 1) / parts + 7) / 8 * 8;
  const int used = (V + width - 1) / width;            // a last part may fall away by the rounding
  uint64_t* keys = (uint64_t*)workspace;
  float2* stat = (float2*)(keys + (int64_t)R * parts * k);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == UNOK_BF16)
    hipLaunchKernelGGL(row_topk_kernel<bf16_t>, dim3((unsigned)(R * used)), dim3(256), 0, st, (const bf16_t*)z, ldz, V, k, used,
                       width, values, cols, lse, keys, stat);
  else
    hipLaunchKernelGGL(row_topk_kernel<float>, dim3((unsigned)(R * used)), dim3(256), 0, st, (const float*)z, ldz, V, k, used,
                       width, values, cols, lse, keys, stat);
  int rc = unok::check_launch("row_topk");
  if (rc || used == 1) return rc;
  hipLaunchKernelGGL(topk_merge_kernel, dim3((unsigned)R), dim3(256), 0, st, keys, stat, k, used, values, cols, lse);
  return unok::check_launch("topk_merge");
}

UNOK_EXPORT int64_t unok_distill_workspace(int R, int V) {
  if (R <= 0 || V <= 0) return 0;
  const int64_t parts = distill_parts(R, V);
  return (int64_t)R * ((parts > 1 ? parts * 8 : 0) + 4);
}

UNOK_EXPORT int unok_distill_fwd(int dtype, int R, int V, int k, const void* z, int64_t ldz, const float* t, const int64_t* idx,
                                 float tau, const float* inv_n, float scale, float* row_stat, float* loss, void* workspace,
                                 int64_t ws_bytes, void* stream) {
  int rc = distill_check("distill_fwd", dtype, R, V, k, ldz, tau);
  if (rc) return rc;
  UNOK_REQUIRE(loss && (R == 0 || (z && t && idx && row_stat)), UNOK_EINVAL, "distill_fwd: null operand");
  const int64_t need = unok_distill_workspace(R, V);
  UNOK_REQUIRE(need == 0 || (workspace && ws_bytes >= need && ((uintptr_t)workspace & 7) == 0), UNOK_EINVAL,
               "distill_fwd: workspace of %lld bytes (8-byte aligned) required, got %lld", (long long)need, (long long)ws_bytes);
  int parts = 1, width = V;
  if (R > 0) distill_split(R, V, parts, width);
  UNOK_REQUIRE((int64_t)R * parts < (1ll << 31), UNOK_EINVAL, "distill_fwd: R=%d", R);
  float2* stat = parts > 1 ? (float2*)workspace : (float2*)row_stat;
  float* row_loss = (float*)workspace + (parts > 1 ? 2ll * R * parts : 0);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto* zt) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(zt)>>;
    hipLaunchKernelGGL(distill_stats_kernel<T>, dim3((unsigned)(R * parts)), dim3(256), 0, st, zt, ldz, V, parts, width, k, t,
                       idx, 1.f / tau, stat, row_loss);
    if (parts > 1)
      hipLaunchKernelGGL(distill_rows_kernel<T>, dim3((unsigned)((R + 3) / 4)), dim3(256), 0, st, zt, ldz, R, V, parts, k, stat,
                         t, idx, 1.f / tau, (float2*)row_stat, row_loss);
  };
  if (R > 0) {
    if (dtype == UNOK_BF16) go((const bf16_t*)z);
    else go((const float*)z);
  }
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(1024), 0, st, R, row_loss, inv_n, scale, loss);
  return unok::check_launch("distill_fwd");
}

UNOK_EXPORT int unok_distill_bwd(int dtype, int R, int V, int k, const void* z, int64_t ldz, const float* t, const int64_t* idx,
                                 float tau, const float* row_stat, const float* gscale, const float* inv_n, float scale,
                                 void* grad, int64_t ldg, void* stream) {
  int rc = distill_check("distill_bwd", dtype, R, V, k, ldz, tau);
  if (rc || R == 0) return rc;
  UNOK_REQUIRE(R <= 1 || ldg >= V, UNOK_EINVAL, "distill_bwd: ldg=%lld", (long long)ldg);
  UNOK_REQUIRE(z && t && idx && row_stat && gscale && grad, UNOK_EINVAL, "distill_bwd: null operand");
  int parts, width;
  distill_split(R, V, parts, width);
  UNOK_REQUIRE((int64_t)R * parts < (1ll << 31), UNOK_EINVAL, "distill_bwd: R=%d", R);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto* zt, auto* gt) {
    using T = std::remove_pointer_t<decltype(gt)>;
    hipLaunchKernelGGL(distill_bwd_kernel<T>, dim3((unsigned)(R * parts)), dim3(256), 0, st, zt, ldz, V, parts, width, k,
                       (const float2*)row_stat, t, idx, 1.f / tau, gscale, inv_n, scale, gt, ldg);
  };
  if (dtype == UNOK_BF16) go((const bf16_t*)z, (bf16_t*)grad);
  else go((const float*)z, (float*)grad);
  return unok::check_launch("distill_bwd");
}
