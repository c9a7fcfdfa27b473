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

// Logits of more than the memory-side cache's 256 MB are read past it (NT), as they cannot be there: 4096 x 151936 bf16
// (1.2 GB), k = 10 255 -> 239 us, and the distillation's gradient of 1024 x 151936 (311 MB) 196 -> 176 us with its forward;
// logits that fit are found there: 512 x 151936 (155 MB) 96 us when read past it, 88 when not.
constexpr int64_t MEMORY_CACHE = 256ll << 20;
template <bool NT> __device__ __forceinline__ u32x4_t load16(const u32x4_t* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
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

// The greatest t with at least k of the wave's N x 64 values v >= t (0: a value that does not count, which no t may reach; the
// callers see to it that k do, as with fewer t is the least of them). SH low bits of t are not looked for, and come as 0.
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

// Candidates of one wave of a row's four: (value key, ~column) pairs in TK_CAP entries of LDS, of which the wave's k
// largest are always among the first `cnt` unless they are known not to be among the row's. Nothing with a value
// key <= `floor` can still enter. SH: value keys differ in their upper 32 - SH bits only (bf16: 16).
//
// The waves share what they know: `whole`, a key that k of the wave's elements reach, and `quarter`, one that a quarter
// of k reach. k elements of the row reach the greatest `whole`, and the least `quarter`, which for rows without an order is
// close to the row's k-th largest value so far. (Whenever a wave sees them: the k largest are the same.)
constexpr int TK_CAP = 512, TK_KEEP = 384, TK_MAX = 256;

struct Shared { uint32_t whole[4], quarter[4]; };

#define TK_LDS __attribute__((address_space(3)))
typedef TK_LDS uint64_t* LdsKeys;
typedef TK_LDS Shared* LdsShared;

__device__ __forceinline__ uint32_t tk_read(const TK_LDS uint32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// A key that k elements of the row reach (0: none known).
__device__ __forceinline__ uint32_t known(LdsShared s) {
  uint32_t w = 0, q = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w = max(w, tk_read(&s->whole[i]));
    q = min(q, tk_read(&s->quarter[i]));
  }
  return max(w, q);
}

struct Cut { int cnt; uint32_t floor, next_floor; };

// Looks for higher keys among a wave's cnt entries and drops those below them: keeps the entries whose value is among the k
// largest, ties included; with `exact`, or when ties leave more than TK_KEEP, the k largest entries and no more. Takes
// up to 64 NE entries. Not inlined: it is rare, and four copies would not fit the instruction cache beside the walk.
template <int SH, int NE>
__device__ __attribute__((noinline)) Cut cut_candidates(LdsKeys buf, LdsShared shared, int wid, int k, int cnt, uint32_t floor,
                                                        uint32_t next_floor, bool exact) {
  const int lane = threadIdx.x & 63, quarter = (k + 3) / 4;
  cnt = __builtin_amdgcn_readfirstlane(cnt);
  k = __builtin_amdgcn_readfirstlane(k);
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
  uint32_t t = 0, u = 0;                                 // the k-th largest key; the least ~column of its kept ties
  if (cnt > k) {
    t = kth_largest<NE, SH>(hi, used, k);
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
    if (above + tied > k && (exact || above + tied > TK_KEEP)) {
      uint32_t tie[NE];
#pragma unroll
      for (int j = 0; j < NE; ++j) tie[j] = hi[j] == t ? lo[j] : 0u;
      u = kth_largest<NE, 0>(tie, used, k - above);
    }
    floor = t - 1 > floor ? t - 1 : floor;
    next_floor = t > next_floor ? t : next_floor;
  }
  if (cnt >= quarter) {
    const uint32_t q = kth_largest<NE, SH>(hi, used, quarter);
    if (lane == 0) {                                     // (both only ever grow; no other wave writes them)
      if (next_floor > tk_read(&shared->whole[wid]))
        __hip_atomic_store(&shared->whole[wid], next_floor, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (q > tk_read(&shared->quarter[wid]))
        __hip_atomic_store(&shared->quarter[wid], q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
  const uint32_t least = known(shared);
  __builtin_amdgcn_wave_barrier();
  int at = 0;
#pragma unroll
  for (int j = 0; j < NE; ++j) {
    if (j >= used) continue;
    const bool keep = hi[j] >= least && hi[j] != 0 && (hi[j] > t || (hi[j] == t && lo[j] >= u));
    const uint64_t mask = __ballot(keep);
    if (keep) buf[at + lanes_below(mask)] = ((uint64_t)hi[j] << 32) | lo[j];
    at += __popcll(mask);
  }
  __builtin_amdgcn_wave_barrier();
  if (least > 0 && least - 1 > floor) floor = least - 1;
  return Cut{at, floor, next_floor};
}

template <int SH> struct Candidates {
  LdsKeys buf;
  LdsShared shared;
  int wid, k, cnt, next;                                 // next: the count at which to look for higher keys
  uint32_t floor, next_floor;

  __device__ __forceinline__ Candidates(uint64_t* b, Shared* s, int w, int kk)
      : buf((LdsKeys)(b + w * TK_CAP)), shared((LdsShared)s), wid(w), k(kk), cnt(0), next((kk + 3) / 4), floor(0), next_floor(0) {}

  // Appends the lanes' candidates with `on`; the caller sees to it that there is room for 64.
  __device__ __forceinline__ void push(bool on, uint32_t key, uint32_t col) {
    on = on && key > floor;
    const uint64_t mask = __ballot(on);
    if (on) buf[cnt + lanes_below(mask)] = ((uint64_t)key << 32) | (uint32_t)~col;
    cnt += __popcll(mask);
  }
  __device__ __forceinline__ bool full() const { return cnt > TK_CAP - 64; }

  // Between two steps all candidates lie left of what follows, so of equal values only the old ones count.
  __device__ __forceinline__ void step_end() { floor = next_floor > floor ? next_floor : floor; }

  __device__ __forceinline__ void learn() {
    const uint32_t t = known(shared);
    if (t > 0 && t - 1 > floor) floor = t - 1;
  }
  __device__ __forceinline__ void cut(bool exact) {
    const Cut c = cnt <= 128 ? cut_candidates<SH, 2>(buf, shared, wid, k, cnt, floor, next_floor, exact)
                             : cut_candidates<SH, TK_CAP / 64>(buf, shared, wid, k, cnt, floor, next_floor, exact);
    cnt = __builtin_amdgcn_readfirstlane(c.cnt);
    floor = (uint32_t)__builtin_amdgcn_readfirstlane((int)c.floor);
    next_floor = (uint32_t)__builtin_amdgcn_readfirstlane((int)c.next_floor);
    next = cnt + (k + 3) / 4;
  }
};

// The least float that may pass `floor` (a value equal to the result passes the first test, and push decides).
__device__ __forceinline__ float floor_value(uint32_t floor) {
  if (floor == 0) return __uint_as_float(0xff800000u);            // -inf: everything passes
  return key_value(floor);
}

// Ranks n distinct entries in LDS: an entry's rank is the number of larger ones.
template <typename F> __device__ __forceinline__ void rank_entries(LdsKeys all, int n, int k, F emit) {
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t e = all[i];
    int rank = 0;
#pragma unroll 8
    for (int q = 0; q < n; ++q) rank += all[q] > e;
    if (rank < k) emit(rank, e);
  }
}

// Merges the waves' candidates of a row into the k largest in order. If the waves hold many, each first drops what the
// others' keys rule out.
template <int SH, typename F>
__device__ __forceinline__ void merge_waves(uint64_t* all, int* wave_cnt, Candidates<SH>& c, int k, F emit) {
  const int lane = threadIdx.x & 63;
  int first[4], n = 0;
  auto counts = [&] {
    if (lane == 0) wave_cnt[c.wid] = c.cnt;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      first[w] = n;
      n += wave_cnt[w];
    }
  };
  counts();
  if (n > 256) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {                        // the second time with what every wave found in the first
      if (c.cnt > 0) c.cut(i > 0);
      __syncthreads();
    }
    counts();
  }
  // dense: every entry is read before any is written
  uint64_t e[TK_CAP / 64];
#pragma unroll
  for (int j = 0; j < TK_CAP / 64; ++j) e[j] = j * 64 + lane < c.cnt ? c.buf[j * 64 + lane] : 0;
  __syncthreads();
  LdsKeys dense = (LdsKeys)all;
  const int at = c.wid == 0 ? first[0] : c.wid == 1 ? first[1] : c.wid == 2 ? first[2] : first[3];
#pragma unroll
  for (int j = 0; j < TK_CAP / 64; ++j)
    if (j * 64 + lane < c.cnt) dense[at + j * 64 + lane] = e[j];
  __syncthreads();
  rank_entries(dense, n, k, emit);
}

// The sum of e^(z - m) over a lane's elements of a row's part, as row_topk_kernel hands them out.
constexpr float TK_FAR = 1048576.f, LOG2E = 1.4426950408889634f;
template <typename T>
__device__ __attribute__((noinline)) float far_sum(const T* p, int n, Span<T> sp, int wid, int lane, float m) {
  const float ref = m == -INFINITY ? 0.f : m;
  const u32x4_t* pv = (const u32x4_t*)(p + sp.head);
  float s = 0.f;
  if (wid == 0)
    for (int i = lane; i < sp.head; i += 64) s += fast_expf(Elem<T>::load(p + i) - ref);
#pragma unroll 1
  for (int q = wid * 256 + lane; q < sp.nv; q += (q & 192) == 192 ? 1024 - 192 : 64) {   // four vectors of each step
    float v[VN<T>];
    unpack16<T>(pv[q], v);
#pragma unroll
    for (int e = 0; e < VN<T>; ++e) s += fast_expf(v[e] - ref);
  }
  if (wid == 3)
    for (int i = sp.tail() + lane; i < n; i += 64) s += fast_expf(Elem<T>::load(p + i) - ref);
  return s;
}

// The k largest of a row's columns [c0, c0 + width) and the part's softmax statistics, one workgroup per (row, part).
// parts == 1 writes values, columns and log-sum-exp; otherwise the part's sorted entries (missing ones 0) and
// (max, sum of e^(z - max)) go to the workspace for topk_merge_kernel.
//
// One pass: a wave takes every fourth step of 4 x 64 16-byte loads. A group of 16 bytes is looked into only
// if its largest value can pass the wave's floor; the first step sets the floor to the k-th largest of its
// 256 groups' maxima (each is one element, so k elements reach it). Bound by its vector instructions: unpacking, comparing,
// the exponential (4096 x 151936 bf16, k = 64: 285 us, 4.4 TB/s; with a subtraction and a product before the exponential 325;
// six waves a SIMD: with five 310, held to seven or eight 333 and 493 for spilled registers).
template <typename T, bool NT>
__global__ __launch_bounds__(256, 6) void row_topk_kernel(const T* __restrict__ z, int64_t ldz, int V, int k, int parts,
                                                       int width, float* __restrict__ values, int64_t* __restrict__ cols,
                                                       float* __restrict__ lse, uint64_t* __restrict__ ws_key,
                                                       float2* __restrict__ ws_stat) {
  constexpr int U = 4, N = VN<T>, STEP = 64 * U;       // vectors per step
  __shared__ uint64_t buf[4 * TK_CAP];
  __shared__ float red[32];
  __shared__ int wave_cnt[4];
  __shared__ Shared shared;
  if (threadIdx.x < 4) shared.whole[threadIdx.x] = shared.quarter[threadIdx.x] = 0;
  __syncthreads();
  const int64_t row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int c0 = part * width, n = min(width, V - c0);
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const T* p = z + row * ldz + c0;
  const Span<T> sp(p, n);
  constexpr int SH = sizeof(T) == 2 ? 16 : 0;
  Candidates<SH> cand(buf, &shared, wid, k);
  // s: the lane's sum of 2^(z log2 e - shift) with shift = m log2 e as rounded, one fused multiply-add an element. What the
  // rounding of shift left out is put right at the end.
  float m = -INFINITY, s = 0.f, shift = 0.f;
  auto raise = [&](float to) {
    // (terms that far below weigh nothing, and their sum is no number where m log2 e is too coarse or overflows: masked columns)
    const bool drop = to - m > 200.f;
    const float before = shift;
    m = to;
    shift = m == -INFINITY ? 0.f : m * LOG2E;            // -inf then adds 0, and a NaN is seen
    s = drop ? 0.f : s * __builtin_amdgcn_exp2f(before - shift);
  };
  auto power = [&](float v) { return __builtin_amdgcn_exp2f(fmaf(v, LOG2E, -shift)); };

  constexpr uint32_t NOTHING = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;   // -inf
  // elements outside the vectors: the head by wave 0 before its steps, the tail by wave 3 after its steps
  auto single = [&](int first, int cnt) {
    for (int i = 0; i < cnt; i += 64) {
      const bool in = i + lane < cnt;
      const float v = in ? Elem<T>::load(p + first + i + lane) : -INFINITY;
      if (cand.full()) cand.cut(false);
      cand.push(in, value_key(v), (uint32_t)(c0 + first + i + lane));
      if (v > m) raise(v);
      s += power(v);
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
      raw[i] = q < sp.nv ? load16<NT>(pv + q) : u32x4_t{NOTHING, NOTHING, NOTHING, NOTHING};
    }
    float gm[U], sm = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float v[N];
      unpack16<T>(raw[i], v);
      gm[i] = v[0];
#pragma unroll
      for (int e = 1; e < N; ++e) gm[i] = fmaxf(gm[i], v[e]);
      sm = fmaxf(sm, gm[i]);
    }
    if (sm > m) raise(sm);
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float v[N];
      unpack16<T>(raw[i], v);
#pragma unroll
      for (int e = 0; e < N; ++e) part[e % 4] += power(v[e]);
    }
    s += (part[0] + part[1]) + (part[2] + part[3]);
    if (fresh) {
      // the first step's 256 largest-of-a-vector: each is one element
      fresh = false;
      uint32_t key[U];
      int cnt = 0;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        key[i] = q0 + i * 64 + lane < sp.nv ? value_key(gm[i]) : 0u;
        cnt += __popcll(__ballot(key[i] != 0));
      }
      // (the keys' low bits come as zeros: bounds all the same)
      if (cnt >= (k + 3) / 4) {
        const uint32_t whole = cnt >= k ? kth_largest<U, SH>(key, U, k) : 0u, quarter = kth_largest<U, SH>(key, U, (k + 3) / 4);
        if (lane == 0) {
          __hip_atomic_store(&shared.whole[wid], whole, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          __hip_atomic_store(&shared.quarter[wid], quarter, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
    }
    cand.learn();
    // bit e of may[i]: element e of vector i may enter. (A lane that has met a NaN, which fmaxf drops, looks into
    // every vector from then on.)
    const float least = floor_value(cand.floor);
    uint32_t may[U];
    bool any = false;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool look = q0 + i * 64 + lane < sp.nv && (!(gm[i] < least) || s != s);
      may[i] = 0;
      if (__ballot(look) == 0) continue;
      any = true;
      float v[N];
      unpack16<T>(raw[i], v);
#pragma unroll
      for (int e = 0; e < N; ++e) may[i] |= look && !(v[e] < least) ? 1u << e : 0u;
    }
    while (any) {
      any = false;
#pragma unroll
      for (int i = 0; i < U; ++i) {
        while (!cand.full() && __ballot(may[i] != 0)) {
          const bool on = may[i] != 0;
          const int e = on ? __builtin_ctz(may[i]) : 0;
          may[i] &= may[i] - 1;                          // (0 stays 0)
          const int word = e * (int)sizeof(T) / 4;
          const uint32_t w01 = word & 1 ? raw[i][1] : raw[i][0], w23 = word & 1 ? raw[i][3] : raw[i][2];
          uint32_t w = word & 2 ? w23 : w01;
          if constexpr (sizeof(T) == 2) w = e & 1 ? w & 0xffff0000u : w << 16;
          cand.push(on, value_key(__uint_as_float(w)),
                    (uint32_t)(c0 + sp.head + (q0 + i * 64 + lane) * N + e));
        }
        any |= __ballot(may[i] != 0) != 0;
      }
      // (higher keys cost less than the candidates under them)
      if (any || cand.cnt >= cand.next) cand.cut(false);
    }
    cand.step_end();
  }
  if (wid == 3) single(sp.tail(), n - sp.tail());

  // The rounding left m log2 e - shift out of every exponent, at most 2^-25 |shift|. Far from 0 that is more than a
  // factor near 1 (or no number at all): the lane's elements are then read again.
  if (__ballot(!(fabsf(m) < TK_FAR) && m != -INFINITY)) s = far_sum(p, n, sp, wid, lane, m);
  else if (m != -INFINITY) s *= __builtin_amdgcn_exp2f(-fmaf(m, LOG2E, -shift));
  const float mb = block_max(m, red);
  s = block_sum(m == -INFINITY ? s : s * fast_expf(m - mb), red);
  if (parts == 1) {
    merge_waves(buf, wave_cnt, cand, k, [&](int rank, uint64_t e) {
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
    merge_waves(buf, wave_cnt, cand, k, [&](int rank, uint64_t e) { o[rank] = e; });
  }
}

// The parts' entries (sorted, at most TK_MERGE together) and statistics of a row, merged; one workgroup per row. k elements reach
// the greatest of the parts' last entries, and the least of their ceil(k / parts)-th ones: what lies below is dropped, and the
// rest ranked. Bound by latency: 16 rows of 32 parts, k = 10, 5.9 us.
constexpr int TK_MERGE = 1024;

__global__ __launch_bounds__(256) void topk_merge_kernel(const uint64_t* __restrict__ ws_key,
                                                         const float2* __restrict__ ws_stat, int k, int parts,
                                                         float* __restrict__ values, int64_t* __restrict__ cols,
                                                         float* __restrict__ lse) {
  __shared__ uint64_t buf[TK_MERGE];
  __shared__ uint64_t red[8];
  __shared__ float fred[32];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const uint64_t* src = ws_key + row * parts * k;
  const int n = parts * k, nth = (k + parts - 1) / parts - 1;
  uint64_t e[TK_MERGE / 256];
#pragma unroll
  for (int i = 0; i < TK_MERGE / 256; ++i) {
    const int at = i * 256 + (int)threadIdx.x;
    e[i] = at < n ? src[at] : 0;
  }
  uint64_t most = 0, least = ~0ull;
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x; i < parts; i += 256) {
    most = max(most, src[(int64_t)i * k + k - 1]);
    least = min(least, src[(int64_t)i * k + nth]);
    const float2 st = ws_stat[row * parts + i];
    if (st.x > m) { s = s * fast_expf(m - st.x) + st.y; m = st.x; }
    else s += st.x == -INFINITY ? st.y : st.y * fast_expf(st.x - m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    most = max(most, (uint64_t)__shfl_xor((unsigned long long)most, o, 64));
    least = min(least, (uint64_t)__shfl_xor((unsigned long long)least, o, 64));
  }
  if (lane == 0) { red[wid] = most; red[4 + wid] = least; }
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  most = max(max(red[0], red[1]), max(red[2], red[3]));
  least = min(min(red[4], red[5]), min(red[6], red[7]));
  most = max(most, least);
#pragma unroll
  for (int i = 0; i < TK_MERGE / 256; ++i) {
    const bool on = e[i] != 0 && e[i] >= most;
    const uint64_t mask = __ballot(on);
    int at = 0;
    if (lane == 0) at = atomicAdd(&count, __popcll(mask));
    at = __builtin_amdgcn_readfirstlane(at);
    if (on) buf[at + lanes_below(mask)] = e[i];          // (in any order: the entries' ranks decide)
  }
  const float mb = block_max(m, fred);
  s = block_sum(m == -INFINITY ? s : s * fast_expf(m - mb), fred);
  rank_entries((LdsKeys)buf, count, k, [&](int rank, uint64_t x) {
    const float v = key_value((uint32_t)(x >> 32));
    values[row * k + rank] = v;
    cols[row * k + rank] = (int64_t)(uint32_t)~(uint32_t)x;
    if (rank == 0) lse[row] = v - v == 0.f ? mb + logf(s) : v;
  });
}

// Parts of a row: with fewer rows than fill the chip (two workgroups per CU), as many as do, of at least 4096 columns, whose
// entries the merge holds. Rows of 151936, k = 10: 16 rows 18.6 us, 128 rows 33 (for one workgroup per CU 19.4 and 41, for four
// 19.6 and 31); 4 rows 17 us (parts of 2048 columns 25), one row, k = 5, 14.8 (parts of 8192 columns 16.6).
int topk_parts(int R, int V, int k) {
  const int want = (512 + R - 1) / (R > 0 ? R : 1), most = V / 4096, room = TK_MERGE / k;
  int p = want < most ? want : most;
  p = p < room ? p : room;
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
      const float v = t[e];
      if (c >= 0 && c < V && !(v == -INFINITY)) { col[i] = (int)c; x[i] = v; m = fmaxf(m, v); any = true; }
    }
  }
  if (__ballot(any) == 0) return false;
  m = wave_max(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < DK_MAX / 64; ++i)
    if (col[i] >= 0) { x[i] = (x[i] - m) * inv_tau; s += expf(x[i]); }
  s = wave_sum(s);
  const float l = logf(s);
  // (from x and s: m / tau + log s would be rounded to its size, and p by as much)
#pragma unroll
  for (int i = 0; i < DK_MAX / 64; ++i) use(lane + 64 * i, col[i], x[i] - l, col[i] >= 0 ? expf(x[i]) / s : 0.f);
  return true;
}

// sum_i p_i (log p_i - log q_i) of a row, in one wave, from the row's (max, sum of e^((z - max) / tau)).
template <typename T>
__device__ __forceinline__ float distill_row(const T* __restrict__ z, const float* __restrict__ t,
                                             const int64_t* __restrict__ idx, int k, int V, float inv_tau, int lane, float m,
                                             float s) {
  const float l = logf(s);
  float acc = 0.f;
  teacher_row(t, idx, k, V, inv_tau, lane, [&](int, int col, float logp, float pr) {
    if (col < 0) return;
    if (!(pr == 0.f)) acc += pr * (logp - (Elem<T>::load(z + col) - m) * inv_tau + l);
  });
  return wave_sum(acc);
}

// e^x of a logit less its row's maximum. fp32 gradients show what the product x log2 e and log2 e itself leave out,
// (|x| + 1) 2^-24 together, so their part is put back; a bf16 gradient is rounded to 2^-8.
template <typename T> __device__ __forceinline__ float distill_exp(float x) {
  if constexpr (sizeof(T) == 2) return fast_expf(x);
  constexpr float L = 1.4426950408889634f, LOW = (float)(1.4426950408889634 - (double)L);
  const float h = x * L, r = fmaf(x, LOW, fmaf(x, L, -h)), e = __builtin_amdgcn_exp2f(h);
  return x < -150.f ? 0.f : fmaf(e, r * 0.69314718f, e);
}

// (max, sum of e^((z - max) / tau)) over a part of a row; one workgroup per (row, part). A row in one part also gets its loss.
// (Differences first: z / tau of the types' largest and lowest numbers may be no number.) Bound by HBM: 4096 x 151936 bf16
// 227-240 us, 5.2-5.5 TB/s.
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
    for (int e = 0; e < N; ++e) g = fmaxf(g, v[e]);
    if (g > m) { s *= distill_exp<T>((m - g) * inv_tau); m = g; }
    const float ref = m == -INFINITY ? 0.f : m;        // -inf then adds 0, and a NaN is seen
#pragma unroll
    for (int e = 0; e < N; ++e) s += distill_exp<T>((v[e] - ref) * inv_tau);
  }
  auto single = [&](float v) {
    if (v > m) { s *= distill_exp<T>((m - v) * inv_tau); m = v; }
    s += distill_exp<T>((v - (m == -INFINITY ? 0.f : m)) * inv_tau);
  };
  for (int j = threadIdx.x; j < sp.head; j += 256) single(Elem<T>::load(p + j));
  for (int j = sp.tail() + threadIdx.x; j < n; j += 256) single(Elem<T>::load(p + j));
  const float mb = block_max(m, red);
  s = block_sum(m == -INFINITY ? s : s * distill_exp<T>((m - mb) * inv_tau), red);
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
    s += st.x == -INFINITY ? st.y : st.y * fast_expf((st.x - m) * inv_tau);
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
// all their probabilities. The gradient is stored past the caches: it is the size of the logits, which the writes would drive
// out (512 x 151936 bf16 with its forward 99 -> 88 us, 4096 x 151936 785 -> 742, and 711 with loads past them too). Bound by HBM.
template <typename T, bool NT>
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
    const bool any = teacher_row(t + row * k, idx + row * k, k, V, inv_tau, threadIdx.x, [&](int e, int col, float, float pr) {
      cols[e] = col;
      prob[e] = pr;
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
  auto one = [&](float v) { return cq * distill_exp<T>((v - m) * inv_tau); };
  if (aligned) {
    const u32x4_t* pv = (const u32x4_t*)(p + sp.head);
    u32x4_t* gv = (u32x4_t*)(g + sp.head);
    for (int q = threadIdx.x; q < sp.nv; q += 256) {
      float v[N];
      unpack16<T>(load16<NT>(pv + q), v);
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = one(v[e]);
      __builtin_nontemporal_store(pack16<T>(v), gv + q);
    }
    for (int j = threadIdx.x; j < sp.head; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
    for (int j = sp.tail() + threadIdx.x; j < n; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
  } else {
    for (int j = threadIdx.x; j < n; j += 256) Elem<T>::store(g + j, one(Elem<T>::load(p + j)));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the columns' first values are stored before the second ones
  __syncthreads();
  if (mine) Elem<T>::store(g + col, distill_exp<T>((zc - m) * inv_tau) / rs.y * c - psum * c);
}

// Parts of a row of the statistics and the gradient, as topk_parts, for four workgroups per CU, of at least 8192 columns. 300 rows of
// 151936, forward and backward: 61 us (for two or eight per CU 65); 16 rows of 32000 23 us (of 16384 columns 25, of 4096 21; no other case
// moves by more than 1 us).
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

int distill_check(const char* what, int dtype, int R, int V, int k, int64_t ldz, float tau, float scale) {
  UNOK_REQUIRE(R >= 0 && V >= 1 && (R <= 1 || ldz >= V), UNOK_EINVAL, "%s: R=%d V=%d ldz=%lld", what, R, V, (long long)ldz);
  UNOK_REQUIRE(k >= 1 && k <= DK_MAX, UNOK_EINVAL, "%s: k=%d must lie in [1, %d]", what, k, DK_MAX);
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "%s: bad dtype %d", what, dtype);
  UNOK_REQUIRE(tau > 0.f && tau < INFINITY && 1.f / tau < INFINITY, UNOK_EINVAL, "%s: temperature %g must be positive", what,
               (double)tau);
  UNOK_REQUIRE(scale - scale == 0.f, UNOK_EINVAL, "%s: scale %g (temperature %g) must be finite", what, (double)scale, (double)tau);
  return 0;
}

}  // namespace

UNOK_EXPORT int64_t unok_row_topk_workspace(int R, int V, int k) {
  if (R <= 0 || V <= 0 || k <= 0) return 0;
  const int64_t parts = topk_parts(R, V, k);
  return parts == 1 ? 0 : R * parts * (8ll * k + 8);
}

UNOK_EXPORT int unok_row_topk(int dtype, int R, int V, int k, const void* z, int64_t ldz, float* values, int64_t* cols,
                              float* lse, void* workspace, int64_t ws_bytes, void* stream) {
  UNOK_REQUIRE(R >= 0 && V >= 0 && (R <= 1 || ldz >= V), UNOK_EINVAL, "row_topk: R=%d V=%d ldz=%lld", R, V, (long long)ldz);
  UNOK_REQUIRE(k >= 1 && k <= TK_MAX && k <= V, UNOK_EINVAL, "row_topk: k=%d must lie in [1, min(%d, V=%d)]", k, TK_MAX, V);
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "row_topk: bad dtype %d", dtype);
  if (R == 0) return 0;
  UNOK_REQUIRE(z && values && cols && lse, UNOK_EINVAL, "row_topk: null operand");
  const int parts = topk_parts(R, V, k);
  const int64_t need = unok_row_topk_workspace(R, V, k);
  UNOK_REQUIRE(need == 0 || (workspace && ws_bytes >= need && ((uintptr_t)workspace & 7) == 0), UNOK_EINVAL,
               "row_topk: workspace of %lld bytes (8-byte aligned) required, got %lld", (long long)need, (long long)ws_bytes);
  UNOK_REQUIRE((int64_t)R * parts < (1ll << 31), UNOK_EINVAL, "row_topk: R=%d", R);
  const int width = ((V + parts - 1) / parts + 7) / 8 * 8;
  const int used = (V + width - 1) / width;            // a last part may fall away by the rounding
  uint64_t* keys = (uint64_t*)workspace;
  float2* stat = (float2*)(keys + (int64_t)R * parts * k);
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto* zt, auto nt) {
    using T = std::remove_cv_t<std::remove_pointer_t<decltype(zt)>>;
    hipLaunchKernelGGL((row_topk_kernel<T, decltype(nt)::value>), dim3((unsigned)(R * used)), dim3(256), 0, st, zt, ldz, V, k, used,
                       width, values, cols, lse, keys, stat);
  };
  auto by_size = [&](auto* zt) {
    if ((int64_t)R * V * (int64_t)sizeof(*zt) > MEMORY_CACHE) go(zt, std::true_type{});
    else go(zt, std::false_type{});
  };
  if (dtype == UNOK_BF16) by_size((const bf16_t*)z);
  else by_size((const float*)z);
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
  int rc = distill_check("distill_fwd", dtype, R, V, k, ldz, tau, scale);
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
  int rc = distill_check("distill_bwd", dtype, R, V, k, ldz, tau, scale);
  if (rc || R == 0) return rc;
  UNOK_REQUIRE(R <= 1 || ldg >= V, UNOK_EINVAL, "distill_bwd: ldg=%lld", (long long)ldg);
  UNOK_REQUIRE(z && t && idx && row_stat && gscale && grad, UNOK_EINVAL, "distill_bwd: null operand");
  const int64_t es = dtype == UNOK_BF16 ? 2 : 4;
  UNOK_REQUIRE((grad == z && (ldg == ldz || R == 1)) || !unok::rows_overlap(z, ldz * es, grad, ldg * es, R, V * es), UNOK_EINVAL,
               "distill_bwd: the gradient overlaps the logits");
  int parts, width;
  distill_split(R, V, parts, width);
  UNOK_REQUIRE((int64_t)R * parts < (1ll << 31), UNOK_EINVAL, "distill_bwd: R=%d", R);
  hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto* zt, auto* gt, auto nt) {
    using T = std::remove_pointer_t<decltype(gt)>;
    hipLaunchKernelGGL((distill_bwd_kernel<T, decltype(nt)::value>), dim3((unsigned)(R * parts)), dim3(256), 0, st, zt, ldz, V,
                       parts, width, k, (const float2*)row_stat, t, idx, 1.f / tau, gscale, inv_n, scale, gt, ldg);
  };
  auto go = [&](auto* zt, auto* gt) {
    if ((int64_t)R * V * es > MEMORY_CACHE) launch(zt, gt, std::true_type{});
    else launch(zt, gt, std::false_type{});
  };
  if (dtype == UNOK_BF16) go((const bf16_t*)z, (bf16_t*)grad);
  else go((const float*)z, (float*)grad);
  return unok::check_launch("distill_bwd");
}
