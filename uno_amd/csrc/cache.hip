// Row moves in KV caches: keeping the accepted path of a drafted tree, copying sequences between slots.
//
// A cache tensor is [batch, nk, max_len, D], contiguous, one per layer for K and one for V. Both
// operations touch the same rows in every layer, so one launch serves all of them: the tensors'
// addresses travel as kernel arguments (a model of 36 layers has 72).
#include "common.h"
#include "../../include/unok.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

constexpr int KEEP_TENSORS = 128, KEEP_PATH = 256;   // per launch; longest path
constexpr int COPY_TENSORS = 96, COPY_DST = 64;      // per launch

struct KeepArgs {
  char* t[KEEP_TENSORS];
  int nk, max_len, P, cpr;                            // cpr: units (16 bytes, or a row of less) per row
  const int64_t *lengths, *nodes, *counts;
};

// Row n + nodes[b, i] -> row n + i for i < counts[b], n = lengths[b]: one workgroup per (tensor, sequence, K/V
// head). It reads everything it moves into registers (NI 16-byte chunks per thread) before the barrier and writes
// after it, so that any list of nodes (descending, the same node twice) means the gather it says. Entries
// outside [0, max_len - n) and rows at or past max_len are skipped.
//
// Bound by latency: length, count, node list and rows are four dependent loads, and few bytes move (72 tensors of 8 heads
// of 128 bf16, 8 sequences, paths of 6: 12 MB, 5 us). The three NI are the registers that paths of up to 16, 64 and 256 rows of 256
// bytes need. Rows of 2, 4 or 8 bytes (the scales of 4-bit rows) are one unit U each.
template <typename U, int NI>
__global__ __launch_bounds__(256) void cache_keep_kernel(const KeepArgs p) {
  const int pair = blockIdx.x, b = pair / p.nk;
  const int64_t n = p.lengths[b];
  if (n < 0 || n >= p.max_len) return;
  const int64_t room = p.max_len - n;
  const int64_t want = p.counts[b];
  const int cnt = (int)(want < 0 ? 0 : want < p.P ? want : p.P);
  const int rows = (int)(cnt < room ? cnt : room);
  U* base = (U*)p.t[blockIdx.y] + ((int64_t)pair * p.max_len + n) * p.cpr;
  const int64_t* nodes = p.nodes + (int64_t)b * p.P;
  // (the room is at least one row, so a load that nothing needs reads row n)
  U v[NI];
  int64_t from[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (threadIdx.x + i * blockDim.x) / p.cpr;
    from[i] = r < rows ? nodes[r] : -1;
  }
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int c = (threadIdx.x + i * blockDim.x) % p.cpr;
    from[i] = from[i] < room ? from[i] : -1;
    v[i] = base[(from[i] < 0 ? 0 : from[i]) * p.cpr + c];
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every row is here before any wave writes
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NI; ++i)
    if (from[i] >= 0) base[(int64_t)(threadIdx.x + i * blockDim.x)] = v[i];
}

struct CopyArgs {
  const char* src[COPY_TENSORS];
  char* dst[COPY_TENSORS];
  int nk, src_max, dst_max, cpr, groups;
  const int64_t* src_lengths;
  int64_t* dst_lengths;
  int group_src[COPY_DST], group_first[COPY_DST + 1], slot[COPY_DST];   // slots of a group: first[g] .. first[g + 1]
};

// Rows [0, length) of a source slot into every destination slot of its group. Grid: (pieces, groups x K/V heads,
// tensors); a workgroup strides over its (slot, head)'s rows, one run of contiguous bytes, in pieces of 32 KB
// held in registers: the source is read once for all its destinations. The first workgroup of a group sets
// the destinations' lengths (no destination is a source where the two lie in the same memory).
//
// Bound by HBM: (1 + destinations) x rows. Stores of up to 2 GB go past the caches, where they would drive out a source that is
// there, as one just written or copied before: the same copy again, 72 tensors of 8 heads of 128 bf16, 2048 rows to one slot (604 MB)
// 121 -> 99-106 us, to four (1.5 GB) 305 -> 289-297, to six (2.1 GB) 430 -> 416-427, and no difference from seven slots on. A source
// that no cache holds gains nothing (three copies in turn, 0.6 and 1.2 GB written: 1.00 to 1.06 of the plain stores' time).
// Above 2 GB no cache holds what matters, and plain stores are the faster ones on the whole (past the caches 1.03 of their time on
// average, 0.94 to 1.21, over 20 shapes in one allocation and in 72; one prompt of 2048 rows to eight slots in turn 576 and 550 us).
// (Loads past the caches too: slower at every size.)
constexpr int64_t COPY_PAST = 2000000000;
constexpr int COPY_U = 8, COPY_PIECE = 256 * COPY_U;   // 16-byte chunks

// U: 16 bytes, or the whole row where it is 2, 4 or 8.
template <typename U> __global__ __launch_bounds__(256) void cache_copy_kernel(const CopyArgs p) {
  const int g = blockIdx.y / p.nk, h = blockIdx.y % p.nk;
  const int s = p.group_src[g], d0 = p.group_first[g], d1 = p.group_first[g + 1];
  int64_t rows = p.src_lengths[s];
  rows = rows < 0 ? 0 : rows;
  rows = rows < p.src_max ? rows : p.src_max;
  rows = rows < p.dst_max ? rows : p.dst_max;
  const int64_t total = rows * p.cpr;                  // units
  const U* src = (const U*)p.src[blockIdx.z] + ((int64_t)s * p.nk + h) * p.src_max * p.cpr;
  U* dst = (U*)p.dst[blockIdx.z];
  // (the branch stands outside: of two stores of one value, the compiler makes one, plain)
  auto move = [&](auto past) {
    for (int64_t c0 = (int64_t)blockIdx.x * COPY_PIECE; c0 < total; c0 += (int64_t)gridDim.x * COPY_PIECE) {
      U v[COPY_U];
#pragma unroll
      for (int i = 0; i < COPY_U; ++i) {
        const int64_t c = c0 + i * 256 + threadIdx.x;
        v[i] = src[c < total ? c : total - 1];
      }
      for (int d = d0; d < d1; ++d) {
        U* o = dst + ((int64_t)p.slot[d] * p.nk + h) * p.dst_max * p.cpr;
#pragma unroll
        for (int i = 0; i < COPY_U; ++i) {
          const int64_t c = c0 + i * 256 + threadIdx.x;
          if (c >= total) continue;
          if constexpr (decltype(past)::value) __builtin_nontemporal_store(v[i], o + c);
          else o[c] = v[i];
        }
      }
    }
  };
  if (total * (int64_t)sizeof(U) * p.nk * gridDim.z * p.group_first[p.groups] < COPY_PAST) move(std::true_type{});   // (a group's rows for all)
  else move(std::false_type{});
  if (blockIdx.x == 0 && blockIdx.z == 0 && h == 0 && p.dst_lengths)
    for (int d = d0 + threadIdx.x; d < d1; d += 256) p.dst_lengths[p.slot[d]] = rows;
}

// Bytes of a row's units; 0: not a row that these kernels move.
int unit_bytes(int row_bytes) {
  return row_bytes > 0 && row_bytes % 16 == 0 ? 16 : row_bytes == 2 || row_bytes == 4 || row_bytes == 8 ? row_bytes : 0;
}

// Runs f with a value of the unit's type.
template <typename F> void with_unit(int bytes, F f) {
  if (bytes == 16) f(u32x4_t{});
  else if (bytes == 8) f(uint64_t{});
  else if (bytes == 4) f(uint32_t{});
  else f(uint16_t{});
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

}  // namespace

UNOK_EXPORT int unok_cache_keep(int ntensors, void* const* caches, int row_bytes, int B, int nk, int max_len, int P,
                                const int64_t* lengths, const int64_t* nodes, const int64_t* counts, void* stream) {
  UNOK_REQUIRE(ntensors >= 0 && B >= 0 && nk > 0 && max_len >= 0 && P >= 0, UNOK_EINVAL,
               "cache_keep: tensors=%d B=%d nk=%d max_len=%d P=%d", ntensors, B, nk, max_len, P);
  UNOK_REQUIRE(P <= KEEP_PATH, UNOK_EUNSUPPORTED, "cache_keep: paths hold at most %d nodes (got %d)", KEEP_PATH, P);
  UNOK_REQUIRE(unit_bytes(row_bytes) && row_bytes <= 512, UNOK_EALIGN,
               "cache_keep: rows of %d bytes (2, 4, 8 or a multiple of 16, at most 512)", row_bytes);
  UNOK_REQUIRE((int64_t)B * nk < (1ll << 31), UNOK_EINVAL, "cache_keep: B=%d nk=%d", B, nk);
  if (ntensors == 0 || B == 0 || P == 0 || max_len == 0) return 0;
  UNOK_REQUIRE(caches && lengths && nodes && counts, UNOK_EINVAL, "cache_keep: null operand");
  const int64_t bytes = (int64_t)B * nk * max_len * row_bytes;
  for (int i = 0; i < ntensors; ++i) {
    UNOK_REQUIRE(caches[i] && ((uintptr_t)caches[i] & 15) == 0, UNOK_EALIGN, "cache_keep: cache %d must be 16-byte aligned", i);
    for (int j = 0; j < i; ++j)
      UNOK_REQUIRE(!overlap(caches[i], bytes, caches[j], bytes), UNOK_EINVAL, "cache_keep: caches %d and %d overlap", j, i);
  }
  KeepArgs a{};
  a.nk = nk; a.max_len = max_len; a.P = P; a.cpr = row_bytes / unit_bytes(row_bytes);
  a.lengths = lengths; a.nodes = nodes; a.counts = counts;
  const int items = P * a.cpr, nt = items <= 64 ? 64 : items <= 128 ? 128 : 256, ni = (items + nt - 1) / nt;
  hipStream_t st = (hipStream_t)stream;
  for (int t0 = 0; t0 < ntensors; t0 += KEEP_TENSORS) {
    const int nt_here = ntensors - t0 < KEEP_TENSORS ? ntensors - t0 : KEEP_TENSORS;
    for (int i = 0; i < nt_here; ++i) a.t[i] = (char*)caches[t0 + i];
    const dim3 grid((unsigned)(B * nk), (unsigned)nt_here), block((unsigned)nt);
    with_unit(unit_bytes(row_bytes), [&](auto u) {
      using U = decltype(u);
      if (ni <= 1) hipLaunchKernelGGL((cache_keep_kernel<U, 1>), grid, block, 0, st, a);
      else if constexpr (sizeof(U) == 16) {              // (a path of smaller rows is one unit to a thread)
        if (ni <= 4) hipLaunchKernelGGL((cache_keep_kernel<U, 4>), grid, block, 0, st, a);
        else hipLaunchKernelGGL((cache_keep_kernel<U, 32>), grid, block, 0, st, a);
      }
    });
  }
  return unok::check_launch("cache_keep");
}

UNOK_EXPORT int unok_cache_copy(int ntensors, const void* const* src, void* const* dst, int row_bytes, int nk, int src_batch,
                                int src_max, int dst_batch, int dst_max, const int64_t* src_lengths, int64_t* dst_lengths,
                                int npairs, const int* pairs, void* stream) {
  UNOK_REQUIRE(ntensors >= 0 && nk > 0 && src_batch >= 0 && src_max >= 0 && dst_batch >= 0 && dst_max >= 0 && npairs >= 0,
               UNOK_EINVAL, "cache_copy: tensors=%d nk=%d batch %d -> %d max_len %d -> %d pairs=%d", ntensors, nk, src_batch,
               dst_batch, src_max, dst_max, npairs);
  UNOK_REQUIRE(unit_bytes(row_bytes), UNOK_EALIGN, "cache_copy: rows of %d bytes (2, 4, 8 or a multiple of 16)", row_bytes);
  UNOK_REQUIRE(nk <= 65535 / COPY_DST, UNOK_EINVAL, "cache_copy: nk=%d", nk);
  if (npairs == 0 || ntensors == 0) return 0;
  UNOK_REQUIRE(src && dst && src_lengths && pairs, UNOK_EINVAL, "cache_copy: null operand");
  const int64_t sbytes = (int64_t)src_batch * nk * src_max * row_bytes, dbytes = (int64_t)dst_batch * nk * dst_max * row_bytes;
  bool same = dst_lengths && overlap(src_lengths, 8ll * src_batch, dst_lengths, 8ll * dst_batch);
  UNOK_REQUIRE(!same || src_lengths == dst_lengths, UNOK_EINVAL, "cache_copy: the lengths overlap");
  for (int i = 0; i < ntensors; ++i) {
    UNOK_REQUIRE(src[i] && dst[i] && ((uintptr_t)src[i] & 15) == 0 && ((uintptr_t)dst[i] & 15) == 0, UNOK_EALIGN,
                 "cache_copy: cache %d must be 16-byte aligned", i);
    for (int j = 0; j < ntensors; ++j) {
      UNOK_REQUIRE(i <= j || !overlap(dst[i], dbytes, dst[j], dbytes), UNOK_EINVAL,
                   "cache_copy: destinations %d and %d overlap", j, i);
      if (overlap(src[j], sbytes, dst[i], dbytes)) {
        UNOK_REQUIRE(i == j && src[i] == dst[i] && src_batch == dst_batch && src_max == dst_max, UNOK_EINVAL,
                     "cache_copy: source %d and destination %d overlap", j, i);
        same = true;
      }
    }
  }
  for (int i = 0; i < npairs; ++i) {
    const int s = pairs[2 * i], d = pairs[2 * i + 1];
    UNOK_REQUIRE(s >= 0 && s < src_batch && d >= 0 && d < dst_batch, UNOK_EINVAL,
                 "cache_copy: slots %d -> %d of batches %d -> %d", s, d, src_batch, dst_batch);
    for (int j = 0; j < npairs; ++j) {
      UNOK_REQUIRE(j >= i || pairs[2 * j + 1] != d, UNOK_EINVAL, "cache_copy: slot %d is written twice", d);
      UNOK_REQUIRE(!same || pairs[2 * j] != d, UNOK_EINVAL, "cache_copy: slot %d is read and written", d);
    }
  }
  CopyArgs a{};
  a.nk = nk; a.src_max = src_max; a.dst_max = dst_max; a.cpr = row_bytes / unit_bytes(row_bytes);
  a.src_lengths = src_lengths; a.dst_lengths = dst_lengths;
  const int64_t most = (int64_t)(src_max < dst_max ? src_max : dst_max) * a.cpr;
  hipStream_t st = (hipStream_t)stream;
  for (int p0 = 0; p0 < npairs; p0 += COPY_DST) {
    // the next destinations, grouped by source
    const int* pr = pairs + 2 * p0;
    const int np = npairs - p0 < COPY_DST ? npairs - p0 : COPY_DST;
    int nd = 0;
    a.groups = 0;
    for (int i = 0; i < np; ++i) {
      bool seen = false;
      for (int j = 0; j < i; ++j) seen |= pr[2 * j] == pr[2 * i];
      if (seen) continue;
      a.group_src[a.groups] = pr[2 * i];
      a.group_first[a.groups++] = nd;
      for (int j = i; j < np; ++j)
        if (pr[2 * j] == pr[2 * i]) a.slot[nd++] = pr[2 * j + 1];
    }
    a.group_first[a.groups] = nd;
    for (int t0 = 0; t0 < ntensors; t0 += COPY_TENSORS) {
      const int nt = ntensors - t0 < COPY_TENSORS ? ntensors - t0 : COPY_TENSORS;
      for (int i = 0; i < nt; ++i) { a.src[i] = (const char*)src[t0 + i]; a.dst[i] = (char*)dst[t0 + i]; }
      a.dst_lengths = t0 == 0 ? dst_lengths : nullptr;
      const int64_t gy = (int64_t)a.groups * nk, pieces = (most + COPY_PIECE - 1) / COPY_PIECE;
      int64_t gx = 8192 / (gy * nt);                   // a few rounds of workgroups; each strides over its pieces
      gx = gx > pieces ? pieces : gx;
      with_unit(unit_bytes(row_bytes), [&](auto u) {
        hipLaunchKernelGGL(cache_copy_kernel<decltype(u)>, dim3((unsigned)(gx < 1 ? 1 : gx), (unsigned)gy, (unsigned)nt),
                           dim3(256), 0, st, a);
      });
    }
  }
  return unok::check_launch("cache_copy");
}
