// Rows put into 4-bit caches, and read back (see cache4.h for the format).
#include "common.h"
#include "cache4.h"
#include "../../include/unok.h"

#include <type_traits>

namespace {

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

static_assert(GROUP4 == 32, "rows have 2^(log_d - 5) scales");
constexpr int TENSORS4 = 16;                          // per launch (their addresses are arguments)

// n / d for 0 <= n < 2^31, d > 0: with 2^(bits - 1) < d <= 2^bits, 2^(31 + bits) / d rounded up has at most 32 bits, and exceeds the quotient
// by less than 2^bits / 2^(31 + bits) of n, below 1 / d.
struct Divisor {
  uint32_t d, factor, bits;
  __host__ __device__ Divisor() {}
  explicit Divisor(uint32_t d_) : d(d_), bits(0) {
    while ((1ull << bits) < d) ++bits;
    factor = (uint32_t)(((1ull << (31 + bits)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (uint32_t)((uint64_t)n * factor >> (31 + bits)); }
};

struct Move4 {
  void* rows[TENSORS4]; int64_t ld[TENSORS4];         // [B T, nk D]
  uint8_t *codes[TENSORS4], *scales[TENSORS4];        // [B, nk, max_len, D / 2], [.., D / GROUP4]
  const int64_t* starts;
  int nk, max_len, log_d;
  Divisor per_row, per_sequence;                      // items to a row, rows to a sequence
  uint32_t items;                                     // eight elements each
};

// Eight elements: their row, their offset in it, their cache row (none: negative), and their offset in that.
struct Eight { int64_t row, cache; int at, d; };
__device__ __forceinline__ Eight eight(const Move4& p, uint32_t i) {
  Eight e;
  const uint32_t row = p.per_row.quotient(i), b = p.per_sequence.quotient(row);
  e.row = row;
  e.at = (int)(i - row * p.per_row.d) * 8;
  e.d = e.at & ((1 << p.log_d) - 1);
  const int64_t start = p.starts[b], r = start < p.max_len && start > INT32_MIN ? start + (row - b * p.per_sequence.d) : -1;
  e.cache = r >= 0 && r < p.max_len ? ((int64_t)b * p.nk + (e.at >> p.log_d)) * p.max_len + r : -1;
  return e;
}
// A thread's items, both on their way before the first is worked on (8192 rows of 1024, K and V: stored in 10.3 us and loaded in 10.7,
// with one item 11.1 and 11.2, with four 10.9 and 10.7; one row 0.2 us more). Past the last one: none (whole groups of four lanes, as the
// items are a multiple of four).
constexpr int MOVES = 2;
__device__ __forceinline__ uint32_t item(int n) { return blockIdx.x * (256u * MOVES) + 256u * n + threadIdx.x; }

template <typename E> __device__ __forceinline__ void store_eight(const Move4& p, const Eight& e, const float (&x)[8]) {
  // the largest magnitude's bits, of four lanes by two exchanges: NaN and infinity are above every number
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
  top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
  if (e.cache < 0) return;
  const uint32_t byte = scale4_of(__uint_as_float(top));
  const float s = scale4(byte == SCALE4_NAN ? 127 : byte);
  uint32_t codes = codes4<0>(0u, x[0], x[1], s);
  codes = codes4<1>(codes, x[2], x[3], s);
  codes = codes4<2>(codes, x[4], x[5], s);
  codes = codes4<3>(codes, x[6], x[7], s);
  *(uint32_t*)(p.codes[blockIdx.y] + (e.cache << (p.log_d - 1)) + e.d / 2) = byte == SCALE4_NAN ? 0u : codes;
  if (e.d % GROUP4 == 0) p.scales[blockIdx.y][(e.cache << (p.log_d - 5)) + e.d / GROUP4] = (uint8_t)byte;
}

// Four lanes to a group. Bound by HBM, or by latency where rows are few.
template <typename E> __global__ __launch_bounds__(256) void cache4_store_kernel(const Move4 p) {
  typedef uint32_t Words __attribute__((ext_vector_type(2 * sizeof(E)), aligned(16)));
  Eight e[MOVES];
  Words v[MOVES];
#pragma unroll
  for (int n = 0; n < MOVES; ++n) {
    e[n] = eight(p, min(item(n), p.items - 1));
    if (item(n) >= p.items) e[n].cache = -1;
    v[n] = *(const Words*)((const E*)p.rows[blockIdx.y] + e[n].row * p.ld[blockIdx.y] + e[n].at);
  }
#pragma unroll
  for (int n = 0; n < MOVES; ++n) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(E) == 4) x[k] = __uint_as_float(v[n][k]);
      else x[k] = __uint_as_float(k % 2 ? v[n][k / 2] & 0xffff0000u : v[n][k / 2] << 16);
    }
    store_eight<E>(p, e[n], x);
  }
}

// Cache rows that do not exist read as zeros.
template <typename E> __global__ __launch_bounds__(256) void cache4_load_kernel(const Move4 p) {
  Eight e[MOVES];
  uint32_t codes[MOVES], byte[MOVES];
#pragma unroll
  for (int n = 0; n < MOVES; ++n) {
    e[n] = eight(p, min(item(n), p.items - 1));
    codes[n] = 0;
    byte[n] = SCALE4_MIN;
    if (e[n].cache >= 0) {
      codes[n] = *(const uint32_t*)(p.codes[blockIdx.y] + (e[n].cache << (p.log_d - 1)) + e[n].d / 2);
      byte[n] = p.scales[blockIdx.y][(e[n].cache << (p.log_d - 5)) + e[n].d / GROUP4];
    }
  }
#pragma unroll
  for (int n = 0; n < MOVES; ++n) {
    if (item(n) >= p.items) continue;
    const float s = scale4(byte[n]);
    const u32x4_t v = {pair4<0>(codes[n], s), pair4<1>(codes[n], s), pair4<2>(codes[n], s), pair4<3>(codes[n], s)};
    E* dst = (E*)p.rows[blockIdx.y] + e[n].row * p.ld[blockIdx.y] + e[n].at;
    if constexpr (sizeof(E) == 2) *(u32x4_t*)dst = v;
    else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *(f32x4_t*)(dst + 4 * h) = f32x4_t{__uint_as_float(v[2 * h] << 16), __uint_as_float(v[2 * h] & 0xffff0000u),
                                           __uint_as_float(v[2 * h + 1] << 16), __uint_as_float(v[2 * h + 1] & 0xffff0000u)};
    }
  }
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

int move4(const char* what, bool store, int dtype, int ntensors, void* const* rows, const int64_t* ld, void* const* codes,
          void* const* scales, int B, int T, int nk, int D, int max_len, const int64_t* starts, void* stream) {
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "%s: bad dtype %d", what, dtype);
  UNOK_REQUIRE(ntensors >= 0 && B >= 0 && T >= 0 && nk > 0 && max_len >= 0, UNOK_EINVAL, "%s: tensors=%d B=%d T=%d nk=%d max_len=%d",
               what, ntensors, B, T, nk, max_len);
  UNOK_REQUIRE(D == 64 || D == 128, UNOK_EINVAL, "%s: head dim %d not in {64,128}", what, D);
  UNOK_REQUIRE(nk < (1 << 20) && (int64_t)B * T < (1ll << 31) && (int64_t)B * T * nk * (D / 8) < (1ll << 31), UNOK_EINVAL,
               "%s: B=%d T=%d nk=%d D=%d: grid too large", what, B, T, nk, D);
  if (ntensors == 0 || B == 0 || T == 0 || (store && max_len == 0)) return 0;
  UNOK_REQUIRE(rows && ld && codes && scales && starts, UNOK_EINVAL, "%s: null operand", what);
  const int64_t es = dtype == UNOK_BF16 ? 2 : 4, n = (int64_t)B * T, width = (int64_t)nk * D;
  const int64_t cbytes = (int64_t)B * nk * max_len * (D / 2), sbytes = (int64_t)B * nk * max_len * (D / GROUP4);
  for (int i = 0; i < ntensors; ++i) {
    UNOK_REQUIRE(rows[i] && ((codes[i] && scales[i]) || max_len == 0), UNOK_EINVAL, "%s: null operand", what);
    UNOK_REQUIRE((((uintptr_t)rows[i] | (uintptr_t)codes[i] | (uintptr_t)scales[i]) & 15) == 0 && ld[i] * es % 16 == 0, UNOK_EALIGN,
                 "%s: rows, codes and scales of tensor %d and the rows' stride must be multiples of 16 bytes", what, i);
    UNOK_REQUIRE(n == 1 || ld[i] >= width, UNOK_EINVAL, "%s: rows of %lld elements, %lld apart", what, (long long)width,
                 (long long)ld[i]);
    const int64_t rbytes = ((n - 1) * ld[i] + width) * es;
    for (int j = 0; j <= i; ++j) {
      // what is written shares no memory with anything else (rows that are read may share theirs)
      bool bad = overlap(rows[i], rbytes, codes[j], cbytes) || overlap(rows[i], rbytes, scales[j], sbytes) ||
                 overlap(codes[i], cbytes, scales[j], sbytes) || overlap(scales[i], sbytes, codes[j], cbytes);
      if (j < i) {
        const int64_t rj = ((n - 1) * ld[j] + width) * es;
        bad |= overlap(rows[j], rj, codes[i], cbytes) || overlap(rows[j], rj, scales[i], sbytes);
        if (store) bad |= overlap(codes[i], cbytes, codes[j], cbytes) || overlap(scales[i], sbytes, scales[j], sbytes);
        else bad |= unok::rows_overlap(rows[i], ld[i] * es, rows[j], ld[j] * es, n, width * es);
      }
      UNOK_REQUIRE(!bad, UNOK_EINVAL, "%s: tensors %d and %d overlap", what, j, i);
    }
  }
  Move4 p{};
  p.starts = starts;
  p.nk = nk; p.max_len = max_len;
  p.log_d = D == 128 ? 7 : 6;
  p.per_row = Divisor((uint32_t)(nk * (D / 8)));
  p.per_sequence = Divisor((uint32_t)T);
  p.items = (uint32_t)(n * nk * (D / 8));
  hipStream_t st = (hipStream_t)stream;
  for (int t0 = 0; t0 < ntensors; t0 += TENSORS4) {
    const int here = ntensors - t0 < TENSORS4 ? ntensors - t0 : TENSORS4;
    for (int i = 0; i < here; ++i) {
      p.rows[i] = rows[t0 + i]; p.ld[i] = ld[t0 + i];
      p.codes[i] = (uint8_t*)codes[t0 + i]; p.scales[i] = (uint8_t*)scales[t0 + i];
    }
    const dim3 grid((p.items + 256 * MOVES - 1) / (256 * MOVES), (unsigned)here), block(256);
    if (store) {
      if (dtype == UNOK_BF16) hipLaunchKernelGGL(cache4_store_kernel<bf16_t>, grid, block, 0, st, p);
      else hipLaunchKernelGGL(cache4_store_kernel<float>, grid, block, 0, st, p);
    } else {
      if (dtype == UNOK_BF16) hipLaunchKernelGGL(cache4_load_kernel<bf16_t>, grid, block, 0, st, p);
      else hipLaunchKernelGGL(cache4_load_kernel<float>, grid, block, 0, st, p);
    }
  }
  return unok::check_launch(what);
}

}  // namespace

UNOK_EXPORT int unok_cache4_store(int dtype, int ntensors, const void* const* rows, const int64_t* ld, void* const* codes,
                                  void* const* scales, int B, int T, int nk, int D, int max_len, const int64_t* starts,
                                  void* stream) {
  return move4("cache4_store", true, dtype, ntensors, (void* const*)rows, ld, codes, scales, B, T, nk, D, max_len, starts, stream);
}

UNOK_EXPORT int unok_cache4_load(int dtype, int ntensors, void* const* rows, const int64_t* ld, const void* const* codes,
                                 const void* const* scales, int B, int T, int nk, int D, int max_len, const int64_t* starts,
                                 void* stream) {
  return move4("cache4_load", false, dtype, ntensors, rows, ld, (void* const*)codes, (void* const*)scales, B, T, nk, D, max_len,
               starts, stream);
}
