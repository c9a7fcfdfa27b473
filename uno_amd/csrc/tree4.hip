// Attention of a tree of drafted tokens over a KV cache in 4 bits: tree.hip's operator over rows as cache4.h describes them.
//
// The numbers of a 4-bit row are exact in bf16, so the products are bf16 ones, and the conversion is one instruction for two elements
// and their scale. Each of a workgroup's four waves walks its own tiles of a range: codes come into its part of LDS, are converted in
// registers, and serve the wave's 16 QT query rows; no barrier in the walk. (Converted tiles shared through LDS, as the bf16 cache's are,
// cost LDS reads of numbers four times as large as their codes: 16 sequences, 64 nodes of 32 / 8 heads of 128 over 16384 rows 418 us,
// this 257 at the time.)
//
// Measured (32 / 8 heads of 128, sequences from the given number of rows down to half of it): one node of 4 sequences, 65536 rows 45 us (232
// MB of codes and scales, 5.2 TB/s: what a large copy reaches); 64 nodes of 16 sequences, 16384 rows 241 to 249 us with their merge (210
// GFLOP, 850 to 880 TFLOP/s; conversions, weights and their rounding, some 190 vector instructions to 32 keys and 32 rows, bound it: the
// products alone would take 173); 16 nodes of 8 sequences, 4096 rows 21.5 us (6 at the copy's rate: eight tiles to a wave, the rest is the
// queries, the join and the launch). fp32 queries, 64 nodes of 8 sequences, 8192 rows 170 us (the three products alone 133).
//
// bf16 queries: a weight is rounded to bf16 for the product with V, off by at most 2^-8 of itself, and the weights' sum is that of the
// rounded ones, so that an output is off by the roundings' scatter alone: 2.1e-3 to 2.3e-3 of its size with its own rounding, which alone
// makes 1.7e-3. Scores, sums and outputs are fp32 until the end. (A second product with what a rounding leaves would add half to the
// products, which bind long caches; tree.hip measured that.)
//
// fp32 queries: a query is the sum of three bf16 numbers (each what the ones before it leave, 8 of its 24 bits), and so is a weight;
// three products take the place of one, exact but for their sums.
#include "tree.h"
#include "cache4.h"
#include "../../include/unok.h"

namespace {

// A range's rows of K or V of one (sequence, K/V head) pair, wave-uniform addresses.
struct Rows4 {
  uintptr_t codes, scales;
};
template <int D> __device__ __forceinline__ Rows4 rows4(const void* codes, const uint8_t* scales, int64_t row) {
  auto uniform = [](uintptr_t at) {
    return ((uintptr_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(at >> 32)) << 32) |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at);
  };
  return {uniform((uintptr_t)codes + row * (D / 2)), uniform((uintptr_t)scales + row * (D / GROUP4))};
}
// The rows from `key` on, of `rows` in all, as a buffer that ends behind the last: what lies past it reads as zeros, and of a tile past it
// nothing is loaded. A tile's place is in its buffer's base, so that a lane's offset alone is held against the buffer's size. (In the loads'
// scalar offset it would pass that size for tiles past the end, where the size less the scalar offset, which a raw buffer's range check
// uses, is below zero.)
__host__ __device__ constexpr int rows_left(int key, int rows) { return key < rows ? rows - key : 0; }
static_assert(rows_left(0, 130) == 130 && rows_left(128, 130) == 2 && rows_left(130, 130) == 0 && rows_left(512, 130) == 0,
              "no row past the last is in a buffer");
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer4(uintptr_t first, int key, int rows, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(first + (int64_t)key * bytes), (short)0, rows_left(key, rows) * bytes, 0x00020000);
}

// Tiles of 32 keys: codes and scales go from memory straight into LDS, NST - 1 tiles ahead, each wave's into its own part, so that
// nothing but the wave's own counter of loads is waited for. (Two tiles in registers, one of them on its way: 16 sequences, 64 nodes over
// 16384 rows 309 us, three spill: 518.) A stage: K's codes, V's codes, a dword to a key for its scales of K, and of V. A lane (m, g),
// m < 16, g < 4, reads
//   K (S^T = K Q^T, first operand: 16 keys x 8 dims a lane): the dims of a product may come in any order that Q takes too; lane group g
//     has dims D/4 g .. of key m and of key 16 + m: one read each, of one scale;
//   V (O^T = V^T P^T, first operand: one dim x 8 keys): lane m has dims D/16 m .. of keys 4 g .. + 3 and 16 + 4 g .. + 3, which are
//     those of its accumulators of S^T. Row 4 g + j of each 16 lies at place 4 j + g, so that the four rows read together are in
//     different banks. Four keys' scales are one read, and a rotation brings the byte of the lane's dims into the exponent (the
//     conversions read no other bit).
template <int D> struct Tile4 {
  static constexpr int KT = 32, KS = D / 32, NDT = D / 16, CR = D / 2, SR = D / GROUP4, NST = 3;
  static constexpr int CODES = KT * CR, SCALES = 256, STAGE = 2 * CODES + 2 * SCALES, LOADS = 2 * CODES / 1024 + 2;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  typedef uint32_t u2 __attribute__((ext_vector_type(2)));
  typedef std::conditional_t<D == 128, u4, u2> KCodes;
  KCodes k[2];
  uint32_t ks[2], v[8];
  u4 vs[2];

  // The wave's loads of the tile at `key`, of `rows` rows in all, into a stage; lane offsets as `places` gives them.
  static __device__ __forceinline__ int2 places(int lane) {
    const int place = lane * 16 / CR, q = place % 16, row = place / 16 * 16 + 4 * (q % 4) + q / 4;
    return make_int2(lane * 16, row * CR + lane * 16 % CR);
  }
  static __device__ __forceinline__ void issue(const Rows4& k, const Rows4& v, int key, int rows, int2 at, int lane, char* stage) {
    typedef __attribute__((address_space(3))) void* Lds;
    const __amdgpu_buffer_rsrc_t kc = buffer4(k.codes, key, rows, CR), vc = buffer4(v.codes, key, rows, CR);
    const __amdgpu_buffer_rsrc_t ks = buffer4(k.scales, key, rows, SR), vs = buffer4(v.scales, key, rows, SR);
#pragma unroll
    for (int i = 0; i < CODES / 1024; ++i) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(kc, (Lds)(stage + 1024 * i), 16, at.x + 1024 * i, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vc, (Lds)(stage + CODES + 1024 * i), 16, at.y + 1024 * i, 0, 0, 0);
    }
    const Lds kx = (Lds)(stage + 2 * CODES), vx = (Lds)(stage + 2 * CODES + SCALES);
    if constexpr (D == 128) {                            // (the size has to be a literal)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, kx, 4, lane * SR, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, vx, 4, lane * SR, 0, 0, 0);
    } else {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ks, kx, 2, lane * SR, 0, 0, 0);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vs, vx, 2, lane * SR, 0, 0, 0);
    }
  }
  // Reads the stage at LDS address `at` once its loads have arrived (the later tiles' may be on their way; the compiler, which cannot
  // tell the stages apart, would wait for those too).
  __device__ __forceinline__ void read(uint32_t at, int m, int g) {
    const uint32_t ka = at + m * CR + CR / 4 * g, kx = at + 2 * CODES + 4 * m + D / 4 * g / GROUP4;
    const uint32_t va = at + CODES + g * CR + NDT / 2 * m, vx = at + 2 * CODES + SCALES + 16 * g;
    if constexpr (D == 128) {
      u2 a, b, c, d;
      asm volatile(
          "s_waitcnt vmcnt(%14)\n\t"
          "ds_read_b128 %0, %10\n\tds_read_b128 %1, %10 offset:1024\n\t"
          "ds_read_u8 %2, %11\n\tds_read_u8 %3, %11 offset:64\n\t"
          "ds_read2st64_b32 %4, %12 offset0:0 offset1:1\n\tds_read2st64_b32 %5, %12 offset0:2 offset1:3\n\t"
          "ds_read2st64_b32 %6, %12 offset0:4 offset1:5\n\tds_read2st64_b32 %7, %12 offset0:6 offset1:7\n\t"
          "ds_read_b128 %8, %13\n\tds_read_b128 %9, %13 offset:64\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(k[0]), "=&v"(k[1]), "=&v"(ks[0]), "=&v"(ks[1]), "=&v"(a), "=&v"(b), "=&v"(c), "=&v"(d), "=&v"(vs[0]), "=&v"(vs[1])
          : "v"(ka), "v"(kx), "v"(va), "v"(vx), "i"((NST - 1) * LOADS)
          : "memory");
      v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
      v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
    } else {
      asm volatile(
          "s_waitcnt vmcnt(%18)\n\t"
          "ds_read_b64 %0, %14\n\tds_read_b64 %1, %14 offset:512\n\t"
          "ds_read_u8 %2, %15\n\tds_read_u8 %3, %15 offset:64\n\t"
          "ds_read_u16 %4, %16\n\tds_read_u16 %5, %16 offset:128\n\tds_read_u16 %6, %16 offset:256\n\t"
          "ds_read_u16 %7, %16 offset:384\n\tds_read_u16 %8, %16 offset:512\n\tds_read_u16 %9, %16 offset:640\n\t"
          "ds_read_u16 %10, %16 offset:768\n\tds_read_u16 %11, %16 offset:896\n\t"
          "ds_read_b128 %12, %17\n\tds_read_b128 %13, %17 offset:64\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(k[0]), "=&v"(k[1]), "=&v"(ks[0]), "=&v"(ks[1]), "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]),
            "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]), "=&v"(vs[0]), "=&v"(vs[1])
          : "v"(ka), "v"(kx), "v"(va), "v"(vx), "i"((NST - 1) * LOADS)
          : "memory");
    }
  }
  // Key j's scale of V for the conversions (more than its exponent bits may be set), and its byte.
  static __device__ __forceinline__ int group(int m) { return NDT * m / GROUP4; }
  __device__ __forceinline__ float v_scale(int j, int m) const {
    return __uint_as_float(__builtin_amdgcn_alignbit(vs[j / 4][j % 4], vs[j / 4][j % 4], (8 * group(m) + 9) & 31));
  }
  __device__ __forceinline__ uint32_t v_byte(int j, int m) const { return vs[j / 4][j % 4] >> (8 * group(m)) & 255; }
  __device__ __forceinline__ static int slot_key(int j, int g) { return j < 4 ? 4 * g + j : 12 + 4 * g + j; }
};

// Eight elements of codes as a product's operand.
__device__ __forceinline__ bf16x8_t eight4(uint32_t codes, float scale) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(bf16x8_t, u4{pair4<0>(codes, scale), pair4<1>(codes, scale), pair4<2>(codes, scale), pair4<3>(codes, scale)});
}

// The ancestors of node t (itself among them) in lane t, of a tree of at most 64 nodes, as tree_ancestors finds them; each wave does it
// for itself, with no barrier. `p` is the lane's parent, below -1 in the lanes from T on. (With tree_ancestors for all, and a bit read from
// LDS to a score: 37 fp32 nodes of three sequences over 901 rows 10.4 us, this way 8.2.)
__device__ __forceinline__ uint64_t tree_ancestors64(int p) {
  const int lane = threadIdx.x & 63;
  uint64_t w = p >= -1 ? 1ull << lane : 0;
  const int above = __shfl(p, p & 63, 64);
  int far = p < 0 || p >= lane || above < -1 ? -1 : p;
  while (__ballot(far >= 0)) {
    const uint64_t more = __shfl(w, far & 63, 64);
    const int next = __shfl(far, far & 63, 64);
    w |= far >= 0 ? more : 0;
    far = far >= 0 ? next : -1;
  }
  return w;
}

template <typename E, int D, int QT>
__global__ __launch_bounds__(256, sizeof(E) == 2 || D == 64 ? 2 : 1) void tree_attn4_kernel(const TreeAttn a) {
  using Tile = Tile4<D>;
  constexpr int KT = Tile::KT, KS = Tile::KS, NDT = Tile::NDT, ROWS = 16 * QT, PARTS = sizeof(E) == 4 ? 3 : 1;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  extern __shared__ __attribute__((aligned(1024))) char lds[];          // the waves' stages; at the end [4][ROWS][D + 4] floats
  __shared__ float merge_ml[4][ROWS][2];
  __shared__ bool merge_pad[ROWS];
  __shared__ uint32_t anc[TREE_MAX * TREE_WORDS];
  __shared__ int next[TREE_MAX];

  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
  const int rep = a.nq / a.nk, T = a.T, NR = rep * T;
  int tile, h, id;
  tree_place(a, tile, h, id);
  const Range range = tree_range(a, id, Tile::CR + Tile::SR);
  if (range.b < 0 || range.lo >= range.hi) return;
  const int b = range.b, n = range.n, lo = range.lo, hi = range.hi;
  tree_note(a, range, id, h, tile);

  // this lane's query of each 16-row subtile (rows past the pair's last repeat it; their results are dropped), and its parent
  typedef E Raw __attribute__((ext_vector_type(8), aligned(16)));
  Raw raw[QT][KS];
  int node[QT], parent[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = tile * ROWS + 16 * i + m, rc = r < NR ? r : NR - 1;
    node[i] = rc % T;
    parent[i] = a.parents[b * a.ldp + node[i]];
    const E* row = (const E*)a.q + ((int64_t)b * T + node[i]) * a.ldq + ((int64_t)h * rep + rc / T) * D + D / 4 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) raw[i][s] = *(const Raw*)(row + 8 * s);
  }
  const bool tree = hi > n, small = T <= 64;
  const int up = tree && small && lane < T ? a.parents[b * a.ldp + lane] : -2;

  const int64_t row0 = ((int64_t)b * a.nk + h) * a.max_len + lo;
  const Rows4 kr = rows4<D>(a.k, a.ks, row0), vr = rows4<D>(a.v, a.vs, row0);
  // committed rows, which every query sees, and rows, of this range
  const int full = __builtin_amdgcn_readfirstlane(min(hi, n) - lo), all = __builtin_amdgcn_readfirstlane(hi - lo);
  char* const mine = lds + wid * Tile::NST * Tile::STAGE;
  const int2 place = Tile::places(lane);
  int key = wid * KT, stage = 0;
  if (tree && !small) tree_ancestors(a.parents + b * a.ldp, T, anc, next);
#pragma unroll
  for (int i = 0; i < Tile::NST; ++i) Tile::issue(kr, vr, key + 4 * i * KT, all, place, lane, mine + i * Tile::STAGE);

  // what the queries see of the tree, of at most 64 nodes in registers (written to LDS, they would wait for the loads on their way there)
  const int W = (T + 31) / 32;
  uint64_t sees[QT];
  {
    const uint64_t w = tree_ancestors64(up);
#pragma unroll
    for (int i = 0; i < QT; ++i) sees[i] = __shfl(w, node[i] & 63, 64);
  }
  bf16x8_t q[QT][PARTS][KS];
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (PARTS == 1) {
        q[i][0][s] = __builtin_bit_cast(bf16x8_t, raw[i][s]);
        if (a.q_factor != 1.f) q[i][0][s] *= (__bf16)a.q_factor;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = raw[i][s][e] * a.q_factor;
#pragma unroll
          for (int p = 0; p < PARTS; ++p) {
            const uint32_t u = __float_as_uint(x) & 0xffff0000u;
            x -= __uint_as_float(u);
            q[i][p][s][e] = __builtin_bit_cast(__bf16, (uint16_t)(u >> 16));
          }
        }
      }
    }
  f32x4_t o[QT][NDT];
  float mref[QT];
  f32x4_t l[QT];                                         // sums of the weights, as a product with ones (254 us; as 16 additions to a tile 260)
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    mref[i] = -INFINITY;
    l[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NDT; ++c) o[i][c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  auto scores = [&](const Tile& t, f32x4_t (&s)[QT][2]) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float f = scale4(t.ks[x]);
#pragma unroll
      for (int i = 0; i < QT; ++i) s[i][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const bf16x8_t kf = eight4(t.k[x][k], f);
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)               // small parts first
#pragma unroll
          for (int i = 0; i < QT; ++i) s[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, q[i][p][k], s[i][x], 0, 0, 0);
      }
    }
  };
  // V's operands: keys in pairs, two dims of eight keys by a permute to a dim and pair.
  auto values = [&](const Tile& t, const float (&vf)[8], bf16x8_t (&v)[NDT]) {
    auto dims = [&](auto pair) {
      constexpr int C = decltype(pair)::value;
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pair4<C>(t.v[j], vf[j]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u4 u;
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], c ? 0x07060302u : 0x05040100u);
        v[2 * C + c] = __builtin_bit_cast(bf16x8_t, u);
      }
    };
    dims(std::integral_constant<int, 0>{});
    dims(std::integral_constant<int, 1>{});
    if constexpr (D == 128) {
      dims(std::integral_constant<int, 2>{});
      dims(std::integral_constant<int, 3>{});
    }
  };
  // The reference that a row's weights are relative to moves only where a score exceeds it by 2^8 (see tree.hip).
  auto reference = [&](const f32x4_t (&s)[QT][2]) {
    float mx[QT];
    bool grow = false;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      // (a maximum that NaN passes through: a row with a NaN score is NaN whatever its reference)
      mx[i] = s[i][0][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx[i] = __builtin_elementwise_maximum(mx[i], s[i][j / 4][j % 4]);
      mx[i] *= a.walk_scale;
      grow |= mx[i] > mref[i] + 8.f;
    }
    if (__ballot(grow)) {
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        mx[i] = __builtin_elementwise_maximum(mx[i], __shfl_xor(mx[i], 16, 64));
        mx[i] = __builtin_elementwise_maximum(mx[i], __shfl_xor(mx[i], 32, 64));
        // (for the queries that need it alone: a row's result does not depend on the rows beside it)
        const float to = mx[i] > mref[i] + 8.f ? mx[i] : mref[i];
        const float f = to == mref[i] ? 1.f : mref[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mref[i] - to);
        mref[i] = to;
        l[i] *= f;
#pragma unroll
        for (int c = 0; c < NDT; ++c) o[i][c] *= f;
      }
    }
  };
  auto weights = [&](int i, const f32x4_t (&s)[2], float (&p)[8]) {
    const float ref = mref[i] == -INFINITY ? 0.f : -mref[i];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[j / 4][j % 4], a.walk_scale, ref));
  };
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, u4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
  auto add_pv = [&](int i, const bf16x8_t (&v)[NDT], float (&p)[8]) {
    bf16x8_t pf[PARTS];
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      u4 u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (PARTS == 1) u[j] = pack2_bf16(p[2 * j], p[2 * j + 1]);
        else {
          const uint32_t x = __float_as_uint(p[2 * j]) & 0xffff0000u, y = __float_as_uint(p[2 * j + 1]) & 0xffff0000u;
          p[2 * j] -= __uint_as_float(x);
          p[2 * j + 1] -= __uint_as_float(y);
          u[j] = x >> 16 | y;
        }
      }
      pf[part] = __builtin_bit_cast(bf16x8_t, u);
    }
#pragma unroll
    for (int part = PARTS - 1; part >= 0; --part) {
      l[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[part], l[i], 0, 0, 0);
#pragma unroll
      for (int c = 0; c < NDT; ++c) o[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[c], pf[part], o[i][c], 0, 0, 0);
    }
  };

  const uint32_t at = lds_addr(mine);
  auto next_tile = [&] {                                  // its stage gets the tile NST behind it (zeros past the end)
    Tile::issue(kr, vr, key + 4 * Tile::NST * KT, all, place, lane, mine + stage * Tile::STAGE);
    key += 4 * KT;
    stage = stage + 1 < Tile::NST ? stage + 1 : 0;
  };
  // Tiles of committed rows.
#pragma unroll 1
  while (key + KT <= full) {
    Tile t;
    t.read(at + stage * Tile::STAGE, m, g);
    f32x4_t s[QT][2];
    float vf[8];
    bf16x8_t v[NDT];
#pragma unroll
    for (int j = 0; j < 8; ++j) vf[j] = t.v_scale(j, m);
    scores(t, s);
    values(t, vf, v);
    // the scores' products run while the codes are converted (held here: the compiler would move V's behind the
    // branch; 16 sequences, 64 nodes over 16384 rows 257 us, 267 without)
#pragma unroll
    for (int c = 0; c < NDT; ++c) {
      u4 u = __builtin_bit_cast(u4, v[c]);
      asm volatile("" : "+v"(u));
      v[c] = __builtin_bit_cast(bf16x8_t, u);
    }
    reference(s);
    // and the weighted values' while the next rows' weights are formed
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float p[8];
      weights(i, s[i], p);
      add_pv(i, v, p);
    }
    next_tile();
  }
  // Tiles with tree rows, and rows at or past hi, which read as zeros, at weight 0.
#pragma unroll 1
  while (key < all) {
    Tile t;
    t.read(at + stage * Tile::STAGE, m, g);
    f32x4_t s[QT][2];
    scores(t, s);
    // bit j: whether the query sees row key + j
    uint32_t seen[QT];
    const int x = key + lo - n, w0 = x >> 5;               // (the first row's place in the tree)
    const uint32_t rows = all - key >= KT ? ~0u : (1u << (all - key)) - 1;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      auto word = [&](int w) {
        if (w < 0) return ~0u;
        if (w >= W) return 0u;
        return small ? (uint32_t)(sees[i] >> (32 * w)) : anc[node[i] * W + w];
      };
      seen[i] = __builtin_amdgcn_alignbit(word(w0 + 1), word(w0), x & 31) & rows;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s[i][j / 4][j % 4] = seen[i] >> (4 * g) & 1u << Tile::slot_key(j, 0) ? s[i][j / 4][j % 4] : -INFINITY;
    }
    reference(s);
    // A scale of NaN, or one too large for numbers, in a row that some queries do not see: 0 in the product, and added where it is
    // seen. The weights go through the tile's stage, 16 rows at a time.
    bool odd = false;
    float vf[8];
    bf16x8_t v[NDT];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t byte = t.v_byte(j, m);
      odd |= byte > SCALE4_MAX;
      vf[j] = scale4(byte > SCALE4_MAX ? 0 : byte);
    }
    odd = __ballot(odd) != 0;
    values(t, vf, v);
    float* ps = (float*)(mine + stage * Tile::STAGE);
    static_assert(16 * (KT + 1) * 4 <= Tile::STAGE, "the weights of 16 rows fit in a stage");
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float p[8];
      weights(i, s[i], p);
      if (odd) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ps[m * (KT + 1) + Tile::slot_key(j, g)] = p[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int j = 0; j < KT && key + j < all; ++j) {
          const int64_t r = row0 + key + j;
          const Row4 row{(const uint8_t*)a.v + r * Tile::CR, a.vs + r * Tile::SR};
          const float w = ps[m * (KT + 1) + j];
#pragma unroll
          for (int c = 0; c < NDT; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int d = (4 * g + e) * NDT + c;
              if (seen[i] >> j & 1 && row.scales[d / GROUP4] > SCALE4_MAX) o[i][c][e] += w * value4(row, d);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      add_pv(i, v, p);
    }
    next_tile();
  }
  if (threadIdx.x < 16)
#pragma unroll
    for (int i = 0; i < QT; ++i) merge_pad[16 * i + m] = parent[i] < -1;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // no load is on its way into what becomes the merge's
  float sum[QT];                                         // (each lane has its query's whole sum; the merge adds four lanes')
#pragma unroll
  for (int i = 0; i < QT; ++i) sum[i] = g == 0 ? l[i][0] : 0.f;
  tree_merge<E, D, QT>(a, range, tile, h, id, o, mref, sum, (float*)lds, merge_ml, merge_pad,
                       [](int c, int e, int g) { return (4 * g + e) * NDT + c; });
}

// Query rows of a workgroup, and one round of workgroups (`share`, two to a CU; fp32 with 128 dims has the registers for one). 32 rows: 64
// to a wave share a conversion among more products, but leave one wave to a SIMD: 16 sequences, 64 nodes over 16384 rows 273 us (32
// rows 266), 8 sequences, 16 nodes over 4096 26.2 (22.5).
// The ranges are those of tree.h, whose figures are of 16/32-bit rows. On these rows (us with the merge, in a graph; ranges of at least one /
// two / four blocks): one sequence, one node over 1150 rows 10.0 / 9.4 / 9.7, over 2000 10.4 / 9.7 / 10.8, over 4096 14.8 / 11.8 / 11.7; 8
// sequences, 16 nodes over 500 rows 17.9 / 15.7 / 15.1, over 1000 18.8 / 18.9 / 15.9, from 2000 on alike. Single blocks for sequences of
// three to eight (with them / without): one node over 1000 rows 8.9 / 9.6, 16 nodes 12.6 / 12.9 (fp32 14.3 / 15.2), fp32 37 nodes of
// three sequences over 901 11.3 / 12.0; they lose for 16 nodes of four sequences over 500 rows, 13.7 / 13.2.
TreePlan tree_plan4(int dtype, int B, int T, int nq, int nk, int D, int max_len) {
  const int NR = nq / nk * T;
  TreePlan p;
  p.rows = NR <= 16 ? 16 : 32;
  p.rt = (NR + p.rows - 1) / p.rows;
  const int64_t share = (dtype == UNOK_F32 && D == 128 ? 256 : 512) / ((int64_t)nk * p.rt);
  p.share = share > 1 ? (int)share : 1;
  p.ranges = max_len <= TREE_LEAST * TB ? B : B + p.share;
  return p;
}

template <typename E, int D> void launch_tree4(const TreeAttn& a, const TreePlan& plan, hipStream_t st) {
  const dim3 grid((unsigned)tree_blocks(a, plan));
  auto walk = [&](auto t) {
    constexpr int QT = decltype(t)::value;
    constexpr size_t merge = 4ull * 16 * QT * (D + 4) * sizeof(float), stages = 4ull * Tile4<D>::NST * Tile4<D>::STAGE;
    constexpr size_t lds = merge > stages ? merge : stages;
    UNOK_SET_LDS_ONCE((tree_attn4_kernel<E, D, QT>), lds);
    hipLaunchKernelGGL((tree_attn4_kernel<E, D, QT>), grid, dim3(256), lds, st, a);
  };
  if (plan.rows == 16) walk(std::integral_constant<int, 1>{});
  else walk(std::integral_constant<int, 2>{});
  launch_combine<E, D>(a, plan, st);
}

int sizes_ok(int B, int T, int nq, int nk, int D, int max_len) {
  UNOK_REQUIRE(max_len <= 1 << 24, UNOK_EINVAL, "tree_attn4: caches hold at most 2^24 rows (got %d)", max_len);   // (32-bit offsets)
  return tree_sizes_ok("tree_attn4", B, T, nq, nk, D, max_len);
}

}  // namespace

UNOK_EXPORT int64_t unok_tree_attn4_workspace(int dtype, int B, int T, int nq, int nk, int D, int max_len) {
  if (sizes_ok(B, T, nq, nk, D, max_len)) return -1;
  if (B == 0 || T == 0) return 0;
  return plan_workspace(tree_plan4(dtype, B, T, nq, nk, D, max_len), B, T, nq, D);
}

UNOK_EXPORT int unok_tree_attn4(int dtype, int B, int T, int nq, int nk, int D, const void* q, int64_t ldq, const void* k,
                                const void* k_scales, const void* v, const void* v_scales, int max_len, const int64_t* lengths,
                                const int32_t* parents, int64_t ldp, float scale, void* o, int64_t ldo, void* workspace,
                                int64_t ws_bytes, void* stream) {
  int rc = sizes_ok(B, T, nq, nk, D, max_len);
  if (rc) return rc;
  UNOK_REQUIRE(dtype == UNOK_BF16 || dtype == UNOK_F32, UNOK_EINVAL, "tree_attn4: bad dtype %d", dtype);
  if (B == 0 || T == 0) return 0;
  UNOK_REQUIRE(k && v && k_scales && v_scales, UNOK_EINVAL, "tree_attn4: null operand");
  UNOK_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_scales | (uintptr_t)v_scales) & 15) == 0, UNOK_EALIGN,
               "tree_attn4: codes and scales must be 16-byte aligned");
  const TreePlan plan = tree_plan4(dtype, B, T, nq, nk, D, max_len);
  TreeAttn a{};
  a.k = k; a.v = v;
  a.ks = (const uint8_t*)k_scales; a.vs = (const uint8_t*)v_scales;
  rc = tree_setup(a, "tree_attn4", plan, dtype, B, T, nq, nk, D, q, ldq, max_len, lengths, parents, ldp, scale, o, ldo, workspace,
                  ws_bytes);
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == UNOK_BF16) D == 128 ? launch_tree4<bf16_t, 128>(a, plan, st) : launch_tree4<bf16_t, 64>(a, plan, st);
  else D == 128 ? launch_tree4<float, 128>(a, plan, st) : launch_tree4<float, 64>(a, plan, st);
  return unok::check_launch("tree_attn4");
}
