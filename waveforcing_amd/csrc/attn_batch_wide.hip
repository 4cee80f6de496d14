// Batched attention, many rows over pages: tiles of 256 (row, head) rows of a sequence over one key head.  Bound by the
// matrix cores and by the issue of the vector work between their instructions.
//
// Eight waves of 32 rows; keys in tiles of 64 through three LDS stages, staged by all threads (thread t: key t / 8, 16
// values t % 8 of its row) one tile ahead of the products, with the loads of the tile after in flight.  S^T = K Q^T on
// 32x32 products leaves a lane with one row and 32 keys, so a row's sums are in-lane, and its weights are directly the
// second operand of O^T += V^T P^T, whose first operand comes from the staged rows by transposing reads (attn_paged.hip
// has the layouts).
//
// 3 x 4680 rows over up to 37440 keys of 12 heads: 2.17-2.23 ms, 0.97 PFLOP/s (one sequence at a time, csrc/attn_paged.hip: 1.0
// PFLOP/s with bf16 keys and weights).  Of the cycles in which a CU has work (85 % of the kernel's) the matrix cores are busy
// 51 % and the vector unit issues 59 %, the matrix instructions' own 5 % among them.  Over 18720 keys 1.10 PFLOP/s on
// zeros and 0.98 on N(0, 1) data, int8 0.97 and 0.88: instructions first, power close behind.
//
// What is rounded, and where:
//   e4m3 keys  the codes go to the fp8 matrix cores as they are, Q as the sum of two e4m3 parts under a power-of-two scale
//              of the row: q = 2^e (q1 + q2 / 16), exact where q's last bit is not below 2^-13 of 2^e (|q| < 2^8 2^e);
//              the product is that of the codes with Q in fp32, and s_k c multiplies the score in fp32.  Staging K costs
//              no conversion and half the LDS.
//   int8 keys  the codes are exact in bf16, as Q is.
//   V          the codes are exact in fp16.
//   weights    fp16(p s_v), the product in fp32: 11 significant bits, eight times finer than bf16.  p is relative to a reference
//              of the row, set by the p s_v of the keys that it sees: the largest so far is between 2^6 and 2^15, so bits are
//              lost below 2^-20 of it, 2^-31 of it at most.  (The scale in V instead, under an exponent that the tile shares,
//              saves an instruction a score, but there a key that a row does not see, or gives no weight, takes the bits of
//              those that it does.)  The row sum adds the p in fp32.
// A NaN or infinite scale makes the key's score NaN and its weight of V zero, so the rows that see the key become NaN and
// no others; in tiles that some row does not see whole, so does a NaN code of V.
#include <utility>

#include "attn_batch.hpp"

namespace wf {
namespace attn_batch {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int BKV = 64;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
constexpr int R = 32 * kWaves;
constexpr int kXcds = 8;
// A row's weights p are relative to a reference, set so that the largest p s_v it had seen was 2^kShift; they may grow by
// 2^kGrow before a new one is taken (fp16 ends at 2^16).  A scale of V below 2^kFloor counts as that in the reference, so
// that the p stay below 2^(kShift + kGrow - kFloor) and their sums in fp32.
constexpr float kShift = 6.f, kGrow = 9.f, kFloor = -80.f;
constexpr _Float16 kMost = 32768.f;
constexpr float kMostSum = 0x1p95f;
constexpr int kRun = 2;  // neighbouring row tiles that one XCD takes, which read the same keys (1: 0.7 % slower, 4: 2.5 %)
static_assert(kThreads == BKV * 8, "one thread per key and 16 values of its row");

template <int SRC>
struct Lds {
  static constexpr bool codes = SRC == SRC_E4M3;              // K as codes
  static constexpr int k_pitch = codes ? D + 16 : 2 * D + 16;
  static constexpr int v_pitch = 2 * D + 64;
  static constexpr int v_off = BKV * k_pitch;
  static constexpr int u_off = v_off + BKV * v_pitch;         // factor of the scores u [64], scale of V [64]
  static constexpr int stage = u_off + 2 * BKV * 4;
  static constexpr int o_pitch = 2 * D + 8;
  static constexpr int out = kWaves * 32 * o_pitch;
  static constexpr int bytes = 3 * stage;
  static_assert(bytes >= out, "the results are staged in the same LDS");
};

// 4 codes as 4 fp16 (exact), negated if `neg`.
template <int SRC>
__device__ inline uint2 codes_f16(uint32_t w, bool neg) {
  if constexpr (SRC == SRC_E4M3) {
    w ^= neg ? 0x80808080u : 0u;
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)));
  } else {
    // code + 128 as the last byte of 1024 + it, less 1152
    const uint32_t x = w ^ 0x80808080u;
    const _Float16 s1 = static_cast<_Float16>(neg ? -1.0f : 1.0f), k1 = static_cast<_Float16>(neg ? 1152.0f : -1152.0f);
    const v2h s = {s1, s1}, k = {k1, k1};
    const uint32_t lo = __builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u), hi = __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u);
    return make_uint2(__builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, lo), s, k)),
                      __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(v2h, hi), s, k)));
  }
}

// 4 int8 codes as 4 bf16 (exact).
__device__ inline uint2 i8_bf16(uint32_t w) {
  return make_uint2(cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w)), static_cast<float>(static_cast<int8_t>(w >> 8))),
                    cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w >> 16)), static_cast<float>(static_cast<int8_t>(w >> 24))));
}

__device__ inline uint32_t cvt_f16x2(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, v2h));
}

__device__ inline bool finite(float v) { return (f32_bits(v) & 0x7f800000u) != 0x7f800000u; }

// SMALL: pages of fewer than 64 positions, where every lane finds its own key's page.
template <int SRC, bool SMALL>
__global__ __launch_bounds__(kThreads, 1) void attn_wide_kernel(Args a) {
  using L = Lds<SRC>;
  constexpr bool kCodes = SRC == SRC_E4M3;
  __shared__ __attribute__((aligned(16))) uint8_t lds[L::bytes];

  if (blockIdx.x >= a.clear_from) return clear_rest<kThreads>(a);
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, half = lane >> 5;

  // Item: runs of kRun neighbouring row tiles go to the XCDs in turn (workgroups are dealt to them round-robin), the
  // heads of a run one after the other.  The last tiles of a sequence, whose causal rows see most, come first in every
  // head, so that little is left at the end (two clips of 7 frames: 10 % less time than with a head after the other).
  const int runs = (a.n_tiles + kRun - 1) / kRun;
  const int xcd = static_cast<int>(blockIdx.x) % kXcds, slot = static_cast<int>(blockIdx.x) / kXcds;
  const int i_run = (slot / kRun) * kXcds + xcd;
  const int head = i_run % a.n_kv_heads, rs = i_run / a.n_kv_heads;
  const int w = a.n_tiles - 1 - (rs % runs) * kRun - slot % kRun, split = a.n_splits - 1 - rs / runs;
  Tile t;
  if (w < 0 || split < 0 || !find_tile<false>(a, w, t)) return;
  const int lim_max = tile_max(a, t), lim_min = tile_min(a, t);
  const int splits = used_splits(a, lim_max);
  if (split >= splits) return;
  const int k_lo = split * a.split_keys;
  const int k_hi = uniform(split == splits - 1 ? lim_max : k_lo + a.split_keys);
  const int tile_lo = k_lo / BKV, tile_hi = (k_hi + BKV - 1) / BKV;

  // this wave's rows: the lane's own, and the largest limit
  const int my_first = t.first + 32 * wave;
  const int r = my_first + l32;
  const bool row_ok = r < t.count;
  uint32_t qi, gi;
  a.group_div.divmod(static_cast<uint32_t>(row_ok ? r : t.first), qi, gi);
  const int lim = row_ok ? row_limit(a, t, static_cast<int>(qi)) : 0;
  int wave_max = 0;
  if (my_first < t.count) wave_max = row_limit(a, t, static_cast<int>(a.group_div.div(min(my_first + 32, t.count) - 1)));
  wave_max = __builtin_amdgcn_readfirstlane(wave_max);

  // ---- staging: key skey of the tile, values 16 schunk .. + 15
  const int skey = tid >> 3, schunk = tid & 7;
  struct Staged {
    u32x4 k0, v0;
    float sk, sv;  // the key's scales
  };
  Staged sreg;
  // Where a tile's keys live (uniform): the first key's row of K and its scale, those of V at the same distance from
  // their pool's start.  A page boundary inside the tile makes cut < 64, and then every lane finds its own key.
  struct Cursor {
    int at, cut, n;   // place in the page; keys to its end; keys that may be read (0: no page)
    const uint8_t* k;
    const float* sk;
  };
  const int pt = a.geom.page_tokens;
  const int32_t* table = a.geom.tables + static_cast<int64_t>(t.b) * a.geom.ld_table;
  const int64_t key_bytes = static_cast<int64_t>(a.n_kv_heads) * D;
  const int64_t k_to_v = a.v_codes - a.k_codes;
  const int64_t sk_to_sv = reinterpret_cast<const uint8_t*>(a.v_scales) - reinterpret_cast<const uint8_t*>(a.k_scales);
  auto cursor_at = [&](int tile) __attribute__((always_inline)) -> Cursor {
    if constexpr (SMALL) return Cursor{};
    uint32_t lp, at;
    a.geom.page.divmod(static_cast<uint32_t>(tile) * BKV, lp, at);
    const int i = static_cast<int>(lp);
    int page = -1;
    if (i < a.geom.ld_table) page = uniform_page(table, i);
    page = __builtin_amdgcn_readfirstlane(page);
    asm volatile("" ::"s"(page));  // awaited here, not among the LDS reads of the tile
    const bool ok = page >= 0 && page < a.geom.pool_pages;
    const int pg = ok ? page : 0, r0 = static_cast<int>(at);
    return Cursor{r0, min(pt - r0, BKV), ok ? BKV : 0, a.k_codes + (static_cast<int64_t>(pg * pt + r0) * a.n_kv_heads + head) * D,
                  a.k_scales + ((pg * a.n_kv_heads + head) * pt + r0)};
  };
  auto cursor_next = [&](const Cursor& c, int tile) __attribute__((always_inline)) -> Cursor {
    if constexpr (SMALL) return c;
    if (c.at + BKV >= pt) return cursor_at(tile);
    return Cursor{c.at + BKV, min(pt - c.at - BKV, BKV), c.n, c.k + BKV * key_bytes, c.sk + BKV};
  };
  Cursor ahead{};
  const uint32_t lane_row = static_cast<uint32_t>(skey) * static_cast<uint32_t>(key_bytes) + 16 * schunk;  // rows of a tile stay below 2^31 bytes (checked on the host)
  constexpr int kWord3 = 0x00020000;  // raw buffer, 32-bit data format
  // SMALL: the page of this lane's key in the tile that is loaded next (-1: none), asked for a tile ahead
  int page_key = -1;
  auto find_page = [&](int tile) __attribute__((always_inline)) {
    const int j = tile * BKV + skey, lp = static_cast<int>(a.geom.page.div(static_cast<uint32_t>(j)));
    page_key = j < k_hi && lp < a.geom.ld_table ? table[lp] : -1;
  };
  // The loads of a tile.  Within one page (ONE) a buffer of the tile's rows that are there reads the others as zero, and
  // a lane's offset never changes.
  auto load_tile = [&](int tile, const Cursor& c, Staged& x, auto ONE) __attribute__((always_inline)) {
    const int n = uniform(min(max(k_hi - tile * BKV, 0), BKV));
    if (decltype(ONE)::value || (!SMALL && c.cut == BKV)) {
      const int m = min(n, c.n);
      const int bytes = m ? (m - 1) * static_cast<int>(key_bytes) + D : 0;
      const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.k), 0, bytes, kWord3);
      const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.k + k_to_v), 0, bytes, kWord3);
      const auto sk = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(c.sk), 0, 4 * m, kWord3);
      const auto sv = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(c.sk) + sk_to_sv), 0, 4 * m, kWord3);
      x.sk = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sk, 4 * skey, 0, 0));
      x.sv = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sv, 4 * skey, 0, 0));
      x.k0 = __builtin_amdgcn_raw_buffer_load_b128(rk, lane_row, 0, 0);
      x.v0 = __builtin_amdgcn_raw_buffer_load_b128(rv, lane_row, 0, 0);
    } else {
      if constexpr (!SMALL) find_page(tile);
      const uint32_t jk = static_cast<uint32_t>(tile * BKV + skey);
      const u32x4 zero = {0, 0, 0, 0};
      x.k0 = x.v0 = zero;
      x.sk = x.sv = 0.f;
      if (page_key >= 0 && page_key < a.geom.pool_pages) {
        const int at = static_cast<int>(jk - a.geom.page.div(jk) * a.geom.page.d);
        const int64_t off = static_cast<int64_t>((page_key * pt + at) * a.n_kv_heads + head) * D + 16 * schunk;
        const int sc = (page_key * a.n_kv_heads + head) * pt + at;
        x.k0 = *reinterpret_cast<const u32x4*>(a.k_codes + off);
        x.v0 = *reinterpret_cast<const u32x4*>(a.v_codes + off);
        x.sk = a.k_scales[sc];
        x.sv = a.v_scales[sc];
      }
    }
  };

  struct Ready {
    uint4 k0, k1, v0, v1;
    float u, sv;
  };
  // The staged tile as it goes to LDS.  PARTIAL: some row may not see all of it.
  auto convert = [&](Staged x, Ready& y, auto PARTIAL) __attribute__((always_inline)) {
    bool poison = !finite(x.sv) || !finite(x.sk);  // the score is NaN for the rows that see the key, the weight of V zero for the others
    if constexpr (SRC == SRC_E4M3 && decltype(PARTIAL)::value) {
      const bool nan = has_nan_code(x.v0[0]) || has_nan_code(x.v0[1]) || has_nan_code(x.v0[2]) || has_nan_code(x.v0[3]);
      const uint64_t any = __ballot(nan);
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v0[e] = without_nan_codes(x.v0[e]);
      poison = poison || (any >> (lane & 56) & 0xffu);
    }
    y.u = poison ? bits_f32(0x7fc00000u) : x.sk * a.c;
    y.sv = poison ? 0.f : fabsf(x.sv);
    const bool neg = x.sv < 0.f;
    if constexpr (kCodes) {
      y.k0 = make_uint4(x.k0[0], x.k0[1], x.k0[2], x.k0[3]);
    } else {
      const uint2 p = i8_bf16(x.k0[0]), q = i8_bf16(x.k0[1]), s = i8_bf16(x.k0[2]), v = i8_bf16(x.k0[3]);
      y.k0 = make_uint4(p.x, p.y, q.x, q.y);
      y.k1 = make_uint4(s.x, s.y, v.x, v.y);
    }
    const uint2 p = codes_f16<SRC>(x.v0[0], neg), q = codes_f16<SRC>(x.v0[1], neg), s = codes_f16<SRC>(x.v0[2], neg), v = codes_f16<SRC>(x.v0[3], neg);
    y.v0 = make_uint4(p.x, p.y, q.x, q.y);
    y.v1 = make_uint4(s.x, s.y, v.x, v.y);
  };
  auto write = [&](int stage, const Ready& y) __attribute__((always_inline)) {
    uint8_t* st = lds + stage;
    uint4* dv = reinterpret_cast<uint4*>(st + L::v_off + skey * L::v_pitch + schunk * 32);
    if constexpr (kCodes) {
      *reinterpret_cast<uint4*>(st + skey * L::k_pitch + schunk * 16) = y.k0;
    } else {
      uint4* dk = reinterpret_cast<uint4*>(st + skey * L::k_pitch + schunk * 32);
      dk[0] = y.k0;
      dk[1] = y.k1;
    }
    dv[0] = y.v0;
    dv[1] = y.v1;
    float* u = reinterpret_cast<float*>(st + L::u_off);
    u[skey] = y.u;  // (the lanes of one key write the same words)
    u[BKV + skey] = y.sv;
  };

  // ---- Q, the second operand of the scores, for the whole kernel
  v8bf qb[kCodes ? 1 : 8];
  v8i q1[kCodes ? 2 : 1], q2[kCodes ? 2 : 1];
  int q_scale = 127;     // e4m3: E8M0 scale of q1
  {
    const uint16_t* qp = a.q + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldq + (head * a.group + static_cast<int>(gi)) * D;
    uint4 raw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // e4m3: values 64 (i / 4) + 32 half + 8 (i % 4) .. + 7; else 16 i + 8 half .. + 7
      raw[i] = *reinterpret_cast<const uint4*>(qp + (kCodes ? 64 * (i >> 2) + 32 * half + 8 * (i & 3) : 16 * i + 8 * half));
      if (!row_ok) raw[i] = make_uint4(0, 0, 0, 0);
    }
    if constexpr (!kCodes) {
#pragma unroll
      for (int i = 0; i < 8; ++i) qb[i] = __builtin_bit_cast(v8bf, raw[i]);
    } else {
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(fabsf(bf16_lo_to_f32(x[e])), fabsf(bf16_hi_to_f32(x[e]))));
      }
      amax = max32(amax);
      const int e = q_exponent(amax);
      q_scale = 127 + e;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint2 c1[4], c2[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_q(nan_if_infinite(raw[4 * m + i], amax), e, c1[i], c2[i]);
        q1[m] = __builtin_bit_cast(v8i, c1);
        q2[m] = __builtin_bit_cast(v8i, c2);
      }
    }
  }

  // Per-lane LDS offsets: K fragment of key block b, step s; V^T operand of d block db, 16-key step, read 0 / 1
  const int k_lane = kCodes ? l32 * L::k_pitch + half * 32 : l32 * L::k_pitch + half * 16;
  const int v_lane = L::v_off + (4 * half + ((lane & 15) >> 2)) * L::v_pitch + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;

  v16f o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  float m_use = -INFINITY;  // the row's maximum in the exponents, log2 units
  float l_run = 0.f;        // this half's row sum
  float neg_m = kShift;

  // Stages (bytes in LDS) of the tiles t - 1, t and t + 1.
  int st_prev = 0, st_cur = L::stage, st_next = 2 * L::stage;
  v16f s[2];        // scores of a tile, between its products and its weights
  uint32_t pw[16];  // weights of a tile, between them and their product with V
#pragma unroll
  for (int i = 0; i < 16; ++i) pw[i] = 0;

  uint4 vf[2][4];
  auto read_v = [&](int stage, int k) __attribute__((always_inline)) {  // V^T operands of 16-key step k
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      const uint8_t* p = lds + stage + v_lane + 16 * k * L::v_pitch + db * 64;
      vf[k & 1][db] = __builtin_bit_cast(uint4, __builtin_shufflevector(read_tr16(p), read_tr16(p + 8 * L::v_pitch), 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  // O^T += V^T P^T of the tile in `stage`, two of its four 16-key steps; steps 0 and 1 of its V are being read.
  auto pv = [&](int stage, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = k0; k < k0 + 2; ++k) {
      const uint4 w = make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, vf[k & 1][db]), __builtin_bit_cast(v8h, w), o[db], 0, 0, 0);
      }
      if (k < 2) read_v(stage, k + 2);
    }
  };

  // The matrix half of tile t: O += the tile before (steps 0 and 1 of its V have been asked for), the scores of t, and
  // among the products the staging of tile t + 1 and the loads of t + 2.  PARTIAL: some row may not see all of t + 1, the
  // wave may see none of t, or the tile to be loaded may span pages; without it the half is one block of instructions.
  float4 uf[2], sf[2];
  auto read_u = [&](int stage, int j) __attribute__((always_inline)) {  // factors and scales of V of the keys 8 j + 4 half + 0 .. 3
    const float* us = reinterpret_cast<const float*>(lds + stage + L::u_off) + 8 * j + 4 * half;
    uf[j & 1] = *reinterpret_cast<const float4*>(us);
    sf[j & 1] = *reinterpret_cast<const float4*>(us + BKV);
  };
  auto products = [&](int tile, auto PARTIAL) __attribute__((always_inline)) {
    constexpr bool kPartial = decltype(PARTIAL)::value;
    using One = std::bool_constant<!kPartial && !SMALL>;
    const uint8_t* st = lds + st_cur;
    Ready nxt;
    __builtin_amdgcn_s_setprio(1);
    auto scores = [&](const auto& kf) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
      if constexpr (kCodes) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int m = i >> 2, b = i & 1;
          if (i & 2)
            s[b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kf[b][m], q1[m], s[b], 0, 0, 0, 127, 0, q_scale);
          else
            s[b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kf[b][m], q2[m], s[b], 0, 0, 0, 127, 0, q_scale - 4);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            s[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, kf[b][ks]), qb[ks], s[b], 0, 0, 0);
      }
    };
    pv(st_prev, 0);
    convert(sreg, nxt, PARTIAL);
    if constexpr (!kPartial) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction, two LDS reads, some vector work
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // (K's fragments take the registers that V's first steps leave)
    std::conditional_t<kCodes, v8i, uint4> kf[2][kCodes ? 2 : 8];
#pragma unroll
    for (int i = 0; i < (kCodes ? 2 : 8); ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if constexpr (kCodes) {
          const uint8_t* p = st + k_lane + b * 32 * L::k_pitch + 64 * i;
          const v4i lo = *reinterpret_cast<const v4i*>(p), hi = *reinterpret_cast<const v4i*>(p + 16);
          kf[b][i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
          kf[b][i] = *reinterpret_cast<const uint4*>(st + k_lane + b * 32 * L::k_pitch + i * 32);
        }
      }
    pv(st_prev, 2);
    __builtin_amdgcn_sched_barrier(0);
    if (!kPartial || tile * BKV < wave_max) scores(kf);
    write(st_next, nxt);
    load_tile(tile + 2, ahead, sreg, One{});
    if constexpr (SMALL) find_page(tile + 3);
    read_u(st_cur, 0);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };

  // The vector half: the weights of tile t (in `stage`) from its scores.
  auto weigh = [&](int tile, int stage, auto PARTIAL) __attribute__((always_inline)) {
    constexpr bool kPartial = decltype(PARTIAL)::value;
    const float* us = reinterpret_cast<const float*>(lds + stage + L::u_off);
    if (kPartial && tile * BKV >= wave_max) {
#pragma unroll
      for (int i = 0; i < 16; ++i) pw[i] = 0;
      read_v(stage, 0);
      read_v(stage, 1);
      return;
    }
    if constexpr (kPartial) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = tile * BKV + 32 * b + 8 * (e >> 2) + 4 * half + (e & 3) >= lim ? -INFINITY : s[b][e];
    }
    auto factor = [&](float u, float x) __attribute__((always_inline)) {  // a key that the row does not see has a score of -inf and may have any factor
      if constexpr (kPartial) return x == -INFINITY ? 1.f : u;
      return u;
    };
    // The weights against the row's reference so far.  Whether it still serves shows in the largest of the fp16 weights (and in
    // the sum, where scales are near zero); if not, and before a row's first key, the exact maximum is taken and the
    // weights are computed again.  So no tile pays for an exact maximum that does not change.
    float l_tile;
    v2h top;
    auto weights = [&]() __attribute__((always_inline)) {
      l_tile = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < 7) read_u(stage, j + 1);
        const float u[4] = {uf[j & 1].x, uf[j & 1].y, uf[j & 1].z, uf[j & 1].w};
        const float sv[4] = {sf[j & 1].x, sf[j & 1].y, sf[j & 1].z, sf[j & 1].w};
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[j >> 2][4 * (j & 3) + e];
          p[e] = __builtin_amdgcn_exp2f(fmaf(x, factor(u[e], x), neg_m));
          l_tile += p[e];
          p[e] *= sv[e];
        }
        pw[2 * j] = cvt_f16x2(p[0], p[1]);
        pw[2 * j + 1] = cvt_f16x2(p[2], p[3]);
        const v2h lo = __builtin_bit_cast(v2h, pw[2 * j]), hi = __builtin_bit_cast(v2h, pw[2 * j + 1]);
        top = j ? __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, lo), hi) : __builtin_elementwise_maximum(lo, hi);
      }
    };
    weights();
    // (NaN needs no other reference; m_use is -inf until the row has seen a key, and its weights count for nothing)
    if (__ballot(top[0] > kMost || top[1] > kMost || l_tile > kMostSum || m_use == -INFINITY)) {
      float mt = -INFINITY;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 x = *reinterpret_cast<const float4*>(us + 32 * b + 8 * g + 4 * half);
          const float4 z = *reinterpret_cast<const float4*>(us + BKV + 32 * b + 8 * g + 4 * half);
          const float u[4] = {x.x, x.y, x.z, x.w}, sv[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mt = fmaxf(mt, fmaf(s[b][4 * g + e], factor(u[e], s[b][4 * g + e]), fmaxf(__builtin_amdgcn_logf(sv[e]), kFloor)));
          __builtin_amdgcn_sched_barrier(0);
        }
      mt = max32(mt);
      const bool fire = m_use == -INFINITY || mt - m_use > kGrow;
      const float m_new = fire ? fmaxf(m_use, mt) : m_use;
      // (in two steps: a sum of small scales' p may be large, and still count where the step as one is below 2^-126)
      const float alpha = m_new == m_use ? 1.f : m_use == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (m_use - m_new));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] *= alpha * alpha;
      l_run = l_run * alpha * alpha;
      m_use = m_new;
      neg_m = m_new == -INFINITY ? kShift : kShift - m_new;
      read_u(stage, 0);
      weights();
    }
    l_run += l_tile;
    read_v(stage, 0);
    read_v(stage, 1);
    __builtin_amdgcn_sched_barrier(0);
  };

  // The waves of a SIMD (w and w + 4) are half a tile apart: while one runs its products the other computes weights, so
  // neither the matrix cores nor the vector unit waits for the other.  A barrier ends each half; the late waves read V of
  // tile t - 1 while the early ones stage t + 1, hence three stages.
  if (tile_lo < tile_hi) {
    const bool late = wave >= kWaves / 2;
    Cursor c = cursor_at(tile_lo);
    if constexpr (SMALL) find_page(tile_lo);
    load_tile(tile_lo, c, sreg, std::false_type{});
    Ready y;
    convert(sreg, y, std::true_type{});
    write(st_cur, y);
    {  // the tile before the first: no weights, and V that they can multiply
      uint4* dv = reinterpret_cast<uint4*>(lds + st_prev + L::v_off + skey * L::v_pitch + schunk * 32);
      dv[0] = dv[1] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) vf[i >> 2][i & 3] = make_uint4(0, 0, 0, 0);
    c = cursor_next(c, tile_lo + 1);
    if constexpr (SMALL) find_page(tile_lo + 1);
    load_tile(tile_lo + 1, c, sreg, std::false_type{});
    ahead = cursor_next(c, tile_lo + 2);
    if constexpr (SMALL) find_page(tile_lo + 2);
    __syncthreads();
    // whole: tiles that every row sees, and the next one too
    const int whole = min(max(lim_min / BKV - 1, tile_lo), tile_hi);
    auto one_page = [&]() __attribute__((always_inline)) { return SMALL || ahead.cut == BKV; };
    auto rotate = [&](const Cursor& after) __attribute__((always_inline)) {
      const int x = st_prev;
      st_prev = st_cur;
      st_cur = st_next;
      st_next = x;
      ahead = after;
    };
    int tile = tile_lo;
    if (!late) {
      auto step = [&](auto PARTIAL) __attribute__((always_inline)) {
        const Cursor after = cursor_next(ahead, tile + 3);  // (branches come first: behind them the tile is one block)
        products(tile, PARTIAL);
        weigh(tile, st_cur, PARTIAL);
        rotate(after);
        __syncthreads();
        ++tile;
      };
      while (tile < tile_hi) {
        while (tile < whole && one_page()) step(std::false_type{});  // (a loop of its own: O stays in its registers)
        if (tile < tile_hi) step(std::true_type{});
      }
    } else {
      products(tile, std::true_type{});
      rotate(cursor_next(ahead, tile + 3));
      __syncthreads();
      ++tile;
      auto step = [&](auto PARTIAL) __attribute__((always_inline)) {
        const Cursor after = cursor_next(ahead, tile + 3);
        weigh(tile - 1, st_prev, PARTIAL);
        products(tile, PARTIAL);
        rotate(after);
        __syncthreads();
        ++tile;
      };
      while (tile < tile_hi) {
        while (tile < whole && one_page()) step(std::false_type{});
        if (tile < tile_hi) step(std::true_type{});
      }
      weigh(tile - 1, st_prev, std::true_type{});
    }
    pv(st_prev, 0);
    pv(st_prev, 2);
    __syncthreads();
  }

  // the rows' results: through LDS as bf16 rows (every wave its own; the last barrier has retired the stages), or, with
  // several splits, in fp32 to the workspace
  const float l_tot = sum32(l_run);
  const float inv = row_inverse(l_tot, splits > 1 ? 0 : lim);  // (of several splits the join sees whether all are empty)
  if (splits > 1) {
    if (!row_ok) return;
    const int64_t at = ((static_cast<int64_t>(w) * a.n_kv_heads + head) * a.n_splits + split) * R + 32 * wave + l32;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(a.part_o + at * D + 32 * db + 8 * g + 4 * half) =
            make_float4(o[db][4 * g] * inv, o[db][4 * g + 1] * inv, o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv);
    if (half == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m_use, l_tot);
    return;
  }
  uint8_t* ow = lds + wave * 32 * L::o_pitch;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(ow + l32 * L::o_pitch + 64 * db + 16 * g + 8 * half) =
          make_uint2(cvt_bf16x2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv), cvt_bf16x2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv));
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = 2 * i + half;
    const uint2 v = *reinterpret_cast<const uint2*>(ow + row * L::o_pitch + 8 * l32);
    if (my_first + row < t.count) {
      uint32_t qj, gj;
      a.group_div.divmod(static_cast<uint32_t>(my_first + row), qj, gj);
      *reinterpret_cast<uint2*>(a.out + static_cast<int64_t>(t.row0 + static_cast<int>(qj)) * a.ldo +
                                (head * a.group + static_cast<int>(gj)) * D + 4 * l32) = v;
    }
  }
}

}  // namespace

int launch_wide(Args a, int format, bool fresh, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>((a.n_tiles + kRun - 1) / kRun * kRun) * a.n_kv_heads * a.n_splits;
  constexpr int64_t per = kXcds * kRun;
  a.clear_from = static_cast<uint32_t>((items + per - 1) / per * per);
  const dim3 grid(a.clear_from + (fresh ? kClearers : 0));
  const bool small = a.geom.page_tokens < BKV;
  void (*kernel)(Args);
  if (format == WF_KV_E4M3)
    kernel = small ? attn_wide_kernel<SRC_E4M3, true> : attn_wide_kernel<SRC_E4M3, false>;
  else
    kernel = small ? attn_wide_kernel<SRC_INT8, true> : attn_wide_kernel<SRC_INT8, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, a);
  return check_launch("wf_attn_batch (many rows)");
}

}  // namespace attn_batch
}  // namespace wf
