// Batched attention, few rows: up to 64 (row, head) rows of a sequence over one key head (single tokens, a few drafted
// ones, grouped heads).  The cache is read once and little is computed, so HBM bounds it: 264 bytes a key of an 8-bit
// cache, 136 of an MXFP4 one, 512 of a dense one.
//
// A workgroup owns a tile of 16 or 32 rows, one key head and one range of the keys; every wave takes each W-th tile
// of 32 keys of the range by itself (no barrier in the loop).  Its loads are one tile ahead: a tile's K leaves its
// registers with the scores and its V goes to LDS before them, and then the next tile is asked for, so that few
// registers hold what is in flight and three waves share a SIMD (two with 32 rows; a tile of 64 rows spills and was half
// as fast as two of 32, which read the keys twice, once from HBM).  Pages of 32 positions and more are read by buffer
// loads, whose bounds zero what is not there.  The waves' results are joined in LDS, those of several ranges by the
// join kernel.
//
// Per 32 keys: K comes straight from memory as the first operand of the scores' product S^T = K Q^T, which leaves a lane
// (l, g) with row l and the keys 16 b + 4 g + 0..3.  e4m3 codes go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are,
// against Q in two e4m3 parts; int8 codes are exact in bf16 and go to v_mfma_f32_16x16x32_bf16 as dense keys do.  V goes
// through a wave's own LDS rows, whose transposing reads give the V^T operand of O^T += V^T P^T for the same keys, the
// codes of both formats exact in bf16.  The scales are applied in fp32, s_k c to the scores and s_v to the weights, and
// the weights go in as the sum of two bf16 (16 significant bits; the matrix cores are idle most of the time anyway).
//
// MXFP4 keys go to the scaled product as codes with their scale bytes, a lane's 32 values of a head one block of a row, against Q in
// the two e4m3 parts in the order that the codes have (the lanes of a 4-bit and of an 8-bit operand hold different values);
// V goes to LDS as bf16 with its scale, one conversion for two codes, exact for every scale that append writes, so no factor is
// left for the scores or the weights; those have room for V of any scale (attn_batch.hpp: headroom).  The scale words are loaded whole, one a key: as single bytes, widened as soon as they
// arrive, they made each tile wait for its own loads.
//
// Measured: 64 single tokens of 40 heads over 8 key heads and 8192 keys each 219-224 us (4.9-5.1 TB/s), 256 over 2048 208 us
// (5.3), 12 over 37440 of 12 heads 272 us (5.2); the first over MXFP4 keys 124 us (4.6; over 32768 keys 5.0; two tiles ahead or a
// fourth wave 0-4 %).  With 17 to 64 rows the vector work bounds it: 48 sequences of 25 rows
// over 8192 keys of 8 heads 184-189 us (4.4-4.5), of 60 rows 318-322 us; over MXFP4 keys 128-135 us (3.2-3.3 of 428 MB) and 234-248:
// no unit is full (the vector unit issues in 52 % of the cycles, the matrix cores are busy in 29 %), each tile's chain of steps is; above
// 32 rows a second tile of rows reads and decodes the cache again.
#include "attn_batch.hpp"

namespace wf {
namespace attn_batch {
namespace {

constexpr int KT = 32;  // keys of a wave's tile
constexpr int W = 4;    // waves of a workgroup
constexpr int kQPitch = 2 * D + 16;

template <int SRC, int NB>
struct Form {
  static constexpr bool dense = SRC == SRC_DENSE, mx = SRC == SRC_MXFP4;
  static constexpr int row_bytes = dense ? 256 : mx ? 64 : 128;
  static constexpr int k_loads = 2 * row_bytes / 64;   // 16-byte loads a lane makes of the tile's K (and V)
  static constexpr bool v_bf16 = dense || mx;          // V in LDS (else its codes)
  static constexpr int v_pitch = v_bf16 ? 256 + 32 : 128 + 16;
  static constexpr int wave_lds = KT * v_pitch + 64 * 4;  // V rows, then 32 factors of K and 32 of V
  static constexpr bool q_lds = NB > 1;                   // Q is read from LDS at every tile (one row block: registers)
  static constexpr int q_off = W * wave_lds;
  static constexpr int stage = q_off + (q_lds ? 16 * NB * (kQPitch + 4) : 0);  // and a row's exponent
  static constexpr int o_slot = 16 * NB * D * 4;          // a wave's results, as they are joined
  static constexpr int join = W / 2 * o_slot + 2 * W * 16 * NB * 4;
  static constexpr int lds = stage > join ? stage : join;
  // waves of a SIMD the registers are allotted for
  static constexpr int waves = NB == 1 ? 3 : 2;
};

// 8 codes (2 dwords) as 8 bf16.
template <int SRC>
__device__ inline v8bf to_bf16(uint32_t w0, uint32_t w1) {
  uint32_t o[4];
  if constexpr (SRC == SRC_E4M3) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true));
  } else {
    const uint32_t w[2] = {w0, w1};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      o[2 * i] = cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w[i])), static_cast<float>(static_cast<int8_t>(w[i] >> 8)));
      o[2 * i + 1] = cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w[i] >> 16)),
                                static_cast<float>(static_cast<int8_t>(w[i] >> 24)));
    }
  }
  return __builtin_bit_cast(v8bf, make_uint4(o[0], o[1], o[2], o[3]));
}

__device__ inline float absmax8(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(bf16_lo_to_f32(w[i])), fabsf(bf16_hi_to_f32(w[i]))));
  return m;
}

template <int SRC, int NB>
__global__ __launch_bounds__(64 * W, (Form<SRC, NB>::waves)) void attn_few_kernel(Args a) {
  using F = Form<SRC, NB>;
  constexpr bool kDense = F::dense, kMx = F::mx;
  constexpr bool kScaled = !kDense && !kMx;  // one fp32 scale a key, applied to scores and weights
  constexpr int R = 16 * NB;
  __shared__ __attribute__((aligned(16))) uint8_t lds[F::lds];

  if (blockIdx.x >= a.clear_from) return clear_rest<64 * W>(a);
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  // The splits are the slowest index, so that those which short sequences do not have come last and on every XCD; the
  // heads are turned from tile to tile and split to split, so that an XCD (every eighth workgroup) reads all of them:
  // one that read the same 128 of every 1024 bytes would keep only some of its L2 channels busy (64 sequences of up to
  // 8192 keys over 8 heads: 136 us, 158 with the heads as they come, 182 with the splits fastest).
  const int items = a.n_tiles * a.n_kv_heads;
  const int split = static_cast<int>(blockIdx.x) / items, slot = static_cast<int>(blockIdx.x) % items;
  const int w = slot / a.n_kv_heads, head = (slot + w + (w >> 3) + split) % a.n_kv_heads;
  Tile t;
  if (!find_tile<kDense>(a, w, t)) return;
  const int lim_max = tile_max(a, t), lim_min = tile_min(a, t);
  const int splits = used_splits(a, lim_max);
  if (split >= splits) return;
  const int k_lo = split * a.split_keys;
  const int k_hi = split == splits - 1 ? lim_max : k_lo + a.split_keys;

  // One tile in registers: K rows, V rows, the scales of key lane & 31, and which of its keys have no place to be read
  // from (where every lane finds its own).
  struct Regs {
    u32x4 k[F::k_loads], v[F::k_loads];
    float fk, fv;
    uint32_t ek[2], ev[2];  // MXFP4: the scale bytes of K's key 16 i + l16 and V's 16 i + lane / 4
    uint32_t bad;
  };
  // Where a tile's keys live: in one page (uniform; `n` of them to be read, the others read as zero), or each on its own.
  struct Where {
    bool one;
    int n;
    const uint8_t* k;
    const float* sk;
  };
  // Lane & 31's (position, head) row in the pool and its scale; keys past the range or without a page are not there.
  struct Place {
    int row, scale;
    bool there;
  };
  const int pt = a.geom.page_tokens;
  const int64_t key_bytes = kDense ? a.ldkv * 2 : kMx ? F::row_bytes : static_cast<int64_t>(a.n_kv_heads) * F::row_bytes;
  const int64_t k_to_v = kDense ? reinterpret_cast<const uint8_t*>(a.v_dense) - reinterpret_cast<const uint8_t*>(a.k_dense)
                                : a.v_codes - a.k_codes;
  const int64_t sk_to_sv = reinterpret_cast<const uint8_t*>(a.v_scales) - reinterpret_cast<const uint8_t*>(a.k_scales);
  auto where = [&](int t0) __attribute__((always_inline)) -> Where {
    const int n = uniform(min(max(k_hi - t0, 0), KT));
    if constexpr (kDense)
      return Where{true, n, reinterpret_cast<const uint8_t*>(a.k_dense + head * D) + (static_cast<int64_t>(t.key0) + (n ? t0 : 0)) * key_bytes,
                   nullptr};
    uint32_t lp, at;
    a.geom.page.divmod(static_cast<uint32_t>(t0), lp, at);
    int page = -1;
    if (n && static_cast<int>(lp) < a.geom.ld_table) page = uniform_page(a.geom.tables, static_cast<int64_t>(t.b) * a.geom.ld_table + lp);
    page = uniform(page);
    const bool ok = page >= 0 && page < a.geom.pool_pages;
    const int pg = ok ? page : 0, r0 = static_cast<int>(at);
    if constexpr (kMx) {  // (codes are stored as scales are, head by head)
      const int row = (pg * a.n_kv_heads + head) * pt + r0;
      return Where{r0 + n <= pt, ok ? n : 0, a.k_codes + static_cast<int64_t>(row) * F::row_bytes, a.k_scales + row};
    }
    return Where{r0 + n <= pt, ok ? n : 0, a.k_codes + (static_cast<int64_t>(pg * pt + r0) * a.n_kv_heads + head) * D,
                 a.k_scales + ((pg * a.n_kv_heads + head) * pt + r0)};
  };
  auto place = [&](int t0) __attribute__((always_inline)) -> Place {
    const int j = t0 + (lane & 31);
    Place p{0, 0, false};
    int page, at;
    if (j < k_hi && pool_row(a.geom, t.b, j, page, at))
      p = Place{kMx ? (page * a.n_kv_heads + head) * pt + at : (page * pt + at) * a.n_kv_heads + head, (page * a.n_kv_heads + head) * pt + at, true};
    return p;
  };
  // A lane's K bytes of key l16 of each 16: 16 g + 64 i .. + 15; its V bytes: 16 of row lane / C, C lanes to a row
  constexpr int C = F::row_bytes / 16;
  const uint32_t k_off = static_cast<uint32_t>(l16) * static_cast<uint32_t>(key_bytes) + 16 * g4;
  const uint32_t v_off = static_cast<uint32_t>(lane / C) * static_cast<uint32_t>(key_bytes) + 16 * (lane % C);
  const bool small = !kDense && pt < KT;
  Place next_place{};  // pages of fewer than 32 positions: the keys' places of the tile after, asked for a tile ahead
  auto load = [&](int t0, const Where& c, Regs& x) __attribute__((always_inline)) {
    constexpr int kWord3 = 0x00020000;  // raw buffer, 32-bit data format
    if (kDense || c.one) {
      const int bytes = uniform(c.n ? (c.n - 1) * static_cast<int>(key_bytes) + F::row_bytes : 0);
      const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.k), 0, bytes, kWord3);
      const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(c.k + k_to_v), 0, bytes, kWord3);
      if constexpr (!kDense) {
        const auto sk = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(c.sk), 0, 4 * c.n, kWord3);
        const auto sv = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(c.sk) + sk_to_sv), 0, 4 * c.n, kWord3);
        if constexpr (kMx) {  // (whole words: a byte would be awaited where it is widened, with the tile's other loads)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x.ek[i] = __builtin_amdgcn_raw_buffer_load_b32(sk, 64 * i + 4 * l16, 0, 0);
            x.ev[i] = __builtin_amdgcn_raw_buffer_load_b32(sv, 64 * i + (lane & 60), 0, 0);
          }
        } else {
          x.fk = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sk, 4 * (lane & 31), 0, 0));
          x.fv = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sv, 4 * (lane & 31), 0, 0));
        }
      }
#pragma unroll
      for (int i = 0; i < F::k_loads; ++i) {
        constexpr int per = F::k_loads / 2;
        x.k[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, k_off + static_cast<uint32_t>(i / per * 16 * key_bytes) + i % per * 64, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < F::k_loads; ++i)
        x.v[i] = __builtin_amdgcn_raw_buffer_load_b128(rv, v_off + static_cast<uint32_t>(i * (64 / C) * key_bytes), 0, 0);
      x.bad = 0;
    } else {
      const Place p = small ? next_place : place(t0);
      x.bad = static_cast<uint32_t>(__ballot(!p.there));
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint8_t* kp = a.k_codes + static_cast<int64_t>(__shfl(p.row, 16 * b + l16)) * F::row_bytes + 16 * g4;
#pragma unroll
        for (int i = 0; i < F::k_loads / 2; ++i) x.k[F::k_loads / 2 * b + i] = *reinterpret_cast<const u32x4*>(kp + 64 * i);
      }
#pragma unroll
      for (int i = 0; i < F::k_loads; ++i)
        x.v[i] = *reinterpret_cast<const u32x4*>(a.v_codes + static_cast<int64_t>(__shfl(p.row, 64 / C * i + lane / C)) * F::row_bytes + 16 * (lane % C));
      if constexpr (kMx) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x.ek[i] = reinterpret_cast<const uint32_t*>(a.k_scales)[__shfl(p.scale, 16 * i + l16)];
          x.ev[i] = reinterpret_cast<const uint32_t*>(a.v_scales)[__shfl(p.scale, 16 * i + (lane >> 2))];
        }
      } else {
        x.fk = a.k_scales[p.scale];
        x.fv = a.v_scales[p.scale];
      }
    }
  };

  // the first tile is on its way while Q is made ready
  int t0 = k_lo + KT * wave;
  Regs x;
  Where next{};
  if (t0 < k_hi) {
    next = where(t0);
    if (small) next_place = place(t0);
    load(t0, next, x);
    next = where(t0 + W * KT);
    if (small) next_place = place(t0 + W * KT);
  }

  // rows: the lane's row of each 16, where its result goes, and its limit
  int lim[NB];
  int row_at[NB];    // the row of q and out
  int row_head[NB];  // its head's first element
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int r = t.first + 16 * n + l16;
    const bool ok = r < t.count;
    uint32_t qi, gi;
    a.group_div.divmod(static_cast<uint32_t>(ok ? r : t.first), qi, gi);
    lim[n] = ok ? row_limit(a, t, static_cast<int>(qi)) : 0;
    row_at[n] = t.row0 + static_cast<int>(qi);
    row_head[n] = (head * a.group + static_cast<int>(gi)) * D;
  }
  // Q, the second operand of the scores.  e4m3 and MXFP4 keys: q = 2^e (q1 + q2 / 16) as in attn_batch_wide.hip, a lane holding
  // values 16 g .. + 15 and 64 + 16 g .. + 15 (what its two loads of a key hold).  The others: step s of the product takes
  // values 64 (s / 2) + 16 g + 8 (s % 2) .. + 7 (dense: 32 s + 8 g .. + 7).
  constexpr bool kCodes = SRC == SRC_E4M3 || kMx;  // K's codes go to the matrix cores as they are
  auto q_values = [&](int s) { return kDense ? 32 * s + 8 * g4 : 64 * (s >> 1) + 16 * g4 + 8 * (s & 1); };
  constexpr int kFormat = kMx ? 4 : 0;  // of K's codes: e2m1, e4m3
  v8bf qf[4];       // one row block's operands
  v8i qa, qb;       // q1 and q2
  int q_scale[NB];  // E8M0 scale of q1
  uint8_t* qbuf = lds + F::q_off;
  if constexpr (F::q_lds) {
    int32_t* es = reinterpret_cast<int32_t*>(qbuf + R * kQPitch);
    for (int c = static_cast<int>(threadIdx.x); c < R * 16; c += 64 * W) {
      const int r = c >> 4;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (t.first + r < t.count) {
        uint32_t qi, gi;
        a.group_div.divmod(static_cast<uint32_t>(t.first + r), qi, gi);
        v = *reinterpret_cast<const uint4*>(a.q + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldq +
                                            (head * a.group + static_cast<int>(gi)) * D + 8 * (c & 15));
      }
      if constexpr (kCodes) {
        float amax = absmax8(v);
#pragma unroll
        for (int off = 1; off < 16; off *= 2) amax = fmaxf(amax, __shfl_xor(amax, off));
        const int e = q_exponent(amax);
        uint2 c1, c2;
        split_q(nan_if_infinite(v, amax), e, c1, c2);
        *reinterpret_cast<uint2*>(qbuf + r * kQPitch + 8 * (c & 15)) = c1;
        *reinterpret_cast<uint2*>(qbuf + r * kQPitch + D + 8 * (c & 15)) = c2;
        if ((c & 15) == 0) es[r] = 127 + e;
      } else {
        *reinterpret_cast<uint4*>(qbuf + r * kQPitch + 16 * (c & 15)) = v;
      }
    }
    __syncthreads();
    if constexpr (kCodes) {
#pragma unroll
      for (int n = 0; n < NB; ++n) q_scale[n] = es[16 * n + l16];
    }
  } else {
    const bool ok = t.first + l16 < t.count;
    const uint16_t* p = a.q + static_cast<int64_t>(row_at[0]) * a.ldq + row_head[0];
    uint4 v[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      v[s] = *reinterpret_cast<const uint4*>(p + q_values(s));
      if (!ok) v[s] = make_uint4(0, 0, 0, 0);
      qf[s] = __builtin_bit_cast(v8bf, v[s]);
    }
    if constexpr (kCodes) {
      const float amax = max16(max32(fmaxf(fmaxf(absmax8(v[0]), absmax8(v[1])), fmaxf(absmax8(v[2]), absmax8(v[3])))));
      const int e = q_exponent(amax);
      q_scale[0] = 127 + e;
      uint2 c1[4], c2[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) split_q(nan_if_infinite(v[s], amax), e, c1[s], c2[s]);
      qa = __builtin_bit_cast(v8i, c1);
      qb = __builtin_bit_cast(v8i, c2);
    }
  }

  v4f o[NB][8];
  float m[NB], l[NB];  // the row's reference, at most kTau below its maximum (MXFP4: above by `above`), and its lanes' sums
  const float above = kMx ? headroom(lim_max) : 0.f;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[n][i] = v4f{0, 0, 0, 0};
  }

  uint8_t* vbuf = lds + wave * F::wave_lds;
  float* fbuf = reinterpret_cast<float*>(vbuf + KT * F::v_pitch);

  v4f s[NB][2];
  [[maybe_unused]] int ek[2], ev[2];
  // V and the factors to LDS, the scores.
  auto scores = [&](bool masked, Regs& x) __attribute__((always_inline)) {
    if (!kDense && x.bad) {  // keys past the range or without a page: zero K and V
      const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < F::k_loads; ++i) {
        if (x.bad >> (16 * (i / (F::k_loads / 2)) + l16) & 1u) x.k[i] = zero;
        if (x.bad >> (64 / C * i + lane / C) & 1u) x.v[i] = zero;
        if constexpr (kMx) {
          if (x.bad >> (16 * i + l16) & 1u) x.ek[i] = 0;
          if (x.bad >> (16 * i + (lane >> 2)) & 1u) x.ev[i] = 0;
        }
      }
      if (x.bad >> (lane & 31) & 1u) x.fk = x.fv = 0.f;
    }
    if constexpr (kMx) {
      // The lane's bytes: block g4 of K's keys, block lane % 4 of V's.
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ek[i] = static_cast<int>((x.ek[i] >> (8 * g4)) & 0xffu);
        ev[i] = static_cast<int>((x.ev[i] >> (8 * (lane & 3))) & 0xffu);
      }
      // A NaN scale of V, which a weight of zero would not silence, becomes one of K: the score of the key is NaN, and is
      // hidden from the rows that do not see it.
      if (__ballot(max(max(ek[0], ek[1]), max(ev[0], ev[1])) >= kMxNan)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint64_t v_nan = __ballot(ev[i] >= kMxNan);
          if (ek[i] >= kMxNan || (v_nan >> (4 * l16) & 15u)) ek[i] = mx::kNanE;
          if (ev[i] >= kMxNan) ev[i] = 127;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float s = mx::scale_of(ev[i]);
        uint4* p = reinterpret_cast<uint4*>(vbuf + (16 * i + (lane >> 2)) * F::v_pitch + 64 * (lane & 3));
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = mx::decode8(x.v[i][e], s);
      }
    } else if constexpr (kDense) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<u32x4*>(vbuf + (4 * i + (lane >> 4)) * F::v_pitch + 16 * l16) = x.v[i];
    } else {
      fbuf[lane] = lane < 32 ? fmaf(x.fk, 0.f, x.fk * a.c) : x.fv;  // (an infinite scale of K: NaN, whatever the score's sign)
      if (SRC == SRC_E4M3 && masked) {
        // A weight of zero does not silence a NaN of V: where some row does not see some key, a NaN code becomes a NaN
        // scale, which only the weights of rows that see the key meet.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool nan = has_nan_code(x.v[i][0]) || has_nan_code(x.v[i][1]) || has_nan_code(x.v[i][2]) || has_nan_code(x.v[i][3]);
          const uint64_t any = __ballot(nan);
          if (any) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[i][e] = without_nan_codes(x.v[i][e]);
            wave_lds_order();
            if ((lane & 7) == 0 && (any >> lane & 0xffu)) fbuf[32 + 8 * i + (lane >> 3)] = bits_f32(0x7fc00000u);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4*>(vbuf + (8 * i + (lane >> 3)) * F::v_pitch + 16 * (lane & 7)) = x.v[i];
    }
    wave_lds_order();
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n][b] = v4f{0, 0, 0, 0};
    if constexpr (kCodes) {
      v8i kf[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if constexpr (kMx) {
          const v4i c = __builtin_bit_cast(v4i, x.k[b]);
          kf[b] = __builtin_shufflevector(c, c, 0, 1, 2, 3, -1, -1, -1, -1);
        } else {
          kf[b] = __builtin_bit_cast(v8i, *reinterpret_cast<u32x4(*)[2]>(&x.k[2 * b]));
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (F::q_lds) {
          const uint8_t* p = qbuf + (16 * n + l16) * kQPitch + 16 * g4;
          u32x4 q[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const u32x4*>(p + 64 * i);
          qa = __builtin_bit_cast(v8i, *reinterpret_cast<u32x4(*)[2]>(&q[0]));
          qb = __builtin_bit_cast(v8i, *reinterpret_cast<u32x4(*)[2]>(&q[2]));
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) s[n][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf[b], qb, s[n][b], kFormat, 0, 0, kMx ? ek[b] : 127, 0, q_scale[n] - 4);
#pragma unroll
        for (int b = 0; b < 2; ++b) s[n][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf[b], qa, s[n][b], kFormat, 0, 0, kMx ? ek[b] : 127, 0, q_scale[n]);
      }
      return;
    }
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      v8bf kf[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if constexpr (kDense) {
          kf[b] = __builtin_bit_cast(v8bf, x.k[4 * b + ks]);
        } else {
          const u32x4 kk = x.k[2 * b + (ks >> 1)];
          kf[b] = to_bf16<SRC>(kk[2 * (ks & 1)], kk[2 * (ks & 1) + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        v8bf q;
        if constexpr (F::q_lds)
          q = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(qbuf + (16 * n + l16) * kQPitch + 2 * q_values(ks)));
        else
          q = qf[ks];
#pragma unroll
        for (int b = 0; b < 2; ++b) s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[b], q, s[n][b], 0, 0, 0);
      }
    }
  };
  v8bf ph[NB], pl[NB];
  // The weights, as two bf16 parts.
  auto weigh = [&](int t0, bool masked) __attribute__((always_inline)) {
    float u[8], sv[8];
    if constexpr (kScaled) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float4 fu = *reinterpret_cast<const float4*>(fbuf + 16 * b + 4 * g4);
        const float4 fv = *reinterpret_cast<const float4*>(fbuf + 32 + 16 * b + 4 * g4);
        u[4 * b] = fu.x, u[4 * b + 1] = fu.y, u[4 * b + 2] = fu.z, u[4 * b + 3] = fu.w;
        sv[4 * b] = fv.x, sv[4 * b + 1] = fv.y, sv[4 * b + 2] = fv.z, sv[4 * b + 3] = fv.w;
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float x8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x8[e] = s[n][e >> 2][e & 3] * (kScaled ? u[e] : a.c);
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (t0 + 16 * (e >> 2) + 4 * g4 + (e & 3) >= lim[n]) x8[e] = -INFINITY;
      }
      float mt = fmaxf(fmaxf(fmaxf(x8[0], x8[1]), fmaxf(x8[2], x8[3])), fmaxf(fmaxf(x8[4], x8[5]), fmaxf(x8[6], x8[7])));
      mt = max16(max32(mt));
      if constexpr (kMx) mt += above;
      const bool fire = mt > m[n] + kTau;
      if (__ballot(fire)) {
        const float m_new = fire ? mt : m[n];
        const float alpha = fire ? (m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m_new)) : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[n][i] *= alpha;
        l[n] *= alpha;
        m[n] = m_new;
      }
      const float neg = m[n] == -INFINITY ? 0.f : -m[n];
      float hi[8], lo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(x8[e] + neg);
        l[n] += p;
        float wgt = p;
        if constexpr (kScaled) {
          wgt = p * sv[e];
          if (masked && x8[e] == -INFINITY) wgt = 0.f;
        }
        hi[e] = wgt;
      }
      uint32_t wh[4], wl[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wh[e] = cvt_bf16x2(hi[2 * e], hi[2 * e + 1]);
        lo[2 * e] = hi[2 * e] - bf16_lo_to_f32(wh[e]);
        lo[2 * e + 1] = hi[2 * e + 1] - bf16_hi_to_f32(wh[e]);
        wl[e] = cvt_bf16x2(lo[2 * e], lo[2 * e + 1]);
      }
      ph[n] = __builtin_bit_cast(v8bf, make_uint4(wh[0], wh[1], wh[2], wh[3]));
      pl[n] = __builtin_bit_cast(v8bf, make_uint4(wl[0], wl[1], wl[2], wl[3]));
    }
  };
  // O^T += V^T P^T.
  auto pv = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v8bf vf;
      if constexpr (F::v_bf16) {
        const uint8_t* p = vbuf + (4 * g4 + (l16 >> 2)) * F::v_pitch + (16 * i + 4 * (l16 & 3)) * 2;
        vf = __builtin_bit_cast(v8bf, __builtin_shufflevector(read_tr16(p), read_tr16(p + 16 * F::v_pitch), 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        const int j = l16 >> 1;
        const v2i c = read_tr8(vbuf + (16 * (j >> 2) + 4 * g4 + (j & 3)) * F::v_pitch + 16 * i + 8 * (l16 & 1));
        vf = to_bf16<SRC>(static_cast<uint32_t>(c[0]), static_cast<uint32_t>(c[1]));
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph[n], o[n][i], 0, 0, 0);
        o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[n], o[n][i], 0, 0, 0);
      }
      if (i & 1) __builtin_amdgcn_sched_barrier(0);  // (reads of two blocks at a time: registers)
    }
    wave_lds_order();
  };

  for (; t0 < k_hi; t0 += W * KT) {
    const bool masked = t0 + KT > lim_min;
    scores(masked, x);
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + W * KT < k_hi) {
      load(t0 + W * KT, next, x);
      next = where(t0 + 2 * W * KT);
      if (small) next_place = place(t0 + 2 * W * KT);
    }
    __builtin_amdgcn_sched_barrier(0);
    weigh(t0, masked);
    pv();
  }

  // Join the waves: maxima and sums, then the outputs pairwise (wave i takes in wave i + half), in LDS that no wave
  // reads any more.
  __syncthreads();
  float* ms = reinterpret_cast<float*>(lds + W / 2 * F::o_slot);
  float* ls = ms + W * R;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] = sum16(sum32(l[n]));
    if (g4 == 0) {
      ms[wave * R + 16 * n + l16] = m[n];
      ls[wave * R + 16 * n + l16] = l[n];
    }
  }
  __syncthreads();
  float top[NB], sum[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    top[n] = -INFINITY;
    sum[n] = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) top[n] = fmaxf(top[n], ms[i * R + 16 * n + l16]);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float mi = ms[i * R + 16 * n + l16];
      sum[n] += mi == -INFINITY ? 0.f : ls[i * R + 16 * n + l16] * __builtin_amdgcn_exp2f(mi - top[n]);
    }
    const float scale = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - top[n]);
#pragma unroll
    for (int d = 0; d < 8; ++d) o[n][d] *= scale;
  }
#pragma unroll
  for (int half = W / 2; half >= 1; half /= 2) {
    // lane's values 4 floats each, lane-linear: conflict-free
    if (wave >= half && wave < 2 * half) {
      v4f* p = reinterpret_cast<v4f*>(lds + (wave - half) * F::o_slot) + lane;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) p[(8 * n + d) * 64] = o[n][d];
    }
    __syncthreads();
    if (wave < half) {
      const v4f* p = reinterpret_cast<const v4f*>(lds + wave * F::o_slot) + lane;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) o[n][d] += p[(8 * n + d) * 64];
    }
    if (half > 1) __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (t.first + 16 * n + l16 >= t.count) continue;
    const float inv = row_inverse(sum[n], splits > 1 ? 0 : lim[n]);  // (of several splits the join sees whether all are empty)
    if (splits > 1) {
      const int64_t at = ((static_cast<int64_t>(w) * a.n_kv_heads + head) * a.n_splits + split) * R + 16 * n + l16;
#pragma unroll
      for (int d = 0; d < 8; ++d) *reinterpret_cast<v4f*>(a.part_o + at * D + 16 * d + 4 * g4) = o[n][d] * inv;
      if (g4 == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top[n], sum[n]);
    } else {
      uint16_t* p = a.out + static_cast<int64_t>(row_at[n]) * a.ldo + row_head[n] + 4 * g4;
#pragma unroll
      for (int d = 0; d < 8; ++d)
        *reinterpret_cast<uint2*>(p + 16 * d) =
            make_uint2(cvt_bf16x2(o[n][d][0] * inv, o[n][d][1] * inv), cvt_bf16x2(o[n][d][2] * inv, o[n][d][3] * inv));
    }
  }
}

template <int SRC>
void launch(Args& a, int row_blocks, bool fresh, hipStream_t stream) {
  a.clear_from = static_cast<uint32_t>(a.n_tiles) * a.n_kv_heads * a.n_splits;
  const dim3 grid(a.clear_from + (fresh ? kClearers : 0));
  if (row_blocks == 1)
    hipLaunchKernelGGL((attn_few_kernel<SRC, 1>), grid, dim3(64 * W), 0, stream, a);
  else
    hipLaunchKernelGGL((attn_few_kernel<SRC, 2>), grid, dim3(64 * W), 0, stream, a);
}

}  // namespace

int launch_few(Args a, int src, int row_blocks, bool fresh, hipStream_t stream) {
  switch (src) {
    case SRC_E4M3: launch<SRC_E4M3>(a, row_blocks, fresh, stream); break;
    case SRC_MXFP4: launch<SRC_MXFP4>(a, row_blocks, fresh, stream); break;
    case SRC_INT8: launch<SRC_INT8>(a, row_blocks, fresh, stream); break;
    default: launch<SRC_DENSE>(a, row_blocks, fresh, stream); break;
  }
  return check_launch("wf_attn_batch (few rows)");
}

}  // namespace attn_batch
}  // namespace wf
