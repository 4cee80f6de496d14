// Batched attention, many rows over dense bf16 keys: tiles of 128 (row, head) rows of a sequence over one key head.  Bound
// by the matrix cores and the exponentials between their products; over the few hundred keys of a prompt also by the
// time in which q comes and the results go.
//
// Four waves of 32 rows, two workgroups to a CU, which fill each other's waits: while one reads its Q or stores its
// results, or computes weights, the other has the matrix cores.  Keys in tiles of 64 through two LDS stages, filled by
// DMA one tile ahead (dense rows need no conversion, so no register holds them on the way); a barrier per tile.
// S^T = K Q^T on 32x32 products leaves a lane with one row and 32 keys, so a row's sums are in-lane, and its weights
// are directly the second operand of O^T += V^T P^T, whose first operand comes from the staged rows by transposing
// reads.  The 16-byte chunks of a staged row r are permuted by chunk ^= 4 (r % 4) + r / 4 % 4: the reads of K (16 rows
// at one chunk) and the transposing reads of V (4 rows at 4 chunks) then meet no bank twice.
//
// A wave's instructions go out in order, so the vector work is put among the products it does not depend on: the weights of a
// tile's first 32 keys among the scores of the others, theirs among the first half of P V.  A score that passes the
// maximum in use by more than 2^20 (bf16 and fp32 keep their relative precision up to there) has O follow a new one.
//
// Rounded to bf16: the weights p, relative to the maximum in use; the row sum adds the rounded weights.  V is bf16, of any
// magnitude, and the matrix cores take both operands in one type: fp16 weights would need V under a scale of its own, two
// bf16 parts a second product.  It takes a result's error against 64 bits from 1.5e-3 to 1.9e-3 (the bf16 result's own rounding
// is the 1.5e-3) over some hundred keys, to 1.9e-3 from 1.7e-3 over some thousand.
//
// 4 x 4608 rows of 12 heads over the same 256 keys each: 43 us, of which q and the results take 22 at the copy's rate; on
// 256-row tiles with one workgroup to a CU 40 % more, without the order above 6 %.  Over 8192 keys 0.91 ms = 1.02 PFLOP/s, and
// 1.37 with zeros for data: long contexts are bound by the chip's power limit.
#include "attn_batch.hpp"
#include "gemm_core.hpp"

namespace wf {
namespace attn_batch {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int BKV = 64;
constexpr int kWaves = 4;
constexpr int R = 32 * kWaves;
constexpr int kXcds = 8;
constexpr int kRun = 8;  // neighbouring row tiles that one XCD takes, which read the same keys
constexpr int kRowBytes = 2 * D;
constexpr int kVOff = BKV * kRowBytes;
constexpr int kStage = 2 * BKV * kRowBytes;
constexpr int kOutPitch = kRowBytes + 16;
constexpr float kMost = 20.f;  // log2 of the largest weight before the maximum is taken anew
static_assert(kWaves * 32 * kOutPitch <= 2 * kStage, "the results are staged in the same LDS");

// (The parameter is __restrict so that the compiler, which tells the DMA's writes from reads only where an access carries
// alias information, does not wait for the next tile's DMA before each of these.)
__device__ inline v4s read_v(const uint8_t* __restrict p) { return read_tr16(p); }

__global__ __launch_bounds__(64 * kWaves, 2) void attn_dense_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
  if (blockIdx.x >= a.clear_from) return clear_rest<64 * kWaves>(a);
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l32 = lane & 31, half = lane >> 5, l16 = lane & 15;

  // Item: runs of kRun neighbouring row tiles go to the XCDs in turn (workgroups are dealt to them round-robin).
  const int n_items = a.n_tiles * a.n_kv_heads * a.n_splits;
  const int xcd = static_cast<int>(blockIdx.x) % kXcds, slot = static_cast<int>(blockIdx.x) / kXcds;
  const int i_lin = ((slot / kRun) * kXcds + xcd) * kRun + slot % kRun;
  const int w = i_lin % a.n_tiles, hs = i_lin / a.n_tiles;
  const int head = hs % a.n_kv_heads, split = hs / a.n_kv_heads;
  Tile t;
  if (i_lin >= n_items || !find_tile<true>(a, w, t)) return;
  const int splits = used_splits(a, t.kv_len);
  if (split >= splits) return;
  const int k_lo = split * a.split_keys;
  const int k_hi = uniform(split == splits - 1 ? t.kv_len : k_lo + a.split_keys);
  const int tiles = (k_hi - k_lo + BKV - 1) / BKV;

  // ---- DMA of a tile: wave w brings the blocks of 4 rows w, w + 4, .. of K and V; a lane 16 bytes of row lane / 16 of a
  // block.  Rows past the range read as zero.
  const int key_bytes = uniform(static_cast<int>(a.ldkv) * 2);
  const int64_t first = (static_cast<int64_t>(t.key0) + k_lo) * a.ldkv + head * D;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k_dense + first);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v_dense + first);
  int from[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    from[i] = (4 * (4 * i + wave) + (lane >> 4)) * key_bytes + ((l16 ^ (((lane >> 4) << 2) | wave)) << 4);
  int left = k_hi - k_lo;  // keys not asked for yet
  auto fetch = [&](int stage) __attribute__((always_inline)) {
    constexpr int kWord3 = 0x00020000;  // raw buffer, 32-bit data format
    const int bytes = uniform((min(left, BKV) - 1) * key_bytes + kRowBytes);
    const auto rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kp), 0, bytes, kWord3);
    const auto rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vp), 0, bytes, kWord3);
    uint8_t* to = lds + stage + wave * 1024;
#pragma unroll
    for (int i = 0; i < 4; ++i) gemm::dma16(rk, to + i * 4096, from[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) gemm::dma16(rv, to + kVOff + i * 4096, from[i]);
    kp += static_cast<int64_t>(BKV) * key_bytes;
    vp += static_cast<int64_t>(BKV) * key_bytes;
    left -= BKV;
  };
  if (tiles > 0) fetch(0);

  // ---- Q, the second operand of the scores: values 16 i + 8 half .. + 7 of the lane's row
  const int my_first = t.first + 32 * wave;
  const bool row_ok = my_first + l32 < t.count;
  v8bf qb[8];
  {
    uint32_t qi, gi;
    a.group_div.divmod(static_cast<uint32_t>(row_ok ? my_first + l32 : t.first), qi, gi);
    const uint16_t* qp = a.q + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldq + (head * a.group + static_cast<int>(gi)) * D;
#pragma unroll
    for (int i = 0; i < 8; ++i) qb[i] = __builtin_bit_cast(v8bf, *reinterpret_cast<const uint4*>(qp + 16 * i + 8 * half));
  }

  // A lane's LDS offsets: K of row l32 (+ 32 b), chunk 2 s + half, as k_at ^ 32 s; V of row 4 half + l16 / 4
  // (+ 16 k + 8 j), chunk 4 db + 2 (lane / 16 % 2) + l16 % 4 / 2, as v_at ^ (64 db + 32 j).
  const int k_at = l32 * kRowBytes + ((half ^ (((l32 & 3) << 2) | ((l32 >> 2) & 3))) << 4);
  const int v_at = kVOff + (4 * half + (l16 >> 2)) * kRowBytes + ((l16 >> 2) << 6) +
                   (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ half) << 4) + 8 * (lane & 1);

  v16f o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
  float m_use = -INFINITY;  // the row's maximum in the exponents, log2 units
  float neg_m = 0.f;
  float l_run = 0.f;        // this half's row sum

  const float c = fmaxf(a.c, 1.2e-38f);  // not zero, so that a hidden key's -inf stays one
  int stage = 0;
  for (int tile = 0; tile < tiles; ++tile, stage ^= kStage) {
    gemm::wait_counts<0, 15>();  // this wave's part of the tile is there; behind the barrier all of it, and nobody reads the other stage
    __syncthreads();
    if (tile + 1 < tiles) fetch(stage ^ kStage);
    const uint8_t* st = lds + stage;
    const int n = k_hi - k_lo - tile * BKV;  // keys of the tile, if fewer than 64
    auto read_k = [&](int b, int i) __attribute__((always_inline)) {
      return __builtin_bit_cast(v8bf, *reinterpret_cast<const v4i*>(st + (k_at ^ (i << 5)) + b * 32 * kRowBytes));
    };
    auto read_vt = [&](int k, int db) __attribute__((always_inline)) {  // V^T operand of 16 keys k, values 32 db ..
      return __builtin_bit_cast(v8bf, __builtin_shufflevector(read_v(st + (v_at ^ (db << 6)) + 16 * k * kRowBytes),
                                                              read_v(st + (v_at ^ (db << 6 | 32)) + (16 * k + 8) * kRowBytes),
                                                              0, 1, 2, 3, 4, 5, 6, 7));
    };
    v16f s[2];
    v8bf kf[2][8], vf[4][4];
    uint32_t pw[16];
    float l_tile = 0.f;
    // Weights of the keys 32 b + 8 (e / 4) + 4 half + e % 4, values e of s[b]: two of them.
    auto weight2 = [&](int b, int e) __attribute__((always_inline)) {
      const v2bf one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
      uint32_t w2 = cvt_bf16x2(__builtin_amdgcn_exp2f(fmaf(s[b][e], c, neg_m)), __builtin_amdgcn_exp2f(fmaf(s[b][e + 1], c, neg_m)));
      l_tile = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, w2), one, l_tile, false);
      asm volatile("" : "+v"(w2), "+v"(l_tile));  // stays here, among the products
      pw[8 * b + e / 2] = w2;
    };
    // Whether the maximum in use serves the scores s[b]; if not, O, the sum and (b = 1) the first half's weights follow
    // the new one.
    auto follow = [&](int b) __attribute__((always_inline)) {
      if (n < BKV) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = 32 * b + 8 * (e >> 2) + 4 * half + (e & 3) >= n ? -INFINITY : s[b][e];
      }
      float mt = s[b][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mt = fmaxf(mt, s[b][e]);
      mt *= c;
      if (__ballot(mt + neg_m > kMost || m_use == -INFINITY)) {
        mt = max32(mt);
        const bool fire = mt + neg_m > kMost || m_use == -INFINITY;
        const float m_new = fire ? fmaxf(m_use, mt) : m_use;
        const float alpha = !fire || m_new == m_use ? 1.f : m_use == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_use - m_new);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        l_run *= alpha;
        m_use = m_new;
        neg_m = m_new == -INFINITY ? 0.f : -m_new;
        if (b == 1) {
          l_tile = 0.f;
#pragma unroll
          for (int e = 0; e < 16; e += 2) weight2(0, e);
        }
      }
    };
    auto pv = [&](int k, int db) __attribute__((always_inline)) {
      const uint4 p = make_uint4(pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]);
      o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[k][db], __builtin_bit_cast(v8bf, p), o[db], 0, 0, 0);
    };
#pragma unroll
    for (int b = 0; b < 2; ++b) s[b] = v16f{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[0][i] = read_k(0, i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[0][i], qb[i], s[0], 0, 0, 0);
      kf[1][i] = read_k(1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    follow(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[1][i], qb[i], s[1], 0, 0, 0);
      vf[i >> 2][i & 3] = read_vt(i >> 2, i & 3);
      weight2(0, 2 * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    follow(1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pv(i >> 2, i & 3);
      vf[2 + (i >> 2)][i & 3] = read_vt(2 + (i >> 2), i & 3);
      weight2(1, 2 * i);
      __builtin_amdgcn_sched_barrier(0);
    }
    l_run += l_tile;
#pragma unroll
    for (int i = 0; i < 8; ++i) pv(2 + (i >> 2), i & 3);
  }

  // the rows' results: through LDS as bf16 rows, every wave its own, or, with several splits, in fp32 to the workspace
  const float l_tot = sum32(l_run);
  const float inv = row_inverse(l_tot, splits > 1 ? 0 : t.kv_len);  // (of several splits the join sees whether all are empty)
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
  __syncthreads();  // nobody reads the stages any more
  uint8_t* ow = lds + wave * 32 * kOutPitch;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<uint2*>(ow + l32 * kOutPitch + 64 * db + 16 * g + 8 * half) =
          make_uint2(cvt_bf16x2(o[db][4 * g] * inv, o[db][4 * g + 1] * inv), cvt_bf16x2(o[db][4 * g + 2] * inv, o[db][4 * g + 3] * inv));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    typedef u32x4 __attribute__((aligned(8))) u32x4_at8;  // (out and its rows are 8-byte aligned)
    const int row = 4 * i + (lane >> 4);
    const u32x4 v = *reinterpret_cast<const u32x4*>(ow + row * kOutPitch + 16 * l16);
    if (my_first + row < t.count) {
      uint32_t qj, gj;
      a.group_div.divmod(static_cast<uint32_t>(my_first + row), qj, gj);
      *reinterpret_cast<u32x4_at8*>(a.out + static_cast<int64_t>(t.row0 + static_cast<int>(qj)) * a.ldo +
                                    (head * a.group + static_cast<int>(gj)) * D + 8 * l16) = v;
    }
  }
}

}  // namespace

int launch_dense(Args a, bool fresh, hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(a.n_tiles) * a.n_kv_heads * a.n_splits;
  constexpr int64_t per = kXcds * kRun;
  a.clear_from = static_cast<uint32_t>((items + per - 1) / per * per);
  const dim3 grid(a.clear_from + (fresh ? kClearers : 0));
  hipLaunchKernelGGL(attn_dense_kernel, grid, dim3(64 * kWaves), 0, stream, a);
  return check_launch("wf_attn_batch (many rows, dense keys)");
}

}  // namespace attn_batch
}  // namespace wf
