// What the kernels of the batched attention share: arguments, row tiles, limits, splits and partial results.
//
// The n new rows of a sequence and the G = n_heads / n_kv_heads query heads of a key head make n G rows (i, head) over
// the same keys; a workgroup takes a tile of R = 2^tile_shift of them for one key head and one range of the keys.
// Tiles are numbered without gaps over the sequences; the host knows the lengths' sum only, and launches
// (n_rows G >> tile_shift) + n_seqs of them, at least as many as there are (ceil(y) <= floor(y) + 1 for each sequence).
#pragma once

#include "batch_geom.hpp"
#include "fp8_codec.hpp"
#include "wf_common.hpp"

namespace wf {
namespace attn_batch {

constexpr int D = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxKeys = 0x7fffffff - 1024;  // of a sequence: the tiles that are loaded ahead stay below 2^31
constexpr float kTau = 8.0f;  // lazy rescale: a row's maximum in its exponents is raised when exceeded by more than this
enum { SRC_E4M3 = WF_KV_E4M3, SRC_INT8 = WF_KV_INT8, SRC_DENSE = 2 };

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct Args {
  const uint16_t* q;
  uint16_t* out;
  int64_t ldq, ldo;
  const uint8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  const uint16_t *k_dense, *v_dense;
  const int32_t* cu_kv;  // dense: [n_seqs + 1]
  int64_t ldkv;
  int32_t n_kv_rows;
  int32_t n_rows, n_kv_heads, group;
  FastDiv group_div;
  int32_t block;
  uint32_t clear_from;  // workgroups from this one on zero the rows of out that no sequence owns
  float c;  // softmax scale * log2(e)
  int32_t tile_shift, n_tiles;
  int32_t split_keys, n_splits;  // keys of a split (a multiple of 64), splits at most
  float* part_o;                 // [n_tiles][n_kv_heads][n_splits][R][D], each divided by its own sum
  float* part_ml;                // [n_tiles][n_kv_heads][n_splits][R][2]: maximum (log2 units) and sum
  BatchGeom geom;
};

// A value that all lanes hold, in a scalar register.
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A workgroup's rows and keys (all uniform).
struct Tile {
  int b;          // sequence
  int row0;       // its first row in q
  int n_new;      // its rows that are in q
  int pos0;       // position of its first row (the rows of cu count, also those past q's last)
  int first;      // the tile's first (i, head) row of the sequence
  int count;      // (i, head) rows of the sequence
  int kv_len;
  int key0;       // dense: the sequence's first key row
};

// Sum of the lanes up to this one.
__device__ inline int prefix_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1 .. 8 within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lane 15 to the 16 after, 47 likewise
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the 32 after
  return x;
}

// Row tile w of all sequences' tiles, numbered without gaps (so that a grid's surplus workgroups, which hold a place on
// a CU until they have seen that they have no work, come last).  Every lane reads one sequence's starts and length.
template <bool DENSE>
__device__ inline bool find_tile(const Args& a, int w, Tile& t) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int before = 0;  // tiles of the sequences before this turn's
  for (int base = 0; base < a.geom.n_seqs; base += 64) {
    const int i = min(base + lane, a.geom.n_seqs - 1);
    const int r = a.geom.cu[i];
    const int end = a.geom.cu[i + 1];
    const int n = min(end, a.n_rows) - r;
    const int u = DENSE ? a.cu_kv[i] : a.geom.kv_lens[i], v = DENSE ? a.cu_kv[i + 1] : 0;
    const bool some = base + lane < a.geom.n_seqs && r >= 0 && n > 0;
    const int tiles = some ? (n * a.group + (1 << a.tile_shift) - 1) >> a.tile_shift : 0;
    const int sum = before + prefix_sum(tiles);
    const uint64_t past = __ballot(some && sum > w);
    if (past) {
      const int at = __builtin_ctzll(past);
      t.b = base + at;
      t.row0 = __builtin_amdgcn_readlane(r, at);
      t.n_new = __builtin_amdgcn_readlane(n, at);
      t.first = (w - __builtin_amdgcn_readlane(sum - tiles, at)) << a.tile_shift;
      t.count = t.n_new * a.group;
      const int x = __builtin_amdgcn_readlane(u, at), y = __builtin_amdgcn_readlane(v, at);
      if constexpr (DENSE) {
        t.key0 = min(max(x, 0), a.n_kv_rows);
        t.kv_len = min(max(y, t.key0), a.n_kv_rows) - t.key0;
      } else {
        t.key0 = 0;
        t.kv_len = min(max(x, 0), kMaxKeys);
        t.pos0 = t.kv_len - (__builtin_amdgcn_readlane(end, at) - t.row0);
      }
      return t.first >= 0 && t.first < t.count;
    }
    before = __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// Rows that no sequence owns, before the first start and from the last one on, are zeroed in a fresh output by kClearers
// workgroups of their own behind the grid's others.
constexpr int kClearers = 128;
template <int THREADS>
__device__ inline void clear_rest(const Args& a) {
  const int before = min(max(a.geom.cu[0], 0), a.n_rows), from = min(max(a.geom.cu[a.geom.n_seqs], before), a.n_rows);
  const int n = before + a.n_rows - from, width = a.n_kv_heads * a.group * D;
  for (int i = static_cast<int>(blockIdx.x - a.clear_from); i < n; i += kClearers) {
    uint16_t* p = a.out + static_cast<int64_t>(i < before ? i : i - before + from) * a.ldo;
    for (int c = 4 * static_cast<int>(threadIdx.x); c < width; c += 4 * THREADS) *reinterpret_cast<uint2*>(p + c) = make_uint2(0, 0);
  }
}

// Keys that row i of the tile's sequence sees (0 .. lim).
__device__ inline int row_limit(const Args& a, const Tile& t, int i) {
  if (a.block == 0) return t.kv_len;
  const int p = t.pos0 + i;
  if (p < 0) return 0;
  const int64_t end = (static_cast<int64_t>(p / a.block) + 1) * a.block;
  return static_cast<int>(min(static_cast<int64_t>(t.kv_len), end));
}

// Limits of the tile's first and last rows: the smallest and the largest of its rows.
__device__ inline int tile_min(const Args& a, const Tile& t) { return row_limit(a, t, a.group_div.div(t.first)); }
__device__ inline int tile_max(const Args& a, const Tile& t) {
  const int last = min(t.first + (1 << a.tile_shift), t.count) - 1;
  return row_limit(a, t, a.group_div.div(last));
}

// Splits that hold keys of a tile whose rows see up to lim keys.
__device__ inline int used_splits(const Args& a, int lim) {
  return min(a.n_splits, max(lim - 1, 0) / a.split_keys + 1);
}

// 1 / sum of a row's weights.  A row that sees keys and whose weights are all zero has scores of -inf only (an infinite q, or
// dense keys that are): there is no mean of them, and it is NaN.
__device__ inline float row_inverse(float sum, int lim) {
  return sum != 0.f ? 1.0f / sum : lim > 0 ? bits_f32(0x7fc00000u) : 0.f;
}

// Two fp32 -> packed bf16x2, round to nearest even.
__device__ inline uint32_t cvt_bf16x2(float lo, float hi) { return pack_bf16x2_hw(lo, hi); }

// Transposing LDS reads: 4 elements of 16 bits (of 8 bytes of 8 bits) of one column for each lane of a 16-lane group.
__device__ inline v4s read_tr16(const uint8_t* addr) {
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(addr));
}
__device__ inline v2i read_tr8(const uint8_t* addr) {
  typedef __attribute__((address_space(3))) v2i lds_v2i;
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(addr));
}

// Order the wave's own LDS accesses (the hardware keeps them in order; this keeps the compiler to it).
__device__ inline void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// max / sum over lanes l, l ^ 32 and l, l ^ 16.  Inline asm because the compiler reads both results of the swap builtins
// from one register; the s_nop is the wait state that it puts before them.
__device__ inline void swap32(float& lo, float& hi) { asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(lo), "+v"(hi)); }
__device__ inline void swap16(float& lo, float& hi) { asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(lo), "+v"(hi)); }
__device__ inline float max32(float v) {
  float a = v, b = v;
  swap32(a, b);
  return fmaxf(a, b);
}
__device__ inline float max16(float v) {
  float a = v, b = v;
  swap16(a, b);
  return fmaxf(a, b);
}
__device__ inline float sum32(float v) {
  float a = v, b = v;
  swap32(a, b);
  return a + b;
}
__device__ inline float sum16(float v) {
  float a = v, b = v;
  swap16(a, b);
  return a + b;
}

// Q as two e4m3 parts under a power of two: q = 2^e (q1 + q2 / 16) with |q| < 2^8 2^e; q1 holds the 4 leading bits of a
// value, q2 the next 4, exact for a bf16 whose last bit is not below 2^-13 of 2^e.  Exponent of a row from its max|q|:
__device__ inline int q_exponent(float amax) {
  return amax > 0.f ? min(max(__builtin_amdgcn_frexp_expf(amax) - 8, -122), 126) : 0;
}
// 8 values of a row as split_q takes them: a row that holds an infinity becomes NaN, as its scores are.
__device__ inline uint4 nan_if_infinite(const uint4& x, float amax) {
  return amax < INFINITY ? x : make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
}
__device__ inline void split_q(const uint4& x, int e, uint2& q1, uint2& q2) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t c1[2], c2[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float v[4] = {__builtin_ldexpf(bf16_lo_to_f32(w[2 * i]), -e), __builtin_ldexpf(bf16_hi_to_f32(w[2 * i]), -e),
                        __builtin_ldexpf(bf16_lo_to_f32(w[2 * i + 1]), -e), __builtin_ldexpf(bf16_hi_to_f32(w[2 * i + 1]), -e)};
    c1[i] = e4m3_pack4_hw(v[0], v[1], v[2], v[3]);
    float b0, b1, b2, b3;
    e4m3_unpack4_hw(c1[i], b0, b1, b2, b3);
    c2[i] = e4m3_pack4_hw((v[0] - b0) * 16.f, (v[1] - b1) * 16.f, (v[2] - b2) * 16.f, (v[3] - b3) * 16.f);
  }
  q1 = make_uint2(c1[0], c1[1]);
  q2 = make_uint2(c2[0], c2[1]);
}

// True when a byte of w is an e4m3 NaN code; the word with those bytes cleared.
__device__ inline bool has_nan_code(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ inline uint32_t without_nan_codes(uint32_t w) {
  const uint32_t n = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return w & ~(n * 0xffu);
}

// (a by value: each sets clear_from)
int launch_few(Args a, int src, int row_blocks, bool fresh, hipStream_t stream);
int launch_wide(Args a, int format, bool fresh, hipStream_t stream);
int launch_dense(Args a, bool fresh, hipStream_t stream);

}  // namespace attn_batch
}  // namespace wf
