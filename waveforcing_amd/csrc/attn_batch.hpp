// What the kernels of the batched attention share: arguments, row tiles, limits, splits and partial results.
//
// The n new rows of a sequence and the G = n_heads / n_kv_heads query heads of a key head make n G rows (i, head) over
// the same keys; a workgroup takes a tile of R = 2^tile_shift of them for one key head and one range of the keys.
// Tiles are numbered without knowing the lengths on the host: sequence b's begin at (cu[b] G >> tile_shift) + b, which
// leaves room for all of them (floor(y) - floor(x) + 1 >= ceil(y - x)), so a launch over
// (n_rows G >> tile_shift) + n_seqs tiles covers the batch and at most one tile of a sequence stays empty.
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
  float c;  // softmax scale * log2(e)
  int32_t tile_shift, n_tiles;
  int32_t split_keys, n_splits;  // keys of a split (a multiple of 64), splits at most
  float* part_o;                 // [n_tiles][n_kv_heads][n_splits][R][D], each divided by its own sum
  float* part_ml;                // [n_tiles][n_kv_heads][n_splits][R][2]: maximum (log2 units) and sum
  BatchGeom geom;
};

// A value that all lanes hold, in a scalar register.
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Sequence of row tile w (uniform); n_seqs > 0.
__device__ inline int tile_seq(const Args& a, int w) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int n = 0;
  for (int base = 0; base < a.geom.n_seqs; base += 64) {
    const int i = base + lane;
    const int at = i < a.geom.n_seqs ? ((a.geom.cu[i] * a.group) >> a.tile_shift) + i : 0x7fffffff;
    const int here = __popcll(__ballot(at <= w));
    n += here;
    if (here < 64) break;
  }
  return n - 1;
}

// A workgroup's rows and keys (all uniform).
struct Tile {
  int b;          // sequence
  int row0;       // its first row in q
  int n_new;      // its rows
  int first;      // the tile's first (i, head) row of the sequence
  int count;      // (i, head) rows of the sequence
  int kv_len;
  int key0;       // dense: the sequence's first key row
};

template <bool DENSE>
__device__ inline bool find_tile(const Args& a, int w, Tile& t) {
  t.b = uniform(tile_seq(a, w));
  if (t.b < 0) return false;
  t.row0 = uniform(a.geom.cu[t.b]);
  const int end = min(uniform(a.geom.cu[t.b + 1]), a.n_rows);
  t.n_new = end - t.row0;
  if (t.row0 < 0 || t.n_new <= 0) return false;
  t.first = (w - ((t.row0 * a.group) >> a.tile_shift) - t.b) << a.tile_shift;
  t.count = t.n_new * a.group;
  if (t.first < 0 || t.first >= t.count) return false;
  if constexpr (DENSE) {
    t.key0 = min(max(uniform(a.cu_kv[t.b]), 0), a.n_kv_rows);
    t.kv_len = min(max(uniform(a.cu_kv[t.b + 1]), t.key0), a.n_kv_rows) - t.key0;
  } else {
    t.key0 = 0;
    t.kv_len = min(max(uniform(a.geom.kv_lens[t.b]), 0), kMaxKeys);
  }
  return true;
}

// Keys that row i of the tile's sequence sees (0 .. lim).
__device__ inline int row_limit(const Args& a, const Tile& t, int i) {
  if (a.block == 0) return t.kv_len;
  const int p = t.kv_len - t.n_new + i;
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

// Splits that hold keys of a tile whose rows see up to lim keys; the last one takes what is left.
__device__ inline int used_splits(const Args& a, int lim) {
  return lim <= 0 ? 1 : min(a.n_splits, (lim - 1) / a.split_keys + 1);
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

// True when a byte of w is an e4m3 NaN code; the word with those bytes cleared.
__device__ inline bool has_nan_code(uint32_t w) { return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0; }
__device__ inline uint32_t without_nan_codes(uint32_t w) {
  const uint32_t n = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return w & ~(n * 0xffu);
}

int launch_few(const Args& a, int src, int row_blocks, hipStream_t stream);
int launch_wide(const Args& a, int src, hipStream_t stream);

}  // namespace attn_batch
}  // namespace wf
