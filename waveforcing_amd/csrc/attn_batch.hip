// Attention of a batch of sequences: ragged query rows over each sequence's paged quantized keys (e4m3, int8 or MXFP4), or
// over ragged dense bf16 keys.
//
//   out[i, h] = sum_j w_j V[j, g] / sum_j w_j,   w_j = exp(scale <Q[i, h], K[j, g]>),   g = h / (n_heads / n_kv_heads)
//   over the keys j < lim(i) of the row's sequence; K = code_k s_k and V = code_v s_v are products of fp32 numbers (MXFP4: s by
//   blocks of 32).
//   lim = kv_len without a block; min(kv_len, (p / block + 1) block) with one, p = kv_len - new + i the row's position.
//   A row without keys is zero.
//
// Three kernels: attn_batch_few.hip for up to 64 (row, head) rows of a sequence per key head, for more attn_batch_wide.hip
// over pages and attn_batch_dense.hip over dense keys; long caches are split over workgroups, and the join below puts the
// splits' results together in their order.
#include "attn_batch.hpp"
#include "gemm_core.hpp"

#include <algorithm>
#include <cmath>

namespace wf {
namespace attn_batch {
namespace {

constexpr int kJoinRows = 16;    // rows of a workgroup, 16 lanes of 8 values each
constexpr int kJoinSplits = 64;  // splits at most

// out = sum_s l_s 2^(m_s - m) o_s / sum_s l_s 2^(m_s - m) over the splits s of a row tile that used more than one.  Reads
// the partial results once (few of them: 4-5 us, most of it the launch; the rows' 16 lanes keep 8 loads in flight).
template <bool DENSE>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  const int R = 1 << a.tile_shift;
  const int parts = R / kJoinRows;
  const int part = static_cast<int>(blockIdx.x) % parts, item = static_cast<int>(blockIdx.x) / parts;
  const int head = item % a.n_kv_heads, w = item / a.n_kv_heads;
  Tile t;
  if (!find_tile<DENSE>(a, w, t)) return;
  const int splits = used_splits(a, tile_max(a, t));
  if (splits < 2) return;
  const int r = part * kJoinRows + (static_cast<int>(threadIdx.x) >> 4), d = 8 * (static_cast<int>(threadIdx.x) & 15);
  if (t.first + r >= t.count) return;
  const int64_t at = static_cast<int64_t>(item) * a.n_splits * R + r;
  // the splits' maxima and sums: each of the row's 16 lanes reads every 16th, 4 in flight
  const int l16 = static_cast<int>(threadIdx.x) & 15;
  float2 ml[kJoinSplits / 16];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kJoinSplits / 16; ++i) {
    ml[i] = make_float2(-INFINITY, 0.f);
    const int s = 16 * i + l16;
    if (s < splits) ml[i] = *reinterpret_cast<const float2*>(a.part_ml + (at + static_cast<int64_t>(s) * R) * 2);
  }
#pragma unroll
  for (int i = 0; i < kJoinSplits / 16; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
  for (int off = 8; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  float g[kJoinSplits / 16], sum = 0.f, o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kJoinSplits / 16; ++i) {
    const float e = __builtin_amdgcn_exp2f(0.5f * (ml[i].x - top));  // (twice: a sum may be large where its maximum is far below)
    g[i] = ml[i].x == -INFINITY ? 0.f : ml[i].y * e * e;
    sum += g[i];
  }
#pragma unroll
  for (int off = 8; off; off >>= 1) sum += __shfl_xor(sum, off);
  const float* po = a.part_o + at * D + d;
#pragma unroll
  for (int i = 0; i < kJoinSplits / 16; ++i) {
    if (16 * i >= splits) break;
#pragma unroll 8
    for (int j = 0; j < min(16, splits - 16 * i); ++j) {
      const float4* p = reinterpret_cast<const float4*>(po + static_cast<int64_t>(16 * i + j) * R * D);
      const float4 x = p[0], y = p[1];
      const float w = __shfl(g[i], (static_cast<int>(threadIdx.x) & 48) + j);
      const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(w, v[e], o[e]);
    }
  }
  uint32_t qi, gi;
  a.group_div.divmod(static_cast<uint32_t>(t.first + r), qi, gi);
  const float inv = row_inverse(sum, row_limit(a, t, static_cast<int>(qi)));
  uint16_t* p = a.out + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldo + (head * a.group + static_cast<int>(gi)) * D + d;
  *reinterpret_cast<uint2*>(p) = make_uint2(cvt_bf16x2(o[0] * inv, o[1] * inv), cvt_bf16x2(o[2] * inv, o[3] * inv));
  *reinterpret_cast<uint2*>(p + 4) = make_uint2(cvt_bf16x2(o[4] * inv, o[5] * inv), cvt_bf16x2(o[6] * inv, o[7] * inv));
}

// How a call is split: rows of a tile (16 and 32 on the few-rows kernel, 256 and over dense keys 128 on the others),
// tiles, keys of a split.
struct Plan {
  int tile_shift;
  int64_t n_tiles, split_keys, n_splits, bytes;
  bool fits;  // the grids; bytes hold nothing otherwise
};

Plan make_plan(bool dense, int64_t n_rows, int64_t n_heads, int64_t n_kv_heads, int64_t n_seqs, int64_t max_new, int64_t max_kv) {
  const int64_t group = n_heads / n_kv_heads, cus = gemm::device_cus();
  const int64_t most = std::min(max_new, n_rows) * group;
  Plan p;
  p.tile_shift = most <= 16 ? 4 : most <= 64 ? 5 : dense ? 7 : 8;
  p.n_tiles = ((n_rows * group) >> p.tile_shift) + n_seqs;
  const int64_t full = std::max<int64_t>(1, std::min<int64_t>(p.n_tiles, n_seqs * ((most + (1ll << p.tile_shift) - 1) >> p.tile_shift)));
  const int64_t units = full * n_kv_heads;
  p.n_splits = 1;
  if (p.tile_shift > 5) {
    // In times of one 64-key tile of a workgroup (about 2 us; one workgroup to a CU, of 128 rows two): a piece takes its
    // tiles and a fixed part of about 4; the rounds of pieces of one sequence (the pieces of several, whose lengths
    // differ, spread over the CUs, the longest first, with little at the end); partial results of 256 rows are written and
    // read at about 0.03.  Six sequences of up to 10001 keys, 800 tiles: 388 us whole, 466 in two, 494 in four; 8 over up to
    // 4001 dense keys, 216 tiles: 69 whole, 50 in three, 57 in eight.
    const double tiles = static_cast<double>((max_kv + 63) / 64);
    double best = 0;
    for (int64_t s = 1; s <= kJoinSplits && (s == 1 || tiles / s >= 8); ++s) {
      const double pieces = static_cast<double>(units * s), per = tiles / s;
      const double rounds = pieces / (dense ? 2 * cus : cus);
      double cost = n_seqs == 1 ? std::ceil(rounds) * (per + 4) : std::max(rounds, 1.0) * (0.7 * per + 4) + 0.15 * per;
      if (s > 1) cost += 1.5 + (dense ? 0.015 : 0.03) * pieces;
      if (s == 1 || cost < best) {
        best = cost;
        p.n_splits = s;
      }
    }
  } else {
    // A piece costs a workgroup about 5 us besides its keys and the join reads its results: two pieces to a CU if the
    // tiles alone are fewer, of 256 keys at least (12 tiles of 8192 keys: 20 us as 32 pieces each, 121 as one; 128 tiles
    // of 8192 keys: 64 as 4, 147 as one, 68 as 16).  Where the tiles fill the chip, pieces of some 2048 keys, so that a
    // few long sequences do not outlast the rest (512 tiles of 1 to 8192 keys: 138 us, 159 as one; where all are as
    // long, 220 and 214).  One long sequence among many short ones has each of them send as many workgroups that find
    // nothing to do, at some 3 ns each, against 12 ns for a key of the longest piece: at most the square root of 4 max_kv /
    // tiles pieces (256 sequences of 512 keys, one of 131072, 8 heads: 318 us as 16 pieces, 541 as 64, 484 as 4).
    // (The tiles that there are, where sequences differ: half a tile of each is taken to be empty.)
    const int64_t some = std::min(n_seqs, n_rows), likely = ((n_rows * group) >> p.tile_shift) + n_seqs / 2;
    const int64_t tiles = std::max<int64_t>(1, std::min(full, std::max(some, likely))) * n_kv_heads;
    const int64_t even = std::llround(std::sqrt(4.0 * static_cast<double>(max_kv) / static_cast<double>(tiles)));
    p.n_splits = std::max(std::min((max_kv + 2047) / 2048, even), std::min(2 * cus / tiles, (max_kv + 255) / 256));
    p.n_splits = std::min<int64_t>(std::max<int64_t>(1, p.n_splits), kJoinSplits);
  }
  p.split_keys = std::max<int64_t>(128, ((max_kv + p.n_splits - 1) / p.n_splits + 127) / 128 * 128);
  // (a grid holds fewer than 2^32 threads: 512 or fewer of each item, rounded up to 64 items, and kClearers more; 16 x 256 where rows are joined)
  p.fits = product_below({p.n_tiles + 64 + kClearers, n_kv_heads, p.n_splits, 512}, 1ll << 32) &&
           (p.n_splits == 1 || product_below({p.n_tiles, n_kv_heads, 16 * 256}, 1ll << 32));
  p.bytes = p.n_splits == 1 || !p.fits ? 0 : ((p.n_tiles * n_kv_heads * p.n_splits) << p.tile_shift) * (D + 2) * 4;
  return p;
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks that both attentions share; fills the common arguments.
int common_args(const char* fn, Args& a, const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads,
                int64_t ldq, float softmax_scale, void* out, int64_t ldo) {
  WF_REQUIRE(n_heads > 0 && n_heads % n_kv_heads == 0, WF_E_SHAPE, "%s: %d heads do not group over %d key heads", fn,
             n_heads, n_kv_heads);
  WF_REQUIRE(n_heads < (1 << 24), WF_E_SHAPE, "%s: %d heads, 2^24 or more", fn, n_heads);  // (as check_batch's)
  WF_REQUIRE(softmax_scale >= 0.f && std::isfinite(softmax_scale * kLog2e), WF_E_INVALID,
             "%s: softmax_scale=%g must not be negative, and finite as a factor of base-2 exponents too", fn,
             static_cast<double>(softmax_scale));
  const int64_t hd = static_cast<int64_t>(n_heads) * D;
  WF_REQUIRE(ldq >= hd && ldo >= hd, WF_E_INVALID, "%s: ldq/ldo smaller than n_heads*head_dim", fn);
  WF_REQUIRE(product_below({n_rows, n_heads}, (1ll << 31) - 65536), WF_E_SHAPE, "%s: rows=%lld x heads=%d reaches 2^31", fn,
             (long long)n_rows, n_heads);
  WF_REQUIRE(aligned(q, 16) && ldq % 8 == 0 && aligned(out, 8) && ldo % 4 == 0, WF_E_ALIGN,
             "%s: q must be 16-byte aligned (ldq %% 8 == 0), out 8-byte aligned (ldo %% 4 == 0)", fn);
  a = Args{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.ldq = ldq;
  a.ldo = ldo;
  a.n_rows = static_cast<int32_t>(n_rows);
  a.n_kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads;
  a.group_div = FastDiv(static_cast<uint32_t>(a.group));
  a.c = softmax_scale * kLog2e;
  return WF_OK;
}

int launch(const char* fn, Args& a, int src, int64_t n_seqs, int64_t max_new, int64_t max_kv, void* ws, int64_t ws_bytes,
           bool fresh, hipStream_t stream) {
  const Plan p = make_plan(src == SRC_DENSE, a.n_rows, static_cast<int64_t>(a.n_kv_heads) * a.group, a.n_kv_heads, n_seqs, max_new, max_kv);
  WF_REQUIRE(p.fits, WF_E_SHAPE, "%s: %lld row tiles x %d key heads x %lld splits are too many", fn, (long long)p.n_tiles, a.n_kv_heads,
             (long long)p.n_splits);
  WF_REQUIRE(a.ldkv < (1 << 23), WF_E_SHAPE, "%s: key rows of %lld elements", fn, (long long)a.ldkv);
  WF_REQUIRE(ws_bytes >= p.bytes && (p.bytes == 0 || ws), WF_E_INVALID, "%s: a workspace of %lld bytes where %lld are needed", fn,
             (long long)ws_bytes, (long long)p.bytes);
  WF_REQUIRE(aligned(ws, 16), WF_E_ALIGN, "%s: the workspace must be 16-byte aligned", fn);
  a.tile_shift = p.tile_shift;
  a.n_tiles = static_cast<int32_t>(p.n_tiles);
  a.split_keys = static_cast<int32_t>(std::min<int64_t>(p.split_keys, kMaxKeys / 128 * 128));
  a.n_splits = static_cast<int32_t>(p.n_splits);
  a.part_o = static_cast<float*>(ws);
  a.part_ml = a.part_o + ((p.n_tiles * a.n_kv_heads * p.n_splits) << p.tile_shift) * D;
  const int st = p.tile_shift <= 5 ? launch_few(a, src, 1 << (p.tile_shift - 4), fresh, stream)
                 : src == SRC_DENSE ? launch_dense(a, fresh, stream) : launch_wide(a, src, fresh, stream);
  if (st || p.n_splits == 1) return st;
  const dim3 grid(static_cast<uint32_t>((p.n_tiles * a.n_kv_heads) << (p.tile_shift - 4)));
  if (src == SRC_DENSE)
    hipLaunchKernelGGL(join_kernel<true>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(join_kernel<false>, grid, dim3(256), 0, stream, a);
  return check_launch(fn);
}

int paged_batch(const char* fn, bool fresh, const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads,
                int32_t head_dim, int64_t ldq, int32_t format, const uint8_t* k_codes, const uint8_t* v_codes,
                const float* k_scales, const float* v_scales, int64_t pool_pages, int32_t page_tokens,
                const int32_t* cu_new, const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables, int64_t ld_table,
                int64_t max_new, int64_t max_kv, int32_t block, float softmax_scale, void* out, int64_t ldo, void* ws,
                int64_t ws_bytes, void* stream) {
  if (int st = check_batch(fn, n_rows, n_kv_heads, head_dim, cu_new, kv_lens, n_seqs)) return st;
  if (int st = check_pool(fn, format, n_kv_heads, page_tokens, pool_pages, tables, ld_table)) return st;
  WF_REQUIRE(n_rows == 0 || n_seqs == 0 || pool_pages > 0, WF_E_INVALID, "%s: an empty pool", fn);
  WF_REQUIRE(block >= 0, WF_E_INVALID, "%s: block=%d must not be negative", fn, block);
  WF_REQUIRE(max_new >= 0 && max_kv >= 0 && max_kv < (1ll << 31), WF_E_INVALID, "%s: bad bound of the lengths", fn);
  Args a;
  if (int st = common_args(fn, a, q, n_rows, n_heads, n_kv_heads, ldq, softmax_scale, out, ldo)) return st;
  WF_REQUIRE(!fresh || n_rows == 0 || n_seqs > 0, WF_E_INVALID, "%s: rows without a sequence", fn);
  if (n_rows == 0 || n_seqs == 0) return WF_OK;
  WF_REQUIRE(q && out && k_codes && v_codes && k_scales && v_scales, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16), WF_E_ALIGN, "%s: code pools must be 16-byte aligned", fn);
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.block = block;
  a.geom = make_batch_geom(cu_new, kv_lens, n_seqs, tables, ld_table, page_tokens, pool_pages);
  return launch(fn, a, format, n_seqs, max_new, max_kv, ws, ws_bytes, fresh, as_stream(stream));
}

int cross_batch(const char* fn, bool fresh, const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads,
                int32_t head_dim, int64_t ldq, const void* k, const void* v, int64_t n_kv_rows, int64_t ldkv,
                const int32_t* cu_q, const int32_t* cu_kv, int64_t n_seqs, int64_t max_q, int64_t max_kv,
                float softmax_scale, void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  if (int st = check_batch(fn, n_rows, n_kv_heads, head_dim, cu_q, cu_kv, n_seqs)) return st;
  WF_REQUIRE(max_q >= 0 && max_kv >= 0 && max_kv < (1ll << 31), WF_E_INVALID, "%s: bad bound of the lengths", fn);
  WF_REQUIRE(n_kv_rows >= 0 && n_kv_rows < kMaxKeys, WF_E_SHAPE, "%s: %lld key rows", fn, (long long)n_kv_rows);
  WF_REQUIRE(ldkv >= static_cast<int64_t>(n_kv_heads) * head_dim && ldkv % 8 == 0, WF_E_INVALID,
             "%s: ldkv=%lld must be >= n_kv_heads*head_dim and a multiple of 8", fn, (long long)ldkv);
  Args a;
  if (int st = common_args(fn, a, q, n_rows, n_heads, n_kv_heads, ldq, softmax_scale, out, ldo)) return st;
  WF_REQUIRE(!fresh || n_rows == 0 || n_seqs > 0, WF_E_INVALID, "%s: rows without a sequence", fn);
  if (n_rows == 0 || n_seqs == 0) return WF_OK;
  WF_REQUIRE(q && out && (n_kv_rows == 0 || (k && v)), WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(aligned(k, 16) && aligned(v, 16), WF_E_ALIGN, "%s: k and v must be 16-byte aligned", fn);
  a.k_dense = static_cast<const uint16_t*>(k);
  a.v_dense = static_cast<const uint16_t*>(v);
  a.ldkv = ldkv;
  a.n_kv_rows = static_cast<int32_t>(n_kv_rows);
  a.cu_kv = cu_kv;
  a.geom = make_batch_geom(cu_q, cu_kv, n_seqs, nullptr, 0, 1, 0);
  return launch(fn, a, SRC_DENSE, n_seqs, max_q, max_kv, ws, ws_bytes, fresh, as_stream(stream));
}

}  // namespace
}  // namespace attn_batch
}  // namespace wf

extern "C" {

int wf_attn_batch_workspace(int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int64_t n_seqs, int64_t max_new,
                            int64_t max_kv, int64_t* bytes) {
  static const char* fn = "wf_attn_batch_workspace";
  WF_REQUIRE(bytes, WF_E_INVALID, "%s: null result", fn);
  WF_REQUIRE(n_rows >= 0 && n_heads > 0 && n_kv_heads > 0 && n_seqs >= 0 && max_new >= 0 && max_kv >= 0, WF_E_INVALID,
             "%s: negative or zero size", fn);
  WF_REQUIRE(n_heads % n_kv_heads == 0, WF_E_SHAPE, "%s: %d heads do not group over %d key heads", fn, n_heads, n_kv_heads);
  WF_REQUIRE(wf::product_below({n_rows, n_heads}, (1ll << 31) - 65536) && n_seqs < (1ll << 31) && max_kv < (1ll << 31), WF_E_SHAPE,
             "%s: rows=%lld x heads=%d, %lld sequences or %lld keys reach 2^31", fn, (long long)n_rows, n_heads, (long long)n_seqs, (long long)max_kv);
  *bytes = 0;
  bool fits = false;  // one of the two attentions takes them
  for (bool dense : {false, true}) {
    const auto p = wf::attn_batch::make_plan(dense, n_rows, n_heads, n_kv_heads, n_seqs, max_new, max_kv);
    fits = fits || p.fits;
    *bytes = std::max(*bytes, p.bytes);
  }
  WF_REQUIRE(n_rows == 0 || n_seqs == 0 || fits, WF_E_SHAPE, "%s: %lld rows of %lld sequences x %d heads are too many", fn,
             (long long)n_rows, (long long)n_seqs, n_heads);
  return WF_OK;
}

int wf_attn_paged_batch(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t ldq,
                        int32_t format, const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scales,
                        const float* v_scales, int64_t pool_pages, int32_t page_tokens, const int32_t* cu_new,
                        const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables, int64_t ld_table, int64_t max_new,
                        int64_t max_kv, int32_t block, float softmax_scale, void* out, int64_t ldo, void* ws,
                        int64_t ws_bytes, void* stream) {
  return wf::attn_batch::paged_batch("wf_attn_paged_batch", false, q, n_rows, n_heads, n_kv_heads, head_dim, ldq,
                                     format, k_codes, v_codes, k_scales, v_scales, pool_pages, page_tokens, cu_new,
                                     kv_lens, n_seqs, tables, ld_table, max_new, max_kv, block, softmax_scale, out, ldo,
                                     ws, ws_bytes, stream);
}

int wf_attn_paged_batch_fresh(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                              int64_t ldq, int32_t format, const uint8_t* k_codes, const uint8_t* v_codes,
                              const float* k_scales, const float* v_scales, int64_t pool_pages, int32_t page_tokens,
                              const int32_t* cu_new, const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables,
                              int64_t ld_table, int64_t max_new, int64_t max_kv, int32_t block, float softmax_scale,
                              void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return wf::attn_batch::paged_batch("wf_attn_paged_batch_fresh", true, q, n_rows, n_heads, n_kv_heads, head_dim, ldq,
                                     format, k_codes, v_codes, k_scales, v_scales, pool_pages, page_tokens, cu_new,
                                     kv_lens, n_seqs, tables, ld_table, max_new, max_kv, block, softmax_scale, out, ldo,
                                     ws, ws_bytes, stream);
}

int wf_attn_cross_batch(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t ldq,
                        const void* k, const void* v, int64_t n_kv_rows, int64_t ldkv, const int32_t* cu_q,
                        const int32_t* cu_kv, int64_t n_seqs, int64_t max_q, int64_t max_kv, float softmax_scale,
                        void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return wf::attn_batch::cross_batch("wf_attn_cross_batch", false, q, n_rows, n_heads, n_kv_heads, head_dim, ldq, k, v,
                                     n_kv_rows, ldkv, cu_q, cu_kv, n_seqs, max_q, max_kv, softmax_scale, out, ldo, ws,
                                     ws_bytes, stream);
}

int wf_attn_cross_batch_fresh(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                              int64_t ldq, const void* k, const void* v, int64_t n_kv_rows, int64_t ldkv,
                              const int32_t* cu_q, const int32_t* cu_kv, int64_t n_seqs, int64_t max_q, int64_t max_kv,
                              float softmax_scale, void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  return wf::attn_batch::cross_batch("wf_attn_cross_batch_fresh", true, q, n_rows, n_heads, n_kv_heads, head_dim, ldq,
                                     k, v, n_kv_rows, ldkv, cu_q, cu_kv, n_seqs, max_q, max_kv, softmax_scale, out, ldo,
                                     ws, ws_bytes, stream);
}

}  // extern "C"
