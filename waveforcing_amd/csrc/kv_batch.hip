// The paged KV cache of a batch of sequences: new rows quantized into their pages (append) and read back (gather).
// Both stream through HBM: a (row, head) of 128 bf16 values (256 B) against 128 codes and one fp32 scale (132 B).
//
// Work split as in kv_pages.hip: 8 lanes own a (row, head), 16 values each, so a code row is 8 16-byte stores and the
// maximum of |x| is an 8-lane reduction; a workgroup owns 32 consecutive (row, head) of K or of V, and each XCD gets a
// contiguous range of them.  A row's sequence is found by the wave itself (batch_geom.hpp): the rows are ragged and
// the lengths live on the device.
//
// Per (row, head), a = max|x|:
//   e4m3: the arithmetic of kv_pages.hip;
//   int8: s = max(a / 127, 1e-8), code = clamp(rint(x / s), -127, 127), fp32 (rows.hpp's quant_i8).
// The magnitudes of bf16 numbers order as their bits do, and those of infinities and NaN come last, so the integer
// maximum that gives a also tells a row that holds one: it is stored as scale NaN and zero codes, and reads back as NaN
// whole in every format, instead of as a finite row of a scale that its other values set.
//
//   MXFP4: mxfp4_codec.hpp's, a block of 32 values in two lanes (one DPP step), a lane's 16 codes 8 bytes; the four blocks'
//   scale bytes meet in two more steps and take the place of the fp32 scale.  A head's rows of 64 bytes follow one another in
//   a page, two to a cache line (as the other formats have them, position by position, the attention, which reads one head's,
//   took half of every line).
//
// Four chunks of 4680 rows of 12 heads: append 40-41 us (4.3 TB/s of 174 MB), gather 30 us (5.8), MXFP4 33 and 29 (4.4 and 5.1
// TB/s of 146 MB); 64 single rows 4 us each, the launch.
#include "batch_geom.hpp"
#include "kv_row.hpp"
#include "mxfp4_codec.hpp"
#include "rows.hpp"

namespace wf {
namespace {

constexpr int kRowsPerBlock = 32;
constexpr uint32_t kXcds = 8;

struct KvBatchArgs {
  const uint16_t* src[2];  // K, V rows bf16 [n_rows][ld] (append)
  uint16_t* dst[2];        // K, V rows bf16 [n_rows][ld] (gather)
  uint8_t* codes[2];
  float* scales[2];
  int64_t ld;
  int32_t n_heads;
  int32_t n_rows;
  uint32_t n_blocks;  // of K
  uint32_t n_items;   // of K and V
  int32_t fresh;      // gather: rows without a position are zeroed
  FastDiv heads;
  BatchGeom geom;
};

// The (row, head) of this lane's group and where it lives in the pool; false: nowhere.  All lanes take part.
template <bool MX>
__device__ inline bool place(const KvBatchArgs& a, uint32_t blk, int& row, int& head, int64_t& code_row, int64_t& scale) {
  uint32_t t, h;
  a.heads.divmod(blk * kRowsPerBlock + (threadIdx.x >> 3), t, h);
  row = static_cast<int>(t);
  head = static_cast<int>(h);
  const int b = seq_of_group8(a.geom, row);
  if (row >= a.n_rows || b >= a.geom.n_seqs || row < a.geom.cu[0]) return false;  // (rows before the first start are nobody's)
  int page, at;
  if (!pool_row(a.geom, b, a.geom.kv_lens[b] - a.geom.cu[b + 1] + row, page, at)) return false;
  code_row = (static_cast<int64_t>(page) * a.geom.page_tokens + at) * a.n_heads + head;
  scale = (static_cast<int64_t>(page) * a.n_heads + head) * a.geom.page_tokens + at;
  if constexpr (MX) code_row = scale;
  return true;
}

__device__ inline bool item(const KvBatchArgs& a, uint32_t& blk, int& which) {
  const uint32_t per_xcd = (a.n_items + kXcds - 1) / kXcds;
  const uint32_t w = (blockIdx.x % kXcds) * per_xcd + blockIdx.x / kXcds;
  if (w >= a.n_items) return false;
  which = w >= a.n_blocks;
  blk = w - (which ? a.n_blocks : 0u);
  return true;
}

// Maximum over aligned groups of 8 lanes of an integer (wf_common.hpp's group8_max).
__device__ inline uint32_t group8_umax(uint32_t v) {
  int o = __builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), 0xB1, 0xF, 0xF, false);
  v = max(v, static_cast<uint32_t>(o));
  o = __builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), 0x4E, 0xF, 0xF, false);
  v = max(v, static_cast<uint32_t>(o));
  o = __builtin_amdgcn_update_dpp(static_cast<int>(v), static_cast<int>(v), 0x141, 0xF, 0xF, false);
  return max(v, static_cast<uint32_t>(o));
}

// OR of v over pairs of lanes of an aligned group of 8 (each pair holding one value).
__device__ inline uint32_t group8_or_pairs(uint32_t v) {
  v |= static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4E, 0xF, 0xF, false));
  return v | static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x141, 0xF, 0xF, false));
}

template <int FMT>
__global__ __launch_bounds__(256) void kv_append_kernel(KvBatchArgs a) {
  uint32_t blk;
  int which;
  if (!item(a, blk, which)) return;
  int row, head;
  int64_t code_row = 0, scale_at = 0;
  const bool ok = place<FMT == WF_KV_MXFP4>(a, blk, row, head, code_row, scale_at);
  const uint32_t lane8 = threadIdx.x & 7u;
  uint4 x = make_uint4(0, 0, 0, 0), y = x;
  if (ok) {
    const uint4* p = reinterpret_cast<const uint4*>(a.src[which] + static_cast<int64_t>(row) * a.ld + head * kHeadDim);
    x = p[lane8 * 2];
    y = p[lane8 * 2 + 1];
  }
  const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  if constexpr (FMT == WF_KV_MXFP4) {
    const uint32_t block = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xF, 0xF, false)));
    const bool nan = group8_umax(top) >= 0x7f80u;
    const int e = mx::scale_byte(block);
    const float s = mx::scale_of(e);
    const uint32_t bytes = nan ? ~0u : group8_or_pairs(static_cast<uint32_t>(e) << (8 * (lane8 >> 1)));
    if (!ok) return;
    const uint2 c = nan ? make_uint2(0, 0) : make_uint2(mx::encode8(w, s), mx::encode8(w + 4, s));
    reinterpret_cast<uint2*>(a.codes[which] + code_row * (kHeadDim / 2))[lane8] = c;
    if (lane8 == 0) reinterpret_cast<uint32_t*>(a.scales[which])[scale_at] = bytes;
    return;
  }
  top = group8_umax(top);
  if (!ok) return;
  const float amax = bf16_bits_to_f32(static_cast<uint16_t>(top));
  float s;
  uint4 c;
  if constexpr (FMT == WF_KV_INT8) {
    s = rows::i8_scale(amax);
    const double r = 1.0 / static_cast<double>(s);
    float v[16];
    rows::unpack8(x, v);
    rows::unpack8(y, v + 8);
    const uint2 lo = rows::quant8_i8(v, r), hi = rows::quant8_i8(v + 8, r);
    c = make_uint4(lo.x, lo.y, hi.x, hi.y);
  } else {
    s = scale_from_amax(amax);
    const float r = __builtin_amdgcn_rcpf(s);
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {bf16_lo_to_f32(w[2 * i]), bf16_hi_to_f32(w[2 * i]), bf16_lo_to_f32(w[2 * i + 1]),
                          bf16_hi_to_f32(w[2 * i + 1])};
      q[i] = quant4f(v, s, r);
    }
    c = make_uint4(q[0], q[1], q[2], q[3]);
  }
  if (top >= 0x7f80u) {
    s = bits_f32(0x7fc00000u);
    c = make_uint4(0, 0, 0, 0);
  }
  reinterpret_cast<uint4*>(a.codes[which] + code_row * kHeadDim)[lane8] = c;
  if (lane8 == 0) a.scales[which][scale_at] = s;
}

// bf16(float(code) * s) of four int8 codes.
__device__ inline uint2 dequant4_i8(uint32_t w, float s) {
  const float v0 = static_cast<float>(static_cast<int8_t>(w)), v1 = static_cast<float>(static_cast<int8_t>(w >> 8));
  const float v2 = static_cast<float>(static_cast<int8_t>(w >> 16)), v3 = static_cast<float>(static_cast<int8_t>(w >> 24));
  return make_uint2(pack_bf16x2_hw(v0 * s, v1 * s), pack_bf16x2_hw(v2 * s, v3 * s));
}

template <int FMT>
__global__ __launch_bounds__(256) void kv_gather_kernel(KvBatchArgs a) {
  uint32_t blk;
  int which;
  if (!item(a, blk, which)) return;
  int row, head;
  int64_t code_row = 0, scale_at = 0;
  const bool ok = place<FMT == WF_KV_MXFP4>(a, blk, row, head, code_row, scale_at);
  if (!ok && (!a.fresh || row >= a.n_rows)) return;
  const uint32_t lane8 = threadIdx.x & 7u;
  uint4* p = reinterpret_cast<uint4*>(a.dst[which] + static_cast<int64_t>(row) * a.ld + head * kHeadDim) + lane8 * 2;
  if (!ok) {
    p[0] = p[1] = make_uint4(0, 0, 0, 0);
    return;
  }
  if constexpr (FMT == WF_KV_MXFP4) {
    const uint2 c = reinterpret_cast<const uint2*>(a.codes[which] + code_row * (kHeadDim / 2))[lane8];
    const uint32_t bytes = reinterpret_cast<const uint32_t*>(a.scales[which])[scale_at];
    const float s = mx::scale_of((bytes >> (8 * (lane8 >> 1))) & 0xffu);
    p[0] = mx::decode8(c.x, s);
    p[1] = mx::decode8(c.y, s);
    return;
  }
  const uint4 c = reinterpret_cast<const uint4*>(a.codes[which] + code_row * kHeadDim)[lane8];
  const float s = a.scales[which][scale_at];
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint2 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = FMT == WF_KV_INT8 ? dequant4_i8(w[i], s) : dequant4(w[i], s);
  p[0] = make_uint4(o[0].x, o[0].y, o[1].x, o[1].y);
  p[1] = make_uint4(o[2].x, o[2].y, o[3].x, o[3].y);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Checks and launch of both directions; k, v: the dense rows (const-cast for append, which only reads them).
int kv_batch(const char* fn, bool write, bool fresh, void* k, void* v, int64_t n_rows, int32_t n_heads, int32_t head_dim, int64_t ld,
             int32_t format, const int32_t* cu, const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables,
             int64_t ld_table, int32_t page_tokens, uint8_t* k_codes, uint8_t* v_codes, float* k_scales,
             float* v_scales, int64_t pool_pages, void* stream) {
  if (int st = check_batch(fn, n_rows, n_heads, head_dim, cu, kv_lens, n_seqs)) return st;
  if (int st = check_pool(fn, format, n_heads, page_tokens, pool_pages, tables, ld_table)) return st;
  WF_REQUIRE(product_below({n_rows, n_heads}, (1ll << 31) - kRowsPerBlock), WF_E_SHAPE, "%s: rows=%lld x heads=%d reaches 2^31",
             fn, (long long)n_rows, n_heads);
  WF_REQUIRE(!fresh || n_rows == 0 || n_seqs > 0, WF_E_INVALID, "%s: rows without a sequence", fn);
  if (n_rows == 0 || n_seqs == 0) return WF_OK;
  WF_REQUIRE(k && k_codes && k_scales, WF_E_INVALID, "%s: null K pointer", fn);
  WF_REQUIRE(!v || (v_codes && v_scales), WF_E_INVALID, "%s: V given without V pool", fn);
  WF_REQUIRE(ld >= static_cast<int64_t>(n_heads) * head_dim && ld % 8 == 0, WF_E_INVALID,
             "%s: row stride %lld must be >= n_heads*head_dim and a multiple of 8", fn, (long long)ld);
  WF_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_codes) && (!v || aligned16(v_codes)), WF_E_ALIGN,
             "%s: K/V rows and code pools must be 16-byte aligned", fn);
  KvBatchArgs a;
  a.src[0] = static_cast<const uint16_t*>(k);
  a.src[1] = static_cast<const uint16_t*>(v);
  a.dst[0] = static_cast<uint16_t*>(k);
  a.dst[1] = static_cast<uint16_t*>(v);
  a.codes[0] = k_codes;
  a.codes[1] = v_codes;
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.ld = ld;
  a.n_heads = n_heads;
  a.n_rows = static_cast<int32_t>(n_rows);
  a.n_blocks = static_cast<uint32_t>((n_rows * n_heads + kRowsPerBlock - 1) / kRowsPerBlock);
  a.n_items = v ? 2 * a.n_blocks : a.n_blocks;
  a.fresh = fresh;
  a.heads = FastDiv(static_cast<uint32_t>(n_heads));
  a.geom = make_batch_geom(cu, kv_lens, n_seqs, tables, ld_table, page_tokens, pool_pages);
  const dim3 grid((a.n_items + kXcds - 1) / kXcds * kXcds);
  void (*kernel)(KvBatchArgs);
  if (format == WF_KV_MXFP4)
    kernel = write ? kv_append_kernel<WF_KV_MXFP4> : kv_gather_kernel<WF_KV_MXFP4>;
  else if (format == WF_KV_INT8)
    kernel = write ? kv_append_kernel<WF_KV_INT8> : kv_gather_kernel<WF_KV_INT8>;
  else
    kernel = write ? kv_append_kernel<WF_KV_E4M3> : kv_gather_kernel<WF_KV_E4M3>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, as_stream(stream), a);
  return check_launch(fn);
}

}  // namespace
}  // namespace wf

extern "C" {

int wf_kv_batch_append(const void* k, const void* v, int64_t n_rows, int32_t n_kv_heads, int32_t head_dim, int64_t ld_kv,
                       int32_t format, const int32_t* cu_new, const int32_t* kv_lens, int64_t n_seqs,
                       const int32_t* tables, int64_t ld_table, int32_t page_tokens, uint8_t* k_codes,
                       uint8_t* v_codes, float* k_scales, float* v_scales, int64_t pool_pages, void* stream) {
  return wf::kv_batch("wf_kv_batch_append", true, false, const_cast<void*>(k), const_cast<void*>(v), n_rows, n_kv_heads,
                      head_dim, ld_kv, format, cu_new, kv_lens, n_seqs, tables, ld_table, page_tokens, k_codes, v_codes,
                      k_scales, v_scales, pool_pages, stream);
}

int wf_kv_batch_gather(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scales, const float* v_scales,
                       int64_t pool_pages, int32_t format, int32_t page_tokens, const int32_t* cu_new,
                       const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables, int64_t ld_table, int64_t n_rows,
                       int32_t n_kv_heads, int32_t head_dim, void* k_out, void* v_out, int64_t ld_out, void* stream) {
  return wf::kv_batch("wf_kv_batch_gather", false, false, k_out, v_out, n_rows, n_kv_heads, head_dim, ld_out, format, cu_new,
                      kv_lens, n_seqs, tables, ld_table, page_tokens, const_cast<uint8_t*>(k_codes),
                      const_cast<uint8_t*>(v_codes), const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                      pool_pages, stream);
}

int wf_kv_batch_gather_fresh(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scales,
                             const float* v_scales, int64_t pool_pages, int32_t format, int32_t page_tokens,
                             const int32_t* cu_new, const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables,
                             int64_t ld_table, int64_t n_rows, int32_t n_kv_heads, int32_t head_dim,
                             void* k_out, void* v_out, int64_t ld_out, void* stream) {
  return wf::kv_batch("wf_kv_batch_gather_fresh", false, true, k_out, v_out, n_rows, n_kv_heads, head_dim, ld_out, format, cu_new,
                      kv_lens, n_seqs, tables, ld_table, page_tokens, const_cast<uint8_t*>(k_codes),
                      const_cast<uint8_t*>(v_codes), const_cast<float*>(k_scales), const_cast<float*>(v_scales),
                      pool_pages, stream);
}

}  // extern "C"
