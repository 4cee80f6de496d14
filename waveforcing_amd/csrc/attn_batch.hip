// Attention of a batch of sequences: ragged query rows over each sequence's paged quantized keys (e4m3 or int8), or
// over ragged dense bf16 keys.
//
//   out[i, h] = sum_j w_j V[j, g] / sum_j w_j,   w_j = exp(scale <Q[i, h], K[j, g]>),   g = h / (n_heads / n_kv_heads)
//   over the keys j < lim(i) of the row's sequence; K = code_k s_k and V = code_v s_v are products of fp32 numbers.
//   lim = kv_len without a block; min(kv_len, (p / block + 1) block) with one, p = kv_len - new + i the row's position.
//   A row without keys is zero.
//
// One wave per (row, head): 64 keys at a time, one key per lane for the scores, two of the 128 values per lane for the
// sum over V, running maximum and sum in fp32.
#include "batch_geom.hpp"
#include "fp8_codec.hpp"
#include "wf_common.hpp"

namespace wf {
namespace {

constexpr int D = 128;
constexpr float kLog2e = 1.4426950408889634f;
enum { SRC_E4M3 = WF_KV_E4M3, SRC_INT8 = WF_KV_INT8, SRC_DENSE = 2 };

struct AttnBatchArgs {
  const uint16_t* q;
  uint16_t* out;
  int64_t ldq, ldo;
  const uint8_t *k_codes, *v_codes;
  const float *k_scales, *v_scales;
  const uint16_t *k_dense, *v_dense;
  const int32_t* cu_kv;
  int64_t ldkv, n_kv_rows;
  int32_t n_rows, n_heads, n_kv_heads, group;
  int32_t block;
  float c;  // softmax scale * log2(e)
  BatchGeom geom;
};

// Where a key's row of head g begins: codes (or dense elements) and scale; false: an invalid page, read as zero.
template <int SRC>
__device__ inline bool key_row(const AttnBatchArgs& a, int b, int j, int g, int64_t& code, int64_t& scale) {
  if constexpr (SRC == SRC_DENSE) {
    code = static_cast<int64_t>(a.cu_kv[b] + j) * a.ldkv + g * D;
    scale = 0;
    return true;
  } else {
    int page, at;
    if (!pool_row(a.geom, b, j, page, at)) return false;
    code = ((static_cast<int64_t>(page) * a.geom.page_tokens + at) * a.n_kv_heads + g) * D;
    scale = (static_cast<int64_t>(page) * a.n_kv_heads + g) * a.geom.page_tokens + at;
    return true;
  }
}

template <int SRC>
__device__ inline float value(const uint8_t* codes, const uint16_t* dense, int64_t i) {
  if constexpr (SRC == SRC_DENSE) return bf16_bits_to_f32(dense[i]);
  if constexpr (SRC == SRC_INT8) return static_cast<float>(static_cast<int8_t>(codes[i]));
  return e4m3_decode_sw(codes[i]);
}

template <int SRC>
__global__ __launch_bounds__(64) void attn_batch_simple_kernel(AttnBatchArgs a) {
  __shared__ float qs[D], ps[64];
  __shared__ int64_t vs[64];
  const int t = static_cast<int>(blockIdx.x) / a.n_heads, h = static_cast<int>(blockIdx.x) % a.n_heads;
  const int lane = threadIdx.x, g = h / a.group;
  const int b = __builtin_amdgcn_readfirstlane(seq_of_group8(a.geom, t));
  if (b >= a.geom.n_seqs) return;
  const int kv_len = SRC == SRC_DENSE ? max(0, a.cu_kv[b + 1] - a.cu_kv[b]) : a.geom.kv_lens[b];
  int lim = kv_len;
  if (a.block > 0) {
    const int p = kv_len - a.geom.cu[b + 1] + t;
    lim = p < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(kv_len), (static_cast<int64_t>(p) / a.block + 1) * a.block));
  }
  const uint16_t* qp = a.q + static_cast<int64_t>(t) * a.ldq + h * D;
  qs[lane] = bf16_bits_to_f32(qp[lane]);
  qs[lane + 64] = bf16_bits_to_f32(qp[lane + 64]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int j0 = 0; j0 < lim; j0 += 64) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int64_t code = 0, scale = 0;
    bool there = false;
    if (j < lim) {
      there = key_row<SRC>(a, b, j, g, code, scale);
      float dot = 0.f;
      if (there) {
        for (int d = 0; d < D; ++d) dot = fmaf(qs[d], value<SRC>(a.k_codes, a.k_dense, code + d), dot);
        if (SRC != SRC_DENSE) dot *= a.k_scales[scale];
      }
      s = dot * a.c;
    }
    float top = s;
    for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    const float m_new = fmaxf(m, top);
    const float alpha = m_new == -INFINITY ? 1.f : exp2f(m - m_new);
    const float p = j < lim ? exp2f(m_new == -INFINITY ? s : s - m_new) : 0.f;
    float sum = p;
    for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
    l = l * alpha + sum;
    o0 *= alpha;
    o1 *= alpha;
    m = m_new;
    ps[lane] = there && SRC != SRC_DENSE ? p * a.v_scales[scale] : p;
    vs[lane] = there ? code : -1;
    __syncthreads();
    const int n = min(64, lim - j0);
    for (int i = 0; i < n; ++i) {
      const int64_t at = vs[i];
      if (at < 0) continue;
      o0 = fmaf(ps[i], value<SRC>(a.v_codes, a.v_dense, at + 2 * lane), o0);
      o1 = fmaf(ps[i], value<SRC>(a.v_codes, a.v_dense, at + 2 * lane + 1), o1);
    }
    __syncthreads();
  }
  const float inv = lim > 0 ? 1.0f / l : 0.f;
  reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(t) * a.ldo + h * D)[lane] = pack_bf16x2(o0 * inv, o1 * inv);
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks that both attentions share; fills the common arguments.
int common_args(const char* fn, AttnBatchArgs& a, const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads,
                int64_t ldq, float softmax_scale, void* out, int64_t ldo) {
  WF_REQUIRE(n_heads > 0 && n_heads % n_kv_heads == 0, WF_E_SHAPE, "%s: %d heads do not group over %d key heads", fn,
             n_heads, n_kv_heads);
  WF_REQUIRE(softmax_scale >= 0.f && softmax_scale < 3.0e38f, WF_E_INVALID,
             "%s: softmax_scale=%g must be finite and non-negative", fn, static_cast<double>(softmax_scale));
  const int64_t hd = static_cast<int64_t>(n_heads) * D;
  WF_REQUIRE(ldq >= hd && ldo >= hd, WF_E_INVALID, "%s: ldq/ldo smaller than n_heads*head_dim", fn);
  WF_REQUIRE(product_below({n_rows, n_heads}, (1ll << 31) - 65536), WF_E_SHAPE, "%s: rows=%lld x heads=%d reaches 2^31", fn,
             (long long)n_rows, n_heads);
  WF_REQUIRE(aligned(q, 16) && ldq % 8 == 0 && aligned(out, 8) && ldo % 4 == 0, WF_E_ALIGN,
             "%s: q must be 16-byte aligned (ldq %% 8 == 0), out 8-byte aligned (ldo %% 4 == 0)", fn);
  a = AttnBatchArgs{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.ldq = ldq;
  a.ldo = ldo;
  a.n_rows = static_cast<int32_t>(n_rows);
  a.n_heads = n_heads;
  a.n_kv_heads = n_kv_heads;
  a.group = n_heads / n_kv_heads;
  a.c = softmax_scale * kLog2e;
  return WF_OK;
}

template <int SRC>
int launch(const char* fn, const AttnBatchArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(attn_batch_simple_kernel<SRC>, dim3(static_cast<uint32_t>(a.n_rows) * a.n_heads), dim3(64), 0, stream,
                     a);
  return check_launch(fn);
}

}  // namespace
}  // namespace wf

extern "C" {

int wf_attn_batch_workspace(int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int64_t n_seqs, int64_t max_new,
                            int64_t max_kv, int32_t paged, int64_t* bytes) {
  static const char* fn = "wf_attn_batch_workspace";
  WF_REQUIRE(bytes, WF_E_INVALID, "%s: null result", fn);
  WF_REQUIRE(n_rows >= 0 && n_heads > 0 && n_kv_heads > 0 && n_seqs >= 0 && max_new >= 0 && max_kv >= 0, WF_E_INVALID,
             "%s: negative or zero size", fn);
  *bytes = 0;
  return WF_OK;
}

int wf_attn_paged_batch(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t ldq,
                        int32_t format, const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scales,
                        const float* v_scales, int64_t pool_pages, int32_t page_tokens, const int32_t* cu_new,
                        const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables, int64_t ld_table, int64_t max_new,
                        int64_t max_kv, int32_t block, float softmax_scale, void* out, int64_t ldo, void* ws,
                        int64_t ws_bytes, void* stream) {
  static const char* fn = "wf_attn_paged_batch";
  if (int st = wf::check_batch(fn, n_rows, n_kv_heads, head_dim, cu_new, kv_lens, n_seqs)) return st;
  if (int st = wf::check_pool(fn, format, n_kv_heads, page_tokens, pool_pages, tables, ld_table)) return st;
  WF_REQUIRE(block >= 0, WF_E_INVALID, "%s: block=%d must not be negative", fn, block);
  WF_REQUIRE(max_new >= 0 && max_kv >= 0, WF_E_INVALID, "%s: negative bound of the lengths", fn);
  wf::AttnBatchArgs a;
  if (int st = wf::common_args(fn, a, q, n_rows, n_heads, n_kv_heads, ldq, softmax_scale, out, ldo)) return st;
  if (n_rows == 0 || n_seqs == 0) return WF_OK;
  WF_REQUIRE(q && out && k_codes && v_codes && k_scales && v_scales, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(wf::aligned(k_codes, 16) && wf::aligned(v_codes, 16), WF_E_ALIGN, "%s: code pools must be 16-byte aligned", fn);
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_scales = k_scales;
  a.v_scales = v_scales;
  a.block = block;
  a.geom = wf::make_batch_geom(cu_new, kv_lens, n_seqs, tables, ld_table, page_tokens, pool_pages);
  return format == WF_KV_INT8 ? wf::launch<wf::SRC_INT8>(fn, a, wf::as_stream(stream))
                              : wf::launch<wf::SRC_E4M3>(fn, a, wf::as_stream(stream));
}

int wf_attn_cross_batch(const void* q, int64_t n_rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int64_t ldq,
                        const void* k, const void* v, int64_t n_kv_rows, int64_t ldkv, const int32_t* cu_q,
                        const int32_t* cu_kv, int64_t n_seqs, int64_t max_q, int64_t max_kv, float softmax_scale,
                        void* out, int64_t ldo, void* ws, int64_t ws_bytes, void* stream) {
  static const char* fn = "wf_attn_cross_batch";
  if (int st = wf::check_batch(fn, n_rows, n_kv_heads, head_dim, cu_q, cu_kv, n_seqs)) return st;
  WF_REQUIRE(max_q >= 0 && max_kv >= 0, WF_E_INVALID, "%s: negative bound of the lengths", fn);
  WF_REQUIRE(n_kv_rows >= 0 && n_kv_rows < (1ll << 31), WF_E_SHAPE, "%s: %lld key rows", fn, (long long)n_kv_rows);
  WF_REQUIRE(ldkv >= static_cast<int64_t>(n_kv_heads) * head_dim && ldkv % 8 == 0, WF_E_INVALID,
             "%s: ldkv=%lld must be >= n_kv_heads*head_dim and a multiple of 8", fn, (long long)ldkv);
  wf::AttnBatchArgs a;
  if (int st = wf::common_args(fn, a, q, n_rows, n_heads, n_kv_heads, ldq, softmax_scale, out, ldo)) return st;
  if (n_rows == 0 || n_seqs == 0) return WF_OK;
  WF_REQUIRE(q && out && (n_kv_rows == 0 || (k && v)), WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(wf::aligned(k, 16) && wf::aligned(v, 16), WF_E_ALIGN, "%s: k and v must be 16-byte aligned", fn);
  a.k_dense = static_cast<const uint16_t*>(k);
  a.v_dense = static_cast<const uint16_t*>(v);
  a.ldkv = ldkv;
  a.n_kv_rows = n_kv_rows;
  a.cu_kv = cu_kv;
  a.geom = wf::make_batch_geom(cu_q, cu_kv, n_seqs, nullptr, 0, 1, 0);
  return wf::launch<wf::SRC_DENSE>(fn, a, wf::as_stream(stream));
}

}  // extern "C"
