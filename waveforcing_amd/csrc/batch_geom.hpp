// Ragged rows of a batch of sequences over paged caches: which sequence a row belongs to, and where its position lives.
//
// Sequence b owns rows cu[b] .. cu[b+1] of the batch's tensors; kv_lens[b] keys are in its cache, the last
// cu[b+1] - cu[b] of them at the positions of its rows.  Position p lives in physical page
// tables[b][p / page_tokens], row p % page_tokens.  cu, kv_lens and tables are read on the device when the kernel runs
// (a captured graph replays with their present contents), so nothing here trusts them: every index is checked against
// what the host passed.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fastdiv.hpp"
#include "wf_common.hpp"

namespace wf {

struct BatchGeom {
  const int32_t* cu;       // [n_seqs + 1]
  const int32_t* kv_lens;  // [n_seqs]
  const int32_t* tables;   // [n_seqs][ld_table]
  int32_t n_seqs;
  int32_t ld_table;
  int32_t page_tokens;
  int32_t pool_pages;
  FastDiv page;
};

// Sequence of row t, one row per aligned group of 8 lanes: the number of b with cu[b + 1] <= t (n_seqs for rows
// behind the last sequence).  The wave reads 64 ends at a time; every lane has to take part.
__device__ inline int seq_of_group8(const BatchGeom& g, int t) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  int seq = 0;
  for (int base = 0; base < g.n_seqs; base += 64) {
    const int end = base + lane < g.n_seqs ? g.cu[base + lane + 1] : 0x7fffffff;
    bool more = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int ti = __builtin_amdgcn_readlane(t, 8 * i);
      const int n = __popcll(__ballot(end <= ti));
      if ((lane >> 3) == i) seq += n;
      more = more || n == 64;
    }
    if (!more) break;
  }
  return seq;
}

// A page id whose index all lanes hold, by a scalar load.  (Through the constant address space, whose loads the compiler keeps
// scalar whatever the kernel stores elsewhere; a vector load would be awaited behind the keys that are on their way:
// 64 tokens of 8192 keys 140 us instead of 134.)
__device__ inline int uniform_page(const int32_t* table, int64_t i) {
  typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
  return reinterpret_cast<constant_ptr>(reinterpret_cast<uintptr_t>(table))[i];
}

// Pool row (page * page_tokens + row in page) of position p of sequence b; false when it has none.
__device__ inline bool pool_row(const BatchGeom& g, int b, int p, int& page, int& row) {
  if (p < 0) return false;
  uint32_t lp, r;
  g.page.divmod(static_cast<uint32_t>(p), lp, r);
  if (lp >= static_cast<uint32_t>(g.ld_table)) return false;
  page = g.tables[static_cast<int64_t>(b) * g.ld_table + lp];
  row = static_cast<int>(r);
  return page >= 0 && page < g.pool_pages;
}

// Host checks of the geometry that every batch entry point shares.
inline int check_batch(const char* fn, int64_t n_rows, int32_t n_kv_heads, int32_t head_dim, const int32_t* cu,
                       const int32_t* kv_lens, int64_t n_seqs) {
  WF_REQUIRE(n_rows >= 0 && n_kv_heads > 0 && n_seqs >= 0, WF_E_INVALID,
             "%s: negative or zero size (rows=%lld kv_heads=%d seqs=%lld)", fn, (long long)n_rows, n_kv_heads,
             (long long)n_seqs);
  WF_REQUIRE(head_dim == 128, WF_E_SHAPE, "%s: head_dim=%d unsupported (must be 128)", fn, head_dim);
  // (an element's place in its row is counted in 32 bits)
  WF_REQUIRE(n_kv_heads < (1 << 16), WF_E_SHAPE, "%s: %d key heads, 2^16 or more", fn, n_kv_heads);
  WF_REQUIRE(n_seqs < (1ll << 20), WF_E_SHAPE, "%s: more than 2^20 sequences", fn);
  WF_REQUIRE(n_seqs == 0 || n_rows == 0 || (cu && kv_lens), WF_E_INVALID, "%s: null row starts or lengths", fn);
  return WF_OK;
}

inline int check_pool(const char* fn, int32_t format, int32_t n_kv_heads, int32_t page_tokens, int64_t pool_pages,
                      const int32_t* tables, int64_t ld_table) {
  WF_REQUIRE(format == WF_KV_E4M3 || format == WF_KV_INT8 || format == WF_KV_MXFP4, WF_E_INVALID, "%s: unknown cache format %d", fn, format);
  WF_REQUIRE(page_tokens > 0 && pool_pages >= 0 && ld_table >= 0, WF_E_INVALID,
             "%s: negative or zero size (page_tokens=%d pool_pages=%lld ld_table=%lld)", fn, page_tokens,
             (long long)pool_pages, (long long)ld_table);
  WF_REQUIRE(ld_table < (1ll << 31) && pool_pages < (1ll << 31), WF_E_SHAPE, "%s: pool or table too large", fn);
  WF_REQUIRE(product_below({pool_pages, page_tokens, n_kv_heads}, 1ll << 31), WF_E_SHAPE,
             "%s: a pool of 2^31 (token, head) rows or more", fn);
  WF_REQUIRE(ld_table == 0 || tables, WF_E_INVALID, "%s: null page tables", fn);
  return WF_OK;
}

inline BatchGeom make_batch_geom(const int32_t* cu, const int32_t* kv_lens, int64_t n_seqs, const int32_t* tables,
                                 int64_t ld_table, int32_t page_tokens, int64_t pool_pages) {
  return BatchGeom{cu, kv_lens, tables, static_cast<int32_t>(n_seqs), static_cast<int32_t>(ld_table), page_tokens,
                   static_cast<int32_t>(pool_pages), FastDiv(static_cast<uint32_t>(page_tokens))};
}

}  // namespace wf
