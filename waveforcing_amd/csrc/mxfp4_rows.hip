// Rows of bf16 into MXFP4 codes and scales (weights once, activations at every call), and back.  Both stream through HBM:
// 2 bytes a value on one side, 17/32 on the other.
//
// Layout: panels of 16 rows x 128 values, P = ceil(rows / 16) by G = ceil(k / 128) of them.
//   codes  [P][G][4][16][16]: the 16 bytes of (p, g, b, r) are the values 128 g + 32 b .. + 31 of row 16 p + r
//   scales [P][G][16][4]: byte b of (p, g, r) belongs to those
// zero where the rows or their values end.  A panel is what a wave's 16x16x128 matrix instruction takes, 16 bytes a lane in
// the lanes' order, and half of what a 32x32x64 one takes twice: 1 KB in a row, read by one load or DMA of 8 whole cache
// lines.  (Codes row by row cost the few-rows product half its rate: 16 rows' 64 bytes from 16 lines; 64 x 13824 -> 5120 44 us
// for 22, 1 x 5120 -> 13824 12 for 9.6.)
//
// A wave takes 4 rows x 512 values: one 16-byte load a lane and row, a block in 4 lanes, whose maximum is two DPP steps; a
// lane's 8 codes are one word, and the 4 rows' scale words leave as 16 bytes of one lane in 16.  The waves of a workgroup
// fill a panel's lines together.  4680 x 13824 quantized in 36 us (4.5 TB/s), read back in 32 (5.1).
#include "launchers.hpp"
#include "mxfp4_codec.hpp"

namespace wf {
namespace {

constexpr int kRows = 4;        // of a wave
constexpr int kChunk = 512;     // values of a row that a wave takes
constexpr int kWaves = 4;

// The wave's rows and the lane's values.  Neighbouring workgroups take the chunks of the same rows, one after the other: the same
// chunk of all rows first meets few memory channels where the rows' stride is a power of two (16384 x 16384: 3.5 TB/s for 5.1
// quantized, 4.7 for 5.7 read back; 4680 x 13824: 4.2 for 4.6, 4.8 for 5.1).
struct Item {
  int row0, chunk, at;
};
__device__ inline Item item(int k) {
  const int chunks = (k + kChunk - 1) / kChunk, chunk = static_cast<int>(blockIdx.x) % chunks;
  const int panel = static_cast<int>(blockIdx.x) / chunks;
  const int wave = static_cast<int>(threadIdx.x) >> 6, lane = static_cast<int>(threadIdx.x) & 63;
  return Item{(panel * kWaves + wave) * kRows, chunk, chunk * kChunk + 8 * lane};
}

// Where the lane's word of codes of row0 goes (its other rows follow at 16 bytes), and the scale words of 4 rows.
struct Place {
  int64_t codes, scales;
  bool there;  // the lane's group of 128 values exists
};
__device__ inline Place place(int row0, int chunk, int k) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int groups = (k + 127) / 128, g = chunk * (kChunk / 128) + (lane >> 4);
  const int64_t panel = static_cast<int64_t>(row0 >> 4) * groups + g;
  return Place{panel * 1024 + ((lane >> 2) & 3) * 256 + (row0 & 15) * 16 + 4 * (lane & 3), panel * 64 + (row0 & 15) * 4, g < groups};
}

__global__ __launch_bounds__(64 * kWaves) void mxfp4_quant_kernel(const uint16_t* x, int rows, int k, int64_t ldx, uint8_t* codes,
                                                                  uint8_t* scales) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const auto [row0, chunk, at] = item(k);  // (k % 32 == 0: a block is there or not, whole)
  uint4 v[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    v[r] = make_uint4(0, 0, 0, 0);
    if (row0 + r < rows && at < k) v[r] = *reinterpret_cast<const uint4*>(x + (row0 + r) * ldx + at);
  }
  const Place to = place(row0, chunk, k);
  uint32_t word[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const uint32_t w[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
    uint32_t top = mx::max_half(mx::max_bits2(mx::max_bits2(w[0], w[1]), mx::max_bits2(w[2], w[3])));
    top = max(top, mx::dpp_u32<0xB1>(top));  // quad_perm [1,0,3,2], [2,3,0,1]
    top = max(top, mx::dpp_u32<0x4E>(top));
    const int e = mx::scale_byte(top);
    uint32_t c = mx::encode8(w, mx::scale_of(e));
    if (e == mx::kNanE) c = 0;
    if (to.there) *reinterpret_cast<uint32_t*>(codes + to.codes + 16 * r) = c;
    // the four blocks' bytes of 16 lanes as one word
    uint32_t s = row0 + r < rows && at < k ? static_cast<uint32_t>(e) << (8 * ((lane >> 2) & 3)) : 0u;
    s |= mx::dpp_u32<0x124>(s);  // row_ror:4, 8
    s |= mx::dpp_u32<0x128>(s);
    word[r] = s;
  }
  if ((lane & 15) == 0 && to.there) *reinterpret_cast<uint4*>(scales + to.scales) = make_uint4(word[0], word[1], word[2], word[3]);
}

__global__ __launch_bounds__(64 * kWaves) void mxfp4_dequant_kernel(const uint8_t* codes, const uint8_t* scales, int rows, int k,
                                                                    uint16_t* out, int64_t ldo) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const auto [row0, chunk, at] = item(k);
  if (row0 >= rows || at >= k) return;
  const Place from = place(row0, chunk, k);
  const uint4 s = *reinterpret_cast<const uint4*>(scales + from.scales);
  const uint32_t word[kRows] = {s.x, s.y, s.z, s.w};
  uint32_t c[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) c[r] = *reinterpret_cast<const uint32_t*>(codes + from.codes + 16 * r);
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (row0 + r < rows)
      *reinterpret_cast<uint4*>(out + (row0 + r) * ldo + at) = mx::decode8(c[r], mx::scale_of((word[r] >> (8 * ((lane >> 2) & 3))) & 0xffu));
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks that both directions share.
int check_rows(const char* fn, const void* dense, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, int64_t ld) {
  WF_REQUIRE(rows >= 0 && k >= 0 && ld >= k, WF_E_INVALID, "%s: bad sizes rows=%lld k=%lld row stride=%lld", fn, (long long)rows,
             (long long)k, (long long)ld);
  WF_REQUIRE(k % mx::kBlock == 0, WF_E_SHAPE, "%s: k=%lld must be a multiple of 32", fn, (long long)k);
  // (a grid holds fewer than 2^32 threads, 256 for 16 rows x 512 values)
  WF_REQUIRE(rows < (1ll << 28) && k < (1ll << 28) && product_below({(rows + 15) / 16, (k + kChunk - 1) / kChunk, 256}, 1ll << 32),
             WF_E_SHAPE, "%s: rows=%lld or k=%lld too large", fn, (long long)rows, (long long)k);
  if (rows == 0 || k == 0) return WF_OK;
  WF_REQUIRE(dense && codes && scales, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(aligned(dense, 16) && ld % 8 == 0 && aligned(codes, 16) && aligned(scales, 16), WF_E_ALIGN,
             "%s: rows, codes and scales must be 16-byte aligned, the row stride a multiple of 8", fn);
  return WF_OK;
}

dim3 rows_grid(int64_t rows, int64_t k) {
  return dim3(static_cast<uint32_t>((rows + kRows * kWaves - 1) / (kRows * kWaves) * ((k + kChunk - 1) / kChunk)));
}

}  // namespace

int launch_mxfp4_quant(const void* x, int64_t rows, int64_t k, int64_t ldx, uint8_t* codes, uint8_t* scales, hipStream_t stream) {
  hipLaunchKernelGGL(mxfp4_quant_kernel, rows_grid(rows, k), dim3(64 * kWaves), 0, stream, static_cast<const uint16_t*>(x),
                     static_cast<int>(rows), static_cast<int>(k), ldx, codes, scales);
  return check_launch("wf_mxfp4_quant");
}

}  // namespace wf

extern "C" {

int wf_mxfp4_quant(const void* x, int64_t rows, int64_t k, int64_t ldx, uint8_t* codes, uint8_t* scales, void* stream) {
  if (int st = wf::check_rows("wf_mxfp4_quant", x, codes, scales, rows, k, ldx)) return st;
  if (rows == 0 || k == 0) return WF_OK;
  return wf::launch_mxfp4_quant(x, rows, k, ldx, codes, scales, wf::as_stream(stream));
}

int wf_mxfp4_dequant(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* out, int64_t ldo, void* stream) {
  if (int st = wf::check_rows("wf_mxfp4_dequant", out, codes, scales, rows, k, ldo)) return st;
  if (rows == 0 || k == 0) return WF_OK;
  hipLaunchKernelGGL(wf::mxfp4_dequant_kernel, wf::rows_grid(rows, k), dim3(64 * wf::kWaves), 0, wf::as_stream(stream), codes, scales,
                     static_cast<int>(rows), static_cast<int>(k), static_cast<uint16_t*>(out), ldo);
  return wf::check_launch("wf_mxfp4_dequant");
}

}  // extern "C"
