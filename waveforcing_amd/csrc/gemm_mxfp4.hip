// Product of MXFP4 rows: y[m][n] = bf16(act(sum_k a[m,k] w[n,k] + bias[n])), both operands e2m1 codes under E8M0 block scales
// (mxfp4_rows.hip has the layouts), sums and epilogue in fp32, rounded once.  The scaled matrix instruction takes codes and
// scales as they are: v_mfma_scale_f32_32x32x64_f8f6f4 at twice the fp8 rate, products of its sums exact to 2^-24 of sum|a w|.
//
// Many rows (gemm_mxfp4_kernel): the tiles and the K loop of the 8-bit products (gemm_w8a8.hip), whose 128 bytes of a row
// are here 256 values: operands by DMA into XOR-swizzled LDS rows, three stages (the 256-row tile: two), a step of four
// sub-steps, the next sub-step's fragments read and a later step's DMAs issued between the matrix instructions.  A step's
// scales, two words a row (each of 128 values), come with its stage; a lane holds 32 consecutive values of one row in each
// operand, so the byte it needs is 2 s + (its half) of the word: one shift a word, and the instruction's byte select.
//
// Few rows (gemm_mxfp4_few_kernel): up to 64 rows, bound by reading the weight once.  A workgroup takes 16 or 32 columns and
// all rows; its waves split K and go without barriers, operands straight from memory in the layout of the 16x16x128
// instruction (16 bytes of a row a lane), and add up in LDS in the order of the waves.  Up to 16 rows the activations are
// quantized in the same kernel: a lane's operand is one whole block, so the maximum, the scale and the codes need no other
// lane.
#include <algorithm>

#include "gemm_core.hpp"
#include "launchers.hpp"
#include "mxfp4_codec.hpp"

namespace wf {
namespace {

using namespace gemm;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct MxArgs {
  const uint16_t* x;  // few rows: bf16 rows (stride ldx) quantized by the kernel, or null
  int64_t ldx;
  const uint8_t *a, *a_scales, *w, *w_scales;
  const uint16_t* bias;
  uint16_t* y;
  int M, N, K;
  int64_t ldy;
  int gelu;
  int vec16;  // y and ldy allow 16-byte row stores
};

__device__ inline v8i widen(const v4i& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

template <int SEL>
__device__ inline v16f mfma32(const v4i& w, const v4i& a, v16f c, int sw, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(w), widen(a), c, 4, 4, SEL, sw, SEL, sa);
}

// BM x BN outputs of a workgroup of WM x WN waves, ST stages.
template <int BM_, int BN_, int WM_, int WN_, int ST_>
struct MxTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, ST = ST_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
  static constexpr int NBA = BM / 8 / NW, NBB = BN / 8 / NW;       // 1 KB DMA blocks of codes per wave and step
  static constexpr int NSA = (BM + 127) / 128, NSB = (BN + 127) / 128;  // 1 KB DMA blocks of scales per step
  static constexpr int B_OFF = BM * BK, SA_OFF = B_OFF + BN * BK, SB_OFF = SA_OFF + NSA * 1024;
  static constexpr int STAGE = SB_OFF + NSB * 1024;
  static constexpr int WCOLS = BN / WN, WPITCH = WCOLS * 2 + 16;
  static constexpr int EPI = BN * 4;                               // the bias as fp32
  static constexpr int LDS = ST * STAGE + EPI;
  static_assert(NBA * 8 * NW == BM && NBB * 8 * NW == BN && NSA + NSB <= NW, "DMA blocks");
  static_assert(NW * 2 * 32 * WPITCH <= ST * STAGE, "wave staging fits the stages");
  static_assert(LDS <= 160 * 1024, "LDS of one workgroup");
};
using TileBig = MxTile<256, 256, 2, 4, 2>;
using TileStd = MxTile<128, 256, 2, 4, 3>;
using TileMid = MxTile<128, 128, 2, 4, 3>;
using TileSmall = MxTile<64, 64, 2, 2, 3>;

constexpr int SUB = 4;       // sub-steps of a step, 64 values each

template <typename T>
__global__ __launch_bounds__(T::THREADS, 1) void gemm_mxfp4_kernel(MxArgs p) {
  constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN, NW = T::NW, MI = T::MI, NI = T::NI, ST = T::ST;
  constexpr int NBA = T::NBA, NDMA = T::NBA + T::NBB, STAGE = T::STAGE, NS = T::NSA + T::NSB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[T::LDS];
  float* const epi = reinterpret_cast<float*>(lds + ST * STAGE);

  // tiles: an XCD's workgroups (blockIdx % 8) are a contiguous range, walked in bands of GROUP_M tile rows
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
  const int n_tiles = tiles_m * tiles_n, per_xcd = (n_tiles + NUM_XCD - 1) / NUM_XCD;
  const int t = static_cast<int>(blockIdx.x % NUM_XCD) * per_xcd + static_cast<int>(blockIdx.x) / NUM_XCD;
  if (t >= n_tiles || static_cast<int>(blockIdx.x) / NUM_XCD >= per_xcd) return;
  const int per_group = GROUP_M * tiles_n;
  const int first_m = (t / per_group) * GROUP_M;
  const int band = min(tiles_m - first_m, GROUP_M);
  const int m0 = (first_m + (t % per_group) % band) * BM, n0 = ((t % per_group) / band) * BN;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int l32 = lane & 31, half = lane >> 5;

  const int row_bytes = p.K >> 1, groups = (p.K + 127) / 128, M4 = (p.M + 3) & ~3, N4 = (p.N + 3) & ~3;
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a), 0, p.M * row_bytes, kBufferRsrcWord3);
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w), 0, p.N * row_bytes, kBufferRsrcWord3);
  // DMA block j of this wave: rows (j NW + wave) 8 .. + 7 of A (j < NBA) or W; 16-byte chunk c of row r lands at c ^ (r / 2 % 8).
  // The blocks' rows differ by 8 NW, so a lane has one chunk and one offset for each operand.
  static_assert(NW % 2 == 0, "the blocks of a wave share the swizzle");
  const int drow = wave * 8 + (lane >> 3), dcol = 16 * ((lane & 7) ^ ((drow >> 1) & 7));
  const int doff_a = (m0 + drow) * row_bytes + dcol, doff_w = (n0 + drow) * row_bytes + dcol;
  // scales: wave i brings 1 KB (i % (NSA + NSB); the same bytes twice cost less than a branch in the loop) of the step's
  // [2 groups][BM] words of A, then of W's; words past the last group read as zero, those of rows past the last belong to
  // outputs that are not stored
  const int sblk = wave % NS;
  const bool s_is_a = sblk < T::NSA;
  const int srow4 = s_is_a ? M4 : N4;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(s_is_a ? p.a_scales : p.w_scales), 0, groups * srow4 * 4, kBufferRsrcWord3);
  const int sdst = T::SA_OFF + sblk * 1024;
  int soff = kOutOfRange - groups * srow4 * 4;  // (what it grows by over the steps)
  {
    const int word = ((s_is_a ? sblk : sblk - T::NSA) * 64 + lane) * 4, b = s_is_a ? BM : BN, g = word / b;
    if (g < 2) soff = (g * srow4 + (s_is_a ? m0 : n0) + word % b) * 4;
  }
  auto dma = [&](auto J, int step, int stage) __attribute__((always_inline)) {
    constexpr int j = decltype(J)::value;
    const int k0 = step * BK;
    if constexpr (j == NDMA) {
      dma16(rs, lds + stage * STAGE + sdst, soff + __builtin_amdgcn_readfirstlane(step * 2 * srow4 * 4));
    } else {
      // (the uniform part in a scalar register, not a vector register for each block)
      const int by = __builtin_amdgcn_readfirstlane((j < NBA ? j : j - NBA) * NW * 8 * row_bytes + k0);
      const int off = k0 + dcol < row_bytes ? (j < NBA ? doff_a : doff_w) + by : kOutOfRange;
      if constexpr (j < NBA)
        dma16(ra, lds + stage * STAGE + (j * NW + wave) * 1024, off);
      else
        dma16(rw, lds + stage * STAGE + T::B_OFF + ((j - NBA) * NW + wave) * 1024, off);
    }
  };

  // the bias of the tile's columns, for the epilogue (published by the first barrier)
  for (int c = static_cast<int>(threadIdx.x); c < BN; c += T::THREADS)
    epi[c] = p.bias && n0 + c < p.N ? bf16_bits_to_f32(p.bias[n0 + c]) : 0.f;

  // Fragments: sub-step s of a lane's row is its chunk 2 s + half; the rows one lane reads differ by multiples of 32
  const int x = (l32 >> 1) & 7;
  const int lane_a = (wm * (BM / WM) + l32) * BK, lane_b = T::B_OFF + (wn * (BN / WN) + l32) * BK;
  const int lane_sa = T::SA_OFF + (wm * (BM / WM) + l32) * 4, lane_sb = T::SB_OFF + (wn * (BN / WN) + l32) * 4;
  int koff[SUB];
#pragma unroll
  for (int s = 0; s < SUB; ++s) koff[s] = 16 * ((2 * s + half) ^ x);

  v16f acc[NI][MI];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = v16f{};
  v4i fa[2][MI], fw[2][NI];
  int sa[2][MI], sw[2][NI];  // by sub-steps 0, 1 and 2, 3 of a step
  const int shift = 8 * half;

  constexpr int NFR = MI + NI;
  // Read o of sub-step S into buffer S % 2: the fragments, then (even S) the scale words.
  auto frag_read = [&](auto O, auto S, int stage) __attribute__((always_inline)) {
    constexpr int o = decltype(O)::value, s = decltype(S)::value;
    const uint8_t* st = lds + stage * STAGE;
    if constexpr (o < MI)
      fa[s & 1][o] = *reinterpret_cast<const v4i*>(st + lane_a + koff[s] + o * 32 * BK);
    else if constexpr (o < NFR)
      fw[s & 1][o - MI] = *reinterpret_cast<const v4i*>(st + lane_b + koff[s] + (o - MI) * 32 * BK);
    else if constexpr (o < NFR + MI)
      sa[s >> 1][o - NFR] = *reinterpret_cast<const int*>(st + lane_sa + (s >> 1) * BM * 4 + (o - NFR) * 128);
    else
      sw[s >> 1][o - NFR - MI] = *reinterpret_cast<const int*>(st + lane_sb + (s >> 1) * BN * 4 + (o - NFR - MI) * 128);
  };
  // The products of sub-step S and, spread between them, the reads of sub-step (S + 1) % 4 from rstage (RD) and the DMAs
  // of slot SLOT (of SUB; two stages: all in slot 0) of step dstep into dstage (DM).
  auto substep = [&](auto S, int rstage, auto SLOT, int dstep, int dstage, auto RD, auto DM) __attribute__((always_inline)) {
    constexpr int s = decltype(S)::value, slot = decltype(SLOT)::value, nx = (s + 1) % SUB;
    constexpr bool rd = decltype(RD)::value, dm = decltype(DM)::value;
    constexpr int ND = NDMA + 1;
    constexpr int d_lo = ST == 3 ? (slot * ND + SUB - 1) / SUB : 0;
    constexpr int d_hi = !dm ? d_lo : ST == 3 ? ((slot + 1) * ND + SUB - 1) / SUB : (slot == 0 ? ND : 0);
    constexpr int NMF = MI * NI, NRD = rd ? (nx % 2 == 0 ? 2 * NFR : NFR) : 0, NOPS = NRD + d_hi - d_lo;
    if constexpr (s % 2 == 0) {
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[s >> 1][i] = static_cast<int>(static_cast<uint32_t>(sa[s >> 1][i]) >> shift);
#pragma unroll
      for (int j = 0; j < NI; ++j) sw[s >> 1][j] = static_cast<int>(static_cast<uint32_t>(sw[s >> 1][j]) >> shift);
    }
    static_for<NMF>([&](auto Q) {
      constexpr int q = decltype(Q)::value, jj = q / MI, ii = q % MI;
      acc[jj][ii] = mfma32<2 * (s & 1)>(fw[s & 1][jj], fa[s & 1][ii], acc[jj][ii], sw[s >> 1][jj], sa[s >> 1][ii]);
      constexpr int o_lo = (q * NOPS + NMF - 1) / NMF, o_hi = ((q + 1) * NOPS + NMF - 1) / NMF;
      static_for<o_hi - o_lo>([&](auto U) {
        constexpr int o = o_lo + decltype(U)::value;
        if constexpr (o < NRD)
          frag_read(ic<o>{}, ic<nx>{}, rstage);
        else
          dma(ic<d_lo + o - NRD>{}, dstep, dstage);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto barrier = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // Stages 0 and 1; only stage 0 is waited for here (a wave's DMAs land in order).
  const int nk = (row_bytes + BK - 1) / BK;
  static_for<NDMA + 1>([&](auto J) { dma(J, 0, 0); });
  if (nk > 1) static_for<NDMA + 1>([&](auto J) { dma(J, 1, 1); });
  if (nk == 1)
    wait_counts<0, 0>();
  else
    wait_counts<NDMA + 1, 0>();
  barrier();
  if constexpr (ST == 3) {  // slot 0 of step 2
    if (nk >= 3) static_for<(NDMA + 1 + SUB - 1) / SUB>([&](auto J) { dma(J, 2, 2); });
  }
  static_for<2 * NFR>([&](auto O) { frag_read(O, ic<0>{}, 0); });
  __builtin_amdgcn_sched_barrier(0);

  if constexpr (ST == 3) {
    // Step kb: sub-steps 0 .. 2 fetch slots 1 .. 3 of step kb + 2 (PRE), the last one, behind the barrier that frees this
    // step's stage, slot 0 of step kb + 3 (POST).  The last three steps are peeled: nothing past K is fetched.
    int c0 = 0, c1 = 1, c2 = 2;
    auto step = [&](int kb, auto PRE, auto POST, auto LAST) __attribute__((always_inline)) {
      constexpr bool pre = decltype(PRE)::value, last = decltype(LAST)::value;
      static_for<SUB - 1>([&](auto S) { substep(S, c0, ic<decltype(S)::value + 1>{}, kb + 2, c2, ic<1>{}, PRE); });
      if constexpr (!last) {
        // own reads of this stage done, own DMAs of step kb + 1 landed (of step kb + 2 all may be in flight)
        if constexpr (pre)
          wait_counts<NDMA + 1, 0>();
        else
          wait_counts<0, 0>();
        barrier();
      }
      substep(ic<SUB - 1>{}, c1, ic<0>{}, kb + 3, c0, ic<!last>{}, POST);
      const int c = c0;
      c0 = c1;
      c1 = c2;
      c2 = c;
    };
    int kb = 0;
    for (; kb < nk - 3; ++kb) step(kb, ic<1>{}, ic<1>{}, ic<0>{});
    if (nk >= 3) step(kb++, ic<1>{}, ic<0>{}, ic<0>{});
    if (nk >= 2) step(kb++, ic<0>{}, ic<0>{}, ic<0>{});
    step(kb, ic<0>{}, ic<0>{}, ic<1>{});
  } else {
    // Two stages: the barrier before a step's last sub-step has every DMA landed and frees the step's stage, into which
    // that sub-step fetches all of step kb + 2.
    int c0 = 0, c1 = 1;
    auto step = [&](int kb, auto POST, auto LAST) __attribute__((always_inline)) {
      constexpr bool last = decltype(LAST)::value;
      static_for<SUB - 1>([&](auto S) { substep(S, c0, ic<decltype(S)::value + 1>{}, 0, 0, ic<1>{}, ic<0>{}); });
      if constexpr (!last) {
        wait_counts<0, 0>();
        barrier();
      }
      substep(ic<SUB - 1>{}, c1, ic<0>{}, kb + 2, c0, ic<!last>{}, POST);
      const int c = c0;
      c0 = c1;
      c1 = c;
    };
    int kb = 0;
    for (; kb < nk - 2; ++kb) step(kb, ic<1>{}, ic<0>{});
    if (nk >= 2) step(kb++, ic<0>{}, ic<0>{});
    step(kb, ic<0>{}, ic<1>{});
  }

  // Epilogue: every wave converts its sub-tile as 32-row slabs, through its own LDS area (two in turn), stored as whole row
  // segments.  Block (j, i), element (n, m): m = l32, n = 8 (r / 4) + 4 half + r % 4.
  wait_counts<0, 0>();
  barrier();
  uint8_t* const wst = lds + wave * (2 * 32 * T::WPITCH);
  const bool gelu = p.gelu != 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    uint8_t* const slab = wst + (i & 1) * 32 * T::WPITCH;
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int cw = j * 32 + 8 * g + 4 * half;
        const float4 b = *reinterpret_cast<const float4*>(epi + wn * T::WCOLS + cw);
        float v[4] = {acc[j][i][4 * g] + b.x, acc[j][i][4 * g + 1] + b.y, acc[j][i][4 * g + 2] + b.z, acc[j][i][4 * g + 3] + b.w};
        if (gelu) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
        }
        *reinterpret_cast<uint2*>(slab + l32 * T::WPITCH + cw * 2) = make_uint2(pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]));
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int CH = T::WCOLS / 8, RPI = 64 / CH;  // 16-byte chunks of a row, rows of a store
#pragma unroll
    for (int it = 0; it < 32 / RPI; ++it) {
      const int rr = it * RPI + lane / CH, ch = lane % CH;
      const uint4 v = *reinterpret_cast<const uint4*>(slab + rr * T::WPITCH + ch * 16);
      const int gm = m0 + wm * (BM / WM) + i * 32 + rr, gn = n0 + wn * T::WCOLS + ch * 8;
      if (gm < p.M && gn < p.N) {
        uint16_t* dst = p.y + static_cast<int64_t>(gm) * p.ldy + gn;
        if (p.vec16 && gn + 8 <= p.N) {
          *reinterpret_cast<uint4*>(dst) = v;
        } else {  // (N % 4 == 0)
          *reinterpret_cast<uint2*>(dst) = make_uint2(v.x, v.y);
          if (gn + 8 <= p.N) *reinterpret_cast<uint2*>(dst + 4) = make_uint2(v.z, v.w);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- few rows
constexpr int kFewRows = 64, kFusedRows = WF_MXFP4_FUSED_ROWS;

// NB blocks of 16 rows, NC of 16 columns, W waves that share K in turns of 128 values; QUANT: the rows are bf16.
template <int NB, int NC, int W, bool QUANT>
__global__ __launch_bounds__(64 * W) void gemm_mxfp4_few_kernel(MxArgs p) {
  static_assert(!QUANT || NB == 1, "rows quantized in the kernel: one block");
  __shared__ __attribute__((aligned(16))) v4f part[W > 1 ? W - 1 : 1][NB * NC][64];
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int n0 = static_cast<int>(blockIdx.x) * 16 * NC;
  const int row_bytes = p.K >> 1, steps = (p.K + 127) / 128, M4 = (p.M + 3) & ~3, N4 = (p.N + 3) & ~3;
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w), 0, p.N * row_bytes, kBufferRsrcWord3);
  const auto rsw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w_scales), 0, steps * N4 * 4, kBufferRsrcWord3);
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a), 0, QUANT ? 0 : p.M * row_bytes, kBufferRsrcWord3);
  const auto rsa = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a_scales), 0, QUANT ? 0 : steps * M4 * 4, kBufferRsrcWord3);

  v4f acc[NB][NC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[b][c] = v4f{0, 0, 0, 0};
  // a lane's 32 values of a step: those from 128 s + 32 g4 on, of column n0 + 16 c + l16 and row 16 b + l16
  struct Regs {
    u32x4 w[NC], a[QUANT ? 4 : NB];
    int sw[NC], sa[NB];
  };
  const bool row_ok = l16 < p.M;
  const uint16_t* xrow = QUANT ? p.x + static_cast<int64_t>(row_ok ? l16 : 0) * p.ldx + 32 * g4 : nullptr;
  auto load = [&](int s, Regs& r) __attribute__((always_inline)) {
    const bool there = 128 * s + 32 * g4 < p.K;  // (K % 32 == 0; also false past the last step)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int n = n0 + 16 * c + l16;
      r.w[c] = __builtin_amdgcn_raw_buffer_load_b128(rw, there ? n * row_bytes + 64 * s + 16 * g4 : kOutOfRange, 0, 0);
      r.sw[c] = __builtin_amdgcn_raw_buffer_load_b8(rsw, there && n < p.N ? (s * N4 + n) * 4 + g4 : kOutOfRange, 0, 0);
    }
    if constexpr (QUANT) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        r.a[i] = u32x4{0, 0, 0, 0};
        if (row_ok && there) r.a[i] = *reinterpret_cast<const u32x4*>(xrow + 128 * s + 8 * i);
      }
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int m = 16 * b + l16;
        r.a[b] = __builtin_amdgcn_raw_buffer_load_b128(ra, there ? m * row_bytes + 64 * s + 16 * g4 : kOutOfRange, 0, 0);
        r.sa[b] = __builtin_amdgcn_raw_buffer_load_b8(rsa, there && m < p.M ? (s * M4 + m) * 4 + g4 : kOutOfRange, 0, 0);
      }
    }
  };
  auto product = [&](Regs& r) __attribute__((always_inline)) {
    v4i a[NB];
    if constexpr (QUANT) {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = mx::max_bits2(top, mx::max_bits2(mx::max_bits2(r.a[i][0], r.a[i][1]), mx::max_bits2(r.a[i][2], r.a[i][3])));
      const int e = mx::scale_byte(mx::max_half(top));
      const float s = mx::scale_of(e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w[4] = {r.a[i][0], r.a[i][1], r.a[i][2], r.a[i][3]};
        a[0][i] = static_cast<int>(mx::encode8(w, s));  // (whatever the codes, a scale byte of 255 makes the sum NaN)
      }
      r.sa[0] = e;
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) a[b] = __builtin_bit_cast(v4i, r.a[b]);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        acc[b][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(__builtin_bit_cast(v4i, r.w[c])), widen(a[b]), acc[b][c], 4, 4, 0,
                                                                     r.sw[c] & 0xff, 0, r.sa[b] & 0xff);
  };
  constexpr int DEEP = NB == 4 ? 2 : 4;  // steps whose loads are in flight
  Regs r[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) load(wave + W * d, r[d]);
  for (int s = wave; s < steps; s += W * DEEP) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      product(r[d]);
      load(s + W * (DEEP + d), r[d]);
    }
  }

  if constexpr (W > 1) {
    if (wave) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int c = 0; c < NC; ++c) part[wave - 1][b * NC + c][lane] = acc[b][c];
    }
    __syncthreads();
    if (wave) return;
  }
  // wave 0 adds the others' sums, in their order, and stores
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      v4f v = acc[b][c];
      if constexpr (W > 1) {
#pragma unroll
        for (int i = 0; i < W - 1; ++i) v += part[i][b * NC + c][lane];
      }
      const int m = 16 * b + l16, n = n0 + 16 * c + 4 * g4;  // rows of the first operand, 4 to a lane: columns of y
      if (m >= p.M || n >= p.N) continue;
      if (p.bias) {
        const uint2 w = *reinterpret_cast<const uint2*>(p.bias + n);
        v[0] += bf16_lo_to_f32(w.x), v[1] += bf16_hi_to_f32(w.x), v[2] += bf16_lo_to_f32(w.y), v[3] += bf16_hi_to_f32(w.y);
      }
      if (p.gelu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
      }
      *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(m) * p.ldy + n) = make_uint2(pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]));
    }
}

template <int NB, int NC, bool QUANT>
void launch_few_waves(const MxArgs& p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>((p.N + 16 * NC - 1) / (16 * NC)));
  if (p.K <= 128 * 8)
    hipLaunchKernelGGL((gemm_mxfp4_few_kernel<NB, NC, 4, QUANT>), grid, dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((gemm_mxfp4_few_kernel<NB, NC, 8, QUANT>), grid, dim3(512), 0, stream, p);
}

template <int NB, bool QUANT>
void launch_few(const MxArgs& p, hipStream_t stream) {
  if (p.N >= 32 * device_cus())
    launch_few_waves<NB, 2, QUANT>(p, stream);
  else
    launch_few_waves<NB, 1, QUANT>(p, stream);
}

template <typename T>
void launch_tile(const MxArgs& p, hipStream_t stream) {
  const int64_t tiles = static_cast<int64_t>((p.M + T::BM - 1) / T::BM) * ((p.N + T::BN - 1) / T::BN);
  hipLaunchKernelGGL((gemm_mxfp4_kernel<T>), dim3(static_cast<uint32_t>((tiles + NUM_XCD - 1) / NUM_XCD * NUM_XCD)), dim3(T::THREADS), 0,
                     stream, p);
}

int launch_gemm(const MxArgs& p, hipStream_t stream) {
  if (p.x) {
    launch_few<1, true>(p, stream);
  } else if (p.M <= 16) {
    launch_few<1, false>(p, stream);
  } else if (p.M <= 32) {
    launch_few<2, false>(p, stream);
  } else if (p.M <= kFewRows) {
    launch_few<4, false>(p, stream);
  } else {
    auto tiles = [&](int bm, int bn) { return static_cast<int64_t>((p.M + bm - 1) / bm) * ((p.N + bn - 1) / bn); };
    const int64_t cus = device_cus();
    if (tiles(256, 256) >= cus)
      launch_tile<TileBig>(p, stream);
    else if (tiles(128, 256) >= cus)
      launch_tile<TileStd>(p, stream);
    else if (tiles(128, 128) >= cus)
      launch_tile<TileMid>(p, stream);
    else
      launch_tile<TileSmall>(p, stream);
  }
  return check_launch("wf_gemm_mxfp4");
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks and arguments that both entry points share.
int make_args(const char* fn, MxArgs& p, int64_t m, int64_t n, int64_t k, const uint8_t* w, const uint8_t* w_scales, const void* bias,
              void* y, int64_t ldy, int32_t flags) {
  WF_REQUIRE(m < (1ll << 31) - 512 && n < (1ll << 31) - 512 && k < (1ll << 31) && product_below({m + 512, k / 2}, (1ll << 31) - 64) &&
                 product_below({n + 512, k / 2}, (1ll << 31) - 64),
             WF_E_SHAPE, "%s: operands of 2 GiB or more are not supported", fn);
  // (a grid holds fewer than 2^32 threads; outputs of so many tiles are on the largest)
  WF_REQUIRE(product_below({m / 256 + 1, n / 256 + 1, 512}, 1ll << 32), WF_E_SHAPE, "%s: m=%lld x n=%lld is too large", fn, (long long)m,
             (long long)n);
  WF_REQUIRE(k % mx::kBlock == 0 && k > 0, WF_E_SHAPE, "%s: k=%lld must be a positive multiple of 32", fn, (long long)k);
  WF_REQUIRE(n % 4 == 0 && ldy % 4 == 0, WF_E_SHAPE, "%s: n and ldy must be multiples of 4", fn);
  WF_REQUIRE(w && w_scales && y, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(aligned(w, 16) && aligned(w_scales, 16) && aligned(y, 8) && aligned(bias, 8), WF_E_ALIGN,
             "%s: codes and scales must be 16-byte and y, bias 8-byte aligned", fn);
  WF_REQUIRE((flags & ~WF_GEMM_GELU_TANH) == 0, WF_E_INVALID, "%s: unknown flags 0x%x", fn, flags);
  p = MxArgs{};
  p.w = w;
  p.w_scales = w_scales;
  p.bias = static_cast<const uint16_t*>(bias);
  p.y = static_cast<uint16_t*>(y);
  p.M = static_cast<int>(m);
  p.N = static_cast<int>(n);
  p.K = static_cast<int>(k);
  p.ldy = ldy;
  p.gelu = (flags & WF_GEMM_GELU_TANH) != 0;
  p.vec16 = ldy % 8 == 0 && aligned(y, 16);
  return WF_OK;
}

}  // namespace
}  // namespace wf

extern "C" {

int wf_gemm_mxfp4(const uint8_t* a, const uint8_t* a_scales, const uint8_t* w, const uint8_t* w_scales, int64_t m, int64_t n, int64_t k,
                  const void* bias, void* y, int64_t ldy, int32_t flags, void* stream) {
  static const char* fn = "wf_gemm_mxfp4";
  WF_REQUIRE(m >= 0 && n >= 0 && k >= 0 && ldy >= n, WF_E_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld ldy=%lld", fn, (long long)m,
             (long long)n, (long long)k, (long long)ldy);
  if (m == 0 || n == 0) return WF_OK;
  wf::MxArgs p;
  if (int st = wf::make_args(fn, p, m, n, k, w, w_scales, bias, y, ldy, flags)) return st;
  WF_REQUIRE(a && a_scales, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(wf::aligned(a, 16) && wf::aligned(a_scales, 16), WF_E_ALIGN, "%s: codes and scales must be 16-byte aligned", fn);
  p.a = a;
  p.a_scales = a_scales;
  return wf::launch_gemm(p, wf::as_stream(stream));
}

int wf_mxfp4_linear(const void* x, int64_t m, int64_t k, int64_t ldx, const uint8_t* w, const uint8_t* w_scales, const void* bias,
                    int64_t n, void* y, int64_t ldy, int32_t flags, uint8_t* ws_codes, uint8_t* ws_scales, void* stream) {
  static const char* fn = "wf_mxfp4_linear";
  WF_REQUIRE(m >= 0 && n >= 0 && k > 0 && ldx >= k && ldy >= n, WF_E_INVALID, "%s: bad sizes m=%lld n=%lld k=%lld ldx=%lld ldy=%lld", fn,
             (long long)m, (long long)n, (long long)k, (long long)ldx, (long long)ldy);
  if (m == 0 || n == 0) return WF_OK;
  wf::MxArgs p;
  if (int st = wf::make_args(fn, p, m, n, k, w, w_scales, bias, y, ldy, flags)) return st;
  WF_REQUIRE(x, WF_E_INVALID, "%s: null pointer", fn);
  WF_REQUIRE(wf::aligned(x, 16) && ldx % 8 == 0, WF_E_ALIGN, "%s: x must be 16-byte aligned with ldx %% 8 == 0", fn);
  if (m <= wf::kFusedRows) {
    p.x = static_cast<const uint16_t*>(x);
    p.ldx = ldx;
  } else {
    WF_REQUIRE(ws_codes && ws_scales, WF_E_INVALID, "%s: null workspace", fn);
    WF_REQUIRE(wf::aligned(ws_codes, 16) && wf::aligned(ws_scales, 16), WF_E_ALIGN, "%s: the workspaces must be 16-byte aligned", fn);
    if (int st = wf::launch_mxfp4_quant(x, m, k, ldx, ws_codes, ws_scales, wf::as_stream(stream))) return st;
    p.a = ws_codes;
    p.a_scales = ws_scales;
  }
  return wf::launch_gemm(p, wf::as_stream(stream));
}

}  // extern "C"
