// Product of MXFP4 rows: y[m][n] = bf16(act(sum_k a[m,k] w[n,k] + bias[n])), both operands e2m1 codes under E8M0 block scales
// (mxfp4_rows.hip has the layouts), sums and epilogue in fp32, rounded once.  The scaled matrix instruction takes codes and
// scales as they are: v_mfma_scale_f32_32x32x64_f8f6f4 at twice the fp8 rate, products of its sums exact to 2^-24 of sum|a w|.
//
// Many rows (gemm_mxfp4_kernel): the K loop of the 8-bit products (gemm_w8a8.hip), whose 128 bytes of a row are here 256
// values: operands by DMA into LDS, three stages (the 256-row tile and the smallest: four), a step of four sub-steps (the
// 256-row tile: two), the next sub-step's fragments read and a later step's DMAs issued between the matrix instructions.  A panel
// (16 rows x 128 values, 1 KB in the order of the lanes) is one DMA, and 16 lanes' fragments are 256 bytes in a row: no swizzle,
// and every place in LDS is a constant from the lane's first.  The scales, a word a row and panel, come with their stage; the
// byte a lane needs is 2 s + (its half) of the word: one shift a word, and the instruction's byte select.
//
// It is bound by the matrix cores and the power limit: 16384^3 at 4.9 PFLOP/s on N(0, 1) operands, 7.6 on zeros; 4680 x 13824 -> 5120
// 155-162 us by box (4.1-4.3; whole rounds of 256 x 256 tiles, then smaller ones), 5120 -> 13824 173-180 (3.7-3.8).
//
// Few rows, or a small output (gemm_mxfp4_few_kernel): bound by reading the weight once, or by the way from the first load to
// the last store.  A workgroup takes 16 or 32 columns (64 in one case) and 16 or 32 rows; its waves split K and go without
// barriers, operands straight from memory, and add up in LDS in the order of the waves.  Up to WF_MXFP4_FUSED_ROWS rows the
// activations are quantized in the same kernel.  1 x 5120 -> 13824 9.1 us (37.6 MB, 4.1 TB/s), 1 x 13824 -> 5120 10.3, 1 x 1536 -> 4608
// 3.4 (an empty launch 3), 64 x 13824 -> 5120 16.
#include <algorithm>
#include <type_traits>

#include "gemm_core.hpp"
#include "launchers.hpp"
#include "mxfp4_codec.hpp"

namespace wf {
namespace {

using namespace gemm;
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// A part of the output that one tile covers: rows [m0, m1), columns [n0, n1), from m0 and n0 on in whole tiles.
struct Rect {
  int m0, m1, n0, n1;
};

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
  Rect rect[4];  // of the first tile: 0, 1; of the second: 2, 3
  int count[4];  // their tiles
};

__device__ inline v8i widen(const v4i& v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

template <int SEL>
__device__ inline v16f mfma32(const v4i& w, const v4i& a, v16f c, int sw, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(w), widen(a), c, 4, 4, SEL, sw, SEL, sa);
}

// BM x BN outputs of a workgroup of WM x WN waves; steps of KG panels' depth (128 values each), ST stages of one.
template <int BM_, int BN_, int WM_, int WN_, int KG_, int ST_>
struct MxTile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KG = KG_, ST = ST_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int MI = BM / WM / 32, NI = BN / WN / 32;
  static constexpr int SUB = 2 * KG;                               // sub-steps of 64 values
  static constexpr int NBA = BM / 16 * KG / NW, NBB = BN / 16 * KG / NW;  // 1 KB DMA blocks of codes per wave and step
  static constexpr int NSA = (BM * KG + 255) / 256, NSB = (BN * KG + 255) / 256;  // and of scales per step, the last may be half used
  static constexpr int B_OFF = BM * KG * 64, SA_OFF = B_OFF + BN * KG * 64, SB_OFF = SA_OFF + NSA * 1024;
  static constexpr int STAGE = SB_OFF + NSB * 1024;
  static constexpr int WCOLS = BN / WN, WPITCH = WCOLS * 2 + 16;
  static constexpr int EPI = BN * 4;                               // the bias as fp32
  static constexpr int LDS = ST * STAGE + EPI;
  static_assert(NBA * 16 * NW == BM * KG && NBB * 16 * NW == BN * KG && NSA + NSB <= NW && NW % KG == 0, "DMA blocks");
  static_assert(NW * 2 * 32 * WPITCH <= ST * STAGE, "wave staging fits the stages");
  static_assert(LDS <= 160 * 1024, "LDS of one workgroup");
};
using TileBig = MxTile<256, 256, 2, 4, 1, 4>;  // (two stages of 256 values: 5-20 % slower)
using TileStd = MxTile<128, 256, 2, 4, 2, 3>;
using TileMid = MxTile<128, 128, 2, 4, 2, 3>;
using TileHalf = MxTile<64, 128, 2, 2, 2, 3>;
using TileSmall = MxTile<64, 64, 2, 2, 2, 4>;   // (three: up to 15 % slower over long K)

constexpr uint32_t kFar = 0x7ffffff0u;

// Tile t of rect r.
template <typename T>
__device__ __attribute__((always_inline)) inline void mx_tile(const MxArgs& p, const Rect& r, int t, uint8_t* lds) {
  constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN, NW = T::NW, MI = T::MI, NI = T::NI, ST = T::ST;
  constexpr int KG = T::KG, SUB = T::SUB, NBA = T::NBA, NDMA = T::NBA + T::NBB, ND = NDMA + 1, STAGE = T::STAGE, NS = T::NSA + T::NSB;
  float* const epi = reinterpret_cast<float*>(lds + ST * STAGE);

  // in bands of GROUP_M tile rows
  const int tiles_m = (r.m1 - r.m0 + BM - 1) / BM, tiles_n = (r.n1 - r.n0 + BN - 1) / BN;
  const int per_group = GROUP_M * tiles_n;
  const int first_m = (t / per_group) * GROUP_M;
  const int band = min(tiles_m - first_m, GROUP_M);
  const int m0 = r.m0 + (first_m + (t % per_group) % band) * BM, n0 = r.n0 + ((t % per_group) / band) * BN;
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int l32 = lane & 31, half = lane >> 5;

  const int groups = (p.K + 127) / 128, pa = (p.M + 15) / 16, pw = (p.N + 15) / 16;  // panels
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a), 0, pa * groups * 1024, kBufferRsrcWord3);
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w), 0, pw * groups * 1024, kBufferRsrcWord3);

  // DMA block j of this wave: panel (j NW + wave) / KG of the tile's rows, the step's 128 values (wave % KG).  Panels past the
  // last row are past the buffer's end and read as zero.
  const uint32_t doff_a = static_cast<uint32_t>(((m0 / 16 + wave / KG) * groups + wave % KG) * 1024 + 16 * lane);
  const uint32_t doff_w = static_cast<uint32_t>(((n0 / 16 + wave / KG) * groups + wave % KG) * 1024 + 16 * lane);
  // scales: wave i brings 1 KB (i % (NSA + NSB); the same bytes twice cost less than a branch in the loop), 64 KG bytes a panel
  const int sblk = wave % NS;
  const bool s_is_a = sblk < T::NSA;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(s_is_a ? p.a_scales : p.w_scales), 0,
                                                    (s_is_a ? pa : pw) * groups * 64, kBufferRsrcWord3);
  const int sdst = T::SA_OFF + sblk * 1024;
  const int schunk = (s_is_a ? sblk : sblk - T::NSA) * 64 + lane, spanel = schunk / (4 * KG);
  // Offsets are unsigned: kFar more is out of every buffer's range.  (In scalar registers where they are uniform, not a vector
  // register for each block; and no branch in the loop.)
  const bool s_in = spanel < (s_is_a ? BM : BN) / 16;
  const uint32_t soff = s_in ? static_cast<uint32_t>((((s_is_a ? m0 : n0) / 16 + spanel) * groups) * 64 + 16 * (schunk % (4 * KG))) : kFar;
  const uint32_t s_second = s_in && schunk % (4 * KG) >= 4 ? kFar : 0u;  // the words of the second 128 values
  auto dma = [&](auto J, int step, int stage) __attribute__((always_inline)) {
    constexpr int j = decltype(J)::value;
    // (a last step of 128 values of 256: nothing in the place of the second 128, not the next panel's first)
    if constexpr (j == NDMA) {
      uint32_t far = 0;
      if constexpr (KG == 2) far = __builtin_amdgcn_readfirstlane(2 * step + 1 < groups ? 0 : -1) & s_second;
      dma16(rs, lds + stage * STAGE + sdst, static_cast<int>(soff + static_cast<uint32_t>(step) * (64u * KG) + far));
    } else {
      const uint32_t at = static_cast<uint32_t>((j < NBA ? j : j - NBA) * (NW / KG) * groups * 1024 + step * (1024 * KG));
      const uint32_t by = __builtin_amdgcn_readfirstlane(KG == 1 || 2 * step + (wave & 1) < groups ? at : kFar);
      if constexpr (j < NBA)
        dma16(ra, lds + stage * STAGE + (j * NW + wave) * 1024, static_cast<int>(doff_a + by));
      else
        dma16(rw, lds + stage * STAGE + T::B_OFF + ((j - NBA) * NW + wave) * 1024, static_cast<int>(doff_w + by));
    }
  };

  // the bias of the tile's columns, for the epilogue (published by the first barrier)
  for (int c = static_cast<int>(threadIdx.x); c < BN; c += T::THREADS)
    epi[c] = p.bias && n0 + c < p.N ? bf16_bits_to_f32(p.bias[n0 + c]) : 0.f;

  // Fragments: a lane's 32 values of sub-step s are block 2 (s % 2) + half of its row in the panel of the step's first (s < 2)
  // or second 128 values
  constexpr int PANEL = 1024 * KG, WORDS = 64 * KG;  // LDS bytes of a panel's codes and scales
  const int lane_a = (wm * (BM / WM) / 16 + (l32 >> 4)) * PANEL + half * 256 + (l32 & 15) * 16;
  const int lane_b = T::B_OFF + (wn * (BN / WN) / 16 + (l32 >> 4)) * PANEL + half * 256 + (l32 & 15) * 16;
  const int lane_sa = T::SA_OFF + (wm * (BM / WM) / 16 + (l32 >> 4)) * WORDS + (l32 & 15) * 4;
  const int lane_sb = T::SB_OFF + (wn * (BN / WN) / 16 + (l32 >> 4)) * WORDS + (l32 & 15) * 4;

  v16f acc[NI][MI];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int i = 0; i < MI; ++i) acc[j][i] = v16f{};
  v4i fa[2][MI], fw[2][NI];
  uint32_t sa_next[MI], sw_next[NI];  // scale words as they are read, and from the lane's byte on
  int sa[MI], sw[NI];
  const int shift = 8 * half;

  constexpr int NFR = MI + NI;
  // Read o of sub-step S into buffer S % 2: the fragments, then (even S) the scale words.
  auto frag_read = [&](auto O, auto S, int stage) __attribute__((always_inline)) {
    constexpr int o = decltype(O)::value, s = decltype(S)::value;
    const uint8_t* st = lds + stage * STAGE;
    if constexpr (o < MI)
      fa[s & 1][o] = *reinterpret_cast<const v4i*>(st + lane_a + (s >> 1) * 1024 + (s & 1) * 512 + o * 2 * PANEL);
    else if constexpr (o < NFR)
      fw[s & 1][o - MI] = *reinterpret_cast<const v4i*>(st + lane_b + (s >> 1) * 1024 + (s & 1) * 512 + (o - MI) * 2 * PANEL);
    else if constexpr (o < NFR + MI)
      sa_next[o - NFR] = *reinterpret_cast<const uint32_t*>(st + lane_sa + (s >> 1) * 64 + (o - NFR) * 2 * WORDS);
    else
      sw_next[o - NFR - MI] = *reinterpret_cast<const uint32_t*>(st + lane_sb + (s >> 1) * 64 + (o - NFR - MI) * 2 * WORDS);
  };
  // The products of sub-step S and, spread between them, the reads of sub-step (S + 1) % SUB from rstage (RD) and the DMAs
  // of slot SLOT (of SUB; two stages: all in slot 0) of step dstep into dstage (DM).
  auto substep = [&](auto S, int rstage, auto SLOT, int dstep, int dstage, auto RD, auto DM) __attribute__((always_inline)) {
    constexpr int s = decltype(S)::value, slot = decltype(SLOT)::value, nx = (s + 1) % SUB;
    constexpr bool rd = decltype(RD)::value, dm = decltype(DM)::value;
    constexpr int d_lo = ST > 2 ? (slot * ND + SUB - 1) / SUB : 0;
    constexpr int d_hi = !dm ? d_lo : ST > 2 ? ((slot + 1) * ND + SUB - 1) / SUB : (slot == 0 ? ND : 0);
    constexpr int NMF = MI * NI, NRD = rd ? (nx % 2 == 0 ? 2 * NFR : NFR) : 0, NOPS = NRD + d_hi - d_lo;
    if constexpr (s % 2 == 0) {
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = static_cast<int>(sa_next[i] >> shift);
#pragma unroll
      for (int j = 0; j < NI; ++j) sw[j] = static_cast<int>(sw_next[j] >> shift);
    }
    static_for<NMF>([&](auto Q) {
      constexpr int q = decltype(Q)::value, jj = q / MI, ii = q % MI;
      acc[jj][ii] = mfma32<2 * (s & 1)>(fw[s & 1][jj], fa[s & 1][ii], acc[jj][ii], sw[jj], sa[ii]);
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

  // The first steps; only step 0 is waited for here (a wave's DMAs land in order).
  const int nk = (groups + KG - 1) / KG;
  constexpr int FIRST = ST > 2 ? ST - 1 : 2;
  static_for<FIRST>([&](auto I) {
    if (decltype(I)::value < nk) static_for<ND>([&](auto J) { dma(J, decltype(I)::value, decltype(I)::value); });
  });
  if (nk >= FIRST)
    wait_counts<(FIRST - 1) * ND, 0>();
  else
    wait_counts<0, 0>();
  barrier();
  if constexpr (ST > 2) {  // slot 0 of the next
    if (nk >= ST) static_for<(ND + SUB - 1) / SUB>([&](auto J) { dma(J, ST - 1, ST - 1); });
  }
  static_for<2 * NFR>([&](auto O) { frag_read(O, ic<0>{}, 0); });
  __builtin_amdgcn_sched_barrier(0);

  // Step kb.  Its last sub-step runs behind the barrier that frees the step's stage.  More than two stages: the sub-steps before
  // it fetch slots 1 .. of step kb + ST - 1 (PRE) into the stage of kb - 1, it slot 0 of kb + ST (POST); two: it fetches all of
  // kb + 2.  Only steps below nk are fetched, so the last ST are peeled.  WAIT: steps beyond kb + 1 that may be in flight.
  int cur = 0;
  auto step = [&](int kb, auto PRE, auto POST, auto WAIT, auto LAST) __attribute__((always_inline)) {
    constexpr bool last = decltype(LAST)::value;
    const int next = cur + 1 == ST ? 0 : cur + 1, before = cur == 0 ? ST - 1 : cur - 1;
    static_for<SUB - 1>([&](auto S) { substep(S, cur, ic<decltype(S)::value + 1>{}, kb + ST - 1, before, ic<1>{}, PRE); });
    if constexpr (!last) {
      wait_counts<decltype(WAIT)::value * ND, 0>();
      barrier();
    }
    substep(ic<SUB - 1>{}, next, ic<0>{}, kb + ST, cur, ic<!last>{}, POST);
    cur = next;
  };
  constexpr bool kPre = ST > 2;
  constexpr int kAhead = ST > 2 ? ST - 2 : 0;
  int kb = 0;
  for (; kb < nk - ST; ++kb) step(kb, ic<kPre>{}, ic<1>{}, ic<kAhead>{}, ic<0>{});
  if constexpr (kPre) {
    if (nk >= ST) step(kb++, ic<1>{}, ic<0>{}, ic<kAhead>{}, ic<0>{});
  }
  constexpr int TAIL = ST > 2 ? ST - 2 : 1;
  static_for<TAIL>([&](auto I) {
    constexpr int w = TAIL - 1 - decltype(I)::value;
    if (nk - kb >= w + 2) step(kb++, ic<0>{}, ic<0>{}, ic<w>{}, ic<0>{});
  });
  step(kb, ic<0>{}, ic<0>{}, ic<0>{}, ic<1>{});

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

// The tiles of T1, then those of T2 (the output's rest), in one launch: a CU takes its next tile as soon as it is done with one.
// An XCD's workgroups (blockIdx % 8) take a contiguous range of each rect's tiles.
template <typename T1, typename T2>
__global__ __launch_bounds__(T1::THREADS, 1) void gemm_mxfp4_kernel(MxArgs p) {
  static_assert(T1::THREADS == T2::THREADS, "one launch");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[T1::LDS > T2::LDS ? T1::LDS : T2::LDS];
  int w = static_cast<int>(blockIdx.x), at = 0, t = 0;
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int per_xcd = (p.count[i] + NUM_XCD - 1) / NUM_XCD, padded = per_xcd * NUM_XCD;
    if (!found && w < padded) {
      found = true;
      at = i;
      t = w % NUM_XCD * per_xcd + w / NUM_XCD;
    }
    w -= padded;
  }
  const Rect r{at == 0 ? p.rect[0].m0 : at == 1 ? p.rect[1].m0 : at == 2 ? p.rect[2].m0 : p.rect[3].m0,
               at == 0 ? p.rect[0].m1 : at == 1 ? p.rect[1].m1 : at == 2 ? p.rect[2].m1 : p.rect[3].m1,
               at == 0 ? p.rect[0].n0 : at == 1 ? p.rect[1].n0 : at == 2 ? p.rect[2].n0 : p.rect[3].n0,
               at == 0 ? p.rect[0].n1 : at == 1 ? p.rect[1].n1 : at == 2 ? p.rect[2].n1 : p.rect[3].n1};
  const int count = at == 0 ? p.count[0] : at == 1 ? p.count[1] : at == 2 ? p.count[2] : p.count[3];
  if (t >= count) return;
  if constexpr (std::is_same<T1, T2>::value)
    mx_tile<T1>(p, r, t, lds);
  else if (at < 2)
    mx_tile<T1>(p, r, t, lds);
  else
    mx_tile<T2>(p, r, t, lds);
}

// ---------------------------------------------------------------- few rows
// Order the wave's own LDS accesses (the hardware keeps them in order; this keeps the compiler to it).
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
constexpr int kFusedRows = WF_MXFP4_FUSED_ROWS;

constexpr int kRun = 2;
constexpr int kXPitch = 80;  // LDS bytes of a quantized row's 128 values (16 rows' 16-byte reads touch every bank alike)

// NB blocks of 16 rows, NC of 16 columns, W waves that share K in turns of 128 values, DEEP turns of a wave in flight; XR: the
// rows are bf16, up to 4 XR of them (0: they are codes).  OCC: waves of a SIMD that the registers are allotted for.
template <int NB, int NC, int W, int DEEP, int OCC, int XR>
__global__ __launch_bounds__(64 * W, OCC) void gemm_mxfp4_few_kernel(MxArgs p) {
  constexpr bool QUANT = XR > 0;
  static_assert(!QUANT || NB == 1, "rows quantized in the kernel: one block");
  constexpr int kPart = (W - 1) * NB * NC * 64 * 16, kX = QUANT ? W * 16 * (kXPitch + 4) : 0;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kPart > kX ? kPart : kX];
  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int n0 = static_cast<int>(blockIdx.x) * 16 * NC;
  const int steps = (p.K + 127) / 128, pa = (p.M + 15) / 16, pw = (p.N + 15) / 16;  // panels
  const auto rw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w), 0, pw * steps * 1024, kBufferRsrcWord3);
  const auto rsw = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.w_scales), 0, pw * steps * 64, kBufferRsrcWord3);
  // rows past the last are out of the buffer's range and read as zero
  const auto ra = QUANT ? __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p.x), 0, static_cast<int>(((p.M - 1) * p.ldx + p.K) * 2), kBufferRsrcWord3)
                        : __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a), 0, pa * steps * 1024, kBufferRsrcWord3);
  const auto rsa = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.a_scales), 0, QUANT ? 0 : pa * steps * 64, kBufferRsrcWord3);
  const int xrow = static_cast<int>(p.ldx) * 2;
  uint8_t* const xbuf = lds + wave * 16 * (kXPitch + 4);

  v4f acc[NB][NC];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[b][c] = v4f{0, 0, 0, 0};
  // A lane's operands of a step are 32 values, from 128 s + 32 g4 on, of column n0 + 16 c + l16 and row 16 b + l16.  bf16 rows
  // are loaded as 256 bytes of 4 rows at a time, quantized by four lanes a block, and change lanes through LDS.
  struct Regs {
    u32x4 w[NC], a[QUANT ? XR : NB];
    int sw[NC], sa[NB];
  };
  const int first = n0 / 16 * steps;  // panel
  const int row_blocks = QUANT ? 0 : NB * static_cast<int>(blockIdx.y);  // before this workgroup's
  auto load = [&](int step, Regs& r) __attribute__((always_inline)) {
    const int s = __builtin_amdgcn_readfirstlane(step);  // (in scalar registers, no vector register for each load's place)
    const bool there = s < steps;
    if constexpr (QUANT) {
      const int at = 128 * s + 8 * l16;
#pragma unroll
      for (int i = 0; i < XR; ++i) r.a[i] = __builtin_amdgcn_raw_buffer_load_b128(ra, at < p.K ? (4 * i + g4) * xrow + 2 * at : kOutOfRange, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int panel = first + c * steps + s;
      r.w[c] = __builtin_amdgcn_raw_buffer_load_b128(rw, (there ? panel * 1024 : kOutOfRange - 1024) + 16 * lane, 0, 0);
      r.sw[c] = __builtin_amdgcn_raw_buffer_load_b32(rsw, (there ? panel * 64 : kOutOfRange - 64) + 4 * l16, 0, 0);
    }
    if constexpr (!QUANT) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int panel = (row_blocks + b) * steps + s;
        r.a[b] = __builtin_amdgcn_raw_buffer_load_b128(ra, (there ? panel * 1024 : kOutOfRange - 1024) + 16 * lane, 0, 0);
        r.sa[b] = __builtin_amdgcn_raw_buffer_load_b32(rsa, (there ? panel * 64 : kOutOfRange - 64) + 4 * l16, 0, 0);
      }
    }
  };
  auto product = [&](Regs& r) __attribute__((always_inline)) {
    v4i a[NB];
    if constexpr (QUANT) {
#pragma unroll
      for (int i = 0; i < XR; ++i) {  // (what LDS holds of other rows belongs to sums that are not stored)
        const uint32_t w[4] = {r.a[i][0], r.a[i][1], r.a[i][2], r.a[i][3]};
        uint32_t top = mx::max_half(mx::max_bits2(mx::max_bits2(w[0], w[1]), mx::max_bits2(w[2], w[3])));
        top = max(top, mx::dpp_u32<0xB1>(top));
        top = max(top, mx::dpp_u32<0x4E>(top));
        const int e = mx::scale_byte(top);
        const int row = 4 * i + g4;  // (whatever the codes, a scale byte of 255 makes the sum NaN)
        *reinterpret_cast<uint32_t*>(xbuf + row * kXPitch + 4 * l16) = mx::encode8(w, mx::scale_of(e));
        xbuf[16 * kXPitch + 4 * row + (l16 >> 2)] = static_cast<uint8_t>(e);  // (the block's four lanes the same: no branch)
      }
      wave_order();
      a[0] = *reinterpret_cast<const v4i*>(xbuf + l16 * kXPitch + 16 * g4);
      r.sa[0] = xbuf[16 * kXPitch + 4 * l16 + g4];
      wave_order();
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) a[b] = __builtin_bit_cast(v4i, r.a[b]);
    }
    // (a lane's own byte of the row's word; loads of single bytes are no cheaper than of 16)
    int sw[NC], sa[NB];
#pragma unroll
    for (int c = 0; c < NC; ++c) sw[c] = static_cast<int>(static_cast<uint32_t>(r.sw[c]) >> (8 * g4));
#pragma unroll
    for (int b = 0; b < NB; ++b) sa[b] = QUANT ? r.sa[b] : static_cast<int>(static_cast<uint32_t>(r.sa[b]) >> (8 * g4));
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        acc[b][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(__builtin_bit_cast(v4i, r.w[c])), widen(a[b]), acc[b][c], 4, 4, 0,
                                                                     sw[c], 0, sa[b]);
  };
  // the wave's i-th turn: runs of kRun neighbouring steps, whose scales share a cache line
  auto step_of = [&](int i) __attribute__((always_inline)) { return (i / kRun * W + wave) * kRun + i % kRun; };
  static_assert(DEEP % kRun == 0, "whole runs in flight");
  Regs r[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) load(step_of(d), r[d]);
  // (the bias of the columns that wave 0 stores, asked for before the sums)
  uint2 bias[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int n = n0 + 16 * c + 4 * g4;
    bias[c] = make_uint2(0, 0);
    if (wave == 0 && p.bias && n < p.N) bias[c] = *reinterpret_cast<const uint2*>(p.bias + n);
  }
  for (int i = 0; step_of(i) < steps; i += DEEP) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      product(r[d]);
      __builtin_amdgcn_sched_barrier(0);  // (the loads take the registers that the product leaves)
      load(step_of(i + DEEP + d), r[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if constexpr (QUANT) __syncthreads();  // the sums take the place of the rows
  v4f* const part = reinterpret_cast<v4f*>(lds) + lane;
  if (wave) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int c = 0; c < NC; ++c) part[((wave - 1) * NB * NC + b * NC + c) * 64] = acc[b][c];
  }
  __syncthreads();
  if (wave) return;
  // wave 0 adds the others' sums, in their order, and stores
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      v4f v = acc[b][c];
#pragma unroll
      for (int i = 0; i < W - 1; ++i) v += part[(i * NB * NC + b * NC + c) * 64];
      const int m = 16 * (row_blocks + b) + l16, n = n0 + 16 * c + 4 * g4;  // rows of the first operand, 4 to a lane: columns of y
      if (m >= p.M || n >= p.N) continue;
      v[0] += bf16_lo_to_f32(bias[c].x), v[1] += bf16_hi_to_f32(bias[c].x), v[2] += bf16_lo_to_f32(bias[c].y), v[3] += bf16_hi_to_f32(bias[c].y);
      if (p.gelu) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
      }
      *reinterpret_cast<uint2*>(p.y + static_cast<int64_t>(m) * p.ldy + n) = make_uint2(pack_bf16x2_hw(v[0], v[1]), pack_bf16x2_hw(v[2], v[3]));
    }
}

constexpr int kDeep = 2;  // (3 or 4 turns in flight: 5-25 % slower at one row, even at 64)

// Columns and waves of a workgroup.  Enough columns that the rows are not read too often, enough waves that the weight is on
// its way everywhere: some 6 waves to a CU.  Columns of 32 from the width on whose workgroups of 16 columns are more than the CUs,
// so that some CU has two (us in columns of 16, of 32; 256 CUs): 16 rows x 13824 -> 4096 13.5, 16.0; -> 4608 21.8, 16.0; -> 5120 21.6, 15.7;
// 16 x 1536 -> 4096 3.8, 4.2; -> 4608 4.8, 4.4; 1 x 13824 -> 4096 9.6, 10.2; -> 4608 10.6, 10.2; -> 5120 11.6, 10.4; 1 x 1536 -> 1536 2.9, 3.2;
// -> 4608 3.4, 3.5.  At 32 columns a CU and more, 16 x 5120 -> 13824 in columns of 32 and 64: 9.9, 9.7; in 4, 8, 16 waves 1 x 5120 -> 13824
// 9.1, 9.4, 10.3; 13824 -> 5120 (columns of 16) 14.4, 10.4, 11.7.
template <int NB, int XR>
void launch_few(const MxArgs& p, hipStream_t stream) {
  auto go = [&](auto C, auto WAVES) {
    constexpr int NC = decltype(C)::value, W = decltype(WAVES)::value;
    hipLaunchKernelGGL((gemm_mxfp4_few_kernel<NB, NC, W, kDeep, 4, XR>), dim3(static_cast<uint32_t>((p.N + 16 * NC - 1) / (16 * NC)),
                       static_cast<uint32_t>((p.M + 16 * NB - 1) / (16 * NB))), dim3(64 * W), 0, stream, p);
  };
  // The waves set the order of the sums (the columns do not), so rows quantized here and quantized ones, which are to give the
  // same results, have as many: 8 for 9 to 16 rows, whichever they are (16 quantized rows in 4 and 8 waves: 5120 -> 13824 9.2,
  // 9.9 us, 5120 -> 8192 7.5, 6.7).
  const int cus = device_cus();
  const bool wide = p.N >= 32 * cus;
  if constexpr (XR == 4) {  // (the rows are quantized anew by every workgroup: 16 x 5120 -> 13824 12.9 us in columns of 32, 11.5 of 64)
    if (wide) return go(ic<4>{}, ic<8>{});
  } else {
    if (wide && (NB > 1 || p.M <= 8)) return go(ic<2>{}, ic<4>{});
  }
  if (p.N > 16 * cus)
    go(ic<2>{}, ic<8>{});
  else
    go(ic<1>{}, ic<8>{});
}

int64_t tiles_of(const Rect& r, int bm, int bn) {
  return static_cast<int64_t>((r.m1 - r.m0 + bm - 1) / bm) * ((r.n1 - r.n0 + bn - 1) / bn);
}

template <typename T1, typename T2>
void launch_tiles(MxArgs p, hipStream_t stream) {
  int64_t grid = 0;
  for (int i = 0; i < 4; ++i) {
    p.count[i] = static_cast<int>(i < 2 ? tiles_of(p.rect[i], T1::BM, T1::BN) : tiles_of(p.rect[i], T2::BM, T2::BN));
    grid += (p.count[i] + NUM_XCD - 1) / NUM_XCD * NUM_XCD;
  }
  hipLaunchKernelGGL((gemm_mxfp4_kernel<T1, T2>), dim3(static_cast<uint32_t>(grid)), dim3(T1::THREADS), 0, stream, p);
}

// What a tile costs, in us: `fixed` and `step` for each 256 values of K, with the chip's CUs all busy; `step2` where two share a
// CU.  From single launches of 128 .. 4680 rows at K = 1536, 5120, 13824 (6, 20, 54 steps), a round of tiles on all CUs: 256 x
// 256 16, 36, 80 us; 128 x 256 9, 23, 54; 128 x 128 5.8, 14.4, 33; 64 x 128 5.2, 12, 25 (two to a CU 6, 17, 45); 64 x 64 2.8,
// 8, 18 (two: 4.3, 12.5, 24-30).
struct TileCost {
  int bm, bn;
  double fixed, step, step2;
};
constexpr TileCost kCost[] = {{256, 256, 8., 1.35, 0.}, {128, 256, 3., 0.96, 0.}, {128, 128, 2.2, 0.58, 0.}, {64, 128, 2., 0.44, 0.78}, {64, 64, 1., 0.32, 0.5}};

double round_cost(const TileCost& c, int64_t tiles, int64_t steps, int64_t cus) {
  const int64_t rounds = (tiles + cus - 1) / cus;
  const double one = c.fixed + c.step * static_cast<double>(steps);
  if (c.step2 == 0.) return static_cast<double>(rounds) * one;
  return static_cast<double>(rounds / 2) * (c.fixed + c.step2 * static_cast<double>(steps)) + static_cast<double>(rounds % 2) * one;
}

// The cheapest by these figures: one tile for the whole output, or whole rounds of 256 x 256 tiles (whole tile rows, then a
// part of the next) and 128 x 256 or 128 x 128 ones over the rest, so that no round is mostly idle.  4680 x 13824 -> 5120, 380
// large tiles on 256 CUs: 178 us in them or in 740 of 128 x 256, 162 as 256 large ones and 248 (5120 -> 13824 194 and 180, -> 5120
// 78 and 70).
void launch_many(MxArgs p, hipStream_t stream) {
  const int64_t cus = device_cus(), steps = (p.K + 255) / 256;
  const Rect all{0, p.M, 0, p.N}, none{0, 0, 0, 0};
  int best = 0, rest = 0;
  int64_t big = 0;  // large tiles of a mixed plan
  double cost = 0.;
  for (int i = 0; i < 5; ++i) {
    const double c = round_cost(kCost[i], tiles_of(all, kCost[i].bm, kCost[i].bn), steps, cus);
    if (i == 0 || c < cost) {
      cost = c;
      best = i;
    }
  }
  const int64_t tn = (p.N + 255) / 256, n_big = tiles_of(all, 256, 256);
  Rect mixed[4] = {none, none, none, none};
  for (int64_t n = cus; n < n_big; n += cus) {
    const int row = static_cast<int>(n / tn) * 256, col = static_cast<int>(n % tn) * 256, next = std::min(row + 256, p.M);
    const Rect r[4] = {{0, row, 0, p.N}, col ? Rect{row, next, 0, col} : none, col ? Rect{row, next, col, p.N} : none,
                       {col ? next : row, p.M, 0, p.N}};
    for (int i = 1; i <= 2; ++i) {
      const double c = static_cast<double>(n / cus) * (kCost[0].fixed + kCost[0].step * static_cast<double>(steps)) +
                       round_cost(kCost[i], tiles_of(r[2], kCost[i].bm, kCost[i].bn) + tiles_of(r[3], kCost[i].bm, kCost[i].bn), steps, cus);
      if (c < cost) {
        cost = c;
        big = n;
        rest = i;
        std::copy(r, r + 4, mixed);
      }
    }
  }
  std::fill(p.rect, p.rect + 4, none);
  p.rect[0] = all;
  if (big) {
    std::copy(mixed, mixed + 4, p.rect);
    return rest == 1 ? launch_tiles<TileBig, TileStd>(p, stream) : launch_tiles<TileBig, TileMid>(p, stream);
  }
  switch (best) {
    case 0: return launch_tiles<TileBig, TileStd>(p, stream);
    case 1: return launch_tiles<TileStd, TileStd>(p, stream);
    case 2: return launch_tiles<TileMid, TileMid>(p, stream);
    case 3: return launch_tiles<TileHalf, TileHalf>(p, stream);
    default: return launch_tiles<TileSmall, TileSmall>(p, stream);
  }
}

int launch_gemm(const MxArgs& p, hipStream_t stream) {
  if (p.x) {
    if (p.M <= 4)
      launch_few<1, 1>(p, stream);
    else if (p.M <= 8)
      launch_few<1, 2>(p, stream);
    else
      launch_few<1, 4>(p, stream);
  } else {
    // By the output's blocks of 16 x 16: some 6 to a CU and fewer are left to waves that split K, in blocks of 32 rows where
    // there is one to a CU (us of 16 rows, 32 rows, tiles: 64 x 13824 -> 512 5.6, 6.0, 17; 200 x 13824 -> 512 7.9, 7.1, 17;
    // 200 x 5120 -> 1536 8.6, 7.9, 9.1; 300 x 5120 -> 1536 11.3, 9.7, 9.5; 100 x 5120 -> 5120 12.0, 11.1, 10.2).
    const int64_t blocks = static_cast<int64_t>((p.M + 15) / 16) * ((p.N + 15) / 16), cus = device_cus();
    if (p.M <= 16 || blocks <= cus)
      launch_few<1, 0>(p, stream);
    else if (p.M <= 32 || blocks <= 6 * cus)
      launch_few<2, 0>(p, stream);
    else
      launch_many(p, stream);
  }
  return check_launch("wf_gemm_mxfp4");
}

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Checks and arguments that both entry points share.
int make_args(const char* fn, MxArgs& p, int64_t m, int64_t n, int64_t k, const uint8_t* w, const uint8_t* w_scales, const void* bias,
              void* y, int64_t ldy, int32_t flags) {
  WF_REQUIRE(m < (1ll << 31) - 512 && n < (1ll << 31) - 512 && k < (1ll << 31) && product_below({m + 512, k / 2 + 64}, (1ll << 31) - 4096) &&
                 product_below({n + 512, k / 2 + 64}, (1ll << 31) - 4096),
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
    WF_REQUIRE(ldx < (1 << 26), WF_E_SHAPE, "%s: a row stride of %lld elements", fn, (long long)ldx);  // (offsets of 16 rows in 32 bits)
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
