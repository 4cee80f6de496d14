// Batched attention, few rows: up to 64 (row, head) rows of a sequence over one key head (single tokens, a few drafted
// ones, grouped heads).  The cache is read once and little is computed, so HBM bounds it: 264 bytes a key of an 8-bit
// cache, 512 of a dense one.
//
// A workgroup of four waves owns a tile of 16, 32 or 64 rows, one key head and one range of the keys; every wave takes
// each fourth tile of 32 keys of the range by itself (no barrier in the loop) with the loads of its next tile in
// flight, and the four results are joined in LDS at the end, those of several ranges by the join kernel.
//
// Per 32 keys: K comes straight from memory as the first operand of v_mfma_f32_16x16x32_bf16 (lane (l, g) holds key l,
// codes 64 i + 16 g .. + 15 of its row; Q, the second operand, is held in the same order), so S^T = K Q^T leaves a lane
// with one row and the keys 16 b + 4 g + 0..3.  V goes through a wave's own LDS rows, whose transposing reads give the
// V^T operand of O^T += V^T P^T for the same keys.  The codes of both formats are exact in bf16 (4 and 8 significant
// bits) and so are the products: the scales are applied in fp32, s_k c to the scores and s_v to the weights, and the
// weights go in as the sum of two bf16 (16 significant bits; the matrix cores are idle most of the time anyway).
#include "attn_batch.hpp"

namespace wf {
namespace attn_batch {
namespace {

constexpr int KT = 32;       // keys of a wave's tile
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kOPitch = D + 4;  // floats of a joined row in LDS

template <int SRC>
struct Form {
  static constexpr bool dense = SRC == SRC_DENSE;
  static constexpr int row_bytes = dense ? 256 : 128;
  static constexpr int k_loads = 2 * row_bytes / 64;   // 16-byte loads a lane makes of the tile's K (and V)
  static constexpr int v_pitch = dense ? 256 + 32 : 128 + 16;
  static constexpr int wave_lds = KT * v_pitch + 64 * 4;  // V rows, then 32 factors of K and 32 of V
};

// 8 codes (2 dwords) as 8 bf16.
template <int SRC>
__device__ inline v8bf to_bf16(uint32_t w0, uint32_t w1) {
  uint32_t o[4];
  if constexpr (SRC == SRC_E4M3) {
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, 1.0f, true));
  } else {
    const uint32_t w[2] = {w0, w1};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      o[2 * i] = cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w[i])), static_cast<float>(static_cast<int8_t>(w[i] >> 8)));
      o[2 * i + 1] = cvt_bf16x2(static_cast<float>(static_cast<int8_t>(w[i] >> 16)),
                                static_cast<float>(static_cast<int8_t>(w[i] >> 24)));
    }
  }
  return __builtin_bit_cast(v8bf, make_uint4(o[0], o[1], o[2], o[3]));
}

// Order the wave's own LDS accesses (the hardware keeps them in order; this keeps the compiler to it).
__device__ inline void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int SRC, int NB>
__global__ __launch_bounds__(kThreads) void attn_few_kernel(Args a) {
  using F = Form<SRC>;
  constexpr bool kDense = F::dense;
  constexpr int R = 16 * NB;
  constexpr int kStage = kWaves * F::wave_lds;
  constexpr int kJoin = R * kOPitch * 4 + 2 * kWaves * R * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kStage > kJoin ? kStage : kJoin];

  const int lane = static_cast<int>(threadIdx.x) & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int split = static_cast<int>(blockIdx.x) % a.n_splits;
  const int item = static_cast<int>(blockIdx.x) / a.n_splits;
  const int head = item % a.n_kv_heads, w = item / a.n_kv_heads;
  Tile t;
  if (!find_tile<kDense>(a, w, t)) return;
  const int lim_max = tile_max(a, t), lim_min = tile_min(a, t);
  const int splits = used_splits(a, lim_max);
  if (split >= splits) return;
  const int k_lo = split * a.split_keys;
  const int k_hi = split == splits - 1 ? lim_max : k_lo + a.split_keys;

  // rows: the lane's row of each 16, its query and its limit
  v8bf qf[NB][4];
  int lim[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int r = t.first + 16 * n + l16;
    const bool ok = r < t.count;
    uint32_t qi, gi;
    a.group_div.divmod(static_cast<uint32_t>(ok ? r : t.first), qi, gi);
    lim[n] = ok ? row_limit(a, t, static_cast<int>(qi)) : 0;
    const uint16_t* p = a.q + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldq + (head * a.group + static_cast<int>(gi)) * D;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      // step s of the product takes values 64 (s / 2) + 16 g + 8 (s % 2) .. + 7 (dense: 32 s + 8 g .. + 7) of a key's row
      const int d = kDense ? 32 * s + 8 * g4 : 64 * (s >> 1) + 16 * g4 + 8 * (s & 1);
      const uint4 v = *reinterpret_cast<const uint4*>(p + d);
      qf[n][s] = __builtin_bit_cast(v8bf, ok ? v : make_uint4(0, 0, 0, 0));
    }
  }

  v4f o[NB][8];
  float m[NB], l[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[n][i] = v4f{0, 0, 0, 0};
  }

  uint8_t* vbuf = lds + wave * F::wave_lds;
  float* fbuf = reinterpret_cast<float*>(vbuf + KT * F::v_pitch);

  // one tile in registers: K rows, V rows, factors (lane < 32: s_k of key lane, else s_v of key lane - 32), and which of
  // its keys have no place to be read from
  struct Regs {
    u32x4 k[F::k_loads], v[F::k_loads];
    float f;
    uint32_t bad;
  };
  // Where the keys of the tile at key t0 live: lane & 31's (position, head) row in the pool (dense: its row of k) and its
  // scale; keys past the range or without a page are not there.
  struct Place {
    int row, scale;
    bool there;
  };
  auto locate = [&](int t0) -> Place {
    const int j = t0 + (lane & 31);
    Place p{kDense ? t.key0 : 0, 0, false};
    if (j >= k_hi) return p;
    if constexpr (kDense) {
      p = Place{t.key0 + j, 0, true};
    } else {
      int page, at;
      if (pool_row(a.geom, t.b, j, page, at))
        p = Place{(page * a.geom.page_tokens + at) * a.n_kv_heads + head, (page * a.n_kv_heads + head) * a.geom.page_tokens + at, true};
    }
    return p;
  };
  auto load = [&](const Place& p, Regs& x) {
    x.bad = static_cast<uint32_t>(__ballot(!p.there));
    const int safe = p.row;
    if constexpr (kDense) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint16_t* kp = a.k_dense + static_cast<int64_t>(__shfl(safe, 16 * b + l16)) * a.ldkv + head * D + 8 * g4;
#pragma unroll
        for (int i = 0; i < 4; ++i) x.k[4 * b + i] = *reinterpret_cast<const u32x4*>(kp + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t* vp = a.v_dense + static_cast<int64_t>(__shfl(safe, 4 * i + (lane >> 4))) * a.ldkv + head * D + 8 * l16;
        x.v[i] = *reinterpret_cast<const u32x4*>(vp);
      }
    } else {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint8_t* kp = a.k_codes + static_cast<int64_t>(__shfl(safe, 16 * b + l16)) * D + 16 * g4;
        x.k[2 * b] = *reinterpret_cast<const u32x4*>(kp);
        x.k[2 * b + 1] = *reinterpret_cast<const u32x4*>(kp + 64);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* vp = a.v_codes + static_cast<int64_t>(__shfl(safe, 8 * i + (lane >> 3))) * D + 16 * (lane & 7);
        x.v[i] = *reinterpret_cast<const u32x4*>(vp);
      }
      x.f = (lane < 32 ? a.k_scales : a.v_scales)[p.scale];
    }
  };

  auto compute = [&](int t0, Regs& x) {
    if (x.bad) {  // keys past the range or without a page: zero K and V
      const u32x4 zero = {0, 0, 0, 0};
      constexpr int per = F::k_loads / 2;
#pragma unroll
      for (int i = 0; i < F::k_loads; ++i) {
        if (x.bad >> (16 * (i / per) + l16) & 1u) x.k[i] = zero;
        if (x.bad >> (kDense ? 4 * i + (lane >> 4) : 8 * i + (lane >> 3)) & 1u) x.v[i] = zero;
      }
      if (x.bad >> (lane & 31) & 1u) x.f = 0.f;
    }
    const bool masked = t0 + KT > lim_min;
    if constexpr (kDense) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<u32x4*>(vbuf + (4 * i + (lane >> 4)) * F::v_pitch + 16 * l16) = x.v[i];
    } else {
      if (lane < 32) x.f *= a.c;
      fbuf[lane] = x.f;
      if (SRC == SRC_E4M3 && masked) {
        // A weight of zero does not silence a NaN of V: where some row does not see some key, a NaN code becomes a NaN
        // scale, which only the weights of rows that see the key meet.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool nan = has_nan_code(x.v[i][0]) || has_nan_code(x.v[i][1]) || has_nan_code(x.v[i][2]) || has_nan_code(x.v[i][3]);
          const uint64_t any = __ballot(nan);
          if (any) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x.v[i][e] = without_nan_codes(x.v[i][e]);
            wave_lds_order();
            if ((lane & 7) == 0 && (any >> lane & 0xffu)) fbuf[32 + 8 * i + (lane >> 3)] = bits_f32(0x7fc00000u);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4*>(vbuf + (8 * i + (lane >> 3)) * F::v_pitch + 16 * (lane & 7)) = x.v[i];
    }
    wave_lds_order();
    v4f s[NB][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n][b] = v4f{0, 0, 0, 0};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        v8bf kf;
        if constexpr (kDense) {
          kf = __builtin_bit_cast(v8bf, x.k[4 * b + ks]);
        } else {
          const u32x4 kk = x.k[2 * b + (ks >> 1)];
          kf = to_bf16<SRC>(kk[2 * (ks & 1)], kk[2 * (ks & 1) + 1]);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][ks], s[n][b], 0, 0, 0);
      }
    }
    float u[8], sv[8];
    if constexpr (!kDense) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float4 fu = *reinterpret_cast<const float4*>(fbuf + 16 * b + 4 * g4);
        const float4 fv = *reinterpret_cast<const float4*>(fbuf + 32 + 16 * b + 4 * g4);
        u[4 * b] = fu.x, u[4 * b + 1] = fu.y, u[4 * b + 2] = fu.z, u[4 * b + 3] = fu.w;
        sv[4 * b] = fv.x, sv[4 * b + 1] = fv.y, sv[4 * b + 2] = fv.z, sv[4 * b + 3] = fv.w;
      }
    }
    v8bf ph[NB], pl[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float x8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x8[e] = s[n][e >> 2][e & 3] * (kDense ? a.c : u[e]);
      if (masked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (t0 + 16 * (e >> 2) + 4 * g4 + (e & 3) >= lim[n]) x8[e] = -INFINITY;
      }
      float mt = fmaxf(fmaxf(fmaxf(x8[0], x8[1]), fmaxf(x8[2], x8[3])), fmaxf(fmaxf(x8[4], x8[5]), fmaxf(x8[6], x8[7])));
      mt = max16(max32(mt));
      const bool fire = mt > m[n] + kTau;
      if (__ballot(fire)) {
        const float m_new = fire ? mt : m[n];
        const float alpha = fire ? (m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - m_new)) : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[n][i] *= alpha;
        l[n] *= alpha;
        m[n] = m_new;
      }
      const float neg = m[n] == -INFINITY ? 0.f : -m[n];
      float hi[8], lo[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = __builtin_amdgcn_exp2f(x8[e] + neg);
        l[n] += p;
        float wgt = p;
        if constexpr (!kDense) {
          wgt = p * sv[e];
          if (masked && x8[e] == -INFINITY) wgt = 0.f;
        }
        hi[e] = wgt;
      }
      uint32_t wh[4], wl[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wh[e] = cvt_bf16x2(hi[2 * e], hi[2 * e + 1]);
        lo[2 * e] = hi[2 * e] - bf16_lo_to_f32(wh[e]);
        lo[2 * e + 1] = hi[2 * e + 1] - bf16_hi_to_f32(wh[e]);
        wl[e] = cvt_bf16x2(lo[2 * e], lo[2 * e + 1]);
      }
      ph[n] = __builtin_bit_cast(v8bf, make_uint4(wh[0], wh[1], wh[2], wh[3]));
      pl[n] = __builtin_bit_cast(v8bf, make_uint4(wl[0], wl[1], wl[2], wl[3]));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v8bf vf;
      if constexpr (kDense) {
        const uint8_t* p = vbuf + (4 * g4 + (l16 >> 2)) * F::v_pitch + (16 * i + 4 * (l16 & 3)) * 2;
        vf = __builtin_bit_cast(v8bf, __builtin_shufflevector(read_tr16(p), read_tr16(p + 16 * F::v_pitch), 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        const int j = l16 >> 1;
        const v2i c = read_tr8(vbuf + (16 * (j >> 2) + 4 * g4 + (j & 3)) * F::v_pitch + 16 * i + 8 * (l16 & 1));
        vf = to_bf16<SRC>(static_cast<uint32_t>(c[0]), static_cast<uint32_t>(c[1]));
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph[n], o[n][i], 0, 0, 0);
        o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[n], o[n][i], 0, 0, 0);
      }
    }
    wave_lds_order();
  };

  int t0 = k_lo + KT * wave;
  if (t0 < k_hi) {
    Regs cur, nxt;
    load(locate(t0), cur);
    Place next = locate(t0 + kWaves * KT);
    for (; t0 < k_hi; t0 += kWaves * KT) {
      if (t0 + kWaves * KT < k_hi) {
        load(next, nxt);
        next = locate(t0 + 2 * kWaves * KT);
      }
      compute(t0, cur);
      cur = nxt;
    }
  }

  // join the four waves: their maxima and sums, then the outputs one wave after the other
  __syncthreads();
  float* ob = reinterpret_cast<float*>(lds);
  float* ms = ob + R * kOPitch;
  float* ls = ms + kWaves * R;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] = sum16(sum32(l[n]));
    if (g4 == 0) {
      ms[wave * R + 16 * n + l16] = m[n];
      ls[wave * R + 16 * n + l16] = l[n];
    }
  }
  __syncthreads();
  float scale[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, ms[i * R + 16 * n + l16]);
    scale[n] = m[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[n] - top);
  }
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          v4f* p = reinterpret_cast<v4f*>(ob + (16 * n + l16) * kOPitch + 16 * d + 4 * g4);
          const v4f v = o[n][d] * scale[n];
          *p = i == 0 ? v : *p + v;
        }
    }
    __syncthreads();
  }
  for (int c = static_cast<int>(threadIdx.x); c < R * 16; c += kThreads) {
    const int r = c >> 4, d = 8 * (c & 15);
    if (t.first + r >= t.count) continue;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = fmaxf(top, ms[i * R + r]);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) sum += ms[i * R + r] == -INFINITY ? 0.f : ls[i * R + r] * __builtin_amdgcn_exp2f(ms[i * R + r] - top);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const float* v = ob + r * kOPitch + d;
    if (splits > 1) {
      const int64_t at = (static_cast<int64_t>(item) * a.n_splits + split) * R + r;
      float4* po = reinterpret_cast<float4*>(a.part_o + at * D + d);
      po[0] = make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
      po[1] = make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top, sum);
    } else {
      uint32_t qi, gi;
      a.group_div.divmod(static_cast<uint32_t>(t.first + r), qi, gi);
      uint16_t* p = a.out + static_cast<int64_t>(t.row0 + static_cast<int>(qi)) * a.ldo + (head * a.group + static_cast<int>(gi)) * D + d;
      *reinterpret_cast<uint2*>(p) = make_uint2(cvt_bf16x2(v[0] * inv, v[1] * inv), cvt_bf16x2(v[2] * inv, v[3] * inv));
      *reinterpret_cast<uint2*>(p + 4) = make_uint2(cvt_bf16x2(v[4] * inv, v[5] * inv), cvt_bf16x2(v[6] * inv, v[7] * inv));
    }
  }
}

template <int SRC>
void launch(const Args& a, int row_blocks, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.n_tiles) * a.n_kv_heads * a.n_splits);
  switch (row_blocks) {
    case 1: hipLaunchKernelGGL((attn_few_kernel<SRC, 1>), grid, dim3(kThreads), 0, stream, a); break;
    case 2: hipLaunchKernelGGL((attn_few_kernel<SRC, 2>), grid, dim3(kThreads), 0, stream, a); break;
    default: hipLaunchKernelGGL((attn_few_kernel<SRC, 4>), grid, dim3(kThreads), 0, stream, a); break;
  }
}

}  // namespace

int launch_few(const Args& a, int src, int row_blocks, hipStream_t stream) {
  switch (src) {
    case SRC_E4M3: launch<SRC_E4M3>(a, row_blocks, stream); break;
    case SRC_INT8: launch<SRC_INT8>(a, row_blocks, stream); break;
    default: launch<SRC_DENSE>(a, row_blocks, stream); break;
  }
  return check_launch("wf_attn_batch (few rows)");
}

}  // namespace attn_batch
}  // namespace wf
