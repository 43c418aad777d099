// Attention of up to 16 query rows over dense fp16 / bf16 K/V rows of 128
// channels, 16 NB tokens (NB even) a step of one wave, in registers alone (gfx950):
//   * scores S^T = K . Q^T on v_mfma_f32_16x16x32: 16 tokens a block, the A
//     operand (lane (q, n) = (lane / 16, lane % 16): 8 channels of token n) as
//     it lies in memory;
//   * result lane (q, r) holds tokens 4q .. 4q + 3 of row r, which is the B
//     operand of P^T over two blocks (k slots 4e + i of lane q: token 4q + i of
//     block e): softmax in base 2, P rounded in place to the 16-bit type, in
//     fp16 times 2^15 (weights down to 2^-29 of the largest keep all their bits);
//   * O^T += V^T . P^T: lane (q, n) loads channels 8n .. 8n + 7 of tokens 4q + i,
//     whose 8 x 4 block, transposed in registers, is the A operand of channels
//     8n + c (c < 8): row m of product c is channel 8m + c.
// A hidden token's value takes no part: those at or past n_valid are taken as
// 0, and where rows see different tokens (mixed) values that are not finite are
// too, and added afterwards to the rows that see them.
#pragma once

#include "bmx_prefill.h"
#include "k2b_common.h"

#include <cmath>

namespace bmx {

constexpr int kRwD = 128;
constexpr int kRwPitch = kRwD + 4;  // floats of a partial: sums, m, l

template <int DT>
__device__ __forceinline__ float4_t rw_mma(u32x4_t a, u32x4_t b, float4_t c) {
  if constexpr (DT == BMX_PREFILL_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                  0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t rw_pack2(float x, float y) {
  if constexpr (DT == BMX_PREFILL_F16) {
    const half2_t h = {(_Float16)x, (_Float16)y};
    return as_u32(h);
  } else {
    typedef __bf16 bf2_t __attribute__((ext_vector_type(2)));
    const bf2_t b = {(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, b);
  }
}
template <int DT>
__device__ __forceinline__ uint16_t rw_pack(float x) {
  return (uint16_t)rw_pack2<DT>(x, 0.f);
}
template <int DT>
__device__ __forceinline__ float rw_elem(uint16_t b) {
  if constexpr (DT == BMX_PREFILL_F16) return half_bits_to_float(b);
  return __uint_as_float((uint32_t)b << 16);
}
// nonzero if one of the two values of x is infinite or NaN (its exponent, all
// ones, carries into its sign bit)
template <int DT>
__device__ __forceinline__ uint32_t rw_nonfinite(uint32_t x) {
  constexpr uint32_t e = DT == BMX_PREFILL_F16 ? 0x7c007c00u : 0x7f807f80u;
  constexpr uint32_t one = DT == BMX_PREFILL_F16 ? 0x04000400u : 0x00800080u;
  return ((x & e) + one) & 0x80008000u;
}

// A wave's running softmax and sums of the lane's row n.
struct RowsState {
  float4_t o[8];   // O^T: o[c][i] = channel 8 (4q + i) + c of row n
  float m, l;      // maximum (base 2, unlifted) and the lane's share of the lifted sum
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = float4_t{0.f, 0.f, 0.f, 0.f};
    m = -INFINITY;
    l = 0.f;
  }
};

// One step of 16 NB tokens: kr[j][dc] = channels 32 dc + 8q .. + 7 of token 16j + n,
// vr[j][i] = channels 8n .. 8n + 7 of token 16j + 4q + i; sees(t): token t is
// visible to the lane's row (whole: all tokens to all rows); value(t): its
// value row.
template <int DT, int NB, class See, class Value>
__device__ __forceinline__ void rows_step(RowsState& st, const u32x4_t (&kr)[NB][4], u32x4_t (&vr)[NB][4],
                                          const u32x4_t (&qb)[4], float qscale, bool whole, bool mixed, int n_valid,
                                          See sees, Value value) {
  constexpr float kLift = DT == BMX_PREFILL_F16 ? 15.f : 0.f;
  const int q = (threadIdx.x & 63) >> 4;
  float4_t s[NB];
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    s[j] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) s[j] = rw_mma<DT>(kr[j][dc], qb[dc], s[j]);
    if (!whole)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!sees(16 * j + 4 * q + i)) s[j][i] = -INFINITY;
    mx = fmaxf(mx, fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])));
  }
  mx = fmaxf(mx, __shfl_xor(mx, 16));
  mx = fmaxf(mx, __shfl_xor(mx, 32));
  const float mn = fmaxf(st.m, mx * qscale);
  const float mu = mn == -INFINITY ? 0.f : mn;   // nothing seen yet
  const float al = __builtin_amdgcn_exp2f(st.m - mu);
  st.m = mn;
  st.l *= al;
#pragma unroll
  for (int c = 0; c < 8; ++c) st.o[c] *= al;
  uint32_t pb[NB][2];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][i], qscale, kLift - mu));
      st.l += p[i];
    }
    pb[j][0] = rw_pack2<DT>(p[0], p[1]);
    pb[j][1] = rw_pack2<DT>(p[2], p[3]);
  }
  bool bad = false;
  if (!whole) {
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (16 * j + 4 * q + i >= n_valid) vr[j][i] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= rw_nonfinite<DT>(vr[j][i][e]);
      }
    bad = mixed && __any(any != 0);
    if (bad) {
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) vr[j][i][e] &= ~((rw_nonfinite<DT>(vr[j][i][e]) >> 15) * 0xffffu);
    }
  }
#pragma unroll
  for (int u = 0; u < NB / 2; ++u) {   // blocks 2u, 2u + 1
    const u32x4_t pv = {pb[2 * u][0], pb[2 * u][1], pb[2 * u + 1][0], pb[2 * u + 1][1]};
#pragma unroll
    for (int e = 0; e < 4; ++e) {   // channels 2e, 2e + 1 of the lane's 8
      u32x4_t lo, hi;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4_t(&w)[4] = vr[2 * u + j];
        lo[2 * j] = __builtin_amdgcn_perm(w[1][e], w[0][e], 0x05040100u);
        lo[2 * j + 1] = __builtin_amdgcn_perm(w[3][e], w[2][e], 0x05040100u);
        hi[2 * j] = __builtin_amdgcn_perm(w[1][e], w[0][e], 0x07060302u);
        hi[2 * j + 1] = __builtin_amdgcn_perm(w[3][e], w[2][e], 0x07060302u);
      }
      st.o[2 * e] = rw_mma<DT>(lo, pv, st.o[2 * e]);
      st.o[2 * e + 1] = rw_mma<DT>(hi, pv, st.o[2 * e + 1]);
    }
  }
  if (bad) {   // rare: whatever weight a row gives such a value, its sum is that value's
#pragma unroll 1
    for (int t = 0; t < 16 * NB; ++t) {
      if (!sees(t)) continue;
      const uint16_t* vp = value(t) + 32 * q;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float x = rw_elem<DT>(vp[8 * i + c]);
          if (!(__builtin_fabsf(x) < INFINITY)) st.o[c][i] += x;
        }
    }
  }
}

// The wave's partial of row n (keep: a row that exists) to dst: 128 sums, m, l.
__device__ __forceinline__ void rows_store(RowsState& st, bool keep, float* dst) {
  const int q = (threadIdx.x & 63) >> 4;
  st.l += __shfl_xor(st.l, 16);
  st.l += __shfl_xor(st.l, 32);
  if (!keep) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    *reinterpret_cast<float4_t*>(dst + 32 * q + 8 * i) = float4_t{st.o[0][i], st.o[1][i], st.o[2][i], st.o[3][i]};
    *reinterpret_cast<float4_t*>(dst + 32 * q + 8 * i + 4) = float4_t{st.o[4][i], st.o[5][i], st.o[6][i], st.o[7][i]};
  }
  if (q == 0) *reinterpret_cast<float2*>(dst + kRwD) = make_float2(st.m, st.l);
}

}  // namespace bmx
