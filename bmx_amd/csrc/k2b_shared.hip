// Shared-prefix decode over packed k2b pages (gfx950): one query step of a
// batch whose sequences share their first pages.  k2b_decode_split_kernel
// rebuilds a page once per sequence; here a rebuilt page meets the query rows
// of the whole batch, B * G rows of a KV head, as one matrix product.
//
// shared_kernel<R, NR, DT>: workgroups of 8 waves, of three kinds by block index:
//   * prefix: (split, KV head, block of 16 NR rows);
//   * own: (split, KV head, sequence): the sequence's pages past the prefix, the
//     same code with the head's G rows (NR 1);
//   * window: (KV head, sequence): the dense recent rows (dense_rows.h).
// A packed workgroup walks its pages 8 at a time (a tile of 128 tokens), one page a
// wave up to the weights, one 16-channel block a wave from there:
//   * keys: K_pre^T = V_h Us^T on v_mfma_f32_16x16x32 (channels x tokens), then
//     residual * scale and rotation; lane (q, n) then holds token n, pairs
//     (j, j + 64), j = 16b + 4q + i: the A operand of the scores S^T = K . Q^T,
//     with Q in LDS in the same channel order;
//   * scores: lane (q, r) holds tokens 4q .. 4q + 3 of row r;
//   * weights: p = 2^(s - c), x = p norm in fp16, l = sum p in fp32, with one
//     offset c a row.  c follows the largest p norm, not the largest p (a sink
//     with a value near 0 would otherwise leave the other weights no bits), and
//     keeps p below 2^100: it moves only when some x would pass fp16's range or
//     p that bound (the tile's weights are then taken again by all waves), so
//     the exponential is taken once and sums are seldom rescaled;
//   * x goes through LDS as the B operand of the values' product (k slots 8q + 4e
//     + t: token 4q + t of page e of a pair), the pages' code bytes too; a wave
//     adds its block of rotated channels, O^T += level . x, over all 8 pages, the
//     levels of a code byte's 4 tokens by one 8-byte table read (fp16 levels as an
//     affine image of the codebook: level_map()).
// With the sums spread over the waves by channels a wave keeps 4 NR registers of
// them, and 128 registers in all let two workgroups share a CU (a form with a
// wave's own tiles and all channels kept 32 NR, spilled, and took 177 us where
// this took 65, at 64k tokens and 16 sequences of up to 1,024 more).  One barrier a tile:
// both buffers in LDS are double, and the values of a tile are added during the
// keys and scores of the next (their products and table reads fill the gaps of
// its vector work).
// Rounded to 16 bits: x, Q when bf16 (by a power of two), and K when bf16.  With
// fp16 queries a rebuilt key stays in two fp16 parts, each with a score product:
// one part left the output 2.4 times as far from 64-bit values as its own rounding
// does (rms), two leave 1.4 times, for 10% of the time.  The rotations come in
// 16-bit fixed point, as wide as fp16 and 16 times as close.  Every sum, c and l
// are fp32.
// Vector instructions bound it: at 64k tokens and 16 sequences (73 us) they are
// active in 71% of the cycles, matrix products in 24%, LDS in 38%.
// A workgroup leaves one fp32 partial a row, and shared_merge_kernel joins a row's
// partials, un-rotates the packed ones (H128, signs) and adds the window's.

#include "dense_rows.h"
#include "k2b_common.h"
#include "k2b_general.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace bmx {
namespace {

constexpr int kShWaves = 8;
constexpr int kShThreads = 64 * kShWaves;
constexpr int kShPitch = kD + 4;              // floats of a partial: sums, c, l, w
constexpr int kShBufWord3 = 0x00020000;       // buffer descriptor word 3: raw 32-bit data
constexpr int kShRope = BMX_K2B_ROPE_PAGE_BYTES;

struct SharedArgs {
  int h_kv, G, B, rows;            // rows = B * G
  int n_prefix, n_own;             // workgroups of each kind (the windows' follow)
  int pre_splits, own_splits, row_blocks, n_slots;
  int pre_groups;                  // 64-token groups of the prefix
  int shared_len, max_len, max_pages, n_pool, n_rope;
  int tail_cap, tail_len_value;
  PageLayout L;
  float qscale;                    // sm_scale * log2(e); the packed keys' also times rope_scaling
  float qscale_rope;
  uint32_t level_hi[4];
  float level_mu;
  const void* q;
  const uint8_t* pages;
  const int32_t* page_table;
  const int32_t* packed_len;
  const uint16_t* basis;
  const uint8_t* rope;
  const uint16_t* k_tail;
  const uint16_t* v_tail;
  int64_t ts_b, ts_h, ts_t;
  const int32_t* tail_len;
  float* part;                     // [B][h_kv][G][n_slots][kShPitch]
};

// One key pair (j, j + 64): low-rank part plus residual code times scale, rotated,
// (k_j c - k_{j+64} s, k_{j+64} c + k_j s) in fp32 with c, s times kRopeOne, as
// fp16 k and, where kLow, the fp16 rest (together 2^-22 of a key)
constexpr float kRopeOne = 32767.0f;   // 1 in the rotation table's 16-bit fixed point
template <bool kLow>
__device__ __forceinline__ void key_pair(float lo, float hi, half2_t code, half2_t scale, uint32_t cs, half2_t& k,
                                         half2_t& low) {
  const float a = __builtin_fmaf((float)code[0], (float)scale[0], lo);
  const float b = __builtin_fmaf((float)code[1], (float)scale[1], hi);
  const float c = (float)(int16_t)(cs & 0xffff), s = (float)(int16_t)(cs >> 16);
  const float u = __builtin_fmaf(-b, s, a * c), v = __builtin_fmaf(a, s, b * c), unit = 1.0f / kRopeOne;
  // one instruction a half: the product with 1 / kRopeOne, rounded, then what that left
  uint32_t d;
  asm("v_fma_mixlo_f16 %0, %1, %3, 0\n\tv_fma_mixhi_f16 %0, %2, %3, 0" : "=&v"(d) : "v"(u), "v"(v), "s"(unit));
  k = as_h2(d);
  if constexpr (kLow) {
    uint32_t e;
    asm("v_fma_mixlo_f16 %0, %2, %4, -%1 op_sel_hi:[0,0,1]\n\t"
        "v_fma_mixhi_f16 %0, %3, %4, -%1 op_sel:[0,0,1] op_sel_hi:[0,0,1]"
        : "=&v"(e)
        : "v"(d), "v"(u), "v"(v), "s"(unit));
    low = as_h2(e);
  }
}

constexpr int kTilePages = kShWaves;   // a page a wave

// LDS of a packed workgroup: two workgroups a CU fit.
template <int R, int NR>
struct ShLds {
  static constexpr int kVlut = 0;                               // 256 x 4 levels
  static constexpr int kBasis = kVlut + 256 * 8;                // [8 channel blocks][64 lanes] x R / 4 halfs
  static constexpr int kQ = kBasis + 8 * 64 * (R / 2);          // [NR][4 slices][64 lanes] x 16 B
  static constexpr int kX = kQ + NR * 4 * 64 * 16;              // [2][4 page pairs][NR][64 lanes] x 16 B
  static constexpr int kV = kX + 2 * 4 * NR * 64 * 16;          // [2][8 pages][64 lanes] x 8 B of codes
  static constexpr int kTo = kV + 2 * kTilePages * 64 * 8;      // [8 waves][16 NR rows] offsets asked for
  static constexpr int kLim = kTo + kShWaves * 16 * NR * 4;     // [16 NR] tokens a row sees
  static constexpr int kScale = kLim + 16 * NR * 4;             // [8 waves][64] scale pairs
  static constexpr int kFlag = kScale + kShWaves * 64 * 4;      // [2]
  static constexpr int kBytes = kFlag + 16;
};

// The packed part of a workgroup: rows row0 .. row0 + 16 NR - 1 of head h (a row
// is a (sequence, head of the group) pair b * G + g, those up to n_rows exist),
// 64-token groups g0 .. g1 of the sequence whose table row is ptab; a row sees
// the groups that end within limit(row) tokens.
template <int R, int NR, int DT, class Limit>
__device__ __forceinline__ void packed_rows(const SharedArgs& a, uint8_t* smem, int h, int row0, int n_rows,
                                            const int32_t* ptab, int g0, int g1, int slot, Limit limit) {
  constexpr int KQ = R / 4;   // rank elements of a lane in the key product
  typedef _Float16 hvec_t __attribute__((ext_vector_type(KQ)));
  constexpr bool kLow = DT == BMX_PREFILL_F16;   // keys in two fp16 parts (bf16's own rounding hides the second)
  using Lds = ShLds<R, NR>;
  uint2* vlut = reinterpret_cast<uint2*>(smem + Lds::kVlut);
  hvec_t* s_basis = reinterpret_cast<hvec_t*>(smem + Lds::kBasis);
  uint4* s_q = reinterpret_cast<uint4*>(smem + Lds::kQ);
  uint8_t* s_x = smem + Lds::kX;
  uint8_t* s_v = smem + Lds::kV;
  float* s_to = reinterpret_cast<float*>(smem + Lds::kTo);
  int* s_lim = reinterpret_cast<int*>(smem + Lds::kLim);
  uint32_t* s_scale = reinterpret_cast<uint32_t*>(smem + Lds::kScale);
  int* s_flag = reinterpret_cast<int*>(smem + Lds::kFlag);
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, n = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  g0 = __builtin_amdgcn_readfirstlane(g0);
  g1 = __builtin_amdgcn_readfirstlane(g1);
  const int n_pages = 4 * (g1 - g0), n_tiles = (n_pages + kTilePages - 1) / kTilePages;

  // ---- the group that holds the wave's page of tile t (the table read as scalar
  // loads): the page is its wave % 4; pages past the range read the last group
  typedef const int32_t __attribute__((address_space(4))) ctable;
  const int sub = wave & 3;
  struct Group {
    int id0, id1, id2, id3;   // its pages
    int own;                  // the wave's
    int first;                // entry of the first
  };
  auto find_group = [&](int t) {
    Group r;
    r.first = 4 * g0 + (min(kTilePages * t + wave, n_pages - 1) & ~3);
    ctable* src = (ctable*)(ptab + r.first);
    r.id0 = src[0];
    r.id1 = src[1];
    r.id2 = src[2];
    r.id3 = src[3];
    r.own = src[sub];
    return r;
  };
  Group now{}, next{};
  if (n_tiles > 0) {
    now = find_group(0);
    next = find_group(1);
  }

  // ---- operands
  if (tid < 256) {
    const uint32_t l0 = a.level_hi[0], l1 = a.level_hi[1], l2 = a.level_hi[2], l3 = a.level_hi[3];
    auto lv = [&](int c) { return c == 0 ? l0 : c == 1 ? l1 : c == 2 ? l2 : l3; };
    vlut[tid] = make_uint2(lv(tid & 3) | (lv((tid >> 2) & 3) << 16), lv((tid >> 4) & 3) | (lv(tid >> 6) << 16));
  }
  if (tid < 2) s_flag[tid] = 0;
  s_basis[wave * 64 + lane] = *reinterpret_cast<const hvec_t*>(a.basis + (int64_t)(h * kD + 16 * wave + n) * R + KQ * q);
  // queries as the scores' B operand: half 2 i + e of lane (q, row) in slice bb is
  // channel 16 bb + 4q + i + 64 e.  A lane loads the 32 channels of one row of a
  // row block (NR 4: two waves share a block's slices)
  constexpr int kPer = kShWaves / NR, kBb = kPer >= 4 ? 1 : 4 / kPer;   // waves of a row block, slices of a wave
  float c[NR], l[NR], w[NR];
  const uint16_t* qbase = static_cast<const uint16_t*>(a.q);
  auto row_at = [&](int row, int& b) {   // its query, and its sequence
    b = row / a.G;
    return qbase + (((int64_t)b * a.h_kv + h) * a.G + (row - b * a.G)) * kD;
  };
  const int rb_q = wave / kPer;
  uint2 qr[8];   // channels 16 (i % 4) + 4q .. + 3, + 64 (i / 4)
  {
    int b;
    const uint16_t* qp = row_at(min(row0 + 16 * rb_q + n, n_rows - 1), b);
#pragma unroll
    for (int i = 0; i < 8; ++i) qr[i] = *reinterpret_cast<const uint2*>(qp + 16 * (i & 3) + 4 * q + 64 * (i >> 2));
  }
  float qs = a.qscale_rope;   // what a score is multiplied by
  if constexpr (DT == BMX_PREFILL_BF16) {
    // bf16 to fp16: all rows times one power of two that brings the largest size
    // to 2^13 (sizes of 2^-27 of that and more keep all bits, smaller ones are off
    // by 2^-38 of it at most); infinities and NaN stay what they are
    uint32_t top = 0;
    auto size = [&](uint32_t m) { return m < 0x7f80u ? m : 0u; };
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = max(top, max(size(qr[i].x << 1 >> 17), size(qr[i].x << 17 >> 17)));
      top = max(top, max(size(qr[i].y << 1 >> 17), size(qr[i].y << 17 >> 17)));
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, x));
    if (lane == 0) s_to[wave] = __uint_as_float(top << 16);
    __syncthreads();
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kShWaves; ++i) most = fmaxf(most, s_to[i]);
    const int ex = (int)(__float_as_uint(most) >> 23), up = ex == 0 ? 0 : 140 - ex;   // 13 - (ex - 127)
    auto half_of = [&](uint32_t bits) { return half_bits((_Float16)__builtin_ldexpf(__uint_as_float(bits), up)); };
#pragma unroll
    for (int i = 0; i < 8; ++i)
      qr[i] = make_uint2(half_of(qr[i].x << 16) | half_of(qr[i].x & 0xffff0000u) << 16,
                         half_of(qr[i].y << 16) | half_of(qr[i].y & 0xffff0000u) << 16);
    qs = __builtin_ldexpf(qs, -up);
  }
#pragma unroll
  for (int bb = 0; bb < 4; ++bb)
    if (bb / kBb == wave % kPer) {
      const uint2 lo = qr[bb], hi = qr[4 + bb];
      s_q[(rb_q * 4 + bb) * 64 + lane] =
          make_uint4(__builtin_amdgcn_perm(hi.x, lo.x, 0x05040100u), __builtin_amdgcn_perm(hi.x, lo.x, 0x07060302u),
                     __builtin_amdgcn_perm(hi.y, lo.y, 0x05040100u), __builtin_amdgcn_perm(hi.y, lo.y, 0x07060302u));
    }
  float4_t o[NR];   // O^T: o[rb][i] = rotated channel 16 wave + 4q + i of row 16 rb + n
  int lim_min = 0x7fffffff;   // the fewest tokens that a row sees
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    o[rb] = float4_t{0.f, 0.f, 0.f, 0.f};
    c[rb] = l[rb] = w[rb] = 0.f;
    const int row = row0 + 16 * rb + n;
    const int lim = row < n_rows ? limit(row) : 0x7fffffff;
    if (tid < 16) s_lim[16 * rb + n] = lim;
    lim_min = min(lim_min, lim);
  }
#pragma unroll
  for (int x = 1; x < 16; x <<= 1) lim_min = min(lim_min, __shfl_xor(lim_min, x));
  lim_min = __builtin_amdgcn_readfirstlane(lim_min);
  __syncthreads();
  KresMasks km;
  km.init();

  // ---- loads of a tile's page: one page of the wave
  // through buffer descriptors on the (uniform) page: a lane offset is one
  // register for all sections.  The head's 64 scale pairs of a group, pair l in
  // lane l, lie at f = 128 h + 2 l of C scales spread over its four pages
  auto page_rsrc = [&](int id) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.pages + clamp_page(id, a.n_pool) * a.L.bytes),
                                             (short)0, a.L.bytes, kShBufWord3);
  };
  auto rope_rsrc = [&](const Group& g) {
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(a.rope + (int64_t)min(g.first + sub, a.n_rope - 1) * kShRope), (short)0, kShRope,
        kShBufWord3);
  };
  const int sc_slot = (h * kD + 2 * lane) / (kD * a.h_kv / 4);
  const int sc_off = a.L.kscale + 2 * (h * kD + 2 * lane - sc_slot * (kD * a.h_kv / 4));
  const int kres_at = a.L.kres + h * 768, vcode_at = a.L.vcode + h * 512, norm_at = a.L.vnorm + h * 32;
  hvec_t us;
  uint32_t kres[3], scale, near;
  u32x2_t vcd, nrm;
  typedef uint32_t u32x3_t __attribute__((ext_vector_type(3)));
  auto load_keys = [&](const Group& g) {
    const auto rs = page_rsrc(g.own);
    if constexpr (R == 32)
      us = __builtin_bit_cast(hvec_t, __builtin_amdgcn_raw_buffer_load_b128(rs, lane * 16, 0, 0));
    else
      us = __builtin_bit_cast(hvec_t, __builtin_amdgcn_raw_buffer_load_b64(rs, lane * 8, 0, 0));
    const u32x3_t k3 = __builtin_amdgcn_raw_buffer_load_b96(rs, lane * 12, kres_at, 0);
    kres[0] = k3[0];
    kres[1] = k3[1];
    kres[2] = k3[2];
  };
  auto load_codes = [&](const Group& g) {
    vcd = __builtin_amdgcn_raw_buffer_load_b64(page_rsrc(g.own), lane * 8, vcode_at, 0);
  };
  auto load_norms = [&](const Group& g) {
    nrm = __builtin_amdgcn_raw_buffer_load_b64(page_rsrc(g.own), q * 8, norm_at, 0);
  };
  auto load_scales = [&](const Group& g) {
    const int id = sc_slot == 0 ? g.id0 : sc_slot == 1 ? g.id1 : sc_slot == 2 ? g.id2 : g.id3;
    scale = *reinterpret_cast<const uint32_t*>(a.pages + clamp_page(id, a.n_pool) * a.L.bytes + sc_off);
  };
  if (n_tiles > 0) {
    load_scales(now);
    load_keys(now);
    load_codes(now);
    load_norms(now);
    near = 0;
  }

  // Scores and weights of tile t, and with them (they share no operand) the
  // values of tile t - 1: a slice of channels, 16 bb .. + 15 and + 64, and a pair
  // of the earlier tile's pages at a time.
  float4_t s[NR];
  auto values = [&](int t, int u) {
    const int buf = t & 1;
    const uint8_t* vp = s_v + (buf * kTilePages + 2 * u) * 512 + lane * 8 + wave;
    const uint2 la = vlut[vp[0]], lb = vlut[vp[512]];
    const half8_t av = __builtin_bit_cast(half8_t, make_uint4(la.x, la.y, lb.x, lb.y));
#pragma unroll
    for (int rb = 0; rb < NR; ++rb)
      o[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
          av, __builtin_bit_cast(half8_t, *reinterpret_cast<const uint4*>(s_x + (((buf * 4 + u) * NR + rb) * 64 + lane) * 16)),
          o[rb], 0, 0, 0);
  };
  auto tile = [&](int t, auto first_c) {
    constexpr bool kFirst = decltype(first_c)::value;
    const int buf = t & 1, more = t + 1 < n_tiles;
    // the page's rotations, a slice at a time.  One load a tile ahead (a dword of
    // every 64 bytes) brings the next ones near
    const auto rope = rope_rsrc(now);
    u32x4_t cs[2];   // of slices bb and bb + 1
    cs[0] = __builtin_amdgcn_raw_buffer_load_b128(rope, lane * 16, 0, 0);
    cs[1] = __builtin_amdgcn_raw_buffer_load_b128(rope, lane * 16, 1024, 0);
    asm volatile("" ::"v"(near));
    near = __builtin_amdgcn_raw_buffer_load_b32(rope_rsrc(next), lane * 64, 0, 0);
    now = next;
    if (t + 2 < n_tiles) next = find_group(t + 2);
    *reinterpret_cast<u32x2_t*>(s_v + ((buf * kTilePages + wave) * 64 + lane) * 8) = vcd;
    s_scale[wave * 64 + lane] = scale;   // read by this wave alone
    if (more) {
      load_codes(now);
      load_scales(now);
    }
    wave_lds_order();
    // ---- keys and scores
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) s[rb] = float4_t{0.f, 0.f, 0.f, 0.f};
    auto slice = [&](auto bbc) {
      constexpr int bb = decltype(bbc)::value;
      const float4_t z = {0.f, 0.f, 0.f, 0.f};
      const hvec_t blo = s_basis[bb * 64 + lane], bhi = s_basis[(bb + 4) * 64 + lane];
      float4_t klo, khi;
      if constexpr (R == 32) {
        klo = __builtin_amdgcn_mfma_f32_16x16x32_f16(blo, us, z, 0, 0, 0);
        khi = __builtin_amdgcn_mfma_f32_16x16x32_f16(bhi, us, z, 0, 0, 0);
      } else {
        klo = __builtin_amdgcn_mfma_f32_16x16x16f16(blo, us, z, 0, 0, 0);
        khi = __builtin_amdgcn_mfma_f32_16x16x16f16(bhi, us, z, 0, 0, 0);
      }
      if constexpr (!kFirst) values(t - 1, bb);
      const uint4 s4 = *reinterpret_cast<const uint4*>(s_scale + wave * 64 + 16 * bb + 4 * q);
      const half2_t sc[4] = {as_h2(s4.x), as_h2(s4.y), as_h2(s4.z), as_h2(s4.w)};
      const half2_t cp[4] = {kres_pair<4 * bb + 0>(km, kres[0], kres[1], kres[2]),
                             kres_pair<4 * bb + 1>(km, kres[0], kres[1], kres[2]),
                             kres_pair<4 * bb + 2>(km, kres[0], kres[1], kres[2]),
                             kres_pair<4 * bb + 3>(km, kres[0], kres[1], kres[2])};
      union { half2_t h2[4]; half8_t v; } ka, kb;
#pragma unroll
      for (int i = 0; i < 4; ++i) key_pair<kLow>(klo[i], khi[i], cp[i], sc[i], cs[bb & 1][i], ka.h2[i], kb.h2[i]);
      if constexpr (bb < 2) cs[bb & 1] = __builtin_amdgcn_raw_buffer_load_b128(rope, lane * 16, (bb + 2) * 1024, 0);
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const half8_t qv = __builtin_bit_cast(half8_t, s_q[(rb * 4 + bb) * 64 + lane]);
        s[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka.v, qv, s[rb], 0, 0, 0);
        if constexpr (kLow) s[rb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb.v, qv, s[rb], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    slice(std::integral_constant<int, 0>{});
    slice(std::integral_constant<int, 1>{});
    slice(std::integral_constant<int, 2>{});
    slice(std::integral_constant<int, 3>{});
    if (more) load_keys(now);
    // ---- weights of the wave's page, with the rows' offsets as they are
    const int page = kTilePages * t + wave;            // in the range
    const int end = (g0 + (page >> 2) + 1) * kGroup;   // of its group
    const bool masked = page >= n_pages || end > lim_min;
    const half2_t n01 = as_h2(nrm[0]), n23 = as_h2(nrm[1]);
    const float nv[4] = {(float)n01[0], (float)n01[1], (float)n23[0], (float)n23[1]};
    if (more) load_norms(now);
    float ln[NR], wn[NR], xm = 0.f, lm = 0.f;
    // row block rb: weights to LDS, the sums with them, the largest x and l
    auto weigh = [&](int rb, auto mask_c) {
      constexpr bool kMask = decltype(mask_c)::value;
      const bool on = page < n_pages && end <= s_lim[16 * rb + n];
      float p[4], x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][i], qs, -c[rb]));
        x[i] = p[i] * nv[i];
        if constexpr (kMask) {   // a hidden token's norm may be anything
          p[i] = on ? p[i] : 0.f;
          x[i] = on ? x[i] : 0.f;
        }
        xm = fmaxf(xm, x[i]);
      }
      const half2_t h01 = {(_Float16)x[0], (_Float16)x[1]}, h23 = {(_Float16)x[2], (_Float16)x[3]};
      const half2_t one2 = {(_Float16)1.0f, (_Float16)1.0f};
      *reinterpret_cast<uint2*>(s_x + (((buf * 4 + (wave >> 1)) * NR + rb) * 64 + lane) * 16 + 8 * (wave & 1)) =
          make_uint2(as_u32(h01), as_u32(h23));
      ln[rb] = l[rb] + ((p[0] + p[1]) + (p[2] + p[3]));
      lm = fmaxf(lm, ln[rb]);
      wn[rb] = __builtin_amdgcn_fdot2(h23, one2, __builtin_amdgcn_fdot2(h01, one2, w[rb], false), false);
    };
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      if (masked) weigh(rb, std::true_type{});
      else weigh(rb, std::false_type{});
    }
    if (__any(kFirst || xm > 60000.f || lm > 0x1p110f) && lane == 0) s_flag[buf] = t + 1;
    __syncthreads();
    if (s_flag[buf] == t + 1) {
      // some weight asks for other offsets: all waves agree on the rows' new ones,
      // which take the largest p norm to 2^8 and p to 2^90 at most
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        const bool on = page < n_pages && end <= s_lim[16 * rb + n];
        float my = -INFINITY, ms = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = s[rb][i] * qs;
          ms = fmaxf(ms, on ? y : -INFINITY);
          my = fmaxf(my, on ? y + __builtin_amdgcn_logf(nv[i]) : -INFINITY);
        }
        float to = fmaxf(my - 8.f, ms - 90.f);
        to = fmaxf(to, __shfl_xor(to, 16));
        to = fmaxf(to, __shfl_xor(to, 32));
        if (q == 0) s_to[wave * 16 * NR + 16 * rb + n] = to;
      }
      __syncthreads();
#pragma unroll
      for (int rb = 0; rb < NR; ++rb) {
        float to = -INFINITY;
#pragma unroll
        for (int i = 0; i < kShWaves; ++i) to = fmaxf(to, s_to[i * 16 * NR + 16 * rb + n]);
        const float cn = kFirst ? (to > -INFINITY ? to : 0.f) : fmaxf(c[rb], to);
        const float al = kFirst ? 0.f : __builtin_amdgcn_exp2f(c[rb] - cn);
        c[rb] = cn;
        l[rb] *= al;
        w[rb] *= al;
        o[rb] *= al;
        weigh(rb, std::true_type{});
      }
      __syncthreads();
    }
#pragma unroll
    for (int rb = 0; rb < NR; ++rb) {
      l[rb] = ln[rb];
      w[rb] = wn[rb];
    }
  };
  if (n_tiles > 0) {
    tile(0, std::true_type{});
#pragma unroll 1
    for (int t = 1; t < n_tiles; ++t) tile(t, std::false_type{});
#pragma unroll
    for (int u = 0; u < kTilePages / 2; ++u) values(n_tiles - 1, u);
  }

  // ---- a row's sums l, w over the waves (their tokens), and the partial out
  __syncthreads();
  float* s_lw = reinterpret_cast<float*>(s_x);   // [8 waves][16 NR][2]
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    l[rb] += __shfl_xor(l[rb], 16);
    l[rb] += __shfl_xor(l[rb], 32);
    w[rb] += __shfl_xor(w[rb], 16);
    w[rb] += __shfl_xor(w[rb], 32);
    if (q == 0) *reinterpret_cast<float2*>(s_lw + 2 * (wave * 16 * NR + 16 * rb + n)) = make_float2(l[rb], w[rb]);
  }
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < NR; ++rb) {
    const int row = row0 + 16 * rb + n;
    if (row >= n_rows) continue;
    const int b = row / a.G, g = row - b * a.G;
    float* dst = a.part + ((((int64_t)b * a.h_kv + h) * a.G + g) * a.n_slots + slot) * kShPitch;
    *reinterpret_cast<float4_t*>(dst + 16 * wave + 4 * q) = o[rb];
    if (wave == 0 && q == 0) {
      float ls = 0.f, ws = 0.f;
#pragma unroll
      for (int i = 0; i < kShWaves; ++i) {
        const float2 lw = *reinterpret_cast<const float2*>(s_lw + 2 * (i * 16 * NR + 16 * rb + n));
        ls += lw.x;
        ws += lw.y;
      }
      *reinterpret_cast<float4_t*>(dst + kD) = float4_t{ls == 0.f ? -INFINITY : c[rb], ls, ws, 0.f};
    }
  }
}

constexpr int kWinStep = 32;

// The window of (b, h): its rows dealt to the waves, 32 a step.
template <int DT>
__device__ __forceinline__ void window_rows(const SharedArgs& a, uint8_t* smem, int b, int h, int slot) {
  float* s_part = reinterpret_cast<float*>(smem);   // [waves][G][kRwPitch]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, q = lane >> 4, n = lane & 15;
  const int T = a.tail_len ? min(max(a.tail_len[b], 0), a.tail_cap) : a.tail_len_value;
  const uint16_t* kh = a.k_tail + (int64_t)b * a.ts_b + (int64_t)h * a.ts_h;
  const uint16_t* vh = a.v_tail + (int64_t)b * a.ts_b + (int64_t)h * a.ts_h;
  u32x4_t qb[4];
  {
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) +
                         (((int64_t)b * a.h_kv + h) * a.G + min(n, a.G - 1)) * kD + 8 * q;
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) qb[dc] = *reinterpret_cast<const u32x4_t*>(qp + 32 * dc);
  }
  RowsState st;
  st.init();
#pragma unroll 1
  for (int v0 = wave * kWinStep; v0 < T; v0 += kShWaves * kWinStep) {
    u32x4_t kr[2][4], vr[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint16_t* kp = kh + (int64_t)min(v0 + 16 * j + n, T - 1) * a.ts_t + 8 * q;
#pragma unroll
      for (int dc = 0; dc < 4; ++dc) kr[j][dc] = *reinterpret_cast<const u32x4_t*>(kp + 32 * dc);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vr[j][i] = *reinterpret_cast<const u32x4_t*>(vh + (int64_t)min(v0 + 16 * j + 4 * q + i, T - 1) * a.ts_t + 8 * n);
    rows_step<DT, 2>(st, kr, vr, qb, a.qscale, v0 + kWinStep <= T, false, T - v0, [&](int t) { return v0 + t < T; },
                  [&](int t) { return vh + (int64_t)(v0 + t) * a.ts_t; });
  }
  rows_store(st, n < a.G, s_part + (wave * a.G + n) * kRwPitch);
  __syncthreads();
  for (int e = tid; e < a.G * (kD / 4); e += kShThreads) {
    const int g = e >> 5, c = 4 * (e & 31);
    const float* src = s_part + g * kRwPitch;
    float M = -INFINITY;
    for (int w = 0; w < kShWaves; ++w) M = fmaxf(M, src[w * a.G * kRwPitch + kD]);
    float den = 0.f;
    float4_t num = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < kShWaves; ++w) {
      const float* ws = src + w * a.G * kRwPitch;
      const float2 ml = *reinterpret_cast<const float2*>(ws + kD);
      const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
      den = __builtin_fmaf(f, ml.y, den);
      num += f * *reinterpret_cast<const float4_t*>(ws + c);
    }
    float* dst = a.part + ((((int64_t)b * a.h_kv + h) * a.G + g) * a.n_slots + slot) * kShPitch;
    *reinterpret_cast<float4_t*>(dst + c) = num;
    // (c, l): the fp16 form's sums are lifted by 2^15 (rows_step)
    constexpr float kLift = DT == BMX_PREFILL_F16 ? 15.f : 0.f;
    if (c == 0) *reinterpret_cast<float4_t*>(dst + kD) = float4_t{M - kLift, den, 0.f, 0.f};
  }
}

template <int R, int NR, int DT>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(4)))
void shared_kernel(const SharedArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int w = blockIdx.x;
  auto length = [&](int b) { return min(max(a.packed_len[b], 0), a.max_len) & ~(kGroup - 1); };
  if (w < a.n_prefix) {
    // the splits run fastest: with a multiple of 8 of them a split's heads and
    // row blocks land on one XCD and read its pages and rotations from one L2
    const int split = w % a.pre_splits, rest = w / a.pre_splits;
    const int h = rest % a.h_kv, rb = rest / a.h_kv;
    const int g0 = (int)((int64_t)split * a.pre_groups / a.pre_splits);
    const int g1 = (int)((int64_t)(split + 1) * a.pre_groups / a.pre_splits);
    packed_rows<R, NR, DT>(a, smem, h, 16 * NR * rb, a.rows, a.page_table, g0, g1, split,
                           [&](int row) { return length(row / a.G); });
    return;
  }
  w -= a.n_prefix;
  if (w < a.n_own) {
    const int split = w % a.own_splits, rest = w / a.own_splits;
    const int h = rest % a.h_kv, b = rest / a.h_kv;
    const int first = a.shared_len / kGroup, groups = max(length(b) / kGroup - first, 0);
    const int g0 = first + (int)((int64_t)split * groups / a.own_splits);
    const int g1 = first + (int)((int64_t)(split + 1) * groups / a.own_splits);
    packed_rows<R, 1, DT>(a, smem, h, b * a.G, (b + 1) * a.G, a.page_table + (int64_t)b * a.max_pages, g0, g1,
                          a.pre_splits + split, [&](int) { return 0x7fffffff; });
    return;
  }
  w -= a.n_own;
  window_rows<DT>(a, smem, w / a.h_kv, w % a.h_kv, a.pre_splits + a.own_splits);
}

struct SharedMergeArgs {
  const float* part;
  void* out;
  int n_slots, win_slot;        // win_slot: the window's, or n_slots
  uint32_t v_sign_bits[4];
  float level_mu, packed_scale; // 1 / (128 kappa)
};

// One row: 256 threads, 8 lanes of slots x 32 of 4 channels.
template <int DT>
__global__ __launch_bounds__(256) void shared_merge_kernel(const SharedMergeArgs a) {
  __shared__ __attribute__((aligned(16))) float s_num[8][kD], s_win[kD];
  __shared__ float s_c[8], s_l[8], s_w[8], s_wc, s_wl;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, c4 = 4 * (tid & 31), part = tid >> 5;
  const float* p = a.part + row * a.n_slots * kShPitch;
  float c = -INFINITY, l = 0.f, w = 0.f;
  float4_t num = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < a.win_slot; s0 += 32) {   // 4 slots of the lane in flight
    float4_t st[4], v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* ps = p + (int64_t)min(s0 + 8 * u, a.win_slot - 1) * kShPitch;
      st[u] = *reinterpret_cast<const float4_t*>(ps + kD);
      v[u] = *reinterpret_cast<const float4_t*>(ps + c4);
    }
    float cn = c;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + 8 * u < a.win_slot) cn = fmaxf(cn, st[u][0]);
    if (cn == -INFINITY) continue;
    const float al = __builtin_amdgcn_exp2f(c - cn);
    c = cn;
    l *= al;
    w *= al;
    num *= al;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + 8 * u < a.win_slot && st[u][0] != -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(st[u][0] - c);
        l = __builtin_fmaf(f, st[u][1], l);
        w = __builtin_fmaf(f, st[u][2], w);
        num += f * v[u];
      }
  }
  *reinterpret_cast<float4_t*>(&s_num[part][c4]) = num;
  if (c4 == 0) {
    s_c[part] = c;
    s_l[part] = l;
    s_w[part] = w;
  }
  if (part == 0) {
    float4_t wv = {0.f, 0.f, 0.f, 0.f}, ws = {-INFINITY, 0.f, 0.f, 0.f};
    if (a.win_slot < a.n_slots) {
      const float* ps = p + (int64_t)a.win_slot * kShPitch;
      wv = *reinterpret_cast<const float4_t*>(ps + c4);
      ws = *reinterpret_cast<const float4_t*>(ps + kD);
    }
    *reinterpret_cast<float4_t*>(&s_win[c4]) = wv;
    if (c4 == 0) {
      s_wc = ws[0];
      s_wl = ws[1];
    }
  }
  __syncthreads();
  if (tid >= 64) return;
  // lane: channels tid and tid + 64
  float M = s_wc;
#pragma unroll
  for (int i = 0; i < 8; ++i) M = fmaxf(M, s_c[i]);
  float y0 = 0.f, y1 = 0.f, den = 0.f, wsum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float f = s_c[i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_c[i] - M);
    den = __builtin_fmaf(f, s_l[i], den);
    wsum = __builtin_fmaf(f, s_w[i], wsum);
    y0 = __builtin_fmaf(f, s_num[i][tid], y0);
    y1 = __builtin_fmaf(f, s_num[i][tid + 64], y1);
  }
  const float fw = s_wc == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_wc - M);
  den = __builtin_fmaf(fw, s_wl, den);
  // the levels were kappa * level + mu; then H128: bit 6 in the lane, bits 0-5 across lanes
  y0 -= a.level_mu * wsum;
  y1 -= a.level_mu * wsum;
  const float a0 = y0 + y1, a1 = y0 - y1;
  y0 = a0;
  y1 = a1;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float z0 = __shfl_xor(y0, o), z1 = __shfl_xor(y1, o);
    y0 = tid & o ? z0 - y0 : y0 + z0;
    y1 = tid & o ? z1 - y1 : y1 + z1;
  }
  y0 = (sign_neg(a.v_sign_bits, tid) ? -y0 : y0) * a.packed_scale;
  y1 = (sign_neg(a.v_sign_bits, tid + 64) ? -y1 : y1) * a.packed_scale;
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  uint16_t* out = static_cast<uint16_t*>(a.out) + row * kD;
  out[tid] = rw_pack<DT>((y0 + fw * s_win[tid]) * inv);
  out[tid + 64] = rw_pack<DT>((y1 + fw * s_win[tid + 64]) * inv);
}

// cos and sin of HF's angle: 64 threads a page, one a lane (q, n)
struct RopeArgs {
  float inv_freq[64];
  uint32_t* out;
};
__global__ __launch_bounds__(64) void rope_table_kernel(const RopeArgs a) {
  const int lane = threadIdx.x, q = lane >> 4, n = lane & 15;
  const float pos = (float)((int64_t)blockIdx.x * kPT + n);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float s, c;
      sincosf(a.inv_freq[16 * b + 4 * q + i] * pos, &s, &c);
      w[i] = (uint32_t)(uint16_t)__float2int_rn(kRopeOne * c) | (uint32_t)__float2int_rn(kRopeOne * s) << 16;
    }
    reinterpret_cast<uint4*>(a.out)[((int64_t)blockIdx.x * 4 + b) * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int sh_fail(int code, const std::string& msg) {
  bmx_set_error("bmx_k2b_decode_shared: " + msg);
  return code;
}

std::string sh_check(const bmx_k2b_decode_shared_args* a) {
  if (!a) return "args is NULL";
  const bmx_k2b_geom& g = a->geom;
  if (Geo::from(g).general) return "the recipe's page only (head_dim 128, group 64, 3 bits, rank 16 or 32)";
  if (g.h_kv < 1 || g.h_kv > 16) return "h_kv must be 1..16";
  if (g.n_q_groups < 1 || g.n_q_groups > 16) return "n_q_groups must be 1..16";
  if (a->batch < 1 || a->batch > 65535) return "batch must be 1..65535";
  if (a->io_dtype != BMX_K2B_IO_F16 && a->io_dtype != BMX_K2B_IO_BF16)
    return "io_dtype must be BMX_K2B_IO_F16 or _BF16";
  if (a->max_packed_len < 0 || a->max_packed_len % kCodec != 0) return "max_packed_len must be a multiple of 128";
  if (a->max_packed_len >= 1 << 24) return "max_packed_len must be below 2^24";
  if (a->shared_len < 0 || a->shared_len % kCodec != 0 || a->shared_len > a->max_packed_len)
    return "shared_len must be a multiple of 128 within max_packed_len";
  if (a->tail_cap < 0 || a->tail_cap > 4096) return "tail_cap must be 0..4096";
  if (!a->tail_len && (a->tail_len_value < 0 || a->tail_len_value > a->tail_cap))
    return "with tail_len NULL, tail_len_value must be 0..tail_cap";
  if (!(a->rope_scaling > 0.0f) || !(a->rope_scaling < 1e30f)) return "rope_scaling must be finite and > 0";
  if (!a->q || !a->out || !a->packed_len) return "q/out/packed_len must be non-NULL";
  if (((uintptr_t)a->q | (uintptr_t)a->out) & 15) return "q and out must be 16-byte aligned";
  if (a->max_packed_len > 0) {
    if (!a->pages || !a->basis || !a->page_table || !a->rope) return "pages/basis/page_table/rope must be non-NULL";
    if (((uintptr_t)a->pages | (uintptr_t)a->basis | (uintptr_t)a->rope) & 15)
      return "pages, basis and rope must be 16-byte aligned";
    if (a->n_pool_pages < 1) return "n_pool_pages must be >= 1";
    if ((int64_t)a->max_pages * kPT < a->max_packed_len) return "max_pages*16 < max_packed_len";
    if ((int64_t)a->rope_pages * kPT < a->max_packed_len) return "rope_pages*16 < max_packed_len";
  }
  if (a->tail_cap > 0) {
    if (!a->k_tail || !a->v_tail) return "k_tail/v_tail must be non-NULL when tail_cap > 0";
    if (a->tail_stride_t % 8 || a->tail_stride_h % 8 || a->tail_stride_b % 8)
      return "tail strides must be multiples of 8 elements";
    if (((uintptr_t)a->k_tail | (uintptr_t)a->v_tail) & 15) return "k_tail and v_tail must be 16-byte aligned";
  }
  for (int j = 0; j < 4; ++j)
    if (!(a->codebook[j] == a->codebook[j]) || (j > 0 && !(a->codebook[j] > a->codebook[j - 1])))
      return "codebook must be 4 finite ascending levels";
  return "";
}

struct SharedPlan {
  int nr, row_blocks, pre_splits, own_splits, n_slots;
  int64_t n_prefix, n_own, n_win;
};

// Row blocks of 16, 32 or 64 rows.  The prefix is split over one workgroup a CU,
// over two (as many as fit) where each still walks 6 tiles, and over no more than
// it has tiles: at 16 sequences, G 4, h_kv 8, 64k tokens take 69 us with one a CU
// (16 tiles each) and 60 with two (8), 16k tokens 29 (4) and 32 (2).  A sequence's
// own pages go over workgroups of 8 groups (4 tiles): 1,024 tokens each behind 64k
// 73 us, with 4 groups 74; without a prefix 8 groups 19, 4 groups 18, 2 groups 23;
// longer ones where there would be over 2048.
SharedPlan sh_plan(const bmx_k2b_decode_shared_args* a) {
  SharedPlan p{};
  const int h = a->geom.h_kv, rows = a->batch * a->geom.n_q_groups, cus = bmx_device_cu_count();
  p.nr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.row_blocks = (rows + 16 * p.nr - 1) / (16 * p.nr);
  const int groups = a->shared_len / kGroup;
  if (groups > 0) {
    const int units = p.row_blocks * h;
    const int tiles = (groups + 1) / 2, one = (cus + units - 1) / units, two = (2 * cus + units - 1) / units;
    p.pre_splits = std::max(1, std::min(tiles, tiles >= 6 * two ? two : one));
  }
  const int own = (a->max_packed_len - a->shared_len) / kGroup;
  if (own > 0) {
    const int64_t units = (int64_t)a->batch * h;
    const int per = (int)std::max<int64_t>(8, (own * units + 2047) / 2048);
    p.own_splits = (own + per - 1) / per;
  }
  p.n_prefix = (int64_t)p.pre_splits * h * p.row_blocks;
  p.n_own = (int64_t)p.own_splits * h * a->batch;
  p.n_win = a->tail_cap > 0 ? (int64_t)h * a->batch : 0;
  p.n_slots = p.pre_splits + p.own_splits + (a->tail_cap > 0 ? 1 : 0);
  return p;
}

size_t sh_bytes(const bmx_k2b_decode_shared_args* a, const SharedPlan& p) {
  return (size_t)a->batch * a->geom.h_kv * a->geom.n_q_groups * p.n_slots * kShPitch * sizeof(float);
}

template <int R, int NR, int DT>
hipError_t sh_launch(const SharedArgs& k, unsigned grid, hipStream_t st) {
  const size_t lds = std::max<size_t>(ShLds<R, NR>::kBytes, (size_t)kShWaves * k.G * kRwPitch * sizeof(float));
  const void* fn = (const void*)shared_kernel<R, NR, DT>;
  const hipError_t e = bmx_ensure_dynamic_lds(fn, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((shared_kernel<R, NR, DT>), dim3(grid), dim3(kShThreads), lds, st, k);
  return hipGetLastError();
}
template <int R, int DT>
hipError_t sh_launch_nr(int nr, const SharedArgs& k, unsigned grid, hipStream_t st) {
  if (nr == 1) return sh_launch<R, 1, DT>(k, grid, st);
  if (nr == 2) return sh_launch<R, 2, DT>(k, grid, st);
  return sh_launch<R, 4, DT>(k, grid, st);
}

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" int bmx_k2b_rope_table(const float inv_freq[64], int32_t n_pages, void* out, void* stream) {
  if (!inv_freq || !out || n_pages < 1 || n_pages > 1 << 20 || ((uintptr_t)out & 15)) {
    bmx_set_error("bmx_k2b_rope_table: inv_freq and a 16-byte aligned out must be non-NULL, n_pages 1..2^20");
    return BMX_E_INVALID;
  }
  RopeArgs k{};
  for (int j = 0; j < 64; ++j) k.inv_freq[j] = inv_freq[j];
  k.out = static_cast<uint32_t*>(out);
  hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)n_pages), dim3(64), 0, (hipStream_t)stream, k);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    bmx_set_error(std::string("bmx_k2b_rope_table: kernel launch: ") + hipGetErrorString(e));
    return BMX_E_HIP;
  }
  return BMX_OK;
}

extern "C" size_t bmx_k2b_decode_shared_workspace_bytes(const bmx_k2b_decode_shared_args* a) {
  if (!sh_check(a).empty()) return 0;
  return sh_bytes(a, sh_plan(a));
}

extern "C" int bmx_k2b_decode_shared(const bmx_k2b_decode_shared_args* a, void* stream) {
  const std::string why = sh_check(a);
  if (!why.empty()) return sh_fail(BMX_E_INVALID, why);
  const SharedPlan p = sh_plan(a);
  const size_t need = sh_bytes(a, p);
  if (need && (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
    return sh_fail(BMX_E_WORKSPACE, "workspace missing, unaligned or smaller than "
                                    "bmx_k2b_decode_shared_workspace_bytes()");
  const int64_t grid = p.n_prefix + p.n_own + p.n_win;
  const int64_t out_rows = (int64_t)a->batch * a->geom.h_kv * a->geom.n_q_groups;
  if (grid > INT32_MAX || out_rows > INT32_MAX) return sh_fail(BMX_E_INVALID, "too many workgroups");
  const LevelMap lm = level_map(a->codebook);
  if (lm.err > 4e-6) return sh_fail(BMX_E_INVALID, "no fp16 level map for this codebook");
  hipStream_t st = (hipStream_t)stream;
  SharedArgs k{};
  k.h_kv = a->geom.h_kv; k.G = a->geom.n_q_groups; k.B = a->batch; k.rows = a->batch * a->geom.n_q_groups;
  k.n_prefix = (int)p.n_prefix; k.n_own = (int)p.n_own;
  k.pre_splits = p.pre_splits; k.own_splits = p.own_splits; k.row_blocks = p.row_blocks; k.n_slots = p.n_slots;
  k.pre_groups = a->shared_len / kGroup;
  k.shared_len = a->shared_len; k.max_len = a->max_packed_len; k.max_pages = a->max_pages;
  k.n_pool = a->n_pool_pages; k.n_rope = a->rope_pages;
  k.tail_cap = a->tail_cap; k.tail_len_value = a->tail_len_value;
  k.L = PageLayout::make(a->geom.h_kv, a->geom.rank);
  k.qscale = a->sm_scale * 1.4426950408889634f;
  k.qscale_rope = k.qscale * a->rope_scaling;
  for (int j = 0; j < 4; ++j) k.level_hi[j] = lm.hi[j];
  k.level_mu = lm.mu;
  k.q = a->q; k.pages = a->pages; k.page_table = a->page_table; k.packed_len = a->packed_len;
  k.basis = a->basis; k.rope = static_cast<const uint8_t*>(a->rope);
  k.k_tail = static_cast<const uint16_t*>(a->k_tail); k.v_tail = static_cast<const uint16_t*>(a->v_tail);
  k.ts_b = a->tail_stride_b; k.ts_h = a->tail_stride_h; k.ts_t = a->tail_stride_t;
  k.tail_len = a->tail_len;
  k.part = static_cast<float*>(a->workspace);
  const bool f16 = a->io_dtype == BMX_K2B_IO_F16;
  hipError_t e = hipSuccess;
  if (grid > 0) {
    if (a->geom.rank == 32)
      e = f16 ? sh_launch_nr<32, BMX_PREFILL_F16>(p.nr, k, (unsigned)grid, st)
              : sh_launch_nr<32, BMX_PREFILL_BF16>(p.nr, k, (unsigned)grid, st);
    else
      e = f16 ? sh_launch_nr<16, BMX_PREFILL_F16>(p.nr, k, (unsigned)grid, st)
              : sh_launch_nr<16, BMX_PREFILL_BF16>(p.nr, k, (unsigned)grid, st);
    if (e != hipSuccess) return sh_fail(BMX_E_HIP, std::string("kernel launch: ") + hipGetErrorString(e));
  }
  SharedMergeArgs m{};
  m.part = k.part; m.out = a->out;
  m.n_slots = p.n_slots;
  m.win_slot = p.pre_splits + p.own_splits;
  for (int j = 0; j < 4; ++j) m.v_sign_bits[j] = a->v_sign_bits[j];
  m.level_mu = lm.mu;
  m.packed_scale = (float)(1.0 / (kD * (double)lm.kappa));
  if (f16) hipLaunchKernelGGL(shared_merge_kernel<BMX_PREFILL_F16>, dim3((unsigned)out_rows), dim3(256), 0, st, m);
  else hipLaunchKernelGGL(shared_merge_kernel<BMX_PREFILL_BF16>, dim3((unsigned)out_rows), dim3(256), 0, st, m);
  e = hipGetLastError();
  if (e != hipSuccess) return sh_fail(BMX_E_HIP, std::string("merge kernel launch: ") + hipGetErrorString(e));
  return BMX_OK;
}
