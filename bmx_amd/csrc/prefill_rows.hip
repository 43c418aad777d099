// Windowed attention of few query rows over dense fp16 / bf16 K/V rows on
// gfx950: a token's attention (n_q 1) in a layer with a sliding window and
// sinks, up to kRowsMax rows (positions x heads of a KV head) in all.
//
// What the rows see of a head's keys is two runs, the sinks and the band from
// the first row's window start to the last key: they are walked as one run of
// T tokens (token v is key v, or v + gap past the sinks), and nothing else is
// read.  With 4 rows a K/V element meets 16 flops, so the call is bound by its
// bytes and, at the few MB of a window, by latency: the run is cut over the
// chip so that a wave has all its loads in flight at once.  A window of 4,096 bf16
// keys, 8 heads, G 4: 7.4 + 3.3 us (16.8 MB, 2.3 TB/s in the first kernel).
//
// rows_kernel<DT>: grid (splits, h_kv, blocks of 16 rows), 8 waves where one
// workgroup takes the whole run (no merge), else 4.  A wave takes 64 tokens at a time (rows_step).
// The waves meet in LDS; one split writes the output, several write (sums, m, l)
// partials that rows_merge_kernel joins.

#include "prefill_rows.h"
#include "dense_rows.h"

#include <algorithm>
#include <cmath>

namespace bmx {
namespace {

constexpr int kRowsBlock = 16;      // rows of a workgroup: the columns of one 16x16 matrix product
constexpr int kRwBatch = 64;        // tokens of a wave's step
constexpr int kRwWaves = 4;         // waves of a workgroup, several splits
constexpr int kRwWavesOne = 8;      // one split

struct RowsArgs {
  const uint16_t* q;
  int64_t qsh, qst;      // elements
  const uint16_t* k;
  const uint16_t* v;
  int64_t sh, st;
  uint16_t* out;         // [h_kv * G][n_q][128]
  float* part;           // [h_kv][R][n_split][kRwPitch]
  int G, n_q, R, n_split;
  int T, n_first, gap;   // tokens walked; those from n_first on are keys v + gap
  int p0;                // position of query 0 (its last visible key)
  int window, sinks;
  float qscale;          // sm_scale * log2(e)
};

template <int DT>
__global__ __launch_bounds__(64 * kRwWavesOne) void rows_kernel(const RowsArgs a) {
  extern __shared__ __attribute__((aligned(16))) float s_part[];   // [waves][n_rows][kRwPitch]
  const int split = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, waves = blockDim.x >> 6;
  const int row0 = kRowsBlock * blockIdx.z, n_rows = min(kRowsBlock, a.R - row0);   // the workgroup's rows
  const int wave = tid >> 6, lane = tid & 63, q = lane >> 4, n = lane & 15;
  // the split's tokens in batches, dealt to the waves in turn
  const int n_batches = (a.T + kRwBatch - 1) / kRwBatch;
  const int b0 = (int)((int64_t)split * n_batches / a.n_split), b1 = (int)((int64_t)(split + 1) * n_batches / a.n_split);
  const uint16_t* kh = a.k + (int64_t)h * a.sh;
  const uint16_t* vh = a.v + (int64_t)h * a.sh;
  auto key_of = [&](int v) {   // tokens past the run: its last key
    v = min(v, a.T - 1);
    return v < a.n_first ? v : v + a.gap;
  };
  u32x4_t kr[4][4], vr[4][4];
  auto issue = [&](int b) {
    const int v0 = b * kRwBatch;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint16_t* kp = kh + (int64_t)key_of(v0 + 16 * j + n) * a.st + 8 * q;
#pragma unroll
      for (int dc = 0; dc < 4; ++dc) kr[j][dc] = *reinterpret_cast<const u32x4_t*>(kp + 32 * dc);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        vr[j][i] = *reinterpret_cast<const u32x4_t*>(vh + (int64_t)key_of(v0 + 16 * j + 4 * q + i) * a.st + 8 * n);
  };
  // the lane's row (lanes past the rows repeat the last and are not stored)
  const int row = row0 + min(n, n_rows - 1), pos_i = row / a.G;
  const int last = a.p0 + pos_i, first = last - a.window + 1;
  u32x4_t qb[4];
  {
    const uint16_t* qp = a.q + (int64_t)(h * a.G + row - pos_i * a.G) * a.qsh + (int64_t)pos_i * a.qst + 8 * q;
#pragma unroll
    for (int dc = 0; dc < 4; ++dc) qb[dc] = *reinterpret_cast<const u32x4_t*>(qp + 32 * dc);
  }
  RowsState st;
  st.init();
  const int all_from = a.p0 + a.n_q - a.window;   // keys from here to p0 are seen by every row

#pragma unroll 1
  for (int b = b0 + wave; b < b1; b += waves) {
    issue(b);
    const int v0 = b * kRwBatch;
    const bool whole = v0 + kRwBatch <= a.n_first || (v0 >= a.n_first && v0 + kRwBatch <= a.T &&
                                                      v0 + a.gap >= all_from && v0 + kRwBatch - 1 + a.gap <= a.p0);
    auto sees = [&](int v) {
      const int key = key_of(v);
      return v < a.T && key <= last && (key >= first || key < a.sinks);
    };
    rows_step<DT, 4>(st, kr, vr, qb, a.qscale, whole, a.n_q > 1, a.T - v0, [&](int t) { return sees(v0 + t); },
                  [&](int t) { return vh + (int64_t)key_of(v0 + t) * a.st; });
  }
  // ---- the waves meet in LDS
  rows_store(st, n < n_rows, s_part + (wave * n_rows + n) * kRwPitch);
  __syncthreads();
  for (int e = tid; e < n_rows * (kRwD / 4); e += blockDim.x) {
    const int x = e >> 5, c = 4 * (e & 31);
    const float* src = s_part + x * kRwPitch;
    float M = -INFINITY;
    for (int w = 0; w < waves; ++w) M = fmaxf(M, src[w * n_rows * kRwPitch + kRwD]);
    float den = 0.f;
    float4_t num = {0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < waves; ++w) {
      const float* ws = src + w * n_rows * kRwPitch;
      const float2 ml = *reinterpret_cast<const float2*>(ws + kRwD);
      const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
      den = __builtin_fmaf(f, ml.y, den);
      num += f * *reinterpret_cast<const float4_t*>(ws + c);
    }
    if (a.n_split == 1) {
      const float inv = den == 0.f ? 0.f : 1.0f / den;
      const int i = (row0 + x) / a.G, g = row0 + x - i * a.G;
      *reinterpret_cast<uint2*>(a.out + ((int64_t)(h * a.G + g) * a.n_q + i) * kRwD + c) =
          make_uint2(rw_pack2<DT>(num[0] * inv, num[1] * inv), rw_pack2<DT>(num[2] * inv, num[3] * inv));
    } else {
      float* po = a.part + (((int64_t)h * a.R + row0 + x) * a.n_split + split) * kRwPitch;
      *reinterpret_cast<float4_t*>(po + c) = num;
      if (c == 0) *reinterpret_cast<float2*>(po + kRwD) = make_float2(M, den);
    }
  }
}

// one row's splits: grid (R, h_kv), 256 threads: 8 lanes of splits x 32 of 4 channels
template <int DT>
__global__ __launch_bounds__(256) void rows_merge_kernel(const RowsArgs a) {
  __shared__ __attribute__((aligned(16))) float s_part[8][kRwPitch];
  const int x = blockIdx.x, h = blockIdx.y, c = 4 * (threadIdx.x & 31), part = threadIdx.x >> 5;
  const float* p = a.part + ((int64_t)h * a.R + x) * a.n_split * kRwPitch;
  float m = -INFINITY, den = 0.f;
  float4_t num = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < a.n_split; s0 += 32) {   // 4 splits of the lane in flight
    float2 ml[4];
    float4_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float* ps = p + (int64_t)min(s0 + 8 * u, a.n_split - 1) * kRwPitch;
      ml[u] = *reinterpret_cast<const float2*>(ps + kRwD);
      w[u] = *reinterpret_cast<const float4_t*>(ps + c);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + 8 * u < a.n_split) mn = fmaxf(mn, ml[u].x);
    if (mn == -INFINITY) continue;
    const float al = __builtin_amdgcn_exp2f(m - mn);
    den *= al;
    num *= al;
    m = mn;
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s0 + 8 * u < a.n_split && ml[u].x != -INFINITY) {
        const float f = __builtin_amdgcn_exp2f(ml[u].x - m);
        den = __builtin_fmaf(f, ml[u].y, den);
        num += f * w[u];
      }
  }
  *reinterpret_cast<float4_t*>(&s_part[part][c]) = num;
  if (c == 0) *reinterpret_cast<float2*>(&s_part[part][kRwD]) = make_float2(m, den);
  __syncthreads();
  if (part != 0) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < 8; ++w) M = fmaxf(M, s_part[w][kRwD]);
  den = 0.f;
  num = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float2 ml = *reinterpret_cast<const float2*>(&s_part[w][kRwD]);
    const float f = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);
    den = __builtin_fmaf(f, ml.y, den);
    num += f * *reinterpret_cast<const float4_t*>(&s_part[w][c]);
  }
  const float inv = den == 0.f ? 0.f : 1.0f / den;
  const int i = x / a.G, g = x - i * a.G;
  *reinterpret_cast<uint2*>(a.out + ((int64_t)(h * a.G + g) * a.n_q + i) * kRwD + c) =
      make_uint2(rw_pack2<DT>(num[0] * inv, num[1] * inv), rw_pack2<DT>(num[2] * inv, num[3] * inv));
}

// what the rows see: the sinks before the band, and the band
RowsArgs rows_run(const bmx_prefill_args* a) {
  RowsArgs k{};
  k.p0 = a->n_kv - a->n_q;
  k.window = std::min(a->window, a->n_kv);
  k.sinks = std::min(a->sinks, a->n_kv);
  const int lo = std::max(0, k.p0 - k.window + 1);
  k.n_first = std::min(k.sinks, lo);
  k.gap = lo - k.n_first;
  k.T = k.n_first + a->n_kv - lo;
  k.G = a->n_q_groups;
  k.n_q = a->n_q;
  k.R = a->n_q * a->n_q_groups;
  return k;
}

// One workgroup of 8 waves a head where its waves take the run at one step each:
// 500 keys 8.7 us, 8 splits and their join 7.9, but a launch more.  Else
// workgroups of 4 waves, up to 16 of 2 steps (2,000 keys 8.3 us, of 4 steps 9.2),
// more of 4 steps (4,096 keys 9.0 us, of 2 steps 9.8; 32,000 keys of one head 11.9
// and 14.3), as long as that is no more than 4 workgroups a CU.
int row_blocks(const bmx_prefill_args* a) { return (a->n_q * a->n_q_groups + kRowsBlock - 1) / kRowsBlock; }
int rows_splits(const bmx_prefill_args* a, int T) {
  if (a->n_split > 0) return a->n_split;
  const int batches = (T + kRwBatch - 1) / kRwBatch;
  if (batches <= kRwWavesOne) return 1;
  const int most = std::max(1, 4 * bmx_device_cu_count() / (a->h_kv * row_blocks(a)));
  const int splits = std::max((batches + kRwWaves - 1) / kRwWaves, std::min(16, (batches + 1) / 2));
  return std::max(1, std::min(splits, most));
}

}  // namespace

size_t rows_workspace_bytes(const bmx_prefill_args* a) {
  const RowsArgs k = rows_run(a);
  const int S = rows_splits(a, k.T);
  return S == 1 ? 0 : (size_t)a->h_kv * k.R * S * kRwPitch * sizeof(float);
}

hipError_t rows_launch(const bmx_prefill_args* a, hipStream_t st) {
  RowsArgs k = rows_run(a);
  k.q = static_cast<const uint16_t*>(a->q);
  k.qsh = a->q_stride_h;
  k.qst = a->q_stride_t;
  k.k = static_cast<const uint16_t*>(a->k);
  k.v = static_cast<const uint16_t*>(a->v);
  k.sh = a->kv_stride_h;
  k.st = a->kv_stride_t;
  k.out = static_cast<uint16_t*>(a->out);
  k.part = static_cast<float*>(a->workspace);
  k.n_split = rows_splits(a, k.T);
  k.qscale = a->sm_scale * 1.4426950408889634f;
  const int waves = k.n_split == 1 ? kRwWavesOne : kRwWaves;
  const size_t lds = (size_t)waves * std::min(k.R, kRowsBlock) * kRwPitch * sizeof(float);
  const dim3 grid((unsigned)k.n_split, (unsigned)a->h_kv, (unsigned)row_blocks(a)), rows((unsigned)k.R, (unsigned)a->h_kv);
  const bool f16 = a->dtype == BMX_PREFILL_F16;
  auto launch = [&](auto kernel) {
    const hipError_t e = bmx_ensure_dynamic_lds((const void*)kernel, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), lds, st, k);
    return hipGetLastError();
  };
  const hipError_t e = f16 ? launch(rows_kernel<BMX_PREFILL_F16>) : launch(rows_kernel<BMX_PREFILL_BF16>);
  if (e != hipSuccess || k.n_split == 1) return e;
  if (f16) hipLaunchKernelGGL(rows_merge_kernel<BMX_PREFILL_F16>, rows, dim3(256), 0, st, k);
  else hipLaunchKernelGGL(rows_merge_kernel<BMX_PREFILL_BF16>, rows, dim3(256), 0, st, k);
  return hipGetLastError();
}

}  // namespace bmx
