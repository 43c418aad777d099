// Windowed attention of few query rows over dense fp16 / bf16 K/V rows on
// gfx950: a token's attention (n_q 1) in a layer with a sliding window and
// sinks, up to kRowsMax rows (positions x heads of a KV head) in all.
//
// What the rows see of a head's keys is two runs, the sinks and the band from
// the first row's window start to the last key: they are walked as one run of
// T tokens (token v is key v, or v + gap past the sinks), and nothing else is
// read.  With 4 rows a K/V element meets 16 flops, so the call is bound by its
// bytes and, at the few MB of a window, by latency: the run is cut over the
// chip so that a wave has all its loads in flight at once.
//
// rows_kernel<DT, NR>: grid (splits, h_kv), block 256 (4 waves).  A chunk is 32
// tokens, 8 a wave: the 16 lanes of a row of lanes hold 8 channels each of 2
// tokens (16-byte loads, 256 contiguous bytes a token), and the 4 rows of
// lanes are 4 streams with an online softmax (base 2, fp32) of their own:
// scores by products over the lane's channels summed over the row by DPP, the
// values weighted in fp32.  The streams of a wave meet by lane exchange, the
// waves in LDS; one split writes the output, several write (sums, m, l)
// partials that rows_merge_kernel joins.
// A hidden token's value is left out, not weighted by 0 (it may be infinite
// or NaN).

#include "prefill_rows.h"
#include "k2b_common.h"

#include <algorithm>

namespace bmx {
namespace {

constexpr int kRwD = 128;
constexpr int kRwThreads = 256;
constexpr int kRwChunk = 32;    // tokens of a workgroup step, 8 a wave
constexpr int kRwDepth = 4;     // steps of a wave in flight

struct RowsArgs {
  const uint16_t* q;
  int64_t qsh, qst;      // elements
  const uint16_t* k;
  const uint16_t* v;
  int64_t sh, st;
  uint16_t* out;         // [h_kv * G][n_q][128]
  float* part;           // [h_kv][R][n_split][130]: sums, m, l
  int G, n_q, R, n_split;
  int T, n_first, gap;   // tokens walked; those from n_first on are keys v + gap
  int p0;                // position of query 0 (its last visible key)
  int window, sinks;
  float qscale;          // sm_scale * log2(e)
};

template <int DT>
__device__ __forceinline__ void rw_unpack(u32x4_t w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == BMX_PREFILL_F16) {
      const half2_t h = as_h2(w[i]);
      x[2 * i] = (float)h[0];
      x[2 * i + 1] = (float)h[1];
    } else {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <int DT>
__device__ __forceinline__ uint16_t rw_pack(float x) {
  if constexpr (DT == BMX_PREFILL_F16) return float_to_half_bits(x);
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// sum over the 16 lanes of a row of lanes; every lane gets it
__device__ __forceinline__ float rw_row_sum(float s) {
  s += xor_row16<1>(s);
  s += xor_row16<2>(s);
  s += xor_row16<4>(s);
  s += xor_row16<8>(s);
  return s;
}

template <int DT, int NR>
__global__ __launch_bounds__(kRwThreads) void rows_kernel(const RowsArgs a) {
  __shared__ float s_ml[4][NR][2];
  __shared__ float s_acc[4][NR][kRwD];
  const int split = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int wave = tid >> 6, lane = tid & 63, r = lane >> 4, c8 = lane & 15;
  const int n_chunks = (a.T + kRwChunk - 1) / kRwChunk;
  const int c0 = (int)((int64_t)split * n_chunks / a.n_split), c1 = (int)((int64_t)(split + 1) * n_chunks / a.n_split);
  const int n_steps = c1 - c0;
  const uint16_t* kh = a.k + (int64_t)h * a.sh + 8 * c8;
  const uint16_t* vh = a.v + (int64_t)h * a.sh + 8 * c8;
  // token j of step s, and its key (tokens past the run read its last one)
  auto token = [&](int s, int j) { return (c0 + s) * kRwChunk + 8 * wave + r + 4 * j; };
  auto key_of = [&](int v) {
    v = min(v, a.T - 1);
    return v < a.n_first ? v : v + a.gap;
  };
  u32x4_t kb[kRwDepth][2], vb[kRwDepth][2];
  auto issue = [&](int s, u32x4_t (&kd)[2], u32x4_t (&vd)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t at = (int64_t)key_of(token(s, j)) * a.st;
      kd[j] = *reinterpret_cast<const u32x4_t*>(kh + at);
      vd[j] = *reinterpret_cast<const u32x4_t*>(vh + at);
    }
  };
#pragma unroll
  for (int b = 0; b < kRwDepth - 1; ++b)
    if (b < n_steps) issue(b, kb[b], vb[b]);

  float qf[NR][8];   // the queries' channels 8 c8 .. +7 (rows past R repeat the last)
  int last[NR];      // the row's position, its last visible key
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    const int row = min(x, a.R - 1), i = row / a.G, g = row - i * a.G;
    last[x] = a.p0 + i;
    rw_unpack<DT>(*reinterpret_cast<const u32x4_t*>(a.q + (int64_t)(h * a.G + g) * a.qsh + (int64_t)i * a.qst + 8 * c8),
                  qf[x]);
  }
  float m[NR], l[NR], acc[NR][8];
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[x][c] = 0.f;
  }
  // keys from `safe` to p0 are seen by every row
  const int safe = a.p0 + a.n_q - a.window;

  for (int s0 = 0; s0 < n_steps; s0 += kRwDepth) {
#pragma unroll
    for (int b = 0; b < kRwDepth; ++b) {
      const int s = s0 + b;
      if (s >= n_steps) break;
      if (s + kRwDepth - 1 < n_steps)
        issue(s + kRwDepth - 1, kb[(b + kRwDepth - 1) % kRwDepth], vb[(b + kRwDepth - 1) % kRwDepth]);
      float p[NR][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float kf[8];
        rw_unpack<DT>(kb[b][j], kf);
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          float d = kf[0] * qf[x][0];
#pragma unroll
          for (int c = 1; c < 8; ++c) d = __builtin_fmaf(kf[c], qf[x][c], d);
          p[x][j] = rw_row_sum(d) * a.qscale;
        }
      }
      // one step's tokens v0 .. v0 + 7 of the wave: all seen by all rows?
      const int v0 = (c0 + s) * kRwChunk + 8 * wave;
      const bool whole = v0 + 8 <= a.n_first
                             ? true
                             : v0 >= a.n_first && v0 + 8 <= a.T && v0 + a.gap >= safe && v0 + 7 + a.gap <= a.p0;
      bool see[NR][2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int v = token(s, j), key = key_of(v);
#pragma unroll
        for (int x = 0; x < NR; ++x) {
          see[x][j] = whole || (v < a.T && key <= last[x] && (key > last[x] - a.window || key < a.sinks));
          if (!see[x][j]) p[x][j] = -INFINITY;
        }
      }
#pragma unroll
      for (int x = 0; x < NR; ++x) {
        const float mn = fmaxf(m[x], fmaxf(p[x][0], p[x][1]));
        const float mu = mn == -INFINITY ? 0.f : mn;   // nothing seen yet
        const float al = __builtin_amdgcn_exp2f(m[x] - mu);
        m[x] = mn;
        l[x] *= al;
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[x][c] *= al;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          p[x][j] = __builtin_amdgcn_exp2f(p[x][j] - mu);
          l[x] += p[x][j];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float vf[8];
        rw_unpack<DT>(vb[b][j], vf);
        if (whole) {
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[x][c] = __builtin_fmaf(p[x][j], vf[c], acc[x][c]);
        } else {
#pragma unroll
          for (int x = 0; x < NR; ++x)
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[x][c] = __builtin_fmaf(p[x][j], see[x][j] ? vf[c] : 0.f, acc[x][c]);
        }
      }
    }
  }
  // ---- the wave's 4 streams (lanes 16 and 32 apart), then the waves
#pragma unroll
  for (int x = 0; x < NR; ++x) {
    float mw = fmaxf(m[x], __shfl_xor(m[x], 16));
    mw = fmaxf(mw, __shfl_xor(mw, 32));
    const float w = m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[x] - mw);
    float lw = l[x] * w;
    lw += __shfl_xor(lw, 16);
    lw += __shfl_xor(lw, 32);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      float y = m[x] == -INFINITY ? 0.f : acc[x][c] * w;
      y += __shfl_xor(y, 16);
      y += __shfl_xor(y, 32);
      if (r == 0) s_acc[wave][x][8 * c8 + c] = y;
    }
    if (lane == 0) {
      s_ml[wave][x][0] = mw;
      s_ml[wave][x][1] = lw;
    }
  }
  __syncthreads();
  for (int e = tid; e < a.R * kRwD; e += kRwThreads) {
    const int x = e / kRwD, c = e % kRwD;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) M = fmaxf(M, s_ml[w][x][0]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = s_ml[w][x][0];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      den = __builtin_fmaf(f, s_ml[w][x][1], den);
      num = __builtin_fmaf(f, s_acc[w][x][c], num);
    }
    if (a.n_split == 1) {
      const int i = x / a.G, g = x - i * a.G;
      a.out[((int64_t)(h * a.G + g) * a.n_q + i) * kRwD + c] = rw_pack<DT>(den == 0.f ? 0.f : num / den);
    } else {
      float* po = a.part + (((int64_t)h * a.R + x) * a.n_split + split) * (kRwD + 2);
      po[c] = num;
      if (c == 0) {
        po[kRwD] = M;
        po[kRwD + 1] = den;
      }
    }
  }
}

// one row's splits: grid (R, h_kv), 512 threads: 4 lanes of splits x 128 channels
template <int DT>
__global__ __launch_bounds__(512) void rows_merge_kernel(const RowsArgs a) {
  __shared__ float s_den[4], s_num[4][kRwD];
  const int x = blockIdx.x, h = blockIdx.y, c = threadIdx.x & (kRwD - 1), part = threadIdx.x >> 7;
  const float* p = a.part + ((int64_t)h * a.R + x) * a.n_split * (kRwD + 2);
  float M = -INFINITY;
  for (int s = threadIdx.x & 63; s < a.n_split; s += 64) M = fmaxf(M, p[(int64_t)s * (kRwD + 2) + kRwD]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
  float num = 0.f, den = 0.f;
#pragma unroll 4
  for (int s = part; s < a.n_split; s += 4) {
    const float* ps = p + (int64_t)s * (kRwD + 2);
    const float ms = ps[kRwD];
    const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - M);
    den = __builtin_fmaf(f, ps[kRwD + 1], den);
    num = ms == -INFINITY ? num : __builtin_fmaf(f, ps[c], num);
  }
  s_num[part][c] = num;
  if (c == 0) s_den[part] = den;
  __syncthreads();
  if (part != 0) return;
  den = (s_den[0] + s_den[1]) + (s_den[2] + s_den[3]);
  num = (s_num[0][c] + s_num[1][c]) + (s_num[2][c] + s_num[3][c]);
  const int i = x / a.G, g = x - i * a.G;
  a.out[((int64_t)(h * a.G + g) * a.n_q + i) * kRwD + c] = rw_pack<DT>(den == 0.f ? 0.f : num / den);
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

// a wave's steps in one flight (kRwDepth chunks a workgroup), as long as that
// is no more than 4 workgroups a CU
int rows_splits(const bmx_prefill_args* a, int T) {
  if (a->n_split > 0) return a->n_split;
  const int chunks = (T + kRwChunk - 1) / kRwChunk;
  const int most = std::max(1, 4 * bmx_device_cu_count() / a->h_kv);
  return std::max(1, std::min((chunks + kRwDepth - 1) / kRwDepth, most));
}

}  // namespace

size_t rows_workspace_bytes(const bmx_prefill_args* a) {
  const RowsArgs k = rows_run(a);
  const int S = rows_splits(a, k.T);
  return S == 1 ? 0 : (size_t)a->h_kv * k.R * S * (kRwD + 2) * sizeof(float);
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
  const dim3 grid((unsigned)k.n_split, (unsigned)a->h_kv);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kRwThreads), 0, st, k); };
  if (a->dtype == BMX_PREFILL_F16) {
    if (k.R <= 1) launch(rows_kernel<BMX_PREFILL_F16, 1>);
    else if (k.R <= 2) launch(rows_kernel<BMX_PREFILL_F16, 2>);
    else if (k.R <= 4) launch(rows_kernel<BMX_PREFILL_F16, 4>);
    else launch(rows_kernel<BMX_PREFILL_F16, 8>);
  } else {
    if (k.R <= 1) launch(rows_kernel<BMX_PREFILL_BF16, 1>);
    else if (k.R <= 2) launch(rows_kernel<BMX_PREFILL_BF16, 2>);
    else if (k.R <= 4) launch(rows_kernel<BMX_PREFILL_BF16, 4>);
    else launch(rows_kernel<BMX_PREFILL_BF16, 8>);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || k.n_split == 1) return e;
  const dim3 rows((unsigned)k.R, (unsigned)a->h_kv);
  if (a->dtype == BMX_PREFILL_F16)
    hipLaunchKernelGGL(rows_merge_kernel<BMX_PREFILL_F16>, rows, dim3(512), 0, st, k);
  else
    hipLaunchKernelGGL(rows_merge_kernel<BMX_PREFILL_BF16>, rows, dim3(512), 0, st, k);
  return hipGetLastError();
}

}  // namespace bmx
