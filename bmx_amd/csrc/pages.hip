// Page tables of a batch on the device (gfx950): bmx_pages_update and
// bmx_pages_compact (include/bmx_pages.h).
//
// All of it is whole-number work bound by launches and a few passes over the
// tables and reference counts, and for compact by the bytes of the pages that
// move.  What orders the result (ascending ids, rows in turn) comes from prefix
// sums, never from the order in which atomics arrive: the counts are sums of
// whole numbers, the same in any order.
//
// update, four launches (two without an index: nothing can be freed):
//   rows_kernel     new rows gathered, refs copied;
//   count_kernel    an old row that k new rows continue adds k - 1 to its pages'
//                   refs: a row kept once costs nothing;
//   freed_kernel    freed pages of every chunk of 1024 ids;
//   stack_kernel    the stack with the freed pages on it, and the pages off its
//                   top into the rows that grow (a stack place finds its row in
//                   the prefix sums of grow).
// A pool of up to kPgSmallPool ids and tables of up to kPgSmallCells entries take
// one launch of one workgroup instead, the counts and the stack in its LDS
// (small_kernel): 8 beams of 512 pages over 8,192 ids 10.2 us against 14.7 of the
// four kernels, and 20.4 us a call against 27.3 with their launches.  At the limits
// (32 rows of 512, 8,192 ids) 13.4 us against 11.8, the launches still ahead; past
// them (64 rows of 512, 16,384 ids) 22.7 against 12.3.  64 rows of 4,096 pages over
// 262,144 ids take the four 20 us.
//
// compact, three launches: live pages a chunk; holes below n_live and movers
// from there listed by rank; pages copied, entries and refs rewritten.  A quarter
// of 4,096 pages moved in the pools of 16 layers (376 MB read and written): 67 us in
// move_kernel, 75 in all, 5.0 TB/s, the rate of a large copy.

#include "bmx_pages.h"
#include "k2b_common.h"

#include <algorithm>
#include <string>

namespace bmx {
namespace {

constexpr int kPgThreads = 256;
constexpr int kPgChunk = 1024;    // ids of a counting workgroup, 4 a thread
constexpr int kPgMaxRows = 16384;   // their counts and lengths lie in a workgroup's LDS
constexpr int kPgMax = 1 << 22;   // a workgroup's 256 counts of up to this sum within 31 bits

struct State {
  int32_t *table, *n_pages, *refs, *free, *n_free;
};

struct UpdateArgs {
  State in, out;
  int rows, new_rows, cap, n_pool, chunks;
  const int32_t* index;
  const int32_t* grow;
  int32_t* status;
  int32_t* counts;   // [chunks] freed pages of a chunk
  int32_t* lens;     // [new_rows] pages of a new row before it grows
};

__device__ __forceinline__ int row_len(const State& s, int r, int cap) { return min(max(s.n_pages[r], 0), cap); }

// the old row that new row i continues, or -1
__device__ __forceinline__ int source_row(const UpdateArgs& a, int i) {
  if (!a.index) return i;
  const int r = a.index[i];
  return r >= 0 && r < a.rows ? r : -1;
}

// Sums over a workgroup are chains of latencies here (a launch has little else to
// do): lanes add through DPP moves, not LDS, and the waves' sums are read at once.

// inclusive prefix sum over the wave
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);    // row_shr:1 within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
  return x;
}

// exclusive prefix sum over the workgroup's W waves; total in every thread
template <int W>
__device__ __forceinline__ int block_scan(int v, int (&s_tmp)[W], int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();   // s_tmp may be in use by an earlier sum
  if (lane == 63) s_tmp[wave] = x;
  __syncthreads();
  int before = 0, n[W];
#pragma unroll
  for (int w = 0; w < W; ++w) n[w] = s_tmp[w];
  total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    before += w < wave ? n[w] : 0;
    total += n[w];
  }
  return before + x - v;
}

// sum over the workgroup, in every thread
template <int W>
__device__ __forceinline__ int block_sum(int v, int (&s_tmp)[W]) {
  int total;
  block_scan(v, s_tmp, total);
  return total;
}

// workgroups 0 .. new_rows * pieces - 1: 1024 entries of a new row; then 1024 refs each
__global__ __launch_bounds__(kPgThreads) void rows_kernel(const UpdateArgs a) {
  const int pieces = (a.cap + kPgChunk - 1) / kPgChunk, i = (int)blockIdx.x / pieces;
  if (i >= a.new_rows) {
    const int p0 = ((int)blockIdx.x - a.new_rows * pieces) * kPgChunk + threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int p = p0 + u * kPgThreads;
      if (p < a.n_pool) a.out.refs[p] = a.in.refs[p];
    }
    return;
  }
  const int piece = (int)blockIdx.x - i * pieces;
  const int src = source_row(a, i);
  const int len = src < 0 ? 0 : row_len(a.in, src, a.cap);
  if (piece == 0 && threadIdx.x == 0) a.lens[i] = len;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = piece * kPgChunk + threadIdx.x + u * kPgThreads;
    if (e < a.cap) a.out.table[(int64_t)i * a.cap + e] = e < len ? a.in.table[(int64_t)src * a.cap + e] : 0;
  }
}

// grid (pieces of a row, old rows)
__global__ __launch_bounds__(kPgThreads) void count_kernel(const UpdateArgs a) {
  __shared__ int s_tmp[kPgThreads / 64];
  const int r = blockIdx.y;
  const int len = row_len(a.in, r, a.cap);
  if ((int)blockIdx.x * kPgChunk >= len) return;
  int p[4];   // the row's pages, in flight during the count
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int e = (int)blockIdx.x * kPgChunk + threadIdx.x + u * kPgThreads;
    p[u] = a.in.table[(int64_t)r * a.cap + min(e, len - 1)];
    if (e >= len) p[u] = -1;
  }
  int k = 0;
  for (int i = threadIdx.x; i < a.new_rows; i += kPgThreads) k += a.index[i] == r;
  k = block_sum(k, s_tmp) - 1;
  if (k == 0) return;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (p[u] >= 0 && p[u] < a.n_pool) atomicAdd(a.out.refs + p[u], k);
}

__device__ __forceinline__ bool freed(const UpdateArgs& a, int p) { return a.in.refs[p] > 0 && a.out.refs[p] <= 0; }

__global__ __launch_bounds__(kPgThreads) void freed_kernel(const UpdateArgs a) {
  __shared__ int s_tmp[kPgThreads / 64];
  int n = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int p = (int)blockIdx.x * kPgChunk + 4 * threadIdx.x + u;
    if (p < a.n_pool) n += freed(a, p);
  }
  n = block_sum(n, s_tmp);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

// One workgroup a chunk: the chunk's ids (freed ones go onto the stack) and its
// places of the old stack; workgroup 0 the lengths, counts and status too.
__global__ __launch_bounds__(kPgThreads) void stack_kernel(const UpdateArgs a) {
  __shared__ int s_tmp[kPgThreads / 64];
  extern __shared__ int s_rows[];   // [new_rows] pages given to rows before, then [new_rows] lengths
  int *s_first = s_rows, *s_len = s_rows + a.new_rows;
  const int tid = threadIdx.x, base = (int)blockIdx.x * kPgChunk + 4 * tid;
  // the chunk's own words first, in flight during the sums
  bool gone[4];
  int id[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int p = min(base + u, a.n_pool - 1);
    gone[u] = a.index && freed(a, p) && base + u < a.n_pool;
    id[u] = a.in.free[p];
  }
  int len = tid < a.new_rows ? a.lens[tid] : 0, grow = tid < a.new_rows && a.grow ? max(a.grow[tid], 0) : 0;
  const int n0 = min(max(*a.in.n_free, 0), a.n_pool);
  // freed pages before the chunk, and in all
  int before = 0, all = 0;
  if (a.index) {
    for (int c = tid; c < a.chunks; c += kPgThreads) {
      const int n = a.counts[c];
      all += n;
      before += c < (int)blockIdx.x ? n : 0;
    }
    before = block_sum(before, s_tmp);
    all = block_sum(all, s_tmp);
  }
  const int top = min(n0 + all, a.n_pool);
  // what the rows ask for
  int64_t asked = 0;
  int wide = 0;
  for (int i0 = 0; i0 < a.new_rows; i0 += kPgThreads) {
    const int i = i0 + tid;
    if (i0 > 0) {
      len = i < a.new_rows ? a.lens[i] : 0;
      grow = i < a.new_rows && a.grow ? max(a.grow[i], 0) : 0;
    }
    wide |= grow > a.cap - len;
    int sum;
    const int at = block_scan(min(grow, a.n_pool + 1), s_tmp, sum);   // a larger one fails the call by itself
    if (i < a.new_rows) {
      s_len[i] = len;
      s_first[i] = (int)min(asked + at, (int64_t)a.n_pool + 1);
    }
    asked += sum;
  }
  wide = block_sum(wide, s_tmp);
  const bool ok = wide == 0 && asked <= top;
  const int given = ok ? (int)asked : 0, left = top - given;
  __syncthreads();
  // stack place j holds page p: kept, or given to the row that counts it
  auto place = [&](int j, int p) {
    if (j >= top) return;
    a.out.free[j] = j < left ? p : -1;
    if (j < left) return;
    const int k = top - 1 - j;   // the k-th page given
    int lo = 0, hi = a.new_rows - 1;
    while (lo < hi) {            // the last row whose pages begin at or before k: it has some, as k < given
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    const int at = s_len[lo] + k - s_first[lo];
    if (at < a.cap) a.out.table[(int64_t)lo * a.cap + at] = p;
    if (p >= 0 && p < a.n_pool) a.out.refs[p] = 1;
  };
  if (a.index) {
    int n = 0, sum;
#pragma unroll
    for (int u = 0; u < 4; ++u) n += gone[u];
    int j = n0 + before + block_scan(n, s_tmp, sum);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (gone[u]) place(j++, base + u);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int j = base + u;
    if (j < n0) place(j, id[u]);
    else if (j >= top && j < a.n_pool) a.out.free[j] = -1;
  }
  if (blockIdx.x == 0) {
    for (int i = tid; i < a.new_rows; i += kPgThreads) {
      a.out.n_pages[i] = s_len[i] + (ok && a.grow ? max(a.grow[i], 0) : 0);
    }
    if (tid == 0) {
      *a.out.n_free = left;
      *a.status = wide ? BMX_PAGES_NO_ROOM : ok ? BMX_PAGES_OK : BMX_PAGES_NO_FREE;
    }
  }
}

constexpr int kPgSmallThreads = 1024;
constexpr int kPgSmallPool = 8192;      // 32 KB of counts, as much of the stack
constexpr int kPgSmallRows = kPgSmallThreads;
constexpr int kPgSmallCells = 32768;    // entries of the old and new tables: a few us of one CU's traffic

// LDS of small_kernel: refs, the new stack, which pages were live (a bit each), and
// per row k (new rows that continue it), lengths, sources and first pages.
__host__ __device__ __forceinline__ size_t small_lds(int n_pool, int rows, int new_rows) {
  return 8 * (size_t)((n_pool + 63) / 64) + 4 * (2 * (size_t)n_pool + 2 * (size_t)rows + 3 * (size_t)new_rows);
}

// An update by one workgroup: the passes of the four kernels over LDS. Its time is
// that of its chain of loads, LDS reads and barriers, so rows take 2^lg threads each
// (no division), 4 rows are in flight, and rows are searched only for the pages given.
__global__ __launch_bounds__(kPgSmallThreads) void small_kernel(const UpdateArgs a) {
  constexpr int kWaves = kPgSmallThreads / 64, kU = 4;
  extern __shared__ uint64_t s_live[];       // [n_pool / 64] in.refs > 0, then the freed ones
  const int words = (a.n_pool + 63) / 64;
  int* s_refs = reinterpret_cast<int*>(s_live + words);
  int* s_stack = s_refs + a.n_pool;          // [n_pool]
  int* s_k = s_stack + a.n_pool;             // [rows] new rows that continue the row
  int* s_old = s_k + a.rows;                 // [rows] its pages
  int* s_len = s_old + a.rows;               // [new_rows]
  int* s_first = s_len + a.new_rows;         // [new_rows]
  int* s_src = s_first + a.new_rows;         // [new_rows]
  __shared__ int s_tmp[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per = (words + kWaves - 1) / kWaves, c0 = wave * per, c1 = min(c0 + per, words);   // the wave's ids, by 64
  const int n0 = min(max(*a.in.n_free, 0), a.n_pool);
  const int src = tid < a.new_rows ? source_row(a, tid) : -1;
  const int grow = tid < a.new_rows && a.grow ? max(a.grow[tid], 0) : 0;
  if (tid < a.rows) {
    s_old[tid] = row_len(a.in, tid, a.cap);
    s_k[tid] = 0;
  }
  for (int c = c0; c < c1; c += kU) {
    int v[kU], f[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = min(64 * (c + u) + lane, a.n_pool - 1);
      v[u] = a.in.refs[p];
      f[u] = a.in.free[p];
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int p = 64 * (c + u) + lane;
      const bool on = c + u < c1 && p < a.n_pool;
      const uint64_t live = __ballot(on && v[u] > 0);
      if (on) {
        s_refs[p] = v[u];
        s_stack[p] = p < n0 ? f[u] : -1;
      }
      if (lane == 0 && c + u < c1) s_live[c + u] = live;
    }
  }
  __syncthreads();
  // new rows, one a thread
  const int len = src < 0 ? 0 : s_old[src];
  if (src >= 0) atomicAdd(s_k + src, 1);
  int asked;
  const int at = block_scan(min(grow, a.n_pool + 1), s_tmp, asked);   // a larger one fails the call by itself
  if (tid < a.new_rows) {
    s_len[tid] = len;
    s_src[tid] = src;
    s_first[tid] = min(at, a.n_pool + 1);
  }
  const bool wide = __syncthreads_or(tid < a.new_rows && grow > a.cap - len);   // and the rows' words are in LDS
  // the tables: an old row's pages lose or gain uses, a new row is its source's entries
  const int lg = min(10, 32 - __clz(a.cap - 1)), per_row = 1 << lg;   // >= cap, or all threads
  const int r_first = tid >> lg, r_step = kPgSmallThreads >> lg, e_first = tid & (per_row - 1);
  if (a.index)
    for (int r0 = r_first; r0 < a.rows; r0 += kU * r_step)
      for (int e = e_first; e < a.cap; e += per_row) {
        int p[kU], k[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
          const int r = min(r0 + u * r_step, a.rows - 1);
          k[u] = s_k[r] - 1;
          p[u] = r0 + u * r_step < a.rows && k[u] != 0 && e < s_old[r] ? a.in.table[(int64_t)r * a.cap + e] : -1;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (p[u] >= 0 && p[u] < a.n_pool) atomicAdd(s_refs + p[u], k[u]);
      }
  for (int r0 = r_first; r0 < a.new_rows; r0 += kU * r_step)
    for (int e = e_first; e < a.cap; e += per_row) {
      int p[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int i = min(r0 + u * r_step, a.new_rows - 1);
        p[u] = e < s_len[i] ? a.in.table[(int64_t)s_src[i] * a.cap + e] : 0;
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (r0 + u * r_step < a.new_rows) a.out.table[(int64_t)(r0 + u * r_step) * a.cap + e] = p[u];
    }
  __syncthreads();
  // freed ids onto the stack, 64 a wave step: how many before the wave's, and in all
  int top = n0;
  if (a.index) {
    int mine = 0;
    for (int c = c0; c < c1; ++c) {
      const int p = 64 * c + lane;
      const uint64_t m = s_live[c] & __ballot(p < a.n_pool && s_refs[p] <= 0);
      mine += __popcll(m);
      if (lane == 0) s_live[c] = m;
    }
    int all, j = n0 + block_scan(lane == 0 ? mine : 0, s_tmp, all);
    j = __builtin_amdgcn_readfirstlane(j);
    top = min(n0 + all, a.n_pool);
#pragma unroll 4
    for (int c = c0; c < c1; ++c) {
      const uint64_t m = s_live[c];
      const int place = j + __popcll(m & ((1ull << lane) - 1));
      if ((m >> lane & 1) && place < a.n_pool) s_stack[place] = 64 * c + lane;
      j += __popcll(m);
    }
    __syncthreads();
  }
  const bool ok = !wide && asked <= top;
  const int given = ok ? asked : 0, left = top - given;
  // the pages given: the k-th off the top to the last row whose pages begin at or before k
  for (int k = tid; k < given; k += kPgSmallThreads) {
    const int p = s_stack[top - 1 - k];
    int lo = 0, hi = a.new_rows - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_first[mid] <= k) lo = mid;
      else hi = mid - 1;
    }
    const int e = s_len[lo] + k - s_first[lo];
    if (e < a.cap) a.out.table[(int64_t)lo * a.cap + e] = p;
    if (p >= 0 && p < a.n_pool) s_refs[p] = 1;
  }
  if (tid < a.new_rows) a.out.n_pages[tid] = len + (ok ? grow : 0);
  if (tid == 0) {
    *a.out.n_free = left;
    *a.status = wide ? BMX_PAGES_NO_ROOM : ok ? BMX_PAGES_OK : BMX_PAGES_NO_FREE;
  }
  __syncthreads();
#pragma unroll 4
  for (int p = tid; p < a.n_pool; p += kPgSmallThreads) {
    a.out.refs[p] = s_refs[p];
    a.out.free[p] = p < left ? s_stack[p] : -1;
  }
}

struct CompactArgs {
  State in, out;
  int rows, cap, n_pool, chunks, n_pools;
  int32_t* counts;   // [chunks] live pages of a chunk
  int32_t* src;      // [n_pool] the movers, ascending
  int32_t* dst;      // [n_pool] the holes they fill
  int32_t* rank;     // [n_pool] a mover's place in src
  int32_t* moved;    // [2] movers, n_live
};

struct Pools {
  uint8_t* ptr[BMX_PAGES_MAX_POOLS];
  int32_t bytes16[BMX_PAGES_MAX_POOLS];   // page size in 16-byte units
};

__global__ __launch_bounds__(kPgThreads) void live_kernel(const CompactArgs a) {
  __shared__ int s_tmp[kPgThreads / 64];
  int n = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int p = (int)blockIdx.x * kPgChunk + 4 * threadIdx.x + u;
    if (p < a.n_pool) n += a.in.refs[p] > 0;
  }
  n = block_sum(n, s_tmp);
  if (threadIdx.x == 0) a.counts[blockIdx.x] = n;
}

__global__ __launch_bounds__(kPgThreads) void lists_kernel(const CompactArgs a) {
  __shared__ int s_tmp[kPgThreads / 64];
  const int tid = threadIdx.x;
  int before = 0, n_live = 0;
  for (int c = tid; c < a.chunks; c += kPgThreads) {
    const int n = a.counts[c];
    n_live += n;
    before += c < (int)blockIdx.x ? n : 0;
  }
  before = block_sum(before, s_tmp);
  n_live = block_sum(n_live, s_tmp);
  // live pages below n_live: whole chunks, and those of the chunk it lies in
  const int edge = n_live / kPgChunk;
  int low = 0;
  for (int c = tid; c < min(edge, a.chunks); c += kPgThreads) low += a.counts[c];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int p = edge * kPgChunk + 4 * tid + u;
    if (p < n_live) low += a.in.refs[p] > 0;
  }
  low = block_sum(low, s_tmp);
  const int base = (int)blockIdx.x * kPgChunk + 4 * tid;
  int ref[4], n = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    ref[u] = base + u < a.n_pool ? a.in.refs[base + u] : 0;
    n += ref[u] > 0;
  }
  int sum, at = before + block_scan(n, s_tmp, sum);   // live pages before the id
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int p = base + u;
    if (p >= a.n_pool) break;
    if (p < n_live) {
      if (ref[u] > 0) a.out.refs[p] = ref[u];
      else a.dst[p - at] = p;
    } else {
      a.out.refs[p] = 0;
      if (ref[u] > 0) {
        a.src[at - low] = p;
        a.rank[p] = at - low;
      }
    }
    at += ref[u] > 0;
    a.out.free[p] = p < a.n_pool - n_live ? a.n_pool - 1 - p : -1;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.moved[0] = n_live - low;
    a.moved[1] = n_live;
    *a.out.n_free = a.n_pool - n_live;
  }
}

// Workgroups 0 .. row_wgs - 1 rewrite the tables (one a row) and the filled
// holes' refs; the others take (page, pool) pairs in turn, a page at a time with
// all of a thread's loads of 16 KB ahead of its stores.
__global__ __launch_bounds__(kPgThreads) void move_kernel(const CompactArgs a, const Pools pools, int row_wgs) {
  const int tid = threadIdx.x, moves = a.moved[0], n_live = a.moved[1];
  if ((int)blockIdx.x < row_wgs) {
    for (int r = blockIdx.x; r < a.rows; r += row_wgs) {
      const int len = row_len(a.in, r, a.cap);
      for (int e = tid; e < a.cap; e += kPgThreads) {
        int p = e < len ? a.in.table[(int64_t)r * a.cap + e] : 0;
        if (e < len && p >= n_live && p < a.n_pool && a.in.refs[p] > 0) p = a.dst[a.rank[p]];
        a.out.table[(int64_t)r * a.cap + e] = p;
      }
      if (tid == 0) a.out.n_pages[r] = len;
    }
    for (int m = (int)blockIdx.x * kPgThreads + tid; m < moves; m += row_wgs * kPgThreads)
      a.out.refs[a.dst[m]] = a.in.refs[a.src[m]];
    return;
  }
  const int wgs = gridDim.x - row_wgs;
  const int64_t pairs = (int64_t)moves * a.n_pools;
  for (int64_t t = blockIdx.x - row_wgs; t < pairs; t += wgs) {
    const int l = (int)(t / moves), m = (int)(t - (int64_t)l * moves);
    const int n16 = pools.bytes16[l];
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(pools.ptr[l]) + (int64_t)a.src[m] * n16;
    u32x4_t* to = reinterpret_cast<u32x4_t*>(pools.ptr[l]) + (int64_t)a.dst[m] * n16;
    for (int i0 = tid; i0 < n16; i0 += 4 * kPgThreads) {
      u32x4_t v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * kPgThreads < n16) v[u] = __builtin_nontemporal_load(from + i0 + u * kPgThreads);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * kPgThreads < n16) __builtin_nontemporal_store(v[u], to + i0 + u * kPgThreads);
    }
  }
}

int pg_fail(const char* name, int code, const std::string& msg) {
  bmx_set_error(std::string(name) + ": " + msg);
  return code;
}

bool whole(const bmx_pages_state& s) { return s.table && s.n_pages && s.refs && s.free && s.n_free; }

State state_of(const bmx_pages_state& s) { return {s.table, s.n_pages, s.refs, s.free, s.n_free}; }

std::string check_sizes(const bmx_pages_state& in, const bmx_pages_state& out, int rows, int cap, int n_pool) {
  if (!whole(in) || !whole(out)) return "the states' pointers must be non-NULL";
  if (rows < 1 || rows > kPgMaxRows) return "rows must be 1..16384";
  if (cap < 1 || cap > kPgMax) return "cap must be 1..2^22";
  if (n_pool < 1 || n_pool > kPgMax) return "n_pool must be 1..2^22";
  if (in.table == out.table || in.n_pages == out.n_pages || in.refs == out.refs || in.free == out.free ||
      in.n_free == out.n_free)
    return "the new state needs buffers of its own";
  return "";
}

std::string check_update(const bmx_pages_update_args* a) {
  if (!a) return "args is NULL";
  const std::string why = check_sizes(a->in, a->out, a->rows, a->cap, a->n_pool);
  if (!why.empty()) return why;
  if (a->new_rows < 1 || a->new_rows > kPgMaxRows) return "new_rows must be 1..16384";
  if (!a->index && a->new_rows != a->rows) return "without an index new_rows must be rows";
  if (!a->status) return "status must be non-NULL";
  return "";
}

std::string check_compact(const bmx_pages_compact_args* a) {
  if (!a) return "args is NULL";
  const std::string why = check_sizes(a->in, a->out, a->rows, a->cap, a->n_pool);
  if (!why.empty()) return why;
  if (a->n_pools < 0 || a->n_pools > BMX_PAGES_MAX_POOLS) return "n_pools must be 0..128";
  for (int l = 0; l < a->n_pools; ++l) {
    if (!a->pools[l] || ((uintptr_t)a->pools[l] & 15)) return "pools must be non-NULL and 16-byte aligned";
    if (a->page_bytes[l] < 16 || a->page_bytes[l] % 16 || a->page_bytes[l] > 1 << 30)
      return "page_bytes must be a multiple of 16, up to 2^30";
  }
  return "";
}

int chunks_of(int n_pool) { return (n_pool + kPgChunk - 1) / kPgChunk; }

}  // namespace
}  // namespace bmx

using namespace bmx;

extern "C" size_t bmx_pages_update_workspace_bytes(const bmx_pages_update_args* a) {
  return check_update(a).empty() ? ((size_t)chunks_of(a->n_pool) + a->new_rows) * 4 : 0;
}

extern "C" int bmx_pages_update(const bmx_pages_update_args* a, void* stream) {
  const char* name = "bmx_pages_update";
  const std::string why = check_update(a);
  if (!why.empty()) return pg_fail(name, BMX_PAGES_E_INVALID, why);
  if (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < bmx_pages_update_workspace_bytes(a))
    return pg_fail(name, BMX_PAGES_E_WORKSPACE, "workspace missing, unaligned or smaller than "
                                                "bmx_pages_update_workspace_bytes()");
  hipStream_t st = (hipStream_t)stream;
  UpdateArgs k{};
  k.in = state_of(a->in);
  k.out = state_of(a->out);
  k.rows = a->rows;
  k.new_rows = a->new_rows;
  k.cap = a->cap;
  k.n_pool = a->n_pool;
  k.chunks = chunks_of(a->n_pool);
  k.index = a->index;
  k.grow = a->grow;
  k.status = a->status;
  k.counts = static_cast<int32_t*>(a->workspace);
  k.lens = k.counts + k.chunks;
  const char* launched = "kernel launch: ";
  if (a->n_pool <= kPgSmallPool && a->rows <= kPgSmallRows && a->new_rows <= kPgSmallRows &&
      ((int64_t)a->rows + a->new_rows) * a->cap <= kPgSmallCells) {
    const size_t lds = small_lds(a->n_pool, a->rows, a->new_rows);
    if (bmx_ensure_dynamic_lds((const void*)small_kernel, lds) != hipSuccess)
      return pg_fail(name, BMX_PAGES_E_HIP, "cannot reserve the kernel's LDS");
    hipLaunchKernelGGL(small_kernel, dim3(1), dim3(kPgSmallThreads), lds, st, k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return pg_fail(name, BMX_PAGES_E_HIP, std::string(launched) + hipGetErrorString(e));
    return 0;
  }
  const unsigned pieces = (unsigned)((a->cap + kPgChunk - 1) / kPgChunk);
  const size_t lds = 2 * (size_t)a->new_rows * sizeof(int);
  if (lds > 48 * 1024 && bmx_ensure_dynamic_lds((const void*)stack_kernel, lds) != hipSuccess)
    return pg_fail(name, BMX_PAGES_E_HIP, "too many rows for the device's LDS");
  const int64_t row_wgs = (int64_t)a->new_rows * pieces + k.chunks;
  if (row_wgs > INT32_MAX) return pg_fail(name, BMX_PAGES_E_INVALID, "too many table entries");
  hipLaunchKernelGGL(rows_kernel, dim3((unsigned)row_wgs), dim3(kPgThreads), 0, st, k);
  if (a->index) {
    hipLaunchKernelGGL(count_kernel, dim3(pieces, (unsigned)a->rows), dim3(kPgThreads), 0, st, k);
    hipLaunchKernelGGL(freed_kernel, dim3((unsigned)k.chunks), dim3(kPgThreads), 0, st, k);
  }
  hipLaunchKernelGGL(stack_kernel, dim3((unsigned)k.chunks), dim3(kPgThreads), lds, st, k);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pg_fail(name, BMX_PAGES_E_HIP, std::string("kernel launch: ") + hipGetErrorString(e));
  return 0;
}

extern "C" size_t bmx_pages_compact_workspace_bytes(const bmx_pages_compact_args* a) {
  return check_compact(a).empty() ? ((size_t)chunks_of(a->n_pool) + 3 * (size_t)a->n_pool + 2) * 4 : 0;
}

extern "C" int bmx_pages_compact(const bmx_pages_compact_args* a, void* stream) {
  const char* name = "bmx_pages_compact";
  const std::string why = check_compact(a);
  if (!why.empty()) return pg_fail(name, BMX_PAGES_E_INVALID, why);
  if (!a->workspace || ((uintptr_t)a->workspace & 15) || a->workspace_bytes < bmx_pages_compact_workspace_bytes(a))
    return pg_fail(name, BMX_PAGES_E_WORKSPACE, "workspace missing, unaligned or smaller than "
                                                "bmx_pages_compact_workspace_bytes()");
  hipStream_t st = (hipStream_t)stream;
  CompactArgs k{};
  k.in = state_of(a->in);
  k.out = state_of(a->out);
  k.rows = a->rows;
  k.cap = a->cap;
  k.n_pool = a->n_pool;
  k.chunks = chunks_of(a->n_pool);
  k.n_pools = a->n_pools;
  k.src = static_cast<int32_t*>(a->workspace);
  k.dst = k.src + a->n_pool;
  k.rank = k.dst + a->n_pool;
  k.counts = k.rank + a->n_pool;
  k.moved = k.counts + k.chunks;
  Pools pools{};
  for (int l = 0; l < a->n_pools; ++l) {
    pools.ptr[l] = static_cast<uint8_t*>(a->pools[l]);
    pools.bytes16[l] = (int32_t)(a->page_bytes[l] / 16);
  }
  hipLaunchKernelGGL(live_kernel, dim3((unsigned)k.chunks), dim3(kPgThreads), 0, st, k);
  hipLaunchKernelGGL(lists_kernel, dim3((unsigned)k.chunks), dim3(kPgThreads), 0, st, k);
  // at most half the pool moves; 8 workgroups a CU keep the copies in flight
  const int row_wgs = std::min(a->rows, 1024);
  const int64_t most = (int64_t)(a->n_pool / 2) * a->n_pools;
  const int copy_wgs = (int)std::min<int64_t>(most, 8 * (int64_t)bmx_device_cu_count());
  hipLaunchKernelGGL(move_kernel, dim3((unsigned)(row_wgs + copy_wgs)), dim3(kPgThreads), 0, st, k, pools, row_wgs);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pg_fail(name, BMX_PAGES_E_HIP, std::string("kernel launch: ") + hipGetErrorString(e));
  return 0;
}
