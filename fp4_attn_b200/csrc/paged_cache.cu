// paged_cache.cu -- the paged NVFP4 KV cache: append (quantize into pages),
// truncate / release, compact, fork and gather.
//
// Page bookkeeping is on the device, so a serving step never waits for the
// host.  It is deterministic: new pages are the lowest-numbered free ones, in
// order of (row, position), found with prefix sums; the only atomics are
// integer reference counts, whose order does not matter.
//
// Few tokens are bound by launches (13 tokens of 8 sequences: truncate, append,
// compact and gather are six launches, 23 us, 2.4 us' worth of bytes), many by bytes
// and by the quantizer's instructions: the data kernels read and write whole
// 16-byte or 8-byte runs of a (token, head) row.
#include <stdint.h>

#include <algorithm>

#include "paged.cuh"
#include "status.h"

namespace fp4 {
namespace {

constexpr int PLAN_THREADS = 1024;
constexpr int SCAN_PER_THREAD = 16;  // reference counts a thread reads at a time: four loads in flight

// The int32 scratch of a cache.
struct Work {
  int32_t* off;    // [max_seqs] first new page of a row, exclusive prefix
  int32_t* start;  // [max_seqs] append: position of a row's first new token; compact: tokens that the row ends with
  int32_t* count;  // [max_seqs] append: its new tokens; compact: the row's error bits; fork: a mark
  int32_t* total;  // [4] total[0]: new pages of the call
  int32_t* ids;    // [num_pages] the pages taken
  int32_t* from;   // [num_pages] fork: the page each is copied from
};

__host__ __device__ __forceinline__ Work work_of(const fp4paged_cache& c) {
  Work w;
  w.off = c.work;
  w.start = w.off + c.max_seqs;
  w.count = w.start + c.max_seqs;
  w.total = w.count + c.max_seqs;
  w.ids = w.total + 4;
  w.from = w.ids + c.num_pages;
  return w;
}

// Inclusive prefix sum over the block's threads; `sum` gets the block's total.
__device__ __forceinline__ int block_scan(int v, int* part, int& sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) part[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int p = part[lane];
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int u = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) p += u;
    }
    part[lane] = p;
  }
  __syncthreads();
  if (warp) v += part[warp - 1];
  sum = part[31];
  __syncthreads();
  return v;
}

// ids[0 .. need) = the lowest-numbered free pages; false if there are fewer.
__device__ bool find_free(const fp4paged_cache& c, int need, int32_t* ids, int* part) {
  int got = 0;
  for (int p0 = 0; p0 < c.num_pages && got < need; p0 += PLAN_THREADS * SCAN_PER_THREAD) {
    const int mine = p0 + threadIdx.x * SCAN_PER_THREAD;
    int32_t r[SCAN_PER_THREAD];
    if (mine + SCAN_PER_THREAD <= c.num_pages) {
#pragma unroll
      for (int i = 0; i < SCAN_PER_THREAD / 4; ++i)
        *reinterpret_cast<int4*>(r + 4 * i) = *reinterpret_cast<const int4*>(c.refs + mine + 4 * i);
    } else {
#pragma unroll
      for (int i = 0; i < SCAN_PER_THREAD; ++i) r[i] = mine + i < c.num_pages ? c.refs[mine + i] : 1;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < SCAN_PER_THREAD; ++i) n += r[i] == 0;
    int sum, at = got + block_scan(n, part, sum) - n;
#pragma unroll
    for (int i = 0; i < SCAN_PER_THREAD; ++i)
      if (r[i] == 0) {
        if (at < need) ids[at] = mine + i;
        ++at;
      }
    got += sum;
  }
  return got >= need;
}

// The row whose new pages hold page number i (off: exclusive prefixes, non-decreasing; rows without new pages
// share their successor's prefix, so the last row with off <= i is the one).
__device__ __forceinline__ int row_of(const int32_t* off, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (off[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

// Whether another row of the call names row b's sequence s: two rows would change one sequence at the same time.  The
// block looks through all rows; every thread of it takes part.
__device__ __forceinline__ bool named_twice(const int32_t* seqs, int B, int b, int s) {
  if (!seqs) return false;
  bool twice = false;
  for (int j = threadIdx.x; j < B; j += blockDim.x) twice |= j != b && seqs[j] == s;
  return __syncthreads_or(twice);
}

// ------------------------------------------------------------------ append
__global__ void __launch_bounds__(PLAN_THREADS) append_plan_kernel(fp4paged_cache c, const int32_t* seqs,
                                                                   const int32_t* counts, int B, int T) {
  __shared__ int part[32];
  __shared__ int err;
  const Work w = work_of(c);
  const int P = c.page_size;
  if (threadIdx.x == 0) err = 0;
  __syncthreads();
  if (seqs) {  // no two rows name one sequence: each finds its own mark
    for (int b = threadIdx.x; b < B; b += PLAN_THREADS)
      if (const int s = pg_seq(c, seqs, b); s >= 0) w.off[s] = b;
    __syncthreads();
    for (int b = threadIdx.x; b < B; b += PLAN_THREADS)
      if (const int s = pg_seq(c, seqs, b); s >= 0 && w.off[s] != b) atomicOr(&err, PG_BAD_SEQ);
    __syncthreads();
  }
  int need = 0;
  for (int b0 = 0; b0 < B; b0 += PLAN_THREADS) {
    const int b = b0 + threadIdx.x;
    int n = 0;
    if (b < B) {
      const int s = pg_seq(c, seqs, b), k = counts ? max(0, min(counts[b], T)) : T;
      int len = 0, cnt = 0;
      if (s < 0) {
        atomicOr(&err, PG_BAD_SEQ);
      } else {
        len = c.lens[s], cnt = k;
        if ((int64_t)len + cnt > (int64_t)c.max_pages * P) atomicOr(&err, PG_TOO_LONG);
        else if (cnt && len % P && c.refs[c.page_table[(int64_t)s * c.max_pages + len / P]] > 1)
          atomicOr(&err, PG_SHARED);  // a shared sequence that was shortened into a full page
        else n = (len + cnt + P - 1) / P - (len + P - 1) / P;
      }
      w.start[b] = len;
      w.count[b] = cnt;
    }
    int sum;
    const int at = block_scan(n, part, sum) - n;
    if (b < B) w.off[b] = need + at;
    need += sum;  // n <= max_pages, B <= max_seqs: below 2^31 (checked when the cache is described)
  }
  __syncthreads();
  bool ok = err == 0;
  if (ok && need > c.num_pages) ok = false, need = 0;
  if (ok && need > 0 && !find_free(c, need, w.ids, part)) ok = false;
  __syncthreads();
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(c.status, err ? err : PG_NO_PAGES);
    for (int b = threadIdx.x; b < B; b += PLAN_THREADS) w.count[b] = 0;
    return;
  }
  for (int i = threadIdx.x; i < need; i += PLAN_THREADS) {
    const int b = row_of(w.off, B, i), s = pg_seq(c, seqs, b), page = w.ids[i];
    c.page_table[(int64_t)s * c.max_pages + (w.start[b] + P - 1) / P + (i - w.off[b])] = page;
    c.refs[page] = 1;
  }
  for (int b = threadIdx.x; b < B; b += PLAN_THREADS) c.lens[pg_seq(c, seqs, b)] = w.start[b] + w.count[b];
}

struct AppendArgs {
  const void* x[2];
  int64_t sB[2], sH[2], sT[2];
  int B, T;
};

// A warp per (token, K or V): the token's blocks are quantized under one g and written to its slot.  They stay in
// registers between the maximum and the codes, so that a token is read once.  3 x 8192 tokens of 8 heads, bf16: 35 us,
// 3.7 TB/s of the 129 MB that go in and out; bound by instructions (22.6 million of a warp), which is why products
// and roundings go in pairs (with gather below, 95 us one by one, 80 in pairs,
// when that still had four tokens a thread).
template <int DT, bool VEC, int NB>
__global__ void __launch_bounds__(256) append_quant_kernel(fp4paged_cache c, const int32_t* seqs, AppendArgs a) {
  using E = typename In<DT>::T;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int kv = blockIdx.y, H = c.num_kv_heads, P = c.page_size;
  if (id >= (int64_t)a.B * a.T) return;
  const int b = (int)(id / a.T), t = (int)(id % a.T);
  const Work w = work_of(c);
  const E* x = static_cast<const E*>(a.x[kv]) + b * a.sB[kv] + t * a.sT[kv];
  const int64_t sH = a.sH[kv];
  int64_t page = 0;
  int slot = 0;
  uint8_t *codes = nullptr, *scales = nullptr;
  bool live = false;
  const float g = pg_quantize_token<DT, VEC, NB>(
      H * PG_SF, [&](int i) { return x + (i >> 3) * sH + (i & 7) * 16; },
      [&]() {
        live = t < w.count[b];
        if (!live) return false;
        const int pos = w.start[b] + t;
        page = c.page_table[(int64_t)pg_seq(c, seqs, b) * c.max_pages + (pos >> (__ffs(P) - 1))];  // P is a power of 2
        slot = pos & (P - 1);
        codes = (kv ? c.v_codes : c.k_codes) + (page * H * P + slot) * PG_ROW;
        scales = (kv ? c.v_scales : c.k_scales) + (page * H * P + slot) * PG_SF;
        return true;
      },
      [&](int i, uint2 v, uint32_t s) {
        const int64_t row = (int64_t)(i >> 3) * P;
        *reinterpret_cast<uint2*>(codes + row * PG_ROW + (i & 7) * 8) = v;
        scales[row * PG_SF + (i & 7)] = (uint8_t)s;
      });
  if (live && (threadIdx.x & 31) == 0) (kv ? c.v_g : c.k_g)[page * P + slot] = g;
}

template <int DT>
int launch_append(const fp4paged_cache& c, const int32_t* seqs, const AppendArgs& a, bool vec, cudaStream_t st) {
  const dim3 grid((unsigned)(((int64_t)a.B * a.T + 7) / 8), 2);
  const int nblk = c.num_kv_heads * PG_SF;
  // up to 64 blocks (8 heads) a token stays in its warp's registers; wider ones are read twice (L1)
  if (!vec) append_quant_kernel<DT, false, 0><<<grid, 256, 0, st>>>(c, seqs, a);
  else if (nblk <= 32) append_quant_kernel<DT, true, 1><<<grid, 256, 0, st>>>(c, seqs, a);
  else if (nblk <= 64) append_quant_kernel<DT, true, 2><<<grid, 256, 0, st>>>(c, seqs, a);
  else append_quant_kernel<DT, true, 0><<<grid, 256, 0, st>>>(c, seqs, a);
  return check_launch("append_quant_kernel");
}

// ------------------------------------------------- truncate, release, compact
// (a few integers per sequence: a launch's time.)  Rows that name one sequence are refused, all of them: two blocks
// would drop the same pages, the second one by what the first has left in the page table.
// Sequence s keeps its first len tokens; the block drops the pages past them.
__device__ __forceinline__ void drop_pages(const fp4paged_cache& c, int s, int old, int len) {
  const int P = c.page_size;
  int32_t* row = c.page_table + (int64_t)s * c.max_pages;
  for (int j = (len + P - 1) / P + threadIdx.x; j < (old + P - 1) / P; j += blockDim.x) {
    atomicSub(c.refs + row[j], 1);
    row[j] = -1;
  }
  if (threadIdx.x == 0) c.lens[s] = len;
}

__global__ void __launch_bounds__(128) truncate_kernel(fp4paged_cache c, const int32_t* lens, const int32_t* seqs) {
  const int s = pg_seq(c, seqs, blockIdx.x);
  const int old = s < 0 ? 0 : c.lens[s], len = lens ? max(0, min(lens[blockIdx.x], old)) : 0;
  if (named_twice(seqs, gridDim.x, blockIdx.x, s) || s < 0) {
    if (threadIdx.x == 0) atomicOr(c.status, PG_BAD_SEQ);
    return;
  }
  __syncthreads();  // every thread has read lens[s]
  drop_pages(c, s, old, len);
}

struct CompactArgs {
  const int32_t *keep, *counts, *tails, *seqs;
  int N;
};

// What a row's compaction does: base = its tail's first position, n kept tokens.  Returns the error bits, the
// same in every block that asks while no reference count changes; every thread of the block takes part.
__device__ int compact_row(const fp4paged_cache& c, const CompactArgs& a, int b, int s, int& base, int& n) {
  const int len = c.lens[s], tail = a.tails ? a.tails[b] : a.N, P = c.page_size;
  const int32_t* keep = a.keep + (int64_t)b * a.N;
  n = a.counts[b];
  base = len - tail;
  int err = 0;
  if (tail < 0 || tail > len || n < 0 || n > a.N || n > tail) {
    err = PG_BAD_KEEP;
  } else {
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
      const int k = keep[j];
      if (k < 0 || k >= tail || (j > 0 && keep[j - 1] >= k)) err |= PG_BAD_KEEP;
      else if (k != j && c.refs[c.page_table[(int64_t)s * c.max_pages + (base + j) / P]] > 1) err |= PG_SHARED;
    }
  }
  // (a block-wide or answers only whether any is not 0)
  const int bad = __syncthreads_or(err & PG_BAD_KEEP), shared = __syncthreads_or(err & PG_SHARED);
  return (bad ? PG_BAD_KEEP : 0) | (shared ? PG_SHARED : 0);
}

// A block per (row, head, K or V) moves the kept tokens of its head down, 64 at a time: all of a chunk is read
// before any of it is written.  keep is increasing, so token j moves from keep[j] >= j, and what later chunks
// read lies past everything that earlier ones wrote.  The row's verdict goes to the scratch: the next kernel lowers
// reference counts, of pages that other rows of the call hold too, so it cannot come to one of its own.
constexpr int MOVE_TOKENS = 64;
__global__ void __launch_bounds__(4 * MOVE_TOKENS) compact_move_kernel(fp4paged_cache c, CompactArgs a) {
  const int b = blockIdx.x, h = blockIdx.y, kv = blockIdx.z, s = pg_seq(c, a.seqs, b);
  const Work w = work_of(c);
  const bool tells = h == 0 && kv == 0 && threadIdx.x == 0;
  if (named_twice(a.seqs, gridDim.x, b, s) || s < 0) {
    if (tells) w.count[b] = PG_BAD_SEQ;
    return;
  }
  int base, n;
  const int err = compact_row(c, a, b, s, base, n);
  if (tells) w.start[b] = base + n, w.count[b] = err;
  if (err) return;
  const int P = c.page_size, H = c.num_kv_heads;
  const int32_t* row = c.page_table + (int64_t)s * c.max_pages;
  const int32_t* keep = a.keep + (int64_t)b * a.N;
  uint4* codes = reinterpret_cast<uint4*>(kv ? c.v_codes : c.k_codes);
  uint2* scales = reinterpret_cast<uint2*>(kv ? c.v_scales : c.k_scales);
  float* g = kv ? c.v_g : c.k_g;
  const int q = threadIdx.x & 3;
  for (int j0 = 0; j0 < n; j0 += MOVE_TOKENS) {
    const int j = j0 + (threadIdx.x >> 2);
    const bool move = j < n && keep[j] != j;
    uint4 v;
    uint2 sc;
    float gv;
    if (move) {
      const int pos = base + keep[j];
      const int64_t at = ((int64_t)row[pos / P] * H + h) * P + pos % P;
      v = codes[at * 4 + q];
      if (q == 0) sc = scales[at];
      if (h == 0 && q == 1) gv = g[(int64_t)row[pos / P] * P + pos % P];
    }
    __syncthreads();
    if (move) {
      const int pos = base + j;
      const int64_t at = ((int64_t)row[pos / P] * H + h) * P + pos % P;
      codes[at * 4 + q] = v;
      if (q == 0) scales[at] = sc;
      if (h == 0 && q == 1) g[(int64_t)row[pos / P] * P + pos % P] = gv;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(128) compact_drop_kernel(fp4paged_cache c, const int32_t* seqs) {
  const Work w = work_of(c);
  const int b = blockIdx.x, err = w.count[b];
  if (err) {
    if (threadIdx.x == 0) atomicOr(c.status, err);
    return;
  }
  const int s = pg_seq(c, seqs, b), old = c.lens[s];
  __syncthreads();  // every thread has read lens[s]
  drop_pages(c, s, old, w.start[b]);
}

// -------------------------------------------------------------------- fork
// One block, since a page's number follows from all before it: 4 sequences to 32 copies, 14 us with release and the
// copies, which are short there.
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(fp4paged_cache c, const int32_t* src,
                                                                 const int32_t* dst, int n, int deep) {
  __shared__ int part[32];
  __shared__ int err;
  const Work w = work_of(c);
  const int P = c.page_size;
  if (threadIdx.x == 0) err = 0;
  for (int r = threadIdx.x; r < n; r += PLAN_THREADS)
    if (const int d = pg_seq(c, dst, r); d >= 0) w.count[d] = r;  // a mark: no two rows go to one sequence
  __syncthreads();
  int need = 0;
  for (int r0 = 0; r0 < n; r0 += PLAN_THREADS) {
    const int r = r0 + threadIdx.x;
    int m = 0;
    if (r < n) {
      const int s = pg_seq(c, src, r), d = pg_seq(c, dst, r);
      int len = 0;
      if (s < 0 || d < 0 || c.lens[d] != 0 || w.count[d] != r) atomicOr(&err, PG_BAD_SEQ);
      else len = c.lens[s], m = (len + P - 1) / P - (deep ? 0 : len / P);
      w.start[r] = len;
    }
    int sum;
    const int at = block_scan(m, part, sum) - m;
    if (r < n) w.off[r] = need + at;
    need += sum;
  }
  __syncthreads();
  bool ok = err == 0;
  if (ok && need > c.num_pages) ok = false;
  if (ok && need > 0 && !find_free(c, need, w.ids, part)) ok = false;
  __syncthreads();
  if (threadIdx.x == 0) w.total[0] = ok ? need : 0;
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(c.status, err ? err : PG_NO_PAGES);
    return;
  }
  // full pages are shared: a warp per row
  const int lane = threadIdx.x & 31;
  if (!deep)
    for (int r = threadIdx.x >> 5; r < n; r += PLAN_THREADS / 32) {
      const int32_t* from = c.page_table + (int64_t)src[r] * c.max_pages;
      int32_t* to = c.page_table + (int64_t)dst[r] * c.max_pages;
      for (int j = lane; j < w.start[r] / P; j += 32) {
        const int page = from[j];
        to[j] = page;
        atomicAdd(c.refs + page, 1);
      }
    }
  for (int i = threadIdx.x; i < need; i += PLAN_THREADS) {
    const int r = row_of(w.off, n, i), page = w.ids[i];
    const int j = (deep ? 0 : w.start[r] / P) + (i - w.off[r]);
    w.from[i] = c.page_table[(int64_t)src[r] * c.max_pages + j];
    c.page_table[(int64_t)dst[r] * c.max_pages + j] = page;
    c.refs[page] = 1;
  }
  for (int r = threadIdx.x; r < n; r += PLAN_THREADS) c.lens[dst[r]] = w.start[r];
}

// Copies the planned pages.  A page's codes of all heads are contiguous, as are its scales and its g; a block takes a
// quarter of a page's codes and scales of one kind at a time, four 16-byte loads in flight a thread.  Bound by bytes:
// 216 MB in and out (eight sequences of up to 16384 tokens, 8 heads) take 39 us, 5.5 TB/s (52 by (token, head) rows).
__device__ __forceinline__ void copy16(uint4* to, const uint4* from, int n) {
  int j = threadIdx.x;
  for (; j + 768 < n; j += 1024) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = from[j + 256 * i];
#pragma unroll
    for (int i = 0; i < 4; ++i) to[j + 256 * i] = v[i];
  }
  for (; j < n; j += 256) to[j] = from[j];
}
__global__ void __launch_bounds__(256) fork_copy_kernel(fp4paged_cache c) {
  const Work w = work_of(c);
  const int P = c.page_size, total = w.total[0], quarter = c.num_kv_heads * P;  // 16-byte units of a quarter's codes
  for (int i = blockIdx.x; i < total * 8; i += gridDim.x) {
    const int64_t p0 = w.from[i >> 3], p1 = w.ids[i >> 3];
    const int kv = i & 1, q = (i >> 1) & 3;
    uint4 *codes = reinterpret_cast<uint4*>(kv ? c.v_codes : c.k_codes) + (int64_t)q * quarter,
          *scales = reinterpret_cast<uint4*>(kv ? c.v_scales : c.k_scales) + (int64_t)q * (quarter / 8);
    copy16(codes + p1 * quarter * 4, codes + p0 * quarter * 4, quarter);
    copy16(scales + p1 * (quarter / 2), scales + p0 * (quarter / 2), quarter / 8);
    if (q == 0) {
      float* g = kv ? c.v_g : c.k_g;
      for (int j = threadIdx.x; j < P; j += 256) g[p1 * P + j] = g[p0 * P + j];
    }
  }
}

// ------------------------------------------------------------------ gather
// A thread per block of 16 channels of GT tokens, 32 apart: 8 code bytes, a scale byte and g in, 16 values out.  A
// token's data is three trips to memory away (length, page, bytes), so two tokens' trips are made together, and few
// registers leave room for many warps: 3 x 8192 tokens of 8 heads, 129 MB, with append 71.8 us (four tokens a thread
// 77.6, one 72.2), about 28 of them here, 4.6 TB/s.
constexpr int GT = 2;
template <int DT>
__global__ void __launch_bounds__(256) gather_kernel(fp4paged_cache c, void* k_out, void* v_out, const int32_t* seqs,
                                                     int T) {
  using E = typename In<DT>::T;
  const int H = c.num_kv_heads, P = c.page_size, bh = blockIdx.y, b = bh / H, h = bh % H, kv = blockIdx.z;
  const int shift = __ffs(P) - 1;  // P is a power of 2
  const int t0 = blockIdx.x * 32 * GT + (threadIdx.x >> 3), j = threadIdx.x & 7;
  const int s = pg_seq(c, seqs, b), len = s < 0 ? 0 : min(c.lens[s], T);
  if (s < 0 && h == 0 && kv == 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(c.status, PG_BAD_SEQ);
  const uint8_t *codes = kv ? c.v_codes : c.k_codes, *scales = kv ? c.v_scales : c.k_scales;
  const float* gs = kv ? c.v_g : c.k_g;
  int64_t page[GT];
#pragma unroll
  for (int i = 0; i < GT; ++i) {
    const int t = t0 + 32 * i;
    page[i] = t < len ? c.page_table[(int64_t)s * c.max_pages + (t >> shift)] : -1;
  }
  uint2 w[GT];
  float sc[GT], g[GT];
#pragma unroll
  for (int i = 0; i < GT; ++i) {
    const int slot = (t0 + 32 * i) & (P - 1);
    const int64_t row = ((page[i] * H + h) << shift) + slot;
    w[i] = page[i] >= 0 ? __ldg(reinterpret_cast<const uint2*>(codes + row * PG_ROW) + j) : make_uint2(0u, 0u);
    sc[i] = page[i] >= 0 ? e4m3_to_f32(__ldg(scales + row * PG_SF + j)) : 0.0f;
    g[i] = page[i] >= 0 ? __ldg(gs + (page[i] << shift) + slot) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < GT; ++i) {
    const int t = t0 + 32 * i;
    if (t >= T) break;
    uint4 raw[sizeof(E)];
    uint32_t o[8];  // codes as fp16; times their scale they are exact
    e2m1x8_f16(w[i].x, o), e2m1x8_f16(w[i].y, o + 4);
    const __half2 s2 = __half2half2(__float2half_rn(sc[i]));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 v = __half22float2(__hmul2(*reinterpret_cast<const __half2*>(&o[e]), s2));
      const float x0 = __fmul_rn(v.x, g[i]), x1 = __fmul_rn(v.y, g[i]);
      if constexpr (DT == FP4_DT_F32) reinterpret_cast<float2*>(raw)[e] = make_float2(x0, x1);
      else if constexpr (DT == FP4_DT_BF16) reinterpret_cast<__nv_bfloat162*>(raw)[e] = __floats2bfloat162_rn(x0, x1);
      else reinterpret_cast<__half2*>(raw)[e] = __floats2half2_rn(x0, x1);
    }
    uint4* out = reinterpret_cast<uint4*>(static_cast<E*>(kv ? v_out : k_out) + ((int64_t)bh * T + t) * PG_D + j * 16);
#pragma unroll
    for (int e = 0; e < (int)sizeof(E); ++e) out[e] = raw[e];
  }
}

int check_cache(const fp4paged_cache* c) {
  if (!c) return set_error(FP4ATTN_ERR_ARG, "cache is null");
  if (!c->k_codes || !c->k_scales || !c->k_g || !c->v_codes || !c->v_scales || !c->v_g || !c->page_table ||
      !c->lens || !c->refs || !c->status || !c->work)
    return set_error(FP4ATTN_ERR_ARG, "null pointer in the cache");
  if (((uintptr_t)c->k_codes | (uintptr_t)c->k_scales | (uintptr_t)c->k_g | (uintptr_t)c->v_codes |
       (uintptr_t)c->v_scales | (uintptr_t)c->v_g | (uintptr_t)c->page_table | (uintptr_t)c->lens |
       (uintptr_t)c->refs | (uintptr_t)c->work) % 16)
    return set_error(FP4ATTN_ERR_ARG, "cache buffers must be 16-byte aligned");
  if (c->head_dim != PG_D) return set_error(FP4ATTN_ERR_UNSUPPORTED, "head_dim must be %d", PG_D);
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return set_error(FP4ATTN_ERR_ARG, "page_size must be 16, 32, 64 or 128");
  if (c->num_pages <= 0 || c->num_pages > 1 << 27 || c->num_kv_heads <= 0 || c->num_kv_heads > 1024 || c->max_seqs <= 0 || c->max_pages <= 0)
    return set_error(FP4ATTN_ERR_ARG, "bad cache shape");
  // positions, and the sum of the pages that one call can ask for, are 32-bit
  if ((int64_t)c->max_pages * c->page_size > INT32_MAX || (int64_t)c->max_seqs * c->max_pages > INT32_MAX)
    return set_error(FP4ATTN_ERR_ARG, "max_pages * page_size and max_seqs * max_pages must be below 2^31");
  return FP4ATTN_OK;
}

int check_rows(const fp4paged_cache* c, int B, const int32_t* seqs) {
  if (B < 0 || B > c->max_seqs || (!seqs && B > c->max_seqs))
    return set_error(FP4ATTN_ERR_ARG, "%d rows, the cache has %d sequences", B, c->max_seqs);
  return FP4ATTN_OK;
}

}  // namespace

int paged_check(const fp4paged_cache* c, int B, const int32_t* seqs) {
  if (int e = check_cache(c)) return e;
  return check_rows(c, B, seqs);
}

}  // namespace fp4

using namespace fp4;

extern "C" int64_t fp4paged_work_size(int num_pages, int max_seqs) {
  if (num_pages <= 0 || max_seqs <= 0) return -1;
  return 3 * (int64_t)max_seqs + 4 + 2 * (int64_t)num_pages;
}

extern "C" int fp4paged_append(const fp4paged_cache* cache, const void* k, const void* v, int in_dtype, int B, int T,
                               int64_t k_sB, int64_t k_sH, int64_t k_sT, int64_t v_sB, int64_t v_sH, int64_t v_sT,
                               const int32_t* seqs, const int32_t* counts, void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  if (T < 0) return set_error(FP4ATTN_ERR_ARG, "bad shape");
  if (B == 0 || T == 0) return FP4ATTN_OK;
  if (!k || !v) return set_error(FP4ATTN_ERR_ARG, "k or v is null");
  if (in_dtype < 0 || in_dtype > 2) return set_error(FP4ATTN_ERR_ARG, "bad in_dtype");
  const AppendArgs a{{k, v}, {k_sB, v_sB}, {k_sH, v_sH}, {k_sT, v_sT}, B, T};
  const int64_t esz = in_dtype == FP4_DT_F32 ? 4 : 2;
  bool vec = ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
  for (int i = 0; i < 2; ++i)
    vec = vec && (a.sB[i] * esz % 16 == 0 || B == 1) && (a.sT[i] * esz % 16 == 0 || T == 1) &&
          (a.sH[i] * esz % 16 == 0 || cache->num_kv_heads == 1);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  append_plan_kernel<<<1, PLAN_THREADS, 0, st>>>(*cache, seqs, counts, B, T);
  if (int e = check_launch("append_plan_kernel")) return e;
  switch (in_dtype) {
    case FP4_DT_F32: return launch_append<FP4_DT_F32>(*cache, seqs, a, vec, st);
    case FP4_DT_BF16: return launch_append<FP4_DT_BF16>(*cache, seqs, a, vec, st);
    default: return launch_append<FP4_DT_F16>(*cache, seqs, a, vec, st);
  }
}

extern "C" int fp4paged_truncate(const fp4paged_cache* cache, const int32_t* lens, const int32_t* seqs, int B,
                                 void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  if (B == 0) return FP4ATTN_OK;
  truncate_kernel<<<B, 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(*cache, lens, seqs);
  return check_launch("truncate_kernel");
}

extern "C" int fp4paged_compact(const fp4paged_cache* cache, const int32_t* keep, const int32_t* counts,
                                const int32_t* tails, const int32_t* seqs, int B, int N, void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  if (N < 0) return set_error(FP4ATTN_ERR_ARG, "bad shape");
  if (B == 0) return FP4ATTN_OK;
  if (!counts || (N > 0 && !keep)) return set_error(FP4ATTN_ERR_ARG, "keep or counts is null");
  const CompactArgs a{keep, counts, tails, seqs, N};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid = N > 0 ? dim3(B, cache->num_kv_heads, 2) : dim3(B);  // (N 0: nothing to move, a verdict all the same)
  compact_move_kernel<<<grid, 4 * MOVE_TOKENS, 0, st>>>(*cache, a);
  if (int e = check_launch("compact_move_kernel")) return e;
  compact_drop_kernel<<<B, 128, 0, st>>>(*cache, seqs);
  return check_launch("compact_drop_kernel");
}

extern "C" int fp4paged_fork(const fp4paged_cache* cache, const int32_t* src, const int32_t* dst, int n, int deep,
                             void* stream) {
  clear_error();
  if (int e = paged_check(cache, n, src)) return e;
  if (n == 0) return FP4ATTN_OK;
  if (!src || !dst) return set_error(FP4ATTN_ERR_ARG, "src or dst is null");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  fork_plan_kernel<<<1, PLAN_THREADS, 0, st>>>(*cache, src, dst, n, deep ? 1 : 0);
  if (int e = check_launch("fork_plan_kernel")) return e;
  // the host does not know how many pages there are: enough blocks to fill the card walk what the plan left
  fork_copy_kernel<<<148 * 8, 256, 0, st>>>(*cache);
  return check_launch("fork_copy_kernel");
}

extern "C" int fp4paged_gather(const fp4paged_cache* cache, void* k_out, void* v_out, int out_dtype,
                               const int32_t* seqs, int B, int T, void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  if (T < 0) return set_error(FP4ATTN_ERR_ARG, "bad shape");
  if (B == 0 || T == 0) return FP4ATTN_OK;
  if (!k_out || !v_out) return set_error(FP4ATTN_ERR_ARG, "k_out or v_out is null");
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16) return set_error(FP4ATTN_ERR_ARG, "outputs must be 16-byte aligned");
  if ((int64_t)B * cache->num_kv_heads > 65535) return set_error(FP4ATTN_ERR_ARG, "more than 65535 (row, head) pairs");
  const dim3 grid((unsigned)((T + 32 * GT - 1) / (32 * GT)), (unsigned)(B * cache->num_kv_heads), 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case FP4_DT_F32: gather_kernel<FP4_DT_F32><<<grid, 256, 0, st>>>(*cache, k_out, v_out, seqs, T); break;
    case FP4_DT_BF16: gather_kernel<FP4_DT_BF16><<<grid, 256, 0, st>>>(*cache, k_out, v_out, seqs, T); break;
    case FP4_DT_F16: gather_kernel<FP4_DT_F16><<<grid, 256, 0, st>>>(*cache, k_out, v_out, seqs, T); break;
    default: return set_error(FP4ATTN_ERR_ARG, "bad out_dtype");
  }
  return check_launch("gather_kernel");
}
