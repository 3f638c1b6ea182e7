// sampling.cu -- sampling from logits with given random numbers, and the walk
// that accepts drafted tokens.
//
// Weights w = exp((x - max) / T) are rounded to whole multiples of 2^-34 of the
// largest: every sum is then an exact integer sum, the same for any split of a
// row, and a result depends neither on the grid nor on an order of atomics.
//
// No sort: a histogram over x finds the bin that the threshold of top-k or top-p
// falls into, and only that bin's few logits are ranked; the draw is a search in
// the running sums of what is kept, in index order.
//
// Few rows: a cluster of CTAs reads a row once and holds it in shared memory; the
// CTAs exchange their maxima, sums, histograms and the bin's logits over
// distributed shared memory, and each draws the same conclusions from them.  Many rows: one
// CTA per row, or a cluster of two or four, goes over it twice, the second time mostly in L2, and
// keeps the logits near the maximum, which are what the rest needs, in shared memory.
//
// One row of 32000: 16 us, a chain of about a dozen exchanges and barriers.  512 rows of 131072 fp32 under
// top_p: 180 us, 1.5 TB/s (41 us at a plain copy's rate).  There the first pass (maximum) runs at the
// memory's rate and is a fifth of a row's time; the second (weights, sum, histogram), half of it, is bound
// by instructions (about 16 per logit, half of them for the weight); what follows by latencies.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attn_softmax.cuh"
#include "common.cuh"
#include "fp4attn.h"
#include "status.h"

namespace fp4 {
namespace {

constexpr int SP_MAX_V = 262144;  // 16 CTAs of 16384 logits
constexpr float SP_ONE = 17179869184.0f;  // 2^34
typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int R, V;
  int64_t ld;
  const float *u, *temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  int64_t* tokens;
  float* logprobs;
};

// Larger keys for larger logits (-0 below +0 would split equal logits: + 0 first).
__device__ __forceinline__ uint32_t sp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t q) { return __uint_as_float(q & 0x80000000u ? q & 0x7fffffffu : ~q); }

constexpr int SP_BINS = 512;    // of x's distance from the maximum
constexpr int SP_LIST = 1024;   // logits of a bin that are ranked directly; more of them are searched bit by bit
constexpr int SP_SHORT = 256;   // that many, and all bins down to one are ranked together
constexpr int SP_RANKS = 16;    // CTAs of a cluster
constexpr int SP_LIMB = 17;     // a weight as two parts of 17 bits,
constexpr int SP_HELD = 32767;  // of which this many add up within 32 bits: logits that a CTA holds
constexpr float SP_FAR = 3.402823466e38f;

// The last kept logit in the order (x descending, index ascending).
struct Cut {
  uint32_t key;
  int index;
};

struct alignas(16) SampleShared {  // (16-byte loads follow it)
  uint32_t count[SP_BINS], lo[SP_BINS], hi[SP_BINS];  // this CTA's histogram
  uint32_t total[SP_BINS];                            // the row's
  u64 mass[SP_BINS];
  u64 list[SP_LIST];  // (key, not index): larger first
  u64 list_w[SP_LIST];
  uint32_t mine_key[SP_LIST];  // this CTA's part of the list
  int mine_index[SP_LIST];
  int listed, found, last;
  u64 last_mass;
  Cut cut;
  float rank_max[SP_RANKS], rank_min[SP_RANKS];
  u64 rank_sum[4][SP_RANKS];  // by turns; a slot is written anew only several barriers after it was read
  int rank_first[SP_RANKS];
  u64 part[32], warp_sum[32];  // a value per warp
  int ipart[32];
  float fpart[2][32];
};

template <int NT, typename T>
__device__ __forceinline__ T sp_block_sum(T v, T* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & ((NT / 32) - 1)];
#pragma unroll
  for (int o = (NT / 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The first bin at which the running sum of v reaches `target`, and the sum before it; SP_BINS if it never does.
template <int NT, typename T>
__device__ __forceinline__ int sp_find_bin(SampleShared& sh, const T* v, double target) {
  static_assert(SP_BINS <= NT, "a bin per thread");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const u64 own = threadIdx.x < SP_BINS ? v[threadIdx.x] : 0;
  u64 inc = own;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) sh.part[warp] = inc;
  if (threadIdx.x == 0) sh.found = SP_BINS;
  __syncthreads();
  u64 at = inc - own;
#pragma unroll
  for (int i = 0; i < SP_BINS / 32; ++i) at += i < warp ? sh.part[i] : 0;
  if ((double)at < target && (double)(at + own) >= target) sh.found = threadIdx.x;
  __syncthreads();
  return sh.found;
}

// STREAM: CTAs that read their part anew for each pass (1024 threads, one CTA on an SM: the rows under way then fit
// L2; with two they did not, and 512 rows of 131072 fp32 took 277 us); else a cluster's CTAs hold it.
constexpr int SP_HELD_THREADS = 512, SP_STREAM_THREADS = 1024;
constexpr int SP_NEAR = 640;  // logits of a band that a warp keeps (160 KB in all); more: the row is read again instead
template <int DT, bool STREAM, bool ALONE>
__global__ void __launch_bounds__(STREAM ? SP_STREAM_THREADS : SP_HELD_THREADS, STREAM ? 1 : 2)
    sample_kernel(SampleArgs a, int loads) {
  constexpr int SP_THREADS = STREAM ? SP_STREAM_THREADS : SP_HELD_THREADS, SP_WARPS = SP_THREADS / 32;
  using T = typename In<DT>::T;
  constexpr int VEC = 16 / (int)sizeof(T);
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  static_assert(sizeof(SampleShared) % 16 == 0, "what follows is read 16 bytes at a time");
  uint4* held = reinterpret_cast<uint4*>(smem + sizeof(SampleShared));  // [warp][loads][lane]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = ALONE ? 1 : (int)cluster.num_blocks(), rank = ALONE ? 0 : (int)cluster.block_rank();
  auto peer = [&](int c) -> SampleShared& { return ALONE ? sh : *cluster.map_shared_rank(&sh, c); };
  auto barrier = [&]() {
    if (ALONE || C == 1) __syncthreads();
    else cluster.sync();
  };
  const int r = (int)(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // this CTA runs; waited for before the first access to another one's memory
  if constexpr (!ALONE) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  // A warp has consecutive positions, VEC per lane and load.  Positions count from the 16-byte boundary at or below
  // the row, so that loads are aligned whatever the row's start.
  const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.ld;
  const int skip = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(row - skip);
  const int pos0 = ((rank * SP_WARPS + warp) * loads * 32 + lane) * VEC, end = a.V + skip;
  uint4* mine = held + warp * loads * 32 + lane;  // only this thread's
  const T none = In<DT>::t(-INFINITY);
  auto fetch = [&](int j) {
    const int pos = pos0 + j * 32 * VEC;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (pos < end) raw = __ldg(base + pos / VEC);
    if (pos < skip || pos + VEC > end) {
      T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = pos + i >= skip && pos + i < end ? t[i] : none;
    }
    return raw;
  };
  // NaN counts as -inf, +inf as the largest finite value.  Where it matters: comparisons pass over NaN by themselves,
  // and only few logits go further than a comparison.
  auto clean = [](float v) { return fminf(fmaxf(v, -INFINITY), SP_FAR); };
  auto value = [&](const uint4& raw, int i) { return In<DT>::f(reinterpret_cast<const T*>(&raw)[i]); };
  u64* kept_near = reinterpret_cast<u64*>(held) + warp * SP_NEAR;  // (x or NaN, index), this warp's
  int near_n = 0;
  bool have_near = false;  // all warps have all down to near_reach below the maximum
  float near_reach = 0.0f;
  auto index_of = [&](int j) { return pos0 + j * 32 * VEC - skip; };
  auto load = [&](int j) { return STREAM ? fetch(j) : mine[j * 32]; };
  // Calls see(x, y), which answers with two bits, for each two of this thread's logits (not cleaned), and some(hits, j)
  // with the bits of up to 16 of them, from load j on; all lanes of a warp call it together.
  constexpr int STEP = STREAM ? 16 / VEC : 8 / VEC;
  const bool inner = (rank * SP_WARPS + warp) * loads * 32 * VEC >= skip && (rank * SP_WARPS + warp + 1) * loads * 32 * VEC <= end;
  auto walk = [&](auto see, auto some) {
#pragma unroll 1
    for (int j = 0; j < loads; j += STEP) {
      uint4 raw[STEP];
      if (STREAM && inner && j + STEP <= loads) {
        const uint4* p = base + (pos0 / VEC + j * 32);
#pragma unroll
        for (int i = 0; i < STEP; ++i) raw[i] = __ldg(p + 32 * i);
      } else {
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          if (j + i < loads) {
            raw[i] = load(j + i);
          } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) reinterpret_cast<T*>(&raw[i])[v] = none;
          }
        }
      }
      uint32_t hits = 0u;
#pragma unroll
      for (int i = 0; i < STEP * VEC; i += 2) hits |= see(value(raw[i / VEC], i % VEC), value(raw[i / VEC], i % VEC + 1)) << i;
      some(hits, j);
    }
  };
  auto place = [&](int j, int i) { return pos0 + (j + i / VEC) * 32 * VEC + i % VEC; };
  auto real = [&](int j, int i) { return j + i / VEC < loads && place(j, i) >= skip && place(j, i) < end; };  // else a stand-in
  // Calls got(x, index) (cleaned) for those that see(x) is true for.
  auto each = [&](auto see, auto got) {
    walk([&](float x, float y) { return (see(x) ? 1u : 0u) | (see(y) ? 2u : 0u); }, [&](uint32_t hits, int j) {
#pragma unroll 1
      while (hits) {
        const int i = __ffs(hits) - 1;
        hits &= hits - 1;
        if (!real(j, i)) continue;
        const int index = place(j, i) - skip;
        const T v = STREAM ? __ldg(row + index) : reinterpret_cast<const T*>(mine + (j + i / VEC) * 32)[i % VEC];
        got(clean(In<DT>::f(v)), index);
      }
    });
  };

  // each() over what is known to have all that see() is true for: the kept ones, if all of those are asked for
  auto each_near = [&](bool enough, auto see, auto got) {
    if (STREAM && enough && have_near) {
      for (int e = lane; e < near_n; e += 32) {
        const u64 c = kept_near[e];
        const float v = __uint_as_float((uint32_t)(c >> 32));
        if (see(v)) got(v, (int)(uint32_t)c);
      }
    } else {
      each(see, got);
    }
  };

  // A streamed row's hits are few, in some lanes: got(x, index) for them one by one would take longer than all else.
  // Their indices go to the warp's list (behind those that are there), and got is called for 32 of them at a time; what
  // it is false for counts no longer.  A list that is too long is given up, and each() takes its place.
  auto take = [&](auto see, auto also, auto got) {
    const int n0 = near_n;
    walk([&](float x, float y) { also(x, y); return (see(x) ? 1u : 0u) | (see(y) ? 2u : 0u); },
         [&](uint32_t hits, int j) {
#pragma unroll 1
           while (__ballot_sync(0xffffffffu, hits != 0u) != 0u) {
             const int i = __ffs(hits) - 1;
             // (-inf that stands in for what a step has past the warp's loads is a hit where see() has no lower end)
             const bool hit = hits != 0u && ((inner && j + STEP <= loads) || real(j, i));
             const unsigned all = __ballot_sync(0xffffffffu, hit);
             const int at = near_n + __popc(all & ((1u << lane) - 1u));
             if (hit && at < SP_NEAR) kept_near[at] = (u64)(place(j, i) - skip);
             hits &= hits - 1;
             near_n += __popc(all);
           }
         });
    __syncwarp();
    if (near_n > SP_NEAR) {
      each(see, got);
      return;
    }
#pragma unroll 1
    for (int e0 = n0 + lane; e0 < near_n; e0 += 128) {
      int index[4];
      T v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) index[i] = e0 + 32 * i < near_n ? (int)kept_near[e0 + 32 * i] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __ldg(row + index[i]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e0 + 32 * i < near_n) kept_near[e0 + 32 * i] = (u64)__float_as_uint(clean(In<DT>::f(v[i]))) << 32 | (uint32_t)index[i];
    }
#pragma unroll 1
    for (int e = n0 + lane; e < near_n; e += 32) {
      const uint32_t index = (uint32_t)kept_near[e];
      if (!got(__uint_as_float((uint32_t)(kept_near[e] >> 32)), (int)index)) kept_near[e] = (u64)0x7fc00000u << 32 | index;
    }
    __syncwarp();
  };

  // --------------------------------------------------------- maximum, minimum
  if constexpr (!STREAM) {
#pragma unroll 4
    for (int j = 0; j < loads; ++j) mine[j * 32] = fetch(j);
  }
  for (int i = tid; i < SP_BINS; i += SP_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
  if (tid == 0) sh.listed = 0;
  float mx = -INFINITY, mn = INFINITY;  // mn: of those above -inf
  each(
      [&](float v) {
        mx = fmaxf(mx, v), mn = fminf(mn, v == -INFINITY ? INFINITY : v);
        return false;
      },
      [](float, int) {});
  mx = fminf(mx, SP_FAR), mn = fminf(mn, SP_FAR);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) sh.fpart[0][warp] = mx, sh.fpart[1][warp] = mn;
  __syncthreads();
  if constexpr (!ALONE) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all CTAs have started
  if (warp == 0) {
    mx = sh.fpart[0][lane & (SP_WARPS - 1)], mn = sh.fpart[1][lane & (SP_WARPS - 1)];
#pragma unroll
    for (int o = SP_WARPS / 2; o > 0; o >>= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane < C) peer(lane).rank_max[rank] = mx, peer(lane).rank_min[rank] = mn;
  }
  barrier();
  mx = sh.rank_max[0], mn = sh.rank_min[0];
  for (int i = 1; i < C; ++i) mx = fmaxf(mx, sh.rank_max[i]), mn = fminf(mn, sh.rank_min[i]);
  if (mx == -INFINITY) {  // the same in every CTA
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  const float t0 = a.temperature ? a.temperature[r] : 1.0f, temp = t0 > 0.0f ? fmaxf(t0, 1e-30f) : 1.0f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const bool greedy = !(t0 > 0.0f);
  const bool by_k = !greedy && k > 0 && k < a.V, by_p = !greedy && top_p < 1.0f;
  // w = 2^((x - max) log2(e) / T): the factor in two parts, so that the product is rounded once
  const double f = 1.4426950408889634 / (double)temp;
  const float f1 = (float)f, f2 = (float)(f - (double)f1);
  auto weight = [&](float v) -> u64 {
    float e;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(e) : "f"(v), "f"(SP_FAR));  // (stays NaN)
    const float d = e - mx;  // (a NaN or an infinite d gives NaN or -inf, and so 0)
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaxf(fmaf(d, f1, d * f2), -150.0f)));
    return __float2ull_rn(e * SP_ONE);  // (2^34 in the exponent's argument would cost it four bits)
  };
  // weigh(x, y) adds two weights to zh 2^17 + zl without conversions to 64 bits, which run at a fraction of the other
  // instructions' rate: w 2^17 is rounded to an integer by adding 1.5 2^23, the remainder, which is exact, times 2^17
  // likewise, and together they are w 2^34 rounded to the nearest integer, as in weight().  What the sums of the bit
  // patterns have of 1.5 2^23's comes off at the end.
  constexpr float SHIFT = 12582912.0f;
  const uint64_t mx2 = pk2(-mx, -mx), f1x2 = pk2(f1, f1), f2x2 = pk2(f2, f2), limb2 = pk2(131072.0f, 131072.0f);
  const uint64_t shift2 = pk2(SHIFT, SHIFT), minus2 = pk2(-1.0f, -1.0f);
  uint32_t zh = 0u, zl = 0u;
  auto weigh = [&](float x, float y) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(x) : "f"(SP_FAR));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(y) : "f"(SP_FAR));
    const uint64_t d = add2(pk2(x, y), mx2);
    float e0, e1, h0, h1, l0, l1;
    upk2(fma2(d, f1x2, mul2(d, f2x2)), e0, e1);
    const uint64_t e = pk2(ex2(fmaxf(e0, -150.0f)), ex2(fmaxf(e1, -150.0f))), h = fma2(e, limb2, shift2);
    const uint64_t l = fma2(fma2(e, limb2, fma2(h, minus2, shift2)), limb2, shift2);
    upk2(h, h0, h1), upk2(l, l0, l1);
    zh += __float_as_uint(h0) + __float_as_uint(h1), zl += __float_as_uint(l0) + __float_as_uint(l1);
  };
  auto weighed = [&]() -> u64 {  // what a walk() over weigh() has added up
    const uint32_t off = (uint32_t)((loads + STEP - 1) / STEP * STEP * VEC) * __float_as_uint(SHIFT);
    return ((u64)(zh - off) << SP_LIMB) + (u64)(int64_t)(int32_t)(zl - off);
  };
  int turn = 0;
  // The cluster's sum of a number per thread.
  auto row_sum = [&](u64 v) -> u64 {
    v = sp_block_sum<SP_THREADS>(v, sh.part);
    if (tid < C) peer(tid).rank_sum[turn & 3][rank] = v;
    barrier();
    u64 sum = 0;
    for (int i = 0; i < C; ++i) sum += sh.rank_sum[turn & 3][i];
    ++turn;
    return sum;
  };
  // The sum of what comes before this warp, in index order, and the row's; `own`: this thread's.
  struct Before {
    u64 before, warp, total;
  };
  auto row_scan = [&](u64 own) -> Before {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    __syncthreads();
    if (lane == 0) sh.warp_sum[warp] = own;
    __syncthreads();
    u64 block = 0;
    Before s{0, own, 0};
#pragma unroll
    for (int i = 0; i < SP_WARPS; ++i) {
      block += sh.warp_sum[i];
      if (i < warp) s.before += sh.warp_sum[i];
    }
    if (tid < C) peer(tid).rank_sum[turn & 3][rank] = block;
    barrier();
    for (int i = 0; i < C; ++i) {
      if (i < rank) s.before += sh.rank_sum[turn & 3][i];
      s.total += sh.rank_sum[turn & 3][i];
    }
    ++turn;
    return s;
  };
  // Calls hit(x, index) for the logit at which the running sum of fn(x, index) passes `target`, in its warp.
  auto row_find = [&](const Before& s, u64 target, auto fn, auto hit) {
    if (!(s.before <= target && target < s.before + s.warp)) return;
    u64 before = s.before;
#pragma unroll 1
    for (int j = 0; j < loads; ++j) {
      const uint4 raw = load(j);
      u64 here = 0;
#pragma unroll 1
      for (int i = 0; i < VEC; ++i) here += fn(clean(value(raw, i)), index_of(j) + i);
      u64 inc = here;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      u64 at = before + inc - here;
      if (at <= target && target < at + here)
#pragma unroll 1
        for (int i = 0; i < VEC; ++i) {
          const float v = clean(value(raw, i));
          const u64 w = fn(v, index_of(j) + i);
          if (at <= target && target < at + w) hit(v, index_of(j) + i);
          at += w;
        }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (before > target) break;
    }
  };

  // ------------------------------- sum, first largest logit, first histogram
  // of what can hold the thresholds: first the logits within 7 (or 7 T) of the maximum, which are few and mostly
  // enough; a logit in the histogram costs as much as three that are only summed, a second histogram a pass over the row
  const float full = fminf(24.6f * temp, mx - mn);  // weights further away are 0
  const float near = full <= 8.0f ? full : fminf(fmaxf(7.0f * temp, 7.0f), full);
  float from = -1.0f, reach = near, per = reach > 0.0f ? (float)SP_BINS / reach : 0.0f;  // the band (from, reach] below mx
  // more than the roundings of mx - distance and of mx - v, for a v near it, come to (2^-24 of |mx| + distance each)
  auto slack = [&](float distance) { return (fabsf(mx) + distance) * 4.8e-7f; };
  auto in_band = [&](float v) { return mx - v > from && mx - v <= reach; };
  auto bin_of = [&](float v) { return max(0, min(SP_BINS - 1, (int)((mx - v - fmaxf(from, 0.0f)) * per))); };
  auto add = [&](float v) {
    const int b = bin_of(v);
    const u64 w = weight(v);
    atomicAdd(&sh.count[b], 1u);
    atomicAdd(&sh.lo[b], (uint32_t)w & ((1u << SP_LIMB) - 1));
    atomicAdd(&sh.hi[b], (uint32_t)(w >> SP_LIMB));
  };
  u64 z = 0;
  int first = INT32_MAX;
  {
    // hits: what the histogram takes, or a greedy row's largest
    const float low = greedy ? mx : by_k || by_p ? mx - reach - slack(reach) : INFINITY;
    auto hit = [&](float v, int index) {
      if (greedy) first = min(first, index);
      else if (in_band(v)) return add(v), true;
      return false;
    };
    if constexpr (STREAM) {
      take([&](float v) { return v >= low; }, weigh, hit);
      z = weighed();
      have_near = __syncthreads_and(near_n <= SP_NEAR && (by_k || by_p));
      near_reach = reach;
    } else {
      each([&](float v) { z += weight(v); return v >= low; }, hit);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.ipart[warp] = first;
    z = sp_block_sum<SP_THREADS>(z, sh.part);
    if (tid < C) {
      int m = INT32_MAX;
#pragma unroll
      for (int i = 0; i < SP_WARPS; ++i) m = min(m, sh.ipart[i]);
      peer(tid).rank_sum[3][rank] = z, peer(tid).rank_first[rank] = m;
    }
  }
  barrier();
  z = 0, first = INT32_MAX;
  for (int i = 0; i < C; ++i) z += sh.rank_sum[3][i], first = min(first, sh.rank_first[i]);
  const float logz = logf((float)((double)z / (double)SP_ONE));
  if (greedy) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = first;
      if (a.logprobs) a.logprobs[r] = -logz;
    }
    return;  // (the barrier above was behind the last access to another CTA)
  }

  Cut cut{0u, INT32_MAX};
  bool search = false;
  // what has to go before a logit for top_p to drop it; the first always stays
  auto p_target = [&](u64 mass) { return fmax((double)top_p * (double)mass, 1.0); };
  if (by_k || by_p) {
    // Every CTA has the row's whole histogram and, of the bin it then needs, all logits: all of them come to the same cut.
    auto merge = [&]() -> bool {
      bool fine = true;
      for (int i = tid; i < SP_BINS; i += SP_THREADS) {
        uint32_t n = 0;
        u64 lo = 0, hi = 0;
        for (int c0 = 0; c0 < C; c0 += 8) {  // (eight CTAs' at a time: a trip over the cluster takes long)
          uint32_t m[8], l[8], h[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const SampleShared& from = peer(min(c0 + c, C - 1));
            m[c] = from.count[i], l[c] = from.lo[i], h[c] = from.hi[i];
          }
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c0 + c < C) {
              fine = fine && m[c] <= SP_HELD;  // more may have run over (a row that is read anew)
              n += m[c], lo += l[c], hi += h[c];
            }
        }
        sh.total[i] = n, sh.mass[i] = lo + (hi << SP_LIMB);
      }
      return __syncthreads_and(fine);
    };
    u64 base_n = 0, base_w = 0;  // above the band
    bool merged = merge();
    // another band's histogram; false if it cannot be had
    auto band = [&](float lo, float hi) -> bool {
      from = lo, reach = hi, per = (float)SP_BINS / (reach - fmaxf(from, 0.0f));
      barrier();  // (the histograms have been read)
      for (int i = tid; i < SP_BINS; i += SP_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
      __syncthreads();
      const float upper = from < 0.0f ? INFINITY : mx - from + slack(from), lower = mx - reach - slack(reach);
      auto see = [&](float v) { return v >= lower && v <= upper; };
      auto hit = [&](float v, int) { return in_band(v) ? add(v), true : false; };
      if (STREAM && have_near && reach > near_reach) {  // (bands follow one another)
        take(see, [](float, float) {}, hit);
        have_near = __syncthreads_and(near_n <= SP_NEAR);
        near_reach = reach;
      } else {
        each_near(reach <= near_reach, see, hit);
      }
      barrier();
      return merge();
    };
    // the bin where the count, or the mass, reaches the target, in this band or one further away; SP_BINS: nowhere
    auto locate = [&](bool by_mass, double target) -> int {
      for (;;) {
        const int b = by_mass ? sp_find_bin<SP_THREADS>(sh, sh.mass, target - (double)base_w) : sp_find_bin<SP_THREADS>(sh, sh.total, target - (double)base_n);
        if (b < SP_BINS || reach >= full) return b;
        u64 sn = 0, sw = 0;
        for (int i = tid; i < SP_BINS; i += SP_THREADS) sn += sh.total[i], sw += sh.mass[i];
        base_n += sp_block_sum<SP_THREADS>(sn, sh.part), base_w += sp_block_sum<SP_THREADS>(sw, sh.part);
        // how much further: counts grow by about e^1.4 for a unit of x, or less
        const double more = by_mass ? 1.0 : target / (double)(base_n + 1);
        const float further = more < 2.0 ? 1.15f : more < 8.0 ? 1.3f : 1.6f;
        if (!(merged = merged && band(reach, fminf(full, reach * further)))) return SP_BINS;
      }
    };
    int listed_bin = -1, listed_from = 0, n = 0;  // the bins that are listed
    u64 above_n = 0, above_w = 0;
    int at_n[SP_LIST / SP_THREADS];
    u64 at_w[SP_LIST / SP_THREADS];
    // The logits of a bin -- or, where they are few, of all bins of the band up to it: top_p then finds its cut among
    // them too -- and how many and how much goes before each of this thread's.
    auto list = [&](int bin) {
      if (listed_bin >= 0) {
        barrier();  // (the last list has been read)
        if (tid == 0) sh.listed = 0;
        barrier();
      }
      u64 sn = 0, sw = 0;
      for (int i = tid; i < bin; i += SP_THREADS) sn += sh.total[i], sw += sh.mass[i];
      sn = sp_block_sum<SP_THREADS>(sn, sh.part);
      const bool all = by_k && by_p && sn + sh.total[bin] <= SP_SHORT;
      above_n = base_n + (all ? 0 : sn), above_w = base_w + (all ? 0 : sp_block_sum<SP_THREADS>(sw, sh.part));
      listed_bin = bin, listed_from = all ? 0 : bin;
      // (a range that surely has the bin, to pass over the others quickly)
      const float wide = slack(reach), at0 = mx - fmaxf(from, 0.0f);
      const float hi = listed_from ? at0 - (float)(listed_from - 1) / per + wide : INFINITY;
      const float lo = per > 0.0f ? at0 - (float)(bin + 2) / per - wide : -INFINITY;
      each_near(
           reach <= near_reach, [&](float v) { return v >= lo && v <= hi; },
           [&](float v, int index) {
             if (in_band(v) && bin_of(v) >= listed_from && bin_of(v) <= bin) {
               const int at = atomicAdd(&sh.listed, 1);
               if (at < SP_LIST) sh.mine_key[at] = sp_key(v), sh.mine_index[at] = index;
             }
           });
      barrier();
      // everybody's, one after the other
      if (tid < C) sh.rank_first[tid] = peer(tid).listed;
      __syncthreads();
      n = 0;
      for (int c = 0; c < C; ++c) n += sh.rank_first[c];
      n = min(n, SP_LIST);
      for (int e = tid; e < n; e += SP_THREADS) {
        int c = 0, i = e;
        while (i >= sh.rank_first[c]) i -= sh.rank_first[c++];
        const uint32_t q = peer(c).mine_key[i];
        sh.list[e] = (u64)q << 32 | (uint32_t)~peer(c).mine_index[i], sh.list_w[e] = weight(logit_of(q));
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < SP_LIST / SP_THREADS; ++t) {
        const int e = tid + t * SP_THREADS;
        at_n[t] = 0, at_w[t] = 0;
        if (e < n) {
          const u64 own = sh.list[e];
#pragma unroll 4
          for (int i = 0; i < n; ++i) {
            const bool ahead = sh.list[i] > own;
            at_n[t] += ahead, at_w[t] += ahead ? sh.list_w[i] : 0ull;
          }
        }
      }
    };
    // the cut behind the listed logits that keeps(t) holds for, and the mass down to it
    auto settle = [&](auto keeps) -> u64 {
      __syncthreads();
      if (tid == 0) sh.last = -1;
      __syncthreads();
#pragma unroll
      for (int t = 0; t < SP_LIST / SP_THREADS; ++t)
        if (tid + t * SP_THREADS < n && keeps(t)) atomicMax(&sh.last, at_n[t]);
      __syncthreads();
#pragma unroll
      for (int t = 0; t < SP_LIST / SP_THREADS; ++t) {
        const int e = tid + t * SP_THREADS;
        if (e < n && at_n[t] == sh.last) {
          sh.cut = {(uint32_t)(sh.list[e] >> 32), (int)~(uint32_t)sh.list[e]};
          sh.last_mass = above_w + at_w[t] + sh.list_w[e];
        }
      }
      __syncthreads();
      cut = sh.cut;
      return sh.last_mass;
    };
    u64 mass = z;  // what is kept so far
    if (by_k && merged) {
      const int b = locate(false, (double)k);
      if (b < SP_BINS && merged) {  // (else fewer than k weights are not 0)
        if (sh.total[b] > SP_LIST) search = true;
        else list(b), mass = settle([&](int t) { return above_n + at_n[t] < (u64)k; });
      }
    }
    if (by_p && merged && !search) {
      const double target = p_target(mass);
      if ((double)base_w >= target) {  // top_k went past the band that has it
        base_n = base_w = 0;
        listed_bin = listed_from = SP_BINS;
        merged = band(-1.0f, near);
      }
      const int b = merged ? locate(true, target) : SP_BINS;
      if (b == SP_BINS || sh.total[b] > SP_LIST) {
        search = true;
      } else {
        if (b > listed_bin || b < listed_from) list(b);
        // (what top_k dropped has all of `mass` before it, more than the target)
        settle([&](int t) { return (double)(above_w + at_w[t]) < target; });
      }
    }
    search = search || !merged;
    if (search) {
      // Too many logits in one bin (flat rows): the thresholds bit by bit.
      cut = {0u, INT32_MAX};
      auto above = [&](uint32_t q, bool by_mass) {
        u64 s = 0;
        each(
            [&](float v) {
              if (v > -INFINITY && sp_key(clean(v)) > q) s += by_mass ? weight(v) : 1ull;
              return false;
            },
            [](float, int) {});
        return row_sum(s);
      };
      auto largest = [&](bool by_mass, double target) {  // the largest key whose own and larger ones reach the target
        uint32_t lo = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t c = lo | (1u << bit);
          if ((double)above(c - 1, by_mass) >= target) lo = c;
        }
        return lo;
      };
      // the cut at the n-th (from 0) logit of key q
      auto nth = [&](uint32_t q, u64 n) {
        auto is = [&](float v, int) -> u64 { return v != -INFINITY && sp_key(v) == q; };
        u64 own = 0;
        each([&](float v) { return v > -INFINITY && sp_key(clean(v)) == q; }, [&](float v, int index) { own += is(v, index); });
        row_find(row_scan(own), n, is, [&](float, int index) {
          for (int c = 0; c < C; ++c) peer(c).cut = {q, index};
        });
        barrier();
        const Cut c = sh.cut;
        barrier();
        return c;
      };
      auto key_weight = [&](uint32_t q) { return weight(logit_of(q)); };
      mass = z;
      if (by_k && above(0u, false) > (u64)k) {
        const uint32_t q = largest(false, (double)k);
        const u64 more = above(q, false);
        mass = above(q, true) + ((u64)k - more) * key_weight(q);
        cut = nth(q, (u64)k - more - 1);
      }
      if (by_p) {
        const double target = p_target(mass);
        const uint32_t q = max(largest(true, target), cut.key);
        const u64 before = above(q, true), w = key_weight(q);
        // how many of key q have less than the target before them
        u64 lo = 0, hi = w > 0 ? (u64)a.V : 0;
        while (lo < hi) {
          const u64 mid = (lo + hi) / 2;
          if ((double)(before + mid * w) < target) lo = mid + 1;
          else hi = mid;
        }
        if (lo > 0) {  // (else q is where top_k cut, and the target is reached before it)
          const Cut c = nth(q, min(lo, above(q - 1, false) - above(q, false)) - 1);
          if (c.key > cut.key || (c.key == cut.key && c.index < cut.index)) cut = c;
        }
      }
    }
  }

  // ----------------------------------------------------------------- the draw
  // min_p above 1 leaves the first of the largest: they are what is kept, and the draw takes its lowest
  const bool only_first = !(min_p <= 1.0f);
  if (only_first) cut = {sp_key(mx), INT32_MAX};
  const u64 least = (u64)ceil((double)fmaxf(fminf(min_p, 1.0f), 0.0f) * (double)SP_ONE);
  // (key 0 is below every logit's)
  const float edge = cut.key == 0u ? -INFINITY : logit_of(cut.key);
  auto kept = [&](float v, int index) -> u64 {
    if (!(v > edge || (v == edge && index <= cut.index))) return 0ull;
    const u64 w = weight(v);
    return w >= least ? w : 0ull;
  };
  u64 own = 0;
  if (cut.key == 0u) {
    each(
        [&](float v) {
          const u64 w = weight(v);
          own += w >= least ? w : 0ull;
          return false;
        },
        [](float, int) {});
  } else {
    each_near(mx - edge <= near_reach, [&](float v) { return v >= edge; }, [&](float v, int index) { own += kept(v, index); });
  }
  const Before s = row_scan(own);  // its barrier is behind the last access to another CTA's memory
  const u64 target = only_first ? 0 : min((u64)floor((double)a.u[r] * (double)s.total), s.total - 1);
  row_find(s, target, kept, [&](float v, int index) {
    a.tokens[r] = index;
    if (a.logprobs) a.logprobs[r] = (v - mx) / temp - logz;
  });
}

// A row is held by a cluster of CTAs of 512 threads, two to an SM, or streamed by CTAs of 1024 threads, one to an SM.
// Times in us with top_k and top_p, bf16, held / streamed by 1, 2, 4 CTAs:
//   rows x V      16 x 100003         36 x 100003        64 x 32000         64 x 131072        148 x 131072
//                 29 / 60, 43, 37     46 / 58, 43, 62    37 / 34, 35, 47    59 / 55, 39, 58    130 / 61, 75
// Held is the shortest way while few CTAs are needed (up to 128; rows that one CTA holds always: 148 x 8000 31 / 33):
// the row is read once, at the price of less room for anything else.  Then as many CTAs hold a row as there is room for, but at most 8
// unless it needs more, since every exchange over the cluster costs about a microsecond.  Streamed rows get a cluster
// while all of them run at the same time; from 196608 logits on two CTAs in any case, since the lists of one do not
// hold the logits near the maximum (148 x 256000: 149 / 127 us with 1 / 2).
template <int DT>
int launch_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int VEC = DT == FP4_DT_F32 ? 4 : 8;
  // a row can begin VEC - 1 logits past a 16-byte boundary
  const bool aligned = (uintptr_t)a.logits % 16 == 0 && (a.ld % VEC == 0 || a.R == 1);
  const int n = a.V + (aligned ? 0 : VEC - 1);
  const int most = DT == FP4_DT_F32 ? 16384 : 28672;  // 64 or 56 KB: two CTAs on an SM
  int C = 1;
  while (C < SP_RANKS && C * most < n) C *= 2;
  const bool stream = C > 1 && (int64_t)a.R * C > 128;
  if (stream) {
    C = a.R <= 32 ? 4 : a.R <= 64 || n > 196608 ? 2 : 1;
  } else
    while (C < 8 && (int64_t)a.R * C * 2 <= 296 && C * 4096 < n) C *= 2;
  const int threads = stream ? SP_STREAM_THREADS : SP_HELD_THREADS;
  const int per_load = C * threads * VEC, loads = (n + per_load - 1) / per_load;
  const size_t smem = sizeof(SampleShared) + (stream ? (size_t)32 * SP_NEAR * 8 : (size_t)loads * threads * 16);
  auto* fn = !stream ? sample_kernel<DT, false, false> : C == 1 ? sample_kernel<DT, true, true> : sample_kernel<DT, true, false>;
  if (int e = set_smem_attr((const void*)fn, (int)sizeof(SampleShared) + (stream ? 32 * SP_NEAR * 8 : 73728), true)) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.R * C)), cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, fn, a, loads);
  return check_launch("sample_kernel");
}

// A warp per row: node by node, the children's tokens are compared 32 at a time.
__global__ void __launch_bounds__(128) accept_tree_kernel(const int32_t* parents, const int64_t* tokens,
                                                          const int64_t* sampled, const int32_t* counts, int B, int N,
                                                          int32_t* keep, int32_t* n, int64_t* next) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (b >= B) return;
  const int c = counts ? max(0, min(counts[b], N)) : N;
  const int64_t at = (int64_t)b * N;
  int cur = c > 0 ? 0 : -1, m = 0;
  int64_t want = -1;
  while (cur >= 0) {
    if (lane == 0) keep[at + m] = cur;
    ++m;
    want = sampled[at + cur];
    int found = -1;
    for (int j0 = cur + 1; j0 < c && found < 0; j0 += 32) {
      const int j = j0 + lane;
      const unsigned hit = __ballot_sync(0xffffffffu, j < c && parents[at + j] == cur && tokens[at + j] == want);
      if (hit) found = j0 + __ffs(hit) - 1;
    }
    cur = found;
  }
  for (int j = m + lane; j < N; j += 32) keep[at + j] = N - 1;
  if (lane == 0) n[b] = m, next[b] = want;
}

}  // namespace
}  // namespace fp4

using namespace fp4;

extern "C" int fp4_sample(const void* logits, int in_dtype, int R, int V, int64_t ld, const float* u,
                          const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                          int64_t* tokens, float* logprobs, void* stream) {
  clear_error();
  if (R < 0 || V <= 0 || ld < 0) return set_error(FP4ATTN_ERR_ARG, "bad shape");
  if ((int64_t)R * 16 > INT32_MAX) return set_error(FP4ATTN_ERR_UNSUPPORTED, "too many rows");
  if (V > SP_MAX_V) return set_error(FP4ATTN_ERR_UNSUPPORTED, "more than %d logits in a row", SP_MAX_V);
  if (R == 0) return FP4ATTN_OK;
  if (!logits || !u || !tokens) return set_error(FP4ATTN_ERR_ARG, "null pointer");
  const SampleArgs a{logits, R, V, ld, u, temperature, top_k, top_p, min_p, tokens, logprobs};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (in_dtype) {
    case FP4_DT_F32: return launch_sample<FP4_DT_F32>(a, st);
    case FP4_DT_BF16: return launch_sample<FP4_DT_BF16>(a, st);
    case FP4_DT_F16: return launch_sample<FP4_DT_F16>(a, st);
  }
  return set_error(FP4ATTN_ERR_ARG, "bad in_dtype");
}

extern "C" int fp4_accept_tree(const int32_t* parents, const int64_t* tokens, const int64_t* sampled,
                               const int32_t* counts, int B, int N, int32_t* keep, int32_t* n, int64_t* next,
                               void* stream) {
  clear_error();
  if (B < 0 || N <= 0) return set_error(FP4ATTN_ERR_ARG, "bad shape");
  if (B == 0) return FP4ATTN_OK;
  if (!parents || !tokens || !sampled || !keep || !n || !next) return set_error(FP4ATTN_ERR_ARG, "null pointer");
  accept_tree_kernel<<<(B + 3) / 4, 128, 0, reinterpret_cast<cudaStream_t>(stream)>>>(parents, tokens, sampled, counts,
                                                                                   B, N, keep, n, next);
  return check_launch("accept_tree_kernel");
}
