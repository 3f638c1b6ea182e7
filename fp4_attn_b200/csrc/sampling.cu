// sampling.cu -- sampling from logits with given random numbers, and the walk
// that accepts drafted tokens.
//
// Weights w = exp((x - max) / T) are rounded to whole multiples of 2^-34 of the
// largest: every sum is then an exact integer sum, the same for any split of a
// row, and a result depends neither on the grid nor on an order of atomics.
//
// A row is read once: a cluster of CTAs holds it in shared memory (up to 16384
// logits a CTA, in their own type), and everything after that -- the maximum, the sum, the
// thresholds of top-k and top-p, the draw -- works on chip, with what the CTAs
// have to tell each other in distributed shared memory.  No sort: a histogram
// over x finds the bin that the threshold falls into, and only that bin's few
// logits are ranked.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

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

// NaN counts as -inf, +inf as the largest finite value.
__device__ __forceinline__ float sp_clean(float x) { return x != x ? -INFINITY : fminf(x, 3.402823466e38f); }

// Larger keys for larger logits (-0 below +0 would split equal logits: + 0 first).
__device__ __forceinline__ uint32_t sp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b >> 31) ? ~b : b | 0x80000000u;
}

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32;
constexpr int SP_BINS = 1024;   // of x's distance from the maximum
constexpr int SP_LIST = 1024;   // logits of a bin that are ranked directly; more of them are searched bit by bit
constexpr int SP_RANKS = 16;    // CTAs of a cluster
constexpr int SP_LIMB = 17;     // a weight as two parts of 17 bits: up to 32767 of either add up within 32 bits

// The last kept logit in the order (x descending, index ascending).
struct Cut {
  uint32_t key;
  int index;
};

// What the leader (rank 0) tells the cluster to do next.
enum : int { SP_DONE = 0, SP_GATHER = 1, SP_WIDER = 2, SP_SEARCH = 3 };
struct Plan {
  int what, bin, pad[2];
  Cut cut;
};

struct SampleShared {
  uint32_t count[SP_BINS], lo[SP_BINS], hi[SP_BINS];  // this CTA's histogram
  // leader: the row's
  uint32_t total[SP_BINS];
  u64 mass[SP_BINS];
  uint32_t list_key[SP_LIST];
  int list_index[SP_LIST];
  u64 list_w[SP_LIST];
  int listed;
  Plan plan;
  float rank_max[SP_RANKS], rank_min[SP_RANKS];
  u64 rank_sum[4][SP_RANKS];  // by turns; each slot is written anew only two barriers after it was read
  int rank_first[SP_RANKS];
  u64 warp_sum[SP_WARPS];
  u64 part[SP_WARPS];
  float fpart[2][SP_WARPS];
};

template <typename T>
__device__ __forceinline__ T sp_block_sum(T v, T* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & (SP_WARPS - 1)];
#pragma unroll
  for (int o = SP_WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The first bin at which the running sum of v (SP_BINS / SP_THREADS bins a thread) reaches `target`, and the sum before
// it; SP_BINS if it never does.
template <typename T>
__device__ __forceinline__ int sp_find_bin(const T* v, double target, T* part, int* found, u64* before) {
  constexpr int PER = SP_BINS / SP_THREADS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  T own[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += own[i] = v[threadIdx.x * PER + i];
  T inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const T u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  if (threadIdx.x == 0) *found = SP_BINS;
  __syncthreads();
  T at = inc - sum;
  for (int i = 0; i < warp; ++i) at += part[i];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if ((double)at < target && (double)(at + own[i]) >= target) *found = threadIdx.x * PER + i, *before = (u64)at;
    at += own[i];
  }
  __syncthreads();
  return *found;
}

template <int DT>
__global__ void __launch_bounds__(SP_THREADS) sample_kernel(SampleArgs a, int loads) {
  using T = typename In<DT>::T;
  constexpr int VEC = 16 / (int)sizeof(T);
  namespace cg = cooperative_groups;
  extern __shared__ __align__(16) uint8_t smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  uint4* held = reinterpret_cast<uint4*>(smem + sizeof(SampleShared));  // [warp][loads][lane]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  SampleShared& lead = *cluster.map_shared_rank(&sh, 0);
  const int r = (int)(blockIdx.x / C), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // A warp holds consecutive positions, VEC per lane and load.  Positions count from the 16-byte boundary at or below
  // the row, so that loads are aligned whatever the row's start.
  const T* row = static_cast<const T*>(a.logits) + (int64_t)r * a.ld;
  const int skip = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(row - skip);
  const int pos0 = ((rank * SP_WARPS + warp) * loads * 32 + lane) * VEC, end = a.V + skip;
  uint4* mine = held + warp * loads * 32 + lane;  // only this thread's
  const T none = In<DT>::t(-INFINITY);
#pragma unroll 4
  for (int j = 0; j < loads; ++j) {
    const int pos = pos0 + j * 32 * VEC;
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    if (pos < end) raw = __ldg(base + pos / VEC);
    T* t = reinterpret_cast<T*>(&raw);
    if (pos < skip || pos + VEC > end)
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = pos + i >= skip && pos + i < end ? t[i] : none;
    mine[j * 32] = raw;
  }
  // calls fn(x, index) for this thread's logits of load j, in order
  auto load = [&](int j, auto fn) {
    const uint4 raw = mine[j * 32];
    const int index = pos0 + j * 32 * VEC - skip;
#pragma unroll
    for (int i = 0; i < VEC; ++i) fn(sp_clean(In<DT>::f(reinterpret_cast<const T*>(&raw)[i])), index + i);
  };
  auto each = [&](auto fn) {
#pragma unroll 2
    for (int j = 0; j < loads; ++j) load(j, fn);
  };

  // --------------------------------------------------------- maximum, minimum
  float mx = -INFINITY, mn = INFINITY;
  each([&](float v, int) { mx = fmaxf(mx, v), mn = fminf(mn, v == -INFINITY ? INFINITY : v); });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
  }
  if (lane == 0) sh.fpart[0][warp] = mx, sh.fpart[1][warp] = mn;
  for (int i = tid; i < SP_BINS; i += SP_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
  if (tid == 0) sh.listed = 0;
  __syncthreads();
  if (warp == 0) {
    mx = sh.fpart[0][lane & (SP_WARPS - 1)], mn = sh.fpart[1][lane & (SP_WARPS - 1)];
#pragma unroll
    for (int o = SP_WARPS / 2; o > 0; o >>= 1) {
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
    }
    if (lane < C) {  // to every CTA
      SampleShared& to = *cluster.map_shared_rank(&sh, lane);
      to.rank_max[rank] = mx, to.rank_min[rank] = mn;
    }
  }
  cluster.sync();
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
  const bool greedy = !(t0 > 0.0f);
  const int k = a.top_k ? a.top_k[r] : 0;
  const float top_p = a.top_p ? a.top_p[r] : 1.0f, min_p = a.min_p ? a.min_p[r] : 0.0f;
  const bool by_k = !greedy && k > 0 && k < a.V, by_p = !greedy && top_p < 1.0f;
  // w = 2^((x - max) log2(e) / T): the factor in two parts, so that the product is rounded once
  const double f = 1.4426950408889634 / (double)temp;
  const float f1 = (float)f, f2 = (float)(f - (double)f1);
  auto weight = [&](float v) -> u64 {
    const float d = v - mx;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaxf(fmaf(d, f1, d * f2), -150.0f)));  // (NaN: both parts infinite)
    return v == -INFINITY ? 0ull : __float2ull_rn(e * SP_ONE);
  };
  int turn = 0;
  // The cluster's sum of a number per thread.
  auto cluster_sum = [&](u64 v) -> u64 {
    v = sp_block_sum(v, sh.part);
    if (tid < C) cluster.map_shared_rank(&sh, tid)->rank_sum[turn & 3][rank] = v;
    cluster.sync();
    u64 sum = 0;
    for (int i = 0; i < C; ++i) sum += sh.rank_sum[turn & 3][i];
    ++turn;
    return sum;
  };

  // ------------------------------------------------- sum, first largest logit
  u64 z = 0;
  int first = INT32_MAX;
  each([&](float v, int index) {
    z += weight(v);
    if (v == mx) first = min(first, index);
  });
  first = __reduce_min_sync(0xffffffffu, first);
  if (lane == 0) sh.list_index[warp] = first;  // (the list is not in use yet)
  z = sp_block_sum(z, sh.part);
  if (tid < C) {
    int m = INT32_MAX;
    for (int i = 0; i < SP_WARPS; ++i) m = min(m, sh.list_index[i]);
    SampleShared& to = *cluster.map_shared_rank(&sh, tid);
    to.rank_sum[3][rank] = z, to.rank_first[rank] = m;
  }
  // the histogram of what can hold the thresholds: first the logits within 10 T of the maximum
  const float full = fminf(24.6f * temp, mx - mn);  // weights further away are 0
  float reach = fminf(10.0f * temp, full);
  auto bin_of = [&](float v, float per) { return min(SP_BINS - 1, (int)((mx - v) * per)); };
  auto histogram = [&](float per) {
    each([&](float v, int) {
      if (mx - v <= reach) {
        const int b = bin_of(v, per);
        const u64 w = weight(v);
        atomicAdd(&sh.count[b], 1u);
        atomicAdd(&sh.lo[b], (uint32_t)w & ((1u << SP_LIMB) - 1));
        atomicAdd(&sh.hi[b], (uint32_t)(w >> SP_LIMB));
      }
    });
  };
  float per = reach > 0.0f ? (float)SP_BINS / reach : 0.0f;
  if (by_k || by_p) histogram(per);
  cluster.sync();
  z = 0;
  first = INT32_MAX;
  for (int i = 0; i < C; ++i) z += sh.rank_sum[3][i], first = min(first, sh.rank_first[i]);
  const float logz = logf((float)((double)z / (double)SP_ONE));
  if (greedy) {
    if (rank == 0 && tid == 0) {
      a.tokens[r] = first;
      if (a.logprobs) a.logprobs[r] = -logz;
    }
    cluster.sync();  // no CTA leaves while another may still write to it
    return;
  }

  Cut cut{0u, INT32_MAX};
  // Kept so far: everything down to the cut.
  auto within = [&](uint32_t q, int index) { return q > cut.key || (q == cut.key && index <= cut.index); };

  // what has to go before a logit for top_p to drop it; the first always stays
  auto p_target = [&](u64 mass) { return fmax((double)top_p * (double)mass, 1.0); };

  if (by_k || by_p) {
    bool k_done = !by_k;  // the leader's: top_k is settled
    u64 kept_mass = z;    // and what it leaves
    for (;;) {
      // the row's histogram, a share of the bins per CTA
      const int share = SP_BINS / C;
      for (int i = rank * share + tid; i < (rank + 1) * share; i += SP_THREADS) {
        uint32_t n = 0;
        u64 lo = 0, hi = 0;
        for (int c = 0; c < C; ++c) {
          const SampleShared& from = *cluster.map_shared_rank(&sh, c);
          n += from.count[i], lo += from.lo[i], hi += from.hi[i];
        }
        lead.total[i] = n, lead.mass[i] = lo + (hi << SP_LIMB);
      }
      cluster.sync();
      // the leader finds the bin
      auto choose = [&]() {
        __shared__ int found;
        __shared__ u64 before;
        Plan p{SP_DONE, 0, {0, 0}, cut};
        int b = SP_BINS;
        if (!k_done) {
          b = sp_find_bin(sh.total, (double)k, reinterpret_cast<uint32_t*>(sh.part), &found, &before);
          if (b == SP_BINS && reach < full) {
            p.what = SP_WIDER;
            return p;
          }
          if (b == SP_BINS) k_done = true;  // fewer than k weights are not 0
        }
        if (k_done) {
          if (!by_p) return p;
          b = sp_find_bin(sh.mass, p_target(kept_mass), sh.part, &found, &before);
        }
        // (the full reach has all of the mass)
        if (b == SP_BINS) p.what = reach < full ? SP_WIDER : SP_SEARCH;
        else p.what = sh.total[b] <= SP_LIST ? SP_GATHER : SP_SEARCH, p.bin = b;
        return p;
      };
      auto tell = [&](const Plan& p) {
        if (tid < C) cluster.map_shared_rank(&sh, tid)->plan = p;
        if (tid == 0) sh.listed = 0;
      };
      if (rank == 0) tell(choose());
      cluster.sync();
      while (sh.plan.what == SP_GATHER) {
        const int bin = sh.plan.bin;
        each([&](float v, int index) {
          if (mx - v <= reach && bin_of(v, per) == bin) {
            const int at = atomicAdd(&lead.listed, 1);
            if (at < SP_LIST) lead.list_key[at] = sp_key(v), lead.list_index[at] = index, lead.list_w[at] = weight(v);
          }
        });
        cluster.sync();
        if (rank == 0) {
          // rank the listed ones: how many, and how much, goes before each
          const int n = min(sh.listed, SP_LIST);
          u64 above_n = 0, above_w = 0;
          for (int i = tid; i < bin; i += SP_THREADS) above_n += sh.total[i], above_w += sh.mass[i];
          above_n = sp_block_sum(above_n, sh.part), above_w = sp_block_sum(above_w, sh.part);
          int at_n[SP_LIST / SP_THREADS];
          u64 at_w[SP_LIST / SP_THREADS];
#pragma unroll
          for (int t = 0; t < SP_LIST / SP_THREADS; ++t) {
            const int e = tid + t * SP_THREADS;
            at_n[t] = 0, at_w[t] = 0;
            if (e < n) {
              const uint32_t q = sh.list_key[e];
              const int id = sh.list_index[e];
              for (int i = 0; i < n; ++i)
                if (sh.list_key[i] > q || (sh.list_key[i] == q && sh.list_index[i] < id)) ++at_n[t], at_w[t] += sh.list_w[i];
            }
          }
          // the last one kept is the one with the most kept ones before it
          __shared__ int last;
          auto settle = [&](auto keeps) {
            __syncthreads();
            if (tid == 0) last = -1;
            __syncthreads();
#pragma unroll
            for (int t = 0; t < SP_LIST / SP_THREADS; ++t)
              if (tid + t * SP_THREADS < n && keeps(t)) atomicMax(&last, at_n[t]);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < SP_LIST / SP_THREADS; ++t)
              if (tid + t * SP_THREADS < n && at_n[t] == last) {
                sh.plan.cut = {sh.list_key[tid + t * SP_THREADS], sh.list_index[tid + t * SP_THREADS]};
                sh.part[0] = above_w + at_w[t] + sh.list_w[tid + t * SP_THREADS];
              }
            __syncthreads();
            cut = sh.plan.cut;
            const u64 mass = sh.part[0];
            __syncthreads();
            return mass;
          };
          if (!k_done) {
            kept_mass = settle([&](int t) { return above_n + at_n[t] < (u64)k; });
            k_done = true;
            if (by_p) {
              Plan p = choose();
              // (the mass up to the cut reaches the target, so the bin is this one or an earlier one)
              if (p.what == SP_GATHER && p.bin == bin) {
                const double target = p_target(kept_mass);
                settle([&](int t) { return above_n + at_n[t] < (u64)k && (double)(above_w + at_w[t]) < target; });
                p.what = SP_DONE, p.cut = cut;
              }
              tell(p);
            } else {
              tell({SP_DONE, 0, {0, 0}, cut});
            }
          } else {
            const double target = p_target(kept_mass);
            settle([&](int t) { return (double)(above_w + at_w[t]) < target; });
            tell({SP_DONE, 0, {0, 0}, cut});
          }
        }
        cluster.sync();
      }
      cut = sh.plan.cut;
      if (sh.plan.what != SP_WIDER) break;
      reach = full, per = (float)SP_BINS / reach;
      cluster.sync();  // (the histograms have been read)
      for (int i = tid; i < SP_BINS; i += SP_THREADS) sh.count[i] = sh.lo[i] = sh.hi[i] = 0u;
      __syncthreads();
      histogram(per);
      cluster.sync();
    }
    if (sh.plan.what == SP_SEARCH) {
      // Too many logits in one bin (flat rows): the thresholds bit by bit, on the logits in registers.
      cut = {0u, INT32_MAX};
      auto above = [&](uint32_t q, bool by_mass) {
        u64 s = 0;
        each([&](float v, int) {
          if (v != -INFINITY && sp_key(v) > q) s += by_mass ? weight(v) : 1ull;
        });
        return cluster_sum(s);
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
      // the index of the n-th (from 0) logit of key q
      auto nth = [&](uint32_t q, u64 n) {
        u64 own = 0;
        each([&](float v, int) { own += v != -INFINITY && sp_key(v) == q; });
        // before this warp: in lower CTAs and lower warps
        u64 w = own;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        __syncthreads();
        if (lane == 0) sh.warp_sum[warp] = w;
        __syncthreads();
        u64 block = 0, before = 0;
        for (int i = 0; i < SP_WARPS; ++i) block += sh.warp_sum[i], before += i < warp ? sh.warp_sum[i] : 0;
        if (tid < C) cluster.map_shared_rank(&sh, tid)->rank_sum[turn & 3][rank] = block;
        cluster.sync();
        for (int i = 0; i < rank; ++i) before += sh.rank_sum[turn & 3][i];
        ++turn;
        if (before <= n && n < before + w) {
          for (int j = 0; j < loads; ++j) {
            u64 here = 0;
            load(j, [&](float v, int) { here += v != -INFINITY && sp_key(v) == q; });
            u64 inc = here;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
              const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
              if (lane >= o) inc += u;
            }
            u64 at = before + inc - here;
            load(j, [&](float v, int index) {
              if (v != -INFINITY && sp_key(v) == q) {
                if (at == n)
                  for (int c = 0; c < C; ++c) cluster.map_shared_rank(&sh, c)->plan.cut = {q, index};
                ++at;
              }
            });
            before += __shfl_sync(0xffffffffu, inc, 31);
          }
        }
        cluster.sync();
        const Cut found = sh.plan.cut;
        cluster.sync();
        return found;
      };
      auto key_weight = [&](uint32_t q) { return weight(__uint_as_float(q & 0x80000000u ? q & 0x7fffffffu : ~q)); };
      u64 mass = z;
      if (by_k) {
        const u64 all = above(0u, false);
        if (all > (u64)k) {
          const uint32_t q = largest(false, (double)k);
          const u64 more = above(q, false);
          mass = above(q, true) + ((u64)k - more) * key_weight(q);
          cut = nth(q, (u64)k - more - 1);
        }
      }
      if (by_p) {
        const double target = p_target(mass);
        const uint32_t q = max(largest(true, target), cut.key);
        const u64 before = above(q, true), w = key_weight(q);
        // how many of key q have less than the target before them
        u64 n = 0;
        if (w > 0) {
          u64 lo = 0, hi = (u64)a.V;
          while (lo < hi) {
            const u64 mid = (lo + hi) / 2;
            if ((double)(before + mid * w) < target) lo = mid + 1; else hi = mid;
          }
          n = lo;
        }
        // none: the target is 0, or reached before q by the cut that top_k made
        if (n > 0) {
          const Cut c2 = nth(q, min(n, above(q - 1, false) - above(q, false)) - 1);
          if (c2.key > cut.key || (c2.key == cut.key && c2.index < cut.index)) cut = c2;
        } else if (before == 0) {
          cut = {sp_key(mx), first};
        }
      }
    }
    if (cut.key > sp_key(mx) || (cut.key == sp_key(mx) && cut.index < first)) cut = {sp_key(mx), first};
  }

  // ----------------------------------------------------------------- the draw
  const double least = (double)fminf(min_p, 1.0f) * (double)SP_ONE;
  auto kept = [&](float v, int index) -> u64 {
    if (v == -INFINITY || !within(sp_key(v), index)) return 0ull;
    const u64 w = weight(v);
    return (double)w >= least ? w : 0ull;
  };
  u64 own = 0;
  each([&](float v, int index) { own += kept(v, index); });
  u64 w = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
  __syncthreads();
  if (lane == 0) sh.warp_sum[warp] = w;
  __syncthreads();
  u64 block = 0, before = 0;
  for (int i = 0; i < SP_WARPS; ++i) block += sh.warp_sum[i], before += i < warp ? sh.warp_sum[i] : 0;
  if (tid < C) cluster.map_shared_rank(&sh, tid)->rank_sum[turn & 3][rank] = block;
  cluster.sync();  // the last access to another CTA's memory is behind this barrier
  u64 total = 0;
  for (int i = 0; i < C; ++i) {
    const u64 s = sh.rank_sum[turn & 3][i];
    total += s;
    if (i < rank) before += s;
  }
  const u64 target = min((u64)floor((double)a.u[r] * (double)total), total - 1);
  if (before <= target && target < before + w) {
    // this warp has it
    for (int j = 0; j < loads; ++j) {
      u64 here = 0;
      load(j, [&](float v, int index) { here += kept(v, index); });
      u64 inc = here;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const u64 u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      u64 at = before + inc - here;
      if (at <= target && target < at + here)
        load(j, [&](float v, int index) {
          const u64 w1 = kept(v, index);
          if (at <= target && target < at + w1) {
            a.tokens[r] = index;
            if (a.logprobs) a.logprobs[r] = (v - mx) / temp - logz;
          }
          at += w1;
        });
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

// CTAs of a row's cluster: enough for 16384 logits each (and a load more where the row is not aligned), more
// where rows are few: the card has 148 SMs, and a row's time is that of its slowest CTA.
template <int DT>
int launch_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int VEC = DT == FP4_DT_F32 ? 4 : 8;
  const int n = a.V + VEC - 1;  // a row can begin VEC - 1 logits past a 16-byte boundary
  int C = 1;
  while (C < SP_RANKS && C * 16384 < n) C *= 2;
  while (C < 8 && (int64_t)a.R * C < 148 && C * 4096 < n) C *= 2;
  const int per_load = C * SP_THREADS * VEC, loads = (n + per_load - 1) / per_load;
  const size_t smem = sizeof(SampleShared) + (size_t)loads * SP_THREADS * 16;
  if (int e = set_smem_attr((const void*)sample_kernel<DT>, (int)(sizeof(SampleShared) + 65536 + SP_THREADS * 16), true)) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.R * C)), cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)C, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, sample_kernel<DT>, a, loads);
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
