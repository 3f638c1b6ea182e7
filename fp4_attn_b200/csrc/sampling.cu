// sampling.cu -- sampling from logits with given random numbers, and the walk
// that accepts drafted tokens.
//
// Weights w = exp((x - max) / T) are rounded to whole multiples of 2^-34: every
// sum is then an exact 64-bit integer sum, the same for any split of a row.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "common.cuh"
#include "fp4attn.h"
#include "status.h"

namespace fp4 {
namespace {

constexpr int SP_MAX_V = 262144;
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

constexpr int SS_THREADS = 1024;

template <typename T>
__device__ __forceinline__ T ss_sum(T v, T* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The simplest form: a block per row that reads the row once for every bit of a threshold.
template <int DT>
__global__ void __launch_bounds__(SS_THREADS) sample_simple_kernel(SampleArgs a) {
  using E = typename In<DT>::T;
  __shared__ u64 part[32];
  __shared__ float fpart[32];
  const int r = blockIdx.x, tid = threadIdx.x;
  const E* row = static_cast<const E*>(a.logits) + (int64_t)r * a.ld;
  auto at = [&](int i) { return sp_clean(In<DT>::f(row[i])); };
  float m = -INFINITY;
  for (int i = tid; i < a.V; i += SS_THREADS) m = fmaxf(m, at(i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((tid & 31) == 0) fpart[tid >> 5] = m;
  __syncthreads();
  m = fpart[tid & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m == -INFINITY) {
    if (tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }
  const float t0 = a.temperature ? a.temperature[r] : 1.0f, T = t0 > 0.0f ? t0 : 1.0f;
  auto weight = [&](float x) -> u64 {
    return x == -INFINITY ? 0ull : __float2ull_rn(expf((x - m) / T) * SP_ONE);
  };
  u64 z = 0;
  for (int i = tid; i < a.V; i += SS_THREADS) z += weight(at(i));
  z = ss_sum(z, part);
  // kept: key > K, or key == K and one of the first `ties` of that key in index order
  uint32_t K = 0;
  int ties = a.V;
  const int k = t0 > 0.0f ? (a.top_k ? a.top_k[r] : 0) : 1;
  const float tp = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? a.min_p[r] : 0.0f;
  auto above = [&](uint32_t key, bool mass, uint32_t low, int lties) {  // mass or count of keys > key, kept before
    u64 s = 0;
    for (int i = tid; i < a.V; i += SS_THREADS) {
      const uint32_t q = sp_key(at(i));
      if (q > key) s += mass ? weight(at(i)) : 1ull;
    }
    (void)low, (void)lties;
    return ss_sum(s, part);
  };
  auto equal = [&](uint32_t key) {
    u64 s = 0;
    for (int i = tid; i < a.V; i += SS_THREADS) s += sp_key(at(i)) == key;
    return ss_sum(s, part);
  };
  auto find = [&](bool mass, double target) {  // largest key with mass or count of keys >= key reaching the target
    uint32_t lo = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = lo | (1u << bit);
      if ((double)above(c - 1, mass, 0, 0) >= target) lo = c;
    }
    return lo;
  };
  if (k > 0 && k < a.V) {
    K = find(false, (double)k);
    ties = k - (int)above(K, false, 0, 0);
  }
  auto key_weight = [&](uint32_t key) {
    return weight(__uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key));
  };
  if (t0 > 0.0f && tp < 1.0f) {
    const u64 ge = above(K, true, 0, 0);
    const u64 n_eq = equal(K);
    const u64 mass = ge + (u64)min((u64)ties, n_eq) * key_weight(K);
    const double target = (double)tp * (double)mass;
    // shortest prefix whose earlier members sum to less than the target
    const uint32_t Kp = max(find(true, target), K);
    const u64 before = above(Kp, true, 0, 0), w = key_weight(Kp);
    int q = Kp == K ? ties : a.V;
    if ((double)before >= target) {
      q = 0;
    } else if (w > 0) {
      int n = 0;  // members of Kp whose predecessors sum to less than the target
      const int most = (int)min((u64)q, equal(Kp));
      int lo = 0, hi = most;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if ((double)(before + (u64)mid * w) < target) lo = mid + 1; else hi = mid;
      }
      n = lo;
      q = min(q, n);
    }
    K = Kp, ties = q;
  }
  const double wmin = t0 > 0.0f ? (double)mp * (double)SP_ONE : 0.0;
  const uint32_t top = sp_key(m);
  if (K > top || (K == top && ties < 1)) K = top, ties = 1;
  // index order: count ties, sum kept weights, then find the crossing
  __shared__ u64 s_w[SS_THREADS];
  __shared__ int s_t[SS_THREADS];
  const int chunk = (a.V + SS_THREADS - 1) / SS_THREADS, i0 = tid * chunk, i1 = min(a.V, i0 + chunk);
  int nt = 0;
  for (int i = i0; i < i1; ++i) nt += sp_key(at(i)) == K;
  s_t[tid] = nt;
  __syncthreads();
  int seen = 0;
  for (int j = 0; j < tid; ++j) seen += s_t[j];
  const int seen0 = seen;
  u64 w = 0;
  auto kept = [&](int i, int& seen) -> u64 {
    const float x = at(i);
    const uint32_t q = sp_key(x);
    bool ok = q > K;
    if (q == K) ok = seen++ < ties;
    const u64 v = weight(x);
    return ok && (((double)v >= wmin) || q == top) ? v : 0ull;
  };
  for (int i = i0; i < i1; ++i) w += kept(i, seen);
  s_w[tid] = w;
  __syncthreads();
  const u64 total = ss_sum(w, part);
  u64 target = (u64)floor((double)a.u[r] * (double)total);
  target = min(target, total - 1);
  u64 before = 0;
  for (int j = 0; j < tid; ++j) before += s_w[j];
  if (before <= target && before + w > target) {
    seen = seen0;
    for (int i = i0; i < i1; ++i) {
      before += kept(i, seen);
      if (before > target) {
        a.tokens[r] = i;
        if (a.logprobs) a.logprobs[r] = (at(i) - m) / T - (float)log((double)z / (double)SP_ONE);
        break;
      }
    }
  }
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
  if (V > SP_MAX_V) return set_error(FP4ATTN_ERR_UNSUPPORTED, "more than %d logits in a row", SP_MAX_V);
  if (R == 0) return FP4ATTN_OK;
  if (!logits || !u || !tokens) return set_error(FP4ATTN_ERR_ARG, "null pointer");
  const SampleArgs a{logits, R, V, ld, u, temperature, top_k, top_p, min_p, tokens, logprobs};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (in_dtype) {
    case FP4_DT_F32: sample_simple_kernel<FP4_DT_F32><<<R, SS_THREADS, 0, st>>>(a); break;
    case FP4_DT_BF16: sample_simple_kernel<FP4_DT_BF16><<<R, SS_THREADS, 0, st>>>(a); break;
    case FP4_DT_F16: sample_simple_kernel<FP4_DT_F16><<<R, SS_THREADS, 0, st>>>(a); break;
    default: return set_error(FP4ATTN_ERR_ARG, "bad in_dtype");
  }
  return check_launch("sample_simple_kernel");
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
