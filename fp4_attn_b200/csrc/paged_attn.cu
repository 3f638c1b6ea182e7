// paged_attn.cu -- attention of the drafted tokens (the last N of each
// sequence) over the paged NVFP4 cache.
#include <stdint.h>

#include <algorithm>

#include "paged.cuh"
#include "status.h"

namespace fp4 {

int paged_check(const fp4paged_cache* c, int B, const int32_t* seqs);

namespace {

struct AttnArgs {
  fp4paged_cache c;
  const uint8_t* q_codes;   // [B*N][Hq*D/2]
  const uint8_t* q_scales;  // [B*N][Hq*D/16]
  const float* q_g;         // [B*N]
  const uint8_t* mask;
  int64_t m_sB, m_sI, m_sJ;
  const int32_t *counts, *seqs;
  int B, Hq, N;
  float scaling;
  void* out;
};

// q, a warp per token
template <int DT, bool VEC, int NB>
__global__ void __launch_bounds__(256) paged_quant_q_kernel(const void* q, int B, int Hq, int N, int64_t sB, int64_t sH,
                                                            int64_t sT, uint8_t* codes, uint8_t* scales, float* g) {
  using E = typename In<DT>::T;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (id >= (int64_t)B * N) return;
  const E* x = static_cast<const E*>(q) + (id / N) * sB + (id % N) * sT;
  const int64_t row = id * Hq;
  const float gv = pg_quantize_token<DT, VEC, NB>(
      Hq * PG_SF, [&](int i) { return x + (i >> 3) * sH + (i & 7) * 16; },
      [&](int i, uint2 v, uint32_t s) {
        *reinterpret_cast<uint2*>(codes + row * PG_ROW + i * 8) = v;
        scales[row * PG_SF + i] = (uint8_t)s;
      });
  if ((threadIdx.x & 31) == 0) g[id] = gv;
}

// Two values of a byte of codes under a scale.
__device__ __forceinline__ float2 pair_value(uint32_t byte, float s) {
  return make_float2(e2m1_value(byte & 15u) * s, e2m1_value((byte >> 4) & 15u) * s);
}

// The simplest form: a block of four warps per (head, node, row), each warp every fourth key; a lane holds
// channels 4 lane .. 4 lane + 3; running maximum and sum, joined over the warps at the end.
template <int DT>
__global__ void __launch_bounds__(128) paged_attn_simple_kernel(AttnArgs a) {
  __shared__ float sm_m[4], sm_l[4], sm_o[4][PG_D];
  const fp4paged_cache& c = a.c;
  const int hq = blockIdx.x, i = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = c.num_kv_heads, h = hq / (a.Hq / H), P = c.page_size;
  const int s = pg_seq(c, a.seqs, b);
  const int n = a.counts ? max(0, min(a.counts[b], a.N)) : a.N;
  const int len = s < 0 || i >= n ? 0 : c.lens[s], base = len - n;
  const int64_t tok = (int64_t)b * a.N + i, qrow = tok * a.Hq + hq;
  const float gq = a.q_g[tok];
  const float qs = e4m3_to_f32(a.q_scales[qrow * PG_SF + lane / 4]);
  const uint32_t qc = reinterpret_cast<const uint16_t*>(a.q_codes)[qrow * (PG_ROW / 2) + lane];
  const float2 q0 = pair_value(qc & 255u, qs), q1 = pair_value(qc >> 8, qs);
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int t = warp; t < len; t += 4) {
    const int j = t - base;
    if (j >= 0 && !(a.mask ? a.mask[b * a.m_sB + i * a.m_sI + j * a.m_sJ] != 0 : j <= i)) continue;
    const int64_t page = c.page_table[(int64_t)s * c.max_pages + t / P];
    const int64_t row = (page * H + h) * P + t % P;
    const uint32_t kc = reinterpret_cast<const uint16_t*>(c.k_codes)[row * (PG_ROW / 2) + lane];
    const float ks = e4m3_to_f32(c.k_scales[row * PG_SF + lane / 4]);
    const float2 k0 = pair_value(kc & 255u, ks), k1 = pair_value(kc >> 8, ks);
    float x = q0.x * k0.x + q0.y * k0.y + q1.x * k1.x + q1.y * k1.y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    x = x * gq * c.k_g[page * P + t % P] * a.scaling;
    const float mn = nanmax(m, x), f = m == mn ? 1.0f : __expf(m - mn), p = x == mn ? 1.0f : expf(x - mn);
    const uint32_t vc = reinterpret_cast<const uint16_t*>(c.v_codes)[row * (PG_ROW / 2) + lane];
    const float vs = e4m3_to_f32(c.v_scales[row * PG_SF + lane / 4]) * c.v_g[page * P + t % P];
    const float2 v0 = pair_value(vc & 255u, vs), v1 = pair_value(vc >> 8, vs);
    o[0] = o[0] * f + p * v0.x, o[1] = o[1] * f + p * v0.y, o[2] = o[2] * f + p * v1.x, o[3] = o[3] * f + p * v1.y;
    l = l * f + p;
    m = mn;
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
#pragma unroll
  for (int d = 0; d < 4; ++d) sm_o[warp][4 * lane + d] = o[d];
  __syncthreads();
  float mx = sm_m[0], lt = 0.0f, ot = 0.0f;
#pragma unroll
  for (int w = 1; w < 4; ++w) mx = nanmax(mx, sm_m[w]);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (sm_l[w] == 0.0f) continue;
    const float f = expf(sm_m[w] - mx);
    lt += sm_l[w] * f, ot += sm_o[w][threadIdx.x] * f;
  }
  store_out<DT>(a.out, (tok * a.Hq + hq) * PG_D + threadIdx.x, lt == 0.0f ? 0.0f : ot / lt);
}

template <int DT>
int launch_quant_q(const void* q, const AttnArgs& a, int64_t sB, int64_t sH, int64_t sT, cudaStream_t st) {
  const unsigned grid = (unsigned)(((int64_t)a.B * a.N + 7) / 8);
  const int64_t esz = DT == FP4_DT_F32 ? 4 : 2;
  const bool vec = (uintptr_t)q % 16 == 0 && (sB * esz % 16 == 0 || a.B == 1) && (sT * esz % 16 == 0 || a.N == 1) &&
                   (sH * esz % 16 == 0 || a.Hq == 1);
  uint8_t *codes = const_cast<uint8_t*>(a.q_codes), *scales = const_cast<uint8_t*>(a.q_scales);
  float* g = const_cast<float*>(a.q_g);
  if (!vec) paged_quant_q_kernel<DT, false, 0><<<grid, 256, 0, st>>>(q, a.B, a.Hq, a.N, sB, sH, sT, codes, scales, g);
  else if (a.Hq * PG_SF <= 64)
    paged_quant_q_kernel<DT, true, 2><<<grid, 256, 0, st>>>(q, a.B, a.Hq, a.N, sB, sH, sT, codes, scales, g);
  else paged_quant_q_kernel<DT, true, 0><<<grid, 256, 0, st>>>(q, a.B, a.Hq, a.N, sB, sH, sT, codes, scales, g);
  return check_launch("paged_quant_q_kernel");
}

}  // namespace
}  // namespace fp4

using namespace fp4;

static int64_t q_piece(int64_t bytes) { return (bytes + 255) / 256 * 256; }

extern "C" int64_t fp4paged_attention_workspace_size(int B, int Hq, int Hkv, int N) {
  if (B <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return -1;
  const int64_t rows = (int64_t)B * N;
  return q_piece(rows * Hq * PG_ROW) + q_piece(rows * Hq * PG_SF) + q_piece(rows * 4);
}

extern "C" int fp4paged_attention(const fp4paged_cache* cache, const void* q, int in_dtype, int B, int Hq, int N,
                                  int64_t q_sB, int64_t q_sH, int64_t q_sT, const uint8_t* mask, int64_t m_sB,
                                  int64_t m_sI, int64_t m_sJ, const int32_t* counts, const int32_t* seqs,
                                  float scaling, void* out, int out_dtype, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  if (N < 0 || Hq <= 0 || Hq % cache->num_kv_heads)
    return set_error(FP4ATTN_ERR_ARG, "bad shape: %d query heads, %d KV heads", Hq, cache->num_kv_heads);
  if (B == 0 || N == 0) return FP4ATTN_OK;
  if (!q || !out || !workspace) return set_error(FP4ATTN_ERR_ARG, "null pointer");
  if (in_dtype < 0 || in_dtype > 2 || out_dtype < 0 || out_dtype > 2) return set_error(FP4ATTN_ERR_ARG, "bad dtype");
  const int64_t need = fp4paged_attention_workspace_size(B, Hq, cache->num_kv_heads, N);
  if ((uintptr_t)workspace % 256 || workspace_bytes < need)
    return set_error(FP4ATTN_ERR_ARG, "workspace of %lld bytes, %lld needed (256-byte aligned)",
                     (long long)workspace_bytes, (long long)need);
  const int64_t rows = (int64_t)B * N;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.c = *cache;
  a.q_codes = w;
  a.q_scales = w + q_piece(rows * Hq * PG_ROW);
  a.q_g = reinterpret_cast<float*>(w + q_piece(rows * Hq * PG_ROW) + q_piece(rows * Hq * PG_SF));
  a.mask = mask, a.m_sB = m_sB, a.m_sI = m_sI, a.m_sJ = m_sJ;
  a.counts = counts, a.seqs = seqs;
  a.B = B, a.Hq = Hq, a.N = N, a.scaling = scaling, a.out = out;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int e = in_dtype == FP4_DT_F32    ? launch_quant_q<FP4_DT_F32>(q, a, q_sB, q_sH, q_sT, st)
          : in_dtype == FP4_DT_BF16 ? launch_quant_q<FP4_DT_BF16>(q, a, q_sB, q_sH, q_sT, st)
                                    : launch_quant_q<FP4_DT_F16>(q, a, q_sB, q_sH, q_sT, st);
  if (e) return e;
  const dim3 grid(Hq, N, B);
  if (out_dtype == FP4_DT_F32) paged_attn_simple_kernel<FP4_DT_F32><<<grid, 128, 0, st>>>(a);
  else if (out_dtype == FP4_DT_BF16) paged_attn_simple_kernel<FP4_DT_BF16><<<grid, 128, 0, st>>>(a);
  else paged_attn_simple_kernel<FP4_DT_F16><<<grid, 128, 0, st>>>(a);
  return check_launch("paged_attn_simple_kernel");
}
