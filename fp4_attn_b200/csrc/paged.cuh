// paged.cuh -- what the kernels over the paged NVFP4 cache share: the token
// quantizer and the page lookup.
//
// A token is stored by itself (one row per token and KV head, blocks of 16
// along head_dim, one global scale g per token over all heads), so that it can
// be moved, shared and dropped without touching its neighbours.
#pragma once

#include "common.cuh"
#include "fp4attn.h"

namespace fp4 {

constexpr int PG_D = 128;           // head dim
constexpr int PG_ROW = PG_D / 2;    // code bytes of a (token, head)
constexpr int PG_SF = PG_D / 16;    // scale bytes of a (token, head)
constexpr float PG_TINY = 1.17549435e-38f;  // 2^-126: 1/g of a smaller g overflows

// Device-side error bits of a cache (status[0]); see fp4attn.h.
enum : int { PG_NO_PAGES = 1, PG_TOO_LONG = 2, PG_BAD_KEEP = 4, PG_SHARED = 8, PG_BAD_SEQ = 16 };

// The slot of row b of a call, -1 where seqs names none.
__device__ __forceinline__ int pg_seq(const fp4paged_cache& c, const int32_t* seqs, int b) {
  const int s = seqs ? seqs[b] : b;
  return s >= 0 && s < c.max_seqs ? s : -1;
}

// 16 elements at p (16-byte aligned when VEC), as loaded.
template <int DT, bool VEC>
struct Block16 {
  using T = typename In<DT>::T;
  static constexpr int W = 16 * (int)sizeof(T) / 16;
  uint4 raw[W];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < W; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) reinterpret_cast<T*>(raw)[i] = p[i];
    }
  }
  __device__ __forceinline__ float operator[](int i) const { return In<DT>::f(reinterpret_cast<const T*>(raw)[i]); }
  __device__ __forceinline__ float absmax() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i += 2) m = absmax3(m, (*this)[i], (*this)[i + 1]);
    return m;
  }
};

// g of a token from the maximum of its |x|, and 1/g: a subnormal g counts as
// 0 (1/g would overflow), one that is not finite makes the token NaN.
__device__ __forceinline__ float pg_global(float m, float& r) {
  const bool bad = !(m <= 3.402823466e38f);
  const float g = m < PG_TINY ? 0.0f : m;
  r = bad || g == 0.0f ? 0.0f : __frcp_rn(g);
  return bad ? __int_as_float(0x7fc00000) : g;
}

// Packed fp32 pairs, each rounded like the scalar operation.
__device__ __forceinline__ uint64_t pg_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pg_mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pg_add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Eight floats, in pairs, to eight E2M1 codes (the first in the low nibble).
__device__ __forceinline__ uint32_t pg_codes(const uint64_t (&z)[4]) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t.reg .f32 l, h;\n\t"
      "mov.b64 {l, h}, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b0, h, l;\n\t"
      "mov.b64 {l, h}, %2;\n\tcvt.rn.satfinite.e2m1x2.f32 b1, h, l;\n\t"
      "mov.b64 {l, h}, %3;\n\tcvt.rn.satfinite.e2m1x2.f32 b2, h, l;\n\t"
      "mov.b64 {l, h}, %4;\n\tcvt.rn.satfinite.e2m1x2.f32 b3, h, l;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "l"(z[0]), "l"(z[1]), "l"(z[2]), "l"(z[3]));
  return r;
}

// A block whose largest |x| is m, under 1/g = r (0 in a token of zeros or NaN): eight code bytes and the E4M3 scale
// byte.  The largest |x r| is that of m: rounding keeps order.
template <typename Blk>
__device__ __forceinline__ uint32_t pg_block(const Blk& x, float m, float r, uint2& codes) {
  codes = make_uint2(0u, 0u);
  if (r == 0.0f) return 0u;  // the same for the whole token
  const uint32_t s8 = e4m3_satfinite(__fmul_rn(__fmul_rn(m, r), recip6<FP4_ARITH_F32>()));
  const float s = e4m3_to_f32((uint8_t)s8), rs = s == 0.0f ? 0.0f : __frcp_rn(s);
  const uint64_t r2 = pg_pair(r, r), rs2 = pg_pair(rs, rs), zero = pg_pair(0.0f, 0.0f);
  uint64_t z[2][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)  // + 0: a zero's code has no sign
    z[i >> 2][i & 3] = pg_add2(pg_mul2(pg_mul2(pg_pair(x[2 * i], x[2 * i + 1]), r2), rs2), zero);
  codes = make_uint2(pg_codes(z[0]), pg_codes(z[1]));
  return s8;
}

// Four E2M1 code pairs (the bytes of w, lowest first) as fp16 pairs.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t* o) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}

// A warp quantizes one token of H heads: lane l takes blocks l, l + 32, ...; at(block) is where the block's
// elements are, put(block, codes, scale) stores it.  Returns the token's g.  Up to NB blocks a lane stay in
// registers between the maximum and the codes (NB 0: read twice).  where() finds the token's place, while its loads
// are on their way; if it has none (false), nothing is stored.
template <int DT, bool VEC, int NB, typename At, typename Where, typename Put>
__device__ __forceinline__ float pg_quantize_token(int nblk, At at, Where where, Put put) {
  const int lane = threadIdx.x & 31;
  float m = 0.0f, r;
  if constexpr (NB > 0) {
    Block16<DT, VEC> x[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (lane + 32 * i < nblk) x[i].load(at(lane + 32 * i));
    if (!where()) return 0.0f;
    float top[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (lane + 32 * i < nblk) top[i] = x[i].absmax(), m = nanmax(m, top[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = nanmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float g = pg_global(m, r);
#pragma unroll
    for (int i = 0; i < NB; ++i)
      if (lane + 32 * i < nblk) {
        uint2 c;
        const uint32_t s = pg_block(x[i], top[i], r, c);
        put(lane + 32 * i, c, s);
      }
    return g;
  } else {
    if (!where()) return 0.0f;
    Block16<DT, VEC> x;
    for (int i = lane; i < nblk; i += 32) x.load(at(i)), m = nanmax(m, x.absmax());
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = nanmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float g = pg_global(m, r);
    for (int i = lane; i < nblk; i += 32) {
      x.load(at(i));
      uint2 c;
      const uint32_t s = pg_block(x, x.absmax(), r, c);
      put(i, c, s);
    }
    return g;
  }
}

}  // namespace fp4
