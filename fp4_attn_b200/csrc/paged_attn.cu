// paged_attn.cu -- attention of the drafted tokens (the last N of each
// sequence) over the paged NVFP4 cache.
//
// A KV head's query rows (node i, head g of the group: row i * G + g) are the
// columns of transposed products, so that few rows cost few columns:
//   S^T[key][row] = K^ Q^^T         tcgen05 kind::mxf4nvf4, the cache's codes and scales as they are
//   O^T[d][row]  += V^^T[d][key] W[key][row]   tcgen05 kind::f16
// with x = S scaling log2(e) + log2(g_v), W = 2^(x - m + 9) and, per row, m a
// running maximum of x.  Folding V's per-token scale g_v into the exponent keeps
// W within fp16 whatever the values' sizes, and leaves code * scale for V^,
// exact in fp16.  The row sum is l = sum W / g_v, in fp32.
//
// The work, tiles of 256 keys of every (sequence, KV head, tile of rows), is
// one list that the CTAs (one per SM) share out evenly, whatever the lengths;
// what a CTA did of a list entry that it shares with others goes to the
// workspace as (m, l, O), and the last kernel joins those in a fixed order.
#include <stdint.h>

#include <algorithm>

#include "attn_softmax.cuh"
#include "paged.cuh"
#include "sm100.cuh"
#include "status.h"
#include "tmap.h"

namespace fp4 {

int paged_check(const fp4paged_cache* c, int B, const int32_t* seqs);

FP4_DEFINE_STATUS_READER(paged_status)

namespace {

constexpr int TK = 256, HK = 128;  // keys of a tile, in two halves of 128 (an MMA's rows)
// W is 2^9 at x = m and at most 2^15: m follows, for all rows at once, when a score passes it by 6.  Half of fp16's
// smallest step is then 2^-34 of a row's largest W.  (With 2^12 and 3 the maxima of 32 rows of a few thousand keys
// moved in every second tile, which costs several times a tile without.)
constexpr float W_BIAS = 9.0f, W_SLACK = 6.0f;
constexpr float GV_MIN = 7.888609052e-31f;  // 2^-100: V tokens below count as 0, so that 1/g_v sums stay finite
// 2^-64, the g_v of a token that counts as 0.  It is in l = sum W / g_v as any other (from W's 2^-126 on: while the others'
// g_v are below 2^38, whatever has a share of 2^-24 or more), and should not be what m follows, for then the others' W,
// smaller by g_v, would be rounded away: with 1 those of g_v 2^-25 kept 8 bits and less.
constexpr float GV_ZERO = 5.421010862e-20f;
constexpr float L_SCALE = 0.0009765625f;    // 2^-10, for the same reason

// A row of the call, as the first kernel found it.
struct Row {
  int slot, len, n, pad;  // sequence (-1: none), its tokens, its nodes
};

struct AttnArgs {
  fp4paged_cache c;
  // query rows in the order of the list, [B][H][RT * NB]: codes [D/2], E4M3 scales [D/16], g scaling log2(e)
  const uint8_t* q_codes;
  const uint8_t* q_scales;
  const float* q_f;
  const uint32_t* bits;     // [B][N (key)][nw]: which nodes see node j (mask calls)
  const Row* rows;          // [B]
  const int* first;         // [B+1] tiles before row b
  float* part;              // [grid][2]: O [NB][D], W_BIAS - m [NB], l [NB]
  int B, Hq, G, N, RT, nw;  // RT: tiles of NB rows that N * G rows take; nw: words of a mask row
  bool causal;
  float scaling;
  void* out;
};

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Key tiles of rows [rt * NB, (rt + 1) * NB) of a (sequence, KV head).
__device__ __forceinline__ int tiles_of(const Row& r, int rt, int NB, int G, bool causal) {
  const int rows = r.n * G;
  if (r.len <= 0 || rt * NB >= rows) return 0;
  const int last = (min((rt + 1) * NB, rows) - 1) / G;  // the last node
  const int limit = causal ? min(r.len, r.len - r.n + last + 1) : r.len;
  return (limit + TK - 1) / TK;
}

// --------------------------------------------------------------- preparation
struct PrepArgs {
  const void* q;
  int64_t sB, sH, sT;
  const uint8_t* mask;
  int64_t m_sB, m_sI, m_sJ;
  const int32_t *counts, *seqs;
  int NB, mask_blocks;
};

// A launch's time (a few hundred tokens at most).  Blocks [0, B*N): a block quantizes a query token (one g over its
// Hq * D channels).  Then mask_blocks blocks: a warp per (row, node j) turns the mask's column j into bits over the
// nodes i that see it.  The last block lists the rows and the tiles before each.
constexpr int PREP_THREADS = 256;
template <int DT, bool VEC, int NBLK>
__global__ void __launch_bounds__(PREP_THREADS) paged_prep_kernel(AttnArgs a, PrepArgs p) {
  using E = typename In<DT>::T;
  __shared__ float smax[PREP_THREADS / 32];
  __shared__ long long ssum[PREP_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t tokens = (int64_t)a.B * a.N;
  pdl_launch();
  if (blockIdx.x < tokens) {
    const int64_t id = blockIdx.x;
    const E* x = static_cast<const E*>(p.q) + (id / a.N) * p.sB + (id % a.N) * p.sT;
    const int nblk = a.Hq * PG_SF;
    // row of head hq of this token
    const int64_t RP = (int64_t)a.RT * p.NB, row0 = (id / a.N) * a.c.num_kv_heads * RP + (id % a.N) * a.G;
    auto row_of = [&](int hq) { return row0 + (hq / a.G) * RP + hq % a.G; };
    auto at = [&](int i) { return x + (i >> 3) * p.sH + (i & 7) * 16; };
    constexpr int NR = NBLK > 0 ? NBLK : 1;
    Block16<DT, VEC> blk[NR];
    float m = 0.0f, r;
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int k = 0; k < NBLK; ++k)
        if (threadIdx.x + PREP_THREADS * k < nblk) blk[k].load(at(threadIdx.x + PREP_THREADS * k));
#pragma unroll
      for (int k = 0; k < NBLK; ++k)
        if (threadIdx.x + PREP_THREADS * k < nblk) m = nanmax(m, blk[k].absmax());
    } else {
      for (int i = threadIdx.x; i < nblk; i += PREP_THREADS) blk[0].load(at(i)), m = nanmax(m, blk[0].absmax());
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = nanmax(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) smax[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PREP_THREADS / 32; ++w) m = nanmax(m, smax[w]);
    const float g = pg_global(m, r);
    auto put = [&](int i, const Block16<DT, VEC>& b) {
      uint2 c;
      const uint32_t s = pg_block(b, b.absmax(), r, c);
      const int64_t row = row_of(i >> 3);
      *reinterpret_cast<uint2*>(const_cast<uint8_t*>(a.q_codes) + row * PG_ROW + (i & 7) * 8) = c;
      const_cast<uint8_t*>(a.q_scales)[row * PG_SF + (i & 7)] = (uint8_t)s;
      if ((i & 7) == 0) const_cast<float*>(a.q_f)[row] = g * (a.scaling * 1.4426950408889634f);
    };
    if constexpr (NBLK > 0) {
#pragma unroll
      for (int k = 0; k < NBLK; ++k)
        if (threadIdx.x + PREP_THREADS * k < nblk) put(threadIdx.x + PREP_THREADS * k, blk[k]);
    } else {
      for (int i = threadIdx.x; i < nblk; i += PREP_THREADS) blk[0].load(at(i)), put(i, blk[0]);
    }
  } else if (blockIdx.x < tokens + p.mask_blocks) {
    const int64_t id = (blockIdx.x - tokens) * (PREP_THREADS / 32) + warp;
    if (id >= tokens) return;
    const int64_t b = id / a.N, j = id % a.N;
    const uint8_t* col = p.mask + b * p.m_sB + j * p.m_sJ;
    for (int w = 0; w < a.nw; ++w) {
      const int i = 32 * w + lane;
      const unsigned v = __ballot_sync(0xffffffffu, i < a.N && col[i * p.m_sI] != 0);
      if (lane == 0) const_cast<uint32_t*>(a.bits)[id * a.nw + w] = v;
    }
  } else {
    Row* rows = const_cast<Row*>(a.rows);
    int* first = const_cast<int*>(a.first);
    long long sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += PREP_THREADS) {
      const int b = b0 + threadIdx.x;
      long long t = 0;
      if (b < a.B) {
        Row r;
        r.slot = pg_seq(a.c, p.seqs, b);
        r.len = r.slot < 0 ? 0 : a.c.lens[r.slot];
        if (r.slot < 0) atomicOr(a.c.status, PG_BAD_SEQ);
        // a sequence with fewer tokens than nodes has only those
        r.n = min(r.len, p.counts ? max(0, min(p.counts[b], a.N)) : a.N);
        r.pad = 0;
        rows[b] = r;
        for (int rt = 0; rt < a.RT; ++rt) t += tiles_of(r, rt, p.NB, a.G, a.causal);
        t *= a.c.num_kv_heads;
      }
      long long v = t;
#pragma unroll
      for (int o = 1; o < 32; o *= 2) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      __syncthreads();
      if (lane == 31) ssum[warp] = v;
      __syncthreads();
      long long before = sum;
      for (int w = 0; w < PREP_THREADS / 32; ++w) {
        if (w < warp) before += ssum[w];
        sum += ssum[w];
      }
      if (b < a.B) first[b] = (int)min(before + v - t, (long long)INT32_MAX);
    }
    if (threadIdx.x == 0) first[a.B] = (int)min(sum, (long long)INT32_MAX);
  }
}

// ------------------------------------------------------------- the work list
// A CTA's place in the list: tile `tile` of `tiles` of rows rt of KV head h of row b.
struct Place {
  int b, h, rt, tile, tiles;
  Row row;
};

// Walks the list from tile g0.  The whole warp takes part.
__device__ __forceinline__ Place place_at(const AttnArgs& a, int NB, int g0) {
  Place p;
  // the last row whose first tile is not past g0 (rows without tiles share their successor's); rows come along
  // with the prefixes, so that the first 32 cost one trip to memory
  p.b = 0;
  int before = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int k = b0 + (threadIdx.x & 31);
    const int f = k < a.B ? a.first[k] : INT32_MAX;
    const int4 r = k < a.B ? *reinterpret_cast<const int4*>(a.rows + k) : make_int4(-1, 0, 0, 0);
    const unsigned m = __ballot_sync(0xffffffffu, f <= g0);
    if (m) {
      const int l = 31 - __clz(m);
      p.b = b0 + l;
      before = __shfl_sync(0xffffffffu, f, l);
      p.row = {__shfl_sync(0xffffffffu, r.x, l), __shfl_sync(0xffffffffu, r.y, l), __shfl_sync(0xffffffffu, r.z, l), 0};
    }
    if (m != 0xffffffffu) break;
  }
  int rem = g0 - before, per = 0;
#pragma unroll 1
  for (int rt = 0; rt < a.RT; ++rt) per += tiles_of(p.row, rt, NB, a.G, a.causal);
  p.h = per ? rem / per : 0;
  rem -= p.h * per;
#pragma unroll 1
  for (p.rt = 0;; ++p.rt) {
    p.tiles = tiles_of(p.row, p.rt, NB, a.G, a.causal);
    if (rem < p.tiles || p.rt + 1 >= a.RT) break;
    rem -= p.tiles;
  }
  p.tile = rem;
  return p;
}

// The next tile; only called while there is one.
__device__ __forceinline__ void advance(const AttnArgs& a, int NB, Place& p) {
  if (++p.tile < p.tiles) return;
  p.tile = 0;
  do {
    if (++p.rt >= a.RT) {
      p.rt = 0;
      if (++p.h >= a.c.num_kv_heads) {
        p.h = 0;
        if (++p.b >= a.B) return;
        p.row = a.rows[p.b];
      }
    }
    p.tiles = tiles_of(p.row, p.rt, NB, a.G, a.causal);
  } while (p.tiles == 0);
}

// The list's tiles are shared out evenly, the first total % grid CTAs having one more.
struct Share {
  int base, more;
  __device__ __forceinline__ Share(int total, int grid) : base(total / grid), more(total % grid) {}
  __device__ __forceinline__ int start(int cta) const { return cta * base + min(cta, more); }
  __device__ __forceinline__ int owner(int g) const {
    const int big = more * (base + 1);
    return g < big ? g / (base + 1) : more + (g - big) / base;
  }
};

// ------------------------------------------------------------------ attention
// Warp 0 walks the work list and brings a tile's pages by TMA (a lane per page); warp 1 builds the K scale atoms
// and issues S^T; warp 2 issues O^T; the softmax warps, two keys (one of each half) and 16 rows a lane at a time,
// turn S^T into W; the V warps widen V's codes to fp16.
//
// What bounds it is instructions.  At first their fetching (with the list walked by every role and all rows of a
// warp unrolled, 110 to 220 KB of code, the instruction caches were 80 % busy and a third of the stalls), hence
// one walker that hands on what the others need through the stage, and apart what is rare (a moved maximum, masks,
// an entry's end).  Then their number: a softmax warp's waits, arrivals and addresses cost about 210 a tile, its
// 16 rows and 32 keys only 90, hence tiles of 256 keys and as many rows per warp as its registers hold.
// With 64 rows it is about 10300 warp instructions a tile, 2500 of them V's widening and 1400 the exponentials.
// Measured, all three kernels: 8 x 32768 keys, 8 heads, 8 rows: 99 us, 3.1 TB/s of 304 MB (46 us at a plain copy's
// rate); 2 x 65536 keys, 8 heads, 512 rows: 568 us, 242 TFLOP/s in O^T (83 us at the fp16 rate of a large product).
//
// Roundings to fewer than 32 bits.  fp32 outputs (PL 2): W is two fp16 planes, 2^-22 of it together, and each tile's
// product is added up in registers.  16-bit outputs (PL 1): W is one plane, off by up to 2^-11 of itself, as an fp16
// output is of its own and a quarter of what a bf16 one is, and the keys' errors average out (drafted trees in fp16,
// relative error against 64 bits: 2.3e-4, with W in 32 bits 2.1e-4; in bf16 the same); O adds up in the tensor cores,
// which cut off, 2e-6 of it after 14 tiles of 128 keys.  A second plane would double the O^T products.
constexpr uint32_t KC = TK * PG_ROW, KS = TK * PG_SF, KG = TK * 4;
constexpr uint32_t O_VC = KC, O_KS = 2 * KC, O_VS = O_KS + KS, O_KG = O_VS + KS, O_VG = O_KG + KG;
constexpr uint32_t STAGE = O_VG + KG;  // K codes, V codes, K scales, V scales, K g, V g: 38 KB
static_assert(STAGE % 1024 == 0, "stage");
constexpr uint32_t V16 = HK * PG_D * 2;  // widened V of a half: two atoms of 64 channels, [128 keys][128 B]

// A tile of the list, as the producer hands it on.
struct TileInfo {
  int b, h, rt, flags;
  int pos, len, base, rows;  // first key, tokens of the sequence, those before the drafted ones, query rows (n * G)
};
// Of the entry, for this CTA: its first tile, its last, all of its tiles are this CTA's, and which of the CTA's two
// partials it is.
enum : int { T_FIRST = 1, T_LAST = 2, T_WHOLE = 4, T_SLOT = 8 };

template <int NB, int PL>
struct Cfg {
  static constexpr int GROUPS = NB == 16 ? 1 : 2;         // groups of four softmax warps
  static constexpr int NCH = NB / 16 / GROUPS;            // chunks of 16 rows that a group has
  static constexpr int SW = 4 * GROUPS, DW = 12 - SW;     // softmax and V warps; 15 in all, 128 registers
  static constexpr int SW0 = 3, DW0 = SW0 + SW, THREADS = (DW0 + DW) * 32;
  static constexpr int NS = NB == 16 ? 3 : 2;
  static constexpr bool FLUSH = PL == 2;           // O leaves TMEM after every tile (see below)
  static constexpr int OB = FLUSH ? 2 : 1;         // O accumulators
  static constexpr uint32_t PBYTES = HK * NB * 2;  // one plane of W of a half
  static constexpr uint32_t OFF_V = NS * STAGE;
  static constexpr uint32_t OFF_P = OFF_V + 2 * V16;             // [tile & 1][half][plane]
  static constexpr uint32_t OFF_ATOM = OFF_P + 4 * PL * PBYTES;  // K scale atoms, two tiles of 2 KB
  static constexpr uint32_t OFF_Q = OFF_ATOM + 4096;             // query rows, 64-byte swizzle
  static constexpr uint32_t OFF_QSF = OFF_Q + NB * PG_ROW;
  static constexpr uint32_t SMEM = OFF_QSF + 1024 + 1024;  // + alignment slack
  static constexpr uint32_t T_S = 0, T_O = 4 * NB, T_SFA = T_O + OB * NB, T_SFB = T_SFA + 32, T_END = T_SFB + 8;
  static constexpr uint32_t TMEM = T_END <= 128 ? 128 : T_END <= 256 ? 256 : 512;
  static_assert(SMEM <= 227 * 1024 && T_END <= 512 && OFF_QSF % 1024 == 0, "on-chip memory");
};

// MN-major operand tile of NB 16-bit columns: [key][NB], rows of min(NB, 64) columns, swizzled over the row's
// 16-byte chunks.  Byte offset of chunk j (8 columns) of key k.
template <int NB>
__device__ __forceinline__ uint32_t mn_chunk(int k, int j) {
  if constexpr (NB == 16) return k * 32 + ((j ^ ((k >> 2) & 1)) << 4);
  else if constexpr (NB == 32) return k * 64 + ((j ^ ((k >> 1) & 3)) << 4);
  else return k * 128 + ((j ^ (k & 7)) << 4);
}
// Its descriptor (NB 128: two atoms of 64 columns); 16 keys further are `pitch` further in the descriptor.
template <int NB>
struct MnTile {
  static constexpr uint32_t ROW = NB >= 64 ? 128 : NB * 2;
  static constexpr uint64_t STEP = (16 * ROW) >> 4;
  static __device__ __forceinline__ uint64_t desc(uint32_t base) {
    constexpr SmemLayout lay = NB == 16 ? kSwizzle32B : NB == 32 ? kSwizzle64B : kSwizzle128B;
    return smem_desc(base, NB == 128 ? HK * 128 : 8 * ROW, 8 * ROW, lay);
  }
};
// kind::f16, fp16 operands, both MN-major (bits 15 and 16), fp32 accumulators.
__host__ __device__ constexpr uint32_t idesc_f16_mn(int M, int N) { return idesc_f16(M, N) | (1u << 15) | (1u << 16); }

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}

// 16 bytes by cp.async, and this thread's arrival at a barrier once its copies are in.
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// mbar_wait of few instructions: bounded by suspended waits of up to 20 us instead of by the clock, and the waiting
// itself in a function of its own.
__device__ __noinline__ bool wait_longer(uint64_t* bar, uint32_t parity, unsigned int site) {
#pragma unroll 1
  for (int i = 0; i < 100000; ++i) {
    if (mbar_try_wait_suspend(bar, parity, kSuspendNs)) return true;
    if (dev_failed()) return false;
  }
  dev_fail(site);
  return false;
}
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, unsigned int site) {
  return __builtin_expect(mbar_try_wait(bar, parity), 1) || wait_longer(bar, parity, site);
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned int site) {
  return __all_sync(0xffffffffu, wait_for(bar, parity, site));
}

// One lane of the warp, in a way the compiler knows.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// Named barrier that ors a flag over its threads.
__device__ __forceinline__ bool bar_or(uint32_t id, uint32_t count, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(count)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 100000; ++i)
    if (mbar_try_wait_suspend(bar, parity, kSuspendNs)) return;
}
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t two_bytes) {
  uint32_t r;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(r) : "r"(two_bytes));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
}

// Which of the rows r0 .. r0 + 15 see keys pos and pos + HK: bits 0-15 and 16-31.  bits: the row's mask words per
// drafted node (null: node j is seen by node i >= j).
__device__ __noinline__ uint32_t seen_rows(const uint32_t* bits, int nw, int N, int G, int r0, int pos, int base,
                                           int len) {
  uint32_t seen = 0u;
#pragma unroll 1
  for (int hf = 0; hf < 2; ++hf, pos += HK) {
    const int jn = pos - base;
    uint32_t v = 0xffffu;
    if (pos >= len) {
      v = 0u;
    } else if (jn >= 0 && !bits) {
      const int cmin = jn * G - r0;  // rows of node >= jn
      v = cmin >= 16 ? 0u : cmin <= 0 ? v : (v << cmin) & 0xffffu;
    } else if (jn >= 0) {
      const uint32_t* w = bits + (int64_t)jn * nw;
      int i = r0 / G, g = r0 - i * G;
      v = 0u;
#pragma unroll 1
      for (int j = 0; j < 16; ++j) {
        if (i < N) v |= ((w[i >> 5] >> (i & 31)) & 1u) << j;
        if (++g == G) g = 0, ++i;
      }
    }
    seen |= v << (16 * hf);
  }
  return seen;
}

// Sums of 16 values over the lanes: lane l gets that of value l & 15 (half of the values go each step).
__device__ __forceinline__ float lane_sums16(float (&v)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const bool up = lane & o;
      const float keep = up ? v[i + o] : v[i], give = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 16);
}

template <int NB, int PL, int DT>
__global__ void __launch_bounds__(Cfg<NB, PL>::THREADS, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ AttnArgs a) {
  using C = Cfg<NB, PL>;
  constexpr int NS = C::NS, NCH = C::NCH;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[NS], empty[NS], s_full[2], s_free[2], p_full[2], p_done[2], v_full[2], v_done[2],
      o_free, qdrain, drained[2];
  __shared__ __align__(16) float colb[NB], colc[NB], red[NB / 16][4][16];
  __shared__ __align__(16) TileInfo info[NS];
  __shared__ int v_first;                        // the tile of v_full[0] begins a list entry
  __shared__ volatile int gave_up[2][C::GROUPS];  // [tile & 1][group]
  __shared__ uint32_t tslot;
  // (broadcast: the compiler then knows that a warp's role is one, and keeps what is uniform in it out of the lanes)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s)
      mbar_init(&full[s], a.c.page_size < 64 ? 33 : 1), mbar_init(&empty[s], 1 + C::SW + C::DW);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1), mbar_init(&s_free[i], C::SW), mbar_init(&drained[i], 1);
      mbar_init(&p_full[i], C::SW), mbar_init(&p_done[i], 1);
      mbar_init(&v_full[i], 4), mbar_init(&v_done[i], 1);
      for (int g = 0; g < C::GROUPS; ++g) gave_up[i][g] = 0;
    }
    mbar_init(&o_free, C::SW), mbar_init(&qdrain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tslot, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  pdl_wait();  // the query's codes and the work list

  const int total = a.first[a.B], grid = min((int)gridDim.x, total);  // CTAs that have tiles
  int g0 = 0, n_it = 0;
  if ((int)blockIdx.x < grid) {
    const Share share(total, grid);
    g0 = share.start(blockIdx.x), n_it = share.start(blockIdx.x + 1) - g0;
  }

  if (n_it > 0 && warp == 0) {
    // ------------------------------------------------------------- producer
    if (lane == 0) tma_prefetch_desc(&tmK), tma_prefetch_desc(&tmV);
    const int H = a.c.num_kv_heads, P = a.c.page_size, npp = TK / P;  // pages of a tile, a lane each
    // a bulk copy costs about 65 cycles to issue: with small pages the scales and g come by cp.async instead
    const bool small = P < 64;
    const uint32_t page_bytes = P * 2 * (PG_ROW + (small ? 0 : PG_SF + 4));
    Place p = place_at(a, NB, g0);
    auto page_of = [&]() -> int {
      const int k = p.tile * npp + lane;  // page of the sequence
      return lane < npp && k * P < p.row.len ? a.c.page_table[(int64_t)p.row.slot * a.c.max_pages + k] : -1;
    };
    int page = page_of(), issued = 0, s = 0, par = 1;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int h = p.h;
      const TileInfo ti = {p.b, h, p.rt,
                           (it == 0 || p.tile == 0 ? T_FIRST : 0) | (p.tile + 1 == p.tiles || it + 1 == n_it ? T_LAST : 0) |
                               (p.tile + 1 == p.tiles && p.tile <= it ? T_WHOLE : 0) | (p.tile < it ? T_SLOT : 0),
                           p.tile * TK, p.row.len, p.row.len - p.row.n, p.row.n * a.G};
      int next = -1;
      if (it + 1 < n_it) advance(a, NB, p), next = page_of();  // in flight while this tile waits for its stage
      if (it >= NS && !warp_wait(&empty[s], par, 0x601)) break;
      const unsigned live = __ballot_sync(0xffffffffu, page >= 0);
      uint8_t* st = sm + (size_t)s * STAGE;
      if (lane == 0) {
        info[s] = ti;
        mbar_arrive_expect_tx(&full[s], __popc(live) * page_bytes);
      }
      __syncwarp();
      if (page >= 0) {
        const int64_t row = ((int64_t)page * H + h) * P;
        tma_load_2d(st + lane * P * PG_ROW, &tmK, &full[s], 0, (int)row);
        tma_load_2d(st + O_VC + lane * P * PG_ROW, &tmV, &full[s], 0, (int)row);
        if (!small) {
          bulk_load(st + O_KS + lane * P * PG_SF, a.c.k_scales + row * PG_SF, P * PG_SF, &full[s]);
          bulk_load(st + O_VS + lane * P * PG_SF, a.c.v_scales + row * PG_SF, P * PG_SF, &full[s]);
          bulk_load(st + O_KG + lane * P * 4, a.c.k_g + (int64_t)page * P, P * 4, &full[s]);
          bulk_load(st + O_VG + lane * P * 4, a.c.v_g + (int64_t)page * P, P * 4, &full[s]);
        }
      }
      if (small) {
#pragma unroll 1
        for (int i = lane; i < TK / 2; i += 32) {  // 16 bytes: the scales of keys 2 i and 2 i + 1
          const int from = __shfl_sync(0xffffffffu, page, 2 * i / P);
          const int64_t row = (((int64_t)from * H + h) * P + 2 * i % P) * PG_SF;
          if (from >= 0) cp_async16(st + O_KS + i * 16, a.c.k_scales + row), cp_async16(st + O_VS + i * 16, a.c.v_scales + row);
        }
#pragma unroll 1
        for (int i = lane; i < TK / 4; i += 32) {  // the g of four keys
          const int from = __shfl_sync(0xffffffffu, page, 4 * i / P);
          const int64_t at = (int64_t)from * P + 4 * i % P;
          if (from >= 0) cp_async16(st + O_KG + i * 16, a.c.k_g + at), cp_async16(st + O_VG + i * 16, a.c.v_g + at);
        }
        cp_async_arrive(&full[s]);
      }
      page = next;
      issued = it + 1;
      if (++s == NS) s = 0, par ^= 1;
    }
    if (lane == 0)
#pragma unroll 1
      for (int it = issued > NS ? issued - NS : 0; it < issued; ++it) mbar_drain(&full[it % NS], (it / NS) & 1);
  } else if (n_it > 0 && warp == 1) {
    // ------------------------------------------------------------------ S^T
    const uint32_t idesc = idesc_nvf4(128, NB);
    uint8_t *qs = sm + C::OFF_Q, *qsf = sm + C::OFF_QSF;
    const uint64_t qdesc = smem_desc(smem_u32(qs), 16, 512, kSwizzle64B);
    int entries = 0, s = 0, par = 0;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int k = it & 1;
      if (!warp_wait(&full[s], par, 0x602)) break;
      const uint8_t* st = sm + (size_t)s * STAGE;
      if (__builtin_expect(info[s].flags & T_FIRST, 0)) {
        // a new list entry: its query rows (contiguous; rows past the entry's hold anything, as columns do not mix)
        const int64_t q0 = (((int64_t)info[s].b * a.c.num_kv_heads + info[s].h) * a.RT + info[s].rt) * NB;
        uint4 v[NB / 8];
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) v[i] = reinterpret_cast<const uint4*>(a.q_codes + q0 * PG_ROW)[lane + 32 * i];
        uint2 sc[(NB + 31) / 32];
#pragma unroll
        for (int i = 0; i < (NB + 31) / 32; ++i)
          sc[i] = lane + 32 * i < NB ? reinterpret_cast<const uint2*>(a.q_scales + q0 * PG_SF)[lane + 32 * i]
                                     : make_uint2(0u, 0u);
        if (entries > 0) {  // the products with the old rows are done
          if (lane == 0) tc_commit(&qdrain);
          if (!warp_wait(&qdrain, (entries - 1) & 1, 0x603)) break;
        }
        ++entries;
#pragma unroll
        for (int i = 0; i < NB / 8; ++i) {
          const int c = (lane + 32 * i) >> 2, ch = lane & 3;
          *reinterpret_cast<uint4*>(qs + c * 64 + ((ch ^ ((c >> 1) & 3)) << 4)) = v[i];
        }
#pragma unroll
        for (int i = 0; i < (NB + 31) / 32; ++i) {
          *reinterpret_cast<uint32_t*>(qsf + lane * 16 + i * 4) = sc[i].x;
          *reinterpret_cast<uint32_t*>(qsf + 512 + lane * 16 + i * 4) = sc[i].y;
        }
        fence_async_smem();
        __syncwarp();
        if (elect_one()) {
          tc_fence_after();
          tmem_cp_sf_atom(tmem + C::T_SFB, smem_desc(smem_u32(qsf), 16, 128, kSwizzleNone));
          tmem_cp_sf_atom(tmem + C::T_SFB + 4, smem_desc(smem_u32(qsf + 512), 16, 128, kSwizzleNone));
        }
        __syncwarp();
      }
      if (it >= 2 && !warp_wait(&s_free[k], ((it >> 1) - 1) & 1, 0x604)) break;
      uint8_t* at = sm + C::OFF_ATOM + k * 2048;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint2 sc = *reinterpret_cast<const uint2*>(st + O_KS + (lane + 32 * j) * 8);
        uint8_t* to = at + (j >> 2) * 1024 + lane * 16 + (j & 3) * 4;
        *reinterpret_cast<uint32_t*>(to) = sc.x;
        *reinterpret_cast<uint32_t*>(to + 512) = sc.y;
      }
      fence_async_smem();
      __syncwarp();
      if (elect_one()) {
        tc_fence_after();
        const uint32_t sfa = tmem + C::T_SFA + 16 * k, sd = tmem + C::T_S + 2 * NB * k;
        const uint64_t ad = smem_desc(smem_u32(at), 16, 128, kSwizzleNone);
        const uint64_t kd = smem_desc(smem_u32(st), 16, 512, kSwizzle64B);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_cp_sf_atom(sfa + 4 * c, ad + c * (512 >> 4));
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            mma_nvf4(sd + NB * hf, kd + hf * (HK * PG_ROW >> 4) + kk * 2, qdesc + kk * 2, idesc, sfa + 8 * hf + 4 * kk,
                     tmem + C::T_SFB + 4 * kk, kk);
        tc_commit(&s_full[k]);
        tc_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == NS) s = 0, par ^= 1;
    }
    if (lane == 0) {
      tc_commit(&drained[0]);  // what was issued completes before TMEM is released
      mbar_drain(&drained[0], 0);
    }
  } else if (n_it > 0 && warp == 2) {
    // ------------------------------------------------------------------ O^T
    const uint32_t idesc = idesc_f16_mn(128, NB);
    const uint64_t vd0 = MnTile<128>::desc(smem_u32(sm + C::OFF_V)), wd0 = MnTile<NB>::desc(smem_u32(sm + C::OFF_P));
    int entries = 0;
    bool ok = true;
#pragma unroll 1
    for (int it = 0; it < n_it && ok; ++it) {
      const int k = it & 1;
      if (!warp_wait(&v_full[0], it & 1, 0x605)) break;
      bool first = v_first != 0;
      if (first && !C::FLUSH && entries++ > 0 && !warp_wait(&o_free, (entries - 2) & 1, 0x606)) break;
      if (!warp_wait(&p_full[k], (it >> 1) & 1, 0x607)) break;
      if (C::FLUSH) first = true;
      const uint32_t o = tmem + C::T_O + (C::FLUSH ? NB * k : 0);
#pragma unroll 1
      for (int hf = 0; hf < 2; ++hf) {
        if (hf && !(ok = warp_wait(&v_full[1], it & 1, 0x608))) break;
        tc_fence_after();
        const uint64_t vd = vd0 + hf * (V16 >> 4), wd = wd0 + (2 * k + hf) * (PL * C::PBYTES >> 4);
        if (elect_one()) {
#pragma unroll
          for (int ks = 0; ks < HK / 16; ++ks)
#pragma unroll
            for (int pl = 0; pl < PL; ++pl)
              mma_f16_ss(o, vd + ks * MnTile<128>::STEP, wd + ks * MnTile<NB>::STEP + pl * (C::PBYTES >> 4), idesc,
                         ks || pl || hf ? 1u : first ? 0u : 1u);
          tc_commit(&v_done[hf]);
          if (hf) tc_commit(&p_done[k]);
        }
        __syncwarp();
      }
    }
    if (lane == 0) {
      tc_commit(&drained[1]);
      mbar_drain(&drained[1], 0);
    }
  } else if (n_it > 0 && warp < C::DW0) {
    // -------------------------------------------------------------- softmax
    // A group's warps have the chunks of 16 rows group, group + GROUPS, ...; those past the entry's rows are skipped.
    const int group = (warp - C::SW0) >> 2, quarter = warp & 3, key = quarter * 32 + lane;
    const uint32_t bar_id = 1 + group, lanes = (uint32_t)(quarter * 32) << 16;
    auto col_of = [&](int ch) { return (ch * C::GROUPS + group) * 16; };
    uint64_t l2[NCH][8];
    float of[C::FLUSH ? NCH : 1][16];  // O of this lane's channel, when it is summed here
    // fp32 outputs: the tensor cores cut off what they add to an accumulator, always towards 0 (2e-6 of the result
    // after 14 tiles of 128), so each tile's product starts anew and O is summed in registers.
    auto flush = [&](int j) {
      const bool ok = warp_wait(&p_done[j & 1], (j >> 1) & 1, 0x609);
      tc_fence_after();
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        uint32_t o[16];
        tmem_ld16(tmem + lanes + C::T_O + NB * (j & 1) + col_of(ch), o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) of[C::FLUSH ? ch : 0][i] += __uint_as_float(o[i]);
      }
      tc_fence_before();
      return ok;
    };
    int s = 0, par = 0;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int k = it & 1;
      bool ok = warp_wait(&full[s], par, 0x60a);
      const TileInfo ti = info[s];
      const uint8_t* st = sm + (size_t)s * STAGE;
      // the factors of this lane's keys, one of each half; keys past the end are not visible, whatever the stage
      // holds for them
      float ak[2], lg[2], rg[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        ak[hf] = *reinterpret_cast<const float*>(st + O_KG + (hf * HK + key) * 4);
        lg[hf] = *reinterpret_cast<const float*>(st + O_VG + (hf * HK + key) * 4);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == NS) s = 0, par ^= 1;
      const bool first = ti.flags & T_FIRST;
      const bool edge = ti.pos + TK > ti.base;  // drafted tokens, or the sequence's end
      const int live = ti.rows - ti.rt * NB;    // columns in use
      if (__builtin_expect(first, 0)) {
        // the factors of the rows' scores, and m = -inf
        if (key < 16 * NCH) {
          const int c = col_of(key >> 4) + (key & 15);
          colb[c] = c < live ? a.q_f[(((int64_t)ti.b * a.c.num_kv_heads + ti.h) * a.RT + ti.rt) * NB + c] : 0.0f;
          colc[c] = INFINITY;  // W_BIAS - m
        }
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
          for (int i = 0; i < 8; ++i) l2[ch][i] = 0ull;
        if constexpr (C::FLUSH)
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
            for (int i = 0; i < 16; ++i) of[ch][i] = 0.0f;
        named_bar(bar_id, 128);
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        if (ti.pos + hf * HK + key >= ti.len) ak[hf] = 0.0f, lg[hf] = 1.0f;
        const float gs = lg[hf] >= GV_MIN ? lg[hf] : GV_ZERO;  // 0 and NaN: V^ is 0 there
        lg[hf] = lg[hf] != lg[hf] ? lg[hf] : lg2(gs), rg[hf] = rcp(gs) * L_SCALE;
      }
      ok = warp_wait(&s_full[k], (it >> 1) & 1, 0x60b) && ok;
      if (it >= 2) ok = warp_wait(&p_done[k], ((it >> 1) - 1) & 1, 0x60c) && ok;  // W's buffer is free
      tc_fence_after();
      bool flushed = false;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        const int c0 = col_of(ch);
        if (NB > 16 && c0 >= live) continue;
        float *cb = colb + c0, *cc = colc + c0;
        uint32_t seen = 0xffffffffu;  // a bit per row, for each of the two keys
        if (__builtin_expect(edge, 0)) {
          seen = seen_rows(a.causal ? nullptr : a.bits + (int64_t)ti.b * a.N * a.nw, a.nw, a.N, a.G, ti.rt * NB + c0,
                           ti.pos + key, ti.base, ti.len);
        }
        // y = x - m + W_BIAS, x = S scaling log2(e) + log2(g_v); -inf marks what a row does not see.  x is rounded by
        // itself, as where m is made of it, and W_BIAS - m is rounded down: once m has moved, y <= W_BIAS holds to the
        // bit for x of all sizes, and the key that has the maximum keeps a weight of 1 or more.  (Rounded as one sum, y
        // is off by up to x's last place, which passes W_SLACK from 2^27 on; 2 x 65536 keys, 512 rows: 554 us so, 566
        // like this.)
        float y[2][16];
#pragma unroll 1
        for (bool moved = false;; moved = true) {  // twice at most
          uint32_t acc[2][16];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) tmem_ld16(tmem + lanes + C::T_S + 2 * NB * k + NB * hf + c0, acc[hf]);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(&cb[j]);
            const ulonglong2 c4 = *reinterpret_cast<const ulonglong2*>(&cc[j]);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const uint64_t ak2 = pk2(ak[hf], ak[hf]), lgv = pk2(lg[hf], lg[hf]);
              upk2(add2(fma2(mul2(pk2(__uint_as_float(acc[hf][j]), __uint_as_float(acc[hf][j + 1])), ak2), b4.x, lgv),
                        c4.x),
                   y[hf][j], y[hf][j + 1]);
              upk2(add2(fma2(mul2(pk2(__uint_as_float(acc[hf][j + 2]), __uint_as_float(acc[hf][j + 3])), ak2), b4.y, lgv),
                        c4.y),
                   y[hf][j + 2], y[hf][j + 3]);
            }
          }
          if (__builtin_expect(edge, 0)) {
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j >> 4][j & 15] = (seen >> j) & 1u ? y[j >> 4][j & 15] : -INFINITY;
          }
          if (moved) break;
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < 16; ++j) top = max3f(top, y[0][j], y[1][j]);
          if (!ok) gave_up[k][group] = 1;
          if (__builtin_expect(!bar_or(bar_id, 128, top > W_BIAS + W_SLACK), 1)) break;
          // some score passed its row's m: every row's m becomes the maximum so far
          float(&rd)[4][16] = red[c0 / 16];
          float mx = -INFINITY;
          {
            float v[16];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              uint32_t acc[16];
              tmem_ld16(tmem + lanes + C::T_S + 2 * NB * k + NB * hf + c0, acc);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float x = __fmaf_rn(__fmul_rn(__uint_as_float(acc[j]), ak[hf]), cb[j], lg[hf]);
                const float u = (seen >> (16 * hf + j)) & 1u ? x : -INFINITY;
                v[j] = hf ? fmaxf(v[j], u) : u;
              }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const float u = redux_max(v[j]);
              if (lane == j) mx = u;
            }
          }
          if (lane < 16) rd[quarter][lane] = mx;
          named_bar(bar_id, 128);
          const int c = lane & 15;
          const float old = cc[c];
          const float bn = fminf(old, __fsub_rd(W_BIAS, fmaxf(fmaxf(rd[0][c], rd[1][c]), fmaxf(rd[2][c], rd[3][c]))));
          const float f = bn == old ? 1.0f : ex2(bn - old);
          named_bar(bar_id, 128);  // cc and rd have been read
          if (quarter == 0 && lane < 16) cc[c] = bn;
          named_bar(bar_id, 128);
          if (!first) {
            // O of the earlier tiles of this list entry, once they are all in
            uint32_t o[16];
            if constexpr (C::FLUSH) {
              if (!flushed) ok = flush(it - 1) && ok, flushed = true;
            } else {
              ok = warp_wait(&p_done[(it - 1) & 1], ((it - 1) >> 1) & 1, 0x60d) && ok;
              tc_fence_after();
              tmem_ld16(tmem + lanes + C::T_O + c0, o);
              tmem_ld_wait();
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float f0 = __shfl_sync(0xffffffffu, f, j), f1 = __shfl_sync(0xffffffffu, f, j + 1);
              l2[ch][j / 2] = mul2(l2[ch][j / 2], pk2(f0, f1));
              if constexpr (C::FLUSH) {
                of[ch][j] *= f0, of[ch][j + 1] *= f1;
              } else {
                o[j] = __float_as_uint(__uint_as_float(o[j]) * f0);
                o[j + 1] = __float_as_uint(__uint_as_float(o[j + 1]) * f1);
              }
            }
            if constexpr (!C::FLUSH) {
              tmem_st16(tmem + lanes + C::T_O + c0, o);
              tmem_st_wait();
              tc_fence_before();
            }
          }
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          uint8_t* wp = sm + C::OFF_P + (2 * k + hf) * PL * C::PBYTES;
          const uint64_t rg2 = pk2(rg[hf], rg[hf]);
#pragma unroll
          for (int j0 = 0; j0 < 16; j0 += 8) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float e0 = ex2(y[hf][j0 + 2 * j]), e1 = ex2(y[hf][j0 + 2 * j + 1]);
              l2[ch][j0 / 2 + j] = fma2(pk2(e0, e1), rg2, l2[ch][j0 / 2 + j]);
              const __half2 h2 = __floats2half2_rn(e0, e1);
              hi[j] = *reinterpret_cast<const uint32_t*>(&h2);
              if constexpr (PL == 2) {
                const float2 hf2 = __half22float2(h2);
                const __half2 r2 = __floats2half2_rn(e0 - hf2.x, e1 - hf2.y);
                lo[j] = *reinterpret_cast<const uint32_t*>(&r2);
              }
            }
            const uint32_t off = mn_chunk<NB>(key, (c0 + j0) / 8);
            *reinterpret_cast<uint4*>(wp + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (PL == 2)
              *reinterpret_cast<uint4*>(wp + C::PBYTES + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[k]), mbar_arrive(&p_full[k]);
      if constexpr (C::FLUSH)
        if (!first && !flushed) ok = flush(it - 1) && ok;
      // written before a vote of this tile, read after its last, so the same for all warps of this group
      if (gave_up[k][group]) break;
      if (__builtin_expect(ti.flags & T_LAST, 0)) {
        // --------------------------------------------- a list entry's end
        // l of each row: over the lanes here, over the four warps in red
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 8; ++j) upk2(l2[ch][j], v[2 * j], v[2 * j + 1]);
          const float sum = lane_sums16(v);
          if (lane < 16) red[col_of(ch) / 16][quarter][lane] = sum;
        }
        named_bar(bar_id, 128);
        const bool whole = ti.flags & T_WHOLE;
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (ti.flags & T_SLOT ? 1 : 0)) * (NB * (PG_D + 2));
        if constexpr (C::FLUSH) ok = flush(it) && ok;
        else ok = warp_wait(&p_done[k], (it >> 1) & 1, 0x60e) && ok;
        tc_fence_after();
        if constexpr (C::FLUSH) {  // back to TMEM, to be read column by column
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch) {
            uint32_t o[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(of[ch][j]);
            tmem_st16(tmem + lanes + C::T_O + NB * k + col_of(ch), o);
          }
          tmem_st_wait();
        }
        const int all = min(NB, a.N * a.G - ti.rt * NB);  // columns that the output has
#pragma unroll 1
        for (int ch = 0; ch < NCH; ++ch) {
          const int c0 = col_of(ch), r0 = ti.rt * NB + c0;
          if (c0 >= all) break;
          float(&rd)[4][16] = red[c0 / 16];
          // lane j (and j + 16): what row j needs
          const float l = (rd[0][lane & 15] + rd[1][lane & 15]) + (rd[2][lane & 15] + rd[3][lane & 15]);
          const float scale = c0 + (lane & 15) < live && l != 0.0f ? L_SCALE / l : 0.0f;
          if (!whole && key < 16) part[NB * PG_D + c0 + key] = colc[c0 + key], part[NB * (PG_D + 1) + c0 + key] = l;
          int i = r0 / a.G, g = r0 - i * a.G;
          int64_t at = (((int64_t)ti.b * a.N + i) * a.Hq + ti.h * a.G + g) * PG_D + key;  // key: this lane's channel
          const uint32_t to = tmem + lanes + C::T_O + (C::FLUSH ? NB * k : 0) + c0;
          float* pp = part + c0 * PG_D + key;
#pragma unroll 1
          for (int j0 = 0; j0 < 16; j0 += 4) {
            uint32_t o[4];
            tmem_ld4(to + j0, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 4; ++j, pp += PG_D) {
              const float v = __uint_as_float(o[j]), f = __shfl_sync(0xffffffffu, scale, j0 + j);
              if (!whole) *pp = v;
              else if (c0 + j0 + j < all) store_out<DT>(a.out, at, f == 0.0f ? 0.0f : v * f);
              at += PG_D;
              if (++g == a.G) g = 0, at += (int64_t)(a.Hq - a.G) * PG_D;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free);
        named_bar(bar_id, 128);  // colc and red are free
      }
    }
  } else if (n_it > 0) {
    // ---------------------------------------------------------------- V^
    // four warps per half: both halves at once with eight, in turn with four
    const int w = (warp - C::DW0) & 3;
    int s = 0, par = 0;
    bool ok = true;
#pragma unroll 1
    for (int it = 0; it < n_it && ok; ++it) {
      ok = warp_wait(&full[s], par, 0x60f);
      if (!ok) break;
      const uint8_t* st = sm + (size_t)s * STAGE;
      const int left = info[s].len - info[s].pos, fl = info[s].flags;
#pragma unroll 1
      for (int hf = (warp - C::DW0) >> 2; hf < 2; hf += C::DW / 4) {
        if (it >= 1 && !(ok = warp_wait(&v_done[hf], (it - 1) & 1, 0x610))) break;
        if (hf == 0 && w == 0 && lane == 0) v_first = fl & T_FIRST;
        uint8_t* vb = sm + C::OFF_V + hf * V16;
#pragma unroll 2
        for (int i = 0; i < 4; ++i) {
          const int r = (i * 4 + w) * 8 + (lane & 7), key = hf * HK + r, ch = lane >> 3;  // 32 channels from 32 ch
          const uint4 cw = *reinterpret_cast<const uint4*>(st + O_VC + key * 64 + ((ch ^ ((r >> 1) & 3)) << 4));
          uint32_t sc = *reinterpret_cast<const uint16_t*>(st + O_VS + key * 8 + ch * 2);
          const float gv = *reinterpret_cast<const float*>(st + O_VG + key * 4);
          // tokens past the end, NaN tokens and those below GV_MIN contribute nothing (NaN comes in through W)
          if (!(gv >= GV_MIN) || key >= left) sc = 0u;
          const uint32_t s2 = e4m3x2_f16x2(sc), s0 = __byte_perm(s2, s2, 0x1010), s1 = __byte_perm(s2, s2, 0x3232);
          uint32_t o[16];
          e2m1x8_f16(cw.x, o), e2m1x8_f16(cw.y, o + 4), e2m1x8_f16(cw.z, o + 8), e2m1x8_f16(cw.w, o + 12);
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = hmul2_u32(o[j], j < 8 ? s0 : s1);
          const uint32_t row = (ch >> 1) * (HK * 128) + r * 128;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(vb + row + ((((ch & 1) * 4 + j) ^ (r & 7)) << 4)) =
                make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[hf]);
      }
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == NS) s = 0, par ^= 1;
    }
  }
  pdl_launch();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

// ------------------------------------------------------------------- joining
// A block per (8 rows, row tile and KV head, b), a warp per row: O = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i over
// the CTAs that had tiles of the list entry, in their order.  Entries that one CTA did are already out; rows
// without a tile are 0.  A launch's time; done by the attention kernel's last CTA of an entry instead, it took longer
// (6 x 27 nodes: 69 us in all instead of 55): one CTA's warps then join 64 rows at the end.
template <int NB, int DT>
__global__ void __launch_bounds__(256) paged_join_kernel(AttnArgs a, int grid_max) {
  pdl_wait();
  const int lane = threadIdx.x & 31, b = blockIdx.z, rt = blockIdx.y % a.RT, h = blockIdx.y / a.RT;
  const int c = blockIdx.x * 8 + (threadIdx.x >> 5), r = rt * NB + c;
  if (r >= a.N * a.G) return;
  const Row row = a.rows[b];
  const int tiles = tiles_of(row, rt, NB, a.G, a.causal);
  const int total = a.first[a.B];
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (tiles > 0) {
    int per = 0, before = 0;
    for (int i = 0; i < a.RT; ++i) {
      const int t = tiles_of(row, i, NB, a.G, a.causal);
      if (i < rt) before += t;
      per += t;
    }
    const int t0 = a.first[b] + h * per + before, t1 = t0 + tiles - 1;
    const Share share(total, min(grid_max, total));
    const int c0 = share.owner(t0), c1 = share.owner(t1);
    if (c0 == c1) return;
    if (r < row.n * a.G) {
      // CTA c0's share is its first segment if its range starts with this entry, else its last; the others' is
      // their first
      auto slot = [&](int i) {
        return a.part + ((int64_t)i * 2 + (i == c0 && share.start(c0) < t0 ? 1 : 0)) * (NB * (PG_D + 2));
      };
      float m = INFINITY;  // W_BIAS - the largest m
      for (int i = c0 + lane; i <= c1; i += 32) m = fminf(m, slot(i)[NB * PG_D + c]);
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) m = fminf(m, __shfl_xor_sync(0xffffffffu, m, k));
      float l = 0.0f;
      for (int i0 = c0; i0 <= c1; i0 += 32) {
        const int i = i0 + lane;
        float f = 0.0f, li = 0.0f;
        if (i <= c1) {
          const float* s = slot(i);
          li = s[NB * (PG_D + 1) + c];
          const float mi = s[NB * PG_D + c];
          f = li == 0.0f ? 0.0f : mi == m ? 1.0f : ex2(m - mi);
        }
        l += f * li;
        const int n = min(32, c1 - i0 + 1);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const float fk = __shfl_sync(0xffffffffu, f, k);
          const float4 v = reinterpret_cast<const float4*>(slot(i0 + k) + c * PG_D)[lane];
          if (fk != 0.0f) o.x += fk * v.x, o.y += fk * v.y, o.z += fk * v.z, o.w += fk * v.w;
        }
      }
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
      const float s = l == 0.0f ? 0.0f : L_SCALE / l;
      o.x *= s, o.y *= s, o.z *= s, o.w *= s;
    }
  }
  const int64_t at = (((int64_t)b * a.N + r / a.G) * a.Hq + h * a.G + r % a.G) * PG_D + 4 * lane;
  store_out<DT>(a.out, at, o.x), store_out<DT>(a.out, at + 1, o.y);
  store_out<DT>(a.out, at + 2, o.z), store_out<DT>(a.out, at + 3, o.w);
}

// --------------------------------------------------------------------- host
// Rows of a tile: the fewest tiles that hold all rows, as each of them reads the keys again and widens V again (32 rows
// of 4 x 2000 keys and 8 heads: 24.5 us as one tile of 64, 26.6 as two of 16), but no more than need be, as a tile's
// exponentials are made for all of them (8 rows, 8 x 32768 keys: 99.6 us with tiles of 16, 123 with 64).  fp32
// outputs keep W as two planes and O in registers, which leaves room for 32.
int rows_per_tile(int64_t rows, bool fp32) { return rows <= 16 ? 16 : fp32 ? 32 : 64; }

struct Layout {
  int NB, RT, nw, grid;
  int64_t scales, g, bits, rows, first, part, bytes;
};

int64_t piece(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// SMs of the current device (148 where there is none to ask).
int sm_count() {
  int dev = 0, n = 0;
  return cudaGetDevice(&dev) == cudaSuccess &&
                 cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0
             ? n
             : 148;
}

Layout layout_of(int B, int Hq, int Hkv, int N, bool fp32, int sms) {
  Layout L;
  const int64_t rows = (int64_t)N * (Hq / Hkv), tok = (int64_t)B * N;
  L.NB = rows_per_tile(rows, fp32);
  L.RT = (int)((rows + L.NB - 1) / L.NB);
  L.nw = (N + 31) / 32;
  L.grid = sms;
  const int64_t qrows = (int64_t)B * Hkv * L.RT * L.NB;
  L.scales = piece(qrows * PG_ROW);
  L.g = L.scales + piece(qrows * PG_SF);
  L.bits = L.g + piece(qrows * 4);
  L.rows = L.bits + piece(tok * L.nw * 4);
  L.first = L.rows + piece((int64_t)B * sizeof(Row));
  L.part = L.first + piece((int64_t)(B + 1) * 4);
  L.bytes = L.part + piece((int64_t)L.grid * 2 * L.NB * (PG_D + 2) * 4);
  return L;
}

int64_t bytes_of(int B, int Hq, int Hkv, int N, int sms) {
  return std::max(layout_of(B, Hq, Hkv, N, false, sms).bytes, layout_of(B, Hq, Hkv, N, true, sms).bytes);
}

template <typename... KArgs, typename... Args>
int launch_pdl(const char* what, void (*fn)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st,
               Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at, cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, fn, args...);
  return check_launch(what);
}

template <int DT>
int launch_prep(const AttnArgs& a, const PrepArgs& p, cudaStream_t st) {
  const int64_t esz = DT == FP4_DT_F32 ? 4 : 2;
  const bool vec = (uintptr_t)p.q % 16 == 0 && (p.sB * esz % 16 == 0 || a.B == 1) &&
                   (p.sT * esz % 16 == 0 || a.N == 1) && (p.sH * esz % 16 == 0 || a.Hq == 1);
  const unsigned grid = (unsigned)((int64_t)a.B * a.N + p.mask_blocks + 1);
  if (!vec) paged_prep_kernel<DT, false, 0><<<grid, PREP_THREADS, 0, st>>>(a, p);
  else if (a.Hq * PG_SF <= 2 * PREP_THREADS) paged_prep_kernel<DT, true, 2><<<grid, PREP_THREADS, 0, st>>>(a, p);
  else paged_prep_kernel<DT, true, 0><<<grid, PREP_THREADS, 0, st>>>(a, p);
  return check_launch("paged_prep_kernel");
}

template <int NB, int PL, int DT>
int launch_attn(const AttnArgs& a, const Layout& L, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  using C = Cfg<NB, PL>;
  if (int e = set_smem_attr((const void*)paged_attn_kernel<NB, PL, DT>, (int)C::SMEM)) return e;
  if (int e = launch_pdl("paged_attn_kernel", paged_attn_kernel<NB, PL, DT>, dim3(L.grid), C::THREADS, C::SMEM, st, mk,
                         mv, a))
    return e;
  return launch_pdl("paged_join_kernel", paged_join_kernel<NB, DT>, dim3(NB / 8, a.c.num_kv_heads * a.RT, a.B), 256, 0,
                    st, a, L.grid);
}

template <int DT>
int launch_rows(const AttnArgs& a, const Layout& L, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  constexpr int PL = DT == FP4_DT_F32 ? 2 : 1;
  if (L.NB == 16) return launch_attn<16, PL, DT>(a, L, mk, mv, st);
  return launch_attn<PL == 2 ? 32 : 64, PL, DT>(a, L, mk, mv, st);
}

}  // namespace
}  // namespace fp4

using namespace fp4;

extern "C" int64_t fp4paged_attention_workspace_size(int B, int Hq, int Hkv, int N) {
  if (B <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv) return -1;
  return bytes_of(B, Hq, Hkv, N, sm_count());
}

extern "C" int fp4paged_attention(const fp4paged_cache* cache, const void* q, int in_dtype, int B, int Hq, int N,
                                  int64_t q_sB, int64_t q_sH, int64_t q_sT, const uint8_t* mask, int64_t m_sB,
                                  int64_t m_sI, int64_t m_sJ, const int32_t* counts, const int32_t* seqs,
                                  float scaling, void* out, int out_dtype, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  clear_error();
  if (int e = paged_check(cache, B, seqs)) return e;
  const int H = cache->num_kv_heads;
  if (N < 0 || Hq <= 0 || Hq % H)
    return set_error(FP4ATTN_ERR_ARG, "bad shape: %d query heads, %d KV heads", Hq, H);
  if (B == 0 || N == 0) return FP4ATTN_OK;
  if (!q || !out || !workspace) return set_error(FP4ATTN_ERR_ARG, "null pointer");
  if (in_dtype < 0 || in_dtype > 2 || out_dtype < 0 || out_dtype > 2) return set_error(FP4ATTN_ERR_ARG, "bad dtype");
  const int sms = sm_count();
  const int64_t need = bytes_of(B, Hq, H, N, sms);
  if ((uintptr_t)workspace % 256 || workspace_bytes < need)
    return set_error(FP4ATTN_ERR_ARG, "workspace of %lld bytes, %lld needed (256-byte aligned)",
                     (long long)workspace_bytes, (long long)need);
  const Layout L = layout_of(B, Hq, H, N, out_dtype == FP4_DT_F32, sms);
  // grid limits, 32-bit rows, and the tensor maps' 32-bit row coordinate
  if (B > 65535 || (int64_t)H * L.RT > 65535 || (int64_t)N * (Hq / H) > INT32_MAX / 2 ||
      (int64_t)B * N > INT32_MAX / 2)
    return set_error(FP4ATTN_ERR_UNSUPPORTED, "more than 65535 rows or (KV head, row tile) pairs");
  // the work list is counted in 32 bits
  const int64_t most = ((int64_t)cache->max_pages * cache->page_size + TK - 1) / TK * L.RT * H * B;
  if (most > INT32_MAX) return set_error(FP4ATTN_ERR_UNSUPPORTED, "2^31 or more key tiles");
  const int64_t krows = (int64_t)cache->num_pages * H * cache->page_size;
  if (krows > INT32_MAX) return set_error(FP4ATTN_ERR_UNSUPPORTED, "the cache has 2^31 or more (token, head) rows");
  uint8_t* w = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.c = *cache;
  a.q_codes = w, a.q_scales = w + L.scales, a.q_f = reinterpret_cast<float*>(w + L.g);
  a.bits = reinterpret_cast<uint32_t*>(w + L.bits), a.rows = reinterpret_cast<Row*>(w + L.rows);
  a.first = reinterpret_cast<int*>(w + L.first), a.part = reinterpret_cast<float*>(w + L.part);
  a.B = B, a.Hq = Hq, a.G = Hq / H, a.N = N, a.RT = L.RT, a.nw = L.nw;
  a.causal = mask == nullptr, a.scaling = scaling, a.out = out;
  const PrepArgs p{q, q_sB, q_sH, q_sT, mask, m_sB, m_sI, m_sJ, counts, seqs, L.NB,
                   mask ? (int)(((int64_t)B * N + 7) / 8) : 0};
  // K and V codes: a row per (page, head, token), boxes of a page with the 64-byte swizzle
  CUtensorMap mk, mv;
  if (int e = encode_tiled_2d(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, cache->k_codes, PG_ROW, krows, PG_ROW, PG_ROW,
                              cache->page_size, CU_TENSOR_MAP_SWIZZLE_64B))
    return e;
  if (int e = encode_tiled_2d(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, cache->v_codes, PG_ROW, krows, PG_ROW, PG_ROW,
                              cache->page_size, CU_TENSOR_MAP_SWIZZLE_64B))
    return e;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int e = in_dtype == FP4_DT_F32    ? launch_prep<FP4_DT_F32>(a, p, st)
                : in_dtype == FP4_DT_BF16 ? launch_prep<FP4_DT_BF16>(a, p, st)
                                          : launch_prep<FP4_DT_F16>(a, p, st);
  if (e) return e;
  switch (out_dtype) {
    case FP4_DT_F32: return launch_rows<FP4_DT_F32>(a, L, mk, mv, st);
    case FP4_DT_BF16: return launch_rows<FP4_DT_BF16>(a, L, mk, mv, st);
    default: return launch_rows<FP4_DT_F16>(a, L, mk, mv, st);
  }
}
