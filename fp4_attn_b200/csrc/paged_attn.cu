// paged_attn.cu -- attention of the drafted tokens (the last N of each
// sequence) over the paged NVFP4 cache.
//
// A KV head's query rows (node i, head g of the group: row i * G + g) are the
// columns of transposed products, so that few rows cost few columns:
//   S^T[key][row] = K^ Q^^T         tcgen05 kind::mxf4nvf4, the cache's codes and scales as they are
//   O^T[d][row]  += V^^T[d][key] W[key][row]   tcgen05 kind::f16
// with x = S scaling log2(e) + log2(g_v), W = 2^(x - m + 12) and, per row, m a
// running maximum of x.  Folding V's per-token scale g_v into the exponent keeps
// W within fp16 whatever the values' sizes, and leaves code * scale for V^,
// exact in fp16.  The row sum is l = sum W / g_v, in fp32.
//
// The work, tiles of 128 keys of every (sequence, KV head, tile of rows), is
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

constexpr int TK = 128;        // keys of a tile
constexpr float W_BIAS = 12.0f;  // 2^12 of fp16's 2^15 is W at x = m: its smallest step is then 2^-36 of it
constexpr float W_SLACK = 3.0f;  // m follows once a score passes it by this much, so W <= 2^15
constexpr float GV_MIN = 7.888609052e-31f;  // 2^-100: V tokens below count as 0, so that 1/g_v sums stay finite
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
  const long long* first;   // [B+1] tiles before row b
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

// Blocks [0, B*N): a block quantizes a query token (one g over its Hq * D channels).  Then mask_blocks blocks: a
// warp per (row, node j) turns the mask's column j into bits over the nodes i that see it.  The last block lists
// the rows and the tiles before each.
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
      const uint32_t s = pg_block(b, r, c);
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
    long long* first = const_cast<long long*>(a.first);
    long long sum = 0;
    for (int b0 = 0; b0 < a.B; b0 += PREP_THREADS) {
      const int b = b0 + threadIdx.x;
      long long t = 0;
      if (b < a.B) {
        Row r;
        r.slot = pg_seq(a.c, p.seqs, b);
        r.len = r.slot < 0 ? 0 : a.c.lens[r.slot];
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
      if (b < a.B) first[b] = before + v - t;
    }
    if (threadIdx.x == 0) first[a.B] = sum;
  }
}

// ------------------------------------------------------------- the work list
// A CTA's place in the list: tile `tile` of `tiles` of rows rt of KV head h of row b.
struct Place {
  int b, h, rt, tile, tiles;
  Row row;
};

// Walks the list from tile g0.  The whole warp takes part.
__device__ __forceinline__ Place place_at(const AttnArgs& a, int NB, long long g0) {
  Place p;
  // the last row whose first tile is not past g0 (rows without tiles share their successor's)
  int b = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int k = b0 + (threadIdx.x & 31);
    const unsigned m = __ballot_sync(0xffffffffu, k < a.B && a.first[k] <= g0);
    if (m) b = b0 + 31 - __clz(m);
    if (m != 0xffffffffu) break;
  }
  p.b = b;
  p.row = a.rows[b];
  long long rem = g0 - a.first[b];
  int per = 0;
#pragma unroll 1
  for (int rt = 0; rt < a.RT; ++rt) per += tiles_of(p.row, rt, NB, a.G, a.causal);
  p.h = per ? (int)(rem / per) : 0;
  rem -= (long long)p.h * per;
#pragma unroll 1
  for (p.rt = 0;; ++p.rt) {
    p.tiles = tiles_of(p.row, p.rt, NB, a.G, a.causal);
    if (rem < p.tiles || p.rt + 1 >= a.RT) break;
    rem -= p.tiles;
  }
  p.tile = (int)rem;
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

__device__ __forceinline__ long long range_start(long long total, int cta, int grid) { return total * cta / grid; }
// The CTA whose range holds tile g: the largest with range_start <= g.
__device__ __forceinline__ int owner_of(long long total, long long g, int grid) {
  return (int)(((g + 1) * grid - 1) / total);
}

// ------------------------------------------------------------------ attention
// Warp 0 walks the work list and brings a tile's pages by TMA (a lane per page); warp 1 builds the K scale atoms
// and issues S^T; warp 2 issues O^T; softmax warps hold a key per lane and 16 rows and turn S^T into W; V warps
// widen V's codes to fp16.
//
// What bounds it is instructions, and first of all fetching them: with the list walked by every role and the rows
// of a warp unrolled, 110 to 220 KB of code, the instruction caches were 80 % busy.  So one warp walks and hands
// the others what they need through the stage, every softmax warp has the same 16 rows' worth of code, and what
// is rare (a moved maximum, masks, an entry's end) stands apart.
constexpr uint32_t KC = TK * PG_ROW, KS = TK * PG_SF, KG = TK * 4;
constexpr uint32_t O_VC = KC, O_KS = 2 * KC, O_VS = O_KS + KS, O_KG = O_VS + KS, O_VG = O_KG + KG;
constexpr uint32_t STAGE = 19 * 1024;  // K codes, V codes, K scales, V scales, K g, V g
static_assert(O_VG + KG <= STAGE && STAGE % 1024 == 0, "stage");
constexpr uint32_t V16 = TK * PG_D * 2;  // widened V: two atoms of 64 channels, [128 keys][128 B]

// A tile of the list, as the producer hands it on.
struct TileInfo {
  int b, h, rt, flags;
  int pos, len, base, rows;  // first key, tokens of the sequence, those before the drafted ones, query rows (n * G)
};
// Of the entry, for this CTA: its first and second tile, its last and the one before, all of its tiles are this
// CTA's, and which of the CTA's two partials it is.
enum : int { T_FIRST = 1, T_SECOND = 2, T_LAST = 4, T_PENULT = 8, T_WHOLE = 16, T_SLOT = 32 };

template <int NB, int PL>
struct Cfg {
  // Streams: with 16 rows one group of warps would be bound by latency, so two take the tiles in turn, each with
  // an O, m and l of its own, joined at the entry's end.
  static constexpr int ST = NB == 16 ? 2 : 1;
  static constexpr int CHUNKS = NB / 16, GROUPS = CHUNKS * ST;  // groups of four softmax warps, 16 rows each
  static constexpr int TW = 4 * CHUNKS, VW = 4;                 // softmax and V warps that a tile has
  static constexpr int SW0 = 3, DW0 = SW0 + 4 * GROUPS, THREADS = (DW0 + VW * ST) * 32;
  static constexpr int NS = 4;
  static constexpr bool FLUSH = PL == 2;            // O leaves TMEM after every tile (see below)
  static constexpr int OB = FLUSH ? 2 * ST : ST;    // O accumulators
  static constexpr uint32_t PBYTES = TK * NB * 2;  // one plane of W
  static constexpr uint32_t OFF_V = NS * STAGE;
  static constexpr uint32_t OFF_P = OFF_V + 2 * V16;
  static constexpr uint32_t OFF_ATOM = OFF_P + 2 * PL * PBYTES;  // K scale atoms, two tiles of 1 KB
  static constexpr uint32_t OFF_Q = OFF_ATOM + 2048;             // query rows, 64-byte swizzle
  static constexpr uint32_t OFF_QSF = OFF_Q + NB * PG_ROW;
  static constexpr uint32_t OFF_MERGE = OFF_QSF + 1024;  // one stream's O [16][D], c, l on its way to the other
  static constexpr uint32_t SMEM = OFF_MERGE + (ST == 2 ? 16 * (PG_D + 2) * 4 : 0) + 1024;  // + alignment slack
  static constexpr uint32_t T_S = 0, T_O = 2 * NB, T_SFA = T_O + OB * NB, T_SFB = T_SFA + 16, T_END = T_SFB + 8;
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
    return smem_desc(base, NB == 128 ? TK * 128 : 8 * ROW, 8 * ROW, lay);
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

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// mbar_wait of few instructions: bounded by suspended waits of up to 20 us instead of by the clock.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, unsigned int site) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
#pragma unroll 1
  for (int i = 0; i < 100000; ++i) {
    if (mbar_try_wait_suspend(bar, parity, kSuspendNs)) return true;
    if (dev_failed()) return false;
  }
  dev_fail(site);
  return false;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned int site) {
  return __all_sync(0xffffffffu, wait_for(bar, parity, site));
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
// Four E2M1 code pairs (the bytes of w, lowest first) as fp16 pairs.
__device__ __forceinline__ void e2m1x8_f16(uint32_t w, uint32_t* o) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\tcvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\tcvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
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
  constexpr int NS = C::NS, ST = C::ST, OB = C::OB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[NS], empty[NS], s_full[2], s_free[2], p_full[2], v_full[2], pv_done[2],
      o_free[ST], qdrain, drained[2], m_full, m_free;
  __shared__ __align__(16) float colb[ST][NB], colc[ST][NB], red[C::GROUPS][4][16];
  __shared__ __align__(16) TileInfo info[NS];
  __shared__ int v_first[2];  // the tile of v_full[k] begins a list entry
  __shared__ volatile int gave_up[2][C::GROUPS];  // [the group's tile & 1][group]
  __shared__ uint32_t tslot;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) mbar_init(&full[s], 1), mbar_init(&empty[s], 1 + C::TW + C::VW);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1), mbar_init(&s_free[i], C::TW), mbar_init(&drained[i], 1);
      mbar_init(&p_full[i], C::TW), mbar_init(&v_full[i], C::VW), mbar_init(&pv_done[i], 1);
      for (int g = 0; g < C::GROUPS; ++g) gave_up[i][g] = 0;
    }
    for (int i = 0; i < ST; ++i) mbar_init(&o_free[i], C::TW);
    mbar_init(&qdrain, 1), mbar_init(&m_full, 4), mbar_init(&m_free, 4);
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

  const long long total = a.first[a.B];
  const int grid = (int)min((long long)gridDim.x, total);  // CTAs that have tiles
  const long long g0 = (int)blockIdx.x < grid ? range_start(total, blockIdx.x, grid) : 0;
  const int n_it = (int)blockIdx.x < grid ? (int)(range_start(total, blockIdx.x + 1, grid) - g0) : 0;

  if (n_it > 0 && warp == 0) {
    // ------------------------------------------------------------- producer
    if (lane == 0) tma_prefetch_desc(&tmK), tma_prefetch_desc(&tmV);
    const int H = a.c.num_kv_heads, P = a.c.page_size, npp = TK / P;  // pages of a tile, a lane each
    const uint32_t page_bytes = P * 2 * (PG_ROW + PG_SF + 4);
    Place p = place_at(a, NB, g0);
    auto page_of = [&]() -> int {
      const int k = p.tile * npp + lane;  // page of the sequence
      return lane < npp && k * P < p.row.len ? a.c.page_table[(int64_t)p.row.slot * a.c.max_pages + k] : -1;
    };
    int page = page_of(), issued = 0;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int s = it % NS, h = p.h;
      const TileInfo ti = {
          p.b, h, p.rt,
          (it == 0 || p.tile == 0 ? T_FIRST : it == 1 || p.tile == 1 ? T_SECOND : 0) |
              (p.tile + 1 == p.tiles || it + 1 == n_it ? T_LAST : p.tile + 2 == p.tiles || it + 2 == n_it ? T_PENULT : 0) |
              (p.tile + 1 == p.tiles && p.tile <= it ? T_WHOLE : 0) | (p.tile < it ? T_SLOT : 0),
          p.tile * TK, p.row.len, p.row.len - p.row.n, p.row.n * a.G};
      int next = -1;
      if (it + 1 < n_it) advance(a, NB, p), next = page_of();  // in flight while this tile waits for its stage
      if (it >= NS && !warp_wait(&empty[s], ((it / NS) - 1) & 1, 0x601)) break;
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
        bulk_load(st + O_KS + lane * P * PG_SF, a.c.k_scales + row * PG_SF, P * PG_SF, &full[s]);
        bulk_load(st + O_VS + lane * P * PG_SF, a.c.v_scales + row * PG_SF, P * PG_SF, &full[s]);
        bulk_load(st + O_KG + lane * P * 4, a.c.k_g + (int64_t)page * P, P * 4, &full[s]);
        bulk_load(st + O_VG + lane * P * 4, a.c.v_g + (int64_t)page * P, P * 4, &full[s]);
      }
      page = next;
      issued = it + 1;
    }
    if (lane == 0)
#pragma unroll 1
      for (int it = issued > NS ? issued - NS : 0; it < issued; ++it) mbar_drain(&full[it % NS], (it / NS) & 1);
  } else if (n_it > 0 && warp == 1) {
    // ------------------------------------------------------------------ S^T
    const uint32_t idesc = idesc_nvf4(128, NB);
    uint8_t *qs = sm + C::OFF_Q, *qsf = sm + C::OFF_QSF;
    const uint64_t qdesc = smem_desc(smem_u32(qs), 16, 512, kSwizzle64B);
    int entries = 0;
#pragma unroll 1
    for (int it = 0; it < n_it; ++it) {
      const int s = it % NS, k = it & 1;
      if (!warp_wait(&full[s], (it / NS) & 1, 0x602)) break;
      const uint8_t* st = sm + (size_t)s * STAGE;
      if (info[s].flags & T_FIRST) {
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
        if (lane == 0) {
          tc_fence_after();
          tmem_cp_sf_atom(tmem + C::T_SFB, smem_desc(smem_u32(qsf), 16, 128, kSwizzleNone));
          tmem_cp_sf_atom(tmem + C::T_SFB + 4, smem_desc(smem_u32(qsf + 512), 16, 128, kSwizzleNone));
        }
        __syncwarp();
      }
      if (it >= 2 && !warp_wait(&s_free[k], ((it >> 1) - 1) & 1, 0x604)) break;
      uint8_t* at = sm + C::OFF_ATOM + k * 1024;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 sc = *reinterpret_cast<const uint2*>(st + O_KS + (lane + 32 * j) * 8);
        *reinterpret_cast<uint32_t*>(at + lane * 16 + j * 4) = sc.x;
        *reinterpret_cast<uint32_t*>(at + 512 + lane * 16 + j * 4) = sc.y;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tc_fence_after();
        const uint32_t sfa = tmem + C::T_SFA + 8 * k;
        const uint64_t ad = smem_desc(smem_u32(at), 16, 128, kSwizzleNone);
        const uint64_t kd = smem_desc(smem_u32(st), 16, 512, kSwizzle64B);
        tmem_cp_sf_atom(sfa, ad);
        tmem_cp_sf_atom(sfa + 4, ad + (512 >> 4));
        mma_nvf4(tmem + C::T_S + NB * k, kd, qdesc, idesc, sfa, tmem + C::T_SFB, 0u);
        mma_nvf4(tmem + C::T_S + NB * k, kd + (32 >> 4), qdesc + (32 >> 4), idesc, sfa + 4, tmem + C::T_SFB + 4, 1u);
        tc_commit(&s_full[k]);
        tc_commit(&empty[s]);
      }
      __syncwarp();
    }
    if (lane == 0) {
      tc_commit(&drained[0]);  // what was issued completes before TMEM is released
      mbar_drain(&drained[0], 0);
    }
  } else if (n_it > 0 && warp == 2) {
    // ------------------------------------------------------------------ O^T
    if (lane == 0) {
      const uint32_t idesc = idesc_f16_mn(128, NB);
      int entries[2] = {0, 0};
#pragma unroll 1
      for (int it = 0; it < n_it; ++it) {
        const int k = it & 1, j = it % ST;
        if (!wait_for(&v_full[k], (it >> 1) & 1, 0x605)) break;
        bool first = v_first[k] != 0;
        if (first && !C::FLUSH) {
          const int n = j ? entries[1]++ : entries[0]++;
          if (n > 0 && !wait_for(&o_free[j], (n - 1) & 1, 0x606)) break;
        }
        if (!wait_for(&p_full[k], (it >> 1) & 1, 0x607)) break;
        tc_fence_after();
        if (C::FLUSH) first = true;
        const uint32_t o = tmem + C::T_O + NB * (it % OB);
        const uint64_t vd = MnTile<128>::desc(smem_u32(sm + C::OFF_V) + k * V16);
        const uint64_t wd = MnTile<NB>::desc(smem_u32(sm + C::OFF_P) + k * PL * C::PBYTES);
#pragma unroll
        for (int ks = 0; ks < TK / 16; ++ks)
#pragma unroll
          for (int pl = 0; pl < PL; ++pl)
            mma_f16_ss(o, vd + ks * MnTile<128>::STEP, wd + ks * MnTile<NB>::STEP + pl * (C::PBYTES >> 4), idesc,
                       first && ks == 0 && pl == 0 ? 0u : 1u);
        tc_commit(&pv_done[k]);
      }
      tc_commit(&drained[1]);
      mbar_drain(&drained[1], 0);
    }
  } else if (n_it > 0 && warp < C::DW0) {
    // -------------------------------------------------------------- softmax
    const int group = (warp - C::SW0) >> 2, stream = ST == 2 ? group : 0, c0 = ST == 2 ? 0 : group * 16;
    const int quarter = warp & 3, key = quarter * 32 + lane;
    const uint32_t bar_id = 1 + group, lanes = (uint32_t)(quarter * 32) << 16;
    float(&rd)[4][16] = red[group];
    float *cc = &colc[stream][c0], *cb = &colb[stream][c0];
    uint64_t l2[8];
    float of[16];  // O of this lane's channel, when it is summed here
    // fp32 outputs: the tensor cores cut off what they add to an accumulator, always towards 0 (2e-6 of the result
    // after 14 tiles), so each tile's product starts anew and O is summed in registers.
    auto flush = [&](int j) {
      const bool ok = warp_wait(&pv_done[j & 1], (j >> 1) & 1, 0x608);
      tc_fence_after();
      uint32_t o[16];
      tmem_ld16(tmem + lanes + C::T_O + NB * (j % OB) + c0, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) of[i] += __uint_as_float(o[i]);
      tc_fence_before();
      return ok;
    };
    int merges = 0;
#pragma unroll 1
    for (int it = stream; it < n_it; it += ST) {
      const int s = it % NS, k = it & 1, turn = (it / ST) & 1;
      bool ok = warp_wait(&full[s], (it / NS) & 1, 0x609);
      const int flags = info[s].flags, pos0 = info[s].pos, live = info[s].rows - info[s].rt * NB - c0;
      const int base = info[s].base, len = info[s].len;
      const int64_t row0 = (((int64_t)info[s].b * a.c.num_kv_heads + info[s].h) * a.RT + info[s].rt) * NB + c0;
      const int eb = info[s].b, eh = info[s].h, r0 = info[s].rt * NB + c0;
      const uint8_t* st = sm + (size_t)s * STAGE;
      // this key's factors; keys past the end are not visible, whatever the stage holds for them
      float ak = *reinterpret_cast<const float*>(st + O_KG + key * 4);
      float gv = *reinterpret_cast<const float*>(st + O_VG + key * 4);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      const int pos = pos0 + key;
      const bool first = flags & (ST == 2 ? T_FIRST | T_SECOND : T_FIRST);
      const bool edge = pos0 + TK > base;  // drafted tokens, or the sequence's end
      const bool idle = C::CHUNKS > 1 && live <= 0;  // no row of the entry in this chunk
      if (__builtin_expect(first, 0)) {
        // the factors of the rows' scores, and m = -inf
        if (key < 16) {
          cb[key] = key < live ? a.q_f[row0 + key] : 0.0f;
          cc[key] = INFINITY;  // W_BIAS - m
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) l2[i] = 0ull;
#pragma unroll
        for (int i = 0; i < 16; ++i) of[i] = 0.0f;
        named_bar(bar_id, 128);
      }
      if (pos >= len) ak = 0.0f, gv = 1.0f;
      const float gs = gv >= GV_MIN ? gv : 1.0f;  // 0 and NaN: V^ is 0 there
      const float lg = gv != gv ? gv : lg2(gs), rg = rcp(gs) * L_SCALE;
      ok = warp_wait(&s_full[k], (it >> 1) & 1, 0x60a) && ok;
      tc_fence_after();
      uint32_t acc[16];
      tmem_ld16(tmem + lanes + C::T_S + NB * k + c0, acc);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[k]);
      if (!idle) {
        // -inf marks what a row does not see
        uint32_t seen = 0xffffu;
        if (__builtin_expect(edge, 0)) {
          const int jn = pos - base;
          if (pos >= len) {
            seen = 0u;
          } else if (jn >= 0) {
            if (a.causal) {
              const int cmin = jn * a.G - r0;  // rows of node >= jn
              seen = cmin >= 16 ? 0u : cmin <= 0 ? seen : (seen << cmin) & 0xffffu;
            } else {
              const uint32_t* bits = a.bits + ((int64_t)eb * a.N + jn) * a.nw;
              int i = r0 / a.G, g = r0 - i * a.G;
              seen = 0u;
#pragma unroll 1
              for (int j = 0; j < 16; ++j) {
                if (i < a.N) seen |= ((bits[i >> 5] >> (i & 31)) & 1u) << j;
                if (++g == a.G) g = 0, ++i;
              }
            }
          }
        }
        // y = x - m + W_BIAS, x = S scaling log2(e) + log2(g_v)
        float y[16];
        auto scores = [&]() {
          const uint64_t ak2 = pk2(ak, ak), lg2v = pk2(lg, lg);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const ulonglong2 b4 = *reinterpret_cast<const ulonglong2*>(&cb[j]);
            const ulonglong2 c4 = *reinterpret_cast<const ulonglong2*>(&cc[j]);
            upk2(fma2(mul2(pk2(__uint_as_float(acc[j]), __uint_as_float(acc[j + 1])), ak2), b4.x, add2(lg2v, c4.x)), y[j],
                 y[j + 1]);
            upk2(fma2(mul2(pk2(__uint_as_float(acc[j + 2]), __uint_as_float(acc[j + 3])), ak2), b4.y, add2(lg2v, c4.y)),
                 y[j + 2], y[j + 3]);
          }
          if (__builtin_expect(edge, 0)) {
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = (seen >> j) & 1u ? y[j] : -INFINITY;
          }
        };
        scores();
        const float t0 = max3f(max3f(y[0], y[1], y[2]), max3f(y[3], y[4], y[5]), max3f(y[6], y[7], y[8]));
        const float t1 = max3f(max3f(y[9], y[10], y[11]), max3f(y[12], y[13], y[14]), y[15]);
        if (!ok) gave_up[turn][group] = 1;
        bool flushed = false;
        if (__builtin_expect(bar_or(bar_id, 128, fmaxf(t0, t1) > W_BIAS + W_SLACK), 0)) {
          // some score passed its row's m: every row's m becomes the maximum so far
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float v = fmaf(__uint_as_float(acc[j]) * ak, cb[j], lg);
            if (!((seen >> j) & 1u)) v = -INFINITY;
            v = redux_max(v);
            if (lane == j) mx = v;
          }
          if (lane < 16) rd[quarter][lane] = mx;
          named_bar(bar_id, 128);
          const int c = lane & 15;
          const float old = cc[c];
          const float bn = fminf(old, W_BIAS - fmaxf(fmaxf(rd[0][c], rd[1][c]), fmaxf(rd[2][c], rd[3][c])));
          const float f = bn == old ? 1.0f : ex2(bn - old);
          named_bar(bar_id, 128);  // cc and rd have been read
          if (quarter == 0 && lane < 16) cc[c] = bn;
          named_bar(bar_id, 128);
          if (!first) {
            // O of the earlier tiles of this list entry, once they are all in
            uint32_t o[16];
            if constexpr (C::FLUSH) {
              ok = flush(it - ST) && ok, flushed = true;
            } else {
              ok = warp_wait(&pv_done[(it - ST) & 1], ((it - ST) >> 1) & 1, 0x60b) && ok;
              tc_fence_after();
              tmem_ld16(tmem + lanes + C::T_O + NB * (it % OB) + c0, o);
              tmem_ld_wait();
            }
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float f0 = __shfl_sync(0xffffffffu, f, j), f1 = __shfl_sync(0xffffffffu, f, j + 1);
              l2[j / 2] = mul2(l2[j / 2], pk2(f0, f1));
              if constexpr (C::FLUSH) {
                of[j] *= f0, of[j + 1] *= f1;
              } else {
                o[j] = __float_as_uint(__uint_as_float(o[j]) * f0);
                o[j + 1] = __float_as_uint(__uint_as_float(o[j + 1]) * f1);
              }
            }
            if constexpr (!C::FLUSH) {
              tmem_st16(tmem + lanes + C::T_O + NB * (it % OB) + c0, o);
              tmem_st_wait();
              tc_fence_before();
            }
          }
          scores();
        }
        if (it >= 2) ok = warp_wait(&pv_done[k], ((it >> 1) - 1) & 1, 0x60c) && ok;  // W's buffer is free
        uint8_t* wp = sm + C::OFF_P + k * PL * C::PBYTES;
        const uint64_t rg2 = pk2(rg, rg);
#pragma unroll
        for (int j0 = 0; j0 < 16; j0 += 8) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e0 = ex2(y[j0 + 2 * j]), e1 = ex2(y[j0 + 2 * j + 1]);
            l2[j0 / 2 + j] = fma2(pk2(e0, e1), rg2, l2[j0 / 2 + j]);
            const __half2 h2 = __floats2half2_rn(e0, e1);
            hi[j] = *reinterpret_cast<const uint32_t*>(&h2);
            if constexpr (PL == 2) {
              const float2 hf = __half22float2(h2);
              const __half2 r2 = __floats2half2_rn(e0 - hf.x, e1 - hf.y);
              lo[j] = *reinterpret_cast<const uint32_t*>(&r2);
            }
          }
          const uint32_t off = mn_chunk<NB>(key, (c0 + j0) / 8);
          *reinterpret_cast<uint4*>(wp + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (PL == 2) *reinterpret_cast<uint4*>(wp + C::PBYTES + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[k]);
        if constexpr (C::FLUSH)
          if (!first && !flushed) ok = flush(it - ST) && ok;
        // written before this tile's vote, read after it, so the same for all warps of this group
        if (gave_up[turn][group]) break;
      } else {
        if (lane == 0) mbar_arrive(&p_full[k]);
      }
      if (__builtin_expect(flags & (ST == 2 ? T_LAST | T_PENULT : T_LAST), 0)) {
        // --------------------------------------------- a list entry's end
        // l of each row: over the lanes here, over the four warps in rd
        if (!idle) {
          float v[16];
#pragma unroll
          for (int j = 0; j < 8; ++j) upk2(l2[j], v[2 * j], v[2 * j + 1]);
          const float sum = lane_sums16(v);
          if (lane < 16) rd[quarter][lane] = sum;
        } else if (lane < 16) {
          rd[quarter][lane] = 0.0f;
        }
        named_bar(bar_id, 128);
        if constexpr (C::FLUSH) {
          ok = flush(it) && ok;
        } else {
          ok = warp_wait(&pv_done[k], (it >> 1) & 1, 0x60d) && ok;
          tc_fence_after();
          uint32_t o[16];
          tmem_ld16(tmem + lanes + C::T_O + NB * (it % OB) + c0, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) of[j] = __uint_as_float(o[j]);
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_free[stream]);
        float* mg = reinterpret_cast<float*>(sm + C::OFF_MERGE);  // [16][D], c [16], l [16]
        if (ST == 2 && (flags & T_PENULT)) {
          // the other stream has the last tile and takes this one's share
          if (merges > 0) warp_wait(&m_free, (merges - 1) & 1, 0x610);
#pragma unroll
          for (int j = 0; j < 16; ++j) mg[j * PG_D + key] = of[j];
          if (key < 16) mg[16 * PG_D + key] = cc[key], mg[16 * PG_D + 16 + key] = (rd[0][key] + rd[1][key]) + (rd[2][key] + rd[3][key]);
          __syncwarp();
          if (lane == 0) mbar_arrive(&m_full);
        } else {
          const bool other = ST == 2 && !(flags & T_FIRST);
          if (other) warp_wait(&m_full, merges & 1, 0x611);
          const bool whole = flags & T_WHOLE;
          float* part = a.part + ((int64_t)blockIdx.x * 2 + (flags & T_SLOT ? 1 : 0)) * (NB * (PG_D + 2));
          const int all = a.N * a.G - r0;  // columns that the output has
          int i = r0 / a.G, g = r0 - i * a.G;
          int64_t at = (((int64_t)eb * a.N + i) * a.Hq + eh * a.G + g) * PG_D + key;  // key: this lane's channel
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float l = (rd[0][j] + rd[1][j]) + (rd[2][j] + rd[3][j]), v = of[j], c = cc[j];
            if (other) {
              const float l1 = mg[16 * PG_D + 16 + j], cj = mg[16 * PG_D + j], cm = fminf(c, cj);
              const float f0 = c == cm ? 1.0f : ex2(cm - c), f1 = cj == cm ? 1.0f : ex2(cm - cj);
              v = v * f0 + mg[j * PG_D + key] * f1, l = l * f0 + l1 * f1, c = cm;
            }
            if (!whole) {
              part[(c0 + j) * PG_D + key] = v;
              if (key == 0) part[NB * PG_D + c0 + j] = c, part[NB * (PG_D + 1) + c0 + j] = l;
            } else if (j < all) {
              store_out<DT>(a.out, at, j < live && l != 0.0f ? v * (L_SCALE / l) : 0.0f);
            }
            at += PG_D;
            if (++g == a.G) g = 0, at += (int64_t)(a.Hq - a.G) * PG_D;
          }
          __syncwarp();
          if (other && lane == 0) mbar_arrive(&m_free);
        }
        named_bar(bar_id, 128);  // cc and rd are free
      }
      if (ST == 2 && (flags & (T_FIRST | T_LAST)) == T_LAST) ++merges;
      else if (ST == 2 && (flags & T_PENULT)) ++merges;
    }
  } else if (n_it > 0) {
    // ---------------------------------------------------------------- V^
    const int w = (warp - C::DW0) % C::VW;
#pragma unroll 1
    for (int it = (warp - C::DW0) / C::VW; it < n_it; it += ST) {
      const int s = it % NS, k = it & 1;
      if (!warp_wait(&full[s], (it / NS) & 1, 0x60e)) break;
      const uint8_t* st = sm + (size_t)s * STAGE;
      uint8_t* vb = sm + C::OFF_V + k * V16;
      const int left = info[s].len - info[s].pos, fl = info[s].flags;
      if (it >= 2 && !warp_wait(&pv_done[k], ((it >> 1) - 1) & 1, 0x60f)) break;
      if (w == 0 && lane == 0) v_first[k] = fl & (ST == 2 ? T_FIRST | T_SECOND : T_FIRST);
#pragma unroll 1
      for (int i = 0; i < 16 / C::VW; ++i) {
        const int key = (i * C::VW + w) * 8 + (lane & 7), ch = lane >> 3;  // 32 channels from 32 ch
        const uint4 cw = *reinterpret_cast<const uint4*>(st + O_VC + key * 64 + ((ch ^ ((key >> 1) & 3)) << 4));
        uint32_t sc = *reinterpret_cast<const uint16_t*>(st + O_VS + key * 8 + ch * 2);
        const float gv = *reinterpret_cast<const float*>(st + O_VG + key * 4);
        // tokens past the end, NaN tokens and those below GV_MIN contribute nothing (NaN comes in through W)
        if (!(gv >= GV_MIN) || key >= left) sc = 0u;
        const uint32_t s2 = e4m3x2_f16x2(sc), s0 = __byte_perm(s2, s2, 0x1010), s1 = __byte_perm(s2, s2, 0x3232);
        uint32_t o[16];
        e2m1x8_f16(cw.x, o), e2m1x8_f16(cw.y, o + 4), e2m1x8_f16(cw.z, o + 8), e2m1x8_f16(cw.w, o + 12);
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = hmul2_u32(o[j], j < 8 ? s0 : s1);
        const uint32_t row = (ch >> 1) * (TK * 128) + key * 128;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(vb + row + ((((ch & 1) * 4 + j) ^ (key & 7)) << 4)) =
              make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]), mbar_arrive(&v_full[k]);
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
// without a tile are 0.
template <int NB, int DT>
__global__ void __launch_bounds__(256) paged_join_kernel(AttnArgs a, int grid_max) {
  pdl_wait();
  const int lane = threadIdx.x & 31, b = blockIdx.z, rt = blockIdx.y % a.RT, h = blockIdx.y / a.RT;
  const int c = blockIdx.x * 8 + (threadIdx.x >> 5), r = rt * NB + c;
  if (r >= a.N * a.G) return;
  const Row row = a.rows[b];
  const int tiles = tiles_of(row, rt, NB, a.G, a.causal);
  const long long total = a.first[a.B];
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (tiles > 0) {
    int per = 0, before = 0;
    for (int i = 0; i < a.RT; ++i) {
      const int t = tiles_of(row, i, NB, a.G, a.causal);
      if (i < rt) before += t;
      per += t;
    }
    const long long t0 = a.first[b] + (long long)h * per + before, t1 = t0 + tiles - 1;
    const int grid = (int)min((long long)grid_max, total);
    const int c0 = owner_of(total, t0, grid), c1 = owner_of(total, t1, grid);
    if (c0 == c1) return;
    if (r < row.n * a.G) {
      // CTA c0's share is its first segment if its range starts with this entry, else its last; the others' is
      // their first
      auto slot = [&](int i) {
        return a.part + ((int64_t)i * 2 + (i == c0 && range_start(total, c0, grid) < t0 ? 1 : 0)) * (NB * (PG_D + 2));
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
// Rows of a tile: the fewest tiles that hold all rows, as each of them reads the keys again and widens V again.
// fp32 outputs keep W as two planes and O in registers, which leaves room for 32.
int rows_per_tile(int64_t rows, bool fp32) { return rows <= 16 ? 16 : fp32 ? 32 : 64; }

struct Layout {
  int NB, RT, nw, grid;
  int64_t scales, g, bits, rows, first, part, bytes;
};

int64_t piece(int64_t bytes) { return (bytes + 255) / 256 * 256; }

Layout layout_of(int B, int Hq, int Hkv, int N, bool fp32) {
  Layout L;
  const int64_t rows = (int64_t)N * (Hq / Hkv), tok = (int64_t)B * N;
  L.NB = rows_per_tile(rows, fp32);
  L.RT = (int)((rows + L.NB - 1) / L.NB);
  L.nw = (N + 31) / 32;
  static int sms = 0;
  if (!sms) {
    int dev = 0, n = 0;
    sms = cudaGetDevice(&dev) == cudaSuccess &&
                  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0
              ? n
              : 148;
  }
  L.grid = sms;
  const int64_t qrows = (int64_t)B * Hkv * L.RT * L.NB;
  L.scales = piece(qrows * PG_ROW);
  L.g = L.scales + piece(qrows * PG_SF);
  L.bits = L.g + piece(qrows * 4);
  L.rows = L.bits + piece(tok * L.nw * 4);
  L.first = L.rows + piece((int64_t)B * sizeof(Row));
  L.part = L.first + piece((int64_t)(B + 1) * 8);
  L.bytes = L.part + piece((int64_t)L.grid * 2 * L.NB * (PG_D + 2) * 4);
  return L;
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
  return std::max(layout_of(B, Hq, Hkv, N, false).bytes, layout_of(B, Hq, Hkv, N, true).bytes);
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
  const int64_t need = fp4paged_attention_workspace_size(B, Hq, H, N);
  if ((uintptr_t)workspace % 256 || workspace_bytes < need)
    return set_error(FP4ATTN_ERR_ARG, "workspace of %lld bytes, %lld needed (256-byte aligned)",
                     (long long)workspace_bytes, (long long)need);
  const Layout L = layout_of(B, Hq, H, N, out_dtype == FP4_DT_F32);
  // grid limits, 32-bit rows, and the tensor maps' 32-bit row coordinate
  if (B > 65535 || (int64_t)H * L.RT > 65535 || (int64_t)N * (Hq / H) > INT32_MAX / 2 ||
      (int64_t)B * N > INT32_MAX / 2)
    return set_error(FP4ATTN_ERR_UNSUPPORTED, "more than 65535 rows or (KV head, row tile) pairs");
  const int64_t krows = (int64_t)cache->num_pages * H * cache->page_size;
  if (krows > INT32_MAX) return set_error(FP4ATTN_ERR_UNSUPPORTED, "the cache has 2^31 or more (token, head) rows");
  uint8_t* w = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.c = *cache;
  a.q_codes = w, a.q_scales = w + L.scales, a.q_f = reinterpret_cast<float*>(w + L.g);
  a.bits = reinterpret_cast<uint32_t*>(w + L.bits), a.rows = reinterpret_cast<Row*>(w + L.rows);
  a.first = reinterpret_cast<long long*>(w + L.first), a.part = reinterpret_cast<float*>(w + L.part);
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
