// Tree attention over a paged cache on the 5th-generation tensor cores (head dims 64 and 128).
//
// The T * G query rows that share a key head are the rows of one product; keys go through in tiles of
// 64. A block (one per SM) holds two streams, each with its own scores S (two buffers: the next tile's
// scores are formed while this one's exponentials are taken), running maximum and sum, and output O in
// tensor memory:
//   more than 128 rows   the streams are two tiles of 128 rows over the same keys (K and V read once)
//   at most 128 rows     the streams take the even and the odd key tiles of the same rows, joined at the
//                        end: O and O' = O e^(m - M) + O' e^(m' - M)
//
//   S = Q K^T    Q and K in shared memory (128-byte swizzle), S in tensor memory
//   P            a thread per row: maximum, exponentials (fp16, the operand of the next product), sum;
//                P takes S's place in tensor memory
//   O += P V     P from tensor memory, V from shared memory as an MN-major operand
// O is rescaled only when the maximum has risen by more than 2^8: P stays under 2^14 (weights carry a
// factor 2^6, so that the small ones keep their bits), and the sum uses the same factor. P in 16 bits is the price of
// the matrix instruction: each weight is off by 2^-11 at most, the sum is of the unrounded ones, and the output's error
// against 64 bits is 3.3e-4 to 3.6e-4 of its size where fp32 weights give 3.0e-4 (q, k, v and the output are 16 bits).
//
// Work split: the key tiles of all (sequence, key head) pairs in a row are cut into equal runs, one for
// each block, whatever the sequences' lengths; a pair that was cut leaves partial (m, l, O) behind, which
// tree_combine joins in the order of the keys, so the result does not depend on timing. The cut comes
// from lens on the device.
//
// K and V arrive by TMA in boxes of as many rows as divide the page (8..64, or 64 where a sequence is
// one page) into a ring of tiles. Rows before the prefix's end are loaded while tree_append still runs.
// Rows that hold nothing (past the last node, or without a page) are taken out of the scores and zeroed
// in V; nodes whose k or v is not finite are taken out of the products too and added by the row's thread
// at the end, for the rows that see them only.
//
// Roles (384 threads): warps 0-3 and 4-7 the streams' rows, warps 8 and 9 the streams' products (warp 8
// owns the tensor memory), warps 10 and 11 the copies of K (and Q) and of V. Every wait is bounded; a block that
// gives up records AF_DEV_WAIT_TIMEOUT, waits for its copies and products in flight, frees its tensor memory and
// returns.
//
// Bounds, and times of the three kernels together on B200 (8 key heads of 128), 20 calls replayed from a graph:
//   few rows a key     memory. 32 sequences of 8192 rows, one node, groups of 4: 174 us, 6.2 TB/s
//   short or few       latency of the three launches, the copies' first tile and the join: one node at 576 rows
//                      13.4 us, 24 nodes at 4001 rows 21.6 us (tree_append 2.8 and 3 of them)
//   many rows a key    the rows' warps. 8 sequences of 32768 rows, 64 nodes x 4 heads: 313 us, 880 TFLOP/s at 1965 MHz;
//                      called for seconds 375 to 387 us, 720 TFLOP/s: the power limit holds the clock near 1510 MHz.
//                      1.3 us for a tile of 64 keys and 2 x 128 rows, of which the warps of a group work 0.95 us; the
//                      products take 0.76 us at the rate of a large library product, the memory 0.74, the
//                      exponentials alone 0.53 (counters: tensor pipe 48 % of its cycles, memory 45 %, issue 42 %)
//   pages of 16 rows   the copies: four boxes a tile. 12 sequences of 2000..8000 rows, 16 nodes x 8 heads: 77 us,
//                      with pages of 64 rows 63 us
// Tiles of 128 keys with one score buffer took 421 us in the third case; the second buffer keeps the products ahead
// of the exponentials. For at most 128 rows the even / odd streams use both groups of warps.
#include <cuda.h>

#include "af_common.cuh"
#include "af_kernels.h"
#include "tcgen05.cuh"
#include "tree_common.cuh"

namespace af {

namespace tt {
constexpr int BK = TREE_BK;                    // keys per tile
constexpr int THREADS = 384;
constexpr int MMA_WARP = 8, TMA_WARP = 10;     // two warps each
constexpr int QSLICE = 128 * 64 * 2;           // 128 rows x 64 fp16, 128-byte swizzled
constexpr int SLICE = BK * 64 * 2;             // a tile's keys x 64 fp16
constexpr long long LIMIT = 1ll << 26;
constexpr float SHIFT = 6.f, RISE = 8.f;       // log2 of the weights' factor; rise of the maximum that is let pass
constexpr int MAXW = TREE_MAX_NODES / 32;
constexpr int NS = 10;                         // ring slots (K or V tiles)
constexpr int AHEAD = 16;                      // segments that the copies can be ahead: under NS
template <int DH, bool TWO> struct Cfg {
  static constexpr int TILE = SLICE * (DH / 64), QTILE = QSLICE * (DH / 64);
  static constexpr int QT = TWO ? 2 : 1;       // row tiles
  static constexpr int QB = TWO ? 1 : 2;       // Q buffers: few rows come with short segments, whose Q is fetched ahead
  static constexpr int RING = 2 * QTILE;
  static constexpr int SH = RING + NS * TILE;
  // Split streams have half of the ring each: a slot's fills are waited for by one warp, in order. (A parity
  // cannot tell a fill from the one before the last, so nobody may wait for a fill before the last one of its
  // slot has landed.)
  static constexpr int HS = TWO ? NS : NS / 2;
};
constexpr uint32_t S_COL = 0, O_COL = 256;     // S / P of stream w at 128 w (two buffers of 64), O at 256 + 128 w
constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
template <int DH> struct IdescPV {
  static constexpr uint32_t v = (1u << 4) | (1u << 16) | ((uint32_t)(DH >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
};
}  // namespace tt

struct TreeShared {
  uint64_t q_full[2], q_empty[2];
  uint64_t full[tt::NS], empty[tt::NS];
  uint64_t s_full[2][2], p_full[2][2];         // of a stream's buffers
  uint64_t pv_done[2];                         // a stream's O += P V is done (every tile)
  uint64_t o_full[2], acc_free[2];             // a stream's O is complete; read out (every segment with tiles for it)
  uint64_t done;
  float2 ml[2][128];                           // split streams: (m, l) of the other half
  uint32_t vmask[tt::NS];                      // boxes of the tile that have a page
  uint32_t bad[tt::AHEAD][tt::MAXW];           // nodes whose k or v is not finite, of a segment (modulo AHEAD)
  uint32_t tmem;
  int holes;                                   // some row of the segments so far has no page
  int abort;
};

AF_DEV bool tt_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  SpinBudget budget;
  for (long long i = 0; i < tt::LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 255 && (*abort || budget.spent())) return false;
  }
  return false;
}
AF_DEV bool tt_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, tt_wait(bar, parity, abort));
}

// whether the phase is over, without waiting; one answer for the warp
AF_DEV bool tt_done_warp(uint64_t* bar, uint32_t parity) {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
               : "=r"(r) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, r != 0);
}

// barrier of the 256 row threads; true if `ok` holds in all of them
AF_DEV bool rows_all(bool ok) {
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, 1, 256, p;\n selp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(r) : "r"((uint32_t)ok) : "memory");
  return r != 0;
}

AF_DEV float tt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

#define TT_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define TT_R32(v, o) TT_R8(v, o), TT_R8(v, o + 8), TT_R8(v, o + 16), TT_R8(v, o + 24)
#define TT_RW8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
// 32 columns of this warp's 32 lanes, on their way until tmem_ld_wait; the registers are touched after it only
AF_DEV void tmem_ld32_async(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : TT_R32(v, 0)
      : "r"(taddr)
      : "memory");
}
AF_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
AF_DEV void after_wait(uint32_t (&v)[32]) { asm volatile("" : TT_RW8(v, 0), TT_RW8(v, 8), TT_RW8(v, 16), TT_RW8(v, 24)); }

#define TT_IN16(v) "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), \
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
AF_DEV void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "{\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n}\n"
      : TT_R8(v, 0), TT_R8(v, 8)
      : "r"(taddr)
      : "memory");
}
AF_DEV void tmem_st16_async(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::TT_IN16(v),
      "r"(taddr)
      : "memory");
}
AF_DEV void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  tmem_st16_async(taddr, v);
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

AF_DEV void mma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
      ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}

// the same with the accumulation known beforehand
AF_DEV void mma_f16_c(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  if (accumulate)
    asm volatile("{\n .reg .pred p;\n setp.eq.u32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 ::"r"(d), "l"(adesc), "l"(bdesc), "r"(idesc) : "memory");
}
AF_DEV void mma_f16_ts_c(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc) {
  asm volatile("{\n .reg .pred p;\n setp.eq.u32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d), "r"(a), "l"(bdesc), "r"(idesc) : "memory");
}
AF_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// a box of a page: rows from `row`, 64 columns from 64 * half (or all 128 columns, as two slices)
AF_DEV void tma_load_5d(void* dst, const CUtensorMap* map, int row, int half, int h, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(0), "r"(row), "r"(half), "r"(h), "r"(page), "r"(smem_u32(bar)) : "memory");
}

// where a stream's K and V stand in the order in which they are loaded and used: K0 K1 V0 K2 V1 ... (the
// scores are formed two tiles ahead)
AF_DEV int seq_k(int i) { return i < 2 ? i : 2 * i - 1; }
AF_DEV int seq_v(int i, int n) { return i < n - 2 ? 2 + 2 * i : n + i; }

// visibility of the 64 nodes from node number u0 (may be negative: prefix rows) for a node's mask row; the
// three words that this can reach are loaded together
AF_DEV void see64(const int* mask, int words, int t, int u0, uint32_t (&vis)[2]) {
  const int w0 = u0 >> 5, s = u0 & 31;         // floor division: u0 = 32 w0 + s
  uint32_t x[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int w = w0 + k;
    x[k] = 0;
    if (mask && w >= 0 && w < words) x[k] = (uint32_t)__ldg(mask + w);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int w = w0 + k, n = t - 32 * w;      // chain: nodes 0..t
    if (w < 0) x[k] = 0xffffffffu;
    else if (!mask) x[k] = n < 0 ? 0u : n >= 31 ? 0xffffffffu : (2u << n) - 1;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) vis[k] = __funnelshift_r(x[k], x[k + 1], s);
}
AF_DEV uint32_t ones_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// what a row's thread has at the end of a segment: its O (one or two accumulators with their weights), m, l
struct TreeEnd {
  uint32_t o0, o1;
  bool have0, have1;
  float f0, f1, m, l;
  int c0, r, t, pr;
  float* part;                                 // where a cut pair's partial result goes; null: the pair is whole
};

template <int DH, bool TWO> struct EndCols { static constexpr int n = TWO ? DH : DH / 2; };

// 16 columns from c0 of the row's sum (a warp)
AF_DEV void tree_take(const TreeEnd& e, int c0, float (&x)[16]) {
  uint32_t o[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) x[k] = 0.f;
  if (e.have0) {
    tmem_ld16(e.o0 + c0, o);
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = __uint_as_float(o[k]) * e.f0;
  }
  if (e.have1) {
    tmem_ld16(e.o1 + c0, o);
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] = fmaf(__uint_as_float(o[k]), e.f1, x[k]);
  }
}

template <int DH>
AF_DEV void tree_put(const AttnTreeArgs& a, int b, int h, int nodes, const TreeEnd& e, int c0, const float (&x)[16]) {
  const int G = a.H / a.KV;
  if (e.r >= a.T * G) return;
  if (e.part) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      __stcg(reinterpret_cast<float4*>(e.part) + (size_t)(c0 / 4 + q) * a.part_rows + e.pr,
             make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]));
    return;
  }
  const float il = e.t >= nodes || e.l == 0.f ? 0.f : 1.f / e.l;       // NaN stays
  __half* dst = a.out + ((size_t)b * a.T + e.t) * a.ld_out + (size_t)(h * G + e.r - e.t * G) * DH + c0;
  __half2 y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = e.t >= nodes ? __half2() : __floats2half2_rn(x[2 * k] * il, x[2 * k + 1] * il);
  if (a.out16) {
    reinterpret_cast<uint4*>(dst)[0] = reinterpret_cast<const uint4*>(y)[0];
    reinterpret_cast<uint4*>(dst)[1] = reinterpret_cast<const uint4*>(y)[1];
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) { dst[2 * k] = __low2half(y[k]); dst[2 * k + 1] = __high2half(y[k]); }
  }
}

template <int DH, bool TWO>
AF_DEV void tree_store(const AttnTreeArgs& a, int b, int h, int nodes, const TreeEnd& e) {
  if (e.part && (TWO || e.c0 == 0) && e.r < a.T * (a.H / a.KV))
    __stcg(reinterpret_cast<float2*>(e.part + (size_t)a.part_rows * DH) + e.pr, make_float2(e.m, e.l));
#pragma unroll 1
  for (int c0 = e.c0; c0 < e.c0 + EndCols<DH, TWO>::n; c0 += 16) {
    float x[16];
    tree_take(e, c0, x);
    tree_put<DH>(a, b, h, nodes, e, c0, x);
  }
}

// The same where nodes of the sequence are not finite: they were left out of the products, and are added to
// the rows that see them here, key by key.
template <int DH, bool TWO>
__device__ __noinline__ void tree_bad_nodes(const AttnTreeArgs& a, int b, int h, int len, int nodes, const uint32_t* bad,
                                            const int* mrow, TreeEnd e) {
  const int R = a.T * (a.H / a.KV);
  const bool in = e.r < R;
  const float sl2 = a.scale * 1.4426950408889634f;
  auto sees = [&](int u) {
    return (bad[u >> 5] >> (u & 31) & 1) && (mrow ? (__ldg(mrow + (u >> 5)) >> (u & 31)) & 1 : u <= e.t);
  };
  auto row = [&](const __half* c, int u) -> const __half* {
    const int j = len + u, p = __ldg(a.table + (size_t)b * a.W + j / a.page);
    return p < 0 || p >= a.P ? nullptr : c + (size_t)p * a.page_stride + ((size_t)h * a.page + j % a.page) * DH;
  };
  auto score = [&](const __half* k) {
    const __half* q = a.q + (((size_t)b * a.KV + h) * R + e.r) * DH;
    float s = 0.f;
    for (int d = 0; d < DH; ++d) s = fmaf(h2f(__ldcg(q + d)), h2f(__ldcg(k + d)), s);
    return s * sl2;
  };
  float m2 = e.m;
  for (int u = 0; in && u < nodes; ++u)
    if (sees(u))
      if (const __half* k = row(a.kc, u)) m2 = fmaxf(m2, score(k));
  const float c = e.m == -INFINITY ? 0.f : tt_ex2(e.m - m2);
  e.f0 *= c; e.f1 *= c; e.l *= c;
  e.m = m2;
  for (int u = 0; in && u < nodes; ++u)
    if (sees(u))
      if (const __half* k = row(a.kc, u)) e.l += tt_ex2(score(k) - (e.m - tt::SHIFT));
  if (e.part && (TWO || e.c0 == 0) && in)
    __stcg(reinterpret_cast<float2*>(e.part + (size_t)a.part_rows * DH) + e.pr, make_float2(e.m, e.l));
#pragma unroll 1
  for (int c0 = e.c0; c0 < e.c0 + EndCols<DH, TWO>::n; c0 += 16) {
    float x[16];
    tree_take(e, c0, x);
    for (int u = 0; in && u < nodes; ++u)
      if (sees(u))
        if (const __half* k = row(a.kc, u)) {
          const __half* v = row(a.vc, u) + c0;
          const float p = tt_ex2(score(k) - (e.m - tt::SHIFT));
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = fmaf(p, h2f(__ldcg(v + i)), x[i]);
        }
    __syncwarp();
    tree_put<DH>(a, b, h, nodes, e, c0, x);
  }
}

template <int DH, bool TWO>
__global__ void __launch_bounds__(tt::THREADS, 1)
    attn_tree_tc_kernel(const __grid_constant__ AttnTreeArgs a, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap) {
  using namespace tt;
  using C = Cfg<DH, TWO>;
  constexpr int TILE = C::TILE, QTILE = C::QTILE, HS = C::HS;
  // the swizzle's period is 1024 bytes; there is no room to align by hand, so a wrong base is an error
  extern __shared__ __align__(1024) unsigned char tt_raw[];
  unsigned char* smem = tt_raw;
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) af_set_err(a.err, AF_DEV_WAIT_TIMEOUT);
    return;
  }
  TreeShared* sh = reinterpret_cast<TreeShared*>(smem + C::SH);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.KV, R = a.T * G;
  pdl_trigger();
  TreeSched sc;
  if (!sc.init(a, blockIdx.x, gridDim.x, lane)) return;      // fewer tiles than blocks

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&sh->full[s], 1);
      mbar_init(&sh->empty[s], C::QT);         // every stream that reads it
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&sh->q_full[w], 1);
      mbar_init(&sh->q_empty[w], 2);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&sh->s_full[w][k], 1);
        mbar_init(&sh->p_full[w][k], 4);
      }
      mbar_init(&sh->pv_done[w], 1);
      mbar_init(&sh->o_full[w], 1);
      mbar_init(&sh->acc_free[w], 8);
    }
    mbar_init(&sh->done, 2);
    sh->abort = 0;
    sh->holes = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&sh->tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sh->tmem;
  volatile int* abort = &sh->abort;

  if (warp >= TMA_WARP) {
    // ------------------------------------------------------------- copies: a warp for K (and Q), one for V
    const bool is_v = warp == TMA_WARP + 1, leader = elect_one();
    const int nbox = BK >> a.box_shift, per = 32 / nbox;     // boxes of a tile (at most 8), tiles of a page read
    bool waited = false, ok = true;
    int seq0[2] = {0, 0}, nseg = 0, nq = 0;                  // loads of each stream so far (two row tiles: of both)
    uint32_t armed = 0, phase = 0;                           // slots that were filled here, and their last phase
    auto dependency = [&] {                                  // q and the nodes' rows come from tree_append
      if (waited) return;
      pdl_wait();
      asm volatile("fence.proxy.async.global;" ::: "memory");
      waited = true;
    };
    for (bool more = true; ok && more; more = sc.next(a), ++nseg) {
      const int nt = sc.tiles();
      bool have_q = is_v;
      if (!is_v) {
        // only a segment that meets the nodes has any that are not finite
        const bool tail = (sc.t0 + nt) * BK > sc.len && sc.nodes > 0;
        if (tail) dependency();
        for (int k = 0; k < MAXW; ++k) {
          unsigned m = 0;
          if (tail && 32 * k < sc.nodes) {
            const int u = 32 * k + lane;
            m = __ballot_sync(0xffffffffu, u < sc.nodes && __ldcg(a.flags + ((size_t)sc.b * a.KV + sc.h) * a.T + u));
          }
          if (lane == 0) *(volatile uint32_t*)&sh->bad[nseg % AHEAD][k] = m;
        }
      }
      // Q of segment n lies in buffer n mod QB, free once the scores of segment n - QB are done
      const int qb = nseg % C::QB, qn = nseg / C::QB;
      auto load_q = [&]() -> bool {
        dependency();
        if (qn && !tt_wait_warp(&sh->q_empty[qb], (uint32_t)((qn - 1) & 1), abort)) return false;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh->q_full[qb], C::QT * QTILE);
          for (int w = 0; w < C::QT; ++w)
            for (int k = 0; k < DH / 64; ++k)
              tma_load_3d(smem + (qb + w) * QTILE + k * QSLICE, &qmap, 64 * k, sc.rg * 256 + 128 * w, sc.b * a.KV + sc.h,
                          &sh->q_full[qb]);
        }
        have_q = true;
        ++nq;
        return true;
      };
      // the pages of `per` tiles at a time, a lane each; -2: no row in the box
      auto pages_of = [&](int j) {
        const int row = (sc.t0 + j) * BK + lane * a.box_rows;
        const int w = a.page_shift >= 0 ? row >> a.page_shift : row / a.page;
        return j < nt && row < sc.len + sc.nodes ? __ldg(a.table + (size_t)sc.b * a.W + w) : -2;
      };
      int pages = -2, pages1 = pages_of(0);
      for (int j = 0; j < nt; ++j) {
        const int w = TWO ? 0 : j & 1, n = TWO ? nt : (nt + 1 - w) >> 1, i = TWO ? j : j >> 1;
        const int local = is_v ? seq_v(i, n) : seq_k(i), seq = (w ? seq0[1] : seq0[0]) + local, st = w * HS + seq % HS;
        const int g = j % per;
        if (g == 0) {
          pages = pages1;
          pages1 = pages_of(j + per);
          if (pages != -2 && (pages < 0 || pages >= a.P)) {
            pages = -1;
            *(volatile int*)&sh->holes = 1;
            af_set_err(a.err, AF_DEV_BAD_POS);
          }
          __syncwarp();                                      // `holes` is written before the leader's next arrival
        }
        const unsigned live = (__ballot_sync(0xffffffffu, pages >= 0) >> (g * nbox)) & ((1u << nbox) - 1);
        if ((sc.t0 + j + 1) * BK > sc.len) dependency();     // the nodes' rows
        // Q at the latest when the ring is full of this segment; before, once the last one's scores are done
        if (!have_q && (local >= HS || (waited && (!qn || tt_done_warp(&sh->q_empty[qb], (uint32_t)((qn - 1) & 1))))) && !load_q()) {
          ok = false;
          break;
        }
        if (seq >= HS && !tt_wait_warp(&sh->empty[st], (uint32_t)((seq / HS - 1) & 1), abort)) { ok = false; break; }
        if (leader) {
          sh->vmask[st] = live;
          mbar_arrive_expect_tx(&sh->full[st], (uint32_t)(__popc(live) * a.box_rows * (DH * 2)));
        }
        // one lane issues all copies: their operands are the warp's, several lanes would take turns
        const int row = (sc.t0 + j) * BK;
        unsigned char* slot = smem + C::RING + st * TILE;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        int pk[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) pk[k] = __shfl_sync(0xffffffffu, pages, (g * nbox + k) & 31);
        if (leader) {
          if (nbox == 1) {
            if (pk[0] >= 0) tma_load_5d(slot, map, a.page_shift >= 0 ? row & (a.page - 1) : row % a.page, 0, sc.h, pk[0], &sh->full[st]);
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < nbox && pk[k] >= 0) {
                const int y = row + k * a.box_rows, in = a.page_shift >= 0 ? y & (a.page - 1) : y % a.page;
#pragma unroll
                for (int c = 0; c < DH / 64; ++c)
                  tma_load_5d(slot + c * SLICE + k * a.box_rows * 128, map, in, c, sc.h, pk[k], &sh->full[st]);
              }
          }
        }
        __syncwarp();
        armed |= 1u << st;
        phase = (phase & ~(1u << st)) | (uint32_t)((seq / HS) & 1) << st;
      }
      if (ok && !have_q) ok = load_q();
      seq0[0] += 2 * (TWO ? nt : (nt + 1) >> 1);
      seq0[1] += 2 * (nt >> 1);
    }
    if (!ok) *abort = 1;
    dependency();
    // shared memory must outlive every copy issued: a block that gave up waits (bounded) for the last ones
    if (!ok) {
      for (int st = 0; st < NS; ++st) {
        SpinBudget b;
        while ((armed >> st & 1) && !mbar_try_wait(&sh->full[st], phase >> st & 1) && !b.spent()) {
        }
      }
      SpinBudget b;
      for (int k = max(0, nq - C::QB); k < nq; ++k)
        while (!mbar_try_wait(&sh->q_full[k % C::QB], (uint32_t)((k / C::QB) & 1)) && !b.spent()) {
        }
    }
  } else if (warp >= MMA_WARP) {
    // ------------------------------------------------------------- products: a warp for each stream
    // The whole warp walks through them, so that descriptors stay in uniform registers; one lane issues (in a
    // branch of one lane alone every product cost about 70 cycles of moves to uniform registers).
    const int w = warp - MMA_WARP;
    const bool leader = elect_one();
    bool ok = true;
    int seq0 = 0, nseg = 0;
    uint32_t cs = 0, cv = 0;                                 // tiles so far: scores, values
    int nown = 0;                                            // segments with tiles for this stream
    const uint64_t qdesc0 = smem_desc(smem_u32(smem)), kdesc0 = smem_desc(smem_u32(smem + C::RING));
    const uint64_t vdesc0 = smem_desc_mn(smem_u32(smem + C::RING), SLICE, 1024);
    for (bool more = true; ok && more; more = sc.next(a), ++nseg) {
      const int nt = sc.tiles(), qb = nseg % C::QB;
      const int n = TWO ? nt : (nt + 1 - w) >> 1;            // the stream's tiles
      auto scores = [&](int i) -> bool {
        const int seq = seq0 + seq_k(i), st = (TWO ? 0 : w * HS) + seq % HS;
        if (!tt_wait_warp(&sh->full[st], (uint32_t)((seq / HS) & 1), abort)) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t kd = kdesc0 + (uint32_t)(st * (TILE >> 4)), qd = qdesc0 + (uint32_t)((TWO ? w : qb) * (QTILE >> 4));
        const uint32_t buf = cs & 1, d = tmem + S_COL + 128 * w + 64 * buf;
        if (leader) {
#pragma unroll
          for (int ks = 0; ks < DH / 16; ++ks)
            mma_f16_c(d, qd + (uint32_t)(((ks >> 2) * QSLICE + (ks & 3) * 32) >> 4), kd + (uint32_t)(((ks >> 2) * SLICE + (ks & 3) * 32) >> 4),
                      IDESC_S, ks != 0);
          mma_commit(&sh->s_full[w][buf]);
          mma_commit(&sh->empty[st]);
          if (i == n - 1) mma_commit(&sh->q_empty[qb]);
        }
        __syncwarp();
        ++cs;
        return true;
      };
      ok = tt_wait_warp(&sh->q_full[qb], (uint32_t)((nseg / C::QB) & 1), abort);
      for (int i = 0; ok && i < min(2, n); ++i) ok = scores(i);
      if (n == 0 && leader) mbar_arrive(&sh->q_empty[qb]);   // no tile for this stream
      __syncwarp();
      if (ok && n) {                                         // O is free once the stream's last segment was read out
        if (nown) ok = tt_wait_warp(&sh->acc_free[w], (uint32_t)((nown - 1) & 1), abort);
        ++nown;
      }
      for (int i = 0; ok && i < n; ++i) {
        const int seq = seq0 + seq_v(i, n), st = (TWO ? 0 : w * HS) + seq % HS;
        const uint32_t buf = cv & 1;
        ok = tt_wait_warp(&sh->full[st], (uint32_t)((seq / HS) & 1), abort) &&
             tt_wait_warp(&sh->p_full[w][buf], (cv >> 1) & 1, abort);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t vd = vdesc0 + (uint32_t)(st * (TILE >> 4));
        const uint32_t d = tmem + O_COL + 128 * w, p = tmem + S_COL + 128 * w + 64 * buf;
        if (leader) {
          mma_f16_ts(d, p, vd, IdescPV<DH>::v, i != 0);      // the first tile begins O
#pragma unroll
          for (int ks = 1; ks < BK / 16; ++ks) mma_f16_ts_c(d, p + ks * 8, vd + (uint32_t)(ks * 2048 >> 4), IdescPV<DH>::v);
          mma_commit(&sh->pv_done[w]);
          mma_commit(&sh->empty[st]);
          if (i == n - 1) mma_commit(&sh->o_full[w]);
        }
        __syncwarp();
        ++cv;
        if (i + 2 < n) ok = scores(i + 2);
      }
      seq0 += 2 * n;
    }
    if (leader) {
      if (!ok) *abort = 1;
      mma_commit(&sh->done);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- rows (two groups of four warps)
    const int w = warp >> 2, wr = (warp & 3) * 32 + lane;    // stream, row of the tile = TMEM lane
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t scol0 = lanes + S_COL + 128 * w, ocol = lanes + O_COL + 128 * w;
    const float sl2 = a.scale * 1.4426950408889634f;
    bool ok = true;
    int seq0 = 0, nseg = 0;
    uint32_t ns = 0, no0 = 0, no1 = 0;                       // tiles of this stream; segments with tiles for stream 0, 1
    pdl_wait();                                              // q, for the nodes that are added at the end
    for (bool more = true; more; more = sc.next(a), ++nseg) {
      // all rows go on, or none (barriers lie ahead); `bad` is free from here
      ok = rows_all(ok);
      if (!ok) break;
      const int nt = sc.tiles();
      const int r = (TWO ? sc.rg * 256 + 128 * w : 0) + wr;  // row of the pair
      const bool live_warp = r - lane < R, in = r < R;
      const int t = in ? r / G : 0;
      const int* mrow = a.mask ? a.mask + ((size_t)sc.b * a.T + t) * a.mask_words : nullptr;
      const uint32_t* bad = sh->bad[nseg % AHEAD];           // written before the segment's first copy
      float m = -INFINITY, l = 0.f;
      bool first = true;
      for (int j = TWO ? 0 : w; j < nt; j += TWO ? 1 : 2) {
        const int j0 = (sc.t0 + j) * BK;
        const bool odd = j0 + BK > sc.len;                   // reaches past the prefix
        uint32_t vis[2];                                     // visible keys, while the scores are on their way
        if (odd) {
          see64(mrow, a.mask_words, t, j0 - sc.len, vis);
#pragma unroll
          for (int c = 0; c < 2; ++c) vis[c] &= ones_below(sc.len + sc.nodes - j0 - 32 * c);
        }
        const uint32_t buf = ns & 1, scol = scol0 + 64 * buf;
        if (!tt_wait_warp(&sh->s_full[w][buf], (ns >> 1) & 1, abort)) { ok = false; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        bool any_bad = false;
        if (odd || *(volatile int*)&sh->holes) {
#pragma unroll
          for (int k = 0; k < MAXW; ++k) any_bad |= bad[k] != 0;
          // keys that are not there: out of the scores; rows of V that nobody may see become zeros (whatever
          // lies there times a weight of 0 must be 0)
          const int seqv = seq0 + (TWO ? seq_v(j, nt) : seq_v(j >> 1, (nt + 1 - w) >> 1)), stv = (TWO ? 0 : w * HS) + seqv % HS;
          if (!tt_wait_warp(&sh->full[stv], (uint32_t)((seqv / HS) & 1), abort)) { ok = false; break; }
          const uint32_t boxes = *(volatile uint32_t*)&sh->vmask[stv];
          const int u = j0 + wr - sc.len;
          const bool isbad = any_bad && u >= 0 && u < TREE_MAX_NODES && (bad[u >> 5] >> (u & 31) & 1);
          if (wr < BK && (u >= sc.nodes || !(boxes >> (wr >> a.box_shift) & 1) || isbad)) {
            unsigned char* vt = smem + C::RING + stv * TILE;
#pragma unroll 1
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(vt + (c >> 3) * SLICE + sw128(wr, c & 7)) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          if (live_warp) {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t x = !odd ? 0xffffffffu : c ? vis[1] : vis[0];
              for (int e = 0; e < 32; e += 8)                // a box has at least 8 rows
                if (!(boxes >> ((32 * c + e) >> a.box_shift) & 1)) x &= ~(0xffu << e);
              if (any_bad)                                   // not the nodes that are added at the end
#pragma unroll 1
                for (int e = 0; e < 32; ++e) {
                  const int n = j0 + 32 * c + e - sc.len;
                  if (n >= 0 && n < TREE_MAX_NODES && (bad[n >> 5] >> (n & 31) & 1)) x &= ~(1u << e);
                }
              if (__all_sync(0xffffffffu, x == 0xffffffffu)) continue;
              uint32_t v[32];
              tmem_ld32(scol + 32 * c, v);
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = x >> e & 1 ? v[e] : 0xff800000u;
              tmem_st32(scol + 32 * c, v);
            }
          }
        }
        if (live_warp) {
          uint32_t v[2][32];
          tmem_ld32_async(scol, v[0]);
          tmem_ld32_async(scol + 32, v[1]);
          tmem_ld_wait();
          after_wait(v[0]);
          after_wait(v[1]);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(v[0][e]));
            mx[2 + (e & 1)] = fmaxf(mx[2 + (e & 1)], __uint_as_float(v[1][e]));
          }
          const float tm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
          const bool rise = tm > m + (first ? 0.f : RISE) || m == -INFINITY;
          if (__any_sync(0xffffffffu, rise)) {
            const float mn = fmaxf(m, tm);
            const float corr = m == -INFINITY ? 0.f : tt_ex2(m - mn);
            m = mn;
            l *= corr;
            if (!first) {
              // once the products before this tile are done
              if (!tt_wait_warp(&sh->pv_done[w], (ns - 1) & 1, abort)) { ok = false; break; }
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int c0 = 0; c0 < DH; c0 += 16) {
                uint32_t o[16];
                tmem_ld16(ocol + c0, o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                tmem_st16(ocol + c0, o);
              }
            }
          }
          const float mb = m == -INFINITY ? 0.f : m - SHIFT;
          float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {                      // P takes the scores' first columns
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = tt_ex2(fmaf(__uint_as_float(v[h][2 * e]), sl2, -mb));
              const float p1 = tt_ex2(fmaf(__uint_as_float(v[h][2 * e + 1]), sl2, -mb));
              ps[(e & 1) * 2] += p0;
              ps[(e & 1) * 2 + 1] += p1;
              const __half2 hp = __floats2half2_rn(p0, p1);
              pk[e] = *reinterpret_cast<const uint32_t*>(&hp);
            }
            tmem_st16_async(scol + 16 * h, pk);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        }
        first = false;
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[w][buf]);
        ++ns;
      }
      seq0 += 2 * (TWO ? nt : (nt + 1 - w) >> 1);
      // ---- the segment's end
      const bool both = TWO || nt > 1;                       // stream 1 has tiles too
      if (!TWO || w == 0) ok = ok && tt_wait_warp(&sh->o_full[0], no0 & 1, abort);
      if (both && (!TWO || w == 1)) ok = ok && tt_wait_warp(&sh->o_full[1], no1 & 1, abort);
      ++no0;
      no1 += both;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      float f0 = first ? 0.f : 1.f, f1 = 0.f;                // weights of O and of the other stream's O
      if (!TWO) {
        sh->ml[w][wr] = make_float2(m, l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float2 o = sh->ml[w ^ 1][wr];
        const float M = fmaxf(m, o.x);
        f0 = m == -INFINITY ? 0.f : tt_ex2(m - M);
        f1 = o.x == -INFINITY ? 0.f : tt_ex2(o.x - M);
        l = l * f0 + o.y * f1;
        m = M;
      }
      TreeEnd e;
      e.o0 = ocol;
      e.o1 = lanes + O_COL + 128 * (w ^ 1);
      e.have0 = !first;
      e.have1 = !TWO && nt > (w ? 0 : 1);
      e.f0 = f0; e.f1 = f1; e.m = m; e.l = l;
      e.c0 = TWO ? 0 : w * (DH / 2);                         // split streams: each group writes half of the columns
      e.r = r; e.t = t;
      e.pr = (TWO ? 128 * w : 0) + wr;
      e.part = sc.whole() ? nullptr : a.part + (size_t)(blockIdx.x * 2 + sc.slot()) * a.part_rows * (DH + 2);
      if (ok && live_warp) {
        bool any_bad = false;
        if (sc.ends())
#pragma unroll
          for (int k = 0; k < MAXW; ++k) any_bad |= bad[k] != 0;
        if (any_bad) tree_bad_nodes<DH, TWO>(a, sc.b, sc.h, sc.len, sc.nodes, bad, mrow, e);
        else tree_store<DH, TWO>(a, sc.b, sc.h, sc.nodes, e);
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sh->acc_free[0]);
        if (both) mbar_arrive(&sh->acc_free[1]);
      }
    }
    if (!ok) {
      *abort = 1;
      af_set_err(a.err, AF_DEV_WAIT_TIMEOUT);
    }
  }
  // the tensor memory is freed only once the products are idle
  if (warp == MMA_WARP) {
    SpinBudget b;
    if (lane == 0)
      while (!mbar_try_wait(&sh->done, 0) && !b.spent()) {
      }
    __syncwarp();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// joins the parts of the pairs that were cut: grid (row blocks, KV, B), a thread per 4 output elements. The
// parts are found by a thread each, their m and l brought to shared memory together, so that a part costs
// one load of O.
template <int DH>
__global__ void __launch_bounds__(256) tree_combine_kernel(AttnTreeArgs a, int blocks) {
  constexpr int C4 = DH / 4, ROWS = 256 / C4, MAXP = 160;
  __shared__ int part_s[MAXP];
  __shared__ float2 ml_s[MAXP][ROWS];
  const int tid = threadIdx.x, G = a.H / a.KV, R = a.T * G;
  const int row0 = blockIdx.x * ROWS, h = blockIdx.y, b = blockIdx.z;
  const int rg = row0 / 256;                   // ROWS divides 256: one group a block
  TreeSched sc;
  long long first, total;
  sc.find(a, b, tid & 31, first, total);
  blocks = (int)min((long long)blocks, total);
  const long long u0 = first + (long long)(h * a.row_groups + rg) * (sc.nt + TREE_PAIR) + TREE_PAIR, u1 = u0 + sc.nt;
  const int c0 = tree_block_of(u0, total, blocks), c1 = tree_block_of(u1 - 1, total, blocks);
  if (c0 == c1) {                              // the pair is whole
    pdl_wait();                                // a grid that ended sooner would let its dependents read early
    return;
  }
  const int lr = tid % ROWS, c4 = tid / ROWS, r = row0 + lr, pr = r - rg * 256;
  const int n = c1 - c0 + 1;
  for (int k = tid; k < n; k += 256) part_s[k] = (c0 + k) * 2 + (tree_unit(c0 + k, total, blocks) > u0 ? 0 : 1);
  pdl_wait();
  __syncthreads();
  const size_t psize = (size_t)a.part_rows * (DH + 2);
  for (int k = tid; k < n * ROWS; k += 256) {
    const int q = k % ROWS;
    ml_s[k / ROWS][q] = row0 + q < R
        ? __ldcg(reinterpret_cast<const float2*>(a.part + part_s[k / ROWS] * psize + (size_t)a.part_rows * DH) + row0 - rg * 256 + q)
        : make_float2(-INFINITY, 0.f);
  }
  __syncthreads();
  if (r >= R) return;
  float M = -INFINITY;
  for (int k = 0; k < n; ++k) M = fmaxf(M, ml_s[k][lr].x);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < n; ++k) {
    const float2 ml = ml_s[k][lr];
    const float4 x = __ldcg(reinterpret_cast<const float4*>(a.part + part_s[k] * psize) + (size_t)c4 * a.part_rows + pr);
    const bool any = ml.x != -INFINITY || ml.y != 0.f;       // a part in which the row saw nothing
    const float f = any ? tt_ex2(ml.x - M) : 0.f;
    l = fmaf(ml.y, f, l);
    o.x = any ? fmaf(x.x, f, o.x) : o.x;
    o.y = any ? fmaf(x.y, f, o.y) : o.y;
    o.z = any ? fmaf(x.z, f, o.z) : o.z;
    o.w = any ? fmaf(x.w, f, o.w) : o.w;
  }
  const int t = r / G, g = r - t * G;
  float il = l == 0.f ? 0.f : 1.f / l;         // NaN stays
  if (t >= sc.nodes) { il = 0.f; o = make_float4(0.f, 0.f, 0.f, 0.f); }
  __half2 x[2] = {__floats2half2_rn(o.x * il, o.y * il), __floats2half2_rn(o.z * il, o.w * il)};
  __half* dst = a.out + ((size_t)b * a.T + t) * a.ld_out + (size_t)(h * G + g) * DH + 4 * c4;
  if (a.out16) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(x);
  else {
    const __half* e = reinterpret_cast<const __half*>(x);
    for (int k = 0; k < 4; ++k) dst[k] = e[k];
  }
}

// K / V [P][KV][page][dh] as [P][KV][dh / 64][page][64]: boxes of box_rows rows of one head's page and 64
// columns; a box of a whole tile takes both halves of a head of 128, which land as two slices
static bool cache_map(CUtensorMap* map, const AttnTreeArgs& a, const __half* base) {
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[5] = {64, (cuuint64_t)a.page, (cuuint64_t)a.dh / 64, (cuuint64_t)a.KV, (cuuint64_t)a.P};
  const cuuint64_t strides[4] = {(cuuint64_t)a.dh * 2, 128, (cuuint64_t)a.page * a.dh * 2, (cuuint64_t)a.page_stride * 2};
  const cuuint32_t box[5] = {64, (cuuint32_t)a.box_rows, a.box_rows == TREE_BK ? (cuuint32_t)a.dh / 64 : 1u, 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<__half*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static bool q_map(CUtensorMap* map, const AttnTreeArgs& a, int rows) {
  const EncodeTiledFn enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.dh, (cuuint64_t)rows, (cuuint64_t)a.B * a.KV};
  const cuuint64_t strides[2] = {(cuuint64_t)a.dh * 2, (cuuint64_t)rows * a.dh * 2};
  const cuuint32_t box[3] = {64, 128, 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, a.q, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// one block an SM (the parts of a pair are listed in shared memory when they are joined: at most 160)
int attn_tree_tc_blocks() { const int n = device_attr(cudaDevAttrMultiProcessorCount, 148); return n < 160 ? n : 160; }

// rows of a page that one box can cover: a box never crosses a page (unless the sequence is one page,
// where it ends at the map's bound), and starts at a multiple of 8 rows, the swizzle's period
static int box_rows(const AttnTreeArgs& a) {
  return a.W == 1 || (a.page & -a.page) > TREE_BK ? TREE_BK : a.page & -a.page;
}

bool attn_tree_tc_ok(const AttnTreeArgs& a) {
  return (a.dh == 64 || a.dh == 128) && a.scale > 0.f && a.scale < 1e30f && box_rows(a) >= 8;
}

template <int DH, bool TWO>
static cudaError_t tc_launch(const AttnTreeArgs& a, cudaStream_t st) {
  const int R = a.T * (a.H / a.KV);
  CUtensorMap qm, km, vm;
  if (!q_map(&qm, a, R) || !cache_map(&km, a, a.kc) || !cache_map(&vm, a, a.vc)) return cudaErrorInvalidValue;
  constexpr int SMEM = tt::Cfg<DH, TWO>::SH + (int)sizeof(TreeShared);
  static_assert(SMEM <= 227 * 1024, "shared memory");
  static PerDeviceOnce attrs;
  const cudaError_t ae = attrs.run([] {
    return cudaFuncSetAttribute(attn_tree_tc_kernel<DH, TWO>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  });
  if (ae != cudaSuccess) return ae;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  const int blocks = attn_tree_tc_blocks();
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(tt::THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attn_tree_tc_kernel<DH, TWO>, a, qm, km, vm);
  if (e != cudaSuccess) return e;
  constexpr int ROWS = 1024 / DH;
  cfg.gridDim = dim3((R + ROWS - 1) / ROWS, a.KV, a.B);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, tree_combine_kernel<DH>, a, blocks);
}

cudaError_t attn_tree_tc_launch(AttnTreeArgs a, cudaStream_t st) {
  const int R = a.T * (a.H / a.KV);
  a.box_rows = box_rows(a);
  a.page_shift = a.page & (a.page - 1) ? -1 : 31 - __builtin_clz((unsigned)a.page);
  a.box_shift = 31 - __builtin_clz((unsigned)a.box_rows);
  a.row_groups = (R + 255) / 256;
  a.out16 = a.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0;
  if (R <= 128) return a.dh == 128 ? tc_launch<128, false>(a, st) : tc_launch<64, false>(a, st);
  return a.dh == 128 ? tc_launch<128, true>(a, st) : tc_launch<64, true>(a, st);
}

}  // namespace af
