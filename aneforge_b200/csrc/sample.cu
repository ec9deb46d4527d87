// One token per row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number.
//
// With l the row in fp32 (NaN as -inf, -0 as +0), z = l / temperature and e = exp(z - max z), a token's
// weight is the integer w = floor(e * 2^40): sums of weights are exact (those of less than 2^24 tokens fit 64 bits),
// so the token does not depend on how a row is split or summed. Kept are
//   top-k   l >= the k-th largest l (ties stay);
//   top-p   of those, in the order of falling l (ties: lowest index first), the tokens with less than
//           ceil(top_p * total) of the weight before them;
//   min-p   of those, e >= min_p.
// The token is the first in index order whose running sum of kept weights passes floor(u * kept sum).
// temperature <= 0 takes the first largest l. A row without a finite or +inf logit gives -1.
#include <cuda_bf16.h>

#include "af_common.cuh"
#include "af_kernels.h"

namespace af {

typedef unsigned long long u64;

AF_DEV float as_logit(float l) { return fmaxf(l, -INFINITY) + 0.f; }       // the number, of a NaN and a number

template <class T> AF_DEV float load_logit(const void* row, int i);
template <> AF_DEV float load_logit<float>(const void* row, int i) { return as_logit(static_cast<const float*>(row)[i]); }
template <> AF_DEV float load_logit<__half>(const void* row, int i) { return as_logit(h2f(static_cast<const __half*>(row)[i])); }
template <> AF_DEV float load_logit<__nv_bfloat16>(const void* row, int i) {
  return as_logit(__bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]));
}

// order-preserving key of a float (no NaN, no -0)
AF_DEV uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// a row's temperature. An infinite one would make NaN of the logits that are -inf (masked, or past the row's end): it
// counts as the largest finite one, by which every logit under 1e30 in size still weighs as much as the largest. One
// under 2^-124 counts as that, so that 8 / temperature is finite.
AF_DEV float row_temperature(const SampleArgs& a, int r) {
  const float t = a.temperature ? __ldg(a.temperature + r) : a.temperature_s;
  return t > 0.f ? fminf(fmaxf(t, 0x1p-124f), 0x1.fffffep127f) : t;
}

struct RowScale {
  float lmax, zmax, temp;
  AF_DEV void set(float largest, float t) {
    lmax = largest;
    temp = t > 0.f ? t : 1.f;
    zmax = __fdiv_rn(lmax, temp);
    // Where a finite largest logit's quotient overflows, so do those of lower ones. The nearest one is 2^-25 of it below:
    // any power of two under 2^-32 of it, by which quotients are exact, leaves the largest all the weight as well
    if (isinf(zmax) && !isinf(lmax)) {
      temp = __uint_as_float((__float_as_uint(lmax) & 0x7f800000u) - (100u << 23));      // |lmax| >= 16
      zmax = __fdiv_rn(lmax, temp);
    }
  }
  AF_DEV float below(float l) const {           // z - max z, 0 for the largest (also where both are infinite)
    const float z = __fdiv_rn(l, temp);
    return l == lmax || z == zmax ? 0.f : z - zmax;
  }
  AF_DEV float e(float l) const { return expf(below(l)); }
  AF_DEV u64 w(float l) const { return (u64)(e(l) * 1099511627776.f); }
};

// ---- rows held in registers: a cluster of blocks per row
//
// Each thread keeps NV vectors of 16 bytes of the row as fp32 for the whole call, so the row is read
// once. Steps (a cluster barrier after each): the maximum; a histogram of how far the logits lie below
// it, in eighths of a nat (top-k), or the bound that min-p sets; the tokens that can still be kept are
// listed. At most LIST of them: the first block sorts them, and everything else happens there. More:
// the k-th key and the nucleus' last key come from a radix search (8 bits a step, whole-number sums),
// then the token from the blocks' kept sums, over the lists or, where a list overflows, the registers.
// A nucleus without top-k can hold a quarter of the vocabulary: the weights are summed by the upper bits
// of e (exactly: a bin's tokens share an octave, so a count and the sum of the lower bits give their
// weight), only the bin that the limit falls into is sorted, and the kept sums come from the registers.
// Bound by latency: a row of 0.5 MB takes 0.1 us to read, the cluster's barriers, scans and the sort take the rest.
// B200, replayed from a graph, one row of 128256 fp32: greedy 4.6 us, plain 7.4, min-p 9.4, top-k 50 with top-p 12.1,
// top-k 1000 26, nucleus 18.1; 16 rows of 152064 with mixed settings 35.5 (two blocks share an SM; top-k 1000 and the
// nuclei are the slowest). Up to 16 blocks a row, each down to a vector a thread: a single block (below) takes 33 us for the row of top-k, 101 us for the nucleus.
namespace smr {
constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int BINS = 256;                      // 32 nats: what lies further below weighs nothing
constexpr int LIST = 2048, PER = LIST / THREADS;             // tokens that one block puts in order: LIST / C from each
constexpr int PAIRS = 256;                     // up to so many by comparing all pairs
constexpr int LOCAL = 3200;                    // listed tokens of one block
constexpr int MAXC = 16;
// nucleus: weights by the upper bits of e (128 bins an octave, bin 0 is e = 1), down to 2^-24
constexpr int EBITS = 16, EBINS = 24 * 128 + 1;
static_assert(EBINS <= LOCAL, "the bins' weights are summed in the local list's place");
}  // namespace smr

struct SampleShared {
  uint32_t kmax[smr::MAXC];                    // written by every block of the cluster: its maximum,
  uint32_t first[smr::MAXC];                   // first index of the maximum,
  uint32_t count[smr::MAXC];                   // listed tokens,
  u64 total[smr::MAXC];                        // weight
  u64 kept[smr::MAXC];                         // and kept weight
  alignas(16) uint32_t hist[smr::BINS];
  uint32_t ecnt[smr::EBINS], elow[smr::EBINS]; // tokens, and the sum of their weights' lower bits
  u64 radix[2][256];
  u64 sums[smr::WARPS * 12];                   // kept weight (or ties) of a (vector, warp)
  u64 scan[smr::WARPS];
  u64 list[smr::LIST];                         // key << 32 | ~index, LIST / C from each block of the cluster
  u64 local[smr::LOCAL];                       // the same, of this block
  u64 mine[smr::LIST];                         // this block's tokens in the nucleus' last bin
  uint32_t nlocal, kloc, floc, in_bin;
  u64 pick;
  u64 total_w;
  u64 need;                                    // weight that the nucleus takes from its last bin
  int where, bin;
  alignas(16) float edge[3][8];                // one block per row: the first and last vector if not whole; none
};

// 16 bytes where `yes`; no branch, on which the loads after it would wait
AF_DEV uint4 ldg_if(bool yes, const void* p) {
  uint4 r;
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
               "@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p), "r"((uint32_t)yes));
  return r;
}
AF_DEV float ex2(float x) {                    // for estimates
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
AF_DEV float logit_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <class P> AF_DEV P* peer(P* p, int rank) {
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"((uint64_t)p), "r"(rank));
  return reinterpret_cast<P*>(r);
}
AF_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
AF_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// weight in two whole-number parts, w = hi * 2^20 + lo: adding 8 (2^-17) rounds down to a multiple of 2^-20 (2^-40)
AF_DEV void weight_parts(float e, uint32_t& hi, uint32_t& lo) {
  const float t = __fadd_rd(e, 8.f);
  const float t2 = __fadd_rd(e - (t - 8.f), 7.62939453125e-06f);
  hi = __float_as_uint(t) - 0x41000000u;
  lo = __float_as_uint(t2) - 0x37000000u;
}

// Descending bitonic sort of N values (a power of two, 128 to LIST) in shared memory by the whole block: a
// thread holds PER neighbours, a step inside them or inside a warp needs no barrier.
AF_DEV void sort_desc(u64* x, int N) {
  using namespace smr;
  static_assert(PER == 4, "the steps inside a thread are written out");
  const int p0 = PER * threadIdx.x;
  const bool on = p0 < N;                      // whole warps
  u64 v[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) v[q] = on ? x[p0 + q] : 0;
  auto pair = [](u64& a, u64& b, bool desc) {
    const u64 lo = a < b ? a : b, hi = a < b ? b : a;
    a = desc ? hi : lo;
    b = desc ? lo : hi;
  };
#pragma unroll 1
  for (int k = 2; k <= N; k <<= 1) {
    const bool desc = !(p0 & k);
#pragma unroll 1
    for (int j = k >> 1; j >= PER; j >>= 1) {
      const bool top = desc == !(p0 & j);      // this thread's places get the larger ones
      u64 o[PER];
      if (j >= 32 * PER) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; ++q)
          if (on) x[p0 + q] = v[q];
        __syncthreads();
#pragma unroll
        for (int q = 0; q < PER; ++q) o[q] = on ? x[(p0 ^ j) + q] : 0;
      } else {
#pragma unroll
        for (int q = 0; q < PER; ++q) o[q] = __shfl_xor_sync(0xffffffffu, v[q], j / PER);
      }
#pragma unroll
      for (int q = 0; q < PER; ++q) v[q] = (v[q] < o[q]) == top ? o[q] : v[q];
    }
    if (k == 2) {
      pair(v[0], v[1], true);
      pair(v[2], v[3], false);
      continue;
    }
    pair(v[0], v[2], desc);
    pair(v[1], v[3], desc);
    pair(v[0], v[1], desc);
    pair(v[2], v[3], desc);
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (on) x[p0 + q] = v[q];
  __syncthreads();
}

// exclusive sum over the block's threads; `total` gets all of it
AF_DEV u64 scan_excl(u64 v, u64* buf, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) buf[warp] = x;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < smr::WARPS; ++k) {
    const u64 s = buf[k];
    if (k < warp) before += s;
    total += s;
  }
  return before + x - v;
}

// target of the draw among `total`: floor(u * total), inside [0, total)
AF_DEV u64 draw_target(float u, u64 total) {
  const u64 t = (u64)fmax(floor((double)u * (double)total), 0.0);
  return t < total ? t : total - 1;
}
AF_DEV float logp_of(const RowScale& sc, float l, u64 total) { return sc.below(l) - logf((float)total / 1099511627776.f); }

// the blocks' shares of the list one after the other, into `local`
AF_DEV void gather(SampleShared& sh, int C, int share) {
  for (int i = threadIdx.x; i < C * share; i += smr::THREADS) {
    const int k = i / share, j = i - k * share;
    int off = 0;
    for (int q = 0; q < k; ++q) off += (int)sh.count[q];
    if (j < (int)sh.count[k]) sh.local[off + j] = sh.list[i];
  }
  __syncthreads();
}

// The last token in order (falling key, rising index) with less than `need` of the weight before it, of
// the n <= LIST in `local`; by comparing all pairs, or by sorting where those are many.
__device__ __noinline__ u64 last_of(RowScale sc, int n, u64 need) {
  using namespace smr;
  extern __shared__ __align__(16) unsigned char sample_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
  const int tid = threadIdx.x;
  if (n <= PAIRS) {
    int pad = 16;
    while (pad < n) pad <<= 1;
    const int L = THREADS / pad, i = tid / L, part = tid % L;
    for (int k = tid; k < n; k += THREADS) sh.list[k] = sc.w(logit_of((uint32_t)(sh.local[k] >> 32)));
    __syncthreads();
    const u64 x = i < n ? sh.local[i] : ~0ull;
    u64 before = 0;
    for (int j = part; j < n; j += L)
      if (sh.local[j] > x) before += sh.list[j];
    for (int o = L >> 1; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (part == 0 && i < n && before < need && need <= before + sh.list[i]) sh.pick = x;
    __syncthreads();
    return sh.pick;
  }
  int N = 32 * PER;
  while (N < n) N <<= 1;
  for (int k = tid; k < N; k += THREADS) sh.list[k] = k < n ? sh.local[k] : 0;
  __syncthreads();
  sort_desc(sh.list, N);
  u64 w[PER], all, mine = 0;
  const int p0 = PER * tid;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    w[k] = p0 + k < n ? sc.w(logit_of((uint32_t)(sh.list[p0 + k] >> 32))) : 0;
    mine += w[k];
  }
  u64 b = scan_excl(mine, sh.scan, all);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (p0 + k < n && b < need && need <= b + w[k]) sh.pick = sh.list[p0 + k];
    b += w[k];
  }
  __syncthreads();
  return sh.pick;
}

// The whole choice among the n <= LIST tokens in `local`, which hold every token that may be kept (k 0: no
// top-k; without it `limit` is the nucleus' weight).
__device__ __noinline__ void few_tokens(int* tok, float* logp, RowScale sc, int V, int n, int k, bool use_p, float top_p, float min_p,
                                        float u, u64 limit) {
  using namespace smr;
  extern __shared__ __align__(16) unsigned char sample_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
  const int tid = threadIdx.x;
  u64 sum;
  if (n <= PAIRS) {
    int pad = 16;
    while (pad < n) pad <<= 1;
    const int L = THREADS / pad, i = tid / L, part = tid % L;
    for (int q = tid; q < n; q += THREADS) sh.list[q] = sc.w(logit_of((uint32_t)(sh.local[q] >> 32)));
    __syncthreads();
    const u64 x = i < n ? sh.local[i] : ~0ull;
    const uint32_t key = (uint32_t)(x >> 32);
    u64 before = 0;
    int over = 0;                              // larger logits
    for (int j = part; j < n; j += L) {
      const u64 y = sh.local[j];
      if (y > x) before += sh.list[j];
      over += (uint32_t)(y >> 32) > key;
    }
    for (int o = L >> 1; o > 0; o >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      over += __shfl_xor_sync(0xffffffffu, over, o);
    }
    const bool mine = part == 0 && i < n;
    const bool in_k = mine && (k == 0 || over < k);
    const u64 w = in_k ? sh.list[i] : 0;
    if (k && use_p) {
      scan_excl(w, sh.scan, sum);
      limit = (u64)ceil((double)top_p * (double)sum);
    }
    const u64 kept = in_k && (!use_p || before < limit) && sc.e(logit_of(key)) >= min_p ? w : 0;
    scan_excl(kept, sh.scan, sum);             // also the barrier before the weights are replaced
    if (mine) sh.list[i] = kept;
    __syncthreads();
    const u64 target = draw_target(u, sum);
    before = 0;
    for (int j = part; j < n; j += L)
      if ((uint32_t)sh.local[j] > (uint32_t)x) before += sh.list[j];       // a lower index: the complement is larger
    for (int o = L >> 1; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (mine && before <= target && target < before + kept) {
      *tok = (int)~(uint32_t)x;
      if (logp) *logp = logp_of(sc, logit_of(key), sum);
    }
    return;
  }
  int N = 32 * PER;
  while (N < n) N <<= 1;
  for (int q = tid; q < N; q += THREADS) sh.list[q] = q < n ? sh.local[q] : 0;
  __syncthreads();
  sort_desc(sh.list, N);
  const uint32_t kth = k && k <= n ? (uint32_t)(sh.list[k - 1] >> 32) : 0u;
  const int p0 = PER * tid;
  u64 w[PER], mine = 0;
  float e[PER];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const uint32_t key = p0 + q < n ? (uint32_t)(sh.list[p0 + q] >> 32) : 0u;
    const bool ok = p0 + q < n && key >= kth;
    e[q] = ok ? sc.e(logit_of(key)) : -1.f;
    w[q] = ok ? (u64)(e[q] * 1099511627776.f) : 0;
    mine += w[q];
  }
  u64 before = scan_excl(mine, sh.scan, sum);
  if (use_p && k) limit = (u64)ceil((double)top_p * (double)sum);
  u64 kept = 0;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const bool ok = e[q] >= 0.f && (!use_p || before < limit) && e[q] >= min_p;
    before += w[q];
    if (!ok) w[q] = 0;
    kept += w[q];
  }
  scan_excl(kept, sh.scan, sum);
  // index order: the kept weights of 512 equal runs of the vocabulary, then the tokens of the target's run
  u64* cells = sh.radix[0];
  static_assert(THREADS == 512 && sizeof(sh.radix) == 512 * sizeof(u64), "a run for each thread");
  int shift = 0;
  while ((V - 1) >> shift >= THREADS) ++shift;
  cells[tid] = 0;
  if (tid == 0) sh.nlocal = 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (w[q]) atomicAdd(&cells[(int)~(uint32_t)sh.list[p0 + q] >> shift], w[q]);
  __syncthreads();
  const u64 target = draw_target(u, sum);
  mine = cells[tid];
  u64 all;
  before = scan_excl(mine, sh.scan, all);
  if (before <= target && target < before + mine) {
    sh.where = tid;
    sh.pick = target - before;
  }
  __syncthreads();
  const int cell = sh.where;
  const u64 in = sh.pick;
#pragma unroll
  for (int q = 0; q < PER; ++q)
    if (w[q] && (int)~(uint32_t)sh.list[p0 + q] >> shift == cell) {
      const uint32_t at = atomicAdd(&sh.nlocal, 1u);
      sh.mine[at] = sh.list[p0 + q];
      sh.local[at] = w[q];
    }
  __syncthreads();
  const int c = (int)sh.nlocal;
  for (int i = tid; i < c; i += THREADS) {
    const u64 x = sh.mine[i];
    before = 0;
    for (int j = 0; j < c; ++j)
      if ((uint32_t)sh.mine[j] > (uint32_t)x) before += sh.local[j];       // a lower index: the complement is larger
    if (before <= in && in < before + sh.local[i]) {
      *tok = (int)~(uint32_t)x;
      if (logp) *logp = logp_of(sc, logit_of((uint32_t)(x >> 32)), sum);
    }
  }
}

template <class T, int NV>
__global__ void __launch_bounds__(smr::THREADS, NV * 16 / (int)sizeof(T) <= 32 ? 2 : 1) sample_kernel(SampleArgs a, int C) {
  using namespace smr;
  constexpr int VE = 16 / (int)sizeof(T), E = NV * VE;
  extern __shared__ __align__(16) unsigned char sample_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x / C, rank = blockIdx.x % C, V = a.V;
  const float temp = row_temperature(a, r);
  const int top_k = a.top_k ? __ldg(a.top_k + r) : a.top_k_s;
  const float top_p = a.top_p ? __ldg(a.top_p + r) : a.top_p_s;
  const float min_p = fminf(a.min_p ? __ldg(a.min_p + r) : a.min_p_s, 1.f);
  const float u = __ldg(a.u + r);
  if (tid < BINS) sh.hist[tid] = 0;
  if (tid == 0) { sh.nlocal = 0; sh.kloc = 0; sh.floc = 0xffffffffu; sh.in_bin = 0; sh.bin = -1; }
  __syncthreads();
  cluster_arrive();                            // the others may write here from their first wait on
  // ---- the row: vectors from the 16-byte boundary at or before its start, this block's share of them
  const T* row = static_cast<const T*>(a.logits) + (size_t)r * a.ld;
  const int skip = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int nvec = (skip + V + VE - 1) / VE, per = (nvec + C - 1) / C;
  float v[E];
  uint32_t kmax = 0;
  auto load_row = [&] {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int vi = i * THREADS + tid, i0 = (rank * per + vi) * VE - skip;
      if (vi < per && i0 >= 0 && i0 + VE <= V) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + i0));
        const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
        for (int k = 0; k < VE; ++k) v[i * VE + k] = load_logit<T>(e, k);
      } else {
#pragma unroll
        for (int k = 0; k < VE; ++k)
          v[i * VE + k] = vi < per && i0 + k >= 0 && i0 + k < V ? load_logit<T>(row, i0 + k) : -INFINITY;
      }
    }
  };
  load_row();
  auto index_of = [&](int j) { return (rank * per + (j / VE) * THREADS + tid) * VE - skip + j % VE; };
  auto in_row = [&](int j) {
    const int idx = index_of(j);
    return idx >= 0 && idx < V && (j / VE) * THREADS + tid < per;
  };
  const bool use_k = top_k > 0 && top_k < V, use_p = top_p > 0.f && top_p < 1.f, use_m = min_p > 0.f;
  if (use_p && !use_k)                         // while the row is on its way
    for (int k = tid; k < EBINS; k += THREADS) sh.ecnt[k] = sh.elow[k] = 0;
  {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) m = fmaxf(m, v[j]);
    kmax = __reduce_max_sync(0xffffffffu, key_of(m));
  }
  if (lane == 0) atomicMax(&sh.kloc, kmax);
  __syncthreads();
  cluster_wait();
  if (tid < C) *peer(&sh.kmax[rank], tid) = sh.kloc;
  cluster_arrive();
  cluster_wait();
  kmax = sh.kmax[0];
  for (int k = 1; k < C; ++k) kmax = max(kmax, sh.kmax[k]);
  RowScale sc;
  sc.set(logit_of(kmax), temp);
  if (sc.lmax == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.tok[r] = -1;
      if (a.logp) a.logp[r] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {
    uint32_t f = 0xffffffffu;
#pragma unroll
    for (int j = E - 1; j >= 0; --j)
      if (v[j] == sc.lmax) f = (uint32_t)index_of(j);
    f = __reduce_min_sync(0xffffffffu, f);
    if (lane == 0) atomicMin(&sh.floc, f);
    __syncthreads();
    if (tid == 0) *peer(&sh.first[rank], 0) = sh.floc;
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && tid == 0) {
      uint32_t b = sh.first[0];
      for (int k = 1; k < C; ++k) b = min(b, sh.first[k]);
      a.tok[r] = (int)b;
      if (a.logp) a.logp[r] = 0.f;
    }
    return;
  }
  // ---- how far below the maximum the logits lie; total weight
  const bool far = !(sc.zmax < 1e30f && sc.zmax > -1e30f && sc.lmax < 1e30f && sc.lmax > -1e30f);   // no distances then
  const float scale = 8.f / sc.temp;
  float cut = -INFINITY;                       // no token under `cut` can be kept
  u64 total_w = 0, limit = 0;
  // e in the logits' place (past the row's end: 0)
  auto to_e = [&] {
    if (sc.temp == 1.f) {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = expf(v[j] - sc.zmax);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) v[j] = expf(__fdiv_rn(v[j], sc.temp) - sc.zmax);
    }
  };
  // the nucleus of a whole row: e takes the logits' place (a block's 2^15 values keep a bin's sum in 32 bits)
  const bool binned = use_p && !use_k && !far;
  if (use_p && !use_k) {
    uint32_t hi = 0, lo = 0;
    auto add = [&](float e) {
      uint32_t h, l;
      weight_parts(e, h, l);
      hi += h;
      lo += l;
    };
    if (binned) {
      to_e();
#pragma unroll
      for (int j = 0; j < E; ++j) add(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) add(in_row(j) ? sc.e(v[j]) : 0.f);       // -inf may be the largest z
    }
    hi = __reduce_add_sync(0xffffffffu, hi);
    lo = __reduce_add_sync(0xffffffffu, lo);
    if (lane == 0) sh.scan[warp] = ((u64)hi << 20) + lo;
    __syncthreads();
    if (tid == 0) {
      u64 s = 0;
      for (int k = 0; k < WARPS; ++k) s += sh.scan[k];
      sh.total_w = s;
    }
    __syncthreads();
    if (tid < C) *peer(&sh.total[rank], tid) = sh.total_w;
    cluster_arrive();
    cluster_wait();
    for (int k = 0; k < C; ++k) total_w += sh.total[k];
    limit = (u64)ceil((double)top_p * (double)total_w);
    if (binned) {
      // tokens so light that all V of them together would not reach past the nucleus need no bin
      const float light = fmaxf((float)((double)(total_w - limit) / (double)V * (0.999 / 1099511627776.0)), 6.0e-8f);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (v[j] >= light) {
          const uint32_t b = __float_as_uint(v[j]);
          const int bin = (int)((0x3f800000u >> EBITS) - (b >> EBITS)), drop = 110 - (int)(b >> 23);
          atomicAdd(&sh.ecnt[bin], 1u);
          atomicAdd(&sh.elow[bin], (b & ((1u << EBITS) - 1)) >> max(drop, 0));
        }
      cluster_arrive();
      cluster_wait();
    }
  }
  if (use_k && !far) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float d = (sc.lmax - v[j]) * scale;
      if (d < (float)BINS) atomicAdd(&sh.hist[(int)d], 1u);
    }
    cluster_arrive();
    cluster_wait();
    // each block sums the cluster's histograms, then finds the first bin by which k tokens are there
    u64 n = 0;
    if (tid < BINS)
      for (int k = 0; k < C; ++k) n += *peer(&sh.hist[tid], k);
    u64 all;
    const u64 before = scan_excl(n, sh.scan, all);
    if (tid == 0) sh.where = BINS;
    __syncthreads();
    if (before < (u64)top_k && (u64)top_k <= before + n) sh.where = tid;
    __syncthreads();
    cut = -(float)(min(sh.where, BINS - 1) + 1);             // a distance, see below; fewer than k weigh anything: all of those
    if (sh.where == BINS && !(fabsf(sc.zmax) < 16777216.f)) cut = -INFINITY;     // z may round by nats: any may weigh something
  } else if (use_m && !use_p && !use_k && !far) {
    cut = -(-8.f * logf(min_p) * 1.0001f + 1.f + fabsf(sc.zmax) * 0x1p-19f);     // z rounds to 2^-24 of its size
  }
  // a token may be kept if its distance is under -cut: the same product as in the histogram
  auto may = [&](float l) { return cut == -INFINITY || (sc.lmax - l) * scale < -cut; };
  // ---- list the tokens that may be kept
  bool listed = false, small = false;
  uint32_t n_local = 0, n_all = 0;
  const int share = LIST / C;                  // of sh.list, for each block
  if (cut != -INFINITY) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool yes = may(v[j]);
      const unsigned who = __ballot_sync(0xffffffffu, yes);
      if (!who) continue;
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&sh.nlocal, (uint32_t)__popc(who));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
      if (yes && at < (uint32_t)LOCAL) sh.local[at] = (u64)key_of(v[j]) << 32 | (uint32_t)~index_of(j);
    }
    __syncthreads();
    n_local = sh.nlocal;
    if (n_local <= (uint32_t)share) {
      u64* list0 = peer(sh.list + rank * share, 0);
      for (uint32_t i = tid; i < n_local; i += THREADS) list0[i] = sh.local[i];
    }
    if (tid < C) *peer(&sh.count[rank], tid) = n_local;
    cluster_arrive();
    cluster_wait();
    bool fits = true;
    small = true;                              // the same answers in every block
    for (int k = 0; k < C; ++k) {
      n_all += sh.count[k];
      fits &= sh.count[k] <= (uint32_t)LOCAL;
      small &= sh.count[k] <= (uint32_t)share;
    }
    listed = fits;
    if (small) {
      if (rank) return;                        // nobody reads the other blocks' memory any more
      gather(sh, C, share);
      few_tokens(a.tok + r, a.logp ? a.logp + r : nullptr, sc, V, (int)n_all, use_k ? top_k : 0, use_p, top_p, min_p, u,
                 use_k ? 0 : limit);
      return;
    }
  }
  // ---- the general way: f(value, index) for each token that may be kept (the value is the logit, or e once
  // the registers hold that)
  auto each = [&](auto f) {
    if (listed) {
      for (uint32_t i = tid; i < n_local; i += THREADS) {
        const u64 x = sh.local[i];
        f(logit_of((uint32_t)(x >> 32)), (int)~(uint32_t)x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (in_row(j)) f(v[j], index_of(j));
    }
  };
  // the largest key such that the weights (or counts) of the keys over it stay under `want`; `left` gets
  // what is wanted of that key itself
  int round = 0;
  auto search = [&](bool counts, uint32_t floor_key, u64 want, u64& left) -> uint32_t {
    uint32_t lo = floor_key, hi = kmax;
    left = want;
    while (true) {
      const uint32_t range = hi - lo;
      const int bits = 32 - __clz(range | 1u), shift = bits > 8 ? bits - 8 : 0;
      u64* hist = sh.radix[round & 1];
      ++round;
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      each([&](float l, int) {
        const uint32_t k = key_of(l);
        if (k >= lo && k <= hi) atomicAdd(&hist[(hi - k) >> shift], counts ? 1ull : sc.w(l));
      });
      cluster_arrive();
      cluster_wait();
      u64 s = 0;
      if (tid < 256)
        for (int k = 0; k < C; ++k) s += *peer(&hist[tid], k);
      u64 all;
      const u64 before = scan_excl(s, sh.scan, all);
      if (tid == 0) sh.where = 255;
      __syncthreads();
      if (tid < 256 && before < left && left <= before + s) {
        sh.where = tid;
        sh.pick = before;
      }
      __syncthreads();
      const int bin = sh.where;
      left -= sh.pick;
      hi -= (uint32_t)bin << shift;
      if (shift == 0) return hi;
      const uint32_t width = (1u << shift) - 1;
      lo = hi - lo > width ? hi - width : lo;
    }
  };
  // the weights of f's results (0: not kept) summed in index order, and the first token whose running sum
  // passes `target`; -1 in the blocks that do not have it
  auto find = [&](auto f, u64* totals, auto target_of, u64& total) -> int {
    // sums of each (vector, warp): index order is (block, vector, warp, lane, element)
    if (listed) {
      for (int k = tid; k < NV * WARPS; k += THREADS) sh.sums[k] = 0;
      __syncthreads();
      each([&](float x, int idx) {
        const u64 w = (u64)(f(x, idx) * 1099511627776.f);
        const int vi = (idx + skip) / VE - rank * per;
        if (w) atomicAdd(&sh.sums[(vi / THREADS) * WARPS + (vi % THREADS) / 32], w);
      });
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint32_t hi = 0, lo = 0;               // 32 * VE values of at most 2^20 each
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const int idx = index_of(i * VE + k);
          uint32_t h, l;
          const float e = f(v[i * VE + k], idx);          // past the row's end: of -inf
          weight_parts(far && !in_row(i * VE + k) ? 0.f : e, h, l);
          hi += h;
          lo += l;
        }
        hi = __reduce_add_sync(0xffffffffu, hi);
        lo = __reduce_add_sync(0xffffffffu, lo);
        if (lane == 0) sh.sums[i * WARPS + warp] = ((u64)hi << 20) + lo;
      }
    }
    __syncthreads();
    u64 mine = tid < NV * WARPS ? sh.sums[tid] : 0;
    u64 all;
    const u64 before = scan_excl(mine, sh.scan, all);
    if (tid < C) *peer(&totals[rank], tid) = all;
    cluster_arrive();
    cluster_wait();
    total = 0;
    u64 base = 0;
    for (int k = 0; k < C; ++k) {
      if (k < rank) base += totals[k];
      total += totals[k];
    }
    const u64 target = target_of(total);
    if (target < base || target >= base + all) return -1;       // another block's (the same answer in all threads)
    if (tid < NV * WARPS && base + before <= target && target < base + before + mine) {
      sh.where = tid;
      sh.pick = target - base - before;
    }
    __syncthreads();
    // inside one (vector, warp): VE * 32 consecutive tokens
    const int cell = sh.where;
    const u64 in = sh.pick;
    const int first = (rank * per + (cell / WARPS) * THREADS + (cell % WARPS) * 32) * VE - skip;
    for (int k = tid; k < 32 * VE; k += THREADS) sh.list[k] = 0;
    __syncthreads();
    each([&](float x, int idx) {
      if (idx >= first && idx < first + 32 * VE) sh.list[idx - first] = (u64)(f(x, idx) * 1099511627776.f);
    });
    __syncthreads();
    mine = tid < 32 * VE ? sh.list[tid] : 0;
    const u64 b2 = scan_excl(mine, sh.scan, all);
    if (tid < 32 * VE && b2 <= in && in < b2 + mine) sh.where = first + tid;
    __syncthreads();
    return sh.where;
  };
  auto finish = [&](int at, u64 sum) {
    if (at >= 0 && tid == 0) {
      a.tok[r] = at;
      if (a.logp) a.logp[r] = logp_of(sc, load_logit<T>(row, at), sum);
    }
    cluster_arrive();                          // peers may still read this block's histograms
    cluster_wait();
  };
  u64 sum;
  // the draw where e is in the registers: kept are the tokens whose e has at least the bits `least`, and of
  // the n_in in `mine` those from `last` on
  auto draw_e = [&](uint32_t least, int n_in, u64 last) {
    auto extra = [&](int i, int& vi, int& idx) -> u64 {
      const u64 x = sh.mine[i];
      const float e = sc.e(logit_of((uint32_t)(x >> 32)));
      idx = (int)~(uint32_t)x;
      vi = (idx + skip) / VE - rank * per;
      return x >= last && e >= min_p ? (u64)(e * 1099511627776.f) : 0;
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      uint32_t hi = 0, lo = 0;                 // 32 * VE values of at most 2^20 each
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        const float e = v[i * VE + k];
        uint32_t h, l;
        weight_parts(__float_as_uint(e) >= least ? e : 0.f, h, l);
        hi += h;
        lo += l;
      }
      hi = __reduce_add_sync(0xffffffffu, hi);
      lo = __reduce_add_sync(0xffffffffu, lo);
      if (lane == 0) sh.sums[i * WARPS + warp] = ((u64)hi << 20) + lo;
    }
    __syncthreads();
    for (int i = tid; i < n_in; i += THREADS) {
      int vi, idx;
      const u64 w = extra(i, vi, idx);
      if (w) atomicAdd(&sh.sums[(vi / THREADS) * WARPS + (vi % THREADS) / 32], w);
    }
    __syncthreads();
    u64 mine = tid < NV * WARPS ? sh.sums[tid] : 0, all;
    u64 before = scan_excl(mine, sh.scan, all);
    if (tid < C) *peer(&sh.total[rank], tid) = all;
    if (tid == 0) sh.where = -1;
    cluster_arrive();
    cluster_wait();
    u64 base = 0;
    sum = 0;
    for (int k = 0; k < C; ++k) {
      if (k < rank) base += sh.total[k];
      sum += sh.total[k];
    }
    // nobody reads another block's memory from here on
    const u64 target = draw_target(u, sum);
    if (target < base || target >= base + all) return;
    before += base;
    if (tid < NV * WARPS && before <= target && target < before + mine) {
      sh.where = tid;
      sh.pick = target - before;
    }
    __syncthreads();
    const int cell = sh.where;
    const u64 in = sh.pick;
    // the 32 * VE consecutive tokens of one (vector, warp)
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (i * WARPS + warp == cell) {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const float e = v[i * VE + k];
          sh.list[lane * VE + k] = __float_as_uint(e) >= least ? (u64)(e * 1099511627776.f) : 0;
        }
      }
    __syncthreads();
    for (int i = tid; i < n_in; i += THREADS) {
      int vi, idx;
      const u64 w = extra(i, vi, idx);
      if (w && (vi / THREADS) * WARPS + (vi % THREADS) / 32 == cell) sh.list[(vi % 32) * VE + (idx + skip) % VE] = w;
    }
    __syncthreads();
    mine = tid < 32 * VE ? sh.list[tid] : 0;
    before = scan_excl(mine, sh.scan, all);
    if (tid < 32 * VE && before <= in && in < before + mine) {
      const int at = (rank * per + (cell / WARPS) * THREADS + (cell % WARPS) * 32) * VE - skip + tid;
      a.tok[r] = at;
      if (a.logp) a.logp[r] = logp_of(sc, load_logit<T>(row, at), sum);
    }
  };
  if (!use_k && !use_p && !far) {
    to_e();
    draw_e(use_m ? __float_as_uint(min_p) : 0u, 0, 0);
    return;
  }
  if (binned) {
    // ---- nucleus: e is in the registers, the blocks' bins are filled. Each block adds up its share of the
    // bins over the cluster; the one whose share the limit falls into tells the others which bin it is
    const int bins = (EBINS + C - 1) / C, b0 = rank * bins, b1 = min(EBINS, b0 + bins);
    for (int b = b0 + tid; b < b1; b += THREADS) {
      u64 cnt = 0, low = 0;
#pragma unroll 4
      for (int k = 0; k < C; ++k) {
        cnt += *peer(&sh.ecnt[b], k);
        low += *peer(&sh.elow[b], k);
      }
      // e = mantissa * 2^(octave - 23), a weight counts 2^-40: 2^(17 + octave) of them a mantissa unit
      const uint32_t bits = 0x3f800000u - ((uint32_t)b << EBITS);
      const int up = 17 + (int)(bits >> 23) - 127;
      const u64 base = (bits & 0x7fffffu) | 0x800000u;
      sh.local[b - b0] = up >= 0 ? (cnt * base + low) << up : cnt * (base >> -up) + low;
    }
    __syncthreads();
    const int run = (bins + THREADS - 1) / THREADS, k0 = b0 + tid * run;
    u64 mine = 0, all;
    for (int k = k0; k < min(k0 + run, b1); ++k) mine += sh.local[k - b0];
    u64 before = scan_excl(mine, sh.scan, all);
    if (tid < C) *peer(&sh.kept[rank], tid) = all;
    cluster_arrive();
    cluster_wait();
    for (int k = 0; k < rank; ++k) before += sh.kept[k];
    if (before < limit && limit <= before + mine)
      for (int k = k0; k < min(k0 + run, b1); ++k) {
        const u64 w = sh.local[k - b0];
        if (before < limit && limit <= before + w)
          for (int c = 0; c < C; ++c) {
            *peer(&sh.bin, c) = k;
            *peer(&sh.need, c) = limit - before;
          }
        before += w;
      }
    cluster_arrive();
    cluster_wait();
    // its tokens, to every block
    const int bin = sh.bin;
    const u64 need = sh.need;
    const uint32_t q = (0x3f800000u >> EBITS) - (uint32_t)bin;
    if (bin >= 0) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (__float_as_uint(v[j]) >> EBITS == q) {
          const uint32_t at = atomicAdd(&sh.in_bin, 1u);
          if (at < (uint32_t)share) sh.mine[at] = (uint32_t)~index_of(j);
        }
      __syncthreads();
      const int n = (int)sh.in_bin;
      if (n <= share)
        for (int i = tid; i < n; i += THREADS) {
          const u64 x = (u64)key_of(load_logit<T>(row, (int)~(uint32_t)sh.mine[i])) << 32 | (uint32_t)sh.mine[i];
          sh.mine[i] = x;
          for (int c = 0; c < C; ++c) *peer(&sh.list[rank * share + i], c) = x;
        }
      if (tid < C) *peer(&sh.count[rank], tid) = (uint32_t)n;
    }
    cluster_arrive();
    cluster_wait();
    bool fit = bin >= 0;
    int n_bin = 0;
    for (int k = 0; fit && k < C; ++k) {
      fit = sh.count[k] <= (uint32_t)share;
      n_bin += (int)sh.count[k];
    }
    if (fit) {                                 // the same in every block
      gather(sh, C, share);
      const u64 last = last_of(sc, n_bin, need);
      draw_e(max((q + 1) << EBITS, __float_as_uint(fmaxf(min_p, 0.f))), (int)sh.in_bin, last);
      return;
    }
    load_row();                                // a bin too full to be sorted: by keys
  }
  uint32_t kth = 0, pth = 0;
  int pidx = V;
  u64 left;
  if (use_k && (!listed || (uint32_t)top_k <= n_all)) kth = search(true, 0u, (u64)top_k, left);
  if (use_p) {
    if (use_k) {
      // total weight of the top k
      u64 mine = 0;
      each([&](float l, int) { if (key_of(l) >= kth) mine += sc.w(l); });
      u64 all;
      scan_excl(mine, sh.scan, all);
      if (tid < C) *peer(&sh.total[rank], tid) = all;
      cluster_arrive();
      cluster_wait();
      total_w = 0;
      for (int k = 0; k < C; ++k) total_w += sh.total[k];
      limit = (u64)ceil((double)top_p * (double)total_w);
    }
    pth = search(false, kth, limit, left);
    // of the tokens with exactly this key the first ceil(left / weight) are kept
    const u64 w1 = sc.w(logit_of(pth));
    const u64 ties = w1 ? (left + w1 - 1) / w1 : 1;
    u64 count;
    // (a tie counts as the smallest weight, 2^-40)
    const int at = find([&](float l, int) -> float { return key_of(l) == pth ? 9.094947017729282e-13f : 0.f; }, sh.kept,
                        [&](u64 n) { return ties - 1 < n ? ties - 1 : n - 1; }, count);
    if (at >= 0 && tid < C) *peer(&sh.first[0], tid) = (uint32_t)at;
    cluster_arrive();
    cluster_wait();
    pidx = (int)sh.first[0];
  }
  const int at = find(
      [&](float l, int idx) -> float {
        const uint32_t k = key_of(l);
        if (k < kth || k < pth || (k == pth && idx > pidx)) return 0.f;
        const float e = sc.e(l);
        return e >= min_p ? e : 0.f;
      },
      sh.total, [&](u64 n) { return draw_target(u, n); }, sum);
  finish(at, sum);
}

// ---- many rows, and rows too long for a cluster's registers: one block per row, which reads the row again
// for each step (from L2, mostly). A step has no barrier between its loads, so the loads of a row flow without
// a pause, where a cluster waits for its peers several times a row. Steps: the maximum, with an estimate of
// the total weight; top-k: the k-th largest of the threads' maxima bounds the k-th largest logit from below, so
// that few more than k tokens are listed; nucleus: the bins of e as in a cluster; then the kept weight of each
// run ("cell") of the row, and the one cell that the target falls into. What does not fit its list or bin goes
// the general way: a radix search, a pass over the row for each 8 bits.
// B200, 256 rows of 128256 fp32 (131 MB, 20 us at the rate of a copy): greedy 25 us, min-p 65, top-k 50 with top-p
// 70, top-k 1000 133, plain 74, nucleus 159. The first pass comes from memory at 5.3 TB/s; the passes that need every token's exact
// e are bound by their instructions (16 warps a row, about 40 a token) and not by L2. A nucleus walks the whole row three
// times: maximum and an estimate of the total, with every token's approximate e; every token's exact weight, and the
// bins; and, to sum the kept weights, every logit against the limit's bin, of which only those that reach it are queued
// for an exact e, 32 to a warp (this walk takes about as long as the second). Counters: an instruction in 69 % of the
// issue slots, memory at 26 %.
namespace smw {
constexpr int CELLS = 1024;                    // runs of 32 * K vectors
}

template <class T>
__global__ void __launch_bounds__(smr::THREADS, 2) sample_wide_kernel(SampleArgs a) {
  using namespace smr;
  constexpr int VE = 16 / (int)sizeof(T), U = 4, U1 = 32 / VE;         // U, U1: vectors of a thread on their way
  extern __shared__ __align__(16) unsigned char sample_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(sample_raw);
  u64* cells = reinterpret_cast<u64*>(sh.ecnt);              // after the bins
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x, V = a.V;
  const float temp = row_temperature(a, r);
  const int top_k = a.top_k ? __ldg(a.top_k + r) : a.top_k_s;
  const float top_p = a.top_p ? __ldg(a.top_p + r) : a.top_p_s;
  const float min_p = fminf(a.min_p ? __ldg(a.min_p + r) : a.min_p_s, 1.f);
  const bool use_k = top_k > 0 && top_k < V, use_p = top_p > 0.f && top_p < 1.f;
  const float u = __ldg(a.u + r);
  if (tid == 0) { sh.nlocal = 0; sh.kloc = 0; sh.floc = 0xffffffffu; sh.in_bin = 0; sh.bin = -1; sh.first[0] = 0xffffffffu; }
  const T* row = static_cast<const T*>(a.logits) + (size_t)r * a.ld;
  const int skip = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const int nvec = (skip + V + VE - 1) / VE;
  // vector vi as logits (-inf outside the row)
  const int full0 = skip ? 1 : 0, nfull = max((skip + V) / VE - full0, 0);
  auto is_full = [&](int vi) { return (unsigned)(vi - full0) < (unsigned)nfull; };
  auto unpack = [&](bool full, const uint4& x, int vi, float (&l)[VE]) {
    if (full) {
      const T* e = reinterpret_cast<const T*>(&x);
#pragma unroll
      for (int k = 0; k < VE; ++k) l[k] = load_logit<T>(e, k);
    } else {
      const float* e = sh.edge[vi == 0 ? 0 : vi == nvec - 1 ? 1 : 2];
#pragma unroll
      for (int k = 0; k < VE; ++k) l[k] = e[k];
    }
  };
  if (tid < 3 * 8) {
    const int i = (tid < 8 ? 0 : nvec - 1) * VE - skip + tid % 8;
    sh.edge[tid / 8][tid % 8] = tid < 16 && tid % 8 < VE && i >= 0 && i < V ? load_logit<T>(row, i) : -INFINITY;
  }
  __syncthreads();
  auto fetch = [&](int vi) { return ldg_if(is_full(vi), row + vi * VE - skip); };
  // f(logits, vector) for the n vectors from v0 in steps of `step`, U loads on their way together. The loop is not
  // unrolled: with U bodies a step the warps waited for instructions (96 rows of 50257, min-p: 25.7 us, 18.3 us so)
  auto run = [&](int v0, int n, int step, auto f) {
    uint4 x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) x[j] = fetch(j < n ? v0 + j * step : nvec);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const uint4 y = x[0];
#pragma unroll
      for (int j = 0; j + 1 < U; ++j) x[j] = x[j + 1];
      const int vi = v0 + i * step;
      x[U - 1] = fetch(i + U < n ? vi + U * step : nvec);
      float l[VE];
      unpack(is_full(vi), y, vi, l);
      f(l, vi);
    }
  };
  auto walk = [&](auto f) { run(tid, (nvec - tid + THREADS - 1) / THREADS, THREADS, f); };
  // ---- the maximum, and about how much all tokens weigh
  float m = -INFINITY, s = 0.f;
  int at = 0;                                  // the first vector that holds m
  const bool estimate = use_p && !use_k && temp > 0.f;
  const float c2 = 1.4426950408889634f / temp;
  auto first_pass = [&](const float (&l)[VE], int vi) {
    float x = l[0];
#pragma unroll
    for (int k = 1; k < VE; ++k) x = fmaxf(x, l[k]);
    if (x > m) {
      if (estimate) s = m == -INFINITY ? 0.f : s * exp2f((m - x) * c2);
      m = x;
      at = vi;
    }
    if (estimate && m != -INFINITY)
#pragma unroll
      for (int k = 0; k < VE; ++k) s += ex2((l[k] - m) * c2);
  };
  for (int base = tid; base < nvec; base += U1 * THREADS) {       // the row comes from memory: more loads on their way
    uint4 x[U1];
#pragma unroll
    for (int j = 0; j < U1; ++j) x[j] = fetch(base + j * THREADS);
#pragma unroll
    for (int j = 0; j < U1; ++j) {
      const int vi = base + j * THREADS;
      float l[VE];
      unpack(is_full(vi), x[j], vi, l);
      first_pass(l, vi);
    }
  }
  const uint32_t mine_key = key_of(m);
  uint32_t kmax = __reduce_max_sync(0xffffffffu, mine_key);
  __syncthreads();
  if (lane == 0) atomicMax(&sh.kloc, kmax);
  __syncthreads();
  kmax = sh.kloc;
  RowScale sc;
  sc.set(logit_of(kmax), temp);
  if (sc.lmax == -INFINITY) {
    if (tid == 0) {
      a.tok[r] = -1;
      if (a.logp) a.logp[r] = -INFINITY;
    }
    return;
  }
  if (!(temp > 0.f)) {
    if (mine_key == kmax) atomicMin(&sh.first[0], (uint32_t)at);
    __syncthreads();
    if (tid == 0) {
      const int vi = (int)sh.first[0];
      int i = max(vi * VE - skip, 0);
      while (load_logit<T>(row, i) != sc.lmax) ++i;          // it is in this vector
      a.tok[r] = i;
      if (a.logp) a.logp[r] = 0.f;
    }
    return;
  }
  const bool far = !(sc.zmax < 1e30f && sc.zmax > -1e30f && sc.lmax < 1e30f && sc.lmax > -1e30f);   // no distances then
  auto e_of = [&](float l) {
    if (far) return sc.e(l);
    return expf((sc.temp == 1.f ? l : __fdiv_rn(l, sc.temp)) - sc.zmax);
  };
  // of a vector: the branches once, the exponentials side by side
  auto es_of = [&](const float (&l)[VE], float (&e)[VE]) {
    if (far) {
#pragma unroll
      for (int k = 0; k < VE; ++k) e[k] = sc.e(l[k]);
      return;
    }
    if (sc.temp == 1.f) {
#pragma unroll
      for (int k = 0; k < VE; ++k) e[k] = l[k];
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k) e[k] = __fdiv_rn(l[k], sc.temp);
    }
#pragma unroll
    for (int k = 0; k < VE; ++k) e[k] = expf(e[k] - sc.zmax);
  };
  auto parts_of = [&](const float (&e)[VE], uint32_t& hi, uint32_t& lo) {
    hi = 0u - VE * 0x41000000u;
    lo = 0u - VE * 0x37000000u;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const float t = __fadd_rd(e[k], 8.f);
      hi += __float_as_uint(t);
      lo += __float_as_uint(__fadd_rd(e[k] - (t - 8.f), 7.62939453125e-06f));
    }
  };
  auto w_of = [&](float e) { return (u64)(e * 1099511627776.f); };
  auto order = [&](float l, int idx) { return (u64)key_of(l) << 32 | (uint32_t)~idx; };
  // ---- sums of f(logit, index) over the cells, and the token of a cell that passes a target
  const int K = max(8, (nvec + 32 * smw::CELLS - 1) / (32 * smw::CELLS)), ncell = (nvec + 32 * K - 1) / (32 * K);
  auto warp_sum64 = [&](u64 w) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    return w;
  };
  // (f(logits, e, vector) gives e, or 0 for a token that is not kept)
  auto group = [&](auto f, int v0) -> u64 {                  // one lane's part of 32 vectors from v0
    const int vi = v0 + lane;
    uint32_t hi = 0, lo = 0;
    if (vi < nvec) {
      const bool full = is_full(vi);
      const uint4 x = fetch(vi);
      float l[VE], e[VE];
      unpack(full, x, vi, l);
      f(l, e, vi);
      parts_of(e, hi, lo);
    }
    return ((u64)hi << 20) + lo;
  };
  auto cell_rows = [&](int c) { return min(K, (nvec - c * K * 32 + 31) / 32); };      // runs of 32 vectors
  auto sum_cells = [&](auto f) {
    __syncthreads();
    for (int c = warp; c < ncell; c += WARPS) {
      u64 w = 0;
      run(c * K * 32 + lane, cell_rows(c), 32, [&](const float (&l)[VE], int vi) {
        float e[VE];
        uint32_t hi, lo;
        f(l, e, vi);
        parts_of(e, hi, lo);
        w += ((u64)hi << 20) + lo;
      });
      w = warp_sum64(w);
      if (lane == 0) cells[c] = w;
    }
    __syncthreads();
  };
  // the same where only tokens from l_lo on count: those of 32 vectors are queued, and a full warp of them is
  // looked at together. f(logit, index, e) gives e or 0
  auto sum_above = [&](float l_lo, auto f) {
    static_assert(LIST + 64 * WARPS <= LOCAL, "the warps' queues lie after the list");
    u64* queue = sh.local + LIST + 64 * warp;
    __syncthreads();
    for (int c = warp; c < ncell; c += WARPS) {
      u64 w = 0;
      int n = 0;
      auto flush = [&](bool mine) {
        __syncwarp();
        uint32_t h = 0, g = 0;
        if (mine) {
          const u64 x = queue[lane];
          const float l = logit_of((uint32_t)(x >> 32));
          weight_parts(f(l, (int)~(uint32_t)x, e_of(l)), h, g);
        }
        w += ((u64)h << 20) + g;
        __syncwarp();                          // the places may be written again
      };
      run(c * K * 32 + lane, cell_rows(c), 32, [&](const float (&l)[VE], int vi) {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const bool yes = l[k] >= l_lo;
          const unsigned who = __ballot_sync(0xffffffffu, yes);
          if (!who) continue;
          if (yes) queue[n + __popc(who & ((1u << lane) - 1))] = order(l[k], vi * VE - skip + k);
          n += __popc(who);
          if (n >= 32) {
            flush(true);
            n -= 32;
            const u64 x = queue[32 + lane];
            __syncwarp();
            queue[lane] = x;
            __syncwarp();                      // before another lane's next token takes a place among them
          }
        }
      });
      flush(lane < n);
      w = warp_sum64(w);
      if (lane == 0) cells[c] = w;
    }
    __syncthreads();
  };
  auto total_cells = [&](u64& before) {        // all cells' sum; this thread's two cells begin after `before`
    u64 all;
    const u64 w = (2 * tid < ncell ? cells[2 * tid] : 0) + (2 * tid + 1 < ncell ? cells[2 * tid + 1] : 0);
    before = scan_excl(w, sh.scan, all);
    return all;
  };
  auto locate = [&](auto f, u64 before, u64 target) -> int {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int c = 2 * tid + j;
      const u64 w = c < ncell ? cells[c] : 0;
      if (before <= target && target < before + w) {
        sh.where = c;
        sh.pick = target - before;
      }
      before += w;
    }
    __syncthreads();
    const int c = sh.where;
    for (int k = warp; k < K; k += WARPS) {
      const u64 w = warp_sum64(group(f, (c * K + k) * 32));
      if (lane == 0) sh.radix[0][k] = w;       // K <= 129 (V < 2^24) of 256 places
    }
    __syncthreads();
    if (warp == 0) {
      u64 in = sh.pick;
      int k = 0;
      while (k + 1 < K && in >= sh.radix[0][k]) in -= sh.radix[0][k++];
      const int v0 = (c * K + k) * 32;
      const u64 w = group(f, v0);
      u64 x = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      u64 b = x - w;
      if (b <= in && in < x) {
        const int vi = v0 + lane;
        float l[VE], e[VE];
        unpack(is_full(vi), fetch(vi), vi, l);
        f(l, e, vi);
        int i = 0;
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          b += w_of(e[k]);
          if (b <= in) i = k + 1;
        }
        sh.where = vi * VE - skip + i;
      }
    }
    __syncthreads();
    return sh.where;
  };
  // kept: l over l_last, or l_last itself up to index i_last, and e >= min_p
  float l_last = -INFINITY;
  int i_last = V;
  auto inside = [&](int idx) { return idx >= 0 && idx < V; };
  bool narrow = far || use_k || use_p || min_p > 0.f;        // else every token is kept
  auto kept = [&](const float (&l)[VE], float (&e)[VE], int vi) {
    es_of(l, e);
    if (!narrow) return;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      const int idx = vi * VE - skip + k;
      const bool yes = (l[k] > l_last || (l[k] == l_last && idx <= i_last)) && e[k] >= min_p && (!far || inside(idx));
      e[k] = yes ? e[k] : 0.f;
    }
  };
  auto finish = [&](u64 before, u64 sum) {
    const int i = locate(kept, before, draw_target(u, sum));
    if (tid == 0) {
      a.tok[r] = i;
      if (a.logp) a.logp[r] = logp_of(sc, load_logit<T>(row, i), sum);
    }
  };
  u64 before;
  bool listed = false;                         // every token that may be kept is in `local`
  uint32_t n_list = 0;
  if (use_k && (top_k <= THREADS * 3 / 4 || !far)) {
    float least = -INFINITY, cut = INFINITY;
    const float scale = 8.f / sc.temp;
    if (top_k <= THREADS * 3 / 4) {
      // at least k tokens are as large as the k-th largest of the threads' maxima
      uint32_t* keys = sh.hist;
      static_assert(THREADS <= BINS + EBINS, "the threads' maxima lie over the histogram and the bins");
      keys[tid] = mine_key;
      __syncthreads();
      int over = 0;
      for (int k = 0; k < THREADS; k += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(keys + k);
        over += (x.x > mine_key) + (x.y > mine_key) + (x.z > mine_key) + (x.w > mine_key);
      }
      if (over < top_k) atomicMin(&sh.floc, mine_key);
      __syncthreads();
      least = logit_of(sh.floc);
    } else {
      // the eighth of a nat that the k-th lies in
      if (tid < BINS) sh.hist[tid] = 0;
      if (tid == 0) sh.where = BINS - 1;
      __syncthreads();
      walk([&](const float (&l)[VE], int) {
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const float d = (sc.lmax - l[k]) * scale;
          if (d < (float)BINS) atomicAdd(&sh.hist[(int)d], 1u);
        }
      });
      u64 all;
      __syncthreads();
      const u64 n = tid < BINS ? sh.hist[tid] : 0;
      before = scan_excl(n, sh.scan, all);
      if (before < (u64)top_k && (u64)top_k <= before + n) sh.where = tid;
      __syncthreads();
      cut = (float)(sh.where + 1);             // fewer than k weigh anything: all of those
      if (all < (u64)top_k && !(fabsf(sc.zmax) < 16777216.f)) cut = INFINITY;    // z may round by nats: any may
    }
    walk([&](const float (&l)[VE], int vi) {
      float most = l[0];
#pragma unroll
      for (int k = 1; k < VE; ++k) most = fmaxf(most, l[k]);
      if (most < least) return;
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        const int i = vi * VE - skip + k;
        if (l[k] >= least && (cut == INFINITY || (sc.lmax - l[k]) * scale < cut) && inside(i)) {
          const uint32_t n = atomicAdd(&sh.nlocal, 1u);
          if (n < (uint32_t)LOCAL) sh.local[n] = order(l[k], i);
        }
      }
    });
    __syncthreads();
    n_list = sh.nlocal;
    if (n_list <= (uint32_t)LIST) {
      few_tokens(a.tok + r, a.logp ? a.logp + r : nullptr, sc, V, (int)n_list, top_k, use_p, top_p, min_p, u, 0);
      return;
    }
    listed = n_list <= (uint32_t)LOCAL;
  }
  // a logit under this one has a smaller e (logf, product and quotient are off by far less than the margin)
  auto under = [&](float e) { return sc.lmax + sc.temp * (logf(e) - 1e-3f) - 1e-5f * fabsf(sc.lmax); };
  u64 total = 0, limit = 0;
  if (estimate && !far) {
    // ---- nucleus: the weights by the upper bits of e
    s = m == -INFINITY ? 0.f : s * exp2f((m - sc.lmax) * c2);
    s = warp_sum(s);
    __syncthreads();
    if (lane == 0) sh.scan[warp] = __float_as_uint(s);
    __syncthreads();
    s = 0.f;
    for (int k = 0; k < WARPS; ++k) s += __uint_as_float((uint32_t)sh.scan[k]);
    __syncthreads();
    // tokens so light that all V of them together would not reach past the nucleus need no bin
    const float sure = fmaxf((1.f - top_p) * 0.99f * s / (float)V, 6.0e-8f);
    // most likely all under `light` do not either: of every 16th vector (one of 16 in turn) the weights, by
    // eighths of a nat, say under which the tail weighs 0.7 of what the nucleus leaves (a few heavy tokens, which
    // the choice may have missed, are not taken for a tail: 64 of those chosen have to be over `light`)
    float light = sure;
    {
      const float scale = 8.f / sc.temp;
      if (tid < BINS) sh.hist[tid] = 0;
      if (tid == 0) sh.where = BINS;
      __syncthreads();
      for (int j = tid; j < nvec / 16; j += THREADS) {
        const int vi = 16 * j + (int)((uint32_t)j * 0x9e3779b1u >> 28);
        float l[VE];
        unpack(is_full(vi), fetch(vi), vi, l);
#pragma unroll
        for (int k = 0; k < VE; ++k) {
          const float d = (sc.lmax - l[k]) * scale;
          if (d < (float)BINS) atomicAdd(&sh.hist[(int)d], 1u);
        }
      }
      __syncthreads();
      const float unit = 16.f * 1073741824.f;
      const u64 n = tid < BINS ? (u64)((float)sh.hist[tid] * expf(-0.125f * (float)tid - 0.0625f) * unit) : 0;
      u64 all, many;
      const u64 over = scan_excl(tid < BINS ? sh.hist[tid] : 0u, sh.scan, many);
      before = scan_excl(n, sh.scan, all);
      if (tid < BINS && over >= 64 && (float)(all - before) <= 0.7f * (1.f - top_p) * s * 1073741824.f) atomicMin(&sh.where, tid);
      __syncthreads();
      light = fmaxf(sure, expf(-0.125f * (float)sh.where));
    }
    u64 w;
    while (true) {
      for (int k = tid; k < EBINS; k += THREADS) sh.ecnt[k] = sh.elow[k] = 0;
      __syncthreads();
      w = 0;
      walk([&](const float (&l)[VE], int) {
        float e[VE];
        uint32_t hi, lo;
        es_of(l, e);
        parts_of(e, hi, lo);
        w += ((u64)hi << 20) + lo;
        float most = e[0];
#pragma unroll
        for (int k = 1; k < VE; ++k) most = fmaxf(most, e[k]);
        if (most >= light)
#pragma unroll
          for (int k = 0; k < VE; ++k)
            if (e[k] >= light) {
              const uint32_t b = __float_as_uint(e[k]);
              const int bin = (int)((0x3f800000u >> EBITS) - (b >> EBITS)), drop = 110 - (int)(b >> 23);
              atomicAdd(&sh.ecnt[bin], 1u);
              atomicAdd(&sh.elow[bin], (b & ((1u << EBITS) - 1)) >> max(drop, 0));
            }
      });
      u64 none;
      scan_excl(w, sh.scan, total);
      limit = (u64)ceil((double)top_p * (double)total);
      const int run = (EBINS + THREADS - 1) / THREADS, b0 = tid * run, b1 = min(b0 + run, EBINS);
      // (the sum of 2^16 lower bits fits 32; past so many tokens in a bin: the general way)
      auto weight = [&](int b) -> u64 {
        const uint32_t bits = 0x3f800000u - ((uint32_t)b << EBITS);
        const int up = 17 + (int)(bits >> 23) - 127;
        const u64 mant = (bits & 0x7fffffu) | 0x800000u, cnt = sh.ecnt[b], low = sh.elow[b];
        return up >= 0 ? (cnt * mant + low) << up : cnt * (mant >> -up) + low;
      };
      w = 0;
      bool full = false;
      for (int b = b0; b < b1; ++b) {
        w += weight(b);
        full |= sh.ecnt[b] > 65536u;
      }
      full = __syncthreads_or(full);
      before = scan_excl(w, sh.scan, none);
      if (!full && before < limit && limit <= before + w)
        for (int b = b0; b < b1; ++b) {
          const u64 x = weight(b);
          if (before < limit && limit <= before + x) {
            sh.bin = b;
            sh.need = limit - before;
          }
          before += x;
        }
      __syncthreads();
      if (sh.bin >= 0 || light == sure) break;               // the same answer in all threads
      light = sure;
      __syncthreads();
    }
    if (sh.bin >= 0) {
      const uint32_t q = (0x3f800000u >> EBITS) - (uint32_t)sh.bin;
      const float lo_e = __uint_as_float(q << EBITS);
      sum_above(under(lo_e), [&](float l, int idx, float e) {
        const uint32_t b = __float_as_uint(e) >> EBITS;
        if (b == q) {
          const uint32_t n = atomicAdd(&sh.in_bin, 1u);
          if (n < (uint32_t)LIST) sh.local[n] = order(l, idx);
        }
        return b > q && e >= min_p ? e : 0.f;
      });
      const int n = (int)min(sh.in_bin, (uint32_t)LIST + 1);
      if (n <= LIST) {
        const u64 last = last_of(sc, n, sh.need);
        l_last = logit_of((uint32_t)(last >> 32));
        i_last = (int)~(uint32_t)last;
        for (int k = tid; k < n; k += THREADS) {
          const u64 x = sh.local[k];
          const float e = e_of(logit_of((uint32_t)(x >> 32)));
          if (x >= last && e >= min_p) atomicAdd(&cells[((int)~(uint32_t)x + skip) / VE / (32 * K)], w_of(e));
        }
        __syncthreads();
        const u64 sum = total_cells(before);
        finish(before, sum);
        return;
      }
      __syncthreads();
    }
  }
  // ---- the general way, over the list or the row
  auto each = [&](auto f) {
    if (listed) {
      for (uint32_t i = tid; i < n_list; i += THREADS) {
        const u64 x = sh.local[i];
        f(logit_of((uint32_t)(x >> 32)));
      }
    } else {
      walk([&](const float (&l)[VE], int vi) {
#pragma unroll
        for (int k = 0; k < VE; ++k)
          if (inside(vi * VE - skip + k)) f(l[k]);
      });
    }
  };
  // the largest key such that the weights (or counts) of the keys over it stay under `want`; `left` gets what
  // is wanted of that key itself
  uint32_t kth = 0;
  auto search = [&](bool counts, u64 want, u64& left) -> uint32_t {
    uint32_t key = 0;
    left = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) sh.radix[0][tid] = 0;
      if (tid == 0) { sh.where = 0; sh.pick = 0; }
      __syncthreads();
      each([&](float l) {
        const uint32_t x = key_of(l);
        if (x >= kth && (shift == 24 || (x >> (shift + 8)) == (key >> (shift + 8))))
          atomicAdd(&sh.radix[0][(x >> shift) & 255], counts ? 1ull : w_of(e_of(l)));
      });
      __syncthreads();
      const u64 n = tid < 256 ? sh.radix[0][255 - tid] : 0;
      u64 all;
      const u64 over = scan_excl(n, sh.scan, all);
      if (over < left && left <= over + n) {
        sh.where = 255 - tid;
        sh.pick = over;
      }
      __syncthreads();
      left -= sh.pick;
      key |= (uint32_t)sh.where << shift;
    }
    return key;
  };
  u64 left;
  if (use_k && (!listed || (uint32_t)top_k <= n_list)) {
    kth = search(true, (u64)top_k, left);
    l_last = logit_of(kth);
  }
  if (use_p) {
    u64 w = 0;
    each([&](float l) { if (key_of(l) >= kth) w += w_of(e_of(l)); });
    scan_excl(w, sh.scan, total);
    const uint32_t pth = search(false, (u64)ceil((double)top_p * (double)total), left);
    // of the tokens with exactly this key the first ceil(left / weight) in index order are kept
    const u64 w1 = w_of(e_of(logit_of(pth)));
    const u64 ties = w1 ? (left + w1 - 1) / w1 : 1;
    l_last = logit_of(pth);
    auto tie = [&](const float (&l)[VE], float (&e)[VE], int vi) {       // 2^-40 each
#pragma unroll
      for (int k = 0; k < VE; ++k) e[k] = l[k] == l_last && inside(vi * VE - skip + k) ? 9.094947017729282e-13f : 0.f;
    };
    sum_cells(tie);
    const u64 n = total_cells(before);
    i_last = locate(tie, before, min(ties, n) - 1);
  }
  if (use_k || use_p || far || !(min_p > 0.f)) sum_cells(kept);
  else sum_above(under(min_p), [&](float, int, float e) { return e >= min_p ? e : 0.f; });
  const u64 sum = total_cells(before);
  finish(before, sum);
}

template <class T>
static cudaError_t launch_wide(const SampleArgs& a, cudaStream_t st) {
  static PerDeviceOnce attrs;
  const cudaError_t ae = attrs.run([] {
    return cudaFuncSetAttribute(sample_wide_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleShared));
  });
  if (ae != cudaSuccess) return ae;
  sample_wide_kernel<T><<<a.R, smr::THREADS, sizeof(SampleShared), st>>>(a);
  return cudaGetLastError();
}

template <class T, int NV>
static cudaError_t launch_rows(const SampleArgs& a, int C, cudaStream_t st) {
  static PerDeviceOnce attrs;
  const cudaError_t ae = attrs.run([] {
    cudaError_t e = cudaFuncSetAttribute(sample_kernel<T, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleShared));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(sample_kernel<T, NV>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return e;
  });
  if (ae != cudaSuccess) return ae;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(a.R * C));
  cfg.blockDim = dim3(smr::THREADS);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, NV>, a, C);
}

template <class T>
static cudaError_t launch_sample(const SampleArgs& a, cudaStream_t st) {
  constexpr int VE = 16 / (int)sizeof(T);
  const int nvec = (a.V + 2 * VE - 2) / VE;    // one more than the row's own where it starts off a boundary
  // blocks per row: few rows are spread over all SMs (down to a vector a thread), many take as few blocks
  // as hold a row at 32 values a thread, two blocks an SM
  const int sms = device_attr(cudaDevAttrMultiProcessorCount, 148);
  int C = 1;
  while (C < smr::MAXC && ((nvec + C - 1) / C > smr::THREADS * (32 / VE) ||
                           ((long long)a.R * C * 2 <= sms && (nvec + C - 1) / C > smr::THREADS)))
    C <<= 1;
  const int NV = ((nvec + C - 1) / C + smr::THREADS - 1) / smr::THREADS;
  // one block per row from five rows for eight SMs on (B200, us, clusters / single blocks: 128256 fp32, 64 rows:
  // top-k 46 / 33, nucleus 71 / 101, min-p 34 / 34, plain 26 / 37; 96 rows 64 / 33, 105 / 101, 47 / 34, 37 / 37; 256
  // rows 171 / 71, 288 / 161, 129 / 66, 106 / 75; 50257 fp16, 96 rows: 39 / 18, 65 / 40, 28 / 19, 21 / 18)
  if (NV > 48 / VE || 8ll * a.R >= 5ll * sms) return launch_wide<T>(a, st);
  if (NV <= 8 / VE) return launch_rows<T, 8 / VE>(a, C, st);
  if (NV <= 16 / VE) return launch_rows<T, 16 / VE>(a, C, st);
  if (NV <= 32 / VE) return launch_rows<T, 32 / VE>(a, C, st);
  return launch_rows<T, 48 / VE>(a, C, st);
}

cudaError_t sample_launch(const SampleArgs& a, cudaStream_t st, bool pdl) {
  (void)pdl;
  if (a.R < 0 || a.V < 1 || a.ld < a.V || a.V >= (1 << 24) || a.dtype < 0 || a.dtype > 2) return cudaErrorInvalidValue;
  if (a.R == 0) return cudaSuccess;
  if (!a.logits || !a.u || !a.tok) return cudaErrorInvalidValue;
  switch (a.dtype) {
    case 0: return launch_sample<float>(a, st);
    case 1: return launch_sample<__half>(a, st);
    default: return launch_sample<__nv_bfloat16>(a, st);
  }
}

}  // namespace af
