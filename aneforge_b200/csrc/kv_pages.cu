// Pages of a key/value cache: forking, growing, shrinking and compacting sequences.
//
// The cache of every layer is one pool [layers][2][P][KV][page][dh] (K, then V). Sequence slot s owns
// the pages table[s][0..), of which the first lens[s] rows hold keys and values; refs[p] counts the
// slots that hold page p (0: free). Entries of table past the pages in use are -1 or pages held by that
// slot alone, so of the pages that a slot may write to only the one that row lens[s] falls into can be
// shared.
//
//   fork     dst gives back what it holds and takes src's pages over (counts only; no row is copied)
//   reserve  rows [lens, lens + n) of a slot get pages of its own: free pages for the missing entries
//            (lowest number first, in the order of the slots given and of their rows), and a copy of a
//            shared page that holds rows up to lens - of k listed sharers of a page with r holders the
//            first max(0, min(k, r - 1)) copy it, the last holder keeps it
//   free     rows from `keep` on (all of them by default): their pages are given back
//   compact  the rows lens + path[j] of an accepted path through a drafted tree move to lens + j, in
//            every layer, K and V
//
// fork, reserve and free change a few kilobytes of counters: one block each, whole-number sums only, so
// the result does not depend on an order of atomics. The copies that reserve asks for and compact's
// moves are bound by memory; a block moves the rows of one (layer, K or V), of fewer heads where that would
// leave SMs idle.
//
// B200, 32 layers of 8 key heads of 128, pages of 64 rows (4 KB a row and layer, K and V together): fork of one
// sequence into three 3.7 us, the pages for their next rows 5.1 us and three copies of 33 rows 8.2 us; 56 copies of 53
// rows (389 MB written, 56 MB of sources read) 81 us, 5.5 TB/s. Compacting 5 rows of one sequence 4.4 us (replayed
// from a graph), 7 rows of 48 sequences in 80 layers (110 MB each way) 36.7 us, 6.0 TB/s. The small calls are bound by launches: the copies
// start behind the reservation without a gap (dependent launch), and compact sets the new lengths itself.
#include "af_common.cuh"
#include "af_kernels.h"

namespace af {

namespace pages {
constexpr int THREADS = 1024;
}

// block-wide exclusive scan of one int per thread (1024 threads); `total` gets the sum
AF_DEV int block_scan_excl(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();                              // warp_sums may still be read from the last scan
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// thread i's slot, or -1 where there is none: out of range or listed before (recorded as an error)
AF_DEV int own_slot(const int* slots, int n, int S, int* list, int* err) {
  const int i = threadIdx.x;
  int s = -1;
  if (i < n) {
    s = slots[i];
    if (s < 0 || s >= S) { af_set_err(err, AF_DEV_BAD_SLOT); s = -1; }
  }
  list[i] = s;
  __syncthreads();
  bool twice = false;
  if (s >= 0)
    for (int j = 0; j < i; ++j) twice |= list[j] == s;
  if (twice) { af_set_err(err, AF_DEV_BAD_SLOT); s = -1; }
  return s;
}

// rows from keep[i] on (0 without `keep`) of each listed slot: pages given back, the length cut
__global__ void __launch_bounds__(pages::THREADS) kv_free_kernel(KvPagesArgs a) {
  __shared__ int list[pages::THREADS], from[pages::THREADS];
  const int i = threadIdx.x;
  const int s = own_slot(a.slots, a.n, a.S, list, a.err);
  __syncthreads();
  list[i] = s;
  if (s >= 0) {
    const int len = max(a.lens[s], 0);
    const int keep = a.rows ? min(max(a.rows[i], 0), len) : 0;
    from[i] = (keep + a.page - 1) / a.page;
    a.lens[s] = keep;
  }
  __syncthreads();
  for (long long e = i; e < (long long)a.n * a.W; e += pages::THREADS) {
    const int j = (int)(e / a.W), w = (int)(e % a.W), sj = list[j];
    if (sj < 0 || w < from[j]) continue;
    int* t = a.table + (size_t)sj * a.W + w;
    const int p = *t;
    if (p >= 0 && p < a.P) atomicSub(a.refs + p, 1);
    *t = -1;
  }
}

// slots = dst, rows = src: pairs are independent, dst slots distinct and none of them a source
__global__ void __launch_bounds__(pages::THREADS) kv_fork_kernel(KvPagesArgs a) {
  __shared__ int list[pages::THREADS], from[pages::THREADS], full[pages::THREADS];
  const int i = threadIdx.x;
  int d = own_slot(a.slots, a.n, a.S, list, a.err);
  __syncthreads();
  list[i] = d;
  __syncthreads();
  int src = -1;
  if (i < a.n) {
    src = a.rows[i];
    bool bad = src < 0 || src >= a.S;
    for (int j = 0; j < a.n && !bad; ++j) bad = list[j] == src;
    if (bad) { af_set_err(a.err, AF_DEV_BAD_SLOT); src = -1; }
  }
  __syncthreads();
  if (src < 0) d = -1;
  list[i] = d;
  from[i] = src;
  if (d >= 0) full[i] = (a.lens[src] + a.page - 1) / a.page;
  __syncthreads();
  const long long E = (long long)a.n * a.W;
  for (long long e = i; e < E; e += pages::THREADS) {
    const int j = (int)(e / a.W), w = (int)(e % a.W);
    if (list[j] < 0) continue;
    const int p = a.table[(size_t)list[j] * a.W + w];
    if (p >= 0 && p < a.P) atomicSub(a.refs + p, 1);
  }
  __syncthreads();
  for (long long e = i; e < E; e += pages::THREADS) {
    const int j = (int)(e / a.W), w = (int)(e % a.W);
    if (list[j] < 0) continue;
    int p = w < full[j] ? a.table[(size_t)from[j] * a.W + w] : -1;
    if (p < 0 || p >= a.P) p = -1;
    else atomicAdd(a.refs + p, 1);
    a.table[(size_t)list[j] * a.W + w] = p;
  }
  if (d >= 0) a.lens[d] = a.lens[src];
}

// scratch: copies [n][4] = (old page, new page, rows, -), then the numbers of the free pages handed out
__global__ void __launch_bounds__(pages::THREADS) kv_reserve_kernel(KvPagesArgs a) {
  __shared__ int list[pages::THREADS], warp_sums[32];
  pdl_trigger();                                // the copies' blocks may take their places
  const int i = threadIdx.x;
  const int s = own_slot(a.slots, a.n, a.S, list, a.err);
  int c0 = 0, c1 = 0, fill = 0, tail = -1;
  int* t = nullptr;
  if (s >= 0) {
    const int len = a.lens[s], need = max(a.rows[i], 0);
    t = a.table + (size_t)s * a.W;
    const long long end = ((long long)len + need + a.page - 1) / a.page;
    if (len < 0 || end > a.W || need == 0) {    // nothing for this slot
      if (need) af_set_err(a.err, AF_DEV_BAD_POS);
    } else {
      c0 = len / a.page;
      c1 = (int)end;
      fill = len - c0 * a.page;
      if (fill) tail = t[c0];
      if (tail >= a.P) tail = -1;
    }
  }
  __syncthreads();
  list[i] = tail;
  __syncthreads();
  bool copy = false;
  if (tail >= 0) {
    int before = 0;
    for (int j = 0; j < i; ++j) before += list[j] == tail;
    copy = a.refs[tail] - before > 1;
  }
  int want = 0;
  for (int c = c0; c < c1; ++c) want += (c == c0 && copy) || t[c] < 0;
  int total;
  const int at = block_scan_excl(want, warp_sums, total);
  int* copies = a.scratch;
  int* fresh = a.scratch + 4 * (size_t)a.n;
  // the first `total` free pages, in order
  int found = 0;
  for (int base = 0; base < a.P && found < total; base += pages::THREADS * 4) {
    const int p = base + 4 * i;
    int free4[4], cnt = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      free4[k] = p + k < a.P && a.refs[p + k] == 0;
      cnt += free4[k];
    }
    int sum;
    int r = found + block_scan_excl(cnt, warp_sums, sum);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (free4[k]) {
        if (r < total) fresh[r] = p + k;
        ++r;
      }
    found += sum;
  }
  __syncthreads();
  const bool enough = found >= total;           // all or nothing
  if (!enough && i == 0) af_set_err(a.err, AF_DEV_NO_PAGES);
  if (i < a.n) {
    int4 c = make_int4(-1, -1, 0, 0);
    if (enough && s >= 0) {
      int r = at;
      for (int k = c0; k < c1; ++k) {
        const bool cow = k == c0 && copy;
        if (!cow && t[k] >= 0) continue;
        const int p = fresh[r++];
        a.refs[p] = 1;
        t[k] = p;
        if (cow) {
          atomicSub(a.refs + tail, 1);
          c = make_int4(tail, p, fill, 0);
        }
      }
    }
    reinterpret_cast<int4*>(copies)[i] = c;
  }
}

// grid (n, 2 * layers, head groups): the filled rows of one copied page, one layer's K or V, a.heads heads.
// A head's rows are contiguous; four 16-byte pieces a thread are on their way together.
__global__ void __launch_bounds__(256) kv_copy_kernel(KvPagesArgs a) {
  pdl_wait();                                   // the list comes from kv_reserve
  const int4 c = __ldcg(reinterpret_cast<const int4*>(a.scratch) + blockIdx.x);
  if (c.x < 0) return;
  const size_t head = (size_t)a.page * a.row16, pg = head * a.KV;
  const int h0 = blockIdx.z * a.heads, h1 = min(a.KV, h0 + a.heads);
  uint4* plane = static_cast<uint4*>(a.pool) + (size_t)blockIdx.y * a.P * pg;
  const int per = c.z * a.row16;                // pieces of a head's filled rows
  for (int h = h0; h < h1; ++h) {
    const uint4* from = plane + (size_t)c.x * pg + h * head;
    uint4* to = plane + (size_t)c.y * pg + h * head;
    for (int e = threadIdx.x; e < per; e += 4 * 256) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + 256 * k < per) v[k] = __ldcs(from + e + 256 * k);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + 256 * k < per) __stcs(to + e + 256 * k, v[k]);
    }
  }
}

// whether rows j, j + step, ... of a path can be taken: its nodes rise (parents come before children), its rows
// have pages, and none of slots j, j + step, ... before it is the same one (whose block moves rows meanwhile)
AF_DEV bool path_bad(const KvPagesArgs& a, int b, int s, int n, int len, int j, int step) {
  bool bad = s < 0 || s >= a.S || n < 0 || n > a.D;
  if (bad) return true;
  for (int k = j; k < b; k += step) bad |= a.slots[k] == s;
  const int* table = a.table + (size_t)s * a.W;
  for (; j < n && !bad; j += step) {
    const int at = a.path[(size_t)b * a.D + j];
    const long long from = (long long)len + at;
    bad = at < j || (j && at <= a.path[(size_t)b * a.D + j - 1]) || from >= (long long)a.W * a.page;
    if (!bad) {
      const int p = table[from / a.page], q = table[(len + j) / a.page];
      bad = p < 0 || p >= a.P || q < 0 || q >= a.P;
    }
  }
  return bad;
}

// grid (B, 2 * layers + 1): one layer's K or V of one sequence; block (0, 2 * layers) writes the new
// lengths. A thread moves one 16-byte column of one head through the rows of the path in order: row j is
// written after row path[j] >= j is read and no later row is read from it, so that no other thread's
// access meets it.
__global__ void __launch_bounds__(256) kv_compact_kernel(KvPagesArgs a) {
  if (blockIdx.y == 2 * a.layers) {
    if (blockIdx.x) return;
    for (int s = threadIdx.x; s < a.S; s += blockDim.x) a.lens_out[s] = a.lens[s];
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int b = threadIdx.x >> 5; b < a.n; b += blockDim.x >> 5) {
      const int s = a.slots[b], n = a.rows[b], len = s >= 0 && s < a.S ? a.lens[s] : 0;
      const bool bad = __any_sync(0xffffffffu, path_bad(a, b, s, n, max(len, 0), lane, 32)) || len < 0;
      if (lane == 0) {
        if (bad) af_set_err(a.err, AF_DEV_BAD_SLOT);
        else a.lens_out[s] = len + n;
      }
    }
    return;
  }
  const int b = blockIdx.x;
  const int s = a.slots[b], n = a.rows[b];
  const int len = s >= 0 && s < a.S ? a.lens[s] : 0;
  __shared__ size_t from_s[256], to_s[256];     // places of the rows, 256 at a time
  if (__syncthreads_or(path_bad(a, b, s, n, max(len, 0), threadIdx.x, blockDim.x)) || len < 0) return;
  const int* table = a.table + (size_t)s * a.W;
  const size_t head = (size_t)a.page * a.row16, pg = head * a.KV;
  uint4* plane = static_cast<uint4*>(a.pool) + (size_t)blockIdx.y * a.P * pg;
  for (int base = 0; base < n; base += 256) {
    const int m = min(256, n - base);
    __syncthreads();
    if ((int)threadIdx.x < m) {
      const int r = len + a.path[(size_t)b * a.D + base + threadIdx.x], w = len + base + threadIdx.x;
      from_s[threadIdx.x] = (size_t)table[r / a.page] * pg + (size_t)(r % a.page) * a.row16;
      to_s[threadIdx.x] = (size_t)table[w / a.page] * pg + (size_t)(w % a.page) * a.row16;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.KV * a.row16; e += blockDim.x) {
      uint4* col = plane + (size_t)(e / a.row16) * head + e % a.row16;
      constexpr int U = 8;
      for (int j0 = 0; j0 < m; j0 += U) {
        uint4 v[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (j0 + k < m) v[k] = col[from_s[j0 + k]];
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (j0 + k < m) col[to_s[j0 + k]] = v[k];
      }
    }
  }
}

static bool pages_ok(const KvPagesArgs& a) {
  return a.table && a.lens && (a.slots || a.n == 0) && a.S > 0 && a.W > 0 && a.P > 0 && a.page > 0 && a.n >= 0;
}

cudaError_t kv_free_launch(const KvPagesArgs& a, cudaStream_t st) {
  if (!pages_ok(a) || !a.refs || a.n > pages::THREADS) return cudaErrorInvalidValue;
  if (a.n == 0) return cudaSuccess;
  kv_free_kernel<<<1, pages::THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t kv_fork_launch(const KvPagesArgs& a, cudaStream_t st) {
  if (!pages_ok(a) || !a.refs || (!a.rows && a.n) || a.n > pages::THREADS) return cudaErrorInvalidValue;
  if (a.n == 0) return cudaSuccess;
  kv_fork_kernel<<<1, pages::THREADS, 0, st>>>(a);
  return cudaGetLastError();
}

size_t kv_reserve_scratch_bytes(int n, int P) { return 4 * (4 * (size_t)n + (size_t)P); }

static bool pool_ok(const KvPagesArgs& a) {
  return a.pool && a.layers > 0 && a.KV > 0 && a.row16 > 0 && (reinterpret_cast<uintptr_t>(a.pool) & 15) == 0 &&
         a.layers < 32767 && (long long)a.page * a.KV * a.row16 < (1ll << 30);
}

cudaError_t kv_reserve_launch(const KvPagesArgs& a, cudaStream_t st) {
  if (!pages_ok(a) || !a.refs || (!a.rows && a.n) || a.n > pages::THREADS || !pool_ok(a) || !a.scratch ||
      (reinterpret_cast<uintptr_t>(a.scratch) & 15))
    return cudaErrorInvalidValue;
  if (a.n == 0) return cudaSuccess;
  kv_reserve_kernel<<<1, pages::THREADS, 0, st>>>(a);
  // blocks of all heads where there are plenty, of fewer where the copies would not fill the GPU
  KvPagesArgs c = a;
  c.heads = a.KV;
  while (c.heads > 1 && (long long)a.n * 2 * a.layers * ((a.KV + c.heads - 1) / c.heads) < 8 * 148) c.heads = (c.heads + 1) / 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3(a.n, 2 * a.layers, (a.KV + c.heads - 1) / c.heads);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  return cudaLaunchKernelEx(&cfg, kv_copy_kernel, c);
}

cudaError_t kv_compact_launch(const KvPagesArgs& a, cudaStream_t st) {
  if (!pages_ok(a) || ((!a.rows || !a.path) && a.n) || !pool_ok(a) || a.D < 1 || !a.lens_out || a.lens_out == a.lens ||
      a.n > pages::THREADS)
    return cudaErrorInvalidValue;
  if (a.n == 0) return cudaMemcpyAsync(a.lens_out, a.lens, 4 * (size_t)a.S, cudaMemcpyDeviceToDevice, st);
  kv_compact_kernel<<<dim3(a.n, 2 * a.layers + 1), 256, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace af
