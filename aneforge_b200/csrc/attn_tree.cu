// Attention of a tree of drafted tokens over a paged key/value cache.
//
// Node t of sequence b is cache row lens[b] + t; row j of the sequence lies in page table[b][j / page],
// row j % page, of K and V [P][KV][page][dh]. The node's rotary position is lens[b] + depth[b][t], and
// it sees every row before lens[b] and the nodes u with bit u set in mask[b][t] (no mask: u <= t, a
// chain). One node is the ordinary decode step. A node that sees nothing (an empty prefix and no bit)
// gives zeros, as do the nodes from nodes[b] on, which are not written either.
//
//   tree_append  q, k: optional per-head RMSNorm, then RoPE at the node's position, rounded to fp16 (the
//                matmul operand and the cache format); k and v into their cache rows, q into a buffer
//                [B][KV][T * G][dh] (row t * G + g), so that the G heads which share a key head are rows
//                of one product
//   attn_tree    softmax(scale q k^T) v over the prefix and the visible nodes; scores, maximum, sum and
//                output in fp32
//
// attn_tree_tc.cu has the second kernel for head dims 64 and 128 whose pages are of a multiple of 8 rows (or one page a
// sequence); the one here takes the rest: head dims 16 and 32, pages of 100, 37 or 4 rows and the like, and scales that
// are not positive (the other's running maximum is of unscaled scores). It is the simple one: a warp has a query row's
// keys to itself, 32 at a time, and is bound by their dot products one after the other. B200, 8 key heads of 128: 24
// nodes x 4 heads at 4001 rows in pages of 100 took 1170 us (pages of 64, the other kernel: 21.6 us), 12 x 16 nodes x 8
// heads over 2000..8000 rows 8.3 ms (63 us), one node x 4 heads at 576 rows 163 us (13.4 us).
//
// A table entry outside the pool ends the sequence there for reading (its rows count as masked) and is
// recorded as an error; nothing is read or written through it.
#include "af_common.cuh"
#include "af_kernels.h"
#include "attn_common.cuh"
#include "tree_common.cuh"

namespace af {

// page of cache row j of sequence b, or -1
AF_DEV int tree_page(const AttnTreeArgs& a, int b, int j) {
  const int w = j / a.page;
  if (w >= a.W) return -1;
  const int p = __ldg(a.table + (size_t)b * a.W + w);
  return p >= 0 && p < a.P ? p : -1;
}

// grid (B * T, ceil((H + KV) / 8)), a warp per head; latency of one dependent chain of loads for few rows (2.8 us for
// one node of 32 + 8 heads of 128), fp32 in and fp16 out for many (8 MB read in 8 us for 192 nodes of 64 + 8 heads)
template <int DH>
__global__ void __launch_bounds__(256) tree_append_kernel(AttnTreeArgs a) {
  using HL = HeadLayout<DH>;
  constexpr int EPL = HL::EPL;
  const int row = blockIdx.x, b = row / a.T, t = row - b * a.T;
  const int y = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (y >= a.H + a.KV) return;
  const bool active = lane < HL::LANES;
  // triggered after the wait: a dependent that starts now may read everything written before this kernel
  pdl_wait();
  pdl_trigger();
  // the row, the extent and the depth are on their way together
  float rc[EPL], rs[EPL], v[EPL], vv[EPL];
  const float* x = a.qkv + (size_t)row * a.ld_qkv;
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    v[e] = active ? __ldcg(x + (size_t)y * DH + lane * EPL + e) : 0.f;
    vv[e] = active && y >= a.H ? __ldcg(x + (size_t)(y + a.KV) * DH + lane * EPL + e) : 0.f;
  }
  const int depth = a.depth ? __ldg(a.depth + row) : t;
  int len, nodes;
  tree_extent(a, b, len, nodes);
  if (t >= nodes) {
    const bool cut = t < (a.nodes ? min(__ldcg(a.nodes + b), a.T) : a.T);
    if (cut && lane == 0) af_set_err(a.err, AF_DEV_BAD_POS);
    return;
  }
  const int pos = len + depth;
  const bool rope = a.cos_t != nullptr;
  const bool lost = rope && (pos < 0 || pos >= a.rope_rows);       // no such position: the node's q and k are zeros
  if (lost) {
    if (lane == 0) af_set_err(a.err, AF_DEV_BAD_POS);
#pragma unroll
    for (int e = 0; e < EPL; ++e) v[e] = 0.f;
  }
  load_rope_row<DH>(a.cos_t, a.sin_t, rope && !lost ? pos : 0, lane, rc, rs);
  if (y < a.H) {
    norm_rope_head_pre<DH>(v, lane, a.qn_g, a.qn_floor, rope, rc, rs);
    const int G = a.H / a.KV;
    __half* q = a.q + (((size_t)b * a.KV + y / G) * a.T * G + (size_t)t * G + y % G) * DH;
    if (active)
#pragma unroll
      for (int e = 0; e < EPL; ++e) q[lane * EPL + e] = f2h(v[e]);
    return;
  }
  const int kvh = y - a.H, j = len + t, p = tree_page(a, b, j);
  if (p < 0) {
    if (lane == 0) {
      af_set_err(a.err, AF_DEV_BAD_POS);
      a.flags[((size_t)b * a.KV + kvh) * a.T + t] = 0;
    }
    return;
  }
  norm_rope_head_pre<DH>(v, lane, a.kn_g, a.kn_floor, rope, rc, rs);
  const size_t o = (size_t)p * a.page_stride + ((size_t)kvh * a.page + j % a.page) * DH + lane * EPL;
  bool finite = true;
  if (active)
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      const __half kh = f2h(v[e]), vh = f2h(vv[e]);
      a.kc[o + e] = kh;
      a.vc[o + e] = vh;
      finite &= isfinite(h2f(kh)) && isfinite(h2f(vh));
    }
  finite = __all_sync(0xffffffffu, finite);
  if (lane == 0) a.flags[((size_t)b * a.KV + kvh) * a.T + t] = !finite;
}

// grid (ceil(T * G / 8), KV, B), a warp per query row: 32 keys at a time, a key per lane for the scores,
// then the lanes share out the head's elements for the sum over values
template <int DH>
__global__ void __launch_bounds__(256) attn_tree_kernel(AttnTreeArgs a) {
  using HL = HeadLayout<DH>;
  constexpr int EPL = HL::EPL;
  __shared__ float q_s[8][DH];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.H / a.KV, kvh = blockIdx.y, b = blockIdx.z;
  const int r = blockIdx.x * 8 + warp;
  pdl_wait();
  if (r >= a.T * G) return;
  const int t = r / G, g = r - t * G;
  int len, nodes;
  tree_extent(a, b, len, nodes);
  __half* out = a.out + ((size_t)b * a.T + t) * a.ld_out + (size_t)(kvh * G + g) * DH;
  const bool active = lane < HL::LANES;
  float acc[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
  float m = -INFINITY, l = 0.f;
  if (t < nodes) {
    const __half* q = a.q + (((size_t)b * a.KV + kvh) * a.T * G + r) * DH;
    for (int d = lane; d < DH; d += 32) q_s[warp][d] = h2f(__ldcg(q + d));
    __syncwarp();
    const int n = len + nodes;
    for (int base = 0; base < n; base += 32) {
      const int j = base + lane;
      int p = j < n ? tree_page(a, b, j) : -1;
      if (j < n && p < 0) af_set_err(a.err, AF_DEV_BAD_POS);
      if (j >= len) {
        const int u = j - len;
        const bool sees = u < nodes && (a.mask ? (__ldg(a.mask + ((size_t)b * a.T + t) * a.mask_words + (u >> 5)) >> (u & 31)) & 1
                                               : u <= t);
        if (!sees) p = -1;
      }
      const size_t o = p < 0 ? 0 : (size_t)p * a.page_stride + ((size_t)kvh * a.page + j % a.page) * DH;
      float s = -INFINITY;
      if (p >= 0) {
        float dot = 0.f;
#pragma unroll 4
        for (int d = 0; d < DH; d += 8) {
          float f[8];
          h8_to_f32(__ldcg(reinterpret_cast<const uint4*>(a.kc + o + d)), f);
#pragma unroll
          for (int k = 0; k < 8; ++k) dot = fmaf(q_s[warp][d + k], f[k], dot);
        }
        s = dot * a.scale;
      }
      const unsigned live = __ballot_sync(0xffffffffu, p >= 0);
      if (!live) continue;
      const float mn = fmaxf(m, warp_max(s));
      const float mb = mn == -INFINITY ? 0.f : mn;           // only scores of -inf so far, or NaN, which stays
      const float corr = m == -INFINITY ? 0.f : expf(m - mn);
      const float pe = p >= 0 ? expf(s - mb) : 0.f;
      l = l * corr + warp_sum(pe);
      m = mn;
#pragma unroll
      for (int e = 0; e < EPL; ++e) acc[e] *= corr;
      for (int k = 0; k < 32; ++k) {
        if (!(live >> k & 1)) continue;
        const float pk = __shfl_sync(0xffffffffu, pe, k);
        const size_t ok = __shfl_sync(0xffffffffu, (unsigned long long)o, k);
        float f[EPL];
        load_row_f16<DH>(a.vc + ok, lane, f);
#pragma unroll
        for (int e = 0; e < EPL; ++e) acc[e] = fmaf(pk, f[e], acc[e]);
      }
    }
  }
  const float il = l == 0.f ? 0.f : 1.f / l;   // NaN stays
  if (active)
#pragma unroll
    for (int e = 0; e < EPL; ++e) out[lane * EPL + e] = f2h(acc[e] * il);
}

// scratch: q, flags, and for the tensor-core form two partial results a block (a pair that a block does
// not have whole: one at the start of its run, one at the end)
struct TreeScratch {
  size_t flags, part, bytes;
  int part_rows;
};
static TreeScratch tree_scratch(int B, int T, int H, int KV, int dh) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  const int R = T * (H / KV);
  TreeScratch s;
  s.flags = up((size_t)B * T * H * dh * 2);
  s.part = s.flags + up((size_t)B * KV * T);
  s.part_rows = R > 128 ? 256 : (R + 7) / 8 * 8;
  s.bytes = s.part + (dh == 64 || dh == 128 ? (size_t)attn_tree_tc_blocks() * 2 * s.part_rows * (dh + 2) * 4 : 0);
  return s;
}

size_t attn_tree_scratch_bytes(int B, int T, int H, int KV, int dh) {
  if (B < 0 || T < 1 || KV < 1 || H % KV || dh < 1) return 0;
  return tree_scratch(B, T, H, KV, dh).bytes;
}

template <int DH>
static cudaError_t tree_launch(const AttnTreeArgs& a, cudaStream_t st, bool pdl) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  cfg.stream = st;
  cfg.blockDim = dim3(256);
  cfg.gridDim = dim3(a.B * a.T, (a.H + a.KV + 7) / 8);
  cudaError_t e = cudaLaunchKernelEx(&cfg, tree_append_kernel<DH>, a);
  if (e != cudaSuccess) return e;
  if constexpr (DH >= 64)
    if (attn_tree_tc_ok(a)) return attn_tree_tc_launch(a, st);
  cfg.gridDim = dim3((a.T * (a.H / a.KV) + 7) / 8, a.KV, a.B);
  cfg.numAttrs = 0;
  return cudaLaunchKernelEx(&cfg, attn_tree_kernel<DH>, a);
}

cudaError_t attn_tree_launch(const AttnTreeArgs& a0, cudaStream_t st, bool pdl) {
  AttnTreeArgs a = a0;
  if (a.KV < 1 || a.H < 1 || a.H % a.KV || a.B < 0 || a.T < 1 || a.T > TREE_MAX_NODES || a.page < 1 || a.W < 1 || a.P < 1 ||
      (long long)a.W * a.page > (1ll << 30) || a.page_stride < (long long)a.KV * a.page * a.dh || a.page_stride % 8 ||
      a.ld_qkv < (a.H + 2 * a.KV) * a.dh || a.ld_out < a.H * a.dh || (a.mask && a.mask_words < (a.T + 31) / 32) ||
      (a.cos_t == nullptr) != (a.sin_t == nullptr) || (a.cos_t && a.rope_rows < 1) ||
      (reinterpret_cast<uintptr_t>(a.kc) & 15) || (reinterpret_cast<uintptr_t>(a.vc) & 15))
    return cudaErrorInvalidValue;
  if (a.B == 0) return cudaSuccess;
  if (!a.qkv || !a.kc || !a.vc || !a.table || !a.lens || !a.out || !a.scratch ||
      a.scratch_bytes < attn_tree_scratch_bytes(a.B, a.T, a.H, a.KV, a.dh) || a.B > 65535 || a.KV > 65535)
    return cudaErrorInvalidValue;
  const TreeScratch s = tree_scratch(a.B, a.T, a.H, a.KV, a.dh);
  char* base = static_cast<char*>(a.scratch);
  if (reinterpret_cast<uintptr_t>(base) & 15) return cudaErrorInvalidValue;
  a.q = reinterpret_cast<__half*>(base);
  a.flags = reinterpret_cast<unsigned char*>(base + s.flags);
  a.part = reinterpret_cast<float*>(base + s.part);
  a.part_rows = s.part_rows;
  switch (a.dh) {
    case 16: return tree_launch<16>(a, st, pdl);
    case 32: return tree_launch<32>(a, st, pdl);
    case 64: return tree_launch<64>(a, st, pdl);
    case 128: return tree_launch<128>(a, st, pdl);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace af
