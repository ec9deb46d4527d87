// One token per row of logits: temperature, top-k, top-p and min-p, drawn with a given uniform number.
//
// With l the row in fp32 (NaN as -inf, -0 as +0), z = l / temperature and e = exp(z - max z), a token's
// weight is the integer w = floor(e * 2^40): sums of weights are exact (2^40 * 2^24 tokens fit 64 bits),
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

namespace smp {
constexpr int THREADS = 1024;
}

AF_DEV float as_logit(float l) { return l != l ? -INFINITY : l + 0.f; }

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

struct RowScale {
  float lmax, zmax, temp;
  AF_DEV float below(float l) const {           // z - max z, 0 for the largest (also where both are infinite)
    const float z = __fdiv_rn(l, temp);
    return l == lmax || z == zmax ? 0.f : z - zmax;
  }
  AF_DEV float e(float l) const { return expf(below(l)); }
  AF_DEV u64 w(float l) const { return (u64)(e(l) * 1099511627776.f); }
};

template <class T>
AF_DEV T block_sum(T v, T* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = 0;
  for (int k = 0; k < smp::THREADS / 32; ++k) s += buf[k];
  return s;
}

// grid: one block per row
template <class T>
__global__ void __launch_bounds__(smp::THREADS) sample_kernel(SampleArgs a) {
  __shared__ u64 sum_s[32];
  __shared__ u64 hist[256];
  __shared__ u64 best_s;
  __shared__ u64 pick_s[4];
  const int r = blockIdx.x, V = a.V, tid = threadIdx.x;
  const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.ld * sizeof(T);
  const float temp = a.temperature ? a.temperature[r] : a.temperature_s;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_s;
  const float top_p = a.top_p ? a.top_p[r] : a.top_p_s;
  const float min_p = fminf(a.min_p ? a.min_p[r] : a.min_p_s, 1.f);
  // the first largest logit: the greatest (key, ~index)
  u64 best = 0;
  for (int i = tid; i < V; i += smp::THREADS) {
    const u64 k = (u64)key_of(load_logit<T>(row, i)) << 32 | (uint32_t)~i;
    best = k > best ? k : best;
  }
  if (tid == 0) best_s = 0;
  __syncthreads();
  atomicMax(&best_s, best);
  __syncthreads();
  best = best_s;
  const int first = (int)~(uint32_t)best;
  RowScale sc;
  sc.lmax = load_logit<T>(row, first);
  sc.temp = temp > 0.f ? temp : 1.f;
  sc.zmax = __fdiv_rn(sc.lmax, sc.temp);
  if (sc.lmax == -INFINITY || !(temp > 0.f)) {
    if (tid == 0) {
      const bool none = sc.lmax == -INFINITY;
      a.tok[r] = none ? -1 : first;
      if (a.logp) a.logp[r] = none ? -INFINITY : 0.f;
    }
    return;
  }
  // top-k: the k-th largest key, byte by byte
  uint32_t kth = 0;
  if (top_k > 0 && top_k < V) {
    u64 left = top_k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += smp::THREADS) {
        const uint32_t k = key_of(load_logit<T>(row, i));
        if (shift == 24 || (k >> (shift + 8)) == (kth >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1ull);
      }
      __syncthreads();
      int d = 255;
      for (; d > 0 && left > hist[d]; --d) left -= hist[d];
      kth |= (uint32_t)d << shift;
    }
  }
  // top-p: the key that the limit falls into, and how much of it is left for the ties
  uint32_t pth = 0;
  int pidx = V;
  if (top_p > 0.f && top_p < 1.f) {
    u64 total = 0;
    for (int i = tid; i < V; i += smp::THREADS) {
      const float l = load_logit<T>(row, i);
      if (key_of(l) >= kth) total += sc.w(l);
    }
    total = block_sum(total, sum_s);
    u64 left = (u64)ceil((double)top_p * (double)total);
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += smp::THREADS) {
        const float l = load_logit<T>(row, i);
        const uint32_t k = key_of(l);
        if (k >= kth && (shift == 24 || (k >> (shift + 8)) == (pth >> (shift + 8))))
          atomicAdd(&hist[(k >> shift) & 255], sc.w(l));
      }
      __syncthreads();
      int d = 255;
      for (; d > 0 && left > hist[d]; --d) left -= hist[d];
      pth |= (uint32_t)d << shift;
    }
    // of the tokens with exactly this key, the first ceil(left / weight) in index order
    const u64 w1 = sc.w(__uint_as_float(pth & 0x80000000u ? pth & 0x7fffffffu : ~pth));
    const u64 ties = w1 ? (left + w1 - 1) / w1 : 0;
    u64 seen = 0;
    for (int base = 0; base < V; base += smp::THREADS) {
      const int i = base + tid;
      const bool tie = i < V && key_of(load_logit<T>(row, i)) == pth;
      const unsigned ball = __ballot_sync(0xffffffffu, tie);
      __syncthreads();
      if ((tid & 31) == 0) sum_s[tid >> 5] = __popc(ball);
      __syncthreads();
      u64 before = seen + __popc(ball & ((1u << (tid & 31)) - 1));
      for (int k = 0; k < 32; ++k) {
        if (k < (tid >> 5)) before += sum_s[k];
        seen += sum_s[k];
      }
      if (tie && before + 1 == ties) pick_s[0] = i;
      if (seen >= ties) break;
    }
    __syncthreads();
    pidx = (int)pick_s[0];
  }
  // kept weights in index order: every thread a run of consecutive tokens
  const int per = (V + smp::THREADS - 1) / smp::THREADS, i0 = tid * per, i1 = min(V, i0 + per);
  auto kept = [&](int i) -> u64 {
    const float l = load_logit<T>(row, i);
    const uint32_t k = key_of(l);
    if (k < kth || k < pth || (k == pth && i > pidx) || !(sc.e(l) >= min_p)) return 0;
    return sc.w(l);
  };
  u64 mine = 0;
  for (int i = i0; i < i1; ++i) mine += kept(i);
  const u64 total = block_sum(mine, sum_s);
  u64 target = (u64)fmax(floor((double)a.u[r] * (double)total), 0.0);
  target = target < total ? target : total - 1;
  u64 x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, x, o);
    if ((tid & 31) >= o) x += y;
  }
  u64 before = x - mine;
  for (int k = 0; k < (tid >> 5); ++k) before += sum_s[k];
  if (before <= target && target < before + mine) {
    int i = i0;
    for (; i < i1; ++i) {
      before += kept(i);
      if (before > target) break;
    }
    a.tok[r] = i;
    if (a.logp) {
      const float l = load_logit<T>(row, i);
      a.logp[r] = sc.below(l) - logf((float)total / 1099511627776.f);
    }
  }
}

cudaError_t sample_launch(const SampleArgs& a, cudaStream_t st, bool pdl) {
  (void)pdl;
  if (a.R < 0 || a.V < 1 || a.ld < a.V || a.V > (1 << 24) || a.dtype < 0 || a.dtype > 2) return cudaErrorInvalidValue;
  if (a.R == 0) return cudaSuccess;
  if (!a.logits || !a.u || !a.tok) return cudaErrorInvalidValue;
  switch (a.dtype) {
    case 0: sample_kernel<float><<<a.R, smp::THREADS, 0, st>>>(a); break;
    case 1: sample_kernel<__half><<<a.R, smp::THREADS, 0, st>>>(a); break;
    default: sample_kernel<__nv_bfloat16><<<a.R, smp::THREADS, 0, st>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace af
