// Drawing a token from each row of logits: temperature, top-k, top-p and
// min-p filters, then the maximum of x / T + noise over the tokens that are
// left (with standard Gumbel noise that is a draw from their softmax).
//
// Order the row by (logit descending, index ascending).  With weights
// w_i = exp((x_i - max) / T), every filter keeps a leading run of that order:
// top-k the first k; top-p those whose predecessors' weights sum to less than
// p times the weight of the first k; min-p those with w_i >= min_p.  So a
// row is described by one cut, the last (logit, index) pair that stays.
//
// One block per row.  The cut is found by bisection over the pairs, as 52-bit
// integers (32 bits of the logit in an order-preserving form, 20 of the
// index), counting or summing the row at every step.
#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace sampling {

constexpr int kThreads = 1024;
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;

// Order-preserving integer of a float; NaN sorts below -inf, -0 equals +0.
MNB_DEVICE uint32_t key_of(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
constexpr uint32_t kKeyNegInf = 0x007fffffu;
// (logit, index) as one integer: larger comes first in the row's order.
MNB_DEVICE uint64_t pair_of(uint32_t key, int i) {
  return (static_cast<uint64_t>(key) << kIndexBits) | (kIndexMask - static_cast<uint32_t>(i));
}

template <typename T>
MNB_DEVICE float load(const T* p, int i);
template <>
MNB_DEVICE float load<float>(const float* p, int i) { return p[i]; }
template <>
MNB_DEVICE float load<__nv_bfloat16>(const __nv_bfloat16* p, int i) { return bf16_to_f32(p[i]); }

// Sum over the block in a fixed order.
template <typename V>
MNB_DEVICE V block_sum(V v, V* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  V s = sh[threadIdx.x % 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  return s;
}
MNB_DEVICE uint64_t block_max(uint64_t v, uint64_t* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  uint64_t s = sh[threadIdx.x % 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s = max(s, __shfl_xor_sync(0xffffffffu, s, o));
  __syncthreads();
  return s;
}

// One value for all rows, or one for each.
template <typename S>
MNB_DEVICE auto at(const S& s, int r) {
  return s.each ? s.each[r] : s.all;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T* __restrict__ logits, long long ld,
                                                          const float* __restrict__ noise, long long noise_ld, int V,
                                                          Setting temperature, WholeSetting top_k, Setting top_p,
                                                          Setting min_p, long long* __restrict__ token,
                                                          float* __restrict__ logprob) {
  __shared__ uint64_t sh64[32];
  __shared__ float shf[32];
  __shared__ int shi[32];
  const int r = blockIdx.x;
  const T* x = logits + r * ld;
  uint64_t best = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) best = max(best, pair_of(key_of(load(x, i)), i));
  best = block_max(best, sh64);
  const uint32_t top_key = static_cast<uint32_t>(best >> kIndexBits);
  const float t = at(temperature, r);
  if (top_key <= kKeyNegInf) {  // no token left
    if (threadIdx.x == 0) {
      token[r] = -1;
      if (logprob) logprob[r] = -INFINITY;
    }
    return;
  }
  const int first = static_cast<int>(kIndexMask - (best & kIndexMask));
  if (!(t > 0.f)) {
    if (threadIdx.x == 0) {
      token[r] = first;
      if (logprob) logprob[r] = 0.f;
    }
    return;
  }
  const float mx = load(x, first);
  const float scale = 1.4426950408889634f / t;
  // weight of a logit; an infinite maximum takes all of it
  auto weight = [&](float v) { return v == mx ? 1.f : ex2_approx((v - mx) * scale); };

  uint64_t cut = static_cast<uint64_t>(kKeyNegInf + 1) << kIndexBits;  // tokens at -inf are never kept
  const int k = at(top_k, r);
  if (k > 0 && k < V) {
    uint64_t lo = cut, hi = best;  // smallest pair with fewer than k before it
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      int n = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) n += pair_of(key_of(load(x, i)), i) > mid;
      if (block_sum(n, shi) < k) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  const float p = at(top_p, r);
  if (p < 1.f) {
    float z = 0.f;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float v = load(x, i);
      if (pair_of(key_of(v), i) >= cut) z += weight(v);
    }
    const float limit = p * block_sum(z, shf);
    uint64_t lo = cut, hi = best;  // smallest pair with less than the limit before it
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      float before = 0.f;
      for (int i = threadIdx.x; i < V; i += kThreads) {
        const float v = load(x, i);
        if (pair_of(key_of(v), i) > mid) before += weight(v);
      }
      if (block_sum(before, shf) < limit) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  const float least = at(min_p, r);
  float z = 0.f;
  uint64_t chosen = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float v = load(x, i);
    const uint64_t pair = pair_of(key_of(v), i);
    const float w = weight(v);
    if (pair == best || (pair >= cut && w >= least)) {
      z += w;
      const float score = __fadd_rn(__fdiv_rn(v, t), noise[r * noise_ld + i]);
      chosen = max(chosen, pair_of(key_of(score == score ? score : -INFINITY), i));
    }
  }
  z = block_sum(z, shf);
  chosen = block_max(chosen, sh64);
  if (threadIdx.x == 0) {
    const int i = static_cast<int>(kIndexMask - (chosen & kIndexMask));
    token[r] = i;
    if (logprob) {
      const float v = load(x, i);
      logprob[r] = (v == mx ? 0.f : __fdiv_rn(v - mx, t)) - logf(z);
    }
  }
}

template <typename T>
static cudaError_t launch(const Sample& a, cudaStream_t stream) {
  sample_kernel<T><<<static_cast<unsigned>(a.rows), kThreads, 0, stream>>>(
      static_cast<const T*>(a.logits), a.ld, a.noise, a.noise_ld, a.vocab, a.temperature, a.top_k, a.top_p, a.min_p, a.token,
      a.logprob);
  return cudaGetLastError();
}

cudaError_t launch_sample(const Sample& a, cudaStream_t stream) {
  return a.bf16 ? launch<__nv_bfloat16>(a, stream) : launch<float>(a, stream);
}

}  // namespace sampling

}  // namespace mnb
