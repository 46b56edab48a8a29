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
// One block of 512 threads per row, two or three blocks per SM so that one
// row's loads run under another's arithmetic; every pass reads the row in
// 16-byte pieces, after the first one from L2.  No pass sorts the row:
//   - pass 1 finds the maximum.  Greedy rows end there.
//   - rows without top-k and top-p need one more pass (sum and best score).
//   - a small top-k takes the k-th largest of the threads' own maxima as a
//     bound: at least k tokens reach it, and few more do.  Pass 2 lists them,
//     and the list is sorted, summed and searched on its own.
//   - otherwise pass 2 counts the row in 2048 bins of the log-weight.  The
//     counts bound the mass above every bin from both sides, which leaves a
//     narrow band of weights that the cut can be in.  Pass 3 sums what lies
//     above the band, scores it, and lists the band; the sorted list gives the
//     exact cut.  A band with too many tokens is counted again in finer bins.
//   - what is left (thousands of equal logits at the cut, infinite logits) is
//     found by bisection over the pairs, slowly.
// Weights and sums are fp32, in a fixed order, so results do not depend on
// scheduling; the scores are IEEE fp32 division and addition.
#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace sampling {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;        // tokens a list can hold
constexpr int kSmallK = 384;       // top-k by the threads' maxima: 3/4 of the threads bound about 1.4 x 512 tokens
constexpr float kRange = 36.f;     // bins cover weights down to 2^-36 of the largest
constexpr int kLevels = 3;         // times a band is divided
constexpr uint32_t kIndexMask = (1u << kIndexBits) - 1;

// Order-preserving integer of a float; NaN sorts below -inf, -0 equals +0.
MNB_DEVICE uint32_t key_of(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
MNB_DEVICE float value_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key); }
constexpr uint32_t kKeyNegInf = 0x007fffffu;
// (logit, index) as one integer: larger comes first in the row's order.
MNB_DEVICE uint64_t pair_of(uint32_t key, int i) {
  return (static_cast<uint64_t>(key) << kIndexBits) | (kIndexMask - static_cast<uint32_t>(i));
}
MNB_DEVICE int index_of(uint64_t pair) { return static_cast<int>(kIndexMask - (static_cast<uint32_t>(pair) & kIndexMask)); }
MNB_DEVICE float logit_of(uint64_t pair) { return value_of(static_cast<uint32_t>(pair >> kIndexBits)); }

// One value for all rows, or one for each.
template <typename S>
MNB_DEVICE auto at(const S& s, int r) {
  return s.each ? s.each[r] : s.all;
}

struct Shared {
  union {
    uint64_t u64[kWarps];
    float f32[kWarps];
    int i32[kWarps];
  } red;
  int n_list;
  int bin_from, bin_to, bin_count;
  uint64_t cut;
  int hist[kBins];
  uint64_t list[kList];
};

template <typename V, typename F>
MNB_DEVICE V block_reduce(V v, V* sh, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  V s = sh[threadIdx.x % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) s = f(s, __shfl_xor_sync(0xffffffffu, s, o));
  __syncthreads();
  return s;
}
MNB_DEVICE float block_sum(float v, Shared& sh) {
  return block_reduce(v, sh.red.f32, [](float a, float b) { return a + b; });
}
MNB_DEVICE int block_sum(int v, Shared& sh) {
  return block_reduce(v, sh.red.i32, [](int a, int b) { return a + b; });
}
MNB_DEVICE float block_max(float v, Shared& sh) {
  return block_reduce(v, sh.red.f32, [](float a, float b) { return fmaxf(a, b); });
}
MNB_DEVICE uint64_t block_max(uint64_t v, Shared& sh) {
  return block_reduce(v, sh.red.u64, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
// Sum over the threads before this one.
template <typename V>
MNB_DEVICE V block_before(V v, V* sh) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  V x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  V base = 0;
  for (int i = 0; i < warp; ++i) base += sh[i];
  __syncthreads();
  return base + (x - v);
}

// A row read in 16-byte pieces.  The first and last piece may reach past the
// row; elements outside it read as NaN, which no filter keeps.
template <typename T>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  int V, lead, pieces;
  MNB_DEVICE Row(const T* p, int n) : x(p), V(n) {
    lead = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    pieces = (n + lead + kVec - 1) / kVec;
  }
  MNB_DEVICE float one(int i) const;
  MNB_DEVICE void piece(int c, float* v) const {
    const int i0 = c * kVec - lead;
    if (i0 >= 0 && i0 + kVec <= V) {
      const uint4 w = *reinterpret_cast<const uint4*>(x + i0);
      unpack(w, v);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = i0 + j >= 0 && i0 + j < V ? one(i0 + j) : __uint_as_float(0x7fc00000u);
    }
  }
  MNB_DEVICE static void unpack(uint4 w, float* v);
  // f(values, index of the first) over the thread's pieces
  template <typename F>
  MNB_DEVICE void scan(F f) const {
#pragma unroll 2
    for (int c = threadIdx.x; c < pieces; c += kThreads) {
      float v[kVec];
      piece(c, v);
      f(v, c * kVec - lead);
    }
  }
};
template <>
MNB_DEVICE float Row<float>::one(int i) const { return x[i]; }
template <>
MNB_DEVICE float Row<__nv_bfloat16>::one(int i) const { return bf16_to_f32(x[i]); }
template <>
MNB_DEVICE void Row<float>::unpack(uint4 w, float* v) {
  v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}
template <>
MNB_DEVICE void Row<__nv_bfloat16>::unpack(uint4 w, float* v) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(a[j] << 16);
    v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
  }
}

// The best score so far of the tokens that a thread has seen.
struct Best {
  float t, inv_t, score = -INFINITY;
  int index = -1;
  const float* noise;
  MNB_DEVICE void see(float v, float g, int i) {
    // the division is only needed where the product, good to 2^-22 of either term, comes near the best
    const float a = v * inv_t;
    if (index >= 0 && a + g < score - 1e-6f * (fabsf(a) + fabsf(g))) return;
    float s = __fadd_rn(__fdiv_rn(v, t), g);
    if (s != s) s = -INFINITY;
    if (index < 0 || s > score || (s == score && i < index)) score = s, index = i;
  }
  MNB_DEVICE uint64_t pair() const { return index < 0 ? 0 : pair_of(key_of(score), index); }
};

// The list in descending order (bitonic, n <= kList, one compare per thread and step).
MNB_DEVICE int sort_list(Shared& sh, int n) {
  int n2 = 32;
  while (n2 < n) n2 <<= 1;
  for (int i = n + threadIdx.x; i < n2; i += kThreads) sh.list[i] = 0;
  __syncthreads();
  const bool one_warp = n2 <= 64;  // only warp 0 has work: its steps need no block barrier
  if (!one_warp || threadIdx.x < 32) {
    for (int size = 2; size <= n2; size <<= 1)
      for (int stride = size / 2; stride > 0; stride >>= 1) {
        if (threadIdx.x < n2 / 2) {
          const int i = 2 * threadIdx.x - (threadIdx.x & (stride - 1)), j = i + stride;
          const uint64_t a = sh.list[i], b = sh.list[j];
          if ((a < b) == ((i & size) == 0)) sh.list[i] = b, sh.list[j] = a;
        }
        if (one_warp) __syncwarp();
        else __syncthreads();
      }
  }
  __syncthreads();
  return n2;
}

// Bisection over the pairs: right for every row, some 50 passes.
template <typename T>
__device__ __noinline__ uint64_t slow_cut(const Row<T>& row, float mx, float scale, int k, float p, Shared& sh) {
  auto weight = [&](float v) { return v == mx ? 1.f : ex2_approx((v - mx) * scale); };  // an infinite maximum takes all
  uint64_t best = 0;
  row.scan([&](const float* v, int i0) {
#pragma unroll
    for (int j = 0; j < Row<T>::kVec; ++j)
      if (v[j] == mx) best = max(best, pair_of(key_of(v[j]), i0 + j));
  });
  best = block_max(best, sh);
  uint64_t cut = static_cast<uint64_t>(kKeyNegInf + 1) << kIndexBits;
  if (k > 0 && k < row.V) {
    uint64_t lo = cut, hi = best;  // smallest pair with fewer than k before it
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      int n = 0;
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < Row<T>::kVec; ++j) n += v[j] == v[j] && pair_of(key_of(v[j]), i0 + j) > mid;
      });
      if (block_sum(n, sh) < k) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  if (p < 1.f) {
    auto mass = [&](uint64_t from) {  // of the pairs above `from`
      float s = 0.f;
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < Row<T>::kVec; ++j)
          if (v[j] == v[j] && pair_of(key_of(v[j]), i0 + j) > from) s += weight(v[j]);
      });
      return block_sum(s, sh);
    };
    const float limit = p * mass(cut - 1);
    uint64_t lo = cut, hi = best;  // smallest pair with less than the limit before it
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      if (mass(mid) < limit) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  return cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ Sample a) {
  constexpr int kVec = Row<T>::kVec;
  __shared__ Shared sh;
  const int r = blockIdx.x, tid = threadIdx.x;
  const Row<T> row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab);

  float mine = -INFINITY;
  row.scan([&](const float* v, int) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) mine = fmaxf(mine, v[j]);
  });
  const float mx = block_max(mine, sh);
  const float t = at(a.temperature, r);
  if (mx == -INFINITY || !(t > 0.f)) {  // no token left, or the first one
    uint64_t first = 0;
    if (mx != -INFINITY)
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (v[j] == mx) first = max(first, pair_of(1, i0 + j));
      });
    first = block_max(first, sh);
    if (tid == 0) {
      a.token[r] = first ? index_of(first) : -1;
      if (a.logprob) a.logprob[r] = first ? 0.f : -INFINITY;
    }
    return;
  }
  const float scale = 1.4426950408889634f / t;  // weights are 2^-y, y = (max - x) scale
  const float p = at(a.top_p, r), least = fminf(at(a.min_p, r), 1.f);
  int k = at(a.top_k, r);
  if (k <= 0 || k >= a.vocab) k = 0;
  Best best;
  best.t = t, best.inv_t = 1.f / t;
  best.noise = a.noise + r * a.noise_ld;
  float z = 0.f;  // weight of the kept tokens that this thread has seen

  // Keeps the elements of a piece that `kept` accepts and that pass min-p.
  const bool noise_vec = (reinterpret_cast<uintptr_t>(best.noise - row.lead) & 15) == 0;
  auto keep = [&](const float* v, int i0, auto kept) {
    float w[kVec];
    bool any = false;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      w[j] = -1.f;
      if (kept(v[j], i0 + j)) {
        const float x = v[j] == mx ? 1.f : ex2_approx((v[j] - mx) * scale);
        if (x >= least) w[j] = x, any = true;
      }
    }
    if (!any) return;
    float g[kVec];
    if (noise_vec && i0 >= 0 && i0 + kVec <= a.vocab) {
#pragma unroll
      for (int j = 0; j < kVec; j += 4) *reinterpret_cast<float4*>(g + j) = *reinterpret_cast<const float4*>(best.noise + i0 + j);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) g[j] = w[j] >= 0.f ? best.noise[i0 + j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if (w[j] >= 0.f) {
        z += w[j];
        best.see(v[j], g[j], i0 + j);
      }
  };
  auto finish = [&]() {
    const uint64_t chosen = block_max(best.pair(), sh);
    const float total = block_sum(z, sh);
    if (tid == 0) {
      const int i = index_of(chosen);
      a.token[r] = i;
      if (a.logprob) {
        const float v = row.one(i);
        a.logprob[r] = (v == mx ? 0.f : __fdiv_rn(v - mx, t)) - logf(total);
      }
    }
  };

  const bool cut_by_mass = p < 1.f;
  if (!k && !cut_by_mass) {
    row.scan([&](const float* v, int i0) { keep(v, i0, [&](float x, int) { return x > -INFINITY; }); });
    finish();
    return;
  }

  uint64_t cut = static_cast<uint64_t>(kKeyNegInf + 1) << kIndexBits;
  bool settled = false;
  if (mx < INFINITY && scale < 1e30f) {
    if (k && (k <= kSmallK || a.vocab <= kList)) {
      // the bound: the k-th largest of the threads' maxima, or a little less
      uint32_t lo = kKeyNegInf + 1;
      if (a.vocab > kList) {
        const uint32_t key = key_of(mine);
        uint32_t hi = key_of(mx);
        while (lo < hi) {  // the largest bound that at least k maxima reach
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          const int n = __syncthreads_count(key >= mid);
          if (n >= k) {
            lo = mid;
            if (n <= k + k / 8) break;
          } else {
            hi = mid - 1;
          }
        }
      }
      const float bound = value_of(lo);
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (v[j] >= bound) {
            const int n = atomicAdd(&sh.n_list, 1);
            if (n < kList) sh.list[n] = pair_of(key_of(v[j]), i0 + j);
          }
      });
      __syncthreads();
      const int n = sh.n_list;
      if (n <= kList) {
        sort_list(sh, n);
        const int have = min(n, k);
        // two neighbouring places per thread
        float w[2], sum = 0.f;
        uint64_t pair[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * tid + e;
          pair[e] = i < have ? sh.list[i] : 0;
          const float v = logit_of(pair[e]);
          w[e] = i < have ? (v == mx ? 1.f : ex2_approx((v - mx) * scale)) : 0.f;
          sum += w[e];
        }
        float before = block_before(sum, sh.red.f32);
        const float limit = cut_by_mass ? p * block_sum(sum, sh) : INFINITY;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * tid + e;
          if (i < have && (i == 0 || before < limit) && w[e] >= least) {
            z += w[e];
            best.see(logit_of(pair[e]), best.noise[index_of(pair[e])], index_of(pair[e]));
          }
          before += w[e];
        }
        finish();
        return;
      }
    }
    // Count and mass bands: first the cut of top-k (if any), then that of top-p.
    bool ok = true;
    float limit = 0.f;
    for (int stage = k ? 0 : 1; stage < (cut_by_mass ? 2 : 1) && ok; ++stage) {
      const bool by_mass = stage == 1, last = by_mass || !cut_by_mass;
      const bool filtered = by_mass && k;  // only what top-k left
      float y0 = 0.f, y1 = kRange;
      ok = false;
      for (int level = 0; level < kLevels && !ok; ++level) {
        for (int b = tid; b < kBins; b += kThreads) sh.hist[b] = 0;
        __syncthreads();
        const float per = kBins / (y1 - y0);
        float mass = 0.f;  // level 0: of everything; later: of what lies above the band
        int above = 0;
        row.scan([&](const float* v, int i0) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const float y = (mx - v[j]) * scale;
            if (filtered && !(v[j] > -INFINITY && pair_of(key_of(v[j]), i0 + j) >= cut)) continue;
            if (level == 0) {
              if (by_mass && v[j] > -INFINITY) mass += ex2_approx(-y);
            } else if (y < y0) {
              ++above;
              if (by_mass) mass += ex2_approx(-y);
            }
            if (y >= y0 && y <= y1) {
              // adding 2^23 leaves the bin, rounded to the nearest, in the low bits
              const float b = fminf(fmaxf((y - y0) * per, 0.f), kBins - 1.f) + 8388608.f;
              atomicAdd(&sh.hist[__float_as_uint(b) & (kBins - 1)], 1);
            }
          }
        });
        mass = block_sum(mass, sh);
        if (!by_mass && level) above = block_sum(above, sh);
        if (by_mass && level == 0) limit = p * mass;
        // this thread's bins, in order
        constexpr int kPer = kBins / kThreads;
        const float head = level ? mass : 0.f;
        int c[kPer], sum_c = 0;
        float sum_hi = 0.f, sum_lo = 0.f;  // with every token at the bin's upper / lower weight
        const float step = 1.f / per;
        auto upper = [&](int b) { return ex2_approx(-(y0 + (b - 0.5f) * step)); };
        auto lower = [&](int b) { return ex2_approx(-(y0 + (b + (b == kBins - 1 ? 1.f : 0.5f)) * step)); };
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int b = tid * kPer + e;
          c[e] = sh.hist[b];
          sum_c += c[e];
          sum_hi += c[e] * upper(b);
          sum_lo += c[e] * lower(b);
        }
        if (tid == 0) sh.bin_from = kBins, sh.bin_to = kBins, sh.bin_count = 0;
        int n = block_before(sum_c, sh.red.i32);
        if (!by_mass) {
          n += level ? above : 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (n < k && n + c[e] >= k) sh.bin_from = sh.bin_to = tid * kPer + e, sh.bin_count = c[e];
            n += c[e];
          }
          __syncthreads();
        } else {
          float hi = head + block_before(sum_hi, sh.red.f32), lo = head + block_before(sum_lo, sh.red.f32);
          // from the other end too: behind a bin lie at most the upper weights of the later bins and of what no bin counts
          const float all_hi = block_sum(sum_hi, sh);
          float behind = level == 0 ? all_hi - (hi - head) + a.vocab * ex2_approx(-kRange) : INFINITY;
          const float all = level == 0 ? mass * (1.f - 2e-6f) : 0.f;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int b = tid * kPer + e;
            hi += c[e] * upper(b);
            lo += c[e] * lower(b);
            behind -= c[e] * upper(b);
            if (c[e] && hi >= limit * (1.f - 1e-5f)) atomicMin(&sh.bin_from, b);
            if (c[e] && (lo >= limit * (1.f + 1e-5f) || all - behind * (1.f + 1e-4f) >= limit * (1.f + 1e-5f)))
              atomicMin(&sh.bin_to, b);
          }
          __syncthreads();
          if (sh.bin_to == kBins && tid == 0) sh.bin_to = kBins - 1;
          __syncthreads();
          int inside = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int b = tid * kPer + e;
            if (b >= sh.bin_from && b <= sh.bin_to) inside += c[e];
          }
          inside = block_sum(inside, sh);
          if (tid == 0) sh.bin_count = inside;
          __syncthreads();
        }
        const int from = sh.bin_from, to = sh.bin_to, count = sh.bin_count;
        __syncthreads();
        if (from >= kBins) break;  // the cut lies below the range
        const float wide = 1e-6f * (y0 + to * step) + 1e-6f * step;
        y1 = to == kBins - 1 ? y1 : y0 + (to + 0.5f) * step + wide;
        y0 = fmaxf(y0, y0 + (from - 0.5f) * step - wide);
        ok = count <= kList - kList / 8;  // the widened edges may let a few more in
      }
      if (!ok) break;
      // what lies above the band, and the band itself as a list
      if (tid == 0) sh.n_list = 0;
      __syncthreads();
      float mass = 0.f;
      int above = 0;
      auto inside = [&](float x, int i) {
        return x > -INFINITY && !(filtered && pair_of(key_of(x), i) < cut);
      };
      row.scan([&](const float* v, int i0) {
        bool any = false;
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float y = (mx - v[j]) * scale;
          if (!(y <= y1) || !inside(v[j], i0 + j)) continue;
          if (y < y0) {
            any = true;
            ++above;
            if (cut_by_mass) mass += ex2_approx(-y);
          } else {
            const int n = atomicAdd(&sh.n_list, 1);
            if (n < kList) sh.list[n] = pair_of(key_of(v[j]), i0 + j);
          }
        }
        if (last && any)
          keep(v, i0, [&](float x, int i) { return (mx - x) * scale < y0 && inside(x, i); });
      });
      mass = block_sum(mass, sh);
      above = block_sum(above, sh);
      const int n = sh.n_list;
      __syncthreads();
      if (n > kList) {
        ok = false;
        break;
      }
      sort_list(sh, n);
      float w[2], sum = 0.f;
      uint64_t pair[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        pair[e] = i < n ? sh.list[i] : 0;
        const float v = logit_of(pair[e]);
        w[e] = i < n ? (v == mx ? 1.f : ex2_approx((v - mx) * scale)) : 0.f;
        sum += w[e];
      }
      float before = mass + block_before(sum, sh.red.f32);
      const float total = mass + block_sum(sum, sh);
      // The first token that goes has to be in the list, and the tokens above it have to stay.
      if (by_mass ? !(mass < limit || above == 0) || !(total >= limit * (1.f - 1e-6f)) : !(above < k && above + n >= k)) {
        ok = false;
        break;
      }
      if (tid == 0) sh.cut = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        const bool stays = i < n && (by_mass ? before < limit || above + i == 0 : above + i < k);
        if (stays && last && w[e] >= least) {
          z += w[e];
          best.see(logit_of(pair[e]), best.noise[index_of(pair[e])], index_of(pair[e]));
        }
        if (!by_mass && above + i == k - 1 && i < n) sh.cut = pair[e];
        before += w[e];
      }
      __syncthreads();
      if (!last) cut = sh.cut;
      __syncthreads();
    }
    settled = ok;
  }
  if (!settled) {
    z = 0.f;
    best.index = -1, best.score = -INFINITY;
    cut = slow_cut(row, mx, scale, k, p, sh);
    row.scan([&](const float* v, int i0) {
      keep(v, i0, [&](float x, int i) { return x == x && pair_of(key_of(x), i) >= cut; });
    });
  }
  finish();
}

template <typename T>
static cudaError_t launch(const Sample& a, cudaStream_t stream) {
  sample_kernel<T><<<static_cast<unsigned>(a.rows), kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_sample(const Sample& a, cudaStream_t stream) {
  return a.bf16 ? launch<__nv_bfloat16>(a, stream) : launch<float>(a, stream);
}

}  // namespace sampling

}  // namespace mnb
