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
// A cluster of 1 to 8 blocks of 512 threads takes a row.  Each block brings
// its slice of the row into shared memory once, by bulk copies, and the passes
// below read it there; block results meet through distributed shared memory.
// No pass sorts the row:
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
//     found by bisection over the pairs, slowly: 1 x 50304 bf16 around 20 with
//     a spread of 1, top-p 0.9, 167 us where the same around 0 takes 22.
// Measured (GPU time): 1 x 50304 bf16, top-k 50: 11 us; 64 x 50304 fp32 with
// mixed settings 27 us; 512 x 50304 bf16, top-p 0.9 to 0.95: 80 us (52 MB of
// logits and about as much noise); 129 x 130003 fp32, min-p: 43 us (67 MB).
// None is bound by its bytes: a row is a chain of passes, and the instructions
// of the passes (12 an element to count, 13 to split, 11 to score) fill the
// issue slots of the two blocks that share an SM.  A row's blocks exchange
// values four to eight times at about a microsecond each, so where
// rows fill the GPU each gets the fewest blocks that hold it: 512 rows of 50304 in clusters of 1, 2, 4 and 8
// blocks took 112, 171, 298 and 562 us.
// Weights and sums are fp32, in a fixed order, so results do not depend on
// scheduling; the winning score is IEEE fp32 division and addition.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "generation.h"
#include "launch.cuh"

namespace mnb {

namespace sampling {

namespace cg = cooperative_groups;

constexpr int kMaxCluster = 8;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;        // tokens a list can hold
constexpr int kPlaces = kList / kThreads;
constexpr int kSmallK = 3 * kThreads / 4;  // top-k by the threads' maxima: those of one block bound about 1.4 x 512 tokens
constexpr int kMostK = 600;                // more maxima than 512 bound under 700 tokens then, which a list holds
constexpr int kChunk = 2 * kThreads;       // pieces of 16 bytes per bulk copy
constexpr int kChunks = 14;
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

template <bool B>
struct Flag {
  static constexpr bool value = B;
};

// One value for all rows, or one for each.
template <typename S>
MNB_DEVICE auto at(const S& s, int r) {
  return s.each ? s.each[r] : s.all;
}

// A block on its own counts and lists in place; the blocks of a cluster have parts of their own.
template <bool Multi>
struct Lists;
template <>
struct Lists<false> {
  union {
    int hist[kBins];
    uint64_t list[kList];
  };
  MNB_DEVICE int* bins() { return hist; }
  MNB_DEVICE uint64_t* mine() { return list; }
};
template <>
struct Lists<true> {
  uint64_t part[kList];
  union {
    float maxima[kMaxCluster][kThreads];
    struct {
      int counts[kBins];
      int hist[kBins];
    };
    uint64_t list[kList];
  };
  MNB_DEVICE int* bins() { return counts; }
  MNB_DEVICE uint64_t* mine() { return part; }
};

template <bool Multi>
struct Shared : Lists<Multi> {
  union {
    uint64_t u64[kWarps];
    float f32[kWarps];
    int i32[kWarps];
    struct {
      int n[kWarps];
      float hi[kWarps], lo[kWarps];
    } sums;
  } red;
  uint64_t from[2][kMaxCluster];  // one value of every block of the cluster, in turn in two places
  uint64_t from_too[2][kMaxCluster];
  int counted[2][kWarps];         // warps' counts, in turn in two places
  uint64_t joined[2];             // mbarriers of these exchanges
  uint64_t arrived[kChunks];      // mbarriers of the bulk copies
  int n_mine;
  int bin_from, bin_to, bin_count;
  uint64_t cut;
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
// The sum with one barrier; the next call takes other places.
MNB_DEVICE int block_count(int n, int* sh) {
  n = __reduce_add_sync(0xffffffffu, n);
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = n;
  __syncthreads();
  const int lane = threadIdx.x % 32;
  return __reduce_add_sync(0xffffffffu, lane < kWarps ? sh[lane] : 0);
}
// The same over the cluster: every block sends its value to all by asynchronous remote stores, which the receivers'
// mbarriers count, and joins what it got in the blocks' order.
template <bool Multi>
struct Team {
  Shared<Multi>& sh;
  int size, rank;
  int* status;
  int exchanges = 0;
  // everything written to shared memory before is there for every block after
  MNB_DEVICE void sync() const {
    if (Multi) cg::this_cluster().sync();
    else __syncthreads();
  }
  template <typename T>
  MNB_DEVICE T* peer(T* p, int q) const {
    return Multi ? cg::this_cluster().map_shared_rank(p, q) : p;
  }
  MNB_DEVICE static uint64_t bits(float v) { return __float_as_uint(v); }
  MNB_DEVICE static uint64_t bits(int v) { return static_cast<uint32_t>(v); }
  MNB_DEVICE static uint64_t bits(uint64_t v) { return v; }
  MNB_DEVICE static void of_bits(uint64_t b, float& v) { v = __uint_as_float(static_cast<uint32_t>(b)); }
  MNB_DEVICE static void of_bits(uint64_t b, int& v) { v = static_cast<int>(static_cast<uint32_t>(b)); }
  MNB_DEVICE static void of_bits(uint64_t b, uint64_t& v) { v = b; }
  // 8 bytes to the same place in block q, counted by its mbarrier
  MNB_DEVICE static void send(uint64_t* place, uint64_t v, uint32_t bar, int q) {
    uint32_t to, to_bar;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(place)), "r"(q));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to_bar) : "r"(bar), "r"(q));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(v), "r"(to_bar)
                 : "memory");
  }
  // Until every block's values are there.  Not given up because another wait of the device has run out: the blocks of a
  // cluster have to agree on every value, or one would end while another still reads its memory.
  MNB_DEVICE void receive(uint32_t bar) {
    if (!mbar_wait(bar, (exchanges >> 1) & 1, nullptr)) atomicCAS(status, 0, kErrPipelineTimeout);
    ++exchanges;
  }
  template <typename V, typename F>
  MNB_DEVICE V join(V v, V* red, F f) {
    v = block_reduce(v, red, f);
    if (!Multi) return v;
    const int turn = exchanges & 1;
    const uint32_t bar = smem_u32(sh.joined + turn);
    if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, 8 * size);
    if (threadIdx.x < size) send(&sh.from[turn][rank], bits(v), bar, threadIdx.x);
    receive(bar);
    V s, x;
    of_bits(*const_cast<volatile uint64_t*>(&sh.from[turn][0]), s);
    for (int q = 1; q < size; ++q) {
      of_bits(*const_cast<volatile uint64_t*>(&sh.from[turn][q]), x);
      s = f(s, x);
    }
    return s;
  }
  MNB_DEVICE float sum(float v) {
    return join(v, sh.red.f32, [](float a, float b) { return a + b; });
  }
  MNB_DEVICE int sum(int v) {
    return join(v, sh.red.i32, [](int a, int b) { return a + b; });
  }
  MNB_DEVICE float max(float v) {
    return join(v, sh.red.f32, [](float a, float b) { return fmaxf(a, b); });
  }
  MNB_DEVICE uint64_t max(uint64_t v) {
    return join(v, sh.red.u64, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
  }
  // The largest `best` and the sum of `z` of all threads, in one exchange.
  MNB_DEVICE uint64_t max_and_sum(uint64_t best, float* z) {
    best = block_reduce(best, sh.red.u64, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    *z = block_reduce(*z, sh.red.f32, [](float a, float b) { return a + b; });
    if (!Multi) return best;
    const int turn = exchanges & 1;
    const uint32_t bar = smem_u32(sh.joined + turn);
    if (threadIdx.x == 0) mbar_arrive_expect_tx(bar, 16 * size);
    if (threadIdx.x < size) {
      send(&sh.from[turn][rank], best, bar, threadIdx.x);
      send(&sh.from_too[turn][rank], bits(*z), bar, threadIdx.x);
    }
    receive(bar);
    *z = 0.f;
    for (int q = 0; q < size; ++q) {
      best = ::max(best, *const_cast<volatile uint64_t*>(&sh.from[turn][q]));
      float x;
      of_bits(*const_cast<volatile uint64_t*>(&sh.from_too[turn][q]), x);
      *z += x;
    }
    return best;
  }
  // The blocks' lists into everybody's `list`; returns the length, more than kList if they do not fit.
  // The next change of a part has to lie behind another sync().
  MNB_DEVICE int gather_list() {
    sync();
    if (!Multi) return sh.n_mine;
    int n = 0;
    for (int q = 0; q < size; ++q) {
      const int m = *peer(&sh.n_mine, q);
      const uint64_t* from = peer(sh.mine(), q);
      if (n + m <= kList)
        for (int i = threadIdx.x; i < m; i += kThreads) sh.list[n + i] = from[i];
      n += m;
    }
    __syncthreads();
    return n;
  }
};
// Sums over the threads before this one, and over all.
struct Sums {
  int n;
  float hi, lo;
};
template <typename S>
MNB_DEVICE Sums sums_before(Sums v, S& sh, Sums* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto scan = [&](auto x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const auto y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const Sums x{scan(v.n), scan(v.hi), scan(v.lo)};
  if (lane == 31) sh.red.sums.n[warp] = x.n, sh.red.sums.hi[warp] = x.hi, sh.red.sums.lo[warp] = x.lo;
  __syncthreads();
  const bool in = lane < kWarps;
  const Sums w{in ? sh.red.sums.n[lane % kWarps] : 0, in ? sh.red.sums.hi[lane % kWarps] : 0.f,
               in ? sh.red.sums.lo[lane % kWarps] : 0.f};
  const Sums p{scan(w.n), scan(w.hi), scan(w.lo)};
  auto at = [](auto x, int i) { return __shfl_sync(0xffffffffu, x, i); };
  *total = {at(p.n, 31), at(p.hi, 31), at(p.lo, 31)};
  const Sums head{at(p.n, (warp + 31) % 32), at(p.hi, (warp + 31) % 32), at(p.lo, (warp + 31) % 32)};
  __syncthreads();
  // (x - v would lose what cancels: shift the scan by a lane instead)
  Sums before{__shfl_up_sync(0xffffffffu, x.n, 1), __shfl_up_sync(0xffffffffu, x.hi, 1), __shfl_up_sync(0xffffffffu, x.lo, 1)};
  if (lane == 0) before = {0, 0.f, 0.f};
  if (warp > 0) before = {before.n + head.n, before.hi + head.hi, before.lo + head.lo};
  return before;
}

MNB_DEVICE float to_float(float v) { return v; }
MNB_DEVICE float to_float(__nv_bfloat16 v) { return bf16_to_f32(v); }
MNB_DEVICE void unpack_piece(uint4 w, float (&v)[4]) {
  v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
}
MNB_DEVICE void unpack_piece(uint4 w, float (&v)[8]) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(a[j] << 16);
    v[2 * j + 1] = __uint_as_float(a[j] & 0xffff0000u);
  }
}
MNB_DEVICE float widest_of(uint4 w, float m, float) {
  return max3f(max3f(__uint_as_float(w.x), __uint_as_float(w.y), m), __uint_as_float(w.z), __uint_as_float(w.w));
}
MNB_DEVICE float widest_of(uint4 w, float m, __nv_bfloat16) {
  auto pair = [](uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); };
  const __nv_bfloat162 a = __hmax2(__hmax2(pair(w.x), pair(w.y)), __hmax2(pair(w.z), pair(w.w)));
  return max3f(m, __low2float(a), __high2float(a));
}
MNB_DEVICE uint4 pack_piece(const float* x, int i0, int V) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = i0 + j >= 0 && i0 + j < V ? __float_as_uint(x[i0 + j]) : 0x7fc00000u;
  return make_uint4(w[0], w[1], w[2], w[3]);
}
MNB_DEVICE uint4 pack_piece(const __nv_bfloat16* x, int i0, int V) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = i0 + 2 * j;
    const uint32_t lo = i >= 0 && i < V ? __bfloat16_as_ushort(x[i]) : 0x7fc0u;
    const uint32_t hi = i + 1 >= 0 && i + 1 < V ? __bfloat16_as_ushort(x[i + 1]) : 0x7fc0u;
    w[j] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// This block's slice of a row, in 16-byte pieces.  The row's first and last
// piece may reach past it; elements outside read as NaN, which no filter keeps.
template <typename T, bool Staged>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  const T* x;
  int V, lead;
  int first, count;  // pieces
  uint4* slice;      // in shared memory, if Staged; otherwise every pass reads global memory (L2)
  MNB_DEVICE Row(const T* p, int n, int rank, int size, uint4* smem) : x(p), V(n), slice(smem) {
    lead = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    const int all = (n + lead + kVec - 1) / kVec, per = (all + size - 1) / size;
    first = min(all, rank * per);
    count = min(all - first, per);
  }
  MNB_DEVICE int start(int c) const { return (first + c) * kVec - lead; }  // element of piece c
  MNB_DEVICE bool whole(int c) const { return start(c) >= 0 && start(c) + kVec <= V; }
  // One thread starts the copies of the whole pieces; the thread that reads a row's edge fills it in.
  MNB_DEVICE void stage(uint64_t* arrived) const {
    if (!Staged || count == 0) return;
    const int from = whole(0) ? 0 : 1, to = whole(count - 1) ? count : count - 1;
    if (threadIdx.x == 0)
      for (int j = 0; j * kChunk < count; ++j) {
        const int a = max(j * kChunk, from), b = min((j + 1) * kChunk, to);
        const uint32_t bar = smem_u32(arrived + j), bytes = a < b ? static_cast<uint32_t>(b - a) * 16 : 0;
        mbar_arrive_expect_tx(bar, bytes);
        if (bytes) bulk_load(smem_u32(slice + a), x + start(a), bytes, bar);
      }
    if (from == 1 && threadIdx.x == 0) slice[0] = edge(start(0));
    if (to < count && count > from && (count - 1) % kThreads == threadIdx.x) slice[count - 1] = edge(start(count - 1));
  }
  MNB_DEVICE static void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
  }
  MNB_DEVICE uint4 piece(int c) const {
    if (Staged) return slice[c];
    return whole(c) ? *reinterpret_cast<const uint4*>(x + start(c)) : edge(start(c));
  }
  MNB_DEVICE float one(int i) const { return to_float(x[i]); }
  // the largest of m and the piece's elements (NaN does not count)
  MNB_DEVICE static float widest(uint4 w, float m) { return widest_of(w, m, T{}); }
  // a piece that reaches past the row
  MNB_DEVICE uint4 edge(int i0) const { return pack_piece(x, i0, V); }
  // f(values, index of the first) over the thread's pieces
  template <typename F>
  MNB_DEVICE void scan(F f) const {
#pragma unroll 2
    for (int c = threadIdx.x; c < count; c += kThreads) {
      float v[kVec];
      unpack_piece(piece(c), v);
      f(v, start(c));
    }
  }
  // f(values, noise, index of the first) over the pieces with an element of at least `least`.  The next piece's noise
  // is on its way while this one is worked on, in two sets of registers by turns (a copy from one to the other would
  // wait for the loads).
  template <typename F>
  MNB_DEVICE void scan_noise(float least, const float* noise, F f) const {
    const bool vec = (reinterpret_cast<uintptr_t>(noise - lead) & 15) == 0;
    constexpr int kUnit = 8 / kVec, kStep = kUnit * kThreads;  // pieces per turn: eight values
    auto fetch = [&](int c0, float (&g)[8]) {
      unsigned have = 0;
#pragma unroll
      for (int u = 0; u < kUnit; ++u) {
        const int c = c0 + u * kThreads;
        if (c >= count || !(widest(piece(c), -INFINITY) >= least)) continue;
        const int i0 = start(c);
        if (vec && whole(c)) {
#pragma unroll
          for (int j = 0; j < kVec; j += 4) {
            const float4 t = *reinterpret_cast<const float4*>(noise + i0 + j);
            float* to = g + u * kVec + j;
            to[0] = t.x, to[1] = t.y, to[2] = t.z, to[3] = t.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) g[u * kVec + j] = i0 + j >= 0 && i0 + j < V ? noise[i0 + j] : 0.f;
        }
        have |= 1u << u;
      }
      return have;
    };
    auto work = [&](int c0, const float (&g)[8], unsigned have) {
#pragma unroll
      for (int u = 0; u < kUnit; ++u) {
        if (!(have >> u & 1)) continue;
        const int c = c0 + u * kThreads;
        float v[kVec];
        unpack_piece(piece(c), v);
#pragma unroll
        for (int j = 0; j < kVec; j += 4) f(v + j, g + u * kVec + j, start(c) + j);  // four at a time: fewer values held at once
      }
    };
    float g0[8], g1[8];
    int c = threadIdx.x;
    unsigned have0 = fetch(c, g0), have1;
    while (c < count) {
      have1 = fetch(c + kStep, g1);
      work(c, g0, have0);
      have0 = fetch(c + 2 * kStep, g0);
      work(c + kStep, g1, have1);
      c += 2 * kStep;
    }
  }
  // f(values, index of the first) over those pieces
  template <typename F>
  MNB_DEVICE void scan_from(float least, F f) const {
#pragma unroll 4
    for (int c = threadIdx.x; c < count; c += kThreads) {
      const uint4 w = piece(c);
      if (!(widest(w, -INFINITY) >= least)) continue;
      float v[kVec];
      unpack_piece(w, v);
      f(v, start(c));
    }
  }
};
// v / t, rounded as IEEE division rounds it, from the reciprocal inv_t = 1 / t (itself rounded to nearest): two
// steps q += (v - q t) inv_t with the remainder exact by fused multiply-add, after which the quotient is the correctly
// rounded one (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990).  Where
// a step could overflow, underflow or meet an infinity the division itself is called.
MNB_DEVICE float divide(float v, float t, float inv_t) {
  float q = v * inv_t;
  q = fmaf(fmaf(-q, t, v), inv_t, q);
  q = fmaf(fmaf(-q, t, v), inv_t, q);
  const float m = fabsf(q);
  if (!(m > 1e-25f && m < 1e25f)) q = __fdiv_rn(v, t);
  return q;
}

// The best score so far of the tokens that a thread has seen.
struct Best {
  float t, inv_t, score = -INFINITY;
  int index = -1;
  const float* noise;
  MNB_DEVICE void see(float v, float g, int i) {
    float s = __fadd_rn(divide(v, t, inv_t), g);
    s = s != s ? -INFINITY : s;
    const bool better = s > score || index < 0 || (s == score && i < index);
    score = better ? s : score;
    index = better ? i : index;
  }
  MNB_DEVICE uint64_t pair() const { return index < 0 ? 0 : pair_of(key_of(score), index); }
};

// Puts the n <= kList pairs of the list in descending order; the log-weights lie between y0 and y1.  A counting sort by
// finer bins of the log-weight, after which each pair is ranked among those of its own bin.  (The list and the counts
// may share their memory: the pairs wait in registers.)
template <typename S>
MNB_DEVICE void sort_list(S& sh, int n, float mx, float scale, float y0, float y1) {
  const float per = y1 > y0 ? kBins / (y1 - y0) : 0.f;
  uint64_t pair[kPlaces];
  int bin[kPlaces], start[kPlaces], end[kPlaces], slot[kPlaces];
#pragma unroll
  for (int e = 0; e < kPlaces; ++e) {
    const int i = threadIdx.x + e * kThreads;
    pair[e] = i < n ? sh.list[i] : 0;
    const float y = (mx - logit_of(pair[e])) * scale;
    bin[e] = static_cast<int>(fminf(fmaxf((y - y0) * per, 0.f), kBins - 1.f));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e)
    if (pair[e]) atomicAdd(sh.hist + bin[e], 1);
  __syncthreads();
  constexpr int kPer = kBins / kThreads;
  int c[kPer], sum = 0;
#pragma unroll
  for (int e = 0; e < kPer; ++e) sum += c[e] = sh.hist[threadIdx.x * kPer + e];
  Sums all;
  int at = sums_before(Sums{sum, 0.f, 0.f}, sh, &all).n;
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    sh.hist[threadIdx.x * kPer + e] = at;
    at += c[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e) {
    start[e] = sh.hist[bin[e]];
    end[e] = bin[e] + 1 < kBins ? sh.hist[bin[e] + 1] : n;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e) slot[e] = pair[e] ? atomicAdd(sh.hist + bin[e], 1) : 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e)
    if (pair[e]) sh.list[slot[e]] = pair[e];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e) {
    slot[e] = start[e];
    if (pair[e])
      for (int i = start[e]; i < end[e]; ++i) slot[e] += sh.list[i] > pair[e];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kPlaces; ++e)
    if (pair[e]) sh.list[slot[e]] = pair[e];
  __syncthreads();
}

// Bisection over the pairs: right for every row, some 50 passes.
// (By value: a reference would keep the row and the team in memory, not in registers, wherever the kernel uses them.)
struct Cut {
  uint64_t pair;
  int exchanges;
};
template <typename T, bool Staged, bool Multi>
__device__ __noinline__ Cut slow_cut(Row<T, Staged> row, float mx, float scale, int k, float p, Team<Multi> team) {
  auto weight = [&](float v) { return v == mx ? 1.f : ex2_approx((v - mx) * scale); };  // an infinite maximum takes all
  uint64_t best = 0;
  row.scan([&](const float* v, int i0) {
#pragma unroll
    for (int j = 0; j < Row<T, Staged>::kVec; ++j)
      if (v[j] == mx) best = max(best, pair_of(key_of(v[j]), i0 + j));
  });
  best = team.max(best);
  uint64_t cut = static_cast<uint64_t>(kKeyNegInf + 1) << kIndexBits;
  if (k > 0 && k < row.V) {
    uint64_t lo = cut, hi = best;  // smallest pair with fewer than k before it
    while (lo < hi) {
      const uint64_t mid = lo + (hi - lo) / 2;
      int n = 0;
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < Row<T, Staged>::kVec; ++j) n += v[j] == v[j] && pair_of(key_of(v[j]), i0 + j) > mid;
      });
      if (team.sum(n) < k) hi = mid;
      else lo = mid + 1;
    }
    cut = lo;
  }
  if (p < 1.f) {
    auto mass = [&](uint64_t from) {  // of the pairs above `from`
      float s = 0.f;
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < Row<T, Staged>::kVec; ++j)
          if (v[j] == v[j] && pair_of(key_of(v[j]), i0 + j) > from) s += weight(v[j]);
      });
      return team.sum(s);
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
  return {cut, team.exchanges};
}

template <typename T, bool Staged, bool Multi>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ Sample a, int cluster) {
  using R = Row<T, Staged>;
  constexpr int kVec = R::kVec;
  extern __shared__ uint4 slice[];
  __shared__ Shared<Multi> sh;
  const int r = blockIdx.x / cluster, tid = threadIdx.x;
  if (!Multi) cluster = 1;
  Team<Multi> team{sh, cluster, static_cast<int>(blockIdx.x) % cluster, a.status};
  const R row(static_cast<const T*>(a.logits) + r * a.ld, a.vocab, team.rank, cluster, slice);
  if (Staged || Multi) {
    if (tid == 0) {
      for (int j = 0; j < kChunks; ++j) mbar_init(smem_u32(sh.arrived + j), 1);
      for (int j = 0; j < 2; ++j) mbar_init(smem_u32(sh.joined + j), 1);
      fence_mbar_init();
    }
    __syncthreads();
    if (Multi) cg::this_cluster().barrier_arrive();  // this block runs and its mbarriers are there
    row.stage(sh.arrived);
  }

  float mine = -INFINITY;
  for (int c = tid, j = 0; c < row.count; ++j) {  // a chunk holds two of a thread's pieces
    // (not given up because another wait of the device has run out: a block may not end before its copies have)
    if (Staged && !mbar_wait(smem_u32(sh.arrived + j), 0, nullptr)) {
      atomicCAS(a.status, 0, kErrPipelineTimeout);
      break;
    }
#pragma unroll
    for (int e = 0; e < kChunk / kThreads; ++e, c += kThreads)
      if (c < row.count) mine = R::widest(row.piece(c), mine);
  }
  if (Multi) cg::this_cluster().barrier_wait();
  const float mx = team.max(mine);
  const float t = at(a.temperature, r);
  if (mx == -INFINITY || !(t > 0.f)) {  // no token left, or the first one
    uint64_t first = 0;
    if (mx != -INFINITY)
      row.scan([&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (v[j] == mx) first = max(first, pair_of(1, i0 + j));
      });
    first = team.max(first);
    if (tid == 0 && team.rank == 0) {
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
  // `z`, summed over the threads, is added to the weight of the kept
  auto finish = [&](float total, float z) {
    const uint64_t chosen = team.max_and_sum(best.pair(), &z);
    total += z;
    if (tid == 0 && team.rank == 0) {
      const int i = chosen ? index_of(chosen) : -1;  // (nothing: the row did not arrive in time, which is in the status word)
      a.token[r] = i;
      if (a.logprob) {
        const float v = i >= 0 ? row.one(i) : -INFINITY;
        a.logprob[r] = (v == mx ? 0.f : __fdiv_rn(v - mx, t)) - logf(total);
      }
    }
  };

  const bool cut_by_mass = p < 1.f;
  float total = 0.f;  // weight of what the cut keeps
  uint64_t cut = static_cast<uint64_t>(kKeyNegInf + 1) << kIndexBits;  // keeps all but -inf and NaN
  bool settled = !k && !cut_by_mass;
  if (!settled && mx < INFINITY && scale < 1e30f) {
    if (k && (k <= min(kSmallK * cluster, kMostK) || a.vocab <= kList)) {
      // the bound: the k-th largest of the threads' maxima, or a little less
      uint32_t lo = kKeyNegInf + 1;
      if (a.vocab > kList) {
        constexpr int kSets = Multi ? kMaxCluster : 1;
        uint32_t key[kSets];
        key[0] = key_of(mine);
        if constexpr (Multi) {  // every block gets all the maxima, so the search needs no further exchange
          for (int q = 0; q < cluster; ++q) team.peer(&sh.maxima[team.rank][tid], q)[0] = mine;
          team.sync();
#pragma unroll
          for (int q = 0; q < kSets; ++q) key[q] = q < cluster ? key_of(sh.maxima[q][tid]) : 0u;
        }
        uint32_t hi = key_of(mx);
        int turn = 0;
        while (lo < hi) {  // the largest bound that at least k maxima reach
          const uint32_t mid = lo + (hi - lo + 1) / 2;
          int n;
          if constexpr (Multi) {
            n = 0;
#pragma unroll
            for (int q = 0; q < kSets; ++q) n += key[q] >= mid;  // (mid is above the 0 of blocks that are not there)
            n = block_count(n, sh.counted[turn]);
            turn ^= 1;
          } else {
            n = __syncthreads_count(key[0] >= mid);
          }
          if (n >= k) {
            lo = mid;
            if (n <= k + k / 8) break;
          } else {
            hi = mid - 1;
          }
        }
      }
      const float bound = value_of(lo);
      if (tid == 0) sh.n_mine = 0;
      __syncthreads();
      row.scan_from(bound, [&](const float* v, int i0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (v[j] >= bound) {
            const int n = atomicAdd(&sh.n_mine, 1);
            if (n < kList) sh.mine()[n] = pair_of(key_of(v[j]), i0 + j);
          }
      });
      const int n = team.gather_list();
      if (n <= kList) {
        sort_list(sh, n, mx, scale, 0.f, (mx - bound) * scale);
        const int have = min(n, k);
        // neighbouring places per thread
        float w[kPlaces], sum = 0.f;
        uint64_t pair[kPlaces];
#pragma unroll
        for (int e = 0; e < kPlaces; ++e) {
          const int i = kPlaces * tid + e;
          pair[e] = i < have ? sh.list[i] : 0;
          const float v = logit_of(pair[e]);
          w[e] = i < have ? (v == mx ? 1.f : ex2_approx((v - mx) * scale)) : 0.f;
          sum += w[e];
        }
        Sums all;
        float before = sums_before(Sums{0, sum, 0.f}, sh, &all).hi;
        const float limit = cut_by_mass ? p * all.hi : INFINITY;
        float z = 0.f;
#pragma unroll
        for (int e = 0; e < kPlaces; ++e) {
          const int i = kPlaces * tid + e;
          if (i < have && (i == 0 || before < limit) && w[e] >= least) {
            z += w[e];
            best.see(logit_of(pair[e]), best.noise[index_of(pair[e])], index_of(pair[e]));
          }
          before += w[e];
        }
        sums_before(Sums{0, z, 0.f}, sh, &all);  // (every block of a cluster has the whole list)
        finish(all.hi, 0.f);
        return;
      }
    }
    // Count and mass bands: first the cut of top-k (if any), then that of top-p.
    using Yes = Flag<true>;
    using No = Flag<false>;
    bool ok = true;
    float limit = 0.f;
    for (int stage = k ? 0 : 1; stage < (cut_by_mass ? 2 : 1) && ok; ++stage) {
      const bool by_mass = stage == 1;
      const bool filtered = by_mass && k;  // only what top-k left
      float y0 = 0.f, y1 = kRange;
      ok = false;
      for (int level = 0; level < kLevels && !ok; ++level) {
        if (level) team.sync();  // everybody has read the last level's counts
        for (int b = tid; b < kBins; b += kThreads) sh.bins()[b] = 0;
        __syncthreads();
        const float per = kBins / (y1 - y0);
        float mass = 0.f;  // level 0: of everything; later: of what lies above the band
        int above = 0;
        // At first the last bin also takes what lies beyond the range, and NaN.
        auto tally = [&](auto filter, auto masses, auto first) {
          row.scan([&](const float* v, int i0) {
            const float2 mx2 = splat2(mx), scale2 = splat2(scale), per2 = splat2(per), y02 = splat2(y0);
#pragma unroll
            for (int j = 0; j < kVec; j += 2) {
              const float2 y2 = mul2(sub2(mx2, make_float2(v[j], v[j + 1])), scale2);
              const float2 b2 = mul2(first.value ? y2 : sub2(y2, y02), per2);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float y = e ? y2.y : y2.x;
                if (filter.value && !(v[j + e] > -INFINITY && pair_of(key_of(v[j + e]), i0 + j + e) >= cut)) continue;
                if (masses.value) {
                  const float w = ex2_approx(-y);
                  if (first.value ? y < INFINITY : y < y0) mass += w;
                } else if (!first.value) {
                  above += y < y0;
                }
                // adding 2^23 leaves the bin, rounded to the nearest, in the low bits
                const float b = fminf(e ? b2.y : b2.x, kBins - 1.f) + 8388608.f;
                if (first.value || (y >= y0 && y <= y1)) atomicAdd(sh.bins() + (__float_as_uint(b) & (kBins - 1)), 1);
              }
            }
          });
        };
        if (filtered) level ? tally(Yes{}, Yes{}, No{}) : tally(Yes{}, Yes{}, Yes{});
        else if (by_mass) level ? tally(No{}, Yes{}, No{}) : tally(No{}, Yes{}, Yes{});
        else level ? tally(No{}, No{}, No{}) : tally(No{}, No{}, Yes{});
        if (by_mass) mass = team.sum(mass);
        else if (level) above = team.sum(above);
        team.sync();
        if constexpr (Multi) {
          for (int b = tid; b < kBins; b += kThreads) {
            int c = 0;
            for (int q = 0; q < cluster; ++q) c += *team.peer(sh.bins() + b, q);
            sh.hist[b] = c;
          }
          __syncthreads();
        }
        if (by_mass && level == 0) limit = p * mass;
        // this thread's bins, in order
        constexpr int kPer = kBins / kThreads;
        const float head = level ? mass : 0.f;
        int c[kPer], sum_c = 0;
        float sum_hi = 0.f, sum_lo = 0.f;  // with every token at the bin's upper / lower weight
        const float step = 1.f / per;
        const float w0 = ex2_approx(-(y0 + (tid * kPer - 0.5f) * step)), ratio = ex2_approx(-step);
        // (the last bin of the first level has no lower end)
        auto lower = [&](int b, float upper) { return b == kBins - 1 && !level ? 0.f : upper * ratio * (b == kBins - 1 ? ratio : 1.f); };
        float upper = w0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int b = tid * kPer + e;
          c[e] = sh.hist[b];
          sum_c += c[e];
          sum_hi += c[e] * upper;
          sum_lo += c[e] * lower(b, upper);
          upper *= ratio;
        }
        if (tid == 0) sh.bin_from = kBins, sh.bin_to = kBins - 1, sh.bin_count = 0;
        Sums all;
        const Sums before = sums_before(Sums{sum_c, sum_hi, sum_lo}, sh, &all);
        if (!by_mass) {
          int n = before.n + (level ? above : 0);
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            if (n < k && n + c[e] >= k) sh.bin_from = sh.bin_to = tid * kPer + e, sh.bin_count = c[e];
            n += c[e];
          }
          __syncthreads();
        } else {
          // The mass down to and with a bin is bounded from above and below by the weights at its bins' ends, and,
          // where everything is counted (level 0), by the whole mass less such bounds of the bins behind it, which is
          // far sharper where little lies behind.
          float hi = head + before.hi, lo = head + before.lo;
          float behind_hi = all.hi - before.hi, behind_lo = all.lo - before.lo;
          const float slack = 3e-6f * mass;
          upper = w0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int b = tid * kPer + e;
            hi += c[e] * upper;
            lo += c[e] * lower(b, upper);
            behind_hi -= c[e] * upper;
            behind_lo -= c[e] * lower(b, upper);
            upper *= ratio;
            const float most = level ? hi : fminf(hi, mass - behind_lo * (1.f - 1e-4f));
            const float fewest = level ? lo : fmaxf(lo, mass - behind_hi * (1.f + 1e-4f));
            if (c[e] && most + slack >= limit) atomicMin(&sh.bin_from, b);
            if (c[e] && fewest - slack >= limit) atomicMin(&sh.bin_to, b);
          }
          __syncthreads();
          int inside = 0;
#pragma unroll
          for (int e = 0; e < kPer; ++e) {
            const int b = tid * kPer + e;
            if (b >= sh.bin_from && b <= sh.bin_to) inside += c[e];
          }
          inside = __reduce_add_sync(0xffffffffu, inside);
          if (tid % 32 == 0 && inside) atomicAdd(&sh.bin_count, inside);
          __syncthreads();
        }
        const int from = sh.bin_from, to = sh.bin_to, count = sh.bin_count;
        __syncthreads();
        if (from >= kBins || (to == kBins - 1 && level == 0)) break;  // the cut may lie below the range
        const float wide = 1e-6f * (y0 + to * step) + 1e-6f * step;
        y1 = to == kBins - 1 ? y1 : y0 + (to + 0.5f) * step + wide;
        y0 = fmaxf(y0, y0 + (from - 0.5f) * step - wide);
        ok = count <= kList - kList / 8;  // the widened edges may let a few more in
      }
      if (!ok) break;
      // what lies above the band, and the band itself as a list
      if (tid == 0) sh.n_mine = 0;
      __syncthreads();
      float mass = 0.f;
      int above = 0;
      const float bound = mx - (y1 * 1.0001f + 0.01f) / scale;  // what lies below the band is skipped by the piece
      auto split = [&](auto filter, auto masses) {
        row.scan_from(bound, [&](const float* v, int i0) {
          const float2 mx2 = splat2(mx), scale2 = splat2(scale);
          float y[kVec];
          int in = 0;
#pragma unroll
          for (int j = 0; j < kVec; j += 2) {
            const float2 y2 = mul2(sub2(mx2, make_float2(v[j], v[j + 1])), scale2);
            y[j] = y2.x, y[j + 1] = y2.y;
          }
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            if (filter.value && !(v[j] > -INFINITY && pair_of(key_of(v[j]), i0 + j) >= cut)) y[j] = INFINITY;
            if (masses.value) {
              const float w = ex2_approx(-y[j]);
              if (y[j] < y0) mass += w;
            } else {
              above += y[j] < y0;
            }
            in += y[j] >= y0 && y[j] <= y1;
          }
          // the last pass will want this noise
          asm volatile("prefetch.global.L2 [%0];" ::"l"(best.noise + min(max(i0, 0), a.vocab - 1)));
          if (in) {  // one place in the list for all of them: the counter's answer takes long
            int n = atomicAdd(&sh.n_mine, in);
#pragma unroll
            for (int j = 0; j < kVec; ++j)
              if (y[j] >= y0 && y[j] <= y1) {
                if (n < kList) sh.mine()[n] = pair_of(key_of(v[j]), i0 + j);
                ++n;
              }
          }
        });
      };
      if (filtered) split(Yes{}, Yes{});
      else if (by_mass) split(No{}, Yes{});
      else split(No{}, No{});
      if (by_mass) mass = team.sum(mass);
      else above = team.sum(above);
      const int n = team.gather_list();
      if (n > kList) {
        ok = false;
        break;
      }
      sort_list(sh, n, mx, scale, y0, y1);
      float w[kPlaces], sum = 0.f;
      uint64_t pair[kPlaces];
#pragma unroll
      for (int e = 0; e < kPlaces; ++e) {
        const int i = kPlaces * tid + e;
        pair[e] = i < n ? sh.list[i] : 0;
        const float v = logit_of(pair[e]);
        w[e] = i < n ? (v == mx ? 1.f : ex2_approx((v - mx) * scale)) : 0.f;
        sum += w[e];
      }
      Sums all;
      float before = mass + sums_before(Sums{0, sum, 0.f}, sh, &all).hi;
      // What lies above the band has to stay, and the last that stays has to be in it.
      if (by_mass ? !(mass < limit || mass == 0.f) || !(mass + all.hi >= limit * (1.f - 1e-6f)) : !(above < k && above + n >= k)) {
        ok = false;
        break;
      }
      if (tid == 0) sh.bin_count = 0;
      __syncthreads();
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < kPlaces; ++e) {
        const int i = kPlaces * tid + e;
        const bool stays = i < n && (by_mass ? before < limit || (mass == 0.f && i == 0) : above + i < k);
        if (stays) {
          z += w[e];
          atomicMax(&sh.bin_count, i);
        }
        before += w[e];
      }
      sums_before(Sums{0, z, 0.f}, sh, &all);
      cut = sh.list[sh.bin_count];
      total = mass + all.hi;
      __syncthreads();
    }
    settled = ok;
  }
  if (!settled) {
    const Cut found = slow_cut(row, mx, scale, k, p, team);
    cut = found.pair;
    team.exchanges = found.exchanges;
  }

  // The best score of what is kept: by a product with 1 / T at first, of which a thread keeps the best and the second
  // best group of four.
  const float cut_x = logit_of(cut), next_x = value_of(static_cast<uint32_t>(cut >> kIndexBits) + 1);
  const int cut_i = index_of(cut);
  const bool weigh = least > 0.f || !settled || !cut_by_mass;  // min-p, or a total that is not known yet
  // what min-p drops is far enough below this bound to be skipped by the piece
  const float least_x = least > 0.f && mx < INFINITY && scale < 1e30f ? mx - (0.01f - 1.0001f * log2f(least)) / scale : cut_x;
  float z = 0.f, near = -INFINITY, second = -INFINITY, widest_noise = 0.f;
  int near_at = -1;
  auto kept = [&](float v, int i) { return v > cut_x || (v == cut_x && i <= cut_i); };
  auto weight = [&](float v) { return v == mx ? 1.f : ex2_approx((v - mx) * scale); };
  auto rank = [&](auto weighs) {
    row.scan_noise(fmaxf(cut_x, least_x), best.noise, [&](const float* x, const float* g, int i0) {
      const float from = i0 <= cut_i ? cut_x : next_x;  // equal logits stay up to the cut's index
      float v[4], s = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x[j];
      if (i0 <= cut_i && cut_i < i0 + 3) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i0 + j > cut_i && v[j] == cut_x) v[j] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bool in = v[j] >= from;
        if (weighs.value) {
          const float w = weight(v[j]);
          in = in && w >= least;
          if (in) z += w;
        }
        s = fmaxf(s, fmaf(v[j], best.inv_t, in ? g[j] : -INFINITY));
        widest_noise = fmaxf(widest_noise, fabsf(g[j]));
      }
      second = fmaxf(second, fminf(near, s));
      near_at = s > near ? i0 : near_at;
      near = fmaxf(near, s);
    });
  };
  if (weigh) rank(Flag<true>{});
  else rank(Flag<false>{});
  // A product is off by less than `off`; a group that comes that near the block's top is scored exactly, and if a
  // thread's second best does too (or a score is infinite), all of the block's are.
  const auto larger = [](float a, float b) { return fmaxf(a, b); };
  const float top = block_reduce(near, sh.red.f32, larger);
  const float off = 2e-6f * (fabsf(mx * best.inv_t) + fabsf(top) + block_reduce(widest_noise, sh.red.f32, larger));
  const bool unclear = second >= top - off || !(fabsf(top) < 1e30f) || !(off < 1e30f);
  if (__syncthreads_or(unclear)) {
    row.scan_noise(fmaxf(cut_x, least_x), best.noise, [&](const float* v, const float* g, int i0) {
      for (int j = 0; j < 4; ++j)
        if (kept(v[j], i0 + j) && weight(v[j]) >= least) best.see(v[j], g[j], i0 + j);
    });
  } else if (near >= top - off) {
    for (int i = max(near_at, 0); i < min(near_at + 4, a.vocab); ++i) {
      const float v = row.one(i);
      if (kept(v, i) && weight(v) >= least) best.see(v, best.noise[i], i);
    }
  }
  finish(weigh ? 0.f : total, z);
}

template <typename T, bool Staged, bool Multi>
static cudaError_t launch_with(const Sample& a, int cluster, int bytes, cudaStream_t stream) {
  static SharedMemory allowed;
  if (Staged)
    if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(sample_kernel<T, Staged, Multi>), bytes,
                                               227 * 1024 - 1024 - static_cast<int>(sizeof(Shared<Multi>)));
        e != cudaSuccess)
      return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * cluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, Staged, Multi>, a, cluster);
}

template <typename T>
static cudaError_t launch(const Sample& a, cudaStream_t stream) {
  // Blocks per row: as few as hold it, because what the blocks of a cluster exchange costs several microseconds a row;
  // a block has an SM to itself while there are at most 148, then half of one.  More only while SMs are idle and a
  // thread has over 16 pieces to go through.  Where no row asks for top-k (whose exchange is the dearest) and a thread
  // would have over 6 of the whole row, as many as fit 128 SMs: 1 x 50304 bf16, 1 and 8 blocks, takes 13.7 and 7.6 us
  // without filters, 26.7 and 21.9 with top-p, 10.5 and 14.5 with top-k 50; 1 x 16384 with top-p 15.9 and 19.9; 18
  // rows of 32000 in 8 blocks (144, which clusters of 8 do not fill in one wave) 24.7, in 4 19.9.
  auto room = [](size_t shared, int per_sm) { return (227 * 1024 / per_sm - static_cast<int>(shared) - 1024) / 16; };  // pieces
  const int pieces = static_cast<int>((static_cast<long long>(a.vocab) * sizeof(T) + 15) / 16 + 1);
  const bool spread = !a.top_k.each && !a.top_k.all && pieces > 6 * kThreads;
  int cluster = 1, slice = pieces;
  for (;; cluster *= 2) {
    slice = (pieces + cluster - 1) / cluster;
    const long long blocks = static_cast<long long>(a.rows) * cluster;
    const bool fits = slice <= room(cluster > 1 ? sizeof(Shared<true>) : sizeof(Shared<false>), blocks <= 148 ? 1 : 2);
    const bool more = (slice > 16 * kThreads && 2 * blocks <= 148) || (spread && 2 * blocks <= 128);
    if (cluster == kMaxCluster || (fits && !more)) break;
  }
  const bool staged = slice <= std::min(kChunk * kChunks, room(sizeof(Shared<true>), 1));
  if (cluster == 1) return launch_with<T, true, false>(a, 1, slice * 16, stream);
  return staged ? launch_with<T, true, true>(a, cluster, slice * 16, stream) : launch_with<T, false, true>(a, cluster, 0, stream);
}

cudaError_t launch_sample(const Sample& a, cudaStream_t stream) {
  return a.bf16 ? launch<__nv_bfloat16>(a, stream) : launch<float>(a, stream);
}

}  // namespace sampling

}  // namespace mnb
