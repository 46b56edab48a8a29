// The shared prefix's part of the paged attention on the 5th-generation tensor
// cores, for more query rows than a few warps can feed (prefix_attention.cu
// has the mathematics, the other parts and the choice between them).
//
// A block owns up to 256 query rows of one kv head (rows of all sequences and
// grouped heads side by side: no row of the prefix part is masked) and a range
// of keys.  Its two streams have a softmax warpgroup, 128 columns of scores
// and an output accumulator in TMEM each, and take turns on the tensor core:
// while one stream's products run, the other's exponentials are computed.
//   more than 128 rows: stream s has rows [128 s, 128 s + 128) and every key
//     tile; a tile of K and V is loaded once for both.
//   up to 128 rows: both streams have the same rows, and stream s the key
//     tiles s, s + 2, ...; they are joined through shared memory at the end.
// Per 128-key tile and stream:  S = Q K^T (TMEM) -> softmax: thread = row, no
// exchange between threads; P (bf16) goes over S in TMEM -> O += P V with P as
// the TMEM operand.  The base that scores are taken relative to is a running
// maximum that only moves when a row's scores pass it by 2^8, so O is rarely
// rescaled (exact either way: the final division uses the same base); it is
// held in fp32, because a rounded one lies up to a 2^-8th of itself above the
// scores, which for large ones is more than any weight survives.  Sums are
// fp32.
//
// Measured: 16 sequences of 4 grouped heads (64 rows) over 65,537 keys of 8 kv
// heads, 268 MB: 48 us, 5.6 TB/s, bound by the bytes.  2388 rows of 32 heads
// over 4001 keys, 157 GFLOP: about 185 us, 0.85 PFLOP/s (0.52 of the measured bf16
// peak).  A step of both streams (256 rows, 128 keys) takes some 3300 cycles,
// of which the products take 2048 and the exponentials as long on their unit;
// what is left is the chain S -> maximum -> P -> O -> next S of each stream,
// which two streams overlap only in part.  One warpgroup per stream (128 keys
// a thread) took 3200 to 3800 cycles, and issuing the products from a
// lane-divergent branch 3800.
//
// K and V tiles come page by page through a TMA tensor map of the pool
// (head_dim, heads, tokens, pages) into a ring of 128-byte-swizzled stages, in
// the order in which the products use them.  The MMA warp zeroes V rows past
// the prefix's end (pages hold anything there); keys past it are masked.
#include "common.cuh"
#include "generation.h"
#include "launch.cuh"
#include "warp_mma.cuh"

namespace mnb {

namespace prefix {

namespace tc {

constexpr int kTile = 128;             // rows per stream and keys per tile
constexpr int kSoftmax = 512;            // threads: two warpgroups for each stream, each with half the keys of a tile
constexpr int kThreads = 64 + kSoftmax;  // and the producer and MMA warps
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;        // log2 units that the scores may pass the running maximum by

template <int D>
struct Smem {
  static constexpr uint32_t q_tile = kTile * D * 2;
  static constexpr uint32_t kv_tile = kTile * D * 2;
  static constexpr int stages = D == 128 ? 5 : 8;
  static constexpr uint32_t q_off = 0, kv_off = 2 * q_tile;
  static constexpr uint32_t bar_off = kv_off + stages * kv_tile;
  static constexpr int n_bars = 2 * stages + 10;
  static constexpr uint32_t max_off = bar_off + n_bars * 8 + 16;  // row maxima so far: [stream][row], as order_of()
  static constexpr uint32_t total = max_off + 2 * kTile * 4 + 1024;
  static_assert(total <= 227 * 1024, "a block's shared memory");
};

MNB_DEVICE void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
MNB_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
// 2^x of a pair on the FMA and integer pipes.  x = n + f with n the nearest whole number (adding and subtracting
// 1.5 * 2^23 rounds to it; shifted left by 23 the sum's bits are n in the exponent's place, the rest shifted out) and
// 2^f from 1 + c1 f + ... + c5 f^5, a least-squares fit of the relative error on [-1/2, 1/2] reweighted until level
// (computed for this kernel; off by at most 1.1e-7, with its roundings 1.7e-7).  Below -126 the result is about 2^-126
// where 0 would be right, and NaN is not kept.
MNB_DEVICE float2 exp2_fma(float2 x) {
  x = make_float2(fmaxf(x.x, -126.f), fmaxf(x.y, -126.f));
  const float2 round = splat2(12582912.f);
  const float2 t = add2(x, round), f = sub2(x, sub2(t, round));
  float2 p = fma2(f, splat2(0.001326472614891827f), splat2(0.009671512991189957f));
  p = fma2(p, f, splat2(0.05550733581185341f));
  p = fma2(p, f, splat2(0.24022242426872253f));
  p = fma2(p, f, splat2(0.6931470036506653f));
  p = fma2(p, f, splat2(1.f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}
MNB_DEVICE void tmem_st_8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// One lane of a converged warp, the same one every time: the products are issued from warp-uniform code, so their
// descriptors stay in uniform registers (a `lane == 0` branch moved them there one by one: 110 cycles a product
// instead of the 64 it takes).
MNB_DEVICE bool elected() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
// The largest of three, or NaN where one is.
MNB_DEVICE float max3_or_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Whole numbers in the floats' order (and back): what atomicMax on shared memory takes.  NaN (as the maximum gives it) comes last.
MNB_DEVICE int order_of(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
MNB_DEVICE float of_order(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
// A warp's wait, given up by all of its lanes or by none.
MNB_DEVICE bool warp_wait(uint32_t bar, uint32_t parity, int* abort) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort)); }
MNB_DEVICE void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kSoftmax) : "memory"); }
MNB_DEVICE void stream_sync(int s) { asm volatile("bar.sync %0, %1;" ::"r"(2 + s), "n"(kSoftmax / 2) : "memory"); }

// A lane's part of a row, moved at once.
template <int N>
struct Vec {
  struct alignas(4 * N) type {
    float v[N];
  };
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v, int whole) {
  using S = Smem<D>;
  constexpr int kStages = S::stages;
  constexpr uint32_t kIdescS = idesc_bf16(kTile, kTile, false, false);
  constexpr uint32_t kIdescO = idesc_bf16(kTile, D, false, true);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(sm);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::bar_off);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::n_bars);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kStages, q_full = empty0 + 8 * kStages,
                 s_full0 = q_full + 8, o_full0 = s_full0 + 16, p_full0 = o_full0 + 16,  // (p_full: two halves per stream)
                 drained = p_full0 + 32;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // The first `whole` blocks take 256 rows, the others half as many: a last wave that fills less than half of the SMs
  // is done in half the time (2484 rows of 32 heads over 4001 keys: 320 blocks in three waves 284 us the whole call, the
  // third with half the rows 257 us).
  int unit = blockIdx.x, most = 2 * kTile, skip = 0;
  if (unit >= whole) {
    skip = (unit - whole) % 2 * kTile;
    most = kTile;
    unit = whole + (unit - whole) / 2;
  }
  const int rt = unit % a.row_tiles;
  const int h = (unit / a.row_tiles) % a.kv_heads;
  const int split = unit / (a.row_tiles * a.kv_heads);
  const int r0 = rt * 2 * kTile + skip;
  const int n_rows = min(most, a.n * a.group - r0);
  if (n_rows <= 0) return;
  const bool shared = n_rows > kTile;  // both streams use every key tile
  const int k0 = split * a.prefix_chunk, k1 = min(a.prefix_len, k0 + a.prefix_chunk);
  const int n_tiles = (k1 - k0 + kTile - 1) / kTile;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(q_full, kSoftmax);
    mbar_init(drained, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full0 + 8 * s, 1);
      mbar_init(p_full0 + 16 * s, 128);
      mbar_init(p_full0 + 16 * s + 8, 128);
      mbar_init(o_full0 + 8 * s, 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (threadIdx.x < 2 * kTile) reinterpret_cast<int*>(sm + S::max_off)[threadIdx.x] = order_of(-INFINITY);
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  const uint32_t tmem = *tmem_slot;  // S_0, S_1: 128 columns each, then O_0, O_1

  if (warp == 0) {
    int pos = 0;
    auto load = [&](const CUtensorMap* map, int tile) -> bool {
      const int st = pos % kStages;
      if (!warp_wait(empty0 + 8 * st, ((pos / kStages) & 1) ^ 1, a.status)) return false;
      ++pos;
      const int j0 = k0 + tile * kTile;
      const int per = min(1 << a.page_shift, 64);  // tokens of a box
      const int boxes = (min(kTile, k1 - j0) + per - 1) / per;
      if (lane == 0) mbar_arrive_expect_tx(full0 + 8 * st, boxes * per * D * 2);
      __syncwarp();
      if (lane < boxes) {
        const int j = j0 + lane * per;
        int page = a.prefix_pages[j >> a.page_shift];
        if (page < 0 || page >= a.pages) {
          atomicCAS(a.errors, 0, kErrBadIndex);
          page = a.no_page;
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(sbase + S::kv_off + st * S::kv_tile + c * (kTile * 128) + lane * per * 128, map, c * 64, h,
                      j & ((1 << a.page_shift) - 1), page, full0 + 8 * st);
      }
      return true;
    };
    bool ok = true;
    if (shared) {
      for (int t = 0; t < n_tiles && ok; ++t) ok = load(&map_k, t) && load(&map_v, t);
    } else {
      ok = load(&map_k, 0) && (n_tiles < 2 || load(&map_k, 1));
      for (int t = 0; t < n_tiles && ok; ++t) ok = load(&map_v, t) && (t + 2 >= n_tiles || load(&map_k, t + 2));
    }
    // The block does not end before its last copies have arrived, also where another warp's wait was given up.
    for (int p = max(0, pos - kStages); p < pos; ++p) mbar_wait(full0 + 8 * (p % kStages), (p / kStages) & 1, nullptr);
  } else if (warp == 1) {
    int pos = 0;
    // Whether this lane's waits have all ended well.  The lanes agree on it once a step (`settle`): a vote at each wait made
    // the kernel 2 % slower, and what a step computes past a wait that was given up is in bounds.
    bool good = true;
    auto settle = [&] { return __all_sync(0xffffffffu, good); };
    auto wait_full = [&](int p) { good = mbar_wait(full0 + 8 * (p % kStages), (p / kStages) & 1, a.status) && good; };
    // (adding bytes / 16 to a descriptor moves its address: the tiles lie below 256 KB, so nothing carries)
    const uint64_t q_desc = smem_desc_sw128(sbase + S::q_off, 16, 1024);
    const uint64_t k_desc = smem_desc_sw128(sbase + S::kv_off, 16, 1024);
    const uint64_t v_desc = smem_desc_sw128(sbase + S::kv_off, kTile * 128, 1024);
    auto tile_of = [&](int p) { return static_cast<uint64_t>(p % kStages) * (S::kv_tile / 16); };
    // S_s = Q_s K^T
    auto scores = [&](int s, int p) {
      const uint64_t qa = q_desc + (shared ? s : 0) * (S::q_tile / 16), kb = k_desc + tile_of(p);
      if (elected()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t at = ((kk / 4) * (kTile * 128) + (kk % 4) * 32) / 16;
          tc_mma(tmem + s * kTile, qa + at, kb + at, kIdescS, kk > 0 ? 1u : 0u);
        }
        tc_commit(s_full0 + 8 * s);
      }
      __syncwarp();
    };
    // O_s (+)= P_s V, the first half of the keys while the second half's probabilities are still computed
    auto values = [&](int s, int p, int step) {
      const uint64_t vb = v_desc + tile_of(p);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        good = mbar_wait(p_full0 + 16 * s + 8 * half, step & 1, a.status) && good;
        tc_fence_after();
        if (elected()) {
#pragma unroll
          for (int kk = half * kTile / 32; kk < (half + 1) * kTile / 32; ++kk)
            tc_mma_tmem_a(tmem + 2 * kTile + s * D, tmem + s * kTile + kk * 8, vb + kk * (2048 / 16), kIdescO,
                          step == 0 && kk == 0 ? 0u : 1u);
        }
        __syncwarp();
      }
    };
    auto done_with = [&](int p) {
      if (elected()) tc_commit(empty0 + 8 * (p % kStages));
      __syncwarp();
    };
    // rows of V past the end of the keys
    auto clean = [&](int tile, int p) {
      const int valid = k1 - k0 - tile * kTile;
      if (valid >= kTile) return;
      uint8_t* v = sm + S::kv_off + (p % kStages) * S::kv_tile;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
        for (int i = valid * 8 + lane; i < kTile * 8; i += 32)
          *reinterpret_cast<uint4*>(v + c * (kTile * 128) + i * 16) = make_uint4(0, 0, 0, 0);
      fence_async_smem();
      __syncwarp();
    };
    bool ok = warp_wait(q_full, 0, a.status);
    tc_fence_after();
    if (shared) {
      if (ok) {
        wait_full(pos);
        scores(0, pos);
        scores(1, pos);
        done_with(pos++);
        ok = settle();
      }
      for (int t = 0; t < n_tiles && ok; ++t) {
        const int v = pos++, k = pos;
        const bool more = t + 1 < n_tiles;
        if (more) ++pos;
        wait_full(v);
        clean(t, v);
        values(0, v, t);
        if (more) {
          wait_full(k);
          scores(0, k);
        } else if (elected()) {
          tc_commit(o_full0);
        }
        values(1, v, t);
        done_with(v);
        if (more) {
          scores(1, k);
          done_with(k);
        } else if (elected()) {
          tc_commit(o_full0 + 8);
        }
        ok = settle();
      }
    } else {
      for (int s = 0; s < 2 && s < n_tiles && ok; ++s) {
        wait_full(pos);
        scores(s, pos);
        done_with(pos++);
        ok = settle();
      }
      for (int t = 0; t < n_tiles && ok; ++t) {
        const int s = t & 1;
        wait_full(pos);
        clean(t, pos);
        values(s, pos, t >> 1);
        done_with(pos++);
        if (t + 2 < n_tiles) {
          wait_full(pos);
          scores(s, pos);
          done_with(pos++);
        } else if (elected()) {
          tc_commit(o_full0 + 8 * s);
        }
        ok = settle();
      }
    }
    if (!ok) {  // a wait was given up: nor do products end after their TMEM is freed
      if (elected()) tc_commit(drained);
      __syncwarp();
      mbar_wait(drained, 0, nullptr);
    }
  } else {
    const int s = (warp - 2) / 8, half = (warp - 2) / 4 % 2, quad = warp % 4;
    const int r = quad * 32 + lane;                 // row of the stream's tile
    {  // Q, swizzled as TMA would leave it; rows past the last are zeros
      constexpr int kChunks = D / 8, kStep = kSoftmax / kChunks;  // a thread keeps its chunk and goes through the rows
      const int c = (threadIdx.x - 64) % kChunks, end = shared ? 2 * kTile : kTile;
      for (int i = (threadIdx.x - 64) / kChunks; i < end; i += kStep) {
        const bool in = i < n_rows;
        const int x = i % kTile, j = in ? r0 + i : r0;
        cp_async16(sbase + S::q_off + (i / kTile) * S::q_tile + (c / 8) * (kTile * 128) + x * 128 + (((c % 8) ^ (x % 8)) << 4),
                   a.q + (j / a.group) * a.q_ld + (h * a.group + j % a.group) * a.q_head + c * 8, in);
      }
      cp_async_commit();
      cp_async_wait_all();
      fence_async_smem();
      mbar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    volatile int* seen = reinterpret_cast<int*>(sm + S::max_off) + s * kTile + r;
    const uint32_t t_s = tmem + s * kTile + lanes, t_o = tmem + 2 * kTile + s * D + lanes;
    const int steps = shared ? n_tiles : (n_tiles - s + 1) / 2;
    const bool padding = (shared ? s * kTile : 0) + quad * 32 >= n_rows;  // a warp without rows leaves P as it is
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t < steps; ++t) {
      // (a wait that gave up is in the status word; the loop goes on, because the other warps meet this one at barriers)
      mbar_wait(s_full0 + 8 * s, t & 1, a.status);
      __syncwarp();
      tc_fence_after();
      if (padding) {
        tc_fence_before();
        stream_sync(s);
        mbar_arrive(p_full0 + 16 * s + 8 * half);
        continue;
      }
      const int valid = k1 - k0 - (shared ? t : 2 * t + s) * kTile - half * 64;  // keys of this half tile (or more, or none)
      float v[64];
      tmem_ld_64(t_s + half * 64, v);
      if (valid < 64) {
#pragma unroll
        for (int i = 0; i < 64; ++i)
          if (i >= valid) v[i] = -INFINITY;
      }
      float mx = v[0], mx2 = v[1];
#pragma unroll
      for (int i = 2; i < 64; i += 4) {
        mx = max3_or_nan(mx, v[i], v[i + 1]);
        if (i + 3 < 64) mx2 = max3_or_nan(mx2, v[i + 2], v[i + 3]);
      }
      mx = max3_or_nan(mx, mx2, mx2);  // (a score of NaN makes the row NaN, by its base)
      // The halves' maxima meet in the row's maximum so far.  Past this barrier both halves' scores are in registers, so
      // P may go over them.  (Neither half is ahead: S of a step was issued after both halves of the last one had read
      // their maximum and written P.)
      atomicMax(const_cast<int*>(seen), order_of(mx * a.scale_log2));
      tc_fence_before();
      stream_sync(s);
      tc_fence_after();
      mx = of_order(*seen);
      const bool grows = !(mx <= m + kRescale) || m == -INFINITY;
      if (__any_sync(0xffffffffu, grows)) {
        const float to = grows ? mx : m;
        const float alpha = ex2_approx(m - (to == -INFINITY ? 0.f : to));
        if (t > 0 && half == 0) {
          // The first half's threads rescale O: the products of this step wait for their probabilities.  Every product
          // issued so far has finished: S of this step was issued after them.
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            float x[16];
            uint32_t w[16];
            tmem_ld_16(t_o + c * 16, x);
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(x[i] * alpha);
            tmem_st_16(t_o + c * 16, w);
          }
        }
        l *= alpha;
        m = to;
      }
      float2 scale2 = splat2(a.scale_log2);
      const float2 base2 = splat2(m == -INFINITY ? 0.f : -m);
      if (__any_sync(0xffffffffu, fabsf(m) >= 16777216.f)) {
        // Here rounding a scaled score moves it by whole units, and by more than a float's range later: round the scores as
        // their maximum was.
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] *= a.scale_log2;
        scale2 = splat2(1.f);
      }
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 y = fma2(make_float2(v[c * 16 + i], v[c * 16 + i + 1]), scale2, base2);
          // one pair of eight on the FMA pipe: the exponential unit alone takes as long as the products (none of eight
          // measured 3 % slower, two equal)
          const float2 p = i == 6 ? exp2_fma(y) : make_float2(ex2_approx(y.x), ex2_approx(y.y));
          sum = add2(sum, p);
          w[i / 2] = pack_bf16x2(p.x, p.y);
        }
        tmem_st_8(t_s + half * 32 + c * 8, w);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full0 + 16 * s + 8 * half);
      l += sum.x + sum.y;
    }
    if (steps > 0) {
      mbar_wait(o_full0 + 8 * s, 0, a.status);
      __syncwarp();
      tc_fence_after();
    }
    // Outputs, maxima and sums pass through the ring, which nobody uses any more once both streams have theirs, so that
    // a warp can write whole rows; streams of the same rows meet there.
    constexpr int kPitch = D + 4, kPer = D / 32;
    float* meet = reinterpret_cast<float*>(sm + S::kv_off);
    float2* meet_ml = reinterpret_cast<float2*>(meet + 2 * kTile * kPitch);
    struct Row {  // where a row goes, and the factors of its parts
      int at;
      float top, mine, met, inv;
    };
    Row* info = reinterpret_cast<Row*>(meet_ml + 2 * kTile);
    float* meet_l = reinterpret_cast<float*>(info + 2 * kTile);  // the second half's sums
    static_assert(2 * kTile * (kPitch * 4 + 8 + sizeof(Row) + 4) <= S::stages * S::kv_tile, "the meeting place fits the ring");
    softmax_sync();
#pragma unroll
    for (int c = half * D / 32; c < (half + 1) * D / 32; ++c) {
      float v[16];
      if (steps > 0) tmem_ld_16(t_o + c * 16, v);
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(meet + (s * kTile + r) * kPitch + c * 16 + i) =
            steps > 0 ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (half == 1) meet_l[s * kTile + r] = l;
    softmax_sync();
    if (half == 0) {
      l += meet_l[s * kTile + r];
      meet_ml[s * kTile + r] = make_float2(m, l);
    }
    softmax_sync();
    using Part = typename Vec<kPer>::type;
    const long long rows = static_cast<long long>(a.n) * a.heads;
    wait_for_previous();  // the own keys' pieces
    const int own = own_count(a) ? a.own_splits : 0;
    const bool alone = a.prefix_splits == 1;  // then this block joins the rows with their own keys' pieces and finishes them
    if (const int i = s * kTile + r; i < n_rows && half == 0) {  // (without `shared`, the first stream's threads)
      const int j = r0 + i, token = j / a.group;
      Row x{token * a.heads + h * a.group + j - token * a.group, m, 1.f, 0.f, 1.f};
      if (!shared) {
        const float2 other = meet_ml[kTile + i];
        x.top = fmaxf(m, other.x);
        const float base = x.top == -INFINITY ? 0.f : x.top;
        x.mine = ex2_approx(m - base), x.met = ex2_approx(other.x - base);
        l = l * x.mine + other.y * x.met;
      }
      if (alone) {
        const float prefix_top = x.top;
        for (int p = 1; p < 1 + own; ++p) x.top = fmaxf(x.top, a.part_ml[p * rows + x.at].x);
        const float base = x.top == -INFINITY ? 0.f : x.top, f = ex2_approx(prefix_top - base);
        l *= f;
        for (int p = 1; p < 1 + own; ++p) {
          const float2 ml = a.part_ml[p * rows + x.at];
          l = fmaf(ex2_approx(ml.x - base), ml.y, l);
        }
        x.inv = l == 0.f ? 0.f : 1.f / l;  // (NaN stays NaN)
        x.mine *= f * x.inv, x.met *= f * x.inv;
        if (a.lse) a.lse[x.at] = l == 0.f ? -INFINITY : kLn2 * (x.top + log2f(l));
      } else {
        a.part_ml[split * rows + x.at] = make_float2(x.top, l);
      }
      info[i] = x;
    }
    softmax_sync();
    constexpr int kBatch = 2;  // rows whose loads are under way together
    for (int i0 = (warp - 2) * kBatch; i0 < n_rows; i0 += kSoftmax / 32 * kBatch) {
      Part o[kBatch];
      Row x[kBatch];
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        const int i = min(i0 + e, n_rows - 1);
        x[e] = info[i];
        o[e] = *reinterpret_cast<const Part*>(meet + i * kPitch + lane * kPer);
        Part met;
        if (!shared) met = *reinterpret_cast<const Part*>(meet + (kTile + i) * kPitch + lane * kPer);
#pragma unroll
        for (int d = 0; d < kPer; ++d) o[e].v[d] = o[e].v[d] * x[e].mine + (shared ? 0.f : met.v[d] * x[e].met);
      }
      if (!alone) {
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          if (i0 + e < n_rows) *reinterpret_cast<Part*>(a.part_o + (split * rows + x[e].at) * D + lane * kPer) = o[e];
        continue;
      }
      for (int p = 1; p < 1 + own; ++p) {
        float top[kBatch];
        Part y[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          top[e] = a.part_ml[p * rows + x[e].at].x;
          y[e] = *reinterpret_cast<const Part*>(a.part_o + (p * rows + x[e].at) * D + lane * kPer);
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const float g = top[e] == -INFINITY ? 0.f : ex2_approx(top[e] - x[e].top) * x[e].inv;
#pragma unroll
          for (int d = 0; d < kPer; ++d) o[e].v[d] += g == 0.f ? 0.f : y[e].v[d] * g;  // (nothing was written without keys)
        }
      }
#pragma unroll
      for (int e = 0; e < kBatch; ++e) {
        if (i0 + e >= n_rows) break;
        uint32_t w[kPer / 2];
#pragma unroll
        for (int d = 0; d < kPer; d += 2) w[d / 2] = pack_bf16x2(o[e].v[d], o[e].v[d + 1]);
        uint32_t* out = reinterpret_cast<uint32_t*>(a.o + static_cast<long long>(x[e].at) * D) + lane * (kPer / 2);
        if constexpr (kPer == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
        else *out = w[0];
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D>
static cudaError_t launch(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  constexpr int bytes = Smem<D>::total;
  static SharedMemory allowed;
  if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(prefix_tc_kernel<D>), bytes); e != cudaSuccess) return e;
  const int units = a.row_tiles * a.kv_heads * a.prefix_splits, last = units % 148;
  const int whole = a.prefix_splits == 1 && 2 * last <= 148 ? units - last : units;
  const int blocks = whole + 2 * (units - whole);
  if (a.own_splits > 0) return launch_after(prefix_tc_kernel<D>, blocks, kThreads, bytes, stream, a, mk, mv, whole);
  prefix_tc_kernel<D><<<blocks, kThreads, bytes, stream>>>(a, mk, mv, whole);
  return cudaGetLastError();
}

__global__ void exp2_kernel(const float* __restrict__ x, float* __restrict__ y, int pairs) {
  for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < pairs; i += gridDim.x * blockDim.x) {
    const float2 p = exp2_fma(make_float2(x[2 * i], x[2 * i + 1]));
    y[2 * i] = p.x, y[2 * i + 1] = p.y;
  }
}

}  // namespace tc

cudaError_t launch_exp2(const float* x, float* y, int pairs, cudaStream_t stream) {
  tc::exp2_kernel<<<148, 256, 0, stream>>>(x, y, pairs);
  return cudaGetLastError();
}

cudaError_t launch_prefix_tc(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, int head_dim, cudaStream_t stream) {
  return head_dim == 64 ? tc::launch<64>(a, mk, mv, stream) : tc::launch<128>(a, mk, mv, stream);
}

}  // namespace prefix

}  // namespace mnb
