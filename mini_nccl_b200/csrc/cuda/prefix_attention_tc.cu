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
// the TMEM operand.  The running maximum only moves when a row's scores pass
// it by 2^8, so O is rarely rescaled (exact either way: the final division
// uses the same maximum); sums are fp32.
//
// K and V tiles come page by page through a TMA tensor map of the pool
// (head_dim, heads, tokens, pages) into a ring of 128-byte-swizzled stages, in
// the order in which the products use them.  The MMA warp zeroes V rows past
// the prefix's end (pages hold anything there); keys past it are masked.
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace prefix {

namespace tc {

constexpr int kTile = 128;             // rows per stream and keys per tile
constexpr int kThreads = 32 * 12;      // producer, MMA, two idle warps, two softmax warpgroups
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRescale = 8.f;        // log2 units that the scores may pass the running maximum by

template <int D>
struct Smem {
  static constexpr uint32_t q_tile = kTile * D * 2;
  static constexpr uint32_t kv_tile = kTile * D * 2;
  static constexpr int stages = D == 128 ? 5 : 8;
  static constexpr uint32_t q_off = 0, kv_off = 2 * q_tile;
  static constexpr uint32_t bar_off = kv_off + stages * kv_tile;
  static constexpr int n_bars = 2 * stages + 7;
  static constexpr uint32_t total = bar_off + n_bars * 8 + 16 + 1024;
};

MNB_DEVICE void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
MNB_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
MNB_DEVICE void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v) {
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
                 s_full0 = q_full + 8, p_full0 = s_full0 + 16, o_full0 = p_full0 + 16;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rt = blockIdx.x % a.row_tiles;
  const int h = (blockIdx.x / a.row_tiles) % a.kv_heads;
  const int split = blockIdx.x / (a.row_tiles * a.kv_heads);
  const int r0 = rt * 2 * kTile;
  const int n_rows = min(2 * kTile, a.n * a.group - r0);
  const bool shared = n_rows > kTile;  // both streams use every key tile
  const int k0 = split * a.prefix_chunk, k1 = min(a.prefix_len, k0 + a.prefix_chunk);
  const int n_tiles = (k1 - k0 + kTile - 1) / kTile;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    mbar_init(q_full, 256);
    for (int s = 0; s < 2; ++s) {
      mbar_init(s_full0 + 8 * s, 1);
      mbar_init(p_full0 + 8 * s, 128);
      mbar_init(o_full0 + 8 * s, 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S_0, S_1: 128 columns each, then O_0, O_1

  if (warp == 0) {
    int pos = 0;
    auto load = [&](const CUtensorMap* map, int tile) -> bool {
      const int st = pos % kStages;
      if (!mbar_wait(empty0 + 8 * st, ((pos / kStages) & 1) ^ 1, a.status)) return false;
      ++pos;
      const int j0 = k0 + tile * kTile;
      const int per = min(1 << a.page_shift, kTile);  // tokens of a box
      const int boxes = (min(kTile, k1 - j0) + per - 1) / per;
      if (lane == 0) mbar_arrive_expect_tx(full0 + 8 * st, boxes * per * D * 2);
      __syncwarp();
      if (lane < boxes) {
        const int j = j0 + lane * per;
        int page = a.prefix_pages[j >> a.page_shift];
        if (page < 0 || page >= a.pages) {
          atomicCAS(a.status, 0, kErrBadIndex);
          page = a.pages;  // outside the map: reads as zeros
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
  } else if (warp == 1) {
    int pos = 0;
    auto stage_of = [&](int p) { return sbase + S::kv_off + (p % kStages) * S::kv_tile; };
    auto wait_full = [&](int p) { return mbar_wait(full0 + 8 * (p % kStages), (p / kStages) & 1, a.status); };
    // S_s = Q_s K^T
    auto scores = [&](int s, int p) {
      if (lane == 0) {
        const uint32_t qa = sbase + S::q_off + (shared ? s : 0) * S::q_tile, kb = stage_of(p);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          tc_mma(tmem + s * kTile, smem_desc_sw128(qa + (kk / 4) * (kTile * 128) + (kk % 4) * 32, 16, 1024),
                 smem_desc_sw128(kb + (kk / 4) * (kTile * 128) + (kk % 4) * 32, 16, 1024), kIdescS, kk > 0 ? 1u : 0u);
        tc_commit(s_full0 + 8 * s);
      }
    };
    // O_s (+)= P_s V
    auto values = [&](int s, int p, bool first) {
      if (lane == 0) {
        const uint32_t vb = stage_of(p);
#pragma unroll
        for (int kk = 0; kk < kTile / 16; ++kk)
          tc_mma_tmem_a(tmem + 2 * kTile + s * D, tmem + s * kTile + kk * 8, smem_desc_sw128(vb + kk * 2048, kTile * 128, 1024),
                        kIdescO, first && kk == 0 ? 0u : 1u);
      }
    };
    auto done_with = [&](int p) {
      if (lane == 0) tc_commit(empty0 + 8 * (p % kStages));
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
    bool ok = mbar_wait(q_full, 0, a.status);
    tc_fence_after();
    if (shared) {
      if (ok && (ok = wait_full(pos))) {
        scores(0, pos);
        scores(1, pos);
        done_with(pos++);
      }
      for (int t = 0; t < n_tiles && ok; ++t) {
        const int v = pos++, k = pos;
        const bool more = t + 1 < n_tiles;
        if (more) ++pos;
        if (!(ok = wait_full(v))) break;
        clean(t, v);
        if (!(ok = mbar_wait(p_full0, t & 1, a.status))) break;
        tc_fence_after();
        values(0, v, t == 0);
        if (more) {
          if (!(ok = wait_full(k))) break;
          scores(0, k);
        } else if (lane == 0) {
          tc_commit(o_full0);
        }
        if (!(ok = mbar_wait(p_full0 + 8, t & 1, a.status))) break;
        tc_fence_after();
        values(1, v, t == 0);
        done_with(v);
        if (more) {
          scores(1, k);
          done_with(k);
        } else if (lane == 0) {
          tc_commit(o_full0 + 8);
        }
      }
    } else {
      for (int s = 0; s < 2 && s < n_tiles && ok; ++s)
        if ((ok = wait_full(pos))) {
          scores(s, pos);
          done_with(pos++);
        }
      for (int t = 0; t < n_tiles && ok; ++t) {
        const int s = t & 1;
        if (!(ok = wait_full(pos))) break;
        clean(t, pos);
        if (!(ok = mbar_wait(p_full0 + 8 * s, (t >> 1) & 1, a.status))) break;
        tc_fence_after();
        values(s, pos, t < 2);
        done_with(pos++);
        if (t + 2 < n_tiles) {
          if (!(ok = wait_full(pos))) break;
          scores(s, pos);
          done_with(pos++);
        } else if (lane == 0) {
          tc_commit(o_full0 + 8 * s);
        }
      }
    }
  } else if (warp >= 4) {
    const int s = (warp - 4) / 4, quad = warp % 4;
    const int r = quad * 32 + lane;                 // row of the stream's tile
    const int row = shared ? s * kTile + r : r;     // row of the block
    auto token_of = [&](int i) { return (r0 + i) / a.group; };
    auto head_of = [&](int i) { return h * a.group + (r0 + i) % a.group; };
    {  // Q, swizzled as TMA would leave it; rows past the last are zeros
      const int t = threadIdx.x - 128;
      const int q_rows = shared ? 2 * kTile : kTile;
      for (int i = t; i < q_rows * (D / 8); i += 256) {
        const int qr = i / (D / 8), c = i % (D / 8);
        uint4 w = make_uint4(0, 0, 0, 0);
        if (qr < n_rows) w = ld_v4(a.q + token_of(qr) * a.q_ld + head_of(qr) * a.q_head + c * 8);
        const int qt = qr / kTile, x = qr % kTile;
        st_v4(sm + S::q_off + qt * S::q_tile + (c / 8) * (kTile * 128) + x * 128 + (((c % 8) ^ (x % 8)) << 4), w);
      }
      fence_async_smem();
      mbar_arrive(q_full);
    }
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + s * kTile + lanes, t_o = tmem + 2 * kTile + s * D + lanes;
    const int steps = shared ? n_tiles : (n_tiles - s + 1) / 2;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int t = 0; t < steps; ++t) {
      ok = __all_sync(0xffffffffu, mbar_wait(s_full0 + 8 * s, t & 1, a.status));
      if (!ok) break;
      tc_fence_after();
      const int valid = k1 - k0 - (shared ? t : 2 * t + s) * kTile;  // keys of this tile (or more)
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float v[64];
        tmem_ld_64(t_s + c * 64, v);
        if (valid < kTile) {
#pragma unroll
          for (int i = 0; i < 64; ++i) mx = fmaxf(mx, c * 64 + i < valid ? v[i] : -INFINITY);
        } else {
#pragma unroll
          for (int i = 0; i < 64; i += 2) mx = max3f(mx, v[i], v[i + 1]);
        }
      }
      mx *= a.scale_log2;
      const bool grows = mx > m + kRescale || m == -INFINITY;
      if (__any_sync(0xffffffffu, grows)) {
        const float to = grows ? mx : m;
        const float alpha = ex2_approx(m - (to == -INFINITY ? 0.f : to));
        if (t > 0) {
          // every product issued so far has finished: S of this step was issued after them
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            float v[16];
            uint32_t w[16];
            tmem_ld_16(t_o + c * 16, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * alpha);
            tmem_st_16(t_o + c * 16, w);
          }
        }
        l *= alpha;
        m = to;
      }
      const float base = m == -INFINITY ? 0.f : m;
      const float2 scale2 = splat2(a.scale_log2), base2 = splat2(-base);
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[32];
        uint32_t w[16];
        tmem_ld_32(t_s + c * 32, v);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const float2 y = fma2(make_float2(v[i], v[i + 1]), scale2, base2);
          float2 p = make_float2(ex2_approx(y.x), ex2_approx(y.y));
          if (valid < kTile) {
            if (c * 32 + i >= valid) p.x = 0.f;
            if (c * 32 + i + 1 >= valid) p.y = 0.f;
          }
          sum = add2(sum, p);
          w[i / 2] = pack_bf16x2(p.x, p.y);
        }
        tmem_st_16(t_s + c * 16, w);  // over columns whose scores have been read
      }
      l += sum.x + sum.y;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full0 + 8 * s);
    }
    if (ok && steps > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(o_full0 + 8 * s, 0, a.status));
      tc_fence_after();
    }
    // Streams of the same rows meet in the ring, which nobody uses any more once both have their outputs.
    constexpr int kPitch = D + 4;
    float* meet = reinterpret_cast<float*>(sm + S::kv_off);
    float2* meet_ml = reinterpret_cast<float2*>(meet + kTile * kPitch);
    static_assert((kTile * kPitch * 4 + kTile * 8) <= S::stages * S::kv_tile, "the meeting place fits the ring");
    if (!shared) {
      softmax_sync();
      if (s == 1) {
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float v[16];
          if (steps > 0) tmem_ld_16(t_o + c * 16, v);
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(meet + r * kPitch + c * 16 + i) =
                steps > 0 ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        meet_ml[r] = make_float2(m, l);
      }
      softmax_sync();
    }
    if (ok && (shared || s == 0)) {
      float f_mine = 1.f, f_met = 0.f;
      if (!shared) {
        const float2 met = meet_ml[r];
        const float to = fmaxf(m, met.x), base = to == -INFINITY ? 0.f : to;
        f_mine = ex2_approx(m - base);
        f_met = ex2_approx(met.x - base);
        l = l * f_mine + met.y * f_met;
        m = to;
      }
      const bool mine = row < n_rows;
      const long long at = static_cast<long long>(token_of(mine ? row : 0)) * a.heads + head_of(mine ? row : 0);
      const long long rows = static_cast<long long>(a.n) * a.heads;
      if (a.prefix_splits > 1) {
        float* out = a.part_o + (split * rows + at) * D;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float v[16];
          tmem_ld_16(t_o + c * 16, v);
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            float4 o = make_float4(v[i] * f_mine, v[i + 1] * f_mine, v[i + 2] * f_mine, v[i + 3] * f_mine);
            if (!shared) {
              const float4 x = *reinterpret_cast<const float4*>(meet + r * kPitch + c * 16 + i);
              o = make_float4(fmaf(x.x, f_met, o.x), fmaf(x.y, f_met, o.y), fmaf(x.z, f_met, o.z), fmaf(x.w, f_met, o.w));
            }
            if (mine) *reinterpret_cast<float4*>(out + c * 16 + i) = o;
          }
        }
        if (mine) a.part_ml[split * rows + at] = make_float2(m, l);
      } else {
        // the prefix in one piece: this block joins the rows with their own keys' pieces and finishes them
        float to = m;
        for (int p = 1; p < 1 + a.own_splits; ++p) to = fmaxf(to, mine ? a.part_ml[p * rows + at].x : -INFINITY);
        const float base = to == -INFINITY ? 0.f : to;
        const float f = ex2_approx(m - base);
        l *= f;
        f_mine *= f;
        f_met *= f;
        for (int p = 1; p < 1 + a.own_splits; ++p)
          if (mine) {
            const float2 ml = a.part_ml[p * rows + at];
            l = fmaf(ex2_approx(ml.x - base), ml.y, l);
          }
        const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          float v[16];
          tmem_ld_16(t_o + c * 16, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] *= f_mine;
          if (!shared) {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = fmaf(meet[r * kPitch + c * 16 + i], f_met, v[i]);
          }
          if (mine) {
            for (int p = 1; p < 1 + a.own_splits; ++p) {
              const float mp = a.part_ml[p * rows + at].x;
              if (mp == -INFINITY) continue;
              const float g = ex2_approx(mp - base);
              const float4* x = reinterpret_cast<const float4*>(a.part_o + (p * rows + at) * D + c * 16);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float4 y = x[i];
                v[4 * i] = fmaf(g, y.x, v[4 * i]);
                v[4 * i + 1] = fmaf(g, y.y, v[4 * i + 1]);
                v[4 * i + 2] = fmaf(g, y.z, v[4 * i + 2]);
                v[4 * i + 3] = fmaf(g, y.w, v[4 * i + 3]);
              }
            }
            uint4 w[2];
            uint32_t* u = reinterpret_cast<uint32_t*>(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = pack_bf16x2(v[2 * i] * inv, v[2 * i + 1] * inv);
            st_v4(a.o + at * D + c * 16, w[0]);
            st_v4(a.o + at * D + c * 16 + 8, w[1]);
          }
        }
        if (mine && a.lse) a.lse[at] = l > 0.f ? kLn2 * (to + log2f(l)) : -INFINITY;
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

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// The pool as (head_dim, heads, tokens, pages); boxes of 64 x 1 x min(page, 128) x 1.
bool pool_map(CUtensorMap* map, const __nv_bfloat16* base, const Args& a, int head_dim) {
  if (!encode_fn()) return false;
  const int page = 1 << a.page_shift;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(a.pages)};
  // an axis of one entry may have any stride: give the map one that it accepts
  auto stride = [](long long n, long long ld) { return static_cast<cuuint64_t>(n > 1 ? ld * 2 : 16); };
  const cuuint64_t strides[3] = {stride(a.kv_heads, a.head_ld), stride(page, a.token_ld), stride(a.pages, a.page_ld)};
  const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(page < kTile ? page : kTile), 1};
  const cuuint32_t each[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(base), dims, strides, box, each,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
cudaError_t launch(const Args& a, cudaStream_t stream) {
  CUtensorMap mk, mv;
  if (!pool_map(&mk, a.k, a, D) || !pool_map(&mv, a.v, a, D)) return cudaErrorInvalidValue;
  constexpr int bytes = Smem<D>::total;
  if (const cudaError_t e = cudaFuncSetAttribute(prefix_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      e != cudaSuccess)
    return e;
  prefix_tc_kernel<D><<<a.row_tiles * a.kv_heads * a.prefix_splits, kThreads, bytes, stream>>>(a, mk, mv);
  return cudaGetLastError();
}

}  // namespace tc

cudaError_t launch_prefix_tc(const Args& a, int head_dim, cudaStream_t stream) {
  return head_dim == 64 ? tc::launch<64>(a, stream) : tc::launch<128>(a, stream);
}

}  // namespace prefix

}  // namespace mnb
