// The shared prefix's part of the paged attention on the 5th-generation tensor
// cores over a cache in 8 bits.  prefix_attention_tc.cu has the scheme (two
// streams of 128 rows, scores, P and O in TMEM) and prefix_attention_8bit.cu the
// mathematics of scales and weights; here the two meet.
//
// Codes come page by page into a ring of raw tiles (128 keys, or their values); four
// warps widen those of keys and four those of values into the swizzled f16 tiles that the
// products read.  (Each group meets every phase of its barriers, in order: a wait by
// parity takes a barrier that is two phases behind for done.)  An f16 tile holds
// code * scale / R, with R the largest scale of the tile's pages: exact while the pages
// of 128 tokens next to one another have scales within a factor of 2^15 (2^17 for int8);
// a value of a page further below R is rounded to a multiple of R 2^-24.  R of the keys
// goes into the factor of the tile's scores, R of the values into their exponent,
//   s'_j = s_j + log2 R_v,  O = sum 2^(s'_j - base) (v_j / R_v),  sum_j 2^(s_j - base) = sum_j 2^(s'_j - base) / R_v,
// one number each for a tile, so the softmax costs what it costs without scales.  The base
// lies 7 below a maximum that scores may pass by 8, so a weight in f16 is at most 2^15.
// Both R come with a tile's keys, before its scores, and one warp makes factors of them.
//
// What bounds it: the widening and the softmax, which share the issue slots and the shared
// memory's bandwidth: 1.4 us for a tile of 128 keys whether one stream has rows or both,
// and 20 us before the first and after the last.  (With few rows raw tiles also lie where
// the second stream's queries would be, so that 64 KB are under way.)  Measured: 48 rows of
// 8 kv heads behind 100003 tokens 92 us (2.4 TB/s of codes), 160 rows of 16 heads behind
// 8003 tokens 86 us with their own keys, 1504 ragged rows of 32 heads 194 us with theirs.
// (The keys' raw tiles two or three deep, with one f16 tile of values less, changed nothing:
// 202 and 96 us.  The two halves of a row meeting alone, not their whole stream, neither.)
#include <type_traits>

#include "launch.cuh"
#include "prefix_attention_8bit.cuh"
#include "prefix_attention_tc.cuh"
#include "warp_mma.cuh"

namespace mnb {

namespace prefix {

namespace tc8 {

using namespace tc;
using namespace q8;

constexpr int kWiden = 256;  // threads that widen codes: keys and values by a group each, a thread a row of a tile
// Warp 0 loads keys, 2 values, 1 issues the products, 3 looks at scales, 4 to 19 do the softmax, 20 to 27 widen.  896 threads
// can have 72 registers each; the softmax takes over what the others do not need.
constexpr int kThreads = 128 + kSoftmax + kWiden, kFirst = 4;
constexpr int kLaunched = 72, kSmall = 48, kLarge = 88;
static_assert((kThreads - kSoftmax) * kSmall + kSoftmax * kLarge <= kThreads * kLaunched, "registers");
constexpr float kBelow = 7.f, kPass = 15.f;       // the base below the maximum, and what a score may lie above the base
constexpr int kInfo = 8;                          // tiles whose factors are kept

template <int D>
struct Smem {
  static constexpr uint32_t q_tile = kTile * D * 2;
  static constexpr uint32_t kv_tile = kTile * D * 2;
  static constexpr uint32_t raw_tile = kTile * D;
  static constexpr int stages = D == 128 ? 4 : 6;
  static constexpr int raws = D == 128 ? 2 : 4, more_raws = D == 128 ? 2 : 0;  // (with one tile of queries there is more room)
  static constexpr uint32_t q_off = 0, kv_off = 2 * q_tile, raw_off = kv_off + stages * kv_tile;
  static constexpr uint32_t bar_off = raw_off + raws * raw_tile;
  static constexpr int n_bars = 2 * stages + 3 * (raws + more_raws) + 10;
  static constexpr uint32_t max_off = bar_off + n_bars * 8 + 16;    // row maxima so far: [stream][row], as order_of()
  static constexpr uint32_t scale_off = max_off + 2 * kTile * 4;    // of the raw tiles' pages: [raw][keys, values][16]
  static constexpr uint32_t info_off = scale_off + (raws + more_raws) * 2 * 16 * 4;  // of tiles: a float4 each
  static constexpr uint32_t total = info_off + kInfo * 16 + 1024;
  static_assert(more_raws * raw_tile <= q_tile, "room");
  static_assert(total <= 227 * 1024, "a block's shared memory");
  static_assert(max_off % 16 == 0, "alignment");
  static_assert(kMeeting<D> <= stages * kv_tile + raws * raw_tile, "the meeting place fits the rings");
};

// Instruction descriptor for kind::f16 with f16 A/B and fp32 D.
constexpr uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn) { return idesc_bf16(m, n, a_mn, b_mn) & ~((1u << 7) | (1u << 10)); }

template <int D, bool kFloat>
__global__ void __launch_bounds__(kThreads, 1)
    prefix8_tc_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, int whole) {
  using S = Smem<D>;
  constexpr int kStages = S::stages;
  constexpr uint32_t kIdescS = idesc_f16(kTile, kTile, false, false);
  constexpr uint32_t kIdescO = idesc_f16(kTile, D, false, true);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(sm);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + S::bar_off);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::n_bars);
  constexpr int kMostRaws = S::raws + S::more_raws;
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kStages, raw_full0 = empty0 + 8 * kStages,
                 raw_empty0 = raw_full0 + 8 * kMostRaws, scaled0 = raw_empty0 + 8 * kMostRaws, q_full = scaled0 + 8 * kMostRaws,
                 s_full0 = q_full + 8,
                 o_full0 = s_full0 + 16, p_full0 = o_full0 + 16,  // (p_full: two halves per stream)
                 drained = p_full0 + 32;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // The first `whole` blocks take 256 rows, the others half as many (a short last wave: prefix_attention_tc.cu).
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
  // Rings of raw and of widened tiles: keys have the even places, values the odd ones.
  const int raw_shift = D == 128 && shared ? 0 : 1, raws = 1 << raw_shift;
  constexpr int kRing = kStages / 2;
  static_assert(S::raws == (D == 64 ? 4 : 2) && kMostRaws == 4 && kRing >= 2, "keys and values have half of them each");
  const int per_shift = min(a.page_shift, 7), per = 1 << per_shift;  // tokens of a box
  auto raw_at = [&](int r) { return r < S::raws ? S::raw_off + r * S::raw_tile : S::q_off + S::q_tile + (r - S::raws) * S::raw_tile; };
  auto valid_of = [&](int tile) { return min(kTile, k1 - k0 - tile * kTile); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, kTile / 32);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int r = 0; r < kMostRaws; ++r) {
      mbar_init(raw_full0 + 8 * r, 33);  // the expected bytes, and every lane's copies of scales
      mbar_init(raw_empty0 + 8 * r, kTile / 32);
      mbar_init(scaled0 + 8 * r, 1);
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
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  const uint32_t tmem = *tmem_slot;  // S_0, S_1: 128 columns each, then O_0, O_1

  if (warp < kFirst) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSmall));
    if (warp % 2 == 0) {
      const bool keys = warp == 0;
      const CUtensorMap* const map = keys ? &map_k : &map_v;
      // Page ids, 32 from `batch` on and the 32 after them, asked for long before they are needed: a trip to memory takes as
      // long as a tile.
      const int ids_end = ((k1 - 1) >> a.page_shift) + 1, in_page = (1 << a.page_shift) - 1;
      auto fetch = [&](int from) { return from + lane < ids_end ? a.prefix_pages[from + lane] : 0; };
      int batch = k0 >> a.page_shift, ids_now = fetch(batch), ids_next = fetch(batch + 32);
      int r = warp / 2;  // the raw tile's place
      uint32_t phase = 1;
      int t = 0;
      for (; t < n_tiles; ++t) {
        const int j0 = k0 + t * kTile, boxes = (valid_of(t) + per - 1) >> per_shift;
        const uint32_t bar = raw_full0 + 8 * r;
        if ((j0 >> a.page_shift) - batch >= 32) {
          batch += 32;
          ids_now = ids_next;
          ids_next = fetch(batch + 32);
        }
        int page = __shfl_sync(0xffffffffu, ids_now, ((j0 >> a.page_shift) - batch + lane) & 31);
        if (!warp_wait(raw_empty0 + 8 * r, phase, a.status)) break;
        if (lane == 0) mbar_arrive_expect_tx(bar, boxes * per * D);
        __syncwarp();
        if (lane < boxes) {
          const bool there = page >= 0 && page < a.pages;
          const long long at = there ? page * a.scale_ld + h * a.scale_head : 0;
          const uint32_t to = sbase + S::scale_off + (r * 2 * 16 + lane) * 4;
          if (!there) {
            atomicCAS(a.errors, 0, kErrBadIndex);
            page = a.no_page;  // reads as zeros
          }
          tma_load_4d(sbase + raw_at(r) + lane * per * D, map, 0, h, (j0 + lane * per) & in_page, page, bar);
          if (keys) copy_float(to, a.k_scales + at, there);
          copy_float(to + 64, a.v_scales + at, there);
        }
        arrive_after_copies(bar);
        if ((r += 2) >= 2 * raws) r -= 2 * raws, phase ^= 1;
      }
      // The block does not end before its last copies have arrived, also where another warp's wait was given up.
      for (int x = max(0, t - raws); x < t; ++x) mbar_wait(raw_full0 + 8 * (2 * (x % raws) + warp / 2), (x / raws) & 1, nullptr);
    } else if (warp == 1) {
      // Whether this lane's waits have all ended well.  The lanes agree on it once a step (`settle`): a vote at each wait made
      // the bf16 kernel 2 % slower, and what a step computes past a wait that was given up is in bounds.
      bool good = true;
      auto settle = [&] { return __all_sync(0xffffffffu, good); };
      auto keys_at = [&](int t) { return 2 * (t % kRing); };
      auto values_at = [&](int t) { return 2 * (t % kRing) + 1; };
      auto wait_full = [&](int st, int t) {
        good = mbar_wait(full0 + 8 * st, (t / kRing) & 1, a.status) && good;
        tc_fence_after();
      };
      // (adding bytes / 16 to a descriptor moves its address: the tiles lie below 256 KB, so nothing carries)
      const uint64_t q_desc = smem_desc_sw128(sbase + S::q_off, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(sbase + S::kv_off, 16, 1024);
      const uint64_t v_desc = smem_desc_sw128(sbase + S::kv_off, kTile * 128, 1024);
      // S_s = Q_s K^T
      auto scores = [&](int s, int t) {
        const uint64_t qa = q_desc + (shared ? s : 0) * (S::q_tile / 16), kb = k_desc + static_cast<uint64_t>(keys_at(t)) * (S::kv_tile / 16);
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
      auto values = [&](int s, int t, int step) {
        const uint64_t vb = v_desc + static_cast<uint64_t>(values_at(t)) * (S::kv_tile / 16);
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
      auto commit = [&](uint32_t bar) {
        if (elected()) tc_commit(bar);
        __syncwarp();
      };
      bool ok = warp_wait(q_full, 0, a.status);
      tc_fence_after();
      if (shared) {
        if (ok) {
          wait_full(keys_at(0), 0);
          scores(0, 0);
          scores(1, 0);
          commit(empty0 + 8 * keys_at(0));
          ok = settle();
        }
        for (int t = 0; t < n_tiles && ok; ++t) {
          const bool more = t + 1 < n_tiles;
          wait_full(values_at(t), t);
          values(0, t, t);
          if (more) {
            wait_full(keys_at(t + 1), t + 1);
            scores(0, t + 1);
          } else {
            commit(o_full0);
          }
          values(1, t, t);
          commit(empty0 + 8 * values_at(t));
          if (more) {
            scores(1, t + 1);
            commit(empty0 + 8 * keys_at(t + 1));
          } else {
            commit(o_full0 + 8);
          }
          ok = settle();
        }
      } else {
        auto next_scores = [&](int t) {
          wait_full(keys_at(t), t);
          scores(t & 1, t);
          commit(empty0 + 8 * keys_at(t));
        };
        if (ok) next_scores(0);
        if (n_tiles > 1 && ok) next_scores(1);
        ok = settle() && ok;
        for (int t = 0; t < n_tiles && ok; ++t) {
          const int s = t & 1;
          wait_full(values_at(t), t);
          values(s, t, t >> 1);
          commit(empty0 + 8 * values_at(t));
          if (t + 2 < n_tiles) next_scores(t + 2);
          else commit(o_full0 + 8 * s);
          ok = settle();
        }
      }
      if (!ok) {  // a wait was given up: nor do products end after their TMEM is freed
        commit(drained);
        mbar_wait(drained, 0, nullptr);
      }
    } else {
      // Scales become the factors of the pages' codes, in place, and the tile's own go to its info.
      int r = 0;
      uint32_t phase = 0;
      float top_v = 0.f;
      for (int t = 0, part = 0; t < n_tiles;) {
        if (!warp_wait(raw_full0 + 8 * (r + part), phase, a.status)) break;
        float* const scales = reinterpret_cast<float*>(sm + S::scale_off) + (r + part) * 2 * 16;
        const int boxes = (valid_of(t) + per - 1) >> per_shift;
        auto largest = [&](float x) {  // of the pages' scales, and at least the least
          const float mine = lane < boxes ? fmaxf(x, kLeastScale) : kLeastScale;  // (also for what is no number)
          return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mine)));
        };
        const float x = scales[part * 16 + (lane & 15)];
        const float top = part ? top_v : largest(x);
        if (!part) top_v = largest(scales[16 + (lane & 15)]);
        __syncwarp();
        if (lane < boxes) scales[part * 16 + lane] = (part ? fmaxf(x, kLeastScale) : x) * rcp_approx(top);
        if (!part && lane == 0) {
          const float b = __log2f(top_v);
          *reinterpret_cast<float4*>(sm + S::info_off + t % kInfo * 16) = make_float4(fminf(top, 3.4e38f) * a.scale_log2, b, ex2_approx(15.f - b), 0.f);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(scaled0 + 8 * (r + part));
        part ^= 1;
        if (part == 0) {
          ++t;
          if ((r += 2) >= 2 * raws) r = 0, phase ^= 1;
        }
      }
    }
  } else if (warp >= kFirst + kSoftmax / 32) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSmall));
    // Widening: a thread has a row of the tile, so one scale.  (Every warp meets every phase of its barriers: one that took
    // tiles out of turn could take a barrier two phases behind for one that is done.)
    const int self = threadIdx.x - (kThreads - kWiden), row = self % kTile, group = self / kTile;
    int r = group, st = group;
    uint32_t raw_phase = 0, phase = 1;
    for (int t = 0; t < n_tiles; ++t) {
      const int valid = valid_of(t);
      // (the factors come from a warp that has waited for the codes)
      if (!warp_wait(scaled0 + 8 * r, raw_phase, a.status)) break;
      const float* const factors = reinterpret_cast<const float*>(sm + S::scale_off) + (r * 2 + group) * 16;
      const float factor = factors[min(row, valid - 1) >> per_shift];
      const uint32_t by = pack_f16x2(factor, factor);
      // int8: (1024 + u) by - 1152 by in one step, which is exact where `by` is a power of two
      const uint32_t less = mul_f16x2(by, 0xe480e480u);
      const bool powers = kFloat || __all_sync(0xffffffffu, (__float_as_uint(factor) & 0x7fffff) == 0);
      const bool there = row < valid;
      const uint8_t* const from = sm + raw_at(r) + row * D;
      uint8_t* const to = sm + S::kv_off + st * S::kv_tile + row * 128;
      const int turn_in = D == 128 ? row & 7 : (row >> 1) & 3, turn_out = row & 7;
      uint4 w[4];
      auto load = [&](int c0) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = ld_v4(from + (((c0 + k) ^ turn_in) << 4));
        if (!there) w[0] = w[1] = w[2] = w[3] = make_uint4(0, 0, 0, 0);  // past the end a page holds anything
      };
      load(0);  // (on their way while the f16 tile's place is waited for)
      if (!warp_wait(empty0 + 8 * st, phase, a.status)) break;
      auto widen_row = [&](auto by_powers) {
#pragma unroll
        for (int c0 = 0; c0 < D / 16; c0 += 4) {
          if (c0 > 0) load(c0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t y[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t v = (&w[k].x)[e];
              if constexpr (kFloat) {
                widen_any<true>(v, y[2 * e], y[2 * e + 1]);  // (in the bytes' order)
                y[2 * e] = mul_f16x2(y[2 * e], by), y[2 * e + 1] = mul_f16x2(y[2 * e + 1], by);
              } else {
                v ^= 0x80808080u;
                y[2 * e] = __byte_perm(v, 0x64646464u, 0x4140), y[2 * e + 1] = __byte_perm(v, 0x64646464u, 0x4342);
                if constexpr (decltype(by_powers)::value) {
                  y[2 * e] = fma_f16x2(y[2 * e], by, less), y[2 * e + 1] = fma_f16x2(y[2 * e + 1], by, less);
                } else {
                  y[2 * e] = mul_f16x2(sub_f16x2(y[2 * e], 0x64806480u), by);
                  y[2 * e + 1] = mul_f16x2(sub_f16x2(y[2 * e + 1], 0x64806480u), by);
                }
              }
            }
            // (dims 16 c on: chunks 2 c and 2 c + 1 of 8 values, eight of them to a 128-byte row)
            uint8_t* const at = to + c0 / 4 * (kTile * 128);
            const int first = (2 * k) ^ turn_out;
            st_v4(at + (first << 4), make_uint4(y[0], y[1], y[2], y[3]));
            st_v4(at + ((first ^ 1) << 4), make_uint4(y[4], y[5], y[6], y[7]));
          }
        }
      };
      if (kFloat || powers) widen_row(std::true_type{});
      else widen_row(std::false_type{});
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full0 + 8 * st);
        mbar_arrive(raw_empty0 + 8 * r);
      }
      if ((r += 2) >= 2 * raws) r -= 2 * raws, raw_phase ^= 1;
      if ((st += 2) >= kStages) st -= kStages, phase ^= 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kLarge));
    const int s = (warp - kFirst) / 8, half = (warp - kFirst) / 4 % 2, quad = warp % 4;
    const int r = quad * 32 + lane;                 // row of the stream's tile
    float* const row_back = reinterpret_cast<float*>(sm + S::max_off);
    {  // Q as f16, each row times a power of two, swizzled as TMA would leave it; rows past the last are zeros
      constexpr int kChunks = D / 8, kStep = kSoftmax / kChunks, kAhead = 8;  // a thread keeps its chunk and goes through the rows
      const int c = (threadIdx.x - 32 * kFirst) % kChunks, rows_end = shared ? 2 * kTile : kTile;
      // (a row's token and which head of the group: kStep rows further without a division each)
      int i0 = (threadIdx.x - 32 * kFirst) / kChunks, token = (r0 + i0) / a.group, member = r0 + i0 - token * a.group;
      const int tokens_on = kStep / a.group, members_on = kStep - tokens_on * a.group;
      for (; i0 < rows_end; i0 += kStep * kAhead) {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          w[k] = make_uint4(0, 0, 0, 0);
          if (i0 + k * kStep < n_rows) w[k] = ld_v4(a.q + token * a.q_ld + (h * a.group + member) * a.q_head + c * 8);
          token += tokens_on, member += members_on;
          if (member >= a.group) ++token, member -= a.group;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * kStep, x = i % kTile;
          uint32_t top = 0;  // of the finite values, as bits
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = (&w[k].x)[e], lo = v & 0x7fffu, hi = v >> 16 & 0x7fffu;
            top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
          }
#pragma unroll
          for (int o = 1; o < kChunks; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int shift = min(141 - static_cast<int>(top >> 7), 126);  // the largest becomes 2^14 to 2^15
          const float up = __int_as_float((127 + shift) << 23);
          uint32_t y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = mul2(unpack_bf16x2((&w[k].x)[e]), splat2(up));
            y[e] = pack_f16x2(v.x, v.y);
          }
          if (i < rows_end) {
            *reinterpret_cast<uint4*>(sm + S::q_off + (i / kTile) * S::q_tile + (c / 8) * (kTile * 128) + x * 128 + (((c % 8) ^ (x % 8)) << 4)) =
                make_uint4(y[0], y[1], y[2], y[3]);
            if (c == 0) row_back[i] = __int_as_float((127 - shift) << 23);
          }
        }
      }
      fence_async_smem();
      mbar_arrive(q_full);
    }
    softmax_sync();
    const float back = row_back[(shared ? s * kTile : 0) + r];
    softmax_sync();
    volatile int* seen = reinterpret_cast<int*>(sm + S::max_off) + s * kTile + r;
    if (half == 0) *seen = order_of(-INFINITY);
    stream_sync(s);
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t t_s = tmem + s * kTile + lanes, t_o = tmem + 2 * kTile + s * D + lanes;
    const int steps = shared ? n_tiles : (n_tiles - s + 1) / 2;
    const bool padding = (shared ? s * kTile : 0) + quad * 32 >= n_rows;  // a warp without rows leaves P as it is
    float m = -INFINITY, l = 0.f;  // the base, and the sum (times 2^15)
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
      const int tile = shared ? t : 2 * t + s;
      const int valid = k1 - k0 - tile * kTile - half * 64;  // keys of this half tile (or more, or none)
      const float4 info = *reinterpret_cast<const float4*>(sm + S::info_off + tile % kInfo * 16);
      // (towards zero, so that past fp32's range it stays finite and 0 times it 0; above 0, so that masked scores stay -inf)
      const float factor = fmaxf(__fmul_rz(info.x, back), 1.2e-38f);
      float v[64];
      tmem_ld_32(t_s + half * 64, v);
      tmem_ld_32(t_s + half * 64 + 32, v + 32);
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
      atomicMax(const_cast<int*>(seen), order_of(valid > 0 ? fmaf(mx, factor, info.y) : -INFINITY));
      tc_fence_before();
      stream_sync(s);
      tc_fence_after();
      mx = of_order(*seen);
      const bool grows = !(mx <= m + kPass) || m == -INFINITY;
      if (__any_sync(0xffffffffu, grows)) {
        const float to = grows ? mx - kBelow : m;
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
      float2 scale2 = splat2(factor);
      float2 base2 = splat2(m == -INFINITY ? 0.f : info.y - m);
      if (__any_sync(0xffffffffu, fabsf(m) >= 16777216.f)) {
        // Here rounding a scaled score moves it by whole units, and by more than a float's range later: round the scores as
        // their maximum was.
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = i >= valid ? -INFINITY : fmaf(v[i], factor, info.y);
        scale2 = splat2(1.f);
        base2 = splat2(m == -INFINITY ? 0.f : -m);
      }
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float2 y = fma2(make_float2(v[c * 16 + i], v[c * 16 + i + 1]), scale2, base2);
          // one pair of eight on the FMA pipe, as in the bf16 kernel, where both streams keep the exponential unit busy
          const float2 p = i == 6 && shared ? exp2_fma(y) : make_float2(ex2_approx(y.x), ex2_approx(y.y));
          sum = add2(sum, p);
          w[i / 2] = pack_f16x2(p.x, p.y);
        }
        tmem_st_8(t_s + half * 32 + c * 8, w);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(p_full0 + 16 * s + 8 * half);
      l = fmaf(sum.x + sum.y, info.z, l);
    }
    if (steps > 0) {
      mbar_wait(o_full0 + 8 * s, 0, a.status);
      __syncwarp();
      tc_fence_after();
    }
    finish_rows<D, 4>(a, sm + S::kv_off, t_o, m, l * 3.0517578125e-5f, steps, s, half, r, warp - kFirst, n_rows, r0, h, split, shared);
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, bool kFloat>
static cudaError_t launch(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  constexpr int bytes = Smem<D>::total;
  static SharedMemory allowed;
  if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(prefix8_tc_kernel<D, kFloat>), bytes); e != cudaSuccess) return e;
  const int units = a.row_tiles * a.kv_heads * a.prefix_splits, last = units % 148;
  const int whole = a.prefix_splits == 1 && 2 * last <= 148 ? units - last : units;
  const int blocks = whole + 2 * (units - whole);
  if (a.own_splits > 0) return launch_after(prefix8_tc_kernel<D, kFloat>, blocks, kThreads, bytes, stream, a, mk, mv, whole);
  prefix8_tc_kernel<D, kFloat><<<blocks, kThreads, bytes, stream>>>(a, mk, mv, whole);
  return cudaGetLastError();
}

}  // namespace tc8

cudaError_t launch_prefix_tc8(const Args& a, int head_dim, cudaStream_t stream) {
  CUtensorMap mk, mv;
  if (!q8::codes_map(&mk, a.k8, a, head_dim, tc::kTile) || !q8::codes_map(&mv, a.v8, a, head_dim, tc::kTile)) return cudaErrorInvalidValue;
  if (a.codes == kE4m3) return head_dim == 64 ? tc8::launch<64, true>(a, mk, mv, stream) : tc8::launch<128, true>(a, mk, mv, stream);
  return head_dim == 64 ? tc8::launch<64, false>(a, mk, mv, stream) : tc8::launch<128, false>(a, mk, mv, stream);
}

}  // namespace prefix

}  // namespace mnb
