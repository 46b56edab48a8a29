// Attention of new tokens over a prefix that every sequence of the batch
// shares and over each sequence's own tokens, both in a paged cache.
//
//   o_r = sum_j exp(s_rj - lse_r) v_j,   s_rj = scale q_r . k_j,
//   lse_r = log sum_j exp(s_rj),         j over prefix and own tokens.
//
// The softmax splits over any partition of the keys: a part contributes its
// maximum m, its sum l = sum exp(s - m) and its unnormalised output
// sum exp(s - m) v, and parts are joined under the common maximum.  So the
// prefix is one product for the rows of ALL sequences (its keys and values
// are read once for the batch, not once for each sequence), each sequence's
// own keys are another part, and both are split along the keys into enough
// pieces to fill the GPU.  A second kernel joins the pieces.
//
// Decoding is bound by the bytes of keys and values.  Blocks of four working
// warps and a loading one go through a list of pieces: the loading warp fills
// a ring of 64-key stages of K and V through a TMA map of the pool (page by
// page, 128-byte swizzle), on into the next piece while the others still work
// on this one, so loads never wait for a piece to end.  The working warps hold
// scores and probabilities in registers (mma.sync m16n8k16); the query rows of
// the heads of one kv head (grouped heads) share a tile of 16, 32 or 64 rows,
// and warps without rows of their own split the keys of a stage.
// Scores, maxima, sums and outputs are fp32; only the probabilities are
// rounded to bf16, as the operand of the product with V.  Many rows go to the
// tensor-core kernel of prefix_attention_tc.cu, which follows the same scheme.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "generation.h"
#include "launch.cuh"
#include "warp_mma.cuh"

namespace mnb {

namespace prefix {

constexpr int kWorkers = 128;
constexpr int kThreads = kWorkers + 32;
constexpr int kKeys = 64;            // keys per stage
constexpr int kTensorCoreRows = 32;  // more rows of a kv head than this go to the tensor-core kernel
constexpr float kLn2 = 0.6931471805599453f;

template <int D, int WR>
struct Ring {
  // Head dim 128: three blocks with two stages fit an SM, or two (tiles of 64 rows need the registers) with three.
  static constexpr int stages = D == 128 ? (WR == 4 ? 3 : 2) : D == 64 ? 3 : 4;
  static constexpr uint32_t tile = kKeys * D * 2;                // of K; V follows
  static constexpr uint32_t bytes = stages * 2 * tile;
  // 16-byte chunk c of row r, as TMA's swizzle leaves it
  MNB_DEVICE static uint32_t at(int r, int c) {
    if (D == 32) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
    return (c / 8) * (kKeys * 128) + r * 128 + (((c % 8) ^ (r % 8)) << 4);
  }
};

MNB_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
MNB_DEVICE void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// One piece: rows r0 .. r0 + n_rows of the rows that start at token n0 (row r is token n0 + r / group, head
// h * group + r % group) over keys [k0, k1) in the pages `ids`.  Row r sees those below limit0 + r / group.
struct Piece {
  int h, n0, r0, n_rows, k0, k1, slot, limit0;
  const int* ids;
};
constexpr int kUnlimited = 1 << 30;

MNB_DEVICE void flag(const Args& a) { atomicCAS(a.errors, 0, kErrBadIndex); }

// Whether q_offsets ascend from 0 to n in steps of at most max_q; for all lanes of a warp.
MNB_DEVICE bool offsets_sound(const Args& a, const int* q_offsets) {
  bool bad = false;
  for (int b = threadIdx.x % 32; b <= a.batch; b += 32) {
    const long long from = q_offsets[b];
    if (b == 0) bad = bad || from != 0;
    if (b == a.batch) bad = bad || from != a.n;
    else bad = bad || q_offsets[b + 1] < from || q_offsets[b + 1] - from > a.max_q;
  }
  return !__any_sync(0xffffffffu, bad);
}

// Item i of the list: first the prefix's (split, kv head, row tile; the row tiles of the same keys side by side), then
// the sequences' own (sequence, row tile, split, kv head).
// With `heads` of 4 an own piece is that of four kv heads, from p.h on.
MNB_DEVICE Piece piece_of(const Args& a, const int* seq_lens, const int* q_offsets, int i, int tile_rows, int heads) {
  Piece p;
  const int of_prefix = a.tensor_cores ? 0 : a.row_tiles * a.kv_heads * a.prefix_splits;
  if (i < of_prefix) {
    const int split = i / (a.row_tiles * a.kv_heads);
    p.h = (i / a.row_tiles) % a.kv_heads;
    p.n0 = 0;
    p.r0 = (i % a.row_tiles) * tile_rows;
    p.n_rows = min(tile_rows, a.n * a.group - p.r0);
    p.k0 = split * a.prefix_chunk;
    p.k1 = min(a.prefix_len, p.k0 + a.prefix_chunk);
    p.slot = split;
    p.limit0 = kUnlimited;
    p.ids = a.prefix_pages;
    return p;
  }
  i -= of_prefix;
  const int groups = (a.kv_heads + heads - 1) / heads;
  p.h = i % groups * heads;
  const int split = (i / groups) % a.own_splits;
  const int rt = (i / (groups * a.own_splits)) % a.own_tiles;
  const int b = i / (groups * a.own_splits * a.own_tiles);
  p.n0 = b;
  int q_len = 1;
  if (a.q_offsets) {
    // (within the rows whatever the offsets say: offsets_sound() has the word on them)
    p.n0 = min(max(q_offsets[b], 0), a.n);
    q_len = min(min(max(q_offsets[b + 1], 0), a.n) - p.n0, a.max_q);
    q_len = max(q_len, 0);
  }
  p.r0 = rt * tile_rows;
  p.n_rows = min(tile_rows, q_len * a.group - p.r0);
  int len = seq_lens[b];
  if (len < 0 || len > a.max_len) {
    flag(a);
    len = 0;  // the sequence's own tokens are left out
  }
  p.limit0 = len - q_len + 1;
  p.k0 = split * a.own_chunk;
  // the newest row of the tile sees the most keys
  p.k1 = p.n_rows > 0 ? min(min(len, max(0, p.limit0 + (p.r0 + p.n_rows - 1) / a.group)), p.k0 + a.own_chunk) : p.k0;
  p.slot = a.prefix_splits + split;
  p.ids = a.page_table + b * a.table_ld;
  return p;
}

// The rows of a block's pieces that are not finite, computed again key by key.  A product over a tile gives a hidden key
// weight 0, and 0 times a value that is no number is NaN; here each row takes only what it sees.  (A row that sees such a
// value comes out as it was.)  Maxima and sums are right already.
template <int D>
__device__ __noinline__ void rows_again(const Args& a, const int* seq_lens, const int* q_offsets, int items, int tile_rows, int heads) {
  constexpr int kPer = D / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    const Piece p = piece_of(a, seq_lens, q_offsets, i, tile_rows, heads);
    if (p.limit0 + p.r0 / a.group >= p.k1) continue;  // every row sees every key
    for (int x = warp; x < p.n_rows * heads; x += kWorkers / 32) {
      const int r = x / heads, head = p.h + x % heads, j = p.r0 + r, token = j / a.group, in_group = j - token * a.group;
      if (head >= a.kv_heads) continue;
      const long long out = (static_cast<long long>(p.slot) * a.n + p.n0 + token) * a.heads + head * a.group + in_group;
      float* to = a.part_o + out * D + lane * kPer;
      float zero = 0.f;
#pragma unroll
      for (int c = 0; c < kPer; ++c) zero = fmaf(to[c], 0.f, zero);
      if (!__any_sync(0xffffffffu, zero != 0.f)) continue;
      const float m = a.part_ml[out].x, base = m == -INFINITY ? 0.f : m;
      const __nv_bfloat16* q = a.q + (p.n0 + token) * a.q_ld + (head * a.group + in_group) * a.q_head + lane * kPer;
      float o[kPer] = {};
      for (int key = p.k0; key < min(p.k1, p.limit0 + token); ++key) {
        const int page = p.ids[key >> a.page_shift];
        if (page < 0 || page >= a.pages) continue;  // reads as zeros
        const long long at = page * a.page_ld + (key & ((1 << a.page_shift) - 1)) * a.token_ld + head * a.head_ld + lane * kPer;
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) s = fmaf(bf16_to_f32(q[c]), bf16_to_f32(a.k[at + c]), s);
        const float w = ex2_approx(warp_sum(s) * a.scale_log2 - base);
#pragma unroll
        for (int c = 0; c < kPer; ++c) o[c] = fmaf(w, bf16_to_f32(a.v[at + c]), o[c]);
      }
#pragma unroll
      for (int c = 0; c < kPer; ++c) to[c] = o[c];
    }
  }
}

// WR: warps that take rows of their own (16 each); the 4 / WR groups of warps split the keys of a stage.
//
// Measured: 192 sequences of 1 to 401 tokens, 16 heads of 128, one row each (314 MB): 72 us, 4.4 TB/s; all of them 384
// long (604 MB): 104 us, 5.8 TB/s, so what short sequences lose is the last stage of each, which costs a warp as much
// as a full one (some 400 instructions at 1.5 a cycle).  Blocks fetching their pieces from the hardware's work queue
// instead of in turn were no faster, and neither were keys laid out head by head.  2388 rows of 24 sequences in tiles
// of 64 (masked triangles): 78 us under ncu (88 with the keys
// that a warp's rows do not see computed too), bound by the latency of eight working warps per SM.
//
// Quad: a piece is four kv heads of one sequence, a stage 16 keys of each, and every warp works on a head of its own,
// without a join: what a piece costs beside its keys is spent once for four heads, which decides where many sequences
// are short (2048 sequences of 4 tokens, 16 heads, behind a prefix of 64: the
// call 261 us without, 86 with).
//
// Chunk: sequences may have several new tokens, and rows not see all the keys of their piece.
template <int D, int WR, bool Quad, bool Chunk>
__global__ void __launch_bounds__(kThreads, WR == 4 ? 2 : 3)
    pieces_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, int items, int join_rows, int known) {
  using R = Ring<D, WR>;
  constexpr int WK = Quad ? 1 : 4 / WR, KW = Quad ? 16 : kKeys / WK, kStages = R::stages, kPitch = D + 4;
  // Tiles of 64 rows of one kv head hold triangles: a warp leaves out the keys that none of its 16 rows sees (16 x 512
  // tokens, 16 heads of 128: 65.6 us with, 69.2 without; 9 x 65 tokens of 24 heads 26.2 and 28.8).  Not at head dim 64
  // (44.8 and 43.6) nor in smaller tiles, where it costs registers (192 single tokens 99 and 95).
  constexpr bool kSkip = WR == 4 && D == 128;
  constexpr int kStep = Quad ? 16 : kKeys, kHeads = Quad ? 4 : 1;  // keys and heads of a stage; head y's keys are rows 16 y on
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * kStages];
  __shared__ int again;  // some row has to be computed again
  const uint32_t ring = smem_u32(sm), full0 = smem_u32(bars), empty0 = full0 + 8 * kStages;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    again = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 4);
    }
    fence_mbar_init();
  }
  // The sequences' lengths, for short lists (`known` of them): finding a piece then costs no trip to memory.
  int* lens = reinterpret_cast<int*>(sm + R::bytes + WK * join_rows * (kPitch * 4 + 8));
  int* offsets = lens + known;
  for (int b = threadIdx.x; b < known; b += kThreads) lens[b] = a.seq_lens[b];
  if (a.q_offsets)
    for (int b = threadIdx.x; b < known + (known > 0); b += kThreads) offsets[b] = a.q_offsets[b];
  const int* const seq_lens = known ? lens : a.seq_lens;
  const int* const q_offsets = known ? offsets : a.q_offsets;
  __syncthreads();
  int pos = 0;  // stages filled, or used, so far
  let_next_start();

  if (warp == 4) {
    const int per = min(1 << a.page_shift, kStep);  // tokens of a box
    const int box = lane / kHeads, head = lane % kHeads;
    bool ok = true;
    for (int i = blockIdx.x; i < items && ok; i += gridDim.x) {
      const Piece p = piece_of(a, seq_lens, q_offsets, i, 16 * WR, kHeads);
      const int heads = min(kHeads, a.kv_heads - p.h);
      for (int j0 = p.k0; j0 < p.k1; j0 += kStep, ++pos) {
        const int st = pos % kStages, boxes = (min(kStep, p.k1 - j0) + per - 1) / per;
        int page = 0;
        const int j = j0 + box * per;
        const bool mine = box < boxes && head < heads;
        if (mine) {
          page = p.ids[j >> a.page_shift];
          if (page < 0 || page >= a.pages) {
            flag(a);
            page = a.no_page;
          }
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * st, ((pos / kStages) & 1) ^ 1, a.status)))) break;
        if (lane == 0) mbar_arrive_expect_tx(full0 + 8 * st, boxes * per * heads * D * 4);
        __syncwarp();
        if (mine) {
          const uint32_t to = ring + st * 2 * R::tile + (head * kStep + box * per) * (D == 32 ? 64 : 128);
#pragma unroll
          for (int c = 0; c < (D + 63) / 64; ++c) {
            const int token = j & ((1 << a.page_shift) - 1);
            tma_load_4d(to + c * (kKeys * 128), &map_k, c * 64, p.h + head, token, page, full0 + 8 * st);
            tma_load_4d(to + R::tile + c * (kKeys * 128), &map_v, c * 64, p.h + head, token, page, full0 + 8 * st);
          }
        }
      }
    }
    // The block does not end before its last copies have arrived, also where a worker's wait was given up.
    for (int k = max(0, pos - kStages); k < pos; ++k) mbar_wait(full0 + 8 * (k % kStages), (k / kStages) & 1, nullptr);
    if (a.sound && blockIdx.x == 0) {  // (here because nobody waits for this warp any more)
      const bool sound = offsets_sound(a, q_offsets);
      if (lane == 0) {
        *a.sound = sound;
        if (!sound) flag(a);
      }
    }
    return;
  }

  const int wk = Quad ? 0 : warp / WR, gq = lane / 4, tg = lane % 4;
  const int row0 = Quad ? warp * 16 : wk * KW;  // of this warp's keys in a stage
  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    const Piece p = piece_of(a, seq_lens, q_offsets, i, 16 * WR, kHeads);
    if (p.n_rows <= 0) continue;
    const int wr = Quad ? 0 : (kSkip ? warp + pos : warp) % WR;  // rows in turn: a triangle's last ones have the most keys
    const int head = Quad ? p.h + warp : p.h;
    const bool idle = Quad && head >= a.kv_heads;  // the last four heads may be fewer
    auto out_of = [&](int r) {
      const int j = p.r0 + r, token = j / a.group;
      return (static_cast<long long>(p.slot) * a.n + p.n0 + token) * a.heads + head * a.group + j - token * a.group;
    };
    if (p.k1 <= p.k0) {  // nothing here: the join skips the piece
      if (!idle)
        for (int r = Quad ? lane : threadIdx.x; r < p.n_rows; r += Quad ? 32 : kWorkers) a.part_ml[out_of(r)] = make_float2(-INFINITY, 0.f);
      continue;
    }
    // Q as the products' first operand, straight from memory
    uint32_t qf[D / 16][4];
    int lim[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = wr * 16 + gq + 8 * e, j = p.r0 + r, token = j / a.group;
      const bool in = r < p.n_rows && !idle;
      lim[e] = min(p.k1, p.limit0 + token);
      const __nv_bfloat16* q = a.q + (p.n0 + token) * a.q_ld + (head * a.group + j - token * a.group) * a.q_head + 2 * tg;
#pragma unroll
      for (int kc = 0; kc < D / 16; ++kc) {
        qf[kc][e] = in ? *reinterpret_cast<const uint32_t*>(q + kc * 16) : 0u;
        qf[kc][e + 2] = in ? *reinterpret_cast<const uint32_t*>(q + kc * 16 + 8) : 0u;
      }
    }
    float acc[D / 8][4];
#pragma unroll
    for (int d = 0; d < D / 8; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.f;
    float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.f, 0.f};
    // the end of the keys that any of this warp's rows sees
    const int top = !kSkip ? p.k1 : wr * 16 < p.n_rows ? min(p.k1, p.limit0 + (p.r0 + min(wr * 16 + 15, p.n_rows - 1)) / a.group) : p.k0;
    const bool lower = p.n_rows > wr * 16 + 8;  // whether the tile's rows 8 to 15 are any of ours

    for (int t0 = p.k0; t0 < p.k1; t0 += kStep, ++pos) {
      const int st = pos % kStages;
      mbar_wait(full0 + 8 * st, (pos / kStages) & 1, a.status);  // (a wait that gave up is in the status word)
      __syncwarp();
      const uint32_t sK = ring + st * 2 * R::tile, sV = sK + R::tile;
      const int key0 = Quad ? t0 : t0 + wk * KW;  // this warp's first key
      const int live = top - key0;
      if (idle || (kSkip && live <= 0)) {
        if (lane == 0) mbar_arrive(empty0 + 8 * st);
        continue;
      }
      const bool part = p.k1 - t0 < kStep;
      if (part) {  // V rows past the end hold anything: this warp's become zeros
        for (int x = lane; x < KW * (D / 8); x += 32) {
          const int r = x / (D / 8);
          if (key0 + r >= p.k1) st_v4(sm + st * 2 * R::tile + R::tile + R::at(row0 + r, x % (D / 8)), make_uint4(0, 0, 0, 0));
        }
        __syncwarp();
      }
      float s[KW / 8][4];
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        if (kSkip && n * 16 >= live) break;
#pragma unroll
        for (int kc = 0; kc < D / 16; ++kc) {
          uint32_t b[4];
          ldsm_x4(b, sK + R::at(row0 + n * 16 + (lane & 7) + (lane >> 4) * 8, kc * 2 + ((lane >> 3) & 1)));
          mma_bf16(s[2 * n], qf[kc], b);
          mma_bf16(s[2 * n + 1], qf[kc], b + 2);
        }
      }
      const int j0 = key0 + 2 * tg;
      float mx[2] = {m_r[0], m_r[1]};
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + n * 8 + (e & 1);
          s[n][e] = j < lim[e >> 1] ? s[n][e] * a.scale_log2 : -INFINITY;
          mx[e >> 1] = fmaxf(mx[e >> 1], s[n][e]);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e == 1 && !lower) break;  // (their weights stay at the scores, which nobody reads)
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
        const float base = mx[e] == -INFINITY ? 0.f : mx[e];  // no key yet: every weight is exp2(-inf) = 0
        const float alpha = ex2_approx(m_r[e] - base);
        m_r[e] = mx[e];
        if (__any_sync(0xffffffffu, alpha != 1.f)) {  // some row of the warp has a new maximum
          l_r[e] *= alpha;
#pragma unroll
          for (int d = 0; d < D / 8; ++d) {
            acc[d][2 * e] *= alpha;
            acc[d][2 * e + 1] *= alpha;
          }
        }
#pragma unroll
        for (int n = 0; n < KW / 8; ++n)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float w = ex2_approx(s[n][2 * e + x] - base);
            s[n][2 * e + x] = w;
            l_r[e] += w;
          }
      }
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        if (kSkip && n * 16 >= live) break;
        const uint32_t pa[4] = {pack_bf16x2(s[2 * n][0], s[2 * n][1]), pack_bf16x2(s[2 * n][2], s[2 * n][3]),
                                pack_bf16x2(s[2 * n + 1][0], s[2 * n + 1][1]), pack_bf16x2(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t b[4];
          ldsm_x4_t(b, sV + R::at(row0 + n * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, d * 2 + (lane >> 4)));
          mma_bf16(acc[2 * d], pa, b);
          mma_bf16(acc[2 * d + 1], pa, b + 2);
        }
      }
      if (part) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes over the zeros next
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * st);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l_r[e] += __shfl_xor_sync(0xffffffffu, l_r[e], 1);
      l_r[e] += __shfl_xor_sync(0xffffffffu, l_r[e], 2);
    }
    // A row that does not see all the keys here and holds something that is no number is computed again.
    if (Chunk && __any_sync(0xffffffffu, min(lim[0], lim[1]) < p.k1) && !idle) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e == 1 && !lower) break;
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int d = 0; d < D / 8; ++d) sum = add2(sum, make_float2(acc[d][2 * e], acc[d][2 * e + 1]));
        if (lim[e] < p.k1 && !(fabsf(sum.x + sum.y) < INFINITY)) again = 1;
      }
    }
    if constexpr (WK > 1) {
      // the key groups of a row join through shared memory
      float* so = reinterpret_cast<float*>(sm + R::bytes);                     // [WK][join_rows][kPitch]
      float2* sml = reinterpret_cast<float2*>(so + WK * join_rows * kPitch);  // [WK][join_rows]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = wr * 16 + gq + 8 * e;
        if (r >= p.n_rows) continue;
        if (tg == 0) sml[wk * join_rows + r] = make_float2(m_r[e], l_r[e]);
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<float2*>(so + (wk * join_rows + r) * kPitch + d * 8 + 2 * tg) = make_float2(acc[d][2 * e], acc[d][2 * e + 1]);
      }
      workers_sync();
      for (int x = threadIdx.x; x < p.n_rows * (D / 4); x += kWorkers) {
        const int r = x / (D / 4), c = x % (D / 4) * 4;
        float m = -INFINITY;
#pragma unroll
        for (int g = 0; g < WK; ++g) m = fmaxf(m, sml[g * join_rows + r].x);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < WK; ++g) {
          const float2 ml = sml[g * join_rows + r];
          const float f = ex2_approx(ml.x - base);
          const float4 v = *reinterpret_cast<const float4*>(so + (g * join_rows + r) * kPitch + c);
          l = fmaf(f, ml.y, l);
          o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
        }
        const long long out = out_of(r);
        *reinterpret_cast<float4*>(a.part_o + out * D + c) = o;
        if (c == 0) a.part_ml[out] = make_float2(m, l);
      }
      workers_sync();
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = wr * 16 + gq + 8 * e;
        if (r >= p.n_rows || idle) continue;
        const long long out = out_of(r);
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<float2*>(a.part_o + out * D + d * 8 + 2 * tg) = make_float2(acc[d][2 * e], acc[d][2 * e + 1]);
        if (tg == 0) a.part_ml[out] = make_float2(m_r[e], l_r[e]);
      }
    }
  }
  if constexpr (Chunk) {
    workers_sync();
    if (again) rows_again<D>(a, seq_lens, q_offsets, items, 16 * WR, kHeads);
  }
}

// A call without pieces of own keys (a bound of 0 for the lengths): reports what the other kernels do not look at.
__global__ void __launch_bounds__(256) check_kernel(const __grid_constant__ Args a) {
  bool bad = a.q_offsets && threadIdx.x < 32 && !offsets_sound(a, a.q_offsets);
  for (int b = threadIdx.x; b < a.batch; b += blockDim.x) bad = bad || a.seq_lens[b] != 0;
  if (bad) flag(a);
}

// Joins the pieces of each (token, head).  With many pieces a block takes a row and its warps the pieces in turn, because
// one warp would wait for one piece after another (512 rows of 20 pieces: 6 us, 9 with a warp each); with few a warp takes
// a row (76,000 rows of one piece: 57 us less than with a block each).
// Checked: the call has offsets, which may not hold.
template <int D, bool Together, bool Checked>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ Args a) {
  constexpr int kPer = D / 32, kStep = Together ? 4 : 1;
  __shared__ float so[4][D];
  __shared__ float sl[4];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long row = Together ? blockIdx.x : blockIdx.x * 4ll + warp, rows = static_cast<long long>(a.n) * a.heads;
  wait_for_previous();
  if (row >= rows) return;
  // Own pieces that do not count are read as empty, so that their loads do not wait for the word on them (16 x 512 tokens of
  // 16 heads of 64: 97.7 us for the call if they do, 88.8 so).
  const int pieces = a.prefix_splits + a.own_splits;
  const bool own = !Checked || own_count(a);
  auto part = [&](int p) {
    const float2 ml = a.part_ml[p * rows + row];
    return !Checked || p < a.prefix_splits || own ? ml : make_float2(-INFINITY, 0.f);
  };
  float m = -INFINITY;
  for (int p = lane; p < pieces; p += 32) m = fmaxf(m, part(p).x);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f, o[kPer] = {};
#pragma unroll 4
  for (int p = Together ? warp : 0; p < pieces; p += kStep) {
    const float2 ml = part(p);
    const float f = ex2_approx(ml.x - base);
    l = fmaf(f, ml.y, l);
    const float* po = a.part_o + (p * rows + row) * D + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(f, ml.x == -INFINITY ? 0.f : po[i], o[i]);  // (a piece without keys is not written)
  }
  if (Together) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    if (warp > 0) return;
    l = sl[0] + sl[1] + sl[2] + sl[3];
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = so[0][lane * kPer + i] + so[1][lane * kPer + i] + so[2][lane * kPer + i] + so[3][lane * kPer + i];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row without keys is zero; one with a score of NaN stays NaN
  __nv_bfloat16* out = a.o + row * D + lane * kPer;
  if constexpr (kPer == 1) *out = f32_to_bf16(o[0] * inv);
#pragma unroll
  for (int i = 0; i + 1 < kPer; i += 2) *reinterpret_cast<uint32_t*>(out + i) = pack_bf16x2(o[i] * inv, o[i + 1] * inv);
  if (a.lse && lane == 0) a.lse[row] = l == 0.f ? -INFINITY : kLn2 * (m + log2f(l));
}

int row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
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

// A pool as (head_dim, heads, tokens, pages) in boxes of 64 values (or the head) and up to `tokens` of one page.
static bool pool_map(CUtensorMap* map, const __nv_bfloat16* base, const Args& a, int head_dim, int tokens) {
  if (!encode_fn()) return false;
  const int page = 1 << a.page_shift;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(std::max(1, a.pages))};
  // an axis of one entry may have any stride: give the map one that it accepts
  auto stride = [](long long n, long long ld) { return static_cast<cuuint64_t>(n > 1 ? ld * 2 : 16); };
  const cuuint64_t strides[3] = {stride(a.kv_heads, a.head_ld), stride(page, a.token_ld), stride(a.pages, a.page_ld)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(std::min(64, head_dim)), 1, static_cast<cuuint32_t>(std::min(page, tokens)), 1};
  const cuuint32_t each[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(base), dims, strides, box, each,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, head_dim == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int WR, bool Quad, bool Chunk>
static cudaError_t launch_pieces(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  const int rows_most = std::max(a.tensor_cores ? 0 : a.n * a.group, a.own_splits > 0 ? a.max_q * a.group : 0);
  const int join_rows = WR == 4 || Quad ? 0 : std::min(16 * WR, rows_most);
  const int known = a.own_splits > 0 && a.batch <= 1024 ? a.batch : 0;
  const int bytes = Ring<D, WR>::bytes + (4 / WR) * join_rows * ((D + 4) * 4 + 8) + (known ? (2 * known + 1) * 4 : 0) + 1024;
  const int items = (a.tensor_cores ? 0 : a.row_tiles * a.kv_heads * a.prefix_splits) +
                    a.batch * a.own_tiles * a.own_splits * (Quad ? ceil_div(a.kv_heads, 4) : a.kv_heads);
  static SharedMemory allowed;
  if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(pieces_kernel<D, WR, Quad, Chunk>), bytes); e != cudaSuccess) return e;
  const int per_sm = std::max(1, std::min(WR == 4 ? 2 : 3, 227 * 1024 / (bytes + 1024 + 64)));
  pieces_kernel<D, WR, Quad, Chunk><<<std::min(items, 148 * per_sm), kThreads, bytes, stream>>>(a, mk, mv, items, join_rows, known);
  return cudaGetLastError();
}

template <int D, bool Chunk>
static cudaError_t launch_pieces_of(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  if (a.quad) return launch_pieces<D, 1, true, Chunk>(a, mk, mv, stream);
  switch (a.tile_rows) {
    case 16: return launch_pieces<D, 1, false, Chunk>(a, mk, mv, stream);
    case 32: return launch_pieces<D, 2, false, Chunk>(a, mk, mv, stream);
    default: return launch_pieces<D, 4, false, Chunk>(a, mk, mv, stream);
  }
}

// Which kernels a call takes.
static bool checks(const Args& a) { return a.own_splits == 0 && a.batch > 0; }
static bool by_warps(const Args& a) { return a.own_splits > 0 || (a.prefix_splits > 0 && !a.tensor_cores); }
static bool by_tensor_cores(const Args& a) { return a.tensor_cores && a.prefix_splits > 0; }
static bool joins(const Args& a) { return !(by_tensor_cores(a) && a.prefix_splits == 1); }
int kernels(const Args& a) { return checks(a) + by_warps(a) + by_tensor_cores(a) + joins(a); }

template <int D>
static cudaError_t launch_for(const Args& a, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  CUtensorMap mk, mv;
  if (checks(a)) {
    check_kernel<<<1, 256, 0, stream>>>(a);
    if (e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  if (by_warps(a)) {
    const int tokens = a.quad ? 16 : kKeys;
    if (!pool_map(&mk, a.k, a, D, tokens) || !pool_map(&mv, a.v, a, D, tokens)) return cudaErrorInvalidValue;
    e = a.max_q > 1 ? launch_pieces_of<D, true>(a, mk, mv, stream) : launch_pieces_of<D, false>(a, mk, mv, stream);
    if (e != cudaSuccess) return e;
  }
  if (by_tensor_cores(a)) {
    if ((!by_warps(a) || a.quad) && (!pool_map(&mk, a.k, a, D, kKeys) || !pool_map(&mv, a.v, a, D, kKeys))) return cudaErrorInvalidValue;
    e = launch_prefix_tc(a, mk, mv, D, stream);
    if (e != cudaSuccess || !joins(a)) return e;
  }
  const int rows = a.n * a.heads;
  if (a.prefix_splits + a.own_splits > 4)
    return launch_after(a.sound ? join_kernel<D, true, true> : join_kernel<D, true, false>, rows, 128, 0, stream, a);
  return launch_after(a.sound ? join_kernel<D, false, true> : join_kernel<D, false, false>, ceil_div(rows, 4), 128, 0, stream, a);
}

// Splits of the tensor-core kernel: whole waves of one block per SM, each taking its tiles and a fixed part, and the
// partial outputs written and read when there are several.
static int tc_splits(int blocks, int tiles, long long rows, int head_dim, bool wide) {
  const double tile_us = wide ? 1.9 : 0.95, fixed_us = 6.0;  // measured: a 128-key tile for 256 rows or for 128, and the rest
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::min(tiles, 64); ++s) {
    const int per = ceil_div(tiles, s), pieces = ceil_div(tiles, per);
    const int units = blocks * pieces, last = units % 148;
    double us = units / 148 * (per * tile_us + fixed_us);
    // (a short last wave of a prefix in one piece has half the rows to a block: prefix_attention_tc.cu)
    if (last > 0) us += per * (pieces == 1 && 2 * last <= 148 ? std::min(tile_us, 0.95) : tile_us) + fixed_us;
    if (pieces > 1) us += 3.0 + pieces * rows * head_dim * 8 / 6.5e6;
    if (us < least * 0.999) least = us, best = s;
  }
  return best;
}

int plan(Args& a, int head_dim) {
  // Without tensor cores, pieces until every SM has about six, so that the last ones are short against the whole.
  constexpr int kWant = 148 * 6;
  a.prefix_splits = a.own_splits = 0;
  a.quad = false;
  const long long rows = static_cast<long long>(a.n) * a.group;
  // (that kernel masks scores before they are scaled, and -inf times a scale of 0 or below is not -inf)
  a.tensor_cores = a.prefix_len > 0 && head_dim != 32 && rows > kTensorCoreRows && a.scale_log2 > 0.f;
  a.tile_rows = 16 * row_warps(static_cast<int>(a.tensor_cores || a.prefix_len == 0 ? static_cast<long long>(a.max_q) * a.group : rows));
  if (a.prefix_len > 0) {
    if (a.tensor_cores) {
      a.row_tiles = ceil_div(rows, 256);
      const int tiles = ceil_div(a.prefix_len, 128);
      const int splits = tc_splits(a.row_tiles * a.kv_heads, tiles, rows * a.kv_heads, head_dim, rows > 128);
      a.prefix_chunk = ceil_div(tiles, splits) * 128;
    } else {
      a.row_tiles = ceil_div(rows, a.tile_rows);
      const int tiles = ceil_div(a.prefix_len, kKeys);
      const int splits = std::max(1, std::min({tiles, 64, ceil_div(kWant, static_cast<long long>(a.row_tiles) * a.kv_heads)}));
      a.prefix_chunk = ceil_div(tiles, splits) * kKeys;
    }
    a.prefix_splits = ceil_div(a.prefix_len, a.prefix_chunk);
  }
  if (a.max_len > 0 && a.max_q > 0 && a.batch > 0) {
    a.own_tiles = ceil_div(static_cast<long long>(a.max_q) * a.group, a.tile_rows);
    const int tiles = ceil_div(a.max_len, kKeys);
    const int splits =
        std::max(1, std::min({tiles, 64, ceil_div(kWant, static_cast<long long>(a.batch) * a.own_tiles * a.kv_heads)}));
    a.own_chunk = ceil_div(tiles, splits) * kKeys;
    a.own_splits = ceil_div(a.max_len, a.own_chunk);
    // Four heads to a piece, where no prefix piece is in the list.  Short sequences (two stages of 64 keys and less) gain
    // as soon as every SM has such a piece: 192 of 4 tokens, 16 heads, 34 us without and 19 with.  Long ones need two for
    // each of an SM's three blocks: 192 of 201 tokens on average, 768 such pieces, lost 4 %.
    const long long quads = static_cast<long long>(a.batch) * a.own_tiles * a.own_splits * ceil_div(a.kv_heads, 4);
    a.quad = (a.tensor_cores || a.prefix_len == 0) && a.tile_rows == 16 && a.kv_heads >= 3 &&
             quads >= (a.max_len <= 2 * kKeys ? 148 : 2 * 3 * 148);
  }
  return a.prefix_splits + a.own_splits;
}

cudaError_t launch_attention(const Args& a, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return launch_for<32>(a, stream);
    case 64: return launch_for<64>(a, stream);
    default: return launch_for<128>(a, stream);
  }
}

}  // namespace prefix

}  // namespace mnb
