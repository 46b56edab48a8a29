// The paged attention over a cache in 8 bits: codes (int8 or e4m3) and one fp32
// scale for each page and kv head; a code stands for code * scale.
// prefix_attention.cu has the mathematics, the pieces and the kernel that joins
// them; prefix_attention_8bit_tc.cu takes the prefix where there are many rows.
//
// With codes c, scales a (keys) and b (values), s_j = scale q . k_j = (scale a_j) (q . c_j),
// and with w_j = b_j exp(s_j) = exp(s_j + log b_j) a part's output is sum w_j c_j: the
// scale of the values rides in the exponent, so weights and codes are both what the
// product takes as f16.  A row's base lies 9 below a maximum of s_j + log2 b_j and moves
// when one passes it by 15, so the largest weight is at most 2^15 and f16 holds weights
// down to 2^-33 of the largest (to 11 bits down to 2^-23).  The sum of exp(s_j) gets
// w_j / b_j in fp32.  Codes are exact in
// f16.  So are queries but for values below 2^-31 of their row's largest: each row is
// scaled by a power of two, which the scores' factor takes back.
//
// What bounds it: the codes' bytes are half of a bf16 cache's, and what is spent on each
// key (widening the codes, products, exponentials) has to fit in half the time.  So the
// products have the keys as their rows: S^T = K Q^T and O^T = V^T P^T (mma.sync
// m16n8k16) for eight or sixteen query rows, where the usual orientation pads one
// query row of a head to sixteen; a warp takes pieces by itself (no barriers between
// warps, no partial results to join in a block) and widens codes in registers: an
// int8 pair by one byte permutation and one subtraction (0x6400 | u is 1024 + u in f16),
// an e4m3 pair by one conversion.
#include <algorithm>
#include <type_traits>

#include "launch.cuh"
#include "prefix_attention_8bit.cuh"
#include "warp_mma.cuh"

namespace mnb {

namespace prefix {

namespace q8 {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStep = 64;  // keys of a stage (2^6)
constexpr float kBelow = 9.f, kPass = 15.f;  // the base below the maximum, and what a score may lie above the base
constexpr int kMostKnown = 1024;  // sequences whose lengths a block keeps

template <int D, int NT>
struct Ring {
  // (sixteen rows need more registers)
  static constexpr int blocks = (D == 128 ? 3 : 4) - (NT == 2 && D > 32);  // per SM
  // A stage's keys and its values each have a place of their own, which the next ones take as soon as it is free: at head dim
  // 128 the keys come while the weights and values are worked on, and the values while the next scores are.
  static constexpr int stages = D == 128 ? 1 : 2;
  static constexpr uint32_t tile = kStep * D;           // of keys, or values
  static constexpr uint32_t bytes = stages * 2 * tile;  // of a warp
  // 16-byte chunk c of row r, as TMA's swizzle leaves it
  MNB_DEVICE static uint32_t at(int r, int c) {
    const int x = D == 128 ? r & 7 : D == 64 ? (r >> 1) & 3 : (r >> 2) & 1;
    return r * D + ((c ^ x) << 4);
  }
};

// Where row i of the products' 8 keys lies among them: rows next to one another meet no bank conflicts when threads read
// 16 bytes each.
template <int D>
MNB_DEVICE int key_of(int i) {
  return D == 128 ? (i >> 1) | ((i & 1) << 2) : i;
}

// (not volatile, as the widening: they may move between the loads)
MNB_DEVICE void mma_f16(float* c, const uint32_t* a, const uint32_t* b) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
MNB_DEVICE uint32_t nan_bytes(uint32_t w) {  // 1 in each byte that is e4m3's NaN
  return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
}
MNB_DEVICE uint32_t transposed(uint32_t x) {  // of an 8 x 8 matrix of 16-bit values, a row's pair in each lane
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// NT: eights of query rows.
template <int D, int NT, bool kFloat>
__global__ void __launch_bounds__(kThreads, Ring<D, NT>::blocks)
    pieces8_kernel(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, int items, int known, int least) {
  using R = Ring<D, NT>;
  // The work takes half a stage at a time: with whole ones the code is so long that fetching it bounds short calls (and
  // sixteen rows lack registers).
  constexpr int kStages = R::stages, kPart = kStep / 2, kU = kPart / 16, kQueue = 4, kRows = 8 * NT, kMt = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[kWarps][2 * kStages];
  __shared__ float scale_of[kWarps][kStages][2][8];  // of a stage's pages: keys, values
  __shared__ float4 factor_of[kWarps][8];            // of each eight keys of the stage that is worked on
  struct Queued {
    Piece p;
    int part_end;
  };
  __shared__ int turns;  // items of this block that are taken
  __shared__ Queued queue[kWarps][kQueue];  // pieces whose loads have begun
  __shared__ uint32_t nan_at[kFloat ? kWarps : 1][kRows][D / 32];  // outputs that have to become NaN, a bit each
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const uint32_t ring = smem_u32(sm) + warp * R::bytes, full_k = smem_u32(bars[warp]), full_v = full_k + 8 * kStages,
                 sc0 = smem_u32(scale_of[warp]);
  if (threadIdx.x == 0) turns = 0;
  if (lane < kStages) {
    mbar_init(full_k + 8 * lane, 33);  // the expected bytes, and every lane's copies of scales
    mbar_init(full_v + 8 * lane, 1);
  }
  fence_mbar_init();
  for (int x = lane; x < kStages * 16; x += 32) (&scale_of[warp][0][0][0])[x] = 1.f;  // (a stage's pages may be fewer than it has room for)
  int* lens = reinterpret_cast<int*>(sm + kWarps * R::bytes);
  int* offsets = lens + known;
  int* tiles_before = offsets + known + 1;  // of 64 keys, of the sequences before each one
  for (int b = threadIdx.x; b < known; b += kThreads) lens[b] = a.seq_lens[b];
  if (a.q_offsets)
    for (int b = threadIdx.x; b < known + (known > 0); b += kThreads) offsets[b] = a.q_offsets[b];
  const int* const seq_lens = known ? lens : a.seq_lens;
  const int* const q_offsets = known ? offsets : a.q_offsets;
  __syncthreads();
  let_next_start();
  // Shares (least > 0: single new tokens).  The tiles of 64 keys of all (part, row tile, kv heads), the prefix first, lie in
  // one row, and every worker takes as many of them, `share`, as every other: a part whose tiles several workers have gets
  // partial results in slots one after another.  (`least` keeps them as few as there are slots.)  A worker is as many warps
  // of a block as heads are taken at once: then they load what lies together in memory (48 sequences of up to 6001 tokens,
  // 8 kv heads: 75 us for a warp and one head each).
  // Otherwise items, pieces of one (part, row tile, kv head, range of keys), in turn over the blocks, whose warps take the
  // next one when they are free (pieces are of 1 to 6 steps in 1504 ragged rows: 199 us,
  // 211 where every warp had its own).
  const int at_once = least == 0 ? 1 : a.kv_heads % 4 == 0 ? 4 : a.kv_heads % 2 == 0 ? 2 : 1, head_groups = a.kv_heads / at_once;
  const int warps = kWarps / at_once * gridDim.x, self = blockIdx.x + warp / at_once * gridDim.x;
  const int own_units = a.own_splits > 0 ? a.own_tiles * head_groups : 0;
  const int prefix_tiles = a.tensor_cores ? 0 : (a.prefix_len + kStep - 1) / kStep, prefix_units = a.row_tiles * head_groups;
  long long of_prefix = 0, from = 0, end = 0, share = 1;
  if (least > 0) {
    if (warp == 0) {
      int sum = 0;
      for (int b0 = 0; b0 < known; b0 += 32) {
        const int len = b0 + lane < known ? lens[b0 + lane] : 0;
        int x = len > 0 && len <= a.max_len ? (len + kStep - 1) / kStep : 0;
        const int mine = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (b0 + lane < known) tiles_before[b0 + lane] = sum + x - mine;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) tiles_before[known] = sum;
    }
    __syncthreads();
    of_prefix = static_cast<long long>(prefix_tiles) * prefix_units;
    const long long all = of_prefix + static_cast<long long>(known ? tiles_before[known] : 0) * own_units;
    share = max((all + warps - 1) / warps, static_cast<long long>(least));
    from = min(all, self * share), end = min(all, from + share);
  }
  // This warp's piece that begins at `at` (a tile, or an item), or else the first one behind it; `at` moves past it.
  auto next = [&](long long& at, Piece& p, int& part_end) {
    if (least == 0) {
      const int turn = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(&turns, 1) : 0, 0);
      at = blockIdx.x + static_cast<long long>(turn) * gridDim.x;
      if (at >= items) return false;
      p = piece_of(a, seq_lens, q_offsets, static_cast<int>(at), kRows, 1);
      part_end = 0;  // (nobody asks)
      return true;
    }
    if (at >= end) return false;
    int unit, tile, tiles, b = -1;
    if (at < of_prefix) {
      tiles = prefix_tiles;
      unit = static_cast<int>(at / tiles), tile = static_cast<int>(at - static_cast<long long>(unit) * tiles);
    } else {
      const long long own = at - of_prefix;
      int lo = 0, hi = known - 1;  // the last sequence whose tiles begin at or before it (those without any come before it)
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (static_cast<long long>(tiles_before[mid]) * own_units <= own) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      tiles = tiles_before[b + 1] - tiles_before[b];
      const long long in = own - static_cast<long long>(tiles_before[b]) * own_units;
      unit = static_cast<int>(in / tiles), tile = static_cast<int>(in - static_cast<long long>(unit) * tiles);
    }
    const int len = b < 0 ? a.prefix_len : lens[b], most = static_cast<int>(min(end - at, static_cast<long long>(tiles - tile)));
    const int segment = self - static_cast<int>((at - tile) / share);
    part_end = len;
    p.h = unit % head_groups * at_once + warp % at_once;
    p.r0 = unit / head_groups * kRows;
    p.k0 = tile * kStep;
    p.k1 = min(len, p.k0 + most * kStep);
    p.limit0 = kUnlimited;
    if (b < 0) {
      p.n0 = 0;
      p.n_rows = min(kRows, a.n * a.group - p.r0);
      p.slot = segment;
      p.ids = a.prefix_pages;
    } else {
      int rows = a.group;
      p.n0 = b;
      if (a.q_offsets) {  // (within the rows whatever the offsets say: offsets_sound() has the word on them)
        p.n0 = min(max(q_offsets[b], 0), a.n);
        rows = max(0, min(min(max(q_offsets[b + 1], 0), a.n) - p.n0, 1)) * a.group;
      }
      p.n_rows = min(kRows, rows - p.r0);
      p.slot = a.prefix_splits + segment;
      p.ids = a.page_table + b * a.table_ld;
    }
    at += most;
    return true;
  };

  // Loading runs ahead of the work, on into the next pieces.
  const int per_shift = min(a.page_shift, 6), per = 1 << per_shift;  // tokens of a box
  long long load_at = least ? from : self;
  bool loading = true;
  int load_key = 0, load_end = 0, load_head = 0, batch = 0, ids_end = 0, issued = 0;
  int ids_now = 0, ids_next = 0;  // this lane's of 32 pages from `batch` on, and of the 32 after them
  const int* ids = nullptr;
  auto fetch = [&](int first) { return first + lane < ids_end ? ids[first + lane] : 0; };
  auto out_of = [&](const Piece& p, int r) {  // where row r's partial results go
    const int j = p.r0 + r, token = j / a.group;
    return (static_cast<long long>(p.slot) * a.n + p.n0 + token) * a.heads + p.h * a.group + j - token * a.group;
  };
  int queued = 0;
  auto next_piece = [&] {
    Piece p;
    int part_end;
    while ((loading = next(load_at, p, part_end))) {
      if (p.n_rows <= 0) continue;
      if (p.k1 <= p.k0) {  // nothing here: the join skips the piece
        if (lane < p.n_rows) a.part_ml[out_of(p, lane)] = make_float2(-INFINITY, 0.f);
        continue;
      }
      load_key = p.k0, load_end = p.k1, load_head = p.h, ids = p.ids;
      batch = p.k0 >> a.page_shift;
      ids_end = ((p.k1 - 1) >> a.page_shift) + 1;
      ids_now = fetch(batch);
      ids_next = fetch(batch + 32);
      // (pieces ahead of the one that is worked on: at most one for each stage, and this)
      if (lane == 0) queue[warp][queued % kQueue] = Queued{p, part_end};
      ++queued;
      return;
    }
  };
  static_assert(kStages + 1 < kQueue, "pieces under way");
  // The keys of the next stage, a box for each of the first lanes, and the scales of both; its values follow.
  int box_page = 0, box_token = 0, box_head = 0, boxes = 0;
  auto issue_keys = [&] {
    boxes = 0;
    if (!loading) return;
    if ((load_key >> a.page_shift) - batch >= 32) {
      batch += 32;
      ids_now = ids_next;
      ids_next = fetch(batch + 32);
    }
    const int st = issued % kStages;
    const uint32_t bar = full_k + 8 * st;
    boxes = (min(kStep, load_end - load_key) + per - 1) >> per_shift;
    box_page = __shfl_sync(0xffffffffu, ids_now, ((load_key >> a.page_shift) - batch + lane) & 31);
    box_token = (load_key + lane * per) & ((1 << a.page_shift) - 1), box_head = load_head;
    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * per * D);
    __syncwarp();
    if (lane < boxes) {
      const bool there = box_page >= 0 && box_page < a.pages;
      const long long at = there ? box_page * a.scale_ld + load_head * a.scale_head : 0;
      if (!there) {
        flag(a);
        box_page = a.no_page;  // reads as zeros
      }
      tma_load_4d(ring + st * 2 * R::tile + lane * per * D, &map_k, 0, load_head, box_token, box_page, bar);
      copy_float(sc0 + (st * 16 + lane) * 4, a.k_scales + at, there);
      copy_float(sc0 + (st * 16 + 8 + lane) * 4, a.v_scales + at, there);
    }
    arrive_after_copies(bar);
    load_key += kStep;
    if (load_key >= load_end) next_piece();
  };
  auto issue_values = [&] {
    if (boxes == 0) return;
    const int st = issued % kStages;
    const uint32_t bar = full_v + 8 * st;
    if (lane == 0) mbar_arrive_expect_tx(bar, boxes * per * D);
    __syncwarp();
    if (lane < boxes) tma_load_4d(ring + (st * 2 + 1) * R::tile + lane * per * D, &map_v, 0, box_head, box_token, box_page, bar);
    ++issued;
  };
  // Where this lane reads: row g (and g + 8) of 16 keys as the first operand of K Q^T, and the rows of ldmatrix for V^T P^T
  const uint32_t at_k = D == 32 ? R::at(g, t >> 1) + (t & 1) * 8 : R::at(key_of<D>(g), t);
  const uint32_t at_v = R::at(((lane >> 3) & 1) * 8 + key_of<D>(lane & 7), lane >> 4);
  next_piece();
  uint32_t qf[NT][kMt][2];
  float back[NT][2];         // what rows n * 8 + 2 t and + 1 were scaled by, taken back
  int lim[NT][2], whole = 0;  // the keys that they see, and those that every row does
  float o[NT][kMt][4], base[NT][2], l[NT][2];
  Piece p;
  int part_end = 0, t0 = 0, taken = 0;
  p.k1 = 0;
  // Stage by stage, the first kStages steps only load.
  for (int pos = -kStages;; ++pos) {
    const bool work = pos >= 0;
    if (work && t0 >= p.k1) {  // the next piece
      if (taken == queued) break;
      __syncwarp();
      p = queue[warp][taken % kQueue].p, part_end = queue[warp][taken % kQueue].part_end;
      ++taken;
      t0 = p.k0;
      // Queries as the products' second operand: row n * 8 + g, four dims (those of a word of codes) for each 16-wide step.
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + g, j = p.r0 + r, token = j / a.group;
        const bool in = r < p.n_rows;
        const __nv_bfloat16* q = a.q + (p.n0 + token) * a.q_ld + (p.h * a.group + j - token * a.group) * a.q_head;
        uint4 w[kMt / 2];
#pragma unroll
        for (int x = 0; x < kMt / 2; ++x) {
          const int dim = D == 32 ? 8 * t : (x / 2) * 64 + 16 * t + (x % 2) * 8;
          w[x] = in ? ld_v4(q + dim) : make_uint4(0, 0, 0, 0);
        }
        uint32_t most = 0;  // of the finite values, as bits
#pragma unroll
        for (int x = 0; x < kMt / 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = (&w[x].x)[e], lo = v & 0x7fffu, hi = (v >> 16) & 0x7fffu;
            most = max(most, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
          }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int shift = min(141 - static_cast<int>(most >> 7), 126);  // the largest becomes 2^14 to 2^15
        const float up = __int_as_float((127 + shift) << 23);
#pragma unroll
        for (int x = 0; x < kMt / 2; ++x)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2 u = unpack_bf16x2((&w[x].x)[2 * e]), v = unpack_bf16x2((&w[x].x)[2 * e + 1]);
            u = mul2(u, splat2(up)), v = mul2(v, splat2(up));
            qf[n][2 * x + e][0] = kFloat ? pack_f16x2(u.x, u.y) : pack_f16x2(u.x, v.x);
            qf[n][2 * x + e][1] = kFloat ? pack_f16x2(v.x, v.y) : pack_f16x2(u.y, v.y);
          }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = n * 8 + 2 * t + e;
          back[n][e] = __int_as_float((127 - __shfl_sync(0xffffffffu, shift, (2 * t + e) * 4)) << 23);
          lim[n][e] = row < p.n_rows ? min(p.k1, p.limit0 + (p.r0 + row) / a.group) : p.k0;
        }
      }
      whole = min(p.k1, p.limit0 + p.r0 / a.group);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        base[n][0] = base[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int m = 0; m < kMt; ++m) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.f;
      }

    }
    const int st = max(pos, 0) % kStages;
    const uint32_t phase = (pos / kStages) & 1;
    if (work) mbar_wait(full_k + 8 * st, phase, a.status);  // (a wait that gave up is in the status word)
    __syncwarp();
    const uint32_t sK = ring + st * 2 * R::tile, sV = sK + R::tile;
    // Each eight keys lie in one page: its factor of the scores, the logarithm of its values' scale, and what turns a
    // weight into its part of the sum (times 2^15, so that nothing leaves the range of fp32).
    if (work && lane < 8) {
      const int box = (lane * 8) >> a.page_shift;
      const float b = __log2f(fmaxf(scale_of[warp][st][1][box], kLeastScale));  // (a page of zeros may have any scale)
      factor_of[warp][lane] = make_float4(scale_of[warp][st][0][box] * a.scale_log2, b, ex2_approx(15.f - b), 0.f);
    }
    __syncwarp();
    bool spoiled = false;
#pragma unroll 1
    for (int part = 0; part < kStep / kPart; ++part) {
      const int t1 = t0 + part * kPart;
      const bool live = work && (part == 0 || t1 < p.k1);
      float s[NT][kU][4];
      if (live) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][u][0] = s[n][u][1] = s[n][u][2] = s[n][u][3] = 0.f;
#pragma unroll
          for (int x = 0; x < (D + 63) / 64; ++x) {
            uint4 ka, kb;  // a row's words: two of them at head dim 32
            const uint32_t from = (sK + (part * kPart + u * 16) * D + at_k) ^ (x * 64);
            if (D == 32) {
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(ka.x), "=r"(ka.y) : "r"(from));
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(kb.x), "=r"(kb.y) : "r"(from + 8 * D));
            } else {
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(ka.x), "=r"(ka.y), "=r"(ka.z), "=r"(ka.w) : "r"(from));
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(kb.x), "=r"(kb.y), "=r"(kb.z), "=r"(kb.w) : "r"(from + 8 * D));
            }
#pragma unroll
            for (int j = 0; j < (D == 32 ? 2 : 4); ++j) {
              uint32_t f[4];
              widen_any<kFloat>((&ka.x)[j], f[0], f[2]);
              widen_any<kFloat>((&kb.x)[j], f[1], f[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma_f16(s[n][u], f, qf[n][x * 4 + j]);
            }
          }
        }
      }
      if (part == kStep / kPart - 1) {
        __syncwarp();  // (the keys and scales have been read)
        issue_keys();
      }
      if (!live) continue;
      float sum_of[kU][2];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 f = factor_of[warp][2 * (part * kU + u) + h];
          sum_of[u][h] = f.z;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              // (towards zero: a factor past fp32's range stays finite, and 0 times it stays 0)
              s[n][u][2 * h + e] = fmaf(s[n][u][2 * h + e], __fmul_rz(f.x, back[n][e]), f.y);
        }
      const bool masked = t1 + kPart > whole;
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int u = 0; u < kU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (t1 + u * 16 + e / 2 * 8 + key_of<D>(g) >= lim[n][e & 1]) s[n][u][e] = -INFINITY;
      }
      float top[NT][2];
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[n][0][e], s[n][0][2 + e]);
#pragma unroll
          for (int u = 1; u < kU; ++u) x = max3f(x, s[n][u][e], s[n][u][2 + e]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          top[n][e] = x;
          grows = grows || x > base[n][e] + kPass || (base[n][e] == -INFINITY && x > -INFINITY);
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float to = top[n][e] > base[n][e] + kPass || base[n][e] == -INFINITY ? top[n][e] - kBelow : base[n][e];
            alpha[e] = to == base[n][e] ? 1.f : ex2_approx(base[n][e] - to);
            l[n][e] *= alpha[e];
            base[n][e] = to;
          }
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][m][e] *= alpha[e & 1];
        }
      }
      uint32_t pf[NT][kU][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        // (no key yet: every weight is exp2(-inf) = 0)
        const float from0 = base[n][0] == -INFINITY ? 0.f : base[n][0], from1 = base[n][1] == -INFINITY ? 0.f : base[n][1];
#pragma unroll
        for (int u = 0; u < kU; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float w0 = ex2_approx(s[n][u][2 * h] - from0), w1 = ex2_approx(s[n][u][2 * h + 1] - from1);
            l[n][0] = fmaf(w0, sum_of[u][h], l[n][0]);
            l[n][1] = fmaf(w1, sum_of[u][h], l[n][1]);
            pf[n][u][h] = transposed(pack_f16x2(w0, w1));
          }
      }
      if (part == 0) {
        mbar_wait(full_v + 8 * st, phase, a.status);
        __syncwarp();
      }
      if constexpr (kFloat) {
        // A key that a row does not see has weight 0, and 0 times NaN (which e4m3 has, also past the end of the keys, where
        // a page holds anything) would be NaN: such codes become zeros here, and rows that do see one become NaN below.
        if (part == 0 && t0 + kStep > whole) {
          uint32_t some = 0;
          for (int x = lane; x < kStep * D / 16; x += 32) {
            uint4 w;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(sV + x * 16));
            some |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
          }
          spoiled = __any_sync(0xffffffffu, some != 0);
          if (spoiled) {
            for (int x = lane; x < kRows * (D / 32); x += 32) (&nan_at[warp][0][0])[x] = 0;
            __syncwarp();
#pragma unroll 1
            for (int x = lane; x < kStep * D / 4; x += 32) {  // word by word
              const int key = x / (D / 4), word = x % (D / 4);
              const uint32_t at = sV + R::at(key, word / 4) + word % 4 * 4;
              uint32_t w;
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at));
              const uint32_t odd = nan_bytes(w);
              if (!odd) continue;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w & ~(odd * 0xffu)) : "memory");
              const uint32_t bits = ((odd & 1u) | (odd >> 7 & 2u) | (odd >> 14 & 4u) | (odd >> 21 & 8u)) << (word % 8 * 4);
              for (int row = 0; row < p.n_rows; ++row)
                if (t0 + key < min(p.k1, p.limit0 + (p.r0 + row) / a.group)) atomicOr(&nan_at[warp][row][word / 8], bits);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes here next
            __syncwarp();
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int c = 0; c < kMt / 2; ++c) {
          uint32_t w[4];
          ldsm_x4_t(w, (sV + (part * kPart + u * 16) * D + at_v) ^ (c * 32));
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint32_t f[4];
            widen<kFloat>(w[2 * m], f[0], f[1]);
            widen<kFloat>(w[2 * m + 1], f[2], f[3]);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * c + m], f, pf[n][u]);
          }
        }
      if (kFloat && spoiled) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int dim = m * 16 + 2 * g + e / 2;
              if (nan_at[warp][n * 8 + 2 * t + e % 2][dim / 32] >> (dim % 32) & 1) o[n][m][e] = NAN;
            }
      }
    }
    __syncwarp();
    issue_values();
    if (!work) continue;
    t0 += kStep;
    if (t0 < p.k1) continue;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = n * 8 + 2 * t + e;
        if (r >= p.n_rows) continue;
        const long long out = out_of(p, r);
#pragma unroll
        for (int m = 0; m < kMt; ++m)
          *reinterpret_cast<float2*>(a.part_o + out * D + m * 16 + 2 * g) = make_float2(o[n][m][e], o[n][m][2 + e]);
        if (g == 0) a.part_ml[out] = make_float2(base[n][e], sum * 3.0517578125e-5f);  // 2^-15
        if (least > 0 && p.k1 == part_end) {  // of shares: the part's other slots have nothing
          const long long step = static_cast<long long>(a.n) * a.heads;
          const int slots = p.slot < a.prefix_splits ? a.prefix_splits : a.prefix_splits + a.own_splits;
          for (int x = p.slot + 1 + g; x < slots; x += 8) a.part_ml[out + (x - p.slot) * step] = make_float2(-INFINITY, 0.f);
        }
      }
  }
  // Sequences without tokens have no partial results at all.
  if (least > 0 && warp % at_once == 0)
    for (int b = self; b < known; b += warps)
      if (tiles_before[b + 1] == tiles_before[b]) {
        if (lane == 0 && lens[b] != 0) flag(a);  // (a length out of its bounds)
        const int n0 = a.q_offsets ? min(max(q_offsets[b], 0), a.n) : b;
        const int rows = a.q_offsets ? max(0, min(min(max(q_offsets[b + 1], 0), a.n) - n0, 1)) : 1;
        for (int x = lane; x < rows * a.own_splits * a.heads; x += 32)
          a.part_ml[(static_cast<long long>(a.prefix_splits + x / a.heads) * a.n + n0) * a.heads + x % a.heads] = make_float2(-INFINITY, 0.f);
      }
  // The block does not end before its last copies have arrived, also where a wait was given up.
  for (int k = max(0, issued - kStages); k < issued; ++k) {
    mbar_wait(full_k + 8 * (k % kStages), (k / kStages) & 1, nullptr);
    mbar_wait(full_v + 8 * (k % kStages), (k / kStages) & 1, nullptr);
  }
  if (a.sound && blockIdx.x == 0 && warp == 0) {
    const bool sound = offsets_sound(a, q_offsets);
    if (lane == 0) {
      *a.sound = sound;
      if (!sound) flag(a);
    }
  }
}

template <int D, int NT, bool kFloat>
static cudaError_t launch(const Args& a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
  using R = Ring<D, NT>;
  const int known = a.own_splits > 0 && a.batch <= kMostKnown ? a.batch : 0;
  const int bytes = kWarps * R::bytes + (known ? (3 * known + 2) * 4 : 0) + 1024;
  long long items = a.batch * static_cast<long long>(a.own_tiles) * a.own_splits * a.kv_heads;
  if (!a.tensor_cores) items += static_cast<long long>(a.row_tiles) * a.kv_heads * a.prefix_splits;
  static SharedMemory allowed;
  if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(pieces8_kernel<D, NT, kFloat>), bytes); e != cudaSuccess) return e;
  const int per_sm = std::max(1, std::min(R::blocks, 227 * 1024 / (bytes + 1024 + 2048)));
  const int blocks = static_cast<int>(std::min<long long>(items, 148 * per_sm));
  pieces8_kernel<D, NT, kFloat><<<blocks, kThreads, bytes, stream>>>(a, mk, mv, static_cast<int>(items), known, a.least_share);
  return cudaGetLastError();
}

template <int D>
static cudaError_t launch_for(const Args& a, cudaStream_t stream) {
  CUtensorMap mk, mv;
  if (!codes_map(&mk, a.k8, a, D, kStep) || !codes_map(&mv, a.v8, a, D, kStep)) return cudaErrorInvalidValue;
  if (a.codes == kE4m3) return a.tile_rows == 8 ? launch<D, 1, true>(a, mk, mv, stream) : launch<D, 2, true>(a, mk, mv, stream);
  return a.tile_rows == 8 ? launch<D, 1, false>(a, mk, mv, stream) : launch<D, 2, false>(a, mk, mv, stream);
}

}  // namespace q8

cudaError_t launch_pieces8(const Args& a, int head_dim, cudaStream_t stream) {
  switch (head_dim) {
    case 32: return q8::launch_for<32>(a, stream);
    case 64: return q8::launch_for<64>(a, stream);
    default: return q8::launch_for<128>(a, stream);
  }
}

int plan8(Args& a, int head_dim) {
  using q8::kStep;
  a.prefix_splits = a.own_splits = a.least_share = 0;
  a.quad = false;
  const long long rows = static_cast<long long>(a.n) * a.group, own_rows = static_cast<long long>(a.max_q) * a.group;
  const bool own = a.max_len > 0 && a.max_q > 0 && a.batch > 0;
  // The tensor-core kernel for more rows than a warp takes, where that comes to enough steps of 16 rows and 64 keys: its blocks
  // take 10 us before and after their tiles, in which the warps do some 2000 steps (20 rows of 16 kv heads over 4096 keys 22
  // us, on tensor cores 25; 160 rows over 4096 keys 72 and 43).  (It takes maxima before it scales.)
  const double steps = static_cast<double>(ceil_div(rows, 16)) * ceil_div(a.prefix_len, kStep) * a.kv_heads;
  a.tensor_cores = a.prefix_len > 0 && head_dim != 32 && rows > 16 && steps > 2048 && a.scale_log2 > 0.f;
  a.tile_rows = std::max(a.prefix_len > 0 && !a.tensor_cores ? rows : 0, own ? own_rows : 0) <= 8 ? 8 : 16;
  const int warps = 148 * q8::kWarps * ((head_dim == 128 ? 3 : 4) - (a.tile_rows == 16 && head_dim > 32));
  const int prefix_tiles = ceil_div(a.prefix_len, kStep), own_tiles = ceil_div(a.max_len, kStep);
  if (a.tensor_cores) plan_prefix_tc(a, head_dim);
  else if (a.prefix_len > 0) a.row_tiles = ceil_div(rows, a.tile_rows);
  if (own) a.own_tiles = ceil_div(own_rows, a.tile_rows);
  // Single new tokens: shares of the tiles, the same for every warp (48 sequences of up to 6001 tokens, 8 heads: 89 us with
  // pieces of 608 keys in turn).  A part of t tiles has at most 1 + ceil((t - 1) / share) warps, and as many slots.  Parts of
  // the average length need one for each warp that it takes to fill the GPU, longer ones (here: up to twice) more.
  const bool shares = a.max_q == 1 && (!own || (a.batch <= q8::kMostKnown && static_cast<long long>(a.batch) * own_tiles < (1ll << 31)));
  constexpr int kMostSlots = 256;
  auto slots = [&](int tiles, long long units, int times) {
    return std::min({tiles, kMostSlots, times * ceil_div(warps, units) + (times == 1 ? 2 : 1)});
  };
  if (a.prefix_len > 0 && !a.tensor_cores) {
    const long long units = static_cast<long long>(a.row_tiles) * a.kv_heads;
    if (shares) {
      a.prefix_splits = slots(prefix_tiles, units, 1);
      if (prefix_tiles > 1) a.least_share = ceil_div(prefix_tiles - 1, a.prefix_splits - 1);
    } else {  // pieces until every warp has about three
      const int splits = std::max(1, std::min({prefix_tiles, 64, ceil_div(3 * warps, units)}));
      a.prefix_chunk = ceil_div(prefix_tiles, splits) * kStep;
      a.prefix_splits = ceil_div(a.prefix_len, a.prefix_chunk);
    }
  }
  if (own) {
    const long long units = static_cast<long long>(a.batch) * a.own_tiles * a.kv_heads;
    if (shares) {
      a.own_splits = slots(own_tiles, units, 2);
      if (own_tiles > 1) a.least_share = std::max(a.least_share, ceil_div(own_tiles - 1, a.own_splits - 1));
    } else {
      const int splits = std::max(1, std::min({own_tiles, 64, ceil_div(3 * warps, units)}));
      a.own_chunk = ceil_div(own_tiles, splits) * kStep;
      a.own_splits = ceil_div(a.max_len, a.own_chunk);
    }
  }
  if (shares) a.least_share = std::max(a.least_share, 1);
  return a.prefix_splits + a.own_splits;
}

}  // namespace prefix

}  // namespace mnb
