// What the kernels of the paged attention share: the list of pieces that a call
// is split into, and the page pools' tensor maps (prefix_attention.cu has the
// mathematics and the choice between the kernels).
#pragma once

#include <cudaTypedefs.h>

#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace prefix {

MNB_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

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

inline int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // or null, without a driver that has it

}  // namespace prefix

}  // namespace mnb
