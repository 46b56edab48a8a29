// Page operations of the paged key / value cache.
//
// The pool is one tensor [..., num_pages, page_size, kv_heads, head_dim]; the
// leading axes (layers, keys / values) are "planes" that every page id names
// at once.  The bookkeeping lives on the device, so no operation waits for
// the host: page_table [sequences, columns] (int32, -1 past a sequence's last
// page), lens [sequences] and refs [num_pages], the number of sequences that
// hold each page.  refs is the only record of what is free; a page is free
// when its count is zero, and the lowest free ids are handed out first, in
// the order of the requests, so results do not depend on scheduling.
//
// Bookkeeping kernels are one block (a few thousand counts); they leave a
// list of copies that a second kernel with many blocks carries out.  Bad
// indices and a pool without room set the status word and leave the request
// out; nothing is read or written out of range.
#include <algorithm>

#include "common.cuh"
#include "generation.h"
#include "launch.cuh"

namespace mnb {

namespace cache {

constexpr int kThreads = 1024;

MNB_DEVICE void flag(int* status, int code) { atomicCAS(status, 0, code); }

// Exclusive scan over the block; *total gets the sum.  `sh` holds 33 ints.
MNB_DEVICE int block_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = lane < blockDim.x / 32 ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    sh[lane] = s;
  }
  __syncthreads();
  const int before = warp == 0 ? 0 : sh[warp - 1];
  *total = sh[blockDim.x / 32 - 1];
  __syncthreads();
  return before + x - v;
}

// The first `want` free pages in ascending order into ids[]; returns how many there are (at most want).
// (`first`: this thread's count of the first kThreads, already read.)
MNB_DEVICE int find_free(const int* refs, int pages, int want, int* ids, int* sh, int first) {
  int found = 0;
  for (int p0 = 0; p0 < pages && found < want; p0 += kThreads) {
    const int p = p0 + threadIdx.x;
    const int is_free = p < pages && (p0 == 0 ? first : refs[p]) == 0;
    int total;
    const int rank = found + block_scan(is_free, sh, &total);
    if (is_free && rank < want) ids[rank] = p;
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

// Marks in owner[slot] the first request that names each slot (requests that
// name it again are refused).
MNB_DEVICE void claim(const int* slot_of, int n, int slots, int* owner) {
  for (int s = threadIdx.x; s < slots; s += kThreads) owner[s] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int s = slot_of[i];
    if (s >= 0 && s < slots) atomicMin(owner + s, i);
  }
  __syncthreads();
}

// fork: child i gets parent i's table row; full pages are shared, the
// part-filled last one gets a page of its own (src / dst / tokens name the copy).
// Few requests keep their state in shared memory: what is left of the time is
// three trips to memory, one after another (the requests, their lengths, the rows):
// 6.6 us for 4 requests with cold caches.  That a parent's row names no page of the pool shows only when the child's is
// written, so such a request is taken back then (the page that it had been given stays free, also for later requests).
constexpr int kFew = 256;
__global__ void __launch_bounds__(kThreads) fork_plan_kernel(Table t, const int* __restrict__ parents,
                                                             const int* __restrict__ children, int n, int* owner,
                                                             int* ids, int* src, int* dst, int* tokens, int* status) {
  __shared__ int sh[33];
  __shared__ int few_ids[kFew], few_src[kFew], few_dst[kFew], few_tokens[kFew], few_len[kFew], few_parent[kFew], few_child[kFew];
  const bool few = n <= kFew;
  int* const of_ids = few ? few_ids : ids;
  int* const of_src = few ? few_src : src;
  int* const of_dst = few ? few_dst : dst;
  int* const of_tokens = few ? few_tokens : tokens;
  const int first_refs = threadIdx.x < t.pages ? t.refs[threadIdx.x] : 1;  // on its way with the requests
  let_next_start();
  if (!few) claim(children, n, t.slots, owner);
  // which requests are sound, and which need a page (its rank is parked in dst)
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0, part = -1;
    int p = -1, c = -1;
    if (i < n) p = parents[i], c = children[i];
    bool ok = p >= 0 && p < t.slots && c >= 0 && c < t.slots;
    const int len = ok ? t.lens[p] : 0, child_len = ok ? t.lens[c] : 0;
    if (few) {
      if (i < n) few_parent[i] = p, few_child[i] = c, few_len[i] = len;
      __syncthreads();
      int clashes = 0;  // (summed without branches, so that the reads follow one another closely)
#pragma unroll 8
      for (int j = 0; j < n; ++j) clashes += (few_child[j] == p) | ((few_child[j] == c) & (j < i));
      ok = ok && clashes == 0;
    } else if (ok) {
      ok = owner[c] == i && owner[p] == 0x7fffffff;  // the child's first request, and a parent that is nobody's child
    }
    if (i < n) {
      ok = ok && child_len == 0 && len >= 0 && len <= t.columns * static_cast<long long>(t.page_size);
      if (ok) {
        part = len % t.page_size;
        need = part > 0;
      } else {
        flag(status, kErrBadIndex);
      }
    }
    int total;
    const int rank = base + block_scan(need, sh, &total);
    if (i < n) {
      of_tokens[i] = part;
      of_dst[i] = need ? rank : -1;
    }
    base += total;
  }
  const int have = find_free(t.refs, t.pages, base, of_ids, sh, first_refs);
  if (base > have && threadIdx.x == 0) flag(status, kErrNoPages);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    of_src[i] = -1;
    if (of_dst[i] >= have) of_tokens[i] = of_dst[i] = -1;  // no page left: the child stays empty
  }
  __syncthreads();
  // f(request, column, the parent's row, its full pages) for the entries of the children's rows, request by request (i and
  // col advance without divisions)
  auto entries = [&](auto f) {
    int i = threadIdx.x / t.columns, col = threadIdx.x % t.columns;
    const int step_i = kThreads / t.columns, step_col = kThreads % t.columns;
    for (; i < n; i += step_i, col += step_col) {
      if (col >= t.columns) {
        col -= t.columns;
        if (++i >= n) break;
      }
      if (of_tokens[i] < 0) continue;
      const int p = few ? few_parent[i] : parents[i];
      f(i, col, t.table + p * t.ld, (few ? few_len[i] : t.lens[p]) / t.page_size);
    }
  };
  auto child_row = [&](int i) { return t.table + (few ? few_child[i] : children[i]) * t.ld; };
  auto of_pool = [&](int page) { return page >= 0 && page < t.pages; };
  bool damaged = false;
  entries([&](int i, int col, const int* row, int full) {
    int page = -1;
    if (col <= full) {
      page = row[col];
      if (col == full) {
        if (of_tokens[i] > 0 && of_pool(page)) of_src[i] = page;
        damaged = damaged || (of_tokens[i] > 0 && !of_pool(page));
        page = of_tokens[i] > 0 ? of_ids[of_dst[i]] : -1;
        if (page >= 0) t.refs[page] = 1;
      } else if (of_pool(page)) {
        atomicAdd(t.refs + page, 1);
      } else {
        damaged = true;
      }
    }
    child_row(i)[col] = page;
  });
  if (__syncthreads_or(damaged)) {
    entries([&](int i, int col, const int* row, int full) {  // which requests it is (-2)
      if (col < full ? !of_pool(row[col]) : col == full && of_tokens[i] > 0 && !of_pool(row[col])) of_src[i] = -2;
    });
    __syncthreads();
    entries([&](int i, int col, const int* row, int full) {
      if (of_src[i] != -2) return;
      if (col < full && of_pool(row[col])) atomicSub(t.refs + row[col], 1);
      if (col == full && of_tokens[i] > 0) t.refs[of_ids[of_dst[i]]] = 0;
      child_row(i)[col] = -1;
    });
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (of_src[i] == -2) {
        of_tokens[i] = of_dst[i] = -1;
        flag(status, kErrBadIndex);
      }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int to = of_tokens[i] >= 0 && of_dst[i] >= 0 ? of_ids[of_dst[i]] : -1;
    if (of_tokens[i] >= 0) t.lens[few ? few_child[i] : children[i]] = few ? few_len[i] : t.lens[parents[i]];
    src[i] = of_src[i];
    dst[i] = to;
    tokens[i] = of_tokens[i];
  }
}

// reserve: slot i grows by counts[i] tokens; new pages fill its row (192 single tokens 4 us; a request's pages are written
// by one thread, one sequence of 4097 pages 205 us).  (A row may hold more tokens than an int32 length
// can say: a sequence ends at 2^31 - 1.)
__global__ void __launch_bounds__(kThreads) reserve_kernel(Table t, const int* __restrict__ slot_of,
                                                           const int* __restrict__ counts, int n, int* owner, int* ids,
                                                           int most, int* rank_of, int* status) {
  __shared__ int sh[33];
  const int first_refs = threadIdx.x < t.pages ? t.refs[threadIdx.x] : 1;
  claim(slot_of, n, t.slots, owner);
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int s = slot_of[i], more = counts[i];
      bool ok = s >= 0 && s < t.slots && owner[s] == i && more >= 0;
      if (ok) {
        const long long len = t.lens[s], to = len + more;
        ok = len >= 0 && to <= min(t.columns * static_cast<long long>(t.page_size), 0x7fffffffll);
        if (ok) need = static_cast<int>((to + t.page_size - 1) / t.page_size - (len + t.page_size - 1) / t.page_size);
      }
      if (!ok) {
        flag(status, kErrBadIndex);
        need = -1;
      }
    }
    int total;
    const int rank = base + block_scan(max(need, 0), sh, &total);
    if (i < n) rank_of[i] = need < 0 ? -1 : rank;
    base += total;
  }
  const int have = find_free(t.refs, t.pages, min(base, most), ids, sh, first_refs);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    if (rank_of[i] < 0) continue;
    const int s = slot_of[i];
    const long long len = t.lens[s], to = len + counts[i];
    const int c0 = static_cast<int>((len + t.page_size - 1) / t.page_size), c1 = static_cast<int>((to + t.page_size - 1) / t.page_size);
    if (c1 > c0 && rank_of[i] + (c1 - c0) > have) {
      flag(status, kErrNoPages);
      continue;
    }
    for (int c = c0; c < c1; ++c) {
      const int page = ids[rank_of[i] + c - c0];
      t.table[s * t.ld + c] = page;
      t.refs[page] = 1;
    }
    t.lens[s] = static_cast<int>(to);
  }
}

// free (a launch's time, 4 us, for 128 rows of 16): every page of the slots'
// rows loses one holder.  The exchange hands
// each entry to one thread, so naming a slot twice frees it once.
__global__ void __launch_bounds__(256) free_kernel(Table t, const int* __restrict__ slot_of, int n, int* status) {
  const long long all = static_cast<long long>(n) * t.columns;
  for (long long x = blockIdx.x * 256ll + threadIdx.x; x < all; x += gridDim.x * 256ll) {
    const int i = static_cast<int>(x / t.columns), col = static_cast<int>(x % t.columns);
    const int s = slot_of[i];
    if (s < 0 || s >= t.slots) {
      flag(status, kErrBadIndex);
      continue;
    }
    const int page = atomicExch(t.table + s * t.ld + col, -1);
    if (col == 0) t.lens[s] = 0;
    if (page < 0) continue;
    if (page >= t.pages) {
      flag(status, kErrBadIndex);
    } else if (atomicSub(t.refs + page, 1) <= 0) {  // nobody held it: put the count back
      atomicAdd(t.refs + page, 1);
      flag(status, kErrBadIndex);
    }
  }
}

// compact: with n pages in use, those with ids >= n move, in ascending order,
// into the free ids below n.  Writes the moves, the new counts, for every old
// id the new one, and the first `entries` of the table under the new ids.
// 8 us for 2048 pages with cold caches, half of it the three passes over refs.
__global__ void __launch_bounds__(kThreads) compact_plan_kernel(const int* __restrict__ refs, int pages,
                                                                int* __restrict__ new_refs, int* __restrict__ to,
                                                                int* __restrict__ src, int* __restrict__ dst,
                                                                int* __restrict__ moves, const int* __restrict__ table,
                                                                long long ld, int columns, int entries,
                                                                int* __restrict__ new_table) {
  __shared__ int sh[33];
  let_next_start();
  int live = 0;
  for (int p0 = 0; p0 < pages; p0 += kThreads) {
    const int p = p0 + threadIdx.x;
    live += __syncthreads_count(p < pages && refs[p] > 0);
  }
  int movers = 0, holes = 0;
  for (int p0 = 0; p0 < pages; p0 += kThreads) {
    const int p = p0 + threadIdx.x;
    const int r = p < pages ? refs[p] : 0;
    const bool mover = p < pages && r > 0 && p >= live, hole = p < live && r <= 0;
    int total;
    const int rank = block_scan((mover ? 1 << 16 : 0) | (hole ? 1 : 0), sh, &total);
    if (mover) src[movers + (rank >> 16)] = p;
    if (hole) dst[holes + (rank & 0xffff)] = p;
    if (p < pages) {
      new_refs[p] = p < live ? r : 0;
      to[p] = r > 0 ? p : -1;
    }
    movers += total >> 16;
    holes += total & 0xffff;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < movers; i += kThreads) {
    new_refs[dst[i]] = refs[src[i]];
    to[src[i]] = dst[i];
  }
  if (threadIdx.x == 0) *moves = movers;
  __syncthreads();
  for (int x = threadIdx.x; x < entries; x += kThreads) {
    const int p = table[(x / columns) * ld + x % columns];
    new_table[x] = p >= 0 && p < pages ? to[p] : -1;
  }
}

// 16-byte chunks of the named pages, in every plane: [planes][moves][chunks].
// Eight loads in flight per thread: 83 us for 477 MB (5.8 TB/s; four 97, two 88).
// `tokens` (or null) gives the leading tokens of each page that hold data.
// The kernel may start while the one that plans the copies still writes src,
// dst, tokens and count, so those are neither const nor __restrict__: nothing
// may read them ahead of wait_for_previous().
constexpr int kPer = 8;
__global__ void __launch_bounds__(256) copy_pages_kernel(uint4* __restrict__ pool, long long plane_chunks,
                                                         int page_chunks, int token_chunks, int planes, int pages,
                                                         int* src, int* dst, int* tokens, int* count, int n_max, int* status) {
  wait_for_previous();
  const int n = count ? min(*count, n_max) : n_max;
  const int runs = (page_chunks + 256 * kPer - 1) / (256 * kPer);
  const long long all = static_cast<long long>(n) * planes * runs;
  for (long long x = blockIdx.x; x < all; x += gridDim.x) {
    // plane by plane, so that a page that several children copy is still in L2 for the next one
    const int run = static_cast<int>(x % runs);
    const int i = static_cast<int>((x / runs) % n);
    const int plane = static_cast<int>(x / (static_cast<long long>(runs) * n));
    const int a = src[i], b = dst[i];
    if (a < 0 || b < 0) continue;
    if (a >= pages || b >= pages) {
      if (threadIdx.x == 0) flag(status, kErrBadIndex);
      continue;
    }
    const int valid = tokens ? min(tokens[i] * token_chunks, page_chunks) : page_chunks;
    const uint4* from = pool + plane * plane_chunks + static_cast<long long>(a) * page_chunks;
    uint4* into = pool + plane * plane_chunks + static_cast<long long>(b) * page_chunks;
    uint4 w[kPer];
    const int c0 = run * 256 * kPer + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (c0 + k * 256 < valid) w[k] = from[c0 + k * 256];
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (c0 + k * 256 < valid) into[c0 + k * 256] = w[k];
  }
}

// Table entries under the new ids.
__global__ void __launch_bounds__(256) remap_kernel(const int* __restrict__ table, long long ld, int columns, long long all,
                                                    const int* __restrict__ to, int pages, int* __restrict__ out) {
  const long long x = blockIdx.x * 256ll + threadIdx.x;
  if (x >= all) return;
  const int p = table[(x / columns) * ld + x % columns];
  out[x] = p >= 0 && p < pages ? to[p] : -1;
}

// One 16-byte chunk of one token's keys and of its values per thread and step:
// bound by the bytes, 216 MB (13,169 tokens, 16 heads of 128) in 39 us, 5.5 TB/s.
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ Append a, int* status) {
  const int per = a.heads * a.chunks;
  const long long all = static_cast<long long>(a.n) * per;
  for (long long x = blockIdx.x * 256ll + threadIdx.x; x < all; x += gridDim.x * 256ll) {
    const int i = static_cast<int>(x / per), r = static_cast<int>(x % per);
    const int pos = a.positions[i];
    if (pos < 0) continue;  // padding
    const int s = a.slot_of ? a.slot_of[i] : i;
    const int col = pos / a.page_size;
    if (s < 0 || s >= a.slots || col >= a.columns) {
      flag(status, kErrBadIndex);
      continue;
    }
    const int page = a.table[s * a.table_ld + col];
    if (page < 0 || page >= a.pages) {
      flag(status, kErrBadIndex);
      continue;
    }
    const int h = r / a.chunks, c = (r % a.chunks) * 8;
    const long long to = page * a.page_ld + (pos % a.page_size) * a.token_ld + h * a.head_ld + c;
    const uint4 wk = ld_v4(a.k + i * a.k_ld + h * a.k_head + c), wv = ld_v4(a.v + i * a.v_ld + h * a.v_head + c);
    st_v4(a.k_pool + to, wk);
    st_v4(a.v_pool + to, wv);
  }
}


namespace {
int copy_blocks(long long units) {
  // 148 SMs x 8 blocks of 256 threads cover the memory latency of a copy
  return static_cast<int>(std::max<long long>(1, std::min<long long>(units, 148 * 8)));
}
}  // namespace

cudaError_t launch_copy(const Pool& p, int* src, int* dst, int* tokens, int* count, int n, int* status, cudaStream_t stream) {
  if (n == 0) return cudaSuccess;
  const long long runs = (p.page_chunks + 256 * kPer - 1) / (256 * kPer);
  return launch_after(copy_pages_kernel, copy_blocks(static_cast<long long>(n) * p.planes * runs), 256, 0, stream,
                      static_cast<uint4*>(p.base), p.plane_chunks, p.page_chunks, p.token_chunks, p.planes, p.pages, src, dst,
                      tokens, count, n, status);
}

cudaError_t launch_fork(const Pool& p, const Table& t, const int* parents, const int* children, int n, int* scratch,
                        int* status, cudaStream_t stream) {
  int* s = scratch;
  fork_plan_kernel<<<1, kThreads, 0, stream>>>(t, parents, children, n, s + 4 * n, s, s + n, s + 2 * n, s + 3 * n, status);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  return launch_copy(p, s + n, s + 2 * n, s + 3 * n, nullptr, n, status, stream);
}

cudaError_t launch_reserve(const Table& t, const int* slots, const int* counts, int n, int* scratch, int* status,
                           cudaStream_t stream) {
  int* s = scratch;
  reserve_kernel<<<1, kThreads, 0, stream>>>(t, slots, counts, n, s + t.pages + n, s, t.pages, s + t.pages, status);
  return cudaGetLastError();
}

cudaError_t launch_free(const Table& t, const int* slots, int n, int* status, cudaStream_t stream) {
  const long long all = static_cast<long long>(n) * t.columns;
  free_kernel<<<copy_blocks((all + 255) / 256), 256, 0, stream>>>(t, slots, n, status);
  return cudaGetLastError();
}

cudaError_t launch_compact(const Pool& p, const int* table, long long table_ld, int rows, int columns, const int* refs,
                           int* new_table, int* new_refs, int* scratch, int* status, cudaStream_t stream) {
  int* s = scratch;
  const long long all = static_cast<long long>(rows) * columns;
  const bool small = all <= kSmallTable;
  compact_plan_kernel<<<1, kThreads, 0, stream>>>(refs, p.pages, new_refs, s, s + p.pages, s + 2 * p.pages, s + 3 * p.pages,
                                                  table, table_ld, columns, small ? static_cast<int>(all) : 0, new_table);
  if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  if (!small) {
    remap_kernel<<<static_cast<unsigned>((all + 255) / 256), 256, 0, stream>>>(table, table_ld, columns, all, s, p.pages,
                                                                               new_table);
    if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
  }
  return launch_copy(p, s + p.pages, s + 2 * p.pages, nullptr, s + 3 * p.pages, p.pages, status, stream);
}

cudaError_t launch_append(const Append& a, int* status, cudaStream_t stream) {
  const long long all = static_cast<long long>(a.n) * a.heads * a.chunks;
  append_kernel<<<copy_blocks((all + 255) / 256), 256, 0, stream>>>(a, status);
  return cudaGetLastError();
}

}  // namespace cache

}  // namespace mnb
