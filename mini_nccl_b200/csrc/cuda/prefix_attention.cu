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
// Decoding is bound by the bytes of keys and values; one block keeps two
// 64-key tiles of K and V in flight with cp.async while warps work on a third
// (mma.sync m16n8k16, scores and probabilities in registers).  Query rows of
// the heads of one kv head (grouped heads) share a tile of 16, 32 or 64 rows.
// Scores, maxima, sums and outputs are fp32; only the probabilities are
// rounded to bf16, as the operand of the product with V.
#include <algorithm>

#include "common.cuh"
#include "generation.h"
#include "warp_mma.cuh"

namespace mnb {

namespace prefix {

constexpr int kThreads = 128;
constexpr int kKeys = 64;  // keys per tile
constexpr int kStages = 3;
constexpr int kTensorCoreRows = 32;  // more rows of a kv head than this go to the tensor-core kernel
constexpr float kLn2 = 0.6931471805599453f;

template <int D, int WR>
struct Smem {
  static constexpr int rows = 16 * WR;
  static constexpr uint32_t q_bytes = rows * D * 2;
  static constexpr uint32_t tile = kKeys * D * 2;
  static constexpr uint32_t total = q_bytes + kStages * 2 * tile;
};

// One piece: rows [0, n_rows) of a tile (row r is token n0 + r / group, head
// h * group + r % group), keys [k0, k1) named by `ids`.  Row r sees all of
// them, or (own tokens) those below limit0 + r / group.
template <int D, int WR, bool Causal>
MNB_DEVICE void attend(const Args& a, uint8_t* sm, int piece, int h, int n0, int r0, int n_rows, const int* ids, int k0,
                       int k1, int limit0) {
  using S = Smem<D, WR>;
  constexpr int WK = 4 / WR;         // key groups: warps that share rows
  constexpr int KW = kKeys / WK;     // keys of a tile per warp
  constexpr int chunks = D / 8;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int wr = warp % WR, wk = warp / WR;
  const int gq = lane / 4, tg = lane % 4;
  const uint32_t sQ = smem_u32(sm);
  const uint32_t sKV = sQ + S::q_bytes;

  auto row_token = [&](int r) { return n0 + (r0 + r) / a.group; };
  auto row_head = [&](int r) { return h * a.group + (r0 + r) % a.group; };

  for (int i = threadIdx.x; i < S::rows * chunks; i += kThreads) {
    const int r = i / chunks, c = i % chunks;
    const bool ok = r < n_rows;
    const int rr = ok ? r : 0;
    cp_async16(sQ + swz<D>(r, c), a.q + row_token(rr) * a.q_ld + row_head(rr) * a.q_head + c * 8, ok);
  }
  auto load_tile = [&](int stage, int j0) {
    const uint32_t sK = sKV + stage * 2 * S::tile, sV = sK + S::tile;
    for (int i = threadIdx.x; i < kKeys * chunks; i += kThreads) {
      const int r = i / chunks, c = i % chunks;
      const int j = j0 + r;
      bool ok = j < k1;
      long long at = 0;
      if (ok) {
        const int page = ids[j >> a.page_shift];
        ok = page >= 0 && page < a.pages;
        if (ok)
          at = page * a.page_ld + (j & ((1 << a.page_shift) - 1)) * a.token_ld + h * a.head_ld + c * 8;
        else
          atomicCAS(a.status, 0, kErrBadIndex);
      }
      cp_async16(sK + swz<D>(r, c), a.k + at, ok);
      cp_async16(sV + swz<D>(r, c), a.v + at, ok);
    }
  };
  const int tiles = (k1 - k0 + kKeys - 1) / kKeys;
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < tiles) load_tile(s, k0 + s * kKeys);
    cp_async_commit();
  }

  float acc[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
  float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.f, 0.f};
  uint32_t qf[D / 16][4];
  // keys below lim[i] are visible to this thread's row i
  int lim[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wr * 16 + gq + 8 * i;
    lim[i] = Causal ? min(k1, limit0 + (r0 + r) / a.group) : k1;
  }

  for (int t = 0; t < tiles; ++t) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (t + kStages - 1 < tiles) load_tile((t + kStages - 1) % kStages, k0 + (t + kStages - 1) * kKeys);
    cp_async_commit();
    if (t == 0) {
#pragma unroll
      for (int kc = 0; kc < D / 16; ++kc)
        ldsm_x4(qf[kc], sQ + swz<D>(wr * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, kc * 2 + (lane >> 4)));
    }
    const uint32_t sK = sKV + (t % kStages) * 2 * S::tile, sV = sK + S::tile;
    float s[KW / 8][4];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kc = 0; kc < D / 16; ++kc)
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        uint32_t b[4];
        ldsm_x4(b, sK + swz<D>(wk * KW + n * 16 + (lane & 7) + (lane >> 4) * 8, kc * 2 + ((lane >> 3) & 1)));
        mma_bf16(s[2 * n], qf[kc], b);
        mma_bf16(s[2 * n + 1], qf[kc], b + 2);
      }
    const int j0 = k0 + t * kKeys + wk * KW + 2 * tg;
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
    for (int i = 0; i < 2; ++i) {
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
      mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
      const float base = mx[i] == -INFINITY ? 0.f : mx[i];  // no key yet: every weight is exp2(-inf) = 0
      const float alpha = ex2_approx(m_r[i] - base);
      m_r[i] = mx[i];
      l_r[i] *= alpha;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        acc[d][2 * i] *= alpha;
        acc[d][2 * i + 1] *= alpha;
      }
#pragma unroll
      for (int n = 0; n < KW / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = ex2_approx(s[n][2 * i + e] - base);
          s[n][2 * i + e] = p;
          l_r[i] += p;
        }
    }
#pragma unroll
    for (int n = 0; n < KW / 16; ++n) {
      const uint32_t pa[4] = {pack_bf16x2(s[2 * n][0], s[2 * n][1]), pack_bf16x2(s[2 * n][2], s[2 * n][3]),
                              pack_bf16x2(s[2 * n + 1][0], s[2 * n + 1][1]), pack_bf16x2(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        uint32_t b[4];
        ldsm_x4_t(b, sV + swz<D>(wk * KW + n * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, d * 2 + (lane >> 4)));
        mma_bf16(acc[2 * d], pa, b);
        mma_bf16(acc[2 * d + 1], pa, b + 2);
      }
    }
  }
  cp_async_wait_all();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l_r[i] += __shfl_xor_sync(0xffffffffu, l_r[i], 1);
    l_r[i] += __shfl_xor_sync(0xffffffffu, l_r[i], 2);
  }
  // The key groups of a row join through shared memory (the K / V stages are free now).
  if constexpr (WK > 1) {
    float* so = reinterpret_cast<float*>(sm + S::q_bytes);        // [4 warps][16][D + 4]
    float2* sml = reinterpret_cast<float2*>(so + 4 * 16 * (D + 4));  // [4 warps][16]
    static_assert(4 * 16 * (D + 4) * 4 + 4 * 16 * 8 <= kStages * 2 * S::tile, "the join fits the stages");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = gq + 8 * i;
      if (tg == 0) sml[warp * 16 + r] = make_float2(m_r[i], l_r[i]);
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(so + (warp * 16 + r) * (D + 4) + d * 8 + 2 * tg) = make_float2(acc[d][2 * i], acc[d][2 * i + 1]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < n_rows * (D / 4); x += kThreads) {
      const int r = x / (D / 4), c = x % (D / 4) * 4;
      const int w0 = r / 16;  // warps w0 + g * WR hold this row
      float m = -INFINITY;
#pragma unroll
      for (int g = 0; g < WK; ++g) m = fmaxf(m, sml[(w0 + g * WR) * 16 + r % 16].x);
      const float base = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int g = 0; g < WK; ++g) {
        const int at = (w0 + g * WR) * 16 + r % 16;
        const float f = ex2_approx(sml[at].x - base);
        const float4 p = *reinterpret_cast<const float4*>(so + at * (D + 4) + c);
        l = fmaf(f, sml[at].y, l);
        o.x = fmaf(f, p.x, o.x);
        o.y = fmaf(f, p.y, o.y);
        o.z = fmaf(f, p.z, o.z);
        o.w = fmaf(f, p.w, o.w);
      }
      const long long out = (static_cast<long long>(piece) * a.n + row_token(r)) * a.heads + row_head(r);
      *reinterpret_cast<float4*>(a.part_o + out * D + c) = o;
      if (c == 0) a.part_ml[out] = make_float2(m, l);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = wr * 16 + gq + 8 * i;
      if (r >= n_rows) continue;
      const long long out = (static_cast<long long>(piece) * a.n + row_token(r)) * a.heads + row_head(r);
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<float2*>(a.part_o + out * D + d * 8 + 2 * tg) = make_float2(acc[d][2 * i], acc[d][2 * i + 1]);
      if (tg == 0) a.part_ml[out] = make_float2(m_r[i], l_r[i]);
    }
  }
}

// Prefix pieces: (split, kv head, row tile), row tiles of the same keys side by side.
template <int D, int WR>
__global__ void __launch_bounds__(kThreads) prefix_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(128) uint8_t sm[];
  const int rt = blockIdx.x % a.row_tiles;
  const int h = (blockIdx.x / a.row_tiles) % a.kv_heads;
  const int split = blockIdx.x / (a.row_tiles * a.kv_heads);
  const int r0 = rt * 16 * WR;
  const int k0 = split * a.prefix_chunk;
  attend<D, WR, false>(a, sm, split, h, 0, r0, min(16 * WR, a.n * a.group - r0), a.prefix_pages, k0,
                min(a.prefix_len, k0 + a.prefix_chunk), 0);
}

// Own pieces: (sequence, row tile, split, kv head).
template <int D, int WR>
__global__ void __launch_bounds__(kThreads) own_kernel(const __grid_constant__ Args a) {
  extern __shared__ __align__(128) uint8_t sm[];
  const int h = blockIdx.x % a.kv_heads;
  const int split = (blockIdx.x / a.kv_heads) % a.own_splits;
  const int rt = (blockIdx.x / (a.kv_heads * a.own_splits)) % a.own_tiles;
  const int b = blockIdx.x / (a.kv_heads * a.own_splits * a.own_tiles);
  int n0 = b, q_len = 1;
  if (a.q_offsets) {
    n0 = min(max(a.q_offsets[b], 0), a.n);
    q_len = min(max(a.q_offsets[b + 1] - n0, 0), a.n - n0);
    if (q_len > a.max_q) {
      if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
      q_len = a.max_q;
    }
  }
  const int r0 = rt * 16 * WR;
  const int n_rows = min(16 * WR, q_len * a.group - r0);
  if (n_rows <= 0) return;
  int len = a.seq_lens[b];
  if (len < 0 || len > a.max_len) {
    if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
    len = min(max(len, 0), a.max_len);
  }
  const int k0 = split * a.own_chunk;
  // the newest row of the tile sees the most keys
  const int seen = max(0, len - q_len + 1 + (r0 + n_rows - 1) / a.group);
  const int k1 = min(min(len, seen), k0 + a.own_chunk);
  const int piece = a.prefix_splits + split;
  if (k1 <= k0) {  // nothing here: the join skips the piece
    for (int r = threadIdx.x; r < n_rows; r += kThreads)
      a.part_ml[(static_cast<long long>(piece) * a.n + n0 + (r0 + r) / a.group) * a.heads + h * a.group + (r0 + r) % a.group] =
          make_float2(-INFINITY, 0.f);
    return;
  }
  attend<D, WR, true>(a, sm, piece, h, n0, r0, n_rows, a.page_table + b * a.table_ld, k0, k1, len - q_len + 1);
}

// One warp joins the pieces of one (token, head).
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Args a) {
  const long long row = blockIdx.x * 8ll + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const long long rows = static_cast<long long>(a.n) * a.heads;
  if (row >= rows) return;
  const int pieces = a.prefix_splits + a.own_splits;
  float m = -INFINITY;
  for (int p = lane; p < pieces; p += 32) m = fmaxf(m, a.part_ml[p * rows + row].x);
  m = warp_max(m);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  constexpr int per = D / 32;
  float o[per];
#pragma unroll
  for (int i = 0; i < per; ++i) o[i] = 0.f;
  for (int p = 0; p < pieces; ++p) {
    const float2 ml = a.part_ml[p * rows + row];
    if (ml.x == -INFINITY) continue;
    const float f = ex2_approx(ml.x - base);
    l = fmaf(f, ml.y, l);
    const float* po = a.part_o + (p * rows + row) * D + lane * per;
#pragma unroll
    for (int i = 0; i < per; ++i) o[i] = fmaf(f, po[i], o[i]);
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;  // a row without keys is zero
#pragma unroll
  for (int i = 0; i < per; ++i) a.o[row * D + lane * per + i] = f32_to_bf16(o[i] * inv);
  if (a.lse && lane == 0) a.lse[row] = l > 0.f ? kLn2 * (m + log2f(l)) : -INFINITY;
}

int row_warps(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
int ceil_div(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

template <int D, int WR>
static cudaError_t launch_prefix(const Args& a, cudaStream_t stream) {
  constexpr int bytes = Smem<D, WR>::total;
  if (const cudaError_t e = cudaFuncSetAttribute(prefix_kernel<D, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      e != cudaSuccess)
    return e;
  prefix_kernel<D, WR><<<a.row_tiles * a.kv_heads * a.prefix_splits, kThreads, bytes, stream>>>(a);
  return cudaGetLastError();
}
template <int D, int WR>
static cudaError_t launch_own(const Args& a, cudaStream_t stream) {
  constexpr int bytes = Smem<D, WR>::total;
  if (const cudaError_t e = cudaFuncSetAttribute(own_kernel<D, WR>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      e != cudaSuccess)
    return e;
  own_kernel<D, WR><<<a.batch * a.own_tiles * a.own_splits * a.kv_heads, kThreads, bytes, stream>>>(a);
  return cudaGetLastError();
}

template <int D>
static cudaError_t launch_for(const Args& a, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (a.own_splits > 0) {
    const int w = row_warps(a.max_q * a.group);
    e = w == 1 ? launch_own<D, 1>(a, stream) : w == 2 ? launch_own<D, 2>(a, stream) : launch_own<D, 4>(a, stream);
  }
  if (e == cudaSuccess && a.prefix_splits > 0) {
    if (a.tensor_cores) {
      e = launch_prefix_tc(a, D, stream);
      if (a.prefix_splits == 1) return e;
    } else {
      const int w = row_warps(a.n * a.group);
      e = w == 1 ? launch_prefix<D, 1>(a, stream) : w == 2 ? launch_prefix<D, 2>(a, stream) : launch_prefix<D, 4>(a, stream);
    }
  }
  if (e != cudaSuccess) return e;
  join_kernel<D><<<ceil_div(static_cast<long long>(a.n) * a.heads, 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

// Splits of the tensor-core kernel: whole waves of one block per SM, each taking its tiles and a fixed part, and the
// partial outputs written and read when there are several.
static int tc_splits(int blocks, int tiles, long long rows, int head_dim, bool wide) {
  const double tile_us = wide ? 1.5 : 0.8, fixed_us = 4.0;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= std::min(tiles, 64); ++s) {
    const int per = ceil_div(tiles, s), pieces = ceil_div(tiles, per);
    double us = ceil_div(static_cast<long long>(blocks) * pieces, 148) * (per * tile_us + fixed_us);
    if (pieces > 1) us += 3.0 + pieces * rows * head_dim * 8 / 6.5e6;
    if (us < least * 0.999) least = us, best = s;
  }
  return best;
}

int plan(Args& a, int head_dim) {
  // Two blocks fit an SM (64 KB of tiles each); split until there are about two waves of them.
  constexpr int kWant = 148 * 2 * 2;
  a.prefix_splits = a.own_splits = 0;
  if (a.prefix_len > 0) {
    const long long rows = static_cast<long long>(a.n) * a.group;
    a.tensor_cores = head_dim != 32 && rows > kTensorCoreRows && a.scale_log2 >= 0.f && a.head_ld > 0 && a.token_ld > 0 && a.page_ld > 0;
    if (a.tensor_cores) {
      a.row_tiles = ceil_div(rows, 256);
      const int tiles = ceil_div(a.prefix_len, 128);
      const int splits = tc_splits(a.row_tiles * a.kv_heads, tiles, rows * a.kv_heads, head_dim, rows > 128);
      a.prefix_chunk = ceil_div(tiles, splits) * 128;
    } else {
      a.row_tiles = ceil_div(rows, 16 * row_warps(a.n * a.group));
      const int tiles = ceil_div(a.prefix_len, kKeys);
      const int splits = std::max(1, std::min({tiles, 64, ceil_div(kWant, static_cast<long long>(a.row_tiles) * a.kv_heads)}));
      a.prefix_chunk = ceil_div(tiles, splits) * kKeys;
    }
    a.prefix_splits = ceil_div(a.prefix_len, a.prefix_chunk);
  }
  if (a.max_len > 0 && a.max_q > 0 && a.batch > 0) {
    a.own_tiles = ceil_div(static_cast<long long>(a.max_q) * a.group, 16 * row_warps(a.max_q * a.group));
    const int tiles = ceil_div(a.max_len, kKeys);
    const int splits =
        std::max(1, std::min({tiles, 64, ceil_div(kWant, static_cast<long long>(a.batch) * a.own_tiles * a.kv_heads)}));
    a.own_chunk = ceil_div(tiles, splits) * kKeys;
    a.own_splits = ceil_div(a.max_len, a.own_chunk);
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
