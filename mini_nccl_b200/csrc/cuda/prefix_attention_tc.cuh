// Device helpers of the shared-prefix attention's tensor-core kernels
// (prefix_attention_tc.cu for bf16 pages, prefix_attention_8bit_tc.cu for codes in 8 bits).
#pragma once

#include "launch.cuh"
#include "prefix_attention.cuh"

namespace mnb {

namespace prefix {

namespace tc {

constexpr int kTile = 128;     // rows per stream and keys per tile
constexpr int kSoftmax = 512;  // threads: two warpgroups for each stream, each with half the keys of a tile
constexpr float kLn2 = 0.6931471805599453f;

MNB_DEVICE void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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

// Shared memory that finish_rows() uses.
template <int D>
constexpr int kMeeting = 2 * kTile * ((D + 4) * 4 + 8 + 20 + 4);

// The end of a block's softmax warps (number `self` of 16): row r of stream s has its base m, its half's sum l and its output
// at t_o in TMEM.  With one prefix piece the rows are joined with their own keys' pieces and finished.  kBatch: rows of a warp
// whose loads are under way together.
template <int D, int kBatch>
MNB_DEVICE void finish_rows(const Args& a, uint8_t* ring, uint32_t t_o, float m, float l, int steps, int s, int half, int r, int self,
                            int n_rows, int r0, int h, int split, bool shared) {
  const int lane = threadIdx.x % 32;
  // Outputs, maxima and sums pass through the ring, which nobody uses any more once both streams have theirs, so that
  // a warp can write whole rows; streams of the same rows meet there.
  constexpr int kPitch = D + 4, kPer = D / 32;
  float* meet = reinterpret_cast<float*>(ring);
  float2* meet_ml = reinterpret_cast<float2*>(meet + 2 * kTile * kPitch);
  struct Row {  // where a row goes, and the factors of its parts
    int at;
    float top, mine, met, inv;
  };
  Row* info = reinterpret_cast<Row*>(meet_ml + 2 * kTile);
  float* meet_l = reinterpret_cast<float*>(info + 2 * kTile);  // the second half's sums
  static_assert(2 * kTile * (kPitch * 4 + 8 + sizeof(Row) + 4) <= kMeeting<D>, "the meeting place");
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
  for (int i0 = self * kBatch; i0 < n_rows; i0 += kSoftmax / 32 * kBatch) {
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
}

}  // namespace tc

}  // namespace prefix

}  // namespace mnb
