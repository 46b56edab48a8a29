// Appending to a paged key / value cache in 8 bits.
//
// A page and kv head share one scale, the least power of two s = 2^e (e from -60 on)
// with |x| <= top s for every value x stored there (top 127 for int8, 448 for e4m3); a
// value is stored as the code nearest to x / s, of two the even one.  A power of two
// costs int8 up to one bit and e4m3 nothing, and makes every step exact but the one
// rounding: x / s, what a code stands for (exact in bf16 too), and, where a later token
// does not fit and the scale grows, the codes' way to the new scale (e4m3 loses
// nothing but below its normal range; int8 at most a step of the last scale in all,
// however often the scale grew).  So the cache does not depend on how its tokens were
// split over calls by more than that, and a call gives the same bits every time.
//
// A warp takes one head of the keys or values of a run, the tokens of a call that go to
// one page: their largest value, the page's scale, the codes held so far where it grows,
// the new codes.  No two warps touch the same page and head, so there are no atomics.
#include <algorithm>

#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace cache {

namespace {

constexpr int kWarps = 2;  // (13 prompts of up to 1001 tokens 23 us; with 8, which start and end together, 25)

MNB_DEVICE uint32_t e4m3_pair(float lo, float hi) {
  uint16_t y;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(y) : "f"(hi), "f"(lo));
  return y;
}
MNB_DEVICE float2 of_e4m3_pair(uint32_t x) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(x)));
  float2 y;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(y.x), "=f"(y.y) : "r"(h));
  return y;
}
// The nearest whole number to x * by (of two the even one), for less than 2^22 of them, in the low bits.
MNB_DEVICE uint32_t nearest(float x, float by) { return __float_as_uint(fmaf(x, by, 12582912.f)); }
// The low bytes of four numbers.
MNB_DEVICE uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Four codes for the bf16 values in two words, times `by`.  (Values beyond every number count as the largest code of
// their sign; NaN is e4m3's NaN, and zero in int8, which has none.)
template <bool kFloat>
MNB_DEVICE uint32_t codes_of(uint32_t a, uint32_t b, float by) {
  const float2 x = unpack_bf16x2(a), y = unpack_bf16x2(b);
  if constexpr (kFloat) {
    return e4m3_pair(x.x * by, x.y * by) | e4m3_pair(y.x * by, y.y * by) << 16;
  } else {
    return bytes_of(nearest(x.x, by), nearest(x.y, by), nearest(y.x, by), nearest(y.y, by));
  }
}
MNB_DEVICE float within(float x) { return x != x ? 0.f : fminf(fmaxf(x, -127.f), 127.f); }

// Four codes under another scale.
template <bool kFloat>
MNB_DEVICE uint32_t rescaled(uint32_t w, float by) {
  if constexpr (kFloat) {
    const float2 x = of_e4m3_pair(w), y = of_e4m3_pair(w >> 16);
    return e4m3_pair(x.x * by, x.y * by) | e4m3_pair(y.x * by, y.y * by) << 16;
  } else {
    const int v = static_cast<int>(w);
    return bytes_of(nearest(static_cast<float>(v << 24 >> 24), by), nearest(static_cast<float>(v << 16 >> 24), by),
                    nearest(static_cast<float>(v << 8 >> 24), by), nearest(static_cast<float>(v >> 24), by));
  }
}

}  // namespace

// kKeep: 16-byte parts of tokens that a lane keeps between the two looks at them.
template <bool kFloat, int kKeep>
__global__ void __launch_bounds__(32 * kWarps) append8_kernel(const __grid_constant__ Append8 a, int window, int* status) {
  constexpr int kTop = kFloat ? 8 : 6;                        // the largest code is kMantissa 2^kTop
  constexpr uint32_t kMantissa = kFloat ? 0x600000 : 0x7e0000;  // 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  const int lane = threadIdx.x % 32;
  const long long unit = blockIdx.x * static_cast<long long>(kWarps) + threadIdx.x / 32;
  const int h = static_cast<int>(unit % a.heads), part = static_cast<int>(unit / a.heads % 2);
  const long long w0 = unit / (2 * a.heads) * window;
  if (w0 >= a.n) return;
  const __nv_bfloat16* const x = part ? a.v + h * a.v_head : a.k + h * a.k_head;
  const long long x_ld = part ? a.v_ld : a.k_ld;
  uint8_t* const pool = (part ? a.v_pool : a.k_pool) + h * a.head_ld;
  float* const scales = (part ? a.v_scales : a.k_scales) + h * a.scale_head;

  // Token i's page, -1 for one that is left out (padding, or a place that is none)
  auto page_of = [&](long long i, int& place) {
    const int pos = a.positions[i], s = a.slot_of ? a.slot_of[i] : static_cast<int>(i);
    if (pos < 0) return -1;
    const int col = pos / a.page_size;
    place = pos - col * a.page_size;
    int page = -1;
    if (s >= 0 && s < a.slots && col < a.columns) page = a.table[s * a.table_ld + col];
    if (page < 0 || page >= a.pages) {
      atomicCAS(status, 0, kErrBadIndex);
      return -1;
    }
    return page;
  };

  // The last lanes take the window's tokens, those before them the tokens before it: a token begins a run where the last
  // one before it that counts is of another page.
  const long long mine = w0 + window - 32 + lane;
  // (their values are on their way to L2 while the pages are looked up: the same prompts 26.3 -> 25.6 us)
  if (mine >= w0 && mine < a.n)
    for (int line = 0; line < a.dim; line += 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(x + mine * x_ld + line));
  int place = 0, next_place = 0;
  const int page = mine >= 0 && mine < a.n ? page_of(mine, place) : -1;
  // ... and the 32 tokens behind the window, where its last run may end
  const int next_page = w0 + window + lane < a.n ? page_of(w0 + window + lane, next_place) : -1;
  const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
  const unsigned below = there & ((1u << lane) - 1);
  int before = __shfl_sync(0xffffffffu, page, below ? 31 - __clz(below) : 0);
  int far = -1;  // of the tokens further back, where all of these are left out
  const bool none = __any_sync(0xffffffffu, lane >= 32 - window && page >= 0 && !below);
  for (long long j = w0 + window - 32; j > 0 && far < 0 && none; j -= 32) {
    int unused;
    const int p = j - 32 + lane >= 0 ? page_of(j - 32 + lane, unused) : -1;
    const unsigned some = __ballot_sync(0xffffffffu, p >= 0);
    if (some) far = __shfl_sync(0xffffffffu, p, 31 - __clz(some));
  }
  if (!below) before = far;
  unsigned begins = __ballot_sync(0xffffffffu, lane >= 32 - window && page >= 0 && before != page);

  const int lanes = a.dim / 8, together = 32 / lanes;  // lanes of a token, and tokens that a warp takes at once
  const int token = lane / lanes, chunk = lane % lanes * 8;
  for (; begins; begins &= begins - 1) {
    const int of = __ffs(begins) - 1;
    const long long i0 = w0 + window - 32 + of;
    const int p = __shfl_sync(0xffffffffu, page, of);
    // A run of a page that had one before it would meet that one's warp there: left out, where it can be seen from here.
    if (__ballot_sync(0xffffffffu, page == p) & ((1u << of) - 1)) {
      if (lane == 0) atomicCAS(status, 0, kErrScattered);
      continue;
    }
    // f(the run's tokens from c0 on: how many of 32 to look at, this lane's page and place)
    auto run = [&](auto f) {
      for (long long c0 = i0;; c0 += 32) {
        const int d = static_cast<int>(min(c0 + lane - (w0 + window), 32ll));  // (from -32 on)
        int q = __shfl_sync(0xffffffffu, page, d & 31), at = __shfl_sync(0xffffffffu, place, d & 31);
        const int next_q = __shfl_sync(0xffffffffu, next_page, d & 31), next_at = __shfl_sync(0xffffffffu, next_place, d & 31);
        if (d >= 0) q = next_q, at = next_at;
        if (c0 + lane >= a.n) q = -2;
        else if (d >= 32) q = page_of(c0 + lane, at);
        const unsigned end = __ballot_sync(0xffffffffu, q != p && q != -1);
        f(c0, end ? __ffs(end) - 1 : 32, q, at);
        if (end) return;
      }
    };
    // The run: how far it goes, whether it has the page's first place, and whether it is nothing but places one after another.
    long long end = i0;
    bool anew = false, plain = true;
    const int at0 = __shfl_sync(0xffffffffu, place, of);
    run([&](long long c0, int count, int q, int at) {
      end = c0 + count;
      anew = anew || __any_sync(0xffffffffu, lane < count && q == p && at == 0);
      plain = plain && __all_sync(0xffffffffu, lane >= count || (q == p && at == at0 + c0 + lane - i0));
    });
    const int count = static_cast<int>(end - i0);
    // The tokens in rounds of kKeep for each lane; those of the last round stay in registers (for pages of 32 tokens and head
    // dim 128 that is all of them).
    uint4 w[kKeep];
    auto load = [&](int from) {
#pragma unroll
      for (int r = 0; r < kKeep; ++r) {
        const int j = from + r * together + token;
        w[r] = make_uint4(0, 0, 0, 0);
        if (token < together && j < count) w[r] = ld_v4(x + (i0 + j) * x_ld + chunk);
      }
    };
    auto largest = [&](uint32_t m) {  // of both halves of a word, with every lane's
      m = max(m & 0xffffu, m >> 16);
      return __reduce_max_sync(0xffffffffu, m);
    };
    const int round = kKeep * together, last = count > 0 ? (count - 1) / round * round : 0;
    uint32_t most = 0;  // pairs, as bits
    if (plain)
      for (int from = 0; from <= last; from += round) {
        load(from);
#pragma unroll
        for (int r = 0; r < kKeep; ++r)
          most = __vmaxu2(most, __vmaxu2(__vmaxu2(w[r].x & 0x7fff7fffu, w[r].y & 0x7fff7fffu), __vmaxu2(w[r].z & 0x7fff7fffu, w[r].w & 0x7fff7fffu)));
      }
    most = largest(most);
    if (!plain || most >= 0x7f80u) {  // padding in between, or something that is no finite number, which does not count
      plain = false;
      most = 0;
      run([&](long long c0, int n, int q, int at) {
        for (int b = 0; b < n; b += together) {
          const int j = b + token;
          const int of_page = __shfl_sync(0xffffffffu, q, min(j, 31));
          if (token >= together || j >= n || of_page != p) continue;
          const uint4 u = ld_v4(x + (c0 + j) * x_ld + chunk);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = (&u.x)[e], lo = v & 0x7fffu, hi = v >> 16 & 0x7fffu;
            most = max(most, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
          }
        }
      });
      most = largest(most);
    }
    most <<= 16;
    const int e = max(static_cast<int>(most >> 23) - 127 - kTop + ((most & 0x7fffff) > kMantissa), -60);
    const float need = __int_as_float((e + 127) << 23);
    float* const scale_at = scales + p * a.scale_ld;
    const float held = anew ? 0.f : *scale_at, now = held > need ? held : need;
    uint8_t* const to = pool + p * a.page_ld;
    if (!anew && now != held) {
      const float by = held > 0.f ? held / now : 0.f;
      for (int b = 0; b < a.page_size; b += together) {
        if (token >= together || b + token >= a.page_size) continue;
        uint2* const c = reinterpret_cast<uint2*>(to + (b + token) * a.token_ld + chunk);
        const uint2 u = *c;
        *c = make_uint2(rescaled<kFloat>(u.x, by), rescaled<kFloat>(u.y, by));
      }
    }
    __syncwarp();  // (also: every lane has read the scale)
    if (lane == 0) *scale_at = now;
    const float by = 1.f / now;
    if (plain) {
      for (int from = last; from >= 0; from -= round) {
        if (from != last) load(from);
#pragma unroll
        for (int r = 0; r < kKeep; ++r) {
          const int j = from + r * together + token;
          if (token < together && j < count)
            *reinterpret_cast<uint2*>(to + (at0 + j) * a.token_ld + chunk) =
                make_uint2(codes_of<kFloat>(w[r].x, w[r].y, by), codes_of<kFloat>(w[r].z, w[r].w, by));
        }
      }
      continue;
    }
    run([&](long long c0, int n, int q, int at) {
      for (int b = 0; b < n; b += together) {
        const int j = b + token;
        const int of_page = __shfl_sync(0xffffffffu, q, min(j, 31)), of_place = __shfl_sync(0xffffffffu, at, min(j, 31));
        bool in = token < together && j < n && of_page == p;
        for (int d = 1; d < together; ++d) {  // a place that is named twice gets the later token
          const int other = __shfl_down_sync(0xffffffffu, in ? of_place : -1, d * lanes);
          if (token + d < together && other == of_place) in = false;
        }
        if (in) {
          const uint4 u = ld_v4(x + (c0 + j) * x_ld + chunk);
          uint2 c = make_uint2(codes_of<kFloat>(u.x, u.y, by), codes_of<kFloat>(u.z, u.w, by));
          if constexpr (!kFloat) {
            uint32_t code[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 v = unpack_bf16x2((&u.x)[k]);
              if (v.x != v.x || v.y != v.y) atomicCAS(status, 0, kErrNotANumber);
              code[2 * k] = nearest(within(v.x * by), 1.f), code[2 * k + 1] = nearest(within(v.y * by), 1.f);
            }
            c = make_uint2(bytes_of(code[0], code[1], code[2], code[3]), bytes_of(code[4], code[5], code[6], code[7]));
          }
          *reinterpret_cast<uint2*>(to + of_place * a.token_ld + chunk) = c;
        }
        __syncwarp();
      }
    });
  }
}

cudaError_t launch_append8(const Append8& a, int* status, cudaStream_t stream) {
  // A warp looks for the runs that begin in `window` tokens: one token each while the GPU has room for their warps, more
  // for long prompts, whose runs are a page.
  int window = 1;
  while (window < 32 && (a.n + window - 1ll) / window * a.heads * 2 > 148 * 48) window *= 2;
  const long long warps = (a.n + window - 1ll) / window * a.heads * 2;
  const unsigned blocks = static_cast<unsigned>((warps + kWarps - 1) / kWarps);
  const auto kernel = a.e4m3 ? (window == 1 ? append8_kernel<true, 2> : append8_kernel<true, 16>)
                             : (window == 1 ? append8_kernel<false, 2> : append8_kernel<false, 16>);
  kernel<<<blocks, 32 * kWarps, 0, stream>>>(a, window, status);
  return cudaGetLastError();
}

}  // namespace cache

}  // namespace mnb
