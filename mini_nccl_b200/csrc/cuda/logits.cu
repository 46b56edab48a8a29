// Penalties, biases and masks on logits before sampling.
//
// With c the number of times that token v is in row r's history and x its logit:
//   x = x > 0 ? x / repetition : x repetition   where v is in the history or the prompt,
//   x = x - (frequency c + presence)            where v is in the history,
//   x = x + bias                                where the row names v,
//   x = -inf                                    where the row's mask does not allow v,
// in fp32, one IEEE operation after another, rounded once to the logits' type.
//
// Bound by the bytes of the logits, once in and once out.  A block takes a run of a
// row's tokens: it copies their logits under the mask (those of tokens that the mask
// forbids are not read), and then rewrites the few that the row's lists name.  For
// that, one word of shared memory for each token counts it (whole numbers, so the order
// does not matter), remembers whether the prompt has it and which bias it gets; whoever
// takes the word out first writes the token.  Only words of named tokens are ever
// touched.  (Penalties applied on the way, in the copying pass, cost every warp the
// arithmetic of each of its lanes' tokens in turn: 512 x 50304 with 1300 tokens named in
// a row, 63 us.)  Measured: 512 x 50304 in bf16 33 us (3.1 TB/s; the lists are read by
// each of a row's seven blocks), 129 x 130003 in fp32 under a mask and biases each
// 33 us (4.1 TB/s), 64 x 50304 in fp32 under masks that leave a twenty-fifth 9 us, one
// row 4 us.
#include <algorithm>

#include "common.cuh"
#include "generation.h"
#include "launch.cuh"

namespace mnb {

namespace logits {

namespace {

constexpr uint32_t kCount = (1u << kCountBits) - 1, kPrompt = 1u << kCountBits;  // and the bias' index + 1 above
constexpr int kBiasShift = kCountBits + 1;

MNB_DEVICE long long id_at(const Ids& t, long long i) {
  return t.wide ? static_cast<const long long*>(t.ids)[i] : static_cast<const int*>(t.ids)[i];
}

MNB_DEVICE float adjusted(float x, uint32_t named, float repetition, float presence, float frequency, const float* bias) {
  const uint32_t count = named & kCount;
  if (named & (kCount | kPrompt)) x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
  if (count) x = __fsub_rn(x, __fadd_rn(__fmul_rn(frequency, static_cast<float>(count)), presence));
  if (named >> kBiasShift) x = __fadd_rn(x, bias[(named >> kBiasShift) - 1]);
  return x;
}

// A block takes kThreads * kPer groups of eight tokens of a row.  (Six blocks to an SM fit fp32, 34 -> 32 us at 129 x 130003, at
// the price of some registers spilled; with bf16 their shared memory would take too much of L1, 34 -> 37 us at 512 x 50304.)
template <bool kBf16, int kThreads, int kPer>
__global__ void __launch_bounds__(kThreads, kBf16 ? 5 : 6) adjust_kernel(const __grid_constant__ Adjust a, int chunks) {
  constexpr int kSize = kBf16 ? 2 : 4, kWords = kBf16 ? 4 : 8, kTokens = kThreads * kPer * 8, kList = 2048;
  static_assert(kTokens <= 1 << 14, "a place's bits");
  extern __shared__ uint32_t named[];  // [kTokens], where some list names tokens
  // Places, and which list names them.  (32 bits each would be room for half as many: 82 rows with a prompt of 2232 tokens 17
  // us, so 11.  More room takes it from L1: 512 x 50304 35 us, so 33.)
  __shared__ uint16_t list[kList];
  __shared__ int listed;
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const char* const in = static_cast<const char*>(a.in) + row * a.in_ld * kSize;
  char* const out = static_cast<char*>(a.out) + row * a.out_ld * kSize;
  // The groups follow the output's alignment to 16 bytes: the row's first token is number `skip` of the first group.
  const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16) / kSize;
  const int first = chunk * kTokens - skip;  // the chunk's first token (below 0: before the row)
  const bool in_aligned = reinterpret_cast<uintptr_t>(in + first * kSize) % 16 == 0;

  int of = -1;  // the row's mask
  if (a.mask_of || a.masks > 0) {
    of = a.mask_of ? a.mask_of[row] : a.masks > 1 ? row : 0;
    if (of >= a.masks) {
      if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
      of = -1;
    }
  }
  const uint32_t* const mask = of >= 0 ? a.allowed + of * a.mask_ld : nullptr;
  const int words = (a.vocab + 31) / 32;

  // The copy, under the mask: its loads are on their way while the lists are looked through.
  const bool copies = !a.in_place || mask;
  auto token_of = [&](int k) { return first + (k * kThreads + static_cast<int>(threadIdx.x)) * 8; };
  uint32_t allowed[kPer];  // of each group's tokens
  uint32_t x[kPer][kWords];
  if (copies) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int v = token_of(k);
      allowed[k] = 0xff;
      if (mask && v < a.vocab && v + 8 > 0) {
        const int at = max(v, 0), w = at >> 5;
        const uint32_t lo = mask[w], hi = w + 1 < words && (at & 31) > 24 ? mask[w + 1] : 0u;
        allowed[k] = (__funnelshift_r(lo, hi, at & 31) << (at - v)) & 0xff;
      }
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int v = token_of(k);
#pragma unroll
      for (int e = 0; e < kWords; ++e) x[k][e] = 0;
      if (v >= a.vocab || !allowed[k] || (a.in_place && allowed[k] == 0xff)) continue;
      if (in_aligned && v >= 0 && v + 8 <= a.vocab) {
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q) {
          const uint4 y = ld_v4(in + static_cast<long long>(v) * kSize + 16 * q);
          x[k][4 * q] = y.x, x[k][4 * q + 1] = y.y, x[k][4 * q + 2] = y.z, x[k][4 * q + 3] = y.w;
        }
        continue;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v + e >= 0 && v + e < a.vocab) {
          if constexpr (kBf16)
            x[k][e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(in)[v + e]) << (e % 2 * 16);
          else
            x[k][e] = reinterpret_cast<const uint32_t*>(in)[v + e];
        }
    }
  }

  // The tokens of the row's lists that lie in the chunk: place, list (0 history, 1 prompt, 2 biases) and, of a bias, which.
  int held = static_cast<int>(a.history.n);
  if (a.history_lens) {
    held = a.history_lens[row];
    if (held < 0 || held > a.history.n) {
      if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
      held = 0;
    }
  }
  const int prompts = static_cast<int>(a.prompt.n), biases = static_cast<int>(a.bias_tokens.n);
  const bool names = prompts > 0 || held > 0 || biases > 0;
  auto scan = [&](const Ids& t, int n, uint32_t kind, auto f) {
    constexpr int kAhead = 4;
    for (int i0 = threadIdx.x; i0 < n; i0 += kAhead * kThreads) {
      long long v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = i0 + k * kThreads < n ? id_at(t, row * t.ld + i0 + k * kThreads) : -1;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint32_t at = static_cast<uint32_t>(v[k]) - static_cast<uint32_t>(first);
        if (static_cast<unsigned long long>(v[k]) >= static_cast<unsigned long long>(a.vocab)) {
          if (v[k] >= 0 && chunk == 0) atomicCAS(a.status, 0, kErrBadIndex);
        } else if (at < kTokens) {
          f(at | kind << 14 | (kind == 2 ? i0 + k * kThreads : 0) << 16);
        }
      }
    }
  };
  auto scan_all = [&](auto f) {
    scan(a.prompt, prompts, 1, f);
    scan(a.history, held, 0, f);
    scan(a.bias_tokens, biases, 2, f);
  };
  // (more of them than the list has room for are looked for again each time)
  auto each = [&](auto f) {
    const int n = listed;
    if (n > kList) scan_all(f);
    else
      for (int i = threadIdx.x; i < n; i += kThreads) f(static_cast<uint32_t>(list[i]));
  };
  auto place = [](uint32_t x) { return x & 0x3fffu; };
  auto kind = [](uint32_t x) { return x >> 14 & 3u; };
  if (names) {
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    scan_all([&](uint32_t x) {
      named[place(x)] = 0;
      const int i = atomicAdd(&listed, 1);
      if (i < kList) list[i] = static_cast<uint16_t>(x);
    });
    __syncthreads();
    if (biases > 0) {  // (the later one of a token that is named twice)
      scan(a.bias_tokens, biases, 2, [&](uint32_t x) { atomicMax(named + place(x), ((x >> 16) + 1) << kBiasShift); });
      __syncthreads();
    }
    each([&](uint32_t x) {
      if (kind(x) == 0) atomicAdd(named + place(x), 1u);
      if (kind(x) == 1) atomicOr(named + place(x), kPrompt);
    });
  }

  // The copy's end
  if (copies) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int v = token_of(k);
      if (v >= a.vocab || (a.in_place && allowed[k] == 0xff)) continue;
      if (allowed[k] != 0xff) {
#pragma unroll
        for (int e = 0; e < kWords; ++e) {
          if constexpr (kBf16) {
            const uint32_t two = allowed[k] >> 2 * e, keep = (two & 1u) * 0xffffu | (two >> 1 & 1u) * 0xffff0000u;
            x[k][e] = (x[k][e] & keep) | (0xff80ff80u & ~keep);
          } else {
            x[k][e] = allowed[k] >> e & 1 ? x[k][e] : 0xff800000u;
          }
        }
      }
      if (v >= 0 && v + 8 <= a.vocab) {
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q)
          st_v4(out + static_cast<long long>(v) * kSize + 16 * q, make_uint4(x[k][4 * q], x[k][4 * q + 1], x[k][4 * q + 2], x[k][4 * q + 3]));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v + e >= 0 && v + e < a.vocab) {
            if constexpr (kBf16)
              reinterpret_cast<uint16_t*>(out)[v + e] = static_cast<uint16_t>(x[k][e / 2] >> (e % 2 * 16));
            else
              reinterpret_cast<uint32_t*>(out)[v + e] = x[k][e];
          }
      }
    }
  }
  if (!names) return;

  // The tokens that the lists name
  const float repetition = a.repetition.each ? a.repetition.each[row] : a.repetition.all;
  const float presence = a.presence.each ? a.presence.each[row] : a.presence.all;
  const float frequency = a.frequency.each ? a.frequency.each[row] : a.frequency.all;
  const float* const bias = a.bias + row * a.bias_tokens.ld;
  __syncthreads();  // (the counts are done, and the block's copies in place)
  each([&](uint32_t x) {
    const uint32_t of_token = atomicExch(named + place(x), 0u);
    if (!of_token) return;
    const int v = first + static_cast<int>(place(x));
    if (mask && !(mask[v >> 5] >> (v & 31) & 1)) return;
    if constexpr (kBf16) {
      const float y = bf16_to_f32(reinterpret_cast<const __nv_bfloat16*>(in)[v]);
      reinterpret_cast<__nv_bfloat16*>(out)[v] = f32_to_bf16(adjusted(y, of_token, repetition, presence, frequency, bias));
    } else {
      reinterpret_cast<float*>(out)[v] = adjusted(reinterpret_cast<const float*>(in)[v], of_token, repetition, presence, frequency, bias);
    }
  });
}

template <bool kBf16, int kThreads, int kPer>
cudaError_t launch(const Adjust& a, cudaStream_t stream) {
  constexpr int kTokens = kThreads * kPer * 8;
  const int chunks = (a.vocab + 7 + kTokens - 1) / kTokens;  // (a row may begin inside its first group)
  const bool names = a.prompt.n > 0 || a.history.n > 0 || a.bias_tokens.n > 0;
  const int bytes = names ? kTokens * 4 : 0;
  static SharedMemory allowed;
  if (const cudaError_t e = allowed.at_least(reinterpret_cast<const void*>(adjust_kernel<kBf16, kThreads, kPer>), bytes, kTokens * 4); e != cudaSuccess) return e;
  adjust_kernel<kBf16, kThreads, kPer><<<static_cast<unsigned>(a.rows) * chunks, kThreads, bytes, stream>>>(a, chunks);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adjust(const Adjust& a, cudaStream_t stream) {
  // 16 KB of a row to a block, so that few blocks read a row's lists (32 KB: 39 us where 16 KB take 34); 4 KB (fp32: 8) where that would leave SMs without one
  const int size = a.bf16 ? 2 : 4;
  const bool few = static_cast<long long>(a.rows) * ((a.vocab * size + 16383) / 16384) < 148;
  if (a.bf16) return few ? launch<true, 256, 1>(a, stream) : launch<true, 256, 4>(a, stream);
  return few ? launch<false, 256, 1>(a, stream) : launch<false, 256, 2>(a, stream);
}

}  // namespace logits

}  // namespace mnb
