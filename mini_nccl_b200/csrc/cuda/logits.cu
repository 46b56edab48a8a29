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
// row's tokens, whose logits wait in registers while the tokens that the row names are
// counted in shared memory (whole numbers, so their order does not matter): one word for
// each token (its count, whether the prompt has it, and which bias it gets) and one bit,
// by which the pass over the logits passes over the many tokens that nobody named.
// Logits of tokens that the mask forbids are not read.
#include <algorithm>

#include "common.cuh"
#include "generation.h"

namespace mnb {

namespace logits {

namespace {

constexpr int kThreads = 256;
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

// Groups of 16 bytes (8 or 4 tokens) of a row, kPer for each thread, one chunk for each block.
template <bool kBf16, int kPer>
__global__ void __launch_bounds__(kThreads) adjust_kernel(const __grid_constant__ Adjust a, int chunks) {
  constexpr int kGroup = kBf16 ? 8 : 4, kSize = kBf16 ? 2 : 4, kTokens = kThreads * kPer * kGroup;
  __shared__ uint32_t named[kTokens];
  __shared__ uint32_t touched[kTokens / 32];
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  const char* const in = static_cast<const char*>(a.in) + row * a.in_ld * kSize;
  char* const out = static_cast<char*>(a.out) + row * a.out_ld * kSize;
  // The groups follow the output's alignment: the row's first token is number `skip` of the first group.
  const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(out) % 16) / kSize;
  const int first = chunk * kTokens - skip;  // the chunk's first token (below 0: before the row)
  const bool in_aligned = reinterpret_cast<uintptr_t>(in + first * kSize) % 16 == 0;

  int of = -1;  // the row's mask
  if (a.masks > 0) {
    of = a.mask_of ? a.mask_of[row] : a.masks > 1 ? row : 0;
    if (of >= a.masks) {
      if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
      of = -1;
    }
  }
  const uint32_t* const mask = of >= 0 ? a.allowed + of * a.mask_ld : nullptr;
  const int words = (a.vocab + 31) / 32;

  // token of the thread's group k, and which of its tokens exist and are allowed
  auto token_of = [&](int k) { return first + (k * kThreads + static_cast<int>(threadIdx.x)) * kGroup; };
  uint32_t allowed[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int v = token_of(k);
    uint32_t bits = (1u << kGroup) - 1;
    if (mask && v < a.vocab && v + kGroup > 0) {
      const int at = max(v, 0), w = at >> 5;
      const uint32_t lo = mask[w], hi = w + 1 < words && (at & 31) + kGroup > 32 ? mask[w + 1] : 0u;
      bits = (__funnelshift_r(lo, hi, at & 31) << (at - v)) & bits;
    }
    allowed[k] = bits;
  }
  uint4 x[kPer];
  auto load = [&](int k) {
    const int v = token_of(k);
    if (in_aligned && v >= 0 && v + kGroup <= a.vocab) {
      x[k] = ld_v4(in + static_cast<long long>(v) * kSize);
      return;
    }
    x[k] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < kGroup; ++e)
      if (v + e >= 0 && v + e < a.vocab) {
        if constexpr (kBf16)
          (&x[k].x)[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(in)[v + e]) << (e % 2 * 16);
        else
          (&x[k].x)[e] = reinterpret_cast<const uint32_t*>(in)[v + e];
      }
  };
  if (!a.in_place) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      x[k] = make_uint4(0, 0, 0, 0);
      if (allowed[k] && token_of(k) < a.vocab) load(k);
    }
  }

  float repetition = 1.f, presence = 0.f, frequency = 0.f;
  const bool names = a.prompt.n > 0 || a.history.n > 0 || a.bias_tokens.n > 0;
  if (names) {
    repetition = a.repetition.each ? a.repetition.each[row] : a.repetition.all;
    presence = a.presence.each ? a.presence.each[row] : a.presence.all;
    frequency = a.frequency.each ? a.frequency.each[row] : a.frequency.all;
    for (int i = threadIdx.x; i < kTokens / 4; i += kThreads) reinterpret_cast<uint4*>(named)[i] = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < kTokens / 32; i += kThreads) touched[i] = 0;
    int held = static_cast<int>(a.history.n);
    if (a.history_lens) {
      held = a.history_lens[row];
      if (held < 0 || held > a.history.n) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, kErrBadIndex);
        held = 0;
      }
    }
    __syncthreads();
    // f(place in the chunk, which one it is) for the tokens of a list
    auto each = [&](const Ids& t, int n, auto f) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const long long v = id_at(t, row * t.ld + i);
        if (v >= a.vocab && chunk == 0) atomicCAS(a.status, 0, kErrBadIndex);
        const long long at = v - first;
        if (v < 0 || v >= a.vocab || at < 0 || at >= kTokens) continue;
        f(static_cast<int>(at), i);
        atomicOr(touched + (at >> 5), 1u << (at & 31));
      }
    };
    if (a.bias_tokens.n > 0) {  // (the later one of a token that is named twice)
      each(a.bias_tokens, static_cast<int>(a.bias_tokens.n), [&](int at, int i) { atomicMax(named + at, static_cast<uint32_t>(i + 1) << kBiasShift); });
      __syncthreads();
    }
    each(a.prompt, static_cast<int>(a.prompt.n), [&](int at, int) { atomicOr(named + at, kPrompt); });
    each(a.history, held, [&](int at, int) { atomicAdd(named + at, 1u); });
    __syncthreads();
  }
  const float* const bias = a.bias + row * a.bias_tokens.ld;

#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int v = token_of(k), at = v - first;
    if (v >= a.vocab) continue;
    const uint32_t here = names ? touched[at >> 5] >> (at & 31) & ((1u << kGroup) - 1) & allowed[k] : 0u;
    const bool all = allowed[k] == (1u << kGroup) - 1;
    if (a.in_place) {
      if (all && !here) continue;
      if (allowed[k]) load(k);
    }
    if (here) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e)
        if (here >> e & 1) {
          uint32_t& w = (&x[k].x)[kBf16 ? e / 2 : e];
          if constexpr (kBf16) {
            const float y = adjusted(__uint_as_float(e % 2 ? w & 0xffff0000u : w << 16), named[at + e], repetition, presence, frequency, bias);
            const uint32_t b = __bfloat16_as_ushort(f32_to_bf16(y));
            w = e % 2 ? (w & 0xffffu) | b << 16 : (w & 0xffff0000u) | b;
          } else {
            w = __float_as_uint(adjusted(__uint_as_float(w), named[at + e], repetition, presence, frequency, bias));
          }
        }
    }
    if (!all) {
#pragma unroll
      for (int e = 0; e < kGroup; ++e)
        if (!(allowed[k] >> e & 1)) {
          uint32_t& w = (&x[k].x)[kBf16 ? e / 2 : e];
          if constexpr (kBf16)
            w = e % 2 ? (w & 0xffffu) | 0xff800000u : (w & 0xffff0000u) | 0xff80u;
          else
            w = 0xff800000u;
        }
    }
    if (v >= 0 && v + kGroup <= a.vocab) {
      st_v4(out + static_cast<long long>(v) * kSize, x[k]);
    } else {
#pragma unroll
      for (int e = 0; e < kGroup; ++e)
        if (v + e >= 0 && v + e < a.vocab) {
          if constexpr (kBf16)
            reinterpret_cast<uint16_t*>(out)[v + e] = static_cast<uint16_t>((&x[k].x)[e / 2] >> (e % 2 * 16));
          else
            reinterpret_cast<uint32_t*>(out)[v + e] = (&x[k].x)[e];
        }
    }
  }
}

template <bool kBf16, int kPer>
cudaError_t launch(const Adjust& a, cudaStream_t stream) {
  constexpr int kGroup = kBf16 ? 8 : 4, kTokens = kThreads * kPer * kGroup;
  const int chunks = (a.vocab + kGroup - 1 + kTokens - 1) / kTokens;  // (a row may begin inside its first group)
  adjust_kernel<kBf16, kPer><<<static_cast<unsigned>(a.rows) * chunks, kThreads, 0, stream>>>(a, chunks);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_adjust(const Adjust& a, cudaStream_t stream) {
  // 8192 tokens to a block, so that few blocks read a row's lists; 2048 where that would leave SMs without one
  const bool few = static_cast<long long>(a.rows) * ((a.vocab + 8191) / 8192) < 148;
  if (a.bf16) return few ? launch<true, 1>(a, stream) : launch<true, 4>(a, stream);
  return few ? launch<false, 2>(a, stream) : launch<false, 8>(a, stream);
}

}  // namespace logits

}  // namespace mnb
