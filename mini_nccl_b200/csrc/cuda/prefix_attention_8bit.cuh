// What the attention's kernels over a cache in 8 bits share: codes as f16, the
// scales' way to shared memory, and the pools' tensor maps.
#pragma once

#include <algorithm>

#include "prefix_attention.cuh"

namespace mnb {

namespace prefix {

namespace q8 {

constexpr float kLeastScale = 8.673617379884035e-19f;  // 2^-60

MNB_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
MNB_DEVICE uint32_t sub_f16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
MNB_DEVICE uint32_t f16_of_e4m3(uint16_t x) {
  uint32_t y;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(y) : "h"(x));
  return y;
}
// Four codes as f16: of bytes 0 and 2 (lo), and 1 and 3 (hi).
template <bool kFloat>
MNB_DEVICE void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kFloat) {
    w = __byte_perm(w, 0, 0x3120);
    lo = f16_of_e4m3(static_cast<uint16_t>(w)), hi = f16_of_e4m3(static_cast<uint16_t>(w >> 16));
  } else {
    w ^= 0x80808080u;
    lo = sub_f16x2(__byte_perm(w, 0x64646464u, 0x4240), 0x64806480u);
    hi = sub_f16x2(__byte_perm(w, 0x64646464u, 0x4341), 0x64806480u);
  }
}
// The same as whichever pairs are cheapest: bytes (0, 1), (2, 3) of e4m3, (0, 2), (1, 3) of int8.
template <bool kFloat>
MNB_DEVICE void widen_any(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (kFloat)
    lo = f16_of_e4m3(static_cast<uint16_t>(w)), hi = f16_of_e4m3(static_cast<uint16_t>(w >> 16));
  else
    widen<false>(w, lo, hi);
}
MNB_DEVICE uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
MNB_DEVICE uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
  return y;
}
MNB_DEVICE void copy_float(uint32_t dst, const float* src, bool there) {  // zero where not
  const int n = there ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
MNB_DEVICE void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// A pool of codes as (head_dim, heads, tokens, pages) in boxes of up to `tokens` of one page and head.
inline bool codes_map(CUtensorMap* map, const uint8_t* base, const Args& a, int head_dim, int tokens) {
  if (!encode_fn()) return false;
  const int page = 1 << a.page_shift;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(page), static_cast<cuuint64_t>(std::max(1, a.pages))};
  // an axis of one entry may have any stride: give the map one that it accepts
  auto stride = [](long long n, long long ld) { return static_cast<cuuint64_t>(n > 1 ? ld : 16); };
  const cuuint64_t strides[3] = {stride(a.kv_heads, a.head_ld), stride(page, a.token_ld), stride(a.pages, a.page_ld)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(head_dim), 1, static_cast<cuuint32_t>(std::min(page, tokens)), 1};
  const cuuint32_t each[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle swizzle = head_dim == 32 ? CU_TENSOR_MAP_SWIZZLE_32B
                                     : head_dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, each,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace q8

}  // namespace prefix

}  // namespace mnb
