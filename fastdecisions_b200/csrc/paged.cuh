// Shared by the kernels that work on a paged KV cache or on pools of states: packed-segment lookup
// and the row codec of the 8-bit cache.
//
// Cache rows: k_cache / v_cache [pages][kv heads][page_size][head_dim], bf16 or e4m3; the 8-bit form
// has one scale byte b per row ([pages][kv heads][page_size]) and stands for e4m3(x) * 2^(b - 127).
// A power of two as the scale makes decoding exact in bf16 (and in fp32): the only rounding of the
// 8-bit cache is the one to e4m3 (at most 2^-4 relative for elements within 2^14 of the row's largest).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace fdk {
namespace paged {

// Largest s with cu[s] <= t for a whole warp (32-ary search: ceil(log32(nseg + 1)) dependent loads);
// -1 when t < cu[0].  `cu` is read on the device only, so it need not be well formed: the caller
// checks cu[s] <= t < cu[s + 1] before it uses s.
__device__ __forceinline__ int find_segment_warp(const int32_t* __restrict__ cu, int nseg, int t, int lane) {
  int lo = 0, n = nseg + 1;  // candidates lo .. lo + n - 1
  while (true) {
    const int step = (n + 31) >> 5;
    const int i = lo + lane * step;
    const bool le = lane * step < n && i <= nseg && cu[i] <= t;
    const unsigned b = __ballot_sync(0xffffffffu, le);
    const int c = (b == 0xffffffffu) ? 32 : __ffs(~b) - 1;  // leading run of true
    if (c == 0) return lo == 0 ? -1 : lo;
    lo += (c - 1) * step;
    if (step == 1) return lo;
    n = min(step, nseg + 1 - lo);
  }
}

// One segment's token range, checked: false (and nothing to do) when cu is not a valid range there.
__device__ __forceinline__ bool segment_range(const int32_t* __restrict__ cu, int s, int64_t tokens, int& begin,
                                              int& end) {
  begin = cu[s];
  end = cu[s + 1];
  return begin >= 0 && end >= begin && end <= tokens;
}

// Scale byte of a row whose largest magnitude is `amax`: the smallest e in [-127, 127] with
// amax <= 448 * 2^e, plus 127.  448 = 1.75 * 2^8, so e is amax's exponent - 8, one more when its
// significand exceeds 1.75.
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, 0), 254);
}
// 2^(127 - b) and 2^(b - 127) for a scale byte b (2^-127 is subnormal).
__device__ __forceinline__ float scale_inverse(int b) { return __uint_as_float((uint32_t)(254 - b) << 23); }
__device__ __forceinline__ float scale_value(int b) {
  return __uint_as_float(b == 0 ? 0x00400000u : (uint32_t)b << 23);
}

// two e4m3 bytes -> two fp16 (exact)
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(v));
  return r;
}
// (lo, hi) -> two e4m3 bytes, lo in the low byte; round to nearest even, saturating
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace paged
}  // namespace fdk
