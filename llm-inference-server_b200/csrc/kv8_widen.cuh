// Payload tiles in shared memory, e4m3 -> fp16 and queries -> fp16: shared by the KV8 attention
// kernels.
#pragma once

#include <stdint.h>

#include "pa_common.cuh"

namespace pa {

// Two e4m3 values (low or high half of a word) as two fp16 values, exactly.
__device__ __forceinline__ uint32_t widen_lo(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %1;\n cvt.rn.f16x2.e4m3x2 %0, h;\n}\n" : "=r"(r) : "r"(w));
  return r;
}

// Two fp16 products; no value of the cache loses a bit in one by its row's scale.
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Two scale bytes as fp16, 2^(b - 127); bytes outside the format's [113, 134] (NaN's 255, those
// behind a context) give its ends, so that a product with a finite payload is finite.
__device__ __forceinline__ uint32_t scale_pair(uint32_t two) {
  const uint32_t b = __vmaxu2(__vminu2(__byte_perm(two, 0u, 0x4140u), 0x00860086u), 0x00710071u);
  return (b - 0x00700070u) << 10;  // the exponent of fp16 is b - 112
}

// Byte offset of 16-byte chunk c of row r in a TMA tile whose rows are D bytes, with the
// swizzle as wide as the row (128 or 64 bytes).
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int c) {
  if constexpr (D == 128) return uint32_t(r * 128 + ((c ^ (r & 7)) << 4));
  return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// The power of two that brings a bf16 row with largest magnitude `big` to [2^14, 2^15), where
// fp16 holds it exactly but for elements 2^-28 below `big`; fp16 rows stay as they are.
template <typename T>
__device__ __forceinline__ float query_power(float big) {
  const uint32_t e = (__float_as_uint(big) >> 23) & 0xffu;
  if (DType<T>::code == PA_DTYPE_F16) return 1.f;
  if (e == 0 || e == 255) return 1.f;
  const int up = 14 - (int(e) - 127);
  return __uint_as_float(uint32_t(127 + max(-126, min(127, up))) << 23);
}

}  // namespace pa
