// Append of new K/V rows quantised to 8 bits: e4m3 payload, one power-of-two scale per row.
//
//   e = the least exponent in [-14, 7] with max|x| <= 448 * 2^e,  payload = e4m3(x * 2^-e)
//
// With a power of two as the scale, x * 2^-e is exact in float32 and the only rounding is
// the one to e4m3, so the payload does not depend on how the division is done; e4m3 is a
// floating type, so a finer scale would not add precision.
//
// A lane holds 8 elements, head_dim / 8 lanes a row; the row's maximum goes around them in
// log2(head_dim / 8) shuffles.  HBM-bound: head_dim * sizeof(T) bytes read and head_dim + 1
// written per row, each once.
#include <cuda_fp8.h>

#include "kv8.h"
#include "pa_common.cuh"

namespace pa {

constexpr int kAppendThreads = 256;

// Scale byte of a row whose largest magnitude is `big` (not NaN): 448 = 1.75 * 2^8, so a
// mantissa above 1.75 needs one exponent more.
__device__ __forceinline__ int kv8_scale_byte(float big) {
  const uint32_t b = __float_as_uint(big);
  const int e = int(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return 127 + max(-14, min(7, e));
}

template <typename T>
__device__ __forceinline__ void load8(const T* src, bool vec, float (&x)[8]) {
  if (vec) {
    VecLoad<T, 4>::run(src, x);
    VecLoad<T, 4>::run(src + 4, x + 4);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(src[i]);
  }
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* src, bool vec, float (&x)[8]) {
  uint4 w;
  if (vec) {
    w = *reinterpret_cast<const uint4*>(src);
  } else {
    __half* h = reinterpret_cast<__half*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = src[i];
  }
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(u[i], (__half*)nullptr);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* src, bool vec, float (&x)[8]) {
  uint4 w;
  if (vec) {
    w = *reinterpret_cast<const uint4*>(src);
  } else {
    __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = src[i];
  }
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(u[i], (__nv_bfloat16*)nullptr);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendParams p) {
  constexpr int LANES = D / 8;  // lanes a row
  const int64_t unit = (int64_t(blockIdx.x) * kAppendThreads + threadIdx.x) / LANES;
  const int64_t rows = int64_t(p.num_tokens) * p.num_kv_heads;
  const bool there = unit < rows;
  const int64_t row = there ? unit : rows - 1;  // a spare lane repeats the last row and stores nothing
  const int t = int(row / p.num_kv_heads), h = int(row - int64_t(t) * p.num_kv_heads);
  const int d = (threadIdx.x % LANES) * 8;
  const bool is_v = blockIdx.y == 1;
  const T* src = is_v ? static_cast<const T*>(p.value) + t * p.v_st + h * p.v_sh + d
                      : static_cast<const T*>(p.key) + t * p.k_st + h * p.k_sh + d;
  const int32_t slot = p.slots[t];
  float x[8];
  load8<T>(src, p.vec16, x);
  float big = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    nan |= x[i] != x[i];
    big = fmaxf(big, fabsf(x[i]));
  }
  big = nan ? INFINITY : big;
  // NaN travels as a flag beside the maximum, which fmaxf would drop.
  int broken = nan;
#pragma unroll
  for (int s = 1; s < LANES; s <<= 1) {
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
    broken |= __shfl_xor_sync(0xffffffffu, broken, s);
  }
  const int byte = broken ? 255 : kv8_scale_byte(big);
  const float inv = broken ? 0.f : __uint_as_float(uint32_t(254 - byte) << 23);  // 2^(127 - byte)
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 lo = make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), hi = make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv);
    if (broken) lo = hi = make_float2(0.f, 0.f);
    w[i] = uint32_t(__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3)) |
           (uint32_t(__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3)) << 16);
  }
  if (!there || slot < 0 || int64_t(slot) >= p.num_slots) return;  // padding tokens carry -1
  uint8_t* pool = is_v ? p.v_pool : p.k_pool;
  *reinterpret_cast<uint2*>(pool + (int64_t(slot) * p.num_kv_heads + h) * D + d) = make_uint2(w[0], w[1]);
  if (d == 0) {
    const int block = slot / p.block_size, at = slot - block * p.block_size;
    (is_v ? p.v_scale : p.k_scale)[(int64_t(block) * p.num_kv_heads + h) * p.block_size + at] = uint8_t(byte);
  }
}

template <typename T>
static cudaError_t append_dim(const Kv8AppendParams& p, cudaStream_t stream) {
  const int64_t lanes = int64_t(p.num_tokens) * p.num_kv_heads * (p.head_dim / 8);
  const dim3 grid(unsigned((lanes + kAppendThreads - 1) / kAppendThreads), 2);
  if (p.head_dim == 64)
    kv8_append_kernel<T, 64><<<grid, kAppendThreads, 0, stream>>>(p);
  else
    kv8_append_kernel<T, 128><<<grid, kAppendThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv8_append(int dtype, const Kv8AppendParams& p, cudaStream_t stream) {
  switch (dtype) {
    case PA_DTYPE_F32: return append_dim<float>(p, stream);
    case PA_DTYPE_F16: return append_dim<__half>(p, stream);
    case PA_DTYPE_BF16: return append_dim<__nv_bfloat16>(p, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace pa
