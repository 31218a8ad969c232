// Append of new K/V rows quantised to 8 bits: e4m3 payload, one power-of-two scale per row.
//
//   e = the least exponent in [-14, 7] with max|x| <= 448 * 2^e,  payload = e4m3(x * 2^-e)
//
// With a power of two as the scale, x * 2^-e is exact in float32 and the only rounding is
// the one to e4m3, so the payload does not depend on how the division is done; e4m3 is a
// floating type, so a finer scale would not add precision.
//
// A lane holds 16 elements (head_dim / 16 lanes a row), so that the arithmetic around the
// loads (places, strides, shuffles) is paid once per 16: with 8 elements a lane the kernel
// was bound by instruction issue, 36 us for 16,384 tokens of 8 heads of 128 in bf16 where
// HBM needs 15.  The row's maximum is taken on packed pairs with the NaN-keeping maximum and
// goes around the lanes in log2(head_dim / 16) shuffles.  HBM-bound: head_dim * sizeof(T)
// bytes read and head_dim + 1 written per row, each once: those 16,384 tokens take 20.5 us
// (4.9 TB/s, 75 % of a plain copy's rate), 32 or 1,000 tokens 4.1, the launch and one latency.
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

// 16 elements of a lane: the loads, the largest magnitude (NaN if there is one) and the
// elements times a power of two as e4m3.
template <typename T> struct Lane16;

template <typename T, typename T2> struct Lane16Half {
  uint4 w[2];
  __device__ __forceinline__ void load(const T* src, bool vec) {
    if (vec) {
      w[0] = reinterpret_cast<const uint4*>(src)[0];
      w[1] = reinterpret_cast<const uint4*>(src)[1];
    } else {
      T* h = reinterpret_cast<T*>(w);
#pragma unroll
      for (int i = 0; i < 16; ++i) h[i] = src[i];
    }
  }
  __device__ __forceinline__ float biggest() const {
    const T2* h = reinterpret_cast<const T2*>(w);
    T2 m = __habs2(h[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, __habs2(h[i]));
    return to_float(__hmax_nan(m.x, m.y));
  }
  __device__ __forceinline__ uint4 quantise(float inv) const {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(u[2 * i], (T*)nullptr), b = unpack2(u[2 * i + 1], (T*)nullptr);
      r[i] = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(a.x * inv, a.y * inv), __NV_SATFINITE, __NV_E4M3)) |
             (uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(b.x * inv, b.y * inv), __NV_SATFINITE, __NV_E4M3)) << 16);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};
template <> struct Lane16<__half> : Lane16Half<__half, __half2> {};
template <> struct Lane16<__nv_bfloat16> : Lane16Half<__nv_bfloat16, __nv_bfloat162> {};
template <> struct Lane16<float> {
  float x[16];
  __device__ __forceinline__ void load(const float* src, bool vec) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      if (vec) {
        VecLoad<float, 4>::run(src + i, x + i);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i + j] = src[i + j];
      }
    }
  }
  __device__ __forceinline__ float biggest() const {
    float m = 0.f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      nan |= x[i] != x[i];
      m = fmaxf(m, fabsf(x[i]));
    }
    return nan ? NAN : m;
  }
  __device__ __forceinline__ uint4 quantise(float inv) const {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE,
                                               __NV_E4M3)) |
             (uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE,
                                                __NV_E4M3))
              << 16);
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const Kv8AppendParams p) {
  constexpr int LANES = D / 16;  // lanes a row
  const uint32_t unit = blockIdx.x * (kAppendThreads / LANES) + threadIdx.x / LANES;
  const uint32_t rows = uint32_t(p.num_tokens) * uint32_t(p.num_kv_heads);  // below 2^31: the host checks
  const bool there = unit < rows;
  const uint32_t row = there ? unit : rows - 1;  // a spare lane repeats the last row and stores nothing
  const uint32_t t = row / uint32_t(p.num_kv_heads), h = row - t * uint32_t(p.num_kv_heads);
  const int d = int(threadIdx.x % LANES) * 16;
  const bool is_v = blockIdx.y == 1;
  const T* src = is_v ? static_cast<const T*>(p.value) + t * p.v_st + h * p.v_sh + d
                      : static_cast<const T*>(p.key) + t * p.k_st + h * p.k_sh + d;
  Lane16<T> x;
  x.load(src, p.vec16);
  const int32_t slot = p.slots[t];
  float big = x.biggest();
  // NaN is the largest bit pattern of a non-negative float, so the maximum of the bits keeps it.
  uint32_t bits = __float_as_uint(big) & 0x7fffffffu;
#pragma unroll
  for (int s = 1; s < LANES; s <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, s));
  const bool broken = bits > 0x7f800000u;
  const int byte = broken ? 255 : kv8_scale_byte(__uint_as_float(bits));
  uint4 w = x.quantise(__uint_as_float(uint32_t(254 - byte) << 23));  // 2^(127 - byte)
  if (broken) w = make_uint4(0, 0, 0, 0);
  if (!there || slot < 0 || int64_t(slot) >= p.num_slots) return;  // padding tokens carry -1
  uint8_t* pool = is_v ? p.v_pool : p.k_pool;
  *reinterpret_cast<uint4*>(pool + (int64_t(slot) * p.num_kv_heads + h) * D + d) = w;
  if (d == 0) {
    const uint32_t block = uint32_t(slot) / uint32_t(p.block_size), at = uint32_t(slot) - block * uint32_t(p.block_size);
    (is_v ? p.v_scale : p.k_scale)[(int64_t(block) * p.num_kv_heads + h) * p.block_size + at] = uint8_t(byte);
  }
}

template <typename T>
static cudaError_t append_dim(const Kv8AppendParams& p, cudaStream_t stream) {
  const int64_t lanes = int64_t(p.num_tokens) * p.num_kv_heads * (p.head_dim / 16);
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
