// Codes and scales of the 8-bit key / value cache, shared by the kernels that write and read it.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace hippo {
constexpr int kMinExp = -100;      // exponent of a block of zeros; 2^(-kMinExp) and every 2^e in between is a normal fp32

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ bool isnan_bits(float x) { return (__float_as_uint(x) & 0x7fffffffu) > 0x7f800000u; }

// Smallest e >= kMinExp with amax <= largest code * 2^e, from the bits of amax = f * 2^x, 1 <= f < 2: 448 = 1.75 * 2^8 (mantissa
// field 0x600000), 127 = 1.984375 * 2^6 (0x7e0000).
template <int E4M3> __device__ __forceinline__ int scale_exponent(uint32_t amax) {
  const int x = (int)(amax >> 23) - 127;
  const uint32_t m = amax & 0x7fffffu;
  const int e = E4M3 ? x - 8 + (m > 0x600000u) : x - 6 + (m > 0x7e0000u);
  return e < kMinExp ? kMinExp : e;
}

template <int E4M3> __device__ __forceinline__ uint8_t encode1(float x) {                // |x| within the codes' range
  if (E4M3) return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  return (uint8_t)(int8_t)__float2int_rn(x);
}
// eight values at once: e4m3 two a conversion; int8 by adding 1.5 * 2^23, which leaves the nearest whole number in the low byte
template <int E4M3> __device__ __forceinline__ uint2 encode8(const float* f) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (E4M3) {
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    } else {
      h[i] = __byte_perm(__float_as_uint(f[2 * i] + 12582912.f), __float_as_uint(f[2 * i + 1] + 12582912.f), 0x0040);
    }
  }
  return make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410));
}
template <int E4M3> __device__ __forceinline__ float decode1(uint8_t c) {
  if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
  return (float)(int8_t)c;
}
}  // namespace hippo
