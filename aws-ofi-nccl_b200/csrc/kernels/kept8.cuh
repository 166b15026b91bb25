// Activations as they are kept in 8 bits: groups of 32 elements of a row (its last group may be shorter) have e4m3 codes and a common power of two, the least
// with which the largest of them is no more than 448, as a byte e of 2^(e - 127). A power of two scales without rounding: what is lost is the rounding
// to e4m3 alone, the same in any arithmetic. Values that are not finite become NaN and count for no power.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "pair_math.cuh"

namespace b200 {

constexpr int KEPT_GROUP = 32;   // elements, four lanes of eight

// Two magnitudes of bf16 each; those that are not finite are above all others.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) f[2 * k] = __uint_as_float(w[k] << 16), f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
}

// Eight bf16 of a lane (f: as floats, which it may change) -> their codes and, in all four lanes of the group, the byte of its power. A whole warp calls it.
__device__ __forceinline__ uint2 keep8(const uint4& v, float (&f)[8], uint32_t& power) {
  uint32_t most = max_u16x2(max_u16x2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), max_u16x2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
  most = max(most >> 16, most & 0xFFFFu);
  if (most >= 0x7F80u) {   // rare: such values become NaN, and the largest of the others is looked for
    most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t m = __float_as_uint(f[k]) >> 16 & 0x7FFFu;
      if (m < 0x7F80u)
        most = max(most, m);
      else
        f[k] = __uint_as_float(0x7FFFFFFFu);
    }
  }
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  // 448 is 1.75 * 2^8: the exponent of the largest less 8, or 7 where its fraction is above 0.75
  power = static_cast<uint32_t>(max(static_cast<int>((most + 0x1Fu) >> 7) - 8, 0));
  const Pair scale = both(__uint_as_float((254u - power) << 23));   // 2^(127 - power)
  uint32_t codes[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float a, b, c, d;
    (Pair(f[4 * k], f[4 * k + 1]) * scale).to(a, b);
    (Pair(f[4 * k + 2], f[4 * k + 3]) * scale).to(c, d);
    codes[k] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
               (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
  }
  return make_uint2(codes[0], codes[1]);
}

// What eight codes stand for
__device__ __forceinline__ void kept8(const uint2& codes, uint32_t power, float (&f)[8]) {
  const Pair scale = both(__uint_as_float(power ? power << 23 : 0x00400000u));   // 2^(power - 127)
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_fp8x2_storage_t pair = static_cast<__nv_fp8x2_storage_t>((k < 2 ? codes.x : codes.y) >> (16 * (k & 1)));
    const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(pair, __NV_E4M3);
    (both(__half22float2(*reinterpret_cast<const __half2*>(&raw))) * scale).to(f[2 * k], f[2 * k + 1]);
  }
}

}  // namespace b200
