// Activations as they are kept in 8 bits: groups of 32 elements of a row (its last group may be shorter) have e4m3 codes and a common power of two, the least
// with which the largest of them is no more than 448, as a byte e of 2^(e - 127). A power of two scales without rounding: what is lost is the rounding
// to e4m3 alone, the same in any arithmetic. Values that are not finite become NaN and count for no power.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace b200 {

constexpr int KEPT_GROUP = 32;   // elements, four lanes of eight

// Two magnitudes of bf16 each; those that are not finite are above all others.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight bf16 of a lane -> their codes and, in all four lanes of the group, the byte of its power. A whole warp calls it.
__device__ __forceinline__ uint2 keep8(const uint4& v, uint32_t& power) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t most = max_u16x2(max_u16x2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), max_u16x2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
  most = max(most >> 16, most & 0xFFFFu);
  if (most >= 0x7F80u) {   // rare: such values become NaN, and the largest of the others is looked for
    most = 0;
#pragma unroll 1
    for (int k = 0; k < 8; ++k) {
      const int at = k >> 1, shift = (k & 1) * 16;
      const uint32_t word = at == 0 ? w[0] : at == 1 ? w[1] : at == 2 ? w[2] : w[3], m = word >> shift & 0x7FFFu;
      if (m < 0x7F80u) {
        most = max(most, m);
        continue;
      }
      const uint32_t nan = 0x7FFFu << shift;
      w[0] |= at == 0 ? nan : 0, w[1] |= at == 1 ? nan : 0, w[2] |= at == 2 ? nan : 0, w[3] |= at == 3 ? nan : 0;
    }
  }
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
  most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
  // 448 is 1.75 * 2^8: the exponent of the largest less 8, or 7 where its fraction is above 0.75
  power = static_cast<uint32_t>(max(static_cast<int>(most >> 7) - ((most & 0x7Fu) > 0x60u ? 7 : 8), 0));
  const float scale = __uint_as_float((254u - power) << 23);   // 2^(127 - power)
  uint32_t codes[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = __uint_as_float(e & 1 ? w[2 * k + e / 2] & 0xFFFF0000u : w[2 * k + e / 2] << 16) * scale;
    codes[k] = static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3)) |
               (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3)) << 16);
  }
  return make_uint2(codes[0], codes[1]);
}

// What eight codes stand for
__device__ __forceinline__ void kept8(const uint2& codes, uint32_t power, float (&f)[8]) {
  const float scale = __uint_as_float(power ? power << 23 : 0x00400000u);   // 2^(power - 127)
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_fp8x2_storage_t pair = static_cast<__nv_fp8x2_storage_t>((k < 2 ? codes.x : codes.y) >> (16 * (k & 1)));
    const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(pair, __NV_E4M3);
    const float2 two = __half22float2(*reinterpret_cast<const __half2*>(&raw));
    f[2 * k] = two.x * scale, f[2 * k + 1] = two.y * scale;
  }
}

}  // namespace b200
