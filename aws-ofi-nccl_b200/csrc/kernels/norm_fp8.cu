// RMSNorm with the residual's addition whose output leaves in 8 bits, with the scales that the fp8 product (one for a row) or the expert
// exchange (one for 128 columns) takes: what rmsnorm and quantize_rows_fp8 make of a row in two passes, without its bf16 values in memory between them.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"

namespace b200 {

constexpr int NORM8_THREADS = 256;
constexpr int NORM8_GROUP = 128;          // columns with a scale of their own, 16 lanes of eight
constexpr int NORM8_MAX_H = NORM8_THREADS * 8 * 8;

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(p[j]), f[2 * j + 1] = __high2float(p[j]);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
         (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
}

// With y = h * r * w the largest |y| of a row is r times the largest |h * w|: it is found together with the sum of squares, in one exchange between the
// row's threads, and a value's code needs h * w alone. The maximum is taken over the numbers' bits, where a NaN is above all others: a row that holds one
// has it as its scale. TPR threads hold a row, VPT 16-byte vectors each, all of whose loads are under way at once.
template <int TPR, int VPT, bool GROUPS>
__global__ void __launch_bounds__(NORM8_THREADS)
    rmsnorm_fp8_kernel(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* res, int64_t ldres, __nv_bfloat16* h_out, const __nv_bfloat16* w,
                       uint8_t* q, float* scale, int64_t T, int H, float eps) {
  __shared__ float sums[NORM8_THREADS / 32];
  __shared__ uint32_t tops[NORM8_THREADS / 32];
  const int lane = threadIdx.x % TPR, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (NORM8_THREADS / TPR) + threadIdx.x / TPR;
  const bool live = row < T;
  grid_wait();
  grid_release();
  uint4 xv[VPT], rv[VPT], wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    xv[i] = rv[i] = wv[i] = make_uint4(0, 0, 0, 0);
    if (live && c * 8 < H) {
      xv[i] = reinterpret_cast<const uint4*>(x + row * ldx)[c];
      if (res) rv[i] = reinterpret_cast<const uint4*>(res + row * ldres)[c];
      wv[i] = reinterpret_cast<const uint4*>(w)[c];
    }
  }
  float ss = 0.f;
  uint32_t top = 0, group_top[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    float f[8], r[8];
    unpack8(xv[i], f);
    if (res) {
      unpack8(rv[i], r);
      __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&xv[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(f[2 * j] + r[2 * j], f[2 * j + 1] + r[2 * j + 1]);
      if (live && c * 8 < H) reinterpret_cast<uint4*>(h_out + row * H)[c] = xv[i];
      unpack8(xv[i], f);   // what is stored is normalised
    }
    unpack8(wv[i], r);
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(f[j], f[j], ss);
      most = max(most, __float_as_uint(f[j] * r[j]) & 0x7fffffffu);
    }
    if constexpr (GROUPS) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      group_top[i] = most;
    } else {
      top = max(top, most);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if constexpr (!GROUPS) top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    if ((threadIdx.x & 31) == 0) {
      sums[warp] = ss;
      tops[warp] = top;
    }
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      ss += sums[(warp & ~(W - 1)) + i];
      if constexpr (!GROUPS) top = max(top, tops[(warp & ~(W - 1)) + i]);
    }
  }
  if (!live) return;
  const float r = rsqrtf(ss / H + eps);
  // a row of zeros has the scale that quantize_rows_fp8 gives it
  auto scale_of = [&](uint32_t bits) {
    const float most = r * __uint_as_float(bits);
    return (most < 1e-12f ? 1e-12f : most) * (1.f / 448.f);
  };
  float s = 0.f, factor = 0.f;
  if constexpr (!GROUPS) {
    s = scale_of(top);
    factor = r * (1.f / s);
    if (lane == 0) scale[row] = s;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    if (c * 8 >= H) continue;
    if constexpr (GROUPS) {
      s = scale_of(group_top[i]);
      factor = r * (1.f / s);
      if (c % (NORM8_GROUP / 8) == 0) scale[row * (H / NORM8_GROUP) + c / (NORM8_GROUP / 8)] = s;
    }
    float f[8], g[8];
    unpack8(xv[i], f);
    unpack8(wv[i], g);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f[j] * g[j] * factor;
    reinterpret_cast<uint2*>(q + row * H)[c] = make_uint2(e4m3x4(f[0], f[1], f[2], f[3]), e4m3x4(f[4], f[5], f[6], f[7]));
  }
}

}  // namespace b200

extern "C" {
using namespace b200;

// x, res: rows of H bf16, ldx and ldres elements apart (multiples of 8); h_out [T][H] where there is a residual; q [T][H]; scale [T], or [T][H / 128] with
// group = 128.
int b200_rmsnorm_fp8(const void* x, long long ldx, const void* res, long long ldres, void* h_out, const void* w, void* q, float* scale, long long T,
                     int H, float eps, int group, void* stream) {
  ensure_context();
  if (T < 0 || H <= 0 || H % 8 || H > NORM8_MAX_H || (group != 0 && group != NORM8_GROUP) || (group && H % NORM8_GROUP)) return B200_ERR_BAD_ARG;
  if (!T) return 0;
  if (!x || !w || !q || !scale || (res && !h_out) || ldx % 8 || (res && ldres % 8)) return B200_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(res ? h_out : nullptr) | reinterpret_cast<uintptr_t>(w)) % 16 ||
      reinterpret_cast<uintptr_t>(q) % 8)
    return B200_ERR_BAD_ARG;
  if (T > 0x7fffffffll) return B200_ERR_TOO_LARGE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto X = static_cast<const __nv_bfloat16*>(x);
  auto R = static_cast<const __nv_bfloat16*>(res);
  auto HO = static_cast<__nv_bfloat16*>(h_out);
  auto W = static_cast<const __nv_bfloat16*>(w);
  auto Q = static_cast<uint8_t*>(q);
#define B200_NORM8(TPR, VPT)                                                                                                                   \
  launch_dependent(group ? rmsnorm_fp8_kernel<TPR, VPT, true> : rmsnorm_fp8_kernel<TPR, VPT, false>,                                          \
                   static_cast<int>((T + NORM8_THREADS / TPR - 1) / (NORM8_THREADS / TPR)), NORM8_THREADS, 0, st, X, static_cast<int64_t>(ldx), \
                   R, static_cast<int64_t>(ldres), HO, W, Q, scale, static_cast<int64_t>(T), H, eps)
  if (H <= 256) B200_NORM8(32, 1);
  else if (H <= 512) B200_NORM8(32, 2);
  else if (H <= 1024) B200_NORM8(64, 2);
  else if (H <= 2048) B200_NORM8(128, 2);
  else if (H <= 4096) B200_NORM8(256, 2);
  else if (H <= 8192) B200_NORM8(256, 4);
  else B200_NORM8(256, 8);
#undef B200_NORM8
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // extern "C"
