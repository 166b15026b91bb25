// RMSNorm with the residual's addition whose output leaves in 8 bits, with the scales that the fp8 product (one for a row) or the expert
// exchange (one for 128 columns) takes: what rmsnorm and quantize_rows_fp8 make of a row in two passes, without its bf16 values in memory between them.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"
#include "pair_math.cuh"

namespace b200 {

constexpr int NORM8_GROUP = 128;          // columns with a scale of their own, 16 lanes of eight
constexpr int NORM8_MAX_H = 16384;

__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(p[j]), f[2 * j + 1] = __high2float(p[j]);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
         (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  (both(a) * both(b)).to(r.x, r.y);
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  fma2(both(a), both(b), both(c)).to(r.x, r.y);
  return r;
}

// With y = h * r * w the largest |y| of a row is r times the largest |h * w|: it is found together with the sum of squares, in one exchange between the
// row's threads, and a value's code needs h * w alone, which stays in registers. Maxima are of the numbers' bits, where a NaN is above all others: a row
// that holds one has it as its scale. A sum of squares beyond 32 bits makes r zero: finite values become zeros, an infinity a NaN of its scale.
// Products of two bf16 lie on a tie of e4m3 exactly in 6 of 10000 elements of normal inputs; there the roundings of r and the scale decide between the two codes.
//
// TPR threads hold a row, VPT 16-byte vectors each, all of whose loads are under way at once; memory bounds it, with what a short kernel takes to come
// up and run out. 4096 x 4096 with a residual 20.0 us (5.9 TB/s; 22.0 in CTAs of 256 threads that pack and unpack more), without 10.2; 5003 x 7168 in
// groups 23.1 (4.7 TB/s; 34.8 in such CTAs). CTAs that stay, with the next row's loads ahead, took 20.4, 10.9 and 22.4 beside 20.0, 10.2 and 22.6: they
// gain where rows are narrow (60000 x 256 12.7 -> 11.2) and lose with a residual (9000 x 5120 50.9 -> 51.9).
template <int TPR, int VPT, int THREADS, bool GROUPS, bool RES>
__global__ void __launch_bounds__(THREADS)
    rmsnorm_fp8_kernel(const __nv_bfloat16* x, int64_t ldx, const __nv_bfloat16* res, int64_t ldres, __nv_bfloat16* h_out, const __nv_bfloat16* w,
                       uint8_t* q, float* scale, int64_t T, int H, float eps) {
  __shared__ float sums[THREADS / 32];
  __shared__ uint32_t tops[THREADS / 32];
  const int lane = threadIdx.x % TPR, warp = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (THREADS / TPR) + threadIdx.x / TPR;
  const bool live = row < T;
  grid_wait();
  grid_release();
  uint4 xv[VPT], rv[RES ? VPT : 1], wv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    xv[i] = wv[i] = make_uint4(0, 0, 0, 0);
    if constexpr (RES) rv[i] = make_uint4(0, 0, 0, 0);
    if (live && c * 8 < H) {
      xv[i] = reinterpret_cast<const uint4*>(x + row * ldx)[c];
      if constexpr (RES) rv[i] = reinterpret_cast<const uint4*>(res + row * ldres)[c];
      wv[i] = reinterpret_cast<const uint4*>(w)[c];
    }
  }
  float2 ss2 = make_float2(0.f, 0.f), y[VPT][4];   // y: h * w
  float top = 0.f;
  uint32_t group_top[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    float f[8], g[8];
    unpack8(xv[i], f);
    if constexpr (RES) {
      unpack8(rv[i], g);
      __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&xv[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(f[2 * j] + g[2 * j], f[2 * j + 1] + g[2 * j + 1]);
      if (live && c * 8 < H) reinterpret_cast<uint4*>(h_out + row * H)[c] = xv[i];
      unpack8(xv[i], f);   // what is stored is normalised
    }
    unpack8(wv[i], g);
    if constexpr (GROUPS) top = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 h = make_float2(f[2 * j], f[2 * j + 1]);
      ss2 = fma2(h, h, ss2);
      y[i][j] = mul2(h, make_float2(g[2 * j], g[2 * j + 1]));
      top = largest(top, y[i][j].x, y[i][j].y);
    }
    if constexpr (GROUPS) {
      uint32_t most = __float_as_uint(top);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      group_top[i] = most;
    }
  }
  float ss = ss2.x + ss2.y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  uint32_t most = 0;
  if constexpr (!GROUPS) most = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    if ((threadIdx.x & 31) == 0) {
      sums[warp] = ss;
      if constexpr (!GROUPS) tops[warp] = most;
    }
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      ss += sums[(warp & ~(W - 1)) + i];
      if constexpr (!GROUPS) most = max(most, tops[(warp & ~(W - 1)) + i]);
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
    s = scale_of(most);
    factor = r * (1.f / s);
    if (lane == 0) scale[row] = s;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = lane + i * TPR;
    if (c * 8 >= H) continue;
    if constexpr (GROUPS) {
      s = scale_of(group_top[i]);
      factor = r * __fdividef(1.f, s);   // within 2 ulp: a code moves where its share is that near to a tie, as by the products' own roundings
      if (c % (NORM8_GROUP / 8) == 0) scale[row * (H / NORM8_GROUP) + c / (NORM8_GROUP / 8)] = s;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) y[i][j] = mul2(y[i][j], make_float2(factor, factor));
    reinterpret_cast<uint2*>(q + row * H)[c] =
        make_uint2(e4m3x4(y[i][0].x, y[i][0].y, y[i][1].x, y[i][1].y), e4m3x4(y[i][2].x, y[i][2].y, y[i][3].x, y[i][3].y));
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
#define B200_NORM8(TPR, VPT, THREADS)                                                                                                          \
  launch_dependent(group ? (res ? rmsnorm_fp8_kernel<TPR, VPT, THREADS, true, true> : rmsnorm_fp8_kernel<TPR, VPT, THREADS, true, false>)       \
                         : (res ? rmsnorm_fp8_kernel<TPR, VPT, THREADS, false, true> : rmsnorm_fp8_kernel<TPR, VPT, THREADS, false, false>),    \
                   static_cast<int>((T + THREADS / TPR - 1) / (THREADS / TPR)), THREADS, 0, st, X, static_cast<int64_t>(ldx), R,                \
                   static_cast<int64_t>(ldres), HO, W, Q, scale, static_cast<int64_t>(T), H, eps)
  // The fewest vectors that hold a row in small CTAs, but for wide rows with a residual, whose registers leave no room for enough of those.
  if (H <= 256) B200_NORM8(32, 1, 256);
  else if (H <= 512) B200_NORM8(32, 2, 256);
  else if (H <= 768) B200_NORM8(32, 3, 128);
  else if (H <= 1024) B200_NORM8(32, 4, 128);
  else if (H <= 1536) B200_NORM8(64, 3, 128);
  else if (H <= 2048) B200_NORM8(64, 4, 128);
  else if (H <= 4096) B200_NORM8(128, 4, 128);
  else if (H <= 5120) B200_NORM8(128, 5, 128);
  else if (!res && H <= 6144) B200_NORM8(128, 6, 128);
  else if (!res && H <= 7168) B200_NORM8(128, 7, 128);
  else if (H <= 6144) B200_NORM8(256, 3, 256);
  else if (H <= 8192) B200_NORM8(256, 4, 256);
  else B200_NORM8(512, 4, 512);
#undef B200_NORM8
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // extern "C"
