// Quotients and roots of pair_math.cuh against IEEE's, over every float of the ranges that their comments name.
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "pair_math.cuh"

using namespace b200;

struct Result {
  unsigned long long inverses, roots, any, seen;   // those that differ, and the numbers looked at
  unsigned int worst[3];                           // largest relative error of roots from 2^-115, 2^-119 and 2^-126 on, as a float's bits
};

__global__ void all_floats(Result* out) {
  unsigned long long inverses = 0, roots = 0, any = 0, seen = 0;
  float worst[3] = {};
  const uint32_t stride = gridDim.x * blockDim.x;
  // every number from 0 to infinity, and NaNs behind it
  for (uint64_t bits = blockIdx.x * blockDim.x + threadIdx.x; bits <= 0x7f800010u; bits += stride) {
    const float v = __uint_as_float(static_cast<uint32_t>(bits));
    ++seen;
    if (v > 0x1p-110f && v < 0x1p120f) inverses += inverse(v) != __frcp_rn(v);
    const Pair m(-v, -v), plain = minus_roots(m);
    float a, b, x, y;
    plain.to(a, b);
    any_minus_roots(m, plain).to(x, y);
    const float want = __fsqrt_rn(v);
    any += v != v ? (x == x || y == y) : (x != -want || y != -want);
    if (v >= 0x1p-100f && v < INFINITY) roots += a != -want || b != -want;
    const float off = fabsf(a + want) / want;
    if (v >= 0x1p-126f && v < 0x1p-100f) {
      worst[2] = fmaxf(worst[2], off);
      if (v >= 0x1p-119f) worst[1] = fmaxf(worst[1], off);
      if (v >= 0x1p-115f) worst[0] = fmaxf(worst[0], off);
    }
  }
  atomicAdd(&out->inverses, inverses);
  atomicAdd(&out->roots, roots);
  atomicAdd(&out->any, any);
  atomicAdd(&out->seen, seen);
  for (int i = 0; i < 3; ++i) atomicMax(&out->worst[i], __float_as_uint(worst[i]));
}

int main() {
  Result* d = nullptr;
  Result r{};
  if (cudaMalloc(&d, sizeof(Result)) != cudaSuccess || cudaMemset(d, 0, sizeof(Result)) != cudaSuccess) return 2;
  all_floats<<<1184, 256>>>(d);
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(&r, d, sizeof(Result), cudaMemcpyDeviceToHost) != cudaSuccess) return 2;
  cudaFree(d);
  float worst[3];
  for (int i = 0; i < 3; ++i) __builtin_memcpy(&worst[i], &r.worst[i], 4);
  printf("of %llu numbers differ: inverses %llu, roots %llu, any roots %llu; largest relative errors below 2^-100: %g, %g, %g\n", r.seen, r.inverses, r.roots,
         r.any, worst[0], worst[1], worst[2]);
  // below 2^-100: with d = 2^-127 / v the unit's reciprocal root is off by d at most, what a Newton step leaves of it is 3/2 d^2, and a rounding
  const bool ok = r.seen == 0x7f800011ull && r.inverses == 0 && r.roots == 0 && r.any == 0 && worst[0] <= 0x1.8p-24f + 0x1p-23f &&
                  worst[1] <= 0x1.8p-16f + 0x1p-23f && worst[2] <= 0.125f;
  return ok ? 0 : 1;
}
