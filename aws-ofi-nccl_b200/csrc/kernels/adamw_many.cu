// One AdamW step over many tensors of their own (the flat buffers' is in llm_ops.cu), bf16 or fp32, with moments in 32 bits or in 8.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// What bounds it is memory: 22 bytes for a bf16 parameter with moments in 32 bits, 10 in 8 bits, 28 and 16 with a master copy. The tensors' addresses travel
// as the kernel's parameter, so that nothing is copied to the device ahead of it and a captured step replays as it was.
//
// Moments in 8 bits: 256 consecutive elements of a tensor, a warp's, are a block with one scale each for m and for v, its largest magnitude over 448; an
// element is the e4m3 code of its share. v is held as its root, which halves the exponents that e4m3 has to span, and never as zero where it is
// none: m / sqrt(v) would be without bounds. Codes are not rounded to nearest: with b2 = 0.95 a root moves by 2.5 % a step at most
// when gradients vanish, half a step of e4m3 is 3 to 6 %, and a moment that moves by less than that would stay where it is for good.
// A value rounds up in that share of elements and steps that is its place between two codes, by a dither that is a function of the element's number and
// the step's, the additive recurrence of Roberts' R2 sequence (2018), whose points fill both directions evenly:
//   d = element * 0xC13FA9A9 + step * 0x91E10DA5 mod 2^32     up where fraction + (d >> 12) / 2^20 >= 1 for m, with ~d for the root
// Scaled by 2^-120 a float has its exponent and upper mantissa where e4m3 has them, denormals included, so the code is the top of a sum of integers.
//
// The update takes the moments of 32 bits, before they are rounded. Each operation on what is held is rounded by itself (no fused multiply-adds, a root
// and a quotient of IEEE's), so that codes do not depend on how the compiler contracts: a neighbouring code is 12 % away.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"

namespace b200 {

constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_BLOCK = 256;                                        // elements of a warp's pass, eight of a lane
constexpr int ADAMW_PASS = ADAMW_THREADS / 32 * ADAMW_BLOCK;            // of a CTA's
constexpr uint32_t DITHER_ELEMENT = 0xC13FA9A9u, DITHER_STEP = 0x91E10DA5u;

enum : uint32_t { ADAMW_P32 = 1, ADAMW_G32 = 2, ADAMW_VECTORS = 4 };

struct AdamwEntry {
  B200AdamwTensor t;
  uint32_t first;   // the tensor's first CTA
  uint32_t flags;
};
struct AdamwNumbers {
  float beta1, rest1, beta2, rest2, lr1, root2, eps, grad_scale;   // rest: 1 - beta; lr1 = lr / (1 - b1^t); root2 = 1 / sqrt(1 - b2^t)
  uint32_t dither;
  int zero_grad;
};
// A launch's parameters are 32764 bytes at most.
template <int N>
struct AdamwTable {
  AdamwEntry e[N];
  AdamwNumbers a;
  int count;
  int chunk;        // elements of a CTA, a multiple of ADAMW_PASS
};
constexpr int ADAMW_MOST = 400;
static_assert(sizeof(AdamwTable<ADAMW_MOST>) <= 32764, "parameters of a launch");

// Eight elements from i on, or as many as are left of n, zeros behind them.
__device__ __forceinline__ void load8(const __nv_bfloat16* p, int64_t i, int64_t n, bool vectors, float (&f)[8]) {
  if (vectors && i + 8 <= n) {
    const uint4 q = *reinterpret_cast<const uint4*>(p + i);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(h[j]), f[2 * j + 1] = __high2float(h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = i + j < n ? __bfloat162float(p[i + j]) : 0.f;
  }
}
__device__ __forceinline__ void load8(const float* p, int64_t i, int64_t n, bool vectors, float (&f)[8]) {
  if (vectors && i + 8 <= n) {
    const float4 a = reinterpret_cast<const float4*>(p + i)[0], b = reinterpret_cast<const float4*>(p + i)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = i + j < n ? p[i + j] : 0.f;
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, int64_t i, int64_t n, bool vectors, const float (&f)[8]) {
  if (vectors && i + 8 <= n) {
    uint4 q;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    *reinterpret_cast<uint4*>(p + i) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = __float2bfloat16_rn(f[j]);
  }
}
__device__ __forceinline__ void store8(float* p, int64_t i, int64_t n, bool vectors, const float (&f)[8]) {
  if (vectors && i + 8 <= n) {
    reinterpret_cast<float4*>(p + i)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p + i)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = f[j];
  }
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int64_t i, int64_t n, bool vectors) {
  if (vectors && i + 8 <= n) return *reinterpret_cast<const uint2*>(p + i);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (i + j < n) w[j / 4] |= static_cast<uint32_t>(p[i + j]) << (8 * (j % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t i, int64_t n, bool vectors, const uint32_t (&code)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) w[h] = code[4 * h] | code[4 * h + 1] << 8 | code[4 * h + 2] << 16 | code[4 * h + 3] << 24;
  if (vectors && i + 8 <= n) {
    *reinterpret_cast<uint2*>(p + i) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) p[i + j] = static_cast<uint8_t>(code[j]);
  }
}
__device__ __forceinline__ void decode8(uint2 q, float scale, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = j < 2 ? q.x : q.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * (j & 1))), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[2 * j] = __fmul_rn(v.x, scale);
    f[2 * j + 1] = __fmul_rn(v.y, scale);
  }
}

constexpr uint32_t E4M3_MOST = 0x7E, E4M3_NAN = 0x7F, INF_BITS = 0x7f800000u;

// Magnitudes' bits -> the scale of a warp's block and the codes. What is not finite is held as NaN and counts for no scale.
__device__ __forceinline__ float hold8(const float (&f)[8], const uint32_t (&dither)[8], uint32_t (&code)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(f[j]) & 0x7fffffffu);
  most = __reduce_max_sync(0xffffffffu, most);
  const bool finite = most < INF_BITS;   // the same in every lane
  if (!finite) {
    most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu;
      most = max(most, b < INF_BITS ? b : 0u);
    }
    most = __reduce_max_sync(0xffffffffu, most);
  }
  const float scale = __fmul_rn(fmaxf(__uint_as_float(most), 1e-30f), 1.f / 448.f);
  const float inv = __fdiv_rn(1.f, scale);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float share = __fmul_rn(__fmul_rn(fabsf(f[j]), inv), 0x1p-120f);
    code[j] = min((__float_as_uint(share) + dither[j]) >> 20, E4M3_MOST);
  }
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((__float_as_uint(f[j]) & 0x7fffffffu) >= INF_BITS) code[j] = E4M3_NAN;
  }
  return scale;
}

template <int BITS, typename P, typename G, bool MASTER>
__device__ __forceinline__ void adamw_chunk(const B200AdamwTensor& t, const AdamwNumbers& a, bool vectors, int64_t begin, int64_t end) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  P* const p = static_cast<P*>(t.p);
  G* const g = static_cast<G*>(t.g);
  const int64_t n = t.n;
  const float keep = t.keep;
  for (int64_t b = begin + warp * ADAMW_BLOCK; b < end; b += ADAMW_PASS) {
    const int64_t i = b + lane * 8, block = b / ADAMW_BLOCK;
    float x[8], gr[8], m[8], v[8], root[8];
    load8(g, i, n, vectors, gr);
    if constexpr (MASTER)
      load8(t.master, i, n, vectors, x);
    else
      load8(p, i, n, vectors, x);
    if constexpr (BITS == 8) {
      const uint2 mc = load_codes(static_cast<const uint8_t*>(t.m), i, n, vectors), vc = load_codes(static_cast<const uint8_t*>(t.v), i, n, vectors);
      const float ms = t.m_scale[block], vs = t.v_scale[block];
      decode8(mc, ms, m);
      decode8(vc, vs, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], v[j]);
    } else {
      load8(static_cast<const float*>(t.m), i, n, vectors, m);
      load8(static_cast<const float*>(t.v), i, n, vectors, v);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = __fmul_rn(gr[j], a.grad_scale);
      m[j] = __fadd_rn(__fmul_rn(m[j], a.beta1), __fmul_rn(d, a.rest1));
      v[j] = __fadd_rn(__fmul_rn(v[j], a.beta2), __fmul_rn(__fmul_rn(d, d), a.rest2));
      root[j] = __fsqrt_rn(v[j]);
      x[j] = fmaf(x[j], keep, -__fdividef(m[j] * a.lr1, fmaf(root[j], a.root2, a.eps)));
    }
    if constexpr (BITS == 8) {
      uint32_t dither[8], code[8];
      const uint32_t d0 = static_cast<uint32_t>(i) * DITHER_ELEMENT + a.dither;
#pragma unroll
      for (int j = 0; j < 8; ++j) dither[j] = (d0 + j * DITHER_ELEMENT) >> 12;
      const float ms = hold8(m, dither, code);
#pragma unroll
      for (int j = 0; j < 8; ++j) code[j] |= __float_as_uint(m[j]) >> 24 & 0x80u;
      store_codes(static_cast<uint8_t*>(t.m), i, n, vectors, code);
#pragma unroll
      for (int j = 0; j < 8; ++j) dither[j] = ~(d0 + j * DITHER_ELEMENT) >> 12;
      const float vs = hold8(root, dither, code);
#pragma unroll
      for (int j = 0; j < 8; ++j) code[j] = max(code[j], root[j] > 0.f ? 1u : 0u);
      store_codes(static_cast<uint8_t*>(t.v), i, n, vectors, code);
      if (lane == 0) {
        t.m_scale[block] = ms;
        t.v_scale[block] = vs;
      }
    } else {
      store8(static_cast<float*>(t.m), i, n, vectors, m);
      store8(static_cast<float*>(t.v), i, n, vectors, v);
    }
    if constexpr (MASTER) store8(t.master, i, n, vectors, x);
    store8(p, i, n, vectors, x);
    if (a.zero_grad) {
      const float zero[8] = {};
      store8(g, i, n, vectors, zero);
    }
  }
}

template <int BITS, int N>
__global__ void __launch_bounds__(ADAMW_THREADS) adamw_many_kernel(const __grid_constant__ AdamwTable<N> table) {
  int lo = 0, hi = table.count - 1;   // the last entry whose first CTA is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (table.e[mid].first <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const AdamwEntry& e = table.e[lo];
  const int64_t begin = static_cast<int64_t>(blockIdx.x - e.first) * table.chunk;
  const int64_t end = begin + table.chunk < e.t.n ? begin + table.chunk : e.t.n;
  const bool vectors = e.flags & ADAMW_VECTORS;
  grid_wait();
  grid_release();
  using bf16 = __nv_bfloat16;
  if (e.flags & ADAMW_P32) {
    if (e.flags & ADAMW_G32)
      adamw_chunk<BITS, float, float, false>(e.t, table.a, vectors, begin, end);
    else
      adamw_chunk<BITS, float, bf16, false>(e.t, table.a, vectors, begin, end);
  } else if (e.t.master) {
    if (e.flags & ADAMW_G32)
      adamw_chunk<BITS, bf16, float, true>(e.t, table.a, vectors, begin, end);
    else
      adamw_chunk<BITS, bf16, bf16, true>(e.t, table.a, vectors, begin, end);
  } else {
    if (e.flags & ADAMW_G32)
      adamw_chunk<BITS, bf16, float, false>(e.t, table.a, vectors, begin, end);
    else
      adamw_chunk<BITS, bf16, bf16, false>(e.t, table.a, vectors, begin, end);
  }
}

static bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Elements of a CTA: as few as fill the chip, up to four passes of it.
static int adamw_chunk_elements(int64_t total) {
  const int64_t per_sm = total / (static_cast<int64_t>(sm_count()) * 8 * ADAMW_PASS);
  return ADAMW_PASS * static_cast<int>(per_sm < 1 ? 1 : per_sm > 4 ? 4 : per_sm);
}

template <int N>
static int launch_adamw(const B200AdamwTensor* list, int count, int bits, const AdamwNumbers& a, int chunk, cudaStream_t stream) {
  AdamwTable<N> table;
  int64_t ctas = 0;
  for (int i = 0; i < count; ++i) {
    AdamwEntry& e = table.e[i];
    e.t = list[i];
    e.first = static_cast<uint32_t>(ctas);
    const int state = bits == 8 ? 8 : 16;
    const bool vectors = on(e.t.p, 16) && on(e.t.g, 16) && on(e.t.master, 16) && on(e.t.m, state) && on(e.t.v, state);
    e.flags = (e.t.p_fp32 ? ADAMW_P32 : 0) | (e.t.g_fp32 ? ADAMW_G32 : 0) | (vectors ? ADAMW_VECTORS : 0);
    ctas += (e.t.n + chunk - 1) / chunk;
  }
  if (ctas > INT_MAX) return B200_ERR_TOO_LARGE;
  table.a = a;
  table.count = count;
  table.chunk = chunk;
  launch_dependent(bits == 8 ? adamw_many_kernel<8, N> : adamw_many_kernel<32, N>, static_cast<int>(ctas), ADAMW_THREADS, 0, stream, table);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace b200

extern "C" {
using namespace b200;

int b200_adamw_many(const B200AdamwTensor* list, int count, int bits, double lr, double beta1, double beta2, double eps, long long step, double grad_scale,
                    int zero_grad, int* launches, void* stream) {
  ensure_context();
  if (launches) *launches = 0;
  if (count < 0 || (count && !list) || (bits != 8 && bits != 32) || step < 1) return B200_ERR_BAD_ARG;
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    const B200AdamwTensor& t = list[i];
    if (t.n <= 0 || !t.p || !t.g || !t.m || !t.v || (bits == 8 && (!t.m_scale || !t.v_scale)) || (t.master && t.p_fp32)) return B200_ERR_BAD_ARG;
    if (!on(t.p, t.p_fp32 ? 4 : 2) || !on(t.g, t.g_fp32 ? 4 : 2) || !on(t.master, 4) || !on(t.m_scale, 4) || !on(t.v_scale, 4)) return B200_ERR_BAD_ARG;
    if (bits == 32 && (!on(t.m, 4) || !on(t.v, 4))) return B200_ERR_BAD_ARG;
    if (t.n > (1ll << 42) - total) return B200_ERR_TOO_LARGE;
    total += t.n;
  }
  const double c1 = 1.0 - pow(beta1, static_cast<double>(step)), c2 = 1.0 - pow(beta2, static_cast<double>(step));
  AdamwNumbers a{};
  a.beta1 = static_cast<float>(beta1);
  a.rest1 = static_cast<float>(1.0 - beta1);
  a.beta2 = static_cast<float>(beta2);
  a.rest2 = static_cast<float>(1.0 - beta2);
  a.lr1 = static_cast<float>(lr / c1);
  a.root2 = static_cast<float>(1.0 / sqrt(c2));
  a.eps = static_cast<float>(eps);
  a.grad_scale = static_cast<float>(grad_scale);
  a.dither = static_cast<uint32_t>(step) * DITHER_STEP;
  a.zero_grad = zero_grad;
  const int chunk = adamw_chunk_elements(total);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int at = 0; at < count; at += ADAMW_MOST) {
    const int some = count - at < ADAMW_MOST ? count - at : ADAMW_MOST;
    const int rc = some <= 16 ? launch_adamw<16>(list + at, some, bits, a, chunk, s)
                 : some <= 128 ? launch_adamw<128>(list + at, some, bits, a, chunk, s)
                               : launch_adamw<ADAMW_MOST>(list + at, some, bits, a, chunk, s);
    if (rc) return rc;
    if (launches) ++*launches;
  }
  return 0;
}

}  // extern "C"
