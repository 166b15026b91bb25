// Activations kept in 8 bits for the backward pass, and the SwiGLU that keeps and reads them: see kept8.cuh for what is kept.
//
// A thread has a vector of eight elements, four neighbouring lanes a group; lanes behind a row's end, where that is not a group's, have zeros. All of
// it is bounded by memory.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "divisor.h"
#include "host_util.h"
#include "kept8.cuh"
#include "swiglu_math.cuh"

namespace b200 {

using bf16 = __nv_bfloat16;

constexpr int KEPT_THREADS = 256;

// Rows of `width` elements as vectors: `vecs` for each, of which the last may lie behind the row's end.
struct KeptRows {
  int rows, width, groups;   // groups: of a row
  Divisor by_vecs;
  KeptRows(int r, int w) : rows(r), width(w), groups((w + KEPT_GROUP - 1) / KEPT_GROUP), by_vecs(groups * 4) {}
};
struct KeptPlace {
  int64_t row;
  int col;
  bool there;
};
__device__ __forceinline__ KeptPlace kept_place(const KeptRows& s, int k) {
  KeptPlace p;
  const int row = s.by_vecs.quotient(k);
  p.row = row;
  p.col = (k - row * s.by_vecs.d) * 8;
  p.there = row < s.rows && p.col < s.width;
  return p;
}
__device__ __forceinline__ uint4 load_once(const void* p) { return __ldcs(static_cast<const uint4*>(p)); }
__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) f[2 * k] = __uint_as_float(w[k] << 16), f[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
    w[k] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_kept(const KeptRows& s, const KeptPlace& p, const uint2& codes, uint32_t power, uint8_t* to, uint8_t* powers) {
  if (!p.there) return;
  *reinterpret_cast<uint2*>(to + p.row * s.width + p.col) = codes;
  if ((p.col & (KEPT_GROUP - 8)) == 0) powers[p.row * s.groups + p.col / KEPT_GROUP] = static_cast<uint8_t>(power);
}

// Rows are numbered from the launch's first; k counts a launch's vectors. All threads of a warp have the same number of turns.
template <class F>
__device__ __forceinline__ void for_vectors(const KeptRows& s, F f) {
  const int64_t total = static_cast<int64_t>(s.rows) * s.by_vecs.d, step = static_cast<int64_t>(gridDim.x) * KEPT_THREADS;
  for (int64_t k = static_cast<int64_t>(blockIdx.x) * KEPT_THREADS; k < total; k += step) f(static_cast<int>(k) + static_cast<int>(threadIdx.x));
}

__global__ void __launch_bounds__(KEPT_THREADS) keep8_kernel(const bf16* x, int64_t pitch, uint8_t* codes, uint8_t* powers, KeptRows s) {
  grid_wait();
  grid_release();
  for_vectors(s, [&](int k) {
    const KeptPlace p = kept_place(s, k);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (p.there) v = *reinterpret_cast<const uint4*>(x + p.row * pitch + p.col);
    uint32_t power;
    const uint2 c = keep8(v, power);
    store_kept(s, p, c, power, codes, powers);
  });
}

__global__ void __launch_bounds__(KEPT_THREADS) kept8_kernel(const uint8_t* codes, const uint8_t* powers, bf16* x, KeptRows s) {
  grid_wait();
  grid_release();
  for_vectors(s, [&](int k) {
    const KeptPlace p = kept_place(s, k);
    if (!p.there) return;
    float f[8];
    kept8(*reinterpret_cast<const uint2*>(codes + p.row * s.width + p.col), powers[p.row * s.groups + p.col / KEPT_GROUP], f);
    *reinterpret_cast<uint4*>(x + p.row * s.width + p.col) = pack8(f);
  });
}

// gate|up [T][2F] -> act = silu(gate) * up, of the values as they come, and both halves as they are kept: rows 2t and 2t + 1 of F elements. s: T rows of F.
__global__ void __launch_bounds__(KEPT_THREADS) swiglu_keep8_kernel(const bf16* gu, bf16* act, uint8_t* codes, uint8_t* powers, KeptRows s) {
  grid_wait();
  grid_release();
  for_vectors(s, [&](int k) {
    KeptPlace p = kept_place(s, k);
    uint4 g = make_uint4(0, 0, 0, 0), u = g;
    if (p.there) {
      const bf16* at = gu + p.row * 2 * s.width + p.col;
      g = load_once(at);
      u = load_once(at + s.width);
      float a[8], b[8];
      unpack8(g, a);
      unpack8(u, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = silu(a[e]) * b[e];
      *reinterpret_cast<uint4*>(act + p.row * s.width + p.col) = pack8(a);
    }
    uint32_t g_power, u_power;
    const uint2 g_codes = keep8(g, g_power), u_codes = keep8(u, u_power);
    p.row *= 2;
    store_kept(s, p, g_codes, g_power, codes, powers);
    p.row += 1;
    store_kept(s, p, u_codes, u_power, codes, powers);
  });
}

// What the backward pass makes of kept halves. GRAD: their gradients [T][2F] from that of act; else the halves themselves (and act, unless null).
template <bool GRAD>
__global__ void __launch_bounds__(KEPT_THREADS)
    swiglu_kept8_kernel(const uint8_t* codes, const uint8_t* powers, const bf16* dout, bf16* to, bf16* act, KeptRows s) {
  grid_wait();
  grid_release();
  for_vectors(s, [&](int k) {
    const KeptPlace p = kept_place(s, k);
    if (!p.there) return;
    const uint8_t* at = codes + p.row * 2 * s.width + p.col;
    const uint8_t* power = powers + p.row * 2 * s.groups + p.col / KEPT_GROUP;
    const uint2 gc = *reinterpret_cast<const uint2*>(at), uc = *reinterpret_cast<const uint2*>(at + s.width);
    uint4 d4;
    if constexpr (GRAD) d4 = load_once(dout + p.row * s.width + p.col);
    float g[8], u[8];
    kept8(gc, power[0], g);
    kept8(uc, power[s.groups], u);
    bf16* row = to + p.row * 2 * s.width + p.col;
    if constexpr (GRAD) {
      float d[8];
      unpack8(d4, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float l = logistic(g[e]), a = g[e] * l;
        const float dg = d[e] * u[e] * (l + a * (1.f - l));
        u[e] = d[e] * a;
        g[e] = dg;
      }
    } else if (act) {
      float a[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = silu(g[e]) * u[e];
      *reinterpret_cast<uint4*>(act + p.row * s.width + p.col) = pack8(a);
    }
    __stcs(reinterpret_cast<uint4*>(row), pack8(g));
    __stcs(reinterpret_cast<uint4*>(row + s.width), pack8(u));
  });
}

// Calls launch(first row, rows) for slices of less than 2^30 vectors, so that their numbers have 32 bits.
template <class F>
static int in_slices(long long rows, int width, F launch) {
  const int vecs = (width + KEPT_GROUP - 1) / KEPT_GROUP * 4;
  const long long most = std::max(1ll, (1ll << 30) / vecs);
  for (long long at = 0; at < rows; at += most) {
    const KeptRows s(static_cast<int>(std::min(most, rows - at)), width);
    const int64_t blocks = (static_cast<int64_t>(s.rows) * vecs + KEPT_THREADS - 1) / KEPT_THREADS;
    launch(at, s, static_cast<int>(std::min<int64_t>(blocks, static_cast<int64_t>(sm_count()) * 64)));
  }
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}
static bool kept_ok(long long rows, int width, std::initializer_list<const void*> vectors, std::initializer_list<const void*> codes) {
  if (rows < 1 || width < 8 || width % 8 || width > 1 << 29) return false;
  for (const void* p : vectors)
    if (!p || reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (const void* p : codes)
    if (!p || reinterpret_cast<uintptr_t>(p) % 8) return false;
  return true;
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_keep8(const void* x, long long pitch, void* codes, void* powers, long long rows, int width, void* stream) {
  if (rows == 0) return 0;
  ensure_context();
  if (!kept_ok(rows, width, {x}, {codes}) || !powers || (rows > 1 && pitch % 8)) return B200_ERR_BAD_ARG;
  return in_slices(rows, width, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(keep8_kernel, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const bf16*>(x) + at * pitch, pitch,
                     static_cast<uint8_t*>(codes) + at * width, static_cast<uint8_t*>(powers) + at * s.groups, s);
  });
}

int b200_kept8(const void* codes, const void* powers, void* x, long long rows, int width, void* stream) {
  if (rows == 0) return 0;
  ensure_context();
  if (!kept_ok(rows, width, {x}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(rows, width, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(kept8_kernel, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * width,
                     static_cast<const uint8_t*>(powers) + at * s.groups, static_cast<bf16*>(x) + at * width, s);
  });
}

int b200_swiglu_keep8(const void* gu, void* act, void* codes, void* powers, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {gu, act}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(T, F, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_keep8_kernel, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const bf16*>(gu) + at * 2 * F,
                     static_cast<bf16*>(act) + at * F, static_cast<uint8_t*>(codes) + at * 2 * F, static_cast<uint8_t*>(powers) + at * 2 * s.groups, s);
  });
}

int b200_swiglu_bwd8(const void* dout, const void* codes, const void* powers, void* dgu, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {dout, dgu}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(T, F, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_kept8_kernel<true>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * 2 * F,
                     static_cast<const uint8_t*>(powers) + at * 2 * s.groups, static_cast<const bf16*>(dout) + at * F, static_cast<bf16*>(dgu) + at * 2 * F,
                     static_cast<bf16*>(nullptr), s);
  });
}

int b200_swiglu_kept8(const void* codes, const void* powers, void* gu, void* act, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {gu}, {codes}) || !powers || reinterpret_cast<uintptr_t>(act) % 16) return B200_ERR_BAD_ARG;
  return in_slices(T, F, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_kept8_kernel<false>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * 2 * F,
                     static_cast<const uint8_t*>(powers) + at * 2 * s.groups, static_cast<const bf16*>(nullptr), static_cast<bf16*>(gu) + at * 2 * F,
                     act ? static_cast<bf16*>(act) + at * F : nullptr, s);
  });
}

}  // extern "C"
