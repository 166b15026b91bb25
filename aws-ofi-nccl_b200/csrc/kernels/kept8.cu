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
// Vectors of a thread, all of whose loads are under way at once. 4096 x 4096 is kept in 13.4 us (3.8 TB/s) and comes back in 8.2, SwiGLU of 4096 x 14336 keeps its
// halves in 83 (5.7 TB/s; issue slots 85 % busy: 30 instructions an element) and makes its gradient of them in 82 to 85 (5.6). With one vector each the first three took
// 17.8, 10.9 and 106 us, before the search for values that are not finite came out of the way of the others; with four 16.9, 9.7 and 101. The gradient, which reads
// three tensors, took 82.2 with one, 82.3 with two and 87.7 with four.
constexpr int KEEP_VECS = 2, KEPT_VECS = 2, SWIGLU_KEEP_VECS = 2, SWIGLU_KEPT_VECS = 1;

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

// A CTA's vectors, VECS for a thread, whose loads are all under way before the first is worked on. k counts a launch's vectors.
template <int VECS>
__device__ __forceinline__ int kept_vector(int i) {
  return (static_cast<int>(blockIdx.x) * VECS + i) * KEPT_THREADS + static_cast<int>(threadIdx.x);
}

template <int VECS>
__global__ void __launch_bounds__(KEPT_THREADS) keep8_kernel(const bf16* x, int64_t pitch, uint8_t* codes, uint8_t* powers, KeptRows s) {
  grid_wait();
  grid_release();
  KeptPlace p[VECS];
  uint4 v[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    p[i] = kept_place(s, kept_vector<VECS>(i));
    v[i] = make_uint4(0, 0, 0, 0);
    if (p[i].there) v[i] = *reinterpret_cast<const uint4*>(x + p[i].row * pitch + p[i].col);
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    uint32_t power;
    float f[8];
    unpack8(v[i], f);
    const uint2 c = keep8(v[i], f, power);
    store_kept(s, p[i], c, power, codes, powers);
  }
}

template <int VECS>
__global__ void __launch_bounds__(KEPT_THREADS) kept8_kernel(const uint8_t* codes, const uint8_t* powers, bf16* x, KeptRows s) {
  grid_wait();
  grid_release();
  KeptPlace p[VECS];
  uint2 c[VECS];
  uint32_t power[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    p[i] = kept_place(s, kept_vector<VECS>(i));
    c[i] = make_uint2(0, 0);
    power[i] = 0;
    if (!p[i].there) continue;
    c[i] = *reinterpret_cast<const uint2*>(codes + p[i].row * s.width + p[i].col);
    power[i] = powers[p[i].row * s.groups + p[i].col / KEPT_GROUP];
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    if (!p[i].there) continue;
    float f[8];
    kept8(c[i], power[i], f);
    *reinterpret_cast<uint4*>(x + p[i].row * s.width + p[i].col) = pack8(f);
  }
}

// gate|up [T][2F] -> act = silu(gate) * up, of the values as they come, and both halves as they are kept: rows 2t and 2t + 1 of F elements. s: T rows of F.
template <int VECS>
__global__ void __launch_bounds__(KEPT_THREADS) swiglu_keep8_kernel(const bf16* gu, bf16* act, uint8_t* codes, uint8_t* powers, KeptRows s) {
  grid_wait();
  grid_release();
  KeptPlace p[VECS];
  uint4 g[VECS], u[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    p[i] = kept_place(s, kept_vector<VECS>(i));
    g[i] = u[i] = make_uint4(0, 0, 0, 0);
    if (!p[i].there) continue;
    const bf16* at = gu + p[i].row * 2 * s.width + p[i].col;
    g[i] = load_once(at);
    u[i] = load_once(at + s.width);
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    float a[8], b[8];
    unpack8(g[i], a);
    unpack8(u[i], b);
    if (p[i].there) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; e += 2) (Pair(silu(a[e]), silu(a[e + 1])) * Pair(b[e], b[e + 1])).to(o[e], o[e + 1]);
      *reinterpret_cast<uint4*>(act + p[i].row * s.width + p[i].col) = pack8(o);
    }
    uint32_t g_power, u_power;
    const uint2 g_codes = keep8(g[i], a, g_power), u_codes = keep8(u[i], b, u_power);
    KeptPlace half = p[i];
    half.row *= 2;
    store_kept(s, half, g_codes, g_power, codes, powers);
    half.row += 1;
    store_kept(s, half, u_codes, u_power, codes, powers);
  }
}

// What the backward pass makes of kept halves. GRAD: their gradients [T][2F] from that of act; else the halves themselves (and act, unless null).
template <bool GRAD, int VECS>
__global__ void __launch_bounds__(KEPT_THREADS)
    swiglu_kept8_kernel(const uint8_t* codes, const uint8_t* powers, const bf16* dout, bf16* to, bf16* act, KeptRows s) {
  grid_wait();
  grid_release();
  KeptPlace p[VECS];
  uint2 gc[VECS], uc[VECS];
  uint32_t gp[VECS], up[VECS];
  uint4 d4[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    p[i] = kept_place(s, kept_vector<VECS>(i));
    if (!p[i].there) continue;
    const uint8_t* at = codes + p[i].row * 2 * s.width + p[i].col;
    const uint8_t* power = powers + p[i].row * 2 * s.groups + p[i].col / KEPT_GROUP;
    gc[i] = *reinterpret_cast<const uint2*>(at), uc[i] = *reinterpret_cast<const uint2*>(at + s.width);
    gp[i] = power[0], up[i] = power[s.groups];
    if constexpr (GRAD) d4[i] = load_once(dout + p[i].row * s.width + p[i].col);
  }
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    if (!p[i].there) continue;
    float g[8], u[8];
    kept8(gc[i], gp[i], g);
    kept8(uc[i], up[i], u);
    bf16* row = to + p[i].row * 2 * s.width + p[i].col;
    if constexpr (GRAD) {
      float d[8];
      unpack8(d4[i], d);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const Pair l(logistic(g[e]), logistic(g[e + 1])), d2(d[e], d[e + 1]), a = Pair(g[e], g[e + 1]) * l;
        const Pair slope = fma2(a, fma2(l, both(-1.f), both(1.f)), l);
        (d2 * Pair(u[e], u[e + 1]) * slope).to(g[e], g[e + 1]);
        (d2 * a).to(u[e], u[e + 1]);
      }
    } else if (act) {
      float a[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) a[e] = silu(g[e]) * u[e];
      *reinterpret_cast<uint4*>(act + p[i].row * s.width + p[i].col) = pack8(a);
    }
    __stcs(reinterpret_cast<uint4*>(row), pack8(g));
    __stcs(reinterpret_cast<uint4*>(row + s.width), pack8(u));
  }
}

// Calls launch(first row, rows, CTAs of so many vectors a thread) for slices of less than 2^30 vectors, so that their numbers have 32 bits.
template <class F>
static int in_slices(long long rows, int width, int vecs_of_thread, F launch) {
  const int vecs = (width + KEPT_GROUP - 1) / KEPT_GROUP * 4, of_cta = KEPT_THREADS * vecs_of_thread;
  const long long most = std::max(1ll, (1ll << 30) / vecs);
  for (long long at = 0; at < rows; at += most) {
    const KeptRows s(static_cast<int>(std::min(most, rows - at)), width);
    launch(at, s, static_cast<int>((static_cast<int64_t>(s.rows) * vecs + of_cta - 1) / of_cta));
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
  return in_slices(rows, width, KEEP_VECS, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(keep8_kernel<KEEP_VECS>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const bf16*>(x) + at * pitch, pitch,
                     static_cast<uint8_t*>(codes) + at * width, static_cast<uint8_t*>(powers) + at * s.groups, s);
  });
}

int b200_kept8(const void* codes, const void* powers, void* x, long long rows, int width, void* stream) {
  if (rows == 0) return 0;
  ensure_context();
  if (!kept_ok(rows, width, {x}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(rows, width, KEPT_VECS, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(kept8_kernel<KEPT_VECS>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * width,
                     static_cast<const uint8_t*>(powers) + at * s.groups, static_cast<bf16*>(x) + at * width, s);
  });
}

int b200_swiglu_keep8(const void* gu, void* act, void* codes, void* powers, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {gu, act}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(T, F, SWIGLU_KEEP_VECS, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_keep8_kernel<SWIGLU_KEEP_VECS>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const bf16*>(gu) + at * 2 * F,
                     static_cast<bf16*>(act) + at * F, static_cast<uint8_t*>(codes) + at * 2 * F, static_cast<uint8_t*>(powers) + at * 2 * s.groups, s);
  });
}

int b200_swiglu_bwd8(const void* dout, const void* codes, const void* powers, void* dgu, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {dout, dgu}, {codes}) || !powers) return B200_ERR_BAD_ARG;
  return in_slices(T, F, SWIGLU_KEPT_VECS, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_kept8_kernel<true, SWIGLU_KEPT_VECS>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * 2 * F,
                     static_cast<const uint8_t*>(powers) + at * 2 * s.groups, static_cast<const bf16*>(dout) + at * F, static_cast<bf16*>(dgu) + at * 2 * F,
                     static_cast<bf16*>(nullptr), s);
  });
}

int b200_swiglu_kept8(const void* codes, const void* powers, void* gu, void* act, long long T, int F, void* stream) {
  if (T == 0) return 0;
  ensure_context();
  if (!kept_ok(T, F, {gu}, {codes}) || !powers || reinterpret_cast<uintptr_t>(act) % 16) return B200_ERR_BAD_ARG;
  return in_slices(T, F, SWIGLU_KEPT_VECS, [&](long long at, const KeptRows& s, int grid) {
    launch_dependent(swiglu_kept8_kernel<false, SWIGLU_KEPT_VECS>, grid, KEPT_THREADS, 0, static_cast<cudaStream_t>(stream), static_cast<const uint8_t*>(codes) + at * 2 * F,
                     static_cast<const uint8_t*>(powers) + at * 2 * s.groups, static_cast<const bf16*>(nullptr), static_cast<bf16*>(gu) + at * 2 * F,
                     act ? static_cast<bf16*>(act) + at * F : nullptr, s);
  });
}

}  // extern "C"
