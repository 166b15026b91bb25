// Tokens sorted by expert and back on one GPU: where a mixture-of-experts layer has all its experts here, its rows need no window, no
// records and no signals (moe.cu), and no atomics: the order is that of a stable sort.
//
// A slot n = t * k + j is token t's j-th choice. Its row is the number of slots that go to an earlier expert, or to the same one and stand
// before it; slots whose expert is none of [0, E) come behind all others, and row_of holds ~row for them. So row_of is a permutation: every
// row has one writer, the zeros of the dropped ones included, and sums over a token's rows run in the order of its choices.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"

namespace b200 {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ the order
// A counting sort in one launch: a cluster of up to eight CTAs, whose counts meet in distributed shared memory. Every warp has a
// range of consecutive slots and counters of its own; it counts its range, takes as its start what the experts before, the CTAs before and
// the warps before it have, and goes over its range again, 32 slots at a time, a slot's place among them being that among the lanes with its expert.
constexpr int ORDER_WARPS = 16;
constexpr int ORDER_THREADS = 32 * ORDER_WARPS;
constexpr int ORDER_AHEAD = 8;   // indices of a lane that are on their way at once
constexpr int ORDER_MAX_EXPERTS = 1024;
constexpr int ORDER_MAX_CTAS = 8;

constexpr int order_smem(int experts) { return (ORDER_WARPS + 2) * (experts + 1) * 4; }

template <typename Index>
__global__ void __launch_bounds__(ORDER_THREADS)
    expert_order_kernel(const Index* idx, int64_t n, int experts, int32_t* row_of, int32_t* offsets) {
  extern __shared__ uint32_t order_shared[];
  __shared__ uint32_t warp_total[ORDER_WARPS];
  const cg::cluster_group cluster = cg::this_cluster();
  const int bins = experts + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t* const mine = order_shared + warp * bins;             // this warp's counts, later the rows that its slots get next
  uint32_t* const total = order_shared + ORDER_WARPS * bins;     // the CTA's counts, read by the cluster
  uint32_t* const start = total + bins;                          // each expert's first row for this CTA
  for (int i = threadIdx.x; i < ORDER_WARPS * bins; i += ORDER_THREADS) order_shared[i] = 0;
  __syncthreads();
  grid_wait();
  grid_release();
  const int64_t parts = static_cast<int64_t>(cluster.num_blocks()) * ORDER_WARPS;
  const int64_t per_warp = ((n + parts - 1) / parts + 31) / 32 * 32;
  const int64_t begin = (static_cast<int64_t>(cluster.block_rank()) * ORDER_WARPS + warp) * per_warp;
  const int64_t end = begin + per_warp < n ? begin + per_warp : n;
  auto bin_of = [&](int64_t i) {
    const Index e = idx[i];
    return e >= 0 && e < experts ? static_cast<int>(e) : experts;
  };
  for (int64_t i0 = begin + lane; i0 < end; i0 += 32 * ORDER_AHEAD) {
    int bin[ORDER_AHEAD];
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u) bin[u] = i0 + 32 * u < end ? bin_of(i0 + 32 * u) : -1;
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u)
      if (bin[u] >= 0) atomicAdd(&mine[bin[u]], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += ORDER_THREADS) {   // counts -> what the CTA's warps before have
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < ORDER_WARPS; ++w) {
      const uint32_t c = order_shared[w * bins + b];
      order_shared[w * bins + b] = sum;
      sum += c;
    }
    total[b] = sum;
  }
  cluster.sync();
  uint32_t carry = 0;   // rows of the experts before this pass's
  for (int b0 = 0; b0 < bins; b0 += ORDER_THREADS) {
    const int b = b0 + threadIdx.x;
    uint32_t before = 0, all = 0;
    if (b < bins)
      for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
        const uint32_t c = cluster.map_shared_rank(total, r)[b];
        before += r < cluster.block_rank() ? c : 0;
        all += c;
      }
    uint32_t sum = all;   // inclusive over the warp's lanes, then over the warps
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint32_t below = __shfl_up_sync(0xffffffffu, sum, o);
      sum += lane >= o ? below : 0;
    }
    if (lane == 31) warp_total[warp] = sum;
    __syncthreads();
    uint32_t first = carry + sum - all;
    for (int w = 0; w < ORDER_WARPS; ++w) {
      first += w < warp ? warp_total[w] : 0;
      carry += warp_total[w];
    }
    __syncthreads();
    if (b < bins) {
      start[b] = first + before;
      if (cluster.block_rank() == 0) offsets[b] = static_cast<int32_t>(first);   // the bin behind the experts begins where they end
    }
  }
  cluster.sync();   // nobody reads this CTA's counts any more, and `start` is whole
  for (int b = lane; b < bins; b += 32) mine[b] += start[b];
  __syncwarp();
  for (int64_t i0 = begin; i0 < end; i0 += 32 * ORDER_AHEAD) {
    int bin[ORDER_AHEAD];
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u) bin[u] = i0 + 32 * u + lane < end ? bin_of(i0 + 32 * u + lane) : -1;
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u) {
      if (i0 + 32 * u >= end) break;
      const unsigned same = __match_any_sync(0xffffffffu, bin[u]);
      const int place = __popc(same & ((1u << lane) - 1));
      uint32_t row = 0;
      if (bin[u] >= 0) row = mine[bin[u]] + place;
      __syncwarp();
      if (bin[u] >= 0) {
        if (place == 0) mine[bin[u]] += __popc(same);
        row_of[i0 + 32 * u + lane] = static_cast<int32_t>(bin[u] < experts ? row : ~row);
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------ there and back
// The rows of a token are written from one read of it, a thread for each 16-byte vector of a token (or each element, where a row is no whole
// number of aligned vectors): the stores, k times the loads, are what bounds it.
constexpr int ROWS_THREADS = 256;

// `scale`: `groups` numbers of a token that go with its rows, or null
template <typename Vec>
__global__ void __launch_bounds__(ROWS_THREADS)
    permute_rows_kernel(const char* x, int64_t pitch, Vec* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups, int64_t tokens,
                        int k, int64_t vecs) {
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(ROWS_THREADS) + threadIdx.x; i < tokens * vecs; i += static_cast<int64_t>(gridDim.x) * ROWS_THREADS) {
    const int64_t t = i / vecs, c = i - t * vecs;
    const Vec v = reinterpret_cast<const Vec*>(x + t * pitch)[c];
    for (int j = 0; j < k; ++j) {
      const int32_t r = row_of[t * k + j];
      const int64_t to = r < 0 ? ~r : r;
      if (to >= slots) continue;   // no order that this library made
      rows[to * vecs + c] = r < 0 ? Vec{} : v;
      for (int64_t q = c; q < groups; q += vecs) row_scale[to * groups + q] = r < 0 ? 0.f : scale[t * groups + q];
    }
  }
}

template <typename T, int V>
struct Values;
template <>
struct Values<__nv_bfloat16, 8> {
  using Vec = uint4;
  static __device__ __forceinline__ void get(const Vec& q, float (&f)[8]) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(p[j]), f[2 * j + 1] = __high2float(p[j]);
  }
  static __device__ __forceinline__ Vec put(const float (&f)[8]) {
    Vec q;
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    return q;
  }
};
template <>
struct Values<__nv_bfloat16, 1> {
  using Vec = __nv_bfloat16;
  static __device__ __forceinline__ void get(const Vec& q, float (&f)[1]) { f[0] = __bfloat162float(q); }
  static __device__ __forceinline__ Vec put(const float (&f)[1]) { return __float2bfloat16_rn(f[0]); }
};
template <>
struct Values<float, 4> {
  using Vec = float4;
  static __device__ __forceinline__ void get(const Vec& q, float (&f)[4]) { f[0] = q.x, f[1] = q.y, f[2] = q.z, f[3] = q.w; }
  static __device__ __forceinline__ Vec put(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <>
struct Values<float, 1> {
  using Vec = float;
  static __device__ __forceinline__ void get(const Vec& q, float (&f)[1]) { f[0] = q; }
  static __device__ __forceinline__ Vec put(const float (&f)[1]) { return f[0]; }
};

// out[t] = sum over j of w[t][j] * rows[row_of[t][j]], in 32 bits and in the order of j; w null: a plain sum. A dropped slot's row is not read.
template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS)
    unpermute_rows_kernel(const T* rows, int64_t pitch, const float* w, const int32_t* row_of, T* out, int64_t tokens, int k, int64_t vecs) {
  using Vec = typename Values<T, V>::Vec;
  constexpr int U = 4;
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(ROWS_THREADS) + threadIdx.x; i < tokens * vecs; i += static_cast<int64_t>(gridDim.x) * ROWS_THREADS) {
    const int64_t t = i / vecs, c = i - t * vecs;
    float acc[V] = {};
    for (int j0 = 0; j0 < k; j0 += U) {
      Vec q[U];
      bool there[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int32_t r = j0 + u < k ? row_of[t * k + j0 + u] : -1;
        there[u] = r >= 0 && r < slots;
        if (there[u]) q[u] = reinterpret_cast<const Vec*>(rows + r * pitch)[c];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!there[u]) continue;
        float f[V];
        Values<T, V>::get(q[u], f);
        const float ws = w ? w[t * k + j0 + u] : 1.f;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(ws, f[e], acc[e]);
      }
    }
    reinterpret_cast<Vec*>(out)[i] = Values<T, V>::put(acc);
  }
}

// What flows back through a weighted sum: drows[row_of[t][j]] = w[t][j] * dout[t] (zeros for a dropped slot, of which nothing is read) and
// dw[t][j] = <dout[t], rows[row_of[t][j]]>, either of them left out where its pointer is null. A team of warps has a token: its gradient is read once for U
// rows, and a row's product is added up over the team in the order of its warps.
constexpr int BACK_WARPS = ROWS_THREADS / 32;
template <typename T, int V>
__global__ void __launch_bounds__(ROWS_THREADS)
    unpermute_rows_bwd_kernel(const T* dout, const T* rows, int64_t pitch, const float* w, const int32_t* row_of, T* drows, float* dw, int64_t tokens,
                              int k, int64_t vecs, int team_warps) {
  using Vec = typename Values<T, V>::Vec;
  constexpr int U = 4;
  __shared__ float parts[BACK_WARPS][U];
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = warp / team_warps * team_warps, teams = BACK_WARPS / team_warps;
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * teams; t0 < tokens; t0 += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t t = t0 + warp / team_warps;   // the same number of passes for every warp of the CTA, for the barriers
    for (int j0 = 0; j0 < k; j0 += U) {
      float acc[U] = {}, ws[U];
      int32_t r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool mine = t < tokens && j0 + u < k;
        r[u] = mine ? row_of[t * k + j0 + u] : INT_MIN;
        ws[u] = mine ? w[t * k + j0 + u] : 0.f;
      }
      if (t < tokens)
        for (int64_t c = (warp - first) * 32 + lane; c < vecs; c += team_warps * 32) {
          float d[V];
          Values<T, V>::get(reinterpret_cast<const Vec*>(dout)[t * vecs + c], d);
          Vec q[U];
          if (dw) {
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (r[u] >= 0 && r[u] < slots) q[u] = reinterpret_cast<const Vec*>(rows + r[u] * pitch)[c];
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int64_t to = r[u] < 0 ? ~r[u] : r[u];
            if (to >= slots) continue;   // INT_MIN is none either: ~INT_MIN is the largest number
            float f[V] = {};
            if (r[u] >= 0) {
#pragma unroll
              for (int e = 0; e < V; ++e) f[e] = ws[u] * d[e];
            }
            if (drows) reinterpret_cast<Vec*>(drows)[to * vecs + c] = Values<T, V>::put(f);
            if (dw && r[u] >= 0) {
              Values<T, V>::get(q[u], f);
#pragma unroll
              for (int e = 0; e < V; ++e) acc[u] = fmaf(d[e], f[e], acc[u]);
            }
          }
        }
      if (!dw) continue;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[u] += __shfl_xor_sync(0xffffffffu, acc[u], o);
        if (lane == 0) parts[warp][u] = acc[u];
      }
      __syncthreads();
      if (warp == first && lane < U && t < tokens && j0 + lane < k) {
        float sum = 0.f;
        for (int q = 0; q < team_warps; ++q) sum += parts[first + q][lane];
        dw[t * k + j0 + lane] = sum;
      }
      __syncthreads();
    }
  }
}

static int rows_grid(int64_t ctas, int per_sm) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(ctas < 1 ? 1 : ctas < cap ? ctas : cap);
}
static bool bad_slots(long long tokens, int k) { return tokens < 0 || k <= 0 || tokens > INT_MAX / k; }
static bool on(const void* p, long long pitch, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch % bytes == 0; }

template <typename Index>
static int launch_order(const void* idx, long long n, int experts, int32_t* row_of, int32_t* offsets, cudaStream_t stream) {
  constexpr auto kern = expert_order_kernel<Index>;
  const int rc = allow_smem<kern>(order_smem(ORDER_MAX_EXPERTS));
  if (rc) return rc;
  int ctas = 1;
  while (ctas < ORDER_MAX_CTAS && n > static_cast<int64_t>(ctas) * ORDER_THREADS * ORDER_AHEAD) ctas *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(ORDER_THREADS);
  cfg.dynamicSmemBytes = order_smem(experts);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, static_cast<const Index*>(idx), static_cast<int64_t>(n), experts, row_of, offsets));
  return 0;
}

template <typename Vec>
static void launch_permute(const void* x, long long pitch, void* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups,
                           long long tokens, int k, long long row_bytes, cudaStream_t stream) {
  const int64_t vecs = row_bytes / sizeof(Vec);
  launch_dependent(permute_rows_kernel<Vec>, rows_grid((tokens * vecs + ROWS_THREADS - 1) / ROWS_THREADS, 64), ROWS_THREADS, 0, stream,
                   static_cast<const char*>(x), static_cast<int64_t>(pitch), static_cast<Vec*>(rows), row_of, scale, row_scale, groups,
                   static_cast<int64_t>(tokens), k, vecs);
}
template <typename T, int V>
static void launch_unpermute(const void* rows, long long pitch, const float* w, const int32_t* row_of, void* out, long long tokens, int k, int H,
                             cudaStream_t stream) {
  const int64_t vecs = H / V;
  launch_dependent(unpermute_rows_kernel<T, V>, rows_grid((tokens * vecs + ROWS_THREADS - 1) / ROWS_THREADS, 64), ROWS_THREADS, 0, stream,
                   static_cast<const T*>(rows), static_cast<int64_t>(pitch), w, row_of, static_cast<T*>(out), static_cast<int64_t>(tokens), k, vecs);
}
template <typename T, int V>
static void launch_unpermute_bwd(const void* dout, const void* rows, long long pitch, const float* w, const int32_t* row_of, void* drows, float* dw,
                                 long long tokens, int k, int H, cudaStream_t stream) {
  const int64_t vecs = H / V;
  int team = 1;
  while (team < BACK_WARPS && team * 128 < vecs) team *= 2;
  const int teams = BACK_WARPS / team;
  launch_dependent(unpermute_rows_bwd_kernel<T, V>, rows_grid((tokens + teams - 1) / teams, 64), ROWS_THREADS, 0, stream, static_cast<const T*>(dout),
                   static_cast<const T*>(rows), static_cast<int64_t>(pitch), w, row_of, static_cast<T*>(drows), dw, static_cast<int64_t>(tokens), k, vecs,
                   team);
}

}  // namespace b200

extern "C" {
using namespace b200;

// row_of [n] and offsets [experts + 1] of the n choices idx, of 32 or 64 bits.
int b200_expert_order(const void* idx, int idx64, long long n, int experts, int* row_of, int* offsets, void* stream) {
  ensure_context();
  if (n < 0 || n > INT_MAX || experts < 1 || experts > ORDER_MAX_EXPERTS || !offsets || (n && (!idx || !row_of))) return B200_ERR_BAD_ARG;
  if (!on(idx, 0, idx64 ? 8 : 4) || !on(row_of, 0, 4) || !on(offsets, 0, 4)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return idx64 ? launch_order<int64_t>(idx, n, experts, row_of, offsets, s) : launch_order<int32_t>(idx, n, experts, row_of, offsets, s);
}

// rows [tokens * k][row_bytes] from x, whose rows lie `pitch` bytes apart; elements of `elem` bytes (1, 2 or 4). With `scale` [tokens][groups]
// row_scale [tokens * k][groups] too.
int b200_permute_rows(const void* x, long long pitch, void* rows, const int* row_of, const float* scale, float* row_scale, int groups, long long tokens,
                      int k, long long row_bytes, int elem, void* stream) {
  ensure_context();
  if (bad_slots(tokens, k) || row_bytes <= 0 || (elem != 1 && elem != 2 && elem != 4) || row_bytes % elem) return B200_ERR_BAD_ARG;
  if (!scale != !row_scale || (scale ? groups <= 0 : groups != 0)) return B200_ERR_BAD_ARG;
  if (!tokens) return 0;
  if (!x || !rows || !row_of || !on(x, pitch, elem) || !on(rows, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (on(x, pitch, 16) && on(rows, row_bytes, 16))
    launch_permute<uint4>(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, row_bytes, s);
  else if (elem == 4)
    launch_permute<uint32_t>(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, row_bytes, s);
  else if (elem == 2)
    launch_permute<uint16_t>(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, row_bytes, s);
  else
    launch_permute<uint8_t>(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, row_bytes, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

// out [tokens][H] = sums over the k rows of each token, weighted by w [tokens][k] unless null; rows lie `pitch` elements apart. bf16, or fp32.
int b200_unpermute_rows(const void* rows, long long pitch, const float* w, const int* row_of, void* out, long long tokens, int k, int H, int fp32,
                        void* stream) {
  ensure_context();
  if (bad_slots(tokens, k) || H <= 0) return B200_ERR_BAD_ARG;
  if (!tokens) return 0;
  const int elem = fp32 ? 4 : 2;
  if (!rows || !row_of || !out || !on(rows, 0, elem) || !on(out, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = on(rows, pitch * elem, 16) && on(out, static_cast<long long>(H) * elem, 16);
  if (fp32)
    (wide ? launch_unpermute<float, 4> : launch_unpermute<float, 1>)(rows, pitch, w, row_of, out, tokens, k, H, s);
  else
    (wide ? launch_unpermute<__nv_bfloat16, 8> : launch_unpermute<__nv_bfloat16, 1>)(rows, pitch, w, row_of, out, tokens, k, H, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

// The gradients of that weighted sum; drows or dw may be null, rows where dw is.
int b200_unpermute_rows_bwd(const void* dout, const void* rows, long long pitch, const float* w, const int* row_of, void* drows, float* dw,
                            long long tokens, int k, int H, int fp32, void* stream) {
  ensure_context();
  if (bad_slots(tokens, k) || H <= 0) return B200_ERR_BAD_ARG;
  if (!tokens || (!drows && !dw)) return 0;
  const int elem = fp32 ? 4 : 2;
  if (!dout || !w || !row_of || (dw && !rows) || !on(dout, 0, elem) || !on(rows, 0, elem) || !on(drows, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = on(dout, static_cast<long long>(H) * elem, 16) && on(drows, 0, 16) && (!dw || on(rows, pitch * elem, 16));
  if (fp32)
    (wide ? launch_unpermute_bwd<float, 4> : launch_unpermute_bwd<float, 1>)(dout, rows, pitch, w, row_of, drows, dw, tokens, k, H, s);
  else
    (wide ? launch_unpermute_bwd<__nv_bfloat16, 8> : launch_unpermute_bwd<__nv_bfloat16, 1>)(dout, rows, pitch, w, row_of, drows, dw, tokens, k, H, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // extern "C"
