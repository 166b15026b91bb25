// Tokens sorted by expert and back on one GPU: where a mixture-of-experts layer has all its experts here, its rows need no window, no
// records and no signals (moe.cu), and no counters in memory: the order is that of a stable sort. Counts are added up by atomics in shared memory, whose
// order no sum depends on.
//
// A slot n = t * k + j is token t's j-th choice. Its row is the number of slots that go to an earlier expert, or to the same one and stand
// before it; slots whose expert is none of [0, E) come behind all others, and row_of holds ~row for them. So row_of is a permutation: every
// row has one writer, the zeros of the dropped ones included, and sums over a token's rows run in the order of its choices.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"

namespace b200 {

namespace cg = cooperative_groups;

// ------------------------------------------------------------------ the order
// A counting sort in one launch: a cluster of CTAs, whose counts meet in distributed shared memory. Every warp has a range of
// consecutive slots and counters of its own; it counts its range, takes as its start what the experts before, the CTAs before and
// the warps before it have, and goes over its range again, 32 slots at a time, a slot's place among them being that among the lanes with its expert.
// Latencies bound it: 32768 slots of 256 experts take 6.2 us, 524288 of 64 33. With the lanes of an expert found by a match of whole numbers they take 6.8 and
// 39, with both passes that way 7.5 and 69.
constexpr int ORDER_WARPS = 16;
constexpr int ORDER_AHEAD = 8;    // indices of a lane that are on their way at once
constexpr int ORDER_MAX_EXPERTS = 1024;
constexpr int ORDER_CTAS = 16;    // more than 8 are not portable, but this GPU has room for them: eight take 1.2 and 1.8 times as long at those sizes

constexpr int order_smem(int warps, int experts) { return (warps + 2) * (experts + 1) * 4; }

template <typename Index, int CTAS>
__global__ void __launch_bounds__(32 * ORDER_WARPS)
    expert_order_kernel(const Index* idx, int64_t n, int experts, int32_t* row_of, int32_t* offsets) {
  extern __shared__ uint32_t order_shared[];
  __shared__ uint32_t warp_total[ORDER_WARPS];
  const cg::cluster_group cluster = cg::this_cluster();
  const int bins = experts + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int warps = CTAS > 1 ? ORDER_WARPS : blockDim.x >> 5, threads = 32 * warps;
  const unsigned rank = CTAS > 1 ? cluster.block_rank() : 0;
  uint32_t* const mine = order_shared + warp * bins;       // this warp's counts, later the rows that its slots get next
  uint32_t* const total = order_shared + warps * bins;     // the CTA's counts, read by the cluster
  uint32_t* const start = total + bins;                    // each expert's first row for this CTA
  for (int i = threadIdx.x; i < warps * bins; i += threads) order_shared[i] = 0;
  __syncthreads();
  grid_wait();
  grid_release();
  const int64_t parts = static_cast<int64_t>(CTAS) * warps;
  const int64_t per_warp = ((n + parts - 1) / parts + 31) / 32 * 32;
  const int64_t begin = (static_cast<int64_t>(rank) * warps + warp) * per_warp;
  const int64_t end = begin + per_warp < n ? begin + per_warp : n;
  auto bin_of = [&](int64_t i) {
    const Index e = idx[i];
    return e >= 0 && e < experts ? static_cast<int>(e) : experts;
  };
  int bin[ORDER_AHEAD];   // of the last batch, which is the only one of most calls
  auto load = [&](int64_t i0) {
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u) bin[u] = i0 + 32 * u + lane < end ? bin_of(i0 + 32 * u + lane) : -1;
  };
  for (int64_t i0 = begin; i0 < end; i0 += 32 * ORDER_AHEAD) {
    load(i0);
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u)
      if (bin[u] >= 0) atomicAdd(&mine[bin[u]], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += threads) {   // counts -> what the CTA's warps before have
    uint32_t sum = 0, c[ORDER_WARPS];
#pragma unroll
    for (int w = 0; w < ORDER_WARPS; ++w) c[w] = w < warps ? order_shared[w * bins + b] : 0;
#pragma unroll
    for (int w = 0; w < ORDER_WARPS; ++w) {
      if (w < warps) order_shared[w * bins + b] = sum;
      sum += c[w];
    }
    total[b] = sum;
  }
  if (CTAS > 1)
    cluster.sync();
  else
    __syncthreads();
  uint32_t carry = 0;   // rows of the experts before this pass's
  for (int b0 = 0; b0 < bins; b0 += threads) {
    const int b = b0 + threadIdx.x;
    uint32_t before = 0, all = 0, c[CTAS];
    if (b < bins) {
#pragma unroll
      for (int r = 0; r < CTAS; ++r) c[r] = CTAS > 1 ? cluster.map_shared_rank(total, r)[b] : total[b];
#pragma unroll
      for (int r = 0; r < CTAS; ++r) {
        before += r < rank ? c[r] : 0;
        all += c[r];
      }
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
#pragma unroll
    for (int w = 0; w < ORDER_WARPS; ++w) {
      const uint32_t c = w < warps ? warp_total[w] : 0;
      first += w < warp ? c : 0;
      carry += c;
    }
    if (b0 + threads < bins) __syncthreads();
    if (b < bins) {
      start[b] = first + before;
      if (rank == 0) offsets[b] = static_cast<int32_t>(first);   // the bin behind the experts begins where they end
    }
  }
  if (CTAS > 1) cluster.barrier_arrive();   // this CTA has read the others' counts
  __syncthreads();                          // and `start` is whole
  for (int b = lane; b < bins; b += 32) mine[b] += start[b];
  __syncwarp();
  const int bits = 32 - __clz(experts);   // of the largest number, the dropped slots'
  for (int64_t i0 = begin; i0 < end; i0 += 32 * ORDER_AHEAD) {
    if (per_warp > 32 * ORDER_AHEAD) load(i0);
#pragma unroll
    for (int u = 0; u < ORDER_AHEAD; ++u) {
      if (i0 + 32 * u >= end) break;
      unsigned same = __ballot_sync(0xffffffffu, bin[u] >= 0);   // the lanes with this one's expert, by a vote for each bit of its number
      for (int k = 0; k < bits; ++k) {
        const bool one = bin[u] >> k & 1;
        const unsigned ones = __ballot_sync(0xffffffffu, one);
        same &= one ? ones : ~ones;
      }
      const int place = __popc(same & ((1u << lane) - 1));
      uint32_t row = 0;
      if (bin[u] >= 0) row = mine[bin[u]] + place;
      __syncwarp();
      if (bin[u] >= 0) {
        if (place == 0) mine[bin[u]] = row + __popc(same);
        row_of[i0 + 32 * u + lane] = static_cast<int32_t>(bin[u] < experts ? row : ~row);
      }
      __syncwarp();
    }
  }
  if (CTAS > 1) cluster.barrier_wait();   // nobody reads this CTA's counts any more
}

// ------------------------------------------------------------------ there and back
// Bound by the rows' bytes. Where rows are whole numbers of aligned 16-byte vectors a thread has one of a token, or some, and goes through the token's
// rows, several of whose loads or stores are under way at once. Other rows go element by element: a warp has a piece of a row, a lane every 32nd
// element of it, so that an access is one stretch of memory whatever it starts at. Whole vectors of which each is put together from the two that it
// straddles cost more in instructions than they save in accesses: the gradient of 2000 x 7169 x 6 in bf16 takes 132 us that way, 102 so, that of
// 3001 x 1283 x 3 in fp32 32 and 23, writing the rows 48 and 44, 15 and 12.
// Aligned, 4096 x 7168 x 8 in bf16: there 91 us (5.8 TB/s), back 87 (6.1), its gradient 159 (6.3); 205 with a team of warps for a token, whose parts of
// the weights' gradient meet behind barriers.
constexpr int ROWS_THREADS = 256;
constexpr int MAX_ROW = 1 << 29;   // elements, so that a piece beyond the last is a number of 32 bits too

// The rows of a token are written from one read of it. `scale`: `groups` numbers of a token that go with its rows, or null
template <typename Index>
__global__ void __launch_bounds__(ROWS_THREADS)
    permute_rows_kernel(const char* x, int64_t pitch, uint4* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups, int64_t tokens,
                        int k, int64_t row_vecs) {
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  const Index vecs = static_cast<Index>(row_vecs), items = static_cast<Index>(tokens) * vecs;
  for (Index i = blockIdx.x * static_cast<Index>(ROWS_THREADS) + threadIdx.x; i < items; i += static_cast<Index>(gridDim.x) * ROWS_THREADS) {
    const Index token = i / vecs;
    const int64_t t = token, c = i - token * vecs;
    const uint4 v = reinterpret_cast<const uint4*>(x + t * pitch)[c];
    for (int j = 0; j < k; ++j) {
      const int32_t r = row_of[t * k + j];
      const int64_t to = r < 0 ? ~r : r;
      if (to >= slots) continue;   // no order that this library made
      rows[to * row_vecs + c] = r < 0 ? make_uint4(0, 0, 0, 0) : v;
      for (int64_t g = c; g < groups; g += row_vecs) row_scale[to * groups + g] = r < 0 ? 0.f : scale[t * groups + g];
    }
  }
}
template <typename E, int U>
__global__ void __launch_bounds__(ROWS_THREADS)
    permute_elements_kernel(const char* x, int64_t pitch, E* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups, int64_t tokens,
                            int k, int H) {
  grid_wait();
  grid_release();
  constexpr int WARPS = ROWS_THREADS / 32;
  const int64_t slots = tokens * k;
  const int lane = threadIdx.x & 31, pieces = (H + 32 * U - 1) / (32 * U);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5); i < tokens * pieces; i += static_cast<int64_t>(gridDim.x) * WARPS) {
    const int64_t t = i / pieces;
    const int piece = static_cast<int>(i - t * pieces), e0 = piece * 32 * U + lane;
    const E* const from = reinterpret_cast<const E*>(x + t * pitch) + e0;
    E v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = e0 + 32 * u < H ? from[32 * u] : E{};
    for (int j = 0; j < k; ++j) {
      const int32_t r = row_of[t * k + j];
      const int64_t to = r < 0 ? ~r : r;
      if (to >= slots) continue;
      E* const row = rows + to * H + e0;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (e0 + 32 * u < H) row[32 * u] = r < 0 ? E{} : v[u];
      for (int64_t g = piece * 32 + lane; g < groups; g += pieces * 32) row_scale[to * groups + g] = r < 0 ? 0.f : scale[t * groups + g];
    }
  }
}

template <typename T>
struct Values;
template <>
struct Values<__nv_bfloat16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void get(const uint4& q, float (&f)[8]) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(p[j]), f[2 * j + 1] = __high2float(p[j]);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[8]) {
    uint4 q;
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    return q;
  }
};
template <>
struct Values<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void get(const uint4& q, float (&f)[4]) {
    f[0] = __uint_as_float(q.x), f[1] = __uint_as_float(q.y), f[2] = __uint_as_float(q.z), f[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 put(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// out[t] = sum over j of w[t][j] * rows[row_of[t][j]], in 32 bits and in the order of j; w null: a plain sum. A dropped slot's row is not read.
// J rows are under way at once, of N vectors of a thread.
template <typename T, typename Index, int J, int N>
__global__ void __launch_bounds__(ROWS_THREADS)
    unpermute_rows_kernel(const T* rows, int64_t pitch, const float* w, const int32_t* row_of, T* out, int64_t tokens, int k, int H) {
  constexpr int V = Values<T>::V;
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  const Index vecs = H / V, each = (vecs + N - 1) / N, items = static_cast<Index>(tokens) * each;
  for (Index i = blockIdx.x * static_cast<Index>(ROWS_THREADS) + threadIdx.x; i < items; i += static_cast<Index>(gridDim.x) * ROWS_THREADS) {
    const Index token = i / each, c0 = i - token * each;
    const int64_t t = token;
    float acc[N][V] = {};
    for (int j0 = 0; j0 < k; j0 += J) {
      uint4 q[J][N];
      float by[J];
      bool there[J];
#pragma unroll
      for (int u = 0; u < J; ++u) {
        const int32_t r = j0 + u < k ? row_of[t * k + j0 + u] : -1;
        there[u] = r >= 0 && r < slots;
        by[u] = w && there[u] ? w[t * k + j0 + u] : 1.f;
#pragma unroll
        for (int v = 0; v < N; ++v)
          if (there[u] && c0 + v * each < vecs) q[u][v] = reinterpret_cast<const uint4*>(rows + r * pitch)[c0 + v * each];
      }
#pragma unroll
      for (int u = 0; u < J; ++u) {
        if (!there[u]) continue;
#pragma unroll
        for (int v = 0; v < N; ++v) {
          float f[V];
          Values<T>::get(q[u][v], f);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[v][e] = fmaf(by[u], f[e], acc[v][e]);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < N; ++v)
      if (c0 + v * each < vecs) reinterpret_cast<uint4*>(out + t * H)[c0 + v * each] = Values<T>::put(acc[v]);
  }
}
// The same for rows that are no whole number of aligned vectors: a warp has U times 32 elements of a token, a lane every 32nd of them.
template <typename T, int J, int U>
__global__ void __launch_bounds__(ROWS_THREADS)
    unpermute_elements_kernel(const T* rows, int64_t pitch, const float* w, const int32_t* row_of, T* out, int64_t tokens, int k, int H) {
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  const int lane = threadIdx.x & 31, pieces = (H + 32 * U - 1) / (32 * U);
  constexpr int WARPS = ROWS_THREADS / 32;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5); i < tokens * pieces; i += static_cast<int64_t>(gridDim.x) * WARPS) {
    const int64_t t = i / pieces;
    const int e0 = static_cast<int>(i - t * pieces) * 32 * U + lane;
    float acc[U] = {};
    for (int j0 = 0; j0 < k; j0 += J) {
      T q[J][U];
      float by[J];
      bool there[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int32_t r = j0 + j < k ? row_of[t * k + j0 + j] : -1;
        there[j] = r >= 0 && r < slots;
        by[j] = w && there[j] ? w[t * k + j0 + j] : 1.f;
        const T* const from = rows + r * pitch + e0;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (there[j] && e0 + 32 * u < H) q[j][u] = from[32 * u];
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (there[j]) acc[u] = fmaf(by[j], static_cast<float>(q[j][u]), acc[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (e0 + 32 * u < H) out[t * H + e0 + 32 * u] = static_cast<T>(acc[u]);
  }
}

// What flows back through a weighted sum: drows[row_of[t][j]] = w[t][j] * dout[t] (zeros for a dropped slot, of which nothing is read) and
// dw[t][j] = <dout[t], rows[row_of[t][j]]>, either of them left out where its pointer is null. LANES lanes of a warp have a slot, so that nothing is joined but
// by shuffles; a token's slots lie in one CTA or two, whose L1 has the gradient that they share. N vectors of a lane are under way at once, or, where rows
// are no whole number of aligned vectors (VECTORS false), N elements.
template <typename T, bool VECTORS, int LANES, int N>
__global__ void __launch_bounds__(ROWS_THREADS)
    unpermute_rows_bwd_kernel(const T* dout, const T* rows, int64_t pitch, const float* w, const int32_t* row_of, T* drows, float* dw, int64_t tokens,
                              int k, int H) {
  using Piece = std::conditional_t<VECTORS, uint4, T>;
  constexpr int V = VECTORS ? Values<T>::V : 1, PER = ROWS_THREADS / LANES;
  grid_wait();
  grid_release();
  const int64_t slots = tokens * k;
  const int lane = threadIdx.x % LANES, pieces = H / V;
  for (int64_t s0 = static_cast<int64_t>(blockIdx.x) * PER; s0 < slots; s0 += static_cast<int64_t>(gridDim.x) * PER) {   // as often for every lane
    const int64_t s = s0 + threadIdx.x / LANES;
    const bool mine = s < slots;
    const int32_t r = mine ? row_of[s] : INT_MIN;
    const float by = mine ? w[s] : 0.f;
    const int64_t t = mine ? s / k : 0, at = r < 0 ? ~r : r;   // ~INT_MIN is no row either: it is the largest number
    const bool there = r >= 0 && r < slots, read = dw && there, write = drows && at < slots;
    const Piece* const d_row = reinterpret_cast<const Piece*>(dout + t * H);
    const Piece* const y_row = reinterpret_cast<const Piece*>(rows + (read ? r * pitch : 0));
    Piece* const to = reinterpret_cast<Piece*>(drows + (write ? at * H : 0));
    float acc = 0.f;
    if (read || write)
      for (int c0 = lane; c0 < pieces; c0 += LANES * N) {
        Piece d[N] = {}, y[N] = {};
#pragma unroll
        for (int v = 0; v < N; ++v) {
          const int c = c0 + v * LANES;
          if (c >= pieces || !there) continue;
          d[v] = d_row[c];
          if (read) y[v] = y_row[c];
        }
#pragma unroll
        for (int v = 0; v < N; ++v) {
          const int c = c0 + v * LANES;
          if (c >= pieces) continue;
          float f[V], g[V];
          if constexpr (VECTORS) {
            Values<T>::get(d[v], f);
            Values<T>::get(y[v], g);
          } else {
            f[0] = static_cast<float>(d[v]);
            g[0] = static_cast<float>(y[v]);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) acc = fmaf(f[e], g[e], acc);
          if (!write) continue;
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] = there ? by * f[e] : 0.f;
          if constexpr (VECTORS)
            to[c] = Values<T>::put(f);
          else
            to[c] = static_cast<T>(f[0]);
        }
      }
    if (!dw) continue;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0 && mine) dw[s] = there ? acc : 0.f;
  }
}

static int rows_grid(int64_t ctas, int per_sm) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(ctas < 1 ? 1 : ctas < cap ? ctas : cap);
}
static bool bad_slots(long long tokens, int k) { return tokens < 0 || k <= 0 || tokens > INT_MAX / k; }
static bool on(const void* p, long long pitch, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0 && pitch % bytes == 0; }
// 32-bit indices hold while a grid's last pass, beyond the last item, stays below 2^32
static bool small_index(int64_t items) { return items < (1ll << 31); }

template <typename Index, int CTAS>
static int launch_order_on(const void* idx, long long n, int experts, int32_t* row_of, int32_t* offsets, int warps, cudaStream_t stream) {
  constexpr auto kern = expert_order_kernel<Index, CTAS>;
  const int rc = allow_smem<kern>(order_smem(ORDER_WARPS, ORDER_MAX_EXPERTS));
  if (rc) return rc;
  if constexpr (CTAS > 8) {
    static OncePerDevice once;
    int dev = -1;
    B200_CUDA_OK(cudaGetDevice(&dev));
    const int rc = once.run(dev, [&]() -> int {
      B200_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
      return 0;
    });
    if (rc) return rc;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CTAS;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(CTAS);
  cfg.blockDim = dim3(32 * warps);
  cfg.dynamicSmemBytes = order_smem(warps, experts);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = CTAS > 1 ? 2 : 1;
  B200_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, static_cast<const Index*>(idx), static_cast<int64_t>(n), experts, row_of, offsets));
  return 0;
}
// One CTA up to 2048 slots (128 take 2.8 us, 2048 4.6 on one or sixteen), where a cluster's barriers cost as much as they share out: 4096 slots take 5.8 us so,
// 4.3 on sixteen CTAs.
template <typename Index>
static int launch_order(const void* idx, long long n, int experts, int32_t* row_of, int32_t* offsets, cudaStream_t stream) {
  // two batches of slots for a warp, and a thread for each expert
  const int64_t wanted = std::max((n + 63) / 64, static_cast<long long>(experts + 32) / 32);
  const int warps = n > 2048 ? ORDER_WARPS : static_cast<int>(std::min<int64_t>(wanted, ORDER_WARPS));
  return n > 2048 ? launch_order_on<Index, ORDER_CTAS>(idx, n, experts, row_of, offsets, warps, stream)
                  : launch_order_on<Index, 1>(idx, n, experts, row_of, offsets, warps, stream);
}

static void launch_permute_rows(const void* x, long long pitch, void* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups,
                                long long tokens, int k, long long bytes, cudaStream_t stream) {
  const int64_t vecs = bytes / 16, items = tokens * vecs;
  launch_dependent(small_index(items) ? permute_rows_kernel<unsigned> : permute_rows_kernel<int64_t>, rows_grid((items + ROWS_THREADS - 1) / ROWS_THREADS, 64),
                   ROWS_THREADS, 0, stream, static_cast<const char*>(x), static_cast<int64_t>(pitch), static_cast<uint4*>(rows), row_of, scale, row_scale, groups,
                   static_cast<int64_t>(tokens), k, vecs);
}
template <typename E, int U>
static void launch_permute_of(const void* x, long long pitch, void* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups,
                              long long tokens, int k, int H, cudaStream_t stream) {
  const int64_t warps = tokens * ((H + 32 * U - 1) / (32 * U));
  launch_dependent(permute_elements_kernel<E, U>, rows_grid((warps + ROWS_THREADS / 32 - 1) / (ROWS_THREADS / 32), 64), ROWS_THREADS, 0, stream,
                   static_cast<const char*>(x), static_cast<int64_t>(pitch), static_cast<E*>(rows), row_of, scale, row_scale, groups,
                   static_cast<int64_t>(tokens), k, H);
}
template <typename E>
static void launch_permute_elements(const void* x, long long pitch, void* rows, const int32_t* row_of, const float* scale, float* row_scale, int groups,
                                    long long tokens, int k, long long bytes, cudaStream_t stream) {
  const int H = static_cast<int>(bytes / sizeof(E));
  auto* const of = H <= 64 ? launch_permute_of<E, 2> : H <= 128 ? launch_permute_of<E, 4> : launch_permute_of<E, 8>;
  of(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, H, stream);
}
template <typename T, int J, int N>
static void launch_unpermute_of(const void* rows, long long pitch, const float* w, const int32_t* row_of, void* out, long long tokens, int k, int H,
                                cudaStream_t stream) {
  const int64_t items = tokens * ((H / Values<T>::V + N - 1) / N);
  launch_dependent(small_index(items) ? unpermute_rows_kernel<T, unsigned, J, N> : unpermute_rows_kernel<T, int64_t, J, N>,
                   rows_grid((items + ROWS_THREADS - 1) / ROWS_THREADS, 64), ROWS_THREADS, 0, stream, static_cast<const T*>(rows), static_cast<int64_t>(pitch),
                   w, row_of, static_cast<T*>(out), static_cast<int64_t>(tokens), k, H);
}
template <typename T, int J, int U>
static void launch_unpermute_elements(const void* rows, long long pitch, const float* w, const int32_t* row_of, void* out, long long tokens, int k, int H,
                                      cudaStream_t stream) {
  const int64_t warps = tokens * ((H + 32 * U - 1) / (32 * U));
  launch_dependent(unpermute_elements_kernel<T, J, U>, rows_grid((warps + ROWS_THREADS / 32 - 1) / (ROWS_THREADS / 32), 64), ROWS_THREADS, 0, stream,
                   static_cast<const T*>(rows), static_cast<int64_t>(pitch), w, row_of, static_cast<T*>(out), static_cast<int64_t>(tokens), k, H);
}
// Two vectors of a thread and up to four of their rows at once; eight rows of one vector where that is all the threads there are (one token of 4096
// and eight rows 2.1 us, 2.6 so; 4096 x 7168 of eight 95 us and 87).
template <typename T>
static void launch_unpermute(bool aligned, const void* rows, long long pitch, const float* w, const int32_t* row_of, void* out, long long tokens, int k, int H,
                             cudaStream_t stream) {
  const bool few = tokens * (static_cast<int64_t>(H) * static_cast<int64_t>(sizeof(T)) / 16) < static_cast<int64_t>(sm_count()) * 1024;
  auto* const of = !aligned ? (H <= 64 ? launch_unpermute_elements<T, 4, 2> : H <= 128 ? launch_unpermute_elements<T, 4, 4> : launch_unpermute_elements<T, 2, 8>)
                   : few    ? launch_unpermute_of<T, 8, 1>
                   : k <= 2 ? launch_unpermute_of<T, 2, 2>
                            : launch_unpermute_of<T, 4, 2>;
  of(rows, pitch, w, row_of, out, tokens, k, H, stream);
}
template <typename T, bool VECTORS, int LANES, int N>
static void launch_bwd_of(const void* dout, const void* rows, long long pitch, const float* w, const int32_t* row_of, void* drows, float* dw, long long tokens,
                          int k, int H, cudaStream_t stream) {
  constexpr int per = ROWS_THREADS / LANES;
  launch_dependent(unpermute_rows_bwd_kernel<T, VECTORS, LANES, N>, rows_grid((tokens * k + per - 1) / per, 64), ROWS_THREADS, 0, stream,
                   static_cast<const T*>(dout), static_cast<const T*>(rows), static_cast<int64_t>(pitch), w, row_of, static_cast<T*>(drows), dw,
                   static_cast<int64_t>(tokens), k, H);
}
// As few lanes as have a row in one go, up to a warp.
template <typename T>
static void launch_unpermute_bwd(bool aligned, const void* dout, const void* rows, long long pitch, const float* w, const int32_t* row_of, void* drows, float* dw,
                                 long long tokens, int k, int H, cudaStream_t stream) {
  const int vecs = H / Values<T>::V;
  auto* const of = !aligned     ? (H <= 64 ? launch_bwd_of<T, false, 32, 2> : launch_bwd_of<T, false, 32, 8>)
                   : vecs <= 8  ? launch_bwd_of<T, true, 8, 1>
                   : vecs <= 32 ? launch_bwd_of<T, true, 8, 4>
                   : vecs <= 64 ? launch_bwd_of<T, true, 16, 4>
                                : launch_bwd_of<T, true, 32, 4>;
  of(dout, rows, pitch, w, row_of, drows, dw, tokens, k, H, stream);
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
  if (bad_slots(tokens, k) || row_bytes <= 0 || (elem != 1 && elem != 2 && elem != 4) || row_bytes % elem ||
      row_bytes / elem > MAX_ROW) return B200_ERR_BAD_ARG;
  if (!scale != !row_scale || (scale ? groups <= 0 : groups != 0)) return B200_ERR_BAD_ARG;
  if (!tokens) return 0;
  if (!x || !rows || !row_of || !on(x, pitch, elem) || !on(rows, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto* const launch = on(x, pitch, 16) && on(rows, row_bytes, 16) ? launch_permute_rows
                       : elem == 4                                 ? launch_permute_elements<uint32_t>
                       : elem == 2                                 ? launch_permute_elements<uint16_t>
                                                                   : launch_permute_elements<uint8_t>;
  launch(x, pitch, rows, row_of, scale, row_scale, groups, tokens, k, row_bytes, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

// out [tokens][H] = sums over the k rows of each token, weighted by w [tokens][k] unless null; rows lie `pitch` elements apart. bf16, or fp32.
int b200_unpermute_rows(const void* rows, long long pitch, const float* w, const int* row_of, void* out, long long tokens, int k, int H, int fp32,
                        void* stream) {
  ensure_context();
  if (bad_slots(tokens, k) || H <= 0 || H > MAX_ROW) return B200_ERR_BAD_ARG;
  if (!tokens) return 0;
  const int elem = fp32 ? 4 : 2;
  if (!rows || !row_of || !out || !on(rows, 0, elem) || !on(out, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = on(rows, pitch * elem, 16) && on(out, static_cast<long long>(H) * elem, 16);
  (fp32 ? launch_unpermute<float> : launch_unpermute<__nv_bfloat16>)(wide, rows, pitch, w, row_of, out, tokens, k, H, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

// The gradients of that weighted sum; drows or dw may be null, rows where dw is.
int b200_unpermute_rows_bwd(const void* dout, const void* rows, long long pitch, const float* w, const int* row_of, void* drows, float* dw,
                            long long tokens, int k, int H, int fp32, void* stream) {
  ensure_context();
  if (bad_slots(tokens, k) || H <= 0 || H > MAX_ROW) return B200_ERR_BAD_ARG;
  if (!tokens || (!drows && !dw)) return 0;
  const int elem = fp32 ? 4 : 2;
  if (!dout || !w || !row_of || (dw && !rows) || !on(dout, 0, elem) || !on(rows, 0, elem) || !on(drows, 0, elem)) return B200_ERR_BAD_ARG;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = on(dout, static_cast<long long>(H) * elem, 16) && on(drows, 0, 16) && (!dw || on(rows, pitch * elem, 16));
  (fp32 ? launch_unpermute_bwd<float> : launch_unpermute_bwd<__nv_bfloat16>)(wide, dout, rows, pitch, w, row_of, drows, dw, tokens, k, H, s);
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // extern "C"
