// What the attention kernels share: which keys a query sees, tiles of [batch][token][head][element] tensors by TMA, products
// whose first operand is in tensor memory.
//
// Query i sees key j where j <= i, and with a window also i - j < window or j < sinks; a sequence of the batch has length[b] tokens,
// and rows behind them are zeros, in the output and in the gradients. Since j <= i, a query in front of the length sees no key behind it.
#pragma once
#include "gemm_tcgen05.cuh"
#include "pair_math.cuh"

namespace b200 {

using bf16 = __nv_bfloat16;

constexpr int ATT_TILE = 128;                         // rows of a tile that stays, lanes of tensor memory
constexpr int ATT_BOX = 64;                           // rows of one TMA box
constexpr int ATT_THREADS = 384;                      // two groups of four warps that compute; warp 8 loads, warp 9 issues products
constexpr float ATT_LOG2E = 1.4426950408889634f;

struct AttnShape {
  int B, S, nq, nkv;   // batch, tokens, heads of q, heads of k and v
  int G;               // heads of q that share one of k and v
  int rows;            // S rounded up to whole tiles: the pitch of lse and delta
  int window, sinks;   // window 0: all keys up to the query (then sinks is 0)
  const int* lengths;  // [B], or null: all sequences have S tokens
  float scale;
};

__device__ __forceinline__ int sequence_length(const AttnShape& s, int b) { return s.lengths ? min(max(s.lengths[b], 0), s.S) : s.S; }

__device__ __forceinline__ void tma_load_4d(uint32_t dst_smem, const CUtensorMap* m, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst_smem),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// ROWS x HD elements of one head, as HD / 64 columns of 128-byte rows (ROWS * 128 bytes each) in the 128-byte swizzle; rows beyond the
// tensor are zeros.
template <int HD, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* m, int b, int head, int row, uint32_t bar) {
#pragma unroll
  for (int c = 0; c < HD / 64; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; r += ATT_BOX) tma_load_4d(dst + c * ROWS * 128 + r * 128, m, c * 64, head, row + r, b, bar);
}
// Descriptors of such a tile for 16 elements of the reduction: of a row's elements (K-major) ...
template <int ROWS>
__device__ __forceinline__ uint64_t desc_rows(uint32_t tile, int k) {
  return make_smem_desc_sw128(tile + (k >> 2) * ROWS * 128 + (k & 3) * 32, 16, 1024);
}
// ... or over its rows (MN-major)
template <int ROWS>
__device__ __forceinline__ uint64_t desc_cols(uint32_t tile, int k) {
  return make_smem_desc_sw128(tile + k * 2048, ROWS * 128, 1024);
}
// Rows from `first` on of a tile become zeros: values that are not finite behind a sequence's end would reach its rows through products with
// zero. By a whole warp, in front of the products that read the tile.
template <int HD, int ROWS>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first) {
  const int lane = threadIdx.x & 31;
  for (int i = first * 8 + lane; i < ROWS * 8; i += 32)
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) st_shared_v4(tile + c * ROWS * 128 + i * 16, 0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// D[tmem] (+)= A[tmem] * B[smem], A as packed pairs of bf16: 16 elements of the reduction are 8 columns.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_unit(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Pair pair_of(uint32_t a, uint32_t b) { return Pair(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ void ld_shared_pairs(uint32_t addr, Pair& a, Pair& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a.bits), "=l"(b.bits) : "r"(addr) : "memory");
}

// What all roles of a CTA share: its tensor memory, barriers and the flag that one of its waits has given up.
struct AttnCta {
  uint32_t smem, bars, tmem;   // aligned tiles; barriers behind them; tensor memory's first column
  volatile int* abort_flag;
  int* err_word;
  __device__ __forceinline__ uint32_t bar(int i) const { return bars + 8u * i; }
  __device__ __forceinline__ bool wait(int i, uint32_t parity, int code) const {
    return mbar_wait_bounded(bar(i), parity, abort_flag, err_word, code, GEMM_WAIT_LIMIT_NS);
  }
};
constexpr int ATT_BAR_BYTES = 256;   // barriers, the slot of tensor memory's address and the flag

// Barrier i is completed by count(i) arrivals. Tensor memory is the last warp's. Every thread calls this.
template <int TILE_BYTES, int BARS, class Count>
__device__ __forceinline__ AttnCta attn_begin(uint8_t* smem_raw, int* err_word, Count count) {
  static_assert(BARS * 8 + 16 <= ATT_BAR_BYTES, "more barriers than room");
  AttnCta c;
  c.smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  c.bars = c.smem + TILE_BYTES;
  uint8_t* at = smem_raw + (c.bars - smem_u32(smem_raw)) + BARS * 8;
  c.abort_flag = reinterpret_cast<volatile int*>(at + 8);
  c.err_word = err_word;
  if (threadIdx.x == 0) {
    for (int i = 0; i < BARS; ++i) mbar_init(c.bar(i), count(i));
    *c.abort_flag = 0;
    fence_barrier_init();
  }
  if (threadIdx.x / 32 == ATT_THREADS / 32 - 1) {
    tmem_alloc(c.bars + BARS * 8, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  c.tmem = *reinterpret_cast<volatile uint32_t*>(at);
  return c;
}
__device__ __forceinline__ void attn_end(const AttnCta& c) {
  tc_fence_before();
  __syncthreads();
  if (*c.abort_flag) {   // copies that may still be in flight land before shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  if (threadIdx.x / 32 == ATT_THREADS / 32 - 1) {
    tc_fence_after();
    tmem_dealloc(c.tmem, 512);
  }
}

}  // namespace b200
