// What the attention kernels share: which keys a query sees, tiles of [batch][token][head][element] tensors by TMA, products
// whose first operand is in tensor memory.
//
// Query i sees key j where j <= i, and with a window also i - j < window or j < sinks; a sequence of the batch has length[b] tokens,
// and rows behind them are zeros, in the output and in the gradients. Since j <= i, a query in front of the length sees no key behind it.
#pragma once
#include <cuda_fp8.h>

#include "divisor.h"
#include "gemm_tcgen05.cuh"
#include "pair_math.cuh"

namespace b200 {

using bf16 = __nv_bfloat16;

constexpr int ATT_TILE = 128;                         // rows of a tile that stays, lanes of tensor memory
constexpr int ATT_BOX = 64;                           // rows of one TMA box
// Warps of a CTA: COMPUTE of them compute, as many for each quarter of a tile's rows; behind them one that loads and one that issues products, a thread
// each, and one that clears what lies behind a sequence's end.
template <int COMPUTE>
struct AttnRoles {
  static constexpr int LOAD = COMPUTE, MMA = COMPUTE + 1, ZERO = COMPUTE + 2, THREADS = 32 * (COMPUTE + 3);
};
constexpr float ATT_LOG2E = 1.4426950408889634f;

struct AttnShape {
  int B, S, nq, nkv;   // batch, tokens, heads of q, heads of k and v
  int G;               // heads of q that share one of k and v
  int rows;            // S rounded up to whole tiles: the pitch of lse and delta
  int window, sinks;   // window 0: all keys up to the query (then sinks is 0)
  const int* lengths;  // [B], or null: all sequences have S tokens
  float scale;
  Divisor by_G, by_nq, by_nkv, by_heads_q, by_heads_kv;   // heads_q: B * nq
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
// Descriptors of such a tile: of 16 of a row's elements (K-major), or over 16 of its rows (MN-major). The high word is the same for all tiles; the low
// one is the address, to which the steps of a reduction are added. One elected thread issues all products of a CTA: beside busy warps, of which its scheduler has four
// more, its instructions are what products wait for (64 clocks each alone; 114 so beside 16 warps of nothing but multiplications, 860 with descriptors put together
// for each product, 1460 where a lane is chosen by its number).
template <int ROWS, bool COLS>
struct TileDesc {
  static constexpr uint32_t HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);   // 8 rows to the next group; version; 128-byte swizzle
  static constexpr uint32_t LEAD = COLS ? ROWS * 128 >> 4 : 1;              // COLS: from 64 columns to the next
  __device__ static __forceinline__ uint32_t low(uint32_t tile) { return (tile >> 4) | (LEAD << 16); }
  __device__ static constexpr uint32_t step(int k) { return (COLS ? k * 2048 : (k >> 2) * ROWS * 128 + (k & 3) * 32) >> 4; }
};
// Rows from `first` on of a tile become zeros: values that are not finite behind a sequence's end would reach its rows through products with
// zero. By a whole warp, in front of the products that read the tile, whose issuing thread waits for `done`.
template <int HD, int ROWS>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first, uint32_t done) {
  const int lane = threadIdx.x & 31;
  for (int i = first * 8 + lane; i < ROWS * 8; i += 32)
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) st_shared_v4(tile + c * ROWS * 128 + i * 16, 0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(done);
}

// D[tmem] (+)= A[smem] * B[smem], descriptors in two words
template <bool ADD>
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_low, uint32_t a_high, uint32_t b_low, uint32_t b_high, uint32_t idesc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 a, b;\n"
      "mov.b64 a, {%1, %2};\n"
      "mov.b64 b, {%3, %4};\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n"
      "}\n" ::"r"(d),
      "r"(a_low), "r"(a_high), "r"(b_low), "r"(b_high), "r"(idesc), "n"(ADD)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], A as packed pairs of bf16: 16 elements of the reduction are 8 columns.
template <bool ADD>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b_low, uint32_t b_high, uint32_t idesc) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 b;\n"
      "mov.b64 b, {%2, %3};\n"
      "setp.ne.b32 p, %5, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b_low), "r"(b_high), "r"(idesc), "n"(ADD)
      : "memory");
}
// A tile's rows times another's, elements of both reduced
template <int HD>
__device__ __forceinline__ void multiply_rows(uint32_t d, uint32_t a_tile, uint32_t b_tile) {
  using D = TileDesc<ATT_TILE, false>;
  constexpr uint32_t idesc = make_instr_desc(1, 1, ATT_TILE, ATT_TILE, 0, 0);
  const uint32_t a = D::low(a_tile), b = D::low(b_tile);
  umma_ss<false>(d, a, D::HIGH, b, D::HIGH, idesc);
#pragma unroll
  for (int k = 1; k < HD / 16; ++k) umma_ss<true>(d, a + D::step(k), D::HIGH, b + D::step(k), D::HIGH, idesc);
}
// d (+)= operand in tensor memory times rows of a tile, 16 rows a step. Its 128 columns are as packed pairs in the first half of each GROUP of columns.
template <int HD, int GROUP>
__device__ __forceinline__ void multiply_step(uint32_t d, uint32_t a, uint32_t b_low, int k, bool add) {
  using D = TileDesc<ATT_TILE, true>;
  constexpr uint32_t idesc = make_instr_desc(1, 1, ATT_TILE, HD, 0, 1);
  const uint32_t at = a + k / (GROUP / 16) * GROUP + k % (GROUP / 16) * 8;
  if (add)
    umma_ts<true>(d, at, b_low + D::step(k), D::HIGH, idesc);
  else
    umma_ts<false>(d, at, b_low + D::step(k), D::HIGH, idesc);
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
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32(taddr, r); }
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld_32x16(taddr, r); }
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st_32x16(taddr, r); }
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[8]) { tmem_st_32x8(taddr, r); }
// 32 rows x 64 elements from shared memory; rows beyond the tensor are left out.
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* m, uint32_t src_smem, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(src_smem), "r"(x),
               "r"(y), "r"(z), "r"(w)
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_unit(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Pair pair_of(uint32_t a, uint32_t b) { return Pair(__uint_as_float(a), __uint_as_float(b)); }

// 2^x of both where x <= 120, in float units beside the one for exponentials, which has a quarter of their rate: 2^n p(f) with n the integer nearest to
// x, f = x - n and p the cubic whose largest relative error on [-1/2, 1/2] is the least (7.5e-5, by Remez' exchange; probabilities are rounded to bf16
// behind it, 3.9e-3). Below -127 it is zero.
__device__ __forceinline__ Pair exp2_cubic(Pair x) {
  constexpr float BIG = 12582912.f;   // 1.5 * 2^23: a sum with it has the integer in its low bits
  float a, b;
  x.to(a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  const Pair y(a, b), t = y + both(BIG), f = fma2(t + both(-BIG), both(-1.f), y);
  const Pair p = fma2(fma2(fma2(both(0.0551716685f), f, both(0.242611125f)), f, both(0.693260968f)), f, both(0.999928057f));
  t.to(a, b);
  return p * pair_of((__float_as_uint(a) << 23) + 0x3F800000u, (__float_as_uint(b) << 23) + 0x3F800000u);
}
// The same of x by the unit, or of every fourth pair of a row (number e / 2) in float units, where the unit bounds a phase: the gradients' kernels take
// 234 and 167 us for 245 and 171 over 4096 tokens of 32 heads, 564 and 388 for 580 and 400 over 16384 with a window of 1024; with every second pair 238 and 170. The forward pass gains nothing by it.
__device__ __forceinline__ void exp2_pair(int e, Pair x, float& a, float& b) {
  if (e / 2 % 4 == 3) {
    exp2_cubic(x).to(a, b);
  } else {
    x.to(a, b);
    a = exp2_unit(a), b = exp2_unit(b);
  }
}
// The largest of three, NaN if there is one
__device__ __forceinline__ float most_of(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Bits 0 to n - 1, none or all of a word where n is outside [0, 32]
__device__ __forceinline__ uint32_t bits_below(int n) {
  uint32_t r;
  asm("shl.b32 %0, 1, %1;" : "=r"(r) : "r"(max(n, 0)));   // PTX: zero from 32 on
  return r - 1u;
}
// Which of 32 columns a row sees: up to `last`, from `first` on or below `sinks`. A bit each, so that a tile on a border costs two instructions for an element:
// with the three comparisons in its place such a tile of the forward pass took 6000 clocks beside 3000.
__device__ __forceinline__ uint32_t columns_seen(int first, int last, int sinks) { return bits_below(last + 1) & (~bits_below(first) | bits_below(sinks)); }

// Two packed bf16, those of columns 2 k and 2 k + 1, where they are seen, else zeros
__device__ __forceinline__ uint32_t seen_pair(uint32_t packed, uint32_t seen, int k) {
  return packed & ((seen >> (2 * k) & 1 ? 0xFFFFu : 0u) | (seen >> (2 * k + 1) & 1 ? 0xFFFF0000u : 0u));
}

// What the rounding of out to bf16 leaves, as e5m2 of 2^12 times it: delta, a sum over out that the gradients of scores lie beside, is made of both. Of out
// alone it is off by 2^-9 of its terms, as much as the gradients' own rounding, and dq and dk of a few keys a row by 2^-8.2 in the mean instead of 2^-8.7.
constexpr float REST_SCALE = 4096.f;
__device__ __forceinline__ uint32_t rest_of(const float (&f)[4], uint32_t packed01, uint32_t packed23) {
  const float2 a = make_float2((f[0] - __uint_as_float(packed01 << 16)) * REST_SCALE, (f[1] - __uint_as_float(packed01 & 0xFFFF0000u)) * REST_SCALE);
  const float2 b = make_float2((f[2] - __uint_as_float(packed23 << 16)) * REST_SCALE, (f[3] - __uint_as_float(packed23 & 0xFFFF0000u)) * REST_SCALE);
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E5M2)) | (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E5M2)) << 16);
}
__device__ __forceinline__ float2 rest_pair(uint32_t codes) {   // of the low two bytes
  const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes), __NV_E5M2);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
  return make_float2(f.x * (1.f / REST_SCALE), f.y * (1.f / REST_SCALE));
}

// What the rounding of two numbers to bf16 left, in bf16; nothing of an infinity
__device__ __forceinline__ uint32_t left_of(float a, float b, uint32_t packed) {
  const float x = __uint_as_float(packed << 16), y = __uint_as_float(packed & 0xFFFF0000u);
  return pack_bf16x2(x == a ? 0.f : a - x, y == b ? 0.f : b - y);
}

// Whether `mine` is true for any thread of two warps that meet at barrier `id`
__device__ __forceinline__ bool any_of_64(int id, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %2, 0;\n"
      "barrier.cta.red.or.pred q, %1, 64, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"(id), "r"(static_cast<uint32_t>(mine))
      : "memory");
  return r;
}
__device__ __forceinline__ void meet_64(int id) { asm volatile("barrier.cta.sync %0, 64;" ::"r"(id) : "memory"); }

// A warp's way out: 32 rows of 32 elements (or 16) in shared memory (in the 64-byte swizzle, or plain), from there to the tensor by TMA. From registers 16 bytes of
// each of 32 rows take the memory pipeline 32 turns a store, of a tile of dk and dv 6000 clocks, and what is spilled waits behind them.
struct RowsOut {
  uint32_t slab;
  __device__ __forceinline__ void free() const {   // of the store before
    if ((threadIdx.x & 31) == 0) tma_store_wait_read<0>();
    __syncwarp();
  }
  template <int WORDS>   // of this lane's row
  __device__ __forceinline__ void put(const uint32_t (&w)[WORDS]) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < WORDS; e += 4)
      st_shared_v4(slab + lane * WORDS * 4 + ((WORDS == 16 ? e / 4 ^ (lane >> 1 & 3) : e / 4) << 4), w[e], w[e + 1], w[e + 2], w[e + 3]);
  }
  __device__ __forceinline__ void out(const CUtensorMap* m, int x, int head, int row, int b) const {
    fence_proxy_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) == 0) {
      tma_store_4d(m, slab, x, head, row, b);
      tma_store_commit();
    }
  }
};

// What all roles of a CTA share: barriers and the flag that one of its waits has given up. It has all of tensor memory, from column 0 on.
struct AttnCta {
  uint32_t smem, bars;   // aligned tiles; barriers behind them
  volatile int* abort_flag;
  int* err_word;
  __device__ __forceinline__ uint32_t bar(int i) const { return bars + 8u * i; }
  // `steps`: of a walk that may pass meanwhile, each of which has the limit that a wait for one has (who waits for a single one of them ends with a stuck CTA
  // all the same, by the flag)
  __device__ __forceinline__ bool wait(int i, uint32_t parity, int code, uint32_t steps = 1) const {
    // Polled: a thread that is suspended for a time comes back later, 5 % of the forward pass and of the gradients
    const uint32_t at = bar(i);
    uint64_t t0 = 0;
    for (uint32_t spins = 0;; ++spins) {
      uint32_t done;
      asm volatile(
          "{\n"
          ".reg .pred P;\n"
          "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n"
          "selp.u32 %0, 1, 0, P;\n"
          "}\n"
          : "=r"(done)
          : "r"(at), "r"(parity)
          : "memory");
      if (done) return true;
      if ((spins & 1023) == 1023) {
        if (*abort_flag) return false;
        const uint64_t t = globaltimer_ns();
        if (!t0) t0 = t;
        if (t - t0 > GEMM_WAIT_LIMIT_NS * steps) {
          *abort_flag = 1;
          if (err_word) atomicCAS(err_word, 0, code);
          return false;
        }
      }
    }
  }
};
constexpr int ATT_BAR_BYTES = 256;   // barriers, the slot of tensor memory's address and the flag

// Barrier i is completed by count(i) arrivals. Tensor memory is the issuing warp's. Every thread calls this.
template <class Roles, int TILE_BYTES, int BARS, class Count>
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
  if (threadIdx.x / 32 == Roles::MMA) {
    tmem_alloc(c.bars + BARS * 8, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  return c;
}
template <class Roles>
__device__ __forceinline__ void attn_end(const AttnCta& c) {
  tc_fence_before();
  __syncthreads();
  if (*c.abort_flag) {   // copies that may still be in flight land before shared memory is released
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  if (threadIdx.x / 32 == Roles::MMA) {
    tc_fence_after();
    tmem_dealloc(0, 512);
  }
}

}  // namespace b200
