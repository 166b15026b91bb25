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
// The update takes the moments of 32 bits, before they are rounded. Each operation on what is held is rounded by itself (no fused multiply-adds, IEEE's
// root and reciprocal), so that a step's codes do not depend on how a compiler contracts: a neighbouring code is 12 % away.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "b200ops.h"
#include "dependent_launch.cuh"
#include "host_util.h"
#include "pair_math.cuh"

namespace b200 {

constexpr int ADAMW_BLOCK = 256;   // elements of a warp's pass, eight of a lane
// With 8-bit moments there are 410 instructions of a warp for a block of it, and latencies between them, beside little memory: small CTAs, which end and
// start one by one, and registers for sixteen of them on an SM. 218 M bf16 parameters take 393 us a pass over some passes (5.6 TB/s; without rounding to codes
// at all 1 % less), 101 M with a master copy 265 (6.1); over 2000 passes in turn, which draw the clock from 1965 down to 1660 and 1490 MHz, 432 and 270. Each
// of these beside 388 and 271 of its own run: CTAs of 128 threads 440 and 298, 14 CTAs (72 registers) 403 and 281, blocks copied ahead into
// shared memory 449 and 346, nothing ahead 415 and 285.
constexpr int adamw_threads(int bits) { return bits == 8 ? 64 : 256; }
constexpr int adamw_ctas(int bits) { return bits == 8 ? 16 : 3; }        // of an SM at least
constexpr int adamw_pass(int bits) { return adamw_threads(bits) * 8; }   // elements of a CTA's pass
constexpr uint32_t DITHER_ELEMENT = 0xC13FA9A9u, DITHER_STEP = 0x91E10DA5u;

struct AdamwEntry {
  B200AdamwTensor t;
  uint32_t first;          // the tensor's first CTA
  uint32_t places;         // how a lane's elements lie (Places)
};
// The step's numbers, those of the float units twice: an instruction that works on two elements takes both.
struct AdamwNumbers {
  float2 beta1, rest1, minus_beta2, minus_rest2, minus_lr1, minus_root2, eps, grad_scale;   // rest: 1 - beta; lr1 = lr / (1 - b1^t); root2 = 1 / sqrt(1 - b2^t)
  float2 one;    // products are added as multiples of it: a product and an addition the assembler makes a fused multiply-add of, whatever their roundings are called
  uint32_t dither;
  int zero_grad;
  int careful;   // eps is so small that roots of the least numbers count beside it
};
// A launch's parameters are 32764 bytes at most.
template <int N>
struct AdamwTable {
  AdamwEntry e[N];
  AdamwNumbers a;
  int count;
  int chunk;        // elements of a CTA, a multiple of its pass
};
constexpr int ADAMW_MOST = 400;
static_assert(sizeof(AdamwTable<ADAMW_MOST>) <= 32764, "parameters of a launch");

// A lane's eight elements of a block of 256:
//  ALIGNED  eight in a row, where all that the step reads and writes of a tensor lies on 16-byte boundaries (8 for codes); they move as vectors.
//  STRIDED  every 32nd, whatever the tensors start at: a warp's access is one piece of memory. 40 M bf16 parameters and 8-bit moments in buffers
//           without padding take 125 us so, 70 aligned; 184 with eight in a row read one by one, 164 with vectors between a block's two ends.
//  LAST     the same in a tensor's last block, with zeros beyond its end.
enum Places { ALIGNED, STRIDED, LAST };
template <Places HOW>
struct Lane {
  uint32_t first, n;      // its first element, from the chunk's beginning, and the chunk's elements
  __device__ __forceinline__ Lane(uint32_t block, uint32_t n_) {
    const uint32_t lane = threadIdx.x & 31;
    n = n_;
    first = HOW == ALIGNED ? block + 8 * lane : block + lane;
  }
  // element j: how far behind the first
  __device__ __forceinline__ uint32_t step(int j) const { return HOW == ALIGNED ? j : 32 * j; }
  __device__ __forceinline__ bool has(int j) const { return HOW != LAST || first + 32 * j < n; }
  __device__ __forceinline__ bool row() const { return HOW == ALIGNED; }
};

template <typename T>
struct Raw8 {   // eight elements as they come from memory
  uint4 q[sizeof(T) / 2];
  __device__ __forceinline__ void to(float (&f)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(q);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[2 * j] = __low2float(h[j]), f[2 * j + 1] = __high2float(h[j]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 w = q[h % (sizeof(T) / 2)];
        f[4 * h] = __uint_as_float(w.x), f[4 * h + 1] = __uint_as_float(w.y), f[4 * h + 2] = __uint_as_float(w.z), f[4 * h + 3] = __uint_as_float(w.w);
      }
    }
  }
  __device__ __forceinline__ void from(const float (&f)[8]) {
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(q);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        q[h % (sizeof(T) / 2)] = make_uint4(__float_as_uint(f[4 * h]), __float_as_uint(f[4 * h + 1]), __float_as_uint(f[4 * h + 2]), __float_as_uint(f[4 * h + 3]));
    }
  }
};
template <>
struct Raw8<uint8_t> {
  uint2 q;
};

template <typename T, Places HOW>
__device__ __forceinline__ void load(Raw8<T>& raw, const T* p, const Lane<HOW>& l) {
  using Element = std::conditional_t<sizeof(T) == 4, uint32_t, std::conditional_t<sizeof(T) == 2, uint16_t, uint8_t>>;
  using Vector = std::conditional_t<sizeof(T) == 1, uint2, uint4>;
  if (l.row()) {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(raw) / sizeof(Vector)); ++h) reinterpret_cast<Vector*>(&raw)[h] = reinterpret_cast<const Vector*>(p + l.first)[h];
  } else {
    const Element* const from = reinterpret_cast<const Element*>(p + l.first);
    uint32_t* const words = reinterpret_cast<uint32_t*>(&raw);
    constexpr int PER = 4 / sizeof(T);
#pragma unroll
    for (int w = 0; w < 8 / PER; ++w) {
      uint32_t bits = 0;
#pragma unroll
      for (int j = w * PER; j < (w + 1) * PER; ++j)
        if (l.has(j)) bits |= static_cast<uint32_t>(from[l.step(j)]) << (8 * sizeof(T) * (j % PER) % 32);
      words[w] = bits;
    }
  }
}
template <typename T, Places HOW>
__device__ __forceinline__ void store(const Raw8<T>& raw, T* p, const Lane<HOW>& l) {
  using Element = std::conditional_t<sizeof(T) == 4, uint32_t, std::conditional_t<sizeof(T) == 2, uint16_t, uint8_t>>;
  using Vector = std::conditional_t<sizeof(T) == 1, uint2, uint4>;
  if (l.row()) {
#pragma unroll
    for (int h = 0; h < static_cast<int>(sizeof(raw) / sizeof(Vector)); ++h) reinterpret_cast<Vector*>(p + l.first)[h] = reinterpret_cast<const Vector*>(&raw)[h];
  } else {
    Element* const to = reinterpret_cast<Element*>(p + l.first);
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(&raw);
    constexpr int PER = 4 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (l.has(j)) to[l.step(j)] = static_cast<Element>(words[j / PER] >> (8 * sizeof(T) * (j % PER) % 32));
  }
}
template <typename T, Places HOW>
__device__ __forceinline__ void store8(const float (&f)[8], T* p, const Lane<HOW>& l) {
  Raw8<T> raw;
  raw.from(f);
  store(raw, p, l);
}

__device__ __forceinline__ void decode8(uint2 q, float scale, Pair (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = j < 2 ? q.x : q.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * (j & 1))), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[j] = Pair(v.x, v.y) * both(scale);
  }
}

constexpr uint32_t E4M3_MOST = 0x7E, E4M3_NAN = 0x7F, INF_BITS = 0x7f800000u;

__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }

// The largest magnitude of a warp's block, as bits; `finite` whether all are numbers, which it counts alone.
__device__ __forceinline__ uint32_t block_most(const float (&f)[8], bool& finite) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) top = largest(top, f[j], f[j + 1]);
  uint32_t most = __reduce_max_sync(0xffffffffu, magnitude(top));   // a NaN's bits are above all others'
  finite = most < INF_BITS;   // the same in every lane
  if (!finite) {
    most = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, magnitude(f[j]) < INF_BITS ? magnitude(f[j]) : 0u);
    most = __reduce_max_sync(0xffffffffu, most);
  }
  return most;
}

// Four words with a code in bits 20 to 27 each -> the four codes, the first lowest
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t even = __byte_perm(a, c, 0x7632), odd = __byte_perm(b, d, 0x7632);   // upper halves
  return (even >> 4 & 0x00ff00ffu) | (odd << 4 & 0xff00ff00u);
}

// Values -> their block's scale and codes; `dither` is 20 bits for each. ROOTS: they are all negative or zero, held without the sign, and what is not
// zero is not held as zero.
template <bool ROOTS>
__device__ __forceinline__ uint2 hold8(const float (&f)[8], const uint32_t (&dither)[8], uint32_t most, bool finite, float& scale) {
  scale = __fmul_rn(fmaxf(__uint_as_float(most), 1e-30f), 1.f / 448.f);
  const float inv = inverse(scale);
  Pair share[4];
  auto shares = [&](float by) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      share[j] = ROOTS ? fma2(Pair(f[2 * j], f[2 * j + 1]), both(-by), both(0.f)) :   // of zeros of either sign the positive one
                  Pair(__fmul_rn(fabsf(f[2 * j]), by), __fmul_rn(fabsf(f[2 * j + 1]), by));
  };
  if (scale < 32.f) {
    shares(inv * 0x1p-120f);
  } else {   // a factor that is denormal itself would not be exact
    shares(inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) share[j] = share[j] * both(0x1p-120f);
  }
  uint32_t word[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float s[2];
    share[j / 2].to(s[0], s[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      word[j + h] = min(__float_as_uint(s[h]) + (ROOTS ? 0xfffffu - dither[j + h] : dither[j + h]), E4M3_MOST << 20 | 0xfffffu);
  }
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (magnitude(f[j]) >= INF_BITS) word[j] = E4M3_NAN << 20;
  }
  uint2 q = make_uint2(pack_codes(word[0], word[1], word[2], word[3]), pack_codes(word[4], word[5], word[6], word[7]));
  if constexpr (ROOTS) {
    auto zeros = [](uint32_t w) { return (w - 0x01010101u) & ~w & 0x80808080u; };   // whether one of four bytes is
    if (zeros(q.x) | zeros(q.y)) {
      uint32_t least[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) least[j] = word[j] >> 20 == 0 && f[j] < 0.f ? 1u << 20 : 0u;
      q.x |= pack_codes(least[0], least[1], least[2], least[3]);
      q.y |= pack_codes(least[4], least[5], least[6], least[7]);
    }
  } else {
    auto signs = [&](int j) {   // the top bytes of four values
      const uint32_t lo = __byte_perm(__float_as_uint(f[j]), __float_as_uint(f[j + 1]), 0x0073);
      const uint32_t hi = __byte_perm(__float_as_uint(f[j + 2]), __float_as_uint(f[j + 3]), 0x0073);
      return __byte_perm(lo, hi, 0x5410) & 0x80808080u;
    };
    q.x |= signs(0);
    q.y |= signs(4);
  }
  return q;
}

// The moments of a lane's eight elements behind the step, v with its sign turned.
__device__ __forceinline__ void moments8(const float (&gr)[8], Pair (&m)[4], Pair (&v)[4], const AdamwNumbers& a) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const Pair d = Pair(gr[2 * j], gr[2 * j + 1]) * both(a.grad_scale);
    m[j] = fma2(m[j] * both(a.beta1), both(a.one), d * both(a.rest1));
    v[j] = fma2(v[j] * both(a.minus_beta2), both(a.one), d * d * both(a.minus_rest2));
  }
}
__device__ __forceinline__ void update8(float (&x)[8], const Pair (&m)[4], const Pair (&minus_root)[4], const AdamwNumbers& a, float keep) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo, hi;
    fma2(minus_root[j], both(a.minus_root2), both(a.eps)).to(lo, hi);
    const Pair update = m[j] * both(a.minus_lr1) * Pair(reciprocal(lo), reciprocal(hi));
    fma2(Pair(x[2 * j], x[2 * j + 1]), both(keep), update).to(x[2 * j], x[2 * j + 1]);
  }
}

// 2^-40: beside a largest root of more, a root that is off by 2^-16 of itself or more (that of a number up to 2^-119) has the
// least code either way, and eps is more than all of it.
constexpr uint32_t CAREFUL_BELOW = 0x2b800000u;

// What a CTA has of a tensor: pointers to its first element, so that places are numbers of 32 bits. X: what the step reads the parameter from.
template <int BITS, typename P, typename G, bool MASTER>
struct Chunk {
  using X = std::conditional_t<MASTER, float, P>;
  using M = std::conditional_t<BITS == 8, uint8_t, float>;
  P* p;
  G* g;
  X* x;
  M *m, *v;
  float *m_scale, *v_scale;
  uint32_t n;        // elements
  uint32_t dither;   // of the first
  float keep;
  __device__ __forceinline__ Chunk(const B200AdamwTensor& t, const AdamwNumbers& a, int64_t begin, int64_t end) {
    p = static_cast<P*>(t.p) + begin;
    g = static_cast<G*>(t.g) + begin;
    x = MASTER ? reinterpret_cast<X*>(t.master) + begin : reinterpret_cast<X*>(p);
    m = static_cast<M*>(t.m) + begin;
    v = static_cast<M*>(t.v) + begin;
    if constexpr (BITS == 8) {
      m_scale = t.m_scale + begin / ADAMW_BLOCK;
      v_scale = t.v_scale + begin / ADAMW_BLOCK;
    }
    n = static_cast<uint32_t>(end - begin);
    dither = static_cast<uint32_t>(begin) * DITHER_ELEMENT + a.dither;
    keep = t.keep;
  }
};

// A lane's part of a block as it is in memory
template <typename C>
struct Held {
  Raw8<typename std::remove_pointer_t<decltype(C::g)>> g;
  Raw8<typename C::X> x;
  Raw8<typename C::M> m, v;
  float m_scale, v_scale;
  template <Places HOW>
  __device__ __forceinline__ void load_from(const C& c, const Lane<HOW>& l, uint32_t block) {
    load(g, c.g, l);
    load(x, c.x, l);
    load(m, c.m, l);
    load(v, c.v, l);
    if constexpr (sizeof(typename C::M) == 1) {
      m_scale = c.m_scale[block];
      v_scale = c.v_scale[block];
    }
  }
};

template <Places HOW, int BITS, typename P, typename G, bool MASTER, typename Next>
__device__ __forceinline__ void step8(const Chunk<BITS, P, G, MASTER>& c, const AdamwNumbers& a, const Lane<HOW>& l, uint32_t block,
                                      const Held<Chunk<BITS, P, G, MASTER>>& held, Next&& next) {
  float gr[8], x[8];
  Pair m[4], v[4], root[4];
  float mf[8], rf[8];
  held.g.to(gr);
  held.x.to(x);
  if constexpr (BITS == 8) {
    decode8(held.m.q, held.m_scale, m);
    decode8(held.v.q, held.v_scale, v);
  } else {
    held.m.to(mf);
    held.v.to(rf);
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = Pair(mf[2 * j], mf[2 * j + 1]), v[j] = Pair(rf[2 * j], rf[2 * j + 1]);
  }
  next();   // what was held is in registers of its own now: the next block's loads
  if constexpr (BITS == 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = v[j] * v[j];
  }
  moments8(gr, m, v, a);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    root[j] = minus_roots(v[j]);
    if constexpr (BITS == 32) root[j] = any_minus_roots(v[j], root[j]);
    root[j].to(rf[2 * j], rf[2 * j + 1]);
    m[j].to(mf[2 * j], mf[2 * j + 1]);
  }
  if constexpr (BITS == 8) {
    bool v_finite, m_finite;
    uint32_t v_most = block_most(rf, v_finite);
    if (a.careful || !v_finite || (v_most < CAREFUL_BELOW && v_most > 0)) {   // the same for the warp
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        root[j] = any_minus_roots(v[j], root[j]);
        root[j].to(rf[2 * j], rf[2 * j + 1]);
      }
      v_most = block_most(rf, v_finite);
    }
    update8(x, m, root, a, c.keep);
    const uint32_t m_most = block_most(mf, m_finite), d0 = l.first * DITHER_ELEMENT + c.dither;
    uint32_t dither[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) dither[j] = (d0 + l.step(j) * DITHER_ELEMENT) >> 12;
    float ms, vs;
    Raw8<uint8_t> code;
    code.q = hold8<false>(mf, dither, m_most, m_finite, ms);
    store(code, c.m, l);
    code.q = hold8<true>(rf, dither, v_most, v_finite, vs);
    store(code, c.v, l);
    if ((threadIdx.x & 31) == 0) {
      c.m_scale[block] = ms;
      c.v_scale[block] = vs;
    }
  } else {
    update8(x, m, root, a, c.keep);
    store8(mf, c.m, l);
#pragma unroll
    for (int j = 0; j < 4; ++j) (v[j] * both(-1.f)).to(rf[2 * j], rf[2 * j + 1]);
    store8(rf, c.v, l);
  }
  if constexpr (MASTER) store8(x, c.x, l);
  store8(x, c.p, l);
  if (a.zero_grad) {
    const float zero[8] = {};
    store8(zero, c.g, l);
  }
}

template <int BITS, typename P, typename G, bool MASTER>
__device__ __forceinline__ void adamw_chunk(const AdamwEntry& e, const AdamwNumbers& a, int64_t begin, int64_t end) {
  const Chunk<BITS, P, G, MASTER> c(e.t, a, begin, end);
  Held<Chunk<BITS, P, G, MASTER>> held;
  constexpr uint32_t PASS = adamw_pass(BITS);
  uint32_t b = (threadIdx.x >> 5) * ADAMW_BLOCK;
  // Whole blocks: with moments in 8 bits each is loaded while the one before it is worked on, which takes as long.
  auto whole = [&](auto how) {
    constexpr Places HOW = decltype(how)::value;
    if (BITS == 8 && b + ADAMW_BLOCK <= c.n) held.load_from(c, Lane<HOW>(b, c.n), b / ADAMW_BLOCK);
    for (; b + ADAMW_BLOCK <= c.n; b += PASS) {
      const Lane<HOW> l(b, c.n);
      if (BITS == 32) held.load_from(c, l, b / ADAMW_BLOCK);
      step8(c, a, l, b / ADAMW_BLOCK, held, [&] {
        if (BITS == 8 && b + PASS + ADAMW_BLOCK <= c.n) held.load_from(c, Lane<HOW>(b + PASS, c.n), (b + PASS) / ADAMW_BLOCK);
      });
    }
  };
  if (e.places == ALIGNED)
    whole(std::integral_constant<Places, ALIGNED>{});
  else
    whole(std::integral_constant<Places, STRIDED>{});
  for (; b < c.n; b += PASS) {
    const Lane<LAST> l(b, c.n);
    held.load_from(c, l, b / ADAMW_BLOCK);
    step8(c, a, l, b / ADAMW_BLOCK, held, [] {});
  }
}

template <int BITS, int N>
__global__ void __launch_bounds__(adamw_threads(BITS), adamw_ctas(BITS)) adamw_many_kernel(const __grid_constant__ AdamwTable<N> table) {
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
  grid_wait();
  grid_release();
  using bf16 = __nv_bfloat16;
  if (e.t.p_fp32) {
    if (e.t.g_fp32)
      adamw_chunk<BITS, float, float, false>(e, table.a, begin, end);
    else
      adamw_chunk<BITS, float, bf16, false>(e, table.a, begin, end);
  } else if (e.t.master) {
    if (e.t.g_fp32)
      adamw_chunk<BITS, bf16, float, true>(e, table.a, begin, end);
    else
      adamw_chunk<BITS, bf16, bf16, true>(e, table.a, begin, end);
  } else {
    if (e.t.g_fp32)
      adamw_chunk<BITS, bf16, float, false>(e, table.a, begin, end);
    else
      adamw_chunk<BITS, bf16, bf16, false>(e, table.a, begin, end);
  }
}

static bool on(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Elements of a CTA: as few as fill the chip, up to some passes of it. With 8-bit moments, in passes enough to draw the clock down, four take 433 and 270 us, eight
// 417 and 266, 32 5 and 10 us more.
static int adamw_chunk_elements(int64_t total, int bits) {
  const int most = bits == 8 ? 8 : 4;
  const int64_t passes = total / (static_cast<int64_t>(sm_count()) * 2048 * 8);
  return adamw_pass(bits) * static_cast<int>(passes < 1 ? 1 : passes > most ? most : passes);
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
    e.places = on(e.t.p, 16) && on(e.t.g, 16) && on(e.t.master, 16) && on(e.t.m, state) && on(e.t.v, state) ? ALIGNED : STRIDED;
    ctas += (e.t.n + chunk - 1) / chunk;
  }
  if (ctas > INT_MAX) return B200_ERR_TOO_LARGE;
  table.a = a;
  table.count = count;
  table.chunk = chunk;
  launch_dependent(bits == 8 ? adamw_many_kernel<8, N> : adamw_many_kernel<32, N>, static_cast<int>(ctas), adamw_threads(bits), 0, stream, table);
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
  auto twice = [](double v) { return make_float2(static_cast<float>(v), static_cast<float>(v)); };
  AdamwNumbers a{};
  a.one = twice(1.0);
  a.beta1 = twice(beta1);
  a.rest1 = twice(1.0 - beta1);
  a.minus_beta2 = twice(-beta2);
  a.minus_rest2 = twice(beta2 - 1.0);
  a.minus_lr1 = twice(-lr / c1);
  a.minus_root2 = twice(-1.0 / sqrt(c2));
  a.eps = twice(eps);
  a.grad_scale = twice(grad_scale);
  a.careful = eps < 1e-12;
  a.dither = static_cast<uint32_t>(step) * DITHER_STEP;
  a.zero_grad = zero_grad;
  const int chunk = adamw_chunk_elements(total, bits);
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
