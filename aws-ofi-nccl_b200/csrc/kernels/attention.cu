// Causal attention with a sliding window and first tokens that stay visible, forward and backward, on tcgen05.
//
//   S = scale q k^T over visible keys, P = softmax(S), out = P v
//   delta = sum(dout * out), dS = P * (dout v^T - delta), dq = scale dS k, dk = scale dS^T q, dv = P^T dout
//
// Scores never leave the SM: the forward pass keeps a running maximum and sum of each row (Milakov and Gimelshein, "Online normalizer calculation for
// softmax", 2018), the backward pass computes P again from the rows' log-sum (in base 2), whose negative the forward pass stores.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "attention.cuh"
#include "b200ops.h"
#include "host_util.h"

namespace b200 {

// Kernels stay: as many CTAs as SMs, each with several items of work (a tile and its walk over the other side), whose loads and first products run
// beside the end of the item before. Items are ordered by their length, longest first, and dealt there and back, so that every CTA has about as much.
__device__ __forceinline__ int dealt(int turn) {
  const int ctas = gridDim.x, cta = blockIdx.x;
  return turn * ctas + (turn & 1 ? ctas - 1 - cta : cta);
}

// A number that the compiler takes for a new one: an item made of it again behind its walk costs less than the registers that keep it along the walk.
__device__ __forceinline__ int anew(int x) {
  asm volatile("" : "+r"(x));
  return x;
}

// Rows of at most 128 keys take probabilities and the gradients of scores into their products as two operands, what they are rounded to and what that left (of few keys
// one rounding of an operand does not average out). These are all rows of a launch with FINE, and the first 128 of every sequence: those that begin in front of row
// 128, whatever the batch is padded to. With a window and its sinks beyond 128 keys no other row sees so few.
__device__ __forceinline__ bool few_keys_from(int row) { return row < ATT_TILE; }
// An operand lies as packed pairs over the first half of each 32 columns of scores that it came from, the second one over the other half.
constexpr int OP_GROUP = 32, OP_SECOND = 16;

// The products of second operands, those steps of which STEPS has a bit. Called, not part of the loops over tiles: there its instructions, hardly ever run, cost 2 to 5 % of
// the time.
template <int HD, uint32_t STEPS>
__device__ __noinline__ void multiply_second(uint32_t d, uint32_t operand, uint32_t b_low) {
#pragma unroll
  for (int k = 0; k < ATT_TILE / 16; ++k)
    if (STEPS >> k & 1) multiply_step<HD, OP_GROUP>(d, operand + OP_SECOND, b_low, k, true);
}

// ------------------------------------------------------------------ forward
// An item are two units of 128 queries of one head each that share a head of k and v: two heads of a group for the same tokens, or where the number
// of heads in a group is odd also neighbouring tokens. So a tile of k and v is loaded once for 256 rows.
struct AttnUnit {
  int head, i0, lo, hi;   // rows from i0; key tiles lo to hi of its window
  bool live, exists;      // has rows in front of the sequence's end, of the tensor's
};
struct AttnFwdItem {
  int b, kv_head, len;
  AttnUnit unit[2];
  // the walk of both: `far` tiles of sinks, then tiles from lo; n in all
  int far, lo, n, sink_tiles;
  int clear_from;   // from which row on its last tile is not the sequence's: what TMA does not fill with zeros by itself
  __device__ __forceinline__ int tile(int j) const { return j < far ? j : lo + j - far; }
  __device__ __forceinline__ bool uses(int u, int t) const { return unit[u].live && t <= unit[u].hi && (t >= unit[u].lo || t < sink_tiles); }

  __device__ __forceinline__ AttnFwdItem(const AttnShape& s, int item) {
    const int heads = s.B * s.nkv, units = s.rows / ATT_TILE * s.G;
    const int nth = s.by_heads_kv.quotient(item), pair = (units + 1) / 2 - 1 - nth, bh = item - nth * heads;
    b = s.by_nkv.quotient(bh), kv_head = bh - b * s.nkv;
    len = sequence_length(s, b);
    sink_tiles = s.window ? (s.sinks + ATT_TILE - 1) / ATT_TILE : 0;
    lo = 1 << 30;
    int hi = -1;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      AttnUnit& r = unit[u];
      const int at = 2 * pair + u, rows = s.by_G.quotient(at);
      r.head = kv_head * s.G + (at - rows * s.G);
      r.i0 = rows * ATT_TILE;
      r.exists = at < units;
      r.live = r.exists && r.i0 < len;
      r.hi = r.live ? (min(r.i0 + ATT_TILE, len) - 1) / ATT_TILE : -1;
      r.lo = s.window ? max(0, r.i0 - s.window + 1) / ATT_TILE : 0;
      if (r.live) lo = min(lo, r.lo);
      hi = max(hi, r.hi);
    }
    far = hi < 0 ? 0 : min(sink_tiles, lo);
    n = hi < 0 ? 0 : far + hi - lo + 1;
    clear_from = n > 0 && len < s.S ? min(len - hi * ATT_TILE, ATT_TILE) : ATT_TILE;
  }
};

using AttnFwdRoles = AttnRoles<16>;
template <int HD>
struct AttnFwd {
  static constexpr int TILE = ATT_TILE * HD * 2;
  static constexpr int STAGES = 4;
  static constexpr int OUT = (2 + STAGES) * TILE;       // 32 rows of 32 elements of each warp on their way out
  static constexpr int TOLD = OUT + 16 * 2048;          // a number for each row, from one of its threads to the other
  static constexpr int TILES = TOLD + 2 * ATT_TILE * 4;
  static constexpr int SMEM = 1024 + TILES + ATT_BAR_BYTES;
  // barriers: stages full and empty; q there and read; scores there; probabilities there (or their row scaled), in two parts; sums of a unit done; rows behind
  // a sequence's end to be cleared, cleared
  static constexpr int FULL = 0, EMPTY = STAGES, Q = 2 * STAGES, QREAD = Q + 2, SCORES = QREAD + 2, PROBS = SCORES + 2, DONE = PROBS + 4, CLEAR = DONE + 2,
                       CLEARED = CLEAR + 1, BARS = CLEARED + 1;
  // tensor memory: scores of a unit (probabilities as bf16 over the first columns of each half), its sums
  static constexpr int S_COL = 0, O_COL = 256;
  static_assert(SMEM <= 232448, "more than a CTA's shared memory");
};

template <int HD, bool FINE>
__global__ void __launch_bounds__(AttnFwdRoles::THREADS, 1)
    attention_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                         const __grid_constant__ CUtensorMap tmSinks, const __grid_constant__ CUtensorMap tmO, const __grid_constant__ CUtensorMap tmR, int with_rest,
                         float* minus_lse, AttnShape s, int items, int* err_word) {
  using L = AttnFwd<HD>;
  using R = AttnFwdRoles;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const AttnCta cta = attn_begin<R, L::TILES, L::BARS>(smem_raw, err_word, [](int i) { return i >= L::PROBS && i < L::DONE ? 8 : 1; });
  grid_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t q_tile = cta.smem, stages = cta.smem + 2 * L::TILE;
  auto stage = [&](uint32_t i) { return stages + i % L::STAGES * L::TILE; };

  if (warp == R::LOAD) {
    // ---------------------------------------------------------------- loads: q, then k and v in turn
    if (elect_one_sync()) {
      uint32_t loaded = 0, q_loaded[2] = {0, 0};
      bool ok = true;
      for (int turn = 0; ok && dealt(turn) < items; ++turn) {
        const AttnFwdItem w(s, dealt(turn));
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (w.unit[u].live && (ok = ok && cta.wait(L::QREAD + u, (q_loaded[u]++ & 1) ^ 1, DEV_ERR_EMPTY_BAR_TIMEOUT))) {
            mbar_expect_tx(cta.bar(L::Q + u), L::TILE);
            load_tile<HD, ATT_TILE>(q_tile + u * L::TILE, &tmQ, w.b, w.unit[u].head, w.unit[u].i0, cta.bar(L::Q + u));
          }
        for (int i = 0; i < 2 * w.n && ok; ++i, ++loaded) {
          const int st = loaded % L::STAGES;
          if (!(ok = cta.wait(L::EMPTY + st, (loaded / L::STAGES & 1) ^ 1, DEV_ERR_EMPTY_BAR_TIMEOUT))) break;
          mbar_expect_tx(cta.bar(L::FULL + st), L::TILE);
          load_tile<HD, ATT_TILE>(stage(loaded), i & 1 ? i >> 1 < w.far ? &tmSinks : &tmV : &tmK, w.b, w.kv_head, w.tile(i >> 1) * ATT_TILE, cta.bar(L::FULL + st));
        }
      }
      grid_release();
    }
  } else if (warp == R::MMA) {
    // ---------------------------------------------------------------- products. Of one thread they run in the order of their issue: probabilities
    // are read before the next scores of their unit are written over them
    if (elect_one_sync()) {
      auto full = [&](uint32_t i) { return cta.wait(L::FULL + i % L::STAGES, i / L::STAGES & 1, DEV_ERR_FULL_BAR_TIMEOUT); };
      uint32_t at = 0, q_used[2] = {0, 0}, turns[2] = {0, 0}, cleared = 0;   // loads, units and their tiles so far
      bool ok = true;
      for (int turn = 0; ok && dealt(turn) < items; ++turn) {
        const AttnFwdItem w(s, dealt(turn));
        if (w.n == 0) continue;
        auto scores = [&](int u, uint32_t i, int t) {
          multiply_rows<HD>(L::S_COL + u * ATT_TILE, q_tile + u * L::TILE, stage(i));
          umma_commit(cta.bar(L::SCORES + u));
          if (t == w.unit[u].hi) umma_commit(cta.bar(L::QREAD + u));
        };
        bool begun[2] = {false, false};   // a unit's sums
        if (!(ok = full(at))) break;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (w.unit[u].live) {
            ok = ok && cta.wait(L::Q + u, q_used[u]++ & 1, DEV_ERR_FULL_BAR_TIMEOUT);
            tc_fence_after();
            if (ok && w.uses(u, w.tile(0))) scores(u, at, w.tile(0));
          }
        umma_commit(cta.bar(L::EMPTY + at % L::STAGES));
        for (int j = 0; j < w.n && ok; ++j, at += 2) {
          const int t = w.tile(j), next = w.tile(j + 1);
          const bool more = j + 1 < w.n;
          if (!(ok = full(at + 1) && (!more || full(at + 2)))) break;
          if (!more && w.clear_from < ATT_TILE) {
            mbar_arrive(cta.bar(L::CLEAR));
            if (!(ok = cta.wait(L::CLEARED, cleared++ & 1, DEV_ERR_FULL_BAR_TIMEOUT))) break;
          }
          const uint32_t v_low = TileDesc<ATT_TILE, true>::low(stage(at + 1));
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (w.uses(u, t)) {
              // in two parts, of 32 columns of both halves, as they are there
#pragma unroll
              for (int part = 0; part < 2; ++part) {
                if (!(ok = ok && cta.wait(L::PROBS + 2 * u + part, turns[u] & 1, DEV_ERR_TMEM_EMPTY_TIMEOUT))) break;
                tc_fence_after();
                auto step = [&](int operand, int k, bool add) {
                  multiply_step<HD, OP_GROUP>(L::O_COL + u * 128, L::S_COL + u * ATT_TILE + operand, v_low, part * 2 + k + (k & 2), add);
                };
                step(0, 0, part || begun[u]);
#pragma unroll
                for (int k = 1; k < 4; ++k) step(0, k, true);
                if constexpr (FINE) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) step(OP_SECOND, k, true);
                } else if (few_keys_from(w.unit[u].i0)) {
                  multiply_second<HD, 0x33>(L::O_COL + u * 128, L::S_COL + u * ATT_TILE + part * OP_GROUP, v_low + part * TileDesc<ATT_TILE, true>::step(2));
                }
              }
              if (!ok) break;
              begun[u] = true;
              ++turns[u];
              if (t == w.unit[u].hi) umma_commit(cta.bar(L::DONE + u));
            }
            if (more && w.uses(u, next)) scores(u, at + 2, next);
          }
          if (!ok) break;
          umma_commit(cta.bar(L::EMPTY + (at + 1) % L::STAGES));
          if (more) umma_commit(cta.bar(L::EMPTY + (at + 2) % L::STAGES));
        }
      }
    }
  } else if (warp == R::ZERO) {
    // ---------------------------------------------------------------- v behind a sequence's end, in the last tile of a walk
    uint32_t at = 0, cleared = 0, before = 0;   // before: loads at the last one
    bool ok = true;
    for (int turn = 0; s.lengths && ok && dealt(turn) < items; ++turn) {
      const AttnFwdItem w(s, dealt(turn));
      at += 2 * w.n;
      if (w.clear_from == ATT_TILE) continue;
      const uint32_t last = at - 1;
      ok = cta.wait(L::CLEAR, cleared++ & 1, DEV_ERR_FULL_BAR_TIMEOUT, at - before) &&
           cta.wait(L::FULL + last % L::STAGES, last / L::STAGES & 1, DEV_ERR_FULL_BAR_TIMEOUT);
      if (ok) zero_rows<HD, ATT_TILE>(stage(last), w.clear_from, cta.bar(L::CLEARED));
      before = at;
    }
  } else {
    // ---------------------------------------------------------------- softmax: a thread has half of a row
    const int u = warp >> 3, half = warp >> 2 & 1, place = (warp & 3) * 32 + lane;
    const int meeting = 1 + u * 4 + (warp & 3);   // of the two warps that have the same rows
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_col = lanes + L::S_COL + u * ATT_TILE + half * 64, o_col = lanes + L::O_COL + u * 128 + half * (HD / 2);
    volatile float* const told = reinterpret_cast<volatile float*>(smem_raw + (cta.smem - smem_u32(smem_raw)) + L::TOLD) + u * ATT_TILE + place;
    const float c = s.scale * ATT_LOG2E;
    const Pair c2 = both(c);
    const RowsOut slab{cta.smem + L::OUT + warp * 2048};
    uint32_t turns = 0, done = 0;   // tiles and units so far
    bool ok = true;                 // where a wait gives up the walks go on without its scores: both warps of some rows meet as often
#pragma unroll 1
    for (int turn = 0; dealt(turn) < items; ++turn) {
      const AttnFwdItem walk(s, dealt(turn));
      const int i0 = u ? walk.unit[1].i0 : walk.unit[0].i0, lo = u ? walk.unit[1].lo : walk.unit[0].lo;
      const bool exists = u ? walk.unit[1].exists : walk.unit[0].exists;
      const int head_of_all = walk.b * s.nq + (u ? walk.unit[1].head : walk.unit[0].head);
      // this unit's own tiles of the walk
      const int far = min(walk.sink_tiles, lo), n = (u ? walk.unit[1].live : walk.unit[0].live) ? far + (u ? walk.unit[1].hi : walk.unit[0].hi) - lo + 1 : 0;
      float top = -INFINITY;   // of the scores times c, as far as the sums are scaled to it
      float sum = 0.f;         // of this half's probabilities, relative to 2^top
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++turns) {
        const int j0 = (j < far ? j : lo + j - far) * ATT_TILE + half * 64;
        ok = cta.wait(L::SCORES + u, turns & 1, DEV_ERR_TMEM_FULL_TIMEOUT) && ok;
        tc_fence_after();
        const bool whole = j0 + 63 <= i0 && (s.window == 0 || i0 + ATT_TILE - 1 - j0 < s.window || j0 + 64 <= s.sinks);
        auto take = [&](auto is_whole, auto in_two) {   // a tile on no border without any of what a border takes
          constexpr bool WHOLE = decltype(is_whole)::value, TWO = decltype(in_two)::value;
          // what a row sees of each 32 columns; blocks of 32 rows and columns of which none is seen are zeros without their scores being looked at
          uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
          if constexpr (!WHOLE) {
            const int last = i0 + place - j0, first = s.window ? last - s.window + 1 : 0, sinks = s.window ? s.sinks - j0 : 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) seen[k] = columns_seen(first - k * 32, last - k * 32, sinks - k * 32);
          }
          const bool some_seen[2] = {WHOLE || __any_sync(0xffffffffu, seen[0]), WHOLE || __any_sync(0xffffffffu, seen[1])};
          auto hide = [&](auto& x, int k, int from) {   // columns `from` on of 32
            if constexpr (!WHOLE) {
              if (__all_sync(0xffffffffu, seen[k] == 0xffffffffu)) return;
#pragma unroll
              for (int e = 0; e < static_cast<int>(sizeof(x) / 4); ++e)
                if (!(seen[k] >> (from + e) & 1)) x[e] = 0xFF800000u;   // -inf
            }
          };
          // Scores are read twice, for their maximum and for the probabilities: all of them with what else is needed are more than a thread has registers
          float some[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (!some_seen[k]) continue;
            uint32_t x[32];
            tmem_ld_32x32(s_col + k * 32, x);
            tmem_ld_wait();
            hide(x, k, 0);
#pragma unroll
            for (int e = 0; e < 32; e += 2) some[e / 2 & 3] = most_of(some[e / 2 & 3], __uint_as_float(x[e]), __uint_as_float(x[e + 1]));
          }
          const float most = most_of(most_of(some[0], some[1], some[2]), some[3], some[3]) * c;
          // The sums are scaled to a new maximum only where one of the two warps' rows has grown by more than 2^8: probabilities beside the old one
          // stay in range. A NaN grows, too, and makes one of everything in its row.
          if (any_of_64(meeting, !(most <= top + 8.f))) {
            if (half) *told = most;
            meet_64(meeting);
            float now = 0.f;
            if (!half) *told = now = most_of(top, most, *told);
            meet_64(meeting);
            if (half) now = *told;
            const float f = now == -INFINITY ? 1.f : exp2_unit(top - now);
            top = now;
            sum *= f;
            if (j) {
#pragma unroll
              for (int k = 0; k < HD / 32; ++k) {
                uint32_t o[16];
                tmem_ld_32x16(o_col + k * 16, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st_32x16(o_col + k * 16, o);
              }
            }
          }
          const Pair ref = both(top == -INFINITY ? 0.f : -top);
          Pair part[2] = {both(0.f), both(0.f)};
          // probabilities of 32 columns come to lie over columns that have been read
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            constexpr int COLS = TWO ? 16 : 32;   // at a time: with 32 the path of one operand spills what two take
            uint32_t left[COLS / 2];
#pragma unroll
            for (int from = 0; from < 32; from += COLS) {
              uint32_t p[COLS / 2];
              if (some_seen[k]) {
                uint32_t x[COLS];
                tmem_ld_cols(s_col + k * 32 + from, x);
                tmem_ld_wait();
                if (TWO && from) tmem_st_cols(s_col + k * OP_GROUP + OP_SECOND, left);   // where scores of these columns were
                hide(x, k, from);
#pragma unroll
                for (int e = 0; e < COLS; e += 2) {
                  float p0, p1;
                  fma2(pair_of(x[e], x[e + 1]), c2, ref).to(p0, p1);
                  p0 = exp2_unit(p0), p1 = exp2_unit(p1);
                  part[e / 2 & 1] = part[e / 2 & 1] + Pair(p0, p1);
                  p[e / 2] = pack_bf16x2(p0, p1);
                  if constexpr (TWO) left[e / 2] = left_of(p0, p1, p[e / 2]);
                }
              } else {
#pragma unroll
                for (int e = 0; e < COLS / 2; ++e) p[e] = left[e] = 0;
                if (TWO && from) tmem_st_cols(s_col + k * OP_GROUP + OP_SECOND, left);
              }
              tmem_st_cols(s_col + k * OP_GROUP + from / 2, p);
            }
            if constexpr (TWO) tmem_st_cols(s_col + k * OP_GROUP + OP_SECOND + 8, left);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(cta.bar(L::PROBS + 2 * u + k));
          }
          float a, d;
          (part[0] + part[1]).to(a, d);
          sum += a + d;
        };
        using Two = std::bool_constant<FINE>;
        if (whole)
          take(std::true_type(), Two());
        else if (!FINE && few_keys_from(i0))   // never whole
          take(std::false_type(), std::true_type());
        else
          take(std::false_type(), Two());
      }
      if (!exists) continue;
      if (half) *told = sum;
      meet_64(meeting);
      if (!half) *told = sum = sum + *told;
      meet_64(meeting);
      if (half) sum = *told;
      if (n) ok = cta.wait(L::DONE + u, done++ & 1, DEV_ERR_TMEM_FULL_TIMEOUT) && ok;
      tc_fence_after();
      const int b = s.by_nq.quotient(head_of_all), head = head_of_all - b * s.nq, i = i0 + place;
      const bool mine = i < sequence_length(s, b);
      if (!half)   // no probability behind the end
        minus_lse[static_cast<int64_t>(head_of_all) * s.rows + i] = mine ? -top - log2f(sum) : -INFINITY;
      const float f = 1.f / sum;
      const bool any = mine && n && ok;
      uint32_t rest[HD / 8];   // of this thread's half of a row
#pragma unroll
      for (int k = 0; k < HD / 64; ++k) {
        uint32_t o[32];
        if (n && ok) {
          tmem_ld_32x32(o_col + k * 32, o);
          tmem_ld_wait();
        }
        uint32_t two[16];
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float f4[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) f4[r] = any ? __uint_as_float(o[e + r]) * f : 0.f;
          two[e / 2] = pack_bf16x2(f4[0], f4[1]), two[e / 2 + 1] = pack_bf16x2(f4[2], f4[3]);
          rest[k * 8 + e / 4] = rest_of(f4, two[e / 2], two[e / 2 + 1]);
        }
        slab.free();
        slab.put(two);
        slab.out(&tmO, half * (HD / 2) + k * 32, head, i0 + (warp & 3) * 32, b);
      }
      if (with_rest) {
        slab.free();
#pragma unroll
        for (int e = 0; e < HD / 8; e += 4) st_shared_v4(slab.slab + lane * (HD / 2) + e * 4, rest[e], rest[e + 1], rest[e + 2], rest[e + 3]);
        slab.out(&tmR, half * (HD / 2), head, i0 + (warp & 3) * 32, b);
      }
      tc_fence_before();   // the sums are read: by the next handing over of probabilities they may be written
    }
    if (lane == 0) tma_store_wait<0>();
  }
  attn_end<R>(cta);
}

// ------------------------------------------------------------------ backward
// minus_delta[b][head][i] = -(sum over a row of dout * (out + what its rounding left, unless rest is null)), 0 behind a sequence's end. 16-byte vectors of a row in neighbouring lanes, two rows of a
// thread at once.
constexpr int DELTA_ROWS = 2;
template <int HD>
__global__ void __launch_bounds__(256) attention_delta_kernel(const bf16* dout, int64_t db, int64_t dt, int64_t dh, const bf16* out, const uint8_t* rest, float* minus_delta,
                                                              AttnShape s, int blocks) {
  constexpr int LANES = HD / 8, STEP = 256 / LANES;
  const int b = blockIdx.x / blocks, v = threadIdx.x % LANES;
  const int64_t first = static_cast<int64_t>(blockIdx.x - b * blocks) * (STEP * DELTA_ROWS);   // over [rows][nq]
  const int token = first < INT_MAX ? s.by_nq.quotient(static_cast<int>(first)) : static_cast<int>(first / s.nq);
  const int beyond = static_cast<int>(first - static_cast<int64_t>(token) * s.nq) + threadIdx.x / LANES;
  grid_wait();
  grid_release();
  const int len = sequence_length(s, b);
  uint4 a[DELTA_ROWS], o[DELTA_ROWS];
  uint2 more_of[DELTA_ROWS];
  int h[DELTA_ROWS], i[DELTA_ROWS];
#pragma unroll
  for (int k = 0; k < DELTA_ROWS; ++k) {
    const int more = s.by_nq.quotient(beyond + k * STEP);
    i[k] = token + more, h[k] = beyond + k * STEP - more * s.nq;
    a[k] = o[k] = make_uint4(0, 0, 0, 0);
    more_of[k] = make_uint2(0, 0);
    if (i[k] < len) {
      a[k] = reinterpret_cast<const uint4*>(dout + b * db + i[k] * dt + h[k] * dh)[v];
      const int64_t at = ((static_cast<int64_t>(b) * s.S + i[k]) * s.nq + h[k]) * HD + v * 8;
      o[k] = *reinterpret_cast<const uint4*>(out + at);
      if (rest) more_of[k] = *reinterpret_cast<const uint2*>(rest + at);
    }
  }
#pragma unroll
  for (int k = 0; k < DELTA_ROWS; ++k) {
    const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162*>(&a[k]), *y = reinterpret_cast<const __nv_bfloat162*>(&o[k]);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 r = rest_pair((e < 2 ? more_of[k].x : more_of[k].y) >> (16 * (e & 1)));
      sum = fmaf(__low2float(x[e]), __low2float(y[e]) + r.x, sum);
      sum = fmaf(__high2float(x[e]), __high2float(y[e]) + r.y, sum);
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (v == 0 && i[k] < s.rows) minus_delta[(static_cast<int64_t>(b) * s.nq + h[k]) * s.rows + i[k]] = -sum;
  }
}

// Both gradient kernels hold a tile of 128 rows and walk over tiles of 128 rows of the other side:
//   KEYS (dk, dv): a tile of k and v; q, dout, lse and delta pass by, over the heads of the group, whose sum is the gradient
//   else (dq):     a tile of q and dout; k and v pass by
// First T1 = held1 passing1^T (scores) and T2 = held2 passing2^T (dout v^T), then P and dS as bf16 operands in tensor memory of
// dv += P dout, dk += dS q or dq += dS k. Four groups of warps have 32 columns each, a thread a row of them. Products and probabilities of neighbouring tiles
// overlap: with KEYS tensor memory is full with T1, T2 and two sums, P lies over T1 and dS over T2; dv's product and the next scores run while dS is
// computed, dk's and the next T2 while the next probabilities are. dq leaves room for two tiles' scores, and dS lies over those. Every sum is made
// in one order: gradients are the same bits in every run.
using AttnBwdRoles = AttnRoles<16>;
template <int HD, bool KEYS>
struct AttnBwd {
  static constexpr int TILE = ATT_TILE * HD * 2;
  // stages of the passing tensors. dq's first one is wanted two tiles ahead, its second one is free again as soon as T2 is there
  static constexpr int N1 = HD == 64 || !KEYS ? 3 : 2, N2 = KEYS ? 2 : 1;
  static constexpr int STATS = 2 * ATT_TILE * 4;                 // lse and delta of a stage's rows
  static constexpr int PASS1 = 2 * TILE, PASS2 = PASS1 + N1 * TILE, OUT = PASS2 + N2 * TILE;
  static constexpr int STAT = OUT + (KEYS ? 0 : 16 * 2048);      // behind each warp's rows on their way out
  static constexpr int TILES = STAT + (KEYS ? N1 * STATS : 0);
  static constexpr int SMEM = 1024 + TILES + ATT_BAR_BYTES;
  static_assert(SMEM <= 232448, "more than a CTA's shared memory");
  static constexpr int FULL1 = 0, EMPTY1 = FULL1 + N1, FULL2 = EMPTY1 + N1, EMPTY2 = FULL2 + N2, THERE = EMPTY2 + N2, HELD_READ = THERE + 1;
  static constexpr int T1 = HELD_READ + 1, T2 = T1 + (KEYS ? 1 : 2), DONE = T2 + 1;            // T1 and T2 there, sums done
  static constexpr int READ = DONE + 1, PROBS = READ, GRADS = PROBS + 2;   // P, in two parts, and dS there: by all warps
  // rows behind a sequence's end are to be cleared, are zeros: of both passing tensors
  static constexpr int CLEAR1 = GRADS + 1, CLEARED1 = CLEAR1 + 1, CLEAR2 = CLEARED1 + 1, CLEARED2 = CLEAR2 + 1, BARS = CLEARED2 + 1;
  // tensor memory: scores (dq: of two tiles), dout v^T, sums
  static constexpr int T1_COL = 0, T2_COL = KEYS ? 128 : 256, ACC1_COL = 256, ACC2_COL = 384;
};
// How the walk of dk and dv over queries that see a tile only through sinks is split: `parts` CTAs take `part_tiles` tiles of queries each, of every
// head, and their sums and those of the tile's own window are joined in order. parts 0: no tile has any.
struct AttnSplit {
  int tiles, parts, part_tiles;
  Divisor by_part;   // items of a part
  float* sums;   // [1 + parts][B * nkv * tiles][dv, dk][128][HD]
};

// An item: a held tile and its walk, `far` passing tiles from 0, then tiles from `lo` on, per_head in all; with KEYS for each head of the group.
template <bool KEYS>
struct AttnBwdItem {
  int b, head, first_head, len, r0;   // first_head: of the passing tensors
  int tile, part, far, lo, per_head, n;
  int clear_from;   // from which row on a head's last tile is not the sequence's: what TMA does not fill with zeros by itself
  bool joined;      // its sums are one part of several
  __device__ __forceinline__ int row(int at) const { return (at < far ? at : lo + at - far) * ATT_TILE; }   // the first one of a head's at-th tile

  __device__ __forceinline__ AttnBwdItem(const AttnShape& s, const AttnSplit& split, int item) {
    const int heads = s.B * (KEYS ? s.nkv : s.nq), tiles = s.rows / ATT_TILE;
    const int split_items = KEYS ? heads * split.tiles * split.parts : 0;
    part = far = 0;
    int index = item;
    const Divisor &by_heads = KEYS ? s.by_heads_kv : s.by_heads_q, &by_head = KEYS ? s.by_nkv : s.by_nq;
    if (index < split_items) {
      part = split.by_part.quotient(index);
      index -= part * heads * split.tiles;
      ++part;
      tile = by_heads.quotient(index);
      index -= tile * heads;
    } else {
      index -= split_items;
      tile = by_heads.quotient(index);
      index -= tile * heads;
      if (!KEYS) tile = tiles - 1 - tile;   // the longest walks first
    }
    b = by_head.quotient(index);
    head = index - b * by_head.d;
    first_head = KEYS ? head * s.G : s.by_G.quotient(head);
    len = sequence_length(s, b), r0 = tile * ATT_TILE;
    joined = KEYS && split.parts > 0 && tile < split.tiles;
    if constexpr (KEYS) {
      // queries of the window: up to the last key's; of the far parts: behind those
      const int end = (len + ATT_TILE - 1) / ATT_TILE;
      const int near = s.window ? min(end, (r0 + ATT_TILE - 1 + s.window - 1) / ATT_TILE + 1) : end;
      lo = tile;
      int hi = near;
      if (part) {
        lo = min(near + (part - 1) * split.part_tiles, end);
        hi = min(lo + split.part_tiles, end);
      } else if (s.window && !joined && r0 < s.sinks) {
        hi = end;   // sinks whose walk is not split
      }
      per_head = r0 < len ? max(0, hi - lo) : 0;
    } else {
      const int last = min(r0 + ATT_TILE, len) - 1;
      lo = s.window ? max(0, r0 - s.window + 1) / ATT_TILE : 0;
      far = s.window ? min((s.sinks + ATT_TILE - 1) / ATT_TILE, lo) : 0;
      per_head = r0 < len ? far + last / ATT_TILE - lo + 1 : 0;
    }
    n = (KEYS ? s.G : 1) * per_head;
    clear_from = n > 0 && len < s.S ? min(len - row(per_head - 1), ATT_TILE) : ATT_TILE;
  }
};

// A warp's values in tensor memory are there for the products behind a barrier.
__device__ __forceinline__ void hand_over(const AttnCta& cta, int barrier) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(cta.bar(barrier));
}
// A warp's part of a tile, 32 columns from c0 on of rows from r0 on of which this thread has row r: from scores and dout v^T to the operands of the second products, with
// TWO both. lse and delta are those of columns (stat) with KEYS, else of the row. False: a wait gave up.
template <class L, bool KEYS, bool TWO>
__device__ __forceinline__ bool tile_gradients(const AttnCta& cta, uint32_t i, uint32_t t1, uint32_t t2, int r, int r0, int c0, int window, int all_sinks, Pair c,
                                               const ulonglong2* stat, float my_lse, float my_delta) {
  // which columns this row's partner sees: those from first to last, and those in front of `sinks`
  bool whole;
  int first, last, sinks = 0;
  if constexpr (KEYS) {   // columns are queries: from the key itself on, up to its window's end
    whole = c0 >= r0 + ATT_TILE - 1 && (window == 0 || c0 + 31 - r0 < window || r0 + ATT_TILE <= all_sinks);
    first = r - c0;
    last = window == 0 || r < all_sinks ? 32 : first + window - 1;
  } else {                // columns are keys
    whole = c0 + 31 <= r0 && (window == 0 || r0 + ATT_TILE - 1 - c0 < window || c0 + 32 <= all_sinks);
    last = r - c0;
    first = window ? last - window + 1 : 0;
    sinks = window ? all_sinks - c0 : 0;
  }
  auto row_numbers = [&](int of, int e, Pair& p0, Pair& p1) {   // of columns e to e + 3: lse (0), delta (1)
    if constexpr (KEYS) {
      const ulonglong2 v = stat[of * (ATT_TILE / 4) + e / 4];
      p0.bits = v.x, p1.bits = v.y;
    } else {
      p0 = p1 = both(of ? my_delta : my_lse);
    }
  };
  auto hide = [&](uint32_t(&packed)[16]) {   // also what zero times is not finite
    const uint32_t seen = columns_seen(first, last, sinks);
    if (__any_sync(0xffffffffu, seen + 1 > 1)) {   // neither none nor all of a row
#pragma unroll
      for (int e = 0; e < 16; ++e) packed[e] = seen_pair(packed[e], seen, e);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) packed[e] &= seen;
    }
  };
  uint32_t p[32];
  tmem_ld_32x32(t1, p);
  tmem_ld_wait();
#pragma unroll
  for (int part = 0; part < 2; ++part) {
#pragma unroll
    for (int e = part * 16; e < part * 16 + 16; e += 4) {
      Pair l0, l1;
      row_numbers(0, e, l0, l1);
      float a, d;
      exp2_pair(e, fma2(pair_of(p[e], p[e + 1]), c, l0), a, d);
      p[e] = __float_as_uint(a), p[e + 1] = __float_as_uint(d);
      exp2_pair(e + 2, fma2(pair_of(p[e + 2], p[e + 3]), c, l1), a, d);
      p[e + 2] = __float_as_uint(a), p[e + 3] = __float_as_uint(d);
    }
    if constexpr (KEYS) {
      uint32_t q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = pack_bf16x2(__uint_as_float(p[part * 16 + 2 * e]), __uint_as_float(p[part * 16 + 2 * e + 1]));
      const uint32_t seen = whole ? 0xffffffffu : columns_seen(first, last, sinks) >> (part * 16);
      if constexpr (TWO) {
        uint32_t left[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) left[e] = seen_pair(left_of(__uint_as_float(p[part * 16 + 2 * e]), __uint_as_float(p[part * 16 + 2 * e + 1]), q[e]), seen, e);
        tmem_st_32x8(t1 + OP_SECOND + part * 8, left);
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] = seen_pair(q[e], seen, e);
      }
      tmem_st_32x8(t1 + part * 8, q);   // over columns that this warp has read
      hand_over(cta, L::PROBS + part);
    }
  }
  if (!cta.wait(L::T2, i & 1, DEV_ERR_TMEM_FULL_TIMEOUT)) return false;
  tc_fence_after();
  uint32_t o[16], left[16];
  constexpr int COLS = TWO ? 16 : 32;   // at a time, as in the forward pass
#pragma unroll
  for (int from = 0; from < 32; from += COLS) {
    uint32_t y[COLS];
    tmem_ld_cols(t2 + from, y);
    tmem_ld_wait();
#pragma unroll
    for (int e = from; e < from + COLS; e += 4) {
      Pair d0, d1;
      row_numbers(1, e, d0, d1);
      float a, d;
      (pair_of(p[e], p[e + 1]) * (pair_of(y[e - from], y[e - from + 1]) + d0)).to(a, d);
      o[e / 2] = pack_bf16x2(a, d);
      if constexpr (TWO) left[e / 2] = left_of(a, d, o[e / 2]);
      (pair_of(p[e + 2], p[e + 3]) * (pair_of(y[e - from + 2], y[e - from + 3]) + d1)).to(a, d);
      o[e / 2 + 1] = pack_bf16x2(a, d);
      if constexpr (TWO) left[e / 2 + 1] = left_of(a, d, o[e / 2 + 1]);
    }
  }
  if (!whole) hide(o);
  tmem_st_32x16(KEYS ? t2 : t1, o);
  if constexpr (TWO) {
    if (!whole) hide(left);
    tmem_st_32x16((KEYS ? t2 : t1) + OP_SECOND, left);
  }
  hand_over(cta, L::GRADS);
  return true;
}
// The same of a sequence's first tile, whose rows see few keys, in a launch with one operand. Called, too: as part of the loop it cost the other tiles 5 to 9 %, as it is 1 %
// over 16384 tokens with a window of 1024 (dk and dv 543 -> 553 us, dq as before) and 5 % over 4096 without (227 -> 239, where such tiles are in the longest walks).
template <class L, bool KEYS>
__device__ __noinline__ bool first_tile_gradients(AttnCta cta, uint32_t i, uint32_t t1, uint32_t t2, int r, int c0, int window, int all_sinks, Pair c, const ulonglong2* stat,
                                                  float my_lse, float my_delta) {
  return tile_gradients<L, KEYS, true>(cta, i, t1, t2, r, 0, c0, window, all_sinks, c, stat, my_lse, my_delta);
}

template <int HD, bool KEYS, bool FINE>
__global__ void __launch_bounds__(AttnBwdRoles::THREADS, 1)
    attention_bwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                         const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmSinks, const __grid_constant__ CUtensorMap tmG,
                         const float* minus_lse, const float* minus_delta,
                         bf16* dv, bf16* dk, AttnShape s,
                         AttnSplit split, int items, int* err_word) {
  using L = AttnBwd<HD, KEYS>;
  using R = AttnBwdRoles;
  using Item = AttnBwdItem<KEYS>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const AttnCta cta = attn_begin<R, L::TILES, L::BARS>(smem_raw, err_word, [](int i) { return i >= L::READ && i < L::CLEAR1 ? R::LOAD : 1; });
  grid_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // numbers of passing tiles count over all items
  auto pass1 = [&](uint32_t i) { return cta.smem + L::PASS1 + i % L::N1 * L::TILE; };
  auto pass2 = [&](uint32_t i) { return cta.smem + L::PASS2 + i % L::N2 * L::TILE; };
  auto full1 = [&](uint32_t i) { return cta.wait(L::FULL1 + i % L::N1, i / L::N1 & 1, DEV_ERR_FULL_BAR_TIMEOUT); };
  auto full2 = [&](uint32_t i) { return cta.wait(L::FULL2 + i % L::N2, i / L::N2 & 1, DEV_ERR_FULL_BAR_TIMEOUT); };

  if (warp == R::LOAD) {
    // ---------------------------------------------------------------- loads
    if (elect_one_sync()) {
      uint32_t i = 0, held = 0;
      bool ok = true;
      for (int turn = 0; ok && dealt(turn) < items; ++turn) {
        const Item w(s, split, dealt(turn));
        if (w.n == 0) continue;
        if (!(ok = cta.wait(L::HELD_READ, (held++ & 1) ^ 1, DEV_ERR_EMPTY_BAR_TIMEOUT))) break;
        mbar_expect_tx(cta.bar(L::THERE), 2 * L::TILE);
        load_tile<HD, ATT_TILE>(cta.smem, KEYS ? &tmK : &tmQ, w.b, w.head, w.r0, cta.bar(L::THERE));
        load_tile<HD, ATT_TILE>(cta.smem + L::TILE, KEYS ? &tmV : &tmD, w.b, w.head, w.r0, cta.bar(L::THERE));
        int at = 0, head = w.first_head;
        for (int k = 0; k < w.n; ++k, ++i) {
          const int row = w.row(at);
          const uint32_t bar1 = cta.bar(L::FULL1 + i % L::N1), bar2 = cta.bar(L::FULL2 + i % L::N2);
          if (!(ok = cta.wait(L::EMPTY1 + i % L::N1, (i / L::N1 & 1) ^ 1, DEV_ERR_EMPTY_BAR_TIMEOUT))) break;
          mbar_expect_tx(bar1, L::TILE + (KEYS ? L::STATS : 0));
          load_tile<HD, ATT_TILE>(pass1(i), KEYS ? &tmQ : at < w.far ? &tmSinks : &tmK, w.b, head, row, bar1);
          if constexpr (KEYS) {
            const uint32_t stats = cta.smem + L::STAT + i % L::N1 * L::STATS;
            const int64_t from = (static_cast<int64_t>(w.b) * s.nq + head) * s.rows + row;
            bulk_load(stats, minus_lse + from, ATT_TILE * 4, bar1);
            bulk_load(stats + ATT_TILE * 4, minus_delta + from, ATT_TILE * 4, bar1);
          }
          if (!(ok = cta.wait(L::EMPTY2 + i % L::N2, (i / L::N2 & 1) ^ 1, DEV_ERR_EMPTY_BAR_TIMEOUT))) break;
          mbar_expect_tx(bar2, L::TILE);
          load_tile<HD, ATT_TILE>(pass2(i), KEYS ? &tmD : &tmV, w.b, head, row, bar2);
          if (++at == w.per_head) at = 0, ++head;
        }
      }
      grid_release();
    }
  } else if (warp == R::MMA) {
    // ---------------------------------------------------------------- products. Of one thread they run in the order of their issue
    if (elect_one_sync()) {
      uint32_t base = 0, held = 0, cleared1 = 0, cleared2 = 0;
      bool ok = true;
      for (int turn = 0; ok && dealt(turn) < items; ++turn) {
        const Item w(s, split, dealt(turn));
        const int n = w.n;
        if (n == 0) continue;
        if (!(ok = cta.wait(L::THERE, held++ & 1, DEV_ERR_FULL_BAR_TIMEOUT))) break;
        int left1 = w.per_head, left2 = w.per_head;   // tiles of a head that are to come, of each of the passing tensors
        auto t1 = [&](int k) {
          const uint32_t i = base + k;
          if (!(ok = full1(i))) return;
          if (--left1 == 0) {
            left1 = w.per_head;
            if (w.clear_from < ATT_TILE) {
              mbar_arrive(cta.bar(L::CLEAR1));
              if (!(ok = cta.wait(L::CLEARED1, cleared1++ & 1, DEV_ERR_FULL_BAR_TIMEOUT))) return;
            }
          }
          tc_fence_after();
          const int two = KEYS ? 0 : i & 1;
          multiply_rows<HD>(L::T1_COL + two * 128, cta.smem, pass1(i));
          umma_commit(cta.bar(L::T1 + two));
        };
        auto t2 = [&](int k) {
          const uint32_t i = base + k;
          if (!(ok = full2(i))) return;
          if (--left2 == 0) {
            left2 = w.per_head;
            if (w.clear_from < ATT_TILE) {
              mbar_arrive(cta.bar(L::CLEAR2));
              if (!(ok = cta.wait(L::CLEARED2, cleared2++ & 1, DEV_ERR_FULL_BAR_TIMEOUT))) return;
            }
          }
          tc_fence_after();
          multiply_rows<HD>(L::T2_COL, cta.smem + L::TILE, pass2(i));
          umma_commit(cta.bar(L::T2));
          if constexpr (!KEYS) umma_commit(cta.bar(L::EMPTY2 + i % L::N2));
          if (k + 1 == n) umma_commit(cta.bar(L::HELD_READ));   // the last product with a held tile
        };
        // sum += operand tile; the operand of each group's 32 columns lies over those columns
        auto add = [&](uint32_t acc, uint32_t operand, uint32_t tile_at, bool begun, bool two, int freed) {
          const uint32_t low = TileDesc<ATT_TILE, true>::low(tile_at);
          multiply_step<HD, OP_GROUP>(acc, operand, low, 0, begun);
#pragma unroll
          for (int k = 1; k < ATT_TILE / 16; ++k) multiply_step<HD, OP_GROUP>(acc, operand, low, k, true);
          if constexpr (FINE) {
#pragma unroll
            for (int k = 0; k < ATT_TILE / 16; ++k) multiply_step<HD, OP_GROUP>(acc, operand + OP_SECOND, low, k, true);
          } else if (two) {
            multiply_second<HD, 0xFF>(acc, operand, low);
          }
          umma_commit(cta.bar(freed));
        };
        t1(0);
        if (ok) t2(0);
        if (!KEYS && ok && n > 1) t1(1);
        // of a sequence's first tile of queries: with KEYS the one that each head begins with, by what t2 has left of a head then
        const bool first = !FINE && few_keys_from(w.r0) && w.part == 0;
        const int left_at_first = !first ? -1 : w.per_head == 1 ? 1 : w.per_head - 1;
        for (int k = 0; k < n && ok; ++k) {
          const uint32_t i = base + k;
          const bool two = KEYS ? left2 == left_at_first : first;
          if constexpr (KEYS) {
            // in two parts, of 16 columns of every group, as they are there
            const uint32_t low = TileDesc<ATT_TILE, true>::low(pass2(i));
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              if (!(ok = ok && cta.wait(L::PROBS + part, i & 1, DEV_ERR_TMEM_EMPTY_TIMEOUT))) break;
              tc_fence_after();
              multiply_step<HD, OP_GROUP>(L::ACC1_COL, L::T1_COL, low, part, part || k > 0);
#pragma unroll
              for (int step = 2; step < ATT_TILE / 16; step += 2) multiply_step<HD, OP_GROUP>(L::ACC1_COL, L::T1_COL, low, step + part, true);
              if constexpr (FINE) {
#pragma unroll
                for (int step = 0; step < ATT_TILE / 16; step += 2) multiply_step<HD, OP_GROUP>(L::ACC1_COL, L::T1_COL + OP_SECOND, low, step + part, true);
              } else if (two) {
                multiply_second<HD, 0x55>(L::ACC1_COL, L::T1_COL + part * 8, low + part * TileDesc<ATT_TILE, true>::step(1));
              }
            }
            if (!ok) break;
            umma_commit(cta.bar(L::EMPTY2 + i % L::N2));
            if (k + 1 < n) t1(k + 1);
          }
          if (!ok || !(ok = cta.wait(L::GRADS, i & 1, DEV_ERR_TMEM_EMPTY_TIMEOUT))) break;
          tc_fence_after();
          if (!KEYS && k + 1 < n) t2(k + 1);
          if (!ok) break;
          add(L::ACC2_COL, KEYS ? L::T2_COL : L::T1_COL + (i & 1) * 128, pass1(i), k > 0, two, L::EMPTY1 + i % L::N1);
          if (k + 1 == n) umma_commit(cta.bar(L::DONE));
          if (KEYS && k + 1 < n) t2(k + 1);
          if (!KEYS && k + 2 < n) t1(k + 2);
        }
        base += n;
      }
    }
  } else if (warp == R::ZERO) {
    // ---------------------------------------------------------------- rows behind a sequence's end, in the last tile of each head
    uint32_t base = 0, cleared = 0, before = 0;   // before: tiles at the last one
    bool ok = true;
    for (int turn = 0; s.lengths && ok && dealt(turn) < items; ++turn) {
      const Item w(s, split, dealt(turn));
      if (w.clear_from < ATT_TILE)
        for (int k = w.per_head - 1; k < w.n && ok; k += w.per_head, ++cleared) {
          const uint32_t i = base + k;
          if (!(ok = cta.wait(L::CLEAR1, cleared & 1, DEV_ERR_FULL_BAR_TIMEOUT, i + 1 - before) && full1(i))) break;
          zero_rows<HD, ATT_TILE>(pass1(i), w.clear_from, cta.bar(L::CLEARED1));
          if (!(ok = cta.wait(L::CLEAR2, cleared & 1, DEV_ERR_FULL_BAR_TIMEOUT, 2) && full2(i))) break;
          zero_rows<HD, ATT_TILE>(pass2(i), w.clear_from, cta.bar(L::CLEARED2));
          before = i;
        }
      base += w.n;
    }
  } else {
    // ---------------------------------------------------------------- probabilities: a thread has 32 columns of a row of the held tile
    const int w = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const Pair c = both(s.scale * ATT_LOG2E);
    const RowsOut slab{cta.smem + L::OUT + warp * 2048};
    const uint8_t* const stat_base = smem_raw + (cta.smem - smem_u32(smem_raw)) + L::STAT + w * 128;
    uint32_t i = 0, done = 0;
    bool ok = true;
    float my_lse = 0.f, my_delta = 0.f;
    auto fetch = [&](int turn) {   // lse and delta of a row of dq's items
      const int index = dealt(turn);
      if (KEYS || index >= items) return;
      const int nth = s.by_heads_q.quotient(index), of_all = index - nth * s.by_heads_q.d;
      const int64_t from = static_cast<int64_t>(of_all) * s.rows + s.rows - (nth + 1) * ATT_TILE + (warp & 3) * 32 + lane;
      my_lse = minus_lse[from];
      my_delta = minus_delta[from];
    };
    fetch(0);
#pragma unroll 1
    for (int turn = 0; ok && dealt(turn) < items; ++turn) {
      const Item walk(s, split, dealt(turn));
      const int r0 = walk.r0, r = r0 + (warp & 3) * 32 + lane, n = walk.n;
      int at = 0, k = 0;
      if (!FINE && !KEYS && few_keys_from(r0) && n > 0) {   // its only one
        const uint32_t t1 = lanes + L::T1_COL + (i & 1) * 128 + w * 32, t2 = lanes + L::T2_COL + w * 32;
        ok = cta.wait(L::T1 + (i & 1), i >> 1 & 1, DEV_ERR_TMEM_FULL_TIMEOUT);
        if (ok) {
          tc_fence_after();
          ok = first_tile_gradients<L, KEYS>(cta, i, t1, t2, r, w * 32, s.window, s.sinks, c, nullptr, my_lse, my_delta);
        }
        k = 1, ++i;
      }
#pragma unroll 1
      for (; k < n; ++k, ++i) {
        const int c0 = walk.row(at) + w * 32;
        // blocks far from the window of which no sink is part are zeros without a look at the scores
        const bool nothing = KEYS ? walk.part > 0 && r0 + (warp & 3) * 32 >= s.sinks : at < walk.far && c0 >= s.sinks;
        const bool first = few_keys_from(KEYS ? c0 - w * 32 : r0);
        if (++at == walk.per_head) at = 0;
        const uint32_t t1 = lanes + L::T1_COL + (KEYS ? 0 : (i & 1) * 128) + w * 32, t2 = lanes + L::T2_COL + w * 32;
        if constexpr (KEYS) {   // lse and delta of the stage
          if (!(ok = full1(i))) break;
        }
        if (!(ok = cta.wait(KEYS ? L::T1 : L::T1 + (i & 1), KEYS ? i & 1 : i >> 1 & 1, DEV_ERR_TMEM_FULL_TIMEOUT))) break;
        tc_fence_after();
        if (nothing) {
          uint32_t zeros[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) zeros[e] = 0;
          tmem_st_32x16(t1, zeros);
          if constexpr (FINE) tmem_st_32x16(t1 + OP_SECOND, zeros);
          if constexpr (KEYS) {
            hand_over(cta, L::PROBS);
            if (lane == 0) mbar_arrive(cta.bar(L::PROBS + 1));
          }
          // T2 comes behind the tile before, whose gradients all warps have handed over then: dq's T1 may be there before that
          if (!(ok = cta.wait(L::T2, i & 1, DEV_ERR_TMEM_FULL_TIMEOUT))) break;
          tc_fence_after();
          if constexpr (KEYS) {
            tmem_st_32x16(t2, zeros);
            if constexpr (FINE) tmem_st_32x16(t2 + OP_SECOND, zeros);
          }
          hand_over(cta, L::GRADS);
          continue;
        }
        const ulonglong2* const stat = reinterpret_cast<const ulonglong2*>(stat_base + i % L::N1 * L::STATS);
        if (!FINE && KEYS && first)
          ok = first_tile_gradients<L, KEYS>(cta, i, t1, t2, r, c0, s.window, s.sinks, c, stat, my_lse, my_delta);
        else
          ok = tile_gradients<L, KEYS, FINE>(cta, i, t1, t2, r, r0, c0, s.window, s.sinks, c, stat, my_lse, my_delta);
        if (!ok) break;
      }
      // ---------------------------------------------------------------- what the sums became
      fetch(turn + 1);   // while the last products run
      const Item it(s, split, dealt(KEYS ? anew(turn) : turn));
      if (ok && it.n > 0) ok = cta.wait(L::DONE, done++ & 1, DEV_ERR_TMEM_FULL_TIMEOUT);
      tc_fence_after();
      const bool full = ok && it.n > 0, mine = it.r0 + (warp & 3) * 32 + lane < it.len;
      // KEYS: the first two groups of warps have dv, the others dk, half of the columns each; dq's columns are shared by four
      constexpr int COLS = KEYS ? HD / 2 : HD / 4;
      const int which = KEYS ? w >> 1 : 1, col = (KEYS ? w & 1 : w) * COLS;
      const uint32_t acc = lanes + (which ? L::ACC2_COL : L::ACC1_COL) + col;
      const float f = which ? s.scale : 1.f;
      const int row0 = it.r0 + (warp & 3) * 32;   // the warp's
      auto load = [&](int c, uint32_t(&o)[16]) {   // 16 columns, scaled
        if (full) {
          tmem_ld_32x16(acc + c, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = full && mine ? __float_as_uint(__uint_as_float(o[e]) * f) : 0u;
      };
      auto two = [](const uint32_t(&o)[16], int e) { return pack_bf16x2(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1])); };
      if constexpr (KEYS) {
        // from registers, 6000 clocks of a tile's 110000: through shared memory the walk's loop is left too few registers (226 -> 284 us)
        bf16* const grad = (which ? dk : dv) + ((static_cast<int64_t>(it.b) * s.S + row0 + lane) * s.nkv + it.head) * HD + col;
        float* sums = nullptr;
        if (it.joined) {
          const int64_t heads = static_cast<int64_t>(s.B) * s.nkv, place = (it.part * split.tiles + it.tile) * heads + it.b * s.nkv + it.head;
          sums = split.sums + ((place * 2 + which) * ATT_TILE + (warp & 3) * 32 + lane) * HD + col;
        }
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
          uint32_t o[16];
          load(c, o);
          if (it.joined) {
            if (it.part == 0 || row0 + lane < s.sinks)   // from far away only sinks are seen
#pragma unroll
              for (int e = 0; e < 4; ++e) reinterpret_cast<uint4*>(sums + c)[e] = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          } else if (row0 + lane < s.S) {
            uint4* const at = reinterpret_cast<uint4*>(grad + c);
            at[0] = make_uint4(two(o, 0), two(o, 1), two(o, 2), two(o, 3));
            at[1] = make_uint4(two(o, 4), two(o, 5), two(o, 6), two(o, 7));
          }
        }
      } else {
        uint32_t o[16], packed[COLS / 2];
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
          load(c, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) packed[c / 2 + e] = two(o, e);
        }
        slab.free();
        slab.put(packed);
        slab.out(&tmG, col, it.head, row0, it.b);
      }
      tc_fence_before();   // the sums are read
    }
    if (!KEYS && lane == 0) tma_store_wait<0>();
  }
  attn_end<R>(cta);
}

// The gradients of tiles whose walk was split: their parts' sums, one after the other.
template <int HD>
__global__ void __launch_bounds__(256) attention_join_kernel(AttnSplit split, bf16* dv, bf16* dk, AttnShape s) {
  grid_wait();
  grid_release();
  constexpr int VECS = ATT_TILE * HD / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, tiles = static_cast<int64_t>(s.B) * s.nkv * split.tiles;
  if (at >= tiles * 2 * VECS) return;
  const int64_t which = at / VECS;
  const int v = static_cast<int>(at % VECS), w = static_cast<int>(which & 1);
  const int64_t place = which >> 1;
  const int tile = static_cast<int>(place / (s.B * s.nkv)), bh = static_cast<int>(place % (s.B * s.nkv));
  const int row = tile * ATT_TILE + v / (HD / 4), col = v % (HD / 4) * 4;
  if (row >= s.S) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* from = reinterpret_cast<const float4*>(split.sums) + at;
  const int parts = row < s.sinks ? split.parts : 0;   // beside the window's, which all rows have
#pragma unroll 8
  for (int p = 0; p <= parts; ++p) {
    const float4 x = from[p * tiles * 2 * VECS];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  bf16* to = (w ? dk : dv) + ((static_cast<int64_t>(bh / s.nkv) * s.S + row) * s.nkv + bh % s.nkv) * HD + col;
  *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
}

// [B][S][heads][hd] with element strides {batch, token, head}. Boxes to load: 64 rows x 64 elements of a head; to store: 32 rows x `store` elements of
// `bytes` bytes, 32 of bf16 in the 64-byte swizzle.
static int attn_map(CUtensorMap* m, const B200AttnTensor& t, int B, int S, int heads, int hd, int store = 0, int bytes = 2) {
  EncodeTiledFn enc = get_encode_tiled();
  if (!enc) return B200_ERR_NO_DRIVER;
  auto pitch = [&](int size, long long stride) { return static_cast<cuuint64_t>(size == 1 ? hd : stride) * bytes; };   // of a single one any will do
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {pitch(heads, t.head), pitch(S, t.token), pitch(B, t.batch)};
  const cuuint32_t box[4] = {store ? static_cast<cuuint32_t>(store) : 64u, 1, store ? 32u : static_cast<cuuint32_t>(ATT_BOX), 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(t.data), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE,
                         store * bytes == 64 && bytes == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : store ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return 0;
  fprintf(stderr, "[b200ops] cuTensorMapEncodeTiled failed: %d (base=%p, %d x %d x %d x %d)\n", static_cast<int>(r), t.data, B, S, heads, hd);
  return B200_ERR_TENSORMAP;
}
static bool attn_tensor_ok(const B200AttnTensor& t, int B, int S, int heads) {
  auto fits = [](int size, long long stride) { return size == 1 || (stride > 0 && stride % 8 == 0 && stride < (1ll << 38)); };
  return t.data && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && fits(B, t.batch) && fits(S, t.token) && fits(heads, t.head);
}
static bool attn_shape(AttnShape& s, const B200AttnArgs& a) {
  if (a.B < 1 || a.S < 1 || a.nkv < 1 || a.nq < 1 || a.nq % a.nkv || (a.hd != 64 && a.hd != 128) || a.window < 0 || a.sinks < 0 || !(a.scale > 0.f)) return false;
  if (static_cast<int64_t>(a.S) > (1 << 30)) return false;
  s.B = a.B, s.S = a.S, s.nq = a.nq, s.nkv = a.nkv, s.G = a.nq / a.nkv;
  s.rows = (a.S + ATT_TILE - 1) / ATT_TILE * ATT_TILE;
  // items' numbers have 32 bits
  if (static_cast<int64_t>(s.B) * s.nq >= (1 << 30) || static_cast<int64_t>(s.B) * s.nq * (s.rows / ATT_TILE) >= (1 << 30)) return false;
  // a window that holds every key, or sinks that are, is none
  s.window = a.window >= a.S || (a.window > 0 && a.sinks >= a.S) ? 0 : a.window;
  s.sinks = s.window ? a.sinks : 0;
  s.lengths = a.lengths;
  s.scale = a.scale;
  s.by_G = Divisor(s.G), s.by_nq = Divisor(s.nq), s.by_nkv = Divisor(s.nkv), s.by_heads_q = Divisor(s.B * s.nq), s.by_heads_kv = Divisor(s.B * s.nkv);
  return true;
}

// Launches all of whose rows see at most 128 keys (FINE) take two operands in every tile; in others the first tile of each sequence does. One rounding of an operand is up
// to 2^-8; many keys make 2^-9.3 in the mean of it, few do not, and in delta, of the output, it comes once more: over 3 to 8 tokens dq and dk were off by 2.6e-3 to 3.4e-3, from 33
// to 128 keys by 2.5e-3, now by 1.7e-3, which is their own rounding. Rows of more keys stay at 2.4e-3: with two
// operands 16384 tokens of 32 heads and a window of 128 take 130 us forward and 396 for dk, dv and dq, with one and a window of 129 97 and 314.
static bool few_keys(const AttnShape& s) { return (s.window ? std::min(s.S, s.window + s.sinks) : s.S) <= ATT_TILE; }

// k or v with no tokens but its sinks, of which tiles far from a window are made: what lies behind the sinks would reach every later row where it is not finite, since
// its products with zero are not zero. TMA fills those rows with zeros. The tensor's own map where no tile is far, or sinks end with a tile.
static int sinks_map(CUtensorMap* m, const CUtensorMap& all, const B200AttnTensor& t, const AttnShape& s, int hd) {
  if (s.sinks % ATT_TILE && s.rows - ATT_TILE - s.window + 1 >= ATT_TILE) return attn_map(m, t, s.B, s.sinks, s.nkv, hd);
  *m = all;
  return 0;
}

template <int HD, bool FINE>
static int attn_fwd(const B200AttnArgs& a, const AttnShape& s, cudaStream_t stream) {
  CUtensorMap q, k, v, sinks, o, r;
  const long long row = static_cast<long long>(s.nq) * HD;
  if (int rc = attn_map(&o, {a.out, s.S * row, row, HD}, s.B, s.S, s.nq, HD, 32)) return rc;
  if (a.rest) {
    if (int rc = attn_map(&r, {a.rest, s.S * row, row, HD}, s.B, s.S, s.nq, HD, HD / 2, 1)) return rc;
  } else {
    r = o;
  }
  if (int rc = attn_map(&q, a.q, s.B, s.S, s.nq, HD)) return rc;
  if (int rc = attn_map(&k, a.k, s.B, s.S, s.nkv, HD)) return rc;
  if (int rc = attn_map(&v, a.v, s.B, s.S, s.nkv, HD)) return rc;
  if (int rc = sinks_map(&sinks, v, a.v, s, HD)) return rc;
  if (int rc = allow_smem<attention_fwd_kernel<HD, FINE>>(AttnFwd<HD>::SMEM)) return rc;
  const int items = s.B * s.nkv * ((s.rows / ATT_TILE * s.G + 1) / 2);
  launch_dependent(attention_fwd_kernel<HD, FINE>, std::min(items, sm_count()), AttnFwdRoles::THREADS, AttnFwd<HD>::SMEM, stream, q, k, v, sinks, o,
                   r, a.rest != nullptr, a.lse, s, items, device_status_word());
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

// The walk of a sink's tile is split where it is more than twice as long as a window's: into parts as long as that, but into no more than make some waves.
// Where such tiles alone make two waves they are whole items, the first to be dealt.
static AttnSplit attn_split(const AttnShape& s, float* sums) {
  AttnSplit p{0, 0, 0, Divisor(), sums};
  if (s.sinks == 0) return p;
  const int near = s.window / ATT_TILE + 2, all = s.rows / ATT_TILE;
  if (all <= 2 * near) return p;
  p.tiles = (s.sinks + ATT_TILE - 1) / ATT_TILE;
  const int64_t items = static_cast<int64_t>(s.B) * s.nkv * p.tiles, sms = sm_count();
  if (items >= 2 * sms) {
    p.tiles = 0;
    return p;
  }
  const int64_t most = 4 * sms / items;
  p.parts = static_cast<int>(std::min<int64_t>(most, (all - 1) / near));
  p.part_tiles = (all + p.parts - 1) / p.parts;
  p.by_part = Divisor(static_cast<int>(items));
  return p;
}

template <int HD, bool FINE>
static int attn_bwd(const B200AttnArgs& a, const AttnShape& s, cudaStream_t stream) {
  CUtensorMap q, k, v, d, g;
  if (int rc = attn_map(&q, a.q, s.B, s.S, s.nq, HD)) return rc;
  if (int rc = attn_map(&k, a.k, s.B, s.S, s.nkv, HD)) return rc;
  if (int rc = attn_map(&v, a.v, s.B, s.S, s.nkv, HD)) return rc;
  if (int rc = attn_map(&d, a.dout, s.B, s.S, s.nq, HD)) return rc;
  auto keys = attention_bwd_kernel<HD, true, FINE>;
  auto queries = attention_bwd_kernel<HD, false, FINE>;
  if (int rc = allow_smem<attention_bwd_kernel<HD, true, FINE>>(AttnBwd<HD, true>::SMEM)) return rc;
  if (int rc = allow_smem<attention_bwd_kernel<HD, false, FINE>>(AttnBwd<HD, false>::SMEM)) return rc;
  int* err = device_status_word();
  const int per_block = 256 / (HD / 8) * DELTA_ROWS;
  const int blocks = static_cast<int>((static_cast<int64_t>(s.rows) * s.nq + per_block - 1) / per_block);   // of a sequence
  auto stride = [](int size, long long x) { return size == 1 ? 0 : x; };
  launch_dependent(attention_delta_kernel<HD>, s.B * blocks, 256, 0, stream, static_cast<const bf16*>(a.dout.data),
                   stride(s.B, a.dout.batch), stride(s.S, a.dout.token), stride(s.nq, a.dout.head), static_cast<const bf16*>(a.out), static_cast<const uint8_t*>(a.rest), a.delta, s, blocks);
  const int tiles = s.rows / ATT_TILE;
  if (a.dk) {
    const AttnSplit split = attn_split(s, a.sums);
    const int items = s.B * s.nkv * (tiles + split.tiles * split.parts);
    launch_dependent(keys, std::min(items, sm_count()), AttnBwdRoles::THREADS, AttnBwd<HD, true>::SMEM, stream, q, k, v, d, k, d, a.lse, a.delta,
                     static_cast<bf16*>(a.dv), static_cast<bf16*>(a.dk), s, split, items, err);
    if (split.parts) {
      const int64_t n = static_cast<int64_t>(s.B) * s.nkv * split.tiles * 2 * (ATT_TILE * HD / 4);
      launch_dependent(attention_join_kernel<HD>, static_cast<int>((n + 255) / 256), 256, 0, stream, split, static_cast<bf16*>(a.dv),
                       static_cast<bf16*>(a.dk), s);
    }
  }
  if (a.dq) {
    const long long row = static_cast<long long>(s.nq) * HD;
    if (int rc = attn_map(&g, {a.dq, s.S * row, row, HD}, s.B, s.S, s.nq, HD, HD / 4)) return rc;
    CUtensorMap sinks;
    if (int rc = sinks_map(&sinks, k, a.k, s, HD)) return rc;
    const int items = s.B * s.nq * tiles;
    launch_dependent(queries, std::min(items, sm_count()), AttnBwdRoles::THREADS, AttnBwd<HD, false>::SMEM, stream, q, k, v, d, sinks, g, a.lse, a.delta,
                     static_cast<bf16*>(nullptr), static_cast<bf16*>(nullptr), s, AttnSplit{0, 0, 0, Divisor(), nullptr}, items, err);
  }
  B200_CUDA_OK(cudaGetLastError());
  return 0;
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_attention_fwd(const B200AttnArgs* args, void* stream) {
  ensure_context();
  const B200AttnArgs& a = *args;
  AttnShape s;
  if (!attn_shape(s, a) || !attn_tensor_ok(a.q, a.B, a.S, a.nq) || !attn_tensor_ok(a.k, a.B, a.S, a.nkv) || !attn_tensor_ok(a.v, a.B, a.S, a.nkv) || !a.out ||
      reinterpret_cast<uintptr_t>(a.out) % 16 || reinterpret_cast<uintptr_t>(a.rest) % 16 || !a.lse)
    return B200_ERR_BAD_ARG;
  const auto run = few_keys(s) ? a.hd == 128 ? attn_fwd<128, true> : attn_fwd<64, true> : a.hd == 128 ? attn_fwd<128, false> : attn_fwd<64, false>;
  return run(a, s, static_cast<cudaStream_t>(stream));
}

long long b200_attention_bwd_workspace(const B200AttnArgs* args) {
  AttnShape s;
  if (!attn_shape(s, *args)) return 0;
  const AttnSplit p = attn_split(s, nullptr);
  return p.parts ? static_cast<long long>(1 + p.parts) * s.B * s.nkv * p.tiles * 2 * ATT_TILE * args->hd : 0;
}

int b200_attention_bwd(const B200AttnArgs* args, int* launches, void* stream) {
  ensure_context();
  const B200AttnArgs& a = *args;
  AttnShape s;
  if (!attn_shape(s, a) || !attn_tensor_ok(a.q, a.B, a.S, a.nq) || !attn_tensor_ok(a.k, a.B, a.S, a.nkv) || !attn_tensor_ok(a.v, a.B, a.S, a.nkv) ||
      !attn_tensor_ok(a.dout, a.B, a.S, a.nq) || !a.out || reinterpret_cast<uintptr_t>(a.out) % 16 || !a.lse || reinterpret_cast<uintptr_t>(a.lse) % 16 ||
      !a.delta || reinterpret_cast<uintptr_t>(a.delta) % 16 || !a.dk != !a.dv || reinterpret_cast<uintptr_t>(a.rest) % 16 || reinterpret_cast<uintptr_t>(a.dq) % 16 ||
      reinterpret_cast<uintptr_t>(a.dk) % 16 || reinterpret_cast<uintptr_t>(a.dv) % 16)
    return B200_ERR_BAD_ARG;
  const AttnSplit p = attn_split(s, nullptr);
  if (a.dk && p.parts && (!a.sums || reinterpret_cast<uintptr_t>(a.sums) % 16)) return B200_ERR_BAD_ARG;
  if (launches) *launches = 1 + (a.dk ? 1 + (p.parts > 0) : 0) + (a.dq ? 1 : 0);
  const auto run = few_keys(s) ? a.hd == 128 ? attn_bwd<128, true> : attn_bwd<64, true> : a.hd == 128 ? attn_bwd<128, false> : attn_bwd<64, false>;
  return run(a, s, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
