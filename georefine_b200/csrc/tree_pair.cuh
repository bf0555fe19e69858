// The wide attention of tree_wide.cuh over a 4-bit cache: two tiles of 128 rows (row of the step, query head of the group) share each step's K and V.
//
// A CTA takes all of an SM.  Two warpgroups turn scores into weights, one for each tile, a thread per row; one brings K and one V, which they decode to FP16 in
// shared memory once for both tiles, their codes asked for two steps ahead; two warps issue the products, one for each tile; one looks up where the next unit lies:
//   S = Q K^T (S in tensor memory, two steps of each tile);  weights P = exp2(S' - reference), written over S;  O += P V (P and O in tensor memory).
// A step is 64 positions; K and V of three steps are held.  Arithmetic is that of tree_wide.cuh: K's exponent multiplies the score of its position, V's goes
// into the weight, the sum of the weights takes it out again; the reference of a row moves when its maximum has passed it by 2^8.  Queries and weights are FP16, one term
// each (what that costs: tree_q4.cuh); references, sums and O are FP32.
//
// A unit is a pair of tiles and a part of the positions.  Where a run's last tile has no partner, the products' and the weights' warps of the other half go through
// all waits and arrivals without anything between them.  Barriers of a step are numbered by the step modulo three.  A wait tells a phase from the one before it and
// no more, so nobody may be a round ahead of one who still waits, and nobody waits for a phase whose predecessor is open: everybody waits for every step in turn,
// and the loaders for the products of the step whose place they take.  (tests/test_pair_schedule.py runs these waits and arrivals in any order.)
//
// No single unit bounds it.  A step of two full tiles takes 3100 cycles: the warps that turn scores into weights work 2400 of them, at an instruction in five cycles or
// so each; the products 1380 (two of S at 434 - the queries are read again for every 64 positions - and two of O at 257), shared memory 2800 (the products 1024, the rest
// mostly exponents that the weights' warps read), exp2 1024.  384 prompt rows behind 8000 positions, 40 heads of 8: 126 us, 510 TFLOP/s; 16 trees of 64 nodes
// behind 4096 to 8192: 340, of which 290 are this kernel (over 8 bits 322: 64 nodes are 25 + 25 + 14 rows, so that half of the pairs have one tile).  What lies between units was dear: the queries' addresses with a division each kept a unit waiting for 4500 cycles (142
// and 381).  (Two threads a row: 4 % slower; four threads for both tiles' rows at a time, whose exponents they read once: 40 %; weights by the reference as it is,
// in one pass over the columns, done again where it moves: 17 %; K's exponents in the operands as far as they differ: 3 and 11 %.)
#pragma once
#include "tree_q4.cuh"
#include "tree_wide.cuh"

namespace grb {

constexpr int kPairThreads = 640;                // weights of tile 0, of tile 1: warps 0-3, 4-7; K and the queries: 8-11; V: 12-15; products: 16, 17; units: 18
constexpr uint32_t kPairRing = 3;
constexpr uint32_t kPairScales = 8;              // steps whose exponents are held: the one five before a step whose K may be stored has been weighed
constexpr uint32_t kPairColumns = 512;           // tensor memory: S of two steps (and P over it) of tile 0, of tile 1, O of either

// What everybody is told of a unit.
struct PairInfo {
  uint32_t valid, first, rows, kvh, part, steps;
  uint32_t plain;                  // steps, from the first on, whose positions every row sees
  int32_t start, extent;           // positions start .. extent - 1: what some row sees, up to the last such
};
// What the exponents of a step's entries mean: 2^e of K; e and 2^-e of V.
struct PairScales {
  float k[kWideStep], v[kWideStep], v_inverse[kWideStep];
};
struct PairShared {
  uint64_t bars[2 * kPairRing + 3 * 2 * kPairRing + 3 + 8];      // K stored, V stored; S done, O done, P stored, of either tile; unit set up, unit seen, queries stored; scales
  PairInfo info[2];                              // of a unit and the next
  int64_t where[2][kWideMostPart / kWideStep];   // first entry of each step; -1: none
  uint32_t tmem_at, aborted;
};
constexpr uint32_t kPairSharedBytes = 2048;
static_assert(sizeof(PairShared) <= kPairSharedBytes, "the operands follow");
constexpr uint32_t kPairSmem = kPairSharedBytes + 2 * kWideOperand + 2 * kPairRing * kWideStage + kPairScales * uint32_t(sizeof(PairScales));

__global__ void __launch_bounds__(kPairThreads, 1)
tree_pair_kernel(const TreeArgs a) {
  extern __shared__ __align__(1024) unsigned char wide_smem[];
  PairShared& sm = *reinterpret_cast<PairShared*>(wide_smem);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t qs = smem_u32(wide_smem) + kPairSharedBytes, ks = qs + 2 * kWideOperand, vs = ks + kPairRing * kWideStage;
  PairScales* const scales = reinterpret_cast<PairScales*>(wide_smem + kPairSharedBytes + 2 * kWideOperand + 2 * kPairRing * kWideStage);
  constexpr uint32_t kRound = 8 * kPairRing;
  const uint32_t bar_k = smem_u32(&sm.bars[0]), bar_v = bar_k + kRound, bar_s = bar_v + kRound, bar_o = bar_s + 2 * kRound, bar_p = bar_o + 2 * kRound, bar_u = bar_p + 2 * kRound,
                 bar_w = bar_u + 8, bar_q = bar_w + 8, bar_t = bar_q + 8;
  // (tensor memory is taken before the kernels behind this one may start: see tree_wide_kernel)
  if (tid == 0) {
    for (uint32_t b = 0; b < kRound; b += 8) {
      mbar_init(bar_k + b, 4);
      mbar_init(bar_v + b, 4);
    }
    for (uint32_t b = 0; b < 2 * kRound; b += 8) {
      mbar_init(bar_s + b, 1);
      mbar_init(bar_o + b, 1);
      mbar_init(bar_p + b, 4);
    }
    mbar_init(bar_u, 1);
    mbar_init(bar_w, 18);
    mbar_init(bar_q, 4);
    for (uint32_t b = 0; b < 8 * kPairScales; b += 8) mbar_init(bar_t + b, 8);
    mbar_fence_init();
    sm.aborted = 0u;
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(&sm.tmem_at), kPairColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  step_kernel_entry();
  const uint32_t tiles = a.plan[2], units = a.plan[3], tile_rows = a.wide_rows / 2;
  if (blockIdx.x >= units) {
    if (warp == 16) tmem_dealloc(sm.tmem_at, kPairColumns);
    return;
  }
  // A wait that runs out is everybody's: nobody waits again, every loop runs to its end, and the status says so.
  auto wait = [&](uint32_t bar, uint32_t phase) {
    if (mbar_test_wait(bar, phase & 1u) || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) return;
    if (!mbar_wait(bar, phase & 1u, false)) {
      *reinterpret_cast<volatile uint32_t*>(&sm.aborted) = 1u;
      atomicOr(a.status, kStatusTimeout);
    }
  };
  auto wait3 = [&](uint32_t bars, uint32_t step) { wait(bars + 8 * (step % kPairRing), step / kPairRing); };
  uint32_t step0 = 0;                                        // steps this CTA has taken before the unit
  // registers, of the 96 that each thread of the launch has: 144 for the weights, 72 for loading, 48 for the others
  if (warp >= 8 && warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---- loading: K and the queries, or V -------------------------------------------------------------------------
    const bool of_k = warp < 12;
    const uint32_t lt = tid & 127u, ring = of_k ? ks : vs, stored = of_k ? bar_k : bar_v, left = of_k ? bar_s : bar_o;      // left: a stage's last use
    const uint8_t* const pool = static_cast<const uint8_t*>(of_k ? a.pages.k : a.pages.v);
    // A thread's pieces of a step: the same group of 32 dimensions of every 32nd row; the lanes of the upper two groups take their words in another order, so
    // that no two of eight lanes store to the same banks.  The first 64 threads also bring a position's exponent.
    const uint32_t row0 = lt >> 2, swapped = lt & 2u;
    const uint32_t per_group = 65536u / a.group + 1u;        // a column of 256 over the group, in units of 2^-16
    uint32_t to_word[4];                                     // where a piece's words, eight dimensions each, go
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) to_word[q] = wide_offset<kWideStep>(row0, 4 * (lt & 3u) + (q ^ swapped));
    struct Pieces {
      uint4 x[2];
      uint32_t scale;                                        // of the two, in bits 0-7 and 16-23
      uint32_t exp;
    };
    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1u;
      wait(bar_u, n);
      const PairInfo unit = sm.info[slot];
      if (!unit.valid || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_w);
      const uint32_t steps = unit.steps;
      auto ask = [&](Pieces& p, uint32_t j) {
        const int64_t entry = j < steps ? sm.where[slot][j] : -1;
        const int32_t npos = entry < 0 ? 0 : unit.extent - unit.start - int32_t(j * kWideStep);
        const uint8_t* const page = pool + (entry < 0 ? 0 : q4_page_at(size_t(entry)));
        const uint32_t place = uint32_t(entry) % kKvPage;
        p.scale = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t at = place + row0 + 32 * i;
          const bool in = int32_t(row0 + 32 * i) < npos;
          p.x[i] = in ? reinterpret_cast<const uint4*>(page)[at * (kQ4Codes / 16) + (lt & 3u)] : make_uint4(0u, 0u, 0u, 0u);
          if (in) p.scale |= uint32_t(page[kQ4ScalesAt + at * 4 + (lt & 3u)]) << (16 * i);
        }
        p.exp = lt < kWideStep && entry >= 0 ? page[kQ4ExpsAt + place + lt] : 127u;
      };
      auto store = [&](const Pieces& p, uint32_t g) {
        const uint32_t stage = g % kPairRing, dst = ring + stage * kWideStage;
        if (g >= kPairRing) {
          wait3(left, g - kPairRing);
          wait3(left + kRound, g - kPairRing);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const Q4Factors f = q4_factors((p.scale >> (16 * i) & 0xFFu) * 0x10001u);
          const uint32_t words[4] = {swapped ? p.x[i].z : p.x[i].x, swapped ? p.x[i].w : p.x[i].y, swapped ? p.x[i].x : p.x[i].z, swapped ? p.x[i].y : p.x[i].w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t y[4];
            q4_operands(words[q], f, y);
            sts128(dst + 4096 * i + to_word[q], make_uint4(y[0], y[1], y[2], y[3]));
          }
        }
        if (lt < kWideStep) {                                // (a byte below what an entry has - 0, where nobody wrote - stands for zeros of the smallest size)
          PairScales& s = scales[g % kPairScales];
          if (of_k) {
            s.k[lt] = kv_scale(p.exp);
          } else {
            const uint32_t b = max(p.exp, kKvLeastByte);
            s.v[lt] = b == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(b) - 127);
            s.v_inverse[lt] = kv_inverse(b);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar_t + 8 * (g % kPairScales));
          mbar_arrive(stored + 8 * stage);
        }
      };
      Pieces p0, p1;
      ask(p0, 0);
      ask(p1, 1);
      if (of_k) {                                            // the queries of both tiles, once the scores of the unit before are done
        if (step0) {
          wait3(bar_s, step0 - 1);
          wait3(bar_s + kRound, step0 - 1);
        }
        // (piece lt % 16 of every eighth column; column c of the two tiles lies c + c / group (nq - group) heads behind the first)
        const uint32_t used = unit.rows * a.group, first_tile = tile_rows * a.group;
        const uint16_t* const src = a.q + (size_t(unit.first) * a.nq + unit.kvh * a.group) * kKvDim + 8 * (lt & 15u);
        const uint32_t next_row = (a.nq - a.group) * kKvDim;
#pragma unroll 1
        for (uint32_t y = 0; y < (unit.rows > tile_rows ? 2u : 1u); ++y) {
          const uint32_t dst = qs + y * kWideOperand + wide_offset<kWideTile>(lt >> 4, lt & 15u);
#pragma unroll 4
          for (uint32_t i = 0; i < kWideTile / 8; ++i) {
            const uint32_t m = (lt >> 4) + 8 * i, column = y * first_tile + m;
            const bool in = column < used && m < first_tile;
            cp_async_16(dst + 1024 * i, in ? src + (column * kKvDim + (column * per_group >> 16) * next_row) : src, in ? 16u : 0u);
          }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q);
      }
      for (uint32_t j = 0; j < steps; j += 2) {
        store(p0, step0 + j);
        ask(p0, j + 2);
        if (j + 1 < steps) {
          store(p1, step0 + j + 1);
          ask(p1, j + 3);
        }
      }
      step0 += steps;
    }
  } else if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 18) {
      // ---- units: where the next one lies, while this one is at hand ------------------------------------------------
      uint32_t tile = 0, n = 0;
      for (uint32_t u = blockIdx.x; u < units; ++n) {
        const uint32_t slot = n & 1u;
        for (;;) {
          const uint32_t past = __ballot_sync(0xFFFFFFFFu, tile + 1 + lane < tiles && uint32_t(a.wide_tiles[tile + 1 + lane].z) <= u);
          tile += __popc(past);
          if (past != 0xFFFFFFFFu) break;
        }
        const int4 d = a.wide_tiles[tile];
        const uint32_t local = u - uint32_t(d.z), part_positions = uint32_t(d.w), first = uint32_t(d.x), rows = uint32_t(d.y), kvh = local % a.nkv, part = local / a.nkv;
        const int32_t seq = a.row_seq[first], start = int32_t(part * part_positions);
        int64_t place = 0, entry = 0;                        // (a step's positions lie in one page)
        if (lane < part_positions / kWideStep) {
          place = kv_place(a.table, seq, start + int32_t(lane * kWideStep));
          entry = place < 0 ? -1 : int64_t(kv_entry(place, a.nkv, kvh));
        }
        const bool absent = __any_sync(0xFFFFFFFFu, place < 0);
        int32_t extent = 0, all = 0x7FFFFFFF;
        for (uint32_t i = lane; i < rows; i += 32) {
          const int32_t e = a.extent[first + i];
          extent = max(extent, e);
          all = min(all, a.row_base ? min(max(a.row_base[first + i], 0), e) : e);
        }
#pragma unroll
        for (int off = 16; off; off >>= 1) {
          extent = max(extent, __shfl_xor_sync(0xFFFFFFFFu, extent, off));
          all = min(all, __shfl_xor_sync(0xFFFFFFFFu, all, off));
        }
        extent = min(extent, start + int32_t(part_positions));
        const uint32_t steps = (uint32_t(extent - start) + kWideStep - 1) / kWideStep;       // (a unit has a position at least)
        // (whole steps alone: the last one may reach past what the rows see, even where they all see as far)
        const uint32_t plain = absent ? 0u : uint32_t(max(min(all, extent) - start, 0)) / kWideStep;
        if (n) wait(bar_w, n - 1);                           // everybody has seen the unit before, and is through with the one whose tables are overwritten
        if (lane < part_positions / kWideStep) sm.where[slot][lane] = entry;
        if (lane == 0) sm.info[slot] = PairInfo{1u, first, rows, kvh, part, steps, plain, start, extent};
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_u);
        if (lane == 0) u = gridDim.x + atomicAdd(a.plan + 4, 1u);
        u = __shfl_sync(0xFFFFFFFFu, u, 0);
      }
      if (n) wait(bar_w, n - 1);                             // no unit is left
      if (lane == 0) {
        sm.info[n & 1u].valid = 0u;
        mbar_arrive(bar_u);
      }
      __syncwarp();
    }
    // ---- products: warp 16 of tile 0, warp 17 of tile 1 -----------------------------------------------------------
    // (what these warps do between a wait and the next lies in the chain of every step, and they get an instruction in seven cycles at best: descriptors are one
    // addition apart, stages and rounds are counted, not divided out)
    const uint32_t x = warp - 16;
    constexpr uint32_t kFp16 = ~((1u << 7) | (1u << 10)), kIdesc = umma_idesc_bf16(128) & kFp16 | (1u << 16), kIdescS = umma_idesc_bf16(kWideStep) & kFp16;
    const uint32_t s_tmem = sm.tmem_at + x * 128, o_tmem = sm.tmem_at + 256 + x * 128, s_bars = bar_s + x * kRound, o_bars = bar_o + x * kRound, p_bars = bar_p + x * kRound;
    const uint64_t q_desc = umma_desc_sw128(qs + x * kWideOperand), k_desc = umma_desc_sw128(ks), v_desc = wide_desc_v(vs);
    struct Turn {                                            // a step's place in the ring, and the parity of its round
      uint32_t stage, parity;
      __device__ __forceinline__ void next() {
        const bool last = stage == kPairRing - 1;
        stage = last ? 0u : stage + 1u;
        parity ^= uint32_t(last);
      }
    };
    Turn s_turn{0, 0}, used{0, 0}, o_turn{0, 0};             // of the next scores, of the products two steps before them, of the next outputs
    uint32_t s_at = s_tmem, p_at = s_tmem, behind = 0;       // (the two places of S and P take turns)
    bool on = true;
    auto scores = [&] {
      if (behind == 2) {                                     // the weights there have been used (issue order alone does not say so: the two products differ in shape)
        wait(o_bars + 8 * used.stage, used.parity);
        used.next();
      } else {
        ++behind;
      }
      wait(bar_k + 8 * s_turn.stage, s_turn.parity);
      tc_fence_after();
      if (elect_one()) {
        if (on) {
          const uint64_t k = k_desc + s_turn.stage * (kWideStage >> 4);
#pragma unroll
          for (int d = 0; d < 8; ++d)                        // 16 dimensions each
            umma_bf16(s_at, q_desc + ((d >> 2) * (kWideOperand / 2) + (d & 3) * 32) / 16, k + ((d >> 2) * (kWideStage / 2) + (d & 3) * 32) / 16, kIdescS, d > 0);
        }
        umma_commit(s_bars + 8 * s_turn.stage);              // (of a tile that stands still: at once)
      }
      __syncwarp();
      s_turn.next();
      s_at ^= kWideStep;
    };
    for (uint32_t n = 0; x < 2; ++n) {
      wait(bar_u, n);
      const PairInfo& unit = sm.info[n & 1u];
      if (!unit.valid || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) break;
      const uint32_t steps = unit.steps;
      on = x == 0 || unit.rows > tile_rows;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_w);
      wait(bar_q, n);
      scores();
      for (uint32_t j = 0; j < steps; ++j) {
        if (j + 1 < steps) scores();
        wait(bar_v + 8 * o_turn.stage, o_turn.parity);
        wait(p_bars + 8 * o_turn.stage, o_turn.parity);
        tc_fence_after();
        if (elect_one()) {
          if (on) {
            const uint64_t v = v_desc + o_turn.stage * (kWideStage >> 4);
#pragma unroll
            for (int d = 0; d < 4; ++d) umma_bf16_ts(o_tmem, p_at + 8 * d, v + 2048 / 16 * d, kIdesc, j > 0 || d > 0);        // 16 positions each
          }
          umma_commit(o_bars + 8 * o_turn.stage);
        }
        __syncwarp();
        o_turn.next();
        p_at ^= kWideStep;
      }
      step0 += steps;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // ---- weights: thread = row m of the tile, lane m of tensor memory ------------------------------------------------
    constexpr float kSlack = 8.f, kBias = 7.f;               // FP16: weights up to 2^(7 + 8)
    const uint32_t x = warp >> 2, m = tid & 127u, lanes = ((warp & 3u) * 32u) << 16;
    const uint32_t s_tmem = sm.tmem_at + lanes + x * 128, o_tmem = sm.tmem_at + lanes + 256 + x * 128, s_bars = bar_s + x * kRound, o_bars = bar_o + x * kRound, p_bars = bar_p + x * kRound;
    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1u;
      wait(bar_u, n);
      const PairInfo unit = sm.info[slot];
      if (!unit.valid || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_w);
      const uint32_t steps = unit.steps, plain = unit.plain, rows = x ? (unit.rows > tile_rows ? unit.rows - tile_rows : 0u) : min(unit.rows, tile_rows);
      if (!rows) {                                           // this tile stands still: the same waits and arrivals, nothing in between
        for (uint32_t j = 0; j < steps; ++j) {
          wait3(s_bars, step0 + j);
          __syncwarp();
          if (lane == 0) mbar_arrive(p_bars + 8 * ((step0 + j) % kPairRing));
        }
        wait3(o_bars, step0 + steps - 1);
        step0 += steps;
        continue;
      }
      const uint32_t used = rows * a.group, r = min(m, used - 1) / a.group, row = unit.first + x * tile_rows + r;
      const int32_t start = unit.start;
      const size_t pair = size_t(row) * a.nq + unit.kvh * a.group + (min(m, used - 1) - r * a.group);
      const float scale = a.q_scale[pair];
      const int32_t base = a.row_base ? a.row_base[row] : 0, mine = a.extent[row];
      float ref = -INFINITY;
      float2 sum = make_float2(0.f, 0.f);
      for (uint32_t j = 0; j < steps; ++j) {
        const uint32_t g = step0 + j, s_at = s_tmem + (g & 1u) * kWideStep;
        const int32_t at = start + int32_t(j * kWideStep);
        wait3(s_bars, g);
        tc_fence_after();
        uint32_t v[2][32];
        tmem_ld32(s_at, v[0]);
        tmem_ld32(s_at + 32, v[1]);
        // which of the step's positions the row sees
        const bool every = j < plain;
        uint32_t see[2] = {~0u, ~0u};
        if (!every) {
          const bool there = sm.where[slot][j] >= 0;          // (a page outside the pool: as if nobody saw its positions)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int32_t p = at + 32 * w, most = min(max(mine - p, 0), 32);
            const uint32_t below = most == 32 ? ~0u : (1u << most) - 1u;            // up to the last position the row sees
            uint32_t bits = ~0u;
            if (a.row_base) {
              const int32_t n0 = p - base;                   // node of the word's first bit
              if (n0 + 31 >= 0) {
                auto word = [&](int32_t i) -> uint64_t { return i >= 0 && uint32_t(i) < a.mask_words ? a.row_mask[row * a.ldm + i] : 0ull; };
                if (n0 >= 0) {
                  const uint32_t sh = uint32_t(n0) & 63u;
                  bits = uint32_t(word(n0 >> 6) >> sh);
                  if (sh > 32) bits |= uint32_t(word((n0 >> 6) + 1) << (64 - sh));
                } else {
                  bits = uint32_t(word(0)) << (-n0) | ((1u << (-n0)) - 1u);           // (-n0 is 1 to 31)
                }
              }
            }
            see[w] = there ? bits & below : 0u;
          }
        }
        tmem_ld_wait();
        const float2 scale2 = make_float2(scale, scale);
        const PairScales& of_step = scales[g % kPairScales];
        wait(bar_t + 8 * (g % kPairScales), g / kPairScales);
#pragma unroll
        for (int i = 0; i < 64; i += 4) {                    // S' (a NaN entry's is NaN)
          const float4 k4 = *reinterpret_cast<const float4*>(&of_step.k[i]), v4 = *reinterpret_cast<const float4*>(&of_step.v[i]);
          const float2 s0 = fma2(mul2(make_float2(__uint_as_float(v[i >> 5][i & 31]), __uint_as_float(v[i >> 5][(i & 31) + 1])), make_float2(k4.x, k4.y)), scale2, make_float2(v4.x, v4.y));
          const float2 s1 = fma2(mul2(make_float2(__uint_as_float(v[i >> 5][(i & 31) + 2]), __uint_as_float(v[i >> 5][(i & 31) + 3])), make_float2(k4.z, k4.w)), scale2, make_float2(v4.z, v4.w));
          v[i >> 5][i & 31] = __float_as_uint(s0.x);
          v[i >> 5][(i & 31) + 1] = __float_as_uint(s0.y);
          v[i >> 5][(i & 31) + 2] = __float_as_uint(s1.x);
          v[i >> 5][(i & 31) + 3] = __float_as_uint(s1.y);
        }
        if (!every) {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[w][i] = see[w] >> i & 1u ? v[w][i] : 0xFF800000u;
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 2) tops[i >> 1 & 3] = fmaxf(tops[i >> 1 & 3], fmaxf(__uint_as_float(v[i >> 5][i & 31]), __uint_as_float(v[i >> 5][(i + 1) & 31])));
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const bool move = top > (ref == -INFINITY ? ref : __fadd_rn(ref, kSlack));
        if (__any_sync(0xFFFFFFFFu, move)) {
          const float to = move ? top : ref, f = move ? exp2_approx(__fsub_rn(ref, to)) : 1.f;        // (from -infinity: 0)
          sum.x = __fmul_rn(sum.x, f);
          sum.y = __fmul_rn(sum.y, f);
          ref = to;
          if (j > 0) {
            wait3(o_bars, g - 1);
            tc_fence_after();
#pragma unroll 1
            for (int w = 0; w < 8; ++w) {
              uint32_t o[16];
              tmem_ld16(o_tmem + 16 * w, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__fmul_rn(__uint_as_float(o[i]), f));
              tmem_st16(o_tmem + 16 * w, o);
            }
          }
        }
        const float low = (ref == -INFINITY ? 0.f : ref) - kBias;
        const float2 low2 = make_float2(-low, -low);
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float4 inverse = *reinterpret_cast<const float4*>(&of_step.v_inverse[32 * w + 2 * i]);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float2 e = add2(make_float2(__uint_as_float(v[w][2 * (i + n)]), __uint_as_float(v[w][2 * (i + n) + 1])), low2);
              e.x = exp2_approx(e.x);
              e.y = exp2_approx(e.y);
              sums[n] = fma2(e, n ? make_float2(inverse.z, inverse.w) : make_float2(inverse.x, inverse.y), sums[n]);
              const __half2 h = __floats2half2_rn(e.x, e.y);
              p[i + n] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
          tmem_st16(s_at + 16 * w, p);                       // (over scores that have been read)
        }
        sum = add2(sum, add2(sums[0], sums[1]));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_bars + 8 * (g % kPairRing));
      }
      // ---- the unit's partial result
      wait3(o_bars, step0 + steps - 1);
      tc_fence_after();
      const size_t out = pair * a.max_parts + unit.part;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t o[32];
        tmem_ld32(o_tmem + 32 * w, o);
        tmem_ld_wait();
        if (m < used) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = __uint_as_float(o[i + e]);
            stg256(a.part_acc + out * kKvDim + 32 * w + i, y);
          }
        }
      }
      if (m < used) a.part_ml[out] = make_float2(ref == -INFINITY ? ref : ref - kBias, sum.x + sum.y);
      tc_fence_before();                                     // (the next unit's first product waits for this warp's first weights)
      step0 += steps;
    }
  }
  // (every product has been waited for, or its wait ran out: then the tensor memory is given back after a moment for what may
  // still be under way)
  if (sm.aborted) {
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < kLingerNs) {}
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(sm.tmem_at, kPairColumns);
}

}  // namespace grb
