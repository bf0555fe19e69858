// The attention of tree_attention.cuh for many rows of one sequence at a time: wide trees and prompt chunks, on tcgen05.
//
// A tile is up to 128 rows (row of the step, query head of the group) of one sequence and kv head: the M of one instruction.  A
// unit is a tile and a chunk of the positions, taken 64 at a time:
//   S = Q K^T (Q, K in shared memory, S in tensor memory);  weights P = exp2(S scale - reference), written over S;
//   O += P V (P from tensor memory, V in shared memory, O in tensor memory).
// Four warps, a thread per row, turn scores into weights; four bring K and V: BF16 as it is, 8 bits through registers, where a code
// becomes FP16, exactly (one conversion for two); one issues the products.  K, V and
// S of two steps are held, so a step's scores are computed while the step before is weighed, and the loaders set the next unit up
// while this one ends.  256 columns of tensor memory and 105 KB of shared memory leave room for two CTAs on an SM.
//
// 16 trees of 64 nodes behind 8192 positions, 40 query heads of 8 kv heads, all launches: 322 us in 8 bits, 0.41 PFLOP/s (one step
// at a time and barriers between units: 438; steps of 128 with one S, the products issued by a weights' warp: 340).  What bounds it
// is the chain of a step, in which the loaders wait for a stage, convert 64 positions of K and of V and ask for the next, and the
// weights' warps go through 64 scores a thread: without the scales' arithmetic 307 us.
//
// BF16: Q and the weights go into the products as two terms, what rounding to BF16 leaves and what it leaves out, so that the error
// is the result's rounding (one term each: twice that).  416 us for the trees above, 291 with one term; with four stages of K and V
// instead of three, and therefore one CTA an SM, 558.
//
// 8 bits: K's scale multiplies the score of its position, V's goes into the weight, as in the narrow kernel: S' = S 2^e_k scale + e_v, so
// that the FP16 weights (2^15 at most, down to 2^-24) are largest where the row's own products are, whatever else the chunk holds; the
// sum of the weights takes V's scale out again.
// The reference of a row's weights moves only when its maximum has passed it by 2^8 (then O, in tensor memory, is scaled down).
#pragma once
#include <type_traits>

#include "tree_attention.cuh"

namespace grb {

constexpr int kWideThreads = 384;                // softmax warps 0-3, loading warps 4-7, a warp that issues the products
constexpr uint32_t kWideTile = 128;              // rows of a tile
constexpr uint32_t kWideStep = 64;               // positions of a step
constexpr uint32_t kWideOperand = 32768;         // Q: two halves of 64 dimensions, 128 rows of 128 bytes each; K or V of two steps
constexpr uint32_t kWideStage = kWideOperand / 2;        // K or V of a step: two halves of 64 dimensions, 64 rows each
constexpr uint32_t kWideColumns = 256;           // tensor memory: S of two steps (and P over it), O

// Byte offset of 16-byte piece `piece` (0..15) of row `row` of an operand of ROWS rows: 128-byte swizzle in each half.
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t wide_offset(uint32_t row, uint32_t piece) {
  return (piece >> 3) * (ROWS * 128u) + row * 128u + (((piece ^ row) & 7u) << 4);
}
// V as the B operand with its dimensions contiguous (N-major): 64 dimensions per 128-byte row, the other half 8 KB on, groups of
// eight positions 1024 bytes apart.
__device__ __forceinline__ uint64_t wide_desc_v(uint32_t smem_addr) {
  return uint64_t((smem_addr >> 4) & 0x3FFFu) | (uint64_t(kWideStage / 2 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// 32 bytes, a whole sector: a thread stores its own row, and 16 bytes at a time every sector went out twice (364 us for 16 trees of
// 64 nodes behind 8192 positions instead of 352).
__device__ __forceinline__ void stg256(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}
struct WideUnit {
  uint32_t first, rows, kvh, part;
  int32_t seq, start, extent;      // positions start .. extent - 1 (at most a chunk): what some row sees, up to the last such
};
// What the loading warps tell the others of a unit.
struct WideInfo {
  uint32_t valid, first, rows, kvh, part, steps;
  uint32_t plain;                  // steps, from the first on, whose positions every row sees
  int32_t start;
};
// What the exponents of a step's positions mean: 2^e of K; e and 2^-e (BF16, exact) of V.  (Half as many loads for the last, whose
// latency the weights wait for: 322 us for the trees above instead of 326.)
struct WideScales {
  float k[kWideStep], v[kWideStep];
  uint16_t v_inverse[kWideStep];
};
// Shared memory beside the operands.
template <bool F8>
struct WideShared {
  uint64_t bars[F8 ? 15 : 11];     // of even and odd steps: K stored, V stored, S done, O done, P stored; unit set up; 8 bits, of every fourth step: scales
  WideInfo info[2];                // of a unit and the next
  uint32_t bad[2][F8 ? 1 : kWideMostPart / 32];        // BF16: positions of the chunk whose value is not a number
  typename std::conditional<F8, int64_t, int32_t>::type where[2][kWideMostPart / kWideStep];     // first entry, or (BF16) page, of each step; -1: none
  uint32_t tmem_at, aborted, next_unit;
  uint32_t any_absent;             // the loaders' own, while they set a unit up
};
static_assert(sizeof(WideShared<false>) <= 1024, "two CTAs of the BF16 kernel take all of an SM's shared memory");
constexpr uint32_t kWideSharedBytes = 2048;
// The operands follow.  8 bits: Q, two stages of K, two of V, scales of four steps.  BF16: Q, what its rounding left
// out, a ring of three stages that K and V take in turn (K of step g where V of g - 2 was, V of g where K of g - 1 was).
template <bool F8>
constexpr uint32_t kWideSmem = F8 ? kWideSharedBytes + 3 * kWideOperand + 4 * uint32_t(sizeof(WideScales)) : 1024 + 2 * kWideOperand + 3 * kWideStage;
__device__ __forceinline__ void wide_loaders_meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <bool F8>
__global__ void __launch_bounds__(kWideThreads, 2)
tree_wide_kernel(const TreeArgs a) {
  extern __shared__ __align__(1024) unsigned char wide_smem[];
  WideShared<F8>& sm = *reinterpret_cast<WideShared<F8>*>(wide_smem);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
  const uint32_t qs = smem_u32(wide_smem) + (F8 ? kWideSharedBytes : 1024u), rs = qs + kWideOperand, ks = F8 ? rs : rs + kWideOperand, vs = ks + kWideOperand;
  WideScales* const scales = reinterpret_cast<WideScales*>(wide_smem + kWideSharedBytes + 3 * kWideOperand);     // (8 bits)
  const uint32_t bar_k = smem_u32(&sm.bars[0]), bar_v = smem_u32(&sm.bars[2]), bar_s = smem_u32(&sm.bars[4]), bar_o = smem_u32(&sm.bars[6]),
                 bar_p = smem_u32(&sm.bars[8]), bar_u = smem_u32(&sm.bars[10]), bar_t = smem_u32(&sm.bars[F8 ? 11 : 10]);
  auto k_stage = [&](uint32_t g) { return ks + (F8 ? g & 1u : 2 * g % 3) * kWideStage; };
  auto v_stage = [&](uint32_t g) { return F8 ? vs + (g & 1u) * kWideStage : ks + (2 * g + 1) % 3 * kWideStage; };
  // Tensor memory is taken before the kernels behind this one may start: a matrix product among them takes its own as it starts and
  // keeps it until this kernel is through.
  if (tid == 0) {
    for (uint32_t b = 0; b < 16; b += 8) {
      mbar_init(bar_k + b, 4);
      mbar_init(bar_v + b, 4);
      mbar_init(bar_s + b, 1);
      mbar_init(bar_o + b, 1);
      mbar_init(bar_p + b, 4);
    }
    mbar_init(bar_u, 4);
    if constexpr (F8) {
      for (uint32_t b = 0; b < 32; b += 8) mbar_init(bar_t + b, 4);
    }
    mbar_fence_init();
    sm.aborted = 0u;
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(&sm.tmem_at), kWideColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  step_kernel_entry();
  const uint32_t tiles = a.plan[2], units = a.plan[3];
  if (blockIdx.x >= units) {
    if (warp == 4) tmem_dealloc(sm.tmem_at, kWideColumns);
    return;
  }
  const uint32_t s_tmem = sm.tmem_at, o_tmem = sm.tmem_at + 128;
  // A wait that runs out is everybody's: nobody waits again, every loop runs to its end, and the status says so.
  auto wait = [&](uint32_t bar, uint32_t step) {
    if (mbar_test_wait(bar, step & 1u) || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) return;
    if (!mbar_wait(bar, step & 1u, false)) {
      *reinterpret_cast<volatile uint32_t*>(&sm.aborted) = 1u;
      atomicOr(a.status, kStatusTimeout);
    }
  };
  auto wait2 = [&](uint32_t bars2, uint32_t step) { wait(bars2 + 8 * (step & 1u), step >> 1); };
  // Units differ in length, so a CTA takes the next one when it is through with its own (who computes a unit changes nothing in it);
  // its loaders set the next one up while the last step of this one is multiplied and its result stored.
  uint32_t step0 = 0;                                        // steps this CTA has taken before the unit
  // registers, of the 240 that three threads of the launch have: 112 for the weights, 88 for loading, 40 for the products; BF16, whose
  // loaders hold nothing: 128, 72, 40
  if (warp >= 4 && warp < 8) {
    if constexpr (F8) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---- loading ------------------------------------------------------------------------------------------------
    const uint32_t lt = tid - 128;
    uint32_t tile = 0, slot = 0, steps_before = 0;
    WideUnit t;
    uint32_t steps = 0, plain = 0;
    for (uint32_t u = blockIdx.x; u < units; slot ^= 1u) {
      // the unit (every warp finds it for itself), and where its steps lie
      for (;;) {
        const uint32_t past = __ballot_sync(0xFFFFFFFFu, tile + 1 + lane < tiles && uint32_t(a.wide_tiles[tile + 1 + lane].z) <= u);
        tile += __popc(past);
        if (past != 0xFFFFFFFFu) break;
      }
      const int4 d = a.wide_tiles[tile];
      const uint32_t local = u - uint32_t(d.z), part_positions = uint32_t(d.w);
      t.first = uint32_t(d.x);
      t.rows = uint32_t(d.y);
      t.kvh = local % a.nkv;
      t.part = local / a.nkv;
      t.seq = a.row_seq[t.first];
      t.start = int32_t(t.part * part_positions);
      const uint32_t used = t.rows * a.group;
      if constexpr (!F8) {
        if (lt < kWideMostPart / 32) sm.bad[slot][lt] = 0u;
      }
      if (lt == 0) sm.next_unit = gridDim.x + atomicAdd(a.plan + 4, 1u);
      if (warp == 4) {                                       // (a step's positions lie in one page)
        int64_t place = 0;
        if (lane < part_positions / kWideStep) {
          place = kv_place(a.table, t.seq, t.start + int32_t(lane * kWideStep));
          if constexpr (F8) sm.where[slot][lane] = place < 0 ? -1 : int64_t(kv_entry(place, a.nkv, t.kvh));
          else sm.where[slot][lane] = place < 0 ? -1 : int32_t(place / kKvPage);
        }
        const bool absent = __any_sync(0xFFFFFFFFu, place < 0);
        if (lane == 0) sm.any_absent = absent;
      }
      int32_t extent = 0, all = 0x7FFFFFFF;
      for (uint32_t i = lane; i < t.rows; i += 32) {
        const int32_t e = a.extent[t.first + i];
        extent = max(extent, e);
        all = min(all, a.row_base ? min(max(a.row_base[t.first + i], 0), e) : e);
      }
#pragma unroll
      for (int off = 16; off; off >>= 1) {
        extent = max(extent, __shfl_xor_sync(0xFFFFFFFFu, extent, off));
        all = min(all, __shfl_xor_sync(0xFFFFFFFFu, all, off));
      }
      t.extent = min(extent, t.start + int32_t(part_positions));
      steps = (uint32_t(t.extent - t.start) + kWideStep - 1) / kWideStep;       // (a unit has a position at least)
      wide_loaders_meet();
      u = sm.next_unit;
      // (whole steps alone: the last one may reach past what the tile's rows see, even where they all see as far)
      plain = sm.any_absent ? 0u : uint32_t(max(min(all, t.extent) - t.start, 0)) / kWideStep;
      // entry (of the layer) of step j's first position; -1: none
      auto entry_of = [&](uint32_t j) -> int64_t {
        if constexpr (F8) return sm.where[slot][j];
        const int32_t page = int32_t(sm.where[slot][j]);
        return page < 0 ? -1 : int64_t(kv_entry(int64_t(page) * kKvPage + (uint32_t(t.start) + j * kWideStep) % kKvPage, a.nkv, t.kvh));
      };
      // the queries, sixteen lanes a row, once the scores of the unit before are done
      auto queries = [&]() {
        if (step0) wait2(bar_s, step0 - 1);
        constexpr uint32_t kHalves = F8 ? 1 : 2, kAtOnce = F8 ? 4 : 8;
#pragma unroll 1
        for (uint32_t i0 = 0; i0 < 16 * kHalves; i0 += kAtOnce) {
          const uint32_t half = i0 >> 4, row0 = (lt >> 4) + (i0 & 15u) * 8;
          uint4 x[kAtOnce];
#pragma unroll
          for (uint32_t i = 0; i < kAtOnce; ++i) {
            const uint32_t m = row0 + 8 * i, r = m / a.group;
            const size_t pair = (size_t(t.first + r)) * a.nq + t.kvh * a.group + (m - r * a.group);
            x[i] = m < used ? reinterpret_cast<const uint4*>(a.q + (pair * kHalves + half) * kKvDim)[lt & 15u] : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (uint32_t i = 0; i < kAtOnce; ++i) sts128((half ? rs : qs) + wide_offset<kWideTile>(row0 + 8 * i, lt & 15u), x[i]);
        }
      };
      // everything is there: tells the weights' warps, who have all looked at the unit before once its first step's values have been
      // used (storing the third step's waited for that)
      auto publish = [&]() {
        if (lt == 0) sm.info[slot] = WideInfo{1u, t.first, t.rows, t.kvh, t.part, steps, plain, t.start};
        if (steps_before && steps_before <= 2) wait2(bar_o, step0 - 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_u);
      };
      if constexpr (F8) {
        // A thread's pieces: the same quarter of both halves of every 32nd row.  Eight lanes take four pieces of two neighbouring rows,
        // which the swizzle spreads over all banks when their sixteen values each are stored.
        const uint32_t row0 = lt >> 2;
        uint4 k[4], v[4];
        auto ask = [&](uint4 (&x)[4], const void* pool, uint32_t j) {
          const int64_t entry = j < steps ? entry_of(j) : -1;
          const int32_t npos = entry < 0 ? 0 : t.extent - t.start - int32_t(j * kWideStep);
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pool) + entry * kKvDim) + row0 * 8 + (lt & 3u);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = int32_t(row0 + 32 * (i >> 1)) < npos ? src[256 * (i >> 1) + 4 * (i & 1)] : make_uint4(0u, 0u, 0u, 0u);
        };
        const uint32_t to_lo = wide_offset<kWideStep>(row0, 2 * (lt & 3u)), to_hi = wide_offset<kWideStep>(row0, 2 * (lt & 3u) + 1);     // (32 rows on: 4096 bytes)
        auto store = [&](const uint4 (&x)[4], uint32_t dst, bool clean) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t h[8];
            e4m3_to_half4(x[i].x, h[0], h[1]);
            e4m3_to_half4(x[i].y, h[2], h[3]);
            e4m3_to_half4(x[i].z, h[4], h[5]);
            e4m3_to_half4(x[i].w, h[6], h[7]);
            if (clean) {
#pragma unroll
              for (int q = 0; q < 8; ++q) h[q] = half2_number(h[q]);
            }
            const uint32_t at = dst + 4096 * (i >> 1) + (kWideStage / 2) * (i & 1);
            sts128(at + to_lo, make_uint4(h[0], h[1], h[2], h[3]));
            sts128(at + to_hi, make_uint4(h[4], h[5], h[6], h[7]));
          }
        };
        // exponents: half of the threads a position's of K, the others one's of V.  A byte below what an entry has (0, where nobody wrote)
        // stands for zeros of the smallest size.
        const uint32_t at = lt & (kWideStep - 1);
        const uint8_t* const exps = lt < kWideStep ? a.pages.k_exp : a.pages.v_exp;
        uint32_t byte;
        auto ask_exp = [&](uint32_t j) {
          const int64_t entry = j < steps ? entry_of(j) : -1;
          byte = entry < 0 ? 127u : exps[entry + at];
        };
        auto store_exp = [&](WideScales& s) {
          if (lt < kWideStep) {
            s.k[at] = kv_scale(byte);
          } else {
            const uint32_t b = max(byte, kKvLeastByte);
            s.v[at] = b == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(b) - 127);
            s.v_inverse[at] = uint16_t(__float_as_uint(kv_inverse(b)) >> 16);
          }
        };
        ask_exp(0);
        ask(k, a.pages.k, 0);
        ask(v, a.pages.v, 0);
        wide_loaders_meet();                                 // (the unit after this one and its pages are known to all)
        queries();
        publish();
        for (uint32_t j = 0; j < steps; ++j) {
          const uint32_t g = step0 + j;
          if (g > 1) wait2(bar_s, g - 2);                    // scores have been taken from the stage's K
          store(k, k_stage(g), false);
          store_exp(scales[g & 3u]);                         // (the step four before has been weighed: the one after it was waited for)
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar_t + 8 * (g & 3u));
            mbar_arrive(bar_k + 8 * (g & 1u));
          }
          ask_exp(j + 1);
          ask(k, a.pages.k, j + 1);
          if (g > 1) wait2(bar_o, g - 2);                    // the stage's values have been used
          store(v, v_stage(g), j >= plain);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_v + 8 * (g & 1u));
          ask(v, a.pages.v, j + 1);
        }
      } else {
        auto ask = [&](uint32_t dst, const void* pool, uint32_t j) {
          const int64_t entry = entry_of(j);
          const int32_t npos = entry < 0 ? 0 : t.extent - t.start - int32_t(j * kWideStep);
          const uint8_t* src = static_cast<const uint8_t*>(pool) + (entry < 0 ? 0 : entry) * kKvDim * 2;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t c = lt + 128 * i;
            const bool in = int32_t(c >> 4) < npos;
            cp_async_16(dst + wide_offset<kWideStep>(c >> 4, c & 15u), src + (in ? c * 16 : 0u), in ? 16u : 0u);
          }
          cp_async_commit();
        };
        wide_loaders_meet();                                 // (the unit after this one and its pages are known to all)
        queries();
        publish();
        // a step's values that are not finite would reach, as 0 * infinity, rows that do not see them
        auto values = [&](uint32_t j) {
          if (j < plain) return;
          uint32_t mine = 0;                               // bit i: of the thread's piece i
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const uint32_t c = lt + 128 * i, at = v_stage(step0 + j) + wide_offset<kWideStep>(c >> 4, c & 15u);
            const uint4 x = lds128(at);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            bool b = false;
#pragma unroll
            for (int q = 0; q < 4; ++q) b = b || (w[q] & 0x7F80u) == 0x7F80u || (w[q] & 0x7F800000u) == 0x7F800000u;
            if (b) sts128(at, make_uint4(0u, 0u, 0u, 0u));
            mine |= uint32_t(b) << i;
          }
          // piece i of this warp's lanes lies in positions 8 i + 2 (warp - 4) and the next
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t m = __ballot_sync(0xFFFFFFFFu, mine >> i & 1u);
            const uint32_t p = 8 * i + 2 * (warp - 4);
            if (lane == 0 && m) atomicOr(&sm.bad[slot][j * (kWideStep / 32) + (p >> 5)], (uint32_t((m & 0xFFFFu) != 0) | uint32_t((m >> 16) != 0) << 1) << (p & 31u));
          }
        };
        // (a step's copies are on their way while the step before's land; behind the last one, a group of none keeps the count)
        for (uint32_t j = 0; j <= steps; ++j) {
          const uint32_t g = step0 + j;
          if (j) {
            cp_async_wait<1>();
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_k + 8 * (~g & 1u));
          }
          if (j < steps) {
            if (g > 1) wait2(bar_o, g - 2);
            ask(k_stage(g), a.pages.k, j);
          } else {
            cp_async_commit();
          }
          if (j) {
            cp_async_wait<1>();
            values(j - 1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_v + 8 * (~g & 1u));
          }
          if (j < steps) {
            if (g > 0) wait2(bar_s, g - 1);
            ask(v_stage(g), a.pages.v, j);
          }
        }
      }
      if (steps == 1 && step0) wait2(bar_o, step0 - 1);      // (the unit before is over, whose tables the next one but one overwrites)
      step0 += steps;
      steps_before = steps;
    }
    // no unit is left
    if (lt == 0) sm.info[slot].valid = 0u;
    if (steps_before && steps_before <= 2) wait2(bar_o, step0 - 1);
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_u);
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // ---- products -----------------------------------------------------------------------------------------------
    // (a warp of its own: issuing a step's products takes it as long as the weights take theirs)
    constexpr uint32_t kIdesc = umma_idesc_bf16(128) & (F8 ? ~((1u << 7) | (1u << 10)) : ~0u);      // FP16 or BF16 operands
    constexpr uint32_t kIdescS = umma_idesc_bf16(kWideStep) & (F8 ? ~((1u << 7) | (1u << 10)) : ~0u);
    auto scores = [&](uint32_t g) {
      if (g > 1) wait2(bar_o, g - 2);                        // the weights there have been used (issue order alone does not say so:
      wait2(bar_k, g);                                       // the two products differ in shape)
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int d = 0; d < (F8 ? 8 : 16); ++d) {            // 16 dimensions each; BF16: of what Q's rounding left out, then of Q
          const uint32_t q = F8 || d >= 8 ? qs : rs, half = (d >> 2 & 1) * (kWideOperand / 2), k16 = (d & 3) * 32;
          umma_bf16(s_tmem + (g & 1u) * kWideStep, umma_desc_sw128(q + half + k16),
                    umma_desc_sw128(k_stage(g) + half / 2 + k16), kIdescS, d > 0);
        }
        umma_commit(bar_s + 8 * (g & 1u));
      }
      __syncwarp();
    };
    for (uint32_t n = 0; warp == 8; ++n) {
      wait(bar_u, n);
      if (!sm.info[n & 1u].valid || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) break;
      const uint32_t steps = sm.info[n & 1u].steps;
      scores(step0);
      for (uint32_t j = 0; j < steps; ++j) {
        const uint32_t g = step0 + j;
        if (j + 1 < steps) scores(g + 1);
        wait2(bar_v, g);
        wait2(bar_p, g);
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int d = 0; d < (F8 ? 4 : 8); ++d)             // 16 positions each; BF16: then of what the weights' rounding left out
            umma_bf16_ts(o_tmem, s_tmem + (g & 1u) * kWideStep + 8 * d, wide_desc_v(v_stage(g) + 2048 * (d & 3)), kIdesc | (1u << 16), j > 0 || d > 0);
          umma_commit(bar_o + 8 * (g & 1u));
        }
        __syncwarp();
      }
      step0 += steps;
    }
  } else {
    if constexpr (F8) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
    // ---- weights: thread = row m of the tile, lane m of tensor memory ------------------------------------------------
    constexpr float kSlack = 8.f, kBias = F8 ? 7.f : 0.f;    // FP16: weights up to 2^(7 + 8)
    const uint32_t m = tid, lanes = (warp * 32u) << 16;
    for (uint32_t n = 0;; ++n) {
      const uint32_t slot = n & 1u;
      wait(bar_u, n);
      const WideInfo unit = sm.info[slot];
      if (!unit.valid || *reinterpret_cast<volatile uint32_t*>(&sm.aborted)) break;
      const uint32_t steps = unit.steps, plain = unit.plain, used = unit.rows * a.group, r = min(m, used - 1) / a.group, row = unit.first + r;
      const int32_t start = unit.start;
      const size_t pair = size_t(row) * a.nq + unit.kvh * a.group + (min(m, used - 1) - r * a.group);
      const float scale = a.q_scale[pair];
      const int32_t base = a.row_base ? a.row_base[row] : 0, mine = a.extent[row];
      float ref = -INFINITY;
      float2 sum = make_float2(0.f, 0.f);
      for (uint32_t j = 0; j < steps; ++j) {
        const uint32_t g = step0 + j, s_at = s_tmem + lanes + (g & 1u) * kWideStep;
        const int32_t at = start + int32_t(j * kWideStep);
        wait2(bar_s, g);
        tc_fence_after();
        uint32_t x[2][32];
        tmem_ld32(s_at, x[0]);
        tmem_ld32(s_at + 32, x[1]);
        // which of the step's positions the row sees
        const bool every = j < plain;
        uint32_t see[2] = {~0u, ~0u};
        bool poisoned = false;
        if (!every) {
          if constexpr (!F8) wait2(bar_v, g);                // (`bad` is complete)
          const bool there = sm.where[slot][j] >= 0;          // (a page outside the pool: as if nobody saw its positions)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int32_t p = at + 32 * w, most = min(max(mine - p, 0), 32);
            const uint32_t below = most == 32 ? ~0u : (1u << most) - 1u;            // up to the last position the row sees
            uint32_t bits = ~0u;
            if (a.row_base) {
              const int32_t n0 = p - base;                   // node of the word's first bit
              if (n0 + 31 < 0) bits = ~0u;
              else {
                auto word = [&](int32_t n) -> uint64_t { return n >= 0 && uint32_t(n) < a.mask_words ? a.row_mask[row * a.ldm + n] : 0ull; };
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
        if (!F8 && !every) {
#pragma unroll
          for (int w = 0; w < 2; ++w) poisoned = poisoned || (*reinterpret_cast<volatile uint32_t*>(&sm.bad[slot][j * (kWideStep / 32) + w]) & see[w]);
        }
        tmem_ld_wait();
        const float2 scale2 = make_float2(scale, scale);
        const WideScales& of_step = scales[g & 3u];
        if constexpr (F8) {                                  // S' (a NaN entry's is NaN)
          wait(bar_t + 8 * (g & 3u), g >> 2);
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(&of_step.k[i]), v4 = *reinterpret_cast<const float4*>(&of_step.v[i]);
            const float2 s0 = fma2(mul2(make_float2(__uint_as_float(x[i >> 5][i & 31]), __uint_as_float(x[i >> 5][(i & 31) + 1])), make_float2(k4.x, k4.y)), scale2, make_float2(v4.x, v4.y));
            const float2 s1 = fma2(mul2(make_float2(__uint_as_float(x[i >> 5][(i & 31) + 2]), __uint_as_float(x[i >> 5][(i & 31) + 3])), make_float2(k4.z, k4.w)), scale2, make_float2(v4.z, v4.w));
            x[i >> 5][i & 31] = __float_as_uint(s0.x);
            x[i >> 5][(i & 31) + 1] = __float_as_uint(s0.y);
            x[i >> 5][(i & 31) + 2] = __float_as_uint(s1.x);
            x[i >> 5][(i & 31) + 3] = __float_as_uint(s1.y);
          }
        }
        if (!every) {
#pragma unroll
          for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < 32; ++i) x[w][i] = see[w] >> i & 1u ? x[w][i] : 0xFF800000u;
        }
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 64; i += 2) tops[i >> 1 & 3] = fmaxf(tops[i >> 1 & 3], fmaxf(__uint_as_float(x[i >> 5][i & 31]), __uint_as_float(x[i >> 5][(i + 1) & 31])));
        const float raw = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), top = F8 ? raw : __fmul_rn(raw, scale);
        const bool move = top > (ref == -INFINITY ? ref : __fadd_rn(ref, kSlack));
        if (__any_sync(0xFFFFFFFFu, move)) {
          const float to = move ? top : ref, f = move ? exp2_approx(__fsub_rn(ref, to)) : 1.f;        // (from -infinity: 0)
          sum.x = __fmul_rn(sum.x, f);
          sum.y = __fmul_rn(sum.y, f);
          ref = to;
          if (j > 0) {
            wait2(bar_o, g - 1);
            tc_fence_after();
#pragma unroll 1
            for (int w = 0; w < 8; ++w) {
              uint32_t o[16];
              tmem_ld16(o_tmem + lanes + 16 * w, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__fmul_rn(__uint_as_float(o[i]), f));
              tmem_st16(o_tmem + lanes + 16 * w, o);
            }
          }
        }
        const float low = (ref == -INFINITY ? 0.f : ref) - kBias;
        const float2 low2 = make_float2(-low, -low);
        float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t p[16], rest[F8 ? 1 : 16];
          uint32_t inverse[F8 ? 16 : 1];
          if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 q = *reinterpret_cast<const uint4*>(&of_step.v_inverse[32 * w + 8 * i]);
              inverse[4 * i] = q.x; inverse[4 * i + 1] = q.y; inverse[4 * i + 2] = q.z; inverse[4 * i + 3] = q.w;
            }
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 s = make_float2(__uint_as_float(x[w][2 * i]), __uint_as_float(x[w][2 * i + 1]));
            float2 e = F8 ? add2(s, low2) : fma2(s, scale2, low2);
            e.x = exp2_approx(e.x);
            e.y = exp2_approx(e.y);
            if constexpr (F8) {
              sums[i & 1] = fma2(e, make_float2(bf_lo(inverse[i]), bf_hi(inverse[i])), sums[i & 1]);
              const __half2 h = __floats2half2_rn(e.x, e.y);
              p[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
              sums[i & 1] = add2(sums[i & 1], e);
              p[i] = pack_bf(e.x, e.y);
              rest[i] = pack_bf_rest(e.x, e.y, p[i]);
            }
          }
          tmem_st16(s_at + 16 * w, p);                       // (over scores that have been read)
          if constexpr (!F8) tmem_st16(s_at + 32 + 16 * w, rest);
        }
        sum = add2(sum, add2(sums[0], sums[1]));
        if (poisoned) sum.x = __uint_as_float(0x7FC00000u);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8 * (g & 1u));
      }
      // ---- the unit's partial result
      wait2(bar_o, step0 + steps - 1);
      tc_fence_after();
      const size_t out = pair * a.max_parts + unit.part;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t x[32];
        tmem_ld32(o_tmem + lanes + 32 * w, x);
        tmem_ld_wait();
        if (m < used) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(x[i + e]);
            stg256(a.part_acc + out * kKvDim + 32 * w + i, o);
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
  if (warp == 4) tmem_dealloc(sm.tmem_at, kWideColumns);
}

}  // namespace grb
