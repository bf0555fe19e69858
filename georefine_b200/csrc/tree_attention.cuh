// Attention of a step's rows over a paged cache in BF16, 8 or 4 bits (kv_cache.cuh), for causal rows and for the nodes of
// draft trees: rotary embedding, the append of the rows' keys and values, soft-max attention in parts merged in part order.
//
//   out[r, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(q_rh . k_j / sqrt(128)),  j over the positions that row r sees:
//   causal: j <= row_pos[r];  tree: j < base[r], or bit j - base[r] of the row's mask.  A row that sees nothing gives 0.
//
// Three launches, four where many rows of a sequence may come together.  tree_prep: rotates the queries (once rounded, to the type
// the matrix instruction takes), stores keys and values, and one CTA lays down the plan: tiles of rows of one sequence, and units =
// (tile, part of the positions, kv head).  tree_part (4 bits: tree_q4, tree_q4.cuh): persistent CTAs take runs of units.  tree_wide (tree_wide.cuh;
// 4 bits: tree_pair, tree_pair.cuh): the same for runs of many rows.  tree_combine: merges a row's parts.  Which kernel takes a row and where its parts lie depends on its own
// sequence's rows alone (and on whether the caller's longest_run lets tree_wide run at all), and every sum runs in a fixed order:
// a row's bits do not depend on what else is in the batch.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"

namespace grb {

constexpr uint32_t kTreeMaxRows = 4096, kTreeMaskWords = 4;
// Threads of a tree_prep CTA, up to 256 rows and beyond: the plan's CTA takes as many rows at a time.
constexpr uint32_t kTreePrepThreads = 256, kTreePrepMost = 1024;
constexpr uint32_t kTreeRowAbsent = 0xFFFFFFFFu;             // row_parts of a row that is left out: its output stays as it was
// Positions of a wide tile's unit: the most, for long contexts (a unit's result is as large as 256 positions of an 8-bit cache); fewer
// for short ones and for runs of one or two tiles, whose few units would leave SMs idle.  1024 instead of 2048 behind 8192 positions,
// 8 bits, 40 heads of 8: one run of 16 rows 35 us instead of 51, 16 runs 120 instead of 138; 16 runs of 64 rows (three tiles) 337
// instead of 320, which keep 2048.  (4 bits: no more parts than the narrow kernel's, for as many there is room; parts of one size: 384 prompt rows behind 8000
// positions 126 us instead of 134, the trees of three tiles 340 instead of 346, which would take 332 with 2048, and leave half of
// the SMs idle where one of them is alone.)
constexpr uint32_t kWideMostPart = 2048;
template <int FORMAT>
__device__ __forceinline__ uint32_t wide_part(uint32_t extent, bool many) {
  const uint32_t part = extent <= 1024 && FORMAT != kKvQ4 ? 256u : extent <= 4096 ? 512u : extent <= 16384 && !many ? 1024u : kWideMostPart;
  if constexpr (FORMAT == kKvQ4) {
    // as many parts as come nearest to that (of the largest: as there have to be), all of them alike: a last part of one step costs a unit's beginning and end and
    // a partial result like the others
    const uint32_t parts = part == kWideMostPart ? (extent + part - 1) / part : (extent + part / 2) / part, each = (extent + max(parts, 1u) - 1) / max(parts, 1u);
    return (max(each, 1u) + 63u) & ~63u;
  }
  return part;
}

struct TreeArgs {
  const __nv_bfloat16* qkv;   // [rows][ldq]: nq query heads | nkv key heads | nkv value heads, 128 each
  int64_t ldq;
  const __nv_bfloat16* cos_table;  // [rope_rows][128]
  const __nv_bfloat16* sin_table;
  uint32_t rope_rows;
  const int32_t* row_seq;     // [rows]: slot, or -1: the row is left out
  const int32_t* row_pos;     // [rows]: where the row's key and value are stored
  const int32_t* row_base;    // tree: [rows]; null: causal rows
  const int32_t* row_rope;    // tree: [rows]: the row's rotary position
  const uint64_t* row_mask;   // tree: [rows][ldm], mask_words words of 64 nodes
  int64_t ldm;
  uint32_t mask_words;
  KvTable table;
  KvPagesArgs pages;          // of one layer
  uint16_t* q;                // scratch: rotated queries, (8-bit caches) [rows][nq][128] FP16 times a power of two, or [rows][nq][2][128]
                              // BF16: rounded, and what the rounding left out, rounded
  float* q_scale;             // scratch: [rows][nq]: what a query's scores are multiplied by, in units of log 2
  uint32_t* status;           // scratch: kStatusTimeout where a wait ran out
  int32_t* extent;            // scratch: [rows]: positions up to the last one the row sees
  uint32_t* row_parts;        // scratch: [rows]: parts of the row
  int4* tiles;                // scratch: [rows]: first row, rows, units (4 bits: weight of the units) before it, positions up to the last one its rows see
  int4* wide_tiles;           // scratch: [rows]: first row, rows (4 bits: of a pair of tiles), first unit, positions of a unit
  uint32_t* plan;             // scratch: tiles, units, wide tiles, wide units, wide units taken
  float* part_acc;            // scratch: [rows][nq][max_parts][128]
  float2* part_ml;            // scratch: [rows][nq][max_parts]: maximum and sum of a part
  __nv_bfloat16* out;         // [rows][ldo]: nq * 128
  int64_t ldo;
  uint32_t rows, nq, nkv, group, tile_rows, max_parts;
  uint32_t wide_rows, wide_from;   // rows of a wide tile (4 bits: of a pair of them); a run of so many rows (0: none) is cut into wide tiles
  float scaling;
};

// The place of row r's own entry; -1: the row is left out (slot -1, or a position outside the table, the pool or the rotary
// tables): nothing is stored for it and its output stays as it was.
__device__ __forceinline__ int64_t tree_place(const TreeArgs& a, uint32_t r) {
  const int32_t pos = a.row_pos[r], rope = a.row_base ? a.row_rope[r] : pos;
  return uint32_t(rope) < a.rope_rows ? kv_place(a.table, a.row_seq[r], pos) : -1;
}
// One past the last position that row r sees; -1: left out.
__device__ __forceinline__ int32_t tree_extent(const TreeArgs& a, uint32_t r) {
  int32_t base = 0;                                          // (asked for before the place is known: no load waits for another's check)
  uint64_t mask[kTreeMaskWords] = {};
  if (a.row_base) {
    base = a.row_base[r];
#pragma unroll
    for (uint32_t w = 0; w < kTreeMaskWords; ++w)
      if (w < a.mask_words) mask[w] = a.row_mask[r * a.ldm + w];
  }
  if (tree_place(a, r) < 0) return -1;
  if (!a.row_base) return a.row_pos[r] + 1;
  const int32_t most = int32_t(a.table.max_pages * kKvPage);
  base = min(max(base, 0), most);
  int32_t extent = base;
#pragma unroll
  for (uint32_t w = 0; w < kTreeMaskWords; ++w)
    if (mask[w]) extent = min(most, base + 64 * int32_t(w) + 64 - __clzll(mask[w]));
  return extent;
}
// Whether row r (of `base`) sees position p >= base.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, uint32_t r, int32_t node) {
  return uint32_t(node) < a.mask_words * 64u && (a.row_mask[r * a.ldm + (node >> 6)] >> (node & 63) & 1u);
}

// What rounding two values to BF16 (`rounded`) left out of them, rounded to BF16.
__device__ __forceinline__ uint32_t pack_bf_rest(float a, float b, uint32_t rounded) { return pack_bf(__fsub_rn(a, bf_lo(rounded)), __fsub_rn(b, bf_hi(rounded))); }

// Inclusive scans over the CTA.  Op: sums and maxima of values >= 0 alone (the order is free, and 0 changes nothing).
template <class T, class Op>
__device__ __forceinline__ T warp_scan(T v, Op op) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const T o = __shfl_up_sync(0xFFFFFFFFu, v, off);
    if ((threadIdx.x & 31u) >= uint32_t(off)) v = op(o, v);
  }
  return v;
}
template <class T, class Op>
__device__ __forceinline__ T cta_scan(T v, T* scratch /* warps */, Op op) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  v = warp_scan(v, op);
  __syncthreads();
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  const T before = __shfl_sync(0xFFFFFFFFu, warp_scan(lane < blockDim.x / 32 ? scratch[lane] : T(0), op), int(warp + 31) & 31);
  return warp ? op(before, v) : v;
}

// Weight of a unit of so many positions in the 4-bit kernel: its steps of 128 positions, 2350 cycles each, and three more, for 6600 that its beginning and end take (with one:
// 1 row behind 2048 17.8 us instead of 15.7, 128 rows 78.9 instead of 77.1).
__device__ __forceinline__ uint32_t tree_q4_weight(uint32_t positions) { return (positions + 127) / 128 + 3; }

// A tile is up to tile_rows (wide_rows) consecutive rows of one sequence; rows that are left out or see nothing may be among them.
// What it needs of the rows is read once, side by side; the rest runs in shared memory.
// A tile's units have a weight each, one in the kernels that deal them out by number.
template <int FORMAT>
__device__ __forceinline__ void tree_plan(const TreeArgs& a, uint32_t part_positions) {
  extern __shared__ int32_t extents[];                       // [rows]; -1: left out
  uint16_t* const run_of = reinterpret_cast<uint16_t*>(extents + a.rows);      // [rows]: first row of the row's run (rows of one sequence in a row)
  __shared__ int32_t scratch[kTreePrepMost / 32];
  __shared__ unsigned long long sums[kTreePrepMost / 32], total;
  const uint32_t tid = threadIdx.x;
  int32_t run = 0;
  for (uint32_t lo = 0; lo < a.rows; lo += blockDim.x) {
    const uint32_t r = lo + tid;
    const bool in = r < a.rows;
    const int32_t extent = in ? tree_extent(a, r) : -1;
    const bool start = in && (r == 0 || a.row_seq[r] != a.row_seq[r - 1]);
    const int32_t first = cta_scan(start ? int32_t(r) : run, scratch, [](int32_t x, int32_t y) { return max(x, y); });
    if (in) {
      extents[r] = extent;
      run_of[r] = uint16_t(first);
      a.extent[r] = max(extent, 0);
    }
    __syncthreads();
    run = run_of[min(lo + blockDim.x, a.rows) - 1];
  }
  // how many tiles and units there are before a tile, of either kind: tiles above, units (at most 2^32) below
  unsigned long long done = 0, wide_done = 0;
  for (uint32_t lo = 0; lo < a.rows; lo += blockDim.x) {
    const uint32_t r = lo + tid;
    uint32_t n = 0, parts = 0, positions = part_positions;
    int32_t extent = 0;
    bool wide = false;
    if (r < a.rows) {
      const uint32_t first = run_of[r], last = first + a.wide_from - 1;
      wide = a.wide_from && last < a.rows && run_of[last] == first;
      const uint32_t per = wide ? a.wide_rows : a.tile_rows;
      if ((r - first) % per == 0) {
        for (; n < per && r + n < a.rows && run_of[r + n] == first; ++n) extent = max(extent, extents[r + n]);
        if (wide) positions = wide_part<FORMAT>(uint32_t(extent), first + 2 * a.wide_rows < a.rows && run_of[first + 2 * a.wide_rows] == first);
        parts = (uint32_t(extent) + positions - 1) / positions;
        if (wide)
          for (uint32_t i = 0; i < n; ++i) a.row_parts[r + i] = extents[r + i] < 0 ? kTreeRowAbsent : parts;
      }
      if (!wide) a.row_parts[r] = extents[r] < 0 ? kTreeRowAbsent : (uint32_t(extents[r]) + part_positions - 1) / part_positions;
    }
    uint32_t weight = parts;
    if constexpr (FORMAT == kKvQ4) {
      if (!wide && parts) weight = (parts - 1) * tree_q4_weight(part_positions) + tree_q4_weight(uint32_t(extent) - (parts - 1) * part_positions);
    }
    const unsigned long long mine = parts ? (1ull << 32) + weight * a.nkv : 0ull;
    auto scan = [&](bool counts, unsigned long long before) {
      const auto sum = [](unsigned long long x, unsigned long long y) { return x + y; };
      const unsigned long long upto = before + cta_scan(counts ? mine : 0ull, sums, sum);
      if (tid == blockDim.x - 1) total = upto;
      return upto;
    };
    const unsigned long long upto = scan(!wide, done);
    if (parts && !wide) a.tiles[(upto >> 32) - 1] = make_int4(int32_t(r), int32_t(n), int32_t(uint32_t(upto) - weight * a.nkv), extent);
    __syncthreads();
    done = total;
    if (a.wide_from) {
      const unsigned long long wide_upto = scan(wide, wide_done);
      if (parts && wide) a.wide_tiles[(wide_upto >> 32) - 1] = make_int4(int32_t(r), int32_t(n), int32_t(uint32_t(wide_upto) - parts * a.nkv), int32_t(positions));
      __syncthreads();
      wide_done = total;
    }
  }
  if (tid == 0) a.plan[4] = 0u;                              // units that CTAs of the wide kernel have taken beyond their first
  if (tid == 0) a.plan[0] = uint32_t(done >> 32), a.plan[1] = uint32_t(done), a.plan[2] = uint32_t(wide_done >> 32), a.plan[3] = uint32_t(wide_done);
}

// Entries of 4-bit pages from a warp whose lanes hold dimensions 2 l, 2 l + 1, 64 + 2 l and 64 + 2 l + 1 of each; no page: nothing is stored.  N entries side by
// side, whose chains of exchanges and divisions would follow one another.
template <int N>
__device__ __forceinline__ void tree_store_q4(uint8_t* const (&page)[N], uint32_t at, float (&x)[N][4], uint32_t lane) {
  float group[N][2];                                         // of dimensions 32 (l / 16) .. and 64 + 32 (l / 16) ..
  bool fine[N];
  uint32_t exp[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    fine[i] = true;
#pragma unroll
    for (int k = 0; k < 4; ++k) fine[i] = fine[i] && fabsf(x[i][k]) <= 3.4028234e38f;
    fine[i] = __all_sync(0xFFFFFFFFu, fine[i]);
#pragma unroll
    for (int h = 0; h < 2; ++h) group[i][h] = fine[i] ? fmaxf(fabsf(x[i][2 * h]), fabsf(x[i][2 * h + 1])) : 0.f;
  }
#pragma unroll
  for (int off = 8; off; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) group[i][h] = fmaxf(group[i][h], __shfl_xor_sync(0xFFFFFFFFu, group[i][h], off));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float top = fmaxf(group[i][0], group[i][1]);
    exp[i] = q4_exp_byte(fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 16)), true);
  }
  uint32_t code[N][2], scale[N][2];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float step;
      scale[i][h] = q4_scale_byte<false>(group[i][h], exp[i], step);
      // dimensions 2 l and 2 l + 1 are nibble l % 4 of either half of word l / 4
      const uint32_t c = q4_nibble(__fdiv_rn(x[i][2 * h], step)) | q4_nibble(__fdiv_rn(x[i][2 * h + 1], step)) << 16;
      code[i][h] = (fine[i] ? c : 0x00080008u) << 4 * (lane & 3u);
    }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) code[i][h] |= __shfl_xor_sync(0xFFFFFFFFu, code[i][h], off);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!page[i]) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if ((lane & 3u) == 0) reinterpret_cast<uint32_t*>(page[i])[at * (kQ4Codes / 4) + 8 * h + (lane >> 2)] = code[i][h];
      if ((lane & 15u) == 0) page[i][kQ4ScalesAt + at * 4 + 2 * h + (lane >> 4)] = uint8_t(scale[i][h]);
    }
    if (lane == 0) page[i][kQ4ExpsAt + at] = uint8_t(fine[i] ? exp[i] : kKvNanByte);
  }
}

// Rotated queries of `count` neighbouring heads for caches that are decoded to FP16: times a power of two that brings the largest component to [2^14, 2^15): 11 bits
// where BF16 has 8 (one term: a component is off by 2^-11 of itself at most, outputs by 2.2 10^-4, an eighth of what their own rounding to BF16 makes), and
// what falls below FP16's normal range is 2^-28 of the largest.  (Magnitudes compare as their bits do; those of numbers that are not finite
// are the largest.)
template <int N>
__device__ __forceinline__ void tree_store_queries(const TreeArgs& a, uint32_t row, uint32_t head, uint32_t count, const float (&x)[N][4], float log2_scale, uint32_t lane) {
  uint32_t most[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    auto size = [&](int k) { return __float_as_uint(x[i][k]) & 0x7FFFFFFFu; };
    most[i] = __reduce_max_sync(0xFFFFFFFFu, max(max(size(0), size(1)), max(size(2), size(3))));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (uint32_t(i) >= count) break;
    const size_t pair = size_t(row) * a.nq + head + i;
    uint32_t* const dst = reinterpret_cast<uint32_t*>(a.q + pair * kKvDim) + lane;
    const bool fine = most[i] < 0x7F800000u;
    const int e = max(int(most[i] >> 23) - 127 - 14, -100);  // (<= 113)
    const float down = __uint_as_float(uint32_t(127 - e) << 23);
    const __half2 h0 = fine ? __floats2half2_rn(x[i][0] * down, x[i][1] * down) : __floats2half2_rn(0.f, 0.f);
    const __half2 h1 = fine ? __floats2half2_rn(x[i][2] * down, x[i][3] * down) : __floats2half2_rn(0.f, 0.f);
    dst[0] = *reinterpret_cast<const uint32_t*>(&h0);
    dst[32] = *reinterpret_cast<const uint32_t*>(&h1);
    if (lane == 0) a.q_scale[pair] = fine ? __fmul_rn(log2_scale, __uint_as_float(uint32_t(127 + e) << 23)) : __uint_as_float(0x7FC00000u);
  }
}

// The first CTA lays down the plan; in the others a warp takes up to eight neighbouring heads of a row, all their loads on their
// way together.  A lane owns dimensions 2 l, 2 l + 1 and the two that the rotation pairs with them.  The products of BF16 values are
// exact in FP32, so the rotation rounds once before the result is rounded to its type.  1024 rows of 56 heads: 15 us (one head a
// warp 43; 256 rows of the plan at a time 27).  One row: 7 us, the plan's chain of dependent loads.  4 bits: 21 us (the
// entries of a warp one after another: 23; 128 rows 9.5 and 11.4).
constexpr uint32_t kTreeHeadsPerWarp = 8;
template <int FORMAT>
__global__ void __launch_bounds__(kTreePrepMost)
tree_prep_kernel(const TreeArgs a, uint32_t part_positions) {
  constexpr bool F8 = FORMAT != kKvBf16;                   // queries in FP16, as for all caches that are decoded to it
  step_kernel_entry();
  if (blockIdx.x == 0) return tree_plan<FORMAT>(a, part_positions);
  const uint32_t heads = a.nq + 2 * a.nkv, lane = threadIdx.x & 31u, per_row = (heads + kTreeHeadsPerWarp - 1) / kTreeHeadsPerWarp;
  const uint32_t at = (blockIdx.x - 1) * (blockDim.x / 32) + (threadIdx.x >> 5), row = at / per_row, head0 = at % per_row * kTreeHeadsPerWarp;
  if (row >= a.rows) return;
  const uint32_t n = min(kTreeHeadsPerWarp, heads - head0);
  const uint32_t* src = reinterpret_cast<const uint32_t*>(a.qkv + row * a.ldq + size_t(head0) * kKvDim) + lane;
  uint32_t lo[kTreeHeadsPerWarp], hi[kTreeHeadsPerWarp];
#pragma unroll
  for (uint32_t i = 0; i < kTreeHeadsPerWarp; ++i)
    if (i < n) { lo[i] = src[i * (kKvDim / 2)]; hi[i] = src[i * (kKvDim / 2) + 32]; }
  const int32_t rope = a.row_base ? a.row_rope[row] : a.row_pos[row];
  const int64_t place = tree_place(a, row);
  if (place < 0) return;
  const uint32_t* cs = reinterpret_cast<const uint32_t*>(a.cos_table + size_t(rope) * kKvDim) + lane;
  const uint32_t* sn = reinterpret_cast<const uint32_t*>(a.sin_table + size_t(rope) * kKvDim) + lane;
  const float c[4] = {bf_lo(cs[0]), bf_hi(cs[0]), bf_lo(cs[32]), bf_hi(cs[32])};
  const float s[4] = {bf_lo(sn[0]), bf_hi(sn[0]), bf_lo(sn[32]), bf_hi(sn[32])};
  const float log2_scale = __fmul_rn(a.scaling, 1.4426950408889634f);
  if constexpr (FORMAT == kKvQ4) {                           // four at a time, the keys' and values' together
    constexpr uint32_t kSide = 4;
#pragma unroll
    for (uint32_t i0 = 0; i0 < kTreeHeadsPerWarp; i0 += kSide) {
      if (i0 >= n) break;
      float x[kSide][4];
#pragma unroll
      for (uint32_t i = 0; i < kSide; ++i) {
        const uint32_t l = i0 + i < n ? lo[i0 + i] : 0u, h = i0 + i < n ? hi[i0 + i] : 0u;
        const float y[4] = {bf_lo(l), bf_hi(l), bf_lo(h), bf_hi(h)};
        const bool value = head0 + i0 + i >= a.nq + a.nkv;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          x[i][k] = value ? y[k] : __fsub_rn(__fmul_rn(y[k], c[k]), __fmul_rn(y[k + 2], s[k]));
          x[i][k + 2] = value ? y[k + 2] : __fadd_rn(__fmul_rn(y[k + 2], c[k + 2]), __fmul_rn(y[k], s[k + 2]));
        }
      }
      if (head0 + i0 < a.nq) tree_store_queries<kSide>(a, row, head0 + i0, min(a.nq - head0 - i0, n - i0), x, log2_scale, lane);
      if (head0 + min(n, i0 + kSide) > a.nq) {
        uint8_t* page[kSide];
#pragma unroll
        for (uint32_t i = 0; i < kSide; ++i) {
          const uint32_t head = head0 + i0 + i;
          const bool value = head >= a.nq + a.nkv;
          page[i] = i0 + i < n && head >= a.nq ? static_cast<uint8_t*>(value ? a.pages.v : a.pages.k) + q4_page_at(kv_entry(place, a.nkv, value ? head - a.nq - a.nkv : head - a.nq)) : nullptr;
        }
        tree_store_q4<kSide>(page, uint32_t(place % kKvPage), x, lane);
      }
    }
    return;
  }
#pragma unroll
  for (uint32_t i = 0; i < kTreeHeadsPerWarp; ++i) {
    const uint32_t head = head0 + i;
    if (i >= n) break;
    float x[4] = {bf_lo(lo[i]), bf_hi(lo[i]), bf_lo(hi[i]), bf_hi(hi[i])};
    const bool query = head < a.nq, value = head >= a.nq + a.nkv;
    if (!value) {
      float y[4];
      if (!F8 && !query) {    // keys of a BF16 cache: the bits that attn_prep_kernel stores, each product and the sum rounded
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          y[k] = round_bf(__fadd_rn(round_bf(__fmul_rn(x[k], c[k])), round_bf(__fmul_rn(-x[k + 2], s[k]))));
          y[k + 2] = round_bf(__fadd_rn(round_bf(__fmul_rn(x[k + 2], c[k + 2])), round_bf(__fmul_rn(x[k], s[k + 2]))));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          y[k] = __fsub_rn(__fmul_rn(x[k], c[k]), __fmul_rn(x[k + 2], s[k]));
          y[k + 2] = __fadd_rn(__fmul_rn(x[k + 2], c[k + 2]), __fmul_rn(x[k], s[k + 2]));
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = y[k];
    }
    if (query) {
      if constexpr (F8) {
        float one[1][4] = {{x[0], x[1], x[2], x[3]}};
        tree_store_queries<1>(a, row, head, 1, one, log2_scale, lane);
      } else {
        const size_t pair = size_t(row) * a.nq + head;
        uint32_t* dst = reinterpret_cast<uint32_t*>(a.q + pair * 2 * kKvDim) + lane;
        const uint32_t h0 = pack_bf(x[0], x[1]), h1 = pack_bf(x[2], x[3]);
        dst[0] = h0;
        dst[32] = h1;
        dst[64] = pack_bf_rest(x[0], x[1], h0);
        dst[96] = pack_bf_rest(x[2], x[3], h1);
        if (lane == 0) a.q_scale[pair] = log2_scale;
      }
      continue;
    }
    const size_t entry = kv_entry(place, a.nkv, value ? head - a.nq - a.nkv : head - a.nq);
    void* const pages = value ? a.pages.v : a.pages.k;
    if constexpr (F8) {
      const uint32_t byte = kv_warp_byte(x);
      uint16_t* dst = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(pages) + entry * kKvDim) + lane;
      dst[0] = uint16_t(kv_codes(x[0], x[1], byte));
      dst[32] = uint16_t(kv_codes(x[2], x[3], byte));
      if (lane == 0) (value ? a.pages.v_exp : a.pages.k_exp)[entry] = uint8_t(byte);
    } else {
      uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(pages) + entry * kKvDim) + lane;
      dst[0] = pack_bf(x[0], x[1]);
      dst[32] = pack_bf(x[2], x[3]);
    }
  }
}

// ---- one part of the positions for one kv head and a tile of rows ---------------------------------------------------
// 128 threads, 64 KB of K and V per unit (256 positions in 8 bits, 128 in BF16), three CTAs per SM.  The M = 16 rows of a
// warp-level MMA are (row of the tile, query head of the group); each warp takes a quarter of the part's positions:
//   scores  S = Q K^T;  weights w = exp2(S' - max);  O = w V;  the four warps' (max, sum, O) merged in warp order.
// 8 bits: a code becomes FP16 exactly (one conversion for two), straight from shared memory to the MMA's B registers.
// K's scale multiplies the score of its position.  V's goes into the weight: S' = S + e_v, so that the FP16 weights are
// largest where the products are, whatever sizes the values have; the sum of the weights takes it out again.
// 128 rows behind 2048 positions each, 40 heads of 8, 8 bits (410 MB): 100 us, 4.1 TB/s.  With one sequence's five heads in sixteen
// MMA rows, what bounds it is the instructions that turn codes into operands and scores into weights, not their products.
template <bool F8>
struct TreePart {
  static constexpr int kThreads = 128;
  static constexpr uint32_t kPositions = F8 ? 256 : 128;
  static constexpr uint32_t kWarpPositions = kPositions / 4;
  static constexpr int kTiles = kWarpPositions / 8;             // score tiles (8 positions) of a warp
  static constexpr uint32_t kTileBytes = 32768;                 // K or V of a part
  static constexpr uint32_t kExpAt = 2 * kTileBytes;            // exponent bytes of K, then V
  static constexpr uint32_t kSmem = 2 * kTileBytes + (F8 ? 512 : 0);
  static constexpr uint32_t kRowBytes = F8 ? 128 : 256;
  // 16-byte pieces of a row are permuted by the row so that the reads of a warp's eight-lane phases hit all banks: keys two
  // neighbouring rows x four pieces, values four even (or odd) rows x two pieces; BF16: the eight rows of an 8 x 8 matrix
  static __device__ __forceinline__ uint32_t offset(uint32_t row, uint32_t piece) {
    if constexpr (F8) return row * 128u + ((piece ^ (((row >> 1) & 3u) << 1) ^ ((row & 1u) << 2)) << 4);
    else return attn_tile_offset(row, piece);
  }
};

__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The larger of two FP16 pairs' components, a NaN giving way: codes that no entry has (memory nobody wrote) become numbers.
__device__ __forceinline__ uint32_t half2_number(uint32_t v) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x5F005F00u));   // 448
  return r;
}

// Units are numbered tile by tile, part by part, kv head by kv head; a CTA takes a run of them, so that it looks up a tile, and the page
// of a part, once for all kv heads (units dealt round in turn spent longer in chains of look-ups than in arithmetic).
struct TreeUnit {
  int64_t k;                // byte offset of the part's K and V tile in its pool
  int64_t place;            // of the part's first position; -1: no page
  uint32_t tile, first, rows, kvh, part, parts;
  int32_t seq, extent, start;
  uint32_t npos;            // positions of the part up to the tile's last visible one; 0: none
};
// First places of the part the unit is at.
template <bool F8>
__device__ __forceinline__ void tree_look_up(const TreeArgs& a, TreeUnit& t) {
  t.start = int32_t(t.part * TreePart<F8>::kPositions);
  t.place = kv_place(a.table, t.seq, t.start);             // (a part starts on a page or in its middle; outside the pool: as if nobody saw it)
  t.npos = t.place < 0 || t.extent <= t.start ? 0u : min(TreePart<F8>::kPositions, uint32_t(t.extent - t.start));
}
template <bool F8>
__device__ __forceinline__ void tree_set_tile(const TreeArgs& a, TreeUnit& t, const int4& d) {
  t.first = uint32_t(d.x);
  t.rows = uint32_t(d.y);
  t.extent = d.w;
  t.parts = (uint32_t(t.extent) + TreePart<F8>::kPositions - 1) / TreePart<F8>::kPositions;
  t.seq = a.row_seq[t.first];
}
template <bool F8>
__device__ __forceinline__ void tree_locate(const TreeArgs& a, TreeUnit& t) {
  t.k = t.npos ? int64_t(kv_entry(t.place, a.nkv, t.kvh)) * TreePart<F8>::kRowBytes : 0;
}
// The tile of unit number u.  Whole warp.
__device__ __forceinline__ uint32_t tree_tile_of(const TreeArgs& a, uint32_t u, uint32_t tiles) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t lo = 0, n = tiles;                              // the tile is one of n from lo on
  while (n > 1) {
    const uint32_t step = (n + 31) / 32, at = lo + lane * step;
    const uint32_t past = __ballot_sync(0xFFFFFFFFu, lane * step < n && uint32_t(a.tiles[at].z) <= u);      // (lane 0 always)
    const uint32_t k = __popc(past) - 1;
    lo += k * step;
    n = min(step, n - k * step);
  }
  return lo;
}
// The unit of number u.  Whole warp.
template <bool F8>
__device__ __forceinline__ TreeUnit tree_unit(const TreeArgs& a, uint32_t u, uint32_t tiles) {
  TreeUnit t;
  t.tile = tree_tile_of(a, u, tiles);
  const int4 d = a.tiles[t.tile];
  tree_set_tile<F8>(a, t, d);
  const uint32_t local = u - uint32_t(d.z);
  t.kvh = local % a.nkv;
  t.part = local / a.nkv;
  tree_look_up<F8>(a, t);
  tree_locate<F8>(a, t);
  return t;
}
template <bool F8>
__device__ __forceinline__ void tree_next(const TreeArgs& a, TreeUnit& t) {
  if (++t.kvh == a.nkv) {
    t.kvh = 0;
    if (++t.part == t.parts) {
      t.part = 0;
      tree_set_tile<F8>(a, t, a.tiles[++t.tile]);
    }
    tree_look_up<F8>(a, t);
  }
  tree_locate<F8>(a, t);
}

// A thread takes the same piece of every sixteenth (BF16: eighth) row, whose places in shared memory are equally far apart.
template <bool F8>
__device__ __forceinline__ void tree_request(uint32_t dst, const void* pool, const TreeUnit& t, uint32_t tid) {
  constexpr uint32_t kPieces = TreePart<F8>::kRowBytes / 16, kRows = TreePart<F8>::kThreads / kPieces;
  const uint32_t r0 = tid / kPieces;
  const uint8_t* src = static_cast<const uint8_t*>(pool) + t.k + tid * 16;
  dst += TreePart<F8>::offset(r0, tid % kPieces);
  if (t.npos == TreePart<F8>::kPositions) {
#pragma unroll
    for (int i = 0; i < 16; ++i) cp_async_16(dst + i * TreePart<F8>::kThreads * 16, src + i * TreePart<F8>::kThreads * 16, 16u);
  } else {
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      const bool in = r0 + i * kRows < t.npos;
      cp_async_16(dst + i * TreePart<F8>::kThreads * 16, in ? src + i * TreePart<F8>::kThreads * 16 : src, in ? 16u : 0u);
    }
  }
}
// K with both exponent runs (positions beyond the last visible one: bytes of the same page, under a mask)
template <bool F8>
__device__ __forceinline__ void tree_request_k(const TreeArgs& a, uint32_t smem, const TreeUnit& t, uint32_t tid) {
  if (t.npos) {
    tree_request<F8>(smem, a.pages.k, t, tid);
    if constexpr (F8) {
      if (tid < 32) cp_async_16(smem + TreePart<F8>::kExpAt + tid * 16, (tid < 16 ? a.pages.k_exp : a.pages.v_exp) + t.k / 128 + (tid & 15u) * 16, 16u);
    }
  }
  cp_async_commit();
}
template <bool F8>
__device__ __forceinline__ void tree_request_v(const TreeArgs& a, uint32_t smem, const TreeUnit& t, uint32_t tid) {
  if (t.npos) tree_request<F8>(smem + TreePart<F8>::kTileBytes, a.pages.v, t, tid);
  cp_async_commit();
}

// Float index of (MMA row m, 16-byte piece i of its 128 outputs) in a warp's block of the merge buffer, spread over the banks
// for the writers (eight lanes: two rows, pieces 8 apart) and the readers (a row at a time) alike.
__device__ __forceinline__ uint32_t tree_merge_index(uint32_t m, uint32_t piece) { return m * 128u + ((piece ^ ((piece >> 3) | ((m & 1u) << 2))) << 2); }

template <bool CLEAN>
__device__ __forceinline__ void tree_values_f8(float (&o)[16][4], const uint32_t (&pa)[4][4], uint32_t vs, uint32_t p_warp, uint32_t lane) {
  const uint32_t g = lane >> 2, c = lane & 3u;
  const uint32_t even = vs + TreePart<true>::offset(p_warp + 2 * c, g), odd = vs + TreePart<true>::offset(p_warp + 2 * c + 1, g);
#pragma unroll
  for (int t = 0; t < 4; ++t) {                    // 16 positions per step
    uint4 r[4];
    r[0] = lds128(even + 2048 * t);
    r[1] = lds128(odd + 2048 * t);
    r[2] = lds128(even + 2048 * t + 1024);
    r[3] = lds128(odd + 2048 * t + 1024);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t x0 = (&r[0].x)[w], x1 = (&r[1].x)[w], x2 = (&r[2].x)[w], x3 = (&r[3].x)[w];
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // dimensions 16 g + 4 w + 2 half and the next
        uint32_t b00, b01, b10, b11;
        e4m3_to_half4(__byte_perm(x0, x1, half ? 0x7362 : 0x5140), b00, b10);
        e4m3_to_half4(__byte_perm(x2, x3, half ? 0x7362 : 0x5140), b01, b11);
        if (CLEAN) { b00 = half2_number(b00); b01 = half2_number(b01); b10 = half2_number(b10); b11 = half2_number(b11); }
        mma_f16_16816(o[4 * w + 2 * half], pa[t], b00, b01);
        mma_f16_16816(o[4 * w + 2 * half + 1], pa[t], b10, b11);
      }
    }
  }
}

template <bool F8>
__global__ void __launch_bounds__(TreePart<F8>::kThreads, 3)
tree_part_kernel(const TreeArgs a) {
  step_kernel_entry();
  using P = TreePart<F8>;
  constexpr int NT = P::kTiles;
  extern __shared__ __align__(128) unsigned char tree_smem[];
  __shared__ float ml_sm[4][16][2];
  __shared__ uint32_t bad_sm[P::kPositions / 32];     // BF16: positions of the part whose value is not finite
  __shared__ __align__(16) float scales_sm[F8 ? 3 : 1][F8 ? P::kPositions : 4];     // 8 bits: 2^e of K, e and 2^-e of V
  const uint32_t smem = smem_u32(tree_smem), vs = smem + P::kTileBytes;
  float* const merge = reinterpret_cast<float*>(tree_smem + P::kTileBytes);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, c = lane & 3u;
  const uint32_t m0 = lane >> 2, m1 = m0 + 8;         // the two MMA rows whose scores and outputs this lane holds
  const uint32_t tiles = a.plan[0], units = a.plan[1];
  const uint32_t u0 = uint32_t(uint64_t(units) * blockIdx.x / gridDim.x), u1 = uint32_t(uint64_t(units) * (blockIdx.x + 1) / gridDim.x);
  if (u0 == u1) return;
  TreeUnit t = tree_unit<F8>(a, u0, tiles);
  tree_request_k<F8>(a, smem, t, tid);
  tree_request_v<F8>(a, smem, t, tid);
  uint32_t qa[8][4];
  float scale0 = 0.f, scale1 = 0.f;
  // BF16: the queries of a unit, or what their rounding left out (half 1)
  auto ask_bf = [&](const TreeUnit& n, uint32_t half, uint32_t (&x)[8][4]) {
    const uint32_t used = n.rows * a.group, rl0 = m0 / a.group, rl1 = m1 / a.group;
    const bool ok0 = m0 < used, ok1 = m1 < used;
    const uint16_t* s0 = a.q + (2 * (ok0 ? size_t(n.first + rl0) * a.nq + n.kvh * a.group + (m0 - rl0 * a.group) : 0) + half) * kKvDim + c * 2;
    const uint16_t* s1 = a.q + (2 * (ok1 ? size_t(n.first + rl1) * a.nq + n.kvh * a.group + (m1 - rl1 * a.group) : 0) + half) * kKvDim + c * 2;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      x[k][0] = ok0 ? *reinterpret_cast<const uint32_t*>(s0 + 16 * k) : 0u;
      x[k][1] = ok1 ? *reinterpret_cast<const uint32_t*>(s1 + 16 * k) : 0u;
      x[k][2] = ok0 ? *reinterpret_cast<const uint32_t*>(s0 + 16 * k + 8) : 0u;
      x[k][3] = ok1 ? *reinterpret_cast<const uint32_t*>(s1 + 16 * k + 8) : 0u;
    }
  };
  // the queries of a unit as A fragments, MMA row m = (row of the tile) * group + (query head of the group), and their scales
  auto ask_q = [&](const TreeUnit& n) {
    const uint32_t used = n.rows * a.group, rl0 = m0 / a.group, rl1 = m1 / a.group;
    const bool ok0 = m0 < used, ok1 = m1 < used;
    const size_t q0 = ok0 ? size_t(n.first + rl0) * a.nq + n.kvh * a.group + (m0 - rl0 * a.group) : 0;
    const size_t q1 = ok1 ? size_t(n.first + rl1) * a.nq + n.kvh * a.group + (m1 - rl1 * a.group) : 0;
    if constexpr (F8) {       // step 4 h + j of the product takes dimensions 64 h + 16 c + 4 j .. + 3 of lane group c
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 x[2] = {}, y[2] = {};
        if (ok0) { const uint4* s = reinterpret_cast<const uint4*>(a.q + q0 * kKvDim + 64 * h + 16 * c); x[0] = s[0]; x[1] = s[1]; }
        if (ok1) { const uint4* s = reinterpret_cast<const uint4*>(a.q + q1 * kKvDim + 64 * h + 16 * c); y[0] = s[0]; y[1] = s[1]; }
        const uint32_t xs[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
        const uint32_t ys[8] = {y[0].x, y[0].y, y[0].z, y[0].w, y[1].x, y[1].y, y[1].z, y[1].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qa[4 * h + j][0] = xs[2 * j]; qa[4 * h + j][1] = ys[2 * j];
          qa[4 * h + j][2] = xs[2 * j + 1]; qa[4 * h + j][3] = ys[2 * j + 1];
        }
      }
    } else {
      ask_bf(n, 0, qa);
    }
    scale0 = ok0 ? a.q_scale[q0] : 0.f;
    scale1 = ok1 ? a.q_scale[q1] : 0.f;
  };
  ask_q(t);
  for (uint32_t u = u0; u < u1; ++u) {
    TreeUnit next = t;
    const bool more = u + 1 < u1;
    if (more) tree_next<F8>(a, next);
    else next.npos = 0;
    if (!t.npos) {            // a page outside the pool: as if no row saw the part (alike in the whole CTA)
      for (uint32_t m = warp; m < t.rows * a.group; m += 4) {
        const size_t at = (size_t(t.first + m / a.group) * a.nq + t.kvh * a.group + m % a.group) * a.max_parts + t.part;
        *reinterpret_cast<float4*>(a.part_acc + at * kKvDim + lane * 4) = make_float4(0.f, 0.f, 0.f, 0.f);
        if (lane == 0) a.part_ml[at] = make_float2(-INFINITY, 0.f);
      }
      cp_async_wait<0>();
      __syncthreads();
      tree_request_k<F8>(a, smem, next, tid);
      tree_request_v<F8>(a, smem, next, tid);
      if (more) ask_q(next);
      t = next;
      continue;
    }
    const uint32_t used = t.rows * a.group, rl0 = m0 / a.group, rl1 = m1 / a.group;
    const bool ok0 = m0 < used, ok1 = m1 < used;
    const uint32_t row0 = t.first + (ok0 ? rl0 : 0), row1 = t.first + (ok1 ? rl1 : 0);
    // positions of this part below which rows m0 and m1 see everything; behind them, in a tree, the mask decides
    const int32_t base0 = a.row_base ? a.row_base[row0] : 0, base1 = a.row_base ? a.row_base[row1] : 0;
    const int32_t seen0 = ok0 ? min(a.row_base ? base0 : a.extent[row0], a.extent[row0]) - t.start : 0;
    const int32_t seen1 = ok1 ? min(a.row_base ? base1 : a.extent[row1], a.extent[row1]) - t.start : 0;
    // whether some row of the tile does not see the whole part
    uint32_t rest[F8 ? 1 : 8][4];     // BF16: of the queries; needed for the scores alone, so asked for here
    if constexpr (!F8) ask_bf(t, 1, rest);
    const bool holes = __syncthreads_or((ok0 && seen0 < int32_t(P::kPositions)) || (ok1 && seen1 < int32_t(P::kPositions)));
    if (!F8 && holes) {       // values that are not finite would reach, as 0 * infinity, the rows that do not see them
      if (tid < P::kPositions / 32) bad_sm[tid] = 0u;
      cp_async_wait<0>();
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < 16; ++i) {
        const uint32_t piece = tid + i * P::kThreads, r = piece >> 4, at = vs + P::offset(r, piece & 15u);
        const uint4 v = lds128(at);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad = bad || (w[j] & 0x7F80u) == 0x7F80u || (w[j] & 0x7F800000u) == 0x7F800000u;
        if (bad) {
          sts128(at, make_uint4(0u, 0u, 0u, 0u));
          atomicOr(&bad_sm[r >> 5], 1u << (r & 31u));
        }
      }
    } else {
      cp_async_wait<1>();     // all but the newest request: this unit's K
    }
    __syncthreads();
    const uint32_t p_warp = warp * P::kWarpPositions;
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[nt][e] = 0.f;
    if constexpr (F8) {
      // what the positions' exponents mean, a thread two positions of K or of V: 2^e; e and 2^-e
      {
        const uint32_t pair = lds_u16(smem + P::kExpAt + tid * 2), b0 = pair & 0xFFu, b1 = pair >> 8;        // K: this thread's two positions
        // (V's bytes below what an entry has - 0, where nobody wrote - stand for zeros of the smallest size: 2^127 would leave the sums' range)
        const uint32_t vpair = lds_u16(smem + P::kExpAt + 256 + tid * 2), v0 = max(vpair & 0xFFu, kKvLeastByte), v1 = max(vpair >> 8, kKvLeastByte);
        *reinterpret_cast<float2*>(&scales_sm[0][2 * tid]) = make_float2(kv_scale(b0), kv_scale(b1));
        *reinterpret_cast<float2*>(&scales_sm[1][2 * tid]) = make_float2(v0 == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(v0) - 127),
                                                                         v1 == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(v1) - 127));
        *reinterpret_cast<float2*>(&scales_sm[2][2 * tid]) = make_float2(kv_inverse(v0), kv_inverse(v1));
      }
      const uint32_t k0 = smem + P::offset(p_warp + (lane >> 2), c), k1 = smem + P::offset(p_warp + (lane >> 2), c + 4);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 k = lds128((h ? k1 : k0) + 1024 * nt);
          const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t lo, hi;
            e4m3_to_half4(w[j], lo, hi);
            mma_f16_16816(sc[nt], qa[4 * h + j], lo, hi);
          }
        }
      }
      __syncthreads();                              // scales_sm is complete
    } else {
#pragma unroll
      for (int kq = 0; kq < 4; ++kq)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t b[4];
          ldsm_x4(smem + P::offset(p_warp + 8 * nt + (lane & 7u), 4 * kq + (lane >> 3)), b);
          mma_bf16_16816(sc[nt], rest[2 * kq], b[0], b[1]);
          mma_bf16_16816(sc[nt], rest[2 * kq + 1], b[2], b[3]);
          mma_bf16_16816(sc[nt], qa[2 * kq], b[0], b[1]);
          mma_bf16_16816(sc[nt], qa[2 * kq + 1], b[2], b[3]);
        }
    }
    // scores in units of log 2, masked where the part has holes; then the weights
    float mx0 = -INFINITY, mx1 = -INFINITY;
    const bool two = used > 8;      // (otherwise the MMA's upper eight rows are nobody's)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (F8) {
        const uint32_t p = p_warp + 8 * nt + 2 * c;
        const float2 k = *reinterpret_cast<const float2*>(&scales_sm[0][p]), v = *reinterpret_cast<const float2*>(&scales_sm[1][p]);
        sc[nt][0] = __fmaf_rn(__fmul_rn(sc[nt][0], scale0), k.x, v.x);
        sc[nt][1] = __fmaf_rn(__fmul_rn(sc[nt][1], scale0), k.y, v.y);
        if (two) {
          sc[nt][2] = __fmaf_rn(__fmul_rn(sc[nt][2], scale1), k.x, v.x);
          sc[nt][3] = __fmaf_rn(__fmul_rn(sc[nt][3], scale1), k.y, v.y);
        }
      } else {
        sc[nt][0] = __fmul_rn(sc[nt][0], scale0);
        sc[nt][1] = __fmul_rn(sc[nt][1], scale0);
        sc[nt][2] = __fmul_rn(sc[nt][2], scale1);
        sc[nt][3] = __fmul_rn(sc[nt][3], scale1);
      }
    }
    if (holes) {
#pragma unroll 1
      for (int nt = 0; nt < NT; ++nt) {
        const uint32_t p = p_warp + 8 * nt + 2 * c;
        float x[4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (n == nt) { x[0] = sc[n][0]; x[1] = sc[n][1]; x[2] = sc[n][2]; x[3] = sc[n][3]; }
        uint32_t bad = 0;
        if constexpr (!F8) bad = bad_sm[p >> 5] >> (p & 31u);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int32_t pos = int32_t(p) + j;
          bool see0 = pos < seen0, see1 = pos < seen1;
          if (a.row_base) {
            see0 = ok0 && (see0 || tree_sees(a, row0, t.start + pos - base0));
            see1 = ok1 && (see1 || tree_sees(a, row1, t.start + pos - base1));
          }
          if (bad >> j & 1u) x[j] = x[2 + j] = __uint_as_float(0x7FC00000u);
          if (!see0) x[j] = -INFINITY;
          if (!see1) x[2 + j] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
          if (n == nt) { sc[n][0] = x[0]; sc[n][1] = x[1]; sc[n][2] = x[2]; sc[n][3] = x[3]; }
      }
    }
    uint32_t pa[NT / 2][4], pr[F8 ? 1 : NT / 2][4];       // weights; BF16: and what their rounding left out
    float l0 = 0.f, l1 = 0.f;
    // one of the lane's two rows: its maximum over the warp's positions, its weights as A fragments, their sum
    auto weigh = [&](int r, float& mx, float& l) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mx = fmaxf(mx, fmaxf(sc[nt][2 * r], sc[nt][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
      const float low = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float p0 = exp2_approx(__fsub_rn(sc[nt][2 * r], low)), p1 = exp2_approx(__fsub_rn(sc[nt][2 * r + 1], low));
        if constexpr (F8) {
          const float2 i = *reinterpret_cast<const float2*>(&scales_sm[2][p_warp + 8 * nt + 2 * c]);
          l = __fmaf_rn(p0, i.x, __fmaf_rn(p1, i.y, l));
          const __half2 h = __floats2half2_rn(p0, p1);
          pa[nt >> 1][(nt & 1) * 2 + r] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          l = __fadd_rn(l, __fadd_rn(p0, p1));
          pa[nt >> 1][(nt & 1) * 2 + r] = pack_bf(p0, p1);
          pr[nt >> 1][(nt & 1) * 2 + r] = pack_bf_rest(p0, p1, pa[nt >> 1][(nt & 1) * 2 + r]);
        }
      }
      l = __fadd_rn(l, __shfl_xor_sync(0xFFFFFFFFu, l, 1));
      l = __fadd_rn(l, __shfl_xor_sync(0xFFFFFFFFu, l, 2));
    };
    weigh(0, mx0, l0);
    if (two) {
      weigh(1, mx1, l1);
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pa[nt >> 1][(nt & 1) * 2 + 1] = 0u;
        if constexpr (!F8) pr[nt >> 1][(nt & 1) * 2 + 1] = 0u;
      }
    }
    cp_async_wait<0>();
    __syncthreads();                                // V is in shared memory, and every warp is done with K
    tree_request_k<F8>(a, smem, next, tid);
    if (more) ask_q(next);                          // (this unit's scores are done)
    float o[16][4];
#pragma unroll
    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
    if constexpr (F8) {
      // (a tile of one causal row has nothing behind what the row sees; between several rows there may be places that nobody wrote)
      if (holes && (a.row_base || t.rows > 1)) tree_values_f8<true>(o, pa, vs, p_warp, lane);
      else tree_values_f8<false>(o, pa, vs, p_warp, lane);
    } else {
#pragma unroll
      for (int s = 0; s < NT / 2; ++s) {
        const uint32_t vrow = p_warp + 16 * s + ((lane >> 3) & 1u) * 8 + (lane & 7u);
#pragma unroll
        for (int dn = 0; dn < 8; ++dn) {
          uint32_t b[4];
          ldsm_x4_trans(vs + P::offset(vrow, 2 * dn + (lane >> 4)), b);
          mma_bf16_16816(o[2 * dn], pr[s], b[0], b[1]);
          mma_bf16_16816(o[2 * dn + 1], pr[s], b[2], b[3]);
          mma_bf16_16816(o[2 * dn], pa[s], b[0], b[1]);
          mma_bf16_16816(o[2 * dn + 1], pa[s], b[2], b[3]);
        }
      }
    }
    __syncthreads();                                // every warp is done with V: the merge buffer takes its place
    {
      float* mine = merge + size_t(warp) * 16 * kKvDim;
      if constexpr (F8) {                           // the lane holds dimensions 32 c .. 32 c + 31 of its two rows
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *reinterpret_cast<float4*>(mine + tree_merge_index(m0, 8 * c + i)) = make_float4(o[4 * i][0], o[4 * i + 1][0], o[4 * i + 2][0], o[4 * i + 3][0]);
          *reinterpret_cast<float4*>(mine + tree_merge_index(m0, 8 * c + 4 + i)) = make_float4(o[4 * i][1], o[4 * i + 1][1], o[4 * i + 2][1], o[4 * i + 3][1]);
          if (!two) continue;
          *reinterpret_cast<float4*>(mine + tree_merge_index(m1, 8 * c + i)) = make_float4(o[4 * i][2], o[4 * i + 1][2], o[4 * i + 2][2], o[4 * i + 3][2]);
          *reinterpret_cast<float4*>(mine + tree_merge_index(m1, 8 * c + 4 + i)) = make_float4(o[4 * i][3], o[4 * i + 1][3], o[4 * i + 2][3], o[4 * i + 3][3]);
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
          const uint32_t col = 8 * nt + c * 2;
          *reinterpret_cast<float2*>(mine + attn_merge_index(m0, col)) = make_float2(o[nt][0], o[nt][1]);
          if (two) *reinterpret_cast<float2*>(mine + attn_merge_index(m1, col)) = make_float2(o[nt][2], o[nt][3]);
        }
      }
      if (c == 0) {
        ml_sm[warp][m0][0] = mx0; ml_sm[warp][m0][1] = l0;
        ml_sm[warp][m1][0] = mx1; ml_sm[warp][m1][1] = l1;
      }
    }
    __syncthreads();
    for (uint32_t m = warp; m < used; m += 4) {
      float wm[4], mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) { wm[w] = ml_sm[w][m][0]; mx = fmaxf(mx, wm[w]); }
      float den = 0.f;
      float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (a warp that saw nothing adds zeros; one whose scores were all NaN has no maximum either and adds NaN)
        const float e = wm[w] == -INFINITY ? 1.f : exp2_approx(__fsub_rn(wm[w], mx));
        den = __fmaf_rn(e, ml_sm[w][m][1], den);
        const float4 v = *reinterpret_cast<const float4*>(merge + size_t(w) * 16 * kKvDim + (F8 ? tree_merge_index(m, lane) : attn_merge_index(m, lane * 4)));
        num.x = __fmaf_rn(e, v.x, num.x);
        num.y = __fmaf_rn(e, v.y, num.y);
        num.z = __fmaf_rn(e, v.z, num.z);
        num.w = __fmaf_rn(e, v.w, num.w);
      }
      const uint32_t rl = m / a.group;
      const size_t at = (size_t(t.first + rl) * a.nq + t.kvh * a.group + (m - rl * a.group)) * a.max_parts + t.part;
      *reinterpret_cast<float4*>(a.part_acc + at * kKvDim + lane * 4) = num;
      if (lane == 0) a.part_ml[at] = make_float2(mx, den);
    }
    __syncthreads();                                // the merge buffer has been read: V of the next unit may land there
    tree_request_v<F8>(a, smem, next, tid);
    t = next;
  }
  cp_async_wait<0>();
}

// The parts of a (row, query head) merged under their common maximum, in part order, one division, BF16 out.  One warp each; what it
// loads first depends on the number of parts alone.
constexpr int kTreeCombineWarps = 4;
__global__ void __launch_bounds__(kTreeCombineWarps * 32)
tree_combine_kernel(const TreeArgs a) {
  step_kernel_entry();
  constexpr uint32_t kAtOnce = 8;
  const uint32_t pair = blockIdx.x * kTreeCombineWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
  if (pair >= a.rows * a.nq) return;
  const uint32_t row = pair / a.nq, head = pair % a.nq, parts = a.row_parts[row];
  if (parts == kTreeRowAbsent) return;
  const size_t base = size_t(pair) * a.max_parts;
  const float4* acc = reinterpret_cast<const float4*>(a.part_acc + base * kKvDim) + lane;
  float4 v[kAtOnce];
  auto load = [&](uint32_t s0) {
#pragma unroll
    for (uint32_t k = 0; k < kAtOnce; ++k) v[k] = s0 + k < parts ? acc[(s0 + k) * (kKvDim / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  load(0);
  float2 ml = lane < parts ? a.part_ml[base + lane] : make_float2(-INFINITY, 0.f);    // of part s0 + lane, s0 a multiple of 32
  float mx = ml.x;
  for (uint32_t s = lane + 32; s < parts; s += 32) mx = fmaxf(mx, a.part_ml[base + s].x);
  mx = warp_max(mx);
  float den = 0.f;
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t s0 = 0; s0 < parts; s0 += kAtOnce) {
    if (s0) load(s0);
    if (s0 && s0 % 32 == 0) ml = s0 + lane < parts ? a.part_ml[base + s0 + lane] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (uint32_t k = 0; k < kAtOnce; ++k) {
      const float m = __shfl_sync(0xFFFFFFFFu, ml.x, (s0 + k) & 31u), l = __shfl_sync(0xFFFFFFFFu, ml.y, (s0 + k) & 31u);
      const float e = m == -INFINITY ? 1.f : exp2f(__fsub_rn(m, mx));      // (a part that saw nothing adds zeros)
      den = __fmaf_rn(e, l, den);
      num.x = __fmaf_rn(e, v[k].x, num.x);
      num.y = __fmaf_rn(e, v[k].y, num.y);
      num.z = __fmaf_rn(e, v[k].z, num.z);
      num.w = __fmaf_rn(e, v[k].w, num.w);
    }
  }
  if (den == 0.f) den = 1.f;      // nothing seen: zeros
  const uint32_t lo = pack_bf(__fdiv_rn(num.x, den), __fdiv_rn(num.y, den)), hi = pack_bf(__fdiv_rn(num.z, den), __fdiv_rn(num.w, den));
  *reinterpret_cast<uint2*>(a.out + row * a.ldo + head * kKvDim + lane * 4) = make_uint2(lo, hi);
}

}  // namespace grb
