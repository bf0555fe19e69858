// Attention of a step's rows over a paged cache in BF16 or in 8 bits (kv_cache.cuh), for causal rows and for the nodes of
// draft trees: rotary embedding, the append of the rows' keys and values, soft-max attention in parts merged in part order.
//
//   out[r, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(q_rh . k_j / sqrt(128)),  j over the positions that row r sees:
//   causal: j <= row_pos[r];  tree: j < base[r], or bit j - base[r] of the row's mask.  A row that sees nothing gives 0.
//
// Three launches, four where many rows of a sequence may come together.  tree_prep: rotates the queries (once rounded, to the type the matrix instruction takes), stores keys and
// values, and one CTA lays down the plan: tiles of rows of one sequence, and units = (tile, part of the positions, kv head).
// tree_part: persistent CTAs take units in turn.  tree_wide (tree_wide.cuh) does for runs of many rows.
// tree_combine: merges a row's parts.  The parts of a row depend on its own sequence alone (in tree_part on its
// own positions), and every sum runs in a fixed order, so a row's bits do not depend on the batch it is in.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"

namespace grb {

constexpr uint32_t kTreeMaxRows = 4096, kTreeMaskWords = 4;
constexpr int kTreePrepThreads = 256;
// Positions of a wide tile's unit: the most, for long contexts (a unit's result is as large as 256 positions of an 8-bit cache); fewer
// for short ones, whose few units would leave SMs idle.
constexpr uint32_t kWideMostPart = 2048;
__device__ __forceinline__ uint32_t wide_part(uint32_t extent) { return extent <= 1024 ? 256u : extent <= 4096 ? 512u : kWideMostPart; }

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
  uint16_t* q;                // scratch: [rows][nq][128]: rotated queries, BF16 or (8-bit caches) FP16 times a power of two
  float* q_scale;             // scratch: [rows][nq]: what a query's scores are multiplied by, in units of log 2
  uint32_t* status;           // scratch: kStatusTimeout where a wait ran out
  int32_t* extent;            // scratch: [rows]: positions up to the last one the row sees
  uint32_t* row_parts;        // scratch: [rows]: parts of the row
  int4* tiles;                // scratch: [rows]: first row, rows, first unit, positions of a unit
  int4* wide_tiles;           // scratch: [rows]: the same of wide tiles
  uint32_t* plan;             // scratch: tiles, units, wide tiles, wide units
  float* part_acc;            // scratch: [rows][nq][max_parts][128]
  float2* part_ml;            // scratch: [rows][nq][max_parts]: maximum and sum of a part
  __nv_bfloat16* out;         // [rows][ldo]: nq * 128
  int64_t ldo;
  uint32_t rows, nq, nkv, group, tile_rows, max_parts;
  uint32_t wide_rows, wide_from;   // rows of a wide tile; a run of so many rows (0: none) is cut into wide tiles
  float scaling;
};

// The place of row r's own entry; -1: the row is left out (slot -1, or a position outside the table, the pool or the rotary
// tables): nothing is stored for it and its output stays as it was.
__device__ __forceinline__ int64_t tree_place(const TreeArgs& a, uint32_t r) {
  const int32_t pos = a.row_pos[r], rope = a.row_base ? a.row_rope[r] : pos;
  return uint32_t(rope) < a.rope_rows ? kv_place(a.table, a.row_seq[r], pos) : -1;
}
// One past the last position that row r sees.
__device__ __forceinline__ int32_t tree_extent(const TreeArgs& a, uint32_t r) {
  if (tree_place(a, r) < 0) return 0;
  if (!a.row_base) return a.row_pos[r] + 1;
  const int32_t most = int32_t(a.table.max_pages * kKvPage);
  const int32_t base = min(max(a.row_base[r], 0), most);
  for (int w = int(a.mask_words) - 1; w >= 0; --w) {
    const uint64_t m = a.row_mask[r * a.ldm + w];
    if (m) return min(most, base + 64 * w + 64 - __clzll(m));
  }
  return base;
}
// Whether row r (of `base`) sees position p >= base.
__device__ __forceinline__ bool tree_sees(const TreeArgs& a, uint32_t r, int32_t node) {
  return uint32_t(node) < a.mask_words * 64u && (a.row_mask[r * a.ldm + (node >> 6)] >> (node & 63) & 1u);
}

// Inclusive scans over the CTA.
template <class T, class Op>
__device__ __forceinline__ T cta_scan(T v, T* scratch /* warps */, Op op) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const T o = __shfl_up_sync(0xFFFFFFFFu, v, off);
    if (lane >= uint32_t(off)) v = op(o, v);
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = v;
  __syncthreads();
  for (uint32_t w = 0; w < warp; ++w) v = op(scratch[w], v);   // (only sums and maxima of values >= 0 run here: the order is free)
  return v;
}

// A tile is up to tile_rows (wide_rows) consecutive rows of one sequence; rows that are left out or see nothing may be among them.
// What it needs of the rows is read once, side by side; the rest runs in shared memory.
__device__ __forceinline__ void tree_plan(const TreeArgs& a, uint32_t part_positions) {
  extern __shared__ int32_t extents[];                       // [rows]
  uint16_t* const run_of = reinterpret_cast<uint16_t*>(extents + a.rows);      // [rows]: first row of the row's run (rows of one sequence in a row)
  __shared__ int32_t scratch[kTreePrepThreads / 32];
  const uint32_t tid = threadIdx.x;
  const auto larger = [](int32_t x, int32_t y) { return max(x, y); };
  const auto sum = [](int32_t x, int32_t y) { return x + y; };
  int32_t run = 0;
  for (uint32_t lo = 0; lo < a.rows; lo += kTreePrepThreads) {
    const uint32_t r = lo + tid;
    const bool in = r < a.rows;
    const int32_t extent = in ? tree_extent(a, r) : 0;
    const bool start = in && (r == 0 || a.row_seq[r] != a.row_seq[r - 1]);
    const int32_t first = cta_scan(start ? int32_t(r) : run, scratch, larger);
    if (in) {
      extents[r] = extent;
      run_of[r] = uint16_t(first);
      a.extent[r] = extent;
    }
    __syncthreads();
    run = run_of[min(lo + kTreePrepThreads, a.rows) - 1];
  }
  int32_t tiles = 0, units = 0, wide_tiles = 0, wide_units = 0;
  for (uint32_t lo = 0; lo < a.rows; lo += kTreePrepThreads) {
    const uint32_t r = lo + tid;
    uint32_t n = 0, parts = 0, positions = part_positions;
    bool wide = false;
    if (r < a.rows) {
      const uint32_t first = run_of[r], last = first + a.wide_from - 1;
      wide = a.wide_from && last < a.rows && run_of[last] == first;
      const uint32_t per = wide ? a.wide_rows : a.tile_rows;
      if ((r - first) % per == 0) {
        int32_t extent = 0;
        for (; n < per && r + n < a.rows && run_of[r + n] == first; ++n) extent = max(extent, extents[r + n]);
        if (wide) positions = wide_part(uint32_t(extent));
        parts = (uint32_t(extent) + positions - 1) / positions;
        for (uint32_t i = 0; i < n; ++i) a.row_parts[r + i] = wide ? parts : (uint32_t(extents[r + i]) + positions - 1) / positions;
      }
    }
    const int32_t mine = int32_t(parts * a.nkv);
    const int32_t t = cta_scan(int32_t(parts && !wide), scratch, sum), u = cta_scan(wide ? 0 : mine, scratch, sum);
    int32_t wt = 0, wu = 0;
    if (a.wide_from) {
      wt = cta_scan(int32_t(parts && wide), scratch, sum);
      wu = cta_scan(wide ? mine : 0, scratch, sum);
    }
    if (parts) {
      if (wide) a.wide_tiles[wide_tiles + wt - 1] = make_int4(int32_t(r), int32_t(n), wide_units + wu - mine, int32_t(positions));
      else a.tiles[tiles + t - 1] = make_int4(int32_t(r), int32_t(n), units + u - mine, int32_t(positions));
    }
    // the last thread's sums go to everybody
    __shared__ int32_t totals[4];
    __syncthreads();
    if (tid == kTreePrepThreads - 1) totals[0] = t, totals[1] = u, totals[2] = wt, totals[3] = wu;
    __syncthreads();
    tiles += totals[0];
    units += totals[1];
    wide_tiles += totals[2];
    wide_units += totals[3];
  }
  if (tid == 0) a.plan[0] = uint32_t(tiles), a.plan[1] = uint32_t(units), a.plan[2] = uint32_t(wide_tiles), a.plan[3] = uint32_t(wide_units);
}

// The first CTA lays down the plan; in the others a warp takes up to eight neighbouring heads of a row, all their loads on their
// way together (one head a warp: 43 us for 1024 rows of 56 heads).  A lane owns dimensions 2 l, 2 l + 1 and the two that the
// rotation pairs with them.  The products of BF16 values are exact in FP32, so the rotation rounds once before the result is
// rounded to its type.
constexpr uint32_t kTreeHeadsPerWarp = 8;
template <bool F8>
__global__ void __launch_bounds__(kTreePrepThreads)
tree_prep_kernel(const TreeArgs a, uint32_t part_positions) {
  step_kernel_entry();
  if (blockIdx.x == 0) return tree_plan(a, part_positions);
  const uint32_t heads = a.nq + 2 * a.nkv, lane = threadIdx.x & 31u, per_row = (heads + kTreeHeadsPerWarp - 1) / kTreeHeadsPerWarp;
  const uint32_t at = (blockIdx.x - 1) * (kTreePrepThreads / 32) + (threadIdx.x >> 5), row = at / per_row, head0 = at % per_row * kTreeHeadsPerWarp;
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
      const size_t pair = size_t(row) * a.nq + head;
      uint32_t* dst = reinterpret_cast<uint32_t*>(a.q + pair * kKvDim) + lane;
      if constexpr (F8) {
        // FP16 times a power of two that brings the largest component to [2^14, 2^15): 11 bits where BF16 has 8, and what falls
        // below FP16's normal range is 2^-28 of the largest.
        const float m = warp_max(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        bool fine = true;
#pragma unroll
        for (int k = 0; k < 4; ++k) fine = fine && fabsf(x[k]) <= 3.4028234e38f;
        fine = __all_sync(0xFFFFFFFFu, fine);
        const int e = max(int(__float_as_uint(m) >> 23) - 127 - 14, -100);        // (<= 113)
        const float down = __uint_as_float(uint32_t(127 - e) << 23);
        const __half2 h0 = fine ? __floats2half2_rn(x[0] * down, x[1] * down) : __floats2half2_rn(0.f, 0.f);
        const __half2 h1 = fine ? __floats2half2_rn(x[2] * down, x[3] * down) : __floats2half2_rn(0.f, 0.f);
        dst[0] = *reinterpret_cast<const uint32_t*>(&h0);
        dst[32] = *reinterpret_cast<const uint32_t*>(&h1);
        if (lane == 0) a.q_scale[pair] = fine ? __fmul_rn(log2_scale, __uint_as_float(uint32_t(127 + e) << 23)) : __uint_as_float(0x7FC00000u);
      } else {
        dst[0] = pack_bf(x[0], x[1]);
        dst[32] = pack_bf(x[2], x[3]);
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

struct TreeUnit {
  int64_t k;                // byte offset of the part's K and V tile in its pool
  size_t exps;
  uint32_t first, rows, kvh, part;
  int32_t start;
  uint32_t npos;            // positions of the part up to the tile's last visible one; 0: no unit
};

template <bool F8>
__device__ __forceinline__ TreeUnit tree_unit(const TreeArgs& a, uint32_t u, uint32_t units, uint32_t tiles, uint32_t& tile) {
  TreeUnit t{};
  if (u >= units) return t;
  // tiles are in the order of their units; this CTA's units ascend
  const uint32_t lane = threadIdx.x & 31u;
  for (;;) {
    const uint32_t next = tile + 1 + lane;
    const uint32_t past = __ballot_sync(0xFFFFFFFFu, next < tiles && uint32_t(a.tiles[next].z) <= u);
    tile += __popc(past);
    if (past != 0xFFFFFFFFu) break;
  }
  const int4 d = a.tiles[tile];
  const uint32_t local = u - uint32_t(d.z);
  t.first = uint32_t(d.x);
  t.rows = uint32_t(d.y);
  t.kvh = local % a.nkv;
  t.part = local / a.nkv;
  t.start = int32_t(t.part * TreePart<F8>::kPositions);
  int32_t extent = 0;
  for (uint32_t i = lane; i < t.rows; i += 32) extent = max(extent, a.extent[t.first + i]);
#pragma unroll
  for (int off = 16; off; off >>= 1) extent = max(extent, __shfl_xor_sync(0xFFFFFFFFu, extent, off));
  const int64_t place = kv_place(a.table, a.row_seq[t.first], t.start);   // (a part starts on a page or in its middle)
  if (place < 0 || extent <= t.start) return t;                  // (a page outside the pool: as if nobody saw the part)
  t.npos = min(TreePart<F8>::kPositions, uint32_t(extent - t.start));
  const size_t entry = kv_entry(place, a.nkv, t.kvh);
  t.k = int64_t(entry) * TreePart<F8>::kRowBytes;
  t.exps = entry;
  return t;
}

template <bool F8>
__device__ __forceinline__ void tree_request(uint32_t dst, const void* pool, const TreeUnit& t, uint32_t tid) {
  const uint8_t* src = static_cast<const uint8_t*>(pool) + t.k;
  constexpr uint32_t kPieces = TreePart<F8>::kRowBytes / 16;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t c = tid + i * TreePart<F8>::kThreads, r = c / kPieces, piece = c % kPieces;
    cp_async_16(dst + TreePart<F8>::offset(r, piece), src + (r < t.npos ? c * 16 : 0u), r < t.npos ? 16u : 0u);
  }
}
// K with both exponent runs (positions beyond the last visible one: bytes of the same page, under a mask)
template <bool F8>
__device__ __forceinline__ void tree_request_k(const TreeArgs& a, uint32_t smem, const TreeUnit& t, uint32_t tid) {
  if (t.npos) {
    tree_request<F8>(smem, a.pages.k, t, tid);
    if constexpr (F8) {
      if (tid < 32) cp_async_16(smem + TreePart<F8>::kExpAt + tid * 16, (tid < 16 ? a.pages.k_exp : a.pages.v_exp) + t.exps + (tid & 15u) * 16, 16u);
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

template <bool F8, bool CLEAN>
__device__ __forceinline__ void tree_values_f8(float (&o)[16][4], const uint32_t (&pa)[4][4], uint32_t vs, uint32_t p_warp, uint32_t lane) {
  const uint32_t g = lane >> 2, c = lane & 3u;
#pragma unroll
  for (int t = 0; t < 4; ++t) {                    // 16 positions per step
    const uint32_t p = p_warp + 16 * t + 2 * c;
    uint4 r[4];
    r[0] = lds128(vs + TreePart<true>::offset(p, g));
    r[1] = lds128(vs + TreePart<true>::offset(p + 1, g));
    r[2] = lds128(vs + TreePart<true>::offset(p + 8, g));
    r[3] = lds128(vs + TreePart<true>::offset(p + 9, g));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t x0 = (&r[0].x)[w], x1 = (&r[1].x)[w], x2 = (&r[2].x)[w], x3 = (&r[3].x)[w];
#pragma unroll
      for (int half = 0; half < 2; ++half) {       // dimensions 16 g + 4 w + 2 half and the next
        const uint32_t lo = __byte_perm(x0, x1, half ? 0x7362 : 0x5140), hi = __byte_perm(x2, x3, half ? 0x7362 : 0x5140);
        uint32_t b00 = e4m3_to_half2(lo & 0xFFFFu), b01 = e4m3_to_half2(hi & 0xFFFFu), b10 = e4m3_to_half2(lo >> 16), b11 = e4m3_to_half2(hi >> 16);
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
  const uint32_t smem = smem_u32(tree_smem), vs = smem + P::kTileBytes;
  float* const merge = reinterpret_cast<float*>(tree_smem + P::kTileBytes);
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u, c = lane & 3u;
  const uint32_t m0 = lane >> 2, m1 = m0 + 8;         // the two MMA rows whose scores and outputs this lane holds
  const uint32_t tiles = a.plan[0], units = a.plan[1];
  uint32_t tile = 0;
  TreeUnit t = tree_unit<F8>(a, blockIdx.x, units, tiles, tile);
  tree_request_k<F8>(a, smem, t, tid);
  tree_request_v<F8>(a, smem, t, tid);
  for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
    const TreeUnit next = tree_unit<F8>(a, u + gridDim.x, units, tiles, tile);
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
      t = next;
      continue;
    }
    // MMA row m = (row of the tile) * group + (query head of the group)
    const uint32_t used = t.rows * a.group, rl0 = m0 / a.group, rl1 = m1 / a.group;
    const bool ok0 = m0 < used, ok1 = m1 < used;
    const uint32_t row0 = t.first + (ok0 ? rl0 : 0), row1 = t.first + (ok1 ? rl1 : 0);
    const size_t q0 = size_t(row0) * a.nq + t.kvh * a.group + (ok0 ? m0 - rl0 * a.group : 0);
    const size_t q1 = size_t(row1) * a.nq + t.kvh * a.group + (ok1 ? m1 - rl1 * a.group : 0);
    uint32_t qa[8][4];
    if constexpr (F8) {       // step 4 h + j of the product takes dimensions 64 h + 16 c + 4 j .. + 3 of lane group c
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 x[2] = {}, y[2] = {};
        if (ok0) { const uint4* s = reinterpret_cast<const uint4*>(a.q + q0 * kKvDim + 64 * h + 16 * c); x[0] = s[0]; x[1] = s[1]; }
        if (ok1) { const uint4* s = reinterpret_cast<const uint4*>(a.q + q1 * kKvDim + 64 * h + 16 * c); y[0] = s[0]; y[1] = s[1]; }
        const uint32_t* xs = &x[0].x;
        const uint32_t* ys = &y[0].x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          qa[4 * h + j][0] = xs[2 * j]; qa[4 * h + j][1] = ys[2 * j];
          qa[4 * h + j][2] = xs[2 * j + 1]; qa[4 * h + j][3] = ys[2 * j + 1];
        }
      }
    } else {
      const uint16_t* s0 = a.q + q0 * kKvDim + c * 2;
      const uint16_t* s1 = a.q + q1 * kKvDim + c * 2;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qa[k][0] = ok0 ? *reinterpret_cast<const uint32_t*>(s0 + 16 * k) : 0u;
        qa[k][1] = ok1 ? *reinterpret_cast<const uint32_t*>(s1 + 16 * k) : 0u;
        qa[k][2] = ok0 ? *reinterpret_cast<const uint32_t*>(s0 + 16 * k + 8) : 0u;
        qa[k][3] = ok1 ? *reinterpret_cast<const uint32_t*>(s1 + 16 * k + 8) : 0u;
      }
    }
    const float scale0 = ok0 ? a.q_scale[q0] : 0.f, scale1 = ok1 ? a.q_scale[q1] : 0.f;
    // positions of this part below which rows m0 and m1 see everything; behind them, in a tree, the mask decides
    const int32_t base0 = a.row_base ? a.row_base[row0] : 0, base1 = a.row_base ? a.row_base[row1] : 0;
    const int32_t seen0 = ok0 ? min(a.row_base ? base0 : a.extent[row0], a.extent[row0]) - t.start : 0;
    const int32_t seen1 = ok1 ? min(a.row_base ? base1 : a.extent[row1], a.extent[row1]) - t.start : 0;
    // whether the part holds positions that some row of the tile does not see
    const bool holes = __syncthreads_or((ok0 && seen0 < int32_t(t.npos)) || (ok1 && seen1 < int32_t(t.npos)));
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
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 k = lds128(smem + P::offset(p_warp + 8 * nt + (lane >> 2), c + 4 * h));
          const uint32_t w[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_f16_16816(sc[nt], qa[4 * h + j], e4m3_to_half2(w[j] & 0xFFFFu), e4m3_to_half2(w[j] >> 16));
        }
      }
    } else {
#pragma unroll
      for (int kq = 0; kq < 4; ++kq)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          uint32_t b[4];
          ldsm_x4(smem + P::offset(p_warp + 8 * nt + (lane & 7u), 4 * kq + (lane >> 3)), b);
          mma_bf16_16816(sc[nt], qa[2 * kq], b[0], b[1]);
          mma_bf16_16816(sc[nt], qa[2 * kq + 1], b[2], b[3]);
        }
    }
    // scores in units of log 2, masked; then the weights
    float mx0 = -INFINITY, mx1 = -INFINITY;
    uint32_t evs[F8 ? NT : 1];      // exponent bytes of the lane's two positions of every tile: values'
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t p = p_warp + 8 * nt + 2 * c;
      float k0 = 1.f, k1 = 1.f, v0 = 0.f, v1 = 0.f;
      if constexpr (F8) {
        const uint32_t eks = lds_u16(smem + P::kExpAt + p);
        evs[nt] = lds_u16(smem + P::kExpAt + 256 + p);
        k0 = kv_scale(eks & 0xFFu); k1 = kv_scale(eks >> 8);
        const uint32_t b0 = evs[nt] & 0xFFu, b1 = evs[nt] >> 8;
        v0 = b0 == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(b0) - 127);
        v1 = b1 == kKvNanByte ? __uint_as_float(0x7FC00000u) : float(int(b1) - 127);
      } else if (holes) {
        const uint32_t bad = bad_sm[p >> 5] >> (p & 31u);
        if (bad & 1u) v0 = __uint_as_float(0x7FC00000u);
        if (bad & 2u) v1 = __uint_as_float(0x7FC00000u);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int32_t pos = int32_t(p) + j;
        bool see0 = pos < seen0, see1 = pos < seen1;
        if (holes && a.row_base) {
          see0 = ok0 && (see0 || tree_sees(a, row0, t.start + pos - base0));
          see1 = ok1 && (see1 || tree_sees(a, row1, t.start + pos - base1));
        }
        const float k = j ? k1 : k0, v = j ? v1 : v0;
        sc[nt][j] = see0 ? __fmaf_rn(__fmul_rn(sc[nt][j], scale0), k, v) : -INFINITY;
        sc[nt][2 + j] = see1 ? __fmaf_rn(__fmul_rn(sc[nt][2 + j], scale1), k, v) : -INFINITY;
        mx0 = fmaxf(mx0, sc[nt][j]);
        mx1 = fmaxf(mx1, sc[nt][2 + j]);
      }
    }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xFFFFFFFFu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xFFFFFFFFu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xFFFFFFFFu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xFFFFFFFFu, mx1, 2));
    const float low0 = mx0 == -INFINITY ? 0.f : mx0, low1 = mx1 == -INFINITY ? 0.f : mx1;
    float l0 = 0.f, l1 = 0.f;
    uint32_t pa[NT / 2][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float p00 = exp2_approx(__fsub_rn(sc[nt][0], low0)), p01 = exp2_approx(__fsub_rn(sc[nt][1], low0));
      const float p10 = exp2_approx(__fsub_rn(sc[nt][2], low1)), p11 = exp2_approx(__fsub_rn(sc[nt][3], low1));
      if constexpr (F8) {
        const float i0 = kv_inverse(evs[nt] & 0xFFu), i1 = kv_inverse(evs[nt] >> 8);
        l0 = __fmaf_rn(p00, i0, __fmaf_rn(p01, i1, l0));
        l1 = __fmaf_rn(p10, i0, __fmaf_rn(p11, i1, l1));
        const __half2 h0 = __floats2half2_rn(p00, p01), h1 = __floats2half2_rn(p10, p11);
        pa[nt >> 1][(nt & 1) * 2] = *reinterpret_cast<const uint32_t*>(&h0);
        pa[nt >> 1][(nt & 1) * 2 + 1] = *reinterpret_cast<const uint32_t*>(&h1);
      } else {
        l0 = __fadd_rn(l0, __fadd_rn(p00, p01));
        l1 = __fadd_rn(l1, __fadd_rn(p10, p11));
        pa[nt >> 1][(nt & 1) * 2] = pack_bf(p00, p01);
        pa[nt >> 1][(nt & 1) * 2 + 1] = pack_bf(p10, p11);
      }
    }
    l0 = __fadd_rn(l0, __shfl_xor_sync(0xFFFFFFFFu, l0, 1));
    l0 = __fadd_rn(l0, __shfl_xor_sync(0xFFFFFFFFu, l0, 2));
    l1 = __fadd_rn(l1, __shfl_xor_sync(0xFFFFFFFFu, l1, 1));
    l1 = __fadd_rn(l1, __shfl_xor_sync(0xFFFFFFFFu, l1, 2));
    cp_async_wait<0>();
    __syncthreads();                                // V is in shared memory, and every warp is done with K
    tree_request_k<F8>(a, smem, next, tid);
    float o[16][4];
#pragma unroll
    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][e] = 0.f;
    if constexpr (F8) {
      if (holes && a.row_base) tree_values_f8<F8, true>(o, pa, vs, p_warp, lane);
      else tree_values_f8<F8, false>(o, pa, vs, p_warp, lane);
    } else {
#pragma unroll
      for (int s = 0; s < NT / 2; ++s) {
        const uint32_t vrow = p_warp + 16 * s + ((lane >> 3) & 1u) * 8 + (lane & 7u);
#pragma unroll
        for (int dn = 0; dn < 8; ++dn) {
          uint32_t b[4];
          ldsm_x4_trans(vs + P::offset(vrow, 2 * dn + (lane >> 4)), b);
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
          *reinterpret_cast<float4*>(mine + tree_merge_index(m1, 8 * c + i)) = make_float4(o[4 * i][2], o[4 * i + 1][2], o[4 * i + 2][2], o[4 * i + 3][2]);
          *reinterpret_cast<float4*>(mine + tree_merge_index(m1, 8 * c + 4 + i)) = make_float4(o[4 * i][3], o[4 * i + 1][3], o[4 * i + 2][3], o[4 * i + 3][3]);
        }
      } else {
#pragma unroll
        for (int nt = 0; nt < 16; ++nt) {
          const uint32_t col = 8 * nt + c * 2;
          *reinterpret_cast<float2*>(mine + attn_merge_index(m0, col)) = make_float2(o[nt][0], o[nt][1]);
          *reinterpret_cast<float2*>(mine + attn_merge_index(m1, col)) = make_float2(o[nt][2], o[nt][3]);
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

// The parts of a (row, query head) merged under their common maximum, in part order, one division, BF16 out.  One warp each.
constexpr int kTreeCombineWarps = 4;
template <int UNROLL>
__global__ void __launch_bounds__(kTreeCombineWarps * 32)
tree_combine_kernel(const TreeArgs a) {
  step_kernel_entry();
  const uint64_t pair = uint64_t(blockIdx.x) * kTreeCombineWarps + (threadIdx.x >> 5);
  const uint32_t lane = threadIdx.x & 31u;
  if (pair >= uint64_t(a.rows) * a.nq) return;
  const uint32_t row = uint32_t(pair / a.nq), head = uint32_t(pair % a.nq);
  if (tree_place(a, row) < 0) return;
  const uint32_t parts = a.row_parts[row];
  const size_t base = size_t(pair) * a.max_parts;
  float mx = -INFINITY;
  for (uint32_t s = lane; s < parts; s += 32) mx = fmaxf(mx, a.part_ml[base + s].x);
  mx = warp_max(mx);
  float den = 0.f;
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  for (uint32_t s0 = 0; s0 < parts; s0 += UNROLL) {
    float4 v[UNROLL];
    float2 ml[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const bool in = s0 + j < parts;
      v[j] = in ? *(reinterpret_cast<const float4*>(a.part_acc + (base + s0 + j) * kKvDim) + lane) : make_float4(0.f, 0.f, 0.f, 0.f);
      ml[j] = in ? a.part_ml[base + s0 + j] : make_float2(-INFINITY, 0.f);
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const float e = ml[j].x == -INFINITY ? 1.f : exp2f(__fsub_rn(ml[j].x, mx));
      den = __fmaf_rn(e, ml[j].y, den);
      num.x = __fmaf_rn(e, v[j].x, num.x);
      num.y = __fmaf_rn(e, v[j].y, num.y);
      num.z = __fmaf_rn(e, v[j].z, num.z);
      num.w = __fmaf_rn(e, v[j].w, num.w);
    }
  }
  if (den == 0.f) den = 1.f;      // nothing seen: zeros
  const uint32_t lo = pack_bf(__fdiv_rn(num.x, den), __fdiv_rn(num.y, den)), hi = pack_bf(__fdiv_rn(num.z, den), __fdiv_rn(num.w, den));
  *reinterpret_cast<uint2*>(a.out + row * a.ldo + head * kKvDim + lane * 4) = make_uint2(lo, hi);
}

}  // namespace grb
