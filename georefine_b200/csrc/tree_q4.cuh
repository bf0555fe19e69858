// The narrow attention of tree_attention.cuh over a 4-bit cache: one part of the positions for one kv head and a tile of rows.
//
// Columns of a warp-level MMA are (row of the tile, query head of the group), at most 16 in one or two blocks of eight; positions and
// dimensions are its rows, so that the five heads of a decode row fill five of eight columns, not of sixteen rows, and an operand of codes
// meets all columns at once:
//   scores  S^T = K Q^T (16 positions x 16 dimensions a step);  weights w = exp2(S' - reference);  outputs  O^T = V^T w^T.
// A warp takes every fourth 32 positions of a part and keeps its reference, sum and O from its first to its last; the four warps
// are merged in warp order.  The reference moves when a score has passed it by 2^8; then O is scaled down.  Each warp copies its own codes into a
// ring of its own, three chunks ahead and across units, so warps meet at the end of a unit alone and nothing waits for another CTA.
//
// A code becomes an FP16 operand with 1.1 instructions (q4_operands).  A group's scale goes into the operand, where it is exact; K's exponent
// multiplies the score of its position, V's goes into the weight, as in 8 bits: S' = S 2^e_k scale + e_v, and the sum of the weights takes it out again.
#pragma once
#include "tree_attention.cuh"

namespace grb {

struct TreeQ4 {
  static constexpr int kThreads = 128;
  static constexpr uint32_t kPositions = 512;                // of a part
  static constexpr uint32_t kChunk = 32;                     // positions of a warp's step
  static constexpr uint32_t kStages = 4;
  static constexpr uint32_t kVAt = kChunk * kQ4Codes, kKScalesAt = 2 * kVAt, kVScalesAt = kKScalesAt + kChunk * 4, kKExpsAt = kVScalesAt + kChunk * 4,
                            kVExpsAt = kKExpsAt + kChunk, kStage = kVExpsAt + kChunk;
  static constexpr uint32_t kSmem = 4 * kStages * kStage;
};
static_assert(TreeQ4::kStage >= 8 * kKvDim * 4, "a warp's stage holds its part of the merge, eight columns at a time");
static_assert(TreeQ4::kStage % 16 == 0 && kKvPage % TreeQ4::kChunk == 0, "copies of 16 bytes; a chunk lies in one page");

__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// An 8 x 8 matrix of 16-bit values across the warp, transposed.
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// What two scales (bytes in bits 0-7 and 16-23) make of nibbles: F, F / 16, -8 F 2^-24.  The byte moved to the upper end of an FP16's
// fraction and four bits of exponent is F 2^-15, below 16 a subnormal one.
struct Q4Factors {
  uint32_t low, high, offset;
};
__device__ __forceinline__ Q4Factors q4_factors(uint32_t bytes) {
  const uint32_t f = mul_f16x2(bytes << 6, 0x78007800u);     // 2^15
  return Q4Factors{f, mul_f16x2(f, 0x2C002C00u), mul_f16x2(f, 0x80088008u)};
}
// Nibble j of both halves of a word as a pair of FP16 numbers, code F 2^-24: the nibbles are subnormals u 2^-24 (or u 2^-20, times F / 16).
__device__ __forceinline__ void q4_operands(uint32_t w, const Q4Factors& f, uint32_t (&y)[4]) {
  const uint32_t upper = w >> 8;
  y[0] = fma_f16x2(w & 0x000F000Fu, f.low, f.offset);
  y[1] = fma_f16x2(w & 0x00F000F0u, f.high, f.offset);
  y[2] = fma_f16x2(upper & 0x000F000Fu, f.low, f.offset);
  y[3] = fma_f16x2(upper & 0x00F000F0u, f.high, f.offset);
}

// Units are numbered as in tree_part_kernel: tile by tile, part by part, kv head by kv head; a CTA takes a run of them.
struct Q4Unit {
  uint32_t tile, first, rows, kvh, part, parts;
  int32_t seq, extent;
};
__device__ __forceinline__ void q4_set_tile(const TreeArgs& a, Q4Unit& t) {
  const int4 d = a.tiles[t.tile];
  t.first = uint32_t(d.x);
  t.rows = uint32_t(d.y);
  t.extent = d.w;
  t.parts = (uint32_t(t.extent) + TreeQ4::kPositions - 1) / TreeQ4::kPositions;
  t.seq = a.row_seq[t.first];
}
__device__ __forceinline__ void q4_next(const TreeArgs& a, Q4Unit& t) {
  if (++t.kvh < a.nkv) return;
  t.kvh = 0;
  if (++t.part < t.parts) return;
  t.part = 0;
  ++t.tile;
  q4_set_tile(a, t);
}
// Chunks that a warp takes of the unit: positions 512 part + 128 i + 32 warp .. + 31 for i below this.
__device__ __forceinline__ uint32_t q4_chunks(const Q4Unit& t, uint32_t warp) {
  const int32_t n = min(t.extent - int32_t(t.part * TreeQ4::kPositions), int32_t(TreeQ4::kPositions)) - int32_t(warp * TreeQ4::kChunk);
  return uint32_t(max(n, 0) + 4 * TreeQ4::kChunk - 1) / (4 * TreeQ4::kChunk);
}

// What a lane keeps of a unit's columns: of block b, the queries of column 8 b + lane / 4 as B operands, and of its score columns
// 8 b + 2 (lane % 4) + j the factor, the row, and the position below which the row sees everything.
template <int NB>
struct Q4Columns {
  uint4 q[NB][4];
  float scale[NB][2];
  int32_t below[NB][2];            // behind it, in a tree, the mask decides; columns that are nobody's see everything
};

struct Q4Warp {                    // a lane's places, the same for all units
  uint32_t warp, lane, r, c, place;      // place: of MMA row r (and, 8 further, of row r + 8) among a tile's 16 positions
};

template <int NB>
__device__ __forceinline__ void q4_ask_columns(const TreeArgs& a, const Q4Unit& t, const Q4Warp& w, Q4Columns<NB>& k) {
  const uint32_t used = t.rows * a.group;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t n = 8 * b + w.r, rl = n / a.group;
    const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t(t.first + rl) * a.nq + t.kvh * a.group + (n - rl * a.group)) * kKvDim + 32 * w.c);
#pragma unroll
    for (int i = 0; i < 4; ++i) k.q[b][i] = n < used ? src[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t m = 8 * b + 2 * w.c + j, ml = m / a.group, row = t.first + ml;
      const bool in = m < used;
      k.scale[b][j] = in ? a.q_scale[size_t(row) * a.nq + t.kvh * a.group + (m - ml * a.group)] : 0.f;
      k.below[b][j] = in ? a.row_base ? min(a.row_base[row], a.extent[row]) : a.extent[row] : 0x7FFFFFFF;
    }
  }
}

// One warp's 32 positions from `at` on, against NB blocks of eight columns.
template <int NB>
__device__ __forceinline__ void q4_chunk(const TreeArgs& a, const Q4Unit& t, const Q4Warp& w, uint32_t stage, int32_t at, const Q4Columns<NB>& k, float (&ref)[NB][2],
                                         float (&sum)[NB][2], float (&o)[NB][8][4]) {
  constexpr float kSlack = 8.f, kBias = 7.f;                 // FP16 weights: up to 2^(7 + 8)
  using P = TreeQ4;
  float s[2][NB][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {                              // 16 positions
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][b][e] = 0.f;
    const uint32_t p = 16 * i + w.place;
    const uint4 k0 = lds128(stage + p * kQ4Codes + 16 * w.c), k1 = lds128(stage + (p + 8) * kQ4Codes + 16 * w.c);
    // (a lane's 16 bytes are a group of 32 dimensions of one position: one scale)
    const Q4Factors f0 = q4_factors(lds_u8(stage + P::kKScalesAt + 4 * p + w.c) * 0x10001u), f1 = q4_factors(lds_u8(stage + P::kKScalesAt + 4 * (p + 8) + w.c) * 0x10001u);
    const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t x[4], y[4];
      q4_operands(w0[j], f0, x);
      q4_operands(w1[j], f1, y);
      const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mma_f16_16816(s[i][b], a0, k.q[b][j].x, k.q[b][j].y);
        mma_f16_16816(s[i][b], a1, k.q[b][j].z, k.q[b][j].w);
      }
    }
  }
  // scores in units of log 2, with V's exponent; masked where some row does not see the whole chunk
  float inverse[2][2];                                       // 2^-e of V
  bool hole = false;
#pragma unroll
  for (int b = 0; b < NB; ++b) hole = hole || min(k.below[b][0], k.below[b][1]) < at + int32_t(P::kChunk);
  const bool holes = __any_sync(0xFFFFFFFFu, hole);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t p = 16 * i + 8 * h + w.place;
      const uint32_t kb = lds_u8(stage + P::kKExpsAt + p), vb = max(lds_u8(stage + P::kVExpsAt + p), kKvLeastByte);
      const float up = kv_scale(kb), add = vb == kKvNanByte ? __uint_as_float(0x7FC00000u) : __fsub_rn(__uint_as_float(0x4B000000u | vb), 8388735.f);      // 2^23 + 127
      inverse[i][h] = kv_inverse(vb);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) s[i][b][2 * h + j] = __fmaf_rn(__fmul_rn(s[i][b][2 * h + j], k.scale[b][j]), up, add);
    }
  if (holes) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t m = 8 * b + 2 * w.c + j;
        if (m >= t.rows * a.group) continue;
        const uint32_t row = t.first + m / a.group;
        const int32_t base = a.row_base ? a.row_base[row] : 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int32_t pos = at + int32_t(16 * i + 8 * h + w.place);
            if (pos >= k.below[b][j] && !(a.row_base && tree_sees(a, row, pos - base))) s[i][b][2 * h + j] = -INFINITY;
          }
      }
  }
  float top[NB][2];
  bool move = false;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      top[b][j] = fmaxf(fmaxf(s[0][b][j], s[0][b][2 + j]), fmaxf(s[1][b][j], s[1][b][2 + j]));
      move = move || top[b][j] > (ref[b][j] == -INFINITY ? ref[b][j] : __fadd_rn(ref[b][j], kSlack));
    }
  if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {                          // (the eight lanes of a column agree)
        float v = top[b][j];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
        if (!(v > (ref[b][j] == -INFINITY ? ref[b][j] : __fadd_rn(ref[b][j], kSlack)))) continue;
        const float f = exp2_approx(__fsub_rn(ref[b][j], v));      // (from -infinity: 0)
        ref[b][j] = v;
        sum[b][j] = __fmul_rn(sum[b][j], f);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          o[b][d][j] = __fmul_rn(o[b][d][j], f);
          o[b][d][2 + j] = __fmul_rn(o[b][d][2 + j], f);
        }
      }
  }
  uint32_t weights[2][NB][2];                                // B operands: positions by columns
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const float low0 = (ref[b][0] == -INFINITY ? 0.f : ref[b][0]) - kBias, low1 = (ref[b][1] == -INFINITY ? 0.f : ref[b][1]) - kBias;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float e0 = exp2_approx(__fsub_rn(s[i][b][2 * h], low0)), e1 = exp2_approx(__fsub_rn(s[i][b][2 * h + 1], low1));
        sum[b][0] = __fmaf_rn(e0, inverse[i][h], sum[b][0]);
        sum[b][1] = __fmaf_rn(e1, inverse[i][h], sum[b][1]);
        const __half2 pair = __floats2half2_rn(e0, e1);
        weights[i][b][h] = movmatrix(*reinterpret_cast<const uint32_t*>(&pair));
      }
  }
  // MMA row r of these products is a dimension of 16 r .. 16 r + 15, whose 8 bytes the lane reads of the four positions of its columns c
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t p0 = 16 * i + w.c, p1 = 16 * i + 4 + (w.c ^ 1u);      // places of MMA rows 2 c and 2 c + 1; 8 further those of 2 c + 8 and 2 c + 9
    const uint32_t codes = stage + P::kVAt + 8 * w.r, scales = stage + P::kVScalesAt + (w.r >> 1);
    const uint2 x0 = lds64(codes + p0 * kQ4Codes), x1 = lds64(codes + p1 * kQ4Codes), x2 = lds64(codes + (p0 + 8) * kQ4Codes), x3 = lds64(codes + (p1 + 8) * kQ4Codes);
    const Q4Factors f01 = q4_factors(lds_u8(scales + 4 * p0) | lds_u8(scales + 4 * p1) << 16), f23 = q4_factors(lds_u8(scales + 4 * (p0 + 8)) | lds_u8(scales + 4 * (p1 + 8)) << 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {                            // eight dimensions
      const uint32_t y0 = h ? x0.y : x0.x, y1 = h ? x1.y : x1.x, y2 = h ? x2.y : x2.x, y3 = h ? x3.y : x3.x;
#pragma unroll
      for (int odd = 0; odd < 2; ++odd) {                    // dimensions odd, odd + 2, odd + 4, odd + 6 of them
        uint32_t u[4], v[4];
        q4_operands(__byte_perm(y0, y1, odd ? 0x7632 : 0x5410), f01, u);
        q4_operands(__byte_perm(y2, y3, odd ? 0x7632 : 0x5410), f23, v);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t x[4] = {u[2 * q], u[2 * q + 1], v[2 * q], v[2 * q + 1]};
#pragma unroll
          for (int b = 0; b < NB; ++b) mma_f16_16816(o[b][4 * h + 2 * odd + q], x, weights[i][b][0], weights[i][b][1]);
        }
      }
    }
  }
}

// Float index of (column m of eight, 16-byte piece i of its 128 outputs) in a warp's block of the merge, spread over the banks.
__device__ __forceinline__ uint32_t q4_merge_index(uint32_t m, uint32_t piece) { return m * 128u + ((piece ^ (m >> 1)) << 2); }

__global__ void __launch_bounds__(TreeQ4::kThreads, 3)
tree_q4_kernel(const TreeArgs a) {
  step_kernel_entry();
  using P = TreeQ4;
  extern __shared__ __align__(128) unsigned char tree_smem[];
  __shared__ float ml_sm[4][16][2];
  const uint32_t tid = threadIdx.x;
  Q4Warp w;
  w.warp = tid >> 5;
  w.lane = tid & 31u;
  w.r = w.lane >> 2;
  w.c = w.lane & 3u;
  // Places are dealt so that neighbouring MMA rows lie in entries of different parity: 64-byte rows, two of which share all banks.
  w.place = w.r & 1u ? 4u + ((w.r >> 1) ^ 1u) : w.r >> 1;
  const uint32_t tiles = a.plan[0], units = a.plan[1];
  const uint32_t u0 = uint32_t(uint64_t(units) * blockIdx.x / gridDim.x), u1 = uint32_t(uint64_t(units) * (blockIdx.x + 1) / gridDim.x);
  if (u0 == u1) return;
  const uint32_t ring = smem_u32(tree_smem) + w.warp * P::kStages * P::kStage;
  Q4Unit t;
  t.tile = tree_tile_of(a, u0, tiles);
  q4_set_tile(a, t);
  {
    const uint32_t local = u0 - uint32_t(a.tiles[t.tile].z);
    t.kvh = local % a.nkv;
    t.part = local / a.nkv;
  }
  // The chunks of the run in their order: where the next one to be copied lies is looked up while the one before is on its way.
  Q4Unit ahead = t;
  uint32_t left = u1 - u0, chunk = 0, asked = 0, there = 0;  // units left; of the unit; chunks asked for; whether the last 32 of them have a page
  int32_t page = -1;                                         // (looked at a chunk later: nothing waits for the load)
  auto position = [&]() { return ahead.part * P::kPositions + chunk * 4 * P::kChunk + w.warp * P::kChunk; };
  auto find = [&]() {                                        // the next chunk, from (ahead, chunk) on
    while (left && chunk >= q4_chunks(ahead, w.warp)) {
      chunk = 0;
      if (--left) q4_next(a, ahead);
    }
    const uint32_t p = position() / kKvPage;
    page = left && uint32_t(ahead.seq) < a.table.slots && p < a.table.max_pages ? a.table.table[ahead.seq * a.table.ld + p] : -1;
  };
  auto request = [&]() {
    if (left) {
      const bool in = uint32_t(page) < a.table.pages;
      there = (there & ~(1u << (asked & 31u))) | uint32_t(in) << (asked & 31u);
      if (in) {
        const size_t block = (size_t(page) * a.nkv + ahead.kvh) * kQ4Page;
        const uint32_t at = position() % kKvPage, dst = ring + (asked % P::kStages) * P::kStage;
        const uint8_t* const k = static_cast<const uint8_t*>(a.pages.k) + block;
        const uint8_t* const v = static_cast<const uint8_t*>(a.pages.v) + block;
#pragma unroll
        for (int i = 0; i < 4; ++i) cp_async_16(dst + (w.lane + 32 * i) * 16, k + at * kQ4Codes + (w.lane + 32 * i) * 16, 16u);
#pragma unroll
        for (int i = 0; i < 4; ++i) cp_async_16(dst + P::kVAt + (w.lane + 32 * i) * 16, v + at * kQ4Codes + (w.lane + 32 * i) * 16, 16u);
        if (w.lane < 20) {                                   // 8 pieces of either's scales, 2 of either's exponents
          const bool scales = w.lane < 16;
          const uint32_t i = scales ? w.lane : w.lane - 16, half = scales ? 8u : 2u, piece = i % half;
          const uint8_t* const src = (i < half ? k : v) + (scales ? kQ4ScalesAt + at * 4 : kQ4ExpsAt + at) + piece * 16;
          cp_async_16(dst + (scales ? P::kKScalesAt : P::kKExpsAt) + i * 16, src, 16u);
        }
      }
      ++asked;
      ++chunk;
      find();
    }
    cp_async_commit();
  };
  find();
  for (uint32_t i = 0; i + 1 < P::kStages; ++i) request();

  uint32_t g = 0;                                            // chunks this warp has taken
  auto run = [&](auto blocks, const Q4Unit& unit) {
    constexpr int NB = decltype(blocks)::value;
    Q4Columns<NB> columns;
    q4_ask_columns<NB>(a, unit, w, columns);
    float ref[NB][2], sum[NB][2], o[NB][8][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int j = 0; j < 2; ++j) { ref[b][j] = -INFINITY; sum[b][j] = 0.f; }
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[b][d][e] = 0.f;
    }
    const uint32_t n = q4_chunks(unit, w.warp);
    const int32_t start = int32_t(unit.part * P::kPositions + w.warp * P::kChunk);
    for (uint32_t i = 0; i < n; ++i, ++g) {
      request();                                             // (into the stage that the chunk before has left)
      cp_async_wait<P::kStages - 1>();
      __syncwarp();
      // a page outside the pool: as if nobody saw the chunk
      if (there >> (g & 31u) & 1u) q4_chunk<NB>(a, unit, w, ring + (g % P::kStages) * P::kStage, start + int32_t(i * 4 * P::kChunk), columns, ref, sum, o);
      __syncwarp();
    }
    // the warps' results merged, eight columns at a time, through the stage of each that is free
    const uint32_t used = unit.rows * a.group, free_stage = (g + P::kStages - 1) % P::kStages;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = sum[b][j];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l = __fadd_rn(l, __shfl_xor_sync(0xFFFFFFFFu, l, off));
        if (w.r == 0) {
          ml_sm[w.warp][8 * b + 2 * w.c + j][0] = ref[b][j] == -INFINITY ? ref[b][j] : ref[b][j] - 7.f;
          ml_sm[w.warp][8 * b + 2 * w.c + j][1] = l;
        }
      }
      float* const mine = reinterpret_cast<float*>(tree_smem + (w.warp * P::kStages + free_stage) * P::kStage);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {                        // dimensions 16 r + 4 q ..: of word q / 2, 4 (q % 2) on
          const int d = 4 * (q >> 1) + (q & 1);
          *reinterpret_cast<float4*>(mine + q4_merge_index(2 * w.c + j, 4 * w.r + q)) = make_float4(o[b][d][j], o[b][d + 2][j], o[b][d][2 + j], o[b][d + 2][2 + j]);
        }
      // (where the other warps put theirs: their own free stages)
      __shared__ uint32_t stage_sm[4];
      if (w.lane == 0) stage_sm[w.warp] = (w.warp * P::kStages + free_stage) * P::kStage;
      __syncthreads();
      for (uint32_t m = w.warp; m < 8 && 8 * b + m < used; m += 4) {
        float wm[4], mx = -INFINITY, den = 0.f;
        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 4; ++x) { wm[x] = ml_sm[x][8 * b + m][0]; mx = fmaxf(mx, wm[x]); }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // (a warp that saw nothing adds zeros; one whose scores were all NaN has no reference either and adds NaN)
          const float e = wm[x] == -INFINITY ? 1.f : exp2_approx(__fsub_rn(wm[x], mx));
          den = __fmaf_rn(e, ml_sm[x][8 * b + m][1], den);
          const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(tree_smem + stage_sm[x]) + q4_merge_index(m, w.lane));
          num.x = __fmaf_rn(e, v.x, num.x);
          num.y = __fmaf_rn(e, v.y, num.y);
          num.z = __fmaf_rn(e, v.z, num.z);
          num.w = __fmaf_rn(e, v.w, num.w);
        }
        const uint32_t col = 8 * b + m, rl = col / a.group;
        const size_t at = (size_t(unit.first + rl) * a.nq + unit.kvh * a.group + (col - rl * a.group)) * a.max_parts + unit.part;
        *reinterpret_cast<float4*>(a.part_acc + at * kKvDim + w.lane * 4) = num;
        if (w.lane == 0) a.part_ml[at] = make_float2(mx, den);
      }
      __syncthreads();                                       // the stages are free again
    }
  };
  for (uint32_t u = u0; u < u1; ++u) {
    if (t.rows * a.group > 8) run(std::integral_constant<int, 2>{}, t);
    else run(std::integral_constant<int, 1>{}, t);
    if (u + 1 < u1) q4_next(a, t);
  }
  cp_async_wait<0>();
}

}  // namespace grb
