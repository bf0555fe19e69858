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
//
// Queries and weights are FP16, one term each, as over 8 bits: rounded by 2^-11 of themselves at most, they put outputs behind 2048 normal entries 2.9 10^-4 off (relative),
// which are then rounded to BF16, 1.63 10^-3: 1.66 in all.  A second term of either would double its products.  References, sums and O are FP32.
//
// Instructions bound it, and the chains between them: 560 for 32 positions of a head, of which 288 make operands of codes and 32 are the products; the four warps of a
// scheduler issue in 58 % of the cycles.  6600 of a unit's 15000 cycles (44 %) go to its beginning and end - the next one found, its columns, the merge.  128 rows
// behind 1024 to 2048 positions, 40 heads of 8 (221 MB): 70 us, 3.2 TB/s; all launches 77, where the 8-bit cache takes 107 with 410 MB; 8 rows behind
// 16384 to 32768 (230 MB): 69.  (Heads as rows of the products, as in 8 bits, would fill five rows of sixteen with twice the operands; a warp's four chunks written out one after
// another no longer fit the instruction cache: 84.)
#pragma once
#include "tree_attention.cuh"

namespace grb {

struct TreeQ4 {
  static constexpr int kThreads = 128;
  static constexpr uint32_t kPositions = 512;                // of a part
  static constexpr uint32_t kChunk = 32;                     // positions of a warp's step
  static constexpr uint32_t kChunks = 4;                     // of a warp and unit
  static constexpr uint32_t kStages = 3;
  static constexpr uint32_t kVAt = kChunk * kQ4Codes, kKScalesAt = 2 * kVAt, kVScalesAt = kKScalesAt + kChunk * 4, kKExpsAt = kVScalesAt + kChunk * 4,
                            kVExpsAt = kKExpsAt + kChunk, kStage = kVExpsAt + kChunk;
  static constexpr uint32_t kWarp = kStages * kStage + kChunk * 16;    // and what the exponents of the chunk at hand mean
  static constexpr uint32_t kSmem = 4 * kWarp;
};
static_assert(TreeQ4::kChunks * 4 * TreeQ4::kChunk == TreeQ4::kPositions && TreeQ4::kPositions == 2 * kKvPage, "a unit is two pages, four chunks a warp");
static_assert(TreeQ4::kStage >= 8 * kKvDim * 4, "a warp's stage holds its part of the merge, eight columns at a time");
static_assert(TreeQ4::kStage % 16 == 0 && kKvPage % TreeQ4::kChunk == 0, "copies of 16 bytes; a chunk lies in one page");

constexpr float kQ4Bias = 7.f;                               // FP16 weights: up to 2^(7 + the 8 by which a score may pass the reference)

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
// The product of mma_f16_16816, and loads from shared memory, that the compiler may move: a tile's loads go before the products of the tile
// before it.
__device__ __forceinline__ void mma_q4(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <class T>
__device__ __forceinline__ T q4_ld(const unsigned char* p) { return *reinterpret_cast<const T*>(p); }
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

// Units follow one another tile by tile, part by part, kv head by kv head; a CTA takes those that start in its share of the plan's weights.
struct Q4Unit {
  uint32_t tile, first, rows, kvh, part, parts;
  uint32_t at;              // where the unit starts, in weights
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
__device__ __forceinline__ uint32_t q4_unit_weight(const Q4Unit& t) { return tree_q4_weight(min(TreeQ4::kPositions, uint32_t(t.extent) - t.part * TreeQ4::kPositions)); }
__device__ __forceinline__ void q4_next(const TreeArgs& a, Q4Unit& t, uint32_t end) {
  t.at += q4_unit_weight(t);
  if (++t.kvh < a.nkv || t.at >= end) return;
  t.kvh = 0;
  if (++t.part < t.parts) return;
  t.part = 0;
  ++t.tile;
  q4_set_tile(a, t);
}
// The first unit that starts at weight `from` or behind it, below `end`; none: one that starts at `end` or behind it.  Whole warp.
__device__ __forceinline__ Q4Unit q4_first(const TreeArgs& a, uint32_t from, uint32_t end, uint32_t tiles) {
  Q4Unit t;
  t.tile = tree_tile_of(a, from, tiles);
  q4_set_tile(a, t);
  const uint32_t before = uint32_t(a.tiles[t.tile].z), part = tree_q4_weight(TreeQ4::kPositions) * a.nkv;     // (of all parts but the last)
  t.part = (from - before) / part;
  t.kvh = 0;
  t.at = before + t.part * part;
  const uint32_t unit = q4_unit_weight(t), skip = (from - t.at + unit - 1) / unit;
  if (skip) {
    t.kvh = skip - 1;
    t.at += (skip - 1) * unit;
    q4_next(a, t, end);
  }
  return t;
}
// Chunks that a warp takes of the unit: positions 512 part + 128 i + 32 warp .. + 31 for i below this.
__device__ __forceinline__ uint32_t q4_chunks(const Q4Unit& t, uint32_t warp) {
  const int32_t n = min(t.extent - int32_t(t.part * TreeQ4::kPositions), int32_t(TreeQ4::kPositions)) - int32_t(warp * TreeQ4::kChunk);
  return uint32_t(max(n, 0) + 4 * TreeQ4::kChunk - 1) / (4 * TreeQ4::kChunk);
}

// What a lane keeps of a unit's columns: of block b, the queries of column 8 b + lane / 4 as B operands, the factors of its score columns
// 8 b + 2 (lane % 4) and the next; and the position below which all rows see everything.
template <int NB>
struct Q4Columns {
  uint4 q[NB][4];
  float2 scale[NB];
  int32_t plain;
};
constexpr float kQ4Nothing = -3.4028234e38f;       // the reference of a column that has seen nothing

struct Q4Warp {                    // a lane's places, the same for all units
  uint32_t warp, lane, r, c, place;      // place: of MMA row r (and, 8 further, of row r + 8) among a tile's 16 positions
  uint32_t per_group;                    // a number below 16 over the group, in units of 2^-16
  unsigned char* meaning;                // the warp's table of what exponents mean
  __device__ __forceinline__ uint32_t row_of(uint32_t column) const { return column * per_group >> 16; }
};

template <int NB>
__device__ __forceinline__ void q4_ask_columns(const TreeArgs& a, const Q4Unit& t, const Q4Warp& w, Q4Columns<NB>& k) {
  const uint32_t used = t.rows * a.group;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const uint32_t n = 8 * b + w.r, rl = w.row_of(n);
    const uint4* src = reinterpret_cast<const uint4*>(a.q + (size_t(t.first + rl) * a.nq + t.kvh * a.group + (n - rl * a.group)) * kKvDim + 32 * w.c);
#pragma unroll
    for (int i = 0; i < 4; ++i) k.q[b][i] = n < used ? src[i] : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t m = 8 * b + 2 * w.c, m0 = w.row_of(m), m1 = w.row_of(m + 1), head = t.kvh * a.group;
    k.scale[b] = make_float2(m < used ? a.q_scale[size_t(t.first + m0) * a.nq + head + (m - m0 * a.group)] : 0.f,
                             m + 1 < used ? a.q_scale[size_t(t.first + m1) * a.nq + head + (m + 1 - m1 * a.group)] : 0.f);
  }
  k.plain = t.extent;
  if (t.rows > 1 || a.row_base) {
    for (uint32_t i = 0; i < t.rows; ++i) {
      const int32_t e = a.extent[t.first + i];
      k.plain = min(k.plain, a.row_base ? min(a.row_base[t.first + i], e) : e);
    }
  }
}

// One warp's 32 positions from `at` on, against NB blocks of eight columns.
template <int NB>
__device__ __forceinline__ void q4_chunk(const TreeArgs& a, const Q4Unit& t, const Q4Warp& w, unsigned char* stage, int32_t at, bool first, const Q4Columns<NB>& k, float2 (&ref)[NB],
                                         float2 (&sum)[NB], float (&o)[NB][8][4]) {
  constexpr float kSlack = 8.f;
  using P = TreeQ4;
  {                                                          // each lane a position: 2^e of K; e and 2^-e of V
    const uint32_t kb = q4_ld<uint8_t>(stage + P::kKExpsAt + w.lane), vb = max(uint32_t(q4_ld<uint8_t>(stage + P::kVExpsAt + w.lane)), kKvLeastByte);
    const float add = vb == kKvNanByte ? __uint_as_float(0x7FC00000u) : __fsub_rn(__uint_as_float(0x4B000000u | vb), 8388735.f);      // 2^23 + 127
    *reinterpret_cast<uint4*>(w.meaning + 16 * w.lane) = make_uint4(kb << 23, __float_as_uint(add), __float_as_uint(kv_inverse(vb)), 0u);
    __syncwarp();
  }
  float s[2][NB][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {                              // 16 positions
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][b][e] = 0.f;
    const uint32_t p = 16 * i + w.place;
    const uint4 k0 = q4_ld<uint4>(stage + p * kQ4Codes + 16 * w.c), k1 = q4_ld<uint4>(stage + (p + 8) * kQ4Codes + 16 * w.c);
    // (a lane's 16 bytes are a group of 32 dimensions of one position: one scale)
    const Q4Factors f0 = q4_factors(q4_ld<uint8_t>(stage + P::kKScalesAt + 4 * p + w.c) * 0x10001u), f1 = q4_factors(q4_ld<uint8_t>(stage + P::kKScalesAt + 4 * (p + 8) + w.c) * 0x10001u);
    const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t x[4], y[4];
      q4_operands(w0[j], f0, x);
      q4_operands(w1[j], f1, y);
      const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        mma_q4(s[i][b], a0, k.q[b][j].x, k.q[b][j].y);
        mma_q4(s[i][b], a1, k.q[b][j].z, k.q[b][j].w);
      }
    }
  }
  // scores in units of log 2, with V's exponent; masked where some row does not see the whole chunk
  float inverse[2][2];                                       // 2^-e of V
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 e = q4_ld<uint4>(w.meaning + 16 * (16 * i + 8 * h + w.place));
      const float2 up = make_float2(__uint_as_float(e.x), __uint_as_float(e.x)), add = make_float2(__uint_as_float(e.y), __uint_as_float(e.y));
      inverse[i][h] = __uint_as_float(e.z);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const float2 x = fma2(mul2(make_float2(s[i][b][2 * h], s[i][b][2 * h + 1]), k.scale[b]), up, add);
        s[i][b][2 * h] = x.x;
        s[i][b][2 * h + 1] = x.y;
      }
    }
  if (at + int32_t(P::kChunk) > k.plain) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t m = 8 * b + 2 * w.c + j;
        if (m >= t.rows * a.group) continue;
        const uint32_t row = t.first + w.row_of(m);
        const int32_t base = a.row_base ? a.row_base[row] : 0, below = a.row_base ? min(base, a.extent[row]) : a.extent[row];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int32_t pos = at + int32_t(16 * i + 8 * h + w.place);
            if (pos >= below && !(a.row_base && tree_sees(a, row, pos - base))) s[i][b][2 * h + j] = -INFINITY;
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
      move = move || top[b][j] > __fadd_rn(j ? ref[b].y : ref[b].x, kSlack);
    }
  if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {                          // (the eight lanes of a column agree)
        float v = top[b][j];
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
        float& r = j ? ref[b].y : ref[b].x;
        float& l = j ? sum[b].y : sum[b].x;
        if (!(v > __fadd_rn(r, kSlack))) continue;
        const float f = exp2_approx(__fsub_rn(r, v));        // (from nothing: 0)
        r = v;
        if (first) continue;                                 // (nothing to scale)
        l = __fmul_rn(l, f);
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
    const float2 up = make_float2(kQ4Bias - ref[b].x, kQ4Bias - ref[b].y);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float2 e = add2(make_float2(s[i][b][2 * h], s[i][b][2 * h + 1]), up);
        e.x = exp2_approx(e.x);
        e.y = exp2_approx(e.y);
        sum[b] = fma2(e, make_float2(inverse[i][h], inverse[i][h]), sum[b]);
        const __half2 pair = __floats2half2_rn(e.x, e.y);
        weights[i][b][h] = movmatrix(*reinterpret_cast<const uint32_t*>(&pair));
      }
  }
  // MMA row r of these products is a dimension of 16 r .. 16 r + 15, whose 8 bytes the lane reads of the four positions of its columns c
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t p0 = 16 * i + w.c, p1 = 16 * i + 4 + (w.c ^ 1u);      // places of MMA rows 2 c and 2 c + 1; 8 further those of 2 c + 8 and 2 c + 9
    const unsigned char* const codes = stage + P::kVAt + 8 * w.r;
    const unsigned char* const scales = stage + P::kVScalesAt + (w.r >> 1);
    const uint2 x0 = q4_ld<uint2>(codes + p0 * kQ4Codes), x1 = q4_ld<uint2>(codes + p1 * kQ4Codes), x2 = q4_ld<uint2>(codes + (p0 + 8) * kQ4Codes), x3 = q4_ld<uint2>(codes + (p1 + 8) * kQ4Codes);
    const Q4Factors f01 = q4_factors(q4_ld<uint8_t>(scales + 4 * p0) | q4_ld<uint8_t>(scales + 4 * p1) << 16), f23 = q4_factors(q4_ld<uint8_t>(scales + 4 * (p0 + 8)) | q4_ld<uint8_t>(scales + 4 * (p1 + 8)) << 16);
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
          for (int b = 0; b < NB; ++b) mma_q4(o[b][4 * h + 2 * odd + q], x, weights[i][b][0], weights[i][b][1]);
        }
      }
    }
  }
}

// Float index of (column m of eight, 16-byte piece i of its 128 outputs) in a warp's block of the merge, spread over the banks.
__device__ __forceinline__ uint32_t q4_merge_index(uint32_t m, uint32_t piece) { return m * 128u + ((piece ^ (m >> 1)) << 2); }

// NB: blocks of eight columns.  Calls whose tiles have eight at most - decode rows - take one.
template <int NB>
__global__ void __launch_bounds__(TreeQ4::kThreads, NB == 1 ? 4 : 3)
tree_q4_kernel(const TreeArgs a) {
  step_kernel_entry();
  using P = TreeQ4;
  extern __shared__ __align__(128) unsigned char tree_smem[];
  __shared__ float ml_sm[4][8][2];
  const uint32_t tid = threadIdx.x;
  Q4Warp w;
  w.warp = tid >> 5;
  w.lane = tid & 31u;
  w.r = w.lane >> 2;
  w.c = w.lane & 3u;
  // Places are dealt so that neighbouring MMA rows lie in entries of different parity: 64-byte rows, two of which share all banks.
  w.place = w.r & 1u ? 4u + ((w.r >> 1) ^ 1u) : w.r >> 1;
  w.per_group = 65536u / a.group + 1u;
  const uint32_t tiles = a.plan[0], weights = a.plan[1];
  const uint32_t from = uint32_t(uint64_t(weights) * blockIdx.x / gridDim.x), end = uint32_t(uint64_t(weights) * (blockIdx.x + 1) / gridDim.x);
  if (from == end) return;
  Q4Unit t = q4_first(a, from, end, tiles);
  if (t.at >= end) return;
  const uint32_t ring = smem_u32(tree_smem) + w.warp * P::kWarp;
  unsigned char* const stages = tree_smem + w.warp * P::kWarp;
  w.meaning = stages + P::kStages * P::kStage;
  // a lane's places in a chunk's copies: 16-byte pieces of codes; the first 20 lanes take the scales (8 pieces of either) and the exponents (2)
  const bool of_scales = w.lane < 16, of_k = of_scales ? w.lane < 8 : w.lane < 18;
  const uint8_t* const k_codes = static_cast<const uint8_t*>(a.pages.k) + w.warp * P::kChunk * kQ4Codes + w.lane * 16;
  const uint8_t* const v_codes = static_cast<const uint8_t*>(a.pages.v) + w.warp * P::kChunk * kQ4Codes + w.lane * 16;
  const uint8_t* const others = static_cast<const uint8_t*>(of_k ? a.pages.k : a.pages.v) +
                                (of_scales ? kQ4ScalesAt + w.warp * P::kChunk * 4 + (w.lane & 7u) * 16 : kQ4ExpsAt + w.warp * P::kChunk + (w.lane & 1u) * 16);
  const uint32_t to_others = of_scales ? P::kKScalesAt + w.lane * 16 : P::kKExpsAt + (w.lane - 16) * 16, page_bytes = a.nkv * kQ4Page;
  const uint32_t half = of_scales ? 4 * P::kChunk * 4 : 4 * P::kChunk;       // to the second 128 positions of a page
  // Two chunks are on their way while a third is at hand; units with fewer chunks, and pages outside the pool, leave their stages empty.  Where the
  // next unit's pages lie is looked up at this unit's beginning, two chunks before it is needed.
  auto request = [&](uint32_t stage, int32_t page, uint32_t kvh, uint32_t i, uint32_t chunks) {
    if (i < chunks && uint32_t(page) < a.table.pages) {
      const uint64_t block = uint64_t(uint32_t(page)) * page_bytes + kvh * kQ4Page;
      const uint32_t dst = ring + stage + w.lane * 16, up = (i & 1u) * (4 * P::kChunk * kQ4Codes);
      const uint8_t* const k = k_codes + block + up;
      const uint8_t* const v = v_codes + block + up;
#pragma unroll
      for (int x = 0; x < 4; ++x) cp_async_16(dst + 512 * x, k + 512 * x, 16u);
#pragma unroll
      for (int x = 0; x < 4; ++x) cp_async_16(dst + P::kVAt + 512 * x, v + 512 * x, 16u);
      if (w.lane < 20) cp_async_16(ring + stage + to_others, others + block + (i & 1u) * half, 16u);
    }
    cp_async_commit();
  };
  auto page_of = [&](const Q4Unit& u, uint32_t i) {
    const uint32_t p = u.part * 2 + i;
    return u.at < end && uint32_t(u.seq) < a.table.slots && p < a.table.max_pages ? a.table.table[u.seq * a.table.ld + p] : -1;
  };
  auto after = [&](uint32_t stage) { return stage == (P::kStages - 1) * P::kStage ? 0u : stage + P::kStage; };
  int32_t page0 = page_of(t, 0), page1 = page_of(t, 1);
  uint32_t stage = 0, chunks = q4_chunks(t, w.warp);
  request(0, page0, t.kvh, 0, chunks);
  request(P::kStage, page0, t.kvh, 1, chunks);
  Q4Columns<NB> columns;
  q4_ask_columns<NB>(a, t, w, columns);
  while (t.at < end) {
    float2 ref[NB], sum[NB];
    float o[NB][8][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      ref[b] = make_float2(kQ4Nothing, kQ4Nothing);
      sum[b] = make_float2(0.f, 0.f);
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[b][d][e] = 0.f;
    }
    Q4Unit next = t;
    q4_next(a, next, end);
    const int32_t next0 = page_of(next, 0), next1 = page_of(next, 1);
    const uint32_t next_chunks = next.at < end ? q4_chunks(next, w.warp) : 0u;
    int32_t at = int32_t(t.part * P::kPositions + w.warp * P::kChunk);
    bool first = true;
#pragma unroll 1
    for (uint32_t i = 0; i < P::kChunks; ++i, at += 4 * P::kChunk) {
      // (into the stage that the chunk before has left)
      const bool same = i < 2;
      request(after(after(stage)), same ? page1 : next0, same ? t.kvh : next.kvh, i ^ 2u, same ? chunks : next_chunks);
      cp_async_wait<P::kStages - 1>();
      __syncwarp();
      // (a page outside the pool: as if nobody saw the chunk)
      if (i < chunks && uint32_t(same ? page0 : page1) < a.table.pages) {
        q4_chunk<NB>(a, t, w, stages + stage, at, first, columns, ref, sum, o);
        first = false;
      }
      stage = after(stage);
      __syncwarp();
    }
    // the next unit's columns are on their way while the warps' results are merged, eight columns at a time, in the stage that was left last
    const uint32_t used = t.rows * a.group, first_row = t.first, heads = t.kvh * a.group, part = t.part, merge_at = after(after(stage));
    t = next;
    page0 = next0;
    page1 = next1;
    chunks = next_chunks;
    if (t.at < end) q4_ask_columns<NB>(a, t, w, columns);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b && 8u * b >= used) break;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float l = j ? sum[b].y : sum[b].x;
        const float r = j ? ref[b].y : ref[b].x;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l = __fadd_rn(l, __shfl_xor_sync(0xFFFFFFFFu, l, off));
        if (w.r == 0) *reinterpret_cast<float2*>(ml_sm[w.warp][2 * w.c + j]) = make_float2(r == kQ4Nothing ? -INFINITY : r - kQ4Bias, l);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {                        // dimensions 16 r + 4 q ..: of word q / 2, 4 (q % 2) on
          const int d = 4 * (q >> 1) + (q & 1);
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(tree_smem + w.warp * P::kWarp + merge_at) + q4_merge_index(2 * w.c + j, 4 * w.r + q)) =
              make_float4(o[b][d][j], o[b][d + 2][j], o[b][d][2 + j], o[b][d + 2][2 + j]);
        }
      __syncthreads();
      for (uint32_t m = w.warp; m < 8 && 8 * b + m < used; m += 4) {
        float2 ml[4];
        float mx = -INFINITY, den = 0.f;
        float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < 4; ++x) { ml[x] = *reinterpret_cast<const float2*>(ml_sm[x][m]); mx = fmaxf(mx, ml[x].x); }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // (a warp that saw nothing adds zeros; one whose scores were all NaN has no reference either and adds NaN)
          const float e = ml[x].x == -INFINITY ? 1.f : exp2_approx(__fsub_rn(ml[x].x, mx));
          den = __fmaf_rn(e, ml[x].y, den);
          const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(tree_smem + x * P::kWarp + merge_at) + q4_merge_index(m, w.lane));
          num.x = __fmaf_rn(e, v.x, num.x);
          num.y = __fmaf_rn(e, v.y, num.y);
          num.z = __fmaf_rn(e, v.z, num.z);
          num.w = __fmaf_rn(e, v.w, num.w);
        }
        const uint32_t col = 8 * b + m, rl = w.row_of(col);
        const size_t to = (size_t(first_row + rl) * a.nq + heads + (col - rl * a.group)) * a.max_parts + part;
        *reinterpret_cast<float4*>(a.part_acc + to * kKvDim + w.lane * 4) = num;
        if (w.lane == 0) a.part_ml[to] = make_float2(mx, den);
      }
      __syncthreads();                                       // the stages are free again
    }
  }
  cp_async_wait<0>();
}

}  // namespace grb
