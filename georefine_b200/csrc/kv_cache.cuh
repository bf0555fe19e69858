// A paged KV cache in BF16, in 8 or in 4 bits: storing rows, reading them back, and moving what a draft tree keeps.
//
// A page holds 256 positions of one sequence as [kv head][position][128]; an entry is the 128 values of one key or value head
// at one position.  In 8 bits an entry is 128 e4m3 codes and one exponent byte (pages of exponents: [kv head][position]):
// with a = max |x|, e = clamp(ceil(log2(a / 448)), -40, 7), code = e4m3 nearest to x 2^-e (ties to even, at most 448), byte =
// e + 127, value = code 2^e.  A power of two scales without rounding, so an entry is off by the e4m3 rounding alone - half a
// step, 2^-4 of the value - whatever its size, and the same input gives the same codes everywhere.  The scale goes with the
// entry because a cache is appended to one entry at a time: nothing stored before is touched again.  An entry with an
// infinity or a NaN is stored as byte 255 with codes 0 and reads as NaN throughout.
//
// In 4 bits an entry is 128 whole numbers in -7 .. 7, a scale byte for each 32 of them and an exponent byte: 69 bytes.  With a = max |x|
// of the entry, e = clamp(floor(log2(a / 7)) + 9, -40, 22), kept as e + 127; a group's scale F is the number nearest to (its max |x|) / 7 2^(24 - e)
// among (16 + m) 2^k, m 0 .. 15, k 0 .. 11, kept as the byte 64 + 16 k + m; code = x / (F 2^(e - 24)) to the nearest (ties to even) in -7 .. 7;
// value = code F 2^(e - 24).  Uniform steps, because the largest of 32 values is about two standard deviations: a normal entry is held to
// 20.2 dB (e2m1 codes under the same scales: 19.9).  A value is off by g / 14 (1 + 1/32) at most, g the largest magnitude of its group, or by a / 28672, half of
// the smallest scale, where that is more, or by 2^-61 under the smallest exponent; beyond 111104, the largest value, it is held as that.
// A nibble holds code + 8: nibbles masked out of a word are FP16 subnormals, so that one
// fused multiply-add makes two FP16 operands of them - u 2^-24 F - 8 F 2^-24, exact, as F is a whole number of at most 16 bits, five of them
// significant, which is also why the scales stay in twelve binades.  The exponent keeps the operands of an entry near the top of that range
// whatever its size, as in 8 bits.  A scale byte below 16 reads as byte / 8, so that memory of zeros reads as zeros.
// A page of one head is 17664 bytes in a piece: the codes of its 256 positions, 64 bytes each, then their scales, 4 bytes each, then their
// exponents.  The codes of dimensions 8 w .. 8 w + 7 are 32-bit word w: nibble j of the lower half is dimension 2 j of the eight, of the upper
// half 2 j + 1 - the two that share an operand register.
//
// The kernels here move bytes, and memory bounds them; nothing is kept between calls.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr uint32_t kKvDim = 128, kKvPage = 256;
constexpr uint32_t kKvNanByte = 255, kKvLeastByte = 127 - 40, kQ4MostByte = 127 + 22;

enum : int { kKvBf16 = 0, kKvE4m3 = 1, kKvQ4 = 4 };      // formats, numbered as in the C interface
constexpr uint32_t kQ4Codes = kKvDim / 2;                // bytes of an entry's codes
constexpr uint32_t kQ4ScalesAt = kKvPage * kQ4Codes, kQ4ExpsAt = kQ4ScalesAt + kKvPage * 4, kQ4Page = kQ4ExpsAt + kKvPage;    // of one head's page

struct KvPagesArgs {
  void* k;                  // [layers][pages][nkv][256][128] BF16 or e4m3, [layers][pages][nkv][17664] in 4 bits; layers `layer_stride` elements apart
  void* v;
  uint8_t* k_exp;           // [layers][pages][nkv][256], layers `exp_stride` bytes apart (8-bit caches)
  uint8_t* v_exp;
  int64_t layer_stride, exp_stride;
  uint32_t layers, pages, nkv;
};

// Where position `pos` of the sequence in slot `seq` lies: its page times 256 plus the place in it; -1 where a caller's row
// is marked as absent (slot -1) or names something outside the table or the pool.
struct KvTable {
  const int32_t* table;     // [slots][ld]
  int64_t ld;
  uint32_t slots, max_pages, pages;
};
__device__ __forceinline__ int64_t kv_place(const KvTable& t, int32_t seq, int32_t pos) {
  if (uint32_t(seq) >= t.slots || pos < 0 || uint32_t(pos) / kKvPage >= t.max_pages) return -1;
  const int32_t page = t.table[seq * t.ld + uint32_t(pos) / kKvPage];
  return uint32_t(page) < t.pages ? int64_t(page) * kKvPage + uint32_t(pos) % kKvPage : -1;
}
// Index of an entry (in entries of its layer) from its place.
__device__ __forceinline__ size_t kv_entry(int64_t place, uint32_t nkv, uint32_t head) {
  return (size_t(place / kKvPage) * nkv + head) * kKvPage + size_t(place % kKvPage);
}

// Exponent byte of an entry whose largest magnitude is `amax`; `finite`: no component is an infinity or a NaN.
// amax = 1.f 2^(E - 127), and 448 = 1.75 2^8: ceil(log2(amax / 448)) = E - 135 + (1.f > 1.75).
__device__ __forceinline__ uint32_t kv_exp_byte(float amax, bool finite) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = int(bits >> 23) - 135 + ((bits & 0x7FFFFFu) > 0x600000u);
  return finite ? uint32_t(min(max(e, -40), 7) + 127) : kKvNanByte;
}
// 2^-e for the byte's e (0 for the NaN byte), and 2^e (infinity for the NaN byte: with codes 0 the product is NaN).
__device__ __forceinline__ float kv_inverse(uint32_t byte) { return __uint_as_float((254u - min(byte, 254u)) << 23); }
__device__ __forceinline__ float kv_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(pair)));
  return r;
}
// Four codes as two pairs.
__device__ __forceinline__ void e4m3_to_half4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, off));
  return v;
}
// Exponent byte of the entry of which this lane holds four values.  Whole warp.
__device__ __forceinline__ uint32_t kv_warp_byte(const float (&x)[4]) {
  const float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  bool fine = true;
#pragma unroll
  for (int i = 0; i < 4; ++i) fine = fine && fabsf(x[i]) <= 3.4028234e38f;
  return kv_exp_byte(warp_max(m), __all_sync(0xFFFFFFFFu, fine));
}
// Two neighbouring values as codes.
__device__ __forceinline__ uint32_t kv_codes(float lo, float hi, uint32_t byte) {
  if (byte == kKvNanByte) return 0u;
  const float s = kv_inverse(byte);
  return e4m3_pair(__fmul_rn(lo, s), __fmul_rn(hi, s));
}


// ---- 4 bits ---------------------------------------------------------------------------------------------------------
// Exponent byte of an entry whose largest magnitude is `amax` = 1.f 2^(E - 127): 7 = 1.75 2^2, so floor(log2(amax / 7)) = E - 127 - 3 + (1.f >= 1.75).
__device__ __forceinline__ uint32_t q4_exp_byte(float amax, bool finite) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = int(bits >> 23) - 127 - 3 + ((bits & 0x7FFFFFu) >= 0x600000u) + 9;
  return finite ? uint32_t(min(max(e, -40), 22) + 127) : kKvNanByte;
}
// Scale byte of a group whose largest magnitude is `amax`, and the scale times the entry's unit, 2^(e - 24).  (A quotient by 7 that lies on no border
// between two scales does not round to one: values next to seven times a border are farther apart than seven halves of a step of the quotient.)
// EIGHT: amax has eight significant bits.  Then the quotient lies on a border, or 2^-9 of it or more from all of them, and the product with
// the rounded seventh, taken to 12 bits first, lands where the quotient does (all 128 fractions agree).
template <bool EIGHT>
__device__ __forceinline__ uint32_t q4_scale_byte(float amax, uint32_t exp_byte, float& step) {
  const float to_unit = __uint_as_float((127u + 24u + 127u - exp_byte) << 23);
  const float want = fminf(fmaxf(__fmul_rn(EIGHT ? __fmul_rn(amax, 0.14285715f) : __fdiv_rn(amax, 7.f), to_unit), 16.f), 63488.f);
  uint32_t bits = __float_as_uint(want);
  if constexpr (EIGHT) bits = (bits + 0x400u) & ~0x7FFu;
  const uint32_t five = (bits + 0x3FFFFu + (bits >> 19 & 1u)) >> 19;     // five bits, ties to even
  step = __fmul_rn(__uint_as_float(five << 19), __uint_as_float((exp_byte - 24u) << 23));
  return five - 127u * 16u;
}
// code + 8 of a value whose quotient by the step is q.
__device__ __forceinline__ uint32_t q4_nibble(float q) { return uint32_t(__float2int_rn(fminf(fmaxf(q, -7.f), 7.f)) + 8); }
// What a scale byte stands for.
__device__ __forceinline__ float q4_scale(uint32_t byte) {
  return byte < 16u ? __fmul_rn(float(byte), 0.125f) : __uint_as_float((byte + 127u * 16u) << 19);
}
// 2^(e - 24) of an exponent byte; bytes below what an entry has (0, where nobody wrote) stand for the smallest.
__device__ __forceinline__ float q4_unit(uint32_t byte) {
  return byte == kKvNanByte ? __uint_as_float(0x7FC00000u) : __uint_as_float((max(byte, kKvLeastByte) - 24u) << 23);
}
// Bytes from the pool's start to the page of one head that entry `entry` is in.
__device__ __forceinline__ size_t q4_page_at(size_t entry) { return entry / kKvPage * kQ4Page; }

constexpr int kKvWarps = 8;

struct KvRowsArgs {
  KvPagesArgs pages;
  KvTable table;
  const int32_t* row_seq;
  const int32_t* row_pos;
  __nv_bfloat16* k;         // [rows][ld][128]: heads of a row side by side
  __nv_bfloat16* v;
  int64_t ldk, ldv;
  uint32_t rows;
};

// Rows into the cache (READ false) or out of it (READ true).  A warp takes eight neighbouring entries of a row (keys, then
// values), two at a time with 16 bytes of BF16 a lane; all its loads are on their way before the first is used, which is what
// keeps enough bytes in flight.  32768 rows of 8 heads, 8 bits: 45 us in, 36 out, 4.5 and 5.6 TB/s (one entry a warp, 8 bytes a
// lane: 106 and 100).  On the way in, 118 instructions for two entries take two thirds of the issue slots; warps are numbered and
// divided in 32 bits for their sake.
constexpr uint32_t kKvEntriesPerWarp = 8;

template <bool READ, int FORMAT>
__global__ void __launch_bounds__(kKvWarps * 32)
kv_rows_kernel(const KvRowsArgs a) {
  step_kernel_entry();
  constexpr int N = kKvEntriesPerWarp / 2;
  const uint32_t lane = threadIdx.x & 31u, half = lane >> 4, l = lane & 15u, heads = 2 * a.pages.nkv;
  const uint32_t per_row = (heads + kKvEntriesPerWarp - 1) / kKvEntriesPerWarp;
  const uint32_t at = blockIdx.x * kKvWarps + (threadIdx.x >> 5), row = at / per_row, head0 = (at - row * per_row) * kKvEntriesPerWarp + half;
  if (row >= a.rows) return;
  const int64_t place = kv_place(a.table, a.row_seq[row], a.row_pos[row]);
  if (place < 0) return;
  const size_t first_entry = kv_entry(place, a.pages.nkv, 0);
  uint4* const keys = reinterpret_cast<uint4*>(a.k + row * a.ldk) + l;
  uint4* const values = reinterpret_cast<uint4*>(a.v + row * a.ldv) + l;
  size_t entry[N];
  bool value[N], in[N];
  uint4* rows[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t head = head0 + 2 * i;
    in[i] = head < heads;
    value[i] = head >= a.pages.nkv;
    const uint32_t h = in[i] ? value[i] ? head - a.pages.nkv : head : 0u;
    entry[i] = first_entry + h * kKvPage;
    rows[i] = (value[i] ? values : keys) + h * (kKvDim / 8);
  }
  if constexpr (FORMAT == kKvBf16) {
    uint4 x[N];
    auto held = [&](int i) { return reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(value[i] ? a.pages.v : a.pages.k) + entry[i] * kKvDim) + l; };
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) x[i] = READ ? *held(i) : *rows[i];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) *(READ ? rows[i] : held(i)) = x[i];
  } else {
    auto held = [&](int i) { return reinterpret_cast<uint2*>(static_cast<uint8_t*>(value[i] ? a.pages.v : a.pages.k) + entry[i] * kKvDim) + l; };
    auto exps = [&](int i) { return (value[i] ? a.pages.v_exp : a.pages.k_exp) + entry[i]; };
    if constexpr (READ) {
      uint2 code[N];
      uint32_t byte[N];
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (in[i]) { code[i] = *held(i); byte[i] = *exps(i); }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!in[i]) continue;
        const float s = kv_scale(byte[i]);
        auto two = [&](uint32_t pair) {               // (exact: four bits times a power of two)
          const uint32_t h = e4m3_to_half2(pair);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          return pack_bf(__fmul_rn(f.x, s), __fmul_rn(f.y, s));
        };
        *rows[i] = make_uint4(two(code[i].x & 0xFFFFu), two(code[i].x >> 16), two(code[i].y & 0xFFFFu), two(code[i].y >> 16));
      }
    } else {
      uint4 x[N];
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = in[i] ? *rows[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        // magnitudes of BF16 values compare as integers; an infinity or a NaN is above all others
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
        m = max(m & 0xFFFFu, m >> 16);
#pragma unroll
        for (int off = 8; off; off >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
        const uint32_t byte = kv_exp_byte(__uint_as_float(m << 16), m < 0x7F80u);
        const float s = kv_inverse(byte);
        uint32_t c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = e4m3_pair(__fmul_rn(bf_lo(w[j]), s), __fmul_rn(bf_hi(w[j]), s));
        if (in[i]) {
          *held(i) = byte == kKvNanByte ? make_uint2(0u, 0u) : make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
          if (l == 0) *exps(i) = uint8_t(byte);
        }
      }
    }
  }
}

// The same in 4 bits.  Eight lanes share an entry, sixteen neighbouring values each, two lanes a scale; a warp takes sixteen entries of a row, four at a time.
// What is found once for a lane's values - the two maxima, the scale, its reciprocal - costs as much as eight of them do.  32768 rows of 8 heads: 37 us in, 37
// out (sixteen lanes an entry, eight entries a warp: 57 and 40); out, the stores alone - 134 MB - take 35 at the 3.8 TB/s that a fill reaches here.
constexpr uint32_t kQ4EntriesPerWarp = 16;
template <bool READ>
__global__ void __launch_bounds__(kKvWarps * 32)
kv_rows_q4_kernel(const KvRowsArgs a) {
  step_kernel_entry();
  constexpr int N = kQ4EntriesPerWarp / 4;
  const uint32_t lane = threadIdx.x & 31u, l = lane & 7u, heads = 2 * a.pages.nkv, per_row = (heads + kQ4EntriesPerWarp - 1) / kQ4EntriesPerWarp;
  const uint32_t id = blockIdx.x * kKvWarps + (threadIdx.x >> 5), row = id / per_row, head0 = (id - row * per_row) * kQ4EntriesPerWarp + (lane >> 3);
  if (row >= a.rows) return;
  const int64_t place = kv_place(a.table, a.row_seq[row], a.row_pos[row]);
  if (place < 0) return;
  const uint32_t at = uint32_t(place % kKvPage);
  const size_t first = size_t(place / kKvPage) * a.pages.nkv * kQ4Page;       // of the page's first head
  uint4* const keys = reinterpret_cast<uint4*>(a.k + row * a.ldk);
  uint4* const values = reinterpret_cast<uint4*>(a.v + row * a.ldv);
  uint8_t* page[N];
  uint4* rows[N];
  bool in[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t head = head0 + 4 * i;
    in[i] = head < heads;
    const bool value = head >= a.pages.nkv;
    const uint32_t h = in[i] ? value ? head - a.pages.nkv : head : 0u;
    page[i] = static_cast<uint8_t*>(value ? a.pages.v : a.pages.k) + first + size_t(h) * kQ4Page;
    rows[i] = (value ? values : keys) + h * (kKvDim / 8);
  }
  if constexpr (READ) {     // (a lane's words are 8 apart, so that eight lanes store 128 bytes in a row)
    uint32_t code[N][2], scale[N][2], exp[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (in[i]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          code[i][j] = reinterpret_cast<const uint32_t*>(page[i] + at * kQ4Codes)[l + 8 * j];
          scale[i][j] = page[i][kQ4ScalesAt + at * 4 + (l >> 2) + 2 * j];
        }
        exp[i] = page[i][kQ4ExpsAt + at];
      }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float step = __fmul_rn(q4_scale(scale[i][j]), q4_unit(exp[i]));   // (exact, as is its product with a code: eight bits)
        // code + 8 in the lowest bits of 2^23; the sum with -(2^23 + 8) is the code
        auto one = [&](uint32_t nibble) { return __fmul_rn(__fadd_rn(__uint_as_float(0x4B000000u | (code[i][j] >> (4 * nibble) & 15u)), -8388616.f), step); };
        rows[i][int(l) + 8 * j] = make_uint4(pack_bf(one(0), one(4)), pack_bf(one(1), one(5)), pack_bf(one(2), one(6)), pack_bf(one(3), one(7)));
      }
    }
  } else {
    uint4 x[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) x[i][j] = in[i] ? rows[i][2 * l + j] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t w[8] = {x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w, x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w};
      uint32_t m = 0;                                 // (magnitudes of BF16 values compare as integers)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = __vmaxu2(m, w[j] & 0x7FFF7FFFu);
      m = max(m & 0xFFFFu, m >> 16);
      m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
      const float group = __uint_as_float(m << 16);
      m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
      m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
      const bool finite = m < 0x7F80u;
      const uint32_t exp = q4_exp_byte(__uint_as_float(m << 16), finite);
      float step;
      uint32_t scale = q4_scale_byte<true>(finite ? group : 0.f, finite ? exp : 127u, step);
      if (exp == kQ4MostByte) {                       // (the only entries with values beyond 7 steps and a half; 7 steps are a BF16 number)
        const __nv_bfloat162 most = __float2bfloat162_rn(__fmul_rn(step, 7.f)), least = __hneg2(most);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const __nv_bfloat162 v = __hmax2(__hmin2(*reinterpret_cast<__nv_bfloat162*>(&w[j]), most), least);
          w[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
      // The quotient of a value of eight bits and a step of five lies on a border between two codes, or 2^-11 or more from all of them.  A product with the
      // reciprocal, 2^-19 of it off at most, rounded to 2^-13 - by adding 1536 - lands on the right side; added to 2^23 1.5 + 8, it is the code.
      float inverse;
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(step));
      uint32_t code[2] = {0, 0};
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        auto nibble = [&](float v) { return __float_as_uint(__fadd_rn(__fmaf_rn(v, inverse, 1536.f), 12582920.f - 1536.f)); };     // code + 8 in the lowest byte, 0 in the next
        code[j >> 2] = code[j >> 2] * 16 + __byte_perm(nibble(bf_lo(w[j])), nibble(bf_hi(w[j])), 0x5410);
      }
      if (!finite) { code[0] = code[1] = 0x88888888u; scale = 64u; }
      if (in[i]) {
        reinterpret_cast<uint2*>(page[i] + at * kQ4Codes)[l] = make_uint2(code[0], code[1]);
        if ((l & 1u) == 0) page[i][kQ4ScalesAt + at * 4 + (l >> 1)] = uint8_t(scale);
        if (l == 0) page[i][kQ4ExpsAt + at] = uint8_t(exp);
      }
    }
  }
}

// What a draft tree keeps: entry base + path[i] of a sequence goes to base + i, for i = 1 .. count - 1, in every layer, keys
// and values.  Paths ascend, so an entry never lands on one that is still to be read (base + i <= base + path[i] <
// base + path[i + 1]) as long as each batch is read before it is written.  Grid (layers * 2 / 4, sequences): where an entry
// lies is looked up once for four planes, whose pieces are then in flight together (64 paths of 64 layers, 8 bits: 19 us; a plane a CTA: 29).
constexpr int kKeepThreads = 256;
constexpr int kKeepPlanes = 4;      // planes (a layer's keys or values) of a CTA, one 16-byte piece of each a thread at a time

struct KvKeepArgs {
  KvPagesArgs pages;
  KvTable table;
  const int32_t* seqs;      // [n]: slots
  const int32_t* base;      // [n]
  const int32_t* path;      // [n][ldp]
  const int32_t* count;     // [n]
  int64_t ldp;
  uint32_t width;
};

template <int FORMAT>
__global__ void __launch_bounds__(kKeepThreads)
kv_keep_kernel(const KvKeepArgs a) {
  step_kernel_entry();
  const uint32_t s = blockIdx.y, tid = threadIdx.x, plane0 = blockIdx.x * kKeepPlanes, planes = min(uint32_t(kKeepPlanes), 2 * a.pages.layers - plane0);
  const int32_t count = min(a.count[s], int32_t(a.width)), seq = a.seqs[s], base = a.base[s];
  constexpr bool F8 = FORMAT == kKvE4m3, Q4 = FORMAT == kKvQ4;
  constexpr uint32_t kPieces = (Q4 ? kQ4Codes : (F8 ? 1 : 2) * kKvDim) / 16;       // of an entry
  const uint32_t per_node = a.pages.nkv * kPieces, nodes = max(1u, kKeepThreads / per_node);
  // plane p: keys (even) or values of layer p / 2
  auto pieces = [&](uint32_t p) {
    return reinterpret_cast<uint4*>(static_cast<uint8_t*>(p & 1u ? a.pages.v : a.pages.k) + int64_t(p >> 1) * a.pages.layer_stride * (FORMAT == kKvBf16 ? 2 : 1));
  };
  // index of an entry's first piece (4 bits: in its plane, whose pages hold scales and exponents behind the codes)
  auto first_piece = [&](size_t entry) { return Q4 ? (q4_page_at(entry) + entry % kKvPage * kQ4Codes) / 16 : entry * kPieces; };
  auto scales = [&](uint32_t p, size_t entry) { return reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(pieces(p)) + q4_page_at(entry) + kQ4ScalesAt) + entry % kKvPage; };
  auto q4_exps = [&](uint32_t p, size_t entry) { return reinterpret_cast<uint8_t*>(pieces(p)) + q4_page_at(entry) + kQ4ExpsAt + entry % kKvPage; };
  auto exps = [&](uint32_t p) { return (p & 1u ? a.pages.v_exp : a.pages.k_exp) + int64_t(p >> 1) * a.pages.exp_stride; };
  for (int32_t first = 1; first < count; first += nodes) {
    const uint32_t items = min(nodes, uint32_t(count - first)) * per_node;
    for (uint32_t round = 0; round < items; round += kKeepThreads) {   // (one round, but for more heads than a batch has threads for)
      const uint32_t item = round + tid, i = first + item / per_node, head = item % per_node / kPieces, piece = item % kPieces;
      size_t src = 0, dst = 0;
      bool on = item < items;
      if (on) {
        const int32_t node = a.path[s * a.ldp + i];
        on = node >= 0 && base >= 0 && node <= 0x7FFFFFFF - base;
        const int64_t from = on ? kv_place(a.table, seq, base + node) : -1, to = on ? kv_place(a.table, seq, base + int32_t(i)) : -1;
        on = from >= 0 && to >= 0 && from != to;
        if (on) {
          src = kv_entry(from, a.pages.nkv, head);
          dst = kv_entry(to, a.pages.nkv, head);
        }
      }
      uint4 x[kKeepPlanes];
      uint8_t byte[kKeepPlanes];
      uint32_t scale[Q4 ? kKeepPlanes : 1];
      if (on) {
#pragma unroll
        for (int p = 0; p < kKeepPlanes; ++p)
          if (uint32_t(p) < planes) {
            x[p] = pieces(plane0 + p)[first_piece(src) + piece];
            if (F8 && piece == 0) byte[p] = exps(plane0 + p)[src];
            if constexpr (Q4) {
              if (piece == 0) { scale[p] = *scales(plane0 + p, src); byte[p] = *q4_exps(plane0 + p, src); }
            }
          }
      }
      __syncthreads();
      if (on) {
#pragma unroll
        for (int p = 0; p < kKeepPlanes; ++p)
          if (uint32_t(p) < planes) {
            pieces(plane0 + p)[first_piece(dst) + piece] = x[p];
            if (F8 && piece == 0) exps(plane0 + p)[dst] = byte[p];
            if constexpr (Q4) {
              if (piece == 0) { *scales(plane0 + p, dst) = scale[p]; *q4_exps(plane0 + p, dst) = byte[p]; }
            }
          }
      }
      __syncthreads();
    }
  }
}

}  // namespace grb
