// A paged KV cache in BF16 or in 8 bits: storing rows, reading them back, and moving what a draft tree keeps.
//
// A page holds 256 positions of one sequence as [kv head][position][128]; an entry is the 128 values of one key or value head
// at one position.  In 8 bits an entry is 128 e4m3 codes and one exponent byte (pages of exponents: [kv head][position]):
// with a = max |x|, e = clamp(ceil(log2(a / 448)), -40, 7), code = e4m3 nearest to x 2^-e (ties to even, at most 448), byte =
// e + 127, value = code 2^e.  A power of two scales without rounding, so an entry is off by the e4m3 rounding alone - half a
// step, 2^-4 of the value - whatever its size, and the same input gives the same codes everywhere.  The scale goes with the
// entry because a cache is appended to one entry at a time: nothing stored before is touched again.  An entry with an
// infinity or a NaN is stored as byte 255 with codes 0 and reads as NaN throughout.
//
// The kernels here move bytes, and memory bounds them; nothing is kept between calls.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr uint32_t kKvDim = 128, kKvPage = 256;
constexpr uint32_t kKvNanByte = 255, kKvLeastByte = 127 - 40;

struct KvPagesArgs {
  void* k;                  // [layers][pages][nkv][256][128] BF16 or e4m3; layers `layer_stride` elements apart
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

template <bool READ, bool F8>
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
  if constexpr (!F8) {
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

template <bool F8>
__global__ void __launch_bounds__(kKeepThreads)
kv_keep_kernel(const KvKeepArgs a) {
  step_kernel_entry();
  const uint32_t s = blockIdx.y, tid = threadIdx.x, plane0 = blockIdx.x * kKeepPlanes, planes = min(uint32_t(kKeepPlanes), 2 * a.pages.layers - plane0);
  const int32_t count = min(a.count[s], int32_t(a.width)), seq = a.seqs[s], base = a.base[s];
  constexpr uint32_t kPieces = (F8 ? 1 : 2) * kKvDim / 16;       // of an entry
  const uint32_t per_node = a.pages.nkv * kPieces, nodes = max(1u, kKeepThreads / per_node);
  // plane p: keys (even) or values of layer p / 2
  auto pieces = [&](uint32_t p) {
    return reinterpret_cast<uint4*>(static_cast<uint8_t*>(p & 1u ? a.pages.v : a.pages.k) + int64_t(p >> 1) * a.pages.layer_stride * (F8 ? 1 : 2));
  };
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
      if (on) {
#pragma unroll
        for (int p = 0; p < kKeepPlanes; ++p)
          if (uint32_t(p) < planes) {
            x[p] = pieces(plane0 + p)[src * kPieces + piece];
            if (F8 && piece == 0) byte[p] = exps(plane0 + p)[src];
          }
      }
      __syncthreads();
      if (on) {
#pragma unroll
        for (int p = 0; p < kKeepPlanes; ++p)
          if (uint32_t(p) < planes) {
            pieces(plane0 + p)[dst * kPieces + piece] = x[p];
            if (F8 && piece == 0) exps(plane0 + p)[dst] = byte[p];
          }
      }
      __syncthreads();
    }
  }
}

}  // namespace grb
