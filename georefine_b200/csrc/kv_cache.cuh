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
// The kernels here move bytes: a warp per entry, 8 bytes of BF16 a lane, and nothing kept between calls.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr uint32_t kKvDim = 128, kKvPage = 256;
constexpr uint32_t kKvNanByte = 255;

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

// Rows into the cache (READ false) or out of it (READ true).  A warp per (row, key or value head).
template <bool READ, bool F8>
__global__ void __launch_bounds__(kKvWarps * 32)
kv_rows_kernel(const KvRowsArgs a) {
  step_kernel_entry();
  const uint32_t lane = threadIdx.x & 31u, heads = 2 * a.pages.nkv;
  const uint64_t at = uint64_t(blockIdx.x) * kKvWarps + (threadIdx.x >> 5);
  const uint32_t row = uint32_t(at / heads), head = uint32_t(at % heads);
  if (row >= a.rows) return;
  const int64_t place = kv_place(a.table, a.row_seq[row], a.row_pos[row]);
  if (place < 0) return;
  const bool value = head >= a.pages.nkv;
  const uint32_t h = value ? head - a.pages.nkv : head;
  const size_t entry = kv_entry(place, a.pages.nkv, h);
  uint2* rows = reinterpret_cast<uint2*>((value ? a.v + row * a.ldv : a.k + row * a.ldk) + h * kKvDim) + lane;
  void* const pages = value ? a.pages.v : a.pages.k;
  if constexpr (!F8) {
    uint2* held = reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(pages) + entry * kKvDim) + lane;
    if (READ) *rows = *held;
    else *held = *rows;
  } else {
    uint32_t* held = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(pages) + entry * kKvDim) + lane;
    uint8_t* exps = value ? a.pages.v_exp : a.pages.k_exp;
    if (READ) {
      const uint32_t code = *held, byte = exps[entry];
      const float s = kv_scale(byte);
      const uint32_t lo = e4m3_to_half2(code & 0xFFFFu), hi = e4m3_to_half2(code >> 16);
      const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&lo)), a1 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      *rows = make_uint2(pack_bf(__fmul_rn(a0.x, s), __fmul_rn(a0.y, s)), pack_bf(__fmul_rn(a1.x, s), __fmul_rn(a1.y, s)));   // (exact: 4 bits)
    } else {
      const uint2 r = *rows;
      const float x[4] = {bf_lo(r.x), bf_hi(r.x), bf_lo(r.y), bf_hi(r.y)};
      const uint32_t byte = kv_warp_byte(x);
      *held = kv_codes(x[0], x[1], byte) | (kv_codes(x[2], x[3], byte) << 16);
      if (lane == 0) exps[entry] = uint8_t(byte);
    }
  }
}

// What a draft tree keeps: entry base + path[i] of a sequence goes to base + i, for i = 1 .. count - 1, in every layer, keys
// and values.  Paths ascend, so an entry never lands on one that is still to be read (base + i <= base + path[i] <
// base + path[i + 1]) as long as each batch is read before it is written.  Grid (layers * 2, sequences).
constexpr int kKeepThreads = 256;
constexpr int kKeepChunks = 4;      // 16-byte pieces a thread holds between a batch's reads and its writes

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
  const uint32_t s = blockIdx.y, layer = blockIdx.x >> 1, tid = threadIdx.x;
  const bool value = blockIdx.x & 1u;
  const int32_t count = min(a.count[s], int32_t(a.width)), seq = a.seqs[s], base = a.base[s];
  constexpr uint32_t kPieces = (F8 ? 1 : 2) * kKvDim / 16;       // of an entry
  uint4* pages = reinterpret_cast<uint4*>(static_cast<uint8_t*>(value ? a.pages.v : a.pages.k) + layer * a.pages.layer_stride * (F8 ? 1 : 2));
  uint8_t* exps = F8 ? (value ? a.pages.v_exp : a.pages.k_exp) + layer * a.pages.exp_stride : nullptr;
  const uint32_t per_node = a.pages.nkv * kPieces, nodes = max(1u, kKeepThreads * kKeepChunks / per_node);
  auto moved = [&](uint32_t i, int64_t& from, int64_t& to) {
    const int32_t node = a.path[s * a.ldp + i];
    if (node < 0 || base < 0 || node > 0x7FFFFFFF - base) return false;
    from = kv_place(a.table, seq, base + node);
    to = kv_place(a.table, seq, base + int32_t(i));
    return from >= 0 && to >= 0 && from != to;
  };
  for (int32_t first = 1; first < count; first += nodes) {
    const uint32_t items = min(nodes, uint32_t(count - first)) * per_node;
    uint4 x[kKeepChunks];
    uint32_t byte[kKeepChunks];
    size_t dst[kKeepChunks];
    bool on[kKeepChunks];
    for (uint32_t round = 0; round < items; round += kKeepThreads * kKeepChunks) {   // (one round, but for more than 64 KV heads)
#pragma unroll
      for (int j = 0; j < kKeepChunks; ++j) {
        const uint32_t item = round + tid + j * kKeepThreads, i = first + item / per_node, head = item % per_node / kPieces, piece = item % kPieces;
        int64_t from = 0, to = 0;
        on[j] = item < items && moved(i, from, to);
        if (on[j]) {
          const size_t src = kv_entry(from, a.pages.nkv, head);
          dst[j] = kv_entry(to, a.pages.nkv, head);
          x[j] = pages[src * kPieces + piece];
          if (F8) byte[j] = exps[src];
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kKeepChunks; ++j) {
        const uint32_t piece = (round + tid + j * kKeepThreads) % kPieces;
        if (on[j]) {
          pages[dst[j] * kPieces + piece] = x[j];
          if (F8 && piece == 0) exps[dst[j]] = uint8_t(byte[j]);
        }
      }
      __syncthreads();
    }
  }
}

}  // namespace grb
