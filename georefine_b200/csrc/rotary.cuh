// Rotary positions of heads that lie in memory with any distance between rows and between heads: the first `turned` dimensions of each are pairs
// that turn by an angle of their own,
//   (a, b) -> factor (a cos - b sin, b cos + a sin),  angle = position * frequency[pair],
// paired (i, i + turned / 2) or (2 i, 2 i + 1); the rest is left as it is (copied, where the result goes elsewhere).  Backward: the same, turned the other
// way.
//
// A frequency is held as the fraction of a turn that one position adds, to the nearest 2^-64; its product with the position is exact and wraps where
// whole turns do, and the upper 32 bits are the angle: off by 2^-32 of a turn, and 2^-65 for every position - as much again at 2^33, 2^-25 at 2^40.
// (In FP32 a million times one radian is off by 0.03.)  Values and sums are FP32, rounded once.
//
// Memory bounds it: a value is read and written once.  A thread takes a piece of four neighbouring heads of a row; their loads are on their way while
// it works the piece's angles out, for itself: shared by the heads of a row through shared memory, they kept the row's loads and stores
// waiting for one another (8192 rows of 48 heads, 201 MB: 53 us, a CTA a row; 126 with the next row asked for meanwhile, in too many registers).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr int kRotaryThreads = 128;
constexpr uint32_t kRotaryMaxDim = 1024, kRotaryHeads = 4;

struct RotaryArgs {
  const void* x;              // [rows][heads][dim], rows ldx and heads ldxh elements apart
  void* out;
  int64_t ldx, ldxh, ldo, ldoh;
  const void* positions;      // [rows], 32 or 64 bits
  const uint64_t* turns;      // [turned / 2]: turns a position, in units of 2^-64
  float factor;               // negative sines: backward
  uint32_t rows, heads, dim, turned, wide_positions, backward;
  uint32_t items;             // pieces of a head: vectors of the pairs' first halves (or of pairs), then of the rest if that is copied
  uint32_t groups, groups_per_cta;   // of kRotaryHeads heads: of a row; a CTA's threads are items x groups
};

// BYTES of memory that are read and written together, as 32-bit words.
template <int BYTES>
struct RotaryWords {
  uint32_t v[BYTES < 4 ? 1 : BYTES / 4];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (BYTES == 16) { const uint4 x = *static_cast<const uint4*>(p); v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
    else if constexpr (BYTES == 8) { const uint2 x = *static_cast<const uint2*>(p); v[0] = x.x; v[1] = x.y; }
    else if constexpr (BYTES == 4) v[0] = *static_cast<const uint32_t*>(p);
    else v[0] = *static_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (BYTES == 16) *static_cast<uint4*>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    else if constexpr (BYTES == 8) *static_cast<uint2*>(p) = make_uint2(v[0], v[1]);
    else if constexpr (BYTES == 4) *static_cast<uint32_t*>(p) = v[0];
    else *static_cast<uint16_t*>(p) = uint16_t(v[0]);
  }
};
// The values of a word (one FP32, two of 16 bits), and the word of values.
template <class T>
__device__ __forceinline__ float2 rotary_in(uint32_t w) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w), 0.f);
  else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(bf_lo(w), bf_hi(w));
}
template <class T>
__device__ __forceinline__ uint32_t rotary_out(float lo, float hi) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(lo);
  else if constexpr (std::is_same_v<T, __half>) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }
  else return pack_bf(lo, hi);
}
__device__ __forceinline__ float rotary_left(float a, float b, float2 t) { return __fmaf_rn(a, t.x, -__fmul_rn(b, t.y)); }
__device__ __forceinline__ float rotary_right(float a, float b, float2 t) { return __fmaf_rn(b, t.x, __fmul_rn(a, t.y)); }

// Cosine and sine of an angle in units of 2^-32 of a turn, to 2^-24 or so: the nearest quarter turn aside, the rest is an eighth of a turn at
// most, where the powers to x^9 and x^10 of either series leave 2e-9.
__device__ __forceinline__ float2 rotary_cos_sin(uint32_t angle) {
  const uint32_t quarter = (angle + 0x20000000u) >> 30;
  const float x = __fmul_rn(float(int32_t(angle - (quarter << 30))), 1.4629180792671596e-9f), z = __fmul_rn(x, x);     // 2 pi 2^-32
  float s = __fmaf_rn(z, 2.7557319e-6f, -1.9841270e-4f);     // 1 / 9!, 1 / 7!, ...
  s = __fmaf_rn(z, s, 8.3333333e-3f);
  s = __fmaf_rn(z, s, -0.16666667f);
  s = __fmaf_rn(__fmul_rn(z, x), s, x);
  float c = __fmaf_rn(z, -2.7557319e-7f, 2.4801587e-5f);
  c = __fmaf_rn(z, c, -1.3888889e-3f);
  c = __fmaf_rn(z, c, 4.1666667e-2f);
  c = __fmaf_rn(z, c, -0.5f);
  c = __fmaf_rn(z, c, 1.f);
  const float a = quarter & 1u ? s : c, b = quarter & 1u ? c : s;
  return make_float2(__uint_as_float(__float_as_uint(a) ^ ((quarter + 1u) << 30 & 0x80000000u)), __uint_as_float(__float_as_uint(b) ^ (quarter << 30 & 0x80000000u)));
}

// V values of T a piece.  HALF: pairs (i, i + turned / 2); a piece is V first and V second components.  Otherwise neighbours: a piece is V / 2 pairs, one at V = 1,
// which is for memory that is aligned to nothing but its type.
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(kRotaryThreads, 5)
rotary_kernel(const RotaryArgs a) {
  step_kernel_entry();
  using Words = RotaryWords<V * int(sizeof(T))>;
  constexpr int kWords = sizeof(Words) / 4, kIn = sizeof(T) == 4 ? 1 : 2;      // values of a word
  constexpr bool kTwo = HALF || V == 1;                      // a piece is two loads
  constexpr uint32_t kFirst = HALF || V == 1 ? V : V / 2;    // pairs of a piece
  const uint32_t pairs = a.turned / 2, turning = pairs / kFirst, per_group = min(a.items, uint32_t(kRotaryThreads)), slot = threadIdx.x / per_group;
  const uint64_t id = uint64_t(blockIdx.x) * a.groups_per_cta + slot;
  const uint32_t row = uint32_t(id / a.groups), head0 = uint32_t(id - uint64_t(row) * a.groups) * kRotaryHeads;
  if (slot >= a.groups_per_cta || id >= uint64_t(a.rows) * a.groups) return;
  const int64_t pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[row] : static_cast<const int32_t*>(a.positions)[row];
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx + head0 * a.ldxh;
  T* const out = static_cast<T*>(a.out) + row * a.ldo + head0 * a.ldoh;
  for (uint32_t item = threadIdx.x % per_group; item < a.items; item += per_group) {
    // where a piece's parts lie: of the turning dimensions, or of the rest
    const bool turn = item < turning;
    const uint32_t first = !turn ? a.turned + (item - turning) * V : HALF ? item * V : kTwo ? 2 * item : item * V, second = first + (HALF ? pairs : 1u);
    Words u[kRotaryHeads], w[kRotaryHeads];
#pragma unroll
    for (uint32_t i = 0; i < kRotaryHeads; ++i)
      if (head0 + i < a.heads) {
        u[i].load(x + i * a.ldxh + first);
        if (kTwo && turn) w[i].load(x + i * a.ldxh + second);
      }
    if (turn) {
      float2 t[kFirst];
#pragma unroll
      for (uint32_t k = 0; k < kFirst; ++k) {
        const float2 f = rotary_cos_sin(uint32_t(uint64_t(pos) * a.turns[item * kFirst + k] >> 32));
        t[k] = make_float2(__fmul_rn(f.x, a.factor), __fmul_rn(f.y, a.backward ? -a.factor : a.factor));
      }
#pragma unroll
      for (uint32_t i = 0; i < kRotaryHeads; ++i)
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          if constexpr (kTwo) {                              // first components in u, second ones in w
            const float2 p = rotary_in<T>(u[i].v[k]), q = rotary_in<T>(w[i].v[k]);
            const float2 t0 = t[k * kIn], t1 = t[V == 1 ? 0 : k * kIn + kIn - 1];
            u[i].v[k] = rotary_out<T>(rotary_left(p.x, q.x, t0), rotary_left(p.y, q.y, t1));
            w[i].v[k] = rotary_out<T>(rotary_right(p.x, q.x, t0), rotary_right(p.y, q.y, t1));
          } else if constexpr (kIn == 2) {                   // a word is a pair
            const float2 p = rotary_in<T>(u[i].v[k]);
            u[i].v[k] = rotary_out<T>(rotary_left(p.x, p.y, t[k]), rotary_right(p.x, p.y, t[k]));
          } else if (k % 2 == 0) {                           // two words are
            const float p = __uint_as_float(u[i].v[k]), q = __uint_as_float(u[i].v[k + 1 < kWords ? k + 1 : k]);
            u[i].v[k] = __float_as_uint(rotary_left(p, q, t[k / 2]));
            u[i].v[k + 1 < kWords ? k + 1 : k] = __float_as_uint(rotary_right(p, q, t[k / 2]));
          }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kRotaryHeads; ++i)
      if (head0 + i < a.heads) {
        u[i].store(out + i * a.ldoh + first);
        if (kTwo && turn) w[i].store(out + i * a.ldoh + second);
      }
  }
}

}  // namespace grb
