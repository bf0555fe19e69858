// Rotary positions of heads that lie in memory with any distance between rows and between heads: the first `turned` dimensions of each are pairs
// that turn by an angle of their own,
//   (a, b) -> factor (a cos - b sin, b cos + a sin),  angle = position * frequency[pair],
// paired (i, i + turned / 2) or (2 i, 2 i + 1); the rest is left as it is (copied, where the result goes elsewhere).  Backward: the same, turned the other
// way.
//
// An angle is exact however far the position: a frequency is held as the 64-bit fraction of a turn that one position adds, the product with the
// position wraps where whole turns do, and its upper 32 bits are the angle to 2^-32 of a turn.  (In FP32 a million times one radian is off by
// 0.03.)  Sine and cosine are taken once for a row and pair, into shared memory, and serve all heads; values and sums are FP32, rounded once.
//
// Memory bounds it: a value is read and written once.  A thread's loads for up to four heads are on their way while the angles are worked out.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr int kRotaryThreads = 128;
constexpr uint32_t kRotaryMaxDim = 1024;

struct RotaryArgs {
  const void* x;              // [rows][heads][dim], rows ldx and heads ldxh elements apart
  void* out;
  int64_t ldx, ldxh, ldo, ldoh;
  const void* positions;      // [rows], 32 or 64 bits
  const uint64_t* turns;      // [turned / 2]: turns a position, in units of 2^-64
  float factor;               // negative sines: backward
  uint32_t rows, heads, dim, turned, wide_positions, backward;
  uint32_t items;             // pieces of a head: vectors of the pairs' first halves (or of pairs), then of the rest if that is copied
  uint32_t rows_per_cta, heads_at_once;      // threads: items x heads_at_once x rows_per_cta
};

template <class T>
__device__ __forceinline__ float rotary_in(T v) { return float(v); }
template <class T>
__device__ __forceinline__ T rotary_out(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
// V values that are read and written together.
template <class T, int V>
struct __align__(sizeof(T) * V) RotaryVector {
  T v[V];
};

// V values of T a piece.  HALF: pairs (i, i + turned / 2); a piece is V first and V second components.  Otherwise neighbours: a piece is V / 2 pairs, one at V = 1,
// which is for memory that is aligned to nothing but its type.
template <class T, int V, bool HALF>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const RotaryArgs a) {
  step_kernel_entry();
  extern __shared__ float2 rotary_table[];                   // [rows_per_cta][turned / 2]: cosine and sine times the factor
  using Vec = RotaryVector<T, V>;
  constexpr bool kTwo = HALF || V == 1;                      // a piece is two loads
  constexpr uint32_t kFirst = HALF || V == 1 ? V : V / 2;    // pairs of a piece
  constexpr uint32_t kAtOnce = 4;
  const uint32_t tid = threadIdx.x, pairs = a.turned / 2, turning = pairs / kFirst;      // pieces that turn
  const uint32_t per_row = min(a.items, uint32_t(kRotaryThreads)), slot = tid / per_row, local = slot / a.heads_at_once, head0 = slot % a.heads_at_once;
  const uint32_t row0 = blockIdx.x * a.rows_per_cta, row = row0 + local;
  const bool in = local < a.rows_per_cta && row < a.rows;
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  T* const out = static_cast<T*>(a.out) + row * a.ldo;
  Vec u[kAtOnce], w[kAtOnce];
  // where a piece's parts lie: of the turning dimensions, or of the rest
  auto place = [&](uint32_t item, uint32_t& first, uint32_t& second) {
    if (item >= turning) first = second = a.turned + (item - turning) * V;
    else if (HALF) first = item * V, second = first + pairs;
    else first = kTwo ? 2 * item : item * V, second = first + 1;
  };
  auto load = [&](uint32_t item, uint32_t head) {
    uint32_t first, second;
    place(item, first, second);
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) {
      const uint32_t h = head + i * a.heads_at_once;
      if (h >= a.heads) break;
      u[i] = *reinterpret_cast<const Vec*>(x + h * a.ldxh + first);
      if (kTwo && item < turning) w[i] = *reinterpret_cast<const Vec*>(x + h * a.ldxh + second);
    }
  };
  const uint32_t item0 = tid % per_row;
  if (in) load(item0, head0);
  for (uint32_t i = tid; i < a.rows_per_cta * pairs; i += kRotaryThreads) {
    const uint32_t r = i / pairs, p = i - r * pairs;
    if (row0 + r >= a.rows) break;
    const int64_t pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[row0 + r] : static_cast<const int32_t*>(a.positions)[row0 + r];
    const int32_t angle = int32_t(uint64_t(pos) * a.turns[p] >> 32);                    // of a turn, in units of 2^-32
    float s, c;
    sincospif(__fmul_rn(float(angle), 4.656612873077393e-10f), &s, &c);                 // 2^-31: in half turns
    rotary_table[i] = make_float2(__fmul_rn(c, a.factor), __fmul_rn(a.backward ? -s : s, a.factor));
  }
  __syncthreads();
  if (!in) return;
  for (uint32_t item = item0; item < a.items; item += per_row) {
    const bool turn = item < turning;
    float2 t[kFirst];
#pragma unroll
    for (uint32_t i = 0; i < kFirst; ++i)
      if (turn) t[i] = rotary_table[local * pairs + item * kFirst + i];
    uint32_t first, second;
    place(item, first, second);
    for (uint32_t head = head0; head < a.heads; head += kAtOnce * a.heads_at_once) {
      if (item != item0 || head != head0) load(item, head);
#pragma unroll
      for (uint32_t i = 0; i < kAtOnce; ++i) {
        const uint32_t h = head + i * a.heads_at_once;
        if (h >= a.heads) break;
        if (turn) {
#pragma unroll
          for (uint32_t k = 0; k < kFirst; ++k) {
            T& left = kTwo ? u[i].v[k < V ? k : 0] : u[i].v[2 * k < V ? 2 * k : 0];
            T& right = kTwo ? w[i].v[k < V ? k : 0] : u[i].v[2 * k + 1 < V ? 2 * k + 1 : 0];
            const float p = rotary_in(left), q = rotary_in(right);
            left = rotary_out<T>(__fmaf_rn(p, t[k].x, -__fmul_rn(q, t[k].y)));
            right = rotary_out<T>(__fmaf_rn(q, t[k].x, __fmul_rn(p, t[k].y)));
          }
        }
        *reinterpret_cast<Vec*>(out + h * a.ldoh + first) = u[i];
        if (kTwo && turn) *reinterpret_cast<Vec*>(out + h * a.ldoh + second) = w[i];
      }
    }
  }
}

}  // namespace grb
