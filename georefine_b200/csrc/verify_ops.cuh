// Verification of drafted tokens against the target's probabilities, from random numbers that the caller gives.
//
// A sequence's rows are the nodes of its draft tree in an order that puts parents first (a chain: each below the one before);
// row 0 is the pending token.  With p = softmax(logits / T) of a node's row, its children c are tried in order: c is kept when
// u_keep[c] (1 - S) < p[t_c], S being the mass of the tokens tried before it at this node (a token tried twice is not kept).
// Where none is kept, the last token is drawn from p without the tried ones: the first t whose cumulative mass exceeds
// u_draw times the whole.  With the drafter's own probabilities q (chains): kept when u q[t] < p[t], else drawn from max(p - q, 0).
//
// Two launches.  verify_rows: sums of every row's eighths in one pass over the logits - this is where the time goes, and memory
// bounds it.  verify_draw: a cluster per sequence walks the tree and draws from the one row where the walk ends.  A draw has a
// border at every token, so the masses there are summed in 64 bits: in 32 the borders of a flat distribution over 150000 tokens
// move by per mille of a token's width.  Rows and sequences are computed on their own, in a fixed order.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "step_utils.cuh"

namespace grb {

constexpr uint32_t kVerifyMaxNodes = 256;      // rows of one sequence
constexpr uint32_t kVerifyRegions = 128;       // runs of tiles that verify_draw sums: cut by the vocabulary alone
constexpr uint32_t kVerifySlices = 8;          // CTAs of a row in verify_rows
constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kVerifyDrawThreads = 512;
constexpr uint32_t kVerifyTile = 256;          // tokens a warp takes at a time, eight consecutive ones a lane
constexpr uint32_t kVerifyMaxVocab = 524288;
// log2(e) / T fits 32 bits with room, 2^104 of it is above 100 (see widen)
constexpr double kVerifyLeastTemperature = 1e-30, kVerifyMostTemperature = 1e20;

struct VerifyArgs {
  const void* logits;       // [rows][ldl] BF16 or FP32
  int64_t ldl;
  const int32_t* tokens;    // [rows]
  const int32_t* parent;    // [rows], within the sequence; null: chains
  const int32_t* starts;    // [seqs + 1]
  const float* u_keep;      // [rows]
  const float* u_draw;      // [seqs]
  const float* q;           // [rows][ldq] or null: what row i's token was drawn from
  int64_t ldq;
  double2* stats;           // scratch [rows][8]: (m, Z) of an eighth of the row: its largest logit, Z = sum of 2^((l[t] - m) log2_scale) over it
  int32_t* out_tokens;      // [seqs][width]
  int32_t* out_rows;        // [seqs][width]
  int32_t* out_count;       // [seqs]
  uint32_t rows, seqs, vocab, width;
  double log2_scale;        // log2(e) / T
};

template <bool F32>
__device__ __forceinline__ float verify_logit(const void* row, uint32_t t) {
  if constexpr (F32) return static_cast<const float*>(row)[t];
  else return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[t]);
}
// Eight consecutive values from t (a multiple of 8), `beyond` outside the vocabulary.  VEC: rows start on 16-byte boundaries.
template <bool F32, bool VEC>
__device__ __forceinline__ void verify_load8(const void* row, uint32_t t, uint32_t vocab, float (&x)[8], float beyond = -INFINITY) {
  if (VEC && t + 8 <= vocab) {
    if constexpr (F32) {
      const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(row) + t)[0], b = reinterpret_cast<const float4*>(static_cast<const float*>(row) + t)[1];
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(row) + t);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { x[2 * i] = bf_lo(w[i]); x[2 * i + 1] = bf_hi(w[i]); }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = t + i < vocab ? verify_logit<F32>(row, t + i) : beyond;
}
template <bool F32>
__device__ __forceinline__ const void* verify_row(const VerifyArgs& a, uint32_t row) {
  return static_cast<const uint8_t*>(a.logits) + int64_t(row) * a.ldl * (F32 ? 4 : 2);
}

__device__ __forceinline__ double lds_f64_cluster(uint32_t a) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
  return v;
}

// Eight consecutive logits as they are loaded, -infinity beyond the vocabulary.
template <bool F32>
struct VerifyOctet;
template <>
struct VerifyOctet<false> {
  uint32_t w[4];
  template <bool VEC>
  __device__ __forceinline__ void load(const void* row, uint32_t t, uint32_t vocab) {
    const auto* p = static_cast<const __nv_bfloat16*>(row) + t;
    if (VEC && t + 8 <= vocab) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      return;
    }
    const auto* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (t + 2 * i < vocab ? u[2 * i] : 0xFF80u) | (t + 2 * i + 1 < vocab ? uint32_t(u[2 * i + 1]) << 16 : 0xFF800000u);
  }
  __device__ __forceinline__ float max(float m) const {
    uint32_t x = w[0];
#pragma unroll
    for (int i = 1; i < 4; ++i) asm("max.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(w[i]));
    return fmaxf(m, fmaxf(bf_lo(x), bf_hi(x)));
  }
  __device__ __forceinline__ float operator[](int i) const { return i & 1 ? bf_hi(w[i >> 1]) : bf_lo(w[i >> 1]); }
};
template <>
struct VerifyOctet<true> {
  float x[8];
  template <bool VEC>
  __device__ __forceinline__ void load(const void* row, uint32_t t, uint32_t vocab) { verify_load8<true, VEC>(row, t, vocab, x); }
  __device__ __forceinline__ float max(float m) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, x[i]);
    return m;
  }
  __device__ __forceinline__ float operator[](int i) const { return x[i]; }
};

// Grid (8, rows): each CTA takes an eighth of the row, a thread up to ten octets of it at a time (all of its share of 152064
// BF16 logits), loaded together: the CTA's maximum of them, then one multiply-add, one exponential and one addition each.
// Bound by memory, the exponentials (16 per SM and cycle) not far behind.  The eighths are put together by whoever needs the
// row: doing it here, in a cluster, left the SMs waiting for chains of exponentials and remote reads (546 rows of 152064 BF16
// logits: 54 us, this 34, 4.9 TB/s).
// The exponent is (l - m) hi, the difference first: whatever the logits' size (a mask of the type's lowest value) and however small
// the temperature, it is 0 for the maximum and negative or -infinity for the others.  Two roundings and what hi (log2_scale in 32 bits)
// leaves out are 2.5 2^-24 of an exponent whose weight falls with it.  Eight exponentials are added in 32 bits, the eights in 64: a
// probability is off by the exponentials' 2^-22 at most.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads)
verify_rows_kernel(const VerifyArgs a) {
  step_kernel_entry();
  constexpr int B = F32 ? 3 : 5;
  __shared__ float tops[kVerifyThreads / 32];
  __shared__ double sums[kVerifyThreads / 32];
  const uint32_t row = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const void* const src = verify_row<F32>(a, row);
  const float hi = float(a.log2_scale);
  const uint32_t octets = (a.vocab + 7) / 8, per = (octets + kVerifySlices - 1) / kVerifySlices;
  const uint32_t first = min(octets, blockIdx.x * per), last = min(octets, first + per);
  const float2 hi2 = make_float2(hi, hi);
  float m = -INFINITY;
  double sum = 0.0;
#pragma unroll 1
  for (uint32_t o0 = first + tid; o0 < last; o0 += B * kVerifyThreads) {
    VerifyOctet<F32> x[B];
#pragma unroll
    for (int b = 0; b < B; ++b) x[b].template load<VEC>(src, (o0 + b * kVerifyThreads < last ? o0 + b * kVerifyThreads : octets) * 8, a.vocab);
    float top = m;
#pragma unroll
    for (int b = 0; b < B; ++b) top = x[b].max(top);
    if (top == -INFINITY) continue;
    if (top > m) {
      sum *= double(exp2_approx(__fmul_rn(__fsub_rn(m, top), hi)));      // (from -infinity: 0)
      m = top;
    }
    const float2 less = make_float2(-m, -m);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      float eight = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 e = mul2(add2(make_float2(x[b][i], x[b][i + 1]), less), hi2);
        eight = __fadd_rn(__fadd_rn(eight, exp2_approx(e.x)), exp2_approx(e.y));
      }
      sum += double(eight);
    }
  }
  // all under the CTA's maximum
  float top = warp_max(m);
  if (lane == 0) tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < int(kVerifyThreads / 32); ++w) top = fmaxf(top, tops[w]);
  if (m < top) sum *= double(exp2_approx(__fmul_rn(__fsub_rn(m, top), hi)));
#pragma unroll
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < int(kVerifyThreads / 32); ++w) sum += sums[w];
    a.stats[size_t(row) * kVerifySlices + blockIdx.x] = make_double2(double(top), sum);
  }
}

// 2^(d scale16 / 16) to 2^-42, for exponents in (-101, 0]: d scale16 = k + f with k whole, 2^(k / 16) from a table and a shift, 2^(f / 16) by
// the first six terms of the exponential series in f ln 2 / 16 (|f| <= 1 / 2: the seventh is 1.4e-13).  Sixteen entries lie in as many
// pairs of banks, so a warp's look-ups never collide; 64 of them and one term less took as long.  (The exponent comes as a product so
// that no operation goes into it alone.)
constexpr uint32_t kExpTable = 16;
__device__ __forceinline__ double exp2_f64(double d, double scale16, const double* table) {
  constexpr double kRound = 6755399441055744.0;     // 1.5 * 2^52: what is added to it rounds to a whole number in its low bits
  const double t = __fma_rn(d, scale16, kRound);
  const int k = __double2loint(t);                  // (whole and fraction: the bits above and below the table's)
  const double f = __fma_rn(d, scale16, -(t - kRound));
  double q = __fma_rn(f, 1.2715871950558131e-09, 1.467610032291943e-07);      // L^5 / 120, L^4 / 24 with L = ln 2 / 16
  q = __fma_rn(f, q, 1.3550807779497457e-05);                               // L^3 / 6
  q = __fma_rn(f, q, 0.0009383847928089872);                               // L^2 / 2
  q = __fma_rn(f, q, 0.04332169878499658);
  const double r = table[k & int(kExpTable - 1)] * __fma_rn(f, q, 1.0);
  return __hiloint2double(__double2hiint(r) + ((k & -int(kExpTable)) << 16), __double2loint(r));
}

// x 2^-896 in 64 bits, exactly, for a finite x, by integer operations in place of a conversion; -infinity becomes -2^128 2^-896, which is
// 2^104 2^-896 below every number.
__device__ __forceinline__ double widen(float x) {
  const int u = __float_as_int(x);
  return __hiloint2double((u >> 3) & int(0x8FFFFFFFu), int(uint32_t(u) << 29));
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  return v;
}
// Inclusive prefix sums over the lanes.
__device__ __forceinline__ double warp_scan_f64(double v, uint32_t lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = __shfl_up_sync(0xFFFFFFFFu, v, off);
    if (lane >= uint32_t(off)) v += o;
  }
  return v;
}

// What verify_draw draws from: masses of a row's tokens.  A mass below 2^-100 of the likeliest token's counts as that much, which no
// draw can feel (a draw's target is at least 2^-75).  The bound is put on the difference l - top in 64 bits: one on the logit, rounded
// to its 32 bits, may be the top itself where the logits are large or the temperature is small.
constexpr double kLeastMass = 8.077935669463161e-28, kLeastTarget = 2.6469779601696886e-23;    // 2^-90, 2^-75
struct VerifyMasses {
  const float* q;           // refused draft's distribution, or null
  const int32_t* tried;     // the tried tokens
  const double* table;
  uint32_t tried_count, vocab;
  bool q_vec;               // rows of q start on 16-byte boundaries
  uint32_t least;           // upper half of the difference that stands for 2^-100
  double top, scale16, inverse;   // top: the likeliest token's logit, times 2^-896; scale16: 16 log2_scale, times 2^896; inverse: of the sum of the masses without q, where q is subtracted

  // Eight consecutive tokens from t.  `plain`: without q.  `some`: of them were tried.  (No branch between the exponentials: each
  // is a chain of a dozen dependent operations, and only side by side do they keep the unit busy.)
  template <bool F32>
  __device__ __forceinline__ void eight(const VerifyOctet<F32>& x, uint32_t t, bool plain, bool some, double (&m)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double d = widen(x[i]) - top;
      // from the bound to 0: of numbers that are not positive, the bits of the larger magnitude are the larger integer (positive is a NaN's alone)
      m[i] = exp2_f64(__hiloint2double(int(min(max(uint32_t(__double2hiint(d)), 0x80000000u), least)), __double2loint(d)), scale16, table);
    }
    if (q && !plain) {
      float o[8];
      if (q_vec) verify_load8<true, true>(q, t, vocab, o, 0.f);
      else verify_load8<true, false>(q, t, vocab, o, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = fmax(__fma_rn(m[i], inverse, -double(o[i])), 0.0);
    } else if (some && !q) {
#pragma unroll 1
      for (uint32_t j = 0; j < tried_count; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (tried[j] == int32_t(t) + i) m[i] = 0.0;
    }
  }
};

// Grid (CTAs of a sequence, sequences), a cluster per sequence: every warp of the cluster sums its regions of the row in 64 bits;
// the sums are exchanged, and the warp in whose region the draw falls goes through it again, tile by tile.  All three passes
// (the middle one for every draw, the first where q is subtracted, the last) run the same loop: unrolled, or written out for each,
// the kernel was slowed by the fetching of its own instructions.
// One sequence: 13 us, a chain of dependent loads, barriers and the walk more than the sums.  128 sequences: 43 us, of which the
// 64-bit operations, twelve a token, take 12.  The cluster is as large (8, 4 or 2 CTAs) as lets all sequences be resident at once:
// with that chain a second wave costs more than the larger share of a CTA in the first.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kVerifyDrawThreads, 2)
verify_draw_kernel(const VerifyArgs a) {
  step_kernel_entry();
  extern __shared__ uint32_t struck[];              // ceil(vocab / 256) words: one bit for every eight tokens that hold a tried one
  __shared__ int32_t token[kVerifyMaxNodes], up[kVerifyMaxNodes], next[kVerifyMaxNodes], tried[kVerifyMaxNodes];
  __shared__ double node_top[kVerifyMaxNodes], node_sum[kVerifyMaxNodes];
  __shared__ double node_mass[kVerifyMaxNodes];     // the parent's probability of a node's token; 0 for one tried before
  __shared__ __align__(128) double table[kExpTable];
  __shared__ double sums[kVerifyRegions], region[kVerifyRegions];
  __shared__ uint32_t at_end, tried_count, path_count;
  __shared__ int32_t last_tried;
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const float u_draw = a.u_draw[seq];
  const int64_t begin = a.starts[seq], end = a.starts[seq + 1];
  const bool some = begin >= 0 && end > begin && end <= int64_t(a.rows);
  const uint32_t first = some ? uint32_t(begin) : 0u, n = some ? uint32_t(min(end - begin, int64_t(kVerifyMaxNodes))) : 0u;
  int32_t* const out_tokens = a.out_tokens + size_t(seq) * a.width;
  int32_t* const out_rows = a.out_rows + size_t(seq) * a.width;
  if (!n) {                                         // (the whole cluster alike)
    if (blockIdx.x == 0) {
      for (uint32_t i = tid; i < a.width; i += kVerifyDrawThreads) out_tokens[i] = out_rows[i] = -1;
      if (tid == 0) a.out_count[seq] = 0;
    }
    return;
  }
  // every node's token, parent, and row sum; then the parent's probability of the token
  const uint32_t tiles = (a.vocab + kVerifyTile - 1) / kVerifyTile, per = (tiles + kVerifyRegions - 1) / kVerifyRegions;
  float u_keep = 0.f;
  if (tid < n) {
    const int32_t t = a.tokens[first + tid];
    int32_t p = tid == 0 ? -1 : a.parent ? a.parent[first + tid] : int32_t(tid) - 1;
    if (p < 0 || p >= int32_t(tid)) p = -1;
    u_keep = a.u_keep[first + tid];
    double2 part[kVerifySlices];
#pragma unroll
    for (int i = 0; i < int(kVerifySlices); ++i) part[i] = a.stats[size_t(first + tid) * kVerifySlices + i];
    double top = part[0].x, sum = 0.0;
#pragma unroll
    for (int i = 1; i < int(kVerifySlices); ++i) top = fmax(top, part[i].x);
#pragma unroll
    for (int i = 0; i < int(kVerifySlices); ++i)
      if (part[i].x > -INFINITY) sum += part[i].y * double(exp2_approx(float((part[i].x - top) * a.log2_scale)));
    node_top[tid] = top;
    node_sum[tid] = sum;
    token[tid] = t;
    up[tid] = p;
    next[tid] = 0x7FFFFFFF;
  }
  for (uint32_t i = tid; i < tiles; i += kVerifyDrawThreads) struck[i] = 0u;
  if (tid >= kVerifyDrawThreads - kExpTable) table[tid - (kVerifyDrawThreads - kExpTable)] = exp2(double(tid - (kVerifyDrawThreads - kExpTable)) / kExpTable);
  if (tid == 0) tried_count = 0u, last_tried = -1;
  __syncthreads();
  const int32_t mine_up = tid < n ? up[tid] : -1;
  float q_mine = 0.f;
  double mass = 0.0;
  if (mine_up >= 0 && uint32_t(token[tid]) < a.vocab) {
    if (a.q) q_mine = a.q[int64_t(first + tid) * a.ldq + token[tid]];
    mass = exp2((double(verify_logit<F32>(verify_row<F32>(a, first + mine_up), uint32_t(token[tid]))) - node_top[mine_up]) * a.log2_scale) / node_sum[mine_up];
  }
  if (a.parent && mine_up >= 0)                     // a token tried before at this node
    for (uint32_t j = uint32_t(mine_up) + 1; j < tid; ++j)
      if (up[j] == mine_up && token[j] == token[tid]) mass = 0.0;
  if (tid < n) node_mass[tid] = mass;
  __syncthreads();
  if (mine_up >= 0) {
    double left = double(u_keep);
    if (a.q) {
      left *= double(q_mine);
    } else if (a.parent) {
      double before = 0.0;
      for (uint32_t j = uint32_t(mine_up) + 1; j < tid; ++j) before += up[j] == mine_up ? node_mass[j] : 0.0;
      left *= 1.0 - before;
    }
    if (left < mass) atomicMin(&next[mine_up], int32_t(tid));
  }
  __syncthreads();
  if (tid == 0) {
    uint32_t node = 0, count = 1;
    if (blockIdx.x == 0) out_rows[0] = 0;
    while (count < a.width && next[node] < int32_t(n)) {
      node = uint32_t(next[node]);
      if (blockIdx.x == 0) { out_tokens[count - 1] = token[node]; out_rows[count] = int32_t(node); }
      ++count;
    }
    at_end = node;
    path_count = count;
    if (blockIdx.x == 0) a.out_count[seq] = int32_t(count);
  }
  __syncthreads();
  const uint32_t node = at_end, count = path_count;
  if (blockIdx.x == 0)
    for (uint32_t i = count + tid; i < a.width; i += kVerifyDrawThreads) { out_tokens[i] = -1; out_rows[i] = -1; }
  // the children of the last node were tried and refused (where the outputs' width cut the walk short, they were not tried)
  if (mine_up == int32_t(node) && next[node] >= int32_t(n)) {
    tried[atomicAdd(&tried_count, 1u)] = token[tid];
    atomicMax(&last_tried, int32_t(tid));
    if (uint32_t(token[tid]) < a.vocab) atomicOr(&struck[token[tid] >> 8], 1u << ((token[tid] >> 3) & 31));
  }
  __syncthreads();
  VerifyMasses masses;
  masses.q = a.q && tried_count ? a.q + int64_t(first + node + 1) * a.ldq : nullptr;
  masses.q_vec = (reinterpret_cast<uintptr_t>(masses.q) & 15) == 0;
  masses.tried = tried;
  masses.table = table;
  masses.tried_count = tried_count;
  masses.vocab = a.vocab;
  masses.scale16 = a.log2_scale * 16 * 0x1p896;
  masses.least = uint32_t(__double2hiint(-100.0 / a.log2_scale * 0x1p-896));
  masses.top = node_top[node] * 0x1p-896;
  masses.inverse = 1.0;
  const void* const row = verify_row<F32>(a, first + node);
  constexpr uint32_t kWarps = kVerifyDrawThreads / 32, kLane = kVerifyRegions / 32;     // regions of a lane, where one looks them over
  const uint32_t of_cta = kVerifyRegions / gridDim.x, of_warp = of_cta / kWarps;
  uint32_t region0 = blockIdx.x * of_cta + warp * of_warp, region1 = region0 + of_warp;
  double target = 0.0, at = 0.0;                    // last pass: the mass to pass, and the mass before the tile
  int32_t fallback = -1;                            // last pass: where rounding leaves no such place, the last token with any mass
#pragma unroll 1
  for (int pass = masses.q ? 0 : 1; pass < 3; ++pass) {
#pragma unroll 1
    for (uint32_t r = region0; r < region1; ++r) {
      const uint32_t tile0 = min(tiles, r * per), tile1 = min(tiles, tile0 + per);
      double total = 0.0;
      VerifyOctet<F32> x;
      x.template load<VEC>(row, tile0 < tile1 ? tile0 * kVerifyTile + lane * 8 : a.vocab, a.vocab);
#pragma unroll 1
      for (uint32_t tile = tile0; tile < tile1; ++tile) {
        const VerifyOctet<F32> now = x;
        const uint32_t t0 = tile * kVerifyTile + lane * 8;
        x.template load<VEC>(row, tile + 1 < tile1 ? t0 + kVerifyTile : a.vocab, a.vocab);
        const bool any = struck[tile] >> lane & 1u;
        double m[8];
        masses.eight(now, t0, pass == 0, any, m);
        const double eight = ((m[0] + m[1]) + (m[2] + m[3])) + ((m[4] + m[5]) + (m[6] + m[7]));
        if (pass < 2) {
          total += eight;
          continue;
        }
        const double upto = at + warp_scan_f64(eight, lane);
        const uint32_t with = __ballot_sync(0xFFFFFFFFu, eight > kLeastMass), past = __ballot_sync(0xFFFFFFFFu, eight > kLeastMass && upto > target);
        at = __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (!with) continue;
        const uint32_t owner = past ? uint32_t(__ffs(past)) - 1u : 31u - __clz(with);
        double running = upto - eight;
        int32_t t = -1;                             // of this lane: the last token that the running mass had not passed before
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (m[i] > kLeastMass && (running <= target || t < 0)) t = int32_t(t0) + i;
          running += m[i];
        }
        fallback = __shfl_sync(0xFFFFFFFFu, t, owner);
        if (past) break;
      }
      if (pass < 2) {
        total = warp_sum_f64(total);
        if (lane == 0) sums[r - blockIdx.x * of_cta] = total;
      }
    }
    if (pass == 2) break;
    cluster_sync();
    if (tid < kVerifyRegions) region[tid] = lds_f64_cluster(cluster_map(smem_u32(&sums[tid % of_cta]), tid / of_cta));
    cluster_sync();                                 // all sums have been read: the next pass may write its own
    double share[kLane], of_lane = 0.0;
#pragma unroll
    for (uint32_t r = 0; r < kLane; ++r) of_lane += share[r] = region[kLane * lane + r];
    const double upto = warp_scan_f64(of_lane, lane), whole = __shfl_sync(0xFFFFFFFFu, upto, 31);
    if (!pass) {
      masses.inverse = 1.0 / whole;
      continue;
    }
    // the region where the running mass passes the target, or the last one with any mass
    target = fmax(double(u_draw) * whole, kLeastTarget);
    if (!(whole > kLeastTarget) || masses.top == -INFINITY) {      // nothing left to draw from (a drafted token of probability 1 that was refused), or no token in the row
      if (blockIdx.x == 0 && tid == 0) out_tokens[count - 1] = last_tried >= 0 ? token[last_tried] : 0;
      return;
    }
    const uint32_t past = __ballot_sync(0xFFFFFFFFu, of_lane > kLeastMass && upto > target), with = __ballot_sync(0xFFFFFFFFu, of_lane > kLeastMass);
    const uint32_t holder = past ? uint32_t(__ffs(past)) - 1u : 31u - __clz(with);
    double run = __shfl_sync(0xFFFFFFFFu, upto - of_lane, holder);
    uint32_t chosen = 0;
    bool there = false;
#pragma unroll
    for (uint32_t r = 0; r < kLane; ++r) {
      const double s = __shfl_sync(0xFFFFFFFFu, share[r], holder);
      if (!there && s > kLeastMass) { chosen = kLane * holder + r; at = run; }
      run += s;
      there = there || (s > kLeastMass && run > target);
    }
    if (chosen < region0 || chosen >= region1) return;
    region0 = chosen;
    region1 = chosen + 1;
  }
  if (lane == 0) out_tokens[count - 1] = fallback;
}

}  // namespace grb
