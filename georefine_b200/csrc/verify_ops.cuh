// Verification of drafted tokens against the target's probabilities, from random numbers that the caller gives.
//
// A sequence's rows are the nodes of its draft tree in an order that puts parents first (a chain: each below the one before);
// row 0 is the pending token.  With p = softmax(logits / T) of a node's row, its children c are tried in order: c is kept when
// u_keep[c] (1 - S) < p[t_c], S being the mass of the tokens tried before it at this node (a token tried twice is not kept).
// Where none is kept, the last token is drawn from p without the tried ones: the first t whose cumulative mass exceeds
// u_draw times the whole.  With the drafter's own probabilities q (chains): kept when u q[t] < p[t], else drawn from max(p - q, 0).
//
// Two launches.  verify_rows: maximum and sum of every row in one pass over the logits - this is where the time goes, and memory
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
constexpr uint32_t kVerifyCluster = 8;
constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kVerifyTile = 256;          // tokens a warp takes at a time, eight consecutive ones a lane
constexpr uint32_t kVerifyWarps = kVerifyCluster * kVerifyThreads / 32;
constexpr uint32_t kVerifyMaxVocab = kVerifyWarps * 32 * kVerifyTile;

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
  double2* stats;           // scratch [rows]: maximum, sum of exp((l - maximum) / T)
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
// Eight consecutive logits from t (a multiple of 8); beyond the vocabulary -infinity.  VEC: rows start on 16-byte boundaries.
template <bool F32, bool VEC>
__device__ __forceinline__ void verify_load8(const void* row, uint32_t t, uint32_t vocab, float (&x)[8]) {
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
  for (int i = 0; i < 8; ++i) x[i] = t + i < vocab ? verify_logit<F32>(row, t + i) : -INFINITY;
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

// (maximum, sum under it) of two shares
struct VerifyShare {
  float max;
  double sum;
};
// 2^(d scale) for d <= 0, the product to 2^-24 of itself.  (-infinity times the scale's low part may have either sign.)
__device__ __forceinline__ float verify_exp(float d, float scale_hi, float scale_lo) {
  d = fmaxf(d, -1e30f);
  return exp2_approx(__fmaf_rn(d, scale_hi, __fmul_rn(d, scale_lo)));
}
__device__ __forceinline__ VerifyShare verify_join(VerifyShare x, VerifyShare y, float hi, float lo) {
  const float m = fmaxf(x.max, y.max);
  if (m == -INFINITY) return x;
  return {m, x.sum * double(verify_exp(__fsub_rn(x.max, m), hi, lo)) + y.sum * double(verify_exp(__fsub_rn(y.max, m), hi, lo))};
}

// Grid (8, rows), clusters of 8: each CTA takes an eighth of the row.  Eight exponentials are added in 32 bits, the eights in 64:
// a probability is then off by its exponentials' rounding alone, 2^-22 at most, which is what a comparison with u_keep can feel.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads)
verify_rows_kernel(const VerifyArgs a) {
  step_kernel_entry();
  __shared__ VerifyShare shares[kVerifyThreads / 32];
  __shared__ __align__(8) double mine[2];
  const uint32_t row = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const void* const src = verify_row<F32>(a, row);
  const float hi = float(a.log2_scale), lo = float(a.log2_scale - double(hi));
  const uint32_t octets = (a.vocab + 7) / 8, per = (octets + kVerifyCluster - 1) / kVerifyCluster;
  const uint32_t first = blockIdx.x * per, last = min(octets, first + per);
  VerifyShare s{-INFINITY, 0.0};
  for (uint32_t o = first + tid; o < last; o += kVerifyThreads) {
    float x[8];
    verify_load8<F32, VEC>(src, o * 8, a.vocab, x);
    float m = s.max;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, x[i]);
    if (m == -INFINITY) continue;
    if (m > s.max) {
      s.sum *= double(verify_exp(__fsub_rn(s.max, m), hi, lo));
      s.max = m;
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = __fadd_rn(sum, verify_exp(__fsub_rn(x[i], m), hi, lo));
    s.sum += double(sum);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    const VerifyShare o{__shfl_xor_sync(0xFFFFFFFFu, s.max, off), __shfl_xor_sync(0xFFFFFFFFu, s.sum, off)};
    s = verify_join(s, o, hi, lo);
  }
  if (lane == 0) shares[warp] = s;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < int(kVerifyThreads / 32); ++w) s = verify_join(s, shares[w], hi, lo);
    mine[0] = double(s.max);
    mine[1] = s.sum;
  }
  cluster_sync();
  if (blockIdx.x == 0 && tid == 0) {
    for (uint32_t r = 1; r < kVerifyCluster; ++r) {
      const uint32_t at = cluster_map(smem_u32(mine), r);
      s = verify_join(s, VerifyShare{float(lds_f64_cluster(at)), lds_f64_cluster(at + 8)}, hi, lo);
    }
    a.stats[row] = make_double2(double(s.max), s.sum);
  }
  cluster_sync();                                   // (a CTA may not leave while its share is read)
}

__device__ __forceinline__ double shfl_up_f64(double v, int off) { return __shfl_up_sync(0xFFFFFFFFu, v, off); }
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  return v;
}
// Inclusive prefix sums over the lanes.
__device__ __forceinline__ double warp_scan_f64(double v, uint32_t lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const double o = shfl_up_f64(v, off);
    if (lane >= uint32_t(off)) v += o;
  }
  return v;
}

// What verify_draw draws from: eight consecutive tokens' masses.
template <bool F32, bool VEC>
struct VerifyMasses {
  const void* row;
  const float* q;           // refused draft's distribution, or null
  const uint32_t* struck;   // one bit for every eight tokens that hold a tried one
  const int32_t* tried;     // the tried tokens
  uint32_t tried_count, vocab;
  double maximum, scale, total;   // total: of the masses without q, where q is subtracted

  __device__ __forceinline__ void whole(uint32_t t, double (&m)[8]) const {
    float x[8];
    verify_load8<F32, VEC>(row, t, vocab, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double y = (double(x[i]) - maximum) * scale;
      m[i] = y > -100.0 ? exp2(y) : 0.0;           // below 2^-100 of the likeliest: none
    }
  }
  __device__ __forceinline__ void operator()(uint32_t t, double (&m)[8]) const {
    whole(t, m);
    if (q) {
#pragma unroll
      for (int i = 0; i < 8; ++i) m[i] = t + i < vocab ? fmax(m[i] / total - double(q[t + i]), 0.0) : 0.0;
    } else if (struck[t >> 8] >> ((t >> 3) & 31u) & 1u) {
      for (uint32_t j = 0; j < tried_count; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (tried[j] == int32_t(t) + i) m[i] = 0.0;
    }
  }
};

// Grid (8, sequences), clusters of 8.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads)
verify_draw_kernel(const VerifyArgs a) {
  step_kernel_entry();
  extern __shared__ uint32_t struck[];              // ceil(vocab / 256) words
  __shared__ int32_t token[kVerifyMaxNodes], up[kVerifyMaxNodes], next[kVerifyMaxNodes], tried[kVerifyMaxNodes];
  __shared__ double node_mass[kVerifyMaxNodes];     // the parent's probability of a node's token; 0 for one tried before
  __shared__ double warp_total[kVerifyThreads / 32], region[kVerifyWarps];
  __shared__ uint32_t at_end, tried_count, path_count;
  __shared__ int32_t refused;
  const uint32_t seq = blockIdx.y, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const int64_t begin = a.starts[seq], end = a.starts[seq + 1];
  const bool some = begin >= 0 && end > begin && end <= int64_t(a.rows);
  const uint32_t first = some ? uint32_t(begin) : 0u, n = some ? uint32_t(min(end - begin, int64_t(kVerifyMaxNodes))) : 0u;
  int32_t* const out_tokens = a.out_tokens + size_t(seq) * a.width;
  int32_t* const out_rows = a.out_rows + size_t(seq) * a.width;
  if (!n) {                                         // (the whole cluster alike)
    if (blockIdx.x == 0) {
      for (uint32_t i = tid; i < a.width; i += kVerifyThreads) out_tokens[i] = out_rows[i] = -1;
      if (tid == 0) a.out_count[seq] = 0;
    }
    return;
  }
  // every node's token, parent, and the parent's probability of the token
  const uint32_t words = (a.vocab + 255) / 256;
  for (uint32_t i = tid; i < words; i += kVerifyThreads) struck[i] = 0u;
  if (tid < n) {
    const int32_t t = a.tokens[first + tid];
    int32_t p = tid == 0 ? -1 : a.parent ? a.parent[first + tid] : int32_t(tid) - 1;
    if (p < 0 || p >= int32_t(tid)) p = -1;
    token[tid] = t;
    up[tid] = p;
    next[tid] = 0x7FFFFFFF;
    double mass = 0.0;
    if (p >= 0 && uint32_t(t) < a.vocab) {
      const double2 st = a.stats[first + p];
      mass = exp2((double(verify_logit<F32>(verify_row<F32>(a, first + p), uint32_t(t))) - st.x) * a.log2_scale) / st.y;
    }
    node_mass[tid] = mass;
  }
  __syncthreads();
  const int32_t mine_up = tid > 0 && tid < n ? up[tid] : -1;
  bool again = false;                               // a token tried before at this node
  if (mine_up >= 0 && a.parent)
    for (uint32_t j = uint32_t(mine_up) + 1; j < tid; ++j) again = again || (up[j] == mine_up && token[j] == token[tid]);
  __syncthreads();
  if (again) node_mass[tid] = 0.0;
  __syncthreads();
  if (mine_up >= 0) {
    bool keep;
    if (a.q) {
      const int32_t t = token[tid];
      keep = uint32_t(t) < a.vocab && double(a.u_keep[first + tid]) * double(a.q[int64_t(first + tid) * a.ldq + t]) < node_mass[tid];
    } else {
      double before = 0.0;
      if (a.parent)
        for (uint32_t j = uint32_t(mine_up) + 1; j < tid; ++j) before += up[j] == mine_up ? node_mass[j] : 0.0;
      keep = double(a.u_keep[first + tid]) * (1.0 - before) < node_mass[tid];
    }
    if (keep) atomicMin(&next[mine_up], int32_t(tid));
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
    // cut short by the width of the outputs: the node's children were not tried
    const bool cut = next[node] < int32_t(n);
    uint32_t k = 0;
    for (uint32_t j = node + 1; j < n && !cut; ++j)
      if (up[j] == int32_t(node)) tried[k++] = token[j];
    at_end = node;
    path_count = count;
    tried_count = k;
    refused = k ? tried[k - 1] : 0;
    if (blockIdx.x == 0) {
      for (uint32_t i = count; i < a.width; ++i) { out_tokens[i] = -1; out_rows[i] = -1; }
      a.out_count[seq] = int32_t(count);
    }
  }
  __syncthreads();
  if (tid < tried_count && uint32_t(tried[tid]) < a.vocab) atomicOr(&struck[tried[tid] >> 8], 1u << ((tried[tid] >> 3) & 31));
  __syncthreads();
  const uint32_t node = at_end, count = path_count;
  VerifyMasses<F32, VEC> masses;
  masses.row = verify_row<F32>(a, first + node);
  masses.q = a.q && tried_count ? a.q + int64_t(first + node + 1) * a.ldq : nullptr;
  masses.struck = struck;
  masses.tried = tried;
  masses.tried_count = tried_count;
  masses.vocab = a.vocab;
  masses.scale = a.log2_scale;
  masses.maximum = a.stats[first + node].x;
  masses.total = 1.0;
  const uint32_t tiles = (a.vocab + kVerifyTile - 1) / kVerifyTile, per = (tiles + kVerifyWarps - 1) / kVerifyWarps;   // (per <= 32)
  const uint32_t unit = blockIdx.x * (kVerifyThreads / 32) + warp, tile0 = min(tiles, unit * per), tile1 = min(tiles, tile0 + per);
  double of_tile = 0.0;                             // lane i: of the warp's tile i
  double r0 = 0.0, r1 = 0.0, upto_region = 0.0;     // lane i: regions 2 i and 2 i + 1, and their running sum
  for (int pass = masses.q ? 0 : 1; pass < 2; ++pass) {
    of_tile = 0.0;
    for (uint32_t tile = tile0; tile < tile1; ++tile) {
      double m[8], sum = 0.0;
      if (pass) masses(tile * kVerifyTile + lane * 8, m);
      else masses.whole(tile * kVerifyTile + lane * 8, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += m[i];
      sum = warp_sum_f64(sum);
      if (lane == tile - tile0) of_tile = sum;
    }
    const double total = warp_sum_f64(of_tile);
    if (lane == 0) warp_total[warp] = total;
    cluster_sync();
    if (tid < kVerifyWarps) region[tid] = lds_f64_cluster(cluster_map(smem_u32(&warp_total[tid & 7u]), tid >> 3));
    cluster_sync();                                 // all shares have been read: the next pass may write its own
    r0 = region[2 * lane];
    r1 = region[2 * lane + 1];
    upto_region = warp_scan_f64(r0 + r1, lane);
    if (!pass) masses.total = __shfl_sync(0xFFFFFFFFu, upto_region, 31);
  }
  // the region (a warp's tiles), the tile, the lane and the token where the running mass passes the target; rounding that
  // leaves no such place falls back to the last one with any mass
  const double whole = __shfl_sync(0xFFFFFFFFu, upto_region, 31), target = double(a.u_draw[seq]) * whole;
  if (!(whole > 0.0)) {                             // nothing left to draw from (a drafted token of probability 1 that was refused)
    if (blockIdx.x == 0 && tid == 0) out_tokens[count - 1] = refused;
    return;
  }
  const double from_region = upto_region - r1 - r0, half_region = upto_region - r1;
  const uint32_t past0 = __ballot_sync(0xFFFFFFFFu, r0 > 0.0 && half_region > target), past1 = __ballot_sync(0xFFFFFFFFu, r1 > 0.0 && upto_region > target);
  const uint32_t with0 = __ballot_sync(0xFFFFFFFFu, r0 > 0.0), with1 = __ballot_sync(0xFFFFFFFFu, r1 > 0.0);
  uint32_t chosen;
  if (past0 | past1) {
    const uint32_t l = __ffs(past0 | past1) - 1;
    chosen = 2 * l + (past0 >> l & 1u ? 0u : 1u);
  } else {
    const uint32_t l = 31 - __clz(with0 | with1);
    chosen = 2 * l + (with1 >> l & 1u);
  }
  if (chosen != unit) return;
  const double before = __shfl_sync(0xFFFFFFFFu, chosen & 1u ? half_region : from_region, chosen >> 1);
  const double upto_tile = before + warp_scan_f64(of_tile, lane);
  const uint32_t with_tile = __ballot_sync(0xFFFFFFFFu, of_tile > 0.0), past_tile = __ballot_sync(0xFFFFFFFFu, of_tile > 0.0 && upto_tile > target);
  const uint32_t pick = past_tile ? uint32_t(__ffs(past_tile)) - 1u : 31u - __clz(with_tile);
  const double before_tile = __shfl_sync(0xFFFFFFFFu, upto_tile - of_tile, pick);
  const uint32_t t0 = (tile0 + pick) * kVerifyTile + lane * 8;
  double m[8], sum = 0.0;
  masses(t0, m);
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += m[i];
  const double upto = before_tile + warp_scan_f64(sum, lane);
  const uint32_t with = __ballot_sync(0xFFFFFFFFu, sum > 0.0), past = __ballot_sync(0xFFFFFFFFu, sum > 0.0 && upto > target);
  const uint32_t owner = past ? uint32_t(__ffs(past)) - 1u : 31u - __clz(with);
  if (lane == owner) {
    double run = upto - sum;
    uint32_t t = t0;
    for (int i = 0; i < 8; ++i) {
      run += m[i];
      if (m[i] > 0.0) {
        t = t0 + i;
        if (run > target) break;
      }
    }
    out_tokens[count - 1] = int32_t(t);
  }
}

}  // namespace grb
