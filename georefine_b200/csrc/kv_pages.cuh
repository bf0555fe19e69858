// Pages of a paged KV cache as a whole: copied, shared between sequences that begin alike, given back, and moved together.
//
// Whose a page is says the page table alone: refs[p] counts the table's places that name page p.  A fork of a sequence of n positions
// names the parent's n / 256 whole pages too (nothing is stored to them any more) and gets a page of its own for the n % 256 positions
// behind them, copied in every layer.  Compacting moves the pages in use to the front of the pool: with u in use, the i-th of them at u or behind goes
// to the i-th free one before u, so every page moves once at most and nothing moves onto a page that is still to be read.
//
// Memory bounds the copies.  A piece of work is one head's part of one page in one plane (a layer's keys or values), whose bytes lie together; warps take the
// pieces, eight loads of 16 bytes a lane on their way.  Forks of one parent run side by side, so that its bytes come from L2 after the first: what bounds
// them is the stores.  64 forks in 64 layers, 400 MB written: 106 us, at the 3.8 TB/s that a fill reaches (a CTA a piece, which looks up where the piece lies
// before its first byte can move: 204).  941 MB read and written by a compaction: 156 us, 6.0 TB/s.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_cache.cuh"

namespace grb {

constexpr int kPageThreads = 256;

// The first `count` positions of one head's part of a page of plane p (keys, even, or values of layer p / 2).  Whole warp.  Codes, scales and exponents are one
// row of 16-byte pieces, so that their loads are on their way together; what is left of a piece goes by words and bytes.
template <int FORMAT>
__device__ __forceinline__ void kv_copy_head(const KvPagesArgs& a, uint32_t p, uint32_t head, uint32_t from, uint32_t to, uint32_t count, uint32_t lane) {
  constexpr uint32_t kEntry = FORMAT == kKvQ4 ? kQ4Codes : FORMAT == kKvE4m3 ? kKvDim : 2 * kKvDim, kBlock = FORMAT == kKvQ4 ? kQ4Page : kEntry * kKvPage;
  uint8_t* const plane = static_cast<uint8_t*>(p & 1u ? a.v : a.k) + int64_t(p >> 1) * a.layer_stride * (FORMAT == kKvBf16 ? 2 : 1);
  const size_t from_block = size_t(from) * a.nkv + head, to_block = size_t(to) * a.nkv + head;
  const uint8_t* const src = plane + from_block * kBlock;
  uint8_t* const dst = plane + to_block * kBlock;
  // where scales and exponents lie behind (or beside) the codes
  uint8_t* const exp_plane = FORMAT == kKvE4m3 ? (p & 1u ? a.v_exp : a.k_exp) + int64_t(p >> 1) * a.exp_stride : nullptr;
  const uint8_t* const src_exp = FORMAT == kKvE4m3 ? exp_plane + from_block * kKvPage : src + kQ4ExpsAt;
  uint8_t* const dst_exp = FORMAT == kKvE4m3 ? exp_plane + to_block * kKvPage : dst + kQ4ExpsAt;
  const uint32_t codes = count * kEntry / 16, scales = FORMAT == kKvQ4 ? count / 4 : 0u, exps = FORMAT == kKvBf16 ? 0u : count / 16, pieces = codes + scales + exps;
  const uint32_t words = FORMAT == kKvQ4 ? count % 4 : 0u, bytes = FORMAT == kKvBf16 ? 0u : count % 16;
  uint32_t word = 0, byte = 0;
  if (lane < words) word = reinterpret_cast<const uint32_t*>(src + kQ4ScalesAt)[scales * 4 + lane];
  if (lane < bytes) byte = src_exp[exps * 16 + lane];
  constexpr uint32_t kAtOnce = 8;
  for (uint32_t i0 = lane; i0 < pieces; i0 += kAtOnce * 32) {
    uint4 x[kAtOnce];
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) {
      const uint32_t n = i0 + i * 32;
      if (n < pieces) x[i] = n < codes ? reinterpret_cast<const uint4*>(src)[n] : n < codes + scales ? reinterpret_cast<const uint4*>(src + kQ4ScalesAt)[n - codes]
                                                                                                    : reinterpret_cast<const uint4*>(src_exp)[n - codes - scales];
    }
#pragma unroll
    for (uint32_t i = 0; i < kAtOnce; ++i) {
      const uint32_t n = i0 + i * 32;
      if (n < pieces) (n < codes ? reinterpret_cast<uint4*>(dst)[n] : n < codes + scales ? reinterpret_cast<uint4*>(dst + kQ4ScalesAt)[n - codes]
                                                                                        : reinterpret_cast<uint4*>(dst_exp)[n - codes - scales]) = x[i];
    }
  }
  if (lane < words) reinterpret_cast<uint32_t*>(dst + kQ4ScalesAt)[scales * 4 + lane] = word;
  if (lane < bytes) dst_exp[exps * 16 + lane] = uint8_t(byte);
}

struct KvCopyArgs {
  KvPagesArgs pages;
  const int32_t* src;       // [n]; a page outside the pool, or one onto itself: left out
  const int32_t* dst;
  const int32_t* positions; // [n]: of each page, from its first on; null: all
  const int32_t* moves;     // null, or how many of the n there are
  uint32_t n;
};

template <int FORMAT>
__global__ void __launch_bounds__(kPageThreads, 4)
kv_copy_kernel(const KvCopyArgs a) {
  step_kernel_entry();
  const uint32_t n = a.moves ? min(uint32_t(max(*a.moves, 0)), a.n) : a.n, parts = 2 * a.pages.layers * a.pages.nkv;
  const uint64_t warps = uint64_t(gridDim.x) * (kPageThreads / 32);
  for (uint64_t item = uint64_t(blockIdx.x) * (kPageThreads / 32) + (threadIdx.x >> 5); item < uint64_t(n) * parts; item += warps) {
    const uint32_t part = uint32_t(item / n), i = uint32_t(item - uint64_t(part) * n);
    const uint32_t from = uint32_t(a.src[i]), to = uint32_t(a.dst[i]);
    if (from >= a.pages.pages || to >= a.pages.pages || from == to) continue;
    const int32_t count = a.positions ? min(max(a.positions[i], 0), int32_t(kKvPage)) : int32_t(kKvPage);
    kv_copy_head<FORMAT>(a.pages, part / a.pages.nkv, part % a.pages.nkv, from, to, uint32_t(count), threadIdx.x & 31u);
  }
}

struct KvForkArgs {
  KvPagesArgs pages;
  int32_t* table;           // [slots][ld]
  int64_t ld;
  uint32_t slots, max_pages;
  const int32_t* parents;   // [n]: slots
  const int32_t* children;  // [n]
  const int32_t* lengths;   // [n]: positions of the parent that the child begins with
  const int32_t* fresh;     // [n]: a page for those behind the last whole one
  int32_t* refs;            // [pages]
  int32_t empty;            // what a place without a page holds
  uint32_t n;
};

template <int FORMAT>
__global__ void __launch_bounds__(kPageThreads, 4)
kv_fork_kernel(const KvForkArgs a) {
  step_kernel_entry();
  // a CTA is one fork's: where it lies is looked up once for all of the CTA's pieces
  const uint32_t parts = 2 * a.pages.layers * a.pages.nkv, i = blockIdx.x % a.n, slice = blockIdx.x / a.n, slices = gridDim.x / a.n;
  const uint32_t parent = uint32_t(a.parents[i]), child = uint32_t(a.children[i]), length = uint32_t(a.lengths[i]);
  // a fork that names what is not there is left out
  if (parent >= a.slots || child >= a.slots || parent == child || length > a.max_pages * kKvPage) return;
  const int32_t* const from = a.table + parent * a.ld;
  const uint32_t whole = length / kKvPage, rest = length % kKvPage;
  const uint32_t fresh = rest ? uint32_t(a.fresh[i]) : 0xFFFFFFFFu, source = rest ? uint32_t(from[whole]) : 0xFFFFFFFFu;
  if (slice == 0) {
    int32_t* const to = a.table + child * a.ld;
    for (uint32_t p = threadIdx.x; p < a.max_pages; p += kPageThreads) {
      const int32_t page = p < whole ? from[p] : p == whole && fresh < a.pages.pages ? int32_t(fresh) : a.empty;
      to[p] = page;
      if (page != a.empty && uint32_t(page) < a.pages.pages) atomicAdd(a.refs + page, 1);
    }
  }
  if (fresh >= a.pages.pages || source >= a.pages.pages || source == fresh) return;
  for (uint32_t part = slice * (kPageThreads / 32) + (threadIdx.x >> 5); part < parts; part += slices * (kPageThreads / 32))
    kv_copy_head<FORMAT>(a.pages, part / a.pages.nkv, part % a.pages.nkv, source, fresh, rest, threadIdx.x & 31u);
}

// A slot's pages counted down and its places emptied.  (An exchange: a slot named twice gives its pages back once.)
struct KvFreeArgs {
  int32_t* table;
  int64_t ld;
  uint32_t slots, max_pages;
  const int32_t* which;     // [n]: slots; -1: left out
  int32_t* refs;
  uint32_t pages, n;
  int32_t empty;
};
__global__ void __launch_bounds__(kPageThreads, 4)
kv_free_kernel(const KvFreeArgs a) {
  step_kernel_entry();
  const uint64_t places = uint64_t(a.n) * a.max_pages;
  for (uint64_t i = uint64_t(blockIdx.x) * kPageThreads + threadIdx.x; i < places; i += uint64_t(gridDim.x) * kPageThreads) {
    const uint32_t slot = uint32_t(a.which[i / a.max_pages]);
    if (slot >= a.slots) continue;
    const int32_t page = atomicExch(a.table + slot * a.ld + i % a.max_pages, a.empty);
    if (page != a.empty && uint32_t(page) < a.pages) atomicSub(a.refs + page, 1);
  }
}

// The plan of a compaction, by one CTA: where each page goes, and the moves in order.
struct KvCompactArgs {
  int32_t* table;
  int64_t ld;
  uint32_t slots, max_pages, pages;
  int32_t* refs;
  int32_t* where;           // [pages]: a page's new number; -1: it is not in use
  int32_t* used;            // pages in use
  int32_t* moves;           // scratch: how many
  int32_t* src;             // scratch: [pages]
  int32_t* dst;
};
constexpr int kCompactThreads = 1024;
__global__ void __launch_bounds__(kCompactThreads)
kv_compact_plan_kernel(const KvCompactArgs a) {
  step_kernel_entry();
  __shared__ uint32_t sums[2][kCompactThreads / 32];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  uint32_t mine = 0;
  for (uint32_t p = tid; p < a.pages; p += kCompactThreads) mine += a.refs[p] > 0;
  mine = __reduce_add_sync(0xFFFFFFFFu, mine);
  if (lane == 0) sums[0][warp] = mine;
  __syncthreads();
  const uint32_t used = __reduce_add_sync(0xFFFFFFFFu, sums[0][lane]);
  uint32_t sources = 0, targets = 0;                         // before the pages at hand
  for (uint32_t lo = 0; lo < a.pages; lo += kCompactThreads) {
    const uint32_t p = lo + tid;
    const bool in = p < a.pages, held = in && a.refs[p] > 0, source = held && p >= used, target = in && !held && p < used;
    const uint32_t s = __ballot_sync(0xFFFFFFFFu, source), t = __ballot_sync(0xFFFFFFFFu, target);
    __syncthreads();                                         // (the sums before have been read)
    if (lane == 0) { sums[0][warp] = __popc(s); sums[1][warp] = __popc(t); }
    __syncthreads();
    const uint32_t below = (1u << lane) - 1u;
    const uint32_t s_before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sums[0][lane] : 0u), t_before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sums[1][lane] : 0u);
    if (source) a.src[sources + s_before + __popc(s & below)] = int32_t(p);
    if (target) a.dst[targets + t_before + __popc(t & below)] = int32_t(p);
    if (in) a.where[p] = held ? int32_t(p) : -1;
    sources += __reduce_add_sync(0xFFFFFFFFu, sums[0][lane]);
    targets += __reduce_add_sync(0xFFFFFFFFu, sums[1][lane]);
  }
  __syncthreads();                                           // (there are as many pages to move as free ones before `used`)
  for (uint32_t i = tid; i < sources; i += kCompactThreads) a.where[a.src[i]] = a.dst[i];
  if (tid == 0) { *a.used = int32_t(used); *a.moves = int32_t(sources); }
}
// Behind the copies: the table names the new places, and the counts go along.
__global__ void __launch_bounds__(kPageThreads, 4)
kv_compact_table_kernel(const KvCompactArgs a) {
  step_kernel_entry();
  const uint64_t places = uint64_t(a.slots) * a.max_pages, stride = uint64_t(gridDim.x) * kPageThreads, first = uint64_t(blockIdx.x) * kPageThreads + threadIdx.x;
  for (uint64_t i = first; i < places; i += stride) {
    int32_t* const place = a.table + i / a.max_pages * a.ld + i % a.max_pages;
    const uint32_t page = uint32_t(*place);
    if (page < a.pages && a.where[page] >= 0) *place = a.where[page];
  }
  const uint64_t moves = uint64_t(*a.moves);
  for (uint64_t i = first; i < moves; i += stride) {
    a.refs[a.dst[i]] = a.refs[a.src[i]];
    a.refs[a.src[i]] = 0;
  }
}

}  // namespace grb
