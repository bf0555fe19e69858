// extern "C" entry points of rotary positions and of the pages of a KV cache: argument validation and launch geometry.
// No allocation and no host synchronisation happen here; errors are returned, never thrown.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/georefine_b200.h"
#include "kv_arguments.h"
#include "kv_pages.cuh"
#include "launch_utils.h"
#include "rotary.cuh"

namespace {

using namespace grb;

// So many CTAs, or as many as stay resident.
uint32_t copy_ctas(uint64_t ctas) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  return uint32_t(std::min<uint64_t>(ctas, uint64_t(std::max(device_sm_count(dev), 0)) * 4));
}
uint64_t parts_of(const KvPagesArgs& p) { return 2ull * p.layers * p.nkv; }

template <class Args>
int launch_copies(void (*bf16)(Args), void (*e4m3)(Args), void (*q4)(Args), uint32_t format, uint32_t ctas, cudaStream_t stream, const Args& a) {
  if (!ctas) return GRB_ERR_CUDA;
  return launch_step(format == GRB_KV_Q4 ? q4 : format == GRB_KV_E4M3 ? e4m3 : bf16, dim3(ctas), dim3(kPageThreads), 0, stream, a);
}
constexpr uint32_t kWarps = kPageThreads / 32;
int copies(uint32_t format, uint64_t pieces, cudaStream_t stream, const KvCopyArgs& a) {
  return launch_copies(kv_copy_kernel<kKvBf16>, kv_copy_kernel<kKvE4m3>, kv_copy_kernel<kKvQ4>, format, copy_ctas((pieces + kWarps - 1) / kWarps), stream, a);
}
// A table that a call writes to.
int own_table_of(const grb_kv_table* t) {
  if (!t || !t->table || !t->slots || !t->max_pages || t->ld < int64_t(t->max_pages)) return GRB_ERR_ARGUMENT;
  return t->max_pages > 0x7FFFFFu || t->slots > 0x7FFFFFFFu ? GRB_ERR_UNSUPPORTED : GRB_OK;
}
// What whole pages are copied in: pieces of 16 bytes, numbered in 31 bits.  (What goes by entries moves exponents byte by byte, and takes layers of
// them that lie any distance apart.)
int copied_pages_of(const grb_kv_pages* pages, KvPagesArgs& a) {
  if (int st = pages_of(pages, a)) return st;
  if (pages->format == GRB_KV_E4M3 && pages->layers > 1 && (pages->exp_stride & 15)) return GRB_ERR_ARGUMENT;
  return parts_of(a) <= 0x7FFFFFFFull ? GRB_OK : GRB_ERR_UNSUPPORTED;
}

template <class T, int V, bool HALF>
int rotary_launch(RotaryArgs a, bool copy, cudaStream_t stream) {
  a.items = a.turned / 2 / (HALF || V == 1 ? V : V / 2) + (copy ? (a.dim - a.turned) / V : 0);
  a.groups = (a.heads + kRotaryHeads - 1) / kRotaryHeads;
  a.groups_per_cta = kRotaryThreads / std::min<uint32_t>(a.items, kRotaryThreads);
  const uint64_t ctas = (uint64_t(a.rows) * a.groups + a.groups_per_cta - 1) / a.groups_per_cta;
  if (ctas > 0x7FFFFFFFull) return GRB_ERR_UNSUPPORTED;
  return launch_step(rotary_kernel<T, V, HALF>, dim3(uint32_t(ctas)), dim3(kRotaryThreads), 0, stream, a);
}
template <class T, bool HALF>
int rotary_width(const RotaryArgs& a, bool copy, cudaStream_t stream) {
  // the widest pieces that everything is a multiple of: sizes, distances and addresses
  constexpr int kWide = 16 / int(sizeof(T));
  const uint64_t sizes = uint64_t(HALF ? a.turned / 2 : a.turned) | (copy ? a.dim - a.turned : 0u) | uint64_t(a.ldx) | uint64_t(a.ldo) | (a.heads > 1 ? uint64_t(a.ldxh) | uint64_t(a.ldoh) : 0ull) |
                         (copy ? a.turned : 0u);
  const uint64_t bytes = sizes * sizeof(T) | reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.out);
  if (bytes % 16 == 0) return rotary_launch<T, kWide, HALF>(a, copy, stream);
  if (bytes % (2 * sizeof(T)) == 0) return rotary_launch<T, 2, HALF>(a, copy, stream);
  return rotary_launch<T, 1, HALF>(a, copy, stream);
}

}  // namespace

extern "C" {

int grb_rotary(const grb_rotary_step* s, void* cuda_stream) {
  if (!s || !s->x || !s->out || !s->positions || !s->turns) return GRB_ERR_ARGUMENT;
  if (s->dtype > GRB_ROTARY_FP16 || s->layout > 1 || s->positions_64 > 1 || s->backward > 1) return GRB_ERR_ARGUMENT;
  if (!s->heads || !s->turned || (s->turned & 1) || s->turned > s->dim) return GRB_ERR_ARGUMENT;
  if (s->dim > kRotaryMaxDim || s->heads > 65535) return GRB_ERR_UNSUPPORTED;
  const uint32_t size = s->dtype == GRB_ROTARY_FP32 ? 4 : 2;
  if (s->rows > 0x7FFFFFFFu || (reinterpret_cast<uintptr_t>(s->x) % size) || (reinterpret_cast<uintptr_t>(s->out) % size) || (reinterpret_cast<uintptr_t>(s->turns) & 7) ||
      (reinterpret_cast<uintptr_t>(s->positions) & (s->positions_64 ? 7 : 3)))
    return GRB_ERR_ARGUMENT;
  // heads and rows of the result may not overlap: heads within a row, or rows within a head's distance
  const auto apart = [&](int64_t row, int64_t head) {
    const int64_t heads = head * int64_t(s->heads - 1) + s->dim, rows = row * (int64_t(s->rows) - 1) + s->dim;
    return (s->heads == 1 || head >= int64_t(s->dim)) && (s->rows <= 1 || row >= heads || (s->heads > 1 && row >= int64_t(s->dim) && head >= rows));
  };
  if (s->ldx < 0 || s->ldx_head < 0 || !apart(s->ldo, s->ldo_head)) return GRB_ERR_ARGUMENT;
  // (in place: where it lies)
  if (s->x == s->out && ((s->rows > 1 && s->ldx != s->ldo) || (s->rows && s->heads > 1 && s->ldx_head != s->ldo_head))) return GRB_ERR_ARGUMENT;
  if (!s->rows) return GRB_OK;
  RotaryArgs a{};
  a.x = s->x;
  a.out = s->out;
  a.ldx = s->ldx;
  a.ldxh = s->ldx_head;
  a.ldo = s->ldo;
  a.ldoh = s->ldo_head;
  a.positions = s->positions;
  a.turns = s->turns;
  a.factor = s->factor;
  a.rows = s->rows;
  a.heads = s->heads;
  a.dim = s->dim;
  a.turned = s->turned;
  a.wide_positions = s->positions_64;
  a.backward = s->backward;
  const bool copy = s->x != s->out && s->turned < s->dim;
  const auto stream = static_cast<cudaStream_t>(cuda_stream);
  if (s->layout == GRB_ROTARY_HALF)
    return s->dtype == GRB_ROTARY_FP32 ? rotary_width<float, true>(a, copy, stream) : s->dtype == GRB_ROTARY_FP16 ? rotary_width<__half, true>(a, copy, stream) : rotary_width<__nv_bfloat16, true>(a, copy, stream);
  return s->dtype == GRB_ROTARY_FP32 ? rotary_width<float, false>(a, copy, stream) : s->dtype == GRB_ROTARY_FP16 ? rotary_width<__half, false>(a, copy, stream) : rotary_width<__nv_bfloat16, false>(a, copy, stream);
}

int grb_kv_copy(const grb_kv_pages* pages, const int32_t* src, const int32_t* dst, const int32_t* positions, uint32_t n, void* cuda_stream) {
  KvCopyArgs a{};
  if (int st = copied_pages_of(pages, a.pages)) return st;
  if (!src || !dst) return GRB_ERR_ARGUMENT;
  if (!n) return GRB_OK;
  a.src = src;
  a.dst = dst;
  a.positions = positions;
  a.n = n;
  return copies(pages->format, n * parts_of(a.pages), static_cast<cudaStream_t>(cuda_stream), a);
}

int grb_kv_fork(const grb_kv_pages* pages, const grb_kv_table* table, const int32_t* parents, const int32_t* children, const int32_t* lengths, const int32_t* fresh,
                int32_t* refs, int32_t empty, uint32_t n, void* cuda_stream) {
  KvForkArgs a{};
  if (int st = copied_pages_of(pages, a.pages)) return st;
  if (int st = own_table_of(table)) return st;
  if (!parents || !children || !lengths || !fresh || !refs) return GRB_ERR_ARGUMENT;
  if (!n) return GRB_OK;
  a.table = const_cast<int32_t*>(table->table);
  a.ld = table->ld;
  a.slots = table->slots;
  a.max_pages = table->max_pages;
  a.parents = parents;
  a.children = children;
  a.lengths = lengths;
  a.fresh = fresh;
  a.refs = refs;
  a.empty = empty;
  a.n = n;
  // CTAs of a fork: as many as there are pieces for their warps, and as stay resident together
  const uint64_t most = (parts_of(a.pages) + kWarps - 1) / kWarps, slices = std::max<uint64_t>(1, std::min<uint64_t>(most, copy_ctas(~0ull) / n));
  if (n * slices > 0x7FFFFFFFull) return GRB_ERR_UNSUPPORTED;
  return launch_copies(kv_fork_kernel<kKvBf16>, kv_fork_kernel<kKvE4m3>, kv_fork_kernel<kKvQ4>, pages->format, uint32_t(n * slices), static_cast<cudaStream_t>(cuda_stream), a);
}

int grb_kv_free(const grb_kv_table* table, const int32_t* slots, int32_t* refs, uint32_t pages, int32_t empty, uint32_t n, void* cuda_stream) {
  if (int st = own_table_of(table)) return st;
  if (!slots || !refs || !pages) return GRB_ERR_ARGUMENT;
  if (!n) return GRB_OK;
  const KvFreeArgs a{const_cast<int32_t*>(table->table), table->ld, table->slots, table->max_pages, slots, refs, pages, n, empty};
  const uint32_t ctas = copy_ctas((uint64_t(n) * table->max_pages + kPageThreads - 1) / kPageThreads);
  if (!ctas) return GRB_ERR_CUDA;
  return launch_step(kv_free_kernel, dim3(ctas), dim3(kPageThreads), 0, static_cast<cudaStream_t>(cuda_stream), a);
}

uint64_t grb_kv_compact_scratch_bytes(uint32_t pages) { return 16 + uint64_t(pages) * 8; }

int grb_kv_compact(const grb_kv_pages* pages, const grb_kv_table* table, int32_t* refs, int32_t* where, int32_t* used, void* scratch, uint64_t scratch_bytes, void* cuda_stream) {
  KvCopyArgs moves{};
  if (int st = copied_pages_of(pages, moves.pages)) return st;
  if (int st = own_table_of(table)) return st;
  if (!refs || !where || !used || !scratch || !aligned16(scratch)) return GRB_ERR_ARGUMENT;
  if (scratch_bytes < grb_kv_compact_scratch_bytes(pages->pages)) return GRB_ERR_WORKSPACE;
  KvCompactArgs a{const_cast<int32_t*>(table->table), table->ld, table->slots, table->max_pages, pages->pages, refs, where, used, static_cast<int32_t*>(scratch), nullptr, nullptr};
  a.src = a.moves + 4;
  a.dst = a.src + pages->pages;
  const auto stream = static_cast<cudaStream_t>(cuda_stream);
  if (int st = launch_step(kv_compact_plan_kernel, dim3(1), dim3(kCompactThreads), 0, stream, a)) return st;
  moves.src = a.src;
  moves.dst = a.dst;
  moves.moves = a.moves;
  moves.n = pages->pages;
  if (int st = copies(pages->format, moves.n * parts_of(moves.pages), stream, moves)) return st;
  const uint32_t ctas = copy_ctas((std::max(uint64_t(table->slots) * table->max_pages, uint64_t(pages->pages)) + kPageThreads - 1) / kPageThreads);
  if (!ctas) return GRB_ERR_CUDA;
  return launch_step(kv_compact_table_kernel, dim3(ctas), dim3(kPageThreads), 0, stream, a);
}

}  // extern "C"
