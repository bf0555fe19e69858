// extern "C" entry points of serving over a paged KV cache in BF16, 8 or 4 bits, and of speculation: argument validation and launch geometry.
// No allocation and no host synchronisation happen here; errors are returned, never thrown.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "../../include/georefine_b200.h"
#include "kv_arguments.h"
#include "kv_cache.cuh"
#include "launch_utils.h"
#include "tree_attention.cuh"
#include "tree_pair.cuh"
#include "tree_q4.cuh"
#include "tree_wide.cuh"
#include "verify_ops.cuh"

namespace {

using namespace grb;

template <bool READ>
int kv_rows(const grb_kv_pages* pages, const grb_kv_table* table, const int32_t* row_seq, const int32_t* row_pos, void* k, int64_t ldk, void* v,
            int64_t ldv, uint32_t rows, void* stream) {
  KvRowsArgs a{};
  if (int st = pages_of(pages, a.pages)) return st;
  if (int st = table_of(table, a.pages, a.table)) return st;
  const int64_t width = int64_t(a.pages.nkv) * kKvDim;
  if (!row_seq || !row_pos || !k || !v || ldk < width || ldv < width || (ldk & 7) || (ldv & 7) || !aligned16(k) || !aligned16(v)) return GRB_ERR_ARGUMENT;
  if (!rows) return GRB_OK;
  a.row_seq = row_seq;
  a.row_pos = row_pos;
  a.k = static_cast<__nv_bfloat16*>(k);
  a.v = static_cast<__nv_bfloat16*>(v);
  a.ldk = ldk;
  a.ldv = ldv;
  a.rows = rows;
  const uint32_t entries = pages->format == GRB_KV_Q4 ? kQ4EntriesPerWarp : kKvEntriesPerWarp;
  const uint64_t warps = uint64_t(rows) * ((2 * a.pages.nkv + entries - 1) / entries), ctas = (warps + kKvWarps - 1) / kKvWarps;
  if (warps > 0xFFFFFF00ull) return GRB_ERR_UNSUPPORTED;   // (numbered in 32 bits)
  const auto kernel = pages->format == GRB_KV_E4M3 ? kv_rows_kernel<READ, kKvE4m3> : pages->format == GRB_KV_Q4 ? kv_rows_q4_kernel<READ> : kv_rows_kernel<READ, kKvBf16>;
  return launch_step(kernel, dim3(uint32_t(ctas)), dim3(kKvWarps * 32), 0, static_cast<cudaStream_t>(stream), a);
}

// Positions of a part of the narrow kernels.
constexpr uint32_t part_positions(uint32_t format) {
  return format == GRB_KV_Q4 ? TreeQ4::kPositions : format == GRB_KV_E4M3 ? TreePart<true>::kPositions : TreePart<false>::kPositions;
}
uint64_t parts_of(uint32_t max_pages, uint32_t format) { return (uint64_t(max_pages) * kKvPage + part_positions(format) - 1) / part_positions(format); }

template <int FORMAT>
int tree_launch(const TreeArgs& a, cudaStream_t stream) {
  constexpr bool F8 = FORMAT != kKvBf16;
  using P = std::conditional_t<FORMAT == kKvQ4, TreeQ4, TreePart<F8>>;
  void (*part)(TreeArgs);
  int resident = 3;                                          // CTAs an SM
  if constexpr (FORMAT == kKvQ4) {
    const bool one = a.tile_rows * a.group <= 8;
    part = one ? tree_q4_kernel<1> : tree_q4_kernel<2>;
    resident = one ? 4 : 3;
  } else {
    part = tree_part_kernel<F8>;
  }
  void (*wide)(TreeArgs);
  uint32_t wide_smem, wide_threads, wide_resident;
  if constexpr (FORMAT == kKvQ4) {
    wide = tree_pair_kernel;
    wide_smem = kPairSmem;
    wide_threads = kPairThreads;
    wide_resident = 1;
  } else {
    wide = tree_wide_kernel<F8>;
    wide_smem = kWideSmem<F8>;
    wide_threads = kWideThreads;
    wide_resident = 2;
  }
  static std::once_flag once[64];
  static int prepared[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return GRB_ERR_CUDA;
  std::call_once(once[dev], [&] {
    if constexpr (FORMAT == kKvQ4) {
      for (auto kernel : {tree_q4_kernel<1>, tree_q4_kernel<2>})
        if (!prepared[dev]) prepared[dev] = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::kSmem)));
    } else {
      prepared[dev] = cuda_status(cudaFuncSetAttribute(part, cudaFuncAttributeMaxDynamicSharedMemorySize, int(P::kSmem)));
    }
    if (!prepared[dev]) prepared[dev] = cuda_status(cudaFuncSetAttribute(wide, cudaFuncAttributeMaxDynamicSharedMemorySize, int(wide_smem)));
  });
  if (prepared[dev]) return prepared[dev];
  const int sms = device_sm_count(dev);
  if (sms <= 0) return GRB_ERR_CUDA;
  const uint32_t warps = a.rows * ((a.nq + 2 * a.nkv + kTreeHeadsPerWarp - 1) / kTreeHeadsPerWarp);
  const uint32_t threads = a.rows > kTreePrepThreads ? kTreePrepMost : kTreePrepThreads;
  if (int st = launch_step(tree_prep_kernel<FORMAT>, dim3((warps + threads / 32 - 1) / (threads / 32) + 1), dim3(threads), a.rows * 6, stream, a, P::kPositions)) return st;
  const uint64_t units = uint64_t(a.rows) * a.max_parts * a.nkv;      // at most
  if (int st = launch_step(part, dim3(uint32_t(std::min<uint64_t>(units, uint64_t(sms) * resident))), dim3(P::kThreads), P::kSmem, stream, a)) return st;
  if (a.wide_from) {
    if (int st = launch_step(wide, dim3(uint32_t(std::min<uint64_t>(units, uint64_t(sms) * wide_resident))), dim3(wide_threads), wide_smem, stream, a)) return st;
  }
  const uint64_t pairs = uint64_t(a.rows) * a.nq;
  return launch_step(tree_combine_kernel, dim3(uint32_t((pairs + kTreeCombineWarps - 1) / kTreeCombineWarps)), dim3(kTreeCombineWarps * 32), 0, stream, a);
}

template <class... Params>
int launch_clusters(void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t smem, uint32_t cluster, cudaStream_t stream, Params... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, args...));
}

template <bool F32, bool VEC>
int verify_launch(const VerifyArgs& a, cudaStream_t stream) {
  if (int st = launch_step(verify_rows_kernel<F32, VEC>, dim3(kVerifySlices, a.rows), dim3(kVerifyThreads), 0, stream, a)) return st;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return GRB_ERR_CUDA;
  const uint32_t resident = 2 * uint32_t(device_sm_count(dev)), cluster = a.seqs * 8 <= resident ? 8 : a.seqs * 4 <= resident ? 4 : 2;
  return launch_clusters(verify_draw_kernel<F32, VEC>, dim3(cluster, a.seqs), kVerifyDrawThreads, (a.vocab + 255) / 256 * 4, cluster, stream, a);
}

}  // namespace

extern "C" {

int grb_kv_write(const grb_kv_pages* pages, const grb_kv_table* table, const int32_t* row_seq, const int32_t* row_pos, const void* k, int64_t ldk,
                 const void* v, int64_t ldv, uint32_t rows, void* cuda_stream) {
  return kv_rows<false>(pages, table, row_seq, row_pos, const_cast<void*>(k), ldk, const_cast<void*>(v), ldv, rows, cuda_stream);
}

int grb_kv_read(const grb_kv_pages* pages, const grb_kv_table* table, const int32_t* row_seq, const int32_t* row_pos, void* k, int64_t ldk, void* v,
                int64_t ldv, uint32_t rows, void* cuda_stream) {
  return kv_rows<true>(pages, table, row_seq, row_pos, k, ldk, v, ldv, rows, cuda_stream);
}

int grb_kv_keep(const grb_kv_pages* pages, const grb_kv_table* table, const int32_t* seqs, const int32_t* base, const int32_t* path, int64_t ldp,
                const int32_t* count, uint32_t n, uint32_t width, void* cuda_stream) {
  KvKeepArgs a{};
  if (int st = pages_of(pages, a.pages)) return st;
  if (int st = table_of(table, a.pages, a.table)) return st;
  if (!seqs || !base || !path || !count || ldp < int64_t(width)) return GRB_ERR_ARGUMENT;
  if (!n || width < 2) return GRB_OK;       // nothing lies behind a root
  if (n > 65535 || a.pages.layers > 0x3FFFFFFFu) return GRB_ERR_UNSUPPORTED;
  a.seqs = seqs;
  a.base = base;
  a.path = path;
  a.count = count;
  a.ldp = ldp;
  a.width = width;
  const auto kernel = pages->format == GRB_KV_E4M3 ? kv_keep_kernel<kKvE4m3> : pages->format == GRB_KV_Q4 ? kv_keep_kernel<kKvQ4> : kv_keep_kernel<kKvBf16>;
  return launch_step(kernel, dim3((a.pages.layers * 2 + kKeepPlanes - 1) / kKeepPlanes, n), dim3(kKeepThreads), 0, static_cast<cudaStream_t>(cuda_stream), a);
}

uint64_t grb_attn_tree_scratch_bytes(uint32_t rows, uint32_t nq, uint32_t max_pages, uint32_t format) {
  if (!rows || rows > kTreeMaxRows || !nq || !max_pages || (format > GRB_KV_E4M3 && format != GRB_KV_Q4)) return 0;
  const uint64_t parts = parts_of(max_pages, format);
  const uint64_t pairs = uint64_t(rows) * nq;
  return ((48 + rows * 40ull + pairs * 4 + 255) & ~uint64_t(255)) + pairs * kKvDim * (format == GRB_KV_BF16 ? 4 : 2) + 16 + pairs * parts * (kKvDim * 4 + 8);
}

int grb_attn_tree(const grb_attn_tree_step* s, void* cuda_stream) {
  if (!s || !s->qkv || !s->cos_table || !s->sin_table || !s->row_seq || !s->row_pos || !s->scratch || !s->out) return GRB_ERR_ARGUMENT;
  TreeArgs a{};
  if (int st = pages_of(&s->pages, a.pages)) return st;
  if (int st = table_of(&s->table, a.pages, a.table)) return st;
  a.nkv = s->pages.nkv;
  a.nq = s->nq;
  if (!s->nq || s->nq % a.nkv || s->head_dim != kKvDim || !s->rope_rows || !(s->scaling > 0.f) || s->scaling > 1e30f) return GRB_ERR_ARGUMENT;
  a.group = a.nq / a.nkv;
  if (a.group > 16 || s->rows > kTreeMaxRows || s->nq + 2 * a.nkv > 65535 || s->mask_words > kTreeMaskWords) return GRB_ERR_UNSUPPORTED;
  if (s->row_base && (!s->row_rope || !s->row_mask || !s->mask_words || s->ldm < int64_t(s->mask_words))) return GRB_ERR_ARGUMENT;
  if (s->ldq < int64_t(s->nq + 2 * a.nkv) * kKvDim || (s->ldq & 1) || s->ldo < int64_t(s->nq) * kKvDim || (s->ldo & 3) ||
      ((reinterpret_cast<uintptr_t>(s->qkv) | reinterpret_cast<uintptr_t>(s->cos_table) | reinterpret_cast<uintptr_t>(s->sin_table)) & 3) ||
      (reinterpret_cast<uintptr_t>(s->out) & 7) || !aligned16(s->scratch) || (reinterpret_cast<uintptr_t>(s->row_mask) & 7))
    return GRB_ERR_ARGUMENT;
  if (!s->rows) return GRB_OK;
  if (s->scratch_bytes < grb_attn_tree_scratch_bytes(s->rows, s->nq, s->table.max_pages, s->pages.format)) return GRB_ERR_WORKSPACE;
  const uint32_t format = s->pages.format;
  a.qkv = static_cast<const __nv_bfloat16*>(s->qkv);
  a.ldq = s->ldq;
  a.cos_table = static_cast<const __nv_bfloat16*>(s->cos_table);
  a.sin_table = static_cast<const __nv_bfloat16*>(s->sin_table);
  a.rope_rows = s->rope_rows;
  a.row_seq = s->row_seq;
  a.row_pos = s->row_pos;
  a.row_base = s->row_base;
  a.row_rope = s->row_rope;
  a.row_mask = s->row_mask;
  a.ldm = s->ldm;
  a.mask_words = s->mask_words;
  a.rows = s->rows;
  a.max_parts = uint32_t(parts_of(s->table.max_pages, format));
  // (4 bits: a tile of eight columns where the caller says that one row of a sequence comes at a time, whatever comes then; a row's bits are the same)
  a.tile_rows = (format == GRB_KV_Q4 && s->longest_run == 1 && a.group <= 8 ? 8 : 16) / a.group;
  a.wide_rows = (format == GRB_KV_Q4 ? 2 : 1) * (kWideTile / a.group);       // (4 bits: tiles in pairs)
  // Runs for the wide kernel: trees of more rows than two tiles of the narrow one take; of causal rows prompt chunks, so that the
  // rows of a speculative chain keep the bits of single steps.  A run's rows alone decide, whatever else is in the call, so one run
  // pays for what many gain.  Eight nodes of five heads a kv head, 8 bits, us narrow / wide: one tree behind 1000 positions 18 / 21,
  // four behind 2000 37 / 27, sixteen behind 4000 127 / 69; 16 nodes: 20 / 22, 48 / 28, 214 / 80.  128 rows of a prompt: behind 2000
  // 67 / 37, behind 8000 190 / 75; at its start 20 / 22.
  // Causal rows are taken to be decode rows where the caller does not say (an empty launch of the wide kernel costs a batch of 128 rows
  // behind 2048 positions 148 us instead of 135); guessing from the other rows of the call would have them change a run's bits.
  const uint32_t longest = s->longest_run ? s->longest_run : s->row_base ? s->rows : 1u;
  a.wide_from = s->row_base ? 32 / a.group + 1 : 64;
  if (a.wide_from > s->rows || a.wide_from > longest) a.wide_from = 0;
  a.scaling = s->scaling;
  a.out = static_cast<__nv_bfloat16*>(s->out);
  a.ldo = s->ldo;
  uint8_t* at = static_cast<uint8_t*>(s->scratch);
  const uint64_t pairs = uint64_t(a.rows) * a.nq;
  a.status = reinterpret_cast<uint32_t*>(at);                // (first of the scratch: the caller reads it there)
  a.plan = a.status + 4;
  a.tiles = reinterpret_cast<int4*>(at + 48);
  a.wide_tiles = a.tiles + a.rows;
  a.extent = reinterpret_cast<int32_t*>(a.wide_tiles + a.rows);
  a.row_parts = reinterpret_cast<uint32_t*>(a.extent + a.rows);
  a.q_scale = reinterpret_cast<float*>(a.row_parts + a.rows);
  at += (48 + a.rows * 40ull + pairs * 4 + 255) & ~uint64_t(255);
  a.q = reinterpret_cast<uint16_t*>(at);
  at += pairs * kKvDim * (format == GRB_KV_BF16 ? 4 : 2);
  at += reinterpret_cast<uintptr_t>(at) & 16;                // (the scratch starts on 16 bytes, the parts on 32)
  a.part_acc = reinterpret_cast<float*>(at);
  at += pairs * a.max_parts * kKvDim * 4;
  a.part_ml = reinterpret_cast<float2*>(at);
  const auto stream = static_cast<cudaStream_t>(cuda_stream);
  return format == GRB_KV_Q4 ? tree_launch<kKvQ4>(a, stream) : format == GRB_KV_E4M3 ? tree_launch<kKvE4m3>(a, stream) : tree_launch<kKvBf16>(a, stream);
}

int grb_verify_drafts(const grb_verify_step* s, void* cuda_stream) {
  if (!s || !s->logits || !s->tokens || !s->starts || !s->u_keep || !s->u_draw || !s->stats || !s->out_tokens || !s->out_rows || !s->out_count)
    return GRB_ERR_ARGUMENT;
  if (!s->vocab || !s->width || s->ldl < int64_t(s->vocab) || !(s->temperature >= kVerifyLeastTemperature) || s->temperature > kVerifyMostTemperature || s->dtype > 1 || (reinterpret_cast<uintptr_t>(s->stats) & 15))
    return GRB_ERR_ARGUMENT;
  if (s->draft_probs && (s->parent || s->ldq < int64_t(s->vocab))) return GRB_ERR_ARGUMENT;
  if (s->vocab > kVerifyMaxVocab || s->rows > 65535 || s->seqs > 65535 || s->width > kVerifyMaxNodes) return GRB_ERR_UNSUPPORTED;
  if (!s->seqs) return GRB_OK;
  if (!s->rows) return GRB_ERR_ARGUMENT;
  VerifyArgs a{};
  a.logits = s->logits;
  a.ldl = s->ldl;
  a.tokens = s->tokens;
  a.parent = s->parent;
  a.starts = s->starts;
  a.u_keep = s->u_keep;
  a.u_draw = s->u_draw;
  a.q = s->draft_probs;
  a.ldq = s->ldq;
  a.stats = reinterpret_cast<double2*>(s->stats);
  a.out_tokens = s->out_tokens;
  a.out_rows = s->out_rows;
  a.out_count = s->out_count;
  a.rows = s->rows;
  a.seqs = s->seqs;
  a.vocab = s->vocab;
  a.width = s->width;
  a.log2_scale = 1.4426950408889634 / s->temperature;
  const uint32_t size = s->dtype ? 4 : 2;
  const bool vec = aligned16(s->logits) && (s->ldl * size) % 16 == 0;
  const auto stream = static_cast<cudaStream_t>(cuda_stream);
  if (s->dtype) return vec ? verify_launch<true, true>(a, stream) : verify_launch<true, false>(a, stream);
  return vec ? verify_launch<false, true>(a, stream) : verify_launch<false, false>(a, stream);
}

}  // extern "C"
