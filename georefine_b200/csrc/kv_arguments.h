// What the C entry points of a paged KV cache refuse, and the kernels' forms of what they accept.
#pragma once
#include "../../include/georefine_b200.h"
#include "kv_cache.cuh"

namespace grb {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline int pages_of(const grb_kv_pages* p, KvPagesArgs& a) {
  if (!p || !p->k || !p->v || !p->layers || !p->pages || !p->nkv) return GRB_ERR_ARGUMENT;
  if (p->format > GRB_KV_E4M3 && p->format != GRB_KV_Q4) return GRB_ERR_UNSUPPORTED;
  if (p->format == GRB_KV_E4M3 ? !p->k_exp || !p->v_exp || !aligned16(p->k_exp) || !aligned16(p->v_exp) : p->k_exp || p->v_exp) return GRB_ERR_ARGUMENT;
  const int64_t entries = int64_t(p->pages) * p->nkv * kKvPage, elements = p->format == GRB_KV_Q4 ? int64_t(p->pages) * p->nkv * kQ4Page : entries * int64_t(kKvDim);
  if (!aligned16(p->k) || !aligned16(p->v) || (p->layers > 1 && (p->layer_stride < elements || (p->layer_stride & 15)))) return GRB_ERR_ARGUMENT;
  if (p->format == GRB_KV_E4M3 && p->layers > 1 && p->exp_stride < entries) return GRB_ERR_ARGUMENT;
  if (p->pages > 0x7FFFFFu || p->nkv > 4096) return GRB_ERR_UNSUPPORTED;
  a = KvPagesArgs{p->k, p->v, p->k_exp, p->v_exp, p->layer_stride, p->exp_stride, p->layers, p->pages, p->nkv};
  return GRB_OK;
}

inline int table_of(const grb_kv_table* t, const KvPagesArgs& pages, KvTable& a) {
  if (!t || !t->table || !t->slots || !t->max_pages || t->ld < int64_t(t->max_pages)) return GRB_ERR_ARGUMENT;
  if (t->max_pages > 0x7FFFFFu || t->slots > 0x7FFFFFFFu) return GRB_ERR_UNSUPPORTED;
  a = KvTable{t->table, t->ld, t->slots, t->max_pages, pages.pages};
  return GRB_OK;
}

}  // namespace grb
