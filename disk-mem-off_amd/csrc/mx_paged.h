// Shared by the paged-cache kernels: argument checks, the batch's rows and their pages.
#pragma once

#include "mx_common.h"

// How a launch holds the cache and the batch (by value).
struct PkCache {
  char* k;
  char* v;
  float* ks;
  float* vs;
  int n_pages, ps, ps_log, nkv, hd, dt;
};
struct PkBatch {
  const int* q_start;
  const int* kv_len;
  const int* pages;
  int n_seqs, max_pages, rows, max_kv;
};

static inline int pk_esz(int dt) { return dt == MX_DT_F32 ? 4 : dt == MX_DT_F16 ? 2 : 1; }

// Field checks that need no device.
static inline int pk_check_cache(const MxKvCache* c) {
  if (!c || !c->k || !c->v || c->n_pages <= 0 || c->page_size <= 0 || c->n_kv_heads <= 0 ||
      c->head_dim <= 0)
    return MX_ERR_INVALID;
  if (c->dtype != MX_DT_F32 && c->dtype != MX_DT_F16 && c->dtype != MX_DT_I8) return MX_ERR_INVALID;
  if (c->dtype == MX_DT_I8 && (!c->k_scale || !c->v_scale)) return MX_ERR_INVALID;
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return MX_ERR_UNSUPPORTED;
  if (c->head_dim > 256 || c->head_dim % (c->dtype == MX_DT_I8 ? 16 : 8)) return MX_ERR_UNSUPPORTED;
  if (c->n_kv_heads > (1 << 16)) return MX_ERR_UNSUPPORTED;
  if (!mx_aligned16(c->k) || !mx_aligned16(c->v)) return MX_ERR_ALIGNMENT;
  if (c->dtype == MX_DT_I8 && (!mx_aligned16(c->k_scale) || !mx_aligned16(c->v_scale)))
    return MX_ERR_ALIGNMENT;
  return MX_OK;
}

static inline int pk_check_batch(const MxPagedBatch* b) {
  if (!b || !b->q_start || !b->kv_len || !b->pages || b->n_seqs < 0 || b->rows < 0 ||
      b->max_pages <= 0 || b->max_q <= 0 || b->max_kv < 0)
    return MX_ERR_INVALID;
  return b->n_seqs > 65535 || b->rows >= (1 << 24) ? MX_ERR_UNSUPPORTED : MX_OK;
}

static inline PkCache pk_cache(const MxKvCache* c) {
  PkCache k;
  k.k = (char*)c->k;
  k.v = (char*)c->v;
  k.ks = c->k_scale;
  k.vs = c->v_scale;
  k.n_pages = c->n_pages;
  k.ps = c->page_size;
  k.ps_log = __builtin_ctz((unsigned)c->page_size);
  k.nkv = c->n_kv_heads;
  k.hd = c->head_dim;
  k.dt = c->dtype;
  return k;
}

static inline PkBatch pk_batch(const MxPagedBatch* b) {
  return PkBatch{b->q_start, b->kv_len, b->pages, b->n_seqs, b->max_pages, b->rows,
                 b->max_kv};
}

// The sequence that row t belongs to: the last b with q_start[b] <= t, or n where t is past
// q_start[n].  The whole wave looks: 64 boundaries at once, so up to 64 sequences take one
// load and up to 4096 two.  Callers must be converged.
__device__ __forceinline__ int pk_seq_of(const int* __restrict__ q_start, int n, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;  // the answer is the number of b in (0, n] with q_start[b] <= t
  while (hi > lo) {
    const int step = (hi - lo + 63) >> 6;
    const int at = lo + (lane + 1) * step;  // the boundary this lane looks at
    const bool below = at <= hi && q_start[at] <= t;
    const int c = __popcll(__builtin_amdgcn_ballot_w64(below));
    const int nlo = lo + c * step;
    hi = min(hi, nlo + step - 1);
    lo = nlo;
  }
  return lo;
}
