// Attention of new rows over a paged key/value cache (mx_paged_attn).
#include <math.h>

#include "mx_common.h"
#include "mx_paged.h"

namespace {

struct PaArgs {
  const void* q;
  void* out;
  const float* gate;
  long ldq, ldo, ldg;
  int nh, group;
  float scale;
};

// One wave per (row, head): the keys one after another, the dims over the lanes.
template <typename XT, int DT>
__global__ __launch_bounds__(64) void k_pa_simple(PkCache c, PkBatch b, PaArgs a) {
  const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int seq = __builtin_amdgcn_readfirstlane(pk_seq_of(b.q_start, b.n_seqs, t));
  if (seq >= b.n_seqs) return;
  const int q0 = b.q_start[seq], q1 = b.q_start[seq + 1];
  const int pos = b.kv_len[seq] - (q1 - q0) + (t - q0);
  const int kvh = h / a.group;
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
  const XT* qr = (const XT*)a.q + (long)t * a.ldq + (long)h * c.hd;
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = lane + 64 * e < c.hd ? (float)qr[lane + 64 * e] * a.scale : 0.f;
  float m = -INFINITY, l = 0.f;
  const int n = min(pos + 1, b.max_pages * c.ps);
  for (int j = 0; j < n; ++j) {
    const int page = b.pages[(long)seq * b.max_pages + (j >> c.ps_log)];
    if (page < 0 || page >= c.n_pages) continue;
    const long row = ((long)page * c.nkv + kvh) * c.ps + (j & (c.ps - 1));
    float s = 0.f, v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      v[e] = 0.f;
      if (d >= c.hd) continue;
      const long at = row * c.hd + d;
      if constexpr (DT == MX_DT_I8) {
        s += q[e] * ((float)((const int8_t*)c.k)[at] * c.ks[row]);
        v[e] = (float)((const int8_t*)c.v)[at] * c.vs[row];
      } else {
        s += q[e] * (float)((const XT*)c.k)[at];
        v[e] = (float)((const XT*)c.v)[at];
      }
    }
    s = mx_wave_sum(s);
    const float mn = fmaxf(m, s), al = m == mn ? 1.f : expf(m - mn), p = s == mn ? 1.f : expf(s - mn);
    m = mn;
    l = l * al + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = o[e] * al + p * v[e];
  }
  XT* orow = (XT*)a.out + (long)t * a.ldo + (long)h * c.hd;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 64 * e;
    if (d >= c.hd) continue;
    float r = l > 0.f ? o[e] / l : 0.f;
    if (l != l) r = l;
    if (a.gate) r *= mx_sigmoid(a.gate[(long)t * a.ldg + (long)h * c.hd + d]);
    orow[d] = (XT)r;
  }
}

int check(const MxKvCache* cache, const MxPagedBatch* batch, int n_heads) {
  MX_TRY(pk_check_cache(cache));
  MX_TRY(pk_check_batch(batch));
  if (n_heads <= 0 || n_heads % cache->n_kv_heads) return MX_ERR_INVALID;
  return n_heads > 65535 ? MX_ERR_UNSUPPORTED : MX_OK;
}

}  // namespace

extern "C" int mx_paged_attn_workspace_size(const MxKvCache* cache, const MxPagedBatch* batch,
                                            int32_t n_heads, size_t* nbytes) {
  if (!nbytes) return MX_ERR_INVALID;
  MX_TRY(check(cache, batch, n_heads));
  *nbytes = 0;
  return MX_OK;
}

extern "C" int mx_paged_attn(const MxKvCache* cache, const MxPagedBatch* batch,
                             const MxPagedAttn* args, void* workspace, size_t workspace_bytes,
                             void* stream) {
  if (!args || !args->q || !args->out) return MX_ERR_INVALID;
  MX_TRY(check(cache, batch, args->n_heads));
  const long w = (long)args->n_heads * cache->head_dim;
  if (args->ldq < w || args->ldo < w || (args->gate && args->ldg < w)) return MX_ERR_INVALID;
  const int esz = cache->dtype == MX_DT_F32 ? 4 : 2;
  if (!mx_aligned16(args->q) || !mx_aligned16(args->out) || !mx_aligned16(args->gate) ||
      args->ldq * esz % 16 || args->ldo * esz % 16 || (args->gate && args->ldg * 4 % 16))
    return MX_ERR_ALIGNMENT;
  if (batch->rows == 0 || batch->n_seqs == 0) return MX_OK;
  const PkCache c = pk_cache(cache);
  const PkBatch b = pk_batch(batch);
  const PaArgs a{args->q, args->out, args->gate, args->ldq, args->ldo, args->ldg, args->n_heads,
                 args->n_heads / cache->n_kv_heads, args->scale};
  const hipStream_t s = (hipStream_t)stream;
  auto* kern = cache->dtype == MX_DT_F32   ? k_pa_simple<float, MX_DT_F32>
               : cache->dtype == MX_DT_F16 ? k_pa_simple<half_t, MX_DT_F16>
                                           : k_pa_simple<half_t, MX_DT_I8>;
  mx_clear_error();
  hipLaunchKernelGGL(kern, dim3(b.rows, a.nh), dim3(64), 0, s, c, b, a);
  return mx_launch_status();
}
