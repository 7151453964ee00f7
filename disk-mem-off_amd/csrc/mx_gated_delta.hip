// The gated delta rule over a ragged batch, from and to state slots (mx_gated_delta_rule).
//   S' = e^{g_t} S;  u = beta_t (v_t - k_t^T S');  S = S' + k_t u^T;  o_t = scale q_t^T S
#include <math.h>

#include "mx_common.h"
#include "mx_paged.h"

namespace {

struct GdArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* g;
  const float* beta;
  void* o;
  float* state;
  const int* slot_in;
  const int* slot_out;
  const int* q_start;
  long ldq, ldk, ldv, ldo;
  int n_slots, n_seqs, rows;
  int nk, nv, dk, dv, rep;  // rep: value heads per key head
  int norm;
  float scale;
};

// ------------------------------------------------------------------------------------
// Token by token.  A block holds 32 value columns of one head's state in registers: 8
// lanes of 4 columns, 32 row groups of NR rows (row = group + 32 i).  With S' = e^g S the two
// products that reduce over the rows are taken together, r = k^T S' and p = q^T S', and o =
// scale (p + (q . k) u) follows without a second pass; q . k, |q|^2 and |k|^2 come out of the
// same rows in LDS, so a token costs one exchange between the waves.
//
// For decode steps bound by the state's bytes, read and written once (128 x 32 columns are 16 KiB
// per block, 128-byte pieces of a row).
// ------------------------------------------------------------------------------------
constexpr int kCols = 32;

template <int NR, typename XT>
__global__ __launch_bounds__(256) void k_gd_recurrent(GdArgs a) {
  constexpr int DKP = 32 * NR;
  __shared__ float sk[2][DKP], sq[2][DKP];
  __shared__ float red[2][4][2][kCols];  // [buffer][wave][r, p][column]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int seq = blockIdx.z, h = blockIdx.y, c0 = blockIdx.x * kCols + 4 * (tid & 7);
  const int hk = h / a.rep, grp = tid >> 3;
  const bool col = c0 < a.dv;
  const int t0 = a.q_start[seq], t1 = min(a.q_start[seq + 1], a.rows);
  const int in = a.slot_in[seq], out = a.slot_out[seq];
  const long head = (long)a.dk * a.dv;
  float4 s[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = grp + 32 * i;
    s[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in >= 0 && in < a.n_slots && col && r < a.dk)
      s[i] = *(const float4*)(a.state + ((long)in * a.nv + h) * head + (long)r * a.dv + c0);
  }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    for (int i = tid; i < DKP; i += 256) {
      sk[buf][i] = i < a.dk ? (float)((const XT*)a.k)[(long)t * a.ldk + (long)hk * a.dk + i] : 0.f;
      sq[buf][i] = i < a.dk ? (float)((const XT*)a.q)[(long)t * a.ldq + (long)hk * a.dk + i] : 0.f;
    }
    const float eg = expf(a.g[(long)t * a.nv + h]), beta = a.beta[(long)t * a.nv + h];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = col ? (float)((const XT*)a.v)[(long)t * a.ldv + (long)h * a.dv + c0 + e] : 0.f;
    __syncthreads();
    float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
    for (int i = 0; i < (DKP + 63) / 64; ++i) {
      const int r = lane + 64 * i;
      const float kv = r < DKP ? sk[buf][r] : 0.f, qv = r < DKP ? sq[buf][r] : 0.f;
      kk += kv * kv;
      qq += qv * qv;
      qk += qv * kv;
    }
    kk = mx_wave_sum(kk);
    qq = mx_wave_sum(qq);
    qk = mx_wave_sum(qk);
    const float rk = a.norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.f;
    const float rq = (a.norm ? 1.0f / sqrtf(qq + 1e-6f) : 1.f) * a.scale;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f), p = r;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float kv = sk[buf][grp + 32 * i], qv = sq[buf][grp + 32 * i];
      s[i] = make_float4(s[i].x * eg, s[i].y * eg, s[i].z * eg, s[i].w * eg);
      r.x += kv * s[i].x;
      r.y += kv * s[i].y;
      r.z += kv * s[i].z;
      r.w += kv * s[i].w;
      p.x += qv * s[i].x;
      p.y += qv * s[i].y;
      p.z += qv * s[i].z;
      p.w += qv * s[i].w;
    }
    float rp[8] = {r.x, r.y, r.z, r.w, p.x, p.y, p.z, p.w};
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int o = 8; o < 64; o *= 2) rp[e] += __shfl_xor(rp[e], o);
    if (lane < 8) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        red[buf][wave][0][4 * lane + e] = rp[e];
        red[buf][wave][1][4 * lane + e] = rp[4 + e];
      }
    }
    __syncthreads();
    float u[4];
    const int cl = 4 * (tid & 7);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float rs = (red[buf][0][0][cl + e] + red[buf][1][0][cl + e]) +
                       (red[buf][2][0][cl + e] + red[buf][3][0][cl + e]);
      u[e] = beta * (v[e] - rk * rs);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float kv = sk[buf][grp + 32 * i] * rk;
      s[i].x += kv * u[0];
      s[i].y += kv * u[1];
      s[i].z += kv * u[2];
      s[i].w += kv * u[3];
    }
    if (tid < 8 && col) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float ps = (red[buf][0][1][cl + e] + red[buf][1][1][cl + e]) +
                         (red[buf][2][1][cl + e] + red[buf][3][1][cl + e]);
        ((XT*)a.o)[(long)t * a.ldo + (long)h * a.dv + c0 + e] = (XT)(rq * (ps + qk * rk * u[e]));
      }
    }
  }
  if (out < 0 || out >= a.n_slots || !col) return;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    const int r = grp + 32 * i;
    if (r < a.dk) *(float4*)(a.state + ((long)out * a.nv + h) * head + (long)r * a.dv + c0) = s[i];
  }
}

int check(const MxGatedDelta* d) {
  if (!d || !d->q || !d->k || !d->v || !d->g || !d->beta || !d->o || !d->state || !d->slot_in ||
      !d->slot_out || !d->q_start)
    return MX_ERR_INVALID;
  if (d->n_slots < 0 || d->n_seqs < 0 || d->rows < 0 || d->max_q <= 0 || d->n_k_heads <= 0 ||
      d->n_v_heads <= 0 || d->head_dim_k <= 0 || d->head_dim_v <= 0 || d->n_v_heads % d->n_k_heads)
    return MX_ERR_INVALID;
  if (d->x_dtype != MX_DT_F32 && d->x_dtype != MX_DT_F16) return MX_ERR_INVALID;
  const long kw = (long)d->n_k_heads * d->head_dim_k, vw = (long)d->n_v_heads * d->head_dim_v;
  if (d->ldq < kw || d->ldk < kw || d->ldv < vw || d->ldo < vw) return MX_ERR_INVALID;
  if (d->head_dim_k % 4 || d->head_dim_v % 4 || d->head_dim_k > 256 || d->head_dim_v > 256 ||
      d->n_seqs > 65535 || d->n_v_heads > 65535 || d->rows >= (1 << 24))
    return MX_ERR_UNSUPPORTED;
  const int esz = pk_esz(d->x_dtype);
  if (!mx_aligned16(d->state) || (uintptr_t)d->q % esz || (uintptr_t)d->k % esz ||
      (uintptr_t)d->v % esz || (uintptr_t)d->o % esz)
    return MX_ERR_ALIGNMENT;
  return MX_OK;
}

GdArgs args_of(const MxGatedDelta* d) {
  GdArgs a;
  a.q = d->q;
  a.k = d->k;
  a.v = d->v;
  a.g = d->g;
  a.beta = d->beta;
  a.o = d->o;
  a.state = d->state;
  a.slot_in = d->slot_in;
  a.slot_out = d->slot_out;
  a.q_start = d->q_start;
  a.ldq = d->ldq;
  a.ldk = d->ldk;
  a.ldv = d->ldv;
  a.ldo = d->ldo;
  a.n_slots = d->n_slots;
  a.n_seqs = d->n_seqs;
  a.rows = d->rows;
  a.nk = d->n_k_heads;
  a.nv = d->n_v_heads;
  a.dk = d->head_dim_k;
  a.dv = d->head_dim_v;
  a.rep = d->n_v_heads / d->n_k_heads;
  a.norm = d->qk_norm != 0;
  a.scale = d->scale;
  return a;
}

template <typename XT>
int launch_recurrent(const GdArgs& a, hipStream_t s) {
  auto* kern = a.dk <= 32    ? k_gd_recurrent<1, XT>
               : a.dk <= 64  ? k_gd_recurrent<2, XT>
               : a.dk <= 128 ? k_gd_recurrent<4, XT>
                             : k_gd_recurrent<8, XT>;
  mx_clear_error();
  hipLaunchKernelGGL(kern, dim3(mx_ceil_div(a.dv, kCols), a.nv, a.n_seqs), dim3(256), 0, s, a);
  return mx_launch_status();
}

}  // namespace

extern "C" int mx_gated_delta_rule_workspace_size(const MxGatedDelta* args, size_t* nbytes) {
  if (!nbytes) return MX_ERR_INVALID;
  MX_TRY(check(args));
  *nbytes = 0;
  return MX_OK;
}

extern "C" int mx_gated_delta_rule(const MxGatedDelta* args, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  MX_TRY(check(args));
  if (args->n_seqs == 0) return MX_OK;
  const GdArgs a = args_of(args);
  const hipStream_t s = (hipStream_t)stream;
  return args->x_dtype == MX_DT_F32 ? launch_recurrent<float>(a, s)
                                    : launch_recurrent<half_t>(a, s);
}
