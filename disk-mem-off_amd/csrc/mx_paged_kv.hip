// Rows into a paged key/value cache (mx_kv_append) and copies of pages (mx_copy_pages).
#include <math.h>

#include "mx_common.h"
#include "mx_paged.h"

namespace {

// ------------------------------------------------------------------------------------
// mx_kv_append.  Per head row x of head_dim values: y = x / sqrt(mean(x^2) + eps) * w, then
// with half = rotary_dim / 2 and a_j = position * theta^(-j / half):
//   y_j cos a_j - y_{j + half} sin a_j   (j < half),   y_{j + half} cos a_j + y_j sin a_j.
// The launch passes theta^(-j / half) / (2 pi) as fp64 numbers; a token's angles are taken
// as turns, reduced to [-1/2, 1/2] in fp64 and only then rounded to fp32, so a position
// of a million costs no accuracy.
//
// Bound by its bytes (rows in, rows out).  A block takes one token and some of its head
// rows: DP / 4 lanes per row, 4 dims each, 256 / DP rows per wave at once, one load for the
// lane's dims and one for their rotation partners (the same cache lines).  The token's cos
// and sin are worked out once per block.  2 x 2048 rows of 16 query and 2 key heads of 256: 32.6 us, 3.8 TB/s;
// 64 rows of one token each 7.5 us, a launch.
// ------------------------------------------------------------------------------------
struct PkTurns {
  double f[128];  // turns per position, rotary_dim / 2 of them
};

struct PkRowArgs {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  const void* qw;
  const void* kw;
  long ldq, ldk, ldv, ldqo;
  int nh, half, pdt, rpb;
  float eps;
};

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

template <typename XT, bool VEC>
__device__ __forceinline__ float4 pk_load4(const XT* p) {
  if constexpr (!VEC) return make_float4((float)p[0], (float)p[1], (float)p[2], (float)p[3]);
  if constexpr (sizeof(XT) == 4) return *(const float4*)p;
  const half4_t h = *(const half4_t*)p;
  return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
}

template <bool VEC>
__device__ __forceinline__ float4 pk_param4(const void* w, int dt, int i) {
  if constexpr (VEC) return mx_load_param4(w, dt, i);
  return make_float4(mx_load_param(w, dt, i), mx_load_param(w, dt, i + 1),
                     mx_load_param(w, dt, i + 2), mx_load_param(w, dt, i + 3));
}

template <bool VEC>
__device__ __forceinline__ void pk_store4(void* base, bool f32, long at, const float4& o) {
  if (f32) {
    float* p = (float*)base + at;
    if constexpr (VEC) {
      *(float4*)p = o;
    } else {
      p[0] = o.x;
      p[1] = o.y;
      p[2] = o.z;
      p[3] = o.w;
    }
  } else {
    half_t* p = (half_t*)base + at;
    const half4_t h = {(half_t)o.x, (half_t)o.y, (half_t)o.z, (half_t)o.w};
    if constexpr (VEC) {
      *(half4_t*)p = h;
    } else {
      p[0] = h[0];
      p[1] = h[1];
      p[2] = h[2];
      p[3] = h[3];
    }
  }
}

// VEC: rows, norm weights and q_out on vector boundaries and a rotary half of whole groups
// of 4 dims; the other form takes any address and any even rotary_dim.
template <int DP, typename XT, bool VEC>
__global__ __launch_bounds__(256) void k_pk_append(PkCache c, PkBatch b, PkRowArgs a,
                                                   PkTurns turns) {
  __shared__ __align__(16) float cs[128], sn[128];
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int seq = __builtin_amdgcn_readfirstlane(pk_seq_of(b.q_start, b.n_seqs, t));
  if (seq >= b.n_seqs) return;  // rows behind the last sequence
  const int q0 = b.q_start[seq], q1 = b.q_start[seq + 1];
  const int pos = b.kv_len[seq] - (q1 - q0) + (t - q0);
  if (pos < 0) return;
  const int pi = pos >> c.ps_log;
  const int page = pi < b.max_pages ? b.pages[(long)seq * b.max_pages + pi] : -1;
  const bool stored = page >= 0 && page < c.n_pages;
  for (int j = threadIdx.x; j < a.half; j += 256) {
    const double turn = (double)pos * turns.f[j];
    sincospif((float)(2.0 * (turn - rint(turn))), &sn[j], &cs[j]);
  }
  __syncthreads();

  constexpr int LPR = DP / 4, RPW = 64 / LPR;
  const int i = 4 * (lane % LPR);
  const bool valid = i < c.hd;
  const int ic = valid ? i : 0;
  const int half = a.half;
  const int nq = a.q ? a.nh : 0;
  const int slots = nq + 2 * c.nkv;
  const int end = min(slots, (int)(blockIdx.y + 1) * a.rpb);
  for (int s0 = blockIdx.y * a.rpb + wave * RPW; s0 < end; s0 += 4 * RPW) {
    const bool act = s0 + lane / LPR < end;
    const int sl = min(s0 + lane / LPR, end - 1);
    const int kind = sl < nq ? 0 : sl < nq + c.nkv ? 1 : 2;  // q, k, v
    const int h = kind == 0 ? sl : kind == 1 ? sl - nq : sl - nq - c.nkv;
    const XT* row = kind == 0   ? (const XT*)a.q + (long)t * a.ldq
                    : kind == 1 ? (const XT*)a.k + (long)t * a.ldk
                                : (const XT*)a.v + (long)t * a.ldv;
    row += (long)h * c.hd;
    float4 x = pk_load4<XT, VEC>(row + ic);
    float4 xp = x, cv = make_float4(1.f, 1.f, 1.f, 1.f), sv = make_float4(0.f, 0.f, 0.f, 0.f);
    float4 wp = cv;
    const void* nw = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
    const bool rot = kind != 2 && valid && i < 2 * half;
    if (rot) {
      if constexpr (VEC) {
        const int p = i < half ? i + half : i - half, j = i < half ? i : i - half;
        xp = pk_load4<XT, VEC>(row + p);
        if (nw) wp = pk_param4<VEC>(nw, a.pdt, p);
        cv = *(const float4*)(cs + j);
        sv = *(const float4*)(sn + j);
        if (i < half) sv = make_float4(-sv.x, -sv.y, -sv.z, -sv.w);
      } else {
        float px[4], pw[4], pc[4], ps[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = i + e;
          const bool in = d < 2 * half;
          const int p = in ? (d < half ? d + half : d - half) : d, j = d < half ? d : d - half;
          px[e] = (float)row[p];
          pw[e] = nw ? mx_load_param(nw, a.pdt, p) : 1.f;
          pc[e] = in ? cs[j] : 1.f;
          ps[e] = in ? (d < half ? -sn[j] : sn[j]) : 0.f;
        }
        xp = make_float4(px[0], px[1], px[2], px[3]);
        wp = make_float4(pw[0], pw[1], pw[2], pw[3]);
        cv = make_float4(pc[0], pc[1], pc[2], pc[3]);
        sv = make_float4(ps[0], ps[1], ps[2], ps[3]);
      }
    }
    if (!valid) x = make_float4(0.f, 0.f, 0.f, 0.f);
    float ss = (x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w);
    if constexpr (LPR == 64) {
      ss = mx_wave_sum(ss);
    } else {
#pragma unroll
      for (int o = 1; o < LPR; o *= 2) ss += __shfl_xor(ss, o);
    }
    float4 o = x;
    if (nw) {
      const float r = 1.0f / sqrtf(ss / (float)c.hd + a.eps);
      const float4 w = pk_param4<VEC>(nw, a.pdt, ic);
      o = make_float4(x.x * r * w.x, x.y * r * w.y, x.z * r * w.z, x.w * r * w.w);
      xp = make_float4(xp.x * r * wp.x, xp.y * r * wp.y, xp.z * r * wp.z, xp.w * r * wp.w);
    }
    if (rot)
      o = make_float4(o.x * cv.x + xp.x * sv.x, o.y * cv.y + xp.y * sv.y, o.z * cv.z + xp.z * sv.z,
                      o.w * cv.w + xp.w * sv.w);
    if (kind == 0) {
      if (act && valid)
        pk_store4<VEC>(a.q_out, c.dt == MX_DT_F32, (long)t * a.ldqo + (long)h * c.hd + i, o);
      if (c.dt != MX_DT_I8) continue;
    }
    // k and v rows: row `at` of the pool counts rows of head_dim values
    const long at = ((long)page * c.nkv + h) * c.ps + (pos & (c.ps - 1));
    char* pool = kind == 1 ? c.k : c.v;
    if (c.dt != MX_DT_I8) {
      if (act && valid && stored) pk_store4<true>(pool, c.dt == MX_DT_F32, at * c.hd + i, o);
      continue;
    }
    // As bits: an infinity or a NaN is larger than every number, and makes the row's scale NaN.
    auto size = [](float v) { return (int)(__float_as_uint(v) & 0x7FFFFFFFu); };
    int m = valid ? max(max(size(o.x), size(o.y)), max(size(o.z), size(o.w))) : 0;
#pragma unroll
    for (int d = 1; d < LPR; d *= 2) m = max(m, __shfl_xor(m, d));
    if (kind == 0) continue;  // the shuffles needed every lane
    const float scale = m >= 0x7F800000 ? __builtin_nanf("") : m > 0 ? __uint_as_float((uint32_t)m) / 127.f : 1.f;
    auto q8 = [&](float v) {
      return (uint32_t)((int)fminf(fmaxf(rintf(v / scale), -127.f), 127.f) & 255);
    };
    if (act && stored) {
      if (valid)
        *(uint32_t*)(pool + at * c.hd + i) = q8(o.x) | q8(o.y) << 8 | q8(o.z) << 16 | q8(o.w) << 24;
      if (i == 0) (kind == 1 ? c.ks : c.vs)[at] = scale;
    }
  }
}

bool on_vector(const void* p, long ld, int esz) {
  return ((uintptr_t)p & (4 * esz - 1)) == 0 && ld % 4 == 0;
}

template <typename XT, bool VEC>
int launch_append(const PkCache& c, const PkBatch& b, const PkRowArgs& a, const PkTurns& f,
                  hipStream_t s) {
  const int slots = (a.q ? a.nh : 0) + 2 * c.nkv;
  const dim3 grid(b.rows, mx_ceil_div(slots, a.rpb));
  auto* kern = c.hd <= 32    ? k_pk_append<32, XT, VEC>
               : c.hd <= 64  ? k_pk_append<64, XT, VEC>
               : c.hd <= 128 ? k_pk_append<128, XT, VEC>
                             : k_pk_append<256, XT, VEC>;
  mx_clear_error();
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, b, a, f);
  return mx_launch_status();
}

// ------------------------------------------------------------------------------------
// mx_copy_pages.  Bound by its bytes, each read and written once: a block copies one piece of
// one page of one pool, 16 bytes per lane and load, all loads of a thread ahead of its
// stores.  250 pages of 64 KiB in 24 pools: 154 us, 5.1 TB/s.
// ------------------------------------------------------------------------------------
constexpr int kCopyPools = 64;          // pools per launch (their table travels as an argument)
constexpr int kCopyVec = 4;             // 16-byte loads of a thread in flight
constexpr int kGridX = (1 << 24) - 1;   // blocks of 256 threads along x (2^32 threads)
constexpr int kCopyPiece = 256 * 16 * kCopyVec;

struct PkPools {
  char* base[kCopyPools];
  size_t bytes[kCopyPools];
  int n_pages[kCopyPools];
};

__global__ __launch_bounds__(256) void k_pk_copy(PkPools p, const int* __restrict__ src,
                                                 const int* __restrict__ dst, int pieces) {
  const int pool = blockIdx.y;
  const int pair = blockIdx.x / pieces;
  const size_t off = (size_t)(blockIdx.x - pair * pieces) * kCopyPiece;
  const size_t bytes = p.bytes[pool];
  if (off >= bytes) return;
  const int from = src[pair], to = dst[pair], n = p.n_pages[pool];
  if (from < 0 || from >= n || to < 0 || to >= n) return;
  const int4_t* a = (const int4_t*)(p.base[pool] + from * bytes + off);
  int4_t* o = (int4_t*)(p.base[pool] + to * bytes + off);
  const int left = (int)min((bytes - off) / 16, (size_t)(kCopyPiece / 16));
  int4_t v[kCopyVec];
#pragma unroll
  for (int u = 0; u < kCopyVec; ++u) {
    const int i = threadIdx.x + 256 * u;
    if (i < left) v[u] = a[i];
  }
#pragma unroll
  for (int u = 0; u < kCopyVec; ++u) {
    const int i = threadIdx.x + 256 * u;
    if (i < left) o[i] = v[u];
  }
}

}  // namespace

extern "C" int mx_kv_append(const MxKvCache* cache, const MxPagedBatch* batch,
                            const MxKvRows* rows, void* stream) {
  MX_TRY(pk_check_cache(cache));
  MX_TRY(pk_check_batch(batch));
  const MxKvRows* r = rows;
  if (!r || !r->k || !r->v || (r->q == nullptr) != (r->q_out == nullptr)) return MX_ERR_INVALID;
  if (r->q && r->n_heads <= 0) return MX_ERR_INVALID;
  if (r->x_dtype != MX_DT_F32 && r->x_dtype != MX_DT_F16) return MX_ERR_INVALID;
  if (r->param_dtype != MX_DT_F32 && r->param_dtype != MX_DT_F16) return MX_ERR_INVALID;
  if (r->rotary_dim < 0 || r->rotary_dim % 2 || r->rotary_dim > cache->head_dim)
    return MX_ERR_INVALID;
  if (r->rotary_dim && !(r->rope_theta > 0.0)) return MX_ERR_INVALID;
  const long hd = cache->head_dim;
  if (r->ldk < cache->n_kv_heads * hd || r->ldv < cache->n_kv_heads * hd) return MX_ERR_INVALID;
  if (r->q && (r->ldq < r->n_heads * hd || r->ldqo < r->n_heads * hd)) return MX_ERR_INVALID;
  const int esz = pk_esz(r->x_dtype), osz = cache->dtype == MX_DT_F32 ? 4 : 2;
  if ((uintptr_t)r->q % esz || (uintptr_t)r->k % esz || (uintptr_t)r->v % esz ||
      (uintptr_t)r->q_out % osz || (uintptr_t)r->q_norm_w % pk_esz(r->param_dtype) ||
      (uintptr_t)r->k_norm_w % pk_esz(r->param_dtype))
    return MX_ERR_ALIGNMENT;
  if (batch->rows == 0 || batch->n_seqs == 0) return MX_OK;
  const PkCache c = pk_cache(cache);
  const PkBatch b = pk_batch(batch);
  PkRowArgs a;
  a.q = r->q;
  a.k = r->k;
  a.v = r->v;
  a.q_out = r->q_out;
  a.qw = r->q_norm_w;
  a.kw = r->k_norm_w;
  a.ldq = r->ldq;
  a.ldk = r->ldk;
  a.ldv = r->ldv;
  a.ldqo = r->ldqo;
  a.nh = r->n_heads;
  a.half = r->rotary_dim / 2;
  a.pdt = r->param_dtype;
  a.eps = r->eps;
  const int slots = (a.q ? a.nh : 0) + 2 * c.nkv;
  a.rpb = b.rows >= 512 ? slots : 4 * (256 / (c.hd <= 32 ? 32 : c.hd <= 64 ? 64 : c.hd <= 128 ? 128 : 256));
  PkTurns f;
  if (a.half) {
    const long double step = powl((long double)r->rope_theta, -1.0L / a.half);
    long double v = 0.15915494309189533576888376337251436L;  // 1 / (2 pi)
    for (int j = 0; j < a.half; ++j, v *= step) f.f[j] = (double)v;
  }
  const int psz = pk_esz(r->param_dtype);
  const bool vec = a.half % 4 == 0 && on_vector(r->k, r->ldk, esz) && on_vector(r->v, r->ldv, esz) &&
                   (!r->q || (on_vector(r->q, r->ldq, esz) && on_vector(r->q_out, r->ldqo, osz))) &&
                   on_vector(r->q_norm_w, 0, psz) && on_vector(r->k_norm_w, 0, psz);
  const hipStream_t s = (hipStream_t)stream;
  if (r->x_dtype == MX_DT_F32)
    return vec ? launch_append<float, true>(c, b, a, f, s) : launch_append<float, false>(c, b, a, f, s);
  return vec ? launch_append<half_t, true>(c, b, a, f, s) : launch_append<half_t, false>(c, b, a, f, s);
}

extern "C" int mx_copy_pages(const MxPagePool* pools, int32_t n_pools, const int32_t* src,
                             const int32_t* dst, int32_t n_copies, void* stream) {
  if (!pools || n_pools < 0 || n_copies < 0 || !src || !dst) return MX_ERR_INVALID;
  for (int i = 0; i < n_pools; ++i) {
    if (!pools[i].base || pools[i].n_pages <= 0 || pools[i].page_bytes == 0) return MX_ERR_INVALID;
    if (!mx_aligned16(pools[i].base)) return MX_ERR_ALIGNMENT;
    if (pools[i].page_bytes % 16 || pools[i].page_bytes > ((size_t)1 << 36))
      return MX_ERR_UNSUPPORTED;
  }
  for (int at = 0; at < n_pools && n_copies > 0; at += kCopyPools) {
    PkPools p = {};
    const int n = n_pools - at < kCopyPools ? n_pools - at : kCopyPools;
    size_t most = 0;
    for (int i = 0; i < n; ++i) {
      p.base[i] = (char*)pools[at + i].base;
      p.bytes[i] = pools[at + i].page_bytes;
      p.n_pages[i] = pools[at + i].n_pages;
      if (p.bytes[i] > most) most = p.bytes[i];
    }
    const int pieces = (int)((most + kCopyPiece - 1) / kCopyPiece);
    const int per = kGridX / pieces;  // pairs of a launch
    for (int i = 0; i < n_copies; i += per) {
      const int pairs = n_copies - i < per ? n_copies - i : per;
      mx_clear_error();
      hipLaunchKernelGGL(k_pk_copy, dim3((unsigned)(pieces * pairs), n), dim3(256), 0,
                         (hipStream_t)stream, p, src + i, dst + i, pieces);
      MX_TRY(mx_launch_status());
    }
  }
  return MX_OK;
}
