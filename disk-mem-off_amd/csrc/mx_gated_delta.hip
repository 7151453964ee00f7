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
// same rows in LDS, so a token costs one exchange between the waves.  Eight tokens' rows are
// loaded at once (16 tokens of one sequence: 28 us one by one, 18 so).
//
// For decode steps bound by the state's bytes, read and written once (128 x 32 columns are 16 KiB
// per block, 128-byte pieces of a row): 96 sequences of 32 heads of 128 x 128 in 82 us, 4.9 TB/s.
// ------------------------------------------------------------------------------------
constexpr int kCols = 32, kAhead = 8;

template <int NR>
struct GdRecLds {
  static constexpr int DKP = 32 * NR;
  float k[kAhead][DKP], q[kAhead][DKP], v[kAhead][kCols], g[kAhead], beta[kAhead];
  float red[2][4][2][kCols];  // [buffer][wave][r, p][column]
};

template <int NR, typename XT>
__device__ void gd_recurrent(const GdArgs& a, GdRecLds<NR>& lds, int piece, int h, int seq, int below) {
  constexpr int DKP = 32 * NR;
  auto &sk = lds.k, &sq = lds.q;
  auto& sv = lds.v;
  auto &sg = lds.g, &sb = lds.beta;
  auto& red = lds.red;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int cl = 4 * (tid & 7), c0 = piece * kCols + cl;
  const int hk = h / a.rep, grp = tid >> 3;
  const bool col = c0 < a.dv;
  const int t0 = a.q_start[seq], t1 = min(a.q_start[seq + 1], a.rows);
  if (t1 - t0 >= below) return;
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
  for (int first = t0; first < t1; first += kAhead) {
    const int some = min(kAhead, t1 - first);
    if (first > t0) __syncthreads();  // the rows before are read
    for (int i = tid; i < some * DKP; i += 256) {
      const int d = i % DKP;
      const long t = first + i / DKP;
      sk[i / DKP][d] = d < a.dk ? (float)((const XT*)a.k)[t * a.ldk + (long)hk * a.dk + d] : 0.f;
      sq[i / DKP][d] = d < a.dk ? (float)((const XT*)a.q)[t * a.ldq + (long)hk * a.dk + d] : 0.f;
    }
    {
      const int i = tid / kCols, c = piece * kCols + tid % kCols;  // 8 x 32 threads
      if (i < some) sv[i][tid % kCols] = c < a.dv ? (float)((const XT*)a.v)[(long)(first + i) * a.ldv + (long)h * a.dv + c] : 0.f;
      if (tid < some) {
        sg[tid] = expf(a.g[(long)(first + tid) * a.nv + h]);
        sb[tid] = a.beta[(long)(first + tid) * a.nv + h];
      }
    }
    __syncthreads();
    for (int i = 0; i < some; ++i) {
      const int buf = i & 1;
      const float eg = sg[i], beta = sb[i];
      float4 r = make_float4(0.f, 0.f, 0.f, 0.f), p = r;
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float kv = sk[i][grp + 32 * n], qv = sq[i][grp + 32 * n];
        s[n] = make_float4(s[n].x * eg, s[n].y * eg, s[n].z * eg, s[n].w * eg);
        r.x += kv * s[n].x;
        r.y += kv * s[n].y;
        r.z += kv * s[n].z;
        r.w += kv * s[n].w;
        p.x += qv * s[n].x;
        p.y += qv * s[n].y;
        p.z += qv * s[n].z;
        p.w += qv * s[n].w;
      }
      // The wave's 8 row groups: halves of the lanes, then quarters, each keep half of the 8 sums.
      float x[4] = {r.x, r.y, r.z, r.w}, y[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        mx_swap32(x[e], y[e]);
        x[e] += y[e];  // r in the lower half of the lanes, p in the upper
      }
      mx_swap16(x[0], x[2]);
      mx_swap16(x[1], x[3]);
      float2 z = make_float2(x[0] + x[2], x[1] + x[3]);  // columns 0, 1 in the even rows, 2, 3 in the odd
      z.x += mx_dpp<0x128>(z.x);  // row_ror:8
      z.y += mx_dpp<0x128>(z.y);
      if ((lane & 8) == 0) *(float2*)&red[buf][wave][lane >> 5][cl + 2 * ((lane >> 4) & 1)] = z;
      float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
      for (int n = 0; n < (DKP + 63) / 64; ++n) {
        const int d = lane + 64 * n;
        const float kv = d < DKP ? sk[i][d] : 0.f, qv = d < DKP ? sq[i][d] : 0.f;
        kk += kv * kv;
        qq += qv * qv;
        qk += qv * kv;
      }
      kk = mx_wave_sum(kk);
      qq = mx_wave_sum(qq);
      qk = mx_wave_sum(qk);
      const float rk = a.norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.f;
      const float rq = (a.norm ? 1.0f / sqrtf(qq + 1e-6f) : 1.f) * a.scale;
      __syncthreads();
      auto sum = [&](int w) {
        const float4 x0 = *(const float4*)&red[buf][0][w][cl], x1 = *(const float4*)&red[buf][1][w][cl];
        const float4 x2 = *(const float4*)&red[buf][2][w][cl], x3 = *(const float4*)&red[buf][3][w][cl];
        return make_float4((x0.x + x1.x) + (x2.x + x3.x), (x0.y + x1.y) + (x2.y + x3.y), (x0.z + x1.z) + (x2.z + x3.z),
                           (x0.w + x1.w) + (x2.w + x3.w));
      };
      const float4 rs = sum(0), v = *(const float4*)&sv[i][cl];
      const float4 u = make_float4(beta * (v.x - rk * rs.x), beta * (v.y - rk * rs.y), beta * (v.z - rk * rs.z),
                                   beta * (v.w - rk * rs.w));
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        const float kv = sk[i][grp + 32 * n] * rk;
        s[n].x += kv * u.x;
        s[n].y += kv * u.y;
        s[n].z += kv * u.z;
        s[n].w += kv * u.w;
      }
      if (tid < 8 && col) {
        const float4 ps = sum(1);
        const float f = qk * rk;
        XT* o = (XT*)a.o + (long)(first + i) * a.ldo + (long)h * a.dv + c0;
        o[0] = (XT)(rq * (ps.x + f * u.x));
        o[1] = (XT)(rq * (ps.y + f * u.y));
        o[2] = (XT)(rq * (ps.z + f * u.z));
        o[3] = (XT)(rq * (ps.w + f * u.w));
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

template <int NR, typename XT>
__global__ __launch_bounds__(256) void k_gd_recurrent(GdArgs a) {
  __shared__ __align__(16) GdRecLds<NR> lds;
  gd_recurrent<NR, XT>(a, lds, blockIdx.x, blockIdx.y, blockIdx.z, 1 << 30);
}

// ------------------------------------------------------------------------------------
// Chunk by chunk.  For the tokens t = 1 .. 64 of a chunk, with G_t = g_1 + .. + g_t, S the
// state before it and k, q as they go in (normalised, q scaled):
//   A_ts = beta_t e^{G_t - G_s} k_t.k_s  (s < t)     T = (I + A)^-1
//   u = T x,  x_t = beta_t (v_t - e^{G_t} k_t^T S)   P_ts = e^{G_t - G_s} q_t.k_s  (s <= t)
//   o_t = e^{G_t} q_t^T S + sum_s P_ts u_s           S <- e^{G_64} S + sum_t e^{G_64 - G_t} k_t u_t^T
// k_gd_prep forms T and P of every chunk at once; k_gd_walk takes a sequence's chunks in order,
// 16 columns of a head's state per four waves.  The exponents are differences <= 0 of one prefix
// sum, which is kept in 64 bits: token decays of -256 (e^-256 is 0 in 32 bits) next to
// decays near 0 leave the differences their digits.  The norms and the scale of q and k are
// factors of a token, so the products take q and k as they are stored.
//
// The products run on the fp16 matrix instructions at fp32's precision: x = 2^e (hi + lo), both fp16,
// hi = x 2^-e rounded and lo the rest rounded: 22 bits and the sign of lo, an error of 2^-23 |x|, and
// at least 2^-39 of the largest element that shares the e (of a token's row of k, a row of T, a column
// of S, 16 tokens of a column of x and u).  hi hi + hi lo + lo hi leave out 2^-22 of a product;
// fp16 k and q are exact as they are, and take two products.  Sums are in 32 bits.
// ------------------------------------------------------------------------------------
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t mx_rsrc_t;
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4_t gd_lds_s4;

constexpr int kC = 64;  // tokens of a chunk

// What k_gd_prep leaves of a (chunk, value head): T and P as planes hi, lo, and factors of the
// tokens; of a (chunk, key head): k and q, as they are or as planes.  All of it lane by lane as the
// walk's matrix instructions take it, in 16-byte pieces: a load of the rows themselves has lanes 64 bytes
// apart next to each other and keeps the L1 busy for each (walk of 4 prompts of up to
// 2600 tokens: 278 us, 170 like this).  T and P: [plane][16 rows][2 blocks of 16 columns][lane]; k and q: [plane][16
// rows][32 dims][lane].
enum { kFa, kFb, kFc, kFbeta, kFt, kFp, kFend, kFactors };
constexpr int kPlane = kC * kC * 2, kOffP = 2 * kPlane, kOffF = 4 * kPlane, kRec = kOffF + kFactors * kC * 4;
template <int DK, typename XT>
constexpr int kRows = kC * DK * (sizeof(XT) == 2 ? 2 : 4);  // bytes of k's planes, and of q's

__device__ __forceinline__ float4_t gd_mfma(half8_t a, half8_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float4_t gd_mfma(half4_t a, half4_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ half4_t gd_half(half8_t x, int h) {
  return h ? (half4_t){x[4], x[5], x[6], x[7]} : (half4_t){x[0], x[1], x[2], x[3]};
}
// Over 16 columns: a holds 4 consecutive columns of the lane's A row, b the same of its B column.
__device__ __forceinline__ float4_t gd_mfma(const float4_t& a, const float4_t& b, float4_t c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// 2^-e and 2^e with m 2^-e in [2^14, 2^15): fp16 holds twice that.  Under 2^-112 they stay; an
// infinite or NaN m gives a finite factor.
__device__ __forceinline__ float gd_scale(float m, float& inv) {
  const int e = max((int)((__float_as_uint(m) >> 23) & 255), 15);
  inv = __uint_as_float((uint32_t)(e - 14) << 23);
  return __uint_as_float((uint32_t)(268 - e) << 23);
}

template <int N>
__device__ __forceinline__ void gd_split(const float* x, float s, half_t* hi, half_t* lo) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float y = x[e] * s;
    hi[e] = (half_t)y;
    lo[e] = (half_t)(y - (float)hi[e]);
  }
}

__device__ __forceinline__ float gd_max4(const float4_t& x) {
  return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}
// Sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float gd_sum16(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Chunk slots: sequence i's start at q_start[i] / 64 + i, which leaves it ceil(n / 64) of them.
__device__ __forceinline__ int gd_base(const int* q_start, int i) { return q_start[i] / kC + i; }

// The sequence of chunk slot id: the last i < n with base(i) <= id.  The whole wave looks.
__device__ __forceinline__ int gd_seq_of(const int* __restrict__ q_start, int n, int id) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n - 1;
  while (hi > lo) {
    const int step = (hi - lo + 63) >> 6;
    const int at = lo + (lane + 1) * step;
    const bool below = at <= hi && gd_base(q_start, at) <= id;
    const int nlo = lo + __popcll(__builtin_amdgcn_ballot_w64(below)) * step;
    hi = min(hi, nlo + step - 1);
    lo = nlo;
  }
  return lo;
}

// Elements d .. d + 7 of a row of dk elements as fp32 or fp16, zeros past its end.  WIDE: rows
// of whole 16-byte pieces, d inside.
template <typename XT>
struct GdVec;
template <>
struct GdVec<half_t> {
  typedef half8_t T;
};
template <>
struct GdVec<float> {
  typedef float T __attribute__((ext_vector_type(8)));
};
template <bool WIDE, typename XT>
__device__ __forceinline__ typename GdVec<XT>::T gd_load8(const XT* row, int d, int dk) {
  typename GdVec<XT>::T x;
  if constexpr (WIDE) {
    constexpr int P = sizeof(XT) / 2;
    union {
      int4_t i[P];
      typename GdVec<XT>::T x;
    } u;
#pragma unroll
    for (int p = 0; p < P; ++p) u.i[p] = *(const int4_t*)(row + d + p * 4);
    x = u.x;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = d + e < dk ? row[d + e] : (XT)0;
  }
  return x;
}

// T and P of the chunks, and the sequences that are too short for chunks (token by token, by the
// first blocks: a launch of their own would take its time next to the others').  A block: one chunk of one value
// head; wave w forms the rows 16 w .. of k k^T and q k^T (fp16 rows: exact products; fp32 rows: fp32
// matrix instructions), whose operands are both rows of k and q.  T: the 16 x 16
// blocks on the diagonal by substitution, a column per lane; then pairs, T_10 = -T_11 A_10 T_00,
// twice.  A product's result has the layout of the next one's right operand, so only T's
// pieces go through LDS.  A chain of short steps, each waiting for the one before: 9 us for one chunk, and
// bound by how many blocks a CU holds (4): 4 prompts of up to 2600 tokens in 50 us, 74 with two blocks.
struct GdPrepLds {
  static constexpr int W = kC + 4;
  float a[kC * W], t[kC * W];
  double g[kC];
  float k2[kC], q2[kC], ki[kC], qi[kC], beta[kC], bad[kC];
};

template <int DK, bool FULL, typename XT>
__global__ __launch_bounds__(256, FULL && sizeof(XT) == 2 ? 4 : 3) void k_gd_prep(GdArgs a, char* __restrict__ ws,
                                                                         char* __restrict__ rows_ws, int from, int pieces,
                                                                         int slots) {
  constexpr int W = GdPrepLds::W, M = DK / 32;
  __shared__ __align__(16) union Lds {
    GdPrepLds p;
    GdRecLds<DK / 32> r;
  } lds;
  const long block = (long)blockIdx.y * gridDim.x + blockIdx.x, short_blocks = (long)pieces * a.nv * a.n_seqs;
  if (block < short_blocks) {
    const long hs = block / pieces;
    gd_recurrent<DK / 32, XT>(a, lds.r, (int)(block % pieces), (int)(hs % a.nv), (int)(hs / a.nv), from);
    return;
  }
  const int h = (int)((block - short_blocks) / slots), hk = h / a.rep, id = (int)((block - short_blocks) % slots);
  float *sa = lds.p.a, *st = lds.p.t;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), j = lane & 15, q = lane >> 4;
  const int seq = gd_seq_of(a.q_start, a.n_seqs, id);
  const int t0 = max(a.q_start[seq], 0), n = min(a.q_start[seq + 1], a.rows) - t0;
  const int c0 = (id - gd_base(a.q_start, seq)) * kC;
  if (n < from || c0 >= n || c0 < 0) return;
  const int live = min(n - c0, kC);

  auto row = [&](const void* x, long ld, int t) {
    return (const XT*)x + (long)(t0 + c0 + min(t, live - 1)) * ld + (long)hk * a.dk;
  };
  float4_t kk[4] = {}, qk[4] = {};
  {
    float g = 0.f, beta = 0.f;
    if (w == 0 && lane < live) {
      const long at = (long)(t0 + c0 + lane) * a.nv + h;
      g = a.g[at];
      beta = a.beta[at];
    }
    const int t = 16 * w + j;
    typename GdVec<XT>::T kf[M], qf[M];
    // Fp16 rows through LDS (where T and A come later), a row's 16-byte pieces at piece ^ (row & 7): a
    // fragment's lanes next to each other are in 16 rows, 64 accesses of the L1 for each load.
    half_t *lk = (half_t*)sa, *lq = (half_t*)st;
    auto place = [&](int r, int p) { return r * DK + ((p ^ (r & 7)) << 3); };
    if constexpr (sizeof(XT) == 2) {
      constexpr int PR = DK / 8;
#pragma unroll
      for (int i = 0; i < kC * PR / 256; ++i) {
        const int r = (i * 256 + tid) / PR, p = tid % PR;
        kf[i] = gd_load8<FULL, XT>(row(a.k, a.ldk, r), 8 * p, a.dk);
        qf[i] = gd_load8<FULL, XT>(row(a.q, a.ldq, r), 8 * p, a.dk);
      }
#pragma unroll
      for (int i = 0; i < kC * PR / 256; ++i) {
        const int r = (i * 256 + tid) / PR, p = tid % PR;
        *(half8_t*)&lk[place(r, p)] = kf[i];
        *(half8_t*)&lq[place(r, p)] = qf[i];
      }
      __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if constexpr (sizeof(XT) == 2) {
        kf[m] = *(const half8_t*)&lk[place(t, 4 * m + q)];
        qf[m] = *(const half8_t*)&lq[place(t, 4 * m + q)];
      } else {
        kf[m] = gd_load8<FULL, XT>(row(a.k, a.ldk, t), 32 * m + 8 * q, a.dk);
        qf[m] = gd_load8<FULL, XT>(row(a.q, a.ldq, t), 32 * m + 8 * q, a.dk);
      }
    }
    if (w == 0) {
      double G = g < -256.f ? -256.f : g;
#pragma unroll
      for (int o = 1; o < 64; o *= 2) {
        const double up = __shfl_up(G, o);
        if (lane >= o) G += up;
      }
      lds.p.g[lane] = G;
      lds.p.beta[lane] = beta;
      lds.p.bad[lane] = 0.f;
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b > w) continue;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        typename GdVec<XT>::T bf;
        if constexpr (sizeof(XT) == 2)
          bf = *(const half8_t*)&lk[place(16 * b + j, 4 * m + q)];
        else
          bf = gd_load8<FULL, XT>(row(a.k, a.ldk, 16 * b + j), 32 * m + 8 * q, a.dk);
        if constexpr (sizeof(XT) == 2) {
          kk[b] = gd_mfma(kf[m], bf, kk[b]);
          qk[b] = gd_mfma(qf[m], bf, qk[b]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float4_t x = {bf[e], bf[e + 1], bf[e + 2], bf[e + 3]};
            kk[b] = gd_mfma((float4_t){kf[m][e], kf[m][e + 1], kf[m][e + 2], kf[m][e + 3]}, x, kk[b]);
            qk[b] = gd_mfma((float4_t){qf[m][e], qf[m][e + 1], qf[m][e + 2], qf[m][e + 3]}, x, qk[b]);
          }
        }
      }
    }
    float k2 = 0.f, q2 = 0.f, km = 0.f, qm = 0.f;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (float)kf[m][e], y = (float)qf[m][e];
        k2 += x * x;
        q2 += y * y;
        km = fmaxf(km, fabsf(x));
        qm = fmaxf(qm, fabsf(y));
      }
    k2 = gd_sum16(k2);
    q2 = gd_sum16(q2);
    km = mx_rowmax4(km);
    qm = mx_rowmax4(qm);
    float ki, qi;
    const float ks = gd_scale(km, ki), qs = gd_scale(qm, qi);
    if (h == hk * a.rep) {  // k and q for all value heads of theirs
      char* to = rows_ws + ((long)id * a.nk + hk) * (2 * kRows<DK, XT>) + (w * M * 64 + lane) * 16;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        if constexpr (sizeof(XT) == 2) {
          half8_t x, y;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[e] = (half_t)((float)kf[m][e] * ks);
            y[e] = (half_t)((float)qf[m][e] * qs);
          }
          *(half8_t*)(to + m * 1024) = x;
          *(half8_t*)(to + kRows<DK, XT> + m * 1024) = y;
        } else {
          half8_t x[4];
          gd_split<8>((const float*)&kf[m], ks, (half_t*)&x[0], (half_t*)&x[1]);
          gd_split<8>((const float*)&qf[m], qs, (half_t*)&x[2], (half_t*)&x[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) *(half8_t*)(to + i * (kRows<DK, XT> / 2) + m * 1024) = x[i];
        }
      }
    }
    if (q == 0) {
      lds.p.k2[t] = a.norm ? 1.0f / sqrtf(k2 + 1e-6f) : 1.f;
      lds.p.q2[t] = (a.norm ? 1.0f / sqrtf(q2 + 1e-6f) : 1.f) * a.scale;
      lds.p.ki[t] = ki;
      lds.p.qi[t] = qi;
    }
  }
  __syncthreads();
  {
    float4_t ft, fq;  // beta |k|^-1 and scale |q|^-1 of the rows
    double gt[4];
    bool bad[4] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * w + 4 * q + e;
      gt[e] = lds.p.g[t];
      ft[e] = lds.p.beta[t] * lds.p.k2[t];
      fq[e] = lds.p.q2[t];
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      if (b > w) continue;
      const int s = 16 * b + j;
      const double gs = lds.p.g[s];
      const float ks = lds.p.k2[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int t = 16 * w + 4 * q + e;
        const float decay = expf((float)(gt[e] - gs)) * ks;
        float x = s < t ? ft[e] * decay * kk[b][e] : 0.f;
        // A row that is not finite (a NaN key, gate or decay) leaves T to the rows before it.
        const bool inf = !(fabsf(x) <= 3.0e38f);
        bad[e] |= inf;
        sa[t * W + s] = inf ? 0.f : x;
        qk[b][e] = s <= t ? fq[e] * decay * qk[b][e] : 0.f;  // P
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (bad[e]) lds.p.bad[16 * w + 4 * q + e] = 1.f;
  }
  {  // the diagonal block's inverse: column j, of this wave's own rows
    const float* d = sa + (16 * w) * W + 16 * w;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y[4] = {i == j ? 1.f : 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int m = 0; m < i; m += 4) {
        const float4_t c = *(const float4_t*)(d + i * W + m);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (m + e < i) y[e] -= c[e] * x[m + e];
      }
      x[i] = (y[0] + y[1]) + (y[2] + y[3]);
    }
    if (q == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) st[(16 * w + i) * W + 16 * w + j] = x[i];
  }
  __syncthreads();
  auto rows = [&](const float* x, int I, int J) { return *(const float4_t*)(x + (16 * I + j) * W + 16 * J + 4 * q); };
  auto cols = [&](const float* x, int I, int J) {
    const float* p = x + (16 * I + 4 * q) * W + 16 * J + j;
    return (float4_t){p[0], p[W], p[2 * W], p[3 * W]};
  };
  auto put = [&](int I, int J, const float4_t& z) {
#pragma unroll
    for (int e = 0; e < 4; ++e) st[(16 * I + 4 * q + e) * W + 16 * J + j] = -z[e];
  };
  if (w < 2) {
    const int I = 2 * w + 1, J = 2 * w;
    const float4_t y = gd_mfma(rows(sa, I, J), cols(st, J, J), (float4_t)0.f);
    put(I, J, gd_mfma(rows(st, I, I), y, (float4_t)0.f));
  }
  __syncthreads();
  {
    const int I = 2 + (w >> 1), J = w & 1;
    const float4_t c1 = cols(st, 1, J);
    float4_t y = gd_mfma(rows(sa, 2, 1), c1, (float4_t)0.f), y3 = (float4_t)0.f;
    if (I == 3) y3 = gd_mfma(rows(sa, 3, 1), c1, y3);
    if (J == 0) {
      const float4_t c0 = cols(st, 0, 0);
      y = gd_mfma(rows(sa, 2, 0), c0, y);
      if (I == 3) y3 = gd_mfma(rows(sa, 3, 0), c0, y3);
    }
    float4_t z = gd_mfma(rows(st, I, 2), y, (float4_t)0.f);
    if (I == 3) z = gd_mfma(rows(st, 3, 3), y3, z);
    put(I, J, z);
  }
  __syncthreads();
#pragma unroll
  for (int b = 0; b < 4; ++b) {  // A is done with
    if (b > w) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) sa[(16 * w + 4 * q + e) * W + 16 * b + j] = qk[b][e];
  }
  char* rec = ws + ((long)id * a.nv + h) * kRec;
  float* f = (float*)(rec + kOffF);
  const int t = tid >> 2, part = tid & 3;  // a row, 16 of its columns: both of this wave's own for P
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* x = (i ? sa : st) + t * W + 16 * part;
    float y[16], m = 0.f, inv;
    if (part <= t >> 4) {
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const float4_t c = *(const float4_t*)(x + e);
        m = fmaxf(m, gd_max4(c));
#pragma unroll
        for (int d = 0; d < 4; ++d) y[e + d] = c[d];
      }
    }
    m = fmaxf(m, mx_dpp<MX_DPP_XOR1>(m));
    m = fmaxf(m, mx_dpp<MX_DPP_XOR2>(m));
    const float s = gd_scale(m, inv);
    if (part <= t >> 4) {
      union {
        half_t h[2][16];
        half4_t v[2][4];
      } u;
      gd_split<16>(y, s, u.h[0], u.h[1]);
      // columns 16 part + 4 c of row t: lane 16 c + t % 16, the half of its piece that part says
      char* to = rec + i * kOffP + ((t >> 4) * 2 + (part >> 1)) * 1024 + (t & 15) * 16 + (part & 1) * 8;
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int c = 0; c < 4; ++c) *(half4_t*)(to + p * kPlane + c * 256) = u.v[p][c];
    }
    if (part == 0) f[(i ? kFp : kFt) * kC + t] = inv;
  }
  if (tid < kC) {
    const double G = lds.p.g[tid], end = lds.p.g[kC - 1];
    const float eg = expf((float)G), k2 = lds.p.k2[tid], ki = lds.p.ki[tid];
    f[kFa * kC + tid] = lds.p.bad[tid] != 0.f ? __builtin_nanf("") : eg * k2 * ki;
    f[kFb * kC + tid] = eg * lds.p.q2[tid] * lds.p.qi[tid];
    f[kFc * kC + tid] = expf((float)(end - G)) * k2 * ki;
    f[kFbeta * kC + tid] = lds.p.beta[tid];
    f[kFend * kC + tid] = expf((float)end);
  }
}

// A sequence's chunks in order, 16 columns of a head's state per block.  Wave rt has the tokens 16 rt ..
// of the chunk and the rows 16 SL rt .. of the state, in accumulators.  Per chunk three barriers:
//   the state's planes to LDS  | k^T S and q^T S; x to LDS, k to LDS  | u = T x to LDS  | o and S
// Bound by these steps one after the other: a chunk takes 2.3 us where a CU has one block and 3.3 with
// two (heads of 128 x 128, fp16).  Tried and slower: 32 columns per block of 8 waves (442 us
// against 380 for 4 prompts of up to 2600 tokens, early on), and 8 waves for 16 columns, four
// of them for k and T and four for q and P (180 us against 147).
// The next chunk's loads go out a few at a time (GD_HERE): four waves' 16-byte loads take the L1 about 64
// cycles, and a wave that issues nine in a row waits for most of them.
//
// A column's factor 2^e of the state's planes has to be known before all waves have the new state: from
// the bound e^G max|S| + 64 max|k| max|c u|, whose maxima went through LDS before (k's rows are
// scaled to 2^15, c u's are below 2^15 of their factor).  It may exceed the maximum by 2^15 before
// the 2^-39 above reaches fp32's own 2^-24.
//
// A NaN or infinity in x (a NaN in v is one of its column, in k of every column) would meet the zeros
// above T's diagonal: it is taken out, as it is out of u, and u, o and S from that row on are NaN, as
// token by token.
#define GD_HERE(x)                     \
  do {                                 \
    __builtin_amdgcn_sched_barrier(0); \
    x;                                 \
    __builtin_amdgcn_sched_barrier(0); \
  } while (0)

template <int DK, typename XT>
__global__ __launch_bounds__(256, 2) void k_gd_walk(GdArgs a, const char* __restrict__ ws,
                                                   const char* __restrict__ rows_ws, int from, int groups) {
  constexpr int SL = DK / 64, NP = sizeof(XT) == 2 ? 1 : 2, NC = 16, M = DK / 32;
  __shared__ __align__(16) half_t ss[2][NC * DK];        // the state [column][row]
  __shared__ __align__(16) half_t skey[NP][kC * DK];     // k [token][dim]
  __shared__ __align__(16) half_t sx[2][NC * kC];        // x, u, c u: [column][token]
  __shared__ __align__(16) half_t su[2][NC * kC], sd[2][NC * kC];
  __shared__ float sxi[4][NC], sui[4][NC], sdi[4][NC];   // their 2^e, per 16 tokens
  __shared__ float smax[2][4][NC];
  __shared__ int sfirst[2][NC];
  __shared__ __align__(16) float sf[2][kFactors * kC];
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), rt = wave;
  int seq = blockIdx.y;
  // The longest first: the last to end sets the time (8 ragged prompts of up to 600 rows: 81 us, 92 as they
  // come).  More than a wave looks at in one go come as they are.
  if (a.n_seqs > 1 && a.n_seqs <= 64) {
    const int at = min(lane, a.n_seqs - 1), size = min(a.q_start[at + 1], a.rows) - a.q_start[at];
    int before = 0;
    for (int i = 0; i < a.n_seqs; ++i) {
      const int other = __builtin_amdgcn_readlane(size, i);
      before += other > size || (other == size && i < lane);
    }
    seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < a.n_seqs && before == (int)blockIdx.y));
  }
  // Slices of a key head's value heads next to each other on one XCD: they read the same k, q, T, P.
  int hk, r;
  const int slices = (a.dv + NC - 1) / NC, per = slices * a.rep;
  if (groups) {
    hk = (blockIdx.x >> 3) / per * 8 + (blockIdx.x & 7);
    r = (blockIdx.x >> 3) % per;
  } else {
    hk = blockIdx.x / per;
    r = blockIdx.x % per;
  }
  const int h = hk * a.rep + r / slices, v0 = r % slices * NC;
  const int t0 = max(a.q_start[seq], 0), n = min(a.q_start[seq + 1], a.rows) - t0;
  if (n < from) return;
  const int in = a.slot_in[seq], out = a.slot_out[seq];
  const char* rec = ws + ((long)gd_base(a.q_start, seq) * a.nv + h) * kRec;
  const bool cl = v0 + j < a.dv;
  const long head = (long)a.dk * a.dv;
  const char* kq = rows_ws + ((long)gd_base(a.q_start, seq) * a.nk + hk) * (2 * kRows<DK, XT>) + rt * M * 1024;
  const XT* vp = (const XT*)a.v + (long)t0 * a.ldv + (long)h * a.dv + v0;
  XT* op = (XT*)a.o + (long)t0 * a.ldo + (long)h * a.dv + v0;

  float4_t s[SL];
#pragma unroll
  for (int i = 0; i < SL; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * (SL * rt + i) + 4 * q + e;
      s[i][e] = in >= 0 && in < a.n_slots && cl && d < a.dk
                    ? a.state[((long)in * a.nv + h) * head + (long)d * a.dv + v0 + j]
                    : 0.f;
    }

  // What a chunk reads, a chunk ahead: in registers until the products before it are done.
  half8_t kf[NP][M], qf[NP][M], tf[2][2], pf[2][2];
  XT vf[4];
  float4 ff;
  const int chunks = (n + kC - 1) / kC;
  // Rows past the end: k and q are the last one's again (k_gd_prep), v is 0 and so is beta; where that
  // row is finite so are x = 0 and all that follows of it.  All addresses are a base of the wave's and
  // an offset of the lane's that stays; what lies past a descriptor's end reads as 0 and
  // is not written, so nothing branches and each load is waited for by itself.
  const uint32_t lane16 = lane * 16, tid16 = 16 * min(tid, kFactors * kC / 4 - 1);
  int v_at[4], o_at[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int t = 16 * rt + 4 * q + e;
    v_at[e] = cl ? (t * (int)a.ldv + j) * (int)sizeof(XT) : -(1 << 31);
    o_at[e] = cl ? (t * (int)a.ldo + j) * (int)sizeof(XT) : -(1 << 31);
  }
  auto rows_of = [&](const XT* x, long ld, int c) {
    return __builtin_amdgcn_make_buffer_rsrc(
        (void*)(x + (long)c * kC * ld), (short)0,
        (int)(((min(n - c * kC, kC) - 1) * ld + min(NC, a.dv - v0)) * (long)sizeof(XT)), 0x00020000);
  };
  auto load_rows = [&](int c, int m) {
    const char* p = kq + (long)c * a.nk * (2 * kRows<DK, XT>);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      kf[i][m] = *(const half8_t*)(p + i * (kC * DK * 2) + m * 1024 + lane16);
      qf[i][m] = *(const half8_t*)(p + kRows<DK, XT> + i * (kC * DK * 2) + m * 1024 + lane16);
    }
  };
  auto load_v = [&](int c) {
    const mx_rsrc_t vr = rows_of(vp, a.ldv, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(XT) == 2)
        vf[e] = __builtin_bit_cast(XT, __builtin_amdgcn_raw_buffer_load_b16(vr, v_at[e], 0, 0));
      else
        vf[e] = __builtin_bit_cast(XT, __builtin_amdgcn_raw_buffer_load_b32(vr, v_at[e], 0, 0));
    }
  };
  auto load_tri = [&](int c, int off, half8_t (&x)[2][2]) {
    const char* p = rec + (long)c * a.nv * kRec + off + rt * 2048;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) x[i][b] = *(const half8_t*)(p + i * kPlane + 1024 * min(b, rt >> 1) + lane16);
  };
  auto load_factors = [&](int c) { ff = *(const float4*)(rec + (long)c * a.nv * kRec + kOffF + tid16); };
  auto factor = [&](const float* f, int k) { return *(const float4_t*)(f + k * kC + 16 * rt + 4 * q); };
  // Places in LDS, in halves; the swizzles are xors, so that places differ by xors of constants too.
  // [column][token]: 8-byte piece 4 b + q of the tokens 16 b .., at piece ^ column
  int pieces[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) pieces[b] = j * kC + ((4 * b + q) ^ j) * 4;
  const int pieces_rt = j * kC + ((4 * rt + q) ^ j) * 4;
  // the state [column][row]: 16-byte pieces at piece ^ (column & 7); written by 8 bytes, read by 16
  const int s_put = j * DK + (((2 * SL * rt + (q >> 1)) ^ (j & 7)) << 3) + (q & 1) * 4;
  const int s_get = j * DK + ((q ^ (j & 7)) << 3);
  // k [token][dim]: 16-byte pieces at piece ^ (2 (token & 3) + (token >> 2 & 1)); written by token 16 rt + j,
  // read transposed, 16 dims of the tokens 4 q .. by 16 lanes
  const int k_put = (16 * rt + j) * DK + ((q ^ (2 * (j & 3) + ((j >> 2) & 1))) << 3);
  const int k_get = (4 * q + (j >> 2)) * DK + (((2 * SL * rt + ((j & 3) >> 1)) ^ (2 * (j >> 2) + (q & 1))) << 3) + (j & 1) * 4;
  auto put = [&](half_t (&to)[2][NC * kC], const float4_t& x, float (&inv)[4][NC]) {
    float iv;
    const float sc = gd_scale(mx_rowmax4(gd_max4(x)), iv);
    half4_t p[2];
    gd_split<4>((const float*)&x, sc, (half_t*)&p[0], (half_t*)&p[1]);
    *(half4_t*)&to[0][pieces_rt] = p[0];
    *(half4_t*)&to[1][pieces_rt] = p[1];
    if (q == 0) inv[rt][j] = iv;
  };
  // sum over the token blocks up to rt of x (row planes) times what put() left; the other blocks' x is
  // not there: as zeros they keep the sum free of branches
  auto tri = [&](const half8_t (&x)[2][2], const half_t (&y)[2][NC * kC], const float (&inv)[4][NC]) {
    float4_t hh[4], mix[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const half4_t hi = *(const half4_t*)&y[0][pieces[b]], lo = *(const half4_t*)&y[1][pieces[b]];
      const half4_t zero = (half4_t)(half_t)0;
      const half4_t xh = b <= rt ? gd_half(x[0][b >> 1], b & 1) : zero, xl = b <= rt ? gd_half(x[1][b >> 1], b & 1) : zero;
      mix[b] = gd_mfma(xl, hi, (float4_t)0.f);
      hh[b] = gd_mfma(xh, hi, (float4_t)0.f);
      mix[b] = gd_mfma(xh, lo, mix[b]);
    }
    float4_t z = (float4_t)0.f;
#pragma unroll
    for (int b = 0; b < 4; ++b) z += (hh[b] + mix[b]) * inv[b][j];
    return z;
  };
  // Takes what is not finite out of x, and notes the first such token of the column.
  auto clean = [&](float4_t& x, int (&first)[NC]) {
    const float sum = (fabsf(x[0]) + fabsf(x[1])) + (fabsf(x[2]) + fabsf(x[3]));
    if (__builtin_amdgcn_ballot_w64(!(sum <= 3.0e38f)) == 0) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(fabsf(x[e]) <= 3.0e38f)) {
        atomicMin(&first[j], 16 * rt + 4 * q + e);
        x[e] = 0.f;
      }
  };

#pragma unroll
  for (int m = 0; m < M; ++m) load_rows(0, m);
  load_v(0);
  load_tri(0, 0, tf);
  load_tri(0, kOffP, pf);
  load_factors(0);
  float bound = 0.f;
#pragma unroll
  for (int i = 0; i < SL; ++i) bound = fmaxf(bound, gd_max4(s[i]));
  bound = mx_rowmax4(bound);
  if (q == 0) smax[1][rt][j] = bound;
  if (tid < NC) sfirst[0][tid] = kC;
  if (tid < kFactors * kC / 4) *(float4*)&sf[0][4 * tid] = ff;
  __syncthreads();
  bound = fmaxf(fmaxf(smax[1][0][j], smax[1][1][j]), fmaxf(smax[1][2][j], smax[1][3][j]));

  for (int c = 0; c < chunks; ++c) {
    const float* f = sf[c & 1];
    const int next = min(c + 1, chunks - 1);
    float sinv;
    {  // the state's planes
      const float sc = gd_scale(bound, sinv);
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < SL; ++i) {
        half4_t p[2];
        gd_split<4>((const float*)&s[i], sc, (half_t*)&p[0], (half_t*)&p[1]);
        const int at = s_put ^ (16 * i);
        *(half4_t*)&ss[0][at] = p[0];
        *(half4_t*)&ss[1][at] = p[1];
        m = fmaxf(m, gd_max4(s[i]));
      }
      m = mx_rowmax4(m);
      if (q == 0) smax[c & 1][rt][j] = m;
    }
    __syncthreads();
    float4_t o = (float4_t)0.f;
    {  // k^T S, q^T S
      GD_HERE(load_factors(next));
      float4_t x = (float4_t)0.f;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int at = (s_get ^ (32 * (m & 1))) + 64 * (m >> 1);
        const half8_t hi = *(const half8_t*)&ss[0][at], lo = *(const half8_t*)&ss[1][at];
        if constexpr (NP == 2) {
          x = gd_mfma(kf[NP - 1][m], hi, x);
          o = gd_mfma(qf[NP - 1][m], hi, o);
        }
        x = gd_mfma(kf[0][m], lo, x);
        o = gd_mfma(qf[0][m], lo, o);
        x = gd_mfma(kf[0][m], hi, x);
        o = gd_mfma(qf[0][m], hi, o);
      }
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int i = 0; i < NP; ++i) *(half8_t*)&skey[i][(k_put ^ (32 * (m & 1))) + 64 * (m >> 1)] = kf[i][m];
      GD_HERE(load_rows(next, 0));
      const float4_t fa = factor(f, kFa), fb = factor(f, kFbeta);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = fb[e] * ((float)vf[e] - fa[e] * (x[e] * sinv));
      clean(x, sfirst[c & 1]);
      o = o * sinv * factor(f, kFb);
      put(sx, x, sxi);
      GD_HERE(load_rows(next, 1));
    }
    __syncthreads();
    {  // u
      if constexpr (M > 2) GD_HERE(load_rows(next, 2));
      float4_t u = tri(tf, sx, sxi) * factor(f, kFt);
      if constexpr (M > 2) GD_HERE(load_rows(next, 3));
      clean(u, sfirst[c & 1]);
      put(su, u, sui);
      put(sd, u * factor(f, kFc), sdi);
    }
    GD_HERE(load_tri(next, 0, tf));
    __syncthreads();
    const int first = sfirst[c & 1][j];
    o += tri(pf, su, sui) * factor(f, kFp);
    GD_HERE(load_tri(next, kOffP, pf));
    load_v(next);
    const mx_rsrc_t to = rows_of(op, a.ldo, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const XT y = (XT)(16 * rt + 4 * q + e < first ? o[e] : __builtin_nanf(""));
      if constexpr (sizeof(XT) == 2)
        __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, y), to, o_at[e], 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, y), to, o_at[e], 0, 0);
    }
    const float end = f[kFend * kC];
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      s[i] *= end;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const half4_t hi = *(const half4_t*)&sd[0][pieces[b]], lo = *(const half4_t*)&sd[1][pieces[b]];
        const int at = (k_get ^ (16 * i)) + 16 * b * DK;
        auto key = [&](int p) {
          return __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((gd_lds_s4*)&skey[p][at]));
        };
        const half4_t kh = key(0);
        float4_t z = (float4_t)0.f;
        if constexpr (NP == 2) z = gd_mfma(key(NP - 1), hi, z);
        z = gd_mfma(kh, lo, z);
        z = gd_mfma(kh, hi, z);
        s[i] += z * sdi[b][j];
      }
      if (first < kC) s[i] = (float4_t)__builtin_nanf("");
    }
    bound = fmaxf(fmaxf(smax[c & 1][0][j], smax[c & 1][1][j]), fmaxf(smax[c & 1][2][j], smax[c & 1][3][j]));
    bound = end * bound + 0x1p36f * fmaxf(fmaxf(sdi[0][j], sdi[1][j]), fmaxf(sdi[2][j], sdi[3][j]));
    if (tid < kFactors * kC / 4) *(float4*)&sf[(c + 1) & 1][4 * tid] = ff;
    if (tid < NC) sfirst[(c + 1) & 1][tid] = kC;
  }
  if (out < 0 || out >= a.n_slots || !cl) return;
#pragma unroll
  for (int i = 0; i < SL; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = 16 * (SL * rt + i) + 4 * q + e;
      if (d < a.dk) a.state[((long)out * a.nv + h) * head + (long)d * a.dv + v0 + j] = s[i][e];
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

// Rows from which a sequence goes chunk by chunk.  32 heads of 128 x 128, one sequence: 16 rows 18 us token by token
// (24 rows about 25), any number up to 64 in a chunk 17; 32 sequences: 16 rows 96 us token by token (24 rows
// about 125), a chunk each 116 to 125.
constexpr int kFrom = 24;

bool chunked(const MxGatedDelta* d) {
  // (a chunk's rows of v and o go through a descriptor of 2^31 bytes)
  return d->head_dim_k <= 128 && d->ldv < (1 << 23) && d->ldo < (1 << 23) && (d->max_q < d->rows ? d->max_q : d->rows) >= kFrom;
}

template <int DK, bool FULL, typename XT>
int launch_chunked(const GdArgs& a, char* ws, hipStream_t s) {
  const int slots = a.rows / kC + a.n_seqs;
  char* rows_ws = ws + (size_t)slots * a.nv * kRec;
  mx_clear_error();
  const int pieces = mx_ceil_div(a.dv, kCols);
  hipLaunchKernelGGL((k_gd_prep<DK, FULL, XT>), dim3(pieces * a.n_seqs + slots, a.nv), dim3(256), 0, s, a, ws, rows_ws,
                     kFrom, pieces, slots);
  MX_TRY(mx_launch_status());
  hipLaunchKernelGGL((k_gd_walk<DK, XT>), dim3(mx_ceil_div(a.dv, 16) * a.nv, a.n_seqs), dim3(256), 0, s, a,
                     ws, rows_ws, kFrom, a.nk % 8 == 0);
  return mx_launch_status();
}

// Rows of q and k in whole 16-byte pieces.
template <typename XT>
bool full(const GdArgs& a) {
  const int esz = sizeof(XT);
  return (a.dk == 64 || a.dk == 128) && mx_aligned16(a.q) && mx_aligned16(a.k) && a.ldq * esz % 16 == 0 &&
         a.ldk * esz % 16 == 0;
}

template <typename XT>
int run(const MxGatedDelta* d, const GdArgs& a, char* ws, hipStream_t s) {
  if (!chunked(d)) return launch_recurrent<XT>(a, s);
  if (full<XT>(a)) return a.dk == 64 ? launch_chunked<64, true, XT>(a, ws, s) : launch_chunked<128, true, XT>(a, ws, s);
  return a.dk <= 64 ? launch_chunked<64, false, XT>(a, ws, s) : launch_chunked<128, false, XT>(a, ws, s);
}

}  // namespace

extern "C" int mx_gated_delta_rule_workspace_size(const MxGatedDelta* args, size_t* nbytes) {
  if (!nbytes) return MX_ERR_INVALID;
  MX_TRY(check(args));
  *nbytes = 0;
  if (!chunked(args)) return MX_OK;
  const size_t row = kC * (args->head_dim_k <= 64 ? 64 : 128) * (args->x_dtype == MX_DT_F16 ? 2 : 4);
  *nbytes = ((size_t)args->rows / kC + args->n_seqs) * (args->n_v_heads * (size_t)kRec + args->n_k_heads * 2 * row);
  return MX_OK;
}

extern "C" int mx_gated_delta_rule(const MxGatedDelta* args, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  size_t need;
  MX_TRY(mx_gated_delta_rule_workspace_size(args, &need));
  if (args->n_seqs == 0) return MX_OK;
  if (need && (!workspace || workspace_bytes < need)) return MX_ERR_WORKSPACE;
  if (need && !mx_aligned16(workspace)) return MX_ERR_ALIGNMENT;
  const GdArgs a = args_of(args);
  const hipStream_t s = (hipStream_t)stream;
  return args->x_dtype == MX_DT_F32 ? run<float>(args, a, (char*)workspace, s)
                                    : run<half_t>(args, a, (char*)workspace, s);
}
