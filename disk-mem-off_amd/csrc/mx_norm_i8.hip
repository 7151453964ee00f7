// Residual addition, RMS norm and rows in 8 bits (mx_add_rmsnorm_i8):
//   v = x + res;  y = v / sqrt(mean(v^2) + eps) * w;  s = max|y| / 127;  q = rint(y / s).
//
// One pass over the data: a row's values stay in registers between the reductions and the codes.  With
// p = v w the norm's factor r is common to the row, so max|y| = r max|p|, and the sum of squares and the
// maximum are reduced together, behind one barrier.
//
// 64 bits.  A code is the nearest whole number of y / s; 32-bit sums and products would move some 1e-5 of the values
// over a border, by a whole step each.  Bound by the rows' bytes all the same: 2777 rows of 5120 (fp32 in, residual,
// sum and fp16 rows) 45 us, 4.7 TB/s; 4096 of 2048 29 us; one row 3.9 us, a launch.
#include <float.h>

#include "mx_common.h"

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxHidden = 1024 * 16;  // 1024 threads of 16 values (of 32: spills)
constexpr int kLaunchRows = 1 << 21;   // a launch holds less than 2^32 threads, a row takes up to 1024

struct NormArgs {
  const void* x;
  const void* res;
  void* sum;
  const void* w;
  int8_t* q;
  float* qs;
  half_t* h16;
  long ldx, ldres, ldsum, ldq, ldh;
  int rows, hidden, xdt, rdt, pdt, norm;
  float eps;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const long b = __builtin_bit_cast(long, v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, 0xF, 0xF, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (long)(uint32_t)lo | (long)hi << 32);
}

__device__ __forceinline__ double readlane64(double v, int lane) {
  const long b = __builtin_bit_cast(long, v);
  const int lo = __builtin_amdgcn_readlane((int)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
  return __builtin_bit_cast(double, (long)(uint32_t)lo | (long)hi << 32);
}

__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<MX_DPP_XOR1>(v);
  v += dpp64<MX_DPP_XOR2>(v);
  v += dpp64<MX_DPP_HALF_MIRROR>(v);
  v += dpp64<MX_DPP_MIRROR>(v);
  return (readlane64(v, 0) + readlane64(v, 16)) + (readlane64(v, 32) + readlane64(v, 48));
}

__device__ __forceinline__ double wave_max64(double v) {
  v = fmax(v, dpp64<MX_DPP_XOR1>(v));
  v = fmax(v, dpp64<MX_DPP_XOR2>(v));
  v = fmax(v, dpp64<MX_DPP_HALF_MIRROR>(v));
  v = fmax(v, dpp64<MX_DPP_MIRROR>(v));
  return fmax(fmax(readlane64(v, 0), readlane64(v, 16)), fmax(readlane64(v, 32), readlane64(v, 48)));
}

// Through fp32: 2^-24 on top of the half step of fp16 (a direct rounding is a library routine).
__device__ __forceinline__ half_t f16(double v) { return (half_t)(float)v; }

// Element i (VEC: elements i .. i + 3) of a row.
template <bool VEC>
__device__ __forceinline__ void load(const void* row, int dt, int i, float (&o)[VEC ? 4 : 1]) {
  if constexpr (VEC) {
    const float4 v = mx_load_param4(row, dt, i);
    o[0] = v.x;
    o[1] = v.y;
    o[2] = v.z;
    o[3] = v.w;
  } else {
    o[0] = mx_load_param(row, dt, i);
  }
}

__device__ __forceinline__ const char* row_of(const void* p, long r, long ld, int dt) {
  return (const char*)p + r * ld * (dt == MX_DT_F16 ? 2 : 4);
}

// T threads per row (a wave's worth: four rows per block), each with NC groups of 4 elements: of 4
// consecutive ones (VEC: hidden a multiple of 4, every array on a boundary of 4 elements), or of 4 that
// are T apart.
template <int T, int NC, bool VEC>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_norm_i8(const NormArgs a) {
  constexpr int E = VEC ? 4 : 1, G = 4 / E * NC;  // elements per load, loads
  constexpr int NWV = T / 64;
  __shared__ double part[2][NWV < 4 ? 4 : NWV];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row = T < 256 ? (long)blockIdx.x * 4 + wave : blockIdx.x;
  if (T < 256 && row >= a.rows) return;
  const int t = T < 256 ? lane : threadIdx.x;
  const char* x = row_of(a.x, row, a.ldx, a.xdt);
  const char* res = a.res ? row_of(a.res, row, a.ldres, a.rdt) : nullptr;
  char* sum = a.sum ? (char*)row_of(a.sum, row, a.ldsum, a.rdt) : nullptr;
  const int H = a.hidden;

  float xv[G][E], rv[G][E], wv[G][E];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = (g * T + t) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) xv[g][e] = 0.f, rv[g][e] = 0.f, wv[g][e] = 1.f;
    if (i < H) {
      load<VEC>(x, a.xdt, i, xv[g]);
      if (res) load<VEC>(res, a.rdt, i, rv[g]);
      if (a.w) load<VEC>(a.w, a.pdt, i, wv[g]);
    }
  }
  double p[G][E], ss = 0.0, top = 0.0;
  bool bad = false;  // fmax drops a NaN
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = (g * T + t) * E;
    double v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = (double)xv[g][e] + (double)rv[g][e];
      ss += v[e] * v[e];
      p[g][e] = v[e] * (double)wv[g][e];
      bad |= !(fabs(p[g][e]) <= DBL_MAX);
      top = fmax(top, fabs(p[g][e]));
    }
    if (sum && i < H) {
      if constexpr (VEC) {
        if (a.rdt == MX_DT_F16)
          *(half4_t*)(sum + 2l * i) = (half4_t){f16(v[0]), f16(v[1]), f16(v[2]), f16(v[3])};
        else
          *(float4*)(sum + 4l * i) = make_float4((float)v[0], (float)v[1], (float)v[2], (float)v[3]);
      } else {
        if (a.rdt == MX_DT_F16) *(half_t*)(sum + 2l * i) = f16(v[0]);
        else *(float*)(sum + 4l * i) = (float)v[0];
      }
    }
  }
  if (__builtin_amdgcn_ballot_w64(bad)) top = (double)INFINITY;
  ss = wave_sum64(ss);
  top = wave_max64(top);
  if constexpr (NWV > 1) {
    if (lane == 0) {
      part[0][wave] = ss;
      part[1][wave] = top;
    }
    __syncthreads();
    ss = 0.0;
    top = 0.0;
#pragma unroll
    for (int w = 0; w < NWV; ++w) {
      ss += part[0][w];
      top = fmax(top, part[1][w]);
    }
  }
  // A row of zeros stays one where eps is 0.
  const double mean = ss / (double)H + (double)a.eps;
  const double r = !a.norm ? 1.0 : mean == 0.0 ? 0.0 : 1.0 / sqrt(mean);
  float s = (float)(top * r / 127.0);
  const bool lost = !(top <= DBL_MAX) || !(s <= FLT_MAX);
  s = lost ? __builtin_nanf("") : top * r == 0.0 ? 1.f : fmaxf(s, FLT_MIN);
  const double step = lost ? 0.0 : r / (double)s;
  if (a.qs && t == 0) a.qs[row] = s;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = (g * T + t) * E;
    if (i >= H) continue;
    if (a.q) {
      int c[E];
#pragma unroll
      for (int e = 0; e < E; ++e) c[e] = lost ? 0 : (int)rint(p[g][e] * step);
      int8_t* q = a.q + row * a.ldq + i;
      if constexpr (VEC)
        *(uint32_t*)q = (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 |
                        (uint32_t)(c[3] & 255) << 24;
      else
        *q = (int8_t)c[0];
    }
    if (a.h16) {
      half_t* h = a.h16 + row * a.ldh + i;
      if constexpr (VEC)
        *(half4_t*)h = (half4_t){f16(p[g][0] * r), f16(p[g][1] * r), f16(p[g][2] * r), f16(p[g][3] * r)};
      else
        *h = f16(p[g][0] * r);
    }
  }
}

// Rows as they are, in 8 bits (and fp16): the maximum is exact in 32 bits, and so is a code that lies clear of a
// border: x times the rounded factor is off by 127 2^-23 at most.  One within 1e-4 of a border, 2e-4 of them, is
// worked out in 64 bits.  4096 rows of 4096 fp16 values: 12.4 us, 18.2 in 64 bits throughout.
template <int T, int NC, bool VEC>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_quantise_i8(const NormArgs a) {
  constexpr int E = VEC ? 4 : 1, G = 4 / E * NC;
  constexpr int NWV = T / 64;
  __shared__ float part[NWV < 4 ? 4 : NWV];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row = T < 256 ? (long)blockIdx.x * 4 + wave : blockIdx.x;
  if (T < 256 && row >= a.rows) return;
  const int t = T < 256 ? lane : threadIdx.x;
  const char* x = row_of(a.x, row, a.ldx, a.xdt);
  const int H = a.hidden;
  float xv[G][E], top = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = (g * T + t) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) xv[g][e] = 0.f;
    if (i < H) load<VEC>(x, a.xdt, i, xv[g]);
  }
  bool bad = false;
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      bad |= !(fabsf(xv[g][e]) <= FLT_MAX);
      top = fmaxf(top, fabsf(xv[g][e]));
    }
  if (__builtin_amdgcn_ballot_w64(bad)) top = INFINITY;
  top = mx_wave_max(top);
  if constexpr (NWV > 1) {
    if (lane == 0) part[wave] = top;
    __syncthreads();
    top = 0.f;
#pragma unroll
    for (int w = 0; w < NWV; ++w) top = fmaxf(top, part[w]);
  }
  const bool lost = !(top <= FLT_MAX);
  const float s = lost ? __builtin_nanf("") : top == 0.f ? 1.f : fmaxf((float)((double)top / 127.0), FLT_MIN);
  const double step = lost ? 0.0 : 1.0 / (double)s;
  const float near = (float)step;
  if (a.qs && t == 0) a.qs[row] = s;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int i = (g * T + t) * E;
    if (i >= H) continue;
    if (a.q) {
      int c[E];
      bool border = false;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = xv[g][e] * near, r = rintf(y);
        border |= fabsf(y - r) > 0.4999f;
        c[e] = lost ? 0 : (int)r;
      }
      if (border && !lost) {
#pragma unroll
        for (int e = 0; e < E; ++e) c[e] = (int)rint((double)xv[g][e] * step);
      }
      int8_t* q = a.q + row * a.ldq + i;
      if constexpr (VEC)
        *(uint32_t*)q = (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 |
                        (uint32_t)(c[3] & 255) << 24;
      else
        *q = (int8_t)c[0];
    }
    if (a.h16) {
      half_t* h = a.h16 + row * a.ldh + i;
      if constexpr (VEC) *(half4_t*)h = (half4_t){(half_t)xv[g][0], (half_t)xv[g][1], (half_t)xv[g][2], (half_t)xv[g][3]};
      else *h = (half_t)xv[g][0];
    }
  }
}

template <int T, bool VEC>
void launch(int nc, const NormArgs& a, hipStream_t s) {
  const bool plain = !a.res && !a.sum && !a.norm;
  const dim3 grid(T < 256 ? mx_ceil_div(a.rows, 4) : a.rows), block(T < 256 ? 256 : T);
  auto* kern = plain ? k_quantise_i8<T, 1, VEC> : k_norm_i8<T, 1, VEC>;
  if (nc > 1) kern = plain ? k_quantise_i8<T, 2, VEC> : k_norm_i8<T, 2, VEC>;
  if constexpr (T > 64) {
    if (nc > 2) kern = plain ? k_quantise_i8<T, 3, VEC> : k_norm_i8<T, 3, VEC>;
    if (nc > 3) kern = plain ? k_quantise_i8<T, 4, VEC> : k_norm_i8<T, 4, VEC>;
  }
  hipLaunchKernelGGL(kern, grid, block, 0, s, a);
}

// Threads per row: of many rows as few as leave registers for several rows on a CU (2777 rows of 5120, 512 threads:
// 45.0 us, 256 with 20 values each 46.6; 4096 rows of 4096 the other way round, 13.5 and 12.4), of few as many as
// there are (200 rows of 5120: 6.8 us, 300 on 512 threads 8.4).
template <bool VEC>
void launch_rows(const NormArgs& a, hipStream_t s) {
  if (a.hidden <= 512) return launch<64, VEC>(mx_ceil_div(a.hidden, 256), a, s);
  if (a.hidden <= 4096 && a.rows > 256) return launch<256, VEC>(mx_ceil_div(a.hidden, 1024), a, s);
  if (a.hidden <= 8192 && a.rows > 256) return launch<512, VEC>(mx_ceil_div(a.hidden, 2048), a, s);
  launch<1024, VEC>(mx_ceil_div(a.hidden, 4096), a, s);
}

int esz(int dt) { return dt == MX_DT_F16 ? 2 : 4; }
bool float_type(int dt) { return dt == MX_DT_F32 || dt == MX_DT_F16; }

}  // namespace

extern "C" int mx_add_rmsnorm_i8(const MxNormRows* args, void* stream) {
  const MxNormRows* n = args;
  if (!n || !n->x || n->rows < 0 || n->hidden <= 0 || (n->q == nullptr) != (n->q_scale == nullptr) ||
      (!n->q && !n->h16) || !float_type(n->x_dtype))
    return MX_ERR_INVALID;
  if ((n->res || n->sum) && !float_type(n->res_dtype)) return MX_ERR_INVALID;
  if (n->norm_w && (!n->norm || !float_type(n->param_dtype))) return MX_ERR_INVALID;
  if (n->norm && !(n->eps >= 0.f)) return MX_ERR_INVALID;
  const long H = n->hidden;
  if (n->ldx < H || (n->res && n->ldres < H) || (n->sum && n->ldsum < H) || (n->q && n->ldq < H) ||
      (n->h16 && n->ldh < H))
    return MX_ERR_INVALID;
  // The values a row writes are read by the same thread before: at the same place only.
  if (n->sum && n->sum == n->res && n->ldsum != n->ldres) return MX_ERR_INVALID;
  if (n->sum && n->sum == n->x && (n->ldsum != n->ldx || n->res_dtype != n->x_dtype)) return MX_ERR_INVALID;
  if (H > kMaxHidden || n->rows >= (1 << 24)) return MX_ERR_UNSUPPORTED;
  const int xs = esz(n->x_dtype), rs = esz(n->res_dtype), ps = esz(n->param_dtype);
  if ((uintptr_t)n->x % xs || (uintptr_t)n->res % rs || (uintptr_t)n->sum % rs || (uintptr_t)n->norm_w % ps ||
      (uintptr_t)n->q_scale % 4 || (uintptr_t)n->h16 % 2)
    return MX_ERR_ALIGNMENT;
  if (n->rows == 0) return MX_OK;
  NormArgs a{n->x,   n->res,   n->sum,   n->norm_w, n->q,    n->q_scale,   (half_t*)n->h16, n->ldx,     n->ldres,
             n->ldsum, n->ldq, n->ldh, n->rows,   n->hidden, n->x_dtype, n->res_dtype,    n->param_dtype, n->norm,
             n->eps};
  auto on = [](const void* p, long ld, int e) { return !p || ((uintptr_t)p % (4 * e) == 0 && ld % 4 == 0); };
  const bool vec = H % 4 == 0 && on(n->x, n->ldx, xs) && on(n->res, n->ldres, rs) && on(n->sum, n->ldsum, rs) &&
                   on(n->norm_w, 0, ps) && on(n->q, n->ldq, 1) && on(n->h16, n->ldh, 2);
  for (long r0 = 0; r0 < n->rows; r0 += kLaunchRows) {
    a.rows = (int)(n->rows - r0 < kLaunchRows ? n->rows - r0 : kLaunchRows);
    a.x = (const char*)n->x + r0 * n->ldx * xs;
    if (n->res) a.res = (const char*)n->res + r0 * n->ldres * rs;
    if (n->sum) a.sum = (char*)n->sum + r0 * n->ldsum * rs;
    if (n->q) a.q = n->q + r0 * n->ldq, a.qs = n->q_scale + r0;
    if (n->h16) a.h16 = (half_t*)n->h16 + r0 * n->ldh;
    mx_clear_error();
    if (vec) launch_rows<true>(a, (hipStream_t)stream);
    else launch_rows<false>(a, (hipStream_t)stream);
    MX_TRY(mx_launch_status());
  }
  return MX_OK;
}
