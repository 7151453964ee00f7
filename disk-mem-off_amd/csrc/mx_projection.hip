// Projections of int8 rows by int8 weights, with low-rank adapters (mx_projection).
//
//   y[r, c] = sx[r] sw[c] sum_k q[r, k] w[c, k]  +  alpha_a sum_j t[j] b[a, c, j]  +  res[r, c],
//   t = x[r] a[a]^T, a the adapter of row r's sequence.
//
// The product's sums are int32 on v_mfma_i32_16x16x64_i8, exact at any order (k <= 65536), so splits of the
// reduction change no result.  With adapters a first launch (k_adapter_t) forms t for every row; the product's
// epilogue then adds t b^T to the scaled sums, so y is written once.
#include <float.h>
#include <limits.h>
#include <math.h>

#include "mx_common.h"
#include "mx_lds_copy.h"
#include "mx_paged.h"

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kOob = 0x80000000u;  // an offset outside every descriptor built here
constexpr int kSegs = MX_PROJECTION_MAX_SEGS;
constexpr int kRowsMax = 64;            // rows of k_rows
constexpr int kMaxK = 1 << 16;
constexpr int kMaxRank = 128;
constexpr int kReadRank = 64;           // ranks from which a tile's rows do not read b themselves
constexpr int kMaxLd = 1 << 22;         // 256 rows stay within a descriptor's 2 GiB
constexpr float kLo = 2048.f;           // the low plane of t is held times this
constexpr long kMaxThreads = (1l << 32) - 1;  // of a launch

__device__ __forceinline__ rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, (int)bytes, 0x00020000);
}

struct Seg {
  const int8_t* w;
  const half_t* ws;
  const half_t* a;
  const half_t* b;
  const void* res;
  void* y;
  long ldres, ldy;
  int n, vec;  // vec: 4 columns of y and res at once
  int blk0;    // blocks of the segments before
  int t;       // which of the t arrays (-1: no adapters)
};

// What k_adapter_t leaves.  For k_rows: t alpha in fp32, [seg][row][rr].  For k_tiles: t 2^s = hi + lo / kLo as two fp16
// planes, [seg][64 ranks][plane][row][64], and alpha 2^-s, [seg][row][rr / 32], s per 32 ranks such that the largest is
// in [2^13, 2^14).
struct Low {
  int* id;     // [rows] adapter, -1: none
  char* t;
  float* fac;
  int rr;      // rank rounded up to 32 (k_rows) or 64
};

struct Args {
  const int8_t* q;
  const float* sx;
  long ldq;
  int M, K, nseg, f16;  // f16: y and res are fp16
  int rank;
  Low low;
  Seg seg[kSegs];
};

// The scaled sum: the same roundings in every kernel, whatever is added to it.  sw first: sum sw lies between 2^-24 and
// 2^46, while sx sw may leave the range of fp32 (sx is down to 2^-126) where the result does not.
__device__ __forceinline__ float scaled(int sum, float sx, float sw) {
#pragma clang fp contract(off)
  return (float)sum * sw * sx;
}

// Four columns of row m from column n on, res added.
__device__ __forceinline__ void store4(const Seg& sg, bool f16, long m, int n, float4_t v) {
  if (f16) {
    half_t* y = (half_t*)sg.y + m * sg.ldy + n;
    const half_t* r = sg.res ? (const half_t*)sg.res + m * sg.ldres + n : nullptr;
    if (sg.vec && n + 3 < sg.n) {
      if (r) {
        const half4_t rv = *(const half4_t*)r;
        v += (float4_t){(float)rv[0], (float)rv[1], (float)rv[2], (float)rv[3]};
      }
      *(half4_t*)y = (half4_t){(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < sg.n) y[e] = (half_t)(r ? v[e] + (float)r[e] : v[e]);
    }
    return;
  }
  float* y = (float*)sg.y + m * sg.ldy + n;
  const float* r = sg.res ? (const float*)sg.res + m * sg.ldres + n : nullptr;
  if (sg.vec && n + 3 < sg.n) {
    if (r) v += *(const float4_t*)r;
    *(float4_t*)y = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < sg.n) y[e] = r ? v[e] + r[e] : v[e];
  }
}

// A wave's tile, rows m + 16 mi and columns n + 16 ni; `whole`: all its columns are there, on boundaries of four.  A
// row's residuals are loaded while the row before is stored.
template <typename T, int MF, int NF>
__device__ __forceinline__ void store_tile(const Seg& sg, int m, int n, int M, bool whole, const float4_t (&v)[MF][NF]) {
  typedef T t4 __attribute__((ext_vector_type(4)));
  if (!whole) {
#pragma unroll
    for (int mi = 0; mi < MF; ++mi)
#pragma unroll
      for (int ni = 0; ni < NF; ++ni)
        if (m + 16 * mi < M && n + 16 * ni < sg.n) store4(sg, sizeof(T) == 2, m + 16 * mi, n + 16 * ni, v[mi][ni]);
    return;
  }
  T* const y = (T*)sg.y + n;
  const T* const res = (const T*)sg.res + n;
  t4 r[2][NF];
  auto load = [&](int mi) {
#pragma unroll
    for (int ni = 0; ni < NF; ++ni) r[mi & 1][ni] = *(const t4*)(res + min(m + 16 * mi, M - 1) * sg.ldres + 16 * ni);
  };
  if (sg.res) load(0);
#pragma unroll
  for (int mi = 0; mi < MF; ++mi) {
    if (sg.res && mi + 1 < MF) load(mi + 1);
    float4_t o[NF];
#pragma unroll
    for (int ni = 0; ni < NF; ++ni) {
      o[ni] = v[mi][ni];
      if (sg.res)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[ni][e] += (float)r[mi & 1][ni][e];
    }
    if (m + 16 * mi < M)
#pragma unroll
      for (int ni = 0; ni < NF; ++ni)
        *(t4*)(y + (m + 16 * mi) * sg.ldy + 16 * ni) = (t4){(T)o[ni][0], (T)o[ni][1], (T)o[ni][2], (T)o[ni][3]};
  }
}

// ------------------------------------------------------------------------------------
// Operands in LDS.  A copy instruction moves 8 rows x 128 bytes straight there (the buffer loads' LDS mode); chunk c
// of row r lands in slot c ^ r of the row, which keeps the operand reads (lane (j, g) = (lane % 16, lane / 16) at
// step ks: row j of 16, chunk 4 ks + g) free of bank conflicts.  Read into registers directly, an operand would take
// a cache line for every 16 bytes: 16 rows per quarter wave.
// ------------------------------------------------------------------------------------
constexpr int kStage = 128;

__device__ __forceinline__ int copy_row(int lane) { return lane >> 3; }
__device__ __forceinline__ int copy_byte(int lane) { return ((lane & 7) ^ (lane >> 3)) * 16; }
__device__ __forceinline__ int read_at(int j, int g, int ks) {
  return (j >> 3) * 1024 + (j & 7) * 128 + (((ks * 4 + g) ^ (j & 7)) << 4);
}

// This wave's reads of LDS are done, and all but N of its copies into it; then every wave's.
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A wave's part of a reduction: stages [sb, se) of NT 16-row blocks of a times XG 8-row groups of x (rows of kb
// bytes, strides lda, ldx), through a ring of S slots of its own in LDS; no barrier.  The upper half of the last
// block of x is what follows the slot where XG is odd: its columns belong to no row.
template <int NT, int XG, int S>
struct WaveRing {
  static constexpr int MT = (XG + 1) / 2, NC = 2 * NT + XG, SLOT = NC * 1024;
  char* ring;
  rsrc_t ra, rx;
  uint32_t aoff[2 * NT], xoff[XG];
  int kb, sb, se;

  // Pieces past the row's end, and stages past the last, are zeros.
  __device__ __forceinline__ void issue(int st) const {
    char* slot = ring + (st - sb) % S * SLOT;
    const bool in = st < se && st * kStage + copy_byte(threadIdx.x & 63) < kb;
    const uint32_t at = (uint32_t)(st * kStage);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) mx_copy_to_lds16(ra, slot + i * 1024, in ? aoff[i] + at : kOob);
#pragma unroll
    for (int i = 0; i < XG; ++i) mx_copy_to_lds16(rx, slot + (2 * NT + i) * 1024, in ? xoff[i] + at : kOob);
  }
  __device__ __forceinline__ void start(int arows, uint32_t lda, int xrows, uint32_t ldx) {
    const int lane = threadIdx.x & 63, cr = copy_row(lane), cc = copy_byte(lane);
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) aoff[i] = 8 * i + cr < arows ? (8 * i + cr) * lda + cc : kOob;
#pragma unroll
    for (int i = 0; i < XG; ++i) xoff[i] = 8 * i + cr < xrows ? (8 * i + cr) * ldx + cc : kOob;
#pragma unroll
    for (int i = 0; i < S; ++i) issue(sb + i);
  }
  // use(a fragments, x fragments) per step.
  template <typename Use>
  __device__ __forceinline__ void run(Use use) const {
    const int j = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
    const int at[2] = {read_at(j, g, 0), read_at(j, g, 1)};
    for (int st = sb; st < se; ++st) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"((S - 1) * NC) : "memory");
      const char* slot = ring + (st - sb) % S * SLOT;
      int4_t a[2][NT], x[2][MT];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int i = 0; i < NT; ++i) a[ks][i] = *(const int4_t*)(slot + i * 2048 + at[ks]);
#pragma unroll
        for (int i = 0; i < MT; ++i) x[ks][i] = *(const int4_t*)(slot + (NT + i) * 2048 + at[ks]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the slot is free
      __builtin_amdgcn_sched_barrier(0);
      issue(st + S);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) use(a[ks], x[ks]);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
};

// ------------------------------------------------------------------------------------
// k_adapter_t: t = x a[adapter]^T.  A block takes 8 XG rows, one segment and 16 H ranks; its W waves split the
// reduction.  The adapter's rows are the MFMA's A operand, 16 rows of x the other: lane (j, g) = (lane % 16, lane /
// 16) ends with ranks 4 g .. + 3 of row j.  The rows may belong to several adapters: each of those is multiplied with
// all rows of the block, and a row keeps its own's (columns of the product do not mix, so another adapter's NaN stays
// away).  blockIdx.z deals the adapters of a tile to blocks.  Bound by latency: finding the adapters, the first
// copies and the sums of the W waves follow one another (48 rows of 20 adapters, three segments of rank 16 of 2048:
// 7.3 us; 3099 rows of rank 64: 17, 0.3 PFLOP/s).  The MFMA sums are fp32.
// ------------------------------------------------------------------------------------
struct LowArgs {
  const half_t* x;
  const int* q_start;
  const int* ids;
  const float* alpha;
  long ldx;
  int M, K, n_seqs, n_adapters, rank;
  int parts;  // rank groups of a block's size
  Low low;
  const half_t* a[kSegs];
};

// The adapters of rows t0 + 16 i + lane % 16 (callers converged).  Up to 64 sequences: their ends and adapters in one
// load each, which do not wait for one another.
template <int MT>
__device__ __forceinline__ void adapters_of(const LowArgs& p, int t0, int (&id)[MT]) {
  const int lane = threadIdx.x & 63, j = lane & 15;
  int first = 0, mine[MT];  // sequences that end up to a row, those before `first` aside
#pragma unroll
  for (int mi = 0; mi < MT; ++mi) mine[mi] = 0;
  if (p.n_seqs > 64) first = pk_seq_of(p.q_start, p.n_seqs, t0);
  int own = -1;
  for (int at = first;;) {  // 64 sequences at once
    const int s = at + lane;
    const int end = s < p.n_seqs ? p.q_start[s + 1] : INT_MAX;
    if (at == first && s < p.n_seqs) own = p.ids[s];
    int most = 0;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = __popcll(__builtin_amdgcn_ballot_w64(end <= t0 + 16 * mi + i));
        if (j == i) mine[mi] += c;
        most = max(most, c);
      }
    if (most < 64) break;
    at += 64;
  }
#pragma unroll
  for (int mi = 0; mi < MT; ++mi) {
    const int seq = first + mine[mi];
    int a = __shfl(own, mine[mi] & 63);
    if (mine[mi] >= 64 && seq < p.n_seqs) a = p.ids[seq];  // behind 64 more sequences, most of them empty
    id[mi] = seq < p.n_seqs && t0 + 16 * mi + j < p.M && a >= 0 && a < p.n_adapters ? a : -1;
  }
}

// A row's 8 ranks per lane group (32 in all) as two fp16 planes: v = hi + lo / kLo times the returned power of two, the
// largest in [2^13, 2^14).  The low plane keeps the magnitude of the high one, so both hold 11 bits and a sign down to
// 2^-26 of the largest: v is off by 2^-23 of itself there, and by 2^-49 of the largest below.  (Unscaled, the low
// plane would be subnormal from 2^-16 of the largest on, and columns that meet only small ranks would lose their
// digits.)  An infinity or a NaN stays in hi.
__device__ __forceinline__ float split(const float4_t (&v)[2], half8_t& hi, half8_t& lo) {
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = fabsf(v[k >> 2][k & 3]);
    if (a <= FLT_MAX) top = fmaxf(top, a);
  }
  top = mx_rowmax4(top);
  const int s = top > 0.f ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float u = ldexpf(v[k >> 2][k & 3], s);
    hi[k] = (half_t)u;
    const float left = (u - (float)hi[k]) * kLo;
    lo[k] = left - left == 0.f ? (half_t)left : (half_t)0.f;
  }
  return ldexpf(1.f, -s);
}

// Ranks r .. r + 3 (and, HF 2, 16 further) of a row of t, summed, into the workspace; `mine`: the lane's row is one of
// the adapter's.  Converged over the lanes of a row.
template <bool PLANES, int HF>
__device__ __forceinline__ void put_t(const LowArgs& p, int sg, long row, int r, bool mine, float alpha, const float4_t (&v)[HF]) {
  if constexpr (!PLANES) {
    if (mine) *(float4_t*)((float*)p.low.t + ((long)sg * p.M + row) * p.low.rr + r) = v[0] * alpha;
  } else {
    half8_t hi, lo;
    const float unit = split(v, hi, lo);
    half_t* out = (half_t*)p.low.t + ((((long)sg * (p.low.rr / 64) + r / 64) * 2) * p.M + row) * 64 + (r & 63);
    if (mine) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        *(half4_t*)(out + 16 * h) = (half4_t){hi[4 * h], hi[4 * h + 1], hi[4 * h + 2], hi[4 * h + 3]};
        *(half4_t*)(out + 64l * p.M + 16 * h) = (half4_t){lo[4 * h], lo[4 * h + 1], lo[4 * h + 2], lo[4 * h + 3]};
      }
    }
    if (mine && r % 32 < 4) p.low.fac[((long)sg * p.M + row) * (p.low.rr / 32) + r / 32] = alpha * unit;
  }
}

template <bool PLANES, int H, int XG, int W, int S>
__global__ __launch_bounds__(64 * W) void k_adapter_t(const LowArgs p) {
  constexpr int MT = XG / 2, SLOT = (2 * H + XG) * 1024;
  __shared__ __align__(1024) char lds[W * S * SLOT];
  static_assert(XG % 2 == 0 && H * MT * 1024 <= S * SLOT, "whole blocks, and the partial sums fit");
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = blockIdx.x * 16 * MT, sg = blockIdx.y / p.parts, r0 = blockIdx.y % p.parts * 16 * H;
  int id[MT];
  uint64_t todo[MT];
  adapters_of<MT>(p, t0, id);
#pragma unroll
  for (int mi = 0; mi < MT; ++mi) {
    if (blockIdx.y == 0 && blockIdx.z == 0 && wave == 0 && g == 0 && t0 + 16 * mi + j < p.M) p.low.id[t0 + 16 * mi + j] = id[mi];
    todo[mi] = __builtin_amdgcn_ballot_w64(id[mi] >= 0) & 0xFFFF;
  }
  const int rows = min(16 * MT, p.M - t0), ranks = min(16 * H, p.rank - r0);
  const rsrc_t rx = make_rsrc(p.x + t0 * p.ldx, (uint32_t)(2 * ((rows - 1) * p.ldx + p.K)));
  const int nst = (2 * p.K + kStage - 1) / kStage, sw = (nst + W - 1) / W;
  const int sb = min(nst, wave * sw), se = min(nst, sb + sw);
  for (int d = 0;; ++d) {
    int a = -1;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
      if (a < 0 && todo[mi]) a = __builtin_amdgcn_readlane(id[mi], __builtin_ctzll(todo[mi]));
    if (a < 0) break;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi) todo[mi] &= ~__builtin_amdgcn_ballot_w64(id[mi] == a);
    if (d % (int)gridDim.z != (int)blockIdx.z) continue;
    const float alpha = p.alpha[a];
    const rsrc_t ra = make_rsrc(p.a[sg] + ((long)a * p.rank + r0) * p.K, (uint32_t)(2 * ranks * p.K));
    float4_t acc[MT][H];
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
      for (int h = 0; h < H; ++h) acc[mi][h] = (float4_t){0.f, 0.f, 0.f, 0.f};
    WaveRing<H, XG, S> ring{lds + wave * S * SLOT, ra, rx, {}, {}, 2 * p.K, sb, se};
    ring.start(ranks, 2 * p.K, rows, (uint32_t)(2 * p.ldx));
    ring.run([&](const int4_t (&af)[H], const int4_t (&xf)[MT]) {
#pragma unroll
      for (int mi = 0; mi < MT; ++mi)
#pragma unroll
        for (int h = 0; h < H; ++h)
          acc[mi][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, af[h]),
                                                              __builtin_bit_cast(half8_t, xf[mi]), acc[mi][h], 0, 0, 0);
    });
    __syncthreads();
    float4_t(*const red)[MT][H][64] = (float4_t(*)[MT][H][64])lds;
#pragma unroll
    for (int mi = 0; mi < MT; ++mi)
#pragma unroll
      for (int h = 0; h < H; ++h) red[wave][mi][h][lane] = acc[mi][h];
    __syncthreads();
    // A wave finishes 16 ranks of 16 rows, or 32 with their common factor.  Ranks past the last are zeros.
    constexpr int HF = PLANES ? 2 : 1;
    static_assert(H % HF == 0, "whole parts");
    for (int part = wave; part < MT * H / HF; part += W) {
      const int mi = part / (H / HF), h0 = part % (H / HF) * HF;
      float4_t v[HF];
#pragma unroll
      for (int h = 0; h < HF; ++h) {
        v[h] = red[0][mi][h0 + h][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v[h] += red[w][mi][h0 + h][lane];
        // (rows of zeros by an infinity in x are NaN)
        if (r0 + 16 * (h0 + h) + 4 * g >= p.rank) v[h] = (float4_t){0.f, 0.f, 0.f, 0.f};
      }
      int own = id[0];
#pragma unroll
      for (int m = 1; m < MT; ++m) own = mi == m ? id[m] : own;
      put_t<PLANES, HF>(p, sg, t0 + 16 * mi + j, r0 + 16 * h0 + 4 * g, own == a, alpha, v);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------
// k_rows: up to 64 rows.  Bound by the weights' bytes: a block owns 16 NB columns and its W waves split the
// reduction, each with S stages of its own on their way (4 rows onto 32768 columns of 2048: 12.2 us, 5.5 TB/s; 1 row
// onto 9216: 5.9 us, 3.2 TB/s and a launch).  From some 16 rows on every block's copies of the rows count too.  The
// weights are the A operand, so a lane ends with columns 4 g .. + 3 of row j.
// ------------------------------------------------------------------------------------
template <int XG, int NB, int W, int S>
__global__ __launch_bounds__(64 * W) void k_rows(const Args p) {
  constexpr int MT = (XG + 1) / 2, SLOT = (2 * NB + XG) * 1024, NT = MT * NB;
  __shared__ __align__(1024) char lds[W * S * SLOT + XG % 2 * 1024];
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int s = 0;
#pragma unroll
  for (int i = 1; i < kSegs; ++i)
    if (i < p.nseg && (int)blockIdx.x >= p.seg[i].blk0) s = i;
  const Seg sg = p.seg[s];
  const int n0 = ((int)blockIdx.x - sg.blk0) * 16 * NB;
  const int K = p.K, M = p.M;

  int4_t acc[MT][NB];
#pragma unroll
  for (int mi = 0; mi < MT; ++mi)
#pragma unroll
    for (int f = 0; f < NB; ++f) acc[mi][f] = (int4_t){0, 0, 0, 0};
  const int cols = min(16 * NB, sg.n - n0);
  const int nst = sg.w ? (K + kStage - 1) / kStage : 0, sw = (nst + W - 1) / W;
  const int sb = min(nst, wave * sw), se = min(nst, sb + sw);
  WaveRing<NB, XG, S> ring{lds + wave * S * SLOT, make_rsrc(sg.w + (long)n0 * K, (uint32_t)(cols * K)),
                           make_rsrc(p.q, (uint32_t)((M - 1) * p.ldq + K)), {}, {}, K, sb, se};
  if (sg.w) {
    ring.start(cols, K, M, (uint32_t)p.ldq);
    ring.run([&](const int4_t (&wf)[NB], const int4_t (&xf)[MT]) {
#pragma unroll
      for (int f = 0; f < NB; ++f)
#pragma unroll
        for (int mi = 0; mi < MT; ++mi) acc[mi][f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[f], xf[mi], acc[mi][f], 0, 0, 0);
    });
  }
  // The waves' partial tiles; tile i (row tile i / NB, column tile i % NB) is finished by wave i % W.
  __syncthreads();
  int4_t(*const red)[NT][64] = (int4_t(*)[NT][64])lds;
  static_assert(NT * 1024 <= S * SLOT, "the partial sums fit");
#pragma unroll
  for (int i = 0; i < NT; ++i) red[wave][i][lane] = acc[i / NB][i % NB];
  __syncthreads();
  for (int i = wave; i < NT; i += W) {
    const int m = 16 * (i / NB) + j, n = n0 + 16 * (i % NB) + 4 * g;
    if (m >= M || n >= sg.n) continue;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    if (sg.w) {
      int4_t r = red[0][i][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) r += red[w][i][lane];
      const float sx = p.sx[m];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = scaled(r[e], sx, (float)sg.ws[min(n + e, sg.n - 1)]);
    }
    // Every lane reads its row's b: 16 rows have up to 16 adapters, and one after the other on the matrix unit costs
    // more (48 rows of 13 in a tile, rank 16: 12.7 us so, 14.9).
    const int a = sg.t >= 0 ? p.low.id[m] : -1;
    if (a >= 0) {
      const float* t = (const float*)p.low.t + ((long)sg.t * M + m) * p.low.rr;
      const half_t* b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] = sg.b + ((long)a * sg.n + min(n + e, sg.n - 1)) * p.rank;
      float4_t d = {0.f, 0.f, 0.f, 0.f};
      for (int r = 0; r < p.rank; r += 8) {
        const float4_t ta = *(const float4_t*)(t + r), tb = *(const float4_t*)(t + r + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const half8_t bv = *(const half8_t*)(b[e] + r);
#pragma unroll
          for (int k = 0; k < 8; ++k) d[e] = fmaf(k < 4 ? ta[k & 3] : tb[k & 3], (float)bv[k], d[e]);
        }
      }
      v += d;
    }
    store4(sg, p.f16, m, n, v);
  }
}

// ------------------------------------------------------------------------------------
// k_tiles: more rows.  BM x BN tiles; stages of 128 bytes per row of both operands go through a ring of NS slots that
// the block's waves share.  The weights are the A operand: a lane ends with four consecutive columns of a row.  Bound
// by the copies into LDS (1 KiB takes a CU some 22 cycles) as much as by the matrix units.
// ------------------------------------------------------------------------------------
// A call's tiles, and which of them a launch takes.  Tile t: groups of 4 row blocks, column block by column block, so
// that what runs at once on an XCD shares its operands through its L2.
struct Tiles {
  int mblk, ncol;  // row and column blocks
  int first, end;  // the tiles of the launch
};

template <int BM, int BN>
__device__ __forceinline__ void tile_at(const Args& p, const Tiles& ts, int t, int* m0, int* n0, int* seg) {
  const int grp = t / (4 * ts.ncol), gm = min(ts.mblk - 4 * grp, 4), in = t - grp * 4 * ts.ncol;
  const int cblk = in / gm;
  int s = 0;
#pragma unroll
  for (int i = 1; i < kSegs; ++i)
    if (i < p.nseg && cblk >= p.seg[i].blk0) s = i;
  *m0 = (4 * grp + in - cblk * gm) * BM;
  *n0 = (cblk - p.seg[s].blk0) * BN;
  *seg = s;
}

__device__ __forceinline__ int wave_min(int v) {
  v = min(v, __builtin_amdgcn_update_dpp(v, v, MX_DPP_XOR1, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(v, v, MX_DPP_XOR2, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(v, v, MX_DPP_HALF_MIRROR, 0xF, 0xF, false));
  v = min(v, __builtin_amdgcn_update_dpp(v, v, MX_DPP_MIRROR, 0xF, 0xF, false));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// v += alpha t b^T of a tile.  Adapter after adapter, lowest id first: the planes of t for the tile's rows and the
// adapter's rows of b are staged in LDS as the product's operands are, 64 ranks (128 bytes) at a time, and a row
// takes its own adapter's product.  Where the rows have many adapters and MANY, every lane reads its row's b itself.
// 3099 rows of rank 64 onto 9216 columns: 92 us, without adapters 71; staging and products take turns.  lo and hi are
// multiplied in turn into one sum, lo's scaled back in between (2 of the 92 us): t to 2^-23, where hi alone would be
// off by half a step of fp16.
template <bool MANY, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void add_adapters(const Args& p, const Seg& sg, char* lds, int m0, int n0,
                                             float4_t (&v)[WM / 16][WN / 16]) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN, MF = WM / 16, NF = WN / 16;
  constexpr int FT = BM / 8, FB = BN / 8;  // 1 KiB copies of a plane of t, of b
  const int M = p.M, N = sg.n, rank = p.rank;
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  const int mr = wm * WM + j, nw = n0 + wn * WN, nks = p.low.rr / 32;
  int all[BM / 64];  // adapters of the tile's rows
#pragma unroll
  for (int i = 0; i < BM / 64; ++i) all[i] = m0 + 64 * i + lane < M ? p.low.id[m0 + 64 * i + lane] : -1;
  auto after = [&](int last) {  // the next one
    int next = INT_MAX;
#pragma unroll
    for (int i = 0; i < BM / 64; ++i) next = all[i] > last ? min(next, all[i]) : next;
    return wave_min(next);
  };

  if constexpr (MANY) {
    // Rows of 4096 onto 4096 columns, rank 16.  128 rows in 64 x 64 tiles: 4 adapters 14.8 us staged, 16.0 read; 8 of
    // them 18.3 and 16.5, 64 of them 36.4 and 17.3.  600 rows in 128 x 128 tiles: 16 adapters 39.1 and 38.8, 32 of
    // them 52.4 and 39.6.  Rows of b of 64 ranks fill cache lines of their own, which every row of the tile reads
    // again: 128 rows of 64 adapters of 2048 onto 9216 columns 70.8 and 90.2 (48 ranks 74.3 and 57.1).
    const int most = rank * (BM * BN / 4096) * 3 / 8;
    int n = 0;
    if (rank < kReadRank)
      for (int a = after(-1); a != INT_MAX && n <= most; a = after(a)) ++n;
    if (n > most) {
#pragma unroll
      for (int mi = 0; mi < MF; ++mi) {
        const int m = min(m0 + mr + 16 * mi, M - 1), own = m0 + mr + 16 * mi < M ? p.low.id[m] : -1;
        const half_t* b = sg.b + (long)max(own, 0) * N * rank;
        const half_t* t = (const half_t*)p.low.t + ((long)sg.t * nks * M + m) * 64;
        for (int ks = 0; 32 * ks < rank; ++ks) {
          float d[NF][4] = {};
          for (int r = 32 * ks; r < min(rank, 32 * ks + 32); r += 8) {
            const half_t* tr = t + (long)(r >> 6) * 2 * M * 64 + (r & 63);
            const half8_t hi = *(const half8_t*)tr, lo = *(const half8_t*)(tr + 64l * M);
#pragma unroll
            for (int ni = 0; ni < NF; ++ni)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const half8_t bv = *(const half8_t*)(b + (long)min(nw + 16 * ni + 4 * g + e, N - 1) * rank + r);
#pragma unroll
                for (int k = 0; k < 8; ++k) d[ni][e] = fmaf(fmaf((float)lo[k], 1.f / kLo, (float)hi[k]), (float)bv[k], d[ni][e]);
              }
          }
          const float fac = p.low.fac[((long)sg.t * M + m) * nks + ks];
#pragma unroll
          for (int ni = 0; ni < NF; ++ni)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (own >= 0) v[mi][ni][e] = fmaf(fac, d[ni][e], v[mi][ni][e]);
        }
      }
      return;
    }
  }

  const int cr = copy_row(lane), cc = copy_byte(lane);
  const int rows = min(BM, M - m0), cols = min(BN, N - n0);
  int* const ids = (int*)(lds + (2 * FT + FB) * 1024);  // [BM]
  float* const facs = (float*)(ids + BM);               // [2][BM]
  static_assert(BM <= 64 * NW, "a thread for each row");
  const int first = after(-1);
  for (int r0 = 0; r0 < rank; r0 += 64) {
    const half_t* t = (const half_t*)p.low.t + (((long)sg.t * (nks / 2) + r0 / 64) * 2 * M + m0) * 64;
    for (int a = first; a != INT_MAX; a = after(a)) {
      wait_and_barrier<0>();  // the slots are free
      if (a == first) {
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
          const rsrc_t rt = make_rsrc(t + 64l * M * pl, (uint32_t)(rows * 128));
#pragma unroll
          for (int i = 0; i < FT / NW; ++i) {
            const int f = wave + i * NW;
            mx_copy_to_lds16(rt, lds + (pl * FT + f) * 1024, 8 * f + cr < rows ? (uint32_t)((8 * f + cr) * 128 + cc) : kOob);
          }
        }
        const int r = 64 * wave + lane;
        if (r < BM) {
          const long at = ((long)sg.t * M + m0 + min(r, rows - 1)) * nks + r0 / 32;
          ids[r] = r < rows ? p.low.id[m0 + r] : -1;
          facs[r] = p.low.fac[at];
          facs[BM + r] = p.low.fac[at + 1];
        }
      }
      const rsrc_t rb = make_rsrc(sg.b + ((long)a * N + n0) * rank, (uint32_t)(cols * rank * 2));
#pragma unroll
      for (int i = 0; i < FB / NW; ++i) {
        const int f = wave + i * NW;
        mx_copy_to_lds16(rb, lds + (2 * FT + f) * 1024,
                         8 * f + cr < cols && r0 * 2 + cc < rank * 2 ? (uint32_t)((8 * f + cr) * rank * 2 + r0 * 2 + cc) : kOob);
      }
      wait_and_barrier<0>();
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (r0 + 32 * ks >= rank) continue;
        const int at = read_at(j, g, ks);
        half8_t bf[NF];
#pragma unroll
        for (int ni = 0; ni < NF; ++ni) bf[ni] = *(const half8_t*)(lds + 2 * FT * 1024 + (wn * NF + ni) * 2048 + at);
#pragma unroll
        for (int mi = 0; mi < MF; ++mi) {
          const bool own = ids[mr + 16 * mi] == a;
          if (!__builtin_amdgcn_ballot_w64(own)) continue;
          const half8_t hi = *(const half8_t*)(lds + (wm * MF + mi) * 2048 + at);
          const half8_t lo = *(const half8_t*)(lds + FT * 1024 + (wm * MF + mi) * 2048 + at);
          const float fac = facs[ks * BM + mr + 16 * mi];
#pragma unroll
          for (int ni = 0; ni < NF; ++ni) {
            float4_t d = {0.f, 0.f, 0.f, 0.f};
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[ni], lo, d, 0, 0, 0) * (1.f / kLo);
            d = __builtin_amdgcn_mfma_f32_16x16x32_f16(bf[ni], hi, d, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (own) v[mi][ni][e] = fmaf(fac, d[e], v[mi][ni][e]);
          }
        }
      }
    }
  }
}

// This block's tiles first, first + step, ..: number u of the launch, `at(u)` its place (false: nothing there).
template <bool AD, int BM, int BN, int WM, int WN, int NS, typename At>
__device__ __forceinline__ void run_tiles(const Args& p, char* lds, int first, int end, int step, At at) {
  constexpr int NWN = BN / WN, NW = (BM / WM) * NWN;
  constexpr int MF = WM / 16, NF = WN / 16;
  constexpr int FA = BM / 8, FT = FA + BN / 8;  // 1 KiB copies per stage
  constexpr int SLOT = FT * 1024, DPW = FT / NW;
  static_assert(FA % NW == 0 && FT % NW == 0, "the copies divide among the waves");
  const int M = p.M, K = p.K;
  const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  const int cr = copy_row(lane), cc = copy_byte(lane);
  const int nst = (K + kStage - 1) / kStage;
  constexpr bool MANY = MF * NF <= 8;  // larger tiles would spill

  struct Place {
    int m0, n0, seg;
    rsrc_t rx, rw;
    uint32_t goff[DPW];
    bool mul;
  } now;
  auto go = [&](int u, Place* t) {
    for (; u < end; u += step)
      if (at(u, &t->m0, &t->n0, &t->seg)) break;
    if (u >= end) return u;
    const Seg& sg = p.seg[t->seg];
    t->mul = sg.w != nullptr;
    if (!t->mul) return u;
    const int rows = min(BM, M - t->m0), cols = min(BN, sg.n - t->n0);
    t->rx = make_rsrc(p.q + (long)t->m0 * p.ldq, (uint32_t)((rows - 1) * p.ldq + K));
    t->rw = make_rsrc(sg.w + (long)t->n0 * K, (uint32_t)(cols * K));
#pragma unroll
    for (int i = 0; i < DPW; ++i) {
      const int f = wave + i * NW;
      if (i * NW < FA) {
        const int row = 8 * f + cr;
        t->goff[i] = row < rows ? (uint32_t)(row * p.ldq) + cc : kOob;
      } else {
        const int row = 8 * (f - FA) + cr;
        t->goff[i] = row < cols ? (uint32_t)(row * K) + cc : kOob;
      }
    }
    return u;
  };
  // Copy i of stage st.  Pieces past the row's end, and stages past the last, are zeros.
  auto copy = [&](int st, int i) {
    mx_copy_to_lds16(i * NW < FA ? now.rx : now.rw, lds + (st % NS) * SLOT + (wave + i * NW) * 1024,
                     st * kStage + cc < K ? now.goff[i] + (uint32_t)(st * kStage) : kOob);
  };
  auto first_copies = [&]() {
    if (!now.mul) return;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < DPW; ++i) copy(st, i);
  };
  int rpos[2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) rpos[ks] = read_at(j, g, ks);

  int u = go(first, &now);
  if (u >= end) return;
  first_copies();
  for (;;) {
    int4_t acc[MF][NF];
#pragma unroll
    for (int mi = 0; mi < MF; ++mi)
#pragma unroll
      for (int ni = 0; ni < NF; ++ni) acc[mi][ni] = (int4_t){0, 0, 0, 0};
    if (now.mul) {
      // Operands of a step, weights first: 0 .. NF - 1 of them, then MF of rows.
      struct Frags {
        int4_t w[NF], x[MF];
      } f[2];
      auto read = [&](int st, int ks, Frags& f, int i) {
        const char* slot = lds + (st % NS) * SLOT + rpos[ks];
        if (i < NF) f.w[i] = *(const int4_t*)(slot + FA * 1024 + (wn * NF + i) * 2048);
        else f.x[i - NF] = *(const int4_t*)(slot + (wm * MF + i - NF) * 2048);
      };
      // A step's products, and between them the next step's reads and the copies of stage `ahead`: a wave that
      // issued them in a row would wait for the queues with its matrix unit idle.
      auto multiply = [&](const Frags& f, Frags& next, int st, int ks, int ahead) {
#pragma unroll
        for (int mi = 0; mi < MF; ++mi) {
#pragma unroll
          for (int i = (MF + NF) * mi / MF; i < (MF + NF) * (mi + 1) / MF; ++i) read(st, ks, next, i);
          if (ahead >= 0) {
#pragma unroll
            for (int i = DPW * mi / MF; i < DPW * (mi + 1) / MF; ++i) copy(ahead, i);
          }
#pragma unroll
          for (int ni = 0; ni < NF; ++ni)
            acc[mi][ni] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[ni], f.x[mi], acc[mi][ni], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      wait_and_barrier<(NS - 1) * DPW>();
#pragma unroll
      for (int i = 0; i < MF + NF; ++i) read(0, 0, f[0], i);
      for (int st = 0; st < nst; ++st) {
        multiply(f[0], f[1], st, 1, -1);
        // This wave's copies of stage st + 1 are done and its reads of stage st, then every wave's: the slot is
        // free for stage st + NS.  (Past the last stage the reads and copies are of no use, and of no harm.)
        wait_and_barrier<(NS - 2) * DPW>();
        multiply(f[1], f[0], st + 1, 0, st + NS);
      }
    }
    // Scales ahead of the next tile's copies, which run while this one is stored.
    const int mw = now.m0 + wm * WM + j, nw = now.n0 + wn * WN;
    const Seg sg = p.seg[now.seg];
    const int N = sg.n;
    float sx[MF];
    half_t sw[NF][4];
    if (now.mul) {
#pragma unroll
      for (int mi = 0; mi < MF; ++mi) sx[mi] = p.sx[min(mw + 16 * mi, M - 1)];
#pragma unroll
      for (int ni = 0; ni < NF; ++ni)
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[ni][e] = sg.ws[min(nw + 16 * ni + 4 * g + e, N - 1)];
    }
    const int m0 = now.m0, n0 = now.n0;
    const bool mul = now.mul;
    u = go(u + step, &now);
    const bool adapted = AD && sg.t >= 0;
    if (u < end && !adapted) {
      wait_and_barrier<0>();  // every wave is past its last reads, no copy is on its way
      first_copies();
    }
    const bool whole = sg.vec && nw + WN <= N;
    float4_t v[MF][NF];
#pragma unroll
    for (int mi = 0; mi < MF; ++mi)
#pragma unroll
      for (int ni = 0; ni < NF; ++ni)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[mi][ni][e] = mul ? scaled(acc[mi][ni][e], sx[mi], (float)sw[ni][e]) : 0.f;
    if (adapted) {
      add_adapters<MANY, BM, BN, WM, WN>(p, sg, lds, m0, n0, v);
      if (u < end) {
        wait_and_barrier<0>();
        first_copies();
      }
    }
    if (p.f16) store_tile<half_t, MF, NF>(sg, mw, nw + 4 * g, M, whole, v);
    else store_tile<float, MF, NF>(sg, mw, nw + 4 * g, M, whole, v);
    if (u >= end) break;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy into LDS outlives the block
}

// One tile per block.
template <bool AD, int BM, int BN, int WM, int WN, int NS, int OCC>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, OCC) void k_tiles(const Args p, const Tiles ts) {
  __shared__ __align__(1024) char lds[NS * (BM + BN) * kStage];
  // Consecutive tiles run on one XCD (block b goes to XCD b % 8).
  const int total = gridDim.x, b = blockIdx.x, id = total % 8 == 0 ? (b & 7) * (total >> 3) + (b >> 3) : b;
  run_tiles<AD, BM, BN, WM, WN, NS>(p, lds, id, total, total, [&](int u, int* m0, int* n0, int* seg) {
    tile_at<BM, BN>(p, ts, u, m0, n0, seg);
    return true;
  });
}

// A block per CU, each with the same number of 256 x 256 tiles; what is left of them (ts.first on) in quarters.
// Bound by the matrix units and the copies next to them: 4096 rows onto 9216 columns of 2048 86 us, 1.80 POP/s.
template <bool AD>
__global__ __launch_bounds__(512, 1) void k_rounds(const Args p, const Tiles ts) {
  __shared__ __align__(1024) char lds[2 * 512 * kStage];
  const int per = gridDim.x >> 3, b = blockIdx.x, id = gridDim.x % 8 == 0 ? (b & 7) * per + (b >> 3) : b;
  run_tiles<AD, 256, 256, 128, 64, 2>(p, lds, id, ts.first, gridDim.x, [&](int u, int* m0, int* n0, int* seg) {
    tile_at<256, 256>(p, ts, u, m0, n0, seg);
    return true;
  });
  if (ts.first == ts.end) return;
  __syncthreads();
  run_tiles<AD, 128, 128, 64, 32, 4>(p, lds, 4 * ts.first + id, 4 * ts.end, gridDim.x, [&](int u, int* m0, int* n0, int* seg) {
    tile_at<256, 256>(p, ts, u >> 2, m0, n0, seg);
    *m0 += (u & 2) * 64;
    *n0 += (u & 1) * 128;
    return *m0 < p.M && *n0 < p.seg[*seg].n;
  });
}

// ---- the launch ----------------------------------------------------------------------

struct Plan {
  bool few;           // k_rows
  int rr;             // rank rounded up
  int nt;             // segments with adapters
  size_t t, fac, bytes;  // workspace: offsets and size
};

int min_of(int a, int b) { return a < b ? a : b; }

int check(const MxProjection* p, const MxAdapters* ad) {
  if (!p || !p->segs || p->n_segs < 1 || p->rows < 0 || p->k <= 0 || (p->q == nullptr) != (p->q_scale == nullptr) ||
      (p->y_dtype != MX_DT_F32 && p->y_dtype != MX_DT_F16))
    return MX_ERR_INVALID;
  if (p->n_segs > kSegs || p->rows >= (1 << 24) || p->k > kMaxK || p->k % 16) return MX_ERR_UNSUPPORTED;
  if (p->q && p->ldq < p->k) return MX_ERR_INVALID;
  if (p->q && p->ldq >= kMaxLd) return MX_ERR_UNSUPPORTED;
  if (!mx_aligned16(p->q) || (p->q && p->ldq % 16) || (uintptr_t)p->q_scale % 4) return MX_ERR_ALIGNMENT;
  const int e = p->y_dtype == MX_DT_F16 ? 2 : 4;
  for (int i = 0; i < p->n_segs; ++i) {
    const MxProjectionSeg& s = p->segs[i];
    if (!s.y || s.n <= 0 || s.ldy < s.n || (s.res && s.ldres < s.n) || (!s.w && !s.a)) return MX_ERR_INVALID;
    if ((s.w == nullptr) != (s.w_scale == nullptr) || (s.a == nullptr) != (s.b == nullptr)) return MX_ERR_INVALID;
    if ((s.w && !p->q) || (s.a && !ad) || (s.res == s.y && s.ldres != s.ldy)) return MX_ERR_INVALID;
    if (s.n >= (1 << 24)) return MX_ERR_UNSUPPORTED;
    if (!mx_aligned16(s.w) || !mx_aligned16(s.a) || !mx_aligned16(s.b) || (uintptr_t)s.w_scale % 2 ||
        (uintptr_t)s.y % e || (uintptr_t)s.res % e)
      return MX_ERR_ALIGNMENT;
  }
  if (ad) {
    if (!ad->x || !ad->q_start || !ad->ids || !ad->alpha || ad->n_seqs < 0 || ad->n_adapters <= 0 || ad->rank <= 0 ||
        ad->ldx < p->k)
      return MX_ERR_INVALID;
    if (ad->n_seqs > 65535 || ad->rank % 8 || ad->rank > kMaxRank || ad->ldx >= kMaxLd) return MX_ERR_UNSUPPORTED;
    if (!mx_aligned16(ad->x) || ad->ldx % 8 || (uintptr_t)ad->q_start % 4 || (uintptr_t)ad->ids % 4 ||
        (uintptr_t)ad->alpha % 4)
      return MX_ERR_ALIGNMENT;
  }
  return MX_OK;
}

Plan plan(const MxProjection* p, const MxAdapters* ad) {
  Plan l = {};
  l.few = p->rows <= kRowsMax;
  for (int i = 0; ad && i < p->n_segs; ++i) l.nt += p->segs[i].a != nullptr;
  if (!l.nt || p->rows == 0) return l;
  l.rr = l.few ? (ad->rank + 31) / 32 * 32 : (ad->rank + 63) / 64 * 64;
  const size_t n = (size_t)l.nt * p->rows * l.rr;
  l.t = mx_align_up((size_t)p->rows * 4, 256);
  l.fac = l.t + mx_align_up(n * 4, 256);
  l.bytes = l.fac + n / 32 * 4;
  return l;
}

// Numbers the segments' column blocks of BN columns.
template <int BM, int BN>
long number(Args& a, Tiles* ts) {
  ts->mblk = mx_ceil_div(a.M, BM);
  ts->ncol = 0;
  for (int i = 0; i < a.nseg; ++i) {
    a.seg[i].blk0 = ts->ncol;
    ts->ncol += mx_ceil_div(a.seg[i].n, BN);
  }
  return (long)ts->mblk * ts->ncol;
}

template <int BM, int BN, int WM, int WN, int NS, int OCC, bool ADAPTERS = true>
int launch_tiles(Args& a, hipStream_t s) {
  Tiles ts = {};
  const long blocks = number<BM, BN>(a, &ts);
  if (blocks * (BM / WM) * (BN / WN) * 64 > kMaxThreads) return MX_ERR_UNSUPPORTED;
  auto* kern = k_tiles<false, BM, BN, WM, WN, NS, OCC>;
  if constexpr (ADAPTERS) {
    if (a.low.id) kern = k_tiles<true, BM, BN, WM, WN, NS, OCC>;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3((BM / WM) * (BN / WN) * 64), 0, s, a, ts);
  return mx_launch_status();
}

int launch_rounds(Args& a, hipStream_t s) {
  Tiles ts = {};
  const long tiles = number<256, 256>(a, &ts);
  if (tiles > INT_MAX / 8) return MX_ERR_UNSUPPORTED;
  ts.end = (int)tiles;
  const int left = ts.end % 256;
  ts.first = left > 128 ? ts.end : ts.end - left;
  hipLaunchKernelGGL(a.low.id ? k_rounds<true> : k_rounds<false>, dim3(256), dim3(512), 0, s, a, ts);
  return mx_launch_status();
}

template <bool PLANES, int H, int XG, int W, int S>
void launch_t(LowArgs& p, int nt, int z, hipStream_t s) {
  const int tiles = mx_ceil_div(p.M, 8 * XG);
  p.parts = mx_ceil_div(p.rank, 16 * H);
  if (z == 0) z = mx_ceil_div(2048, tiles * nt * p.parts);
  z = min_of(min_of(z, 16), min_of(p.M, min_of(p.n_adapters, p.n_seqs)));
  hipLaunchKernelGGL((k_adapter_t<PLANES, H, XG, W, S>), dim3(tiles, nt * p.parts, z < 1 ? 1 : z), dim3(64 * W), 0, s, p);
}

// Few blocks: a ring per wave hides the copies' latency (2329 rows onto 32 ranks of 4096: 8.5 us, one slot 11.1).
// Past a block per CU, one slot each and more blocks at once (1500 rows onto three segments of 64 ranks of 2048: 11.8
// us, 13.5).  Many rows of more than 32 ranks: 32 rows by 64 ranks, which halves the copies (3099 rows onto three of
// 64: 16.7 us, 20.7; 1500: 14.1, 11.8).  The grid's third axis deals a tile's adapters to blocks while there are not
// many, since a tile of two takes twice a tile's time otherwise (128 sequences of a row: 39 us with one block, 9 with
// 16; those 3099 rows 22.2 and 16.7; 24000 rows, which keep one: 56 us, 70 with four).  Up to 64 rows a wave has up
// to 16 stages of its reduction, four of them on their way, and eight waves share longer ones (9 rows of 8192 values:
// 10.8 us, 9.4; 64 rows and ranks 16.1, 12.3; of 2048 values 7.5, 7.9; 4096 8.9, 9.3).
void launch_low(LowArgs& p, int nt, bool few, hipStream_t s) {
  if (few) return p.K > 4096 ? launch_t<false, 1, 2, 8, 2>(p, nt, 16, s) : launch_t<false, 1, 2, 4, 4>(p, nt, 16, s);
  const long blocks = (long)mx_ceil_div(p.M, 16) * nt * mx_ceil_div(p.rank, 32);
  if (blocks <= 256) return launch_t<true, 2, 2, 4, 2>(p, nt, 0, s);
  if (p.rank > 32 && blocks > 768) return launch_t<true, 4, 4, 4, 1>(p, nt, 0, s);
  launch_t<true, 2, 2, 4, 1>(p, nt, 0, s);
}

template <int XG, int NB, int S>
void launch_rows(Args& a, hipStream_t s) {
  int blocks = 0;
  for (int i = 0; i < a.nseg; ++i) {
    a.seg[i].blk0 = blocks;
    blocks += mx_ceil_div(a.seg[i].n, 16 * NB);
  }
  hipLaunchKernelGGL((k_rows<XG, NB, 4, S>), dim3(blocks), dim3(256), 0, s, a);
}

// With a block of 16 columns per CU at most, a ring of S slots per wave hides the copies' latency (48 rows onto 2048
// columns of 4096: 6.8 us, one slot 7.9; two blocks still fit a CU's LDS).  Past that, blocks of one slot do: more of
// them share a CU, and they start at once (1 row onto 9216 columns of 2048: 5.9 us, four slots 7.0; 48 rows 8.8, two
// slots 10.0).  Many blocks of more than 16 rows take 32 columns each, to copy the rows half as often (32 rows onto
// 32768: 13.8 us, 16 columns 15.2; onto 9216 both 7.0).
template <int XG, int S>
void launch_rows_by_blocks(Args& a, long blocks, hipStream_t s) {
  if (blocks <= 256) return launch_rows<XG, 1, S>(a, s);
  if constexpr (XG > 2) {
    if (blocks > 640) return launch_rows<XG, 2, 1>(a, s);
  }
  launch_rows<XG, 1, 1>(a, s);
}

long column_blocks(const Args& a, int bn) {
  long n = 0;
  for (int i = 0; i < a.nseg; ++i) n += mx_ceil_div(a.seg[i].n, bn);
  return n;
}

int launch_few(Args& a, hipStream_t s) {
  const long blocks = column_blocks(a, 16);
  if (a.M <= 8) launch_rows_by_blocks<1, 4>(a, blocks, s);
  else if (a.M <= 16) launch_rows_by_blocks<2, 4>(a, blocks, s);
  else if (a.M <= 32) launch_rows_by_blocks<4, 3>(a, blocks, s);
  else if (a.M <= 48) launch_rows_by_blocks<6, 2>(a, blocks, s);
  else launch_rows_by_blocks<8, 2>(a, blocks, s);
  return mx_launch_status();
}

// The smallest tile whose blocks run at once: at few blocks a stage of one is paced by the latency of its copies, so
// small tiles on more CUs are faster (330 rows onto 2048 columns of 4096: 64 x 64 10.4 us, 128 x 128 16.4, 256 x 256
// 26); past one round the larger tile's fewer copies per product count (1700 rows: 28.2, 19.4 and 28).  Past all of
// them rounds of 256 x 256 (4096 rows onto 9216 of 2048: 90 us, 128 x 128 tiles 100), but tiles no higher than the
// rows (128 rows onto 131072: 128 x 128 73 us, 84; 64 rows: 64 x 128 58, 64 x 64 68).
//
// `mix`: adapters that 128 rows may have, on the mean of the batch (where its long sequences lie the device knows alone).
// Where they are many, tiles whose rows can read b themselves (512 sequences of a row onto 9216 columns, rank 16: of 64
// adapters 54 us, 256 x 128 tiles 84; of 256 adapters 74, 180; of 16 48, 44; of 4 32, 29), up to 1024 rows (2048 of 4
// adapters: 89 us, 67).  Tiles of more than 2048 outputs a wave take an adapter after the other, however many: 2048 rows of
// 256 adapters 272 us (187 in 128 x 64 tiles), a prompt of 900 rows beside 100 sequences of a row, 64 adapters, 125 us
// (1000 rows of one adapter 41).
int launch_many(Args& a, int mix, hipStream_t s) {
  auto tiles = [&](int bm, int bn) { return column_blocks(a, bn) * mx_ceil_div(a.M, bm); };
  if (tiles(64, 64) <= 256) return launch_tiles<64, 64, 32, 16, 4, 2>(a, s);
  if (tiles(128, 64) <= 256) return launch_tiles<128, 64, 32, 32, 3, 1>(a, s);
  if (tiles(64, 64) <= 512) return launch_tiles<64, 64, 32, 16, 4, 2>(a, s);  // two per CU
  if (a.rank < kReadRank && mix > 2 * a.rank && a.M <= 1024 && tiles(128, 64) * 512 <= kMaxThreads)
    return launch_tiles<128, 64, 32, 32, 3, 1>(a, s);
  if (a.M <= kRowsMax) return launch_tiles<64, 128, 32, 32, 3, 1, false>(a, s);  // (with adapters: k_rows)
  if (tiles(128, 128) <= 256) return launch_tiles<128, 128, 64, 32, 4, 1>(a, s);
  if (tiles(256, 128) <= 256) return launch_tiles<256, 128, 64, 64, 3, 1>(a, s);
  if (a.M <= 128 || tiles(128, 128) <= 512) return launch_tiles<128, 128, 64, 64, 2, 2>(a, s);
  return launch_rounds(a, s);
}

}  // namespace

extern "C" int mx_projection_workspace_size(const MxProjection* args, const MxAdapters* adapters, size_t* nbytes) {
  if (!nbytes) return MX_ERR_INVALID;
  MX_TRY(check(args, adapters));
  *nbytes = plan(args, adapters).bytes;
  return MX_OK;
}

extern "C" int mx_projection(const MxProjection* args, const MxAdapters* adapters, void* workspace,
                             size_t workspace_bytes, void* stream) {
  MX_TRY(check(args, adapters));
  if (args->rows == 0) return MX_OK;
  const Plan l = plan(args, adapters);
  if (l.bytes && (!workspace || workspace_bytes < l.bytes)) return MX_ERR_WORKSPACE;
  if (l.bytes && !mx_aligned16(workspace)) return MX_ERR_ALIGNMENT;
  const hipStream_t s = (hipStream_t)stream;
  char* const ws = (char*)workspace;
  Args a = {};
  a.q = args->q;
  a.sx = args->q_scale;
  a.ldq = args->ldq;
  a.M = args->rows;
  a.K = args->k;
  a.nseg = args->n_segs;
  a.f16 = args->y_dtype == MX_DT_F16;
  if (l.bytes) a.low = Low{(int*)ws, ws + l.t, (float*)(ws + l.fac), l.rr};
  LowArgs la = {};
  int nt = 0;
  const size_t four = a.f16 ? 8 : 16;
  for (int i = 0; i < a.nseg; ++i) {
    const MxProjectionSeg& g = args->segs[i];
    const bool vec = (uintptr_t)g.y % four == 0 && g.ldy % 4 == 0 &&
                     (!g.res || ((uintptr_t)g.res % four == 0 && g.ldres % 4 == 0));
    a.seg[i] = Seg{(const int8_t*)g.w, (const half_t*)g.w_scale, (const half_t*)g.a, (const half_t*)g.b, g.res, g.y,
                   g.ldres, g.ldy, g.n, vec, 0, g.a ? nt : -1};
    if (g.a) la.a[nt++] = (const half_t*)g.a;
  }
  mx_clear_error();
  if (nt) {
    a.rank = adapters->rank;
    la.x = (const half_t*)adapters->x;
    la.q_start = adapters->q_start;
    la.ids = adapters->ids;
    la.alpha = adapters->alpha;
    la.ldx = adapters->ldx;
    la.M = a.M;
    la.K = a.K;
    la.n_seqs = adapters->n_seqs;
    la.n_adapters = adapters->n_adapters;
    la.rank = adapters->rank;
    la.low = a.low;
    launch_low(la, nt, l.few, s);
    MX_TRY(mx_launch_status());
  }
  // Without adapters, tiles take over from 33 rows where the columns give two blocks of 16 to a CU: their waves share
  // the copies (40 rows onto 9216 columns of 2048: 7.6 us, 8.0; 64 rows 7.8, 9.3; onto 4096 columns 7.1, 5.6).  With
  // adapters the rows' own sums cost less (48 rows with as many adapters onto 16384: 14.1 us, 15.6).
  if (l.few && (nt || a.M <= 32 || column_blocks(a, 16) <= 512)) return launch_few(a, s);
  const int mix = nt ? min_of(adapters->n_adapters, mx_ceil_div(128 * adapters->n_seqs, a.M)) : 0;
  return launch_many(a, mix, s);
}
