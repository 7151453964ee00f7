// Attention of new rows over a paged key/value cache (mx_paged_attn).
//
// Rows.  All query heads of a key/value head read the same keys, so the rows of a sequence and
// key/value head are counted token-major with the head inside: row r is token r / G, head r % G
// of the group (G = n_heads / n_kv_heads).  A decode step of one token fills G rows, a chunk of
// n tokens n G, and a row tile takes consecutive rows.
//
// Products.  Per 32 keys (two sub-tiles of 16, each inside one page):
//   S^T = K Q^T   (A = 16 key rows from memory order, B = 16 query rows): lane (j, g) = (lane %
//                 16, lane / 16) gets S[key 4 g + r][row j], so a row's softmax is in its lanes
//   O^T += V^T P  (A = 16 dims x 32 keys, B = the lane's own probabilities): the k-slot (g, e)
//                 stands for key 4 g + e of sub-tile 0 (e < 4) and key 4 g + e - 4 of sub-tile 1.
// Values lie row-major in the pages; the transposing LDS reads (ds_read_b64_tr) give a lane the
// 8 keys of one dim.
//
// Softmax in the base-2 domain with a lazy reference: a row's reference m moves only when a tile's
// maximum passes it by more than kTau, so probabilities stay below 2^kTau (fp16 holds them)
// and the accumulators are rescaled on few tiles.  Statistics and sums are fp32; the probabilities
// are rounded to fp16 for the second product.
//
// Int8 pages: with a score s in the base-2 domain and the value row's scale w, the weight that
// meets the int8 values is 2^s w = 2^(s + log2 w); its reference is taken over s + log2 w, the
// accumulators take 2^(s + log2 w - m) and the row sum the same divided by w (fp32), so no
// range of scales leaves fp16's.
//
// What is masked stays out: scores of keys past the row, past the cache or on no page are
// replaced before the maximum; value rows no row of the wave sees are replaced by zeros, and
// non-finite values that only some rows of a tile see (a NaN in the newest token) are taken out
// of the matrix product and added to the rows that see them one by one.
#include <math.h>

#include <type_traits>

#include "mx_common.h"
#include "mx_lds_copy.h"
#include "mx_paged.h"

namespace {

constexpr float kTau = 8.f;
constexpr float kLow = -3.0e38f;  // a reference below every score
constexpr float kLog2e = 1.4426950408889634f;

typedef __amdgpu_buffer_rsrc_t pa_rsrc_t;
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef int int2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int pa_ceil(int a, int b) { return (a + b - 1) / b; }

struct PaArgs {
  const void* q;
  void* out;
  const float* gate;
  long ldq, ldo, ldg;
  int nh, group;
  float scale;
};

// A register's value the compiler knows nothing of: what is worked out from it is worked out
// here, per tile, and holds no registers across the loop.
__device__ __forceinline__ int pa_opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ int pa_opaque_s(int v) {  // a uniform one
  asm volatile("" : "+s"(v));
  return v;
}
// The lane's number, from the execution mask: it holds no register where it is not needed.
__device__ __forceinline__ int pa_lane() {
  return pa_opaque(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)));
}

constexpr int kKeysRows = 16;

// Work items.  A call's rows are cut into row tiles (RT rows of one sequence and key/value head) and
// a tile's keys into ranges of `len` keys; an item is one range of one tile.  Every block works
// the same schedule out of the batch's lengths: len such that about `target` items of equal
// size come out (sum over the tiles of their keys / target, within [least, most]), the items in
// order of sequence, range, tile.  A tile's ranges are as long as each other, in whole steps (12 ragged
// chunks over up to 7000 keys: 132 us, 138 with a short last range), and the tiles of every other range come
// in the other order, so that a CU's two blocks get a long and a short one of a causal chunk (2048
// rows over 8192 keys: 260 us, 269).  The blocks of a head take its items in turn.
// An item whose tile fits one range writes its rows; the others leave sums, relative to their
// reference, in a slot for k_pa_join.
struct PaSched {
  int target, least, most;
  int slots;     // at most so many items of a head
  int end;       // rows of sums in all
  float* po;     // [nkv][slots][RT][hd]
  float2* ml;    // [nkv][slots][RT]: reference, sum
  int4_t* rows;  // [rows][nh]: where a row's first partial sum lies in them, the step to the next, how many
};

// A sequence's part, one sequence per lane.
struct PaSeq {
  int q0, m, len;   // first row, rows, cached tokens
  int tiles, keys;  // row tiles; keys its last row sees
  int items;
};

struct PaWork {
  int len, items;   // keys per range, items of a head
  PaSeq own;        // up to 64 sequences: the lane's, and the items before its end
  int incl;
};

// What an item is.
struct PaTile {
  int seq, row0, nrows;  // first row; rows of the sequence and head
  int first;             // q_start of the sequence
  int pos0;              // position of the sequence's row 0
  int kend;              // keys the tile's last row sees
  int k0;                // first key of the range
  int len, ranges;       // keys of its ranges, how many
  int slot, tiles;       // the range's slot for sums; the tile's next range's is `tiles` further
};

template <int RT>
__device__ __forceinline__ PaSeq pa_seq(const PkBatch& b, const PkCache& c, int group, int s) {
  PaSeq q;
  const bool in = s < b.n_seqs;
  const int at = in ? s : 0;
  q.q0 = b.q_start[at];
  q.m = in ? min(b.q_start[at + 1], b.rows) - q.q0 : 0;
  q.len = b.kv_len[at];
  q.tiles = q.m > 0 ? (int)(((long)q.m * group + RT - 1) / RT) : 0;
  q.keys = (int)max(0l, min((long)min(q.len, b.max_kv), (long)b.max_pages << c.ps_log));
  return q;
}

__device__ __forceinline__ int pa_scan(int v) {  // inclusive, over the wave
  const int lane = pa_lane();
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const int up = __shfl_up(v, o);
    if (lane >= o) v += up;
  }
  return v;
}

__device__ __forceinline__ int pa_items(const PaSeq& q, int len) {
  return q.tiles * max(1, pa_ceil(q.keys, len));
}

// The schedule (wave-uniform but for `own`; callers converged).
template <int RT>
__device__ __forceinline__ PaWork pa_schedule(const PkBatch& b, const PkCache& c, const PaSched& sp, int group,
                                              int per) {
  const int lane = pa_lane();
  PaWork w;
  w.own = pa_seq<RT>(b, c, group, lane);
  float total = (float)w.own.tiles * (float)w.own.keys, tiles = (float)w.own.tiles;
  for (int s = 64 + lane; s - lane < b.n_seqs; s += 64) {
    const PaSeq q = pa_seq<RT>(b, c, group, s);
    total += (float)q.tiles * (float)q.keys;
    tiles += (float)q.tiles;
  }
  total = mx_wave_sum(total) * (float)c.nkv;
  tiles = mx_wave_sum(tiles);
  // Every tile rounds its last range up: half an item each is set aside for that.  k_pa_keys and k_pa_f32,
  // bound by the copies that a block has in flight, let the ranges grow instead until one item per block is
  // enough, where there are no more tiles than blocks (48 ragged sequences of up to 12000 keys in fp16:
  // 32 us, 44 with a second item for some).
  const int most = min(per, sp.slots);
  const bool fits = RT == kKeysRows && tiles <= (float)most;
  const int unit = fits ? 64 : 128;
  const float room = fits ? (float)sp.target : max((float)sp.target - 0.5f * tiles * (float)c.nkv, 0.5f * (float)sp.target);
  const int each = (int)min(total / room, 1.0e9f);
  w.len = max(sp.least, min(sp.most, (each + unit) / unit * unit));
  for (;;) {
    w.own.items = pa_items(w.own, w.len);
    w.incl = pa_scan(w.own.items);
    w.items = __builtin_amdgcn_readlane(w.incl, 63);
    for (int s = 64 + lane; s - lane < b.n_seqs; s += 64)
      w.items += __builtin_amdgcn_readlane(pa_scan(pa_items(pa_seq<RT>(b, c, group, s), w.len)), 63);
    if (!fits || w.items <= most || w.len >= sp.most) break;
    w.len = min(sp.most, w.len + max(unit, w.len / 16 / unit * unit));
  }
  w.items = min(w.items, sp.slots);
  return w;
}

// The sequence that `pick` (a lane's cumulative measure past a sequence > it) points at, and
// the items before it: 64 sequences at a time.
template <int RT>
__device__ __forceinline__ PaSeq pa_locate(const PkBatch& b, const PkCache& c, int group, const PaWork& w, int item,
                                           int* seq, int* before) {
  PaSeq q = w.own;
  int incl = w.incl, base = 0, s0 = 0;
  uint64_t past;
  while (!(past = __builtin_amdgcn_ballot_w64(incl > item)) && s0 + 64 < b.n_seqs) {
    s0 += 64;
    base = __builtin_amdgcn_readlane(incl, 63);
    q = pa_seq<RT>(b, c, group, s0 + pa_lane());
    q.items = pa_items(q, w.len);
    incl = base + pa_scan(q.items);
  }
  const int l = past ? __builtin_ctzll(past) : 63;
  *seq = s0 + l;
  *before = __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(q.items, l);
  PaSeq r;
  r.q0 = __builtin_amdgcn_readlane(q.q0, l);
  r.m = __builtin_amdgcn_readlane(q.m, l);
  r.len = __builtin_amdgcn_readlane(q.len, l);
  r.tiles = __builtin_amdgcn_readlane(q.tiles, l);
  r.keys = __builtin_amdgcn_readlane(q.keys, l);
  return r;
}

// Keys that the last row of a tile sees.
template <int RT>
__device__ __forceinline__ int pa_kend(const PaSeq& q, int row0, int group) {
  const int last = min(row0 + RT, q.m * group) - 1;
  return max(0, min(q.len - q.m + last / group + 1, q.keys));
}

// Item `item` < w.items of a head; false where nothing is to be done (a range behind the last key
// that its tile sees).
template <int RT>
__device__ __forceinline__ bool pa_item(const PkBatch& b, const PkCache& c, int group, const PaWork& w, int item,
                                        PaTile* t) {
  int before;
  const PaSeq q = pa_locate<RT>(b, c, group, w, item, &t->seq, &before);
  const int z = (item - before) / q.tiles, i = item - before - z * q.tiles, tile = z & 1 ? i : q.tiles - 1 - i;
  t->slot = before + (z + 1) * q.tiles - 1 - tile;
  t->first = q.q0;
  t->row0 = tile * RT;
  t->nrows = q.m * group;
  t->pos0 = q.len - q.m;
  t->kend = pa_kend<RT>(q, t->row0, group);
  const int n = max(1, pa_ceil(t->kend, w.len));  // at most; rounded up, fewer may do
  constexpr int unit = RT == kKeysRows ? 64 : 128;
  t->len = max(unit, (pa_ceil(t->kend, n) + unit - 1) / unit * unit);
  t->k0 = z * t->len;
  t->ranges = min(n, max(1, pa_ceil(t->kend, t->len)));
  t->tiles = q.tiles;
  return z < t->ranges && t->slot < w.items;
}

// The page ids of 64 sub-tiles, one per lane (the one that holds key `key`), and which of them
// are pages.
struct PaIds {
  int id;
  uint64_t on;
};
__device__ __forceinline__ PaIds pa_ids(const PkBatch& b, const PkCache& c, int seq, int key) {
  PaIds r;
  const int pi = key >> c.ps_log;
  r.id = pi < b.max_pages ? b.pages[(long)seq * b.max_pages + pi] : -1;
  const bool ok = r.id >= 0 && r.id < c.n_pages;
  if (!ok) r.id = 0;
  r.on = __builtin_amdgcn_ballot_w64(ok);
  return r;
}

// The item of a block of a direct schedule's grid (sequence, head, range), with the page ids of its
// range (lane: key k0 + `key`): few enough that all may be there; everything is loaded at once.
__device__ __forceinline__ bool pa_direct(const PkBatch& b, const PkCache& c, int group, int len, int key, PaTile* t,
                                          PaIds* ids) {
  const int z = blockIdx.z, s = blockIdx.x;
  const int q0 = b.q_start[s], q1 = min(b.q_start[s + 1], b.rows), have = b.kv_len[s];
  *ids = pa_ids(b, c, s, z * len + key);
  t->seq = s;
  t->first = __builtin_amdgcn_readfirstlane(q0);
  const int m = __builtin_amdgcn_readfirstlane(q1) - t->first, n = __builtin_amdgcn_readfirstlane(have);
  t->row0 = 0;
  t->nrows = m * group;
  t->pos0 = n - m;
  t->kend = (int)max(0l, min((long)min(n, b.max_kv), (long)b.max_pages << c.ps_log));
  t->k0 = z * len;
  t->len = len;
  t->ranges = max(1, pa_ceil(t->kend, len));
  t->tiles = b.n_seqs;
  t->slot = z * b.n_seqs + s;
  return m > 0 && z < t->ranges;
}

// The head of a block and its place among the head's blocks (`per` of them).  A head's blocks sit
// on as few of the 8 XCDs as there are to go round, so that its keys pass through their caches.
__device__ __forceinline__ void pa_head_of(int nkv, int* kvh, int* place) {
  const int x = blockIdx.x & 7, i = blockIdx.x >> 3;
  if (8 % nkv == 0) {
    const int per = 8 / nkv;
    *kvh = x / per;
    *place = i * per + x % per;
  } else if (nkv % 8 == 0) {
    const int per = nkv / 8;
    *kvh = x * per + i % per;
    *place = i / per;
  } else {
    *kvh = blockIdx.x % nkv;
    *place = blockIdx.x / nkv;
  }
}

__device__ __forceinline__ pa_rsrc_t pa_rsrc(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, bytes, 0x00020000);
}

// Sum over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float pa_rowsum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// 8 int8 -> 8 fp16 (mx_i8_to_f16 of half the width).
__device__ __forceinline__ half8_t pa_i8x8(int2_t v) {
  const half2_t bias = {(half_t)1152.0f, (half_t)1152.0f};
  half2_t h[4];
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const uint32_t u = (uint32_t)v[d] ^ 0x80808080u;
    h[2 * d] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
    h[2 * d + 1] = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  }
  return (half8_t){h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

// ------------------------------------------------------------------------------------
// LDS tiles of 32 rows of RB bytes (RB = 64 .. 512, the padded row), row-major, a row's 16-byte
// chunks permuted by an XOR so that the fragment reads use every bank once: 8 lanes of a
// 16-byte read take one chunk of 8 consecutive rows (keys: chunk ^ row % 8), 16 lanes of an 8-byte
// transposing read take 32 bytes of 4 rows (fp16 values: chunk ^ 2 (row % 4)) or 16 bytes of 8
// rows (int8 values: chunk ^ the row's number among those 8).
// A copy instruction fills 1 KiB, whole rows: the permutation stays inside a row, so it reads
// whole rows of the page in order.  Rows of fewer than RB bytes: the chunks past the row repeat
// its last one (the queries are zero there, and no output is stored).
// ------------------------------------------------------------------------------------
template <int DT>
__device__ __forceinline__ int pa_vxor(int row) {  // row of the 32
  if constexpr (DT == MX_DT_I8) return (row & 3) | ((row >> 4) & 1) << 2;
  return 2 * (row & 3);
}

// Byte offset in a 16-row sub-tile of the page that copy instruction `i` (of RB / 64) loads on this
// lane for row-major rows of rb bytes; XORs by `x(row)`.
template <int RB, typename X>
__device__ __forceinline__ uint32_t pa_copy_off(int i, int lane, int rb, X x) {
  constexpr int CPR = RB / 16, RPI = 1024 / RB;
  const int row = i * RPI + lane / CPR;
  const int chunk = ((lane % CPR) ^ x(row)) & (CPR - 1);
  return (uint32_t)(row * rb + min(chunk * 16, rb - 16));
}

// One lane's reads of a tile's value fragments (16 dims x 32 keys each): the XOR touches the low
// bits of a fragment's number only, so a few addresses and constant offsets serve all of
// them.
template <int RB, int DT>
struct PaV {
  static constexpr int STEP = DT == MX_DT_I8 ? 16 : 32;       // bytes of a fragment in a row
  static constexpr int NB = (DT == MX_DT_I8 ? 8 : 4) * STEP <= RB ? (DT == MX_DT_I8 ? 8 : 4) : RB / STEP;
  const char* at[NB];
  // The lane's place in a tile, fragment 0 (the others: an XOR with f STEP).
  static __device__ __forceinline__ int lane_at(int lane) {
    const int j = lane & 15, g = lane >> 4;
    const int rr = j >> 1;
    const int row = DT == MX_DT_I8 ? (rr < 4 ? 4 * g + rr : 16 + 4 * g + rr - 4) : 4 * g + (j >> 2);
    const int chunk = DT == MX_DT_I8 ? 0 : (j & 3) >> 1;
    return row * RB + ((chunk ^ pa_vxor<DT>(row)) & (RB / 16 - 1)) * 16 + 8 * (j & 1);
  }
  __device__ __forceinline__ PaV(const char* tile, int place) {
#pragma unroll
    for (int e = 0; e < NB; ++e) at[e] = tile + (place ^ (e * STEP));
  }
  __device__ __forceinline__ const char* operator()(int f) const { return at[f % NB] + f / NB * NB * STEP; }
};

typedef __attribute__((address_space(3))) short4_t pa_lds_s4;
typedef __attribute__((address_space(3))) int2_t pa_lds_i2;

template <int RB, int DT>
__device__ __forceinline__ half8_t pa_vfrag(const PaV<RB, DT>& vl, int f) {
  const char* p = vl(f);
  if constexpr (DT == MX_DT_I8) {
    return pa_i8x8(__builtin_amdgcn_ds_read_tr8_b64_v2i32((pa_lds_i2*)p));
  } else {
    const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s4*)p);
    const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s4*)(p + 16 * RB));
    const half4_t x = __builtin_bit_cast(half4_t, a), y = __builtin_bit_cast(half4_t, b);
    return (half8_t){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }
}

// 16-bit masks of the lane's 8 keys of a tile whose last seen key is `top` (relative) and whose
// sub-tiles on a page are `on`.
__device__ __forceinline__ void pa_keep(int top, int on, uint32_t (&keep)[4]) {
  const int g = pa_lane() >> 4;
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int s = d >> 1, k = 16 * s + 4 * g + 2 * (d & 1);
    const bool ok = (on >> s) & 1;
    keep[d] = (ok && k <= top ? 0xFFFFu : 0u) | (ok && k + 1 <= top ? 0xFFFF0000u : 0u);
  }
}

// A fragment of a masked fp16 tile: keys no row of the wave sees become zeros, and with ODD non-
// finite values do too, noted in `odd`.  (Int8 values are finite: a weight of zero suffices.)
template <bool ODD>
__device__ __forceinline__ half8_t pa_clean(half8_t v, const uint32_t (&keep)[4], uint32_t& odd) {
  int4_t u = __builtin_bit_cast(int4_t, v);
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    uint32_t w = (uint32_t)u[d] & keep[d];
    if constexpr (ODD) {
      const uint32_t lo = (w & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u;
      const uint32_t hi = (w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u;
      odd |= lo | hi;
      w &= ~(lo | hi);
    }
    u[d] = (int)w;
  }
  return __builtin_bit_cast(half8_t, u);
}

// The non-finite values that pa_clean took out of a tile, added to the rows that see them (fp16
// values only; rare).  p: the row's probabilities in k-slot order; lim: the last key of the tile
// that the lane's row sees; seen: keys on a page (bit per key).
template <int RB, int NF>
__device__ __forceinline__ void pa_add_odd(const char* tile, half8_t p, int lim, uint32_t seen,
                                           float4_t (&o)[NF]) {
  const int4_t pi = __builtin_bit_cast(int4_t, p);
#pragma nounroll
  for (int key = 0; key < 32; ++key) {
    if (!((seen >> key) & 1)) continue;
    const int lane = pa_lane(), j = lane & 15, g = lane >> 4;
    const int src = ((key & 15) >> 2) * 16 + j, d = (key >> 4) * 2 + ((key >> 1) & 1);
    const int pw = __shfl(d == 0 ? pi[0] : d == 1 ? pi[1] : d == 2 ? pi[2] : pi[3], src);
    const half2_t ph = __builtin_bit_cast(half2_t, pw);
    const float pk = key <= lim ? (float)((key & 1) ? ph[1] : ph[0]) : 0.f;
    // dims 16 f + 4 g ..: chunk 2 f + g / 2, its half g % 2
    const char* row = tile + key * RB + 8 * (g & 1);
    const int x = pa_vxor<MX_DT_F16>(key) * 16 ^ 16 * (g >> 1);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const half4_t v = *(const half4_t*)(row + ((32 * f ^ pa_opaque(x)) & (RB - 1)));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool bad = (__builtin_bit_cast(unsigned short, v[r]) & 0x7C00) == 0x7C00;
        if (bad && key <= lim) o[f][r] += pk * (float)v[r];
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Two sub-tiles' key scales and value scales on this lane's keys (int8 pages).
struct PaScales {
  float4 ks[2], vs[2];
};

// One 32-key step of a row set: scores sc (raw dots) -> probabilities, running reference and
// sum, accumulators rescaled where the reference moved.  lim: last key of the tile (relative)
// that the row sees, relative to 4 g; `on`: bits of the sub-tiles that are on a page.
template <int DT, bool MASK, int NF>
__device__ __forceinline__ half8_t pa_softmax(float4_t (&sc)[2], float rs, const PaScales& q8, int lim,
                                              int on, float& mrun, float& lrun, float4_t (&o)[NF]) {
  float s[8], inv[8];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const float kq[4] = {q8.ks[b].x, q8.ks[b].y, q8.ks[b].z, q8.ks[b].w};
    const float vq[4] = {q8.vs[b].x, q8.vs[b].y, q8.vs[b].z, q8.vs[b].w};
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool out = MASK && (16 * b + r > lim || !((on >> b) & 1));
      float v;
      if constexpr (DT == MX_DT_I8) {
        const float w = vq[r] < 1e-30f ? 1e-30f : vq[r];  // a NaN stays, which fmaxf would drop
        inv[4 * b + r] = out ? 0.f : __builtin_amdgcn_rcpf(w);
        v = __builtin_fmaf(sc[b][r], rs * kq[r], __builtin_amdgcn_logf(w));
      } else {
        v = sc[b][r] * rs;
      }
      s[4 * b + r] = out ? -INFINITY : v;
    }
  }
  float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                   fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
  mt = mx_rowmax4(mt);
  const bool up = mt > mrun + kTau;
  if (__builtin_amdgcn_ballot_w64(up)) {
    const float mnew = up ? mt : mrun;
    const float alpha = __builtin_amdgcn_exp2f(mrun - mnew);  // 1 where it stays
    lrun *= alpha;
    mrun = mnew;
#pragma unroll
    for (int f = 0; f < NF; ++f) o[f] *= alpha;
  }
  half8_t p;
  float ps = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = __builtin_amdgcn_exp2f(s[e] - mrun);
    if constexpr (DT == MX_DT_I8) ps = __builtin_fmaf(v, inv[e], ps);
    else ps += v;
    p[e] = (half_t)v;
  }
  lrun += ps;
  return p;
}

// ------------------------------------------------------------------------------------
// k_pa_keys: a tile of 16 rows, its keys dealt to the block's 4 waves 32 at a time.  For decode
// steps, bound by the bytes of the pages.  A wave's tiles are its own: one LDS buffer for keys,
// one for values, filled by copies of whole rows (key rows read straight into MFMA registers
// would be 16 rows x 16 bytes per quarter wave, a cache line each); the next tile's keys are on
// their way from the moment this tile's scores are formed, its values from the moment this
// tile's are used.  No barrier until the waves' sums are put together at the end.  64 sequences of 8000
// fp16 tokens, 16 heads over 2 of 256: 185 us with the join, 5.7 TB/s; two of 913 tokens 11.7 us, launches; 40
// ragged ones of up to 12000 int8 tokens 32 us, of which 27.5 here (3.3 TB/s, 76 bytes of scratch per lane).
// ------------------------------------------------------------------------------------
constexpr int kKeysMax = 4096;  // keys of a split: 64 sub-tile page ids per wave

template <int RB, int DT, bool DIRECT>
__global__ __launch_bounds__(256, RB < 512 ? 2 : 1) void k_pa_keys(PkCache c, PkBatch b, PaArgs a, PaSched sp, int per) {
  constexpr int ES = DT == MX_DT_I8 ? 1 : 2;
  constexpr int DP = RB / ES, NC = DP / 32, NF = DP / 16, CPR = RB / 16;
  constexpr int NL = RB / 64;             // 1 KiB pieces per 16 rows
  constexpr int TILE = 32 * RB;
  __shared__ __align__(1024) char ldsk[4 * TILE];  // one variable per buffer (see k_pa_rows)
  __shared__ __align__(1024) char ldsv[4 * TILE];
  __shared__ float sm[4][16], sl[4][16];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh = blockIdx.y, first = 0;
  PaWork work;
  if constexpr (DIRECT) {  // one item per block, slot by range and sequence
    first = blockIdx.z * b.n_seqs + blockIdx.x;
    work.len = sp.least;
  } else {
    pa_head_of(c.nkv, &kvh, &first);
    work = pa_schedule<kKeysRows>(b, c, sp, a.group, per);
  }
  for (int item = first; DIRECT || item < work.items; item += per) {
  // Opaque: what follows from the lane is worked out per item and holds nothing across the loop.
  const int lane = pa_lane(), tid = 64 * wave + lane, j = lane & 15, g = lane >> 4;
  PaTile t;
  PaIds ids;  // lane l: the page of sub-tile l % 2 of the wave's tile l / 2
  const int mine = 32 * (wave + 4 * (lane >> 1)) + 16 * (lane & 1);
  if constexpr (DIRECT) {
    if (!pa_direct(b, c, a.group, work.len, mine, &t, &ids)) return;
  } else {
    if (!pa_item<kKeysRows>(b, c, a.group, work, item, &t)) continue;
    ids = pa_ids(b, c, t.seq, t.k0 + mine);
  }
  const int k0 = t.k0, k1 = min(t.kend, k0 + t.len);

  const int row = min(t.row0 + j, t.nrows - 1);
  const int tok = row / a.group, hq = kvh * a.group + row - tok * a.group;
  const int pos = t.pos0 + tok;
  const int rb = c.hd * ES;
  const float rs = mx_readlane(a.scale * kLog2e, 0);  // uniform: a scalar register

  // Queries: B fragments.  Fp16 pages: chunk cc holds dims 32 cc + 8 g ..; int8 pages (16 dims per
  // 16-byte load): chunk pair (2 i, 2 i + 1) dims 64 i + 16 g .. + 7 and + 8 .. + 15.
  half8_t qf[NC];
  const half_t* qrow = (const half_t*)a.q + (long)(t.first + tok) * a.ldq + (long)hq * c.hd;
  auto qdim = [&](int cc) { return DT == MX_DT_I8 ? 64 * (cc >> 1) + 16 * g + 8 * (cc & 1) : 32 * cc + 8 * g; };
#pragma unroll
  for (int cc = 0; cc < NC; ++cc) qf[cc] = *(const half8_t*)(qrow + min(qdim(cc), c.hd - 8));
  const int ntile = pa_ceil(max(0, k1 - k0), 32);
  const int nw = ntile > wave ? (ntile - 1 - wave) / 4 + 1 : 0;
  char* const kbuf = ldsk + wave * TILE;
  char* const vbuf = ldsv + wave * TILE;
  uint32_t koff[NL], voff[NL][2];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    koff[i] = pa_copy_off<RB>(i, lane, rb, [](int r) { return r & 7; });
#pragma unroll
    for (int s = 0; s < 2; ++s)
      voff[i][s] = pa_copy_off<RB>(i, lane, rb, [&](int r) { return pa_vxor<DT>(16 * s + r); });
  }
  auto row_of = [&](int i, int s) {  // the sub-tile's first row in a pool
    const int id = __builtin_amdgcn_readlane(ids.id, 2 * i + s);
    const int key = k0 + 32 * (wave + 4 * i) + 16 * s;
    return (((long)id * c.nkv + kvh) << c.ps_log) + (key & (c.ps - 1));
  };
  PaScales q8n;
  auto issue_k = [&](int i) {
    const long at0 = row_of(i, 0), at1 = row_of(i, 1);
    if constexpr (DT == MX_DT_I8) {  // ahead of the copies: the waits below count those alone
      q8n.ks[0] = *(const float4*)(c.ks + at0 + 4 * g);
      q8n.ks[1] = *(const float4*)(c.ks + at1 + 4 * g);
      q8n.vs[0] = *(const float4*)(c.vs + at0 + 4 * g);
      q8n.vs[1] = *(const float4*)(c.vs + at1 + 4 * g);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const pa_rsrc_t r = pa_rsrc(c.k + (s ? at1 : at0) * rb, 16 * rb);
#pragma unroll
      for (int n = 0; n < NL; ++n) mx_copy_to_lds16(r, kbuf + s * 16 * RB + n * 1024, koff[n]);
    }
  };
  auto issue_v = [&](int i) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const pa_rsrc_t r = pa_rsrc(c.v + row_of(i, s) * rb, 16 * rb);
#pragma unroll
      for (int n = 0; n < NL; ++n) mx_copy_to_lds16(r, vbuf + s * 16 * RB + n * 1024, voff[n][s]);
    }
  };
  constexpr int NK = DT == MX_DT_I8 ? NC / 2 : NC;  // 16-byte fragment reads per key row and lane
  const int vlane = PaV<RB, DT>::lane_at(lane);
  const int klane = j * RB + ((g ^ (j & 7)) & (CPR - 1)) * 16;
  float4_t o[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) o[f] = (float4_t){0.f, 0.f, 0.f, 0.f};
  float mrun = kLow, lrun = 0.f;

  if (nw > 0) {
    issue_k(0);
    issue_v(0);
  }
  __builtin_amdgcn_sched_barrier(0);  // the queries, loaded ahead of the copies, are not waited for before
#pragma unroll
  for (int cc = 0; cc < NC; ++cc)
    if (qdim(cc) >= c.hd) qf[cc] = (half8_t)(half_t)0.f;
  // The last key that every row of the tile sees (rows past the last repeat it), and that any does.
  const int all = t.pos0 + t.row0 / a.group, any = t.kend - 1;
  // MORE: a tile follows.  Its copies are issued without a branch, so that the compiler's own waits
  // leave them in flight too.
  auto step = [&](int i, auto more) {
    constexpr bool MORE = decltype(more)::value;
    // Keys of this tile: all but the value copies behind them.
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
    const PaScales q8 = q8n;
    float4_t sc[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p0 = kbuf + klane + s * 16 * RB;
      const char* p1 = kbuf + (klane ^ (CPR > 4 ? 64 : 0)) + s * 16 * RB;
      float4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const int4_t kf = *(const int4_t*)((n & 1 ? p1 : p0) + 64 * (n & ~1));
        if constexpr (DT == MX_DT_I8) {
          half8_t lo, hi;
          mx_i8_to_f16(kf, lo, hi);
          x[0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qf[2 * n], x[0], 0, 0, 0);
          x[1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qf[2 * n + 1], x[1], 0, 0, 0);
        } else {
          x[n & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, kf), qf[n], x[n & 1], 0, 0, 0);
        }
      }
      sc[s] = x[0] + x[1];
    }
    // The scores are formed (their registers pass through here): the buffer is free.
    asm volatile("" : "+v"(sc[0]), "+v"(sc[1])::"memory");
    if constexpr (MORE) issue_k(i + 1);
    const int tk = k0 + 32 * (wave + 4 * i);  // first key of the tile
    const int on = (int)(ids.on >> (2 * i)) & 3;
    const bool mask = tk + 31 > all || on != 3;
    const int lim = pos - tk;
    half8_t p;
    if (mask) p = pa_softmax<DT, true>(sc, rs, q8, lim - 4 * g, on, mrun, lrun, o);
    else p = pa_softmax<DT, false>(sc, rs, q8, lim, on, mrun, lrun, o);
    // Values of this tile: all but the key copies behind them.
    if constexpr (MORE) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const PaV<RB, DT> vt(vbuf, pa_opaque(vlane));
    if (DT == MX_DT_I8 || !mask) {  // (a weight of zero meets finite int8 values)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa_vfrag<RB, DT>(vt, f), p, o[f], 0, 0, 0);
    } else {
      uint32_t keep[4], odd = 0;
      pa_keep(any - tk, on, keep);
      if (all >= any) {  // one token: what one row does not see, none does
#pragma unroll
        for (int f = 0; f < NF; ++f)
          o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa_clean<false>(pa_vfrag<RB, DT>(vt, f), keep, odd), p,
                                                        o[f], 0, 0, 0);
      } else {
#pragma unroll
        for (int f = 0; f < NF; ++f)
          o[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa_clean<true>(pa_vfrag<RB, DT>(vt, f), keep, odd), p,
                                                        o[f], 0, 0, 0);
        if (__builtin_amdgcn_ballot_w64(odd != 0)) {
          const uint32_t seen = ((on & 1) ? 0xFFFFu : 0u) | ((on & 2) ? 0xFFFF0000u : 0u);
          pa_add_odd<RB, NF>(vbuf, p, lim, seen, o);
        }
      }
    }
    // Every value is read (the products hold them): the buffer is free.
    asm volatile("" : "+v"(o[NF - 1])::"memory");
    if constexpr (MORE) issue_v(i + 1);
  };
#pragma nounroll
  for (int i = 0; i + 1 < nw; ++i) step(i, std::true_type{});
  if (nw > 0) step(nw - 1, std::false_type{});
  lrun = pa_rowsum(lrun);

  // The waves' sums, relative to the largest reference of each row.
  if (g == 0) {
    sm[wave][j] = mrun;
    sl[wave][j] = lrun;
  }
  __syncthreads();
  const float m = fmaxf(fmaxf(sm[0][j], sm[1][j]), fmaxf(sm[2][j], sm[3][j]));
  const float weight = __builtin_amdgcn_exp2f(mrun - m);
  // [16 rows][DP] per wave: waves 0, 1 in the first buffer, 2, 3 in the second
  static_assert(2 * 16 * DP * 4 <= 4 * TILE, "the sums fit the buffers");
  auto part_of = [&](int w) { return (float*)(w < 2 ? ldsk : ldsv) + (w & 1) * 16 * DP; };
  __syncthreads();
  float* const part = part_of(wave);
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const float4_t v = o[f] * weight;
    *(float4_t*)(part + j * DP + 16 * f + 4 * g) = v;
  }
  __syncthreads();
  constexpr int D4 = DP / 4;
  for (int i = tid; i < 16 * D4; i += 256) {
    const int r = i / D4, d = 4 * (i % D4);
    if (t.row0 + r >= t.nrows || d >= c.hd) continue;
    float4_t s = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f, mr = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      s += *(const float4_t*)(part_of(w) + r * DP + d);
      l += sl[w][r] * __builtin_amdgcn_exp2f(sm[w][r] - mr);
    }
    const int rt = (t.row0 + r) / a.group, h = kvh * a.group + (t.row0 + r) - rt * a.group;
    const long tr = t.first + rt;
    const int at = (kvh * sp.slots + t.slot) * kKeysRows + r;
    if (k0 == 0 && d == 0)
      sp.rows[tr * a.nh + h] = (int4_t){at, t.tiles * kKeysRows, t.ranges, 0};
    if (t.ranges > 1) {
      *(float4_t*)(sp.po + (long)at * c.hd + d) = s;
      if (d == 0) sp.ml[at] = make_float2(mr, l);
      continue;
    }
    s *= l == 0.f ? 0.f : 1.f / l;
    if (a.gate) {
      const float4 gv = *(const float4*)(a.gate + tr * a.ldg + (long)h * c.hd + d);
      s = (float4_t){s[0] * mx_sigmoid(gv.x), s[1] * mx_sigmoid(gv.y), s[2] * mx_sigmoid(gv.z),
                     s[3] * mx_sigmoid(gv.w)};
    }
    *(half4_t*)((half_t*)a.out + tr * a.ldo + (long)h * c.hd + d) =
        (half4_t){(half_t)s[0], (half_t)s[1], (half_t)s[2], (half_t)s[3]};
  }
  if constexpr (DIRECT) return;
  __syncthreads();  // the buffers are free
  }
}

// ------------------------------------------------------------------------------------
// k_pa_join: the partial sums of a row's key ranges; the first range's item has noted where they
// lie.  One wave per (row, head), or WIDE, a block's four waves, a quarter of the ranges each: a
// decode step has few rows of many ranges, whose sums were written by other XCDs and take a
// microsecond or two to fetch (40 rows of up to 35 ranges: 11.4 us with one wave, 5.0 with four).
// Bound by the sums' bytes where there are many rows: 2048 rows of 16 heads in two ranges 21 us.
// ------------------------------------------------------------------------------------
template <typename OT, bool WIDE>
__global__ __launch_bounds__(256) void k_pa_join(PkCache c, PkBatch b, PaArgs a, PaSched sp) {
  __shared__ float sml[4][2];
  __shared__ __align__(16) float so[WIDE ? 4 : 1][256];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = WIDE ? blockIdx.y : blockIdx.y * 4 + wave;
  const int t = blockIdx.x;
  if (h >= a.nh) return;
  const int4_t where = sp.rows[(long)t * a.nh + h];
  if (t >= b.q_start[b.n_seqs]) return;  // behind the last sequence
  const int ranges = __builtin_amdgcn_readfirstlane(where[2]);
  // (a row that no sequence has, or two have, left no place for its sums)
  if (ranges <= 1 || where[0] < 0 || where[1] < 0 || where[0] + (ranges - 1l) * where[1] >= sp.end) return;
  // This wave's: every 4th range, or all of them.
  constexpr int HOP = WIDE ? 4 : 1;
  const int n = WIDE ? (ranges - wave + 3) / 4 : ranges;
  const long at = __builtin_amdgcn_readfirstlane(where[0]) + (WIDE ? (long)wave * where[1] : 0);
  const long step = (long)HOP * __builtin_amdgcn_readfirstlane(where[1]);
  const int d = min(4 * lane, c.hd - 4);
  const float* po = sp.po + at * c.hd + d;
  float4 gv = make_float4(0.f, 0.f, 0.f, 0.f);  // on its way with the sums
  if (a.gate) gv = *(const float4*)(a.gate + (long)t * a.ldg + (long)h * c.hd + d);
  float mr = kLow, l = 0.f;
  float4_t s = {0.f, 0.f, 0.f, 0.f};
  // 64 ranges at a time: lane z holds range z's reference and sum, whose weights all lanes
  // then read; 8 partial rows in flight.
  for (int z0 = 0; z0 < n; z0 += 64) {
    const int nz = min(64, n - z0);
    float2 ml = make_float2(kLow, 0.f);
    if (lane < nz) ml = sp.ml[at + (z0 + lane) * step];
    float4_t v[8];
    auto load = [&](int z) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (z + e < nz) v[e] = *(const float4_t*)(po + (z0 + z + e) * step * c.hd);
    };
    load(0);
    const float top = fmaxf(mr, mx_wave_max(ml.x));
    const float w = __builtin_amdgcn_exp2f(ml.x - top), old = __builtin_amdgcn_exp2f(mr - top);
    l = l * old + mx_wave_sum(w * ml.y);
    s *= old;
    mr = top;
    for (int z = 0; z < nz; z += 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (z + e < nz) s += mx_readlane(w, z + e) * v[e];
      load(z + 8);
    }
  }
  if constexpr (WIDE) {
    if (lane == 0) {
      sml[wave][0] = mr;
      sml[wave][1] = l;
    }
    *(float4_t*)(so[wave] + 4 * lane) = s;
    __syncthreads();
    if (wave) return;
    const float top = fmaxf(fmaxf(sml[0][0], sml[1][0]), fmaxf(sml[2][0], sml[3][0]));
    l = 0.f;
    s = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(sml[w][0] - top);
      l += f * sml[w][1];
      s += f * *(const float4_t*)(so[w] + 4 * lane);
    }
  }
  if (4 * lane >= c.hd) return;
  s *= l == 0.f ? 0.f : 1.f / l;
  if (a.gate) {
    s = (float4_t){s[0] * mx_sigmoid(gv.x), s[1] * mx_sigmoid(gv.y), s[2] * mx_sigmoid(gv.z),
                   s[3] * mx_sigmoid(gv.w)};
  }
  typedef OT ot4_t __attribute__((ext_vector_type(4)));
  *(ot4_t*)((OT*)a.out + (long)t * a.ldo + (long)h * c.hd + d) =
      (ot4_t){(OT)s[0], (OT)s[1], (OT)s[2], (OT)s[3]};
}

// ------------------------------------------------------------------------------------
// k_pa_rows: a tile of 64 QS rows (16 QS per wave), every key tile shared by the block's 4 waves.
// For chunks of new tokens, bound by the matrix instructions.  Key and value tiles of 32 keys are
// copied straight into two LDS buffers by the buffer loads' LDS mode; a wave's copies of tile t + 1
// are issued behind the barrier that opens tile t.  Each fragment read from LDS feeds QS query
// sets.  A wave computes up to its own last key and then only keeps the copies going.  2048 rows over 8192
// tokens, 16 heads over 2 of 256: 259 us with the join, 0.93 PFLOP/s.  Two sets of 256 fp16 dims take all 256
// registers and 12 bytes of scratch.
//
// Row tiles of a key/value head run on the XCDs that its keys are dealt to.
// ------------------------------------------------------------------------------------
constexpr int kAheadReads = 2;  // LDS fragment reads in flight ahead of the MFMAs

template <int RB, int DT, int QS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_pa_rows(PkCache c, PkBatch b, PaArgs a, PaSched sp, int per) {
  constexpr int ES = DT == MX_DT_I8 ? 1 : 2;
  constexpr int DP = RB / ES, NC = DP / 32, NF = DP / 16, CPR = RB / 16;
  constexpr int NL = RB / 64;             // 1 KiB pieces per 16 rows
  constexpr int FPW = NL;                 // copies per wave and tile (4 NL pieces, 4 waves)
  constexpr int TILE = 64 * RB;           // keys, then values
  constexpr int NK = DT == MX_DT_I8 ? NC / 2 : NC;  // 16-byte fragment reads per key row and lane
  constexpr int RT = 64 * QS;
  // One variable per buffer: the compiler then knows that a read of one does not wait for copies
  // into the other (a transposing read waits for every copy it may meet).
  __shared__ __align__(1024) char lds0[TILE];
  __shared__ __align__(1024) char lds1[TILE];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh, place;
  pa_head_of(c.nkv, &kvh, &place);
  for (int item = place;; item += per) {
  // Worked out anew for every item: it would hold registers across the loops below.
  PaSched now = sp;
  now.target = pa_opaque_s(sp.target);
  const int group = pa_opaque_s(a.group);
  const PaWork work = pa_schedule<RT>(b, c, now, group, per);
  if (item >= work.items) return;
  // Opaque: what follows from the lane is worked out per item and holds nothing across the loop.
  const int lane = pa_lane(), j = lane & 15, g = lane >> 4;
  PaTile t;
  if (!pa_item<RT>(b, c, group, work, item, &t)) continue;
  const int k0 = t.k0, k1 = min(t.kend, k0 + t.len);
  PaIds ids = pa_ids(b, c, t.seq, k0 + 16 * lane);
  const int ntile = pa_ceil(max(0, k1 - k0), 32);

  const int rb = c.hd * ES;
  const float rs = mx_readlane(a.scale * kLog2e, 0);  // uniform: a scalar register
  // Copies: piece wave + 4 i of the tile's 4 NL (key pieces of both sub-tiles, then values).  A
  // wave's pieces of a sub-tile (NL > 4: two) are 4 pieces, 8 rows, apart: the same lane
  // offsets.  Int8 values' XOR depends on the sub-tile.
  const int n0 = wave % NL;
  const uint32_t offk = pa_copy_off<RB>(n0, lane, rb, [](int r) { return r & 7; });
  uint32_t offv[2];
  offv[0] = pa_copy_off<RB>(n0, lane, rb, [](int r) { return pa_vxor<DT>(r); });
  offv[1] = DT == MX_DT_I8 ? pa_copy_off<RB>(n0, lane, rb, [](int r) { return pa_vxor<DT>(16 + r); }) : offv[0];
  auto row_of = [&](int kt, int s) {  // the sub-tile's first row in a pool
    const int id = __builtin_amdgcn_readlane(ids.id, 2 * (kt & 31) + s);
    return (((long)id * c.nkv + kvh) << c.ps_log) + ((k0 + 32 * kt + 16 * s) & (c.ps - 1));
  };
  PaScales q8n;
  auto issue = [&](int kt, char* buf) {
    const long at0 = row_of(kt, 0), at1 = row_of(kt, 1);
#pragma unroll
    for (int i = 0; i < FPW; ++i) {
      // piece wave + 4 i: key or value, its sub-tile, its rows (8 behind the lane offset's, or not)
      const bool key = NL >= 2 ? i < FPW / 2 : wave < 2;
      const bool second = NL >= 4 ? (4 * i / NL) % 2 : NL == 2 ? wave >= 2 : wave & 1;
      const int more = NL > 4 && (4 * i) % NL >= 4 ? 8 * rb : 0;
      const pa_rsrc_t r = pa_rsrc((key ? c.k : c.v) + (second ? at1 : at0) * rb, 16 * rb);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (mx_lds_void*)(buf + (wave + 4 * i) * 1024), 16,
                                               key ? offk : second ? offv[1] : offv[0], more, 0, 0);
    }
    if constexpr (DT == MX_DT_I8) {
      const long r0 = at0 + 4 * g, r1 = at1 + 4 * g;
      q8n.ks[0] = *(const float4*)(c.ks + r0);
      q8n.ks[1] = *(const float4*)(c.ks + r1);
      q8n.vs[0] = *(const float4*)(c.vs + r0);
      q8n.vs[1] = *(const float4*)(c.vs + r1);
    }
  };
  if (ntile > 0) issue(0, lds0);
  int on_next = (int)(ids.on & 3);

  half8_t qf[QS][NC];
  auto qdim = [&](int cc) { return DT == MX_DT_I8 ? 64 * (cc >> 1) + 16 * g + 8 * (cc & 1) : 32 * cc + 8 * g; };
  const int w0 = t.row0 + wave * 16 * QS;  // the wave's first row
  // Token (of the sequence) and head of the lane's row in set u: worked out where they are needed,
  // behind a barrier to the compiler, so that they hold no registers in between.
  auto where = [&](int u, int& tok, int& hq) {
    const int row = min(w0 + 16 * u + (pa_lane() & 15), t.nrows - 1);
    const int group = pa_opaque_s(a.group);  // (its reciprocal, too)
    tok = row / group;
    hq = kvh * group + row - tok * group;
  };
#pragma unroll
  for (int u = 0; u < QS; ++u) {
    int tok, hq;
    where(u, tok, hq);
    const half_t* qrow = (const half_t*)a.q + (long)(t.first + tok) * a.ldq + (long)hq * c.hd;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) qf[u][cc] = *(const half8_t*)(qrow + min(qdim(cc), c.hd - 8));
#pragma unroll
    for (int cc = 0; cc < NC; ++cc)
      if (qdim(cc) >= c.hd) qf[u][cc] = (half8_t)(half_t)0.f;
  }
  // The keys that every row of the wave sees end at `all`, those that any sees at `any`.
  const int lastrow = min(w0 + 16 * QS, t.nrows) - 1;
  const int all = t.pos0 + min(w0, t.nrows - 1) / group;
  const int any = min(t.pos0 + lastrow / group, t.kend - 1);
  const int nt_w = w0 < t.nrows ? min(ntile, max(0, any + 1 - k0 + 31) / 32) : 0;

  float4_t o[QS][NF];
  float mrun[QS], lrun[QS];
#pragma unroll
  for (int u = 0; u < QS; ++u) {
    mrun[u] = kLow;
    lrun[u] = 0.f;
#pragma unroll
    for (int f = 0; f < NF; ++f) o[u][f] = (float4_t){0.f, 0.f, 0.f, 0.f};
  }
  // Key piece n of a row lies at (place ^ 64 (n % 2)) + 64 (n - n % 2).
  auto key_place = [&]() {
    const int l = pa_lane(), jj = l & 15, gg = l >> 4;
    return jj * RB + ((gg ^ (jj & 7)) & (CPR - 1)) * 16;
  };
  auto value_place = [&]() { return PaV<RB, DT>::lane_at(pa_lane()); };

  auto advance = [&](int kt, char* buf) {  // tile kt + 1 (there is one) on its way
    if (((kt + 1) & 31) == 0) ids = pa_ids(b, c, t.seq, k0 + 32 * (kt + 1) + 16 * pa_lane());
    issue(kt + 1, buf);
    on_next = (int)(ids.on >> (2 * ((kt + 1) & 31))) & 3;
  };
  // Scores of tile kt (its copies have landed): step i is sub-tile i % 2, 16-byte piece i / 2.
  auto scores = [&](const char* kb, float4_t (&sc)[QS][2]) {
    const int kl = key_place();
    const char* const ka[2] = {kb + kl, kb + (kl ^ (CPR > 4 ? 64 : 0))};
    auto kfrag = [&](int i) {
      const int n = i >> 1;
      return *(const int4_t*)(ka[n & 1] + (i & 1) * 16 * RB + 64 * (n & ~1));
    };
#pragma unroll
    for (int u = 0; u < QS; ++u)
#pragma unroll
      for (int s = 0; s < 2; ++s) sc[u][s] = (float4_t){0.f, 0.f, 0.f, 0.f};
    int4_t fr[kAheadReads];
#pragma unroll
    for (int i = 0; i < kAheadReads && i < 2 * NK; ++i) fr[i] = kfrag(i);
#pragma unroll
    for (int i = 0; i < 2 * NK; ++i) {
      const int4_t kf = fr[i % kAheadReads];
      if (i + kAheadReads < 2 * NK) fr[i % kAheadReads] = kfrag(i + kAheadReads);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (DT == MX_DT_I8) {
        half8_t lo, hi;
        mx_i8_to_f16(kf, lo, hi);
#pragma unroll
        for (int u = 0; u < QS; ++u)
          sc[u][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qf[u][2 * (i >> 1)], sc[u][i & 1], 0, 0, 0);
#pragma unroll
        for (int u = 0; u < QS; ++u)
          sc[u][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qf[u][2 * (i >> 1) + 1], sc[u][i & 1], 0, 0, 0);
      } else {
#pragma unroll
        for (int u = 0; u < QS; ++u)
          sc[u][i & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, kf), qf[u][i >> 1],
                                                                sc[u][i & 1], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Three loops, so that no accumulator is merged behind a branch: the tiles that every row of the
  // wave sees whole (in pairs, one per buffer), the ones from the first masked tile on, and those
  // only other waves need.
  auto whole = [&](const char* kb, char* next, int kt) {
    mx_wait_copies_and_barrier<0>();
    const PaScales q8 = q8n;
    advance(kt, next);
    float4_t sc[QS][2];
    scores(kb, sc);
    const PaV<RB, DT> vt(kb + 32 * RB, value_place());
    half8_t vf = pa_vfrag<RB, DT>(vt, 0);
    half8_t p[QS];
#pragma unroll
    for (int u = 0; u < QS; ++u) p[u] = pa_softmax<DT, false>(sc[u], rs, q8, 0, 3, mrun[u], lrun[u], o[u]);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const half8_t v = vf;
      if (f + 1 < NF) vf = pa_vfrag<RB, DT>(vt, f + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < QS; ++u)
        o[u][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[u], o[u][f], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Page ids of tiles kt and kt + 1 (kt even) lie in one load of ids, whose bits are at hand once
  // tile kt is on its way.
  int kt = 0;
  const int seen = all + 1 - k0;  // keys of the range that every row of the wave sees
  auto both_on = [&]() { return ((ids.on >> (2 * (kt & 31))) & 15) == 15; };
  for (; kt + 2 < ntile && kt + 2 <= nt_w && 32 * kt + 64 <= seen && both_on(); kt += 2) {
    whole(lds0, lds1, kt);
    whole(lds1, lds0, kt + 1);
  }
  int pos[QS];
#pragma unroll
  for (int u = 0; u < QS; ++u) {
    int hq;
    where(u, pos[u], hq);
    pos[u] += t.pos0;
  }
  for (; kt < nt_w; ++kt) {
    mx_wait_copies_and_barrier<0>();
    const int on = on_next;
    const PaScales q8 = q8n;
    if (kt + 1 < ntile) advance(kt, kt & 1 ? lds0 : lds1);
    const int tk = k0 + 32 * kt;
    const char* kb = kt & 1 ? lds1 : lds0;
    const char* vb = kb + 32 * RB;
    float4_t sc[QS][2];
    scores(kb, sc);
    const PaV<RB, DT> vt(vb, value_place());
    half8_t p[QS];
#pragma unroll
    for (int u = 0; u < QS; ++u)
      p[u] = pa_softmax<DT, true>(sc[u], rs, q8, pos[u] - tk - 4 * (pa_lane() >> 4), on, mrun[u], lrun[u], o[u]);
    uint32_t keep[4], odd = 0;
    pa_keep(any - tk, on, keep);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      half8_t v = pa_vfrag<RB, DT>(vt, f);
      if constexpr (DT != MX_DT_I8) v = pa_clean<true>(v, keep, odd);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < QS; ++u)
        o[u][f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[u], o[u][f], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (DT != MX_DT_I8)
      if (__builtin_amdgcn_ballot_w64(odd != 0)) {
        const uint32_t seen = ((on & 1) ? 0xFFFFu : 0u) | ((on & 2) ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int u = 0; u < QS; ++u) pa_add_odd<RB, NF>(vb, p[u], pos[u] - tk, seen, o[u]);
      }
  }
  for (; kt < ntile; ++kt) {
    mx_wait_copies_and_barrier<0>();
    if (kt + 1 < ntile) advance(kt, kt & 1 ? lds0 : lds1);
  }
  const int j1 = pa_lane() & 15, g1 = pa_lane() >> 4;
#pragma unroll
  for (int u = 0; u < QS; ++u) {
    const float l = pa_rowsum(lrun[u]);
    if (w0 + 16 * u + j1 >= t.nrows) continue;
    int tok, hq;
    where(u, tok, hq);
    const long tr = t.first + tok;
    const int at = (kvh * sp.slots + t.slot) * RT + (w0 - t.row0) + 16 * u + j1;
    if (k0 == 0 && g1 == 0) sp.rows[tr * a.nh + hq] = (int4_t){at, t.tiles * RT, t.ranges, 0};
    if (t.ranges > 1) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int d = 16 * f + 4 * g1;
        if (d < c.hd) *(float4_t*)(sp.po + (long)at * c.hd + d) = o[u][f];
      }
      if (g1 == 0) sp.ml[at] = make_float2(mrun[u], l);
      continue;
    }
    const float il = l == 0.f ? 0.f : 1.f / l;
    const float* gate = a.gate ? a.gate + tr * a.ldg + (long)hq * c.hd : nullptr;
    half_t* orow = (half_t*)a.out + tr * a.ldo + (long)hq * c.hd;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const int d = 16 * f + 4 * g1;
      if (d >= c.hd) continue;
      float4_t v = o[u][f] * il;
      if (gate) {
        const float4 gv = *(const float4*)(gate + d);
        v = (float4_t){v[0] * mx_sigmoid(gv.x), v[1] * mx_sigmoid(gv.y), v[2] * mx_sigmoid(gv.z),
                       v[3] * mx_sigmoid(gv.w)};
      }
      *(half4_t*)(orow + d) = (half4_t){(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
    }
  }
  __syncthreads();  // the buffers are free
  }
}

// ------------------------------------------------------------------------------------
// k_pa_f32: fp32 pages on v_mfma_f32_16x16x4_f32 (full fp32 products and sums), k_pa_keys' way: 16
// rows, keys dealt to the waves 16 at a time, keys in registers, values through the wave's LDS
// buffers.  The MFMA k-slot of lane group g at step r is key 4 g + r on both operands.  Bound by those
// instructions (a sixteenth of fp16's rate) and, in small calls, by their latency: 3 x 130 rows over 1500 tokens,
// 32 heads over 8 of 128: 131 us, 70 TFLOP/s.  Heads of 256 dims: 60 bytes of scratch.
// ------------------------------------------------------------------------------------
template <int DP, bool DIRECT>
__global__ __launch_bounds__(256, DP < 256 ? 2 : 1) void k_pa_f32(PkCache c, PkBatch b, PaArgs a, PaSched sp, int per) {
  constexpr int RB = DP * 4, NC = DP / 16, NL = RB / 64, CPR = RB / 16;
  constexpr int TILE = 16 * RB;
  __shared__ __align__(1024) char lds[4 * 2 * TILE];
  __shared__ float sm[4][16], sl[4][16];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kvh = blockIdx.y, first = 0;
  PaWork work;
  if constexpr (DIRECT) {  // one item per block, slot by range and sequence
    first = blockIdx.z * b.n_seqs + blockIdx.x;
    work.len = sp.least;
  } else {
    pa_head_of(c.nkv, &kvh, &first);
    work = pa_schedule<kKeysRows>(b, c, sp, a.group, per);
  }
  for (int item = first; DIRECT || item < work.items; item += per) {
  // Opaque: what follows from the lane is worked out per item and holds nothing across the loop.
  const int lane = pa_lane(), tid = 64 * wave + lane, j = lane & 15, g = lane >> 4;
  PaTile t;
  PaIds ids;  // lane l: the page of the wave's tile l
  const int mine = 16 * (wave + 4 * lane);
  if constexpr (DIRECT) {
    if (!pa_direct(b, c, a.group, work.len, mine, &t, &ids)) return;
  } else {
    if (!pa_item<kKeysRows>(b, c, a.group, work, item, &t)) continue;
    ids = pa_ids(b, c, t.seq, t.k0 + mine);
  }
  const int k0 = t.k0, k1 = min(t.kend, k0 + t.len);
  const int row = min(t.row0 + j, t.nrows - 1);
  const int tok = row / a.group, hq = kvh * a.group + row - tok * a.group;
  const int pos = t.pos0 + tok;
  const int rb = c.hd * 4;
  const float rs = mx_readlane(a.scale * kLog2e, 0);  // uniform: a scalar register
  float4 qf[NC];
  const float* qrow = (const float*)a.q + (long)(t.first + tok) * a.ldq + (long)hq * c.hd;
#pragma unroll
  for (int n = 0; n < NC; ++n) qf[n] = *(const float4*)(qrow + min(16 * n + 4 * g, c.hd - 4));
#pragma unroll
  for (int n = 0; n < NC; ++n)
    if (16 * n + 4 * g >= c.hd) qf[n] = make_float4(0.f, 0.f, 0.f, 0.f);

  const int ntile = pa_ceil(max(0, k1 - k0), 16);
  const int nw = ntile > wave ? (ntile - 1 - wave) / 4 + 1 : 0;
  char* const buf = lds + wave * 2 * TILE;
  uint32_t voff[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    // rows of a copy: 64 / CPR; value chunks XORed by 4 (row / 4), so the four rows of a read
    // lie in different banks
    const int r = i * (64 / CPR) + lane / CPR;
    voff[i] = (uint32_t)(r * rb + min(((lane % CPR) ^ ((r & 12) & (CPR - 1))) * 16, rb - 16));
  }
  auto base_of = [&](int i) {  // byte offset of the tile's first row in a pool
    const int key = k0 + 16 * (wave + 4 * i);
    const long row = (((long)__builtin_amdgcn_readlane(ids.id, i) * c.nkv + kvh) << c.ps_log) + (key & (c.ps - 1));
    return row * rb;
  };
  auto issue_v = [&](int i) {
    const pa_rsrc_t r = pa_rsrc(c.v + base_of(i), 16 * rb);
#pragma unroll
    for (int n = 0; n < NL; ++n) mx_copy_to_lds16(r, buf + (i & 1) * TILE + n * 1024, voff[n]);
  };
  float4 kr[NC];
  auto load_k = [&](int i) {
    const char* p = c.k + base_of(i);
#pragma unroll
    for (int n = 0; n < NC; ++n) kr[n] = *(const float4*)(p + (uint32_t)(j * rb + min(64 * n + 16 * g, rb - 16)));
  };
  // value of key 4 g + r, dim 16 f + j
  const int vlane = 4 * g * RB + (((j >> 2) ^ ((4 * g) & (CPR - 1))) * 16) + 4 * (j & 3);
  float4_t o[NC];
#pragma unroll
  for (int f = 0; f < NC; ++f) o[f] = (float4_t){0.f, 0.f, 0.f, 0.f};
  float mrun = kLow, lrun = 0.f;
  const int all = t.pos0 + t.row0 / a.group;
  if (nw > 0) {
    issue_v(0);
    load_k(0);
  }
  // `more`: a tile follows, issued without a branch, so that the waits leave it in flight.
  auto step = [&](int i, auto more) {
    constexpr bool MORE = decltype(more)::value;
    if constexpr (MORE) issue_v(i + 1);
    float4_t x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      x[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n].x, qf[n].x, x[0], 0, 0, 0);
      x[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n].y, qf[n].y, x[1], 0, 0, 0);
      x[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n].z, qf[n].z, x[2], 0, 0, 0);
      x[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[n].w, qf[n].w, x[3], 0, 0, 0);
    }
    const float4_t sc = (x[0] + x[1]) + (x[2] + x[3]);
    const int tk = k0 + 16 * (wave + 4 * i);
    const bool on = (ids.on >> i) & 1;
    if constexpr (MORE) load_k(i + 1);
    const bool mask = tk + 15 > all || !on;
    const int lim = pos - tk;
    float4_t s = sc * rs;
    if (mask) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * g + r > lim || !on) s[r] = -INFINITY;
    }
    const float mt = mx_rowmax4(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const bool up = mt > mrun + kTau;
    if (__builtin_amdgcn_ballot_w64(up)) {
      const float mnew = up ? mt : mrun;
      const float alpha = __builtin_amdgcn_exp2f(mrun - mnew);
      lrun *= alpha;
      mrun = mnew;
#pragma unroll
      for (int f = 0; f < NC; ++f) o[f] *= alpha;
    }
    float4_t p;
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(s[r] - mrun);
    lrun += (p[0] + p[1]) + (p[2] + p[3]);
    if constexpr (MORE) asm volatile("s_waitcnt vmcnt(%1)" : "+v"(p) : "n"(NL + NC) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" : "+v"(p) : : "memory");
    const char* tile = buf + (i & 1) * TILE;
    const int top = t.kend - 1 - tk;  // the last key any row sees
    bool odd = false;
    if (!mask) {
#pragma unroll
      for (int f = 0; f < NC; ++f)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          o[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(*(const float*)(tile + (vlane ^ (f * 64)) + r * RB), p[r],
                                                      o[f], 0, 0, 0);
      return;
    }
#pragma unroll
    for (int f = 0; f < NC; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = *(const float*)(tile + (vlane ^ (f * 64)) + r * RB);
        {
          const bool fin = (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u;
          const bool in = on && 4 * g + r <= top;
          odd |= in && !fin;
          v = in && fin ? v : 0.f;
        }
        o[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[r], o[f], 0, 0, 0);
      }
    if (__builtin_amdgcn_ballot_w64(odd)) {  // non-finite values that only some rows see
      for (int key = 0; key < 16; ++key) {
        const int e = key & 3;
        const float pe = e == 0 ? p[0] : e == 1 ? p[1] : e == 2 ? p[2] : p[3];
        const float pk = __shfl(pe, (key >> 2) * 16 + j);
        const int x16 = ((key & 12) & (CPR - 1)) * 16;
#pragma unroll
        for (int f = 0; f < NC; ++f) {
          const float4_t v = *(const float4_t*)(tile + key * RB + ((64 * f + 16 * g) ^ x16));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool bad = (__builtin_bit_cast(uint32_t, v[r]) & 0x7F800000u) == 0x7F800000u;
            if (bad && key <= lim) o[f][r] += pk * v[r];
          }
        }
      }
    }
  };
  for (int i = 0; i + 1 < nw; ++i) step(i, std::true_type{});
  if (nw > 0) step(nw - 1, std::false_type{});
  lrun = pa_rowsum(lrun);
  if (g == 0) {
    sm[wave][j] = mrun;
    sl[wave][j] = lrun;
  }
  __syncthreads();
  const float m = fmaxf(fmaxf(sm[0][j], sm[1][j]), fmaxf(sm[2][j], sm[3][j]));
  const float weight = __builtin_amdgcn_exp2f(mrun - m);
  float* const part = (float*)buf;
#pragma unroll
  for (int f = 0; f < NC; ++f) {
    const float4_t v = o[f] * weight;
    *(float4_t*)(part + j * DP + 16 * f + 4 * g) = v;
  }
  __syncthreads();
  constexpr int D4 = DP / 4;
  for (int i = tid; i < 16 * D4; i += 256) {
    const int r = i / D4, d = 4 * (i % D4);
    if (t.row0 + r >= t.nrows || d >= c.hd) continue;
    float4_t s = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f, mr = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      s += *(const float4_t*)((const float*)(lds + w * 2 * TILE) + r * DP + d);
      l += sl[w][r] * __builtin_amdgcn_exp2f(sm[w][r] - mr);
    }
    const int rt = (t.row0 + r) / a.group, h = kvh * a.group + (t.row0 + r) - rt * a.group;
    const long tr = t.first + rt;
    const int at = (kvh * sp.slots + t.slot) * kKeysRows + r;
    if (k0 == 0 && d == 0)
      sp.rows[tr * a.nh + h] = (int4_t){at, t.tiles * kKeysRows, t.ranges, 0};
    if (t.ranges > 1) {
      *(float4_t*)(sp.po + (long)at * c.hd + d) = s;
      if (d == 0) sp.ml[at] = make_float2(mr, l);
      continue;
    }
    s *= l == 0.f ? 0.f : 1.f / l;
    if (a.gate) {
      const float4 gv = *(const float4*)(a.gate + tr * a.ldg + (long)h * c.hd + d);
      s = (float4_t){s[0] * mx_sigmoid(gv.x), s[1] * mx_sigmoid(gv.y), s[2] * mx_sigmoid(gv.z),
                     s[3] * mx_sigmoid(gv.w)};
    }
    *(float4_t*)((float*)a.out + tr * a.ldo + (long)h * c.hd + d) = s;
  }
  if constexpr (DIRECT) return;
  __syncthreads();  // the buffers are free
  }
}

// ---- the launch ----------------------------------------------------------------------

enum PaKind { kKeys, kRows1, kRows2, kF32 };

struct PaPlan {
  PaKind kind;
  int rt;             // rows per tile
  int target, least, most, slots;  // PaSched's
  bool direct;        // one row tile per sequence, a block for every range there may be
  int per;            // blocks of a head
  bool join;          // a tile may have more than one range
  size_t ml, row, bytes;  // workspace: offsets and size
};

// Kernel, row tile and bounds of the schedule of a call, from its sizes alone.
int plan(const MxKvCache* c, const MxPagedBatch* b, int nh, PaPlan* p) {
  const int group = nh / c->n_kv_heads, nkv = c->n_kv_heads;
  const long max_q = b->max_q < b->rows ? b->max_q : b->rows;
  const long seqs = b->n_seqs, rows = (long)b->rows * group;
  if (rows >= (1l << 30)) return MX_ERR_UNSUPPORTED;
  p->kind = c->dtype == MX_DT_F32 ? kF32 : max_q * group <= kKeysRows ? kKeys : kRows1;
  const bool own = p->kind == kKeys || p->kind == kF32;
  // Two query sets per wave (128 rows) halve the LDS reads per product, but also the tiles: from about
  // 160 tiles of 64 rows on (4 x 200 rows over 3000 keys: 200 tiles, 112 us with one set, 86 with
  // two; 1 x 500 rows: 126 tiles, 25 and 30).  Int8 heads over 128 dims would spill.
  if (p->kind == kRows1 && !(c->dtype == MX_DT_I8 && c->head_dim > 128) && (rows / 64 + seqs) * nkv >= 160)
    p->kind = kRows2;
  p->rt = p->kind == kRows1 ? 64 : p->kind == kRows2 ? 128 : kKeysRows;
  const long tiles = rows / p->rt + (seqs < b->rows ? seqs : b->rows);  // at most, of a head
  const long keys = b->max_kv > 0 ? b->max_kv : 1;
  // Items: as many as blocks run at once, by their LDS.  k_pa_keys on rows of 512 bytes: one per CU (64
  // sequences of 8000 keys, 256 items 184 us, 512 items 191; 32 of 4000 57 and 64); 256 bytes: two
  // (int8, 48 ragged sequences, 256 items 33 us, 512 27); shorter rows four.
  const int row_bytes = c->head_dim * pk_esz(c->dtype);
  p->target = !own ? 512 : row_bytes > (c->dtype == MX_DT_F32 ? 512 : 256) ? 256 : row_bytes > 128 ? 512 : 1024;
  // The shortest range.  Up to 256 keys in one need no joining: decode steps over 250 cached tokens 11.0 us,
  // 12.3 in two ranges; but over 500 tokens 12.4 us in ranges of 128 and 14.6 in one.  Fp32 tiles
  // take longer: 2 x 500 tokens 16.1 us in ranges of 64, 19.5 of 128.
  p->least = p->kind == kF32 ? 64 : own && keys <= 256 ? 256 : 128;
  p->most = own ? kKeysMax : 1 << 30;
  // Items of a head, as pa_schedule comes to them: the tiles' ceil(keys / len) add up to at most tiles +
  // (keys of the tiles) / len, and len is above nkv (keys of the tiles) / target, or `most`; one or
  // two roundings of its 32-bit sum do not matter, since the extra are counted twice.
  const long capped = own ? tiles * (keys / kKeysMax) : 0;
  const long fine = tiles * (keys / p->least);
  const long extra = 2 * (p->target / nkv + 1);
  long slots = tiles + (extra > capped ? extra : capped);
  if (slots > tiles + fine) slots = tiles + fine;
  const long ranges = (keys + p->least - 1) / p->least;
  p->direct = own && max_q * group <= kKeysRows && seqs * ranges * nkv <= 256;
  if (p->direct) slots = seqs * ranges;
  if (slots * nkv * p->rt >= (1l << 31)) return MX_ERR_UNSUPPORTED;
  p->slots = (int)slots;
  long per = (p->target + nkv - 1) / nkv;
  if (per > slots || p->direct) per = slots;
  if (8 % nkv == 0) per = (per + 8 / nkv - 1) / (8 / nkv) * (8 / nkv);  // whole rounds of the XCDs
  p->per = (int)per;
  p->join = keys > p->least;
  const size_t n = p->join ? (size_t)slots * nkv * p->rt : 0;
  p->ml = mx_align_up(n * c->head_dim * 4, 256);
  p->row = p->ml + mx_align_up(n * 8, 256);
  p->bytes = p->row + (size_t)b->rows * nh * 16;
  return MX_OK;
}

template <int DT, bool DIRECT>
int launch(const PaPlan& p, const PkCache& c, const PkBatch& b, const PaArgs& a, const PaSched& sp, hipStream_t s) {
  const dim3 grid = DIRECT ? dim3(b.n_seqs, c.nkv, p.slots / b.n_seqs) : dim3(p.per * c.nkv);
  mx_clear_error();
  if constexpr (DT == MX_DT_F32) {
    auto* kern = c.hd <= 32    ? k_pa_f32<32, DIRECT>
                 : c.hd <= 64  ? k_pa_f32<64, DIRECT>
                 : c.hd <= 128 ? k_pa_f32<128, DIRECT>
                               : k_pa_f32<256, DIRECT>;
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, b, a, sp, p.per);
  } else {
    constexpr int ES = DT == MX_DT_I8 ? 1 : 2;
    const int rb = c.hd * ES;
    auto* kern = rb <= 64    ? k_pa_keys<64, DT, DIRECT>
                 : rb <= 128 ? k_pa_keys<128, DT, DIRECT>
                             : k_pa_keys<256, DT, DIRECT>;
    if constexpr (ES == 2)
      if (rb > 256) kern = k_pa_keys<512, DT, DIRECT>;
    if constexpr (!DIRECT) {
      if (p.kind == kRows1)
        kern = rb <= 64 ? k_pa_rows<64, DT, 1> : rb <= 128 ? k_pa_rows<128, DT, 1> : k_pa_rows<256, DT, 1>;
      if (p.kind == kRows2) kern = rb <= 64 ? k_pa_rows<64, DT, 2> : k_pa_rows<128, DT, 2>;
      if constexpr (ES == 2) {
        if (p.kind == kRows2 && rb > 128) kern = k_pa_rows<256, DT, 2>;
        if (p.kind == kRows1 && rb > 256) kern = k_pa_rows<512, DT, 1>;
        if (p.kind == kRows2 && rb > 256) kern = k_pa_rows<512, DT, 2>;
      }
    }
    hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, c, b, a, sp, p.per);
  }
  MX_TRY(mx_launch_status());
  if (!p.join) return MX_OK;
  typedef typename std::conditional<DT == MX_DT_F32, float, half_t>::type OT;
  if (p.rt == kKeysRows)
    hipLaunchKernelGGL((k_pa_join<OT, true>), dim3(b.rows, a.nh), dim3(256), 0, s, c, b, a, sp);
  else
    hipLaunchKernelGGL((k_pa_join<OT, false>), dim3(b.rows, mx_ceil_div(a.nh, 4)), dim3(256), 0, s, c, b, a, sp);
  return mx_launch_status();
}

int check(const MxKvCache* cache, const MxPagedBatch* batch, int n_heads) {
  MX_TRY(pk_check_cache(cache));
  MX_TRY(pk_check_batch(batch));
  if (n_heads <= 0 || n_heads % cache->n_kv_heads) return MX_ERR_INVALID;
  // (a key's number plus a range's length stays below 2^31)
  if (batch->max_kv > (1 << 30)) return MX_ERR_UNSUPPORTED;
  return n_heads > 65535 || (long)n_heads * batch->rows >= (1l << 26) ? MX_ERR_UNSUPPORTED : MX_OK;
}

}  // namespace

extern "C" int mx_paged_attn_workspace_size(const MxKvCache* cache, const MxPagedBatch* batch,
                                            int32_t n_heads, size_t* nbytes) {
  if (!nbytes) return MX_ERR_INVALID;
  MX_TRY(check(cache, batch, n_heads));
  *nbytes = 0;
  if (batch->rows == 0 || batch->n_seqs == 0) return MX_OK;
  PaPlan p;
  MX_TRY(plan(cache, batch, n_heads, &p));
  *nbytes = p.bytes;
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
  PaPlan p;
  MX_TRY(plan(cache, batch, args->n_heads, &p));
  if (!workspace || workspace_bytes < p.bytes) return MX_ERR_WORKSPACE;
  if (!mx_aligned16(workspace)) return MX_ERR_ALIGNMENT;
  const PkCache c = pk_cache(cache);
  const PkBatch b = pk_batch(batch);
  const PaArgs a{args->q, args->out, args->gate, args->ldq, args->ldo, args->ldg, args->n_heads,
                 args->n_heads / cache->n_kv_heads, args->scale};
  char* const ws = (char*)workspace;
  const PaSched sp{p.target, p.least, p.most, p.slots, p.slots * c.nkv * p.rt, (float*)ws, (float2*)(ws + p.ml), (int4_t*)(ws + p.row)};
  const hipStream_t s = (hipStream_t)stream;
  if (cache->dtype == MX_DT_F32)
    return p.direct ? launch<MX_DT_F32, true>(p, c, b, a, sp, s) : launch<MX_DT_F32, false>(p, c, b, a, sp, s);
  if (cache->dtype == MX_DT_F16)
    return p.direct ? launch<MX_DT_F16, true>(p, c, b, a, sp, s) : launch<MX_DT_F16, false>(p, c, b, a, sp, s);
  return p.direct ? launch<MX_DT_I8, true>(p, c, b, a, sp, s) : launch<MX_DT_I8, false>(p, c, b, a, sp, s);
}
