// Attention of a few query rows per request over the scaled 8-bit paged cache
// (gfx950): every key, a sliding window with first tokens that stay visible, or
// selected blocks.
//
// An item is a 16-row tile of a request: rows are (token, query head of the group)
// pairs, so a K/V byte is loaded once for all of them.  A workgroup works for one
// kv head, on one item whole or, where items are long or few, on an equal share of
// the units (32 keys each) of all items together, which leaves no last round of a
// ragged batch: it cuts at most its first and its last item, and
// cache8_merge_kernel joins what was cut.  The waves of a workgroup take an item's
// units in turn, entirely in registers:
//   S^T = K Q^T   v_mfma_f32_16x16x32: A = 16 keys x 32 dims.  The reduction
//         runs over the dims in any order, so a lane takes 16 contiguous bytes
//         of a key row per load (two steps) and Q's operand follows suit.
//   D layout: lane l holds row l % 16 and keys 4 (l / 16) + 0..3 of each of the
//         unit's two 16-key groups, which is an A operand of P with its keys in
//         a fixed order (slot j < 4: group 0, j >= 4: group 1);
//   O += P V  v_mfma_f32_16x16x32_f16: a lane loads D / 16 contiguous bytes of
//         each of its 8 keys (the 16 lanes of a key cover its row), and an 8 x 8
//         byte transpose by v_perm_b32 gives it the 8 keys of one dim per MFMA.
// A 16-key group lies in one page (page sizes are multiples of 16), so the K
// scale joins the softmax scale, and the V scale joins the exponent: with
// z' = z + log2 vs, p' = 2^(z' - m) weighs the bytes of V and p' / vs the sum l,
// so p' needs no range beyond the softmax's own.  p' and V's bytes are multiplied
// in fp16 whatever q's type is: the bytes are exact there and p' keeps 11 bits
// (half a step 2^-12; bf16 would lose 2^-9 of each weight).  The running maximum
// moves only when a z' exceeds it by 2^8 and is kept 2^7 below it, so p' stays
// below 2^15 and only weights under 2^-31 of the largest vanish.
#include <algorithm>

#include "cache8.h"
#include "mfma_common.h"

namespace srswa {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;
constexpr float kBelow = 7.f, kSlack = 8.f;   // the running maximum's place and play (log2)
constexpr int kGroup = 16;     // keys per page lookup; a unit is two groups
constexpr int kMergeWaves = 8;
// units of the smallest share: one request of 9,000 keys 19.2 us with 8, 17.9 with 16,
// 19.9 with 32; of 3,000 keys 14.5, 15.5, 20.4
constexpr int kMinShare = 16;

struct AttendK {
  srswa_cache8_attend_args a;
  int G;                  // query heads per kv head
  int tiles, items;       // row tiles per request at most, items in all
  bool dense;             // items numbered by the rows there are (tile_at), else R * tiles
  int shares;             // workgroups per kv head that share the items' units; 0: one per item
  bool pairs;             // D = 64: neighbouring heads to one XCD
  int rs, rm;             // rows of a record, rows that a workgroup of the merge joins
  int gpp;                // 16-key groups per page
  int64_t most_units;     // of an item
  float scale_l2;         // scale * log2(e)
  float* part;            // records: [shares][HKV][2][rs * (D + 2)], a share's first item and its last
};

// What a row tile reads, the same on every thread and in the merge kernel.
struct Tile {
  int r;                  // request
  int row0, nrows;        // rows of the tile: (token t, head g) = (row / G, row % G)
  int q0;                 // first query token of the request
  int p0;                 // position of the request's first query row
  int pmin, pmax;         // positions of the tile's first and last row
  int kend;               // keys that have a table entry
  int ng0, g1, units;     // groups of the first section, first group of the second, units in all
};

template <bool SEL>
__device__ __forceinline__ Tile tile_of(const AttendK& p, int r, int tile) {
  const srswa_cache8_attend_args& a = p.a;
  Tile t;
  t.r = r;
  const int q0 = a.cu_seqlens_q ? min(max(a.cu_seqlens_q[r], 0), a.total_q) : r * a.max_query_len;
  const int q1 = a.cu_seqlens_q ? min(max(a.cu_seqlens_q[r + 1], q0), a.total_q) : q0 + a.max_query_len;
  const int ql = min(q1 - q0, a.max_query_len);          // (later rows are not written; records hold no more)
  const int sl = max(a.seq_lens[r], 0);
  t.q0 = q0;
  t.p0 = sl - (q1 - q0);
  if constexpr (SEL) {                        // the heads of one token, 16 at a time
    const int per = (p.G + kRows - 1) / kRows;
    const int tok = tile / per, g0 = tile % per * kRows;
    t.row0 = tok * p.G + g0;
    t.nrows = tok < ql ? min(kRows, p.G - g0) : 0;
  } else {
    t.row0 = tile * kRows;
    t.nrows = (int)max((int64_t)0, min((int64_t)kRows, (int64_t)ql * p.G - t.row0));
  }
  t.kend = (int)min((int64_t)sl, (int64_t)a.max_blocks * a.page_size);
  t.pmin = t.p0 + t.row0 / p.G;
  t.pmax = t.nrows > 0 ? t.p0 + (t.row0 + t.nrows - 1) / p.G : -1;
  const int end = min(t.pmax + 1, t.kend);    // keys some row may see: [0, end)
  const int lo = a.window > 0 ? max(t.pmin - a.window + 1, 0) : 0;
  if constexpr (SEL) {
    t.ng0 = a.topk_n * p.gpp;                 // each slot's block, group by group
    t.g1 = lo / kGroup;
  } else {
    t.ng0 = lo > 0 ? (min(min(a.sinks, lo), max(end, 0)) + kGroup - 1) / kGroup : 0;   // first tokens
    t.g1 = max(lo / kGroup, t.ng0);
  }
  const int ng1 = SEL && a.window == 0 ? 0 : max((end + kGroup - 1) / kGroup - t.g1, 0);
  t.units = t.nrows > 0 ? (t.ng0 + ng1 + 1) / 2 : 0;
  return t;
}

// Item number `item`.  Where the requests' lengths are far below their bound, the items
// are numbered by the rows there are: request r's from first(r) = 16-row tiles before
// its first row + r on, which leaves every request as many as its rows can take.
template <bool SEL>
__device__ __forceinline__ Tile tile_at(const AttendK& p, int item) {
  if (!p.dense) return tile_of<SEL>(p, item / p.tiles, item % p.tiles);
  const srswa_cache8_attend_args& a = p.a;
  auto first = [&](int r) {
    return (int)((int64_t)min(max(a.cu_seqlens_q[r], 0), a.total_q) * p.G / kRows) + r;
  };
  int lo = 0, hi = a.R - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (first(mid) <= item) lo = mid;
    else hi = mid - 1;
  }
  return tile_of<SEL>(p, lo, max(item - first(lo), 0));
}

// Units that an item counts for: one at least, so that a row without keys is written.
template <bool SEL>
__device__ __forceinline__ uint32_t item_units(const AttendK& p, int item) {
  if (item >= p.items) return 0u;
  const Tile t = tile_at<SEL>(p, item);
  return t.nrows > 0 ? (uint32_t)max(t.units, 1) : 0u;
}

__device__ __forceinline__ uint32_t wave_prefix(uint32_t v, int lane) {   // inclusive
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint32_t x = __shfl_up(v, o, kWave);
    if (lane >= o) v += x;
  }
  return v;
}

// (a wave's 64 items sum below 2^32: a request holds 2^30 keys at most)
__device__ __forceinline__ int share_count(const AttendK& p, int64_t total) {
  return (int)max((int64_t)1, min((int64_t)p.shares, total / kMinShare));
}

// Share `id` of the items' units, [s, e), and the item that holds its first unit
// with the unit that item starts at; false past the last share.
struct Share {
  int64_t s, e, start;
  int item;
};
template <bool SEL>
__device__ __forceinline__ bool share_at(const AttendK& p, int id, int lane, Share* out) {
  const uint32_t n0 = item_units<SEL>(p, lane), incl0 = wave_prefix(n0, lane);   // of the first 64 items
  int64_t total = (uint32_t)__builtin_amdgcn_readlane((int)incl0, kWave - 1);
  for (int i0 = kWave; i0 < p.items; i0 += kWave) total += (uint32_t)wave_sum_int((int)item_units<SEL>(p, i0 + lane));
  const int n = share_count(p, total);
  if (id >= n) return false;
  out->s = total * id / n;
  out->e = total * (id + 1) / n;
  int64_t before = 0;
  for (int i0 = 0; i0 < p.items; i0 += kWave) {
    const uint32_t v = i0 == 0 ? n0 : item_units<SEL>(p, i0 + lane);
    const uint32_t incl = i0 == 0 ? incl0 : wave_prefix(v, lane);
    const uint64_t past = __ballot(before + (int64_t)incl > out->s);
    if (past) {
      const int i = __ffsll((long long)past) - 1;
      out->item = __builtin_amdgcn_readfirstlane(i0 + i);
      out->start = before + (uint32_t)__builtin_amdgcn_readlane((int)(incl - v), i);
      return true;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)incl, kWave - 1);
  }
  return false;
}

// 4 x 4 byte transpose: word t of the result holds byte t of a, b, c, d
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t* o) {
  const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab1 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd1 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  o[0] = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(cd1, ab1, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(cd1, ab1, 0x07060302u);
}

template <typename T>
__device__ __forceinline__ f32x4_t mfma16(const uint4& a, const uint4& b, f32x4_t c) {
  if constexpr (std::is_same<T, bf16_t>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
}

__device__ __forceinline__ float xor16_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Four or eight e4m3 bytes of V: those that are NaN, and the bytes without them.
__device__ __forceinline__ uint32_t nan_of(uint32_t v) { return nan_bytes4(v); }
__device__ __forceinline__ uint32_t nan_of(uint2 v) { return nan_bytes4(v.x) | nan_bytes4(v.y); }
__device__ __forceinline__ bool is_nan(uint32_t v, int d) { return (nan_bytes4(v) >> (8 * d + 7)) & 1u; }
__device__ __forceinline__ bool is_nan(uint2 v, int d) { return is_nan(d < 4 ? v.x : v.y, d % 4); }
__device__ __forceinline__ uint32_t without_nan(uint32_t v) { return without(v, nan_bytes4(v)); }
__device__ __forceinline__ uint2 without_nan(uint2 v) { return make_uint2(without_nan(v.x), without_nan(v.y)); }
__device__ __forceinline__ uint32_t shfl_bytes(uint32_t v, int l) { return __shfl(v, l, kWave); }
__device__ __forceinline__ uint2 shfl_bytes(uint2 v, int l) {
  return make_uint2(__shfl(v.x, l, kWave), __shfl(v.y, l, kWave));
}

// One unit's K and V bytes of a lane.
template <int D>
struct UnitBytes {
  static constexpr int DV = D / 16;                    // bytes per V key and lane
  uint4 k[2][D / 64];                                  // key l % 16 of each group
  std::conditional_t<DV == 8, uint2, uint32_t> v[8];   // keys 4 (l / 16) + 0..3 of each group
};

// Item rows' attention over units [u_lo, u_end) of theirs: to out and lse, or to a
// record (unnormalised, with m and l) where rec is not null.
// (MIX: a tile's rows may be of several tokens and V may hold NaN.)
template <typename T, int KV, int D, bool SEL, bool MIX, int NW>
__device__ __forceinline__ void attend_item(const AttendK& p, int h, const Tile& t, int u_lo, int u_end, float* rec) {
  constexpr int NT = NW * kWave;
  constexpr int NL = D / 64;      // K loads per group
  constexpr int DV = D / 16;      // V tiles
  using VB = std::conditional_t<DV == 8, uint2, uint32_t>;
  __shared__ float s_m[NW][kRows], s_l[NW][kRows];
  __shared__ __align__(16) float s_o[NW][kRows][D];
  const srswa_cache8_attend_args& a = p.a;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 15, g = lane >> 4, r = t.r;

  // Q operand: lane (row n, g) holds dims 64 i + 16 g + 8 e .. + 7 of step 2 i + e
  const int row = min(t.row0 + n, t.row0 + t.nrows - 1);
  const int tok = row / p.G, hq = h * p.G + row % p.G;
  uint4 qf[2 * NL];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(t.q0 + tok) * a.q_sn + (int64_t)hq * a.q_sh + 16 * g;
#pragma unroll
    for (int s = 0; s < 2 * NL; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + 64 * (s / 2) + 8 * (s % 2));
  }
  const int pr = n < t.nrows ? t.p0 + tok : -1;        // this lane's row position
  const int end = min(t.pmax + 1, t.kend);
  const int wlo = a.window > 0 ? t.pmin - a.window + 1 : 0;    // first key of the first row's window
  // the keys this lane's row sees: [my_lo, my_lo + my_span) and [0, my_first)
  const int my_hi = min(pr, t.kend - 1), my_lo = a.window > 0 ? max(pr - a.window + 1, 0) : 0;
  const uint32_t my_span = (uint32_t)max(my_hi - my_lo + 1, 0), my_first = (uint32_t)max(min(a.sinks, my_hi + 1), 0);
  const int32_t* topk = nullptr;
  const float* bias = nullptr;
  if constexpr (SEL) {
    const int64_t o = (int64_t)h * a.t_sh + (int64_t)(t.q0 + t.row0 / p.G) * a.t_sn;
    topk = a.topk + o;
    bias = a.bias ? a.bias + o : nullptr;
  }

  f32x4_t acc[DV];
#pragma unroll
  for (int d = 0; d < DV; ++d) acc[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, msub = 0.f, thr = -INFINITY, l = 0.f;   // m: the exponent that p' is relative to

  const uint8_t* kcache = reinterpret_cast<const uint8_t*>(a.k_cache) + (int64_t)h * a.k_sh;
  const uint8_t* vcache = reinterpret_cast<const uint8_t*>(a.v_cache) + (int64_t)h * a.v_sh;
  const int64_t koff = (int64_t)n * a.k_st + 16 * g;
  const int64_t voff = (int64_t)(4 * g) * a.v_st + DV * n;

  for (int u0 = u_lo + wave; u0 < u_end; u0 += NW * kWave) {
    // lane i looks up the two groups of this wave's i-th unit from here: first
    // key (-1: nothing to see), byte offsets, scales, bias and bounds
    int dk[2], dlo[2], dhi[2];
    uint64_t dko[2], dvo[2];
    float dks[2], dvi[2], db[2];
    bool whole = true;
    const int du = u0 + NW * lane;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int gi = 2 * du + e;
      int key = -1;
      db[e] = 0.f;
      dlo[e] = 0;
      dhi[e] = INT_MAX;
      if (du < u_end) {
        if (gi < t.ng0) {
          if constexpr (SEL) {
            const int slot = gi / p.gpp, sub = gi % p.gpp;
            const int id = topk[(int64_t)slot * a.t_sk];
            bool ok = id >= 0 && id < a.max_blocks;
            for (int s = 0; s < slot; ++s) ok = ok && topk[(int64_t)s * a.t_sk] != id;
            if (ok) key = id * a.page_size + sub * kGroup;
            dhi[e] = t.pmin - a.window;                // remote keys end before the window
            if (bias) {                                  // the lowest finite value stays finite in log2 units
              const float b = bias[(int64_t)slot * a.t_sk];
              db[e] = b > -INFINITY && b * kLog2e < -3.0e38f ? -3.0e38f : b * kLog2e;
            }
          } else {
            key = gi * kGroup;
          }
        } else {
          key = (t.g1 + gi - t.ng0) * kGroup;
          if constexpr (SEL) dlo[e] = t.pmin - a.window + 1;
        }
        if (key >= end || (SEL && key > dhi[e])) key = -1;
      }
      int page = -1;
      if (key >= 0) page = a.block_table[(int64_t)r * a.bt_sr + key / a.page_size];
      const bool ok = page >= 0 && page < a.num_pages;
      dk[e] = ok ? key : -1;
      const uint32_t pg = ok ? page : 0, rw = ok ? key % a.page_size : 0;   // (strides are below 2^31)
      dko[e] = (uint64_t)pg * (uint32_t)a.k_sp + (uint64_t)rw * (uint32_t)a.k_st;
      dvo[e] = (uint64_t)pg * (uint32_t)a.v_sp + (uint64_t)rw * (uint32_t)a.v_st;
      dks[e] = ok ? p.scale_l2 * a.k_scale[(int64_t)page * a.ks_sp + (int64_t)h * a.ks_sh] : 0.f;
      const float vs = ok ? fmaxf(a.v_scale[(int64_t)page * a.vs_sp + (int64_t)h * a.vs_sh], kScaleMin) : 1.f;
      dvi[e] = 0x1p-12f / vs;                    // (kLift)
      db[e] += __log2f(vs);
      const int last = key + kGroup - 1;
      if constexpr (SEL)
        whole = whole && ok && key >= dlo[e] && last <= dhi[e] && last < end;
      else
        whole = whole && ok && last <= t.pmin && last < t.kend &&
                (a.window == 0 || key > t.pmax - a.window || last < a.sinks);
    }
    const uint64_t whole_bits = __ballot(whole);
    settle(qf);
    const int cnt = min(kWave, (u_end - u0 + NW - 1) / NW);

    // One unit's bytes are held at a time: K's registers are loaded again as soon as
    // the products have read them, V's after the transposes, so a unit's K comes in
    // behind the softmax and its V behind the next products, and three waves fit a SIMD
    // (in the registers of four the loop spills: 48 uneven requests 297 us, not 220)
    UnitBytes<D> b;
    auto load_k = [&](int i) __attribute__((always_inline)) {
      i = min(i, cnt - 1);                       // (past the end: the last unit again, not used)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint8_t* kp = kcache + lane_u64(dko[e], i) + koff;
#pragma unroll
        for (int q = 0; q < NL; ++q) b.k[e][q] = *reinterpret_cast<const uint4*>(kp + 64 * q);
      }
    };
    auto load_v = [&](int i) __attribute__((always_inline)) {
      i = min(i, cnt - 1);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint8_t* vp = vcache + lane_u64(dvo[e], i) + voff;
#pragma unroll
        for (int j = 0; j < 4; ++j) b.v[4 * e + j] = *reinterpret_cast<const VB*>(vp + (int64_t)j * a.v_st);
      }
    };
    // (in this order, as in the loop: the wait for K then leaves V in flight)
    load_k(0);
    __builtin_amdgcn_sched_barrier(0);
    load_v(0);
    __builtin_amdgcn_sched_barrier(0);
    for (int i = 0; i < cnt; ++i) {
      // S^T
      f32x4_t sc[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < NL; ++q) {
          const uint2 k0 = bytes4_to<KV, T>(b.k[e][q].x), k1 = bytes4_to<KV, T>(b.k[e][q].y);
          const uint2 k2 = bytes4_to<KV, T>(b.k[e][q].z), k3 = bytes4_to<KV, T>(b.k[e][q].w);
          sc[e] = mfma16<T>(make_uint4(k0.x, k0.y, k1.x, k1.y), qf[2 * q], sc[e]);
          sc[e] = mfma16<T>(make_uint4(k2.x, k2.y, k3.x, k3.y), qf[2 * q + 1], sc[e]);
        }
      }
      load_k(i + 1);
      __builtin_amdgcn_sched_barrier(0);
      float z[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dks[e]), i));
        const float bl = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(db[e]), i));
#pragma unroll
        for (int j = 0; j < 4; ++j) z[4 * e + j] = fmaf(sc[e][j], ks, bl);
      }
      if (per_lane(!((whole_bits >> i) & 1))) {
        // some key is not visible to some row: its logit is -inf, and a key no
        // row sees has its V bytes cleared (0 * NaN would reach O)
        asm volatile("");                        // (a branch: not computed and selected for every unit)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = __builtin_amdgcn_readlane(dk[e], i) ;
          const int lo = SEL ? __builtin_amdgcn_readlane(dlo[e], i) : 0;
          const int hi = SEL ? __builtin_amdgcn_readlane(dhi[e], i) : 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = key + 4 * g + j;
            bool see, any;
            if constexpr (SEL) {                           // the tile's rows share one position
              see = any = (k >= lo) & (k <= hi) & (k < end);
            } else {
              see = ((uint32_t)(k - my_lo) < my_span) | ((uint32_t)k < my_first);
              any = (k < end) & ((k >= wlo) | (k < a.sinks));
            }
            see = see & (key >= 0);
            any = any & (key >= 0);
            z[4 * e + j] = see ? z[4 * e + j] : -INFINITY;
            if constexpr (DV == 8) {
              b.v[4 * e + j].x = any ? b.v[4 * e + j].x : 0u;
              b.v[4 * e + j].y = any ? b.v[4 * e + j].y : 0u;
            } else {
              b.v[4 * e + j] = any ? b.v[4 * e + j] : 0u;
            }
          }
        }
        if constexpr (MIX) {
          // a NaN of a key that only some of the rows see is set in their O here, and
          // is a zero in the products
          uint32_t nan = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) nan |= nan_of(b.v[j]);
          if (__any(nan != 0u)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int key = __builtin_amdgcn_readlane(dk[j / 4], i) + j % 4;
#pragma unroll 1
              for (int kg = 0; kg < 4; ++kg) {
                const VB w = shfl_bytes(b.v[j], 16 * kg + n);      // key `key + 4 kg`, this lane's dims of O
                if (!__any(nan_of(w) != 0u)) continue;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const int pos = t.p0 + (t.row0 + 4 * g + x) / p.G, k = key + 4 * kg;
                  const bool see = (k <= pos) & ((a.window == 0) | (k > pos - a.window) | (k < a.sinks));
#pragma unroll
                  for (int d = 0; d < DV; ++d) acc[d][x] = (see & is_nan(w, d)) ? NAN : acc[d][x];
                }
              }
              b.v[j] = without_nan(b.v[j]);
            }
          }
        }
      }
      float zm = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
      if (per_lane(__any(zm > thr))) {
        zm = xor32_max(xor16_max(zm));
        const float mn = fmaxf(m, zm - kBelow);
        const float alpha = mn == -INFINITY ? 1.f : exp2f(m - mn);
        m = mn;
        msub = mn == -INFINITY ? 0.f : mn;
        thr = mn + kBelow + kSlack;
        l *= alpha;
        float ar[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) ar[j] = __shfl(alpha, 4 * g + j, kWave);
#pragma unroll
        for (int d = 0; d < DV; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[d][j] *= ar[j];
      }
      const float vi0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dvi[0]), i));
      const float vi1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dvi[1]), i));
      float pe[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pe[j] = __builtin_amdgcn_exp2f(z[j] - msub);
        l = fmaf(pe[j], j < 4 ? vi0 : vi1, l);
      }
      const uint4 pa = make_uint4(pack_f16(pe[0], pe[1]), pack_f16(pe[2], pe[3]), pack_f16(pe[4], pe[5]),
                                  pack_f16(pe[6], pe[7]));
      // O += P V
      uint32_t tv[DV][2];                        // dim d's 8 keys
#pragma unroll
      for (int hf = 0; hf < DV / 4; ++hf) {
        uint32_t w[8], ta[4], tb[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (DV == 8) w[j] = hf ? b.v[j].y : b.v[j].x;
          else w[j] = b.v[j];
        }
        transpose4(w[0], w[1], w[2], w[3], ta);
        transpose4(w[4], w[5], w[6], w[7], tb);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          tv[4 * hf + d][0] = ta[d];
          tv[4 * hf + d][1] = tb[d];
        }
      }
      load_v(i + 1);
#pragma unroll
      for (int d = 0; d < DV; ++d) {
        const uint2 x0 = bytes4_to<KV, __half>(tv[d][0]), x1 = bytes4_to<KV, __half>(tv[d][1]);
        acc[d] = mfma16<__half>(pa, make_uint4(x0.x, x0.y, x1.x, x1.y), acc[d]);
      }
    }
  }

  // the waves' (m, l, O): O lane layout row 4 g + j, dims DV n + d
  l = xor32_sum(xor16_sum(l));
  if (g == 0) {
    s_m[wave][n] = m;
    s_l[wave][n] = l;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (4 * g + j < t.nrows) {
#pragma unroll
      for (int d = 0; d < DV; d += 4)
        *reinterpret_cast<float4*>(&s_o[wave][4 * g + j][DV * n + d]) =
            make_float4(acc[d][j], acc[d + 1][j], acc[d + 2][j], acc[d + 3][j]);
    }
  __syncthreads();
  for (int i = tid; i < t.nrows * (D / 4); i += NT) {
    const int rr = i / (D / 4), c = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_m[w][rr]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = s_m[w][rr] == -INFINITY ? 0.f : exp2f(s_m[w][rr] - M);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][rr][c]);
      L = fmaf(f, s_l[w][rr], L);
      o.x = fmaf(f, x.x, o.x); o.y = fmaf(f, x.y, o.y); o.z = fmaf(f, x.z, o.z); o.w = fmaf(f, x.w, o.w);
    }
    if (!rec) {
      const int ro = t.row0 + rr, ho = h * p.G + ro % p.G;
      const float inv = inv_sum(M, L);
      T* op = reinterpret_cast<T*>(a.out) + (int64_t)(t.q0 + ro / p.G) * a.o_sn + (int64_t)ho * a.o_sh + c;
      uint2 w;
      w.x = Mfma<T>::pack2(o.x * inv, o.y * inv);
      w.y = Mfma<T>::pack2(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(op) = w;
      if (a.lse && c == 0)
        a.lse[(int64_t)(t.q0 + ro / p.G) * a.lse_sn + (int64_t)ho * a.lse_sh] = lse_of(M, L);
    } else {
      *reinterpret_cast<float4*>(rec + rr * D + c) = o;
      if (c == 0) {
        rec[p.rs * D + rr] = M;
        rec[p.rs * D + p.rs + rr] = L;
      }
    }
  }
}

// shares == 0: one workgroup per (item, kv head).  Else workgroup (share, kv head)
// takes its equal part of all items' units.  The heads of one share run side by
// side, on neighbouring XCDs: their rows share DRAM pages (a share's heads on one
// XCD 305 us, one head's shares first 340 us against 261 us, 48 requests of 700 to
// 40,000 keys, ten heads).
template <typename T, int KV, int D, bool SEL, bool MIX, int NW>
__global__ __launch_bounds__(NW * kWave) __attribute__((amdgpu_waves_per_eu(3))) void cache8_decode_kernel(AttendK p) {
  const srswa_cache8_attend_args& a = p.a;
  const int lane = threadIdx.x % kWave;
  int h, id;
  if (D == 64 && p.pairs) {
    // two heads' rows share a 128-byte line: both on one XCD, so it is fetched once
    const int half = a.HKV / 2, pair = (int)blockIdx.x / 16 * 8 + (int)blockIdx.x % 8;
    h = pair % half * 2 + (int)(blockIdx.x / 8 & 1);
    id = pair / half;
    if (id >= (p.shares > 0 ? p.shares : p.items)) return;
  } else {
    h = (int)blockIdx.x % a.HKV;
    id = (int)blockIdx.x / a.HKV;
  }
  if (p.shares == 0) {
    const Tile t = tile_at<SEL>(p, id);
    if (t.nrows > 0) attend_item<T, KV, D, SEL, MIX, NW>(p, h, t, 0, t.units, nullptr);
    return;
  }
  Share sh;
  if (!share_at<SEL>(p, id, lane, &sh)) return;
  int64_t s = sh.s, start = sh.start;
  const int64_t e = sh.e;
  int item = sh.item;
  float* recs = p.part + ((int64_t)id * a.HKV + h) * 2 * p.rs * (D + 2);
  for (bool first = true; s < e; ++item) {
    const Tile t = tile_at<SEL>(p, item);
    if (t.nrows == 0) continue;
    const int64_t end = start + max(t.units, 1);
    const bool whole = s == start && e >= end;
    if (!first) __syncthreads();                 // the item before is written from LDS
    attend_item<T, KV, D, SEL, MIX, NW>(p, h, t, (int)(s - start), (int)min((int64_t)t.units, min(e, end) - start),
                                   whole ? nullptr : recs + (first ? 0 : p.rs * (D + 2)));
    first = false;
    s = start = end;
  }
}

// Joins the shares of an item that was cut: one workgroup per (item, kv head, rm rows),
// D / 64 dims a lane, its eight waves shared among the rows, or a row's records among
// waves where rows are few (one request of 30,000 keys, 59 records a row: 42.9 us with
// one wave, 29.8 with four, 28.8 with eight).  rm is as small as 2,048 workgroups allow
// (16 rows after 30,000 keys: 32 us with a row each, 73 with all 16; 256 requests of 4
// rows 460 and 392).  Share i begins with the item (its first
// record) unless the item starts inside it (its last).
template <typename T, int D, bool SEL>
__global__ __launch_bounds__(kMergeWaves * kWave) void cache8_merge_kernel(AttendK p) {
  constexpr int DL = D / kWave;
  __shared__ float s_o[kMergeWaves][D], s_l[kMergeWaves];
  const srswa_cache8_attend_args& a = p.a;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int parts = (p.rs + p.rm - 1) / p.rm, id = (int)blockIdx.x / parts;
  const int h = id % a.HKV, item = id / a.HKV;
  const Tile t = tile_at<SEL>(p, item);
  const int first = (int)blockIdx.x % parts * p.rm, last = min(first + p.rm, t.nrows);
  if (first >= last) return;
  int64_t start = 0, total = 0;
  for (int i0 = 0; i0 < p.items; i0 += kWave) {
    const int n = (int)item_units<SEL>(p, i0 + lane);
    total += (uint32_t)wave_sum_int(n);
    start += (uint32_t)wave_sum_int(i0 + lane < item ? n : 0);
  }
  const int64_t end = start + max(t.units, 1);
  const int n = share_count(p, total);
  // the shares that hold units start and end - 1: share i is [total i / n, total (i + 1) / n)
  auto share_of = [&](int64_t u) {
    int i = (int)(u * n / total);
    while (total * (i + 1) / n <= u) ++i;
    while (total * i / n > u) --i;
    return i;
  };
  const int s0 = share_of(start), s1 = share_of(end - 1);
  if (s0 == s1) return;                          // not cut
  const int64_t rsz = (int64_t)p.rs * (D + 2);
  const int late = total * s0 / n != start ? 1 : 0;
  auto record = [&](int i) { return p.part + (((int64_t)i * a.HKV + h) * 2 + (i == s0 ? late : 0)) * rsz; };
  int per = kMergeWaves;                         // waves per row
  while (per > 1 && per * (last - first) > kMergeWaves) per >>= 1;
  const int sub = wave % per;
  for (int r0 = first; r0 < last; r0 += kMergeWaves / per) {
    const int rr = r0 + wave / per;
    float M = -INFINITY, o[DL] = {}, L = 0.f;
    if (rr < last) {
      for (int i = s0 + lane; i <= s1; i += kWave) M = fmaxf(M, record(i)[p.rs * D + rr]);
      M = wave_max(M);
#pragma unroll 8
      for (int i = s0 + sub; i <= s1; i += per) {
        const float* rec = record(i);
        const float mk = rec[p.rs * D + rr];
        const float f = mk == -INFINITY ? 0.f : exp2f(mk - M);
        L = fmaf(f, rec[p.rs * D + p.rs + rr], L);
#pragma unroll
        for (int d = 0; d < DL; ++d) o[d] = fmaf(f, rec[rr * D + DL * lane + d], o[d]);
      }
    }
    if (per > 1) {
      if (r0 > first) __syncthreads();           // the rows before are read
#pragma unroll
      for (int d = 0; d < DL; ++d) s_o[wave][DL * lane + d] = o[d];
      if (lane == 0) s_l[wave] = L;
      __syncthreads();
#pragma unroll
      for (int w = 1; w < kMergeWaves; ++w) {
        const int from = min(wave + w, kMergeWaves - 1);
        L += w < per ? s_l[from] : 0.f;
#pragma unroll
        for (int d = 0; d < DL; ++d) o[d] += w < per ? s_o[from][DL * lane + d] : 0.f;
      }
    }
    if (sub > 0 || rr >= last) continue;
    const int ro = t.row0 + rr, ho = h * p.G + ro % p.G;
    const float inv = inv_sum(M, L);
    T* op = reinterpret_cast<T*>(a.out) + (int64_t)(t.q0 + ro / p.G) * a.o_sn + (int64_t)ho * a.o_sh + DL * lane;
    if constexpr (DL == 2) {
      *reinterpret_cast<uint32_t*>(op) = Mfma<T>::pack2(o[0] * inv, o[1] * inv);
    } else {
      *reinterpret_cast<uint16_t*>(op) = (uint16_t)(Mfma<T>::pack2(o[0] * inv, 0.f) & 0xffffu);
    }
    if (a.lse && lane == 0)
      a.lse[(int64_t)(t.q0 + ro / p.G) * a.lse_sn + (int64_t)ho * a.lse_sh] = lse_of(M, L);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int cache8_check(const srswa_cache8_attend_args* a, const char* what) {
  if (!a || !a->q || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->block_table || !a->seq_lens ||
      !a->out) {
    set_error("%s: null argument", what);
    return SRSWA_INVALID;
  }
  if (a->R < 0 || a->total_q < 0 || a->max_query_len < 0 || a->HQ <= 0 || a->HKV <= 0 || a->topk_n < 0 ||
      a->max_blocks <= 0 || a->num_pages <= 0 || a->page_size <= 0 || a->window < 0 || a->sinks < 0 ||
      (!a->cu_seqlens_q && (int64_t)a->R * a->max_query_len != a->total_q)) {
    set_error("%s: bad sizes", what);
    return SRSWA_INVALID;
  }
  if (a->HQ % a->HKV) {
    set_error("%s: HQ=%d must be a multiple of HKV=%d", what, a->HQ, a->HKV);
    return SRSWA_UNSUPPORTED;
  }
  if (!(a->D == 64 || a->D == 128) || !(a->dtype == SRSWA_BF16 || a->dtype == SRSWA_F16) ||
      !(a->kv_dtype == SRSWA_I8 || a->kv_dtype == SRSWA_FP8_E4M3FN)) {
    set_error("%s: D=%d / dtype %d / cache format %d not supported", what, a->D, a->dtype, a->kv_dtype);
    return SRSWA_UNSUPPORTED;
  }
  if (a->page_size % 16 || a->page_size > 1024 || (int64_t)a->max_blocks * a->page_size > (1 << 30) ||
      a->window > (1 << 30) || a->sinks > (1 << 30)) {
    set_error("%s: page size %d must be a multiple of 16 up to 1024, and %d of them at most 2^30 keys", what,
              a->page_size, a->max_blocks);
    return SRSWA_UNSUPPORTED;
  }
  const int64_t qs[] = {a->q_sn, a->q_sh, a->o_sn, a->o_sh};
  for (int64_t s : qs)
    if (s % 8) {
      set_error("%s: strides must keep rows 16-byte aligned", what);
      return SRSWA_UNSUPPORTED;
    }
  const int64_t ks[] = {a->k_sp, a->k_st, a->k_sh, a->v_sp, a->v_st, a->v_sh};
  for (int64_t s : ks)
    if (s % 16 || s < 0 || s > INT32_MAX) {
      set_error("%s: cache strides must keep rows 16-byte aligned and be below 2^31", what);
      return SRSWA_UNSUPPORTED;
    }
  if (a->k_st >= 1 << 28 || a->v_st >= 1 << 28) {     // (16 rows of a group lie within 2^32 bytes)
    set_error("%s: token strides must be below 2^28", what);
    return SRSWA_UNSUPPORTED;
  }
  if (a->ks_sp < 0 || a->ks_sp > INT32_MAX || a->vs_sp < 0 || a->vs_sp > INT32_MAX) {
    set_error("%s: scale strides must be below 2^31", what);
    return SRSWA_UNSUPPORTED;
  }
  if (!al16(a->q) || !al16(a->k_cache) || !al16(a->v_cache) || !al16(a->out)) {
    set_error("%s: pointers must be 16-byte aligned", what);
    return SRSWA_UNSUPPORTED;
  }
  if (a->topk && (a->window <= 0 && a->topk_n == 0)) {
    set_error("%s: selected blocks need slots or a window", what);
    return SRSWA_INVALID;
  }
  return SRSWA_OK;
}

namespace {

// Short items are taken whole, others shared by as many workgroups as the GPU holds
// at once.  Whole needs no second launch and no count of the items, but leaves CUs
// idle where the workgroups are few: one request of ten heads 9.6 us whole against
// 14.9 shared at 777 keys, 21.6 against 15.4 at 3,000 (94 units); four of 1,000 to
// 4,000 keys 24.1 against 20.4, eight 25.4 against 25.0, 24 of 400 to 3,000 keys 23.1
// against 30.9, 24 of 400 to 6,000 keys 48.2 against 43.5.
AttendK plan(const srswa_cache8_attend_args* a) {
  AttendK p{};
  p.a = *a;
  p.G = a->HQ / a->HKV;
  p.gpp = a->page_size / kGroup;
  p.scale_l2 = a->scale * kLog2e;
  const int64_t rows = (int64_t)a->max_query_len * p.G;
  p.tiles = (int)(a->topk ? (int64_t)a->max_query_len * ((p.G + kRows - 1) / kRows) : (rows + kRows - 1) / kRows);
  const int64_t even = (int64_t)a->R * p.tiles, own = (int64_t)a->total_q * p.G / kRows + a->R;
  p.dense = a->cu_seqlens_q && own < even;
  const int64_t items = p.dense ? own : even;
  p.items = (int)std::min<int64_t>(items, INT32_MAX);
  p.rs = (int)std::min<int64_t>(kRows, a->topk ? p.G : rows);
  p.rm = 1;
  while (p.rm < p.rs && items * a->HKV * ((p.rs + p.rm - 1) / p.rm) > 2048) p.rm *= 2;
  int64_t groups = (int64_t)a->max_blocks * a->page_size / kGroup;
  if (a->topk) groups = (int64_t)a->topk_n * p.gpp + std::min<int64_t>(groups, a->window / kGroup + 2);
  else if (a->window > 0)
    groups = std::min<int64_t>(groups, ((int64_t)a->window + a->max_query_len) / kGroup + 2 + (a->sinks + kGroup - 1) / kGroup);
  const int64_t units = (groups + 1) / 2, wgs = items * a->HKV;
  p.most_units = units;
  p.pairs = a->D == 64 && a->HKV % 2 == 0;
  int cus = device_cu_count();
  if (cus <= 0) cus = 256;
  if (units > 128 || (units > 64 && wgs <= 64))
    p.shares = (int)std::min<int64_t>(std::max(1, (a->D == 64 ? 4 : 3) * cus / a->HKV),
                                      (units * p.items + kMinShare - 1) / kMinShare);
  return p;
}

size_t ws_bytes_of(const AttendK& p) {
  return (size_t)p.shares * p.a.HKV * 2 * p.rs * (p.a.D + 2) * sizeof(float);
}

template <typename T, int KV, int D, bool SEL>
void launch(const AttendK& p, unsigned grid, hipStream_t st) {
  // (the code that a NaN of a key which not every row sees takes costs 48 uneven
  // single-token requests 5%)
  constexpr bool kMix = KV == kFp8E4M3FN && !SEL;
  if (kMix && p.a.max_query_len > 1) cache8_decode_kernel<T, KV, D, SEL, kMix, 4><<<grid, 4 * kWave, 0, st>>>(p);
  else cache8_decode_kernel<T, KV, D, SEL, false, 4><<<grid, 4 * kWave, 0, st>>>(p);
  if (p.shares > 0)
    cache8_merge_kernel<T, D, SEL><<<(unsigned)(p.items * p.a.HKV * ((p.rs + p.rm - 1) / p.rm)),
                                     kMergeWaves * kWave, 0, st>>>(p);
}
template <typename T, int KV, int D>
void launch_sel(const AttendK& p, unsigned grid, hipStream_t st) {
  if (p.a.topk) launch<T, KV, D, true>(p, grid, st);
  else launch<T, KV, D, false>(p, grid, st);
}
template <typename T, int KV>
void launch_d(const AttendK& p, unsigned grid, hipStream_t st) {
  if (p.a.D == 64) launch_sel<T, KV, 64>(p, grid, st);
  else launch_sel<T, KV, 128>(p, grid, st);
}
template <typename T>
void launch_kv(const AttendK& p, unsigned grid, hipStream_t st) {
  if (p.a.kv_dtype == SRSWA_I8) launch_d<T, kI8>(p, grid, st);
  else launch_d<T, kFp8E4M3FN>(p, grid, st);
}

}  // namespace

int cache8_decode_run(const srswa_cache8_attend_args* a, void* ws, size_t ws_bytes, void* stream, const char* what) {
  AttendK p = plan(a);
  const size_t need = ws_bytes_of(p);
  if (need > 0 && (!ws || ws_bytes < need)) {
    set_error("%s: workspace of %zu bytes required (got %zu)", what, need, ws_bytes);
    return SRSWA_WORKSPACE;
  }
  p.part = reinterpret_cast<float*>(ws);
  const int64_t wgs = (int64_t)(p.shares > 0 ? p.shares : p.items) * a->HKV;
  const int64_t grid = p.pairs ? (wgs / 2 + 7) / 8 * 16 : wgs;
  if (grid > 0x7fffffff || (int64_t)p.items * a->HKV * ((p.rs + p.rm - 1) / p.rm) > 0x7fffffff) {
    set_error("%s: grid too large", what);
    return SRSWA_UNSUPPORTED;
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->dtype == SRSWA_BF16) launch_kv<bf16_t>(p, (unsigned)grid, st);
  else launch_kv<__half>(p, (unsigned)grid, st);
  return cache8_launched(what);
}

size_t cache8_decode_ws(const srswa_cache8_attend_args* a) { return ws_bytes_of(plan(a)); }

void cache8_decode_load(const srswa_cache8_attend_args* a, int64_t* wgs, int64_t* units, bool* shared) {
  const AttendK p = plan(a);
  *wgs = (int64_t)p.items * a->HKV;
  *units = p.most_units;
  *shared = p.shares > 0;
}

}  // namespace srswa

using namespace srswa;

extern "C" size_t srswa_cache8_decode_workspace(const srswa_cache8_attend_args* a) {
  return cache8_plannable(a) ? cache8_decode_ws(a) : 0;
}
extern "C" int srswa_cache8_decode(const srswa_cache8_attend_args* a, void* ws, size_t ws_bytes, void* stream) {
  const int rc = cache8_check(a, "cache8 decode");
  if (rc != SRSWA_OK || !cache8_plannable(a) || a->total_q == 0) return rc;
  return cache8_decode_run(a, ws, ws_bytes, stream, "cache8 decode");
}
