// Attention of many query rows per request over the scaled 8-bit paged cache
// (gfx950, matrix cores).
//
// One workgroup = (request, kv head, tile of 128 rows, part of its keys): four
// waves of 32 rows, a row being a (token, query head of the group) pair, two
// workgroups per CU.  Per chunk of 64 keys:
//   * the next chunk's bytes, fetched into registers one chunk before, are
//     converted once for all four waves and stored to the other LDS buffer, K in
//     q's type and V in fp16 (both exact), beside the products K Q^T: one barrier
//     per chunk;
//   * S^T = K Q^T on v_mfma_f32_32x32x16: every lane owns one row and 32 keys;
//   * a 16-key group lies in one page, so its scales are uniform: z' = scale ks s
//     + log2 vs - m in one FMA, p' = 2^z' weighs V's bytes, l += p' / vs (see
//     cache8_decode.hip for the range of p');
//   * O^T += V^T P^T in fp16, V^T read by ds_read_b64_tr_b16.
// A chunk that every row of a wave sees whole takes no mask.  Parts (few tiles, long keys) write fp32 records that
// cache8_join_kernel combines.
#include <algorithm>
#include <cstdlib>
#include <cstring>

#include "cache8.h"
#include "mfma_common.h"

namespace srswa {
namespace {

constexpr int kThreads = 256;
constexpr int kRowsWg = 128;
constexpr int kGroup = 16;
constexpr int kXcds = 8;
constexpr int kMinChunks = 4;
constexpr float kBelow = 7.f, kSlack = 8.f;

struct PrefillK {
  srswa_cache8_attend_args a;
  int G, tiles, nsplit;           // tiles: of all requests at most
  uint32_t page_mul;              // key / page_size = umulhi(key, page_mul) >> page_shift
  int page_shift;
  int64_t chunks;                 // of a tile at most
  float scale_l2;
  bool by_group;                  // the tiles of a group to one XCD, else in turn
  float* part;                    // [tiles][HKV][nsplit][128 * (D + 2)]
};

template <int D> struct Lds {
  // row pitches (16-bit elements): K rows 4 banks apart, so 16 lanes' 16 bytes of
  // 16 rows meet no bank twice; V rows 16 banks (of 64) apart, so the two 16-lane
  // groups of a transposing read (4 rows x 64 bytes) do not either
  static constexpr int KP = D + 8, VP = D + 32;
  static constexpr int kBytes = kChunk * KP * 2, vBytes = kChunk * VP * 2;
  static constexpr int buf = kBytes + vBytes + 64;       // + four float4 of the groups
  static constexpr int total = 2 * buf;
};

struct Tile {
  int row0, nrows, q0, p0, pmin, pmax, kend, end, c0, c1, chunks;
};

// What a tile of rows reads: chunks [0, c0) hold the first tokens it sees past
// its window, chunks c1 .. the rest.
__device__ __forceinline__ Tile tile_of(const PrefillK& p, int r, int tile) {
  const srswa_cache8_attend_args& a = p.a;
  Tile t;
  const int q0 = min(max(a.cu_seqlens_q[r], 0), a.total_q), q1 = min(max(a.cu_seqlens_q[r + 1], q0), a.total_q);
  const int ql = min(q1 - q0, a.max_query_len);
  const int sl = max(a.seq_lens[r], 0);
  t.q0 = q0;
  t.p0 = sl - (q1 - q0);
  t.row0 = tile * kRowsWg;
  t.nrows = (int)max((int64_t)0, min((int64_t)kRowsWg, (int64_t)ql * p.G - t.row0));
  t.kend = (int)min((int64_t)sl, (int64_t)a.max_blocks * a.page_size);
  t.pmin = t.p0 + t.row0 / p.G;
  t.pmax = t.nrows > 0 ? t.p0 + (t.row0 + t.nrows - 1) / p.G : -1;
  t.end = min(t.pmax + 1, t.kend);
  const int lo = a.window > 0 ? max(t.pmin - a.window + 1, 0) : 0;
  t.c0 = lo > 0 ? (min(min(a.sinks, lo), max(t.end, 0)) + kChunk - 1) / kChunk : 0;
  t.c1 = max(lo / kChunk, t.c0);
  t.chunks = t.c0 + max((t.end + kChunk - 1) / kChunk - t.c1, 0);
  return t;
}

// Tile number b over all requests' own tiles: its request and place there, the
// same on every lane; false past the last.
__device__ __forceinline__ bool nth_tile(const PrefillK& p, int b, int lane, int* r, int* tile) {
  const srswa_cache8_attend_args& a = p.a;
  int before = 0;
  for (int r0 = 0; r0 < a.R; r0 += kWave) {
    int n = 0;
    if (r0 + lane < a.R) {
      const int q0 = min(max(a.cu_seqlens_q[r0 + lane], 0), a.total_q);
      const int q1 = min(max(a.cu_seqlens_q[r0 + lane + 1], q0), a.total_q);
      n = (int)(((int64_t)min(q1 - q0, a.max_query_len) * p.G + kRowsWg - 1) / kRowsWg);
    }
    int incl = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int x = __shfl_up(incl, o, kWave);
      if (lane >= o) incl += x;
    }
    const uint64_t past = __ballot(before + incl > b);
    if (past) {
      const int i = __ffsll((long long)past) - 1;
      *r = __builtin_amdgcn_readfirstlane(r0 + i);
      *tile = __builtin_amdgcn_readfirstlane(b - before - __shfl(incl - n, i, kWave));
      return true;
    }
    before += __shfl(incl, kWave - 1, kWave);
  }
  return false;
}

// Parts of a tile: at least kMinChunks chunks each.
__device__ __forceinline__ int parts_of(const PrefillK& p, const Tile& t) {
  return max(1, min(p.nsplit, t.chunks / kMinChunks));
}

template <typename T, int KV, int D, bool ONE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void cache8_prefill_kernel(PrefillK p) {
  using L = Lds<D>;
  constexpr int KP = L::KP, VP = L::VP;
  constexpr int KS = D / 16, MT = D / 32;
  constexpr int PPR = D / 8;                     // 8-byte pieces per key row
  constexpr int NP = kChunk * PPR / kThreads;    // pieces of K (and of V) per thread
  constexpr int RPP = kThreads / PPR;            // key rows per pass
  extern __shared__ __align__(16) unsigned char smem[];
  const srswa_cache8_attend_args& a = p.a;
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int rl = lane & 31, hh = lane >> 5;

  // The hardware deals workgroups to the XCDs in turn.  One request: the tiles of
  // one (head, part), which read the same keys, stay on one XCD's L2, the later,
  // longer ones first.  Several: workgroups count only the tiles that the requests
  // have, so every XCD gets as many to one (six requests of 70 to 1,900 rows, ten
  // heads, 500 tiles for 512 places: 81 -> 58 us against tiles up to the longest).
  int r, tile, nth, h, part;
  if (p.by_group) {
    const int gi = (int)(blockIdx.x % kXcds) + kXcds * (int)(blockIdx.x / kXcds / p.tiles);
    if (gi >= a.HKV * p.nsplit) return;
    tile = nth = p.tiles - 1 - (int)(blockIdx.x / kXcds % p.tiles);
    part = gi % p.nsplit;
    h = gi / p.nsplit;
    r = 0;
  } else {
    const int b = (int)blockIdx.x / p.nsplit;
    part = (int)blockIdx.x % p.nsplit;
    h = b % a.HKV;
    nth = b / a.HKV;
    if (!nth_tile(p, nth, lane, &r, &tile)) return;
  }
  const Tile t = tile_of(p, r, tile);
  if (t.nrows == 0) return;
  const int parts = parts_of(p, t);
  if (part >= parts) return;
  const int u_lo = (int)((int64_t)t.chunks * part / parts), u_hi = (int)((int64_t)t.chunks * (part + 1) / parts);

  const int wrow = wave * 32 + rl;
  const int row = t.row0 + min(wrow, t.nrows - 1);
  const int tok = row / p.G, hq = h * p.G + row % p.G;
  uint4 qf[KS];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + (int64_t)(t.q0 + tok) * a.q_sn + (int64_t)hq * a.q_sh + 8 * hh;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + 16 * s);
  }
  const int pr = wrow < t.nrows ? t.p0 + tok : -1;
  // the keys this row sees: [my_lo, my_lo + my_span) and [0, my_first)
  const int my_hi = min(pr, t.kend - 1), my_lo = a.window > 0 ? max(pr - a.window + 1, 0) : 0;
  const uint32_t my_span = (uint32_t)max(my_hi - my_lo + 1, 0), my_first = (uint32_t)max(min(a.sinks, my_hi + 1), 0);
  const bool wave_live = wave * 32 < t.nrows;
  const int wpmin = t.p0 + (t.row0 + min(wave * 32, t.nrows - 1)) / p.G;
  const int wpmax = t.p0 + (t.row0 + min(wave * 32 + 31, t.nrows - 1)) / p.G;

  // staging: piece i of a thread is 8 bytes of row srow + i RPP of the chunk.  A
  // wave's rows of one pass lie in one 16-key group, so its page and the address
  // of the group's first row are scalar, and a lane adds a constant offset.  Every
  // load is unconditional, from clamped pages and keys (a branch around one would
  // have its registers waited for where the paths meet); what no row may see is
  // zeroed as it is stored, for 0 * NaN would reach O.
  const int srow = tid / PPR, scol = tid % PPR * 8;
  const int wgrp = wave * kWave / PPR / kGroup;                     // the wave's group in pass 0
  // (from the chunk's first row where ONE: its 64 rows lie within 2^31 bytes)
  uint32_t kpiece[ONE ? NP : 1], vpiece[ONE ? NP : 1];
#pragma unroll
  for (int i = 0; i < (ONE ? NP : 1); ++i) {
    const uint32_t from = (uint32_t)(ONE ? srow + i * RPP : srow - wgrp * kGroup);
    kpiece[i] = from * (uint32_t)a.k_st + scol;
    vpiece[i] = from * (uint32_t)a.v_st + scol;
  }
  // ONE: read through the scalar cache (constant address space)
  using Table = std::conditional_t<ONE, const __attribute__((address_space(4))) int32_t*, const int32_t*>;
  const Table bt = (Table)(a.block_table + (int64_t)r * a.bt_sr);
  const uint8_t* kcache = reinterpret_cast<const uint8_t*>(a.k_cache) + (int64_t)h * a.k_sh;
  const uint8_t* vcache = reinterpret_cast<const uint8_t*>(a.v_cache) + (int64_t)h * a.v_sh;
  const float *kscale = a.k_scale + (int64_t)h * a.ks_sh, *vscale = a.v_scale + (int64_t)h * a.vs_sh;
  auto base_of = [&](int u) { return (u < t.c0 ? u : t.c1 + u - t.c0) * kChunk; };
  auto block_of = [&](int key) { return (int)(__umulhi((uint32_t)key, p.page_mul) >> p.page_shift); };
  // ONE: pages of a multiple of 64 keys hold whole chunks, whose page and address
  // are scalar (one 64-bit product each: as scalar arithmetic for four groups this
  // took as long as the conversions).  Else lane q of each four finds 16-key group
  // q's, and readlane hands it to the wave.
  auto offset = [](int n, int64_t stride) { return (uint64_t)(uint32_t)n * (uint32_t)stride; };   // (strides below 2^31)
  const int lq = ONE ? 0 : tid & 3;
  int pgn;                           // page id (of group lq) of the chunk to fetch next
  struct Fetched {                   // a chunk's bytes, its page id and scales
    uint2 kb[NP], vb[NP];
    float gk, gv;
    int page;
  };
  Fetched f;
  auto page_of = [&](int u) __attribute__((always_inline)) {
    return bt[block_of(min(base_of(min(u, u_hi - 1)) + lq * kGroup, t.end - 1))];
  };
  auto fetch = [&](int u) __attribute__((always_inline)) {
    const int j = base_of(min(u, u_hi - 1));
    f.page = pgn;
    const int page = pgn >= 0 && pgn < a.num_pages ? pgn : 0;
    f.gk = kscale[offset(page, a.ks_sp)];
    f.gv = vscale[offset(page, a.vs_sp)];
    const int key = ONE ? j : min(j + lq * kGroup, t.end - 1) & ~(kGroup - 1);
    const int rw = key - block_of(key) * a.page_size;
    const uint64_t ko = offset(page, a.k_sp) + offset(rw, a.k_st), vo = offset(page, a.v_sp) + offset(rw, a.v_st);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint8_t *kp, *vp;
      if constexpr (ONE) {
        kp = kcache + ko + kpiece[i];
        vp = vcache + vo + vpiece[i];
      } else {
        const int q = D == 128 ? i : wgrp + 2 * i;                  // the piece's group: RPP is 16 or 32 rows
        kp = kcache + lane_u64(ko, q) + kpiece[0];
        vp = vcache + lane_u64(vo, q) + vpiece[0];
      }
      f.kb[i] = *reinterpret_cast<const uint2*>(kp);
      f.vb[i] = *reinterpret_cast<const uint2*>(vp);
    }
  };
  // rows at positions lo .. hi each see every key of the chunk at j
  auto seen_whole = [&](int j, int lo, int hi) __attribute__((always_inline)) {
    return j + kChunk - 1 <= lo && j + kChunk <= t.kend && (a.window == 0 || j > hi - a.window || j + kChunk <= a.sinks);
  };
  uint32_t nans = 0;                 // not 0: this thread met such a NaN
  auto stage = [&](int u, int buf) __attribute__((always_inline)) {
    const int j = base_of(u);
    const bool ok = f.page >= 0 && f.page < a.num_pages && j + lq * kGroup < t.end;
    const uint32_t oks = ONE ? (ok ? 15u : 0u) : (uint32_t)__ballot(ok) & 15u;
    const bool inside = oks == 15u && j + kChunk <= t.end &&
                        (a.window == 0 || j > t.pmin - a.window || j + kChunk <= a.sinks);
    if (per_lane(!inside)) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int key = j + srow + i * RPP;
        const bool any = (oks >> (D == 128 ? i : wgrp + 2 * i) & 1u) && key < t.end &&
                         (a.window == 0 || key > t.pmin - a.window || key < a.sinks);
        f.kb[i].x = any ? f.kb[i].x : 0u;
        f.kb[i].y = any ? f.kb[i].y : 0u;
        f.vb[i].x = any ? f.vb[i].x : 0u;
        f.vb[i].y = any ? f.vb[i].y : 0u;
      }
    }
    if constexpr (KV == kFp8E4M3FN) {
      // a NaN of a key that only some rows see is a zero in the products and is set
      // in their O after the loop
      if (per_lane(!seen_whole(j, t.pmin, t.pmax))) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const uint32_t nx = nan_bytes4(f.vb[i].x), ny = nan_bytes4(f.vb[i].y);
          nans |= nx | ny;
          f.vb[i].x = without(f.vb[i].x, nx);
          f.vb[i].y = without(f.vb[i].y, ny);
        }
      }
    }
    uint16_t* sK = reinterpret_cast<uint16_t*>(smem + buf * L::buf) + srow * KP + scol;
    uint16_t* sV = reinterpret_cast<uint16_t*>(smem + buf * L::buf + L::kBytes) + srow * VP + scol;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint2 k0 = bytes4_to<KV, T>(f.kb[i].x), k1 = bytes4_to<KV, T>(f.kb[i].y);
      *reinterpret_cast<uint4*>(sK + i * RPP * KP) = make_uint4(k0.x, k0.y, k1.x, k1.y);
      const uint2 v0 = bytes4_to<KV, __half>(f.vb[i].x), v1 = bytes4_to<KV, __half>(f.vb[i].y);
      *reinterpret_cast<uint4*>(sV + i * RPP * VP) = make_uint4(v0.x, v0.y, v1.x, v1.y);
    }
    if (tid < 4) {
      const float vs = ok ? fmaxf(f.gv, kScaleMin) : 1.f;
      reinterpret_cast<float4*>(smem + buf * L::buf + L::kBytes + L::vBytes)[tid] =
          make_float4(ok ? f.gk * p.scale_l2 : 0.f, ok ? __log2f(vs) : -INFINITY, 0x1p-12f * __builtin_amdgcn_rcpf(vs), 0.f);   // (kLift)
    }
  };

  f32x16_t o[MT];
#pragma unroll
  for (int d = 0; d < MT; ++d) o[d] = zero16();
  float m = -INFINITY, msub = 0.f, thr = -INFINITY, l = 0.f;

  if (u_lo < u_hi) {
    const int p0 = page_of(u_lo), p1 = page_of(u_lo + 1), p2 = page_of(u_lo + 2);
    pgn = p0;
    fetch(u_lo);
    stage(u_lo, 0);
    pgn = p1;
    fetch(u_lo + 1);
    pgn = p2;
  }
  settle(qf);
  __syncthreads();
  // One chunk.  The next one (in f) goes to the other buffer first, and f takes the
  // one after: the conversions fill the time of the products K Q^T, 6 of them per
  // product (after the products P V instead: 2,048 rows after 30,720 keys 410 -> 405
  // us, seven short prompts on 16-key pages 22.8 -> 21.6).  405 us are 822 TFLOP/s,
  // and orders, depths and waits of the loads no longer move it: at the clocks that
  // so many products leave, the matrix cores and the vector units are each busy for
  // half of the time.
  auto step = [&](int u, int buf) __attribute__((always_inline)) {
    const uint16_t* sK = reinterpret_cast<const uint16_t*>(smem + buf * L::buf);
    const uint16_t* sV = reinterpret_cast<const uint16_t*>(smem + buf * L::buf + L::kBytes);
    const float4* sg = reinterpret_cast<const float4*>(smem + buf * L::buf + L::kBytes + L::vBytes);
    const int j0 = base_of(u);
    stage(min(u + 1, u_hi - 1), buf ^ 1);
    fetch(u + 2);
    pgn = page_of(u + 3);
    float4 gs[4];                                 // (ONE: four times the same)
#pragma unroll
    for (int q = 0; q < 4; ++q) gs[q] = sg[ONE ? 0 : q];
    // (a group without a page has K zero and an exponent of -inf, and needs no mask)
    const bool whole = seen_whole(j0, wpmin, wpmax);
    f32x16_t s[2];
    // K's operands, kAhead of them in flight
    constexpr int kAhead = 4;
    uint4 kf[kAhead];
    auto k_operand = [&](int i) {
      return *reinterpret_cast<const uint4*>(sK + (32 * (i / KS) + rl) * KP + 16 * (i % KS) + 8 * hh);
    };
#pragma unroll
    for (int f = 0; f < kAhead; ++f) kf[f] = k_operand(f);
    s[0] = s[1] = zero16();
#pragma unroll
    for (int f = 0; f < 2 * KS; ++f) {
      s[f / KS] = Mfma<T>::mac(kf[f % kAhead], qf[f % KS], s[f / KS]);
      if (f + kAhead < 2 * KS) kf[f % kAhead] = k_operand(f + kAhead);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead + (ONE ? 1 : 4), 0);
#pragma unroll
    for (int f = 0; f < 2 * KS; ++f) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (f < 2 * KS - kAhead) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float b = gs[q].y - msub;
#pragma unroll
      for (int j = 0; j < 8; ++j) s[q / 2][8 * (q % 2) + j] = fmaf(s[q / 2][8 * (q % 2) + j], gs[q].x, b);
    }
    if (per_lane(!whole)) {
      const int from = j0 + 4 * hh - my_lo;       // the lane's first key, from its row's window on
      if (per_lane(j0 >= a.sinks)) {              // one range: windowed prefill 51.8 -> 51.1 us
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            s[kt][x] = (uint32_t)(from + 32 * kt + 8 * (x / 4) + x % 4) < my_span ? s[kt][x] : -INFINITY;
      } else {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int k = from + 32 * kt + 8 * (x / 4) + x % 4;
            s[kt][x] = (((uint32_t)k < my_span) | ((uint32_t)(k + my_lo) < my_first)) ? s[kt][x] : -INFINITY;
          }
      }
    }
    float zm = s[0][0];
#pragma unroll
    for (int x = 1; x < 16; ++x) zm = fmaxf(zm, s[0][x]);
#pragma unroll
    for (int x = 0; x < 16; ++x) zm = fmaxf(zm, s[1][x]);
    uint4 vf[MT];
#pragma unroll
    for (int d = 0; d < MT; ++d) vf[d] = a_operand_tr<VP>(sV, 0, 32 * d, lane);
    if (per_lane(__any(zm > thr))) {
      const float mn = fmaxf(m, xor32_max(zm) + msub - kBelow);
      const float alpha = mn == -INFINITY ? 1.f : exp2f(m - mn);
      const float now = mn == -INFINITY ? 0.f : mn, by = msub - now;
      m = mn;
      msub = now;
      thr = mn == -INFINITY ? -INFINITY : kBelow + kSlack;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < MT; ++d)
#pragma unroll
        for (int x = 0; x < 16; ++x) o[d][x] *= alpha;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int x = 0; x < 16; ++x) s[kt][x] += by;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float pe[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) pe[j] = __builtin_amdgcn_exp2f(s[g / 2][8 * (g % 2) + j]);
      const uint4 pf = make_uint4(pack_f16(pe[0], pe[1]), pack_f16(pe[2], pe[3]), pack_f16(pe[4], pe[5]),
                                  pack_f16(pe[6], pe[7]));
      l = fmaf(((pe[0] + pe[1]) + (pe[2] + pe[3])) + ((pe[4] + pe[5]) + (pe[6] + pe[7])), gs[g].z, l);
#pragma unroll
      for (int d = 0; d < MT; ++d) {
        o[d] = Mfma<__half>::mac(vf[d], pf, o[d]);
        if (g < 3) vf[d] = a_operand_tr<VP>(sV, 16 * g + 16, 32 * d, lane);
      }
    }
    __syncthreads();
  };
  for (int u = u_lo; u < u_hi; u += 2) {
    step(u, 0);
    if (u + 1 < u_hi) step(u + 1, 1);
  }

  if constexpr (KV == kFp8E4M3FN) {
    int* met = reinterpret_cast<int*>(smem);               // (the last step's barrier is behind)
    const bool any = __any(nans != 0u);
    if (lane == 0) met[wave] = any;
    __syncthreads();
    if (met[0] | met[1] | met[2] | met[3]) {
      for (int u = u_lo; u < u_hi; ++u) {
        const int j = base_of(u);
        if (seen_whole(j, t.pmin, t.pmax)) continue;
        for (int k = j; k < min(j + kChunk, t.end); ++k) {
          const int page = a.block_table[(int64_t)r * a.bt_sr + block_of(k)];
          if (page < 0 || page >= a.num_pages) continue;
          const bool see = ((uint32_t)(k - my_lo) < my_span) | ((uint32_t)k < my_first);
          const uint8_t* vp = vcache + offset(page, a.v_sp) + offset(k - block_of(k) * a.page_size, a.v_st) + 4 * hh;
#pragma unroll
          for (int d = 0; d < MT; ++d)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const uint32_t n = see ? nan_bytes4(*reinterpret_cast<const uint32_t*>(vp + 32 * d + 8 * x)) : 0u;
#pragma unroll
              for (int e = 0; e < 4; ++e) o[d][4 * x + e] = (n >> (8 * e + 7)) & 1u ? NAN : o[d][4 * x + e];
            }
        }
      }
    }
  }
  l = xor32_sum(l);
  if (!wave_live) return;
  if (p.nsplit > 1 && parts > 1) {
    // record: lane-major float4s, then the rows' (m, l)
    float* rec = p.part + (((int64_t)nth * a.HKV + h) * p.nsplit + part) * kRowsWg * (D + 2);
#pragma unroll
    for (int d = 0; d < MT; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        *reinterpret_cast<float4*>(rec + ((d * 4 + x) * kThreads + tid) * 4) =
            make_float4(o[d][4 * x], o[d][4 * x + 1], o[d][4 * x + 2], o[d][4 * x + 3]);
    if (hh == 0) {
      rec[kRowsWg * D + 2 * wrow] = m;
      rec[kRowsWg * D + 2 * wrow + 1] = l;
    }
    return;
  }
  if (wrow >= t.nrows) return;
  const float inv = inv_sum(m, l);
  T* op = reinterpret_cast<T*>(a.out) + (int64_t)(t.q0 + tok) * a.o_sn + (int64_t)hq * a.o_sh + 4 * hh;
#pragma unroll
  for (int d = 0; d < MT; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<uint2*>(op + 32 * d + 8 * x) =
          make_uint2(Mfma<T>::pack2(o[d][4 * x] * inv, o[d][4 * x + 1] * inv),
                     Mfma<T>::pack2(o[d][4 * x + 2] * inv, o[d][4 * x + 3] * inv));
  if (a.lse && hh == 0)
    a.lse[(int64_t)(t.q0 + tok) * a.lse_sn + (int64_t)hq * a.lse_sh] = lse_of(m, l);
}

// Joins the parts of a tile, lane by lane as they were written: one workgroup per
// 32 rows, D / 32 x 64 threads of 16 dims each.
template <typename T, int D>
__global__ __launch_bounds__(2 * D) void cache8_join_kernel(PrefillK p) {
  const srswa_cache8_attend_args& a = p.a;
  const int wave = (int)blockIdx.x % 4, rt = (int)blockIdx.x / 4;     // the wave that wrote the rows
  const int h = rt % a.HKV;
  int r, tile;
  if (!nth_tile(p, rt / a.HKV, (int)threadIdx.x % kWave, &r, &tile)) return;
  const Tile t = tile_of(p, r, tile);
  const int parts = parts_of(p, t);
  if (wave * 32 >= t.nrows || parts == 1) return;
  const int lane = threadIdx.x % kWave, d = threadIdx.x / kWave, wrow = wave * 32 + (lane & 31), hh = lane >> 5;
  constexpr int64_t rsz = kRowsWg * (D + 2);
  const float* rec = p.part + (int64_t)rt * p.nsplit * rsz;
  const float* ml = rec + kRowsWg * D + 2 * wrow;
  float M = -INFINITY, l = 0.f;
  for (int k = 0; k < parts; ++k) M = fmaxf(M, ml[k * rsz]);
  float4 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int k = 0; k < parts; ++k) {
    const float mk = ml[k * rsz];
    const float f = mk == -INFINITY ? 0.f : exp2f(mk - M);
    l = fmaf(f, ml[k * rsz + 1], l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(rec + k * rsz + ((d * 4 + i) * kThreads + wave * kWave + lane) * 4);
      o[i].x = fmaf(f, x.x, o[i].x); o[i].y = fmaf(f, x.y, o[i].y);
      o[i].z = fmaf(f, x.z, o[i].z); o[i].w = fmaf(f, x.w, o[i].w);
    }
  }
  if (wrow >= t.nrows) return;
  const int row = t.row0 + wrow, tok = row / p.G, hq = h * p.G + row % p.G;
  const float inv = inv_sum(M, l);
  T* op = reinterpret_cast<T*>(a.out) + (int64_t)(t.q0 + tok) * a.o_sn + (int64_t)hq * a.o_sh + 32 * d + 4 * hh;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<uint2*>(op + 8 * i) = make_uint2(Mfma<T>::pack2(o[i].x * inv, o[i].y * inv),
                                                       Mfma<T>::pack2(o[i].z * inv, o[i].w * inv));
  if (a.lse && hh == 0 && d == 0)
    a.lse[(int64_t)(t.q0 + tok) * a.lse_sn + (int64_t)hq * a.lse_sh] = lse_of(M, l);
}

// Parts: the fewest that need the least rounds of the GPU per part, where two
// workgroups share a CU and a (request, head, part)'s tiles an XCD; four chunks of a
// full table are one part's least (eight requests of 128 rows after up to 2,000 keys
// 47 us with eight, 35 with four, 36 with two; of 512 rows alone 31, 31, 53).
PrefillK plan(const srswa_cache8_attend_args* a) {
  PrefillK p{};
  p.a = *a;
  p.G = a->HQ / a->HKV;
  p.scale_l2 = a->scale * kLog2e;
  // as many tiles as the rows can make: the longest request may be shorter than its bound
  p.tiles = (int)std::min<int64_t>((int64_t)a->R * (((int64_t)a->max_query_len * p.G + kRowsWg - 1) / kRowsWg),
                                   (int64_t)a->total_q * p.G / kRowsWg + a->R);
  int lg = 0;
  while ((1 << lg) < a->page_size) ++lg;
  p.page_shift = lg - 1;
  p.page_mul = (uint32_t)(((1ull << (31 + lg)) / a->page_size) + 1);
  int64_t keys = (int64_t)a->max_blocks * a->page_size;
  if (a->window > 0) keys = std::min<int64_t>(keys, (int64_t)a->window + kRowsWg / p.G + 2 * kChunk + a->sinks);
  p.chunks = (keys + kChunk - 1) / kChunk;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(16, keys / kChunk / kMinChunks));
  int cus = device_cu_count();
  if (cus <= 0) cus = 256;
  // rounds of the GPU per part, tiles dealt in turn (half a tile per request is a
  // remainder) or one request's by XCD, and the parts that need the least
  const int64_t in_turn = std::max<int64_t>(1, ((int64_t)a->total_q * p.G / kRowsWg + a->R / 2) * a->HKV);
  double least[2] = {1e30, 1e30};
  int parts[2] = {1, 1};
  for (int g = 0; g < (a->R == 1 ? 2 : 1); ++g)
    for (int n = 1; n <= most; ++n) {
      const int64_t wgs = g ? ((int64_t)a->HKV * n + kXcds - 1) / kXcds * p.tiles : in_turn * n;
      const int64_t slots = g ? std::max(1, cus / kXcds * 2) : 2 * cus;
      const double cost = (double)((wgs + slots - 1) / slots) / n;
      if (cost < least[g] * 0.95) {
        least[g] = cost;
        parts[g] = n;
      }
    }
  p.by_group = least[1] <= least[0] * 1.02;
  p.nsplit = parts[p.by_group];
  return p;
}

size_t ws_bytes_of(const PrefillK& p) {
  return p.nsplit > 1 ? (size_t)p.tiles * p.a.HKV * p.nsplit * kRowsWg * (p.a.D + 2) * sizeof(float) : 0;
}

// Whether decode's form of 16-row items is the faster: a 128-row tile converts each key
// once for eight times the rows, but fills fewer CUs and takes longer to start and end.
// Both are estimated in us from what 24 shapes measured (their keys are the table's
// width here, a call's may be fewer, so near ties go to the items): items 14 shared out
// or 8 whole, and 0.85 per unit of a place (three a CU) or 0.19 of the longest; tiles 10,
// 20 with a join, and per chunk of a part 1.35 alone on a CU, 2.4 beside another.  One
// request of ten heads, items against tiles: 33 against 62 us (16 rows after 30,000
// keys), 64 against 64 (64 rows), 105 against 65 (128 rows), 47 against 34 (128 rows
// after 8,000), 22 against 28 (256 after 2,000), 11 against 21 (512, no prefix); eight:
// 25 against 29 (64 after 2,000), 22 against 16 (256, no prefix); sixteen of 16 rows
// after 30,000 keys 152 against 264.
// SRSWA_CACHE8_PREFILL = items or tiles takes that form for any call.
bool narrow(const srswa_cache8_attend_args* a, const PrefillK& p) {
  if (const char* form = std::getenv("SRSWA_CACHE8_PREFILL")) {
    if (std::strcmp(form, "items") == 0) return true;
    if (std::strcmp(form, "tiles") == 0) return false;
  }
  int64_t wgs, units;
  bool shared;
  cache8_decode_load(a, &wgs, &units, &shared);
  int cus = device_cu_count();
  if (cus <= 0) cus = 256;
  const double by_d = a->D == 128 ? 1.0 : 0.7;
  const double load = 0.85 * (double)wgs * (double)units / (3 * cus);
  const double items = shared ? 14 + by_d * load : 8 + by_d * std::max(0.19 * (double)units, load);
  const int64_t parts = (int64_t)p.tiles * a->HKV * p.nsplit, rounds = (parts + 2 * cus - 1) / (2 * cus);
  const double tiles = (p.nsplit > 1 ? 20 : 10) +
                       by_d * (parts <= cus ? 1.35 : 2.4 * (double)rounds) * (double)((p.chunks + p.nsplit - 1) / p.nsplit);
  return items <= 1.1 * tiles;
}

template <typename T, int KV, int D, bool ONE>
int launch_tiles(const PrefillK& p, unsigned grid, hipStream_t st) {
  static LdsGrant grant;
  if (!ensure_dynamic_lds(cache8_prefill_kernel<T, KV, D, ONE>, Lds<D>::total, &grant)) return SRSWA_LAUNCH;
  cache8_prefill_kernel<T, KV, D, ONE><<<grid, kThreads, Lds<D>::total, st>>>(p);
  return SRSWA_OK;
}
template <typename T, int KV, int D>
int launch(const PrefillK& p, unsigned grid, hipStream_t st) {
  const bool one = p.a.page_size % kChunk == 0 && std::max(p.a.k_st, p.a.v_st) <= INT32_MAX / kChunk;
  const int rc = one ? launch_tiles<T, KV, D, true>(p, grid, st)
                     : launch_tiles<T, KV, D, false>(p, grid, st);
  if (rc != SRSWA_OK) return rc;
  if (p.nsplit > 1)
    cache8_join_kernel<T, D><<<(unsigned)(p.a.HKV * p.tiles * 4), 2 * D, 0, st>>>(p);
  return SRSWA_OK;
}
template <typename T, int KV>
int launch_d(const PrefillK& p, unsigned grid, hipStream_t st) {
  return p.a.D == 64 ? launch<T, KV, 64>(p, grid, st) : launch<T, KV, 128>(p, grid, st);
}
template <typename T>
int launch_kv(const PrefillK& p, unsigned grid, hipStream_t st) {
  return p.a.kv_dtype == SRSWA_I8 ? launch_d<T, kI8>(p, grid, st) : launch_d<T, kFp8E4M3FN>(p, grid, st);
}

}  // namespace
}  // namespace srswa

using namespace srswa;

extern "C" size_t srswa_cache8_prefill_workspace(const srswa_cache8_attend_args* a) {
  if (!cache8_plannable(a)) return 0;
  const PrefillK p = plan(a);
  return narrow(a, p) ? cache8_decode_ws(a) : ws_bytes_of(p);
}

extern "C" int srswa_cache8_prefill(const srswa_cache8_attend_args* a, void* ws, size_t ws_bytes, void* stream) {
  const char* what = "cache8 prefill";
  const int rc = cache8_check(a, what);
  if (rc != SRSWA_OK) return rc;
  if (a->topk) {
    set_error("%s: selected blocks are for decode", what);
    return SRSWA_UNSUPPORTED;
  }
  if (!cache8_plannable(a) || a->total_q == 0) return SRSWA_OK;
  if (!a->cu_seqlens_q) {
    set_error("%s: cu_seqlens_q is null", what);
    return SRSWA_INVALID;
  }
  PrefillK p = plan(a);
  if (narrow(a, p)) return cache8_decode_run(a, ws, ws_bytes, stream, what);
  const size_t need = ws_bytes_of(p);
  if (need > 0 && (!ws || ws_bytes < need)) {
    set_error("%s: workspace of %zu bytes required (got %zu)", what, need, ws_bytes);
    return SRSWA_WORKSPACE;
  }
  p.part = reinterpret_cast<float*>(ws);
  const int64_t parts = (int64_t)a->HKV * p.nsplit;
  const int64_t grid = (p.by_group ? (parts + kXcds - 1) / kXcds * kXcds : parts) * p.tiles;
  if (grid > 0x7fffffff || (int64_t)a->HKV * p.tiles * 4 > 0x7fffffff) {
    set_error("%s: grid too large", what);
    return SRSWA_UNSUPPORTED;
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int ok = a->dtype == SRSWA_BF16 ? launch_kv<bf16_t>(p, (unsigned)grid, st) : launch_kv<__half>(p, (unsigned)grid, st);
  return ok == SRSWA_OK ? cache8_launched(what) : ok;
}
