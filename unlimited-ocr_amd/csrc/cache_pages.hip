// Pages of a pool (gfx950): dealing them out, reordering rows (sharing, copying
// and freeing pages) and compacting, over block_table [R, W], seq_lens [R] and
// ref [num_pages] (rows that hold a page, 0 = free).
//
// Every step reads the old state and writes the new one, and free pages are
// found by rank (the k-th free page in ascending order, from counts per tile of
// kTile pages), so no result depends on the order of execution; the only atomics
// are integer additions into ref.
#include <algorithm>

#include "common.h"

namespace srswa {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 2048;       // pages per tile of the free-page counts
constexpr int kMaxCaches = 64;    // caches per copy launch (the table is a kernel argument)

struct PagesK {
  const int32_t* bt;   int64_t bt_sr;
  const int32_t* sl;
  const int32_t* ref;
  const int32_t* rows;
  int32_t* bto;        int64_t bto_sr;
  int32_t* slo;
  int32_t* refo;
  int32_t* count;
  int R, W, N, page_size, ntiles;
  // workspace
  int32_t* need;       // [R]       pages a row asks for
  int32_t* src;        // [R | N]   reorder: the page row r copies; compact: pair i's source
  int32_t* dst;        // [R | N]   its destination (-1: none)
  int32_t* tfree;      // [ntiles]  free (compact: held) pages per tile
  int32_t* npairs;     // [1]
  uint32_t* bits;      // [ceil(N / 32)] free pages
};

// sum over the workgroup of one value per thread, on every thread
__device__ __forceinline__ int block_sum(int v, int* s) {
  v = wave_sum_int(v);
  __syncthreads();
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  int t = 0;
  for (int w = 0; w < (int)blockDim.x / kWave; ++w) t += s[w];
  return t;
}

// exclusive prefix of one value per thread over the workgroup, and the total
__device__ __forceinline__ int block_scan(int v, int* s, int* total) {
  int incl = v;
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int x = __shfl_up(incl, o, kWave);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == kWave - 1) s[w] = incl;
  __syncthreads();
  int base = 0, t = 0;
  for (int i = 0; i < (int)blockDim.x / kWave; ++i) {
    base += i < w ? s[i] : 0;
    t += s[i];
  }
  *total = t;
  return base + incl - v;
}

__device__ __forceinline__ bool valid_page(const PagesK& p, int id) { return id >= 0 && id < p.N; }

// Marks and counts the free pages of one tile of ref.
__device__ __forceinline__ void mark_tile(const PagesK& p, const int32_t* ref, int tile, int* s) {
  int n = 0;
  for (int i = threadIdx.x; i < kTile; i += (int)blockDim.x) {
    const int page = tile * kTile + i;
    const bool fr = page < p.N && ref[page] == 0;
    const uint64_t b = __ballot(fr);
    if (threadIdx.x % 32 == 0 && page < p.N) p.bits[page / 32] = (uint32_t)(threadIdx.x % kWave ? b >> 32 : b);
    n += fr;
  }
  n = block_sum(n, s);
  if (threadIdx.x == 0) p.tfree[tile] = n;
}

// The free pages of ranks [k0, k0 + n): put(k, page) for each that exists.  The
// tiles that hold them are found from the tile counts (c0: tile threadIdx.x's); a
// wave then takes a tile, a
// lane each of its 64 words.  Every thread of the workgroup calls it.
struct Hit {
  int tile, before;
};
template <typename Put>
__device__ __forceinline__ void find_free(const PagesK& p, int k0, int n, int c0, int* s, Hit* s_hit, int* s_nhit,
                                          Put put) {
  static_assert(kTile == 32 * kWave, "a lane per word of a tile");
  int before = 0;
  for (int t0 = 0; t0 < p.ntiles && before < k0 + n; t0 += (int)blockDim.x) {
    if (threadIdx.x == 0) *s_nhit = 0;
    const int t = t0 + threadIdx.x;
    const int c = t0 == 0 ? c0 : t < p.ntiles ? p.tfree[t] : 0;
    int total;
    const int b = before + block_scan(c, s, &total);
    if (c > 0 && b < k0 + n && b + c > k0) s_hit[atomicAdd(s_nhit, 1)] = Hit{t, b};   // (any order)
    __syncthreads();
    const int hits = *s_nhit, lane = threadIdx.x % kWave;
    for (int i = threadIdx.x / kWave; i < hits; i += (int)blockDim.x / kWave) {
      const int w = s_hit[i].tile * kWave + lane;
      uint32_t x = w < (p.N + 31) / 32 ? p.bits[w] : 0u;
      const int m = __popc(x);
      int incl = m;
#pragma unroll
      for (int o = 1; o < kWave; o <<= 1) {
        const int v = __shfl_up(incl, o, kWave);
        if (lane >= o) incl += v;
      }
      int k = s_hit[i].before + incl - m;
      if (k + m > k0 && k < k0 + n)
        while (x) {
          const int bit = __ffs((int)x) - 1;
          x &= x - 1;
          if (k >= k0 && k < k0 + n) put(k, w * 32 + bit);
          ++k;
        }
    }
    __syncthreads();
    before += total;
  }
}

// ---------------------------------------------------------------- reserve
// rows: the new lengths.  First launch: a workgroup per row copies it and counts
// what it misses, a workgroup per tile copies ref and counts its free pages.
__global__ __launch_bounds__(kThreads) void reserve_count_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  if ((int)blockIdx.x < p.R) {
    const int r = (int)blockIdx.x;
    const int len = p.rows[r];
    const int nb = (int)min((int64_t)p.W, ((int64_t)max(len, 0) + p.page_size - 1) / p.page_size);
    int n = 0;
    for (int b = threadIdx.x; b < p.W; b += kThreads) {
      const int id = p.bt[(int64_t)r * p.bt_sr + b];
      p.bto[(int64_t)r * p.bto_sr + b] = id;
      n += b < nb && id < 0;
    }
    n = block_sum(n, s);
    if (threadIdx.x == 0) {
      p.need[r] = n;
      p.slo[r] = len;
    }
  } else {
    const int tile = (int)blockIdx.x - p.R;
    for (int i = threadIdx.x; i < kTile; i += kThreads)
      if (tile * kTile + i < p.N) p.refo[tile * kTile + i] = p.ref[tile * kTile + i];
    mark_tile(p, p.ref, tile, s);
  }
}

// Second launch: each row that misses pages takes the free pages of its ranks.  What
// the first thread-width of rows, tiles and entries needs is loaded at once, before
// any of it is used.
__global__ __launch_bounds__(kThreads) void reserve_deal_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  __shared__ int s_blk[kThreads];
  __shared__ Hit s_hit[kThreads];
  __shared__ int s_nhit;
  const int r = (int)blockIdx.x, tid = threadIdx.x;
  const bool last = r == p.R - 1;
  const int need = p.need[r], len = p.rows[r];
  const int n0 = tid < p.R ? p.need[tid] : 0;
  const int c0 = tid < p.ntiles ? p.tfree[tid] : 0;
  const int e0 = p.bt[(int64_t)r * p.bt_sr + min(tid, p.W - 1)];
  if (need == 0 && !last) return;
  int before = tid < r ? n0 : 0, all = n0, fr = c0;
  for (int i = tid + kThreads; i < p.R; i += kThreads) {
    const int n = p.need[i];
    before += i < r ? n : 0;
    all += n;
  }
  before = block_sum(before, s);
  if (last) {
    all = block_sum(all, s);
    for (int i = tid + kThreads; i < p.ntiles; i += kThreads) fr += p.tfree[i];
    fr = block_sum(fr, s);
    if (tid == 0) *p.count = max(all - fr, 0);
    if (need == 0) return;
  }
  // the row's missing entries in order: entry of rank k takes the free page of rank before + k
  const int nb = (int)min((int64_t)p.W, ((int64_t)max(len, 0) + p.page_size - 1) / p.page_size);
  int done = 0;
  for (int b0 = 0; b0 < nb && done < need; b0 += kThreads) {
    const int b = b0 + tid;
    const bool miss = b < nb && (b0 == 0 ? e0 : p.bt[(int64_t)r * p.bt_sr + b]) < 0;
    int got;
    const int k = block_scan(miss ? 1 : 0, s, &got);
    if (miss) s_blk[k] = b;
    __syncthreads();
    if (got > 0)
      find_free(p, before + done, got, c0, s, s_hit, &s_nhit, [&](int rank, int page) {
        p.bto[(int64_t)r * p.bto_sr + s_blk[rank - before - done]] = page;
        p.refo[page] = 1;
      });
    __syncthreads();
    done += got;
  }
}

// ---------------------------------------------------------------- reorder
__global__ __launch_bounds__(kThreads) void copy_ref_kernel(PagesK p) {
  const int i = (int)blockIdx.x * kThreads + threadIdx.x;
  if (i < p.N) p.refo[i] = p.ref[i];
}

// rows: the parents.  `threads` threads write row r's new entries, move the
// references from its old pages to its new ones; returns the page it must copy (-1:
// none) to the first of them.
__device__ __forceinline__ int reorder_row(const PagesK& p, int r, int par, int len, int me, int threads, bool first) {
  const bool alive = par >= 0 && par < p.R;
  const int full = max(len, 0) / p.page_size;
  const int begun = max(len, 0) % p.page_size;
  const int32_t* mine = p.bt + (int64_t)r * p.bt_sr;
  const int32_t* theirs = p.bt + (int64_t)(alive ? par : r) * p.bt_sr;
  int src = -1;                                   // (its load is in flight beside the first entries')
  if (me == 0 && alive && !first && begun > 0 && full < p.W) src = theirs[full];
  for (int b0 = me; b0 < p.W; b0 += 8 * threads) {
    int old[8], id[8];                            // (loaded together, before any addition)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int b = min(b0 + k * threads, p.W - 1);
      old[k] = mine[b];
      id[k] = theirs[b];
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int b = b0 + k * threads;
      if (b >= p.W) break;
      const int now = alive && (first || b < full) ? id[k] : -1;
      p.bto[(int64_t)r * p.bto_sr + b] = now;
      if (old[k] != now) {
        if (valid_page(p, old[k])) atomicSub(&p.refo[old[k]], 1);
        if (valid_page(p, now)) atomicAdd(&p.refo[now], 1);
      }
    }
  }
  if (me == 0) p.slo[r] = len;
  return valid_page(p, src) ? src : -1;
}

// Deals free pages to the rows that copy, in row order (one workgroup).
__device__ __forceinline__ void reorder_deal(const PagesK& p, int* s, int* s_row, Hit* s_hit, int* s_nhit) {
  int fr = 0;
  for (int i = threadIdx.x; i < p.ntiles; i += (int)blockDim.x) fr += p.tfree[i];
  fr = block_sum(fr, s);
  int done = 0;
  for (int r0 = 0; r0 < p.R; r0 += (int)blockDim.x) {
    const int r = r0 + threadIdx.x;
    const bool want = r < p.R && p.src[r] >= 0;
    int n;
    const int k = block_scan(want ? 1 : 0, s, &n);
    if (want) s_row[k] = r;
    if (r < p.R) p.dst[r] = -1;
    __syncthreads();
    if (n > 0)
      find_free(p, done, n, (int)threadIdx.x < p.ntiles ? p.tfree[threadIdx.x] : 0, s, s_hit, s_nhit, [&](int rank, int page) {
        const int row = s_row[rank - done];
        p.dst[row] = page;
        p.bto[(int64_t)row * p.bto_sr + p.slo[row] / p.page_size] = page;
        p.refo[page] = 1;
      });
    __syncthreads();
    done += n;
  }
  if (threadIdx.x == 0) {
    *p.count = max(done - fr, 0);
    *p.npairs = p.R;
  }
}

__global__ __launch_bounds__(kThreads) void reorder_rows_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  const int r = (int)blockIdx.x, par = p.rows[r];
  const bool alive = par >= 0 && par < p.R;
  int older = 0;                                  // rows before this one that continue the same parent
  for (int i = threadIdx.x; alive && i < r; i += kThreads) older += p.rows[i] == par;
  older = block_sum(older, s);
  const int src = reorder_row(p, r, par, alive ? p.sl[par] : 0, threadIdx.x, kThreads, older == 0);
  if (threadIdx.x == 0) p.src[r] = src;
}

__global__ __launch_bounds__(kThreads) void mark_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  mark_tile(p, p.refo, (int)blockIdx.x, s);
}

__global__ __launch_bounds__(kThreads) void reorder_deal_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  __shared__ int s_row[kThreads];
  __shared__ Hit s_hit[kThreads];
  __shared__ int s_nhit;
  reorder_deal(p, s, s_row, s_hit, &s_nhit);
}

// The four steps in one workgroup, the marks and the list of free pages in LDS: a power
// of two of threads per row, every row at once where they suffice.  Against the four
// launches, one layer's copies included: 4 rows of 128 pages 9.5 us (17.6), 64 rows 16.5
// (23.1), 128 rows 29.6 (29.3), 256 rows 54 (32); 8 rows of a pool of 32,000 pages 23.5
// (18.6).
constexpr int kWide = 1024;
constexpr int kPlanRows = 128, kPlanEntries = 16384, kPlanPages = 16384;
static_assert(kPlanRows <= kWide && kPlanPages <= 32 * kWide, "a thread per row, a bit per page");
__global__ __launch_bounds__(kWide) void reorder_plan_kernel(PagesK p) {
  __shared__ int s[kWide / kWave];
  __shared__ int s_par[kWide], s_len[kWide], s_src[kWide], s_free[kWide];
  __shared__ uint32_t s_bits[kWide];
  const int tid = threadIdx.x;
  s_bits[tid] = 0u;
  if (tid < p.R) {
    const int par = p.rows[tid];
    s_par[tid] = par;
    s_len[tid] = par >= 0 && par < p.R ? p.sl[par] : 0;
  }
  for (int i = tid; i < p.N; i += kWide) p.refo[i] = p.ref[i];
  __syncthreads();
  int per = kWave;                                // threads per row
  while (per > 1 && per * p.R > kWide) per >>= 1;
  const int me = tid & (per - 1);
  for (int r = tid / per; r < p.R; r += kWide / per) {
    const int par = s_par[r];
    int older = 0;
    for (int i = me; i < r; i += per) older += s_par[i] == par;
    for (int o = 1; o < per; o <<= 1) older += __shfl_xor(older, o, kWave);
    const int src = reorder_row(p, r, par, s_len[r], me, per, older == 0);
    if (me == 0) {
      s_src[r] = src;
      p.src[r] = src;
    }
  }
  __syncthreads();                                // (orders this workgroup's global accesses too)
  for (int i0 = 0; i0 < p.N; i0 += kWide) {
    // the additions went past this CU's cache: so does the load
    const int i = i0 + tid;
    const bool fr = i < p.N && __hip_atomic_load(p.refo + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == 0;
    const uint64_t b = __ballot(fr);
    if (tid % 32 == 0) s_bits[i / 32] = (uint32_t)(tid % kWave ? b >> 32 : b);
  }
  __syncthreads();
  // the rank of a row that copies among them, and the free page of that rank
  int wants, nfree;
  const bool want = tid < p.R && s_src[tid] >= 0;
  const int rank = block_scan(want ? 1 : 0, s, &wants);
  uint32_t x = s_bits[tid];
  int k = block_scan(__popc(x), s, &nfree);
  while (x && k < wants) {
    const int bit = __ffs((int)x) - 1;
    x &= x - 1;
    s_free[k++] = tid * 32 + bit;
  }
  __syncthreads();
  if (tid < p.R) {
    const int page = want && rank < nfree ? s_free[rank] : -1;
    p.dst[tid] = page;
    if (page >= 0) {
      p.bto[(int64_t)tid * p.bto_sr + s_len[tid] / p.page_size] = page;
      p.refo[page] = 1;
    }
  }
  if (tid == 0) {
    *p.count = max(wants - nfree, 0);
    *p.npairs = p.R;
  }
}

// ---------------------------------------------------------------- compact
__global__ __launch_bounds__(kThreads) void held_count_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  int n = 0;
  for (int i = threadIdx.x; i < kTile; i += kThreads) {
    const int page = (int)blockIdx.x * kTile + i;
    n += page < p.N && p.ref[page] > 0;
  }
  n = block_sum(n, s);
  if (threadIdx.x == 0) p.tfree[blockIdx.x] = n;
}

// With n pages held, hole number i (the i-th free page below n) takes mover
// number i (the i-th held page at or past n); there are n - held(< n) of each.
// Page x is hole x - held(< x) or mover held(< x) - held(< n).
__global__ __launch_bounds__(kThreads) void compact_plan_kernel(PagesK p) {
  __shared__ int s[kThreads / kWave];
  const int tile = (int)blockIdx.x;
  int all = 0, before = 0;
  for (int i = threadIdx.x; i < p.ntiles; i += kThreads) {
    const int c = p.tfree[i];
    all += c;
    before += i < tile ? c : 0;
  }
  const int n = block_sum(all, s);
  before = block_sum(before, s);
  // held(< n), for the ranks of this tile's movers
  int below = 0;
  if ((tile + 1) * kTile >= n) {
    const int nt = n / kTile;
    for (int i = threadIdx.x; i < nt; i += kThreads) below += p.tfree[i];
    for (int i = nt * kTile + threadIdx.x; i < n; i += kThreads) below += p.ref[i] > 0;
    below = block_sum(below, s);
  }
  for (int i0 = 0; i0 < kTile; i0 += kThreads) {
    const int x = tile * kTile + i0 + threadIdx.x;
    const bool held = x < p.N && p.ref[x] > 0;
    int got;
    const int hb = before + block_scan(held ? 1 : 0, s, &got);   // held pages below x
    if (x < n && !held) p.dst[x - hb] = x;
    if (x < p.N && x >= n && held) {
      p.src[hb - below] = x;
      p.need[x] = hb - below;
    }
    before += got;
  }
  if (tile == p.ntiles - 1 && threadIdx.x == 0) {
    *p.count = n;
    *p.npairs = n - below;
  }
}

// The table follows and the references move (the last workgroups).
__global__ __launch_bounds__(kThreads) void compact_table_kernel(PagesK p, int row_groups) {
  const int n = *p.count;
  if ((int)blockIdx.x < row_groups) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < (int64_t)p.R * p.W) {
      const int r = (int)(i / p.W), b = (int)(i % p.W);
      const int id = p.bt[(int64_t)r * p.bt_sr + b];
      const bool moves = id >= n && id < p.N && p.ref[id] > 0;
      p.bto[(int64_t)r * p.bto_sr + b] = moves ? p.dst[p.need[id]] : id;
    }
    if (i < p.R) p.slo[i] = p.sl[i];
  } else {
    const int x = ((int)blockIdx.x - row_groups) * kThreads + threadIdx.x;
    if (x < p.N) {
      const int v = p.ref[x];
      if (x < n) {
        if (v > 0) p.refo[x] = v;
      } else {
        p.refo[x] = v > 0 ? 0 : v;
        if (v > 0) p.refo[p.dst[p.need[x]]] = v;
      }
    }
  }
}

// ---------------------------------------------------------------- copy
struct CopyK {
  srswa_page_cache c[kMaxCaches];
  int n, big;                   // caches; the first `big` are cut into slices of kSlice bytes
  int slices;                   // of the largest
  const int32_t* src;
  const int32_t* dst;
  const int32_t* npairs;
  int N;
};

constexpr int kSlice = kThreads * 4 * 16;

// Workgroups take (pair, cache, slice) items of the big caches in turn, four
// 16-byte loads a thread in flight, then pairs whose small caches a wave each
// copies.  A pair whose destination is -1 copies nothing.  No destination is a
// source (a source is held, a destination was free), so the order does not matter.
__global__ __launch_bounds__(kThreads) void copy_pages_kernel(CopyK p) {
  const int np = *p.npairs;
  auto pair = [&](int i, int* s, int* d) {
    *s = p.src[i];
    *d = p.dst[i];
    return *s >= 0 && *s < p.N && *d >= 0 && *d < p.N;
  };
  const int64_t items = (int64_t)np * p.big * p.slices;
  int s, d;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int sl = (int)(it % p.slices);
    const int64_t ic = it / p.slices;
    const srswa_page_cache c = p.c[ic % p.big];
    if (!pair((int)(ic / p.big), &s, &d) || (int64_t)sl * kSlice >= c.bytes) continue;
    const int n = (int)min((int64_t)kSlice, c.bytes - (int64_t)sl * kSlice) / 16;
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const char*>(c.base) + (int64_t)s * c.stride + (int64_t)sl * kSlice);
    uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(c.base) + (int64_t)d * c.stride + (int64_t)sl * kSlice);
    const int i = threadIdx.x, last = n - 1;
    const uint4 v0 = from[min(i, last)], v1 = from[min(i + kThreads, last)], v2 = from[min(i + 2 * kThreads, last)],
                v3 = from[min(i + 3 * kThreads, last)];
    if (i < n) to[i] = v0;
    if (i + kThreads < n) to[i + kThreads] = v1;
    if (i + 2 * kThreads < n) to[i + 2 * kThreads] = v2;
    if (i + 3 * kThreads < n) to[i + 3 * kThreads] = v3;
  }
  const int small = p.n - p.big, lane = threadIdx.x % kWave;
  const int64_t parts = (int64_t)np * small;
  for (int64_t it = (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave; it < parts;
       it += (int64_t)gridDim.x * (kThreads / kWave)) {
    const srswa_page_cache c = p.c[p.big + it % small];
    if (!pair((int)(it / small), &s, &d)) continue;
    const char* from = static_cast<const char*>(c.base) + (int64_t)s * c.stride;
    char* to = static_cast<char*>(c.base) + (int64_t)d * c.stride;
    if (((reinterpret_cast<uintptr_t>(c.base) | (uint64_t)c.stride | (uint64_t)c.bytes) & 3) == 0) {
      for (int64_t k = lane; k < c.bytes / 4; k += kWave)
        reinterpret_cast<uint32_t*>(to)[k] = reinterpret_cast<const uint32_t*>(from)[k];
    } else {
      for (int64_t k = lane; k < c.bytes; k += kWave) to[k] = from[k];
    }
  }
}

struct Layout {
  size_t need, src, dst, tfree, npairs, bits, total;
};
Layout layout_of(const srswa_pages_args* a) {
  const size_t n = (size_t)a->num_pages, r = (size_t)a->R, m = std::max(n, r);
  const size_t tiles = (n + kTile - 1) / kTile;
  auto up = [](size_t b) { return (b + 63) / 64 * 64; };
  Layout l;
  l.need = 0;
  l.src = l.need + up(m * 4);
  l.dst = l.src + up(m * 4);
  l.tfree = l.dst + up(m * 4);
  l.npairs = l.tfree + up(tiles * 4);
  l.bits = l.npairs + 64;
  l.total = l.bits + up((n + 31) / 32 * 4);
  return l;
}

int setup(const srswa_pages_args* a, void* ws, size_t ws_bytes, bool rows, const char* what, PagesK* k) {
  if (!a || !a->block_table || !a->seq_lens || !a->ref || (rows && !a->rows) || !a->block_table_out ||
      !a->seq_lens_out || !a->ref_out || !a->count || (a->ncaches > 0 && !a->caches)) {
    set_error("%s: null argument", what);
    return SRSWA_INVALID;
  }
  if (a->R <= 0 || a->W <= 0 || a->num_pages <= 0 || a->page_size <= 0 || a->ncaches < 0) {
    set_error("%s: bad sizes", what);
    return SRSWA_INVALID;
  }
  if (a->num_pages > (1 << 30) || (int64_t)a->R * a->W > (1ll << 38)) {
    set_error("%s: more than 2^30 pages or 2^38 table entries", what);
    return SRSWA_UNSUPPORTED;
  }
  for (int i = 0; i < a->ncaches; ++i)
    if (!a->caches[i].base || a->caches[i].bytes < 0 || a->caches[i].stride < a->caches[i].bytes) {
      set_error("%s: cache %d is null or its pages overlap", what, i);
      return SRSWA_INVALID;
    }
  const Layout l = layout_of(a);
  if (!ws || ws_bytes < l.total) {
    set_error("%s: workspace of %zu bytes required (got %zu)", what, l.total, ws_bytes);
    return SRSWA_WORKSPACE;
  }
  char* w = reinterpret_cast<char*>(ws);
  *k = PagesK{};
  k->bt = a->block_table;      k->bt_sr = a->bt_sr;
  k->sl = a->seq_lens;         k->ref = a->ref;            k->rows = a->rows;
  k->bto = a->block_table_out; k->bto_sr = a->bto_sr;
  k->slo = a->seq_lens_out;    k->refo = a->ref_out;       k->count = a->count;
  k->R = a->R;  k->W = a->W;  k->N = a->num_pages;  k->page_size = a->page_size;
  k->ntiles = (a->num_pages + kTile - 1) / kTile;
  k->need = reinterpret_cast<int32_t*>(w + l.need);
  k->src = reinterpret_cast<int32_t*>(w + l.src);
  k->dst = reinterpret_cast<int32_t*>(w + l.dst);
  k->tfree = reinterpret_cast<int32_t*>(w + l.tfree);
  k->npairs = reinterpret_cast<int32_t*>(w + l.npairs);
  k->bits = reinterpret_cast<uint32_t*>(w + l.bits);
  return SRSWA_OK;
}

// A cache whose pages are 16-byte aligned and hold 2 KB or more is cut into slices,
// any other copied by a wave a page.
bool is_big(const srswa_page_cache& c) {
  return ((reinterpret_cast<uintptr_t>(c.base) | (uint64_t)c.stride | (uint64_t)c.bytes) & 15) == 0 && c.bytes >= 2048;
}

void copy_pages(const srswa_pages_args* a, const PagesK& k, int64_t most_pairs, hipStream_t st) {
  for (int c0 = 0; c0 < a->ncaches; c0 += kMaxCaches) {
    CopyK c{};
    c.slices = 1;
    const int n = std::min(kMaxCaches, a->ncaches - c0);
    for (int big = 1; big >= 0; --big)
      for (int i = 0; i < n; ++i)
        if (is_big(a->caches[c0 + i]) == (big == 1)) {
          c.c[c.n++] = a->caches[c0 + i];
          if (big) {
            c.big = c.n;
            c.slices = std::max(c.slices, (int)((a->caches[c0 + i].bytes + kSlice - 1) / kSlice));
          }
        }
    c.src = k.src;  c.dst = k.dst;  c.npairs = k.npairs;  c.N = k.N;
    const int64_t items = most_pairs * std::max<int64_t>((int64_t)c.big * c.slices, (c.n - c.big + 3) / 4);
    copy_pages_kernel<<<(unsigned)std::max<int64_t>(1, std::min<int64_t>(items, 8192)), kThreads, 0, st>>>(c);
  }
}

int done(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s launch failed: %s", what, hipGetErrorString(e));
    return SRSWA_LAUNCH;
  }
  return SRSWA_OK;
}

}  // namespace
}  // namespace srswa

using namespace srswa;

extern "C" size_t srswa_pages_workspace(const srswa_pages_args* a) {
  return a && a->R > 0 && a->num_pages > 0 ? layout_of(a).total : 0;
}

extern "C" int srswa_pages_reserve(const srswa_pages_args* a, void* ws, size_t ws_bytes, void* stream) {
  PagesK k;
  const int rc = setup(a, ws, ws_bytes, true, "pages reserve", &k);
  if (rc != SRSWA_OK) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  reserve_count_kernel<<<(unsigned)(k.R + k.ntiles), kThreads, 0, st>>>(k);
  reserve_deal_kernel<<<(unsigned)k.R, kThreads, 0, st>>>(k);
  return done("pages reserve");
}

extern "C" int srswa_pages_reorder(const srswa_pages_args* a, void* ws, size_t ws_bytes, void* stream) {
  PagesK k;
  const int rc = setup(a, ws, ws_bytes, true, "pages reorder", &k);
  if (rc != SRSWA_OK) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (k.R <= kPlanRows && (int64_t)k.R * k.W <= kPlanEntries && k.N <= kPlanPages) {
    reorder_plan_kernel<<<1, kWide, 0, st>>>(k);
  } else {
    copy_ref_kernel<<<(unsigned)((k.N + kThreads - 1) / kThreads), kThreads, 0, st>>>(k);
    reorder_rows_kernel<<<(unsigned)k.R, kThreads, 0, st>>>(k);
    mark_kernel<<<(unsigned)k.ntiles, kThreads, 0, st>>>(k);
    reorder_deal_kernel<<<1, kThreads, 0, st>>>(k);
  }
  copy_pages(a, k, k.R, st);
  return done("pages reorder");
}

extern "C" int srswa_pages_compact(const srswa_pages_args* a, void* ws, size_t ws_bytes, void* stream) {
  PagesK k;
  const int rc = setup(a, ws, ws_bytes, false, "pages compact", &k);
  if (rc != SRSWA_OK) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  held_count_kernel<<<(unsigned)k.ntiles, kThreads, 0, st>>>(k);
  compact_plan_kernel<<<(unsigned)k.ntiles, kThreads, 0, st>>>(k);
  const int64_t rows = ((int64_t)k.R * k.W + kThreads - 1) / kThreads;
  compact_table_kernel<<<(unsigned)(rows + (k.N + kThreads - 1) / kThreads), kThreads, 0, st>>>(k, (int)rows);
  copy_pages(a, k, k.N / 2 + 1, st);
  return done("pages compact");
}
