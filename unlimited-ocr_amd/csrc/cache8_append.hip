// Append to the scaled 8-bit paged cache (gfx950).
//
// One workgroup = (page that a request's new tokens touch, kv head), K and V side by
// side, so the page's scales have one writer, no atomics are needed and the result
// does not depend on the order of execution:
//   a  = max |x| over the page's new finite values          (pass 1)
//   s' = 2^e with a <= QMAX 2^e, at least the old scale where older keys stay
//   old bytes: round(q s / s') when s' > s;  new: round(x / s')   (pass 2)
// With powers of two x / s' is exact in fp32, so each value is rounded once.  The
// new values stay in registers between the passes (pages of up to 64 keys).
#include <algorithm>

#include "cache8.h"

namespace srswa {
namespace {

constexpr int kHeld = 4;          // 16-byte pieces of K, and of V, that a thread holds

struct AppendK {
  srswa_cache8_append_args a;
  int pages_per_req;           // workgroups per request and head; 0: as many as the pages it touches
};

// Request r's new rows and where they go (n = 0 for a negative start).
struct Run {
  int row0;
  uint32_t n, start;
};
__device__ __forceinline__ Run run_of(const srswa_cache8_append_args& a, int r) {
  Run u;
  u.row0 = a.cu_seqlens ? min(max(a.cu_seqlens[r], 0), a.total) : r * a.max_new_len;
  const int row1 = a.cu_seqlens ? min(max(a.cu_seqlens[r + 1], u.row0), a.total) : u.row0 + a.max_new_len;
  const int start = a.start[r];
  u.n = start >= 0 ? (uint32_t)min(row1 - u.row0, a.max_new_len) : 0u;
  u.start = (uint32_t)max(start, 0);
  return u;
}

// Page number b over all requests' runs: its request and place there, the same on
// every lane; false past the last.
__device__ __forceinline__ bool nth_page(const AppendK& p, int b, int lane, int* r, int* t) {
  int64_t before = 0;
  for (int r0 = 0; r0 < p.a.R; r0 += kWave) {
    uint32_t n = 0;
    if (r0 + lane < p.a.R) {
      const Run u = run_of(p.a, r0 + lane);
      const uint32_t ps = (uint32_t)p.a.page_size;
      n = u.n > 0 ? (u.start + u.n - 1) / ps - u.start / ps + 1 : 0u;
    }
    uint32_t incl = n;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const uint32_t x = __shfl_up(incl, o, kWave);
      if (lane >= o) incl += x;
    }
    const uint64_t past = __ballot(before + (int64_t)incl > b);
    if (past) {
      const int i = __ffsll((long long)past) - 1;
      *r = __builtin_amdgcn_readfirstlane(r0 + i);
      *t = __builtin_amdgcn_readfirstlane((int)(b - before - (int64_t)__shfl(incl - n, i, kWave)));
      return true;
    }
    before += __shfl(incl, kWave - 1, kWave);
  }
  return false;
}

// K or V of the page
struct Side {
  const void* x;                // first new row
  int64_t x_sn;
  uint8_t* c;                   // the page's first row
  int64_t c_st;
  float* scale;
};

template <typename T, int KV, int D, int NT>
__global__ __launch_bounds__(NT) void cache8_append_kernel(AppendK p) {
  using V = Vec16<T>;
  constexpr int PP = D / 8;                 // 8-element pieces per row
  __shared__ float s_max[2][NT / kWave];
  const srswa_cache8_append_args& a = p.a;
  const int tid = threadIdx.x;
  const int h = (int)blockIdx.x % a.HKV, nth = (int)blockIdx.x / a.HKV;
  int r, t;                                 // the workgroup's request, and which of its pages
  if (p.pages_per_req > 0) {
    r = nth / p.pages_per_req;
    t = nth % p.pages_per_req;
  } else if (!nth_page(p, nth, tid % kWave, &r, &t)) {
    return;
  }
  const Run u = run_of(a, r);
  const uint32_t blk = u.start / (uint32_t)a.page_size + (uint32_t)t;
  if (u.n == 0 || blk >= (uint32_t)a.max_blocks) return;
  const int64_t start = u.start, base = (int64_t)blk * a.page_size;
  const int64_t lo = max(start, base), hi = min(start + u.n, base + a.page_size);
  if (lo >= hi) return;
  const int page = a.block_table[(int64_t)r * a.bt_sr + blk];
  if (page < 0 || page >= a.num_pages) return;
  const int old_n = (int)(lo - base), n = (int)(hi - lo);
  const int64_t row = u.row0 + (lo - start);
  const Side side[2] = {
      {reinterpret_cast<const T*>(a.k) + row * a.k_sn + h * a.k_sh, a.k_sn,
       reinterpret_cast<uint8_t*>(a.k_cache) + page * a.kc_sp + h * a.kc_sh, a.kc_st,
       a.k_scale + page * a.ks_sp + h * a.ks_sh},
      {reinterpret_cast<const T*>(a.v) + row * a.v_sn + h * a.v_sh, a.v_sn,
       reinterpret_cast<uint8_t*>(a.v_cache) + page * a.vc_sp + h * a.vc_sh, a.vc_st,
       a.v_scale + page * a.vs_sp + h * a.vs_sh}};
  auto piece = [&](int v, int i) {
    return *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(side[v].x) + (int64_t)(i / PP) * side[v].x_sn + i % PP * 8);
  };
  const bool few = n * PP <= NT;            // one piece of each per thread
  uint4 held[2][kHeld];
  float amax[2] = {0.f, 0.f}, old[2];
  auto take = [&](int v, const uint4& w) {
    float f[8];
    V::unpack(w, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax[v] = fabsf(f[e]) < INFINITY ? fmaxf(amax[v], fabsf(f[e])) : amax[v];
  };
  // (the clamped loads read the last piece again, which is no other value)
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    old[v] = *side[v].scale;
    held[v][0] = piece(v, min(tid, n * PP - 1));
  }
  if (!few) {
#pragma unroll
    for (int k = 1; k < kHeld; ++k)
#pragma unroll
      for (int v = 0; v < 2; ++v) held[v][k] = piece(v, min(tid + k * NT, n * PP - 1));
#pragma unroll
    for (int k = 1; k < kHeld; ++k)
#pragma unroll
      for (int v = 0; v < 2; ++v) take(v, held[v][k]);
    for (int i = tid + kHeld * NT; i < n * PP; i += NT) {
      take(0, piece(0, i));
      take(1, piece(1, i));
    }
  }
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    take(v, held[v][0]);
    amax[v] = wave_max(amax[v]);
  }
  if constexpr (NT > kWave) {
    if (tid % kWave == 0) {
      s_max[0][tid / kWave] = amax[0];
      s_max[1][tid / kWave] = amax[1];
    }
    __syncthreads();                        // every thread has read the old scales too
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) {
      amax[0] = fmaxf(amax[0], s_max[0][w]);
      amax[1] = fmaxf(amax[1], s_max[1][w]);
    }
  }
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const float need = scale_for<KV>(amax[v]);
    const float s = old_n > 0 ? fmaxf(old[v], need) : need;
    uint8_t* c = side[v].c;
    const int64_t c_st = side[v].c_st;
    if (tid == 0) *side[v].scale = s;
    if (old_n > 0 && s != old[v]) {
      const float ratio = old[v] / s;
      for (int i = tid; i < old_n * PP; i += NT) {
        uint2* w = reinterpret_cast<uint2*>(c + (int64_t)(i / PP) * c_st + i % PP * 8);
        const uint2 b = *w;
        float f[8];
        from_bytes4<KV>(b.x, f);
        from_bytes4<KV>(b.y, f + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= ratio;
        *w = make_uint2(to_bytes4<KV>(f), to_bytes4<KV>(f + 4));
      }
    }
    // a caller's own scale need not be a power of two: then x / s is a division
    const bool pow2 = (__float_as_uint(s) & 0x7fffffu) == 0u;
    const float inv = 1.f / s;
    auto put = [&](int i, const uint4& w) {
      float f[8];
      V::unpack(w, f);
      if (pow2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= inv;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] /= s;
      }
      *reinterpret_cast<uint2*>(c + (int64_t)(old_n + i / PP) * c_st + i % PP * 8) =
          make_uint2(to_bytes4<KV>(f), to_bytes4<KV>(f + 4));
    };
    if (tid < n * PP) put(tid, held[v][0]);
    if (!few) {
#pragma unroll
      for (int k = 1; k < kHeld; ++k)
        if (tid + k * NT < n * PP) put(tid + k * NT, held[v][k]);
      for (int i = tid + kHeld * NT; i < n * PP; i += NT) put(i, piece(v, i));
    }
  }
}

// One wave where no request brings more than four rows' pieces.
template <typename T, int KV, int D>
void launch_n(const AppendK& k, unsigned grid, hipStream_t st) {
  if (k.a.max_new_len <= kWave / (D / 8)) cache8_append_kernel<T, KV, D, kWave><<<grid, kWave, 0, st>>>(k);
  else cache8_append_kernel<T, KV, D, 256><<<grid, 256, 0, st>>>(k);
}

template <typename T, int KV>
void launch_d(const AppendK& k, unsigned grid, hipStream_t st) {
  if (k.a.D == 64) launch_n<T, KV, 64>(k, grid, st);
  else launch_n<T, KV, 128>(k, grid, st);
}

template <typename T>
void launch_kv(const AppendK& k, unsigned grid, hipStream_t st) {
  if (k.a.kv_dtype == SRSWA_I8) launch_d<T, kI8>(k, grid, st);
  else launch_d<T, kFp8E4M3FN>(k, grid, st);
}

bool al(const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

}  // namespace
}  // namespace srswa

using namespace srswa;

extern "C" int srswa_cache8_append(const srswa_cache8_append_args* a, void* stream) {
  if (!a || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->k_scale || !a->v_scale || !a->block_table ||
      !a->start) {
    set_error("cache8 append: null argument");
    return SRSWA_INVALID;
  }
  if (a->R < 0 || a->total < 0 || a->max_new_len < 0 || a->HKV <= 0 || a->max_blocks <= 0 || a->num_pages <= 0 ||
      a->page_size <= 0 || (!a->cu_seqlens && (int64_t)a->R * a->max_new_len != a->total)) {
    set_error("cache8 append: bad sizes");
    return SRSWA_INVALID;
  }
  if (!(a->D == 64 || a->D == 128) || !(a->dtype == SRSWA_BF16 || a->dtype == SRSWA_F16) ||
      !(a->kv_dtype == SRSWA_I8 || a->kv_dtype == SRSWA_FP8_E4M3FN)) {
    set_error("cache8 append: D=%d / dtype %d / cache format %d not supported", a->D, a->dtype, a->kv_dtype);
    return SRSWA_UNSUPPORTED;
  }
  if (a->page_size % 16 || a->page_size > 1024) {
    set_error("cache8 append: page size %d must be a multiple of 16 up to 1024", a->page_size);
    return SRSWA_UNSUPPORTED;
  }
  if (!al(a->k, 16) || !al(a->v, 16) || a->k_sn % 8 || a->k_sh % 8 || a->v_sn % 8 || a->v_sh % 8 ||
      !al(a->k_cache, 16) || !al(a->v_cache, 16) || a->kc_sp % 16 || a->kc_st % 16 || a->kc_sh % 16 ||
      a->vc_sp % 16 || a->vc_st % 16 || a->vc_sh % 16) {
    set_error("cache8 append: rows must be 16-byte aligned");
    return SRSWA_UNSUPPORTED;
  }
  if (a->R == 0 || a->max_new_len == 0 || a->total == 0) return SRSWA_OK;
  AppendK k{*a, (int)(((int64_t)a->max_new_len - 1 + a->page_size - 1) / a->page_size) + 1};
  // uneven runs: as many workgroups as their pages (each run adds at most two parts
  // of pages), which the workgroups count; five runs of 13 to 8,000 rows 15.7 -> 14.5 us
  const int64_t even = (int64_t)a->R * k.pages_per_req, own = (int64_t)a->total / a->page_size + 2 * (int64_t)a->R;
  if (own < even) k.pages_per_req = 0;
  const int64_t grid = std::min(even, own) * a->HKV;
  if (grid > 0x7fffffff) {
    set_error("cache8 append: grid too large");
    return SRSWA_UNSUPPORTED;
  }
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (a->dtype == SRSWA_BF16) launch_kv<bf16_t>(k, (unsigned)grid, st);
  else launch_kv<__half>(k, (unsigned)grid, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("cache8 append launch failed: %s", hipGetErrorString(e));
    return SRSWA_LAUNCH;
  }
  return SRSWA_OK;
}
