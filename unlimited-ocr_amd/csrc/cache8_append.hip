// Append to the scaled 8-bit paged cache (gfx950).
//
// One workgroup = (page that a request's new tokens touch, kv head, K or V), so
// the page's scale has one writer, no atomics are needed and the result does
// not depend on the order of execution:
//   a  = max |x| over the page's new finite values          (pass 1)
//   s' = 2^e with a <= QMAX 2^e, at least the old scale where older keys stay
//   old bytes: round(q s / s') when s' > s;  new: round(x / s')   (pass 2)
// With powers of two x / s' is exact in fp32, so each value is rounded once.
#include "cache8.h"

namespace srswa {
namespace {

constexpr int kThreads = 256;

struct AppendK {
  srswa_cache8_append_args a;
  int pages_per_req;           // most pages a request's new tokens can touch
};

template <typename T, int KV, int D>
__global__ __launch_bounds__(kThreads) void cache8_append_kernel(AppendK p) {
  using V = Vec16<T>;
  constexpr int PP = D / 8;                 // 8-element pieces per row
  __shared__ float s_max[kThreads / kWave];
  const srswa_cache8_append_args& a = p.a;
  const int tid = threadIdx.x;
  int lid = (int)blockIdx.x;
  const bool is_v = lid & 1;
  lid >>= 1;
  const int h = lid % a.HKV;
  lid /= a.HKV;
  const int t = lid % p.pages_per_req, r = lid / p.pages_per_req;

  const int row0 = a.cu_seqlens ? min(max(a.cu_seqlens[r], 0), a.total) : r * a.max_new_len;
  const int row1 = a.cu_seqlens ? min(max(a.cu_seqlens[r + 1], row0), a.total) : row0 + a.max_new_len;
  const int64_t start = a.start[r];
  if (start < 0) return;
  const int64_t blk = start / a.page_size + t;
  if (blk >= a.max_blocks) return;
  const int64_t base = blk * a.page_size;
  const int64_t lo = max(start, base), hi = min(start + (row1 - row0), base + a.page_size);
  if (lo >= hi) return;
  const int page = a.block_table[(int64_t)r * a.bt_sr + blk];
  if (page < 0 || page >= a.num_pages) return;
  const int old_n = (int)(lo - base), n = (int)(hi - lo);

  const int64_t x_sn = is_v ? a.v_sn : a.k_sn, x_sh = is_v ? a.v_sh : a.k_sh;
  const T* x = reinterpret_cast<const T*>(is_v ? a.v : a.k) + (row0 + (lo - start)) * x_sn + h * x_sh;
  const int64_t c_sp = is_v ? a.vc_sp : a.kc_sp, c_st = is_v ? a.vc_st : a.kc_st, c_sh = is_v ? a.vc_sh : a.kc_sh;
  uint8_t* c = reinterpret_cast<uint8_t*>(is_v ? a.v_cache : a.k_cache) + page * c_sp + h * c_sh;
  float* sp = is_v ? a.v_scale + page * a.vs_sp + h * a.vs_sh : a.k_scale + page * a.ks_sp + h * a.ks_sh;
  const float old = *sp;

  float amax = 0.f;
  for (int i = tid; i < n * PP; i += kThreads) {
    float f[8];
    V::unpack(*reinterpret_cast<const uint4*>(x + (int64_t)(i / PP) * x_sn + i % PP * 8), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fabsf(f[e]) < INFINITY ? fmaxf(amax, fabsf(f[e])) : amax;
  }
  amax = wave_max(amax);
  if (tid % kWave == 0) s_max[tid / kWave] = amax;
  __syncthreads();                          // every thread has read the old scale too
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) amax = fmaxf(amax, s_max[w]);
  const float need = scale_for<KV>(amax);
  const float s = old_n > 0 ? fmaxf(old, need) : need;
  if (tid == 0) *sp = s;

  if (old_n > 0 && s != old) {
    const float ratio = old / s;
    for (int i = tid; i < old_n * PP; i += kThreads) {
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
  for (int i = tid; i < n * PP; i += kThreads) {
    float f[8];
    V::unpack(*reinterpret_cast<const uint4*>(x + (int64_t)(i / PP) * x_sn + i % PP * 8), f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = pow2 ? f[e] * inv : f[e] / s;
    *reinterpret_cast<uint2*>(c + (int64_t)(old_n + i / PP) * c_st + i % PP * 8) =
        make_uint2(to_bytes4<KV>(f), to_bytes4<KV>(f + 4));
  }
}

template <typename T, int KV>
void launch_d(const AppendK& k, unsigned grid, hipStream_t st) {
  if (k.a.D == 64) cache8_append_kernel<T, KV, 64><<<grid, kThreads, 0, st>>>(k);
  else cache8_append_kernel<T, KV, 128><<<grid, kThreads, 0, st>>>(k);
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
  const int64_t grid = (int64_t)a->R * k.pages_per_req * a->HKV * 2;
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
