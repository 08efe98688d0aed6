// Shared pieces of the scaled 8-bit paged cache (float8_e4m3fn or int8 values,
// one fp32 scale per page and kv head): conversions and the page geometry.
#pragma once

#include "common.h"

namespace srswa {

constexpr int kI8 = SRSWA_I8;
constexpr int kScaleMinExp = -100;          // a page of zeros has scale 2^-100
constexpr float kScaleMin = 0x1p-100f;

template <int KV> constexpr float kQMax = KV == kI8 ? 127.f : 448.f;

// The smallest power of two s >= 2^kScaleMinExp with a <= QMAX s, for finite
// a >= 0.  With a = 1.m 2^x (fp32 fields) and QMAX = 1.f 2^w the exponent is
// x - w, one more when m > f: no division and no rounding.  (A subnormal a has
// x = -127 and falls to the minimum.)
template <int KV>
__device__ __forceinline__ float scale_for(float a) {
  constexpr int w = KV == kI8 ? 6 : 8;                          // 127 = 1.984375 2^6, 448 = 1.75 2^8
  constexpr uint32_t f = KV == kI8 ? 0x7e0000u : 0x600000u;
  const uint32_t u = __float_as_uint(a);
  const int e = max((int)(u >> 23) - 127 - w + ((u & 0x7fffffu) > f ? 1 : 0), kScaleMinExp);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// four values in units of the scale -> four bytes, round to nearest even,
// saturating; NaN stays NaN in e4m3 and becomes 0 in int8
template <int KV>
__device__ __forceinline__ uint32_t to_bytes4(const float* y) {
  if constexpr (KV == kI8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = y[i] == y[i] ? fminf(fmaxf(rintf(y[i]), -127.f), 127.f) : 0.f;
      w |= ((uint32_t)(int)c & 0xffu) << (8 * i);
    }
    return w;
  } else {
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = y[i] == y[i] ? fminf(fmaxf(y[i], -448.f), 448.f) : y[i];
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], w, true);
    return (uint32_t)w;
  }
}

__device__ __forceinline__ float i8_f32(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

// four bytes -> fp32, in units of the scale
template <int KV>
__device__ __forceinline__ void from_bytes4(uint32_t w, float* f) {
  if constexpr (KV == kI8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = i8_f32(w, i);
  } else {
    const f32x2_t a = fp8x2_f32<KV, false>(w), b = fp8x2_f32<KV, true>(w);
    f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
  }
}

// 0x80 in each byte of four that holds an e4m3 NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_bytes4(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// w with those bytes zeroed
__device__ __forceinline__ uint32_t without(uint32_t w, uint32_t nan) { return w & ~((nan >> 7) * 0xffu); }

// The sum l holds p' 2^-kLift / vs: between 2^-125 (one key, the largest bf16 value's
// scale 2^120) and 2^127 (2^24 keys at the smallest scale, p' = 2^15) it stays a
// normal number.
constexpr int kLift = 12;

// out = O inv_sum(M, L), lse = lse_of(M, L): M is -inf where no key was seen (L = 0)
// and where every logit was NaN (L too).
__device__ __forceinline__ float inv_sum(float M, float L) { return M == -INFINITY ? 0.f : 0x1p-12f / L; }
__device__ __forceinline__ float lse_of(float M, float L) {
  return M == -INFINITY ? L - INFINITY : (M + (log2f(L) + kLift)) * kLn2;
}

// A wave-uniform condition in a form the compiler must take for a lane's own, so
// that the rare updates under it happen in place: under a uniform branch it copied
// the whole set of accumulators to other registers on the common path.
__device__ __forceinline__ bool per_lane(bool c) {
  int v = c;
  asm("" : "+v"(v));
  return v != 0;
}

// Waits here for loaded values that a loop uses: left alone, the wait stands at
// their first use inside the loop and, counting in order, drains the loop's own
// prefetches in every pass.
template <int N>
__device__ __forceinline__ void settle(uint4 (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(v[i].x), "+v"(v[i].y), "+v"(v[i].z), "+v"(v[i].w));
}

// lane q's value, uniform
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int q) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, q);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), q);
  return (uint64_t)hi << 32 | lo;
}

// two fp32 values -> packed fp16, round to nearest even (v_cvt_pk_f16_f32)
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const f16x2_native_t v = {(_Float16)lo, (_Float16)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// four bytes -> four values of T, two words (exact: every e4m3 and int8 value
// is a bf16 and an fp16 value)
template <int KV, typename T>
__device__ __forceinline__ uint2 bytes4_to(uint32_t w) {
  if constexpr (KV == kI8) {
    if constexpr (std::is_same<T, bf16_t>::value) {
      return make_uint2(pack_bf16x2(i8_f32(w, 0), i8_f32(w, 1)), pack_bf16x2(i8_f32(w, 2), i8_f32(w, 3)));
    } else {
      // x + 128 as a byte b under the exponent of 1024 is the fp16 value 1024 + b
      const uint32_t u = w ^ 0x80808080u;
      const f16x2_native_t k = {(_Float16)-1152.f, (_Float16)-1152.f};
      const f16x2_native_t a = __builtin_bit_cast(f16x2_native_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + k;
      const f16x2_native_t b = __builtin_bit_cast(f16x2_native_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + k;
      return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    }
  } else {
    return make_uint2(fp8x2_to<KV, T, false>(w), fp8x2_to<KV, T, true>(w));
  }
}

// Host side shared by the two attention forms (cache8_decode.hip): the checks of
// the arguments, and the split-over-keys form behind both entry points.
int cache8_check(const srswa_cache8_attend_args* a, const char* what);
int cache8_decode_run(const srswa_cache8_attend_args* a, void* ws, size_t ws_bytes, void* stream, const char* what);
size_t cache8_decode_ws(const srswa_cache8_attend_args* a);
// what that form does for a call: (item, kv head) pairs, units of 32 keys of one at most,
// and whether they are shared out
void cache8_decode_load(const srswa_cache8_attend_args* a, int64_t* wgs, int64_t* units, bool* shared);
inline bool cache8_plannable(const srswa_cache8_attend_args* a) {
  return a && a->R > 0 && a->HQ > 0 && a->HKV > 0 && a->page_size >= 16 && a->max_blocks > 0 && a->max_query_len > 0;
}
inline int cache8_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s launch failed: %s", what, hipGetErrorString(e));
    return SRSWA_LAUNCH;
  }
  return SRSWA_OK;
}

}  // namespace srswa
