// serve_common.cuh — what the serving kernels over a block-scaled cache share:
// status words, element conversions and the search for a row's request.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/marathon_shift.h"

namespace mshift {

// Records the CUDA error's text for mshift_last_cuda_error; returns MSHIFT_ECUDA.
int cuda_fail(cudaError_t e);

namespace serve {

constexpr float kFMax = 448.0f;         // largest finite e4m3 value
constexpr float kScaleFloor = 0x1p-64f;  // smallest block scale append writes, attend divides by

__device__ __forceinline__ void flag(uint32_t* err, uint32_t bit) { atomicOr(err, bit); }

// Two e4m3 codes (the low 16 bits of w) as f16x2; exact, NaN codes stay NaN.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return r;
}

// {lo, hi} rounded to nearest even, saturated at +-448 (infinities too), NaN kept.
__device__ __forceinline__ uint16_t f32x2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// One 32-bit word of bf16 / f16 / f32 elements to fp32 and back (round to nearest even).
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPer = 2;
  __device__ static void unpack(uint32_t w, float* f) {
    f[0] = __uint_as_float(w << 16);
    f[1] = __uint_as_float(w & 0xffff0000u);
  }
  __device__ static uint32_t pack(const float* f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f[0], f[1]);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Elem<__half> {
  static constexpr int kPer = 2;
  __device__ static void unpack(uint32_t w, float* f) {
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w));
    f[0] = p.x;
    f[1] = p.y;
  }
  __device__ static uint32_t pack(const float* f) { return pack_f16x2(f[0], f[1]); }
  __device__ static float get(__half x) { return __half2float(x); }
  __device__ static __half put(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<float> {
  static constexpr int kPer = 1;
  __device__ static void unpack(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
  __device__ static uint32_t pack(const float* f) { return __float_as_uint(f[0]); }
  __device__ static float get(float x) { return x; }
  __device__ static float put(float x) { return x; }
};

// An offset kept inside the call's rows, whatever the caller's array holds; and query_start[i] so.
__device__ __forceinline__ int inside(int offset, int rows) { return min(max(offset, 0), rows); }
__device__ __forceinline__ int row_start(const int32_t* qs, int i, int rows) {
  return inside(qs[i], rows);
}

// The last r in [0, reqs) with key(r) <= x, for a non-decreasing key (0 if there
// is none).  All 32 lanes call it together: each step reads 32 evenly spaced
// keys, so 1,024 requests take two dependent reads instead of ten.
template <typename Key>
__device__ __forceinline__ int find_request(int reqs, long long x, Key key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = reqs;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const bool below = at < hi && key(at) <= x;
    const unsigned m = __ballot_sync(0xffffffffu, below);
    const int last = m ? 31 - __clz(m) : 0;  // lane 0's key is <= x unless there is no answer
    lo = lo + last * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

}  // namespace serve
}  // namespace mshift
