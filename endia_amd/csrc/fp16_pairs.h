// fp32 numbers as pairs of fp16 for the matrix cores.
//
// The fp32 matrix instruction multiplies at 1/16 of the fp16 rate. An fp32 number x that has been scaled by a power of two
// so that the largest of its group lies in [2^13, 2^14) is held as hi = fp16(x), lo = fp16(x - hi): the difference is exact in
// fp32, so hi + lo is off by at most 2^-22 |x| (half a step of fp16, 2^-11, twice), or by 2^-25 where lo is subnormal, which
// is 2^-38 of the group's largest. A product is then three fp16 matrix products accumulated in fp32,
//   x y = hi_x hi_y + hi_x lo_y + lo_x hi_y   (lo_x lo_y, at most 2^-22 |x y|, is left out),
// 3/16 of the time of the fp32 instruction at an error of the size of fp32's own rounding. The scales are powers of two, so
// applying and removing them rounds nothing. Non-finite values take no part in choosing a scale; they reach the result as NaN.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pairs {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kTop = 13;        // the largest of a group is scaled to [2^kTop, 2^(kTop + 1))
constexpr int kMaxShift = 100;  // groups below 2^-87 (zeros among them) are not scaled any further up

__device__ __forceinline__ void split2(float x, float y, half2v& hi, half2v& lo) {
  const float2v f = {x, y};
  hi = __builtin_convertvector(f, half2v);
  const float2v r = {x - (float)hi[0], y - (float)hi[1]};
  lo = __builtin_convertvector(r, half2v);
}

__device__ __forceinline__ void split8(const float (&x)[8], half8& hi, half8& lo) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    half2v a, b;
    split2(x[i], x[i + 1], a, b);
    hi[i] = a[0];
    hi[i + 1] = a[1];
    lo[i] = b[0];
    lo[i + 1] = b[1];
  }
}

// |x| for the choice of a scale: 0 for infinities and NaN
__device__ __forceinline__ float finite_abs(float x) {
  const float a = __builtin_fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// s such that a number of size amax, times 2^s, lies in [2^kTop, 2^(kTop + 1))
__device__ __forceinline__ int shift_of(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23) - 127;
  const int s = kTop - e;
  return s < kMaxShift ? s : kMaxShift;
}

__device__ __forceinline__ float scaled(float x, int shift) { return __builtin_ldexpf(x, shift); }

// three matrix products: acc += a b for a 32 x 16 and a 16 x 32 block held as pairs
__device__ __forceinline__ floatx16 mfma_pairs(half8 ah, half8 al, half8 bh, half8 bl, floatx16 acc) {
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(al, bh, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bl, acc, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(ah, bh, acc, 0, 0, 0);
}

// One wave: 64 lanes x 16 bytes from global memory straight into LDS (lane i's bytes land at lds + 16 i). The caller waits
// (wait_loads) before the barrier behind which the bytes are read.
__device__ __forceinline__ void load_to_lds(const void* global_of_lane, void* lds_of_wave) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)global_of_lane,
                                   (__attribute__((address_space(3))) void*)lds_of_wave, 16, 0, 0);
}
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

}  // namespace pairs
