// Rows of values held in 8 bits: per group of consecutive values one float
// scale s, and per value a code q with value = q * s.
//   int8: s = max|x| / 127, q in [-127, 127] (s a step less where 127 s would
//         pass the largest float);
//   e4m3: s = the smallest power of two (at least 2^-126) with max|x| / s <= 448,
//         so that x / s and q * s are exact and storing stored values again
//         changes nothing.  The format's own exponent covers 2^-9 .. 448 (.. 240
//         with s = 2^120, so that every stored value is finite).
// A group of zeros has s = 0; a group that holds a NaN or an infinity has
// s = NaN and reads back as NaN throughout: nothing non-finite is hidden.
// q is x / s rounded to nearest even or, dithered, floor(|x / s| / step + u)
// steps with u in [0, 1) from a hash of (seed, row, column): the expected
// value of a stored number is then the number, which a moving average whose
// change per step is below half a step needs (rounded to nearest, it stands).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cfloat>
#include <cstdint>

namespace blitz {
namespace quant {

enum Kind : int { kInt8 = 0, kE4m3 = 1 };

// The hash of (seed, row, column): odd multipliers between shifts.  0x9E3779B1 and 0x85EBCA77
// are primes that Y. Collet published for hashing 32-bit words; 0x7FEB352D, 0x846CA68B and
// 0x2C1B3C6D come from C. Wellons's published search for 32-bit mixers of little bias.
__device__ __forceinline__ uint32_t row_key(uint32_t seed, int64_t row) {
  uint32_t k = seed * 0x9E3779B1u + (uint32_t)row * 0x85EBCA77u;
  k = (k ^ (k >> 16)) * 0x7FEB352Du;
  k = (k ^ (k >> 15)) * 0x846CA68Bu;
  return k ^ (k >> 16);
}

// 20 random bits
__device__ __forceinline__ uint32_t random20(uint32_t key, uint32_t col) {
  uint32_t h = key + col * 0x9E3779B1u;
  h = (h ^ (h >> 15)) * 0x2C1B3C6Du;
  h = h ^ (h >> 12);
  return h >> 12;
}

// the group's scale, and what x is multiplied by (e4m3) before it is rounded
template <int KIND>
__device__ __forceinline__ float group_scale(float amax, bool finite) {
  if (!finite) return __int_as_float(0x7fffffff);
  if (KIND == kInt8) {
    const float s = __fdiv_rn(amax, 127.0f);
    // next to the largest float 127 s may round to infinity: one step less
    return __fmul_rn(s, 127.0f) <= FLT_MAX ? s : __int_as_float(__float_as_int(s) - 1);
  }
  const int bits = __float_as_int(amax);
  // amax = 1.f * 2^e: 448 = 1.75 * 2^8, so s = 2^(e-8) while 1.f <= 1.75
  const int e = max((bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), 1);
  return amax > 0.0f ? __int_as_float(e << 23) : 0.0f;
}

// 1 / s of a power of two s >= 2^-126 (s <= 2^120 for any finite group); 0 for 0
__device__ __forceinline__ float inverse_pow2(float s) {
  return s > 0.0f ? __int_as_float((254 << 23) - __float_as_int(s)) : 0.0f;
}

// What the codes of one group are formed with.
template <int KIND>
struct GroupCode {
  float s, inv;    // the scale; inverse_pow2(s) (e4m3 only)
  uint32_t limit;  // largest magnitude code: 448, or 240 where 256 s would be past the largest float
  __device__ __forceinline__ explicit GroupCode(float scale)
      : s(scale), inv(KIND == kE4m3 ? inverse_pow2(scale) : 0.0f), limit(scale >= 0x1p120f ? 0x77u : 0x7eu) {}
};

// two e4m3 codes -> the numbers they stand for (one conversion makes both)
__device__ __forceinline__ float2 e4m3_pair(uint8_t x, uint8_t y) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((uint32_t)x | (uint32_t)y << 8), __NV_E4M3);
  return __half22float2(__half2(h));
}

// |y| -> magnitude code of y dithered by r20 (see encode)
__device__ __forceinline__ uint32_t e4m3_dithered(float y, uint32_t r20) {
  return ((uint32_t)__float_as_int(__fmul_rz(fabsf(y), 0x1p-120f)) + r20) >> 20;
}

// x -> code; r20: random20 (dithered only).
//
// An e4m3 magnitude's 7 bits are the top of the float |y| * 2^-120: the
// exponents then agree, and below 2^-6 both formats count in equal steps (the
// float's are denormal).  The 20 bits behind them are the fraction of a step,
// so dithering is an integer addition of 20 random bits; the multiplication
// rounds towards zero, which does not change floor(fraction + u).
template <int KIND, bool DITHER, bool NEVER_ZERO = false>
__device__ __forceinline__ uint8_t encode(float x, const GroupCode<KIND>& g, uint32_t r20) {
  if (KIND == kInt8) {
    // a true division, so that the rounding is of x / s itself
    const float y = g.s > 0.0f ? __fdiv_rn(x, g.s) : 0.0f;
    const float q = DITHER ? floorf(__fadd_rn(y, __int_as_float(0x3f800000 | (r20 << 3)) - 1.0f)) : rintf(y);
    return (uint8_t)(int8_t)(int)fminf(fmaxf(q, -127.0f), 127.0f);
  } else {
    const float y = __fmul_rn(x, g.inv);
    uint32_t code;
    if (DITHER)
      code = e4m3_dithered(y, r20);
    else
      code = (uint32_t)__nv_cvt_float_to_fp8(fabsf(y), __NV_SATFINITE, __NV_E4M3);
    code = min(code, g.limit);
    // where x > 0, the smallest code at least (x is never negative there)
    if (NEVER_ZERO) code = x > 0.0f ? max(code, 1u) : code;
    return (uint8_t)(code | ((uint32_t)__float_as_int(x) >> 24 & 0x80u));
  }
}

// two codes -> their values.  The e4m3 bytes 0x7f and 0xff, which encode never makes but a
// caller's tensor may hold, are NaN in the format and here.
template <int KIND>
__device__ __forceinline__ float2 decode2(uint8_t x, uint8_t y, float s) {
  const float2 v = KIND == kInt8 ? make_float2((float)(int8_t)x, (float)(int8_t)y) : e4m3_pair(x, y);
  return make_float2(__fmul_rn(v.x, s), __fmul_rn(v.y, s));
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// maximum over LANES neighbouring lanes (a power of two)
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace quant
}  // namespace blitz
