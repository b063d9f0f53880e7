// Reading an update and writing its direction, shared by the orthogonalisation kernels.
#pragma once
#include <type_traits>

#include "kernels.h"
#include "ortho.h"
#include "quant.cuh"

namespace blitz {

// the powers of two that X (at least, see OrthoInfo), A and B are scaled by in f16 terms (see ortho.cu)
constexpr float kScaleX = 16384.0f, kScaleA = 16384.0f, kScaleB = 8192.0f;

// How one matrix is scaled into f16.  u is stored as u * up.x * up.y (ortho_up).  X_i, i > 0,
// is stored times 2^(14 + k[i]), with k[i] > 0 where u is so much smaller than eps (or the
// coefficients so small) that this iterate is small: it would lie among f16's denormals (40 x 60
// with eps = 1e-7 came out 1.6e-3 off for a norm of 1e-15).  X_1 so scaled is B_0 times
// `first` times what is stored of u.
struct OrthoInfo {
  float2 up;
  float first;
  uint8_t k[kMostSteps + 4];
};

__device__ __forceinline__ float ortho_pow2(int e) { return __int_as_float((127 + e) << 23); }

// the exponent that takes a 2-norm into [2^13, 2^14) (less for the largest, whose values are then
// still below 4)
__device__ __forceinline__ int ortho_exponent(double norm) {
  return max(-126, norm > 0.0 && norm <= 1e300 ? 14 - (ilogb(norm) + 1) : 0);
}
// exact, in two factors, since 2^163 is no float
__device__ __forceinline__ float2 ortho_up(double norm) {
  const int e = ortho_exponent(norm);
  return make_float2(ortho_pow2(min(e, 80)), ortho_pow2(max(e - 80, 0)));
}
__device__ __forceinline__ void ortho_scaling(double norm, const OrthoParams& p, OrthoInfo* info) {
  info->up = ortho_up(norm);
  const double a = fabs((double)p.a), b = fabs((double)p.b), c = fabs((double)p.c);
  int first = 0;
  if (norm < (double)p.eps || a + b + c < 1.0) {
    // bounds of the iterates: a step multiplies singular values up to s by at most
    // a + b s^2 + c s^4, and they stay below 1.85 (checked by the caller)
    double s = norm / (norm + (double)p.eps);
    for (int i = 0; i <= p.steps; ++i) {
      const int k = s > 0.0 ? max(0, min(100, ilogb(1.85 / s))) : 0;
      info->k[i] = (uint8_t)k;
      if (i == 1) first = k;
      s = fmin(s * (a + s * s * (b + s * s * c)), 1.85);
    }
  } else {
    for (int i = 0; i <= p.steps; ++i) info->k[i] = 0;
  }
  // zeros stay zeros, whatever eps is
  info->first = norm == 0.0 ? 0.0f
                            : (float)(1.0 / ((norm + (double)p.eps) * ldexp(1.0, ortho_exponent(norm) - 14 - first)));
}
// what a step's sums are multiplied by: those of X X^T squared, to give A; those of B X, to give the
// next X as it is stored, or the direction
struct OrthoFactors {
  float x, next;
};
__device__ __forceinline__ OrthoFactors ortho_factors(const OrthoInfo& info, int step, bool last) {
  const int k = info.k[step], to = info.k[step + 1];
  OrthoFactors f;
  if (step == 0) {
    f.x = info.first * ortho_pow2(-14 - to);
    f.next = (last ? f.x : info.first) / kScaleB;
  } else {
    f.x = ortho_pow2(-14 - k);
    f.next = (last ? f.x : ortho_pow2(to - k)) / kScaleB;
  }
  return f;
}

// whether u needs two f16 terms
__host__ __device__ inline bool ortho_two_in(const OrthoParams& p) { return p.param || p.g_type == kValueF32; }

// What the kernels that stay in 32 bits multiply u with 2-norm `norm` by, in two factors: alone
// 1 / norm would be infinite for norms below 2^-128.  .y is 1 but for the smallest.
__device__ __forceinline__ float2 ortho_inverse(double norm, float eps) {
  const double s = norm == 0.0 ? 0.0 : 1.0 / (norm + (double)eps);
  return s > 0x1p100 ? make_float2((float)(s * 0x1p-80), 0x1p80f) : make_float2((float)s, 1.0f);
}

// 32 bytes of global memory, a whole sector, by one lane
__device__ __forceinline__ void store32(void* p, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void load32(const void* p, uint32_t (&v)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p)
               : "memory");
}
// two values' high terms and, in lo, low ones (one conversion makes a pair)
__device__ __forceinline__ uint32_t split2(float x, float y, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  lo = *(const uint32_t*)&l;
  return *(const uint32_t*)&h;
}
// two values from their terms
__device__ __forceinline__ float2 join2(uint32_t hi, uint32_t lo) {
  const float2 h = __half22float2(*(const __half2*)&hi), l = __half22float2(*(const __half2*)&lo);
  return make_float2(h.x + l.x, h.y + l.y);
}
// 8 values as 8 high terms and 8 low ones
__device__ __forceinline__ void split8(const float* v, uint4& hi, uint4& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = split2(v[2 * e], v[2 * e + 1], l[e]);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// V neighbouring values from memory, in 32 bits (V = 4: aligned to 4 of them)
template <int V>
__device__ __forceinline__ void load_values(const float* p, float (&v)[V]) {
  if constexpr (V == 4) {
    const float4 q = *(const float4*)p;
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  } else {
    v[0] = *p;
  }
}
template <int V, class T>
__device__ __forceinline__ void load_values(const T* p, float (&v)[V]) {
  if constexpr (V == 4) {
    const uint2 q = *(const uint2*)p;
    const T* t = (const T*)&q;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = quant::to_float(t[k]);
  } else {
    v[0] = quant::to_float(*p);
  }
}
template <int V>
__device__ __forceinline__ void store_values(float* p, const float (&v)[V]) {
  if constexpr (V == 4)
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
  else
    *p = v[0];
}
template <int V, class T>
__device__ __forceinline__ void store_values(T* p, const float (&v)[V]) {
  if constexpr (V == 4) {
    T t[4];
#pragma unroll
    for (int k = 0; k < V; ++k) t[k] = quant::from_float<T>(v[k]);
    *(uint2*)p = *(const uint2*)t;
  } else {
    *p = quant::from_float<T>(v[0]);
  }
}

// whether the tensors begin where 4 neighbouring values can be taken at once, and whether every
// row does
inline bool ortho_aligned(const OrthoParams& p) {
  const uintptr_t narrow = (uintptr_t)p.g | (uintptr_t)p.out;
  const uintptr_t wide = (uintptr_t)p.momentum | (uintptr_t)p.param | (p.g_type == kValueF32 ? narrow : 0);
  return wide % 16 == 0 && narrow % 8 == 0;
}
inline bool ortho_by_four(const OrthoParams& p) { return (p.sj == 1 ? p.m : p.n) % 4 == 0 && ortho_aligned(p); }

// f(position, u) for groups of V values of u at first, first + step, ... below `end`,
// K groups loaded before the first is used.  T: type of g; UPDATE: with momentum and
// parameter; ADVANCE: this reading advances the momentum.  (Types are template arguments
// of the kernels: six variants of this in one kernel cost it 1 KB of spills a thread.)
template <class T, bool UPDATE, bool ADVANCE, int V, int K, class F>
__device__ __forceinline__ void ortho_for_u(const OrthoParams& p, int64_t base, int first, int step, int end, F f) {
  const bool need_g = !UPDATE || ADVANCE || p.nesterov;
  const T* g = (const T*)p.g + base;
  float* M = p.momentum + base;
#pragma unroll 1
  for (int e0 = first; e0 < end; e0 += K * step) {
    float u[K][V], old[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int e = e0 + k * step;
      if (e < end) {
        if (need_g) load_values<V>(g + e, u[k]);
        if (UPDATE) load_values<V>(M + e, old[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int e = e0 + k * step;
      if (e < end) {
        if (UPDATE) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float h = need_g ? __fmul_rn(u[k][v], p.one_minus_beta) : 0.0f;
            if (ADVANCE) old[k][v] = __fadd_rn(__fmul_rn(old[k][v], p.beta), h);
            u[k][v] = p.nesterov ? __fadd_rn(h, __fmul_rn(old[k][v], p.beta)) : old[k][v];
          }
          if (ADVANCE) store_values<V>(M + e, old[k]);
        }
        f(e, u[k]);
      }
    }
  }
}

// Directions o(position, values) written out at first, first + step, ... below `end`:
// to out, or along them into the parameter.
template <class T, bool UPDATE, int V, int K, class F>
__device__ __forceinline__ void ortho_for_out(const OrthoParams& p, int64_t base, int first, int step, int end, F o) {
  float* q = p.param + base;
  T* out = (T*)p.out + base;
#pragma unroll 1
  for (int e0 = first; e0 < end; e0 += K * step) {
    float old[K][V];
    if (UPDATE) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (e0 + k * step < end) load_values<V>(q + e0 + k * step, old[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int e = e0 + k * step;
      if (e < end) {
        float d[V];
        o(e, d);
        if (UPDATE) {
#pragma unroll
          for (int v = 0; v < V; ++v) d[v] = __fmaf_rn(-p.alpha, d[v], __fmul_rn(old[k][v], p.keep));
          store_values<V>(q + e, d);
        } else {
          store_values<V>(out + e, d);
        }
      }
    }
  }
}

// f(type tag, is an update) for a call's types
template <class F>
inline auto ortho_dispatch(const OrthoParams& p, F f) {
  if (p.momentum) {
    if (p.g_type == kValueF32) return f(float(), std::true_type());
    if (p.g_type == kValueBf16) return f(__nv_bfloat16(), std::true_type());
    return f(__half(), std::true_type());
  }
  if (p.g_type == kValueF32) return f(float(), std::false_type());
  if (p.g_type == kValueBf16) return f(__nv_bfloat16(), std::false_type());
  return f(__half(), std::false_type());
}

// old: the parameter there, where there is one
__device__ __forceinline__ void ortho_store(const OrthoParams& p, int64_t at, float o, float old) {
  if (p.param) {
    p.param[at] = __fmaf_rn(-p.alpha, o, __fmul_rn(old, p.keep));
  } else if (p.g_type == kValueF32) {
    ((float*)p.out)[at] = o;
  } else if (p.g_type == kValueBf16) {
    ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(o);
  } else {
    ((__half*)p.out)[at] = __float2half_rn(o);
  }
}

__device__ __forceinline__ void ortho_store(const OrthoParams& p, int64_t at, float o) {
  ortho_store(p, at, o, p.param ? p.param[at] : 0.0f);
}

}  // namespace blitz
