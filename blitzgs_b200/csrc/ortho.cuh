// Reading an update and writing its direction, shared by the orthogonalisation kernels.
#pragma once
#include "kernels.h"
#include "ortho.h"
#include "quant.cuh"

namespace blitz {

__device__ __forceinline__ float ortho_g(const OrthoParams& p, int64_t at) {
  if (p.g_type == kValueF32) return ((const float*)p.g)[at];
  if (p.g_type == kValueBf16) return __bfloat162float(((const __nv_bfloat16*)p.g)[at]);
  return __half2float(((const __half*)p.g)[at]);
}

// the matrix to be orthogonalised at `at`; the momentum is advanced where this
// is its first reading (`advance`), else taken as it stands
template <bool ADVANCE>
__device__ __forceinline__ float ortho_u(const OrthoParams& p, int64_t at) {
  if (!p.momentum) return ortho_g(p, at);
  float g = 0.0f;
  if (ADVANCE || p.nesterov) g = __fmul_rn(ortho_g(p, at), p.one_minus_beta);
  float M = p.momentum[at];
  if (ADVANCE) {
    M = __fadd_rn(__fmul_rn(M, p.beta), g);
    p.momentum[at] = M;
  }
  return p.nesterov ? __fadd_rn(g, __fmul_rn(M, p.beta)) : M;
}

__device__ __forceinline__ void ortho_store(const OrthoParams& p, int64_t at, float o) {
  if (p.param) {
    p.param[at] = __fmaf_rn(-p.alpha, o, __fmul_rn(p.param[at], p.keep));
  } else if (p.g_type == kValueF32) {
    ((float*)p.out)[at] = o;
  } else if (p.g_type == kValueBf16) {
    ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(o);
  } else {
    ((__half*)p.out)[at] = __float2half_rn(o);
  }
}

}  // namespace blitz
