// Parameters shared by the orthogonalisation's host side and kernels (ortho.cu, ortho_small.cu).
#pragma once
#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace blitz {

// One call: batch matrices [rows, cols] (contiguous, back to back).  The
// products run on the short side: X is [n, m] with n = min, m = max, and
// element (i, j) of X lies at i * si + j * sj of its matrix.
struct OrthoParams {
  const void* g;      // gradient / input
  int g_type;         // kValueF32 / kValueBf16 / kValueF16
  float* momentum;    // update only
  float* param;       // update only
  void* out;          // orthogonalize only, of g's type
  int64_t batch, n, m, si, sj;
  int steps;
  float a, b, c, eps;
  float beta, one_minus_beta;
  int nesterov;
  float keep, alpha;  // param = param * keep - alpha * direction
  long long wait_limit;  // cycles after which a wait within a kernel gives up
};

constexpr int kMostSteps = 64;

// about two seconds of the SM's clock
constexpr long long kOrthoWaitLimit = 4000000000ll;

size_t ortho_workspace_bytes(const OrthoParams& p);
int launch_ortho(const OrthoParams& p, void* workspace, cudaStream_t st);
// ortho_small.cu: matrices that one thread group or one block holds
bool ortho_small_fits(const OrthoParams& p);
int launch_ortho_small(const OrthoParams& p, cudaStream_t st);
// ortho_resident.cu: matrices that one block holds, on the tensor cores
bool ortho_resident_fits(const OrthoParams& p);
int launch_ortho_resident(const OrthoParams& p, cudaStream_t st);

}  // namespace blitz
