// Orthogonalisation of matrices by Newton-Schulz products.  With X_0 = u /
// (|u|_F + eps), n <= m rows and columns, each of `steps` steps is
//   A = X X^T;   B = a I + b A + c A^2;   X <- B X
// an odd polynomial of X's singular values that drives them towards 1 and
// leaves its singular vectors alone.  3 n^2 m + n^3 multiply-add pairs' worth
// of operations a step once A and B, which are symmetric, are computed on and
// below the diagonal only.
//
// The products run on the fifth-generation tensor cores (tcgen05.mma, f16
// inputs, 32-bit accumulators in tensor memory).  One f16 has 11 bits, and a
// step multiplies what lies in X's weak directions by up to a = 3.44, five
// steps by 485: rounding X to f16 once a step would leave the direction 1e-3
// to 1e-2 off.  So X, A and B are kept as two f16 terms (high + low, 22 bits)
// and a product is high*high + high*low + low*high, which leaves about 4e-6.
// bf16 terms would need three for that.  16-bit inputs are exact in one term, so step 0
// reads one of X; every other operand has two, whatever type the result is rounded to.
// Everything is scaled by powers of two into
// f16's range: |X_ij| <= 1.9 by 2^14 (by more where X is tiny throughout, see OrthoInfo),
// |A_ij| <= 3.7 by 2^14, |B_ij| < 7.9 by 2^13
// (the caller's coefficients are checked to keep to that).
//
// Which kernel runs goes by size: registers or one block's shared memory (ortho_small.cu), one
// block's shared and tensor memory (ortho_resident.cu), or, below and in ortho_split.cu,
// the whole grid. There `sum_kernel` advances the momentum and adds up squares (in 64 bits, in
// a fixed order), `layout_kernel` writes X_0's terms, and one persistent cooperative
// kernel runs all 3 * steps products with a grid-wide barrier between them, so a step
// costs no launch.  In it two warps copy tiles of 64 columns by TMA (128-byte swizzle), two
// issue the products, and eight warps move finished tiles out of tensor memory.
//
// Every wait gives up after two seconds (see wait_limit).  In `resident_kernel` that block's matrix
// is then NaN.  Over the grid the other blocks learn of it at the next barrier, and
// `lost_kernel`, which runs when all of them have ended and so after all that they wrote, makes all
// outputs of the call NaN.  (In a call of 124 us its launch does not show.)
#include <algorithm>

#include "ortho_grid.cuh"

namespace blitz {

namespace {

constexpr int kMaxParts = 256;

// the momentum advanced, and the squares of u added up: block (x, b) takes part x of
// matrix b
template <class T, bool UPDATE, int V>
__global__ void __launch_bounds__(256) sum_kernel(OrthoParams o, double* parts, unsigned* barrier, int n_parts) {
  __shared__ double sums[8];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *barrier = 0u;
  const int size = (int)(o.n * o.m), per = ((size + n_parts - 1) / n_parts + 3) / 4 * 4;
  for (int64_t b = blockIdx.y; b < o.batch; b += gridDim.y) {
    const int lo = (int)min((int64_t)size, (int64_t)blockIdx.x * per), hi = (int)min((int64_t)size, (int64_t)lo + per);
    double sq = 0.0;
    ortho_for_u<T, UPDATE, true, V, 16 / V>(o, b * size, lo + threadIdx.x * V, 256 * V, hi,
                                            [&](int, const float(&u)[V]) {
#pragma unroll
                                              for (int v = 0; v < V; ++v) sq += (double)u[v] * (double)u[v];
                                            });
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, k);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sq;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) sq += sums[w];
      parts[b * n_parts + blockIdx.x] = sq;
    }
  }
}

struct LayoutParams {
  OrthoParams o;
  __half* x;
  const double* parts;
  OrthoInfo* info;
  int n_parts, ldm, two_in;
};

// X_0's terms, scaled: one 64 x 64 tile a block (through shared memory where X is the
// transpose of what is stored)
template <class T, bool UPDATE, int V>
__global__ void __launch_bounds__(256) layout_kernel(LayoutParams p) {
  __shared__ float tile[64 * 65];
  __shared__ float2 up_shared;
  const OrthoParams& o = p.o;
  const int n = (int)o.n, m = (int)o.m, tid = threadIdx.x;
  const int tj = p.ldm / 64, per = (n + 63) / 64 * tj;
  const int64_t b = blockIdx.x / per, base = b * o.n * o.m;
  const int r = blockIdx.x % per, i0 = r / tj * 64, j0 = r % tj * 64;
  const bool wide = o.sj == 1;
  // element (i0 + x, j0 + y) of X: 4 values along the order of the memory, 4 times
  const int inner = wide ? m : n, outer = wide ? n : m, in0 = wide ? j0 : i0, out0 = wide ? i0 : j0;
  const int q = (tid & 15) * 4;
  float u[4][4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int x = out0 + (tid >> 4) + 16 * k, left = x < outer ? inner - (in0 + q) : 0;
    const int64_t at = base + (int64_t)x * inner + in0 + q;
    if constexpr (V == 4) {
      if (left > 0) {
        ortho_for_u<T, UPDATE, false, 4, 1>(o, at, 0, 4, 4, [&](int, const float(&v)[4]) {
#pragma unroll
          for (int e = 0; e < 4; ++e) u[k][e] = v[e];
        });
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[k][e] = 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[k][e] = 0.0f;
        if (e < left)
          ortho_for_u<T, UPDATE, false, 1, 1>(o, at + e, 0, 1, 1, [&](int, const float(&v)[1]) { u[k][e] = v[0]; });
      }
    }
  }
  if (tid < 32) {
    double sq = 0.0;
    for (int k = tid; k < p.n_parts; k += 32) sq += p.parts[b * p.n_parts + k];
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, k);
    if (tid == 0) {
      up_shared = ortho_up(sqrt(sq));
      if (r == 0) ortho_scaling(sqrt(sq), o, p.info + b);
    }
  }
  if (!wide) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[(q + e) * 65 + (tid >> 4) + 16 * k] = u[k][e];
  }
  __syncthreads();
  const float2 up = up_shared;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int x = (tid >> 4) + 16 * k;
    if (i0 + x >= n) continue;
    if (!wide) {
#pragma unroll
      for (int e = 0; e < 4; ++e) u[k][e] = tile[x * 65 + q + e];
    }
    uint2 hi, lo;
    hi.x = split2(u[k][0] * up.x * up.y, u[k][1] * up.x * up.y, lo.x);
    hi.y = split2(u[k][2] * up.x * up.y, u[k][3] * up.x * up.y, lo.y);
    __half* dst = p.x + ((2 * b) * n + i0 + x) * (int64_t)p.ldm + j0 + q;
    *(uint2*)dst = hi;
    if (p.two_in) *(uint2*)(dst + (int64_t)n * p.ldm) = lo;
  }
}

// NaN for every output where a block of the call gave up
__global__ void __launch_bounds__(512) lost_kernel(OrthoParams o, const unsigned* barrier) {
  if (*barrier < kGaveUp) return;
  const int64_t size = o.batch * o.n * o.m;
  for (int64_t e = (int64_t)blockIdx.x * 512 + threadIdx.x; e < size; e += (int64_t)gridDim.x * 512)
    ortho_store(o, e, __int_as_float(0x7fffffff));
}

template <class T, bool UPDATE, int V>
int start_input(const OrthoGrid& p, cudaStream_t st) {
  const OrthoParams& o = p.o;
  sum_kernel<T, UPDATE, V><<<dim3((unsigned)p.n_parts, (unsigned)std::min<int64_t>(o.batch, 65535)), 256, 0, st>>>(
      o, p.parts, p.barrier, p.n_parts);
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  const LayoutParams l{o, p.x[0], p.parts, p.info, p.n_parts, p.ldm, p.two_in};
  layout_kernel<T, UPDATE, V><<<(unsigned)(o.batch * ((o.n + 63) / 64) * (p.ldm / 64)), 256, 0, st>>>(l);
  return (int)cudaGetLastError();
}

struct Plan {
  int ldm, ldn, n_parts;
  size_t x, a, parts, info, total;  // bytes of one X, of A, ...
};

Plan plan_of(const OrthoParams& p) {
  Plan q;
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  q.ldm = (int)((p.m + 63) / 64 * 64);
  q.ldn = (int)((p.n + 63) / 64 * 64);
  q.n_parts = (int)std::min<int64_t>(kMaxParts, (p.n * p.m + 4095) / 4096);
  q.x = up((size_t)2 * p.batch * p.n * q.ldm * sizeof(__half));
  q.a = up((size_t)2 * p.batch * p.n * q.ldn * sizeof(__half));
  q.parts = up((size_t)p.batch * q.n_parts * sizeof(double));
  q.info = up((size_t)p.batch * sizeof(OrthoInfo));
  q.total = 2 * q.x + 2 * q.a + q.parts + q.info + 256;
  return q;
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// [2 * batch][rows][cols] halves, ld apart; boxes of 64 x 64, zeros outside
int make_map(CUtensorMap* map, void* base, int64_t cols, int64_t rows, int64_t ld, int64_t batch) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)(2 * batch)};
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)(ld * rows) * 2};
  const cuuint32_t box[3] = {64, 64, 1}, one[3] = {1, 1, 1};
  EncodeFn fn = encode_fn();
  if (!fn) return (int)cudaErrorNotSupported;
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

}  // namespace

size_t ortho_workspace_bytes(const OrthoParams& p) {
  return ortho_small_fits(p) || ortho_resident_fits(p) ? 0 : plan_of(p).total;
}

int launch_ortho(const OrthoParams& o, void* workspace, cudaStream_t st) {
  if (ortho_small_fits(o)) return launch_ortho_small(o, st);
  if (ortho_resident_fits(o)) return launch_ortho_resident(o, st);
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return (int)e;
  const Plan q = plan_of(o);
  OrthoGrid p;
  p.o = o;
  uint8_t* w = (uint8_t*)workspace;
  p.barrier = (unsigned*)w;
  w += 256;
  p.x[0] = (__half*)w;
  p.x[1] = (__half*)(w + q.x);
  p.a = (__half*)(w + 2 * q.x);
  p.b = (__half*)(w + 2 * q.x + q.a);
  p.parts = (double*)(w + 2 * q.x + 2 * q.a);
  p.info = (OrthoInfo*)(w + 2 * q.x + 2 * q.a + q.parts);
  p.n_parts = q.n_parts;
  p.ldm = q.ldm;
  p.ldn = q.ldn;
  p.two_in = ortho_two_in(o);
  p.four = ortho_by_four(o);
  for (int i = 0; i < 2; ++i)
    if (int rc = make_map(&p.map_x[i], p.x[i], o.m, o.n, q.ldm, o.batch)) return rc;
  if (int rc = make_map(&p.map_a, p.a, o.n, o.n, q.ldn, o.batch)) return rc;
  if (int rc = make_map(&p.map_b, p.b, o.n, o.n, q.ldn, o.batch)) return rc;
  // what can fail does so before the first kernel advances the momentum
  const int split = ortho_split_for(p, sms);
  if (int rc = ortho_split_ready(split)) return rc;
  if (int rc = ortho_dispatch(o, [&](auto type, auto update) {
        using T = decltype(type);
        constexpr bool kUpdate = decltype(update)::value;
        return p.four ? start_input<T, kUpdate, 4>(p, st) : start_input<T, kUpdate, 1>(p, st);
      }))
    return rc;
  if (int rc = launch_ortho_split(p, split, st)) return rc;
  lost_kernel<<<(unsigned)sms, 512, 0, st>>>(o, p.barrier);
  return (int)cudaGetLastError();
}

}  // namespace blitz
