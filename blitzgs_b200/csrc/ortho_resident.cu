// Orthogonalisation of matrices that one block holds from the first step to
// the last (short side <= 128, long side <= 256; see ortho.cu for the formula
// and the two f16 terms).  X lives in shared memory as swizzled tiles of 64
// columns, which serve the tensor cores three ways without being moved: as both
// operands of X X^T (k along a row) and as the right operand of B X (n along a row);
// A, and then B in its place, beside it.  A step is three products issued by
// one thread, each followed by all warps turning the accumulators into f16
// terms; no launch, no grid-wide barrier and no traffic beyond shared memory.  Bound by the
// latency of that chain: what a block cannot overlap, the other blocks of
// the SM do (three at most: every matrix has tiles of 128 rows, 66 KB at least).
//
// One of 128 x 256 in 32 bits takes 52 us, 9 us a step: about 8k cycles of products and 7k of
// conversions; 1000 of 64 x 64 take 99 us.
//
// Within a product the small terms (high * low, low * high) come first: the
// accumulator drops bits below its last one at every addition, so the sum
// should be large for as few of them as possible.
#include <algorithm>

#include "ortho.cuh"
#include "tcgen05.cuh"

namespace blitz {

namespace {

constexpr int kGroup = 128 * 128;  // bytes of 64 columns of one term: 128 rows of 128 bytes

struct Layout {
  int np, mp;           // n and m in whole steps of 16
  int x_term, a_term;   // bytes of one term of X, of A
  int columns;          // tensor memory
  int bytes;
};

__host__ __device__ inline Layout layout_of(int n, int m) {
  Layout l;
  l.np = (n + 15) / 16 * 16;
  l.mp = (m + 15) / 16 * 16;
  l.x_term = (l.mp + 63) / 64 * kGroup;
  l.a_term = (l.np + 63) / 64 * kGroup;
  l.bytes = 2 * (l.x_term + l.a_term) + 1024;
  const int most = l.np > l.mp ? l.np : l.mp;
  l.columns = most <= 32 ? 32 : most <= 64 ? 64 : most <= 128 ? 128 : 256;
  return l;
}

// byte offset of 8 columns from `col` (a multiple of 8) of a row, in a term
__device__ __forceinline__ int chunk_at(int row, int col) {
  return (col >> 6) * kGroup + row * 128 + ((((col & 63) >> 3) ^ (row & 7)) << 4);
}

// row stride, in floats, of the 32-bit direction: whole float4s, rows 4 banks apart
__host__ __device__ inline int stage_stride(int m) { return (m + 31) / 32 * 32 + 4; }

struct Product {
  uint32_t a, b;         // first terms
  uint32_t a_term, b_term;
  bool two_a, two_b;
  int k;                 // steps of 16
  int n;
  bool b_mn;             // b lies with n along a row
};

__device__ __forceinline__ void issue(const Product& q, uint32_t on, uint32_t d, uint32_t bar) {
  const uint32_t idesc = instruction_desc(q.n, q.b_mn);
  // 16 of k further, in units of 16 bytes: 32 bytes along a row and after four of those the next
  // 64 columns, or 16 rows
  const uint32_t b_step = q.b_mn ? 128 : 2, b_four = q.b_mn ? 512 : kGroup >> 4;
  uint32_t add = 0;
#pragma unroll
  for (int t = 0; t < 3; ++t) {
    // low * high, high * low, high * high
    if (t == 0 && !q.two_a || t == 1 && !q.two_b) continue;
    uint32_t a = smem_desc(q.a + (t == 0 ? q.a_term : 0), 16);
    uint32_t b = smem_desc(q.b + (t == 1 ? q.b_term : 0), q.b_mn ? kGroup : 16);
    int k = q.k;
    for (; k >= 4; k -= 4, a += kGroup >> 4, b += b_four) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk, add = 1) mma(on, d, a + 2 * kk, b + b_step * kk, idesc, add);
    }
    for (; k > 0; --k, a += 2, b += b_step, add = 1) mma(on, d, a, b, idesc, add);
  }
  mma_commit(on, bar);
}

// position e of a matrix stored in rows of `inner`, without a division a step
struct Walk {
  int o, k, by_o, by_k, inner;
  __device__ __forceinline__ Walk(int first, int step, int inner_)
      : o(first / inner_), k(first - o * inner_), by_o(step / inner_), by_k(step - by_o * inner_), inner(inner_) {}
  __device__ __forceinline__ void next() {
    o += by_o;
    k += by_k;
    if (k >= inner) {
      k -= inner;
      ++o;
    }
  }
};

template <class T, bool UPDATE, int THREADS, int V>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) resident_kernel(OrthoParams p) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bar_mem;
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  __shared__ double sums[THREADS / 32];
  __shared__ OrthoInfo scaling;
  volatile int* dead = &dead_flag;
  uint8_t* X = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int n = (int)p.n, m = (int)p.m, tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const Layout l = layout_of(n, m);
  uint8_t* A = X + 2 * l.x_term;
  const uint32_t xs = smem_addr(X), as = smem_addr(A), bar = smem_addr(&bar_mem);
  const bool two_in = ortho_two_in(p), wide = p.sj == 1;
  if (tid == 0) {
    dead_flag = 0;
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(&tmem_base, l.columns);
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = tmem_base, on = elected();
  const int row = (warp & 3) * 32 + lane;
  const uint32_t tmem_rows = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  uint32_t parity = 0;
  const int inner = wide ? m : n, total = n * m;

  for (int64_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const int64_t base = b * p.n * p.m;
    {
      for (int e = tid; e < l.x_term / 8; e += THREADS) ((uint4*)X)[e] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      // u's 32 bits lie where its two terms will: the upper half as the high one
      double sq = 0.0;
      Walk at(tid * V, THREADS * V, inner);
      ortho_for_u<T, UPDATE, true, V, 16 / V>(
          p, base, tid * V, THREADS * V, total, [&](int, const float(&u)[V]) {
#pragma unroll
            for (int v = 0; v < V; ++v) sq += (double)u[v] * (double)u[v];
            if (wide) {
              uint8_t* dst = X + chunk_at(at.o, at.k & ~7) + (at.k & 7) * 2;
              if constexpr (V == 4) {
                const uint32_t w[4] = {__float_as_uint(u[0]), __float_as_uint(u[1]), __float_as_uint(u[2]),
                                       __float_as_uint(u[3])};
                *(uint2*)dst = make_uint2(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632));
                *(uint2*)(dst + l.x_term) =
                    make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
              } else {
                *(uint16_t*)dst = (uint16_t)(__float_as_uint(u[0]) >> 16);
                *(uint16_t*)(dst + l.x_term) = (uint16_t)__float_as_uint(u[0]);
              }
            } else {
#pragma unroll
              for (int v = 0; v < V; ++v) {
                uint8_t* dst = X + chunk_at(at.k + v, at.o & ~7) + (at.o & 7) * 2;
                *(uint16_t*)dst = (uint16_t)(__float_as_uint(u[v]) >> 16);
                *(uint16_t*)(dst + l.x_term) = (uint16_t)__float_as_uint(u[v]);
              }
            }
            at.next();
          });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
      if (lane == 0) sums[warp] = sq;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < THREADS / 32; ++w) sq += sums[w];
        ortho_scaling(sqrt(sq), p, &scaling);
      }
      __syncthreads();
      const float2 up = scaling.up;
      // whole rows of 128 bytes, so the swizzle does not matter
      for (int e = tid; e < l.x_term / 16; e += THREADS) {
        uint4* hi = (uint4*)X + e;
        uint4* lo = (uint4*)(X + l.x_term) + e;
        const uint4 h = *hi, w = *lo;
        const uint32_t hs[4] = {h.x, h.y, h.z, h.w}, ls[4] = {w.x, w.y, w.z, w.w};
        float x[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = __uint_as_float(__byte_perm(ls[k], hs[k], 0x5410)) * up.x * up.y;
          x[2 * k + 1] = __uint_as_float(__byte_perm(ls[k], hs[k], 0x7632)) * up.x * up.y;
        }
        uint4 nh, nl;
        split8(x, nh, nl);
        *hi = nh;
        *lo = nl;
      }
    }
    fence_async_shared();
    __syncthreads();

#pragma unroll 1
    for (int s = 0; s < p.steps; ++s) {
      const bool two_x = s > 0 || two_in;
      const bool last = s + 1 == p.steps;
      const OrthoFactors by = ortho_factors(scaling, s, last);
#pragma unroll 1
      for (int which = 0; which < 3; ++which) {
        if (warp == 0) {
          tcgen05_after_sync();
          Product q;
          q.a = which == 0 ? xs : as;
          q.b = which == 1 ? as : xs;
          q.a_term = which == 0 ? l.x_term : l.a_term;
          q.b_term = which == 1 ? l.a_term : l.x_term;
          q.two_a = which == 0 ? two_x : true;
          q.two_b = which == 1 ? true : two_x;
          q.k = (which == 0 ? l.mp : l.np) / 16;
          q.n = which == 2 ? l.mp : l.np;
          q.b_mn = which == 2;
          issue(q, on, tmem, bar);
        }
        mbar_wait(bar, parity, dead, p.wait_limit);
        parity ^= 1;
        tcgen05_after_sync();
        __syncwarp();
        const int width = which == 2 ? l.mp : l.np;
#pragma unroll 1
        for (int c = (warp >> 2) * 32; c < width; c += THREADS / 4) {
          float v[32];
          tmem_load32(tmem_rows + c, v);
          if (which == 2 && last) {
            // the direction in 32 bits over X, in the order of the matrix's own memory
            const float f = by.next;
            if (row < n) {
              if (wide) {
                float* dst = (float*)X + row * stage_stride(m) + c;
#pragma unroll
                for (int k = 0; k < 32; k += 4)
                  *(float4*)(dst + k) = make_float4(v[k] * f, v[k + 1] * f, v[k + 2] * f, v[k + 3] * f);
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  if (c + k < m) ((float*)X)[(c + k) * n + row] = v[k] * f;
              }
            }
            continue;
          }
          // columns past np / mp hold what was left there; nothing reads their terms
          uint8_t* dst = which == 2 ? X : A;
          const int term = which == 2 ? l.x_term : l.a_term;
          const float f = which == 0 ? by.x * by.x * kScaleA : which == 1 ? p.c * (kScaleB / (kScaleA * kScaleA))
                                                                     : by.next;
          const float fb = p.b * (kScaleB / kScaleA);
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            const int at = chunk_at(row, c + k);
            if (which == 1) {
              // B = a I + b A + c A^2 in A's place: this thread alone reads and writes here
              const uint4 h4 = *(const uint4*)(dst + at), l4 = *(const uint4*)(dst + term + at);
              const uint32_t hs[4] = {h4.x, h4.y, h4.z, h4.w}, ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x = join2(hs[e], ls[e]);
                v[k + 2 * e] = fmaf(f, v[k + 2 * e], fb * x.x);
                v[k + 2 * e + 1] = fmaf(f, v[k + 2 * e + 1], fb * x.y);
              }
              if (c == (warp & 3) * 32) {
                // these 32 columns cross the diagonal in this warp's rows
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k + e] += k + e == lane ? p.a * kScaleB : 0.0f;
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[k + e] *= f;
            }
            uint4 hi, lo;
            split8(v + k, hi, lo);
            *(uint4*)(dst + at) = hi;
            *(uint4*)(dst + term + at) = lo;
          }
        }
        tcgen05_before_sync();
        fence_async_shared();
        __syncthreads();
      }
    }
    {
      const int stride = wide ? stage_stride(m) : n;
      // after the step's last barrier every thread sees the same
      const bool lost = *dead != 0;
      Walk at(tid * V, THREADS * V, inner);
      ortho_for_out<T, UPDATE, V, 16 / V>(p, base, tid * V, THREADS * V, total, [&](int, float(&d)[V]) {
        load_values<V>((const float*)X + at.o * stride + at.k, d);
        if (lost)
#pragma unroll
          for (int v = 0; v < V; ++v) d[v] = __int_as_float(0x7fffffff);
        at.next();
      });
    }
    __syncthreads();
  }
  if (dead_flag) {
    // products of this block that are still in flight end within this time
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
  }
  __syncthreads();
  if (warp == 0) tmem_free(tmem, l.columns);
}

template <class T, bool UPDATE, int THREADS, int V>
int start(const OrthoParams& p, cudaStream_t st) {
  const auto kernel = resident_kernel<T, UPDATE, THREADS, V>;
  const int bytes = layout_of((int)p.n, (int)p.m).bytes;
  // one value for every size: calls of other threads set the same
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           layout_of(128, 256).bytes))
    return (int)e;
  kernel<<<(unsigned)std::min<int64_t>(p.batch, 1 << 20), THREADS, bytes, st>>>(p);
  return (int)cudaGetLastError();
}

}  // namespace

bool ortho_resident_fits(const OrthoParams& p) { return p.n <= 128 && p.m <= 256; }

int launch_ortho_resident(const OrthoParams& p, cudaStream_t st) {
  const bool four = ortho_by_four(p);
  return ortho_dispatch(p, [&](auto type, auto update) {
    using T = decltype(type);
    constexpr bool kUpdate = decltype(update)::value;
    if (p.n * p.m <= 4096) return four ? start<T, kUpdate, 128, 4>(p, st) : start<T, kUpdate, 128, 1>(p, st);
    return four ? start<T, kUpdate, 512, 4>(p, st) : start<T, kUpdate, 512, 1>(p, st);
  });
}

}  // namespace blitz
