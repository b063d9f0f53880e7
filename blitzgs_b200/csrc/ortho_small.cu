// Orthogonalisation of small matrices (see ortho.cu for the formula), in 32
// bits from end to end.
//
// thin: short side n <= 4.  LANES neighbouring lanes hold one matrix in
// registers, each its own columns; the n x n products are a few registers and
// one shuffle reduction a step.  Bound by reading and writing the matrices.
//
// block: one block holds one matrix in shared memory.  The iteration never
// leaves it: A = X X^T and B = a I + b A + c A^2 by 4 x 4 register tiles of the
// upper half (both are symmetric), X <- B X in place, a set of whole columns
// at a time.  Bound by the FP32 pipe and shared-memory reads (32 B a lane for
// 64 multiply-adds).
#include <algorithm>

#include "ortho.cuh"

namespace blitz {

namespace {

constexpr int kThinCols = 16;  // columns a lane holds at most
constexpr size_t kSharedMost = 200 * 1024;

// A block's matrices lie one after the other in memory and in shared memory, where they are
// copied whole (threads reading their own matrix from global memory: 77 us for 200000 of
// 15 x 3, of which the arithmetic is a tenth; copied a word at a time 45 us).  `gap`: odd
// distance between matrices there, so that neighbouring lanes read different banks.  V = 4
// where a matrix has an odd number of values: both sides are then alike, and 16 bytes go at a time.
template <class T, bool UPDATE, int N, int LANES, int COLS, int V>
__global__ void __launch_bounds__(128) thin_kernel(OrthoParams p, int gap) {
  extern __shared__ __align__(16) float smem[];
  constexpr int kMatrices = 128 / LANES;
  const int64_t b0 = (int64_t)blockIdx.x * kMatrices;
  const int here = (int)min((int64_t)kMatrices, p.batch - b0), mine = threadIdx.x / LANES;
  const int lane = threadIdx.x & (LANES - 1), m = (int)p.m, size = N * m, total = here * size;
  const int64_t base = b0 * size;
  // position e of the block's values -> shared memory, without a division a step
  const int by_o = 128 / size, by_k = 128 - by_o * size;
  if constexpr (V == 4) {
    const int most = total & ~3;
    ortho_for_u<T, UPDATE, true, 4, 4>(p, base, threadIdx.x * 4, 512, most, [&](int e, const float(&u)[4]) {
      *(float4*)(smem + e) = make_float4(u[0], u[1], u[2], u[3]);
    });
    ortho_for_u<T, UPDATE, true, 1, 1>(p, base, most + threadIdx.x, 128, total,
                                       [&](int e, const float(&u)[1]) { smem[e] = u[0]; });
  } else {
    int o = threadIdx.x / size, k = threadIdx.x - o * size;
    ortho_for_u<T, UPDATE, true, 1, 8>(p, base, threadIdx.x, 128, total, [&](int, const float(&u)[1]) {
      smem[o * gap + k] = u[0];
      o += by_o;
      k += by_k;
      if (k >= size) k -= size, ++o;
    });
  }
  __syncthreads();
  const int si = (int)p.si, sj = (int)p.sj;
  float* X = smem + mine * gap;
  float x[N][COLS];
  double sq = 0.0;
#pragma unroll
  for (int k = 0; k < COLS; ++k) {
    const int j = lane + k * LANES;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i][k] = mine < here && j < m ? X[i * si + j * sj] : 0.0f;
      sq += (double)x[i][k] * (double)x[i][k];
    }
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
  const float2 scale = ortho_inverse(sqrt(sq), p.eps);
#pragma unroll
  for (int k = 0; k < COLS; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i][k] *= scale.y, x[i][k] *= scale.x;
  for (int s = 0; s < p.steps; ++s) {
    float A[N][N], B[N][N];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = i; j < N; ++j) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < COLS; ++k) t = fmaf(x[i][k], x[j][k], t);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        A[i][j] = A[j][i] = t;
      }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = i; j < N; ++j) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < N; ++k) t = fmaf(A[i][k], A[k][j], t);
        B[i][j] = B[j][i] = fmaf(p.c, t, p.b * A[i][j]);
      }
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      float y[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float t = 0.0f;
#pragma unroll
        for (int q = 0; q < N; ++q) t = fmaf(B[i][q], x[q][k], t);
        y[i] = fmaf(p.a, x[i][k], t);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) x[i][k] = y[i];
    }
  }
  if (mine < here) {
#pragma unroll
    for (int k = 0; k < COLS; ++k) {
      const int j = lane + k * LANES;
      if (j < m)
#pragma unroll
        for (int i = 0; i < N; ++i) X[i * si + j * sj] = x[i][k];
    }
  }
  __syncthreads();
  if constexpr (V == 4) {
    const int most = total & ~3;
    ortho_for_out<T, UPDATE, 4, 4>(p, base, threadIdx.x * 4, 512, most,
                                   [&](int e, float(&d)[4]) { load_values<4>(smem + e, d); });
    ortho_for_out<T, UPDATE, 1, 1>(p, base, most + threadIdx.x, 128, total, [&](int e, float(&d)[1]) { d[0] = smem[e]; });
  } else {
    int o = threadIdx.x / size, k = threadIdx.x - o * size;
    ortho_for_out<T, UPDATE, 1, 8>(p, base, threadIdx.x, 128, total, [&](int, float(&d)[1]) {
      d[0] = smem[o * gap + k];
      o += by_o;
      k += by_k;
      if (k >= size) k -= size, ++o;
    });
  }
}

// shared-memory row stride of k values: whole float4s, rows 4 banks apart
__host__ __device__ inline int row_stride(int k) { return (k + 31) / 32 * 32 + 4; }

struct BlockLayout {
  int np, mp, ldx, lda;
  size_t bytes;
};
__host__ __device__ inline BlockLayout block_layout(int n, int m) {
  BlockLayout l;
  l.np = (n + 3) / 4 * 4;
  l.mp = (m + 3) / 4 * 4;
  l.ldx = row_stride(l.mp);
  l.lda = row_stride(l.np);
  l.bytes = sizeof(float) * ((size_t)l.np * l.ldx + 2 * (size_t)l.np * l.lda);
  return l;
}

// R = P P^T over k columns for 4 x 4 interleaved tiles of the upper half (rows
// t, t + q, t + 2 q, t + 3 q: neighbouring lanes read neighbouring rows), then
// R = f(R, i, j) stored on both sides
template <int THREADS, class F>
__device__ __forceinline__ void symmetric_product(const float* P, int ldp, int kp, float* R, int ldr, int q, F f) {
  const int tiles = q * (q + 1) / 2;
  for (int t = threadIdx.x; t < tiles; t += THREADS) {
    int ti = 0, r = t;
    while (r >= q - ti) r -= q - ti++;
    const int tj = ti + r;
    float acc[4][4] = {};
    for (int k = 0; k < kp; k += 4) {
      float4 u[4], v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[e] = *(const float4*)(P + (ti + e * q) * ldp + k);
        v[e] = *(const float4*)(P + (tj + e * q) * ldp + k);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          acc[e][h] = fmaf(u[e].x, v[h].x, acc[e][h]);
          acc[e][h] = fmaf(u[e].y, v[h].y, acc[e][h]);
          acc[e][h] = fmaf(u[e].z, v[h].z, acc[e][h]);
          acc[e][h] = fmaf(u[e].w, v[h].w, acc[e][h]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int i = ti + e * q, j = tj + h * q;
        // a diagonal tile holds both (i, j) and (j, i): the upper one is kept
        if (ti == tj && e > h) continue;
        const float x = f(acc[e][h], i, j);
        R[i * ldr + j] = x;
        R[j * ldr + i] = x;
      }
  }
}

// The same by one warp: 2 x 4 tiles of the whole product, which give all 32 lanes work on 16 x 16
// (4 x 4 tiles of its upper half would give ten).  Both halves come out the same to
// the last bit: the same products, added in the same order.
template <class F>
__device__ __forceinline__ void warp_product(const float* P, int ldp, int kp, float* R, int ldr, int np, F f) {
  const int rows = np / 2, q = np / 4;
  for (int t = threadIdx.x; t < rows * q; t += 32) {
    const int tj = t / rows, ti = t - tj * rows;
    float acc[2][4] = {};
    for (int k = 0; k < kp; k += 4) {
      float4 u[2], v[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) u[e] = *(const float4*)(P + (ti + e * rows) * ldp + k);
#pragma unroll
      for (int h = 0; h < 4; ++h) v[h] = *(const float4*)(P + (tj + h * q) * ldp + k);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          acc[e][h] = fmaf(u[e].x, v[h].x, acc[e][h]);
          acc[e][h] = fmaf(u[e].y, v[h].y, acc[e][h]);
          acc[e][h] = fmaf(u[e].z, v[h].z, acc[e][h]);
          acc[e][h] = fmaf(u[e].w, v[h].w, acc[e][h]);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int i = ti + e * rows, j = tj + h * q;
        R[i * ldr + j] = f(acc[e][h], i, j);
      }
  }
}

template <int THREADS>
__device__ __forceinline__ void block_sync() {
  if (THREADS == 32)
    __syncwarp();
  else
    __syncthreads();
}

template <class T, bool UPDATE, int THREADS>
__global__ void __launch_bounds__(THREADS) block_kernel(OrthoParams p) {
  extern __shared__ __align__(16) float smem[];
  __shared__ double sums[THREADS / 32];
  const int n = (int)p.n, m = (int)p.m, tid = threadIdx.x;
  const BlockLayout l = block_layout(n, m);
  float *X = smem, *A = X + l.np * l.ldx, *B = A + l.np * l.lda;
  const int q = l.np / 4, q4 = l.mp / 4;
  for (int64_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    const int64_t base = b * p.n * p.m;
    double sq = 0.0;
    // in the matrix's own order, whichever side is short
    const int inner = p.sj == 1 ? m : n, total = n * m;
    for (int e = tid; e < l.np * l.ldx; e += THREADS) X[e] = 0.0f;
    block_sync<THREADS>();
    ortho_for_u<T, UPDATE, true, 1, 8>(p, base, tid, THREADS, total, [&](int e, const float(&u)[1]) {
      const int o = e / inner, k = e - o * inner;
      X[p.sj == 1 ? o * l.ldx + k : k * l.ldx + o] = u[0];
      sq += (double)u[0] * (double)u[0];
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    if ((tid & 31) == 0) sums[tid >> 5] = sq;
    block_sync<THREADS>();
    sq = 0.0;
    for (int w = 0; w < THREADS / 32; ++w) sq += sums[w];
    const float2 scale = ortho_inverse(sqrt(sq), p.eps);
    for (int e = tid; e < l.np * l.ldx; e += THREADS) X[e] = X[e] * scale.y * scale.x;
    block_sync<THREADS>();
    for (int s = 0; s < p.steps; ++s) {
      const auto gram = [](float x, int, int) { return x; };
      const auto poly = [&](float x, int i, int j) { return fmaf(p.c, x, p.b * A[i * l.lda + j]); };
      if constexpr (THREADS == 32)
        warp_product(X, l.ldx, l.mp, A, l.lda, l.np, gram);
      else
        symmetric_product<THREADS>(X, l.ldx, l.mp, A, l.lda, q, gram);
      block_sync<THREADS>();
      if constexpr (THREADS == 32)
        warp_product(A, l.lda, l.np, B, l.lda, l.np, poly);
      else
        symmetric_product<THREADS>(A, l.lda, l.np, B, l.lda, q, poly);
      block_sync<THREADS>();
      // X <- a X + B X, `per` column groups of 4 at a time; a column's new values need
      // that column alone, so a set is read whole and then written in place
      constexpr int kRows = THREADS == 32 ? 2 : 4;  // of a lane's tile
      const int across = l.np / kRows, per = max(THREADS / across, 1);
      for (int c0 = 0; c0 < q4; c0 += per) {
        // n <= 16, so there is a set of columns for every row group
        const int cg = tid / across, t = tid - cg * across, col = (c0 + cg) * 4;
        const bool on = cg < per && c0 + cg < q4;
        float acc[kRows][4] = {};
        if (on) {
          for (int k = 0; k < l.np; k += 4) {
            float4 w[kRows], v[4];
#pragma unroll
            for (int e = 0; e < kRows; ++e) w[e] = *(const float4*)(B + (t + e * across) * l.lda + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *(const float4*)(X + (k + e) * l.ldx + col);
#pragma unroll
            for (int e = 0; e < kRows; ++e) {
              const float* wk = (const float*)&w[e];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                acc[e][0] = fmaf(wk[h], v[h].x, acc[e][0]);
                acc[e][1] = fmaf(wk[h], v[h].y, acc[e][1]);
                acc[e][2] = fmaf(wk[h], v[h].z, acc[e][2]);
                acc[e][3] = fmaf(wk[h], v[h].w, acc[e][3]);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < kRows; ++e) {
            const float4 x = *(const float4*)(X + (t + e * across) * l.ldx + col);
            acc[e][0] = fmaf(p.a, x.x, acc[e][0]);
            acc[e][1] = fmaf(p.a, x.y, acc[e][1]);
            acc[e][2] = fmaf(p.a, x.z, acc[e][2]);
            acc[e][3] = fmaf(p.a, x.w, acc[e][3]);
          }
        }
        block_sync<THREADS>();
        if (on)
#pragma unroll
          for (int e = 0; e < kRows; ++e)
            *(float4*)(X + (t + e * across) * l.ldx + col) = make_float4(acc[e][0], acc[e][1], acc[e][2], acc[e][3]);
      }
      block_sync<THREADS>();
    }
    ortho_for_out<T, UPDATE, 1, 8>(p, base, tid, THREADS, total, [&](int e, float(&d)[1]) {
      const int o = e / inner, k = e - o * inner;
      d[0] = X[p.sj == 1 ? o * l.ldx + k : k * l.ldx + o];
    });
    block_sync<THREADS>();
  }
}

template <int N, int LANES, int COLS>
int start_thin(const OrthoParams& p, cudaStream_t st) {
  const int gap = (int)(N * p.m) | 1;
  const unsigned blocks = (unsigned)((p.batch * LANES + 127) / 128);
  const size_t bytes = (size_t)gap * (128 / LANES) * sizeof(float);
  return ortho_dispatch(p, [&](auto type, auto update) {
    using T = decltype(type);
    constexpr bool kUpdate = decltype(update)::value;
    // a block's 128 / LANES matrices begin 16 bytes aligned where there is a multiple of 4 of them
    if (gap == N * p.m && ortho_aligned(p))
      thin_kernel<T, kUpdate, N, LANES, COLS, 4><<<blocks, 128, bytes, st>>>(p, gap);
    else
      thin_kernel<T, kUpdate, N, LANES, COLS, 1><<<blocks, 128, bytes, st>>>(p, gap);
    return (int)cudaGetLastError();
  });
}

template <int N>
int thin(const OrthoParams& p, cudaStream_t st) {
  if (p.m <= 4) return start_thin<N, 1, 4>(p, st);
  if (p.m <= 16) return start_thin<N, 1, 16>(p, st);
  return p.m <= 64 ? start_thin<N, 4, 16>(p, st) : start_thin<N, 32, 16>(p, st);
}

template <int THREADS>
int block(const OrthoParams& p, cudaStream_t st) {
  const size_t bytes = block_layout((int)p.n, (int)p.m).bytes;
  const unsigned blocks = (unsigned)std::min<int64_t>(p.batch, 1 << 20);
  return ortho_dispatch(p, [&](auto type, auto update) {
    const auto kernel = block_kernel<decltype(type), decltype(update)::value, THREADS>;
    // one value for every size: calls of other threads set the same
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSharedMost))
      return (int)e;
    kernel<<<blocks, THREADS, bytes, st>>>(p);
    return (int)cudaGetLastError();
  });
}

}  // namespace

bool ortho_small_fits(const OrthoParams& p) {
  if (p.n <= 4 && p.m <= 32 * kThinCols) return true;
  return p.n <= 16 && p.m <= 4096 && block_layout((int)p.n, (int)p.m).bytes <= kSharedMost;
}

int launch_ortho_small(const OrthoParams& p, cudaStream_t st) {
  if (p.n <= 4 && p.m <= 32 * kThinCols) {
    switch (p.n) {
      case 1: return thin<1>(p, st);
      case 2: return thin<2>(p, st);
      case 3: return thin<3>(p, st);
      default: return thin<4>(p, st);
    }
  }
  if (p.n <= 16 && p.m <= 32) return block<32>(p, st);
  return block<256>(p, st);
}

}  // namespace blitz
