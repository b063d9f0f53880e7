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
// bf16 terms would need three for that.  Where the result is rounded to bf16
// (off by 1.7e-3 itself) the last two steps, whose errors are hardly
// multiplied any more, use the high terms alone; 16-bit inputs are exact in one
// term, so step 0 reads one.  Everything is scaled by powers of two into
// f16's range: |X_ij| <= 1.9 by 2^14, |A_ij| <= 3.7 by 2^14, |B_ij| < 7.9 by 2^13
// (the caller's coefficients are checked to keep to that).
//
// Two launches: `prepare_kernel` advances the momentum and adds up squares
// (in 64 bits, in a fixed order); `ortho_kernel` is one persistent cooperative
// block an SM that runs all 3 * steps products with a grid-wide barrier
// between them, so a step costs no launch.  In it one warp copies tiles of
// 64 columns by TMA (128-byte swizzle), one warp issues the products, and
// eight warps move finished tiles out of tensor memory; tensor memory holds
// two accumulators, so the next tile's products run meanwhile.  Every wait
// gives up after two seconds: the outputs are then NaN.
#include <cuda.h>

#include <algorithm>

#include "ortho.cuh"
#include "tcgen05.cuh"

namespace blitz {

namespace {

constexpr int kBM = 128, kBK = 64;
constexpr int kBox = 64 * kBK * 2;         // bytes of one copied box: 64 rows of 128 bytes
constexpr int kRing = 24 * kBox;           // shared memory of the operand ring
constexpr int kMaxStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;  // warps 0: copies, 1: products, 2: tensor memory, 4..: tiles out
constexpr int kAcc = 256;                  // tensor-memory columns of one accumulator
constexpr int kMaxParts = 256;

struct Info {       // one matrix's scaling, written while X_0 is laid out
  float up, alpha;  // X_0 is stored as u * up; alpha = 1 / ((|u|_F + eps) * up)
  float pad[2];
};

struct KernelParams {
  OrthoParams o;
  CUtensorMap map_x[2], map_a, map_b;
  __half *x[2], *a, *b;   // [2 * batch][n][ld]: high and low terms of each matrix
  double* parts;          // [batch][n_parts]
  Info* info;             // [batch]
  unsigned* barrier;      // [0]: arrivals, [1]: gave up
  int n_parts;
  int ldm, ldn;
  int two_in;             // u needs two terms
  int two_steps;          // steps 0 .. two_steps-1 use two terms
  int bn_s, bn_x;         // tile widths of the symmetric products and of B X
};

// ---- tiles ---------------------------------------------------------------

enum Phase : int { kGram, kPoly, kApply };

struct PhaseShape {
  int which, bn, mt, nt, per, total;  // per: tiles of one matrix
  int k_blocks;
  bool two_a, two_b;                  // terms read of either operand
  bool write_two;                     // terms written
  bool last;
  const CUtensorMap *ma, *mb;
  int stage_bytes, stages;
};

__device__ __forceinline__ int tiles_in_row(int mi, int bn, int nt) { return min(nt, (mi * kBM + kBM - 1) / bn + 1); }

__device__ PhaseShape shape_of(const KernelParams& p, int ph) {
  PhaseShape s;
  const int step = ph / 3;
  const int n = (int)p.o.n, m = (int)p.o.m;
  s.which = ph - 3 * step;
  const bool two = step < p.two_steps;
  const bool two_x = two && (step > 0 || p.two_in);
  s.last = step == p.o.steps - 1 && s.which == kApply;
  s.mt = (n + kBM - 1) / kBM;
  s.bn = s.which == kApply ? p.bn_x : p.bn_s;
  s.nt = ((s.which == kApply ? m : n) + s.bn - 1) / s.bn;
  if (s.which == kApply) {
    s.per = s.mt * s.nt;
  } else {
    s.per = 0;
    for (int i = 0; i < s.mt; ++i) s.per += tiles_in_row(i, s.bn, s.nt);
  }
  s.total = s.per * (int)p.o.batch;
  s.k_blocks = ((s.which == kGram ? m : n) + kBK - 1) / kBK;
  s.two_a = s.which == kGram ? two_x : two;
  s.two_b = s.which == kPoly ? two : two_x;
  // A and B are read by this step's own products, the new X by the next one's
  s.write_two = s.which == kApply ? step + 1 < p.two_steps : two;
  s.ma = s.which == kGram ? &p.map_x[step & 1] : s.which == kPoly ? &p.map_a : &p.map_b;
  s.mb = s.which == kPoly ? &p.map_a : &p.map_x[step & 1];
  s.stage_bytes = ((s.two_a ? 2 : 1) * (kBM / 64) + (s.two_b ? 2 : 1) * (s.bn / 64)) * kBox;
  s.stages = min(kRing / s.stage_bytes, kMaxStages);
  return s;
}

__device__ __forceinline__ void tile_of(const PhaseShape& s, int t, int& b, int& mi, int& ni) {
  b = t / s.per;
  int r = t - b * s.per;
  if (s.which == kApply) {
    // neighbouring blocks take the same columns of X and the rows of B in turn
    ni = r / s.mt;
    mi = r - ni * s.mt;
    return;
  }
  mi = 0;
  for (int k = tiles_in_row(0, s.bn, s.nt); r >= k; k = tiles_in_row(mi, s.bn, s.nt)) {
    r -= k;
    ++mi;
  }
  ni = r;
}

// 32 values of one row as terms at dst (and, the low ones, at dst + low): 16-byte stores
__device__ __forceinline__ void store_row(__half* dst, int64_t low, const float (&v)[32], bool two) {
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    uint4 h, l;
    split8(v + k, h, l);
    *(uint4*)(dst + k) = h;
    if (two) *(uint4*)(dst + low + k) = l;
  }
}

// one finished accumulator tile out of tensor memory; a warp takes 32 of its
// rows and every second group of 32 columns
__device__ void tile_out(const KernelParams& p, const PhaseShape& s, int b, int mi, int ni, int step, uint32_t acc,
                         int warp, int lane) {
  const int quarter = warp & 3, n = (int)p.o.n, m = (int)p.o.m;
  const int row = mi * kBM + quarter * 32 + lane, row_hi = mi * kBM + quarter * 32 + 31;
  const float alpha = step == 0 ? p.info[b].alpha : 1.0f / kScaleX;
  const int64_t low_n = (int64_t)n * p.ldn, low_m = (int64_t)n * p.ldm;
  for (int c = (warp >> 2) * 32; c < s.bn; c += 32 * (kEpiWarps / 4)) {
    const int col = ni * s.bn + c;
    if (s.which == kApply ? col >= m : col >= n || col > row_hi) continue;  // the same for the whole warp
    if (mi * kBM + quarter * 32 >= n) continue;
    float v[32];
    tmem_load32(acc + ((uint32_t)(quarter * 32) << 16) + c, v);
    if (s.which == kApply) {
      if (!s.last) {
        const float f = alpha * (kScaleX / kScaleB);
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] *= f;
        if (row < n)
          store_row(p.x[(step + 1) & 1] + ((int64_t)(2 * b) * n + row) * p.ldm + col, low_m, v, s.write_two);
      } else if (row < n) {
        const float f = alpha / kScaleB;
        const int64_t at = (int64_t)b * n * m + row * p.o.si;
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (col + k < m) ortho_store(p.o, at + (col + k) * p.o.sj, v[k] * f);
      }
      continue;
    }
    __half* const out = (s.which == kGram ? p.a : p.b) + (int64_t)(2 * b) * n * p.ldn;
    if (s.which == kGram) {
      const float f = alpha * alpha * kScaleA;
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] *= f;
    } else {
      // B = a I + b A + c A^2, scaled; A from its terms
      const float fc = p.o.c * (kScaleB / (kScaleA * kScaleA)), fb = p.o.b * (kScaleB / kScaleA);
      const __half* A = p.a + ((int64_t)(2 * b) * n + min(row, n - 1)) * p.ldn + col;
#pragma unroll
      for (int k = 0; k < 32; k += 8) {
        const uint4 hi = *(const uint4*)(A + k);
        uint4 lo = make_uint4(0, 0, 0, 0);
        if (s.two_a) lo = *(const uint4*)(A + low_n + k);
        const __half2* h2 = (const __half2*)&hi;
        const __half2* l2 = (const __half2*)&lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 h = __half22float2(h2[e]), l = __half22float2(l2[e]);
          v[k + 2 * e] = fmaf(fc, v[k + 2 * e], fb * (h.x + l.x));
          v[k + 2 * e + 1] = fmaf(fc, v[k + 2 * e + 1], fb * (h.y + l.y));
        }
      }
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (col + k == row) v[k] += p.o.a * kScaleB;
    }
    // on and below the diagonal; the rest is the mirror image, so that the
    // stored matrix is symmetric to the last bit
    if (row < n) {
      __half* dst = out + (int64_t)row * p.ldn + col;
      if (col + 31 <= row) {
        store_row(dst, low_n, v, s.write_two);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (col + k <= row) {
            const __half h = __float2half_rn(v[k]);
            dst[k] = h;
            if (s.write_two) dst[low_n + k] = __float2half_rn(v[k] - __half2float(h));
          }
      }
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (col + k < row) {
          const __half h = __float2half_rn(v[k]);
          __half* t = out + (int64_t)(col + k) * p.ldn + row;
          *t = h;
          if (s.write_two) t[low_n] = __float2half_rn(v[k] - __half2float(h));
        }
    }
  }
}

// ---- kernels -------------------------------------------------------------

// the momentum advanced, and the squares of u added up: block (x, b) takes
// part x of matrix b
__global__ void __launch_bounds__(256) prepare_kernel(OrthoParams o, double* parts, unsigned* barrier, int n_parts) {
  __shared__ double sums[8];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 2) barrier[threadIdx.x] = 0u;
  const int64_t size = o.n * o.m, per = (size + n_parts - 1) / n_parts;
  for (int64_t b = blockIdx.y; b < o.batch; b += gridDim.y) {
    const int64_t lo = b * size + min(size, (int64_t)blockIdx.x * per), hi = b * size + min(size, (blockIdx.x + 1) * per);
    double sq = 0.0;
    for (int64_t e = lo + threadIdx.x; e < hi; e += 256) {
      const float u = ortho_u<true>(o, e);
      sq += (double)u * (double)u;
    }
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

// every block of the grid has arrived, and what each wrote (for its reads and its copies) is seen
__device__ bool grid_barrier(const KernelParams& p, unsigned target, volatile int* dead) {
  fence_async_global();
  fence_async_shared();
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(p.barrier, 1u);
    const long long t0 = clock64();
    volatile unsigned* arrived = p.barrier;
    while (*arrived < target) {
      if (*dead || ((volatile unsigned*)p.barrier)[1] || clock64() - t0 > kGiveUp) {
        *dead = 1;
        break;
      }
    }
    if (*dead) atomicExch(p.barrier + 1, 1u);
    __threadfence();
  }
  __syncthreads();
  fence_async_global();
  fence_async_shared();
  return *dead == 0;
}

// X_0's terms, scaled; 64 x 64 tiles, through shared memory where X is the
// transpose of what is stored
__device__ void lay_out(const KernelParams& p, float* tile) {
  const OrthoParams& o = p.o;
  const int n = (int)o.n, m = (int)o.m;
  const int ti = (n + 63) / 64, tj = p.ldm / 64, per = ti * tj;
  const int64_t total = (int64_t)per * o.batch;
  __shared__ Info info;
  int64_t have = -1;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int64_t b = t / per;
    const int r = (int)(t - b * per), i0 = r / tj * 64, j0 = (r % tj) * 64;
    if (b != have) {
      __syncthreads();
      if (threadIdx.x < 32) {
        double sq = 0.0;
        for (int k = threadIdx.x; k < p.n_parts; k += 32) sq += p.parts[b * p.n_parts + k];
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, k);
        if (threadIdx.x == 0) {
          ortho_scaling(sqrt(sq), o.eps, info.up, info.alpha);
          if (r == 0) p.info[b] = info;
        }
      }
      __syncthreads();
      have = b;
    }
    const int64_t base = b * o.n * o.m;
    if (o.sj != 1) {
      for (int e = threadIdx.x; e < 64 * 64; e += kThreads) {
        const int i = i0 + (e & 63), j = j0 + (e >> 6);
        tile[(e & 63) * 65 + (e >> 6)] = i < n && j < m ? ortho_u<false>(o, base + i + j * o.sj) : 0.0f;
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < 64 * 32; e += kThreads) {
      const int i = i0 + (e >> 5), j = j0 + 2 * (e & 31);
      if (i >= n) continue;
      float x = 0.0f, y = 0.0f;
      if (o.sj != 1) {
        x = tile[(e >> 5) * 65 + 2 * (e & 31)];
        y = tile[(e >> 5) * 65 + 2 * (e & 31) + 1];
      } else {
        if (j < m) x = ortho_u<false>(o, base + i * o.si + j);
        if (j + 1 < m) y = ortho_u<false>(o, base + i * o.si + j + 1);
      }
      x *= info.up;
      y *= info.up;
      __half* dst = p.x[0] + ((2 * b) * n + i) * (int64_t)p.ldm + j;
      uint32_t lo;
      *(uint32_t*)dst = split2(x, y, lo);
      if (p.two_in) *(uint32_t*)(dst + (int64_t)n * p.ldm) = lo;
    }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kThreads, 1) ortho_kernel(const __grid_constant__ KernelParams p) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 4];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  volatile int* dead = &dead_flag;
  uint8_t* ring = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t full = smem_addr(bars), empty = full + 8 * kMaxStages, acc_full = full + 16 * kMaxStages,
                 acc_empty = acc_full + 16, ring_addr = smem_addr(ring);
  if (threadIdx.x == 0) {
    dead_flag = 0;
    for (int i = 0; i < kMaxStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, kEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) tmem_alloc(&tmem_base, 2 * kAcc);
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = tmem_base;

  lay_out(p, (float*)ring);
  unsigned arrivals = gridDim.x;
  bool alive = grid_barrier(p, arrivals, dead);

  // each role's parities, one bit a stage or accumulator; a fresh barrier's
  // "empty" counts as passed, hence the ones
  uint32_t ph_full = 0, ph_empty = ~0u, ph_accf = 0, ph_acce = ~0u;
  uint32_t stage_no = 0, acc_no = 0;
  const int phases = 3 * p.o.steps;
  for (int ph = 0; alive && ph < phases; ++ph) {
    const PhaseShape s = shape_of(p, ph);
    const int step = ph / 3;
    stage_no = 0;
    if (warp == 0 && lane == 0) {
      const int low = 1;
      for (int t = blockIdx.x; t < s.total && !*dead; t += gridDim.x) {
        int b, mi, ni;
        tile_of(s, t, b, mi, ni);
        for (int k = 0; k < s.k_blocks; ++k) {
          const uint32_t st = stage_no;
          stage_no = stage_no + 1 == (uint32_t)s.stages ? 0 : stage_no + 1;
          if (!mbar_wait(empty + 8 * st, ph_empty >> st & 1, dead)) break;
          ph_empty ^= 1u << st;
          mbar_expect(full + 8 * st, s.stage_bytes);
          uint32_t dst = ring_addr + st * s.stage_bytes;
          for (int term = 0; term < (s.two_a ? 2 : 1); ++term)
            for (int q = 0; q < kBM / 64; ++q, dst += kBox)
              tma_load(dst, s.ma, k * kBK, mi * kBM + q * 64, 2 * b + term * low, full + 8 * st);
          for (int term = 0; term < (s.two_b ? 2 : 1); ++term)
            for (int q = 0; q < s.bn / 64; ++q, dst += kBox) {
              const int at = ni * s.bn + q * 64;
              if (s.which == kApply)
                tma_load(dst, s.mb, at, k * kBK, 2 * b + term * low, full + 8 * st);
              else
                tma_load(dst, s.mb, k * kBK, at, 2 * b + term * low, full + 8 * st);
            }
        }
      }
    } else if (warp == 1) {
      const bool mn = s.which == kApply;
      const uint32_t idesc = instruction_desc(s.bn, mn);
      // 16 of K further: 32 bytes along a row, or 16 rows of 128 bytes
      const uint32_t b_step = mn ? 2048 : 32, b_lead = mn ? kBox : 16;
      const uint32_t a_term = kBM / 64 * kBox, b_term = s.bn / 64 * kBox;
      for (int t = blockIdx.x; t < s.total && !*dead; t += gridDim.x) {
        const uint32_t ac = acc_no;
        acc_no ^= 1;
        if (!mbar_wait(acc_empty + 8 * ac, ph_acce >> ac & 1, dead)) break;
        ph_acce ^= 1u << ac;
        tcgen05_after_sync();
        const uint32_t d = tmem + ac * kAcc;
        for (int k = 0; k < s.k_blocks; ++k) {
          const uint32_t st = stage_no;
          stage_no = stage_no + 1 == (uint32_t)s.stages ? 0 : stage_no + 1;
          if (!mbar_wait(full + 8 * st, ph_full >> st & 1, dead)) break;
          ph_full ^= 1u << st;
          tcgen05_after_sync();
          const uint32_t a0 = ring_addr + st * s.stage_bytes, b0 = a0 + (s.two_a ? 2 : 1) * a_term;
          // high * high, low * high, high * low
          for (int q = 0; q < 3; ++q) {
            if (q == 1 && !s.two_a || q == 2 && !s.two_b) continue;
            const uint32_t aa = a0 + (q == 1 ? a_term : 0), bb = b0 + (q == 2 ? b_term : 0);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              mma(d, smem_desc(aa + 32 * kk, 16, 1024), smem_desc(bb + b_step * kk, b_lead, 1024), idesc,
                  k + q + kk > 0);
          }
          mma_commit(empty + 8 * st);
        }
        mma_commit(acc_full + 8 * ac);
      }
    } else if (warp >= 4) {
      for (int t = blockIdx.x; t < s.total && !*dead; t += gridDim.x) {
        const uint32_t ac = acc_no;
        acc_no ^= 1;
        const bool ok = mbar_wait(acc_full + 8 * ac, ph_accf >> ac & 1, dead);
        if (!__all_sync(0xffffffffu, ok)) break;
        ph_accf ^= 1u << ac;
        tcgen05_after_sync();
        int b, mi, ni;
        tile_of(s, t, b, mi, ni);
        tile_out(p, s, b, mi, ni, step, tmem + ac * kAcc, warp - 4, lane);
        tcgen05_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty + 8 * ac);
      }
    }
    __syncwarp();
    if (ph + 1 < phases) {
      arrivals += gridDim.x;
      alive = grid_barrier(p, arrivals, dead);
    }
  }
  __syncthreads();
  if (dead_flag) {
    // copies and products of this block that are still in flight end within this time
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    const int64_t size = p.o.batch * p.o.n * p.o.m;
    for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < size; e += (int64_t)gridDim.x * kThreads)
      ortho_store(p.o, e, __int_as_float(0x7fffffff));
  }
  __syncthreads();
  if (warp == 2) tmem_free(tmem, 2 * kAcc);
}

// ---- host ----------------------------------------------------------------

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
  q.info = up((size_t)p.batch * sizeof(Info));
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

// The width of a tile: the one whose slowest block has the least to do, a
// wider one (fewer bytes a product) where that is equal.
int pick_width(int64_t tiles64, int64_t tiles128, int64_t tiles256, int sms) {
  const int64_t t[3] = {tiles256, tiles128, tiles64};
  const int w[3] = {256, 128, 64};
  int best = 256;
  int64_t cost = INT64_MAX;
  for (int i = 0; i < 3; ++i) {
    const int64_t c = (t[i] + sms - 1) / sms * w[i];
    if (c < cost) {
      cost = c;
      best = w[i];
    }
  }
  return best;
}

int64_t symmetric_tiles(int64_t n, int bn) {
  const int64_t mt = (n + kBM - 1) / kBM, nt = (n + bn - 1) / bn;
  int64_t k = 0;
  for (int64_t i = 0; i < mt; ++i) k += std::min(nt, (i * kBM + kBM - 1) / bn + 1);
  return k;
}

}  // namespace

size_t ortho_workspace_bytes(const OrthoParams& p) { return ortho_small_fits(p) || ortho_resident_fits(p) ? 0 : plan_of(p).total; }

int launch_ortho(const OrthoParams& o, void* workspace, cudaStream_t st) {
  if (ortho_small_fits(o)) return launch_ortho_small(o, st);
  if (ortho_resident_fits(o)) return launch_ortho_resident(o, st);
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return (int)e;
  const Plan q = plan_of(o);
  KernelParams p;
  p.o = o;
  uint8_t* w = (uint8_t*)workspace;
  p.barrier = (unsigned*)w;
  w += 256;
  p.x[0] = (__half*)w;
  p.x[1] = (__half*)(w + q.x);
  p.a = (__half*)(w + 2 * q.x);
  p.b = (__half*)(w + 2 * q.x + q.a);
  p.parts = (double*)(w + 2 * q.x + 2 * q.a);
  p.info = (Info*)(w + 2 * q.x + 2 * q.a + q.parts);
  p.n_parts = q.n_parts;
  p.ldm = q.ldm;
  p.ldn = q.ldn;
  p.two_in = ortho_two_in(o);
  p.two_steps = ortho_two_steps(o);
  p.bn_s = pick_width(o.batch * symmetric_tiles(o.n, 64), o.batch * symmetric_tiles(o.n, 128),
                      o.batch * symmetric_tiles(o.n, 256), sms);
  const int64_t mt = (o.n + kBM - 1) / kBM;
  p.bn_x = pick_width(o.batch * mt * ((o.m + 63) / 64), o.batch * mt * ((o.m + 127) / 128),
                      o.batch * mt * ((o.m + 255) / 256), sms);
  for (int i = 0; i < 2; ++i)
    if (int rc = make_map(&p.map_x[i], p.x[i], o.m, o.n, q.ldm, o.batch)) return rc;
  if (int rc = make_map(&p.map_a, p.a, o.n, o.n, q.ldn, o.batch)) return rc;
  if (int rc = make_map(&p.map_b, p.b, o.n, o.n, q.ldn, o.batch)) return rc;
  prepare_kernel<<<dim3((unsigned)q.n_parts, (unsigned)std::min<int64_t>(o.batch, 65535)), 256, 0, st>>>(
      o, p.parts, p.barrier, q.n_parts);
  if (cudaError_t e = cudaGetLastError()) return (int)e;
  const int smem = kRing + 1024;
  if (cudaError_t e = cudaFuncSetAttribute(ortho_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
    return (int)e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, ortho_kernel, p);
}

}  // namespace blitz
