// Orthogonalisation of matrices of medium size over the whole grid (see
// ortho.cu for the formula, the terms and the phases).
//
// A matrix of 1024 rows has 36 symmetric tiles of 128 x 128 for 148 SMs, and an
// SM takes in about 64 bytes a cycle: 1 MB of operands for one tile's two terms
// would take 9 us. So a cluster of S blocks shares a tile: each
// copies and multiplies 1/S of its k, hands the columns that are another's to that
// block's shared memory, and finishes 1/S of the columns.  (By bulk copies: stores into a
// peer's shared memory came to 12 bytes a cycle, 5500 cycles a tile.)  Order of the sum: by
// block, so the result does not depend on timing.
//
// Where there are tiles enough (S = 1) a k of 64 takes 760 cycles, the products' own rate; 2048^2 in
// 32 bits takes 468 us, 4096^2 3.8 ms.  (Tiles of 128 x 256 have fewer units in flight and leave
// more SMs without one: 4260 us for 3760 at 4096^2. Pairs of blocks on 256 x 128 took 5530.)
//
// The operands' ring holds the low terms of a k of 64 and the high ones as units of their own:
// the low ones are free after two thirds of the products.  Two warps issue copies, every
// second unit each, and two issue products, every second k of 64 each into accumulators of its
// own: a wait that is already over still takes 125 cycles, a product's issue 45 and a copy's
// 100; one warp each took 1350 cycles a k of 64.
//
// Tensor memory holds four accumulators. Each takes one k of 64 (the low terms first) and
// is then added up in registers: the tensor cores' additions drop the bits below the
// accumulator's last one, those here round. Over
// 1024 columns that is the difference between an error of 4e-5 and of 2e-6.
#include <algorithm>
#include <atomic>

#include "ortho_grid.cuh"

namespace blitz {

namespace {

constexpr int kB = 128;                       // tiles are kB x kB
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;  // warps 0, 1: copies, 2, 3: products, 4..: tiles out
constexpr int kColumns = 512;                 // of tensor memory: all

constexpr int kAccs = kColumns / kB;
constexpr int kUnit = 4 * kBox;               // one term of both operands
template <int S>
constexpr int kUnits = S == 1 ? 6 : 4;        // 192 or 128 KB; even: a slot's units are one warp's
template <int S>
constexpr int kRing = kUnits<S> * kUnit;
// columns that go to other blocks, on their way out; and as they come in
template <int S>
constexpr int kExchange = S > 1 ? (S - 1) * (kB / S) * kB * 4 : 0;

struct Shape {
  OrthoTerms t;
  int mt, nt, per, total;  // per: tiles of one matrix
  int k0, boxes;           // this block's k, in boxes
  int units;               // units of a box: 2 where an operand has two terms
};

template <int S>
__device__ __forceinline__ Shape shape_of(const OrthoGrid& p, int ph, int rank) {
  Shape s;
  s.t = ortho_terms(p, ph);
  const int n = (int)p.o.n, m = (int)p.o.m;
  s.mt = (n + kB - 1) / kB;
  s.nt = (m + kB - 1) / kB;
  if (s.t.which == kApply)
    s.per = s.mt * s.nt;
  else
    s.per = s.mt * (s.mt + 1) / 2;
  s.total = s.per * (int)p.o.batch;
  const int boxes = ((s.t.which == kGram ? m : n) + kBK - 1) / kBK;
  s.k0 = S > 1 ? boxes * rank / S : 0;
  s.boxes = (S > 1 ? boxes * (rank + 1) / S : boxes) - s.k0;
  s.units = s.t.two_a || s.t.two_b ? 2 : 1;
  return s;
}

__device__ __forceinline__ void tile_of(const Shape& s, int t, int& b, int& mi, int& ni) {
  b = t / s.per;
  const int r = t - b * s.per;
  if (s.t.which == kApply) {
    ni = r / s.mt;
    mi = r - ni * s.mt;
    return;
  }
  // r = mi (mi + 1) / 2 + ni
  mi = (int)((sqrtf(8.0f * (float)r + 1.0f) - 1.0f) * 0.5f);
  while (mi * (mi + 1) / 2 > r) --mi;
  while ((mi + 1) * (mi + 2) / 2 <= r) ++mi;
  ni = r - mi * (mi + 1) / 2;
}

// A's terms where a thread will need them for B (read ahead of the sums where there is room)
template <int C>
__device__ __forceinline__ void load_a(const OrthoGrid& p, const OrthoTerms& t, int b, int row, int col,
                                       uint32_t (&hi)[C / 2], uint32_t (&lo)[C / 2]) {
  const int n = (int)p.o.n;
  const __half* A = p.a + ((int64_t)(2 * b) * n + min(row, n - 1)) * p.ldn + col;
#pragma unroll
  for (int k = 0; k < C / 2; k += 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) hi[k + e] = lo[k + e] = 0;
    // rows are a whole number of 64 columns long, so 16 from one below n are in the row
    if (t.which == kPoly && col + 2 * k < n) {
      load32(A + 2 * k, *(uint32_t(*)[8])(hi + k));
      load32(A + (int64_t)n * p.ldn + 2 * k, *(uint32_t(*)[8])(lo + k));
    }
  }
}

// C values' terms to row `dst`, the low ones `low` further, as far as there are columns
template <int C>
__device__ __forceinline__ void store_terms(__half* dst, int64_t low, int left, const uint32_t (&h)[C / 2],
                                            const uint32_t (&l)[C / 2]) {
#pragma unroll
  for (int k = 0; k < C / 2; k += 8) {
    if (2 * k >= left) break;
    store32(dst + 2 * k, *(const uint32_t(*)[8])(h + k));
    store32(dst + low + 2 * k, *(const uint32_t(*)[8])(l + k));
  }
}

// C finished sums of one row (columns col ..) turned into what the phase writes
template <int C>
__device__ __forceinline__ void finish(const OrthoGrid& p, const OrthoTerms& t, int b, int row, int col, bool diagonal,
                                       bool mirror, float (&v)[C], const uint32_t (&old_hi)[C / 2],
                                       const uint32_t (&old_lo)[C / 2], OrthoFactors by) {
  const int n = (int)p.o.n, m = (int)p.o.m, lane = threadIdx.x & 31;
  if (t.which == kApply) {
#pragma unroll
    for (int k = 0; k < C; ++k) v[k] *= by.next;
    if (row >= n) return;
    if (!t.last) {
      uint32_t h[C / 2], l[C / 2];
#pragma unroll
      for (int k = 0; k < C / 2; ++k) h[k] = split2(v[2 * k], v[2 * k + 1], l[k]);
      store_terms<C>(p.x[(t.step + 1) & 1] + ((int64_t)(2 * b) * n + row) * p.ldm + col, (int64_t)n * p.ldm, m - col,
                     h, l);
      return;
    }
    const int64_t at = (int64_t)b * n * m + row * p.o.si;
    if (p.o.sj == 1 && p.four) {
#pragma unroll
      for (int k0 = 0; k0 < C; k0 += 16) {
        // 16 of the parameter's values before the first of them is written
        float old[16];
#pragma unroll
        for (int k = k0; k < k0 + 16; k += 4)
          if (p.o.param && col + k < m) load_values<4>(p.o.param + at + col + k, *(float(*)[4])(old + k - k0));
#pragma unroll
        for (int k = k0; k < k0 + 16; k += 4) {
          if (col + k >= m) break;
          float d[4] = {v[k], v[k + 1], v[k + 2], v[k + 3]};
          const int64_t e = at + col + k;
          if (p.o.param) {
#pragma unroll
            for (int q = 0; q < 4; ++q) d[q] = __fmaf_rn(-p.o.alpha, d[q], __fmul_rn(old[k - k0 + q], p.o.keep));
            store_values<4>(p.o.param + e, d);
          } else if (p.o.g_type == kValueF32) {
            store_values<4>((float*)p.o.out + e, d);
          } else if (p.o.g_type == kValueBf16) {
            store_values<4>((__nv_bfloat16*)p.o.out + e, d);
          } else {
            store_values<4>((__half*)p.o.out + e, d);
          }
        }
      }
    } else {
#pragma unroll
      for (int k0 = 0; k0 < C; k0 += 16) {
        float old[16];
#pragma unroll
        for (int k = 0; k < 16; ++k)
          old[k] = p.o.param && col + k0 + k < m ? p.o.param[at + (col + k0 + k) * p.o.sj] : 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k)
          if (col + k0 + k < m) ortho_store(p.o, at + (col + k0 + k) * p.o.sj, v[k0 + k], old[k]);
      }
    }
    return;
  }
  const int64_t low = (int64_t)n * p.ldn;
  if (t.which == kGram) {
    const float f = by.x * by.x * kScaleA;
#pragma unroll
    for (int k = 0; k < C; ++k) v[k] *= f;
  } else {
    // B = a I + b A + c A^2, scaled; A from its terms
    const float fc = p.o.c * (kScaleB / (kScaleA * kScaleA)), fb = p.o.b * (kScaleB / kScaleA);
#pragma unroll
    for (int k = 0; k < C / 2; ++k) {
      const float2 x = join2(old_hi[k], old_lo[k]);
      v[2 * k] = fmaf(fc, v[2 * k], fb * x.x);
      v[2 * k + 1] = fmaf(fc, v[2 * k + 1], fb * x.y);
    }
    if (diagonal) {
#pragma unroll
      for (int k = 0; k < C; ++k) v[k] += col + k == row ? p.o.a * kScaleB : 0.0f;
    }
  }
  __half* out = (t.which == kGram ? p.a : p.b) + (int64_t)(2 * b) * n * p.ldn;
  uint32_t h[C / 2], l[C / 2];
#pragma unroll
  for (int k = 0; k < C / 2; ++k) h[k] = split2(v[2 * k], v[2 * k + 1], l[k]);
  if (row < n) store_terms<C>(out + (int64_t)row * p.ldn + col, low, n - col, h, l);
  if (!mirror) return;
  // the mirror image: neighbouring lanes (rows) swap halves, so that each writes two
  // rows' values of one column in one word
  const int even = row & ~1;
  __half* to = out + (int64_t)(col + (lane & 1)) * p.ldn + even;
  const uint32_t pick = lane & 1 ? 0x3276u : 0x5410u;
#pragma unroll
  for (int k = 0; k < C / 2; ++k) {
    const uint32_t ho = __shfl_xor_sync(0xffffffffu, h[k], 1), lo = __shfl_xor_sync(0xffffffffu, l[k], 1);
    // even lane: (mine.first, other's first); odd lane: (other's second, mine.second)
    const uint32_t hw = __byte_perm(h[k], ho, pick), lw = __byte_perm(l[k], lo, pick);
    // ldn is even, so a pair that begins below n stays inside its row
    if (even < n) {
      *(uint32_t*)(to + (int64_t)(2 * k) * p.ldn) = hw;
      *(uint32_t*)(to + (int64_t)(2 * k) * p.ldn + low) = lw;
    }
  }
}

template <int S>
__global__ void __launch_bounds__(kThreads, 1) split_kernel(const __grid_constant__ OrthoGrid p) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) uint64_t bars[2 * kUnits<S> + 2 * kAccs + 4];
  __shared__ uint32_t tmem_base;
  __shared__ int dead_flag;
  volatile int* dead = &dead_flag;
  uint8_t* ring = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t full = smem_addr(bars), empty = full + 8 * kUnits<S>, acc_full = empty + 8 * kUnits<S>,
                 acc_empty = acc_full + 8 * kAccs, x_full = acc_empty + 8 * kAccs, x_empty = x_full + 8,
                 token = x_empty + 8;
  const uint32_t ring_addr = smem_addr(ring), exchange = ring_addr + kRing<S>, incoming = exchange + kExchange<S>;
  const int rank = S > 1 ? (int)cluster_rank() : 0;
  const int first = blockIdx.x / S, by = gridDim.x / S;
  if (threadIdx.x == 0) {
    dead_flag = 0;
    for (int i = 0; i < kUnits<S>; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kAccs; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, kEpiWarps);
    }
    for (int i = 0; i < 2; ++i) mbar_init(token + 8 * i, 1);
    mbar_init(x_full, 1);
    mbar_init(x_empty, kEpiWarps * (S > 1 ? S - 1 : 1));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < 2; ++i) prefetch_map(&p.map_x[i]);
    prefetch_map(&p.map_a);
    prefetch_map(&p.map_b);
  }
  if (warp == 0) tmem_alloc(&tmem_base, kColumns);
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  if (S > 1) cluster_sync();
  // all 512 columns are this block's, so they begin at 0 (which the compiler then knows to
  // be the same for the whole warp)
  constexpr uint32_t tmem = 0;
  const uint32_t on = elected();
  const long long limit = p.o.wait_limit;

  // Units and boxes are numbered through the whole run, by every role alike: unit u lies in
  // slot u % kUnits and is that slot's use u / kUnits, whose parity is waited for; box a has
  // accumulator a % kAccs.
  uint32_t unit0 = 0, box0 = 0, ph_xf = 0, ph_xe = 1;
  unsigned arrivals = 0;
  bool alive = true;
  const int phases = 3 * p.o.steps;
#pragma unroll 1
  for (int ph = 0; alive && ph < phases; ++ph) {
    const Shape s = shape_of<S>(p, ph, rank);
    const int tiles = first < s.total ? (s.total - first + by - 1) / by : 0;
    if (warp < 2) {
      uint32_t u = unit0;
      bool go = true;  // until a wait gives up
      for (int t = first; t < s.total && go; t += by) {
        int b, mi, ni;
        tile_of(s, t, b, mi, ni);
        for (int k = s.k0; k < s.k0 + s.boxes && go; ++k) {
          // the low terms, then the high ones
          for (int term = s.units - 1; term >= 0; --term, ++u) {
            if ((u & 1) != (uint32_t)warp) continue;
            const uint32_t slot = u % kUnits<S>;
            // by lane: the one that copies goes on as long as its own waits end
            go = mbar_wait(empty + 8 * slot, (u / kUnits<S> & 1) ^ 1, dead, limit);
            if (!go) break;
            const bool has_a = term == 0 || s.t.two_a, has_b = term == 0 || s.t.two_b;
            const uint32_t bar = full + 8 * slot, dst = ring_addr + slot * kUnit;
            mbar_expect(on, bar, (has_a ? 2 * kBox : 0) + (has_b ? 2 * kBox : 0));
            if (has_a)
              for (int q = 0; q < 2; ++q)
                tma_load(on, dst + q * kBox, s.t.ma, k * kBK, mi * kB + q * 64, 2 * b + term, bar);
            if (has_b)
              for (int q = 0; q < 2; ++q) {
                const int at = ni * kB + q * 64;
                if (s.t.which == kApply)
                  tma_load(on, dst + (2 + q) * kBox, s.t.mb, at, k * kBK, 2 * b + term, bar);
                else
                  tma_load(on, dst + (2 + q) * kBox, s.t.mb, k * kBK, at, 2 * b + term, bar);
              }
          }
        }
      }
    } else if (warp < 4) {
      const bool mn = s.t.which == kApply;
      const uint32_t idesc = instruction_desc(kB, mn);
      // 16 of k further, in units of 16 bytes: 32 bytes along a row, or 16 rows
      const uint32_t b_step = mn ? 128 : 2, b_lead = mn ? kBox : 16;
      // The boxes of the whole run go to the two warps in turn, and a warp waits for one only
      // when the other has what it waited for before it: a parity cannot tell a barrier two
      // uses behind from one that is ready.
      const uint32_t mine = warp - 2;
      uint32_t u0 = unit0, g0 = box0;
      bool go = true;  // until a wait gives up
      for (int t = 0; t < tiles && go; ++t, u0 += s.boxes * s.units, g0 += s.boxes) {
        for (int k = (int)((mine ^ g0) & 1); k < s.boxes; k += 2) {
          const uint32_t a = g0 + k, turn = a >> 1, d = tmem + a % kAccs * kB;
          const uint32_t ul = u0 + k * s.units, uh = ul + s.units - 1;
          const uint32_t lo = ul % kUnits<S>, hi = uh % kUnits<S>;
          go = mbar_wait(token + 8 * mine, (turn + (mine ? 0 : 1)) & 1, dead, limit) &&
               mbar_wait(acc_empty + 8 * (a % kAccs), (a / kAccs & 1) ^ 1, dead, limit) &&
               (s.units == 1 || mbar_wait(full + 8 * lo, ul / kUnits<S> & 1, dead, limit)) &&
               mbar_wait(full + 8 * hi, uh / kUnits<S> & 1, dead, limit);
          go = whole_warp(go);
          if (!go) break;
          uint32_t add = 0;
          mbar_arrive(on, token + 8 * (mine ^ 1));
          tcgen05_after_sync();
          const uint32_t ah = smem_desc(ring_addr + hi * kUnit, 16),
                         bh = smem_desc(ring_addr + hi * kUnit + 2 * kBox, b_lead);
          if (s.units == 2) {
            const uint32_t al = smem_desc(ring_addr + lo * kUnit, 16),
                           bl = smem_desc(ring_addr + lo * kUnit + 2 * kBox, b_lead);
            // low * high, high * low: small terms first
            if (s.t.two_a) {
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk, add = 1) mma(on, d, al + 2 * kk, bh + b_step * kk, idesc, add);
            }
            if (s.t.two_b) {
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk, add = 1) mma(on, d, ah + 2 * kk, bl + b_step * kk, idesc, add);
            }
            mma_commit(on, empty + 8 * lo);
          }
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk, add = 1) mma(on, d, ah + 2 * kk, bh + b_step * kk, idesc, add);
          mma_commit(on, empty + 8 * hi);
          mma_commit(on, acc_full + 8 * (a % kAccs));
        }
      }
    } else {
      uint32_t a = box0;
      // a block finishes W columns of a tile, a thread C of them in one row: the first or
      // second half.  It adds up that half of every block's columns.
      constexpr int W = kB / S, C = W / 2;
      const int quarter = warp & 3, half = (warp >> 2) - 1, local = quarter * 32 + lane;
      const uint32_t rows = tmem + ((uint32_t)(quarter * 32) << 16) + half * C;
      // Warps that gave up go through the rest of the phase without arriving or sending: they
      // meet at a barrier of their own.
      bool ok = true;
      for (int t = first; t < s.total; t += by) {
        int b, mi, ni;
        tile_of(s, t, b, mi, ni);
        const int row = mi * kB + local, col = ni * kB + (S > 1 ? rank * W : 0) + half * C;
        // read ahead of the sums
        const OrthoFactors factors = ortho_factors(p.info[b], s.t.step, s.t.last);
        const bool sym = s.t.which != kApply, diagonal = sym && mi == ni, mirror = sym && mi > ni;
        float acc[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
        for (int j = 0; j < s.boxes; ++j, ++a) {
          const uint32_t ac = a % kAccs;
          ok = whole_warp(mbar_wait(acc_full + 8 * ac, a / kAccs & 1, dead, limit)) && ok;
          tcgen05_after_sync();
          if constexpr (S == 4) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              float v[16];
              tmem_load16(rows + ac * kB + g * W, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[g * 16 + i] += v[i];
            }
          } else {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              float v[32];
              tmem_load32(rows + ac * kB + g * (S == 2 ? W : 32), v);
#pragma unroll
              for (int i = 0; i < 32; ++i) acc[g * 32 + i] += v[i];
            }
          }
          tcgen05_before_sync();
          __syncwarp();
          if (ok) mbar_arrive(on, acc_empty + 8 * ac);
        }
        if constexpr (S == 1) {
#pragma unroll
          for (int c = 0; c < C; c += 32) {
            uint32_t hi[16], lo[16];
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = acc[c + i];
            load_a<32>(p, s.t, b, row, col + c, hi, lo);
            finish<32>(p, s.t, b, row, col + c, diagonal, mirror, v, hi, lo, factors);
          }
        } else {
          // slots of W / 4 columns x 128 rows of 4 columns' sums; one for each other block, in
          // the order of their ranks
          constexpr uint32_t kSlot = W * kB * 4;
          // what this block sent last has been read, so it has also left
          ok = whole_warp(mbar_wait_cluster(x_empty, ph_xe, dead, limit)) && ok;
          ph_xe ^= 1;
          float4* out = (float4*)(ring + kRing<S>);
          float v[C];
#pragma unroll
          for (int to = 0; to < S; ++to) {
            if (to == rank) {
#pragma unroll
              for (int i = 0; i < C; ++i) v[i] = acc[to * C + i];
            } else {
              const int slot = to - (to > rank ? 1 : 0);
#pragma unroll
              for (int g = 0; g < C / 4; ++g)
                out[(slot * (W / 4) + half * (C / 4) + g) * kB + local] =
                    make_float4(acc[to * C + 4 * g], acc[to * C + 4 * g + 1], acc[to * C + 4 * g + 2],
                                acc[to * C + 4 * g + 3]);
            }
          }
          // A's terms, while the sums travel
          uint32_t old_hi[C / 2], old_lo[C / 2];
          load_a<C>(p, s.t, b, row, col, old_hi, old_lo);
          fence_async_shared();
          asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpiWarps) : "memory");
          if (warp == 4 && ok) {
            mbar_expect(on, x_full, (S - 1) * kSlot);
#pragma unroll
            for (int k = 1; k < S; ++k) {
              const int to = (rank + k) % S, slot = to - (to > rank ? 1 : 0), at = rank - (rank > to ? 1 : 0);
              peer_copy(on, peer_addr(incoming + at * kSlot, to), exchange + slot * kSlot, kSlot, peer_addr(x_full, to));
            }
          }
          ok = whole_warp(mbar_wait_cluster(x_full, ph_xf, dead, limit)) && ok;
          ph_xf ^= 1;
          const float4* got = (const float4*)(ring + kRing<S> + kExchange<S>);
          float sum[C];
#pragma unroll
          for (int i = 0; i < C; ++i) sum[i] = 0.0f;
#pragma unroll
          for (int from = 0; from < S; ++from) {
            if (from == rank) {
#pragma unroll
              for (int i = 0; i < C; ++i) sum[i] += v[i];
            } else {
              const int slot = from - (from > rank ? 1 : 0);
#pragma unroll
              for (int g = 0; g < C / 4; ++g) {
                const float4 x = got[(slot * (W / 4) + half * (C / 4) + g) * kB + local];
                sum[4 * g] += x.x;
                sum[4 * g + 1] += x.y;
                sum[4 * g + 2] += x.z;
                sum[4 * g + 3] += x.w;
              }
            }
          }
          __syncwarp();
          if (lane < S && lane != rank && ok) peer_arrive(peer_addr(x_empty, lane));
          finish<C>(p, s.t, b, row, col, diagonal, mirror, sum, old_hi, old_lo, factors);
        }
      }
    }
    __syncwarp();
    unit0 += (uint32_t)(tiles * s.boxes * s.units);
    box0 += (uint32_t)(tiles * s.boxes);
    if (ph + 1 < phases) {
      arrivals += gridDim.x;
      alive = ortho_barrier(p.barrier, arrivals, dead, limit);
    }
  }
  __syncthreads();
  if (dead_flag) {
    // copies and products of this block that are still in flight end within this time
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) __nanosleep(1000);
    // where it was in the last phase nobody has heard of it: lost_kernel does
    if (threadIdx.x == 0) atomicAdd(p.barrier, kGaveUp);
  }
  __syncthreads();
  if (warp == 0) tmem_free(tmem_base, kColumns);
  // a peer may still write to or arrive at this block's shared memory
  if (S > 1) cluster_sync();
}

template <int S>
constexpr int kSharedBytes = kRing<S> + 2 * kExchange<S> + 1024;

template <int S>
int configure(cudaLaunchConfig_t& cfg, cudaLaunchAttribute* attr, int blocks, cudaStream_t st) {
  if (cudaError_t e = cudaFuncSetAttribute(split_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes<S>))
    return (int)e;
  cfg = cudaLaunchConfig_t{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSharedBytes<S>;
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = S;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return 0;
}

// clusters of S blocks that fit the device at once
template <int S>
int clusters(int sms) {
  if (S == 1) return sms;
  static std::atomic<int> known[64] = {};  // by device; the same answer whoever asks first
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (known[dev] == 0) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    int k = 0;
    if (configure<S>(cfg, attr, S, nullptr)) return 0;
    if (cudaOccupancyMaxActiveClusters(&k, split_kernel<S>, &cfg) != cudaSuccess) return 0;
    known[dev] = std::min(k, sms / S);
  }
  return known[dev];
}

int clusters_of(int split, int sms) {
  return split == 1 ? clusters<1>(sms) : split == 2 ? clusters<2>(sms) : clusters<4>(sms);
}

template <int S>
int start(const OrthoGrid& p, int sms, cudaStream_t st) {
  const int64_t mt = (p.o.n + kB - 1) / kB, nt = (p.o.m + kB - 1) / kB;
  const int64_t tiles = p.o.batch * std::max(mt * nt, mt * (mt + 1) / 2);
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  int k = (int)std::min<int64_t>(clusters<S>(sms), tiles);
  if (k < 1) return (int)cudaErrorLaunchOutOfResources;
  // Where the context has fewer SMs than the device (a part of it set aside for others), as
  // many blocks as it takes: a grid of any size goes through all tiles.
  for (;; k = (k + 1) / 2) {
    if (int rc = configure<S>(cfg, attr, S * k, st)) return rc;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, split_kernel<S>, p);
    if (e != cudaErrorCooperativeLaunchTooLarge || k == 1) return (int)e;
    cudaGetLastError();
  }
}

}  // namespace

// The split whose step takes the fewest cycles by a count fitted to what was measured (us for a
// split of 1 / 2 / 4 in 32 bits: 512^2 168 / 160 / 124, 768^2 193 / 178 / 158, 1024^2 222 / 200 /
// 222, 1300^2 261 / 285 / 319, 2048^2 458 / 708 / 759): rounds of tiles, each with a fixed part
// (latencies, the exchange, the tile's end) and one for every box of k.
int ortho_split_for(const OrthoGrid& p, int sms) {
  const int64_t mt = (p.o.n + kB - 1) / kB, nt = (p.o.m + kB - 1) / kB;
  const int64_t km = (p.o.m + kBK - 1) / kBK, kn = (p.o.n + kBK - 1) / kBK;
  const int64_t sym = p.o.batch * mt * (mt + 1) / 2, apply = p.o.batch * mt * nt;
  const struct {
    int split, fixed, box;
  } ways[] = {{1, 13000, 870}, {2, 13700, 1250}, {4, 11800, 1250}};
  int best = 1;
  int64_t cost = INT64_MAX;
  for (const auto& w : ways) {
    const int c = clusters_of(w.split, sms), s = w.split;
    if (c < 1) continue;
    auto phase = [&](int64_t tiles, int64_t k) { return (tiles + c - 1) / c * (w.fixed + w.box * ((k + s - 1) / s)); };
    const int64_t t = phase(sym, km) + phase(sym, kn) + phase(apply, kn);
    if (t < cost) {
      cost = t;
      best = s;
    }
  }
  return best;
}

int ortho_split_ready(int split) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  return split == 1   ? configure<1>(cfg, attr, 1, nullptr)
         : split == 2 ? configure<2>(cfg, attr, 2, nullptr)
                      : configure<4>(cfg, attr, 4, nullptr);
}

int launch_ortho_split(const OrthoGrid& p, int split, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
  if (cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) return (int)e;
  switch (split) {
    case 1: return start<1>(p, sms, st);
    case 2: return start<2>(p, sms, st);
    default: return start<4>(p, sms, st);
  }
}

}  // namespace blitz
