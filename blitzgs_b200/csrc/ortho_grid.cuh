// What the orthogonalisation kernels that spread over the grid share: the
// scratch, the phases of a step and the barrier between them.
#pragma once
#include "ortho.cuh"
#include "tcgen05.cuh"

namespace blitz {

constexpr int kBK = 64;                    // k of one copied box
constexpr unsigned kGaveUp = 1u << 20;     // above all arrivals: 192 phases of a grid of a few hundred blocks
constexpr int kBox = 64 * kBK * 2;         // bytes of 64 of its rows of 128 bytes

struct OrthoGrid {
  OrthoParams o;
  CUtensorMap map_x[2], map_a, map_b;  // boxes of 64 rows (128 rows a box took a quarter longer)
  __half *x[2], *a, *b;   // [2 * batch][n][ld]: high and low terms of each matrix
  double* parts;          // [batch][n_parts] sums of squares
  OrthoInfo* info;        // [batch], written while X_0 is laid out
  unsigned* barrier;      // arrivals, and kGaveUp for a block that gave up
  int n_parts;
  int ldm, ldn;
  int two_in;             // u needs two terms
  int four;               // ortho_by_four
};

enum OrthoPhase : int { kGram, kPoly, kApply };

// which terms a phase reads
struct OrthoTerms {
  int which, step;
  bool two_a, two_b, last;
  const CUtensorMap *ma, *mb;
};
__device__ __forceinline__ OrthoTerms ortho_terms(const OrthoGrid& p, int ph) {
  OrthoTerms t;
  t.step = ph / 3;
  t.which = ph - 3 * t.step;
  const bool two_x = t.step > 0 || p.two_in;
  t.two_a = t.which == kGram ? two_x : true;
  t.two_b = t.which == kPoly ? true : two_x;
  t.last = t.step == p.o.steps - 1 && t.which == kApply;
  t.ma = t.which == kGram ? &p.map_x[t.step & 1] : t.which == kPoly ? &p.map_a : &p.map_b;
  t.mb = t.which == kPoly ? &p.map_a : &p.map_x[t.step & 1];
  return t;
}

// every block of the grid has arrived, and what each wrote (for its reads and its copies) is seen.
// A block that has given up arrives with its word for that in the same addition: whoever passes has
// seen it, and no block goes on from what it left unfinished.
__device__ __forceinline__ bool ortho_barrier(unsigned* counter, unsigned target, volatile int* dead, long long limit) {
  fence_async_global();
  __syncthreads();
  if (threadIdx.x == 0) {
    asm volatile("red.release.gpu.global.add.u32 [%0], %1;" ::"l"(counter), "r"(*dead ? kGaveUp + 1 : 1u) : "memory");
    const long long t0 = clock64();
    for (;;) {
      unsigned seen;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
      if (seen >= kGaveUp) {
        *dead = 1;
        break;
      }
      if (seen >= target) break;
      if (clock64() - t0 > limit) {
        *dead = 1;
        atomicAdd(counter, kGaveUp);
        break;
      }
    }
  }
  __syncthreads();
  fence_async_global();
  return *dead == 0;
}

int launch_ortho_split(const OrthoGrid& p, int split, cudaStream_t st);
// an error if a split's kernel cannot be launched here at all
int ortho_split_ready(int split);
// the split that launch_ortho_split takes for this size
int ortho_split_for(const OrthoGrid& p, int sms);

}  // namespace blitz
