// Rows of values stored in 8 bits and read back (see quant.cuh for the format):
//   write: values [n, D] (32 or 16 bits) -> codes [N, D] and scales [N, G] at
//          the listed rows, G = ceil(D / group);
//   read:  the listed rows (or all) -> [n, D] values in 32 or 16 bits;
//   adam8: the sparse Adam step of adam.cu on moments held so, in one pass.
// All are HBM bound: a write moves D * (4 or 2) + D + 4 G bytes a row, a
// read the same, a step 16 D + 16 G (parameter read and written, gradient read,
// two codes read and written) where 32-bit moments cost 28 D.
//
// One unit is a group of one row, held by LANES neighbouring lanes in
// registers (at most 8 values a lane), so the group's maximum is a shuffle
// reduction and every value is read once.  Few lanes for narrow groups: the
// reduction and the per-group arithmetic are then shared by more rows a warp.
#include "kernels.h"
#include "quant.cuh"

namespace blitz {

namespace {

using namespace quant;

constexpr int kPer = 8;  // values a lane holds

struct Unit {
  int64_t j, row;  // index in the list, row of the store (-1: none)
  int g, c0, width;
};

template <int LANES>
__device__ __forceinline__ Unit unit_of(int64_t n, int64_t N, int64_t D, int G, int group,
                                        const int64_t* __restrict__ rows) {
  const int64_t u = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / LANES;
  Unit t;
  t.j = G == 1 ? u : u / G;
  t.g = G == 1 ? 0 : (int)(u - t.j * G);
  t.row = t.j >= n ? -1 : rows ? rows[t.j] : t.j;
  if (t.row >= N) t.row = -1;
  t.c0 = t.g * group;
  t.width = (int)min((int64_t)group, D - t.c0);
  return t;
}

template <int KIND, int LANES>
__device__ __forceinline__ void scale_of(const float (&x)[kPer], float& s, float& inv) {
  float amax = 0.0f, bad = 0.0f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    amax = fmaxf(amax, fabsf(x[k]));
    // x - x is NaN for NaN and the infinities, which fmaxf would drop
    bad += x[k] - x[k];
  }
  amax = lanes_max<LANES>(amax);
  const float worst = lanes_max<LANES>(bad == 0.0f ? 0.0f : 1.0f);
  s = group_scale<KIND>(amax, worst == 0.0f);
  inv = KIND == kE4m3 ? inverse_pow2(s) : 0.0f;
}

__device__ __forceinline__ uint32_t seed_of(uint32_t seed, const int64_t* seed_ptr) {
  return seed + (seed_ptr ? (uint32_t)*seed_ptr : 0u);
}

template <class T, int KIND, bool DITHER, int LANES>
__global__ void __launch_bounds__(256) write_kernel(QuantParams p) {
  const Unit t = unit_of<LANES>(p.n, p.N, p.D, p.G, p.group, p.rows);
  const int lane = threadIdx.x & (LANES - 1);
  float x[kPer];
  const T* src = (const T*)p.values + t.j * p.value_stride + t.c0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = lane + k * LANES;
    x[k] = t.row >= 0 && c < t.width ? to_float(src[c]) : 0.0f;
  }
  float s, inv;
  scale_of<KIND, LANES>(x, s, inv);
  if (t.row < 0) return;
  uint8_t* dst = p.codes + t.row * p.D + t.c0;
  const uint32_t key = DITHER ? row_key(seed_of(p.seed, p.seed_ptr), t.row) : 0u;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = lane + k * LANES;
    if (c < t.width)
      dst[c] = s == s ? encode<KIND, DITHER>(x[k], s, inv, DITHER ? uniform20(key, t.c0 + c) : 0.0f) : (uint8_t)0;
  }
  if (lane == 0) p.scales[t.row * p.G + t.g] = s;
}

template <class T, int KIND, int LANES>
__global__ void __launch_bounds__(256) read_kernel(QuantParams p) {
  const Unit t = unit_of<LANES>(p.n, p.N, p.D, p.G, p.group, p.rows);
  if (t.j >= p.n) return;
  const int lane = threadIdx.x & (LANES - 1);
  T* dst = (T*)p.out + t.j * p.D + t.c0;
  const uint8_t* src = p.codes + t.row * p.D + t.c0;
  const float s = t.row >= 0 ? p.scales[t.row * p.G + t.g] : 0.0f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = lane + k * LANES;
    if (c < t.width) dst[c] = from_float<T>(t.row >= 0 ? decode<KIND>(src[c], s) : 0.0f);
  }
}

// One group of one row's step.  The moment updates and the parameter's step
// are single rounded operations in the order of the formula (no contraction),
// so the result does not depend on how the compiler fuses them.
template <int LANES>
__global__ void __launch_bounds__(256) adam8_kernel(Adam8Params p) {
  Unit t = unit_of<LANES>(p.n, p.N, p.M, p.G, p.group, p.rows);
  if (t.row >= 0 && p.visible && !p.visible[t.row]) t.row = -1;
  if (__all_sync(0xffffffffu, t.row < 0)) return;
  const int lane = threadIdx.x & (LANES - 1);
  const int64_t at = t.row * p.M + t.c0, grad_at = t.j * p.M + t.c0, sc = t.row * p.G + t.g;
  float m[kPer], r[kPer];
  const float ms = t.row >= 0 ? p.m_scales[sc] : 0.0f, rs = t.row >= 0 ? p.r_scales[sc] : 0.0f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = lane + k * LANES;
    m[k] = r[k] = 0.0f;
    if (t.row >= 0 && c < t.width) {
      const float g = __fmul_rn(p.grad[grad_at + c], p.grad_scale);
      const float r0 = decode<kE4m3>(p.r_codes[at + c], rs);
      m[k] = __fadd_rn(__fmul_rn(decode<kE4m3>(p.m_codes[at + c], ms), p.b1), __fmul_rn(g, p.b1c));
      r[k] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(r0, r0), p.b2), __fmul_rn(__fmul_rn(g, g), p.b2c)));
      p.param[at + c] = __fsub_rn(p.param[at + c], __fdiv_rn(__fmul_rn(m[k], p.lr), __fadd_rn(r[k], p.eps)));
    }
  }
  float sm, im, sr, ir;
  scale_of<kE4m3, LANES>(m, sm, im);
  scale_of<kE4m3, LANES>(r, sr, ir);
  if (t.row < 0) return;
  const uint32_t seed = seed_of(p.seed, p.seed_ptr);
  const uint32_t km = row_key(seed, t.row), kr = row_key(seed ^ 0x5BF03635u, t.row);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int c = lane + k * LANES;
    if (c < t.width) {
      const uint32_t col = t.c0 + c;
      p.m_codes[at + c] = sm == sm ? encode<kE4m3, true>(m[k], sm, im, uniform20(km, col)) : (uint8_t)0;
      // a second moment that has seen a gradient never becomes zero: the next
      // step would divide its first moment by the new gradient alone
      p.r_codes[at + c] = sr == sr ? encode<kE4m3, true, true>(r[k], sr, ir, uniform20(kr, col)) : (uint8_t)0;
    }
  }
  if (lane == 0) {
    p.m_scales[sc] = sm;
    p.r_scales[sc] = sr;
  }
}

// lanes that hold a group of `width` values, at most kPer each
inline int lanes_for(int64_t width) { return width <= 8 ? 2 : width <= 16 ? 4 : width <= 64 ? 8 : 32; }

template <int LANES>
inline unsigned blocks_for(int64_t units) {
  return (unsigned)((units * LANES + 255) / 256);
}

template <class T, int KIND, int LANES>
void start_write(const QuantParams& p, cudaStream_t st) {
  const unsigned b = blocks_for<LANES>(p.n * p.G);
  if (p.dither)
    write_kernel<T, KIND, true, LANES><<<b, 256, 0, st>>>(p);
  else
    write_kernel<T, KIND, false, LANES><<<b, 256, 0, st>>>(p);
}

template <class T, int KIND, int LANES>
void start_read(const QuantParams& p, cudaStream_t st) {
  read_kernel<T, KIND, LANES><<<blocks_for<LANES>(p.n * p.G), 256, 0, st>>>(p);
}

template <class T, int KIND>
void start(const QuantParams& p, bool write, cudaStream_t st) {
  const int lanes = lanes_for(p.D < p.group ? p.D : p.group);
#define BLITZ_LANES(L)                 \
  if (lanes == L) {                    \
    if (write)                         \
      start_write<T, KIND, L>(p, st);  \
    else                               \
      start_read<T, KIND, L>(p, st);   \
    return;                            \
  }
  BLITZ_LANES(2)
  BLITZ_LANES(4)
  BLITZ_LANES(8)
  BLITZ_LANES(32)
#undef BLITZ_LANES
}

template <class T>
void start_kind(const QuantParams& p, bool write, cudaStream_t st) {
  if (p.kind == kInt8)
    start<T, kInt8>(p, write, st);
  else
    start<T, kE4m3>(p, write, st);
}

int launch(const QuantParams& p, bool write, cudaStream_t st) {
  if (p.n <= 0) return 0;
  if (p.type == kValueF32)
    start_kind<float>(p, write, st);
  else if (p.type == kValueBf16)
    start_kind<__nv_bfloat16>(p, write, st);
  else
    start_kind<__half>(p, write, st);
  return (int)cudaGetLastError();
}

}  // namespace

int launch_quant_write(const QuantParams& p, cudaStream_t st) { return launch(p, true, st); }
int launch_quant_read(const QuantParams& p, cudaStream_t st) { return launch(p, false, st); }

int launch_adam8(const Adam8Params& p, cudaStream_t st) {
  if (p.n <= 0) return 0;
  const int64_t units = p.n * p.G;
  const int lanes = lanes_for(p.M < p.group ? p.M : p.group);
  if (lanes == 2)
    adam8_kernel<2><<<blocks_for<2>(units), 256, 0, st>>>(p);
  else if (lanes == 4)
    adam8_kernel<4><<<blocks_for<4>(units), 256, 0, st>>>(p);
  else if (lanes == 8)
    adam8_kernel<8><<<blocks_for<8>(units), 256, 0, st>>>(p);
  else
    adam8_kernel<32><<<blocks_for<32>(units), 256, 0, st>>>(p);
  return (int)cudaGetLastError();
}

}  // namespace blitz
