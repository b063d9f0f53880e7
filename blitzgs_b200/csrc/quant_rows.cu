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
// registers (PER values a lane), so the group's maximum is a shuffle
// reduction and every value is read once.  Few lanes for narrow groups: the
// reduction and the per-group arithmetic are then shared by more rows a warp.
// What is left over the traffic is instructions: a byte costs as many as a
// word, so lanes and values are chosen to fit the group and codes are formed by
// integer operations (see quant.cuh) rather than by conversions.  All loads of a
// unit are issued before the first is used.
#include "kernels.h"
#include "quant.cuh"

namespace blitz {

namespace {

using namespace quant;

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
  t.width = t.row < 0 ? 0 : (int)min((int64_t)group, D - t.c0);
  return t;
}

template <int KIND, int LANES, int PER>
__device__ __forceinline__ float scale_of(const float (&x)[PER]) {
  float amax = 0.0f, bad = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    amax = fmaxf(amax, fabsf(x[k]));
    // x - x is NaN for NaN and the infinities, which fmaxf would drop
    bad += x[k] - x[k];
  }
  // a bad value leaves an infinite maximum behind
  if (bad != 0.0f) amax = __int_as_float(0x7f800000);
  amax = lanes_max<LANES>(amax);
  return group_scale<KIND>(amax, amax <= FLT_MAX);
}

__device__ __forceinline__ uint32_t seed_of(uint32_t seed, const int64_t* seed_ptr) {
  return seed + (seed_ptr ? (uint32_t)*seed_ptr : 0u);
}

template <class T, int KIND, bool DITHER, int LANES, int PER>
__global__ void __launch_bounds__(256) write_kernel(QuantParams p) {
  const Unit t = unit_of<LANES>(p.n, p.N, p.D, p.G, p.group, p.rows);
  const int lane = threadIdx.x & (LANES - 1), left = t.width - lane;
  float x[PER];
  const T* src = (const T*)p.values + t.j * p.value_stride + t.c0 + lane;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    x[k] = k * LANES < left ? to_float(src[k * LANES]) : 0.0f;
  }
  const float s = scale_of<KIND, LANES, PER>(x);
  if (t.row < 0) return;
  uint8_t* dst = p.codes + t.row * p.D + t.c0 + lane;
  const uint32_t key = DITHER ? row_key(seed_of(p.seed, p.seed_ptr), t.row) : 0u;
  const GroupCode<KIND> code(s);
  if (s == s) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (k * LANES < left)
        dst[k * LANES] = encode<KIND, DITHER>(x[k], code, DITHER ? random20(key, t.c0 + lane + k * LANES) : 0u);
    }
  } else {
    for (int k = 0; k * LANES < left; ++k) dst[k * LANES] = 0;
  }
  if (lane == 0) p.scales[t.row * p.G + t.g] = s;
}

template <class T, int KIND, int LANES, int PER>
__global__ void __launch_bounds__(256) read_kernel(QuantParams p) {
  const Unit t = unit_of<LANES>(p.n, p.N, p.D, p.G, p.group, p.rows);
  if (t.j >= p.n) return;
  const int lane = threadIdx.x & (LANES - 1), left = (int)min((int64_t)p.group, p.D - t.c0) - lane;
  T* dst = (T*)p.out + t.j * p.D + t.c0 + lane;
  if (t.row < 0) {
    for (int k = 0; k * LANES < left; ++k) dst[k * LANES] = from_float<T>(0.0f);
    return;
  }
  const uint8_t* src = p.codes + t.row * p.D + t.c0 + lane;
  const float s = p.scales[t.row * p.G + t.g];
  uint8_t c[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    c[k] = k * LANES < left ? src[k * LANES] : (uint8_t)0;
  }
#pragma unroll
  for (int k = 0; k < PER; k += 2) {
    const float2 v = decode2<KIND>(c[k], k + 1 < PER ? c[k + 1] : (uint8_t)0, s);
    if (k * LANES < left) dst[k * LANES] = from_float<T>(v.x);
    if (k + 1 < PER && (k + 1) * LANES < left) dst[(k + 1) * LANES] = from_float<T>(v.y);
  }
}

// V codes of one group by one thread, where rows and groups are whole numbers of
// V and everything is aligned to it: one load and one or two stores for what
// costs V of each above.  1M x 48 e4m3 -> bf16 (148 MB): 28.5 us, 79% of the measured copy rate, where
// read_kernel takes 55.
template <class T, int KIND, int V>
__global__ void __launch_bounds__(256) read_vector_kernel(QuantParams p) {
  const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int per_row = (int)(p.D / V);
  const int64_t j = e / per_row;
  if (j >= p.n) return;
  const int c = (int)(e - j * per_row) * V;
  int64_t row = p.rows ? p.rows[j] : j;
  if (row >= p.N) row = -1;
  uint32_t w[V / 4];
  float s = 0.0f;
  if (row >= 0) {
    s = p.scales[row * p.G + (p.G == 1 ? 0 : c / p.group)];
    const uint8_t* src = p.codes + row * p.D + c;
    if (V == 16) {
      const uint4 q = *(const uint4*)src;
      w[0] = q.x, w[1 % (V / 4)] = q.y, w[2 % (V / 4)] = q.z, w[3 % (V / 4)] = q.w;
    } else {
      w[0] = *(const uint32_t*)src;
    }
  } else {
    for (int k = 0; k < V / 4; ++k) w[k] = 0;
  }
  T o[V];
#pragma unroll
  for (int k = 0; k < V; k += 2) {
    const float2 v = decode2<KIND>((uint8_t)(w[k / 4] >> 8 * (k % 4)), (uint8_t)(w[k / 4] >> 8 * (k % 4 + 1)), s);
    o[k] = from_float<T>(v.x);
    o[k + 1] = from_float<T>(v.y);
  }
  uint8_t* dst = (uint8_t*)((T*)p.out + j * p.D + c);
  constexpr int kBytes = V * (int)sizeof(T);
  if (kBytes % 16 == 0) {
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k) ((uint4*)dst)[k] = ((const uint4*)o)[k];
  } else {
    *(uint2*)dst = *(const uint2*)o;
  }
}

// 320k of 8M rows of 45: 114 us for 411 MB (scattered rows open whole sectors), against 36 us for
// the 238 MB that the rows hold; issue slots 59% busy.  4 or 16 lanes a row took 137 and 131.
// One group of one row's step.  The moment updates are single rounded operations in
// the order of the formula (no contraction), so the codes do not depend on how the
// compiler fuses them.
template <int LANES, int PER>
__device__ __forceinline__ void adam8_unit(const Adam8Params& p, int64_t j, int64_t row, int g, int lane,
                                           uint32_t seed) {
  const int c0 = g * p.group;
  const int left = row < 0 ? 0 : (int)min((int64_t)p.group, p.M - c0) - lane;
  const int64_t at = row * p.M + c0 + lane, sc = row * p.G + g;
  const float* grad = p.grad + j * p.M + c0 + lane;
  float* param = p.param + at;
  uint8_t *mc = p.m_codes + at, *rc = p.r_codes + at;
  float m[PER], r[PER], w[PER], old[PER];
  uint8_t m0[PER], r0[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const bool on = k * LANES < left;
    w[k] = on ? grad[k * LANES] : 0.0f;
    m0[k] = on ? mc[k * LANES] : (uint8_t)0;
    r0[k] = on ? rc[k * LANES] : (uint8_t)0;
    old[k] = on ? param[k * LANES] : 0.0f;
  }
  const float ms = row >= 0 ? p.m_scales[sc] : 0.0f, rs = row >= 0 ? p.r_scales[sc] : 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const float2 held = e4m3_pair(m0[k], r0[k]);
    const float g1 = __fmul_rn(w[k], p.grad_scale), root = __fmul_rn(held.y, rs);
    m[k] = __fadd_rn(__fmul_rn(__fmul_rn(held.x, ms), p.b1), __fmul_rn(g1, p.b1c));
    r[k] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(root, root), p.b2), __fmul_rn(__fmul_rn(g1, g1), p.b2c)));
    // each operation rounded once, as in adam.cu
    if (k * LANES < left)
      param[k * LANES] = __fsub_rn(old[k], __fdiv_rn(__fmul_rn(m[k], p.lr), __fadd_rn(r[k], p.eps)));
  }
  const float sm = scale_of<kE4m3, LANES, PER>(m), sr = scale_of<kE4m3, LANES, PER>(r);
  if (row < 0) return;
  const uint32_t km = row_key(seed, row), kr = row_key(seed ^ 0x5BF03635u, row);
  const float im = inverse_pow2(sm), ir = inverse_pow2(sr);
  uint8_t a[PER], b[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const uint32_t col = c0 + lane + k * LANES;
    a[k] = (uint8_t)(e4m3_dithered(__fmul_rn(m[k], im), random20(km, col)) |
                     ((uint32_t)__float_as_int(m[k]) >> 24 & 0x80u));
    // a second moment that has seen a gradient never becomes zero: the next step would
    // divide its first moment by the new gradient alone (r is not negative, so r > 0
    // where its bits are not 0)
    b[k] = (uint8_t)max(e4m3_dithered(__fmul_rn(r[k], ir), random20(kr, col)),
                        min((uint32_t)__float_as_int(r[k]), 1u));
  }
  if (!(sm < 0x1p120f) || !(sr < 0x1p120f)) {
    // rare: a scale that is not finite, or whose largest code would not be
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      a[k] = sm == sm ? (uint8_t)((a[k] & 0x80u) | min(a[k] & 0x7fu, GroupCode<kE4m3>(sm).limit)) : (uint8_t)0;
      b[k] = sr == sr ? (uint8_t)min((uint32_t)b[k], GroupCode<kE4m3>(sr).limit) : (uint8_t)0;
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (k * LANES < left) {
      mc[k * LANES] = a[k];
      rc[k * LANES] = b[k];
    }
  }
  if (lane == 0) {
    p.m_scales[sc] = sm;
    p.r_scales[sc] = sr;
  }
}

template <int LANES, int PER>
__global__ void __launch_bounds__(256) adam8_rows_kernel(Adam8Params p) {
  const Unit t = unit_of<LANES>(p.n, p.N, p.M, p.G, p.group, p.rows);
  adam8_unit<LANES, PER>(p, t.j, t.row, t.g, threadIdx.x & (LANES - 1), seed_of(p.seed, p.seed_ptr));
}

// A block takes 256 rows and packs the visible ones into a list first, so that
// no lane waits out the step of a row that only its neighbour has.
template <int LANES, int PER>
__global__ void __launch_bounds__(256) adam8_mask_kernel(Adam8Params p) {
  __shared__ int counts[8];
  __shared__ uint8_t list[256];
  const int warp = threadIdx.x >> 5;
  const int64_t row0 = (int64_t)blockIdx.x * 256, mine = row0 + threadIdx.x;
  const bool on = mine < p.N && p.visible[mine];
  const unsigned ballot = __ballot_sync(0xffffffffu, on);
  if ((threadIdx.x & 31) == 0) counts[warp] = __popc(ballot);
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 8; ++w) {
    before += w < warp ? counts[w] : 0;
    all += counts[w];
  }
  if (on) list[before + __popc(ballot & ((1u << (threadIdx.x & 31)) - 1))] = (uint8_t)threadIdx.x;
  __syncthreads();
  const uint32_t seed = seed_of(p.seed, p.seed_ptr);
  const int64_t units = (int64_t)all * p.G;
  // every lane of a warp goes round as often, for the shuffles
  for (int64_t u0 = 0; u0 < units; u0 += 256 / LANES) {
    const int64_t u = u0 + threadIdx.x / LANES;
    const int64_t i = p.G == 1 ? u : u / p.G;
    const int64_t row = u < units ? row0 + list[i] : -1;
    adam8_unit<LANES, PER>(p, row, row, (int)(u - i * p.G), threadIdx.x & (LANES - 1), seed);
  }
}

// Lanes and values a lane by the group's width: 45 to 48 SH coefficients fit 8 x 6.
// (150000 rows of 45 written: 22 us with 8 lanes, 25 with 16, 29 with 4; 100000 rows of 3 x 67
// read: 30 us with 8 x 9, 33 with 16 x 6, 54 with 32 x 3.)
template <int LANES>
inline unsigned blocks_for(int64_t units) {
  return (unsigned)((units * LANES + 255) / 256);
}

template <class T, int KIND, int LANES, int PER>
void start_lanes(const QuantParams& p, bool write, cudaStream_t st) {
  const unsigned b = blocks_for<LANES>(p.n * p.G);
  if (!write)
    read_kernel<T, KIND, LANES, PER><<<b, 256, 0, st>>>(p);
  else if (p.dither)
    write_kernel<T, KIND, true, LANES, PER><<<b, 256, 0, st>>>(p);
  else
    write_kernel<T, KIND, false, LANES, PER><<<b, 256, 0, st>>>(p);
}

template <class T, int KIND, int V>
bool start_vector(const QuantParams& p, cudaStream_t st) {
  const uintptr_t bytes = (uintptr_t)p.codes | (uintptr_t)p.out;
  if (p.D % V || p.group % V && p.G > 1 || bytes % 16 || p.n * (p.D / V) > ((int64_t)1 << 31) * 200) return false;
  read_vector_kernel<T, KIND, V><<<(unsigned)((p.n * (p.D / V) + 255) / 256), 256, 0, st>>>(p);
  return true;
}

template <class T, int KIND>
void start(const QuantParams& p, bool write, cudaStream_t st) {
  if (!write && (start_vector<T, KIND, 16>(p, st) || start_vector<T, KIND, 4>(p, st))) return;
  const int64_t width = p.D < p.group ? p.D : p.group;
  if (width <= 12)
    start_lanes<T, KIND, 2, 6>(p, write, st);
  else if (width <= 24)
    start_lanes<T, KIND, 4, 6>(p, write, st);
  else if (width <= 48)
    start_lanes<T, KIND, 8, 6>(p, write, st);
  else if (width <= 72)
    start_lanes<T, KIND, 8, 9>(p, write, st);
  else if (width <= 96)
    start_lanes<T, KIND, 16, 6>(p, write, st);
  else
    start_lanes<T, KIND, 32, 8>(p, write, st);
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

template <int LANES, int PER>
void start_adam8(const Adam8Params& p, cudaStream_t st) {
  if (p.visible)
    adam8_mask_kernel<LANES, PER><<<(unsigned)((p.N + 255) / 256), 256, 0, st>>>(p);
  else
    adam8_rows_kernel<LANES, PER><<<blocks_for<LANES>(p.n * p.G), 256, 0, st>>>(p);
}

}  // namespace

int launch_quant_write(const QuantParams& p, cudaStream_t st) { return launch(p, true, st); }
int launch_quant_read(const QuantParams& p, cudaStream_t st) { return launch(p, false, st); }

int launch_adam8(const Adam8Params& p, cudaStream_t st) {
  if (p.n <= 0) return 0;
  const int64_t width = p.M < p.group ? p.M : p.group;
  if (width <= 12)
    start_adam8<2, 6>(p, st);
  else if (width <= 24)
    start_adam8<4, 6>(p, st);
  else if (width <= 48)
    start_adam8<8, 6>(p, st);
  else if (width <= 96)
    start_adam8<16, 6>(p, st);
  else
    start_adam8<32, 8>(p, st);
  return (int)cudaGetLastError();
}

}  // namespace blitz
