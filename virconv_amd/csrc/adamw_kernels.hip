// AdamW over many tensors at once, with the two moments in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// in fp32 whatever the parameters' type, every operation rounded by itself (this file is built without contraction), the parameter rounded
// once to its own type.  The step is one pass over its data and nothing else: what bounds it is HBM -- 28 bytes an element with fp32
// parameters and 32-bit moments, 16 with 8-bit ones, 10 with bf16 parameters and 8-bit moments.  Measured: 200 M bf16 parameters with 8-bit
// moments 389 us (5.16 TB/s; a large copy 4.9), 13 M fp32 ones in 193 tensors 81 us with 32-bit moments (4.5 TB/s), 56 us with 8-bit ones (3.7: three
// launches and their ends; with 64 tensors a launch 88 and 62 us); 0.42 M in 87 tensors 18 us of host time, one launch (23 and two).
//
// 8-bit moments.  m and r = sqrt(v) are held as e4m3 values over a power of two per 128 elements: value * 2^(exponent - 7), the block's
// largest magnitude lying in [128, 256) before the power is taken off.  r and not v: the root halves the range that a block has to span.
// A power of two and not the largest magnitude itself: when a block's exponent moves, values that lie on the grid stay on it.  The grid's
// steps (6 to 12 per cent of a value) are far wider than what one step changes of a moment (1 - b2 = 1 per cent of v), so rounding to the
// nearest value would leave a moment where it is for good; it is rounded up with the probability of its distance from the lower
// neighbour instead, which keeps the mean of m and of what r is rounded from.  The mean of v = r^2 is not kept: a rounding to a grid of spacing s adds
// s |d| to it, d what the step changes of r, and the decay holds on to that for 1 / (1 - b2) steps.  Under steady gradients v settles at 1 + 0.48 s / r
// times its value in 32 bits -- s / r lies between 1/16 and 1/8: 4 per cent more on average, 3 to 6 by where r lies in its binade -- whatever b2, and
// the steps are 1 to 2 per cent shorter.  The random numbers are a function of (seed, step, tensor, element), so a run can be
// repeated, and resumed, bit for bit.  An infinite or undefined moment is held as NaN and has no part in its block's exponent.  A NaN in place of
// r beside a number in place of m is a square beyond fp32 (a gradient from 1.8e19 on, not an undefined one): it counts as infinite, m / r as 0, and
// the parameter only decays from then on, as it does with 32-bit moments.
#include "common.h"

#include <math.h>

#include <algorithm>
#include <vector>

namespace vc {

static constexpr int kAdamwChunk = 2048;    // elements of one block: 256 threads x 8
static constexpr int kStateBlock = 128;     // elements that share an exponent: 16 lanes x 8

// A launch's tensors travel in the kernel's arguments, as many as fit: 4 KB.
struct AdamwTensor32 {
  void* param;
  const void* grad;
  void *exp_avg, *exp_avg_sq;
  uint64_t n_place;      // elements (40 bits), place in the model (20 bits), bit 63: the pointers allow 16-byte accesses (8-byte ones of 8-bit states)
};
struct AdamwTensor8 : AdamwTensor32 { int8_t* exponents; };

template <typename Entry>
struct AdamwTable {
  static constexpr int kMost = sizeof(Entry) == 40 ? 88 : 76;
  Entry t[kMost];
  unsigned block0[kMost];
  int n;
};
typedef AdamwTable<AdamwTensor32> AdamwTable32;
typedef AdamwTable<AdamwTensor8> AdamwTable8;

__host__ __device__ static inline uint32_t mix32(uint32_t x) {   // the finalizer of MurmurHash3
  x ^= x >> 16; x *= 0x85ebca6bu; x ^= x >> 13; x *= 0xc2b2ae35u; x ^= x >> 16;
  return x;
}

struct AdamwArgs {
  float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, keep, step_size, inv_bc2_sqrt;
  uint32_t key;          // of the seed and the step
};

static_assert(sizeof(AdamwTable32) + sizeof(AdamwArgs) < 4096 && sizeof(AdamwTable8) + sizeof(AdamwArgs) < 4096, "kernel arguments are limited to 4 KB");

template <typename T> struct Elem;
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};
template <> struct Elem<_Float16> {
  static __device__ __forceinline__ float up(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 down(float x) { return (_Float16)x; }
};
template <> struct Elem<__bf16> {
  static __device__ __forceinline__ float up(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 down(float x) { return (__bf16)x; }
};

// eight consecutive elements: one 16- or two 16-byte accesses where the tensor's pointers allow it
template <typename T> struct alignas(sizeof(T) * 8 < 16 ? sizeof(T) * 8 : 16) Eight { T v[8]; };

template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t i, int64_t n, bool vec, float (&out)[8]) {
  if (vec && i + 8 <= n) {
    const Eight<T> e = *reinterpret_cast<const Eight<T>*>(p + i);
#pragma unroll
    for (int k = 0; k < 8; ++k) out[k] = Elem<T>::up(e.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) out[k] = i + k < n ? Elem<T>::up(p[i + k]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int64_t i, int64_t n, bool vec, const float (&x)[8]) {
  if (vec && i + 8 <= n) {
    Eight<T> e;
#pragma unroll
    for (int k = 0; k < 8; ++k) e.v[k] = Elem<T>::down(x[k]);
    *reinterpret_cast<Eight<T>*>(p + i) = e;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) p[i + k] = Elem<T>::down(x[k]);
  }
}

template <typename Entry>
__device__ __forceinline__ int adamw_find(const AdamwTable<Entry>& B) {
  // the last tensor that begins at or before this block: one lane a tensor, twice
  const int lane = threadIdx.x & 63;
  const unsigned b0 = lane < B.n ? B.block0[lane] : 0xffffffffu, b1 = lane + 64 < B.n ? B.block0[lane + 64] : 0xffffffffu;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(b0 <= blockIdx.x)) + __popcll(__ballot(b1 <= blockIdx.x)) - 1);
}
template <typename Entry>
__device__ __forceinline__ int64_t adamw_size(const Entry& S) { return (int64_t)(S.n_place & ((1ull << 40) - 1)); }

template <typename T>
__global__ void __launch_bounds__(256) adamw32_kernel(AdamwTable32 B, AdamwArgs a) {
  const int s = adamw_find(B);
  const AdamwTensor32& S = B.t[s];
  const int64_t n = adamw_size(S), i = (int64_t)(blockIdx.x - B.block0[s]) * kAdamwChunk + threadIdx.x * 8;
  if (i >= n) return;
  const bool vec = S.n_place >> 63;
  float p[8], g[8], m[8], v[8];
  load8((const T*)S.grad, i, n, vec, g);
  load8((const float*)S.exp_avg, i, n, vec, m);
  load8((const float*)S.exp_avg_sq, i, n, vec, v);
  load8((const T*)S.param, i, n, vec, p);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    m[k] = m[k] * a.beta1 + g[k] * a.one_minus_beta1;
    v[k] = v[k] * a.beta2 + g[k] * g[k] * a.one_minus_beta2;
    p[k] = p[k] * a.keep - a.step_size * (m[k] / (sqrtf(v[k]) * a.inv_bc2_sqrt + a.eps));
  }
  store8((float*)S.exp_avg, i, n, vec, m);
  store8((float*)S.exp_avg_sq, i, n, vec, v);
  store8((T*)S.param, i, n, vec, p);
}

template <int CTRL>
__device__ __forceinline__ uint32_t max_rotated(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t max16(uint32_t x) {   // over the 16 lanes of a row, in every lane: rotations by 8, 4, 2, 1
  x = max_rotated<0x128>(x); x = max_rotated<0x124>(x); x = max_rotated<0x122>(x); x = max_rotated<0x121>(x);
  return x;
}

__device__ __forceinline__ void decode8(const void* codes, int64_t i, int64_t n, bool vec, int exponent, float (&out)[8]) {
  const uint8_t* c = (const uint8_t*)codes;
  uint32_t w[2] = {0, 0};
  if (vec && i + 8 <= n) {
    const uint2 e = *reinterpret_cast<const uint2*>(c + i);
    w[0] = e.x; w[1] = e.y;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) w[k >> 2] |= (uint32_t)c[i + k] << (8 * (k & 3));
  }
  const float unit = __uint_as_float((uint32_t)(max(exponent, -119) + 120) << 23);   // 2^(exponent - 7)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    out[4 * h + 0] = __builtin_amdgcn_cvt_f32_fp8(w[h], 0) * unit;
    out[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(w[h], 1) * unit;
    out[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(w[h], 2) * unit;
    out[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(w[h], 3) * unit;
  }
}

// the magnitude's bits where it is finite, 0 otherwise
__device__ __forceinline__ uint32_t finite_bits(uint32_t magnitude) { return magnitude < 0x7f800000u ? magnitude : 0u; }

// The root of v >= 0: v_rsq_f32 with one correction by the exact residual, 8 issue slots where the library's correctly rounded root takes 17
// (the last bit differs for one value in 280).  Below 2^-126, where v itself has lost bits, it falls with v instead of its root, to 0 at 0.
__device__ __forceinline__ float root(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-126f)), s = v * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, v), 0.5f * y, s);
}

__device__ __forceinline__ void put8(void* codes, int64_t i, int64_t n, bool vec, const int (&w)[2]) {
  uint8_t* c = (uint8_t*)codes;
  if (vec && i + 8 <= n) {
    *reinterpret_cast<int2*>(c + i) = make_int2(w[0], w[1]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k < n) c[i + k] = (uint8_t)((uint32_t)w[k >> 2] >> (8 * (k & 3)));
  }
}

// What bounds this kernel is issue slots as much as HBM: at 16 (fp32) or 10 bytes (bf16 parameters) an element the memory leaves about 105 or 65
// slots for one.  Hence v_cvt_sr_fp8_f32, which is the rounding that the states are defined with (16 random bits on top of the ones it takes),
// v_rsq and v_rcp in place of the library's root and quotient, and the first product of the mixing function from its neighbour's: the eight
// arguments of a lane differ in three bits, so their products differ by +-1, +-2, +-4 times the factor.
template <typename T>
__global__ void __launch_bounds__(256) adamw8_kernel(AdamwTable8 B, AdamwArgs a) {
  const int s = adamw_find(B);
  const AdamwTensor8& S = B.t[s];
  const int64_t n = adamw_size(S), i = (int64_t)(blockIdx.x - B.block0[s]) * kAdamwChunk + threadIdx.x * 8;
  // 16 lanes share an exponent, and all 16 are here for the maximum: the lanes behind the last element carry zeros
  const bool vec = S.n_place >> 63;
  const int64_t blk = i / kStateBlock;
  const bool live = blk * kStateBlock < n;
  float p[8], g[8], m[8], r[8];
  load8((const T*)S.grad, i, n, vec, g);
  load8((const T*)S.param, i, n, vec, p);
  const int8_t em0 = live ? S.exponents[2 * blk] : 0, er0 = live ? S.exponents[2 * blk + 1] : 0;
  decode8(S.exp_avg, i, n, vec, em0, m);
  decode8(S.exp_avg_sq, i, n, vec, er0, r);
  uint32_t mtop = 0, vtop = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    m[k] = m[k] * a.beta1 + g[k] * a.one_minus_beta1;
    const float v = r[k] * r[k] * a.beta2 + g[k] * g[k] * a.one_minus_beta2;
    r[k] = root(v);
    p[k] = p[k] * a.keep - a.step_size * (m[k] * __builtin_amdgcn_rcpf(r[k] * a.inv_bc2_sqrt + a.eps));
    mtop = max(mtop, __float_as_uint(m[k]) & 0x7fffffffu);
    vtop = max(vtop, __float_as_uint(v));
  }
  if (max(mtop, vtop) >= 0x7f800000u) {   // something infinite or undefined: it has no part in the block's exponents
    mtop = vtop = 0;
    float before[8];
    load8((const T*)S.param, i, n, vec, before);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // r = sqrt(v) is not a number then, infinite or not; m is where the gradient was
      if ((__float_as_uint(m[k]) & 0x7fffffffu) < 0x7f800000u && (__float_as_uint(r[k]) & 0x7fffffffu) >= 0x7f800000u) p[k] = before[k] * a.keep;
      mtop = max(mtop, finite_bits(__float_as_uint(m[k]) & 0x7fffffffu));
      vtop = max(vtop, finite_bits(__float_as_uint(r[k] * r[k])));
    }
  }
  store8((T*)S.param, i, n, vec, p);
  // the root's exponent is half of v's, whatever the root's last bit
  mtop = max16(mtop);
  vtop = max16(vtop);
  const int em = max((int)(mtop >> 23) - 127, -119), er = vtop ? ((int)(vtop >> 23) - 127) >> 1 : -119;
  const float mscale = __uint_as_float((uint32_t)(134 - em) << 23), rscale = __uint_as_float((uint32_t)(134 - er) << 23);   // 2^(7 - e)
  constexpr uint32_t kFirst = 0x85ebca6bu, kSecond = 0xc2b2ae35u;
  uint32_t x0 = mix32(a.key + ((uint32_t)(S.n_place >> 40) & 0xfffffu)) ^ (uint32_t)i ^ (uint32_t)(i >> 32) * 0x9e3779b9u;
  x0 ^= x0 >> 16;     // (i is a multiple of 8: the element's three bits come in unshifted)
  const uint32_t p0 = x0 * kFirst, d1 = x0 & 1 ? 0u - kFirst : kFirst, d2 = x0 & 2 ? 0u - 2 * kFirst : 2 * kFirst,
                 d4 = x0 & 4 ? 0u - 4 * kFirst : 4 * kFirst;
  int wm[2] = {0, 0}, wr[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t x = p0 + (k & 1 ? d1 : 0u) + (k & 2 ? d2 : 0u) + (k & 4 ? d4 : 0u);
    x ^= x >> 13;
    x *= kSecond;
    const float ym = m[k] * mscale, yr = r[k] * rscale;
    const int bm = (int)((x ^ (x >> 16)) << 16), br = (int)(x & 0xffff0000u);   // the low and the high half of x ^ (x >> 16), each on top
    switch (k & 3) {
      case 0: wm[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(ym, bm, wm[k >> 2], 0); wr[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(yr, br, wr[k >> 2], 0); break;
      case 1: wm[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(ym, bm, wm[k >> 2], 1); wr[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(yr, br, wr[k >> 2], 1); break;
      case 2: wm[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(ym, bm, wm[k >> 2], 2); wr[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(yr, br, wr[k >> 2], 2); break;
      default: wm[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(ym, bm, wm[k >> 2], 3); wr[k >> 2] = __builtin_amdgcn_cvt_sr_fp8_f32(yr, br, wr[k >> 2], 3);
    }
  }
  put8(S.exp_avg, i, n, vec, wm);
  put8(S.exp_avg_sq, i, n, vec, wr);
  if (live && (threadIdx.x & 15) == 0) {
    S.exponents[2 * blk] = (int8_t)em;
    S.exponents[2 * blk + 1] = (int8_t)er;
  }
}

struct Span {
  uintptr_t a, b;
  bool operator<(const Span& o) const { return a < o.a; }
};

static void fill(AdamwTensor32& e, const vc_adamw_tensor& T, uint64_t n_place) { e = {T.param, T.grad, T.exp_avg, T.exp_avg_sq, n_place}; }
static void fill(AdamwTensor8& e, const vc_adamw_tensor& T, uint64_t n_place) {
  fill(static_cast<AdamwTensor32&>(e), T, n_place);
  e.exponents = T.exponents;
}

template <typename Entry, typename Launch>
static int adamw_tables(const vc_adamw_tensor* tensors, int64_t n_tensors, uintptr_t wide, uintptr_t wide_state, Launch launch) {
  AdamwTable<Entry> B;
  for (int64_t k = 0; k < n_tensors;) {
    B.n = 0;
    unsigned blocks = 0;
    for (; k < n_tensors && B.n < B.kMost; ++k) {
      const vc_adamw_tensor& T = tensors[k];
      if (T.n == 0) continue;
      const int64_t need = cdiv(T.n, kAdamwChunk);
      if (B.n && (int64_t)blocks + need >= (1LL << 24)) break;     // (2^32 threads)
      const bool vec = ((((uintptr_t)T.param | (uintptr_t)T.grad) & wide) | (((uintptr_t)T.exp_avg | (uintptr_t)T.exp_avg_sq) & wide_state)) == 0;
      fill(B.t[B.n], T, (uint64_t)T.n | (uint64_t)T.key << 40 | (uint64_t)vec << 63);
      B.block0[B.n++] = blocks;
      blocks += (unsigned)need;
    }
    if (B.n == 0) break;
    launch(B, blocks);
    VC_CHECK_LAUNCH("adamw_kernel");
  }
  return VC_OK;
}

template <typename T>
static int adamw_launch(const vc_adamw_tensor* tensors, int64_t n_tensors, int state_bits, const AdamwArgs& a, hipStream_t st) {
  if (state_bits == 32)
    return adamw_tables<AdamwTensor32>(tensors, n_tensors, 15, 15, [&](const AdamwTable32& B, unsigned blocks) {
      hipLaunchKernelGGL(adamw32_kernel<T>, dim3(blocks), dim3(256), 0, st, B, a);
    });
  return adamw_tables<AdamwTensor8>(tensors, n_tensors, 15, 7, [&](const AdamwTable8& B, unsigned blocks) {
    hipLaunchKernelGGL(adamw8_kernel<T>, dim3(blocks), dim3(256), 0, st, B, a);
  });
}

}  // namespace vc

using namespace vc;

extern "C" {

int vc_adamw(const vc_adamw_tensor* tensors, int64_t n_tensors, int dtype, int state_bits, double lr, double beta1, double beta2, double eps,
             double weight_decay, int64_t step, uint32_t seed, void* stream) {
  VC_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors), "vc_adamw: %lld tensors at %p", (long long)n_tensors, (const void*)tensors);
  VC_REQUIRE(dtype == VC_F32 || dtype == VC_F16 || dtype == VC_BF16, "vc_adamw: unknown dtype %d", dtype);
  VC_REQUIRE(state_bits == 8 || state_bits == 32, "vc_adamw: states in %d bits (8 or 32)", state_bits);
  VC_REQUIRE(step >= 1, "vc_adamw: step = %lld (the first step is 1)", (long long)step);
  VC_REQUIRE(beta1 >= 0. && beta1 < 1. && beta2 >= 0. && beta2 < 1., "vc_adamw: betas (%g, %g) outside [0, 1)", beta1, beta2);
  const int64_t psize = dtype == VC_F32 ? 4 : 2, ssize = state_bits / 8;
  hipStream_t st = (hipStream_t)stream;
  // what is written must not overlap: two blocks would race on it.  A run of spans for each kind of tensor, by address (a model's tensors mostly come
  // so), and one walk over the runs together: 87 tensors 1.3 us less host time than by one sort of all spans.
  const int kinds = state_bits == 8 ? 4 : 3;
  Span stack[512];
  std::vector<Span> heap;
  Span* spans = stack;
  if (4 * n_tensors > 512) {
    try { heap.resize((size_t)(4 * n_tensors)); } catch (...) { set_error("vc_adamw: out of host memory"); return VC_ECAPACITY; }
    spans = heap.data();
  }
  Span* const run[4] = {spans, spans + n_tensors, spans + 2 * n_tensors, spans + 3 * n_tensors};
  int64_t m = 0;
  for (int64_t k = 0; k < n_tensors; ++k) {
    const vc_adamw_tensor& T = tensors[k];
    VC_REQUIRE(T.n >= 0 && T.n < (1LL << 35), "vc_adamw: tensor %lld has n = %lld", (long long)k, (long long)T.n);
    VC_REQUIRE(T.key < (1u << 20), "vc_adamw: tensor %lld has the place %u (at most 2^20 tensors)", (long long)k, T.key);
    if (T.n == 0) continue;
    VC_REQUIRE(T.param && T.grad && T.exp_avg && T.exp_avg_sq && (state_bits == 32 || T.exponents), "vc_adamw: tensor %lld has a NULL pointer", (long long)k);
    VC_REQUIRE((((uintptr_t)T.param | (uintptr_t)T.grad) & (psize - 1)) == 0 && (((uintptr_t)T.exp_avg | (uintptr_t)T.exp_avg_sq) & (ssize - 1)) == 0,
               "vc_adamw: tensor %lld is not aligned to its element size", (long long)k);
    run[0][m] = {(uintptr_t)T.param, (uintptr_t)T.param + T.n * psize};
    run[1][m] = {(uintptr_t)T.exp_avg, (uintptr_t)T.exp_avg + T.n * ssize};
    run[2][m] = {(uintptr_t)T.exp_avg_sq, (uintptr_t)T.exp_avg_sq + T.n * ssize};
    run[3][m++] = {(uintptr_t)T.exponents, (uintptr_t)T.exponents + 2 * cdiv(T.n, kStateBlock)};
  }
  for (int r = 0; r < kinds; ++r)
    if (!std::is_sorted(run[r], run[r] + m)) std::sort(run[r], run[r] + m);
  int64_t at[4] = {0, 0, 0, 0};
  uintptr_t end = 0;
  for (int64_t k = 0; k < kinds * m; ++k) {
    int first = -1;
    for (int r = 0; r < kinds; ++r)
      if (at[r] < m && (first < 0 || run[r][at[r]] < run[first][at[first]])) first = r;
    const Span s = run[first][at[first]++];
    VC_REQUIRE(s.a >= end, "vc_adamw: two of the parameters and states overlap in memory");
    end = s.b;
  }
  AdamwArgs a;
  a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.one_minus_beta1 = (float)(1.0 - beta1); a.one_minus_beta2 = (float)(1.0 - beta2);
  a.eps = (float)eps;
  a.keep = (float)(1.0 - lr * weight_decay);
  a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
  a.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
  a.key = mix32(mix32(seed) + (uint32_t)step);
  return dtype == VC_F32   ? adamw_launch<float>(tensors, n_tensors, state_bits, a, st)
         : dtype == VC_F16 ? adamw_launch<_Float16>(tensors, n_tensors, state_bits, a, st)
                           : adamw_launch<__bf16>(tensors, n_tensors, state_bits, a, st);
}

}  // extern "C"
