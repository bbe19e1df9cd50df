// Layer norm over the last axis of a row matrix, forward and backward.
//
//   mean = sum(x) / C;  var = sum((x - mean)^2) / C;  rstd = 1 / sqrt(var + eps);  xh = (x - mean) rstd;  y = xh w + b
//   gw = dy w;  dx = rstd (gw - sum(gw) / C - xh sum(gw xh) / C);  dw = sum over rows of dy xh;  db = sum over rows of dy
//
// in fp32 whatever the tensors' types, each output rounded once.  Both directions are bound by HBM: a row is read once, held in registers
// while its sums are formed (the variance from the centred values, not from a difference of two sums), and written once.  The weight
// gradient's sums over the rows ride along in the backward pass: every block walks a fixed share of the rows, keeps its columns' sums in
// registers, and writes them to a row of its own; a second kernel adds those rows in a fixed order, so nothing depends on the order of
// atomics.
//
// A row is held by LPR lanes, each with ITER vectors of VEC elements: as few lanes as there are vectors for short rows (four rows of 64
// channels a wave), a block for wide ones.  A row whose length is no multiple of VEC ends in a vector that overlaps the one before it; the
// elements that are there twice count once in the sums and are written twice with one value.  Rows wider than a block's registers are read
// three times (they come from the cache by then).
//
// Measured, with fp32 weights, tensors cycled through so that nothing is left in a cache (a large copy reaches 4.9 TB/s):
//   forward   16381 x 4096 bf16 54 us (4.9 TB/s), fp32 99 us (5.4); 133578 x 64 fp32 14.5 us (4.7), bf16 8.0 us (4.3)
//   backward  16381 x 4096 bf16 89 us (4.5 TB/s), fp32 163 us (4.9); 133578 x 64 fp32 27 us (3.8), bf16 14.2 us (3.6: as much time goes into the
//             column sums, 2 fused operations an element and the launch that adds them, as into the memory's part)
#include "common.h"

namespace vc {

template <typename T, int VEC> struct __attribute__((packed, aligned(sizeof(T)))) Pack { T v[VEC]; };

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[VEC]) {
  Pack<T, VEC> e;
  __builtin_memcpy(&e, p, sizeof(e));
#pragma unroll
  for (int k = 0; k < VEC; ++k) out[k] = (float)e.v[k];
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[VEC]) {
  Pack<T, VEC> e;
#pragma unroll
  for (int k = 0; k < VEC; ++k) e.v[k] = (T)x[k];
  __builtin_memcpy(p, &e, sizeof(e));
}

// weights in the tensor's type or in fp32
template <int VEC>
__device__ __forceinline__ void load_weight(const void* w, int wtype, int64_t c, float fill, float (&out)[VEC]) {
  if (!w) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) out[k] = fill;
  } else if (wtype == VC_F32) load_vec<float, VEC>((const float*)w + c, out);
  else if (wtype == VC_F16) load_vec<_Float16, VEC>((const _Float16*)w + c, out);
  else load_vec<__bf16, VEC>((const __bf16*)w + c, out);
}

template <int CTRL>
__device__ __forceinline__ float plus_moved(float x) {
  return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }

// the sum over min(LPR, 64) neighbouring lanes, the same in each of them: exchanges within a row of 16 lanes, then between the rows
template <int LPR>
__device__ __forceinline__ float lane_sum(float x) {
  if constexpr (LPR >= 2) x = plus_moved<0xb1>(x);     // neighbours
  if constexpr (LPR >= 4) x = plus_moved<0x4e>(x);     // pairs
  if constexpr (LPR >= 8) x = plus_moved<0x141>(x);    // mirrored in eight
  if constexpr (LPR >= 16) x = plus_moved<0x140>(x);   // mirrored in sixteen
  if constexpr (LPR == 32) x += __shfl_xor(x, 16, 64);
  if constexpr (LPR >= 64) x = (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
  return x;
}

// N sums over the LPR lanes of a row, the same in each of them; rows of several waves meet in LDS: one barrier, the halves of `lds` in turn
template <int LPR, int ROWS, int N>
struct RowSums {
  static constexpr int W = LPR > 64 ? LPR / 64 : 1;
  float lds[2][ROWS][N][W];
};
template <int LPR, int ROWS, int N, int M>
__device__ __forceinline__ void row_sums(float (&x)[M], RowSums<LPR, ROWS, N>& shared, int& half) {
  static_assert(M <= N, "room for the sums");
#pragma unroll
  for (int i = 0; i < M; ++i) x[i] = lane_sum<LPR>(x[i]);
  if constexpr (LPR > 64) {
    constexpr int W = LPR / 64;
    const int r = threadIdx.x / LPR, w = threadIdx.x % LPR / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < M; ++i) shared.lds[half][r][i][w] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < M; ++i) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) s += shared.lds[half][r][i][j];
      x[i] = s;
    }
    half ^= 1;
  }
}

struct NormArgs {
  const void *x, *w, *b;
  void* y;
  float *mean, *rstd;
  int64_t n, stride;
  int c, wtype, btype;
  float eps;
};

// where vector j of a row begins, and from which of its elements on it counts (a last vector that overlaps its neighbour)
template <int VEC>
__device__ __forceinline__ int vec_at(int j, int c, int& first) {
  const int at = min(j * VEC, c - VEC);
  first = j * VEC - at;         // VEC or more: the row has no such vector (it is read all the same, and counts for nothing)
  return at;
}

// A block takes rows until there are none: the weights are read once (a row of 4096 16-bit channels is 8 KB, its two fp32 weights 32 KB), and the
// next row is under way while this one is summed.
template <typename T, int VEC, int LPR, int ITER, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_forward_kernel(NormArgs a) {
  constexpr int kRows = THREADS / LPR;
  __shared__ RowSums<LPR, kRows, 1> shared;
  const int lane = threadIdx.x % LPR, mine = threadIdx.x / LPR;
  int at[ITER], first[ITER], half = 0;
  float w[ITER][VEC], b[ITER][VEC];
  Pack<T, VEC> next[ITER];
  const int64_t step = (int64_t)gridDim.x * kRows;
  auto ask = [&](int64_t row) {     // (behind the last row, that one again)
    const T* x = (const T*)a.x + min(row, a.n - 1) * a.stride;
#pragma unroll
    for (int j = 0; j < ITER; ++j) __builtin_memcpy(&next[j], x + at[j], sizeof(next[j]));
  };
#pragma unroll
  for (int j = 0; j < ITER; ++j) {
    at[j] = vec_at<VEC>(j * LPR + lane, a.c, first[j]);
    load_weight<VEC>(a.w, a.wtype, at[j], 1.f, w[j]);
    load_weight<VEC>(a.b, a.btype, at[j], 0.f, b[j]);
  }
  ask((int64_t)blockIdx.x * kRows + mine);
  for (int64_t base = (int64_t)blockIdx.x * kRows; base < a.n; base += step) {
    const int64_t row = base + mine;
    float v[ITER][VEC], sum[1] = {0.f};
#pragma unroll
    for (int j = 0; j < ITER; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[j][k] = (float)next[j].v[k];
        sum[0] += k >= first[j] ? v[j][k] : 0.f;
      }
    ask(row + step);
    row_sums(sum, shared, half);
    const float mean = sum[0] / (float)a.c;
    sum[0] = 0.f;
#pragma unroll
    for (int j = 0; j < ITER; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        v[j][k] -= mean;
        sum[0] += k >= first[j] ? v[j][k] * v[j][k] : 0.f;
      }
    row_sums(sum, shared, half);
    const float rstd = 1.f / sqrtf(sum[0] / (float)a.c + a.eps);
    if (row >= a.n) continue;
    T* y = (T*)a.y + row * a.c;
#pragma unroll
    for (int j = 0; j < ITER; ++j)
      if (first[j] < VEC) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j][k] = v[j][k] * rstd * w[j][k] + b[j][k];
        store_vec<T, VEC>(y + at[j], v[j]);
      }
    if (a.mean && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// rows wider than a block's registers: three walks over the row
template <typename T>
__global__ void __launch_bounds__(1024) norm_forward_wide_kernel(NormArgs a) {
  __shared__ RowSums<1024, 1, 1> shared;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.stride;
  int half = 0;
  float sum[1] = {0.f};
  for (int c = threadIdx.x; c < a.c; c += 1024) sum[0] += (float)x[c];
  row_sums(sum, shared, half);
  const float mean = sum[0] / (float)a.c;
  sum[0] = 0.f;
  for (int c = threadIdx.x; c < a.c; c += 1024) { const float d = (float)x[c] - mean; sum[0] += d * d; }
  row_sums(sum, shared, half);
  const float rstd = 1.f / sqrtf(sum[0] / (float)a.c + a.eps);
  T* y = (T*)a.y + row * a.c;
  for (int c = threadIdx.x; c < a.c; c += 1024) {
    float w[1], b[1];
    load_weight<1>(a.w, a.wtype, c, 1.f, w);
    load_weight<1>(a.b, a.btype, c, 0.f, b);
    y[c] = (T)(((float)x[c] - mean) * rstd * w[0] + b[0]);
  }
  if (a.mean && threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

struct NormBackArgs {
  const void *x, *dy, *w;
  const float *mean, *rstd;
  void* dx;
  float* partial;        // (blocks, 2, C): dw and db of each block's rows; null: not wanted
  int64_t n, stride, dystride, rows_per_block;
  int c, wtype;
};

template <typename T, int VEC, int LPR, int ITER, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_backward_kernel(NormBackArgs a) {
  constexpr int kRows = THREADS / LPR;
  __shared__ RowSums<LPR, kRows, 2> shared;
  __shared__ float sums[kRows > 1 ? THREADS * VEC * 2 : 1];
  const int lane = threadIdx.x % LPR, mine = threadIdx.x / LPR;
  int at[ITER], first[ITER], half = 0;
  float w[ITER][VEC], dw[ITER][VEC], db[ITER][VEC];
  Pack<T, VEC> nx[ITER], ny[ITER];
  float nmean, nrstd;
#pragma unroll
  for (int j = 0; j < ITER; ++j) {
    at[j] = vec_at<VEC>(j * LPR + lane, a.c, first[j]);
    load_weight<VEC>(a.w, a.wtype, at[j], 1.f, w[j]);
#pragma unroll
    for (int k = 0; k < VEC; ++k) dw[j][k] = db[j][k] = 0.f;
  }
  const int64_t begin = (int64_t)blockIdx.x * a.rows_per_block, end = min(begin + a.rows_per_block, a.n);
  auto ask = [&](int64_t r) {     // (behind the last row, that one again)
    const int64_t row = min(r, a.n - 1);
    const T* x = (const T*)a.x + row * a.stride;
    const T* dy = (const T*)a.dy + row * a.dystride;
#pragma unroll
    for (int j = 0; j < ITER; ++j) {
      __builtin_memcpy(&nx[j], x + at[j], sizeof(nx[j]));
      __builtin_memcpy(&ny[j], dy + at[j], sizeof(ny[j]));
    }
    nmean = a.mean[row];
    nrstd = a.rstd[row];
  };
  ask(begin + mine);
  for (int64_t base = begin; base < end; base += kRows) {
    const int64_t row = base + mine;
    const bool live = row < end;
    const float mean = nmean, rstd = nrstd;
    float h[ITER][VEC], g[ITER][VEC], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < ITER; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        h[j][k] = ((float)nx[j].v[k] - mean) * rstd;
        const float d = live ? (float)ny[j].v[k] : 0.f;
        dw[j][k] += live ? d * h[j][k] : 0.f;      // (a row that is not there must not bring in 0 times something undefined)
        db[j][k] += d;
        g[j][k] = d * w[j][k];
        sum[0] += k >= first[j] ? g[j][k] : 0.f;
        sum[1] += k >= first[j] ? g[j][k] * h[j][k] : 0.f;
      }
    ask(row + kRows);
    row_sums(sum, shared, half);
    const float s = sum[0] / (float)a.c, q = sum[1] / (float)a.c;
    if (a.dx && live) {
      T* dx = (T*)a.dx + row * a.c;
#pragma unroll
      for (int j = 0; j < ITER; ++j)
        if (first[j] < VEC) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) h[j][k] = rstd * (g[j][k] - s - h[j][k] * q);
          store_vec<T, VEC>(dx + at[j], h[j]);
        }
    }
  }
  if (!a.partial) return;
  float* out = a.partial + (int64_t)blockIdx.x * 2 * a.c;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int j = 0; j < ITER; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k)
        if (k >= first[j]) {
          out[at[j] + k] = dw[j][k];
          out[a.c + at[j] + k] = db[j][k];
        }
  } else {
#pragma unroll
    for (int j = 0; j < ITER; ++j) {   // the block's row groups, added in order
      __syncthreads();
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        sums[(2 * k) * THREADS + threadIdx.x] = dw[j][k];
        sums[(2 * k + 1) * THREADS + threadIdx.x] = db[j][k];
      }
      __syncthreads();
      for (int i = threadIdx.x; i < LPR * VEC * 2; i += THREADS) {
        const int l = i % LPR, k2 = i / LPR;
        float s = 0.f;
        for (int r = 0; r < kRows; ++r) s += sums[k2 * THREADS + r * LPR + l];
        int f;
        const int col = vec_at<VEC>(j * LPR + l, a.c, f);
        if ((k2 >> 1) >= f) out[(k2 & 1) * a.c + col + (k2 >> 1)] = s;
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_backward_wide_kernel(NormBackArgs a) {   // dx only; the sums have a kernel of their own
  __shared__ RowSums<1024, 1, 2> shared;
  const int64_t row = blockIdx.x;
  const T* x = (const T*)a.x + row * a.stride;
  const T* dy = (const T*)a.dy + row * a.dystride;
  const float mean = a.mean[row], rstd = a.rstd[row];
  int half = 0;
  float sum[2] = {0.f, 0.f}, w[1];
  for (int c = threadIdx.x; c < a.c; c += 1024) {
    load_weight<1>(a.w, a.wtype, c, 1.f, w);
    const float g = (float)dy[c] * w[0];
    sum[0] += g;
    sum[1] += g * (((float)x[c] - mean) * rstd);
  }
  row_sums(sum, shared, half);
  const float s = sum[0] / (float)a.c, q = sum[1] / (float)a.c;
  T* dx = (T*)a.dx + row * a.c;
  for (int c = threadIdx.x; c < a.c; c += 1024) {
    load_weight<1>(a.w, a.wtype, c, 1.f, w);
    dx[c] = (T)(rstd * ((float)dy[c] * w[0] - s - (((float)x[c] - mean) * rstd) * q));
  }
}

template <typename T>
__global__ void __launch_bounds__(256) norm_column_sums_kernel(NormBackArgs a) {   // the wide rows' column sums: one thread a column
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= a.c) return;
  const int64_t begin = (int64_t)blockIdx.y * a.rows_per_block, end = min(begin + a.rows_per_block, a.n);
  float dw = 0.f, db = 0.f;
  for (int64_t row = begin; row < end; ++row) {
    const float g = (float)((const T*)a.dy)[row * a.dystride + c];
    dw += g * (((float)((const T*)a.x)[row * a.stride + c] - a.mean[row]) * a.rstd[row]);
    db += g;
  }
  float* out = a.partial + (int64_t)blockIdx.y * 2 * a.c;
  out[c] = dw;
  out[a.c + c] = db;
}

// dw and db from the blocks' rows: 16 columns a block, 16 slices of the rows, four loads in flight a thread; added in a fixed order
__global__ void __launch_bounds__(256) norm_param_grad_kernel(const float* __restrict__ partial, int rows, int64_t c, void* dw, int wtype, void* db,
                                                              int btype) {
  __shared__ float lds[16][17];
  const int x = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + x;
  const int per = (rows + 15) / 16, r0 = slice * per, r1 = min(r0 + per, rows);
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (col < 2 * c) {
    const float* p = partial + col + (int64_t)r0 * 2 * c;
    int r = r0;
    for (; r + 4 <= r1; r += 4, p += 8 * c) {
      s0 += p[0];
      s1 += p[2 * c];
      s2 += p[4 * c];
      s3 += p[6 * c];
    }
    for (; r < r1; ++r, p += 2 * c) s0 += *p;
  }
  lds[slice][x] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (slice || col >= 2 * c) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += lds[i][x];
  void* out = col < c ? dw : db;
  const int type = col < c ? wtype : btype;
  const int64_t i = col < c ? col : col - c;
  if (!out) return;
  if (type == VC_F32) ((float*)out)[i] = s;
  else if (type == VC_F16) ((_Float16*)out)[i] = (_Float16)s;
  else ((__bf16*)out)[i] = (__bf16)s;
}

// how a row of c elements is held: VEC elements a vector, LPR lanes, ITER vectors a lane; iter 0: wider than a block's registers
struct NormShape { int vec, lpr, iter; };
static NormShape norm_shape(int64_t c, int dtype) {
  const int full = dtype == VC_F32 ? 4 : 8;
  if (c < full) return {1, 8, 1};
  const int64_t vecs = cdiv(c, full);
  for (int lpr = 2; lpr <= 64; lpr *= 2)
    if (vecs <= lpr) return {full, lpr, 1};
  if (vecs <= 128) return {full, 64, 2};      // (32768 x 1000 bf16: forward 28 us, backward 54; by blocks of 256, one vector a lane, 42 and 60)
  // (two vectors a lane up to 512 and 1024 vectors were no faster in the forward pass, and spill in the backward pass, which holds five values
  // an element: 16381 x 4096 bf16, 138 us and 89)
  for (int lpr = 256; lpr <= 1024; lpr *= 2)
    if (vecs <= lpr) return {full, lpr, 1};
  if (vecs <= 2048) return {full, 1024, 2};
  if (dtype == VC_F32 && vecs <= 4096) return {full, 1024, 4};
  return {1, 1024, 0};
}

// Blocks of the backward pass = rows of its partial sums, which are written and read once more: one a compute unit, of 1024 threads for rows of
// several waves and of 512 for shorter ones.  (133578 x 64 fp32 and bf16, with the weights' gradients: 27 and 14 us; 1024 blocks of 256 threads 29
// and 18, 256 of 1024 threads 26 and 16; 32768 x 1000 bf16: 47, 54 and, as that many threads leave too few registers, 80.)
static int back_threads(const NormShape& s) { return s.lpr > 64 ? 1024 : 512; }
static int64_t norm_blocks(int64_t n, int64_t c, const NormShape& s) {
  const int rows = s.iter ? back_threads(s) / s.lpr : 64;
  const int64_t most = s.iter ? 256 : 512, b = cdiv(n, rows);
  return b < most ? (b > 0 ? b : 1) : most;
}

template <typename T> struct FullVec { static constexpr int value = sizeof(T) == 4 ? 4 : 8; };

#define VC_NORM_SHAPES(DO)                                                                                                                  \
  if (s.vec == 1) { DO(1, 8, 1); }                                                                                                          \
  else if (s.lpr == 2) { DO(V, 2, 1); } else if (s.lpr == 4) { DO(V, 4, 1); } else if (s.lpr == 8) { DO(V, 8, 1); }                         \
  else if (s.lpr == 16) { DO(V, 16, 1); } else if (s.lpr == 32) { DO(V, 32, 1); }                                                           \
  else if (s.lpr == 64 && s.iter == 1) { DO(V, 64, 1); } else if (s.lpr == 64) { DO(V, 64, 2); }                                            \
  else if (s.lpr == 256) { DO(V, 256, 1); } else if (s.lpr == 512) { DO(V, 512, 1); } else if (s.iter == 1) { DO(V, 1024, 1); }             \
  else if (s.iter == 2) { DO(V, 1024, 2); } else if constexpr (V == 4) { DO(V, 1024, 4); }

template <typename T>
static void norm_forward_launch(const NormArgs& a, const NormShape& s, hipStream_t st) {
  constexpr int V = FullVec<T>::value;
  if (!s.iter) {
    hipLaunchKernelGGL(norm_forward_wide_kernel<T>, dim3((unsigned)a.n), dim3(1024), 0, st, a);
    return;
  }
  // as many blocks as the chip holds (2048 threads a compute unit), or as there are rows for
  const int threads = s.lpr > 256 ? s.lpr : 256;
  const int64_t most = 256 * (2048 / threads), need = cdiv(a.n, threads / s.lpr);
  const unsigned blocks = (unsigned)(need < most ? need : most);
#define VC_DO(VEC, LPR, ITER)                                                                                                               \
  hipLaunchKernelGGL((norm_forward_kernel<T, VEC, LPR, ITER, (LPR > 256 ? LPR : 256)>), dim3(blocks), dim3(threads), 0, st, a)
  VC_NORM_SHAPES(VC_DO)
#undef VC_DO
}

template <typename T>
static void norm_backward_launch(const NormBackArgs& a, const NormShape& s, int64_t blocks, hipStream_t st) {
  constexpr int V = FullVec<T>::value;
  if (!s.iter) {
    if (a.dx) hipLaunchKernelGGL(norm_backward_wide_kernel<T>, dim3((unsigned)a.n), dim3(1024), 0, st, a);
    if (a.partial) hipLaunchKernelGGL(norm_column_sums_kernel<T>, dim3((unsigned)cdiv(a.c, 256), (unsigned)blocks), dim3(256), 0, st, a);
    return;
  }
#define VC_DO(VEC, LPR, ITER)                                                                                                               \
  hipLaunchKernelGGL((norm_backward_kernel<T, VEC, LPR, ITER, (LPR > 64 ? 1024 : 512)>), dim3((unsigned)blocks), dim3(back_threads(s)), 0, st, a)
  VC_NORM_SHAPES(VC_DO)
#undef VC_DO
}

// a launch has fewer than 2^32 threads: 1024 for a row beyond a block's registers, 256 for 16 of the two gradients' columns
static bool launches(int64_t n, int64_t c, const NormShape& s, bool sums) { return (s.iter || n < (1LL << 22)) && (!sums || c < (1LL << 27)); }

static bool known_dtype(int t) { return t == VC_F32 || t == VC_F16 || t == VC_BF16; }

}  // namespace vc

using namespace vc;

extern "C" {

int vc_layer_norm_forward(const void* x, int64_t x_stride, int64_t n, int64_t c, int dtype, const void* weight, int weight_dtype,
                          const void* bias, int bias_dtype, float eps, void* y, float* mean, float* rstd, void* stream) {
  VC_REQUIRE(known_dtype(dtype) && known_dtype(weight_dtype) && known_dtype(bias_dtype), "vc_layer_norm_forward: unknown dtype");
  VC_REQUIRE(n >= 0 && n < (1LL << 31) && c >= 1 && c < (1LL << 30), "vc_layer_norm_forward: %lld rows of %lld", (long long)n, (long long)c);
  VC_REQUIRE(x_stride >= c || n <= 1, "vc_layer_norm_forward: row stride %lld below %lld columns", (long long)x_stride, (long long)c);
  VC_REQUIRE((mean == nullptr) == (rstd == nullptr), "vc_layer_norm_forward: mean and rstd come together");
  if (n == 0) return VC_OK;
  VC_REQUIRE(x && y, "vc_layer_norm_forward: NULL pointer");
  NormArgs a{x, weight, bias, y, mean, rstd, n, x_stride, (int)c, weight_dtype, bias_dtype, eps};
  const NormShape s = norm_shape(c, dtype);
  VC_REQUIRE(launches(n, c, s, false), "vc_layer_norm_forward: %lld rows of %lld: too many for one launch", (long long)n, (long long)c);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == VC_F32) norm_forward_launch<float>(a, s, st);
  else if (dtype == VC_F16) norm_forward_launch<_Float16>(a, s, st);
  else norm_forward_launch<__bf16>(a, s, st);
  VC_CHECK_LAUNCH("norm_forward_kernel");
  return VC_OK;
}

size_t vc_layer_norm_backward_workspace_bytes(int64_t n, int64_t c, int dtype) {
  if (n <= 0 || c <= 0 || !known_dtype(dtype)) return 0;
  return (size_t)norm_blocks(n, c, norm_shape(c, dtype)) * 2 * (size_t)c * sizeof(float);
}

int vc_layer_norm_backward(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int64_t n, int64_t c, int dtype,
                           const void* weight, int weight_dtype, int bias_dtype, const float* mean, const float* rstd, void* dx, void* dweight,
                           void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  VC_REQUIRE(known_dtype(dtype) && known_dtype(weight_dtype) && known_dtype(bias_dtype), "vc_layer_norm_backward: unknown dtype");
  VC_REQUIRE(n >= 0 && n < (1LL << 31) && c >= 1 && c < (1LL << 30), "vc_layer_norm_backward: %lld rows of %lld", (long long)n, (long long)c);
  VC_REQUIRE((x_stride >= c && dy_stride >= c) || n <= 1, "vc_layer_norm_backward: row stride below %lld columns", (long long)c);
  hipStream_t st = (hipStream_t)stream;
  const bool sums = dweight || dbias;
  const NormShape s = norm_shape(c, dtype);
  VC_REQUIRE(launches(dx ? n : 0, c, s, sums), "vc_layer_norm_backward: %lld rows of %lld: too many for one launch", (long long)n, (long long)c);
  const int64_t blocks = norm_blocks(n, c, s);
  if (n > 0) {
    VC_REQUIRE(x && dy && mean && rstd, "vc_layer_norm_backward: NULL pointer");
    const size_t need = sums ? (size_t)blocks * 2 * (size_t)c * sizeof(float) : 0;
    VC_REQUIRE(!sums || (workspace && workspace_bytes >= need), "vc_layer_norm_backward: workspace of %zu bytes, need %zu", workspace_bytes, need);
    NormBackArgs a{x, dy, weight, mean, rstd, dx, sums ? (float*)workspace : nullptr, n, x_stride, dy_stride, cdiv(n, blocks), (int)c, weight_dtype};
    if (dx || sums) {
      if (dtype == VC_F32) norm_backward_launch<float>(a, s, blocks, st);
      else if (dtype == VC_F16) norm_backward_launch<_Float16>(a, s, blocks, st);
      else norm_backward_launch<__bf16>(a, s, blocks, st);
      VC_CHECK_LAUNCH("norm_backward_kernel");
    }
  }
  if (sums) {
    hipLaunchKernelGGL(norm_param_grad_kernel, dim3((unsigned)cdiv(2 * c, 16)), dim3(256), 0, st, (const float*)workspace, n > 0 ? (int)blocks : 0, c,
                       dweight, weight_dtype, dbias, bias_dtype);
    VC_CHECK_LAUNCH("norm_param_grad_kernel");
  }
  return VC_OK;
}

}  // extern "C"
