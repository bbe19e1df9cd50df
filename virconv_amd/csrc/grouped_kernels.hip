// Products of ragged row groups with one weight matrix per group: rows [offsets[g], offsets[g + 1]) of x meet W_g (out x in).
//
//   forward         y_r  = W_g x_r + b_g                 a row product, both operands along the inner axis
//   backward input  dx_r = W_g^T dy_r                    a row product, the weights across it
//   backward weight dW_g = sum_r dy_r x_r^T, db_g = sum_r dy_r     both operands across the summed axis (the group's rows)
//
// One output tile per block on v_mfma_f32_16x16x32, fp32 accumulation, one rounding at the end.  The tile's operands go through LDS as
// 16-bit values: as they are where the tensors are f16 or bf16, and cut exactly into three bf16 pieces where they are fp32 -- six of the
// nine cross terms are issued, the dropped ones stay below 2^-24 of a product.  An operand that lies along the summed axis is read back
// with ds_read_b128, one that lies across it with ds_read_b64_tr_b16 (four rows by sixteen columns a 16-lane group, transposed on the way);
// the 16-byte (32-byte) pieces of a row are exchanged by a function of the row, so that either read touches every bank once.
//
// The group sizes are known on the device only (a router's output needs no trip to the host): the grid is sized for the most tiles that
// `rows` and `groups` allow, and every block finds its group by a scan of the offsets.  Offsets are taken as a rising sequence within
// [0, rows]; one that is not is cut to it, so no content of `offsets` leads out of the tensors.  Rows of no group come out as zeros.
#include "common.h"

namespace vc {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

enum { kForward = 0, kBackInput = 1, kBackWeight = 2 };

struct GroupArgs {
  const void *a, *b;         // row products: the rows and the weights; weight product: dy and x
  const void* bias;          // (groups, n) or null (forward)
  const void* offsets;       // (groups + 1) int32 or int64
  void* out;
  float* partial;            // split sums (see the launchers), or null
  void* dbias;               // weight product: (groups, m), or null
  float* partial_bias;
  int64_t lda, ldb;
  int64_t rows;
  int groups, off64, m, n, k;   // m: weight product only
  int ntiles, mtiles, splits, per_split;
  unsigned total;
};

__device__ __forceinline__ int64_t offset_at(const GroupArgs& a, int g) {
  const int64_t o = a.off64 ? ((const int64_t*)a.offsets)[g] : (int64_t)((const int32_t*)a.offsets)[g];
  return o < 0 ? 0 : o > a.rows ? a.rows : o;
}

__device__ __forceinline__ int64_t shfl_up64(int64_t x, int d) {
  int lo = __shfl_up((int)(uint32_t)x, d, 64), hi = __shfl_up((int)(x >> 32), d, 64);
  return ((int64_t)hi << 32) | (uint32_t)lo;
}
__device__ __forceinline__ int64_t shfl64(int64_t x, int l) {
  int lo = __shfl((int)(uint32_t)x, l, 64), hi = __shfl((int)(x >> 32), l, 64);
  return ((int64_t)hi << 32) | (uint32_t)lo;
}

// Tile `target` of the groups' tiles of `per` rows, group after group: its group, the group's rows and the tile's number within it.
// group = groups: behind the groups' tiles; `target` is then what is left of it, [begin, end) the rows behind the last group.
// Every wave of the block runs it for itself.
struct Place { int group; int64_t begin, end, first_row; unsigned tile; };
__device__ __forceinline__ Place find_tile(const GroupArgs& a, int64_t per, unsigned target) {
  const int lane = threadIdx.x & 63;
  int64_t high = 0, first_row = 0;      // rows handed out so far (the running maximum of the offsets), the first group's begin
  for (int g0 = 0; g0 < a.groups; g0 += 64) {
    const int g = g0 + lane;
    int64_t end = g < a.groups ? offset_at(a, g + 1) : 0;
    if (g0 == 0) first_row = high = offset_at(a, 0);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int64_t o = shfl_up64(end, d); if (lane >= d && o > end) end = o; }
    if (end < high) end = high;
    int64_t begin = shfl_up64(end, 1);
    if (lane == 0) begin = high;
    unsigned tiles = g < a.groups ? (unsigned)((end - begin + per - 1) / per) : 0u, upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const unsigned o = __shfl_up(upto, d, 64); if (lane >= d) upto += o; }
    const uint64_t hit = __ballot(target < upto);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      Place p;
      p.group = g0 + l;
      p.begin = shfl64(begin, l);
      p.end = shfl64(end, l);
      p.first_row = first_row;
      p.tile = target - (__shfl(upto, l, 64) - __shfl(tiles, l, 64));
      return p;
    }
    target -= __shfl(upto, 63, 64);
    high = shfl64(end, 63);
  }
  return {a.groups, high, a.rows, first_row, target};
}

// ------------------------------------------------------------------------------------------------ operands
template <typename T> struct OperandOf { static constexpr int planes = 1, bk = 64; typedef T type; };
template <> struct OperandOf<float> { static constexpr int planes = 3, bk = 32; typedef __bf16 type; };

template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Eight { T v[8]; };

template <typename T>
__device__ __forceinline__ void load8(const T* p, int valid, T (&out)[8]) {   // `valid` of eight elements; zeros behind them
  if (valid >= 8) {
    Eight<T> e;
    __builtin_memcpy(&e, p, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = e.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = i < valid ? p[i] : (T)0.f;
  }
}

// the top 16 bits of x as a bf16 (cut, not rounded: x - top is exact and so is what is left of it)
__device__ __forceinline__ uint32_t top16(float x) { return __float_as_uint(x) & 0xffff0000u; }

// eight elements into their place(s) in LDS: one 16-byte piece, or three planes of it
template <typename T>
__device__ __forceinline__ void stage8(char* lds, int plane_bytes, int at, const T (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<v8s*>(lds + at) = *reinterpret_cast<const v8s*>(&x);
  } else {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t h[2][3];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float v = x[2 * i + j];
        h[j][0] = top16(v);
        const float r = v - __uint_as_float(h[j][0]);
        h[j][1] = top16(r);
        h[j][2] = top16(r - __uint_as_float(h[j][1]));
      }
#pragma unroll
      for (int q = 0; q < 3; ++q) w[q][i] = (h[0][q] >> 16) | h[1][q];
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(lds + q * plane_bytes + at) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
}

// A tile of one operand in LDS.  ALONG: [rows][BK], pieces of 8 along the summed axis; else [BK][cols], pieces of 8 across it.
template <typename T, int ROWS, bool ALONG>
struct Tile {
  static constexpr int BK = OperandOf<T>::bk, planes = OperandOf<T>::planes;
  static constexpr int plane_bytes = ROWS * BK * 2, bytes = plane_bytes * planes;
  static constexpr int pieces = ROWS * BK / 8, per_thread = (pieces + 255) / 256;

  static __device__ __forceinline__ int place(int r, int k) {   // byte of element (row r, summed index k); r or k a multiple of 8
    if constexpr (ALONG) {
      constexpr int CH = BK / 8, R = 16 / CH;                   // pieces a row, rows per 256 bytes
      return r * BK * 2 + ((((k >> 3) ^ (r / R)) & (CH - 1)) << 4);
    } else {
      constexpr int SLOTS = ROWS / 16;                          // 32-byte slots a row (of the summed axis)
      const int f = SLOTS >= 8 ? ((k & 3) | ((k >> 1) & 4)) : SLOTS == 4 ? (((k >> 1) & 1) | ((k >> 2) & 2)) : SLOTS == 2 ? ((k >> 3) & 1) : 0;
      return k * ROWS * 2 + ((((r >> 4) ^ f) & (SLOTS - 1)) << 5) + ((r & 15) << 1);
    }
  }

  T reg[per_thread][8];

  // rows [0, rows) and summed indices [0, depth) of the tile exist; p: the tile's first element, ld: the stride of its slow axis
  __device__ __forceinline__ void fetch(const T* p, int64_t ld, int rows, int depth) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * 256 + threadIdx.x;
      if (pieces % 256 && q >= pieces) continue;
      int valid;
      const T* s;
      if constexpr (ALONG) {
        const int r = q / (BK / 8), k = (q % (BK / 8)) * 8;
        valid = r < rows ? depth - k : 0;
        s = p + r * ld + k;
      } else {
        const int k = q / (ROWS / 8), c = (q % (ROWS / 8)) * 8;
        valid = k < depth ? rows - c : 0;
        s = p + k * ld + c;
      }
      load8(s, valid, reg[i]);
    }
  }
  __device__ __forceinline__ void put(char* lds) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * 256 + threadIdx.x;
      if (pieces % 256 && q >= pieces) continue;
      int at;
      if constexpr (ALONG) at = place(q / (BK / 8), (q % (BK / 8)) * 8);
      else at = place((q % (ROWS / 8)) * 8, q / (ROWS / 8));
      stage8(lds, plane_bytes, at, reg[i]);
    }
  }
  // The 16 rows from r0 on (a multiple of 16), 32 summed indices from k0 on (a multiple of 32), as an operand of v_mfma_f32_16x16x32: lane l
  // holds row l % 16, the eight indices from 8 (l / 16) on.  `lane_place` is the lane's part of the address, to be made once per tile row.
  static __device__ __forceinline__ int lane_place(int r0) {
    const int lane = threadIdx.x & 63;
    if constexpr (ALONG) return place(r0 + (lane & 15), (lane >> 4) * 8);
    else return place(r0 + (lane & 3) * 4, (lane >> 4) * 8 + ((lane & 15) >> 2));
  }
  static __device__ __forceinline__ v8s fragment(const char* lds, int plane, int at, int k0) {
    if constexpr (ALONG) {
      return *reinterpret_cast<const v8s*>(lds + plane * plane_bytes + (at ^ (k0 << 1)));   // (32 indices on: bit 6 of the exchanged piece)
    } else {
      typedef __attribute__((address_space(3))) v4s lds4;
      const char* p = lds + at + plane * plane_bytes + k0 * ROWS * 2;
      const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
      const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * ROWS * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <typename O>
__device__ __forceinline__ v4f mfma(v8s a, v8s b, v4f c) {
  if constexpr (__is_same(O, _Float16))
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ v8s ones() {
  const short one = __is_same(T, _Float16) ? (short)0x3c00 : (short)0x3f80;
  return v8s{one, one, one, one, one, one, one, one};
}

// blocks of one XCD (consecutive blocks go to the eight XCDs in turn) take consecutive tiles: neighbours share an operand in its L2
__device__ __forceinline__ unsigned xcd_order(unsigned b, unsigned total) {
  const unsigned per = total / 8, rest = total % 8, x = b % 8, i = b / 8;
  return x * per + (x < rest ? x : rest) + i;
}

template <typename T> __device__ __forceinline__ void store4(T* p, int valid, const float (&x)[4]) {
  if (valid >= 4) {
    struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; } e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.v[i] = (T)x[i];
    __builtin_memcpy(p, &e, sizeof(e));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = (T)x[i];
  }
}

// ------------------------------------------------------------------------------------------------ the kernel
template <typename T, int BM, int BN, int MODE>
__global__ void __launch_bounds__(256, 2) grouped_kernel(GroupArgs a) {
  typedef typename OperandOf<T>::type O;
  constexpr int BK = OperandOf<T>::bk, P = OperandOf<T>::planes;
  typedef Tile<T, BM, MODE != kBackWeight> TileA;
  typedef Tile<T, BN, MODE == kForward> TileB;
  constexpr int WM = BM >= 64 ? 2 : 1, WN = 4 / WM;            // waves along m and n
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;          // fragments of a wave
  __shared__ __align__(16) char lds[TileA::bytes + TileB::bytes];
  char* const la = lds;
  char* const lb = lds + TileA::bytes;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;

  unsigned id = xcd_order(blockIdx.x, a.total);
  const T *pa, *pb;
  int rows_a, rows_b, depth, group;
  int64_t m0, mend;
  int n0, split = 0;
  float* partial = nullptr;
  if constexpr (MODE != kBackWeight) {
    n0 = (int)(id % a.ntiles) * BN;
    id /= a.ntiles;
    split = (int)(id % a.splits);
    const Place w = find_tile(a, BM, id / a.splits);
    if (w.group == a.groups) {   // rows of no group: in front of the first and behind the last
      if (split) return;
      int64_t r = (int64_t)w.tile * BM, front = w.first_row;
      const int64_t front_tiles = (front + BM - 1) / BM;
      const int64_t lo = (int64_t)w.tile < front_tiles ? r : w.begin + (r - front_tiles * BM);
      const int64_t hi = min(lo + BM, (int64_t)w.tile < front_tiles ? front : a.rows);
      for (int64_t e = threadIdx.x; lo < hi && e < (hi - lo) * BN; e += 256) {
        const int n = n0 + (int)(e % BN);
        if (n < a.n) ((T*)a.out)[(lo + e / BN) * a.n + n] = (T)0.f;
      }
      return;
    }
    group = w.group;
    m0 = w.begin + (int64_t)w.tile * BM;
    mend = w.end;
    const int k0 = split * a.per_split;
    depth = min(a.per_split, a.k - k0);
    rows_a = (int)min((int64_t)BM, mend - m0);
    rows_b = min(BN, a.n - n0);
    pa = (const T*)a.a + m0 * a.lda + k0;
    const T* weights = (const T*)a.b + (int64_t)group * a.n * a.k;
    if constexpr (MODE == kForward) pb = weights + (int64_t)n0 * a.k + k0;
    else pb = weights + (int64_t)k0 * a.n + n0;
    if (a.splits > 1) partial = a.partial + ((int64_t)split * a.rows + m0) * a.n + n0;
  } else {
    n0 = (int)(id % a.ntiles) * BN;
    id /= a.ntiles;
    m0 = (int64_t)(id % a.mtiles) * BM;
    mend = a.m;
    id /= a.mtiles;
    int64_t r0, r1;
    if (a.splits > 1) {          // pieces of per_split rows, their sums added by grouped_weight_sum_kernel
      const Place w = find_tile(a, a.per_split, id);
      if (w.group == a.groups) return;
      group = w.group;
      r0 = w.begin + (int64_t)w.tile * a.per_split;
      r1 = min(r0 + a.per_split, w.end);
      partial = a.partial + ((int64_t)id * a.m + m0) * a.n + n0;
    } else {
      group = (int)id;
      r0 = r1 = 0;
      // the group's rows: the running maximum of the offsets up to it
      for (int g0 = 0; g0 <= group; g0 += 64) {
        const int g = g0 + lane;
        int64_t o = g <= group ? offset_at(a, g) : 0;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) { const int64_t q = shfl64(o, lane ^ d); if (q > o) o = q; }
        if (o > r0) r0 = o;
      }
      r1 = max(offset_at(a, group + 1), r0);
    }
    depth = (int)(r1 - r0);
    rows_a = (int)min((int64_t)BM, (int64_t)a.m - m0);
    rows_b = min(BN, a.n - n0);
    pa = (const T*)a.a + r0 * a.lda + m0;
    pb = (const T*)a.b + r0 * a.ldb + n0;
  }
  const int64_t lda = a.lda, ldb = MODE == kForward ? a.k : MODE == kBackInput ? a.n : a.ldb;
  const bool sum_bias = MODE == kBackWeight && a.dbias && n0 == 0 && wn == 0;

  v4f acc[FM][FN], accb[FM];
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    accb[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  int at_a[FM], at_b[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) at_a[i] = TileA::lane_place(wm * (BM / WM) + i * 16);
#pragma unroll
  for (int j = 0; j < FN; ++j) at_b[j] = TileB::lane_place(wn * (BN / WN) + j * 16);
  TileA ta;
  TileB tb;
  ta.fetch(pa, lda, rows_a, depth);
  tb.fetch(pb, ldb, rows_b, depth);
  for (int k0 = 0; k0 < depth; k0 += BK) {
    __syncthreads();
    ta.put(la);
    tb.put(lb);
    __syncthreads();
    if (k0 + BK < depth) {   // the next tile is under way while this one is multiplied
      const int64_t k1 = k0 + BK;
      ta.fetch(MODE == kBackWeight ? pa + k1 * lda : pa + k1, lda, rows_a, depth - (int)k1);
      tb.fetch(MODE == kForward ? pb + k1 : pb + k1 * ldb, ldb, rows_b, depth - (int)k1);
    }
#pragma unroll
    for (int kk = 0; kk < BK; kk += 32) {
      v8s fb[FN][P];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < P; ++q) fb[j][q] = TileB::fragment(lb, q, at_b[j], kk);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        v8s fa[P];
#pragma unroll
        for (int q = 0; q < P; ++q) fa[q] = TileA::fragment(la, q, at_a[i], kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          // the lane's four results are neighbours along n: the n side is the instruction's row operand
          if constexpr (P == 3) {
            acc[i][j] = mfma<O>(fb[j][2], fa[0], acc[i][j]);
            acc[i][j] = mfma<O>(fb[j][0], fa[2], acc[i][j]);
            acc[i][j] = mfma<O>(fb[j][1], fa[1], acc[i][j]);
            acc[i][j] = mfma<O>(fb[j][1], fa[0], acc[i][j]);
            acc[i][j] = mfma<O>(fb[j][0], fa[1], acc[i][j]);
          }
          acc[i][j] = mfma<O>(fb[j][0], fa[0], acc[i][j]);
        }
        if (MODE == kBackWeight && sum_bias) {
#pragma unroll
          for (int q = P - 1; q >= 0; --q) accb[i] = mfma<O>(ones<O>(), fa[q], accb[i]);
        }
      }
    }
  }

  // results: lane l holds row m = l % 16 and the columns n = 4 (l / 16) .. + 3 of each 16 x 16 tile
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wm * (BM / WM) + i * 16 + (lane & 15);
    if (m >= rows_a) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = wn * (BN / WN) + j * 16 + (lane >> 4) * 4;
      if (n >= rows_b) continue;
      float r[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (partial) {
        store4(partial + (int64_t)m * a.n + n, rows_b - n, r);
        continue;
      }
      if (MODE == kForward && a.bias) {
        const T* bias = (const T*)a.bias + (int64_t)group * a.n + n0 + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < rows_b) r[e] += (float)bias[e];
      }
      T* out = (T*)a.out;
      if constexpr (MODE == kBackWeight) out += ((int64_t)group * a.m + m0 + m) * a.n + n0 + n;
      else out += (m0 + m) * a.n + n0 + n;
      store4(out, rows_b - n, r);
    }
    if (MODE == kBackWeight && sum_bias && lane < 16) {
      if (partial) a.partial_bias[(int64_t)id * a.m + m0 + m] = accb[i][0];
      else ((T*)a.dbias)[(int64_t)group * a.m + m0 + m] = (T)accb[i][0];
    }
  }
}

// the sum of `count` values `stride` apart, in order: a chain, its loads four at a time
__device__ __forceinline__ float sum_along(const float* p, unsigned count, int64_t stride) {
  float s = 0.f;
  unsigned q = 0;
  for (; q + 4 <= count; q += 4, p += 4 * stride) {
    const float v0 = p[0], v1 = p[stride], v2 = p[2 * stride], v3 = p[3 * stride];
    s += v0; s += v1; s += v2; s += v3;
  }
  for (; q < count; ++q, p += stride) s += *p;
  return s;
}

// row products: the splits' sums added in order (+ bias); a wave takes 64 columns of a row
template <typename T>
__global__ void __launch_bounds__(256) grouped_row_sum_kernel(GroupArgs a) {
  const int lane = threadIdx.x & 63, chunks = (a.n + 63) / 64;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), row = id / chunks;
  if (row >= a.rows) return;
  // the row's group: the first one whose end lies behind it
  int group = -1;
  int64_t high = 0;
  for (int g0 = 0; g0 < a.groups && group < 0; g0 += 64) {
    const int g = g0 + lane;
    int64_t end = g < a.groups ? offset_at(a, g + 1) : 0;
    if (g0 == 0) {
      high = offset_at(a, 0);
      if (row < high) break;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int64_t o = shfl_up64(end, d); if (lane >= d && o > end) end = o; }
    if (end < high) end = high;
    const uint64_t hit = __ballot(g < a.groups && row < end);
    if (hit) group = g0 + __builtin_ctzll(hit);
    high = shfl64(end, 63);
  }
  const int n = (int)(id % chunks) * 64 + lane;
  if (group < 0 || n >= a.n) return;   // (rows of no group: written by the tiles' kernel)
  float s = sum_along(a.partial + row * a.n + n, a.splits, a.rows * a.n);
  if (a.bias) s += (float)((const T*)a.bias)[(int64_t)group * a.n + n];
  ((T*)a.out)[row * a.n + n] = (T)s;
}

// weight product: the pieces' sums of each group.  64 elements a block; its four waves add a quarter of the pieces each, in order, and the four
// sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256) grouped_weight_sum_kernel(GroupArgs a) {
  __shared__ float part[4][64];
  const int group = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // pieces in front of the group, and its own
  int64_t high = 0;
  unsigned before = 0, mine = 0;
  for (int g0 = 0; g0 <= group; g0 += 64) {
    const int g = g0 + lane;
    int64_t end = g < a.groups ? offset_at(a, g + 1) : 0;
    if (g0 == 0) high = offset_at(a, 0);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int64_t o = shfl_up64(end, d); if (lane >= d && o > end) end = o; }
    if (end < high) end = high;
    int64_t begin = shfl_up64(end, 1);
    if (lane == 0) begin = high;
    const unsigned pieces = (unsigned)((end - begin + a.per_split - 1) / a.per_split);
    unsigned s = g < group ? pieces : 0u;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
    before += s;
    if (group - g0 < 64) mine = __shfl(pieces, group - g0, 64);
    high = shfl64(end, 63);
  }
  const int64_t weights = (int64_t)a.m * a.n, size = weights + (a.dbias ? a.m : 0);
  const unsigned per = (mine + 3) / 4, q0 = min(wave * per, mine), q1 = min(q0 + per, mine);
  for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < size; e0 += (int64_t)gridDim.x * 64) {
    const int64_t e = e0 + lane, i = e - weights;
    if (e < weights) part[wave][lane] = sum_along(a.partial + (int64_t)(before + q0) * weights + e, q1 - q0, weights);
    else if (e < size) part[wave][lane] = sum_along(a.partial_bias + (int64_t)(before + q0) * a.m + i, q1 - q0, a.m);
    __syncthreads();
    if (wave == 0 && e < size) {
      const float s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
      if (e < weights) ((T*)a.out)[group * weights + e] = (T)s;
      else ((T*)a.dbias)[group * (int64_t)a.m + i] = (T)s;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ launch rules
struct GroupPlan { int bm, bn, splits, per_split; int64_t partial_floats, mtiles_most; };

// Row products.  Tiles of 128 rows where the groups have that many on average, of 64 or 16 where they have fewer (a tile of a short group is
// mostly padding); the inner axis is split where there are too few tiles to fill 256 compute units.
static GroupPlan plan_rows(int64_t rows, int64_t groups, int64_t n, int64_t k, int dtype) {
  GroupPlan p;
  const int64_t average = groups > 0 ? rows / groups : rows, bk = dtype == VC_F32 ? 32 : 64;
  p.bm = average > 96 && n > 64 ? 128 : average > 24 ? 64 : 16;
  p.bn = p.bm == 64 ? 64 : 128;
  p.mtiles_most = rows / p.bm + groups + 2;
  // tiles there will be: full ones, and one that is cut short for every group that has rows
  const int64_t tiles = (rows / p.bm + (groups < rows ? groups : rows)) * cdiv(n, p.bn), steps = cdiv(k, bk);
  int64_t splits = 1;
  if (tiles < 256 && steps >= 16) splits = 512 / tiles;
  if (splits > steps / 8) splits = steps / 8 > 0 ? steps / 8 : 1;
  p.per_split = (int)(cdiv(steps, splits) * bk);
  p.splits = (int)cdiv(k, p.per_split);
  if (p.splits < 1) p.splits = 1;
  p.partial_floats = p.splits > 1 ? p.splits * rows * n : 0;
  return p;
}

// Weight product.  The rows are split into pieces where the output has few tiles, a piece being long enough that the sums written for it
// (and read once more) stay small beside the rows that it reads.
static GroupPlan plan_weight(int64_t rows, int64_t groups, int64_t m, int64_t n, int dtype) {
  GroupPlan p;
  p.bm = m > 64 && n > 64 ? 128 : 64;
  p.bn = p.bm;
  const int64_t tiles = cdiv(m, p.bm) * cdiv(n, p.bn);
  int64_t piece = cdiv(rows, cdiv(512, tiles));
  const int64_t least = 4 * m * n / (m + n) > 256 ? 4 * m * n / (m + n) : 256;
  if (piece < least) piece = least;
  piece = cdiv(piece, 64) * 64;
  p.splits = tiles < 512 && groups * piece <= rows ? 2 : 1;
  p.per_split = (int)piece;
  p.mtiles_most = p.splits > 1 ? rows / piece + groups : groups;   // pieces
  p.partial_floats = p.splits > 1 ? p.mtiles_most * (m * n + m) : 0;
  return p;
}

static bool grouped_dtype(int t) { return t == VC_F32 || t == VC_F16 || t == VC_BF16; }

static int grouped_check(const char* who, int64_t rows, int64_t groups, int64_t in, int64_t out, int dtype, int offset_bits, const void* offsets) {
  VC_REQUIRE(grouped_dtype(dtype), "%s: unknown dtype %d", who, dtype);
  VC_REQUIRE(offset_bits == 32 || offset_bits == 64, "%s: offsets of %d bits", who, offset_bits);
  VC_REQUIRE(rows >= 0 && rows < (1LL << 31) && groups >= 0 && groups < (1 << 20), "%s: %lld rows in %lld groups", who, (long long)rows, (long long)groups);
  VC_REQUIRE(in >= 1 && in < (1 << 24) && out >= 1 && out < (1 << 24), "%s: %lld -> %lld channels", who, (long long)in, (long long)out);
  VC_REQUIRE(offsets || groups == 0, "%s: NULL offsets", who);
  return VC_OK;
}

static int launch_rows(const char* who, GroupArgs a, int mode, int dtype, const GroupPlan& p, void* ws, size_t ws_bytes, hipStream_t st) {
  const size_t need = (size_t)p.partial_floats * sizeof(float);
  VC_REQUIRE(need == 0 || (ws && ws_bytes >= need), "%s: workspace of %zu bytes, need %zu", who, ws_bytes, need);
  a.partial = (float*)ws;
  a.splits = p.splits;
  a.per_split = p.per_split;
  a.ntiles = (int)cdiv(a.n, p.bn);
  const int64_t total = p.mtiles_most * a.ntiles * p.splits;
  VC_REQUIRE(total < (1LL << 31), "%s: %lld tiles", who, (long long)total);
  a.total = (unsigned)total;
#define VC_GO(T, BM, BN)                                                                                                          \
  if (mode == kForward) hipLaunchKernelGGL((grouped_kernel<T, BM, BN, kForward>), dim3(a.total), dim3(256), 0, st, a);            \
  else hipLaunchKernelGGL((grouped_kernel<T, BM, BN, kBackInput>), dim3(a.total), dim3(256), 0, st, a);                           \
  if (p.splits > 1) hipLaunchKernelGGL(grouped_row_sum_kernel<T>, dim3((unsigned)cdiv(a.rows * cdiv(a.n, 64), 4)), dim3(256), 0, st, a)
#define VC_TILES(T)                                       \
  if (p.bm == 128) { VC_GO(T, 128, 128); }                \
  else if (p.bm == 64) { VC_GO(T, 64, 64); }              \
  else { VC_GO(T, 16, 128); }
  if (dtype == VC_F32) { VC_TILES(float) } else if (dtype == VC_F16) { VC_TILES(_Float16) } else { VC_TILES(__bf16) }
#undef VC_TILES
#undef VC_GO
  VC_CHECK_LAUNCH(who);
  return VC_OK;
}

}  // namespace vc

using namespace vc;

extern "C" {

size_t vc_grouped_linear_workspace_bytes(int direction, int64_t rows, int64_t groups, int64_t in, int64_t out, int dtype) {
  if (rows <= 0 || groups <= 0 || in <= 0 || out <= 0 || !grouped_dtype(dtype)) return 0;
  const GroupPlan p = direction == kForward ? plan_rows(rows, groups, out, in, dtype)
                      : direction == kBackInput ? plan_rows(rows, groups, in, out, dtype) : plan_weight(rows, groups, out, in, dtype);
  return (size_t)p.partial_floats * sizeof(float);
}

int vc_grouped_linear_forward(const void* x, int64_t x_stride, int64_t rows, const void* weight, const void* bias, const void* offsets,
                              int offset_bits, int64_t groups, int64_t in, int64_t out, int dtype, void* y, void* workspace,
                              size_t workspace_bytes, void* stream) {
  const int ok = grouped_check("vc_grouped_linear_forward", rows, groups, in, out, dtype, offset_bits, offsets);
  if (ok != VC_OK) return ok;
  if (rows == 0) return VC_OK;
  VC_REQUIRE(x && y && (weight || groups == 0), "vc_grouped_linear_forward: NULL pointer");
  VC_REQUIRE(x_stride >= in || rows == 1, "vc_grouped_linear_forward: row stride %lld below %lld channels", (long long)x_stride, (long long)in);
  GroupArgs a{};
  a.a = x; a.lda = x_stride; a.b = weight; a.bias = bias; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = y;
  a.rows = rows; a.groups = (int)groups; a.n = (int)out; a.k = (int)in;
  return launch_rows("vc_grouped_linear_forward", a, kForward, dtype, plan_rows(rows, groups, out, in, dtype), workspace, workspace_bytes, (hipStream_t)stream);
}

int vc_grouped_linear_backward_input(const void* dy, int64_t dy_stride, int64_t rows, const void* weight, const void* offsets, int offset_bits,
                                     int64_t groups, int64_t in, int64_t out, int dtype, void* dx, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  const int ok = grouped_check("vc_grouped_linear_backward_input", rows, groups, in, out, dtype, offset_bits, offsets);
  if (ok != VC_OK) return ok;
  if (rows == 0) return VC_OK;
  VC_REQUIRE(dy && dx && (weight || groups == 0), "vc_grouped_linear_backward_input: NULL pointer");
  VC_REQUIRE(dy_stride >= out || rows == 1, "vc_grouped_linear_backward_input: row stride %lld below %lld channels", (long long)dy_stride, (long long)out);
  GroupArgs a{};
  a.a = dy; a.lda = dy_stride; a.b = weight; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = dx;
  a.rows = rows; a.groups = (int)groups; a.n = (int)in; a.k = (int)out;
  return launch_rows("vc_grouped_linear_backward_input", a, kBackInput, dtype, plan_rows(rows, groups, in, out, dtype), workspace, workspace_bytes, (hipStream_t)stream);
}

int vc_grouped_linear_backward_weight(const void* x, int64_t x_stride, const void* dy, int64_t dy_stride, int64_t rows, const void* offsets,
                                      int offset_bits, int64_t groups, int64_t in, int64_t out, int dtype, void* dweight, void* dbias,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "vc_grouped_linear_backward_weight";
  const int ok = grouped_check(who, rows, groups, in, out, dtype, offset_bits, offsets);
  if (ok != VC_OK) return ok;
  if (groups == 0) return VC_OK;
  VC_REQUIRE(dweight && (rows == 0 || (x && dy)), "%s: NULL pointer", who);
  VC_REQUIRE((x_stride >= in && dy_stride >= out) || rows <= 1, "%s: row strides %lld, %lld below %lld, %lld channels", who, (long long)x_stride,
             (long long)dy_stride, (long long)in, (long long)out);
  const GroupPlan p = plan_weight(rows, groups, out, in, dtype);
  const size_t need = (size_t)p.partial_floats * sizeof(float);
  VC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, need %zu", who, workspace_bytes, need);
  GroupArgs a{};
  a.a = dy; a.lda = dy_stride; a.b = x; a.ldb = x_stride; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = dweight; a.dbias = dbias;
  a.rows = rows; a.groups = (int)groups; a.m = (int)out; a.n = (int)in;
  a.splits = p.splits; a.per_split = p.per_split;
  a.mtiles = (int)cdiv(out, p.bm); a.ntiles = (int)cdiv(in, p.bn);
  a.partial = (float*)workspace;
  a.partial_bias = a.partial + p.mtiles_most * out * in;
  const int64_t total = p.mtiles_most * a.mtiles * a.ntiles;
  VC_REQUIRE(total < (1LL << 31), "%s: %lld tiles", who, (long long)total);
  a.total = (unsigned)total;
  hipStream_t st = (hipStream_t)stream;
  const int64_t sum_blocks = cdiv(out * in + out, 64);
#define VC_GO(T)                                                                                                                              \
  if (p.bm == 128) hipLaunchKernelGGL((grouped_kernel<T, 128, 128, kBackWeight>), dim3(a.total), dim3(256), 0, st, a);                        \
  else hipLaunchKernelGGL((grouped_kernel<T, 64, 64, kBackWeight>), dim3(a.total), dim3(256), 0, st, a);                                      \
  if (p.splits > 1)                                                                                                                           \
    hipLaunchKernelGGL(grouped_weight_sum_kernel<T>, dim3((unsigned)(sum_blocks < 16384 ? sum_blocks : 16384), (unsigned)groups), dim3(256), 0, st, a)
  if (dtype == VC_F32) { VC_GO(float); } else if (dtype == VC_F16) { VC_GO(_Float16); } else { VC_GO(__bf16); }
#undef VC_GO
  VC_CHECK_LAUNCH(who);
  return VC_OK;
}

}  // extern "C"
