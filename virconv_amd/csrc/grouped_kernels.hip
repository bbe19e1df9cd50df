// Products of ragged row groups with one weight matrix per group: rows [offsets[g], offsets[g + 1]) of x meet W_g (out x in).
//
//   forward         y_r  = W_g x_r + b_g                 a row product, both operands along the inner axis
//   backward input  dx_r = W_g^T dy_r                    a row product, the weights across it
//   backward weight dW_g = sum_r dy_r x_r^T, db_g = sum_r dy_r     both operands across the summed axis (the group's rows)
//
// One output tile per block on v_mfma_f32_16x16x32, fp32 accumulation, one rounding at the end.  The tile's operands go through LDS as
// 16-bit values: as they are where the tensors are f16 or bf16, and where they are fp32 as three bf16 pieces x = h + m + l, each rounded to nearest,
// so that |m| <= 2^-8 |x|, |l| <= 2^-17 |x| and nothing is left -- six of the nine cross terms are issued, the dropped ones (m l, l m, l l) stay below
// 2^-24 of a product.  (Pieces that are cut off instead take as many operations and as long, and drop up to 2^-21, always towards zero.)  A number from
// 2^128 - 2^119 on rounds to an infinite h, and its products are undefined; a largest finite h in its place is two operations more for two elements
// and costs 2 to 6 per cent (4096^3: 620 and 665 us).  What lies below 2^-133 of an operand has no bf16 and is lost.  The matrix unit cuts what it
// adds to a larger product at 2^-23 of that, so a sum of one product is within 3 x 2^-24 of it.  An operand that lies along the summed axis is read back
// with ds_read_b128, one that lies across it with ds_read_b64_tr_b16 (four rows by sixteen columns a 16-lane group, transposed on the way);
// the 16-byte (32-byte) pieces of a row are exchanged by a function of the row, so that either read touches every bank once.
//
// The group sizes are known on the device only (a router's output needs no trip to the host): the grid is sized for the most tiles that
// `rows` and `groups` allow, and every block finds its group by a scan of the offsets.  Offsets are taken as a rising sequence within
// [0, rows]; one that is not is cut to it, so no content of `offsets` leads out of the tensors.  Rows of no group come out as zeros.
#include "common.h"

#include <initializer_list>

namespace vc {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
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
};

// ------------------------------------------------------------------------------------------------ the groups
__device__ __forceinline__ int offset_at(const GroupArgs& a, int g) {   // (rows < 2^31)
  const int64_t o = a.off64 ? ((const int64_t*)a.offsets)[g] : (int64_t)((const int32_t*)a.offsets)[g];
  return o < 0 ? 0 : o > a.rows ? (int)a.rows : (int)o;
}

// inclusive scans over the 64 lanes, of values >= 0: shifts within a row of 16, then the rows' last lanes handed on
template <int CTRL, int ROWS> __device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int scan_add(int x) {
  x += moved<0x111, 0xf>(x); x += moved<0x112, 0xf>(x); x += moved<0x114, 0xf>(x); x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x); x += moved<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ int scan_max(int x) {
  x = max(x, moved<0x111, 0xf>(x)); x = max(x, moved<0x112, 0xf>(x)); x = max(x, moved<0x114, 0xf>(x)); x = max(x, moved<0x118, 0xf>(x));
  x = max(x, moved<0x142, 0xa>(x)); x = max(x, moved<0x143, 0xc>(x));
  return x;
}

struct Place { int group, begin, end, tile; };   // group = groups: none

// The groups as a wave sees them, 64 at a time, one a lane: their rows (the offsets as a rising sequence), their tiles of `per` rows and the
// running count of those.  Every wave of a block holds them for itself; up to 64 groups they are read once.
struct Groups {
  int begin, end, tiles, upto;        // the lane's group
  int first_row, last_end, total;     // rows in front of the groups, the groups' last end, their tiles

  __device__ __forceinline__ void load(const GroupArgs& a, int per, int g0, int high) {
    const int g = g0 + (threadIdx.x & 63);
    end = max(scan_max(g < a.groups ? offset_at(a, g + 1) : 0), high);
    begin = __builtin_amdgcn_update_dpp(high, end, 0x138, 0xf, 0xf, false);   // the neighbour's end
    tiles = g < a.groups ? (int)(((int64_t)end - begin + per - 1) / per) : 0;
    upto = scan_add(tiles);
  }
  __device__ __forceinline__ Groups(const GroupArgs& a, int per) {
    begin = end = tiles = upto = first_row = last_end = total = 0;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
      if (g0 == 0) first_row = last_end = offset_at(a, 0);
      load(a, per, g0, last_end);
      total += __builtin_amdgcn_readlane(upto, 63);
      last_end = __builtin_amdgcn_readlane(end, 63);
    }
    first_row = __builtin_amdgcn_readfirstlane(first_row);
  }
  // the group of tile `target` (of the groups' tiles, `times` of them counted for one), and the tile's number in it
  __device__ __forceinline__ Place of_tile(const GroupArgs& a, int per, unsigned target, unsigned times) {
    int high = first_row;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
      if (a.groups > 64) load(a, per, g0, high);
      const uint64_t hit = __ballot(target < (unsigned)upto * times);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        const unsigned before = (unsigned)(__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l)) * times;
        return {g0 + l, __builtin_amdgcn_readlane(begin, l), __builtin_amdgcn_readlane(end, l), (int)(target - before)};
      }
      target -= (unsigned)__builtin_amdgcn_readlane(upto, 63) * times;
      high = __builtin_amdgcn_readlane(end, 63);
    }
    return {a.groups, 0, 0, (int)target};
  }
  // the group with the r-th most rows (up to 64 groups; above, group r)
  __device__ __forceinline__ Place of_rank(const GroupArgs& a, int per, int r) {
    if (a.groups > 64) {
      int high = first_row;
      for (int g0 = 0; g0 < a.groups; g0 += 64) {
        load(a, per, g0, high);
        if (r < g0 + 64) return {r, __builtin_amdgcn_readlane(begin, r - g0), __builtin_amdgcn_readlane(end, r - g0), 0};
        high = __builtin_amdgcn_readlane(end, 63);
      }
    }
    const int lane = threadIdx.x & 63, size = end - begin;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const int other = __builtin_amdgcn_readlane(size, g);
      rank += other > size || (other == size && g < lane);
    }
    const uint64_t hit = __ballot(rank == r && lane < a.groups);
    const int l = hit ? __builtin_ctzll(hit) : 0;
    return {l, __builtin_amdgcn_readlane(begin, l), __builtin_amdgcn_readlane(end, l), 0};
  }
};

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
  } else if (valid > 0) {   // eight loads side by side: the missing ones read the last element that there is
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = p[i < valid ? i : valid - 1];
#pragma unroll
    for (int i = 1; i < 8; ++i)
      if (i >= valid) out[i] = (T)0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = (T)0.f;
  }
}

// two values as bf16, rounded to nearest; and what the two are
__device__ __forceinline__ uint32_t nearest2(float lo, float hi) {
  typedef float v2f __attribute__((ext_vector_type(2)));
  typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2bf));
}
__device__ __forceinline__ float low_half(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// eight elements, as 32-bit words
template <typename T> struct Words { static constexpr int n = sizeof(T) * 2; uint32_t w[n]; };

template <typename T>
__device__ __forceinline__ Words<T> load_words(const void* p) {   // all eight, at any alignment that the elements have
  struct __attribute__((packed, aligned(sizeof(T)))) Raw { uint32_t w[Words<T>::n]; };
  Words<T> x;
  const Raw r = *reinterpret_cast<const Raw*>(p);
#pragma unroll
  for (int i = 0; i < Words<T>::n; ++i) x.w[i] = r.w[i];
  return x;
}

// (by value: a choice between two array elements would be made between their addresses, and put the array into memory)
__device__ __forceinline__ uint32_t choose(bool first, uint32_t x, uint32_t y) { return first ? x : y; }

// the elements `shift` places on (to the front), zeros from the `valid`-th on
template <typename T>
__device__ __forceinline__ void shift_words(Words<T>& x, int shift, int valid) {
  constexpr int n = Words<T>::n, per = 4 / sizeof(T);     // elements a word
#pragma unroll
  for (int step = 4; step >= per; step >>= 1)
#pragma unroll
    for (int k = 0; k + step / per < n; ++k) x.w[k] = choose(shift & step, x.w[k + step / per], x.w[k]);
  if constexpr (per == 2) {
#pragma unroll
    for (int k = 0; k < n; ++k) x.w[k] = choose(shift & 1, __builtin_amdgcn_alignbyte(k + 1 < n ? x.w[k + 1] : 0u, x.w[k], 2), x.w[k]);
  }
#pragma unroll
  for (int k = 0; k < n; ++k) {
    const int left = valid - k * per;
    x.w[k] &= left <= 0 ? 0u : per == 2 && left == 1 ? 0xffffu : 0xffffffffu;
  }
}

// eight elements into their place(s) in LDS: one 16-byte piece, or three planes of it
template <typename T>
__device__ __forceinline__ void stage8(char* lds, int plane_bytes, int at, const Words<T>& x) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(lds + at) = make_uint4(x.w[0], x.w[1], x.w[2], x.w[3]);
  } else {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v0 = __uint_as_float(x.w[2 * i]), v1 = __uint_as_float(x.w[2 * i + 1]);
      w[0][i] = nearest2(v0, v1);
      const float r0 = v0 - low_half(w[0][i]), r1 = v1 - high_half(w[0][i]);
      w[1][i] = nearest2(r0, r1);
      w[2][i] = nearest2(r0 - low_half(w[1][i]), r1 - high_half(w[1][i]));
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(lds + q * plane_bytes + at) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
  }
}

// A tile of one operand in LDS.  ALONG: [rows][BK], pieces of 8 along the summed axis; else [BK][cols], pieces of 8 across it.
template <typename T, int ROWS, bool ALONG, int THREADS = 256>
struct Tile {
  static constexpr int BK = OperandOf<T>::bk, planes = OperandOf<T>::planes;
  static constexpr int plane_bytes = ROWS * BK * 2, bytes = plane_bytes * planes;
  static constexpr int pieces = ROWS * BK / 8, per_thread = (pieces + THREADS - 1) / THREADS;

  static __device__ __forceinline__ int place(int r, int k) {   // byte of element (row r, summed index k); r or k a multiple of 8
    if constexpr (ALONG) {
      constexpr int CH = BK / 8, R = 16 / CH;                   // pieces a row, rows per 256 bytes
      // ds_read_b128 serves lanes 0-3, 12-15, 20-23, 24-27 (and so on) together: with four pieces a row the plain order would let rows 0-3
      // and 4-7 meet, so the four row groups exchange by 0, 2, 3, 1
      const int f = CH == 4 ? 0x78 >> ((r / R & 3) << 1) : r / R;
      return r * BK * 2 + ((((k >> 3) ^ f) & (CH - 1)) << 4);
    } else {
      constexpr int SLOTS = ROWS / 16;                          // 32-byte slots a row (of the summed axis)
      const int f = SLOTS >= 8 ? ((k & 3) | ((k >> 1) & 4)) : SLOTS == 4 ? (((k >> 1) & 1) | ((k >> 2) & 2)) : SLOTS == 2 ? ((k >> 3) & 1) : 0;
      return k * ROWS * 2 + ((((r >> 4) ^ f) & (SLOTS - 1)) << 5) + ((r & 15) << 1);
    }
  }

  Words<T> reg[per_thread];

  // rows [0, rows) and summed indices [0, depth) of the tile exist; p: the tile's first element, ld: the stride of its slow axis
  __device__ __forceinline__ void fetch(const T* p, int64_t ld, int rows, int depth) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * THREADS + threadIdx.x;
      if (pieces % THREADS && q >= pieces) continue;
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
      T e[8];
      load8(s, valid, e);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j) reg[i].w[j] = __builtin_bit_cast(uint32_t, e[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          reg[i].w[j] = (uint32_t)__builtin_bit_cast(uint16_t, e[2 * j]) | (uint32_t)__builtin_bit_cast(uint16_t, e[2 * j + 1]) << 16;
      }
    }
  }
  // The same with as many loads whatever exists (a load in a branch would have to be waited for at its end): a piece that reaches behind the
  // operand is read from where it just fits, a row that is not there as one that is, and `mend` puts the elements in their places and zeros
  // behind the ends.  For operands of at least eight elements either way and ld < 2^22.  `rest`: summed indices from the tile's first on.
  static constexpr int kBias = BK > ROWS ? BK : ROWS;          // keeps the 32-bit offsets positive where a piece begins in front of the tile
  static __device__ __forceinline__ void offsets_for(uint32_t (&from)[per_thread], int64_t ld, int rows, int rest) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = min(i * THREADS + (int)threadIdx.x % THREADS, pieces - 1);
      if constexpr (ALONG) from[i] = ((uint32_t)min(q / (BK / 8), rows - 1) * (uint32_t)ld + (kBias + min(q % (BK / 8) * 8, rest - 8))) * sizeof(T);
      else from[i] = ((uint32_t)min(q / (ROWS / 8), rest - 1) * (uint32_t)ld + (kBias + min(q % (ROWS / 8) * 8, rows - 8))) * sizeof(T);
    }
  }
  __device__ __forceinline__ void load(const T* p, const uint32_t (&from)[per_thread]) {
    const char* base = (const char*)(p - kBias);
#pragma unroll
    for (int i = 0; i < per_thread; ++i) reg[i] = load_words<T>(base + from[i]);
  }
  static __device__ __forceinline__ bool ragged(int rows, int rest) { return rest < BK || (!ALONG && rows < ROWS); }
  __device__ __forceinline__ void mend(int rows, int rest) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * THREADS + (int)threadIdx.x % THREADS;
      int valid;
      if constexpr (ALONG) valid = rest - q % (BK / 8) * 8;
      else valid = q / (ROWS / 8) < rest ? rows - q % (ROWS / 8) * 8 : 0;
      shift_words<T>(reg[i], valid >= 8 ? 0 : 8 - valid, valid);
    }
  }
  __device__ __forceinline__ void put(char* lds) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * THREADS + threadIdx.x;
      if (pieces % THREADS && q >= pieces) continue;
      int at;
      if constexpr (ALONG) at = place(q / (BK / 8), (q % (BK / 8)) * 8);
      else at = place((q % (ROWS / 8)) * 8, q / (ROWS / 8));
      stage8<T>(lds, plane_bytes, at, reg[i]);
    }
  }
  // The tile straight from memory into LDS, 16 bytes a lane (16-bit operands whose pieces are all aligned): the order of the lanes' pieces in
  // LDS is given, so a lane reads the piece that belongs at its place.  Rows that are not there read one that is: they only enter results that
  // are not written.  Every summed index of the tile has to exist.
  // `from`: the byte offsets of the lane's pieces in the tensor's tile, to be made once per tile (256 rows of up to 2^22 elements: 32 bits).
  static __device__ __forceinline__ void offsets(uint32_t (&from)[per_thread], int64_t ld, int rows) {
#pragma unroll
    for (int i = 0; i < per_thread; ++i) {
      const int q = i * THREADS + threadIdx.x;
      if constexpr (ALONG) {
        constexpr int CH = BK / 8, R = 16 / CH;
        const int r = q / CH, k = ((q ^ (r / R)) & (CH - 1)) * 8;
        from[i] = ((uint32_t)min(r, rows - 1) * (uint32_t)ld + k) * 2;
      } else {
        const int k = q / (ROWS / 8), c0 = (q % (ROWS / 8)) * 8;
        const int f = (k & 3) | ((k >> 1) & 4), c = ((((c0 >> 4) ^ f) & (ROWS / 16 - 1)) << 4) | (c0 & 8);
        from[i] = ((uint32_t)k * (uint32_t)ld + (c < rows ? c : 0)) * 2;
      }
    }
  }
  static __device__ __forceinline__ void copy(char* lds, const T* p, const uint32_t (&from)[per_thread]) {
    static_assert(pieces % THREADS == 0 && planes == 1, "whole waves of pieces");
    typedef __attribute__((address_space(1))) const void global_void;
    typedef __attribute__((address_space(3))) void lds_void;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < per_thread; ++i)
      __builtin_amdgcn_global_load_lds((global_void*)((const char*)p + from[i]), (lds_void*)(lds + (i * THREADS + wave * 64) * 16), 16, 0, 0);
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

// The sums of a wave's operands of a tile along the summed axis (dbias from dy), by products with ones.  The WN waves that hold the same FM operands
// take every WN-th.  Each operand's sum of a step stands by itself: with ones in one row of a result that several operands share, an infinite value
// would bring 0 * inf into the sums of the others.  Every row of the result holds the same sums, of which a lane keeps one, that of channel lane % 16
// (kept as the instruction's four, or unrolled, the 256 x 256 tiles spill; in a loop the fp32 tiles are 2 to 5 per cent slower).  The operands are
// read once more: between the other products this would cut those into pieces that wait for their own reads (weight product with a bias or without,
// 8192^3: 1010 TFLOP/s so).
template <int FM, int WN> struct BiasSums { static constexpr int n = (FM + WN - 1) / WN; float acc[n]; };
template <typename T, typename Tile, int FM, int WN>
__device__ __forceinline__ void add_bias_sums(const char* lds, int wm0, int wn, BiasSums<FM, WN>& sums) {
  static_assert(FM % WN == 0, "as many operands a wave");
  constexpr short one = __is_same(T, _Float16) ? (short)0x3c00 : (short)0x3f80;
  constexpr int kTogether = FM < 8 ? BiasSums<FM, WN>::n : 1;
#pragma unroll kTogether
  for (int s = 0; s < sums.n; ++s) {
    const int at = Tile::lane_place(wm0 + (s * WN + wn) * 16);
    v4f step = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kk = 0; kk < Tile::BK; kk += 32)
#pragma unroll
      for (int q = Tile::planes - 1; q >= 0; --q)
        step = mfma<T>(v8s{one, one, one, one, one, one, one, one}, Tile::fragment(lds, q, at, kk), step);
#pragma unroll
    for (int t = 0; t < sums.n; ++t) sums.acc[t] = t == s ? sums.acc[t] + step[0] : sums.acc[t];
  }
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

// ------------------------------------------------------------------------------------------------ tiles of a block
// What a block computes: where its operands begin, how much of them there is, where its results go.
template <typename T> struct Work {
  int64_t pa, pb;          // elements behind a.a and a.b
  int64_t lda, ldb, m0;
  int rows_a, rows_b, depth, group, n0;
  unsigned piece;
  float* partial;
  bool none;
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) { return (int64_t)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x)); }
template <typename T> __device__ __forceinline__ Work<T> uniform(const Work<T>& w) {   // into scalar registers
  return {uniform(w.pa), uniform(w.pb), uniform(w.lda), uniform(w.ldb), uniform(w.m0), uniform(w.rows_a), uniform(w.rows_b), uniform(w.depth),
          uniform(w.group), uniform(w.n0), (unsigned)uniform((int)w.piece), w.partial, (bool)uniform((int)w.none)};
}

// Consecutive blocks go to the eight XCDs in turn; the blocks of one XCD take neighbouring items, which share operands in its L2.
//
// Row products: the items are the tiles (x splits) that the groups really have, each XCD an eighth of them, within a group in bands of four
// column tiles.  Weight products without splits: the groups by their size, the largest first (their tiles take longest), and each group's
// tiles dealt out over all XCDs.
struct Items {
  unsigned count;      // of an XCD: the local items [0, count), item l of XCD x
  unsigned first;      // row products: the XCD's first item
};
template <int MODE>
__device__ __forceinline__ Items items_of(const GroupArgs& a, const Groups& g, int bm, unsigned x) {
  if (MODE == kBackWeight && a.splits == 1) {
    const unsigned tiles = (unsigned)a.mtiles * a.ntiles;
    return {tiles >= 8 ? (tiles + 7) / 8 * a.groups : (tiles * a.groups + 7 - x) / 8, 0u};
  }
  unsigned all;
  if (MODE == kBackWeight) all = (unsigned)g.total * a.mtiles * a.ntiles;
  else all = (unsigned)(g.total + (g.first_row + bm - 1) / bm + (int)((a.rows - g.last_end + bm - 1) / bm)) * a.ntiles * a.splits;
  const unsigned per = all / 8, rest = all % 8;
  return {per + (x < rest ? 1u : 0u), x * per + (x < rest ? x : rest)};
}

template <typename T, int BM, int BN, int MODE, int THREADS>
__device__ __forceinline__ Work<T> find_work(const GroupArgs& a, Groups& g, const Items& items, unsigned x, unsigned l) {
  Work<T> w;
  w.none = true;
  w.partial = nullptr;
  w.piece = 0;
  if constexpr (MODE != kBackWeight) {
    unsigned id = items.first + l;
    const int split = (int)(id % a.splits);
    id /= a.splits;
    const Place at = g.of_tile(a, BM, id, a.ntiles);
    if (at.group == a.groups) {   // rows of no group: in front of the first and behind the last
      if (split) return w;
      const int t = at.tile / a.ntiles, front_tiles = (g.first_row + BM - 1) / BM;
      w.n0 = at.tile % a.ntiles * BN;
      const int64_t lo = t < front_tiles ? (int64_t)t * BM : g.last_end + (int64_t)(t - front_tiles) * BM;
      const int64_t hi = min(lo + BM, t < front_tiles ? (int64_t)g.first_row : a.rows);
      for (int64_t e = threadIdx.x; lo < hi && e < (hi - lo) * BN; e += THREADS) {
        const int n = w.n0 + (int)(e % BN);
        if (n < a.n) ((T*)a.out)[(lo + e / BN) * a.n + n] = (T)0.f;
      }
      return w;
    }
    const int mtiles = (at.end - at.begin + BM - 1) / BM, band = at.tile / (4 * mtiles), wide = min(4, a.ntiles - 4 * band), in = at.tile - 4 * band * mtiles;
    w.n0 = (4 * band + in % wide) * BN;
    w.group = at.group;
    w.m0 = at.begin + (int64_t)(in / wide) * BM;
    const int k0 = split * a.per_split;
    w.depth = min(a.per_split, a.k - k0);
    w.rows_a = (int)min((int64_t)BM, at.end - w.m0);
    w.lda = a.lda;
    w.pa = w.m0 * a.lda + k0;
    const int64_t weights = (int64_t)w.group * a.n * a.k;
    w.ldb = MODE == kForward ? a.k : a.n;
    w.pb = MODE == kForward ? weights + (int64_t)w.n0 * a.k + k0 : weights + (int64_t)k0 * a.n + w.n0;
    if (a.splits > 1) w.partial = a.partial + ((int64_t)split * a.rows + w.m0) * a.n + w.n0;
  } else {
    const unsigned tiles = (unsigned)a.mtiles * a.ntiles;
    unsigned t;
    int64_t r0, r1;
    bool pieces = false;         // the sums of a group of one piece are its result
    if (a.splits > 1) {          // pieces of per_split rows, their sums added by grouped_weight_sum_kernel
      const unsigned id = items.first + l;
      t = id % tiles;
      w.piece = id / tiles;
      const Place at = g.of_tile(a, a.per_split, w.piece, 1);
      if (at.group == a.groups) return w;
      w.group = at.group;
      r0 = at.begin + (int64_t)at.tile * a.per_split;
      r1 = min(r0 + a.per_split, (int64_t)at.end);
      pieces = at.end - at.begin > a.per_split;
    } else {
      const unsigned share = (tiles + 7) / 8;
      const unsigned r = tiles >= 8 ? l / share : (l * 8 + x) / tiles;
      t = tiles >= 8 ? x * share + l % share : (l * 8 + x) % tiles;
      if (t >= tiles) return w;
      const Place at = g.of_rank(a, a.per_split, (int)r);
      w.group = at.group;
      r0 = at.begin;
      r1 = at.end;
    }
    w.n0 = (int)(t % a.ntiles) * BN;
    w.m0 = (int64_t)(t / a.ntiles) * BM;
    if (pieces) w.partial = a.partial + ((int64_t)w.piece * a.m + w.m0) * a.n + w.n0;
    w.depth = (int)(r1 - r0);
    w.rows_a = (int)min((int64_t)BM, (int64_t)a.m - w.m0);
    w.lda = a.lda;
    w.ldb = a.ldb;
    w.pa = r0 * a.lda + w.m0;
    w.pb = r0 * a.ldb + w.n0;
  }
  w.rows_b = min(BN, a.n - w.n0);
  w.none = false;
  return w;
}

// Results of a wave: lane l holds row m = l % 16 and the columns n = 4 (l / 16) .. + 3 of each 16 x 16 tile; (wm0, wn0): the wave's place.
template <typename T, int FM, int FN, int MODE>
__device__ __forceinline__ void write_results(const GroupArgs& a, const Work<T>& w, int wm0, int wn0, const v4f (&acc)[FM][FN]) {
  const int lane = threadIdx.x & 63;
  if (w.rows_a >= wm0 + FM * 16 && w.rows_b >= wn0 + FN * 16) {   // the wave's part of the tile is whole
    const int64_t at = (int64_t)(wm0 + (lane & 15)) * a.n + wn0 + (lane >> 4) * 4;
    float* part = w.partial ? w.partial + at : nullptr;
    T* out = (T*)a.out + ((MODE == kBackWeight ? (int64_t)w.group * a.m : 0) + w.m0) * a.n + w.n0 + at;
    struct __attribute__((packed, aligned(sizeof(T)))) Four { T v[4]; } bias[FN] = {};
    if (MODE == kForward && a.bias && !part) {
#pragma unroll
      for (int j = 0; j < FN; ++j) __builtin_memcpy(&bias[j], (const T*)a.bias + (int64_t)w.group * a.n + w.n0 + wn0 + j * 16 + (lane >> 4) * 4, sizeof(bias[j]));
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        float r[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        if (MODE == kForward) {
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] += (float)bias[j].v[e];
        }
        if (part) store4(part + j * 16, 4, r);
        else store4(out + j * 16, 4, r);
      }
      if (part) part += (int64_t)16 * a.n;
      out += (int64_t)16 * a.n;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int m = wm0 + i * 16 + (lane & 15);
    if (m >= w.rows_a) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = wn0 + j * 16 + (lane >> 4) * 4;
      if (n >= w.rows_b) continue;
      float r[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (w.partial) {
        store4(w.partial + (int64_t)m * a.n + n, w.rows_b - n, r);
        continue;
      }
      if (MODE == kForward && a.bias) {
        const T* bias = (const T*)a.bias + (int64_t)w.group * a.n + w.n0 + n;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < w.rows_b) r[e] += (float)bias[e];
      }
      T* out = (T*)a.out;
      if constexpr (MODE == kBackWeight) out += ((int64_t)w.group * a.m + w.m0 + m) * a.n + w.n0 + n;
      else out += (w.m0 + m) * a.n + w.n0 + n;
      store4(out, w.rows_b - n, r);
    }
  }
}

// ... and what add_bias_sums made of a wave's operands
template <typename T, int FM, int WN>
__device__ __forceinline__ void write_bias(const GroupArgs& a, const Work<T>& w, int wm0, int wn, const BiasSums<FM, WN>& sums) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int s = 0; s < sums.n; ++s) {
    const int m = wm0 + (s * WN + wn) * 16 + (lane & 15);
    if (lane >= 16 || m >= w.rows_a) continue;
    if (w.partial) a.partial_bias[(int64_t)w.piece * a.m + w.m0 + m] = sums.acc[s];
    else ((T*)a.dbias)[(int64_t)w.group * a.m + w.m0 + m] = (T)sums.acc[s];
  }
}

// ------------------------------------------------------------------------------------------------ the kernel for every case
// WM of the four waves lie along m.  STAGES tiles are under way in registers ahead of the one that is multiplied (a short summed axis is asked
// for as a whole, a long one keeps that many times a tile in flight).
// SMALL: operands of fewer than eight elements one way or the other, or with longer strides than 32-bit offsets reach.
template <typename T, int BM, int BN, int WM, int STAGES, bool SMALL, int MODE>
__global__ void __launch_bounds__(256, 2) grouped_kernel(GroupArgs a) {
  typedef typename OperandOf<T>::type O;
  constexpr int BK = OperandOf<T>::bk, P = OperandOf<T>::planes;
  typedef Tile<T, BM, MODE != kBackWeight> TileA;
  typedef Tile<T, BN, MODE == kForward> TileB;
  constexpr int WN = 4 / WM, FM = BM / WM / 16, FN = BN / WN / 16;   // waves along n, fragments of a wave
  constexpr int kBuffer = TileA::bytes + TileB::bytes;
  __shared__ __align__(16) char lds[2 * kBuffer];
  const int wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;

  Groups groups(a, MODE == kBackWeight ? a.per_split : BM);
  const unsigned xcd = blockIdx.x % 8, item = blockIdx.x / 8;
  const Items items = items_of<MODE>(a, groups, BM, xcd);
  if (item >= items.count) return;
  const Work<T> w = find_work<T, BM, BN, MODE, 256>(a, groups, items, xcd, item);
  if (w.none) return;
  const T *const pa = (const T*)a.a + w.pa, *const pb = (const T*)a.b + w.pb;
  const int64_t lda = w.lda, ldb = w.ldb;
  const int rows_a = w.rows_a, rows_b = w.rows_b, depth = w.depth;
  const bool sum_bias = MODE == kBackWeight && a.dbias && w.n0 == 0;

  TileA ta[STAGES];
  TileB tb[STAGES];
  uint32_t from_a[TileA::per_thread], from_b[TileB::per_thread];
  if (!SMALL && depth > 0) {
    TileA::offsets_for(from_a, lda, rows_a, min(depth, BK));
    TileB::offsets_for(from_b, ldb, rows_b, min(depth, BK));
  }
  auto load = [&](int stage, int k0) {
    const int64_t k = k0;
    const T *p = pa + (MODE == kBackWeight ? k * lda : k), *q = pb + (MODE == kForward ? k : k * ldb);
    if constexpr (SMALL) {
      ta[stage].fetch(p, lda, rows_a, depth - k0);
      tb[stage].fetch(q, ldb, rows_b, depth - k0);
    } else {
      if (k0 && depth - k0 < BK) {
        TileA::offsets_for(from_a, lda, rows_a, depth - k0);
        TileB::offsets_for(from_b, ldb, rows_b, depth - k0);
      }
      ta[stage].load(p, from_a);
      tb[stage].load(q, from_b);
    }
  };
  const bool deep = depth > (2 * STAGES - 1) * BK;
  if (deep) {                  // (in the loop that runs on from here every load exists; one that might not would make each wait one for all)
#pragma unroll
    for (int d = 0; d < STAGES; ++d) load(d, d * BK);
  }
  v4f acc[FM][FN];
  BiasSums<FM, WN> bias_sums{};
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  int at_a[FM], at_b[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) at_a[i] = TileA::lane_place(wm * (BM / WM) + i * 16);
#pragma unroll
  for (int j = 0; j < FN; ++j) at_b[j] = TileB::lane_place(wn * (BN / WN) + j * 16);

  // One barrier a step: the two halves of LDS take turns, so that a wave may put the next tile while another still multiplies this one.
  int half = 0;
  auto put = [&](int d, int k0) {
    if constexpr (!SMALL) {
      if (TileA::ragged(rows_a, depth - k0)) ta[d].mend(rows_a, min(depth - k0, BK));
      if (TileB::ragged(rows_b, depth - k0)) tb[d].mend(rows_b, min(depth - k0, BK));
    }
    ta[d].put(lds + half);
    tb[d].put(lds + half + TileA::bytes);
  };
  auto multiply = [&] {
    const char *const la = lds + half, *const lb = la + TileA::bytes;
    half ^= kBuffer;
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
      }
    }
    if constexpr (MODE == kBackWeight) {
      if (sum_bias) add_bias_sums<O, TileA, FM, WN>(la, wm * (BM / WM), __builtin_amdgcn_readfirstlane(wn), bias_sums);
    }
  };
  int kb = 0;
  if (deep) {
    for (; kb + (2 * STAGES - 1) * BK < depth; kb += STAGES * BK) {
#pragma unroll
      for (int d = 0; d < STAGES; ++d) {
        put(d, kb + d * BK);
        __syncthreads();
        load(d, kb + (d + STAGES) * BK);
        multiply();
      }
    }
  } else {
#pragma unroll
    for (int d = 0; d < STAGES; ++d)
      if (d * BK < depth) load(d, d * BK);
  }
  for (; kb < depth; kb += STAGES * BK) {
#pragma unroll
    for (int d = 0; d < STAGES; ++d) {
      const int k0 = kb + d * BK;
      if (k0 >= depth) break;
      put(d, k0);
      __syncthreads();
      if (k0 + STAGES * BK < depth) load(d, k0 + STAGES * BK);
      multiply();
    }
  }
  write_results<T, FM, FN, MODE>(a, w, wm * (BM / WM), wn * (BN / WN), acc);
  if (MODE == kBackWeight && sum_bias) write_bias<T, FM, WN>(a, w, wm * (BM / WM), wn, bias_sums);
}

// ------------------------------------------------------------------------------------------------ large tiles of fp32 operands
// Cutting fp32 operands into three bf16 pieces takes half as many issue slots as their six products take matrix cycles, and in a wave that does
// both the two come one after the other (28 to 40 per cent of the matrix rate).  So each SIMD has one wave that loads, cuts and stores tiles and
// one that multiplies them: four waves of each kind, two halves of LDS, one barrier a step.  The block takes tiles until there are none, and
// the first kind is already at the next tile while the second writes its results.
//
// Measured: 4096^3 forward 223, backward input 219, weight 199 TFLOP/s (1340 of bf16 products; the clock falls with them: 170 to 223 by card); 480 x
// 27648 to 256 columns in 3 ragged groups 64, 75 and 67 us, 106 MB and 41 GFLOP of bf16 products each: tiles of rows that are not there and the
// unequal groups leave the compute units without work for 40 per cent of that time.
template <int BM, int BN, int MODE>
__global__ void __launch_bounds__(512, 2) grouped_f32_kernel(GroupArgs a) {
  constexpr int BK = 32, P = 3, STAGES = 2, WM = 2, WN = 2, FM = BM / WM / 16, FN = BN / WN / 16;
  typedef Tile<float, BM, MODE != kBackWeight> TileA;
  typedef Tile<float, BN, MODE == kForward> TileB;
  constexpr int kBuffer = TileA::bytes + TileB::bytes;
  __shared__ __align__(16) char lds[2 * kBuffer];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  Groups groups(a, MODE == kBackWeight ? a.per_split : BM);
  const unsigned xcd = blockIdx.x % 8, blocks = gridDim.x / 8, block = blockIdx.x / 8;
  const Items items = items_of<MODE>(a, groups, BM, xcd);
  unsigned round = 0;
  auto next = [&](Work<float>& w) {
    for (w.none = true; w.none && round * blocks < items.count; ++round) {
      const unsigned item = round * blocks + (round & 1 ? blocks - 1 - block : block);
      if (item < items.count) w = uniform(find_work<float, BM, BN, MODE, 512>(a, groups, items, xcd, item));
    }
  };
  auto meet = [] {           // what this wave wrote is there for the others, and they have come as far
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  };
  int half = 0;
  Work<float> w;
  next(w);
  if (wave < 4) {
    // The steps of all tiles are one stream: the loads run two steps ahead of the stores, into the next tile where this one ends.
    TileA ta[STAGES];
    TileB tb[STAGES];
    int rest[STAGES], rows_a[STAGES], rows_b[STAGES];        // rest 0: the stream has ended
    uint32_t from_a[TileA::per_thread], from_b[TileB::per_thread];
    int k0 = 0;
    auto settle = [&](bool fresh) {      // (k0 is a step of w, or there is none left)
      while (!w.none && k0 >= w.depth) { next(w); k0 = 0; fresh = true; }
      if (w.none || !(fresh || w.depth - k0 < BK)) return;
      TileA::offsets_for(from_a, w.lda, w.rows_a, min(w.depth - k0, BK));
      TileB::offsets_for(from_b, w.ldb, w.rows_b, min(w.depth - k0, BK));
    };
    int64_t at_pa = 0, at_pb = 0;
    auto fetch = [&](int d) {
      rest[d] = w.none ? 0 : min(w.depth - k0, BK);
      if (!w.none) {
        rows_a[d] = w.rows_a;
        rows_b[d] = w.rows_b;
        at_pa = w.pa + (MODE == kBackWeight ? (int64_t)k0 * w.lda : k0);
        at_pb = w.pb + (MODE == kForward ? k0 : (int64_t)k0 * w.ldb);
      }
      ta[d].load((const float*)a.a + at_pa, from_a);      // (behind the stream's end the last step once more: the number of loads under
      tb[d].load((const float*)a.b + at_pb, from_b);      // way has to be the same on every path, or all of them would be waited for)
      if (!w.none) {
        k0 += BK;
        settle(false);
      }
    };
    settle(true);
    if (w.none) return;
#pragma unroll
    for (int d = 0; d < STAGES; ++d) fetch(d);
    for (bool more = true; more;) {
#pragma unroll
      for (int d = 0; d < STAGES; ++d) {
        if (!rest[d]) { more = false; break; }
        if (TileA::ragged(rows_a[d], rest[d])) ta[d].mend(rows_a[d], rest[d]);
        if (TileB::ragged(rows_b[d], rest[d])) tb[d].mend(rows_b[d], rest[d]);
        ta[d].put(lds + half);
        tb[d].put(lds + half + TileA::bytes);
        half ^= kBuffer;
        fetch(d);
        meet();
      }
    }
    return;
  }
  const int wm = (wave - 4) / WN, wn = (wave - 4) % WN;
  int at_a[FM], at_b[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) at_a[i] = TileA::lane_place(wm * (BM / WM) + i * 16);
#pragma unroll
  for (int j = 0; j < FN; ++j) at_b[j] = TileB::lane_place(wn * (BN / WN) + j * 16);
  while (!w.none) {
    const bool sum_bias = MODE == kBackWeight && a.dbias && w.n0 == 0;
    v4f acc[FM][FN];
    BiasSums<FM, WN> bias_sums{};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < w.depth; k0 += BK) {
      meet();
      const char *la = lds + half, *lb = la + TileA::bytes;
      half ^= kBuffer;
      v8s fb[FN][P];
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int q = 0; q < P; ++q) fb[j][q] = TileB::fragment(lb, q, at_b[j], 0);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        v8s fa[P];
#pragma unroll
        for (int q = 0; q < P; ++q) fa[q] = TileA::fragment(la, q, at_a[i], 0);
        // the smallest terms first, each over all columns: neighbouring products do not wait for one another
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][2], fa[0], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][0], fa[2], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][1], fa[1], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][1], fa[0], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][0], fa[1], acc[i][j]);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<__bf16>(fb[j][0], fa[0], acc[i][j]);
      }
      if constexpr (MODE == kBackWeight) {
        if (sum_bias) add_bias_sums<__bf16, TileA, FM, WN>(la, wm * (BM / WM), wn, bias_sums);
      }
    }
    write_results<float, FM, FN, MODE>(a, w, wm * (BM / WM), wn * (BN / WN), acc);
    if (MODE == kBackWeight && sum_bias) write_bias<float, FM, WN>(a, w, wm * (BM / WM), wn, bias_sums);
    next(w);
  }
}

// ------------------------------------------------------------------------------------------------ large tiles of aligned 16-bit operands
// 256 (or 192) x 256 results a block of eight waves, 128 x 64 a wave: of the tiles that registers allow the one whose fragment reads (24 KB a wave
// and step of 64) stay below what its products take (a 128 x 128 tile of four waves keeps LDS exactly as busy as the matrix units and reached 570
// TFLOP/s).  The next step's operands come by LDS-direct loads into the other buffer while this one is multiplied: no registers, one barrier a
// step.  Within a step each fragment is read while the products of the one before it run.  What is left of the summed axis behind the last whole
// step goes through registers, with zeros behind its end.
//
// Measured, bf16: 8192^3 forward 1340 to 1385, backward input 1350 to 1380, weight 1140 to 1200 TFLOP/s by card (a library product 1313; both operands of the weight product come
// by ds_read_b64_tr_b16, twice the instructions); 32749 x 1024 -> 4096 in 16 ragged groups 960, 910, 970.  A tile's way in and out costs about as
// much as 400 summed indices, so short sums stay below the rate; steps of 32 in a ring of five buffers were 9 per cent slower.
constexpr int kLargeNarrow = 192, kLargeBuffer = (256 + 256) * 64 * 2;
template <typename T, int BM, int MODE>
__device__ __forceinline__ void large_products(const GroupArgs& a, Groups& groups, char* even, char* odd) {
  constexpr int BN = 256, BK = 64, WN = 4, FM = BM / 32, FN = 4;
  typedef Tile<T, BM, MODE != kBackWeight, 512> TileA;
  typedef Tile<T, BN, MODE == kForward, 512> TileB;
  static_assert(TileA::bytes + TileB::bytes <= kLargeBuffer, "");
  const int wave = threadIdx.x >> 6, wm0 = (wave / WN) * (FM * 16), wn0 = (wave % WN) * (FN * 16);
  int at_a[FM], at_b[FN];
#pragma unroll
  for (int i = 0; i < FM; ++i) at_a[i] = TileA::lane_place(wm0 + i * 16);
#pragma unroll
  for (int j = 0; j < FN; ++j) at_b[j] = TileB::lane_place(wn0 + j * 16);

  const unsigned xcd = blockIdx.x % 8, blocks = gridDim.x / 8;
  const Items items = items_of<MODE>(a, groups, BM, xcd);
  const unsigned block = blockIdx.x / 8;
  unsigned round = 0;
  auto next = [&](Work<T>& w) {
    // (there and back: a block that had one of the larger items of a round gets one of the smaller of the next)
    for (w.none = true; w.none && round * blocks < items.count; ++round) {
      const unsigned item = round * blocks + (round & 1 ? blocks - 1 - block : block);
      if (item < items.count) w = uniform(find_work<T, BM, BN, MODE, 512>(a, groups, items, xcd, item));
    }
  };
  uint32_t from_a[TileA::per_thread], from_b[TileB::per_thread];
  struct alignas(8) Four { T v[4]; };
  Four bias[FN];           // of the tile to come: asked for before the stores of the one that ends, which later loads queue behind
  auto copy = [&](char* lds, const Work<T>& w, int t) {
    TileA::copy(lds, (const T*)a.a + (w.pa + t * (MODE == kBackWeight ? BK * w.lda : BK)), from_a);
    TileB::copy(lds + TileA::bytes, (const T*)a.b + (w.pb + t * (MODE == kForward ? BK : BK * w.ldb)), from_b);
  };
  auto begin = [&](const Work<T>& w) {
    if (w.none) return;
    TileA::offsets(from_a, w.lda, w.rows_a);
    TileB::offsets(from_b, w.ldb, w.rows_b);
    if (MODE == kForward && a.bias) {
      const T* p = (const T*)a.bias + (int64_t)w.group * a.n + w.n0;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = wn0 + j * 16 + ((threadIdx.x & 63) >> 4) * 4;
        bias[j] = *reinterpret_cast<const Four*>(p + (n < w.rows_b ? n : 0));   // (sizes and pointers are multiples of eight elements)
      }
    }
    if (w.depth >= BK) copy(even, w, 0);
  };
  auto arrived = [&] {     // this wave's loads have landed, and every wave is done with the buffer that is filled next
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
  };

  Work<T> w;
  next(w);
  begin(w);
  while (!w.none) {
    const bool sum_bias = MODE == kBackWeight && a.dbias && w.n0 == 0;
    v4f acc[FM][FN];
    BiasSums<FM, WN> bias_sums{};
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      v4f start = v4f{0.f, 0.f, 0.f, 0.f};
      if (MODE == kForward && a.bias) start = v4f{(float)bias[j].v[0], (float)bias[j].v[1], (float)bias[j].v[2], (float)bias[j].v[3]};
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[i][j] = start;
    }
    auto multiply = [&](const char* lds) {
      v8s fb[2][FN], fa[2];      // (held in this order by the barriers: left to itself the compiler reads a fragment in front of its products and waits)
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[0][j] = TileB::fragment(lds + TileA::bytes, 0, at_b[j], 0);
      fa[0] = TileA::fragment(lds, 0, at_a[0], 0);
#pragma unroll
      for (int q = 0; q < BK / 32 * FM; ++q) {
        const int i = q % FM, h = q / FM, kk = h * 32;
        if (i + 1 < FM) fa[(q + 1) & 1] = TileA::fragment(lds, 0, at_a[i + 1], kk);
        else if (kk + 32 < BK) {
          fa[(q + 1) & 1] = TileA::fragment(lds, 0, at_a[0], kk + 32);
#pragma unroll
          for (int j = 0; j < FN; ++j) fb[h + 1][j] = TileB::fragment(lds + TileA::bytes, 0, at_b[j], kk + 32);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = mfma<T>(fb[h][j], fa[q & 1], acc[i][j]);
      }
      if constexpr (MODE == kBackWeight) {
        if (sum_bias) add_bias_sums<T, TileA, FM, WN>(lds, wm0, __builtin_amdgcn_readfirstlane(wave % WN), bias_sums);
      }
    };
    const int steps = w.depth / BK, rest = w.depth % BK;
    for (int t = 0; t < steps; t += 2) {
      arrived();
      if (t + 1 < steps) copy(odd, w, t + 1);
      multiply(even);
      if (t + 1 < steps) {
        arrived();
        if (t + 2 < steps) copy(even, w, t + 2);
        multiply(odd);
      }
    }
    if (rest) {
      char* lds = steps & 1 ? odd : even;
      {
        TileA ta;
        ta.fetch((const T*)a.a + w.pa + (int64_t)steps * (MODE == kBackWeight ? BK * w.lda : BK), w.lda, w.rows_a, rest);
        ta.put(lds);
        TileB tb;
        tb.fetch((const T*)a.b + w.pb + (int64_t)steps * (MODE == kForward ? BK : BK * w.ldb), w.ldb, w.rows_b, rest);
        tb.put(lds + TileA::bytes);
      }
      __syncthreads();
      multiply(lds);
    }
    Work<T> after;
    next(after);
    __syncthreads();       // every wave is done with both buffers:
    begin(after);          // the next tile is under way while this one's results are written
    // Two neighbouring column tiles at a time: a lane that holds four columns of either exchanges with its neighbour for eight of one, so that a
    // row's 64 bytes go out together.  The rows' results, of which nothing is read again here, are marked so, which leaves the L2s to the operands
    // (forward, 32768 x 1024 to 4096 columns in 16 groups: 350 us with 32 bytes a store, 333 with 64, 300 marked; 8192^3: 888, 875, 845.  The
    // weight product lost 2 percent by the mark.)
    const int lane = threadIdx.x & 63, m0 = wm0 + (lane & 15), nb = wn0 + (lane >> 4 & 1) * 16 + (lane >> 5) * 8;
    T* out = (T*)a.out + ((MODE == kBackWeight ? (int64_t)w.group * a.m : 0) + w.m0) * a.n + w.n0 + (int64_t)m0 * a.n + nb;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
      for (int j = 0; j < FN; j += 2) {
        uint2 e[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          Four f;
#pragma unroll
          for (int k = 0; k < 4; ++k) f.v[k] = (T)acc[i][j + h][k];
          e[h] = __builtin_bit_cast(uint2, f);
        }
        const auto x = __builtin_amdgcn_permlane16_swap(e[0].x, e[1].x, false, false);   // lanes 16-31 of one with lanes 0-15 of the other,
        const auto y = __builtin_amdgcn_permlane16_swap(e[0].y, e[1].y, false, false);   // and 48-63 with 32-47
        const v4u eight = {x[0], y[0], x[1], y[1]};
        if (m0 + i * 16 < w.rows_a && nb + j * 16 < w.rows_b) {
          if (MODE == kBackWeight) *reinterpret_cast<v4u*>(out + j * 16) = eight;
          else __builtin_nontemporal_store(eight, reinterpret_cast<v4u*>(out + j * 16));
        }
      }
      out += (int64_t)16 * a.n;
    }
    if (MODE == kBackWeight && sum_bias) write_bias<T, FM, WN>(a, w, wm0, wave % WN, bias_sums);
    w = after;
  }
}

// Rows of a tile: 256, or 192 where that takes less time in whole rounds of the blocks: a round costs its products (at 192 rows at a rate that is
// 3 per cent lower) and the way in and out, as much as 400 summed indices of 256 rows.  The groups' real tiles decide (32749 rows in 16 groups, the
// largest three times the smallest, 4096 summed indices, 1024 columns: 2.2 rounds of 256 rows, 355 and 317 us; 2.8 of 192, 334 and 287).
template <typename T, int MODE>
__global__ void __launch_bounds__(512, 2) grouped_large_kernel(GroupArgs a) {
  __shared__ __align__(16) char even[kLargeBuffer];
  __shared__ __align__(16) char odd[kLargeBuffer];
  Groups groups(a, MODE == kBackWeight ? a.per_split : 256);
  if constexpr (MODE != kBackWeight) {
    Groups narrow(a, kLargeNarrow);
    auto rounds = [&](const Groups& g) { return (float)(((unsigned)g.total * a.ntiles + gridDim.x - 1) / gridDim.x); };
    if (rounds(narrow) * (kLargeNarrow * 1.03f * a.k + 256 * 400) < rounds(groups) * (256.f * a.k + 256 * 400)) {
      large_products<T, kLargeNarrow, MODE>(a, narrow, even, odd);
      return;
    }
  }
  large_products<T, 256, MODE>(a, groups, even, odd);
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
  Groups groups(a, 1);     // tiles of one row: the row's group is that of the tile `row`
  int group = a.groups;
  if (row >= groups.first_row && row < groups.last_end) group = groups.of_tile(a, 1, (unsigned)(row - groups.first_row), 1).group;
  const int n = (int)(id % chunks) * 64 + lane;
  if (group == a.groups || n >= a.n) return;   // (rows of no group: written by the tiles' kernel)
  float s = sum_along(a.partial + row * a.n + n, a.splits, a.rows * a.n);
  if (a.bias) s += (float)((const T*)a.bias)[(int64_t)group * a.n + n];
  ((T*)a.out)[row * a.n + n] = (T)s;
}

// weight product: the pieces' sums of each group.  64 elements a block; its waves add a share of the pieces each, in order, and their sums are
// added in order.  Sixteen waves where a group has many pieces, whose sums a wave reads one after the other (133578 rows, 64 x 64 in 4 groups of
// about a hundred: the whole product 26.4 us, 28.2 with four waves); four where few pieces leave the others nothing.
template <typename T, int WAVES>
__global__ void __launch_bounds__(WAVES * 64) grouped_weight_sum_kernel(GroupArgs a) {
  __shared__ float part[WAVES][64];
  const int group = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // pieces in front of the group, and its own
  unsigned before = 0, mine = 0;
  Groups groups(a, a.per_split);
  int high = groups.first_row;
  for (int g0 = 0; g0 <= group; g0 += 64) {
    if (a.groups > 64) groups.load(a, a.per_split, g0, high);
    const int l = min(group - g0, 63);
    mine = (unsigned)__builtin_amdgcn_readlane(groups.tiles, l);
    before += (unsigned)__builtin_amdgcn_readlane(groups.upto, l) - (group - g0 < 64 ? mine : 0u);
    high = __builtin_amdgcn_readlane(groups.end, 63);
  }
  if (mine == 1) return;   // (written by the tiles' kernel; a group without rows is cleared here)
  const int64_t weights = (int64_t)a.m * a.n, size = weights + (a.dbias ? a.m : 0);
  const unsigned per = (mine + WAVES - 1) / WAVES, q0 = min(wave * per, mine), q1 = min(q0 + per, mine);
  for (int64_t e0 = (int64_t)blockIdx.x * 64; e0 < size; e0 += (int64_t)gridDim.x * 64) {
    const int64_t e = e0 + lane, i = e - weights;
    if (e < weights) part[wave][lane] = sum_along(a.partial + (int64_t)(before + q0) * weights + e, q1 - q0, weights);
    else if (e < size) part[wave][lane] = sum_along(a.partial_bias + (int64_t)(before + q0) * a.m + i, q1 - q0, a.m);
    __syncthreads();
    if (wave == 0 && e < size) {
      float s = part[0][lane];
#pragma unroll
      for (int q = 1; q < WAVES; ++q) s += part[q][lane];
      if (e < weights) ((T*)a.out)[group * weights + e] = (T)s;
      else ((T*)a.dbias)[group * (int64_t)a.m + i] = (T)s;
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ launch rules
struct GroupPlan { int bm, bn, splits, per_split; bool two_kinds; double us; int64_t partial_floats, mtiles_most; };

// Row products.  The tile and the number of pieces that the summed axis is cut into are those of the least expected time, in us:
//
//   5 + what the steps take + (4 + the pieces' sums, written and read at 2.6 TB/s, where there is more than one piece)
//
// The blocks of the kernel for every case share compute units, so the steps take the time of all of them at the rate of a full device (`full`, of
// a compute unit) or that of one block alone (`alone`), whichever is more; the two-kind kernel has one block a compute unit and takes its tiles in
// whole rounds.  Tiles of a group of r rows: r / bm and half a one for the last, as the sizes are not known here.  The figures were measured
// over 23 to 26 shapes with every tile and 1 to 48 pieces: what the rule picks takes 3 per cent longer on average than the best of them (times for
// bf16, 64 x 128 tile: 8 groups of 2048 rows in all, 1024 x 1024, 17 us whole, 29 in two pieces, 24 by 16-row tiles; 200 rows in 4 groups 9 us by
// 16-row tiles, 11 by 64; fp32, 480 rows in 3 groups, 27648 summed: two kinds, 24 pieces, 61 us, whole 933, by 64-row tiles 65).
// 128 x 128 tiles of 16-bit operands were at most 6 per cent faster than the best of the others.
static GroupPlan plan_rows(int64_t rows, int64_t groups, int64_t n, int64_t k, int dtype) {
  struct Kind { int dtype_bits, bm, bn; bool two_kinds; double alone, full; };
  static const Kind kinds[] = {{16, 16, 128, false, 0.36, 0.28}, {16, 64, 128, false, 0.48, 0.42},
                               {32, 16, 128, false, 0.63, 0.57}, {32, 64, 128, false, 0.88, 1.0}, {32, 128, 128, true, 1.25, 1.25}, {32, 192, 128, true, 1.65, 1.65}};
  const int bits = dtype == VC_F32 ? 32 : 16;
  const int64_t bk = dtype == VC_F32 ? 32 : 64, steps = cdiv(k, bk), filled = groups < rows ? groups : rows;
  GroupPlan best{};
  for (const Kind& kind : kinds) {
    if (kind.dtype_bits != bits || (kind.two_kinds && n <= 64)) continue;
    const int bn = kind.bm == 64 && n <= 64 ? 64 : kind.bn;
    const double cut = (double)rows / kind.bm + 0.5 * filled, tiles = (cut > filled ? cut : filled) * cdiv(n, bn);
    for (int64_t want = 1; want <= 64; want = want & (want - 1) ? want / 3 * 4 : want == 1 ? 2 : want / 2 * 3) {   // 1, 2, 3, 4, 6, 8, 12, ...
      const int64_t per = cdiv(steps, want), splits = cdiv(steps, per);
      if (want > 1 && per * bk < 256) break;
      double us;
      if (kind.two_kinds) us = (double)(int64_t)((tiles * splits + 255) / 256) * per * kind.full;
      else us = tiles * splits * per / 256 * kind.full;
      if (us < per * kind.alone) us = per * kind.alone;
      us += 5 + (splits > 1 ? 4 + 8e-6 / 2.6 * splits * rows * n : 0);
      if (best.bm == 0 || us < best.us) best = {kind.bm, bn, (int)splits, (int)(per * bk), kind.two_kinds, us, splits > 1 ? splits * rows * n : 0, 0};
    }
  }
  return best;
}

// Weight product.  The rows are split into pieces where the groups' outputs have fewer than 128 tiles in all, or up to three groups, of which one
// may hold nearly all rows, fewer than 512 each; a piece is long enough that the sums written for it (and read once more) stay small beside the
// rows that it reads.  (bf16, groups of which the largest has four times the rows of the smallest: 65536 rows of 512 and 512 channels in 32 groups,
// 512 tiles, 178 us in pieces and 75 whole; 16384 rows in 8 groups, 128 tiles, 66 and 51; 8192 rows of 1024 and 1024 in 2 groups, 128 tiles, 75
// and 92.  128 x 128 tiles from 65 channels a side on, 64 x 64 below.)  From four groups on a group that holds nearly all rows has its own tiles' blocks
// only: bf16, 32768 rows of 512 and 512 channels in 8 groups, 61 us with equal groups, 437 with all rows in one; 32749 of 1024 and 4096 in 16, 276 and 854.
static GroupPlan plan_weight(int64_t rows, int64_t groups, int64_t m, int64_t n, int dtype) {
  GroupPlan p;
  p.two_kinds = dtype == VC_F32 && m > 64 && n > 64;
  p.bm = m > 64 && n > 64 ? 128 : 64;
  p.bn = p.bm;
  const int64_t tiles = cdiv(m, p.bm) * cdiv(n, p.bn);
  int64_t piece = cdiv(rows, cdiv(512, tiles));
  const int64_t least = 4 * m * n / (m + n) > 256 ? 4 * m * n / (m + n) : 256;
  if (piece < least) piece = least;
  piece = cdiv(piece, 64) * 64;
  p.splits = tiles < 512 && (groups < 4 || tiles * groups < 128) && groups * piece <= rows ? 2 : 1;
  p.per_split = (int)piece;
  p.mtiles_most = p.splits > 1 ? rows / piece + groups : groups;   // pieces
  p.partial_floats = p.splits > 1 ? p.mtiles_most * (m * n + m) : 0;
  return p;
}

// Large tiles need every piece of both operands to be aligned, sizes of 192 either way (of a tile's 256), and 32-bit offsets in a tile.
static constexpr unsigned kLargeBlocks = 256;   // one a compute unit, each taking tiles until there are none
static bool large_tiles(int dtype, int64_t m, int64_t n, int64_t longest, std::initializer_list<uintptr_t> aligned) {
  if (longest >= (1 << 22) || dtype == VC_F32 || m < 192 || n < 192) return false;
  for (uintptr_t v : aligned)
    if (v & 15) return false;
  return true;
}
// Their expected time as above, a step of all compute units taking 1.3 us, the way in and out of a round 4 (bf16, 8192 rows in 8 groups, 1024 x 1024:
// 26 us, by 64 x 128 tiles 34; 4096 rows 24 and 22; 2560 rows in 16 groups, 1024 x 4096: 33 and 45).
static double large_us(int64_t rows, int64_t groups, int64_t n, int64_t k) {
  const double filled = (double)(groups < rows ? groups : rows), cut = rows / 256.0 + 0.5 * filled, tiles = (cut > filled ? cut : filled) * cdiv(n, 256);
  return 5 + (tiles > 256 ? tiles / 256 : 1) * (cdiv(k, 64) * 1.3 + 4);
}

static bool small_operands(int64_t n, int64_t k, int64_t longest) { return n < 8 || k < 8 || longest >= (1 << 22) - 1 || n >= (1 << 22) - 1; }

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
  const uintptr_t size = 2;
  const bool large = large_us(a.rows, a.groups, a.n, a.k) < p.us &&
                     large_tiles(dtype, a.rows, a.n, a.lda > a.n ? a.lda : a.n,
                                 {(uintptr_t)a.a, (uintptr_t)a.b, (uintptr_t)a.out, (uintptr_t)a.bias, a.lda * size, a.k * size, a.n * size});
  a.splits = large ? 1 : p.splits;
  a.per_split = large ? a.k : p.per_split;
  const bool small = small_operands(a.n, a.k, a.lda);
  const int bm = large ? kLargeNarrow : small ? 64 : p.bm, bn = large ? 256 : small ? 64 : p.bn;
  a.ntiles = (int)cdiv(a.n, bn);
  const int64_t total = (a.rows / bm + a.groups + 2) * a.ntiles * a.splits;
  VC_REQUIRE(total < (1LL << 24) - 8, "%s: %lld tiles", who, (long long)total);   // (2^32 threads)
  const unsigned blocks = large || (p.two_kinds && !small) ? kLargeBlocks : (unsigned)cdiv(total, 8) * 8;
#define VC_GO(T, ...)                                                                                                             \
  if (mode == kForward) hipLaunchKernelGGL((grouped_kernel<T, __VA_ARGS__, kForward>), dim3(blocks), dim3(256), 0, st, a);        \
  else hipLaunchKernelGGL((grouped_kernel<T, __VA_ARGS__, kBackInput>), dim3(blocks), dim3(256), 0, st, a);                       \
  if (p.splits > 1) hipLaunchKernelGGL(grouped_row_sum_kernel<T>, dim3((unsigned)cdiv(a.rows * cdiv(a.n, 64), 4)), dim3(256), 0, st, a)
#define VC_TILES(T)                                       \
  if (small) { VC_GO(T, 64, 64, 2, 1, true); }                          \
  else if (p.bm == 64 && p.bn == 64) { VC_GO(T, 64, 64, 2, 3, false); }    \
  else if (p.bm == 64) { VC_GO(T, 64, 128, 2, 2, false); }                 \
  else { VC_GO(T, 16, 128, 1, 3, false); }
#define VC_LARGE(T)                                                                                                               \
  if (mode == kForward) hipLaunchKernelGGL((grouped_large_kernel<T, kForward>), dim3(blocks), dim3(512), 0, st, a);              \
  else hipLaunchKernelGGL((grouped_large_kernel<T, kBackInput>), dim3(blocks), dim3(512), 0, st, a)
#define VC_PIECES(BM)                                                                                                                \
  if (mode == kForward) hipLaunchKernelGGL((grouped_f32_kernel<BM, 128, kForward>), dim3(blocks), dim3(512), 0, st, a);           \
  else hipLaunchKernelGGL((grouped_f32_kernel<BM, 128, kBackInput>), dim3(blocks), dim3(512), 0, st, a);                          \
  if (p.splits > 1) hipLaunchKernelGGL(grouped_row_sum_kernel<float>, dim3((unsigned)cdiv(a.rows * cdiv(a.n, 64), 4)), dim3(256), 0, st, a)
  if (large && dtype == VC_F16) { VC_LARGE(_Float16); }
  else if (large) { VC_LARGE(__bf16); }
  else if (!small && p.two_kinds && p.bm == 192) { VC_PIECES(192); }
  else if (!small && p.two_kinds) { VC_PIECES(128); }
  else if (dtype == VC_F32) { VC_TILES(float) } else if (dtype == VC_F16) { VC_TILES(_Float16) } else { VC_TILES(__bf16) }
#undef VC_PIECES
#undef VC_LARGE
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
  a.a = x; a.lda = rows == 1 ? in : x_stride; a.b = weight; a.bias = bias; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = y;
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
  a.a = dy; a.lda = rows == 1 ? out : dy_stride; a.b = weight; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = dx;
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
  if (rows <= 1) { x_stride = in; dy_stride = out; }     // (a single row's stride may be anything; it decides on tiles and offsets all the same)
  const GroupPlan p = plan_weight(rows, groups, out, in, dtype);
  const size_t need = (size_t)p.partial_floats * sizeof(float);
  VC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %zu bytes, need %zu", who, workspace_bytes, need);
  GroupArgs a{};
  a.a = dy; a.lda = dy_stride; a.b = x; a.ldb = x_stride; a.offsets = offsets; a.off64 = offset_bits == 64; a.out = dweight; a.dbias = dbias;
  a.rows = rows; a.groups = (int)groups; a.m = (int)out; a.n = (int)in;
  a.splits = p.splits; a.per_split = p.per_split;
  const uintptr_t size = 2;
  // (from 160 tiles on: of 2048 columns, 1024 and 4 groups of 512 rows 128 tiles took 23 us, 128 x 128 ones 20, and 256 of 4096 columns 25 and 34)
  const bool large = p.splits == 1 && groups * cdiv(out, 256) * cdiv(in, 256) >= 160 &&
                     large_tiles(dtype, out, in, x_stride > dy_stride ? x_stride : dy_stride,
                                 {(uintptr_t)x, (uintptr_t)dy, (uintptr_t)dweight, x_stride * size, dy_stride * size, in * size, out * size});
  const bool small = small_operands(out, in, x_stride > dy_stride ? x_stride : dy_stride);
  a.mtiles = (int)cdiv(out, large ? 256 : small ? 64 : p.bm); a.ntiles = (int)cdiv(in, large ? 256 : small ? 64 : p.bn);
  a.partial = (float*)workspace;
  a.partial_bias = a.partial + p.mtiles_most * out * in;
  const int64_t tiles = (int64_t)a.mtiles * a.ntiles;
  // without splits every XCD takes an eighth of each group's tiles
  const int64_t total = p.splits == 1 && tiles >= 8 ? cdiv(tiles, 8) * 8 * groups : p.mtiles_most * tiles;
  VC_REQUIRE(total < (1LL << 24) - 8, "%s: %lld tiles", who, (long long)total);   // (2^32 threads)
  const unsigned blocks = large || (p.two_kinds && !small) ? kLargeBlocks : (unsigned)cdiv(total, 8) * 8;
  hipStream_t st = (hipStream_t)stream;
  const int64_t sum_blocks = cdiv(out * in + out, 64);
#define VC_GO(T)                                                                                                                              \
  if (small) hipLaunchKernelGGL((grouped_kernel<T, 64, 64, 2, 1, true, kBackWeight>), dim3(blocks), dim3(256), 0, st, a);                     \
  else if (p.two_kinds) hipLaunchKernelGGL((grouped_f32_kernel<128, 128, kBackWeight>), dim3(blocks), dim3(512), 0, st, a);                        \
  else if (p.bm == 128) { if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((grouped_kernel<T, 128, 128, 2, 2, false, kBackWeight>), dim3(blocks), dim3(256), 0, st, a); } \
  else hipLaunchKernelGGL((grouped_kernel<T, 64, 64, 2, 3, false, kBackWeight>), dim3(blocks), dim3(256), 0, st, a);                                      \
  if (p.splits > 1 && p.mtiles_most > 16 * groups)                                                                                            \
    hipLaunchKernelGGL((grouped_weight_sum_kernel<T, 16>), dim3((unsigned)(sum_blocks < 16384 ? sum_blocks : 16384), (unsigned)groups), dim3(1024), 0, st, a);   \
  else if (p.splits > 1)                                                                                                                      \
    hipLaunchKernelGGL((grouped_weight_sum_kernel<T, 4>), dim3((unsigned)(sum_blocks < 16384 ? sum_blocks : 16384), (unsigned)groups), dim3(256), 0, st, a)
  if (large && dtype == VC_F16) hipLaunchKernelGGL((grouped_large_kernel<_Float16, kBackWeight>), dim3(blocks), dim3(512), 0, st, a);
  else if (large) hipLaunchKernelGGL((grouped_large_kernel<__bf16, kBackWeight>), dim3(blocks), dim3(512), 0, st, a);
  else if (dtype == VC_F32) { VC_GO(float); } else if (dtype == VC_F16) { VC_GO(_Float16); } else { VC_GO(__bf16); }
#undef VC_GO
  VC_CHECK_LAUNCH(who);
  return VC_OK;
}

}  // extern "C"
