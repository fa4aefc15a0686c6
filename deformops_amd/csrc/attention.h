// Cross attention (softmax(scale q k^T + mask) v) for gfx950, forward and backward, behind
// deformops_cross_attention_* of include/deformops_amd.h.
//
// Mathematics. With x_ij the scaled and masked score of row i and key j, m_i = max_j x_ij:
//   p_ij = exp(x_ij - m_i) / l_i,   l_i = sum_j exp(x_ij - m_i),   o_i = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,   ds_ij = p_ij (do_i . v_j - delta_i),   delta_i = do_i . o_i
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i
// The forward passes over the keys once with a running maximum and sum, and keeps (m, log2 l)
// of each row, from which the backward forms p again. A row that no key is left for has o = 0
// and no gradient: its m is kept as +inf, which makes every p of it 0.
//
// Rows. The heads that share a key head are one list of rows: row r of (image, key head) is
// query r / G of head r % G in the group, G = heads / key heads. So the states are read once
// for the whole group, a group's gradients of k and v are summed in one place, and a single
// token's G heads fill one tile.
//
// Products. All run on v_mfma_f32_32x32x16_{bf16,f16} (float as three bf16 parts), whose result
// has column = lane % 32 and rows 8 (r / 4) + 4 (lane / 32) + r % 4 in its 16 registers. The
// scores are formed so that the axis of the next product's contraction lies in the registers:
// keys x rows for o and dq, rows x keys for dv and dk. A product contracts over its axis in
// any order as long as both operands agree, so the registers are the next product's operand
// as they are, and the other operand is read from LDS in the registers' order
// (ds_read_b64_tr_b16 turns a row-major 16-bit tile on the way). Scores never touch LDS, and a
// softmax statistic of the keys x rows form is one value per lane.
//
// Measured (this card: a large copy 4.9 TB/s, large bf16 and f16 products 1,147 and 1,112
// TFLOP/s), rates by the operations that a kernel does:
//   forward, 2 x 16,384 rows of 16,384 states, 8 heads of 128, bf16: 2.17 ms, 1,010 TFLOP/s.
//     Bound by the matrix cores and, where heads are narrower, by the exponentials beside them:
//     2 x 16,384 rows of 4,096 states, 8 heads of 64, f16: 333 us, 825 TFLOP/s.
//   grad_q and grad_states of that call: 471 us, 875 TFLOP/s, and 690 us, 797 TFLOP/s.
//   forward, 8 images' single tokens over 21,504 states each at most, 16 heads of 64 on 4, bf16:
//     23 us, 4.8 TB/s, bound by the states' bytes; the join of the pieces 5 us more.
//   forward, and all gradients in one pass (FUSED), 2 x 21,504 rows of 77 states, 8 heads of 64, bf16:
//     32 us, 2.7 TB/s, and 59 us, 3.0 TB/s, bound by the time a tile takes from its loads to its
//     stores.
//   4 x 100 rows of 16,384 states, 8 heads of 32, bf16, bool mask: forward 26 us, grad_q 33 us,
//     2.5 and 2.0 TB/s, grad_states 49 us, 2.7 TB/s: the prologue and epilogue of short walks.

#ifndef DEFORMOPS_AMD_ATTENTION_H_
#define DEFORMOPS_AMD_ATTENTION_H_

#include <algorithm>
#include <math.h>
#include <type_traits>

#include "operators.h"

namespace attention {

using namespace operators;

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -INFINITY;

template <int V> using Const = std::integral_constant<int, V>;

enum MaskKind { kNoMask = 0, kBoolMask = 1, kFloatMask = 2 };

// Rows of channels in memory: element strides of the image, the row and the head. Every row the
// kernels read is aligned to 16 bytes and holds Dp channels (zeros past D); a call whose tensors
// are not like that is packed first.
struct Rows {
  const void* at;
  int64_t batch, row, head;
};

struct Args {
  Rows q, k, v;
  // A bool mask as words of 32 keys each (bit k % 32 of word k / 32, zeros past S; mask_bits_kernel),
  // a float mask as it is, its keys side by side. Strides of the image, the head and the row, 0
  // where it is one for all.
  const void* mask;
  int64_t mask_batch, mask_head, mask_row;
  int mask_row_keys;  // keys of a float mask's row in memory (at least 4)
  int mask_type;      // element type of a float mask
  bool mask_of_keys;  // a bool mask that is one for all rows and heads: it removes states
  const void* lengths;
  bool lengths_i64;
  void* out;
  float2* stats;  // [B][H][Q]: (m, log2 l) of each row, m = +inf for a row without keys
  int B, Q, S, K, G, D;
  int Dp;      // D, rounded up to 16 bytes
  uint32_t R;  // rows of one (image, key head): Q * G
  float scale;
  bool out_vector;  // results may be written four channels at a time
  // The key axis is worked on in `slots` pieces, which belong to images: `splits` of each, or,
  // `balanced`, as many of each as its states need.
  int slots, splits;
  bool balanced;
  float* part;         // [slots][K][R][D] unnormalized sums of each piece
  float2* part_stats;  // [slots][K][R]
  // Backward.
  Rows o, go;
  const float2* row_stats;
  float* delta;  // [B][H][Q]
  void *grad_q, *grad_k, *grad_v;
  int row_splits, near;
  float* part_k;  // [row_splits][B][S][K][D]
  float* part_v;
};

// ---------------------------------------------------------------------------
// Matrix products of one wave.

// Precision of a 16-bit operand made from fp32 scores: p and ds are rounded to the operands'
// type (by half a step: bf16 2^-8, f16 2^-11 relative). f16 has 5 exponent bits: the backward
// scales p by 2^14, so that weights down to 2^-28 stay normal, and ds by a running power of
// two for each lane (Scaled below). The forward's weights exp2(x - m) are scaled by 2^9.
template <typename T> constexpr float kWeightBits = std::is_same_v<T, f16_t> ? 14.0f : 0.0f;
template <typename T> constexpr float kForwardBits = std::is_same_v<T, f16_t> ? 9.0f : 0.0f;

// The forward's running maximum stays where it is until a score passes it by this many powers
// of two: with random scores every tile has a row whose maximum moves by a little, and each
// move costs a multiplication of all sums. Weights then reach 2^8 (f16: 2^5 2^9 = 2^14, in its
// range), in a sum and a product that are as exact for them.
template <typename T> constexpr float kSlack = std::is_same_v<T, f16_t> ? 5.0f : 8.0f;

template <typename T> struct Mma;

template <typename T> struct Mma16 {
  using Vec = std::conditional_t<std::is_same_v<T, bf16_t>, bf16x8, f16x8>;
  static constexpr int kPlanes = 1;
  struct Piece { u32x4 plane[1]; };          // 8 channels of a row
  struct Weights { Vec part[2][1]; };        // 32 contracted positions

  static __device__ f32x16 mma(Vec a, Vec b, f32x16 c) {
    if constexpr (std::is_same_v<T, bf16_t>)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ f32x16 product(const Vec (&a)[1], const Vec (&b)[1], f32x16 c) { return mma(a[0], b[0], c); }
  static __device__ Weights weights(const float (&w)[16]) {
    Weights out;
#pragma unroll
    for (int i = 0; i < 16; ++i) out.part[i / 8][0][i % 8] = static_cast<T>(w[i]);
    return out;
  }
  // 8 channels, 16 bytes, as an operand.
  static __device__ Piece piece(const u32x4 (&memory)[1]) { return Piece{{memory[0]}}; }
};
template <> struct Mma<bf16_t> : Mma16<bf16_t> {};
template <> struct Mma<f16_t> : Mma16<f16_t> {};

// float on the bf16 matrix cores: x = x0 + x1 + x2 exactly, each part the rest rounded to bf16
// (8 bits; the parts of a number below 2^-110 lose their last bits to bf16's range), and a product
// is the sum of the six largest of the nine: what is left out, a1 b2 + a2 b1 + a2 b2, is at most
// 2^-23 of it, float's own rounding. Six products of 32 cycles for 16 contracted channels, where
// v_mfma_f32_32x32x2_f32 takes eight of 64 cycles (4 x 1,501 rows of 2,333 states, 8 heads of
// 64, forward and backward: 1.40 ms with it, 0.90 with these). An infinite operand gives NaN.
template <> struct Mma<float> {
  using Vec = bf16x8;
  static constexpr int kPlanes = 3;
  struct Piece { u32x4 plane[3]; };
  struct Weights { Vec part[2][3]; };

  static __device__ void split(float x, bf16_t (&out)[3]) {
    out[0] = static_cast<bf16_t>(x);
    const float rest = x - static_cast<float>(out[0]);
    out[1] = static_cast<bf16_t>(rest);
    out[2] = static_cast<bf16_t>(rest - static_cast<float>(out[1]));
  }
  // The parts of x (the words' lower halves) and y: one conversion for both.
  static __device__ void split(float x, float y, uint32_t (&out)[3]) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      out[p] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
      x -= __uint_as_float(out[p] << 16);
      y -= __uint_as_float(out[p] & 0xffff0000u);
    }
  }
  static __device__ f32x16 product(const Vec (&a)[3], const Vec (&b)[3], f32x16 c) {
    c = Mma<bf16_t>::mma(a[2], b[0], c);  // the smallest first
    c = Mma<bf16_t>::mma(a[0], b[2], c);
    c = Mma<bf16_t>::mma(a[1], b[1], c);
    c = Mma<bf16_t>::mma(a[1], b[0], c);
    c = Mma<bf16_t>::mma(a[0], b[1], c);
    return Mma<bf16_t>::mma(a[0], b[0], c);
  }
  static __device__ Weights weights(const float (&w)[16]) {
    u32x4 words[2][3];
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      uint32_t parts[3];
      split(w[i], w[i + 1], parts);
#pragma unroll
      for (int p = 0; p < 3; ++p) words[i / 8][p][i % 8 / 2] = parts[p];
    }
    Weights out;
#pragma unroll
    for (int p = 0; p < 6; ++p) out.part[p / 3][p % 3] = __builtin_bit_cast(Vec, words[p / 3][p % 3]);
    return out;
  }
  static __device__ Piece piece(const u32x4 (&memory)[2]) {
    Piece out;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const f32x4 four = __builtin_bit_cast(f32x4, memory[i / 4]);
      uint32_t parts[3];
      split(four[i % 4], four[i % 4 + 1], parts);
#pragma unroll
      for (int p = 0; p < 3; ++p) out.plane[p][i / 2] = parts[p];
    }
    return out;
  }
};

// c += the rows' products over one piece of each: 16 contracted channels, 8 in each half of the
// wave.
template <typename T>
__device__ inline f32x16 multiply(const typename Mma<T>::Piece& a, const typename Mma<T>::Piece& b, f32x16 c) {
  typename Mma<T>::Vec x[Mma<T>::kPlanes], y[Mma<T>::kPlanes];
#pragma unroll
  for (int p = 0; p < Mma<T>::kPlanes; ++p) {
    x[p] = __builtin_bit_cast(typename Mma<T>::Vec, a.plane[p]);
    y[p] = __builtin_bit_cast(typename Mma<T>::Vec, b.plane[p]);
  }
  return Mma<T>::product(x, y, c);
}

// A tile of rows in LDS, DP channels each, as 16-bit elements (float: the three planes of a row
// side by side) in 16-byte pieces that change places within their plane by an exclusive or with
// bits of the row's number. LDS serves 64 banks (256 bytes) a cycle: 16 lanes of a row operand's
// read (one piece of 16 rows), or 32 lanes of a turning read (4 neighbouring pieces of 4 rows, 8
// bytes a lane), have to lie in different sixteenths of 256 bytes. Measured on reads of both
// kinds: 540 and 300-320 bytes/ns a CU with these patterns, 300 and 150 with `row & 7`. (A row of
// three planes is 12, 8, 4 or 0 sixteenths past a multiple of 256 bytes for 32, 64, 96 and 128
// channels, as 192, 128, 64 and 256 bytes are, so the patterns serve it too.)
template <typename T, int DP> struct Tile {
  static constexpr int kPlanes = Mma<T>::kPlanes;
  static constexpr int kPieces = DP / 8;  // of a plane
  static constexpr int kRowBytes = kPlanes * DP * 2;

  static __device__ int offset(int row, int piece, int plane = 0) {
    int turn;
    if constexpr (kPieces == 16)
      turn = ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (kPieces == 8)
      turn = ((row & 2) << 1) | ((row >> 2) & 3);
    else  // 4 or 12: rows r .. r + 3 differ in their sixteenths already
      turn = (row >> 2) & 3;
    return row * kRowBytes + plane * (DP * 2) + ((piece ^ turn) << 4);
  }
};

// The turning read of a tile: 8 contracted rows from `row0` and `row1` (4 each) of 32 channels.
template <typename T, int DP>
__device__ inline void turned(const char* tile, int row0, int row1, int block, typename Mma<T>::Vec (&out)[Mma<T>::kPlanes]) {
  const int lane = threadIdx.x % kWave;
  // Lane c of a 16-lane group gets channel c of the four rows that the group reads.
  const int channel = 32 * block + 16 * ((lane / 16) & 1) + 4 * (lane % 4), within = (lane % 16) / 4;
#pragma unroll
  for (int p = 0; p < Mma<T>::kPlanes; ++p) {
    i16x4 part[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
          tile + Tile<T, DP>::offset((u ? row1 : row0) + within, channel / 8, p) + (channel % 8) * 2));
    out[p] = __builtin_bit_cast(typename Mma<T>::Vec, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// acc (channels x lanes) += tile^T (32 channels from 32 * block, the 32 tile rows from `row`)
// x w: the sum over tile rows of w[row][lane] * tile[row][channel].
template <typename T, int DP>
__device__ inline f32x16 accumulate(const char* tile, int row, int block, const typename Mma<T>::Weights& w,
                                    f32x16 acc) {
  const int half = int(threadIdx.x % kWave) / 32;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    typename Mma<T>::Vec a[Mma<T>::kPlanes];
    const int r = row + 16 * t + 4 * half;
    turned<T, DP>(tile, r, r + 8, block, a);
    acc = Mma<T>::product(a, w.part[t], acc);
  }
  return acc;
}

// The product's row operand: piece 2 * step + half of tile row `row + lane % 32`.
template <typename T, int DP> __device__ inline typename Mma<T>::Piece row_piece(const char* tile, int row, int step) {
  const int lane = threadIdx.x % kWave;
  typename Mma<T>::Piece out;
#pragma unroll
  for (int p = 0; p < Mma<T>::kPlanes; ++p)
    out.plane[p] = *reinterpret_cast<const u32x4*>(tile + Tile<T, DP>::offset(row + lane % 32, 2 * step + lane / 32, p));
  return out;
}

// 16 bytes of a row in memory, from channel c; zero past Dp.
template <typename T> __device__ inline u32x4 load_piece(const T* row, int c, int Dp) {
  u32x4 out = {0, 0, 0, 0};
  if (c < Dp) out = *reinterpret_cast<const u32x4*>(row + c);
  return out;
}

// The largest of a lane's value and its partner's, 32 lanes on.
__device__ inline float half_max(float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ inline float half_sum(float v) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// The keys' (or rows') number in a 32 x 32 result's register r.
__device__ inline int result_row(int r) { return 8 * (r / 4) + 4 * ((threadIdx.x % kWave) / 32) + r % 4; }

// f16 only: ds as operands of the matrix cores, scaled by a power of two for each lane. ds
// spans what p and the incoming gradient span together (p alone reaches 1e-6 at 2^20 keys),
// more than f16's 2^-24 .. 2^16 in ordinary training. A lane's ds all go into sums that the
// lane's column holds, so each lane keeps an exponent of its own, taken from the first values
// (to 2^11 .. 2^12) and lowered, with the sums so far, when a later value would pass 2^15.
template <typename T> struct Scaled {
  static constexpr float power = 1.0f;
  template <int N> __device__ void fit(float (&)[16], f32x16 (&)[N]) {}
  __device__ float undo() const { return 1.0f; }
};
template <> struct Scaled<f16_t> {
  int e = 0;
  bool set = false;
  float power = 1.0f;  // 2^e, which the caller has put into ds
  template <int N> __device__ __forceinline__ void fit(float (&ds)[16], f32x16 (&acc)[N]) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(ds[i]));
    top = half_max(top);
    const int bits = __builtin_amdgcn_frexp_expf(top);  // top = f 2^bits, f in [0.5, 1); 0 for 0, inf and NaN
    const bool change = top > 0.0f && (bits > 15 || !set);
    if (__any(change)) {
      const int by = change ? min(12 - bits, 120 - e) : 0;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] = ldexpf(acc[n][i], by);
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] = ldexpf(ds[i], by);
      e += by;
      power = ldexpf(1.0f, e);
      set |= change;
    }
  }
  __device__ float undo() const { return ldexpf(1.0f, -e); }
};

// ---------------------------------------------------------------------------
// Masks and lengths.

__device__ inline int states_of(const Args& a, int b) {
  if (!a.lengths) return a.S;
  const int64_t n = a.lengths_i64 ? static_cast<const int64_t*>(a.lengths)[b]
                                  : int64_t(static_cast<const int32_t*>(a.lengths)[b]);
  return int(n < 0 ? 0 : n > a.S ? a.S : n);
}

// 16 elements of a float mask, element i at at(i). The type is asked once, so that all loads are
// under way before the first is waited for: 393 us against 486 with a type, and a wait, for each
// element (4 x 1,501 rows of 2,333 states, 8 heads of 64, bf16, forward and backward).
template <typename At> __device__ __forceinline__ void mask_elements(const Args& a, At at, float (&out)[16]) {
  if (a.mask_type == MSDA_F32) {
#pragma unroll
    for (int i = 0; i < 16; ++i) out[i] = static_cast<const float*>(a.mask)[at(i)];
    return;
  }
  uint16_t half[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) half[i] = static_cast<const uint16_t*>(a.mask)[at(i)];
  const bool brain = a.mask_type == MSDA_BF16;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    out[i] = brain ? __uint_as_float(uint32_t(half[i]) << 16) : widen(__builtin_bit_cast(f16_t, half[i]));
}
// One key's bit of a mask of states.
__device__ inline bool state_bit(const Args& a, int b, int key) {
  return (static_cast<const uint32_t*>(a.mask)[b * a.mask_batch + key / 32] >> (key % 32)) & 1;
}

// Mask rows may begin at any byte: global loads take any alignment.
template <typename V> __device__ inline V load_anywhere(const void* p) {
  struct __attribute__((packed)) Any { V v; };
  return static_cast<const Any*>(p)->v;
}

// The bits of the 16 result rows in a lane's word of 32 keys: result row r in bit
// 8 (r / 4) + r % 4.
__device__ inline uint32_t result_bits(uint32_t word) { return word >> (4 * (int(threadIdx.x % kWave) / 32)); }

// v where bit `bit` of `bits` is set, else `other`.
__device__ inline float where_bit(uint32_t bits, int bit, float v, float other) {
  const uint32_t all = uint32_t(__builtin_amdgcn_sbfe(int32_t(bits), uint32_t(bit), 1));
  return __uint_as_float((all & __float_as_uint(v)) | (~all & __float_as_uint(other)));
}

// The additive mask of the 16 result rows; 0 past the row. Four keys a load: where the row ends
// within them, its last four, moved down (2 x 21,404 rows of 77 states, 8 heads of 64, bf16: 54 us
// against 60 with an element a load there).
__device__ __forceinline__ void float_masks(const Args& a, int64_t at, int key, float (&out)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) out[i] = 0.0f;
  if (key >= a.mask_row_keys) return;
  const int k0 = key + 4 * (int(threadIdx.x % kWave) / 32), end = a.mask_row_keys - 4;
  const bool ends = key + 32 > a.mask_row_keys;
  if (a.mask_type == MSDA_F32) {
    f32x4 four[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int k = k0 + 8 * g;
      four[g] = load_anywhere<f32x4>(static_cast<const float*>(a.mask) + at + (k < end ? k : end));
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (ends) {
        const int by = k0 + 8 * g - end;
        f32x4 x = four[g];
        if (by > 0 && (by & 1)) x = f32x4{x[1], x[2], x[3], 0.0f};
        if (by > 0 && (by & 2)) x = f32x4{x[2], x[3], 0.0f, 0.0f};
        if (by >= 4) x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        four[g] = x;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) out[4 * g + i] = four[g][i];
    }
  } else {
    uint64_t four[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int k = k0 + 8 * g;
      const u32x2 two = load_anywhere<u32x2>(static_cast<const uint16_t*>(a.mask) + at + (k < end ? k : end));
      four[g] = uint64_t(two[1]) << 32 | two[0];
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (ends) {
        const int by = k0 + 8 * g - end;
        four[g] = by >= 4 ? 0 : by > 0 ? four[g] >> (16 * by) : four[g];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint16_t h = uint16_t(four[g] >> (16 * i));
        out[4 * g + i] = a.mask_type == MSDA_BF16 ? __uint_as_float(uint32_t(h) << 16) : widen(__builtin_bit_cast(f16_t, h));
      }
    }
  }
}

// Rows of a (image, key head): query and head of row r.
struct RowOf {
  int query, head;
};
__device__ inline RowOf row_of(const Args& a, int kv, uint32_t r) {
  const uint32_t q = a.G == 1 ? r : r / uint32_t(a.G);
  return RowOf{int(q), kv * a.G + int(r - q * uint32_t(a.G))};
}

__device__ inline int64_t mask_row_at(const Args& a, int b, RowOf o) {
  return b * a.mask_batch + int64_t(o.head) * a.mask_head + int64_t(o.query) * a.mask_row;
}
template <typename T> __device__ inline const T* row_at(const Rows& rows, int b, RowOf o) {
  return static_cast<const T*>(rows.at) + b * rows.batch + int64_t(o.query) * rows.row + int64_t(o.head) * rows.head;
}
__device__ inline int64_t stat_at(const Args& a, int b, RowOf o) {
  return (int64_t(b) * (a.K * a.G) + o.head) * a.Q + o.query;
}

// ---------------------------------------------------------------------------
// Staging: tile rows from memory to LDS through registers, so that the next tile's loads are
// under way while this one is worked on. Buffer loads answer zero outside their range, which
// is how rows past the last and channels past Dp become zeros.

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr uint32_t kOutside = 0x80000000u;  // past every range, which is at most 2^31 bytes

template <typename T> __device__ inline const T* uniform(const T* p) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v >> 32));
  return reinterpret_cast<const T*>((uint64_t(hi) << 32) | lo);
}

template <typename T, int DP, int ROWS> struct Stage {
  static constexpr int kPieces = DP * int(sizeof(T)) / 16;
  static constexpr int kEach = ROWS * kPieces / kThreads;
  static_assert(ROWS * kPieces % kThreads == 0);
  u32x4 hold[kEach];
  uint32_t from[kEach];
  uint32_t stride;  // bytes

  static __device__ int row(int i) { return (i * kThreads + int(threadIdx.x)) / kPieces; }
  static __device__ int piece(int i) { return (i * kThreads + int(threadIdx.x)) % kPieces; }

  __device__ void plan(int64_t row_stride, int Dp) {
    stride = uint32_t(row_stride) * uint32_t(sizeof(T));
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      from[i] = piece(i) * (16 / int(sizeof(T))) < Dp ? uint32_t(row(i)) * stride + uint32_t(piece(i)) * 16 : kOutside;
  }
  // ROWS rows from `base` (the same for all lanes), of which `left` exist; `kept(row)` whether
  // a row is read.
  template <typename F> __device__ __forceinline__ void load(const T* base, int left, F kept) {
    const uint32_t bytes = __builtin_amdgcn_readfirstlane(uint32_t(left < ROWS ? left : ROWS) * stride);
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(uniform(base)), 0, bytes, 0x00027000);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      hold[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, kept(row(i)) ? from[i] : kOutside, 0, 0);
  }
  __device__ __forceinline__ void store(char* tile) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4*>(tile + Tile<T, DP>::offset(row(i), piece(i))) = hold[i];
      } else {  // half a piece of each plane
        const f32x4 four = __builtin_bit_cast(f32x4, hold[i]);
        uint32_t low[3], high[3];
        Mma<T>::split(four[0], four[1], low);
        Mma<T>::split(four[2], four[3], high);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          *reinterpret_cast<u32x2*>(tile + Tile<T, DP>::offset(row(i), piece(i) / 2, p) + 8 * (piece(i) % 2)) =
              u32x2{low[p], high[p]};
      }
    }
  }
};

struct All {
  __device__ bool operator()(int) const { return true; }
};

// Two waves of a SIMD hide each other's waits where their registers allow it (256 each).
constexpr int forward_waves(int size, int DP, int mask) {
  return size == 4 ? (DP > 64 ? 1 : 2) : DP == 32 ? (mask ? 3 : 4) : DP == 64 ? (mask ? 2 : 3) : DP == 128 && mask ? 1 : 2;
}
constexpr int grad_q_waves(int size, int DP, int mask) {
  return size == 4 ? (DP > 32 ? 1 : 2) : DP == 32 ? 3 : DP <= (mask ? 64 : 96) ? 2 : 1;
}
constexpr int grad_states_waves(int size, int DP, int mask, bool fused) {
  if (fused && (size == 4 || (DP == 64 && mask == kFloatMask))) return 1;
  return size == 4 ? (DP > 32 ? 1 : 2) : DP == 32 ? (fused && mask ? 2 : 3) : DP == 64 ? 2 : 1;
}

// ---------------------------------------------------------------------------
// Forward. A workgroup has 4 waves: WR of them along the rows (32 each), 4 / WR along the keys
// of a tile (KB blocks of 32 each), whose partial sums meet in LDS at the end. Splits of the
// key axis leave unnormalized sums, which combine_kernel joins.

template <typename T, int DP, int WR> struct ForwardShape {
  static constexpr int WK = kWaves / WR;
  static constexpr int KB = WR == kWaves ? 2 : 1;
  static constexpr int kRows = 32 * WR;
  static constexpr int kKeys = 32 * KB * WK;
  static constexpr int kTile = kKeys * Tile<T, DP>::kRowBytes;
  static constexpr int kBuffers = 4 * kTile <= (forward_waves(sizeof(T), DP, kNoMask) > 1 ? 80 : 160) * 1024 ? 2 : 1;
  static constexpr int kJoin = WK > 1 ? WK * 32 * WR * (DP + 2) * 4 : 0;
  static constexpr int kLds = std::max(2 * kBuffers * kTile, kJoin);
};

// Four consecutive channels of a result, rounded to T.
template <typename T> __device__ inline void store_four(T* p, const float (&v)[4], int left, bool vector) {
  if (vector && left >= 4) {
    T parts[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) parts[i] = static_cast<T>(v[i]);
    if constexpr (sizeof(T) == 2) {
      u32x2 w;
      __builtin_memcpy(&w, parts, 8);
      *reinterpret_cast<u32x2*>(p) = w;
    } else {
      u32x4 w;
      __builtin_memcpy(&w, parts, 16);
      *reinterpret_cast<u32x4*>(p) = w;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = static_cast<T>(v[i]);
}

// The running softmax of one row in each lane, over keys x rows results.
template <int NB> struct Softmax {
  float m = kLowest;  // in log2 units without a float mask, natural ones with it
  float l = 0.0f;     // this half's keys only
  f32x16 acc[NB] = {};

  __device__ void rescale(float factor) {
    l *= factor;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][i] *= factor;
  }
};

// The pieces of image `b`, slots first .. first + count - 1, by the whole wave. With lengths that
// differ, equal pieces for every image would leave most of the card to wait for the longest one:
// so every piece gets the same number of tiles (at least 2), and an image as many pieces as its
// states need, none for none. The sum over images of ceil(tiles / quota) is at most
// (sum of tiles) / quota + B, which the quota keeps within the slots.
struct Pieces {
  int first, count;
};
struct Shares {
  int mine, before;  // of the image of this lane's number
  __device__ Shares(const Args& a, int keys) {
    const int lane = threadIdx.x % kWave;
    const int tiles = lane < a.B ? (states_of(a, lane) + keys - 1) / keys : 0;
    int64_t total = tiles;
    for (int by = 32; by; by /= 2) total += __shfl_xor(total, by);
    const int64_t most = a.slots - a.B, quota = max(int64_t(2), (total + most - 1) / most);
    mine = int((tiles + quota - 1) / quota);
    int upto = mine;
    for (int by = 1; by < kWave; by *= 2) {
      const int other = __shfl_up(upto, by);
      if (lane >= by) upto += other;
    }
    before = upto - mine;
  }
};
__device__ inline Pieces pieces_of(const Args& a, int b, int keys) {
  if (!a.balanced) return Pieces{b * a.splits, a.splits};
  const Shares s(a, keys);
  return Pieces{__builtin_amdgcn_readlane(s.before, b), __builtin_amdgcn_readlane(s.mine, b)};
}

// A wave's operand of 32 rows, straight from memory. By way of LDS, where neighbouring lanes would
// read a row's neighbouring pieces, it was no faster for short calls and 3 % slower for long
// ones (2 x 16,384 rows of 4,096 states: 1.37 and 1.39 ms, more registers).
template <typename T, int DP>
__device__ inline void take_rows(const Args& a, const T* row, bool live, typename Mma<T>::Piece (&out)[DP / 16]) {
  constexpr int N = 16 / int(sizeof(T)), kOfPiece = 8 / N;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    u32x4 memory[kOfPiece];
#pragma unroll
    for (int i = 0; i < kOfPiece; ++i) {
      const u32x4 zero = {0, 0, 0, 0};
      memory[i] = live ? load_piece(row, (2 * s + int(threadIdx.x % kWave) / 32) * 8 + i * N, a.Dp) : zero;
    }
    out[s] = Mma<T>::piece(memory);
  }
}

// The sum of the products of two rows' channels, by the two lanes of the row.
template <typename T, int DP> __device__ inline float row_dot(const Args& a, const T* x, const T* y) {
  constexpr int N = 16 / int(sizeof(T));
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < DP; c += 2 * N) {
    const int at = c + N * (int(threadIdx.x % kWave) / 32);
    const u32x4 p = load_piece(x, at, a.Dp), q = load_piece(y, at, a.Dp);
    T u[N], v[N];
    __builtin_memcpy(u, &p, 16);
    __builtin_memcpy(v, &q, 16);
#pragma unroll
    for (int i = 0; i < N; ++i) sum = fmaf(widen(u[i]), widen(v[i]), sum);
  }
  return half_sum(sum);
}

// A wave's channels x rows result, rounded to T, into the row of each lane (`image`: dense rows).
template <typename T, int DP>
__device__ __forceinline__ void write_row(const Args& a, T* image, RowOf o, const f32x16 (&acc)[DP / 32]) {
  T* out = image + (int64_t(o.query) * (a.K * a.G) + o.head) * a.D;
#pragma unroll
  for (int c = 0; c < DP / 32; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * (int(threadIdx.x % kWave) / 32);
      const float v[4] = {acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
      store_four(out + d, v, a.D - d, a.out_vector);
    }
}

// What a workgroup of the walks over the keys works on. Row tiles of one piece of one key head
// come first, then the heads: their rows share cache lines.
template <typename Shape> struct KeyWalk {
  int b, kv, slot, first, last, states;
  uint32_t row_tile;
  bool leads;  // the first piece of its image

  __device__ explicit KeyWalk(const Args& a) {
    const uint32_t row_tiles = (a.R + Shape::kRows - 1) / Shape::kRows;
    uint32_t id = xcd_order(blockIdx.x, gridDim.x);
    row_tile = id % row_tiles;
    id /= row_tiles;
    kv = int(id % uint32_t(a.K));
    slot = int(id / uint32_t(a.K));
    int split = slot % a.splits, count = a.splits;
    b = slot / a.splits;
    if (a.balanced) {
      const Shares s(a, Shape::kKeys);
      const uint64_t here = __ballot(s.before <= slot && slot < s.before + s.mine);
      b = here ? __builtin_ctzll(here) : -1;
      if (b < 0) return;
      split = slot - __builtin_amdgcn_readlane(s.before, b);
      count = __builtin_amdgcn_readlane(s.mine, b);
    }
    leads = split == 0;
    states = __builtin_amdgcn_readfirstlane(states_of(a, b));
    const int tiles = (states + Shape::kKeys - 1) / Shape::kKeys;
    first = count == 1 ? 0 : int(int64_t(tiles) * split / count);  // 64-bit divisions are long
    last = count == 1 ? tiles : int(int64_t(tiles) * (split + 1) / count);
  }
  __device__ int64_t part_row(const Args& a, uint32_t r) const { return (int64_t(slot) * a.K + kv) * a.R + r; }
};

// The tiles of keys and values on their way to LDS, and a bool mask's bytes of the next tile.
template <typename T, int DP, int MASK, typename Shape> struct KeyStage {
  static constexpr int KB = Shape::KB;
  const Args& a;
  const KeyWalk<Shape>& w;
  Stage<T, DP, Shape::kKeys> k, v;
  const T *k_base, *v_base;
  int64_t mask_at = 0;  // this row's first mask element
  int local;            // this wave's first key in a tile
  uint32_t next[KB];    // this row's mask words

  __device__ KeyStage(const Args& args, const KeyWalk<Shape>& walk, int first_key) : a(args), w(walk), local(first_key) {
    k.plan(a.k.row, a.Dp);
    v.plan(a.v.row, a.Dp);
    k_base = static_cast<const T*>(a.k.at) + w.b * a.k.batch + w.kv * a.k.head;
    v_base = static_cast<const T*>(a.v.at) + w.b * a.v.batch + w.kv * a.v.head;
  }
  __device__ __forceinline__ void load(int tile) {
    const int key = tile * Shape::kKeys, left = w.states - key;
    const T *ks = k_base + int64_t(key) * a.k.row, *vs = v_base + int64_t(key) * a.v.row;
    if (MASK == kBoolMask && a.mask_of_keys) {  // removed states are read as zeros
      auto kept = [&](int row) {
        return row < left && state_bit(a, w.b, key + row);
      };
      k.load(ks, left, kept);
      v.load(vs, left, kept);
    } else {
      k.load(ks, left, All());
      v.load(vs, left, All());
    }
    load_words(tile, next);
  }
  __device__ __forceinline__ void load_words(int tile, uint32_t (&words)[KB]) const {
    if constexpr (MASK == kBoolMask) {
#pragma unroll
      for (int n = 0; n < KB; ++n)
        words[n] = static_cast<const uint32_t*>(a.mask)[mask_at + (tile * Shape::kKeys + local) / 32 + n];
    }
  }
};

template <typename T, int DP, int MASK, int WR>
__global__ __launch_bounds__(kThreads, forward_waves(sizeof(T), DP, MASK)) void attention_forward_kernel(const Args a) {
  using Shape = ForwardShape<T, DP, WR>;
  using TileT = Tile<T, DP>;
  constexpr int KB = Shape::KB, NB = DP / 32, kSteps = TileT::kPieces / 2, kKeys = Shape::kKeys;
  __shared__ __attribute__((aligned(16))) char lds[Shape::kLds];

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wr = wave % WR, wk = wave / WR;
  const KeyWalk<Shape> w(a);
  if (w.b < 0) return;  // a slot that no image needs
  const int local = 32 * KB * wk;
  KeyStage<T, DP, MASK, Shape> stage(a, w, local);

  const uint32_t r = w.row_tile * Shape::kRows + 32 * wr + lane % 32;
  const bool live = r < a.R;
  const RowOf mine = row_of(a, w.kv, live ? r : a.R - 1);
  if constexpr (MASK != kNoMask) stage.mask_at = mask_row_at(a, w.b, mine);
  if (w.first < w.last) stage.load(w.first);
  typename Mma<T>::Piece q[kSteps];
  take_rows<T, DP>(a, row_at<T>(a.q, w.b, mine), live, q);
  Softmax<NB> soft;

  const float factor = MASK == kFloatMask ? a.scale : a.scale * kLog2e;
  constexpr float kStay = MASK == kFloatMask ? kSlack<T> / kLog2e : kSlack<T>;

  auto attend = [&](int tile, auto buffer, const uint32_t (&mask)[KB]) __attribute__((always_inline)) {
    const char* k_tile = lds + decltype(buffer)::value * 2 * Shape::kTile;
    const char* v_tile = k_tile + Shape::kTile;
    const int key0 = tile * kKeys + local;  // this wave's keys
    if constexpr (MASK == kBoolMask) {
      uint32_t any = 0;
#pragma unroll
      for (int n = 0; n < KB; ++n) any |= mask[n];
      if (!__any(any != 0 && live)) return;
    }
    float x[KB][16];
#pragma unroll
    for (int n = 0; n < KB; ++n) {
      float add[16];
      if constexpr (MASK == kFloatMask) float_masks(a, stage.mask_at, key0 + 32 * n, add);
      const uint32_t bits = result_bits(mask[n]);
      f32x16 s = {};
#pragma unroll
      for (int t = 0; t < kSteps; ++t) s = multiply<T>(row_piece<T, DP>(k_tile, local + 32 * n, t), q[t], s);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[n][i] = s[i];
        if constexpr (MASK == kBoolMask) x[n][i] = where_bit(bits, 8 * (i / 4) + i % 4, s[i], kLowest);
        if constexpr (MASK == kFloatMask) x[n][i] = add[i] == kLowest ? kLowest : fmaf(s[i], factor, add[i]);
      }
    }
    if (key0 + 32 * KB > w.states) {
#pragma unroll
      for (int n = 0; n < KB; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[n][i] = key0 + 32 * n + result_row(i) < w.states ? x[n][i] : kLowest;
    }
    float top = kLowest;
#pragma unroll
    for (int n = 0; n < KB; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, x[n][i]);
    top = half_max(top);
    if constexpr (MASK != kFloatMask) top *= factor;
    if (__any(top > soft.m + kStay)) {
      const float m = fmaxf(soft.m, top);
      const float by = m == soft.m ? 0.0f : soft.m - m;  // 0 too where both are -inf
      soft.rescale(__builtin_amdgcn_exp2f(MASK == kFloatMask ? by * kLog2e : by));
      soft.m = m;
    }
    const float base = soft.m == kLowest ? 0.0f : soft.m;  // all -inf: every weight is exp2(-inf)
    const float shift = kForwardBits<T> - base;
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < KB; ++n) {
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = MASK == kFloatMask ? fmaf(x[n][i] - base, kLog2e, kForwardBits<T>) : fmaf(x[n][i], factor, shift);
        p[i] = __builtin_amdgcn_exp2f(y);
        sum += p[i];
      }
      const auto weights = Mma<T>::weights(p);
#pragma unroll
      for (int c = 0; c < NB; ++c) soft.acc[c] = accumulate<T, DP>(v_tile, local + 32 * n, c, weights, soft.acc[c]);
    }
    soft.l += sum;
  };

  auto step = [&](int tile, auto buffer) __attribute__((always_inline)) {
    if (Shape::kBuffers == 1 && tile > w.first) __syncthreads();
    stage.k.store(lds + decltype(buffer)::value * 2 * Shape::kTile);
    stage.v.store(lds + decltype(buffer)::value * 2 * Shape::kTile + Shape::kTile);
    uint32_t words[KB];
#pragma unroll
    for (int n = 0; n < KB; ++n) words[n] = MASK == kBoolMask ? stage.next[n] : 0;
    __syncthreads();
    if (tile + 1 < w.last) stage.load(tile + 1);
    attend(tile, buffer, words);
  };
  for (int tile = w.first; tile < w.last; tile += 2) {
    step(tile, Const<0>());
    if (tile + 1 < w.last) step(tile + 1, Const<Shape::kBuffers - 1>());
  }

  // Join the waves that share rows: each leaves its sums in LDS, wave 0 of them adds.
  soft.l = half_sum(soft.l);
  if constexpr (Shape::WK > 1) {
    __syncthreads();
    float* mine_at = reinterpret_cast<float*>(lds) + wave * 32 * (DP + 2);
    if (lane < 32) {
      mine_at[32 * DP + lane] = soft.m;
      mine_at[32 * DP + 32 + lane] = soft.l;
    }
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine_at[(32 * c + result_row(i)) * 32 + lane % 32] = soft.acc[c][i];
    __syncthreads();
    if (wk > 0) return;
    for (int other = 1; other < Shape::WK; ++other) {
      const float* at = reinterpret_cast<const float*>(lds) + (other * WR + wr) * 32 * (DP + 2);
      const float m2 = at[32 * DP + lane % 32], l2 = at[32 * DP + 32 + lane % 32];
      const float m = fmaxf(soft.m, m2);
      const float unit = MASK == kFloatMask ? kLog2e : 1.0f;
      const float f1 = m == soft.m ? 1.0f : __builtin_amdgcn_exp2f((soft.m - m) * unit);
      const float f2 = m == m2 ? 1.0f : __builtin_amdgcn_exp2f((m2 - m) * unit);
      soft.rescale(f1);
      soft.m = m;
      soft.l = fmaf(l2, f2, soft.l);
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          soft.acc[c][i] = fmaf(at[(32 * c + result_row(i)) * 32 + lane % 32], f2, soft.acc[c][i]);
    }
  }

  if (!live) return;
  if (a.splits > 1) {
    const int64_t at = w.part_row(a, r);
    if (lane < 32) a.part_stats[at] = float2{soft.m, soft.l};
    float* part = a.part + at * a.D;
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * c + 8 * g + 4 * (lane / 32);
        const float v[4] = {soft.acc[c][4 * g], soft.acc[c][4 * g + 1], soft.acc[c][4 * g + 2], soft.acc[c][4 * g + 3]};
        store_four(part + d, v, a.D - d, a.D % 4 == 0);
      }
    return;
  }
  const float inverse = soft.m == kLowest ? 0.0f : 1.0f / soft.l;
  if (a.stats && lane < 32)
    a.stats[stat_at(a, w.b, mine)] = soft.m == kLowest ? float2{INFINITY, 0.0f}
                                                       : float2{soft.m, log2f(soft.l) - kForwardBits<T>};
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) soft.acc[c][i] *= inverse;
  write_row<T, DP>(a, static_cast<T*>(a.out) + w.b * (int64_t(a.Q) * (a.K * a.G) * a.D), mine, soft.acc);
}

// Joins the pieces of the forward's rows. A row has `lanes` lanes of four channels each, `shares`
// of them (both powers of two) for its pieces: a lane takes every shares-th piece, four at a time,
// and the shares meet in LDS in their order. So few rows of many pieces do not wait for one
// lane's loads in turn, and many rows of few pieces fill the workgroup. Bound by the latency of
// its loads: 4 to 8 us for the calls above.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_combine_kernel(const Args a, int lanes, int shares, bool natural,
                                                                     int keys) {
  __shared__ f32x4 sums[kThreads];
  __shared__ float2 stats[kThreads];
  const int b = int(blockIdx.y) / a.K, kv = int(blockIdx.y) % a.K;
  const Pieces pieces = pieces_of(a, b, keys);
  const int rows = kThreads / (lanes * shares);  // of this workgroup
  const int lane = int(threadIdx.x) % lanes, share = (int(threadIdx.x) / lanes) % shares;
  const int64_t r = int64_t(blockIdx.x) * rows + int(threadIdx.x) / (lanes * shares);
  const bool live = r < a.R;
  const int d = lane * 4, left = a.D - d;
  const float unit = natural ? kLog2e : 1.0f;
  const int64_t each = int64_t(a.K) * a.R, first = (int64_t(pieces.first) * a.K + kv) * a.R + r;
  float m = kLowest, l = 0.0f;
  f32x4 v = {0, 0, 0, 0};
  auto join = [&](const float2& st, f32x4 four, float top) __attribute__((always_inline)) {
    const float f = st.x == kLowest ? 0.0f : __builtin_amdgcn_exp2f((st.x - top) * unit);
    l = fmaf(st.y, f, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fmaf(four[i], f, v[i]);
  };
  auto raise = [&](float top) __attribute__((always_inline)) {
    const float f = m == kLowest ? 0.0f : __builtin_amdgcn_exp2f((m - top) * unit);
    m = top;
    l *= f;
    v *= f;
  };
  constexpr int kAhead = 4;
  for (int s = share; s < pieces.count; s += kAhead * shares) {
    float2 st[kAhead];
    f32x4 four[kAhead];
    float top = m;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int piece = s + i * shares;
      const bool here = live && piece < pieces.count;
      const int64_t at = first + piece * each;
      const float* p = a.part + at * a.D + d;
      st[i] = here ? a.part_stats[at] : float2{kLowest, 0.0f};
      four[i] = f32x4{0, 0, 0, 0};
      if (here && left > 0) {
        if (a.D % 4 == 0) {
          four[i] = *reinterpret_cast<const f32x4*>(p);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < left) four[i][j] = p[j];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) top = fmaxf(top, st[i].x);
    raise(top);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) join(st[i], four[i], top);
  }
  if (shares > 1) {
    sums[threadIdx.x] = v;
    stats[threadIdx.x] = float2{m, l};
    __syncthreads();
    if (share > 0) return;
    for (int i = 1; i < shares; ++i) {
      const float2 st = stats[threadIdx.x + i * lanes];
      raise(fmaxf(m, st.x));
      join(st, sums[threadIdx.x + i * lanes], m);
    }
  }
  if (!live) return;
  const float inverse = m == kLowest ? 0.0f : 1.0f / l;
  const float out_v[4] = {v[0] * inverse, v[1] * inverse, v[2] * inverse, v[3] * inverse};
  const RowOf o = row_of(a, kv, uint32_t(r));
  T* out = static_cast<T*>(a.out) + ((int64_t(b) * a.Q + o.query) * (a.K * a.G) + o.head) * a.D;
  store_four(out + d, out_v, left, a.out_vector);
  if (a.stats && lane == 0)
    a.stats[stat_at(a, b, o)] = m == kLowest ? float2{INFINITY, 0.0f} : float2{m, log2f(l) - kForwardBits<T>};
}

// ---------------------------------------------------------------------------
// Backward, queries: the forward's walk over the keys with p formed from the row's statistics.
// It also leaves delta_i = do_i . o_i of its rows for the states' kernel.

template <typename T, int DP, int MASK, int WR>
__global__ __launch_bounds__(kThreads, grad_q_waves(sizeof(T), DP, MASK)) void attention_grad_q_kernel(const Args a) {
  using Shape = ForwardShape<T, DP, WR>;
  using TileT = Tile<T, DP>;
  constexpr int KB = Shape::KB, NB = DP / 32, kSteps = TileT::kPieces / 2, kKeys = Shape::kKeys;
  __shared__ __attribute__((aligned(16))) char lds[Shape::kLds];

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int wr = wave % WR, wk = wave / WR;
  const KeyWalk<Shape> w(a);
  if (w.b < 0) return;  // a slot that no image needs
  const uint32_t r = w.row_tile * Shape::kRows + 32 * wr + lane % 32;
  const bool live = r < a.R;
  const RowOf mine = row_of(a, w.kv, live ? r : a.R - 1);
  int64_t mask_at = 0;
  if constexpr (MASK != kNoMask) mask_at = mask_row_at(a, w.b, mine);
  const int local = 32 * KB * wk;
  KeyStage<T, DP, MASK, Shape> stage(a, w, local);
  stage.mask_at = mask_at;
  if (w.first < w.last) stage.load(w.first);

  typename Mma<T>::Piece q[kSteps], go[kSteps];
  take_rows<T, DP>(a, row_at<T>(a.q, w.b, mine), live, q);
  take_rows<T, DP>(a, row_at<T>(a.go, w.b, mine), live, go);
  // Lanes past the last row repeat it.
  const float delta = row_dot<T, DP>(a, row_at<T>(a.go, w.b, mine), row_at<T>(a.o, w.b, mine));
  const float2 stat = live ? a.row_stats[stat_at(a, w.b, mine)] : float2{INFINITY, 0.0f};
  if (w.leads && wk == 0 && live && lane < 32) a.delta[stat_at(a, w.b, mine)] = delta;

  f32x16 acc[NB] = {};
  Scaled<T> scaled;
  const float factor = MASK == kFloatMask ? a.scale : a.scale * kLog2e;
  const float shift = kWeightBits<T> - (MASK == kFloatMask ? stat.y : stat.x + stat.y);

  auto step = [&](int tile, auto buffer) __attribute__((always_inline)) {
    char* k_tile = lds + decltype(buffer)::value * 2 * Shape::kTile;
    char* v_tile = k_tile + Shape::kTile;
    if (Shape::kBuffers == 1 && tile > w.first) __syncthreads();
    stage.k.store(k_tile);
    stage.v.store(v_tile);
    uint32_t mask[KB];
#pragma unroll
    for (int n = 0; n < KB; ++n) mask[n] = MASK == kBoolMask ? stage.next[n] : 0;
    __syncthreads();
    if (tile + 1 < w.last) stage.load(tile + 1);

#pragma unroll
    for (int n = 0; n < KB; ++n) {
      const int here = local + 32 * n, key0 = tile * kKeys + here;
      if constexpr (MASK == kBoolMask)
        if (!__any(mask[n] != 0 && live)) continue;
      const uint32_t bits = result_bits(mask[n]);
      float add[16];
      if constexpr (MASK == kFloatMask) float_masks(a, mask_at, key0, add);
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        s = multiply<T>(row_piece<T, DP>(k_tile, here, t), q[t], s);
        dp = multiply<T>(row_piece<T, DP>(v_tile, here, t), go[t], dp);
      }
      float ds[16];
      const float low = delta * scaled.power;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = MASK == kFloatMask ? fmaf(fmaf(s[i], factor, add[i]) - stat.x, kLog2e, shift)
                                           : fmaf(s[i], factor, shift);
        ds[i] = __builtin_amdgcn_exp2f(y) * fmaf(dp[i], scaled.power, -low);
        if constexpr (MASK == kBoolMask) ds[i] = where_bit(bits, 8 * (i / 4) + i % 4, ds[i], 0.0f);
        if constexpr (MASK == kFloatMask) ds[i] = add[i] == kLowest ? 0.0f : ds[i];
      }
      if (key0 + 32 > w.states) {
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] = key0 + result_row(i) < w.states ? ds[i] : 0.0f;
      }
      scaled.fit(ds, acc);
      const auto weights = Mma<T>::weights(ds);
#pragma unroll
      for (int c = 0; c < NB; ++c) acc[c] = accumulate<T, DP>(k_tile, here, c, weights, acc[c]);
    }
  };
  for (int tile = w.first; tile < w.last; tile += 2) {
    step(tile, Const<0>());
    if (tile + 1 < w.last) step(tile + 1, Const<Shape::kBuffers - 1>());
  }

  const float unit = a.scale * __builtin_amdgcn_exp2f(-kWeightBits<T>), undo = scaled.undo();
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[c][i] = acc[c][i] * undo * unit;
  if constexpr (Shape::WK > 1) {
    __syncthreads();
    float* mine_at = reinterpret_cast<float*>(lds) + wave * 32 * DP;
#pragma unroll
    for (int c = 0; c < NB; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine_at[(32 * c + result_row(i)) * 32 + lane % 32] = acc[c][i];
    __syncthreads();
    if (wk > 0) return;
    for (int other = 1; other < Shape::WK; ++other) {
      const float* at = reinterpret_cast<const float*>(lds) + (other * WR + wr) * 32 * DP;
#pragma unroll
      for (int c = 0; c < NB; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][i] += at[(32 * c + result_row(i)) * 32 + lane % 32];
    }
  }
  const int64_t of_image = int64_t(a.Q) * (a.K * a.G) * a.D;
  if (!live) return;
  if (a.splits == 1) {
    write_row<T, DP>(a, static_cast<T*>(a.grad_q) + w.b * of_image, mine, acc);
    return;
  }
  // A piece's sums lie in the order of an image's grad_q.
  float* part = a.part + w.slot * of_image + (int64_t(mine.query) * (a.K * a.G) + mine.head) * a.D;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * (lane / 32);
      const float v[4] = {acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]};
      store_four(part + d, v, a.D - d, a.D % 4 == 0);
    }
}

// ---------------------------------------------------------------------------
// Backward, states: a workgroup's 4 waves hold 32 keys each and walk over the queries of each
// head of the group in turn, so that dk and dv of a key are summed by one wave. Row splits
// leave fp32 sums, which sum_kernel adds in their order.

template <typename T, int DP> struct StatesShape {
  static constexpr int kKeys = 32 * kWaves;
  static constexpr int RB = DP * int(sizeof(T)) <= 192 ? 2 : 1;  // blocks of 32 rows in a tile
  static constexpr int kRows = 32 * RB;
  static constexpr int kTile = kRows * Tile<T, DP>::kRowBytes;
  static constexpr int kWords = kRows * kWaves * 4;  // a bool mask: 32 keys' bits for each row and wave
  static constexpr int kBuffer = 2 * kTile + kWords + kRows * 3 * 4;
  static constexpr int kLds = 2 * kBuffer;
  // FUSED: the keys' tile and ds of a tile of rows.
  static constexpr int kKeyTile = kKeys * Tile<T, DP>::kRowBytes;
  static constexpr int kScoreTile = kRows * Tile<T, kKeys>::kRowBytes;
};

// acc (channels x lanes) += tile^T (32 channels from 32 * block) x the rows' pieces `scores`, over
// all kKeys tile rows in their order.
template <typename T, int DP, int KEYS>
__device__ inline f32x16 accumulate_rows(const char* tile, int block, const char* scores, int row, f32x16 acc) {
  const int half = int(threadIdx.x % kWave) / 32;
#pragma unroll
  for (int t = 0; t < KEYS / 16; ++t) {
    typename Mma<T>::Vec a[Mma<T>::kPlanes], b[Mma<T>::kPlanes];
    const auto piece = row_piece<T, KEYS>(scores, row, t);
#pragma unroll
    for (int p = 0; p < Mma<T>::kPlanes; ++p) b[p] = __builtin_bit_cast(typename Mma<T>::Vec, piece.plane[p]);
    const int key = 16 * t + 8 * half;
    turned<T, DP>(tile, key, key + 4, block, a);
    acc = Mma<T>::product(a, b, acc);
  }
  return acc;
}

// FUSED: all states fill one workgroup's keys. Then it forms dq of its rows too, from ds in LDS,
// and delta from the outputs: one pass over the rows' bytes, which bound calls of many rows and
// few states, and 5 products in place of 7. Not in f16, whose ds has a scale for each key that a
// sum over the keys cannot use.
template <typename T, int DP, int MASK, bool FUSED>
__global__ __launch_bounds__(kThreads, grad_states_waves(sizeof(T), DP, MASK, FUSED)) void attention_grad_states_kernel(const Args a) {
  using Shape = StatesShape<T, DP>;
  using TileT = Tile<T, DP>;
  constexpr int NB = DP / 32, kSteps = TileT::kPieces / 2, kRows = Shape::kRows;
  constexpr int N = 16 / int(sizeof(T));
  __shared__ __attribute__((aligned(16))) char lds[Shape::kLds + (FUSED ? Shape::kKeyTile + Shape::kScoreTile : 0)];
  char* const key_rows = lds + Shape::kLds;  // FUSED
  char* const scores = key_rows + Shape::kKeyTile;

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  // The heads whose rows share a cache line first (the key heads are a multiple of `near`),
  // then the tiles, which read the same queries.
  const uint32_t key_tiles = (uint32_t(a.S) + Shape::kKeys - 1) / Shape::kKeys;
  uint32_t id = xcd_order(blockIdx.x, gridDim.x);
  int kv = int(id % uint32_t(a.near));
  id /= a.near;
  const int key_tile = int(id % key_tiles);
  id /= key_tiles;
  const int split = int(id % uint32_t(a.row_splits));
  id /= a.row_splits;
  kv += int(id % uint32_t(a.K / a.near)) * a.near;
  const int b = int(id / uint32_t(a.K / a.near));

  const int states = __builtin_amdgcn_readfirstlane(states_of(a, b));
  const int key = key_tile * Shape::kKeys + 32 * wave + lane % 32;
  const bool words = MASK == kBoolMask && !a.mask_of_keys;
  bool on = key < states;
  if constexpr (MASK == kBoolMask)
    if (a.mask_of_keys && on) on = state_bit(a, b, key);

  // Tiles of every head of the group in turn.
  const int query_tiles = (a.Q + kRows - 1) / kRows;
  const int64_t tiles = int64_t(query_tiles) * a.G;
  int64_t first = 0, last = tiles;
  if (a.row_splits > 1) {  // 64-bit divisions are long
    first = tiles * split / a.row_splits;
    last = tiles * (split + 1) / a.row_splits;
  }
  // Padding only: zeros. FUSED goes on to write dq, which is 0 then.
  if (!FUSED && key_tile * Shape::kKeys >= states) last = first;
  int next_head = first ? int(first / query_tiles) : 0, next_tile = int(first - int64_t(next_head) * query_tiles);

  Stage<T, DP, kRows> q_stage, go_stage, o_stage;
  q_stage.plan(a.q.row, a.Dp);
  go_stage.plan(a.go.row, a.Dp);
  if constexpr (FUSED) {
    o_stage.plan(a.o.row, a.Dp);
    Stage<T, DP, Shape::kKeys> keys;
    keys.plan(a.k.row, a.Dp);
    auto kept = [&](int row) { return MASK != kBoolMask || !a.mask_of_keys || (row < states && state_bit(a, b, row)); };
    keys.load(static_cast<const T*>(a.k.at) + b * a.k.batch + kv * a.k.head, states, kept);
    keys.store(key_rows);
  }
  float2 stat = {INFINITY, 0.0f};
  float delta = 0.0f;
  uint32_t word = 0;
  int64_t float_at = 0, float_next = 0;  // the tile's first mask element, and its rows (float masks)
  int float_rows = 0, float_left = 0;
  int row_head = 0, row_query = 0, row_head_next = 0, row_query_next = 0;
  auto load = [&]() __attribute__((always_inline)) {  // the next tile
    const int head = kv * a.G + next_head, query = next_tile * kRows, left = a.Q - query;
    q_stage.load(static_cast<const T*>(a.q.at) + b * a.q.batch + head * a.q.head + int64_t(query) * a.q.row, left, All());
    go_stage.load(static_cast<const T*>(a.go.at) + b * a.go.batch + head * a.go.head + int64_t(query) * a.go.row, left,
                  All());
    if (threadIdx.x < kRows) {
      const bool live = int(threadIdx.x) < left;
      const int64_t at = (int64_t(b) * (a.K * a.G) + head) * a.Q + query + threadIdx.x;
      stat = live ? a.row_stats[at] : float2{INFINITY, 0.0f};
      if constexpr (!FUSED) delta = live ? a.delta[at] : 0.0f;
    }
    if constexpr (FUSED)
      o_stage.load(static_cast<const T*>(a.o.at) + b * a.o.batch + head * a.o.head + int64_t(query) * a.o.row, left, All());
    row_head_next = head;
    row_query_next = query;
    if constexpr (MASK == kFloatMask) {
      float_next = mask_row_at(a, b, RowOf{query, head});
      float_left = left;
    }
    if (words && threadIdx.x < kRows * kWaves) {  // row threadIdx.x / 4, keys 32 (threadIdx.x % 4) ..
      const int row = threadIdx.x / kWaves;
      const int64_t at = mask_row_at(a, b, RowOf{query + (row < left ? row : left - 1), head});
      word = static_cast<const uint32_t*>(a.mask)[at + key_tile * (Shape::kKeys / 32) + int(threadIdx.x % kWaves)];
    }
    if (++next_tile == query_tiles) {
      next_tile = 0;
      ++next_head;
    }
  };
  if (first < last) load();

  typename Mma<T>::Piece k[kSteps], v[kSteps];
  take_rows<T, DP>(a, static_cast<const T*>(a.k.at) + b * a.k.batch + int64_t(key) * a.k.row + kv * a.k.head, on, k);
  take_rows<T, DP>(a, static_cast<const T*>(a.v.at) + b * a.v.batch + int64_t(key) * a.v.row + kv * a.v.head, on, v);

  f32x16 grad_k[NB] = {}, grad_v[NB] = {};
  Scaled<T> scaled;
  const float factor = MASK == kFloatMask ? a.scale : a.scale * kLog2e;
  auto put_score = [&](int row, float v) __attribute__((always_inline)) {
    const int at = 32 * wave + lane % 32;
    auto put = [&](int plane, auto x) __attribute__((always_inline)) {
      *reinterpret_cast<decltype(x)*>(scores + Tile<T, Shape::kKeys>::offset(row, at / 8, plane) + (at % 8) * 2) = x;
    };
    if constexpr (sizeof(T) == 2) {
      put(0, static_cast<T>(v));
    } else {
      bf16_t parts[3];
      Mma<T>::split(v, parts);
#pragma unroll
      for (int p = 0; p < 3; ++p) put(p, parts[p]);
    }
  };
  auto step = [&](int64_t tile, auto buffer) __attribute__((always_inline)) {
    char* q_tile = lds + decltype(buffer)::value * Shape::kBuffer;
    char* go_tile = q_tile + Shape::kTile;
    uint32_t* row_words = reinterpret_cast<uint32_t*>(go_tile + Shape::kTile);
    float* row_shift = reinterpret_cast<float*>(row_words + Shape::kWords / 4);
    float* row_delta = row_shift + kRows;  // minus delta
    float* row_max = row_delta + kRows;    // float masks only
    q_stage.store(q_tile);
    go_stage.store(go_tile);
    if (threadIdx.x < kRows) {
      row_shift[threadIdx.x] = kWeightBits<T> - (MASK == kFloatMask ? stat.y : stat.x + stat.y);
      if constexpr (!FUSED) row_delta[threadIdx.x] = -delta;
      if constexpr (MASK == kFloatMask) row_max[threadIdx.x] = stat.x;
    }
    if constexpr (FUSED) {  // the lanes of a row, a power of two, add up do . o
#pragma unroll
      for (int i = 0; i < Stage<T, DP, kRows>::kEach; ++i) {
        T x[N], y[N];
        __builtin_memcpy(x, &go_stage.hold[i], 16);
        __builtin_memcpy(y, &o_stage.hold[i], 16);
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) dot = fmaf(widen(x[j]), widen(y[j]), dot);
#pragma unroll
        for (int by = 1; by < Stage<T, DP, kRows>::kPieces; by *= 2) dot += __shfl_xor(dot, by);
        if (o_stage.piece(i) == 0) row_delta[o_stage.row(i)] = -dot;
      }
    }
    if (words && threadIdx.x < kRows * kWaves)
      row_words[(threadIdx.x % kWaves) * kRows + threadIdx.x / kWaves] = word;
    float_at = float_next;
    float_rows = float_left;
    row_head = row_head_next;
    row_query = row_query_next;
    __syncthreads();
    if (tile + 1 < last) load();

    // Two blocks of rows unrolled take more registers than they hide: as fast at 64 channels, 8 %
    // slower at 96 (2 x 452 rows of 1,171 states, 32 heads).
#pragma unroll 1
    for (int n = 0; n < Shape::RB; ++n) {
      const int local = 32 * n;
      float add[16];
      // The rows' words as they are, for 4 x 1,501 rows of 2,333 states, 8 heads of 128: 493 us
      // forward and backward against 519 with the lane's 16 bits packed into one. FUSED has no
      // registers left and packs them: 161 us against 251 for 6 x 5,108 rows of 100 states, 16
      // heads of 64.
      uint32_t bits[MASK == kBoolMask && !FUSED ? 16 : 1];
      auto attended = [&](int i, float x) {
        if constexpr (FUSED) return (bits[0] >> i) & 1 ? x : 0.0f;
        else return where_bit(bits[i], lane % 32, x, 0.0f);
      };
#pragma unroll
      for (uint32_t& word : bits) word = ~0u;
      if (words) {
        uint32_t any = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const u32x4 four = *reinterpret_cast<const u32x4*>(row_words + wave * kRows + local + result_row(4 * g));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (FUSED) any |= ((four[j] >> (lane % 32)) & 1) << (4 * g + j);
            else if constexpr (MASK == kBoolMask) any |= bits[4 * g + j] = four[j];
          }
        }
        if constexpr (FUSED) bits[0] = any;
        else any = (any >> (lane % 32)) & 1;
        if (!__any(on && any != 0)) {
          if constexpr (FUSED) {
#pragma unroll
            for (int i = 0; i < 16; ++i) put_score(local + result_row(i), 0.0f);
          }
          continue;
        }
      } else if constexpr (MASK == kFloatMask) {
        // Rows and keys that are not there take the last one's address.
        const int64_t column = float_at + (key < a.S ? key : a.S - 1);
        mask_elements(a, [&](int i) {
          const int row = local + result_row(i);
          return column + (row < float_rows ? row : float_rows - 1) * a.mask_row;
        }, add);
#pragma unroll
        for (int i = 0; i < 16; ++i) add[i] = on && local + result_row(i) < float_rows ? add[i] : kLowest;
      }
      f32x16 s = {}, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 low = *reinterpret_cast<const f32x4*>(row_delta + local + result_row(4 * g));
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[4 * g + j] = low[j];
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        s = multiply<T>(row_piece<T, DP>(q_tile, local, t), k[t], s);
        dp = multiply<T>(row_piece<T, DP>(go_tile, local, t), v[t], dp);
      }
      float p[16], ds[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = local + result_row(4 * g);
        const f32x4 shift = *reinterpret_cast<const f32x4*>(row_shift + at);
        f32x4 top = {};
        if constexpr (MASK == kFloatMask) top = *reinterpret_cast<const f32x4*>(row_max + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * g + j;
          const float y = MASK == kFloatMask ? fmaf(fmaf(s[i], factor, add[i]) - top[j], kLog2e, shift[j])
                                             : fmaf(s[i], factor, shift[j]);
          p[i] = __builtin_amdgcn_exp2f(y);
          // Without a mask every state of the tile is attended; columns past the last are
          // not written.
          if constexpr (MASK == kBoolMask) p[i] = attended(i, p[i]);
          if constexpr (MASK == kFloatMask) p[i] = add[i] == kLowest ? 0.0f : p[i];
          ds[i] = p[i] * scaled.power * dp[i];
          // A masked state may hold anything: 0 times its NaN or infinity is not 0.
          if constexpr (MASK != kNoMask) ds[i] = p[i] == 0.0f ? 0.0f : ds[i];
        }
      }
      const auto wp = Mma<T>::weights(p);
#pragma unroll
      for (int c = 0; c < NB; ++c) grad_v[c] = accumulate<T, DP>(go_tile, local, c, wp, grad_v[c]);
      if constexpr (FUSED) {
#pragma unroll
        for (int i = 0; i < 16; ++i) put_score(local + result_row(i), on ? ds[i] : 0.0f);
      }
      scaled.fit(ds, grad_k);
      const auto ws = Mma<T>::weights(ds);
#pragma unroll
      for (int c = 0; c < NB; ++c) grad_k[c] = accumulate<T, DP>(q_tile, local, c, ws, grad_k[c]);
    }
    if constexpr (FUSED) {  // dq: blocks of 32 rows x 32 channels, shared by the waves
      __syncthreads();
      for (int job = wave; job < Shape::RB * NB; job += kWaves) {
        const int local = 32 * (job % Shape::RB), block = job / Shape::RB, query = row_query + local + lane % 32;
        const f32x16 acc = accumulate_rows<T, DP, Shape::kKeys>(key_rows, block, scores, local, f32x16{});
        if (query >= a.Q) continue;
        T* to = static_cast<T*>(a.grad_q) + ((int64_t(b) * a.Q + query) * (a.K * a.G) + row_head) * a.D;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = 32 * block + 8 * g + 4 * (lane / 32);
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = acc[4 * g + i] * a.scale;
          store_four(to + d, x, a.D - d, a.out_vector);
        }
      }
    }
  };
  for (int64_t tile = first; tile < last; tile += 2) {
    step(tile, Const<0>());
    if (tile + 1 < last) step(tile + 1, Const<1>());
  }

  if (key >= a.S) return;
  const float unit = __builtin_amdgcn_exp2f(-kWeightBits<T>), undo = scaled.undo();
  const int64_t at = ((int64_t(b) * a.S + key) * a.K + kv) * a.D;
  const int64_t elements = int64_t(a.B) * a.S * a.K * a.D;
#pragma unroll
  for (int c = 0; c < NB; ++c)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * c + 8 * g + 4 * (lane / 32);
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = on ? grad_k[c][4 * g + i] * undo * (unit * a.scale) : 0.0f;
        y[i] = on ? grad_v[c][4 * g + i] * unit : 0.0f;
      }
      if (a.row_splits > 1) {
        store_four(a.part_k + split * elements + at + d, x, a.D - d, a.D % 4 == 0);
        store_four(a.part_v + split * elements + at + d, y, a.D - d, a.D % 4 == 0);
      } else {
        store_four(static_cast<T*>(a.grad_k) + at + d, x, a.D - d, a.out_vector);
        store_four(static_cast<T*>(a.grad_v) + at + d, y, a.D - d, a.out_vector);
      }
    }
}

// out = the sum of fp32 parts of n elements each, in a fixed order: for grad_q (`of_keys` keys in
// a tile) the parts of image blockIdx.y's pieces, for the states all row_splits parts of grad_k
// (blockIdx.y 0) and grad_v. Four waves share the parts of 64 x 4 elements. 5 us for 2 x 77 states
// of 8 heads of 64 in 16 parts: a launch and its loads' latency.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_sum_kernel(const Args a, int64_t n, int of_keys) {
  __shared__ f32x4 sums[kWaves - 1][kWave];
  const int lane = threadIdx.x % kWave, share = threadIdx.x / kWave;
  const int64_t at = (int64_t(blockIdx.x) * kWave + lane) * 4;
  const float* part;
  T* out;
  Pieces pieces = {0, a.row_splits};
  if (of_keys) {
    pieces = pieces_of(a, int(blockIdx.y), of_keys);
    part = a.part;
    out = static_cast<T*>(a.grad_q) + blockIdx.y * n;
  } else {
    part = blockIdx.y ? a.part_v : a.part_k;
    out = static_cast<T*>(blockIdx.y ? a.grad_v : a.grad_k);
  }
  const bool vector = n % 4 == 0;
  f32x4 v = {0, 0, 0, 0};
  if (at < n) {
#pragma unroll 4
    for (int s = pieces.first + share; s < pieces.first + pieces.count; s += kWaves) {
      const float* p = part + s * n + at;
      if (vector) {
        v += *reinterpret_cast<const f32x4*>(p);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + i < n) v[i] += p[i];
      }
    }
  }
  if (share) sums[share - 1][lane] = v;
  __syncthreads();
  if (share || at >= n) return;
#pragma unroll
  for (int s = 0; s < kWaves - 1; ++s) v += sums[s][lane];
  const float four[4] = {v[0], v[1], v[2], v[3]};
  store_four(out + at, four, int(n - at < 4 ? n - at : 4), vector && reinterpret_cast<uintptr_t>(out) % 16 == 0);
}

// A bool mask's bytes as words of 32 keys, `words` of them for a row (a multiple of 4), one
// thread each. The kernels read a row's mask several times (every head of a mask that is one for
// all, forward and backward), as words at an eighth of the bytes, and two operations for each
// score. Bound by the bytes read: 4 us for 6.6 MB, launch included. Axes of stride 0 have size 1.
inline __global__ __launch_bounds__(256) void attention_mask_bits_kernel(const uint8_t* from, uint32_t* to, int64_t batch,
                                                                         int64_t head, int64_t row, int64_t key, int heads,
                                                                         int rows, int S, int words, int64_t count) {
  const int64_t n = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (n >= count) return;
  const int word = int(n % words), k0 = 32 * word;
  int64_t at = n / words;
  const int64_t r = at % rows;
  at /= rows;
  const uint8_t* bytes = from + (at / heads) * batch + (at % heads) * head + r * row;
  uint32_t bits = 0;
  if (key == 1 && k0 + 32 <= S) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const u32x4 four = load_anywhere<u32x4>(bytes + k0 + 16 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t x = four[j] | (four[j] >> 4);  // non-zero bytes to their lowest bits
        x |= x >> 2;
        x |= x >> 1;
        bits |= ((((x & 0x01010101u) * 0x01020408u) >> 24) & 15u) << (16 * i + 4 * j);
      }
    }
  } else {
    for (int i = 0; i < 32 && k0 + i < S; ++i) bits |= uint32_t(bytes[(k0 + i) * key] != 0) << i;
  }
  to[n] = bits;
}

// A float mask whose keys do not lie side by side, or of fewer than 4, as rows of `keys` (a multiple
// of 32), with zeros past S: one thread for each element. Axes of stride 0 have size 1.
template <typename V>
__global__ __launch_bounds__(256) void attention_pack_mask_kernel(const V* from, V* to, int64_t batch, int64_t head,
                                                                  int64_t row, int64_t key, int heads, int rows, int S,
                                                                  int keys, int64_t elements) {
  const int64_t n = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (n >= elements) return;
  const int k = int(n % keys);
  int64_t at = n / keys;
  const int64_t r = at % rows;
  at /= rows;
  to[n] = k < S ? from[(at / heads) * batch + (at % heads) * head + r * row + k * key] : V(0);
}

// Rows of D channels at any strides and alignment, as dense rows of Dp with zeros past D: one
// thread per 16 bytes of the copy.
template <typename T>
__global__ __launch_bounds__(256) void attention_pack_kernel(Rows from, T* to, int64_t rows, int heads, int D, int Dp,
                                                             int64_t pieces) {
  constexpr int N = 16 / int(sizeof(T));
  const int64_t n = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (n >= pieces) return;
  const int each = Dp / N, d = int(n % each) * N;
  int64_t at = n / each;
  const int64_t head = at % heads;
  at /= heads;
  const T* row = static_cast<const T*>(from.at) + (at / rows) * from.batch + (at % rows) * from.row + head * from.head;
  T parts[N];
#pragma unroll
  for (int i = 0; i < N; ++i) parts[i] = d + i < D ? row[d + i] : T(0);
  u32x4 out;
  __builtin_memcpy(&out, parts, 16);
  *reinterpret_cast<u32x4*>(to + n * N) = out;
}

// ---------------------------------------------------------------------------
// Launches, one translation unit for each type (attention_f32.hip and so on): the kernels'
// variants compile side by side.

template <typename F> void with_mask(int kind, F f) {
  if (kind == kNoMask) f(Const<kNoMask>());
  else if (kind == kBoolMask) f(Const<kBoolMask>());
  else f(Const<kFloatMask>());
}

inline int padded(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

template <typename F> void with_channels(int64_t D, F f) {
  switch (padded(D)) {
    case 32: f(Const<32>()); break;
    case 64: f(Const<64>()); break;
    case 96: f(Const<96>()); break;
    default: f(Const<128>()); break;
  }
}

// `groups` and `key_groups`: workgroups of the walk over the keys and over the rows.
// Whether the states' kernel forms dq too where all keys fit its workgroup: not in f16 (its ds
// has a scale for each key), not where a row's pieces are no power of two lanes (96 channels),
// nor in f32 of 128 channels, which it would spill.
constexpr bool fused_shape(bool f16, int size, int DP) { return !f16 && DP != 96 && DP * size < 512; }

// What variant runs, by the plan of the call.
struct Variant {
  bool few_rows, fused;
};
template <typename T>
void launch_forward(const Args& a, int mask_kind, Variant variant, uint32_t groups, hipStream_t s);
template <typename T>
void launch_backward(const Args& a, int mask_kind, Variant variant, uint32_t groups, uint32_t key_groups, hipStream_t s);
template <typename T>
void launch_pack(const Rows& from, void* to, int64_t batch, int64_t rows, int heads, int D, int Dp, hipStream_t s);

#ifdef ATTENTION_DEFINE_LAUNCHES

template <typename T>
void launch_forward(const Args& a, int mask_kind, Variant variant, uint32_t groups, hipStream_t s) {
  with_channels(a.D, [&](auto dp) {
    with_mask(mask_kind, [&](auto kind) {
      constexpr int DP = decltype(dp)::value, MASK = decltype(kind)::value;
      if constexpr (sizeof(T) * DP < 512)
        if (variant.few_rows) return attention_forward_kernel<T, DP, MASK, 1><<<groups, kThreads, 0, s>>>(a);
      attention_forward_kernel<T, DP, MASK, 4><<<groups, kThreads, 0, s>>>(a);
    });
  });
  if (a.splits > 1) {
    int lanes = 1, shares = 1;
    while (4 * lanes < a.D) lanes *= 2;
    while (lanes * shares < kThreads && 4 * shares < a.splits) shares *= 2;
    const int rows = kThreads / (lanes * shares);
    attention_combine_kernel<T><<<dim3(uint32_t(ceil_div(a.R, rows)), uint32_t(a.B * a.K)), kThreads, 0, s>>>(
        a, lanes, shares, mask_kind == kFloatMask, variant.few_rows ? 128 : 64);
  }
}

template <typename T>
void launch_backward(const Args& a, int mask_kind, Variant variant, uint32_t groups, uint32_t key_groups, hipStream_t s) {
  with_channels(a.D, [&](auto dp) {
    with_mask(mask_kind, [&](auto kind) {
      constexpr int DP = decltype(dp)::value, MASK = decltype(kind)::value;
      if constexpr (fused_shape(std::is_same_v<T, f16_t>, sizeof(T), DP))
        if (variant.fused) return attention_grad_states_kernel<T, DP, MASK, true><<<key_groups, kThreads, 0, s>>>(a);
      bool done = groups == 0;
      if constexpr (sizeof(T) * DP < 512)
        if (variant.few_rows && !done) {
          attention_grad_q_kernel<T, DP, MASK, 1><<<groups, kThreads, 0, s>>>(a);
          done = true;
        }
      if (!done) attention_grad_q_kernel<T, DP, MASK, 4><<<groups, kThreads, 0, s>>>(a);
      if (key_groups) attention_grad_states_kernel<T, DP, MASK, false><<<key_groups, kThreads, 0, s>>>(a);
    });
  });
  if (groups && a.splits > 1 && !variant.fused) {
    const int64_t n = int64_t(a.Q) * a.K * a.G * a.D;
    attention_sum_kernel<T><<<dim3(uint32_t(ceil_div(n, 4 * kWave)), uint32_t(a.B)), kThreads, 0, s>>>(
        a, n, variant.few_rows ? 128 : 64);
  }
  if (key_groups && a.row_splits > 1) {
    const int64_t n = int64_t(a.B) * a.S * a.K * a.D;
    attention_sum_kernel<T><<<dim3(uint32_t(ceil_div(n, 4 * kWave)), 2), kThreads, 0, s>>>(a, n, 0);
  }
}

template <typename T>
void launch_pack(const Rows& from, void* to, int64_t batch, int64_t rows, int heads, int D, int Dp, hipStream_t s) {
  const int64_t pieces = batch * rows * heads * (Dp / (16 / int64_t(sizeof(T))));
  if (pieces == 0) return;
  attention_pack_kernel<T><<<uint32_t(ceil_div(pieces, 256)), 256, 0, s>>>(from, static_cast<T*>(to), rows, heads, D, Dp, pieces);
}

#define ATTENTION_INSTANTIATE(T)                                                                        \
  namespace attention {                                                                                 \
  template void launch_forward<T>(const Args&, int, Variant, uint32_t, hipStream_t);                    \
  template void launch_backward<T>(const Args&, int, Variant, uint32_t, uint32_t, hipStream_t);         \
  template void launch_pack<T>(const Rows&, void*, int64_t, int64_t, int, int, int, hipStream_t);       \
  }

#endif

}  // namespace attention

#endif  // DEFORMOPS_AMD_ATTENTION_H_
