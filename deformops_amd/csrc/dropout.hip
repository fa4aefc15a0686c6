// Dropout from a counter-based generator, with the residual's addition, for gfx950:
//   y_i = x_i s + r_i where element i is kept, r_i where it is dropped;  s = 1 / (1 - p)
// Element i is kept where word i % 4 of Philox4x32 with 7 rounds (Salmon, Moraes, Dror and
// Shaw, SC 2011, whose least number of rounds that passes BigCrush is 7), of the counter
// (i / 4, offset) and the key `seed`, is at least p 2^32. The mask is not stored: the
// backward is the same call on the gradient, without a residual.
//
// One thread makes a block's four words for four elements; the words cost 14 products of 32
// bits for four elements. Bytes bound the large calls: 88 million bf16 elements take 56 us, 6.3
// TB/s read and written. Loads and stores pass the caches by, which such a stream only fills.

#include <type_traits>

#include "operators.h"

namespace {

using namespace operators;

struct DropoutArgs {
  const void *x, *residual;
  void* y;
  int64_t n;
  uint64_t seed, offset;
  const int64_t* seed_at;  // the seed in device memory, or null
  uint32_t threshold;
  bool all;  // p = 1
  float scale;
  bool vector;
};

__device__ inline void philox7(uint64_t counter, uint64_t offset, uint64_t seed, uint32_t (&w)[4]) {
  uint32_t c0 = uint32_t(counter), c1 = uint32_t(counter >> 32), c2 = uint32_t(offset), c3 = uint32_t(offset >> 32);
  uint32_t k0 = uint32_t(seed), k1 = uint32_t(seed >> 32);
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const uint64_t a = uint64_t(c0) * 0xD2511F53u, b = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(b >> 32) ^ c1 ^ k0;
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ k1;
    c3 = uint32_t(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// A thread takes VEC elements (16 bytes of them; 4 for the last ones of a call and for rows
// that are not aligned) at a time.
template <typename T, bool RESIDUAL> __global__ __launch_bounds__(256) void dropout_kernel(const DropoutArgs a) {
  constexpr int VEC = 16 / int(sizeof(T));
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);
  T* y = static_cast<T*>(a.y);
  const uint64_t seed = a.seed_at ? uint64_t(*a.seed_at) : a.seed;
  const int64_t pieces = (a.n + VEC - 1) / VEC;
  for (int64_t piece = int64_t(blockIdx.x) * 256 + threadIdx.x; piece < pieces; piece += int64_t(gridDim.x) * 256) {
    const int64_t at = piece * VEC;
    const bool whole = a.vector && at + VEC <= a.n;
    T in[VEC], add[VEC], out[VEC];
    if (whole) {
      const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x + at));
      __builtin_memcpy(in, &w, 16);
      if constexpr (RESIDUAL) {
        const u32x4 r = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(residual + at));
        __builtin_memcpy(add, &r, 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        in[i] = at + i < a.n ? x[at + i] : T(0);
        if constexpr (RESIDUAL) add[i] = at + i < a.n ? residual[at + i] : T(0);
      }
    }
#pragma unroll
    for (int g = 0; g < VEC / 4; ++g) {
      uint32_t w[4];
      philox7(uint64_t(at) / 4 + g, a.offset, seed, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * g + i;
        const bool keep = !a.all && w[i] >= a.threshold;
        // A dropped element leaves nothing of x, also where x is not finite.
        const float v = RESIDUAL ? (keep ? fmaf(widen(in[e]), a.scale, widen(add[e])) : widen(add[e]))
                                 : (keep ? widen(in[e]) * a.scale : 0.0f);
        out[e] = static_cast<T>(v);
      }
    }
    if (whole) {
      u32x4 w;
      __builtin_memcpy(&w, out, 16);
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(y + at));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (at + i < a.n) y[at + i] = out[i];
    }
  }
}

template <typename T> void launch(const DropoutArgs& a, hipStream_t s) {
  const int64_t pieces = ceil_div(a.n, 16 / int(sizeof(T)));
  const uint32_t groups = uint32_t(ceil_div(pieces, 256) < 65536 ? ceil_div(pieces, 256) : 65536);
  if (a.residual)
    dropout_kernel<T, true><<<groups, 256, 0, s>>>(a);
  else
    dropout_kernel<T, false><<<groups, 256, 0, s>>>(a);
}

}  // namespace

extern "C" int deformops_dropout(const void* x, const void* residual, void* y, int dtype, int64_t elements, double p,
                                 uint64_t seed, const void* seed_at, uint64_t offset, void* stream) {
  if (dtype != MSDA_F32 && dtype != MSDA_F16 && dtype != MSDA_BF16)
    return fail(MSDA_ERR_INVALID, "dropout: dtype %d is not float32, float16 or bfloat16", dtype);
  if (elements < 0 || !(p >= 0.0 && p <= 1.0)) return fail(MSDA_ERR_INVALID, "dropout: p must lie in [0, 1]");
  if (elements == 0) return MSDA_OK;
  if (!x || !y) return fail(MSDA_ERR_INVALID, "dropout: null tensor");
  DropoutArgs a = {};
  a.x = x;
  a.residual = residual;
  a.y = y;
  a.n = elements;
  a.seed = seed;
  a.offset = offset;
  a.seed_at = static_cast<const int64_t*>(seed_at);
  a.all = p == 1.0;
  // p 2^32 is exact; the sum rounds half to even, as Python's round().
  const double words = __builtin_nearbyint(p * 4294967296.0);
  a.threshold = words < 4294967295.0 ? uint32_t(words) : 0xFFFFFFFFu;
  a.scale = a.all ? 0.0f : float(1.0 / (1.0 - p));
  a.vector = aligned(x, 16) && aligned(y, 16) && aligned(residual, 16);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MSDA_F32) launch<float>(a, s);
  else if (dtype == MSDA_F16) launch<f16_t>(a, s);
  else launch<bf16_t>(a, s);
  return launched("dropout");
}
