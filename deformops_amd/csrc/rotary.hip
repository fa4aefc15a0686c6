// Rotary positions with several axes for gfx950: each pair of features turns by the angle
// position[axis of the pair] * frequency of the pair,
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),
// with pairs (j, j + R) or, interleaved, (2 j, 2 j + 1); features past 2 R pass through. The
// transpose of a turn is the turn by -t, so the backward is this call on the gradient with
// `inverse`.
//
// Angles. t = position * frequency is formed in 64 bits as turns (t / 2 pi), of which only the
// fraction counts: at position 10^6 a product in 32 bits would be off by up to 0.06 rad. The
// fraction, in [-1/2, 1/2], is exact enough in 32 bits (2^-26 of a turn).
//
// A workgroup takes some tokens with all their heads. It forms their angles once, into LDS, and
// then streams the heads' rows in 16-byte pieces; bytes bound the large calls: 131,072 tokens of 16
// heads of 128 in bf16 take 180 us, 6.0 TB/s read and written. Angles cost small ones: 21,825
// tokens of 8 heads of 32 in float, 11 pairs, take 17.5 us, 2.6 TB/s.

#include "operators.h"

namespace {

using namespace operators;

constexpr int kMaxPairs = 256;

struct RotaryArgs {
  const void* x;
  void* y;
  int64_t x_batch, x_row, x_head;
  const void* positions;
  int64_t p_batch, p_row, p_axis;
  const float* frequencies;
  uint8_t axis[kMaxPairs];
  int64_t L;
  int H, D, R;
  int tokens;  // of one workgroup
  int64_t groups_of_image;
  float sign;
  bool vector;
};

template <typename P> __device__ inline double position(const void* p, int64_t at) {
  return static_cast<double>(static_cast<const P*>(p)[at]);
}

template <typename T, typename P, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 turns[];  // [tokens][R] (cos, sin)
  const int64_t b = blockIdx.x / a.groups_of_image;
  const int64_t first = (blockIdx.x % a.groups_of_image) * a.tokens;
  const int count = int(a.L - first < a.tokens ? a.L - first : a.tokens);
  for (int n = threadIdx.x; n < count * a.R; n += 256) {
    const int token = n / a.R, j = n - token * a.R;
    const double at = position<P>(a.positions, b * a.p_batch + (first + token) * a.p_row + a.axis[j] * a.p_axis);
    const double t = at * double(a.frequencies[j]) * 0.15915494309189535;
    const float f = float(t - rint(t));
    turns[n] = float2{cospif(2.0f * f), a.sign * sinpif(2.0f * f)};
  }
  __syncthreads();

  const T* x = static_cast<const T*>(a.x) + b * a.x_batch;
  T* y = static_cast<T*>(a.y) + b * a.L * a.H * a.D;
  constexpr int VEC = 16 / int(sizeof(T));
  const int rows = count * a.H;
  if (a.vector) {
    // Units of a row: R / VEC pairs of pieces (or 2 R / VEC pieces, interleaved), then the
    // pieces that pass.
    const int turned = INTERLEAVED ? 2 * a.R / VEC : a.R / VEC;
    const int units = turned + (a.D - 2 * a.R) / VEC;
    for (int n = threadIdx.x; n < rows * units; n += 256) {
      const int row = n / units, u = n - row * units, token = row / a.H, head = row - token * a.H;
      const T* from = x + (first + token) * a.x_row + head * a.x_head;
      T* to = y + ((first + token) * a.H + head) * a.D;
      const float2* turn = turns + token * a.R;
      if (u >= turned) {
        const int c = 2 * a.R + (u - turned) * VEC;
        *reinterpret_cast<u32x4*>(to + c) = *reinterpret_cast<const u32x4*>(from + c);
        continue;
      }
      if constexpr (INTERLEAVED) {
        T v[VEC];
        u32x4 w = *reinterpret_cast<const u32x4*>(from + u * VEC);
        __builtin_memcpy(v, &w, 16);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const float2 t = turn[u * (VEC / 2) + i / 2];
          const float p = widen(v[i]), q = widen(v[i + 1]);
          v[i] = static_cast<T>(fmaf(p, t.x, -q * t.y));
          v[i + 1] = static_cast<T>(fmaf(q, t.x, p * t.y));
        }
        __builtin_memcpy(&w, v, 16);
        *reinterpret_cast<u32x4*>(to + u * VEC) = w;
      } else {
        T p[VEC], q[VEC];
        u32x4 w = *reinterpret_cast<const u32x4*>(from + u * VEC);
        __builtin_memcpy(p, &w, 16);
        w = *reinterpret_cast<const u32x4*>(from + a.R + u * VEC);
        __builtin_memcpy(q, &w, 16);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float2 t = turn[u * VEC + i];
          const float c = widen(p[i]), d = widen(q[i]);
          p[i] = static_cast<T>(fmaf(c, t.x, -d * t.y));
          q[i] = static_cast<T>(fmaf(d, t.x, c * t.y));
        }
        __builtin_memcpy(&w, p, 16);
        *reinterpret_cast<u32x4*>(to + u * VEC) = w;
        __builtin_memcpy(&w, q, 16);
        *reinterpret_cast<u32x4*>(to + a.R + u * VEC) = w;
      }
    }
    return;
  }
  const int units = a.R + (a.D - 2 * a.R);  // pairs, then single features
  for (int n = threadIdx.x; n < rows * units; n += 256) {
    const int row = n / units, u = n - row * units, token = row / a.H, head = row - token * a.H;
    const T* from = x + (first + token) * a.x_row + head * a.x_head;
    T* to = y + ((first + token) * a.H + head) * a.D;
    if (u >= a.R) {
      to[a.R + u] = from[a.R + u];
      continue;
    }
    const int c = INTERLEAVED ? 2 * u : u, d = INTERLEAVED ? 2 * u + 1 : u + a.R;
    const float2 t = turns[token * a.R + u];
    const float p = widen(from[c]), q = widen(from[d]);
    to[c] = static_cast<T>(fmaf(p, t.x, -q * t.y));
    to[d] = static_cast<T>(fmaf(q, t.x, p * t.y));
  }
}

template <typename T, typename P> void launch(const RotaryArgs& a, bool interleaved, uint32_t groups, hipStream_t s) {
  const size_t lds = size_t(a.tokens) * a.R * sizeof(float2);
  if (interleaved)
    rotary_kernel<T, P, true><<<groups, 256, lds, s>>>(a);
  else
    rotary_kernel<T, P, false><<<groups, 256, lds, s>>>(a);
}

template <typename T> void launch(const RotaryArgs& a, int type, bool interleaved, uint32_t groups, hipStream_t s) {
  if (type == DEFORMOPS_POSITION_I64) launch<T, int64_t>(a, interleaved, groups, s);
  else if (type == DEFORMOPS_POSITION_I32) launch<T, int32_t>(a, interleaved, groups, s);
  else if (type == DEFORMOPS_POSITION_F32) launch<T, float>(a, interleaved, groups, s);
  else launch<T, double>(a, interleaved, groups, s);
}

}  // namespace

extern "C" int deformops_rotary(const void* x, const int64_t* x_strides, void* y, int dtype, const void* positions,
                                const int64_t* position_strides, int position_type, const void* frequencies,
                                const int64_t* sections, int64_t axes, int64_t batch, int64_t tokens, int64_t heads,
                                int64_t channels, int interleaved, int inverse, void* stream) {
  const int size = dtype == MSDA_F32 ? 4 : dtype == MSDA_F16 || dtype == MSDA_BF16 ? 2 : 0;
  if (!size) return fail(MSDA_ERR_INVALID, "rotary: dtype %d is not float32, float16 or bfloat16", dtype);
  if (position_type < DEFORMOPS_POSITION_I64 || position_type > DEFORMOPS_POSITION_F64)
    return fail(MSDA_ERR_INVALID, "rotary: unknown type of positions");
  if (!x_strides || !position_strides || !sections) return fail(MSDA_ERR_INVALID, "rotary: null strides or sections");
  if (batch < 0 || tokens < 0 || heads < 0 || channels < 0 || axes < 1 || axes > 255)
    return fail(MSDA_ERR_INVALID, "rotary: a size is negative, or no axes");
  RotaryArgs a = {};
  int64_t pairs = 0;
  for (int64_t i = 0; i < axes; ++i) {
    if (sections[i] < 0) return fail(MSDA_ERR_INVALID, "rotary: a section is negative");
    if (pairs + sections[i] > kMaxPairs)
      return fail(MSDA_ERR_UNSUPPORTED, "rotary: more than %d rotated pairs", kMaxPairs);
    for (int64_t j = 0; j < sections[i]; ++j) a.axis[pairs + j] = uint8_t(i);
    pairs += sections[i];
  }
  if (2 * pairs > channels) return fail(MSDA_ERR_INVALID, "rotary: the sections rotate more than the channels");
  constexpr int64_t kMost = int64_t(1) << 20;
  if (heads > kMost || channels > kMost || heads * channels > kMost)
    return fail(MSDA_ERR_UNSUPPORTED, "rotary: a token of more than 2^20 elements");
  if (batch == 0 || tokens == 0 || heads == 0 || channels == 0) return MSDA_OK;
  if (!x || !y || (pairs && (!positions || !frequencies))) return fail(MSDA_ERR_INVALID, "rotary: null tensor");
  a.x = x;
  a.y = y;
  a.x_batch = x_strides[0]; a.x_row = x_strides[1]; a.x_head = x_strides[2];
  a.positions = positions;
  a.p_batch = position_strides[0]; a.p_row = position_strides[1]; a.p_axis = position_strides[2];
  a.frequencies = static_cast<const float*>(frequencies);
  a.L = tokens;
  a.H = int(heads); a.D = int(channels); a.R = int(pairs);
  a.sign = inverse ? -1.0f : 1.0f;
  const int n = 16 / size;
  const int64_t part = interleaved ? 2 * pairs : pairs;
  a.vector = aligned(x, 16) && aligned(y, 16) && channels % n == 0 && part % n == 0 && (2 * pairs) % n == 0 &&
             a.x_batch % n == 0 && a.x_row % n == 0 && a.x_head % n == 0;
  // About 16 KB of x in a workgroup, and no more tokens than fill the card.
  int64_t each = 16384 / (heads * channels * size);
  each = each < ceil_div(batch * tokens, 1024) ? each : ceil_div(batch * tokens, 1024);
  each = each < 1 ? 1 : each > 32 ? 32 : each;
  a.tokens = int(each < tokens ? each : tokens);
  a.groups_of_image = ceil_div(tokens, a.tokens);
  if (a.groups_of_image > kMostGroups / batch)
    return fail(MSDA_ERR_UNSUPPORTED, "rotary: the tokens pass a grid");
  const uint32_t groups = uint32_t(a.groups_of_image * batch);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MSDA_F32) launch<float>(a, position_type, interleaved != 0, groups, s);
  else if (dtype == MSDA_F16) launch<f16_t>(a, position_type, interleaved != 0, groups, s);
  else launch<bf16_t>(a, position_type, interleaved != 0, groups, s);
  return launched("rotary");
}
