// What the operators beside MSDA share: element types, the calling thread's error message,
// launch checks and the mapping of workgroups to XCDs.
#ifndef DEFORMOPS_AMD_OPERATORS_H_
#define DEFORMOPS_AMD_OPERATORS_H_

#include <hip/hip_runtime.h>

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "deformops_amd.h"

namespace operators {

using bf16_t = __bf16;
using f16_t = _Float16;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWave = 64;
constexpr int kXcds = 8;  // gfx950 deals workgroups to its 8 XCDs round-robin

// The calling thread's last failure (deformops_last_error).
inline thread_local char g_error[512] = "";

__attribute__((format(printf, 2, 3))) inline int fail(int status, const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(g_error, sizeof(g_error), format, args);
  va_end(args);
  return status;
}

inline int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MSDA_OK : fail(MSDA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// Workgroups of 256 threads that one launch takes: fewer than 2^32 threads.
constexpr int64_t kMostGroups = (int64_t(1) << 24) - 1;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Consecutive workgroup numbers on one XCD, so that neighbours share its L2: the hardware
// gives workgroup i to XCD i % 8, and the answer numbers each XCD's workgroups in a row.
// A bijection for every count: the first count % 8 XCDs hold one more.
__device__ inline uint32_t xcd_order(uint32_t i, uint32_t count) {
  const uint32_t xcd = i % kXcds, each = count / kXcds, more = count % kXcds;
  return xcd * each + (xcd < more ? xcd : more) + i / kXcds;
}

template <typename T> __device__ inline float widen(T v) { return static_cast<float>(v); }

}  // namespace operators

#endif  // DEFORMOPS_AMD_OPERATORS_H_
