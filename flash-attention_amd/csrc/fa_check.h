// What the entry points of the C ABI check their arguments with.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace fa {

// Leaves a message for fa_last_error() and returns the code.
int fail(int code, const char* fmt, ...);

#define FA_REQUIRE(cond, ...) \
  do {                        \
    if (!(cond)) return ::fa::fail(FA_ERR_INVALID_ARGUMENT, __VA_ARGS__); \
  } while (0)

#define FA_LAUNCH(expr)                                                                              \
  do {                                                                                               \
    hipError_t e_ = (expr);                                                                          \
    if (e_ != hipSuccess) return ::fa::fail(FA_ERR_LAUNCH, "%s failed: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

inline size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// strides are in elements: multiples of 8 (16-byte vectors), non-negative, and below 2^24 so that the kernels' 32-bit
// per-lane byte offsets inside a tile (up to 63 rows) cannot overflow
inline bool stride_ok(int64_t s) { return s % 8 == 0 && s >= 0 && s < ((int64_t)1 << 24); }

}  // namespace fa
