// Device helpers shared by the paged-cache kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlq {

// Inclusive prefix sum over the wave: within the rows of 16 lanes by shifts
// (0x110 + n: from n lanes below, 0 where there is none), then the rows before.
template <int CTRL>
__device__ __forceinline__ int64_t dpp64(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xF, 0xF, false);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t readlane64(int64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t wave_scan64(int64_t v) {
  v += dpp64<0x111>(v);
  v += dpp64<0x112>(v);
  v += dpp64<0x114>(v);
  v += dpp64<0x118>(v);
  const int row = (threadIdx.x & 63) >> 4;
  const int64_t a = readlane64(v, 15), b = a + readlane64(v, 31), c = b + readlane64(v, 47);
  return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}

// a / b for a >= 0, b > 0, in 32 bits where they fit (a 64-bit division is a
// hundred instructions).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

}  // namespace mlq
