// Rows of a paged cache of 4 or 8 bits (MLQ_KV_Q4, MLQ_KV_Q8): a head's elements
// in blocks of 32, x = d (c - z) + m with d and m in fp16 and codes c of 0 .. L
// (q4: L = 15, z = 8; q8: L = 255, z = 128). m lies in the middle of the block's
// range, not at its end: d (c - z) and m are then both about as large as x, and
// sums over them lose no more to cancellation than sums over x.
//
// A row holds NB = 2, 4 or 8 blocks (head dims up to 64, 128, 256; what lies
// behind the head's end has code z, blocks of nothing else d = m = 0): unit
// i * NB + b (i < 16) holds dims 2i and 2i + 1 of block b, a byte (q4, the lower
// dim in its low half) or two (q8), behind the units d and m of each block. So
// lane i of 16 has two dims of every block side by side, which is what both
// products of the attention kernels take from a row: the scores a key's dims
// 8 q .. 8 q + 7 of every block (16 NB / 4 units in a run), the output two dims
// of every block of several keys.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "mlq.h"

namespace mlq {

constexpr __host__ __device__ bool kv_quantised(int type) { return type == MLQ_KV_Q4 || type == MLQ_KV_Q8; }
constexpr __host__ __device__ int kv_blocks(int hd) { return hd <= 64 ? 2 : hd <= 128 ? 4 : 8; }
constexpr __host__ __device__ int kv_row_bytes(int type, int hd) {
  return type == MLQ_KV_Q4 ? 20 * kv_blocks(hd) : type == MLQ_KV_Q8 ? 36 * kv_blocks(hd) : type == MLQ_KV_F32 ? 4 * hd : 2 * hd;
}

struct KvQ4 {
  static constexpr int kType = MLQ_KV_Q4, kLevels = 15, kMiddle = 8, kUnit = 1;
};
struct KvQ8 {
  static constexpr int kType = MLQ_KV_Q8, kLevels = 255, kMiddle = 128, kUnit = 2;
};

// d and m of a block.
struct KvScale {
  _Float16 d, m;
};

// A rounding of its own: the compiler makes one of a sum's to fp32 and its result's
// to fp16 (an instruction that gives fp16 right away), which is off at fp16's ties.
__device__ __forceinline__ _Float16 half_of_float(float x) {
  asm("" : "+v"(x));
  return (_Float16)x;
}

// From the block's least and largest element (-inf and inf where one is not
// finite). A range or middle that fp16 does not hold gives NaN: the whole block
// then reads as NaN.
template <typename Q>
__device__ __forceinline__ KvScale kv_scale(float lo, float hi) {
  KvScale s;
  // (the quotient as a division rounds it: true of 15 and 255 for every fp32
  // mantissa; where exponents end, fp16 has d 0 or NaN either way)
  constexpr float kInv = 1.0f / (float)Q::kLevels;
  const float q = (hi - lo) * kInv;
  s.d = half_of_float(__builtin_fmaf(__builtin_fmaf(-q, (float)Q::kLevels, hi - lo), kInv, q));
  s.m = half_of_float(lo + (float)Q::kMiddle * (float)s.d);
  const float all = (float)s.d * 0.0f + (float)s.m * 0.0f;
  if (!(all == 0.0f)) s.d = s.m = __builtin_bit_cast(_Float16, (uint16_t)0x7e00);
  return s;
}

// The code of x: the nearest of d (c - z) + m, upwards from halfway. Decided
// exactly: fp32 gives it but for a neighbour, and whether x is past that one's
// border is asked in 64 bits, which hold the border (multiples of 2^-25 below
// 2^25) where they do not hold x - m of a tiny x.
// inv: 1 / d to a few units in its last place.
template <typename Q>
__device__ __forceinline__ int kv_code(float x, KvScale s, float inv) {
  constexpr float kLo = -(float)Q::kMiddle, kHi = (float)(Q::kLevels - Q::kMiddle);
  const float d = (float)s.d, m = (float)s.m;
  if (!(d > 0.0f)) return Q::kMiddle;
  float c = floorf(__builtin_fmaf(x - m, inv, 0.5f));
  c = fminf(fmaxf(c, kLo), kHi);
  if ((double)x >= __builtin_fma((double)c + 0.5, (double)d, (double)m)) c += 1.0f;
  else if ((double)x < __builtin_fma((double)c - 0.5, (double)d, (double)m)) c -= 1.0f;
  return (int)fminf(fmaxf(c, kLo), kHi) + Q::kMiddle;
}

// One rounding, of the sum: d (c - z) has at most 19 bits.
template <typename Q>
__device__ __forceinline__ float kv_value(int code, KvScale s) {
  return __builtin_fmaf((float)s.d, (float)(code - Q::kMiddle), (float)s.m);
}

// What an element adds to its block's range: itself, or everything if it is not
// finite (so that fminf and fmaxf, which pass over NaN, cannot lose it).
__device__ __forceinline__ void kv_range(float x, float& lo, float& hi) {
  const bool finite = fabsf(x) <= 3.402823466e38f;
  lo = fminf(lo, finite ? x : -INFINITY);
  hi = fmaxf(hi, finite ? x : INFINITY);
}

}  // namespace mlq
