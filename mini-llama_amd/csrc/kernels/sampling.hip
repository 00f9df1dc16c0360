// A token of each row of logits, by temperature, top-k, top-p and min-p and a
// given random number (contract in include/mlq.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "paged_device.h"
#include "sampling.h"

namespace mlq {
namespace {

// Every filter keeps a first part of the tokens in the order of falling logits,
// so a row needs three places in that order: where the count reaches top_k,
// where the sum of weights reaches top_p of those, and where it passes u times
// what is kept. Sums are whole numbers, weights w = exp((l - max) / T) in units of
// 2^-44: they do not depend on the order in which they are added, so neither does
// the token, and 2^19 of them fit 64 bits. What a unit cannot hold could be asked
// for by no u, whose last step is 2^-24 of the sum.
constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr double kUnits = 17592186044416.0;  // 2^44
constexpr int kDigit = 11, kBins = 1 << kDigit;

// What counts of a logit: NaN and -inf are no candidates (-inf), inf is the
// largest finite number, -0 is 0.
__device__ __forceinline__ float candidate(float l) {
  if (!(l >= -3.402823466e38f)) return -INFINITY;
  return fminf(l, 3.402823466e38f) + 0.0f;
}
// Ascending where logits fall.
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l);
  return b & 0x80000000u ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k : ~k & 0x7fffffffu);
}

struct SampleLds {
  uint32_t count[kBins];
  uint64_t weight[kBins];
  uint64_t scan[2][kSampleWaves];
  uint64_t found[4];
};

// A place in the order: the key there, how many tokens and units lie before the
// first with it, how many have it.
struct Place {
  uint32_t key;
  uint64_t count, weight, ties;
};

struct Row {
  const float* logits;
  int vocab;
  float top;      // the largest
  double inv_t;
  __device__ __forceinline__ float at(int i) const { return candidate(logits[i]); }
  __device__ __forceinline__ double weight(float l) const { return exp(((double)l - (double)top) * inv_t); }
  __device__ __forceinline__ uint64_t units(float l) const { return (uint64_t)(weight(l) * kUnits + 0.5); }
};

// Sums over the workgroup, in every thread.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* lds) {
  const uint64_t s = (uint64_t)readlane64(wave_scan64((int64_t)v), 63);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  uint64_t all = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) all += lds[w];
  return all;
}

// Where the count (BY_COUNT) or the units first reach `target`, at least 1 and
// at most all there are: by histograms of the key's digits, from the first.
template <bool BY_COUNT>
__device__ Place find(const Row& r, SampleLds& lds, uint64_t target) {
  const int tid = threadIdx.x, wave = tid >> 6;
  Place p = {0, 0, 0, 0};
  int shift = 32;
  while (shift > 0) {
    const int bits = shift > kDigit ? kDigit : shift, low = shift - bits;
    for (int i = tid; i < kBins; i += kSampleThreads) {
      lds.count[i] = 0;
      lds.weight[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < r.vocab; i += kSampleThreads) {
      const float l = r.at(i);
      const uint32_t k = key_of(l);
      if (l == -INFINITY || (shift < 32 && k >> shift != p.key)) continue;
      const uint32_t bin = k >> low & ((1u << bits) - 1);
      atomicAdd(&lds.count[bin], 1u);
      atomicAdd((unsigned long long*)&lds.weight[bin], (unsigned long long)r.units(l));
    }
    __syncthreads();
    // two bins a thread
    uint64_t c[2], w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      c[j] = lds.count[2 * tid + j];
      w[j] = lds.weight[2 * tid + j];
    }
    uint64_t ce = (uint64_t)wave_scan64((int64_t)(c[0] + c[1])), we = (uint64_t)wave_scan64((int64_t)(w[0] + w[1]));
    if ((tid & 63) == 63) {
      lds.scan[0][wave] = ce;
      lds.scan[1][wave] = we;
    }
    __syncthreads();
    for (int v = 0; v < wave; ++v) {
      ce += lds.scan[0][v];
      we += lds.scan[1][v];
    }
    uint64_t c0 = p.count + ce - c[0] - c[1], w0 = p.weight + we - w[0] - w[1];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t before = BY_COUNT ? c0 : w0, here = BY_COUNT ? c[j] : w[j];
      if (before < target && target <= before + here) {
        lds.found[0] = 2 * tid + j;
        lds.found[1] = c0;
        lds.found[2] = w0;
        lds.found[3] = c[j];
      }
      c0 += c[j];
      w0 += w[j];
    }
    __syncthreads();
    p = {(shift < 32 ? p.key << bits : 0u) | (uint32_t)lds.found[0], lds.found[1], lds.found[2], lds.found[3]};
    __syncthreads();
    shift = low;
  }
  return p;
}

// The n-th (from 0) index with the key, in every thread.
__device__ int index_of(const Row& r, SampleLds& lds, uint32_t key, uint64_t n) {
  const int tid = threadIdx.x, wave = tid >> 6;
  uint64_t before = 0;
  for (int i0 = 0; i0 < r.vocab; i0 += kSampleThreads) {
    const int i = i0 + tid;
    const float l = i < r.vocab ? r.at(i) : -INFINITY;
    const uint64_t has = __ballot(l != -INFINITY && key_of(l) == key);
    __syncthreads();
    if ((tid & 63) == 0) lds.scan[0][wave] = __builtin_popcountll(has);
    __syncthreads();
    uint64_t mine = before, all = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
      if (w < wave) mine += lds.scan[0][w];
      all += lds.scan[0][w];
    }
    if (before + all > n) {
      const uint64_t lower = has & ((1ull << (tid & 63)) - 1);
      if ((has >> (tid & 63) & 1) != 0 && mine + __builtin_popcountll(lower) == n) lds.found[0] = i;
      __syncthreads();
      return (int)lds.found[0];
    }
    before += all;
  }
  return -1;
}

__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleLds lds;
  const int row = blockIdx.x, tid = threadIdx.x;
  Row r = {a.logits + row * a.stride, a.vocab, -INFINITY, 1.0};

  // ---- the largest logit, the first that is
  float top = -INFINITY;
  int at = 0x7fffffff;
  for (int i = tid; i < a.vocab; i += kSampleThreads) {
    const float l = r.at(i);
    if (l > top) {
      top = l;
      at = i;
    }
  }
  {
    const float best = wave_max(top);
    uint32_t first = top == best ? (uint32_t)at : 0x7fffffffu;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) first = min(first, (uint32_t)__shfl_xor((int)first, d));
    // (the largest first by its key, then the smallest index)
    if ((tid & 63) == 0) lds.scan[0][tid >> 6] = (uint64_t)(best == -INFINITY ? 0xffffffffu : key_of(best)) << 32 | first;
    __syncthreads();
    uint64_t least = ~0ull;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) least = min(least, lds.scan[0][w]);
    __syncthreads();
    at = (int)(uint32_t)least;
    top = (uint32_t)(least >> 32) == 0xffffffffu ? -INFINITY : of_key((uint32_t)(least >> 32));
  }
  const float t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  const int k = a.top_k != nullptr ? a.top_k[row] : 0;
  const float p = a.top_p != nullptr ? a.top_p[row] : 1.0f, least_p = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  if (top == -INFINITY || !(t > 0.0f) || k == 1) {
    if (tid == 0) a.tokens[row] = top == -INFINITY ? -1 : at;
    return;
  }
  r.top = top;
  r.inv_t = 1.0 / (double)t;

  // ---- all candidates, and those that min_p leaves
  uint64_t count = 0, units = 0, n_m = 0, w_m = 0;
  for (int i = tid; i < a.vocab; i += kSampleThreads) {
    const float l = r.at(i);
    if (l == -INFINITY) continue;
    const double w = r.weight(l);
    const uint64_t x = (uint64_t)(w * kUnits + 0.5);
    ++count;
    units += x;
    if (!(least_p > 0.0f) || w >= (double)least_p) {
      ++n_m;
      w_m += x;
    }
  }
  count = block_sum(count, lds.scan[0]);
  units = block_sum(units, lds.scan[0]);
  n_m = block_sum(n_m, lds.scan[0]);
  w_m = block_sum(w_m, lds.scan[0]);
  if (n_m == 0) {  // (the first always stays)
    n_m = 1;
    w_m = (uint64_t)kUnits;
  }
  // ---- how many stay, and their units
  uint64_t n = count, kept = units;
  if (k > 0 && (uint64_t)k < count) {
    const Place c = find<true>(r, lds, k);
    n = k;
    kept = c.weight + (n - c.count) * r.units(of_key(c.key));
  }
  if (p < 1.0f) {
    const double need = (double)p * (double)kept;
    const uint64_t target = need > 1.0 ? min((uint64_t)ceil(need), kept) : 1;
    const Place c = find<false>(r, lds, target);
    const uint64_t x = r.units(of_key(c.key)), ties = (target - c.weight + x - 1) / x;
    n = c.count + ties;
    kept = c.weight + ties * x;
  }
  if (n_m < n) kept = w_m;
  // ---- the first whose sum passes u of them
  const float u = a.uniform[row];
  const double past = u > 0.0f ? (double)u * (double)kept : 0.0;
  const uint64_t target = past < (double)kept ? min((uint64_t)past + 1, kept) : kept;
  const Place c = find<false>(r, lds, target);
  const int token = index_of(r, lds, c.key, (target - c.weight - 1) / r.units(of_key(c.key)));
  if (tid == 0) a.tokens[row] = token;
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(sample_kernel, dim3(a.rows), dim3(kSampleThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mlq
