// A token of each row of logits, by temperature, top-k, top-p and min-p and a
// given random number (contract in include/mlq.h).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "launch.h"
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

// What of a row is asked for.
struct Ask {
  float t, p, least, u;
  int k;
  bool greedy;
};
__device__ __forceinline__ Ask ask_of(const SampleArgs& a, int row) {
  Ask s;
  s.t = a.temperature != nullptr ? a.temperature[row] : 1.0f;
  s.k = a.top_k != nullptr ? a.top_k[row] : 0;
  s.p = a.top_p != nullptr ? a.top_p[row] : 1.0f;
  s.least = a.min_p != nullptr ? a.min_p[row] : 0.0f;
  s.u = a.uniform[row];
  s.greedy = !(s.t > 0.0f) || s.k == 1 || s.least > 1.0f;
  return s;
}
// How many units (of `all`) have to be reached for top_p, and by the token.
__device__ __forceinline__ uint64_t top_p_target(float p, uint64_t all) {
  const double need = (double)p * (double)all;
  return need > 1.0 ? min((uint64_t)ceil(need), all) : 1;
}
__device__ __forceinline__ uint64_t token_target(float u, uint64_t all) {
  const double past = u > 0.0f ? (double)u * (double)all : 0.0;
  return past < (double)all ? min((uint64_t)past + 1, all) : all;
}

// f(l, i) for the candidates l at lo <= i < hi, by the whole workgroup, several
// loads at a time.
template <typename F>
__device__ __forceinline__ void for_each(const float* logits, int lo, int hi, F f) {
  typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int kStep = 4 * kSampleThreads, kAhead = 4;
  int i = lo + 4 * (int)threadIdx.x;
  for (; i + (kAhead - 1) * kStep + 3 < hi; i += kAhead * kStep) {
    v4 x[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x[j] = *(const v4*)(logits + i + j * kStep);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) f(candidate(x[j][c]), i + j * kStep + c);
  }
  for (; i < hi; i += kStep) {
    if (i + 3 < hi) {
      const v4 x = *(const v4*)(logits + i);
#pragma unroll
      for (int c = 0; c < 4; ++c) f(candidate(x[c]), i + c);
    } else {
      for (int c = 0; i + c < hi; ++c) f(candidate(logits[i + c]), i + c);
    }
  }
}

// The largest of a range and the first index with it, as the key and the index
// in one number, in every thread; a range without candidates: all ones.
__device__ uint64_t first_top(const float* logits, int lo, int hi, uint64_t* lds) {
  float top = -INFINITY;
  int at = 0x7fffffff;
  for_each(logits, lo, hi, [&](float l, int i) __attribute__((always_inline)) {
    if (l > top) {
      top = l;
      at = i;
    }
  });
  const float best = wave_max(top);
  uint32_t first = top == best ? (uint32_t)at : 0x7fffffffu;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) first = min(first, (uint32_t)__shfl_xor((int)first, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = best == -INFINITY ? ~0ull : (uint64_t)key_of(best) << 32 | first;
  __syncthreads();
  uint64_t least = ~0ull;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) least = min(least, lds[w]);
  return least;
}

// A row by itself, whatever its logits: everything by histograms of the whole
// row. Other than greedily; `top` is the row's largest logit.
__device__ int sample_row(const SampleArgs& a, int row, const Ask& s, float top, SampleLds& lds) {
  const Row r = {a.logits + row * a.stride, a.vocab, top, 1.0 / (double)s.t};
  // ---- all candidates, and those that min_p leaves
  uint64_t count = 0, units = 0, n_m = 0, w_m = 0;
  for_each(r.logits, 0, a.vocab, [&](float l, int) __attribute__((always_inline)) {
    if (l == -INFINITY) return;
    const double w = r.weight(l);
    const uint64_t x = (uint64_t)(w * kUnits + 0.5);
    ++count;
    units += x;
    if (!(s.least > 0.0f) || w >= (double)s.least) {
      ++n_m;
      w_m += x;
    }
  });
  count = block_sum(count, lds.scan[0]);
  units = block_sum(units, lds.scan[0]);
  n_m = block_sum(n_m, lds.scan[0]);
  w_m = block_sum(w_m, lds.scan[0]);
  // ---- how many stay, and their units
  uint64_t n = count, kept = units;
  if (s.k > 0 && (uint64_t)s.k < count) {
    const Place c = find<true>(r, lds, s.k);
    n = s.k;
    kept = c.weight + (n - c.count) * r.units(of_key(c.key));
  }
  if (s.p < 1.0f) {
    const uint64_t target = top_p_target(s.p, kept);
    const Place c = find<false>(r, lds, target);
    const uint64_t x = r.units(of_key(c.key)), ties = (target - c.weight + x - 1) / x;
    n = c.count + ties;
    kept = c.weight + ties * x;
  }
  if (n_m < n) kept = w_m;
  // ---- the first whose sum passes u of them
  const uint64_t target = token_target(s.u, kept);
  const Place c = find<false>(r, lds, target);
  return index_of(r, lds, c.key, (target - c.weight - 1) / r.units(of_key(c.key)));
}

// ---- rows in parts ---------------------------------------------------------------------
// The logits' read bounds a row: 4 bytes each, once if all goes well, a second
// time out of the caches. Three launches: parts of a row make histograms over
// bins of equal width in the logit, finer where the row is flat; from their sum every
// part learns which bins hold the three places and lists the tokens in them (a
// few hundred); one workgroup a row sorts those and finds the token. With a
// top-k of up to kLightK no weight is asked for before the end: the list is then
// everything down to the bin that holds the k-th. Where the list would be
// longer than kListed, or a place lies behind the last bin, the row is done by
// sample_row.
constexpr int kGrid = 1024;     // bins, the last of them everything behind the others
constexpr int kListed = 4096, kLightK = 1024;
constexpr int kPartLeast = 4096;
constexpr int kRowsAtOnce = 1024;
static_assert(kGrid == kSampleThreads, "a bin a thread");

struct PartHead {
  uint64_t top;    // first_top()
  uint64_t units;  // of all its candidates
  double grid;     // bins a unit of logit, the row's
  uint32_t count;
  uint32_t pad;
};
struct RowState {
  uint32_t listed;  // tokens in the list
  uint32_t slow;    // sample_row's
  uint64_t top;
  double grid;
  int32_t m_bin;    // the first bin that min_p may cut
  uint32_t pad;
};
struct PartsView {
  PartHead* head;      // [rows][parts]
  uint32_t* count;     // [rows][parts][kGrid]
  uint64_t* units;     // [rows][parts][kGrid]
  RowState* state;     // [rows]
  uint64_t* before_w;  // [rows][kGrid + 1] units before each bin
  uint32_t* before_c;  // [rows][kGrid + 1] tokens
  uint32_t* listed;    // [rows][kGrid + 1] listed ones
  uint64_t* list;      // [rows][kListed] key and index
};
__host__ __device__ inline size_t parts_align(size_t n) { return (n + 255) & ~(size_t)255; }
__host__ __device__ inline size_t parts_view(void* ws, int rows, int parts, PartsView* v) {
  size_t at = 0;
  auto take = [&](auto** p, size_t n) {
    typedef typename std::remove_reference<decltype(**p)>::type X;
    *p = (X*)((char*)ws + at);
    at += parts_align(n * sizeof(X));
  };
  take(&v->head, (size_t)rows * parts);
  take(&v->count, (size_t)rows * parts * kGrid);
  take(&v->units, (size_t)rows * parts * kGrid);
  take(&v->state, (size_t)rows);
  take(&v->before_w, (size_t)rows * (kGrid + 1));
  take(&v->before_c, (size_t)rows * (kGrid + 1));
  take(&v->listed, (size_t)rows * (kGrid + 1));
  take(&v->list, (size_t)rows * kListed);
  return at;
}

__device__ __forceinline__ float top_of(uint64_t first) { return first == ~0ull ? -INFINITY : of_key((uint32_t)(first >> 32)); }

// 2^x for -64 < x <= 0 to 2^-50: 2^n times e^f, |f| <= ln 2 / 2, by its series.
__device__ __forceinline__ double exp2_units(double x) {
  const double n = rint(x), f = (x - n) * 0.693147180559945309417;
  double s = 1.0 / 479001600;
  s = __builtin_fma(s, f, 1.0 / 39916800);
  s = __builtin_fma(s, f, 1.0 / 3628800);
  s = __builtin_fma(s, f, 1.0 / 362880);
  s = __builtin_fma(s, f, 1.0 / 40320);
  s = __builtin_fma(s, f, 1.0 / 5040);
  s = __builtin_fma(s, f, 1.0 / 720);
  s = __builtin_fma(s, f, 1.0 / 120);
  s = __builtin_fma(s, f, 1.0 / 24);
  s = __builtin_fma(s, f, 1.0 / 6);
  s = __builtin_fma(s, f, 0.5);
  s = __builtin_fma(s, f, 1.0);
  s = __builtin_fma(s, f, 1.0);
  return __builtin_amdgcn_ldexp(s, (int)n);
}
// The same weights as Row::units, to a unit: 0 where less than half of one.
__device__ __forceinline__ uint64_t quick_units(double y) {  // y = (l - top) log2 e / T
  if (!(y > -46.0)) return 0;
  // (2^44 w + 2^52 has the rounded units as its last bits)
  const double w = __builtin_fma(exp2_units(y), kUnits, 4503599627370496.0);
  return __builtin_bit_cast(uint64_t, w) & ((1ull << 52) - 1);
}

// Bins a unit of logit, for a whole row the same in all its parts: from the
// spread of a thousand of its logits. 32 T are e^-32, less than half a unit.
__device__ double grid_of(const float* logits, int vocab, float t, float* lds) {
  const int tid = threadIdx.x;
  const float l = candidate(logits[(int)((int64_t)tid * vocab / kSampleThreads)]), ref = candidate(logits[0]);
  const float x = l == -INFINITY ? 0.0f : l - (ref == -INFINITY ? 0.0f : ref);
  const float n = wave_sum(l == -INFINITY ? 0.0f : 1.0f), s = wave_sum(x), q = wave_sum(x * x);
  __syncthreads();
  if ((tid & 63) == 0) {
    lds[3 * (tid >> 6)] = n;
    lds[3 * (tid >> 6) + 1] = s;
    lds[3 * (tid >> 6) + 2] = q;
  }
  __syncthreads();
  float an = 0.0f, as = 0.0f, aq = 0.0f;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    an += lds[3 * w];
    as += lds[3 * w + 1];
    aq += lds[3 * w + 2];
  }
  const float var = aq / an - (as / an) * (as / an);
  double span = 32.0 * (double)t;
  // (14 of the spread: the largest lies 5 to 8 above the middle)
  if (var > 0.0f && var < 1e30f) span = fmin(span, 14.0 * (double)sqrtf(var));
  return (double)(kGrid - 1) / span;
}
__device__ __forceinline__ int bin_of(float l, double top_bin, double grid) {
  return (int)fmin(top_bin - floor((double)l * grid), (double)(kGrid - 1));
}

constexpr double kLog2e = 1.44269504088896340736;

__global__ __launch_bounds__(kSampleThreads) void sample_parts_kernel(SampleArgs a, PartsView v, int parts, int part_len) {
  __shared__ uint64_t units[kGrid];
  __shared__ uint32_t count[kGrid];
  __shared__ uint64_t scan[kSampleWaves];
  __shared__ float stats[3 * kSampleWaves];
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const float* logits = a.logits + row * a.stride;
  const int lo = part * part_len, hi = min(lo + part_len, a.vocab);
  const Ask s = ask_of(a, row);
  const size_t at = (size_t)row * parts + part;
  count[tid] = 0;
  units[tid] = 0;
  const uint64_t first = first_top(logits, lo, hi, scan);
  const float top = top_of(first);
  if (part == 0 && tid == 0) v.state[row].listed = 0;
  if (s.greedy || top == -INFINITY) {
    if (tid == 0) v.head[at] = {first, 0, 0.0, 0, 0};
    if (s.greedy) return;
  } else {
    const double grid = grid_of(logits, a.vocab, s.t, stats), top_bin = floor((double)top * grid);
    const double scale = kLog2e / (double)s.t;
    const bool light = s.k > 0 && s.k <= kLightK;
    uint64_t all = 0;
    uint32_t n = 0;
    for_each(logits, lo, hi, [&](float l, int) __attribute__((always_inline)) {
      if (l == -INFINITY) return;
      const int b = bin_of(l, top_bin, grid);
      atomicAdd(&count[b], 1u);
      ++n;
      if (light) return;
      const uint64_t x = quick_units(((double)l - (double)top) * scale);
      if (x == 0) return;
      atomicAdd((unsigned long long*)&units[b], (unsigned long long)x);
      all += x;
    });
    all = block_sum(all, scan);  // (its barriers are the histogram's, too)
    n = (uint32_t)block_sum(n, scan);
    if (tid == 0) v.head[at] = {first, all, grid, n, 0};
  }
  __syncthreads();
  v.count[at * kGrid + tid] = count[tid];
  v.units[at * kGrid + tid] = units[tid];
}

// Exclusive prefix sums over the workgroup.
__device__ __forceinline__ uint64_t block_before(uint64_t x, uint64_t* lds, uint64_t* all) {
  const int wave = threadIdx.x >> 6;
  const uint64_t end = (uint64_t)wave_scan64((int64_t)x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) lds[wave] = end;
  __syncthreads();
  uint64_t before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) {
    if (w < wave) before += lds[w];
    sum += lds[w];
  }
  *all = sum;
  return before + end - x;
}

struct ListLds {
  uint64_t w[kGrid + 1];
  uint32_t c[kGrid + 1];
  uint64_t scan[kSampleWaves];
  int bins[8];
};

__global__ __launch_bounds__(kSampleThreads) void sample_list_kernel(SampleArgs a, PartsView v, int parts, int part_len) {
  __shared__ ListLds lds;
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const float* logits = a.logits + row * a.stride;
  const Ask s = ask_of(a, row);
  uint64_t first = ~0ull;
  double grid = 0.0;
  for (int i = 0; i < parts; ++i) {
    const PartHead h = v.head[(size_t)row * parts + i];
    if (h.top < first) {
      first = h.top;
      grid = h.grid;
    }
  }
  const float top = top_of(first);
  if (part == 0 && tid == 0) v.state[row].top = first;
  if (s.greedy || top == -INFINITY) return;
  const double top_bin = floor((double)top * grid);
  const bool light = s.k > 0 && s.k <= kLightK;

  // ---- the parts' histograms added up, each moved to the row's largest logit
  uint64_t w = 0, all_w = 0;
  uint32_t c = 0, all_c = 0;
  for (int i = 0; i < parts; ++i) {
    const size_t at = (size_t)row * parts + i;
    const PartHead h = v.head[at];
    const float t = top_of(h.top);
    if (t == -INFINITY) continue;
    const double down = top_bin - floor((double)t * grid);
    const int off = (int)fmin(down, (double)kGrid);
    const double f = exp2((((double)t - (double)top) * kLog2e) / (double)s.t);
    if (tid >= off && tid < kGrid - 1) {
      c += v.count[at * kGrid + tid - off];
      if (!light) w += (uint64_t)((double)v.units[at * kGrid + tid - off] * f + 0.5);
    }
    all_c += h.count;
    all_w += (uint64_t)((double)h.units * f + 0.5);
  }
  uint64_t sum_w, sum_c;
  const uint64_t before_w = block_before(w, lds.scan, &sum_w), before_c = block_before(c, lds.scan, &sum_c);
  // (what is not in a bin of its own is in the last one)
  if (tid == kGrid - 1) {
    w = all_w > sum_w ? all_w - sum_w : 0;
    c = all_c - (uint32_t)sum_c;
  }
  lds.w[tid] = before_w;
  lds.c[tid] = (uint32_t)before_c;
  if (tid == kGrid - 1) {
    lds.w[kGrid] = before_w + w;
    lds.c[kGrid] = (uint32_t)before_c + c;
  }
  if (tid < 8) lds.bins[tid] = kGrid - 1;
  __syncthreads();
  const uint64_t end_w = lds.w[tid + 1], end_c = lds.c[tid + 1], total = lds.w[kGrid];
  // the bin in which a count or units are reached, in every thread
  auto bin_by = [&](bool by_count, uint64_t target, int slot) __attribute__((always_inline)) {
    const uint64_t b = by_count ? before_c : before_w, e = by_count ? end_c : end_w;
    if (b < target && target <= e) lds.bins[slot] = tid;
    __syncthreads();
    return lds.bins[slot];
  };
  // ---- the bins in question, from what the units kept are at least and at most
  bool mine = false;
  int m_bin = 0;
  const bool cut = s.k > 0 && (uint32_t)s.k < all_c;
  if (light) {
    const int b = cut ? bin_by(true, s.k, 0) : kGrid - 1;
    mine = tid <= b;
  } else {
    uint64_t lo = total, hi = total;
    if (cut) {
      const int b = bin_by(true, s.k, 0);
      mine = tid == b;
      lo = max(lds.w[b], (uint64_t)1);
      hi = lds.w[b + 1];
    }
    if (s.p < 1.0f) {
      const int b0 = bin_by(false, top_p_target(s.p, lo), 1), b1 = bin_by(false, top_p_target(s.p, hi), 2);
      mine |= tid >= b0 && tid <= b1;
      lo = max(lds.w[b0], (uint64_t)1);
      hi = lds.w[b1 + 1];
    }
    if (s.least > 0.0f) {
      // (the logit of a weight of min_p, and what its logarithm may be off by)
      const double l = (double)top + log((double)s.least) * (double)s.t, off = 1e-12 * (fabs((double)top) + fabs(l));
      auto bin = [&](double x) __attribute__((always_inline)) {
        return (int)fmin(fmax(top_bin - floor(x * grid), 0.0), (double)(kGrid - 1));
      };
      m_bin = bin(l + off);
      const int b1 = bin(l - off);
      mine |= tid >= m_bin && tid <= b1;
      lo = min(lo, max(lds.w[m_bin], (uint64_t)1));
      hi = min(hi, lds.w[b1 + 1]);
    }
    const int b0 = bin_by(false, token_target(s.u, lo), 3), b1 = bin_by(false, token_target(s.u, hi), 4);
    mine |= tid >= b0 && tid <= b1;
  }
  if (c == 0) mine = false;
  uint64_t n_listed;
  const uint64_t listed = block_before(mine ? c : 0, lds.scan, &n_listed);
  // a bin that is behind the grid's end has more in it than its place says
  const bool slow = __syncthreads_or((mine && !light && tid == kGrid - 1) || n_listed > kListed);
  if (part == 0) {
    if (tid == 0) {
      v.state[row].slow = slow;
      v.state[row].grid = grid;
      v.state[row].m_bin = m_bin;
    }
    const size_t at = (size_t)row * (kGrid + 1) + tid;
    v.before_w[at] = before_w;
    v.before_c[at] = (uint32_t)before_c;
    v.listed[at] = (uint32_t)listed;
    if (tid == kGrid - 1) {
      v.before_w[at + 1] = end_w;
      v.before_c[at + 1] = (uint32_t)end_c;
      v.listed[at + 1] = (uint32_t)n_listed;
    }
  }
  if (slow) return;
  // ---- their tokens
  __syncthreads();
  uint32_t* flags = lds.c;
  flags[tid] = mine;
  __syncthreads();
  uint64_t* list = v.list + (size_t)row * kListed;
  for_each(logits, part * part_len, min((part + 1) * part_len, a.vocab), [&](float l, int i) __attribute__((always_inline)) {
    if (l == -INFINITY || flags[bin_of(l, top_bin, grid)] == 0) return;
    const uint32_t at = atomicAdd(&v.state[row].listed, 1u);
    if (at < kListed) list[at] = (uint64_t)key_of(l) << 32 | (uint32_t)i;
  });
}

// 64-bit numbers in ascending order: elements tid + kSampleThreads * q of n (a
// power of two, n / kSampleThreads or 1 a thread; threads past n idle), by a
// bitonic network: within the wave by lane swaps, across waves through LDS.
template <int Q>
__device__ __forceinline__ void sort_list(uint64_t (&x)[Q], uint64_t* lds, int n) {
  const int tid = threadIdx.x;
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 64) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (tid + kSampleThreads * q < n) lds[tid + kSampleThreads * q] = x[q];
        __syncthreads();
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = tid + kSampleThreads * q;
        if (i >= n) continue;  // (n is a multiple of 64: whole waves)
        uint64_t y;
        if (j >= 64) y = lds[i ^ j];
        else y = (uint64_t)__shfl_xor((unsigned long long)x[q], j);
        const bool up = (i & k) == 0, low = (i & j) == 0;
        x[q] = up == low ? min(x[q], y) : max(x[q], y);
      }
    }
}

struct TokenLds {
  union {
    SampleLds row;
    uint64_t list[kListed];
  };
  uint64_t scan[kSampleWaves];
  uint64_t kept[3];
  unsigned long long count[3];
  int token;
};

// DIRECT: the list is the whole row (vocabularies of up to kListed), read here.
template <bool DIRECT>
__global__ __launch_bounds__(kSampleThreads) void sample_token_kernel(SampleArgs a, PartsView v, int parts) {
  constexpr int Q = kListed / kSampleThreads;
  __shared__ TokenLds lds;
  const int row = blockIdx.x, tid = threadIdx.x;
  const Ask s = ask_of(a, row);
  const float* logits = a.logits + row * a.stride;
  const uint64_t first = DIRECT ? first_top(logits, 0, a.vocab, lds.scan) : v.state[row].top;
  if (s.greedy || first == ~0ull) {
    if (tid == 0) a.tokens[row] = first == ~0ull ? -1 : (int32_t)(uint32_t)first;
    return;
  }
  const float top = top_of(first);
  if (!DIRECT && v.state[row].slow) {
    const int token = sample_row(a, row, s, top, lds.row);
    if (tid == 0) a.tokens[row] = token;
    return;
  }
  // ---- the list, in order
  const bool light = DIRECT || (s.k > 0 && s.k <= kLightK);
  int n = DIRECT ? a.vocab : (int)min(v.state[row].listed, (uint32_t)kListed);
  int size = 64;
  while (size < n) size <<= 1;
  uint64_t x[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const int i = tid + kSampleThreads * q;
    x[q] = ~0ull;  // (no token: behind all others)
    if (i >= n) continue;
    if constexpr (DIRECT) {
      const float l = candidate(logits[i]);
      if (l != -INFINITY) x[q] = (uint64_t)key_of(l) << 32 | (uint32_t)i;
    } else {
      x[q] = v.list[(size_t)row * kListed + i];
    }
  }
  sort_list<Q>(x, lds.list, size);
  if (tid < 3) {
    lds.count[tid] = 0;
    lds.kept[tid] = 0;
  }
  __syncthreads();
  // element order from here on: Q neighbours a thread
#pragma unroll
  for (int q = 0; q < Q; ++q) lds.list[tid + kSampleThreads * q] = x[q];
  __syncthreads();
#pragma unroll
  for (int q = 0; q < Q; ++q) x[q] = lds.list[Q * tid + q];
  // ---- weights, ranks and running sums
  const Row r = {logits, a.vocab, top, 1.0 / (double)s.t};
  double weight[Q];
  uint64_t sum[Q], mine = 0;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    weight[q] = x[q] == ~0ull ? 0.0 : r.weight(of_key((uint32_t)(x[q] >> 32)));
    mine += (uint64_t)(weight[q] * kUnits + 0.5);
    sum[q] = mine;
  }
  uint64_t all;
  const uint64_t before = block_before(mine, lds.scan, &all);
  uint32_t rank[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    rank[q] = Q * tid + q;
    sum[q] += before;
  }
  if constexpr (!DIRECT)
    if (!light) {
      // (before each bin what the histogram says; a bin's last token brings it to
      // the next one's)
      __syncthreads();
      uint64_t* sums = lds.list;
#pragma unroll
      for (int q = 0; q < Q; ++q) sums[Q * tid + q] = sum[q];
      __syncthreads();
      const double grid = v.state[row].grid, top_bin = floor((double)top * grid);
      const size_t at = (size_t)row * (kGrid + 1);
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (x[q] == ~0ull) continue;
        const int b = bin_of(of_key((uint32_t)(x[q] >> 32)), top_bin, grid);
        const uint32_t from = v.listed[at + b], to = v.listed[at + b + 1], i = rank[q];
        const uint64_t w0 = v.before_w[at + b], w1 = v.before_w[at + b + 1];
        sum[q] = i + 1 == to ? w1 : min(w0 + sum[q] - (from > 0 ? sums[from - 1] : 0), w1);
        rank[q] = v.before_c[at + b] + i - from;
      }
    }
  // ---- the filters, each by the token with which it ends
  __syncthreads();
  uint64_t count = DIRECT || light ? (uint64_t)n : v.before_c[(size_t)row * (kGrid + 1) + kGrid];
  uint64_t kept = DIRECT || light ? all : v.before_w[(size_t)row * (kGrid + 1) + kGrid];
  if (s.k > 0 && (uint64_t)s.k < count) {
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && rank[q] == (uint32_t)s.k - 1) lds.kept[0] = sum[q];
    __syncthreads();
    if (lds.kept[0] != 0) {
      count = s.k;
      kept = lds.kept[0];
    }
  }
  // the first token that reaches a number of units: one whose sum does and whose
  // predecessor's does not, the lowest rank if there are several
  auto reached = [&](uint64_t target, int slot) __attribute__((always_inline)) {
    uint32_t least = 0xffffffffu;
#pragma unroll
    for (int q = Q - 1; q >= 0; --q)
      if (x[q] != ~0ull && sum[q] >= target) least = rank[q];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = min(least, (uint32_t)__shfl_xor((int)least, d));
    __syncthreads();
    if ((tid & 63) == 0) lds.scan[tid >> 6] = least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) least = min(least, (uint32_t)lds.scan[w]);
    return least;
  };
  if (s.p < 1.0f) {
    const uint32_t last = reached(top_p_target(s.p, kept), 1);
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && rank[q] == last) lds.kept[1] = sum[q];
    __syncthreads();
    count = (uint64_t)last + 1;
    kept = lds.kept[1];
  }
  if (s.least > 0.0f) {
    uint64_t stay = 0, units = 0;
    if (!light) {
      const size_t at = (size_t)row * (kGrid + 1) + v.state[row].m_bin;
      stay = v.before_c[at];
      units = v.before_w[at];
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && weight[q] >= (double)s.least && rank[q] + 1 > stay) {
        stay = rank[q] + 1;
        units = sum[q];
      }
    atomicMax(&lds.count[2], (unsigned long long)stay);
    __syncthreads();
    if (stay == lds.count[2]) lds.kept[2] = units;
    __syncthreads();
    if (lds.count[2] < count) kept = lds.kept[2];
  }
  // ---- the token
  const uint32_t last = reached(token_target(s.u, kept), 2);
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (x[q] != ~0ull && rank[q] == last) a.tokens[row] = (int32_t)(uint32_t)x[q];
}

int parts_of(int rows, int vocab) {
  const int most = std::max(2 * device_cus() / std::min(rows, kRowsAtOnce), 1);
  return std::min(std::min(most, 16), (vocab + kPartLeast - 1) / kPartLeast);
}

}  // namespace

size_t sample_workspace(int rows, int vocab) {
  if (rows == 0 || vocab <= kListed) return 0;
  PartsView v;
  return parts_view(nullptr, std::min(rows, kRowsAtOnce), parts_of(rows, vocab), &v);
}

hipError_t launch_sample(const SampleArgs& all, void* ws, hipStream_t stream) {
  PartsView v = {};
  if (all.vocab <= kListed) {
    hipLaunchKernelGGL(sample_token_kernel<true>, dim3(all.rows), dim3(kSampleThreads), 0, stream, all, v, 1);
    return hipGetLastError();
  }
  const int parts = parts_of(all.rows, all.vocab);
  const int part_len = ((all.vocab + parts - 1) / parts + 3) & ~3;
  parts_view(ws, std::min(all.rows, kRowsAtOnce), parts, &v);
  for (int r0 = 0; r0 < all.rows; r0 += kRowsAtOnce) {
    SampleArgs a = all;
    a.rows = std::min(kRowsAtOnce, all.rows - r0);
    a.logits += r0 * a.stride;
    a.uniform += r0;
    a.tokens += r0;
    if (a.temperature != nullptr) a.temperature += r0;
    if (a.top_k != nullptr) a.top_k += r0;
    if (a.top_p != nullptr) a.top_p += r0;
    if (a.min_p != nullptr) a.min_p += r0;
    const dim3 grid(parts, a.rows);
    hipLaunchKernelGGL(sample_parts_kernel, grid, dim3(kSampleThreads), 0, stream, a, v, parts, part_len);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_list_kernel, grid, dim3(kSampleThreads), 0, stream, a, v, parts, part_len);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(sample_token_kernel<false>, dim3(a.rows), dim3(kSampleThreads), 0, stream, a, v, parts);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mlq
