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
// the token, and 2^19 of them fit 64 bits. Half a unit is rounded off each weight, and
// where the parts' sums are brought together off each bin of each part: sums are off
// by up to (vocab + 2^14) 2^-45 where the largest weight is 1, of 2^19 tokens by 2^-26
// (a quarter of the last step of u before 1), and by 64 bits' roundings.
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

// The value of the lane J away (a power of two).
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t x) {
  if constexpr (J == 1) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppXor1, 0xF, 0xF, false);
  if constexpr (J == 2) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppXor2, 0xF, 0xF, false);
  if constexpr (J == 4)  // (7 away, then 3)
    return (uint32_t)__builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)x, kDppHalfMirror, 0xF, 0xF, false), 0x1B, 0xF, 0xF, false);
  if constexpr (J == 8) return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, kDppRor8, 0xF, 0xF, false);
  if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return threadIdx.x & 16 ? (uint32_t)r[0] : (uint32_t)r[1];
  }
  if constexpr (J == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return threadIdx.x & 32 ? (uint32_t)r[0] : (uint32_t)r[1];
  }
}
// f(l, i) for the candidates l at lo <= i < hi, by the whole workgroup, several
// loads at a time.
template <int THREADS, typename F>
__device__ __forceinline__ void for_each(const float* logits, int lo, int hi, F f) {
  typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int kStep = 4 * THREADS, kAhead = 4;
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
    for_each<kSampleThreads>(r.logits, 0, r.vocab, [&](float l, int) __attribute__((always_inline)) {
      const uint32_t k = key_of(l);
      if (l == -INFINITY || (shift < 32 && k >> shift != p.key)) return;
      const uint32_t bin = k >> low & ((1u << bits) - 1);
      const uint64_t x = r.units(l), who = __ballot(true);
      // (a row is here for its equal logits: a wave's go with one atomic, not 64 in
      // turn; 152064 equal ones with top-k and top-p 2.4 -> 0.8 ms, loads ahead among it)
      const int lead = __builtin_ctzll(who);
      if (__ballot(k != (uint32_t)__builtin_amdgcn_readlane((int)k, lead)) == 0) {
        if ((tid & 63) == lead) {
          const int n = __builtin_popcountll(who);
          atomicAdd(&lds.count[bin], (uint32_t)n);
          atomicAdd((unsigned long long*)&lds.weight[bin], (unsigned long long)(n * x));
        }
      } else {
        atomicAdd(&lds.count[bin], 1u);
        atomicAdd((unsigned long long*)&lds.weight[bin], (unsigned long long)x);
      }
    });
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
  constexpr int kAhead = 8;
  for (int i0 = 0; i0 < r.vocab; i0 += kAhead * kSampleThreads) {
    float l[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) l[j] = r.at(min(i0 + j * kSampleThreads + tid, r.vocab - 1));
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = i0 + j * kSampleThreads + tid;
      const uint64_t has = __ballot(i < r.vocab && l[j] != -INFINITY && key_of(l[j]) == key);
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
  }
  return -1;
}

// What of a row is asked for.
constexpr int kLightK = 1024;
struct Ask {
  float t, p, least, u;
  int k;
  bool greedy;
  // few enough are kept that no weight of others is asked for; tokens are counted
  __device__ __forceinline__ bool light() const { return k > 0 && k <= kLightK; }
  __device__ __forceinline__ bool counts() const { return k > 0; }
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

// The largest of what the threads have and the first index with it, as the key
// and the index in one number; no candidates: all ones.
template <int J>
__device__ __forceinline__ uint64_t wave_least(uint64_t x) {
  x = min(x, (uint64_t)lane_xor<J>((uint32_t)(x >> 32)) << 32 | lane_xor<J>((uint32_t)x));
  if constexpr (J > 1) return wave_least<J / 2>(x);
  return x;
}
__device__ __forceinline__ uint64_t first_of_wave(float top, int at) {
  return wave_least<32>(top == -INFINITY ? ~0ull : (uint64_t)key_of(top) << 32 | (uint32_t)at);
}
// (in every thread of the workgroup)
__device__ __forceinline__ uint64_t first_of(float top, int at, uint64_t* lds) {
  const uint64_t mine = first_of_wave(top, at);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = mine;
  __syncthreads();
  uint64_t least = ~0ull;
#pragma unroll
  for (int w = 0; w < kSampleWaves; ++w) least = min(least, lds[w]);
  return least;
}
// Calls `all` with the f that goes over the candidates of a range: up to QUADS of
// four a thread are asked for at once and stay in registers however often it is
// called.
template <int THREADS, int QUADS, typename A>
__device__ __forceinline__ void over(const float* logits, int lo, int hi, A all) {
  typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int kStep = 4 * THREADS, kHeldQuads = QUADS;
  if (hi - lo > kHeldQuads * kStep) {
    all([&](auto f) __attribute__((always_inline)) { for_each<THREADS>(logits, lo, hi, f); });
    return;
  }
  v4 x[kHeldQuads];
  const int i0 = lo + 4 * (int)threadIdx.x;
#pragma unroll
  for (int j = 0; j < kHeldQuads; ++j) {
    const int i = i0 + j * kStep;
    x[j] = v4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    if (i + 3 < hi) {
      x[j] = *(const v4*)(logits + i);
    } else if (i < hi) {
      x[j].x = logits[i];
      if (i + 1 < hi) x[j].y = logits[i + 1];
      if (i + 2 < hi) x[j].z = logits[i + 2];
    }
  }
  all([&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kHeldQuads; ++j)
      if (i0 + j * kStep < hi) {
#pragma unroll
        for (int c = 0; c < 4; ++c) f(candidate(x[j][c]), i0 + j * kStep + c);
      }
  });
}

// A row by itself, whatever its logits: everything by histograms of the whole
// row. Other than greedily; `top` is the row's largest logit.
__device__ int sample_row(const SampleArgs& a, int row, const Ask& s, float top, SampleLds& lds) {
  const Row r = {a.logits + row * a.stride, a.vocab, top, 1.0 / (double)s.t};
  // ---- all candidates, and those that min_p leaves
  uint64_t count = 0, units = 0, n_m = 0, w_m = 0;
  for_each<kSampleThreads>(r.logits, 0, a.vocab, [&](float l, int) __attribute__((always_inline)) {
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
// Of the histograms' kernel: two workgroups a CU, one's loads beside the other's
// exponentials (64 rows of 152064 logits: 80.0 us, 83.3 with 1024 threads, 85.7 with 256).
constexpr int kPartThreads = 512, kPartWaves = kPartThreads / 64;
// Of four logits that a thread of it holds; longer parts are read again for each
// pass, out of the caches. 48 rows of 152064 logits, 15208 a part, 62.7 us, read again
// 64.4; 65 rows, 21724 a part, 83.8, held (11) 83.2, and beyond that the same.
constexpr int kPartQuads = 10;
constexpr int kGrid = 1024;     // bins, the last of them everything behind the others
constexpr int kListed = 4096;
constexpr int kDirect = kSampleThreads;  // a row is its own list
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
  int32_t m_bin;    // the first bin that min_p may cut; kGrid: none
  uint32_t pad;
};
struct PartsView {
  PartHead* head;      // [rows][parts]
  uint32_t* count;     // [rows][parts][kGrid]
  uint64_t* units;     // [rows][parts][kGrid]
  RowState* state;     // [rows]
  uint64_t* before_w;  // [rows][kGrid + 1] units before each bin
  uint32_t* before_c;  // [rows][kGrid + 1] tokens
  uint64_t* list;      // [rows][kListed] key and index
};
__host__ __device__ inline size_t parts_align(size_t n) { return (n + 255) & ~(size_t)255; }
// (slots: parts of all rows)
__host__ __device__ inline size_t parts_view(void* ws, int rows, int slots, PartsView* v) {
  size_t at = 0;
  auto take = [&](auto** p, size_t n) {
    typedef typename std::remove_reference<decltype(**p)>::type X;
    *p = (X*)((char*)ws + at);
    at += parts_align(n * sizeof(X));
  };
  take(&v->head, (size_t)slots);
  take(&v->count, (size_t)slots * kGrid);
  take(&v->units, (size_t)slots * kGrid);
  take(&v->state, (size_t)rows);
  take(&v->before_w, (size_t)rows * (kGrid + 1));
  take(&v->before_c, (size_t)rows * (kGrid + 1));
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

// Logits' number, sum and sum of squares about the row's first one, kSpread of
// them a thread.
constexpr int kSpread = 1024 / kPartThreads;
struct Spread {
  float n, s, q;
  __device__ __forceinline__ Spread(const float (&l)[kSpread], float ref) {
    n = s = q = 0.0f;
#pragma unroll
    for (int i = 0; i < kSpread; ++i) {
      const float c = candidate(l[i]), x = c == -INFINITY ? 0.0f : c - (ref == -INFINITY ? 0.0f : ref);
      n += c == -INFINITY ? 0.0f : 1.0f;
      s += x;
      q += x * x;
    }
    n = wave_sum(n);
    s = wave_sum(s);
    q = wave_sum(q);
  }
};
// Bins a unit of logit from that. 32 T are e^-32, less than half a unit, and 14
// of the spread reach from the largest, 5 to 8 above the middle, far enough down.
__device__ __forceinline__ double grid_of(float n, float s, float q, float t) {
  const float var = q / n - (s / n) * (s / n);
  double span = 32.0 * (double)t;
  if (var > 0.0f && var < 1e30f) span = fmin(span, 14.0 * (double)sqrtf(var));
  return (double)(kGrid - 1) / span;
}
__device__ __forceinline__ int bin_of(float l, double top_bin, double grid) {
  return (int)fmin(top_bin - floor((double)l * grid), (double)(kGrid - 1));
}

constexpr double kLog2e = 1.44269504088896340736;

__global__ __launch_bounds__(kPartThreads, 4) void sample_parts_kernel(SampleArgs a, PartsView v, int parts, int part_len) {
  __shared__ uint64_t units[kGrid];
  __shared__ uint32_t count[kGrid];
  __shared__ uint64_t first_lds[kPartWaves];
  __shared__ float spread[kPartWaves][3];
  __shared__ uint64_t units_lds[kPartWaves];
  __shared__ uint32_t count_lds[kPartWaves];
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
  const bool leads = (tid & 63) == 0;
  const float* logits = a.logits + row * a.stride;
  const Ask s = ask_of(a, row);
  const size_t at = (size_t)row * parts + part;
  // (the same logits in every part of a row; asked for with the part's own)
  float sampled[kSpread];
#pragma unroll
  for (int i = 0; i < kSpread; ++i) sampled[i] = logits[(int)((int64_t)(kSpread * tid + i) * a.vocab / 1024)];
  const float zeroth = logits[0];
#pragma unroll
  for (int b = tid; b < kGrid; b += kPartThreads) {
    count[b] = 0;
    units[b] = 0;
  }
  if (part == 0 && tid == 0) v.state[row].listed = 0;
  over<kPartThreads, kPartQuads>(logits, part * part_len, min((part + 1) * part_len, a.vocab), [&](auto each) __attribute__((always_inline)) {
    float top = -INFINITY;
    int index = 0x7fffffff;
    each([&](float l, int i) __attribute__((always_inline)) {
      if (l > top) {
        top = l;
        index = i;
      }
    });
    uint64_t first = first_of_wave(top, index);
    const Spread sp(sampled, candidate(zeroth));
    if (leads) {
      first_lds[wave] = first;
      spread[wave][0] = sp.n;
      spread[wave][1] = sp.s;
      spread[wave][2] = sp.q;
    }
    __syncthreads();
    float n3[3] = {};
#pragma unroll
    for (int w = 0; w < kPartWaves; ++w) {
      first = min(first, first_lds[w]);
#pragma unroll
      for (int i = 0; i < 3; ++i) n3[i] += spread[w][i];
    }
    top = top_of(first);
    const double grid = s.greedy ? 0.0 : grid_of(n3[0], n3[1], n3[2], s.t);
    uint64_t all = 0;
    uint32_t n = 0;
    if (!s.greedy && top != -INFINITY) {
      const double top_bin = floor((double)top * grid), scale = kLog2e / (double)s.t;
      if (s.counts())
        each([&](float l, int) __attribute__((always_inline)) {
          if (l == -INFINITY) return;
          atomicAdd(&count[bin_of(l, top_bin, grid)], 1u);
          ++n;
        });
      if (!s.light())
        each([&](float l, int) __attribute__((always_inline)) {
          const uint64_t x = quick_units(((double)l - (double)top) * scale);
          if (x == 0) return;
          atomicAdd((unsigned long long*)&units[bin_of(l, top_bin, grid)], (unsigned long long)x);
          all += x;
        });
    }
    all = (uint64_t)readlane64(wave_scan64((int64_t)all), 63);
    n = (uint32_t)readlane64(wave_scan64((int64_t)n), 63);
    if (leads) {
      units_lds[wave] = all;
      count_lds[wave] = n;
    }
    __syncthreads();  // (and the histogram is whole)
    if (tid == 0) {
      all = n = 0;
      for (int w = 0; w < kPartWaves; ++w) {
        all += units_lds[w];
        n += count_lds[w];
      }
      v.head[at] = {first, all, grid, n, 0};
    }
  });
  if (s.greedy) return;
#pragma unroll
  for (int b = tid; b < kGrid; b += kPartThreads) {
    if (s.counts()) v.count[at * kGrid + b] = count[b];
    if (!s.light()) v.units[at * kGrid + b] = units[b];
  }
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

constexpr int kMaxParts = 16;
struct ListLds {
  uint64_t w[kGrid + 1];
  uint32_t c[kGrid + 1];
  uint64_t scan[kSampleWaves];
  int bins[8];
  uint32_t found, place;
  uint64_t list[kListed];
};

__global__ __launch_bounds__(kSampleThreads, 8) void sample_list_kernel(SampleArgs a, PartsView v, int parts, int part_len) {
  __shared__ ListLds lds;
  const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  const float* logits = a.logits + row * a.stride;
  const Ask s = ask_of(a, row);
  // (lane i of every wave has part i's)
  PartHead h = {~0ull, 0, 0.0, 0, 0};
  if ((tid & 63) < parts) h = v.head[(size_t)row * parts + (tid & 63)];
  // (what is the same in every lane lies in scalar registers: two workgroups a CU
  // have 64 others a lane; 64 rows of 152064 logits 74.9 us, with one a CU 79.8)
  auto uniform = [](double x) __attribute__((always_inline)) {
    return __builtin_bit_cast(double, (uint64_t)readlane64((int64_t)__builtin_bit_cast(uint64_t, x), 0));
  };
  const uint64_t first = (uint64_t)readlane64((int64_t)wave_least<32>(h.top), 0);
  const float top = top_of(first);
  if (part == 0 && tid == 0) v.state[row].top = first;
  if (s.greedy || top == -INFINITY) return;
  const uint64_t grid_bits = __builtin_bit_cast(uint64_t, h.grid);
  const double grid = __builtin_bit_cast(double, (uint64_t)readlane64((int64_t)grid_bits, __builtin_ctzll(__ballot(h.top == first))));
  const double top_bin = uniform(floor((double)top * grid));
  const bool light = s.light();
  // the logit of a weight of min_p (up to 1 here, and an infinite temperature makes
  // every weight 1: nothing falls below it)
  const bool m_cuts = s.least > 0.0f && s.t < INFINITY;
  const double least = m_cuts ? uniform((double)top + log((double)s.least) * (double)s.t) : 0.0;

  // ---- the parts' histograms added up, each moved to the row's largest logit
  const bool any = h.top != ~0ull;
  const float t = any ? top_of(h.top) : top;
  // bins from the row's largest logit to the part's, what a unit of the part is in the row's
  const int off_lane = any ? (int)fmin(top_bin - floor((double)t * grid), (double)kGrid) : kGrid;
  const double f_lane = light || !any ? 0.0 : exp2((((double)t - (double)top) * kLog2e) / (double)s.t);
  const uint32_t all_c = (uint32_t)readlane64(wave_scan64(any ? (int64_t)h.count : 0), 63);
  const uint64_t all_w = (uint64_t)readlane64(wave_scan64((int64_t)((double)h.units * f_lane + 0.5)), 63);
  uint64_t w = 0;
  uint32_t c = 0;
  const uint64_t* row_units = v.units + (size_t)row * parts * kGrid;
  const uint32_t* row_count = v.count + (size_t)row * parts * kGrid;
  // (loads without a condition between them are asked for together: a part that
  // is not there has the last one's, and bins that are none the first one's)
  constexpr int kAhead = 8;
  auto place = [&](int i, bool* in) __attribute__((always_inline)) {
    const int n = min(i, parts - 1), b = tid - __builtin_amdgcn_readlane(off_lane, n);
    *in = i < parts && b >= 0 && tid < kGrid - 1;
    return (uint32_t)(n * kGrid + (b >= 0 ? b : 0));
  };
  if (s.counts())
    for (int i0 = 0; i0 < parts; i0 += kAhead) {
      uint32_t x[kAhead];
      bool in[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = *(const uint32_t*)((const char*)row_count + 4 * place(i0 + i, &in[i]));
#pragma unroll
      for (int i = 0; i < kAhead; ++i) c += in[i] ? x[i] : 0;
    }
  if (!light)
    for (int i0 = 0; i0 < parts; i0 += kAhead) {
      uint64_t x[kAhead];
      bool in[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) x[i] = *(const uint64_t*)((const char*)row_units + 8 * place(i0 + i, &in[i]));
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const double f = __builtin_bit_cast(double, (uint64_t)readlane64((int64_t)__builtin_bit_cast(uint64_t, f_lane), min(i0 + i, parts - 1)));
        w += in[i] ? (uint64_t)((double)x[i] * f + 0.5) : 0;
      }
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
  int m_bin = kGrid, far = kGrid - 1;  // the last bin in question
  const bool cut = s.k > 0 && (uint32_t)s.k < all_c;
  if (light) {
    const int b = cut ? bin_by(true, s.k, 0) : kGrid - 1;
    mine = tid <= b;
    far = b;
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
    if (m_cuts) {
      // (and what its logarithm may be off by, and a logit whose weight is rounded
      // to min_p's: half a step of 64 bits is 1.1e-16 T)
      const double off = 1e-12 * (fabs((double)top) + fabs(least)) + 1e-15 * (double)s.t;
      auto bin = [&](double x) __attribute__((always_inline)) {
        return (int)fmin(fmax(top_bin - floor(x * grid), 0.0), (double)(kGrid - 1));
      };
      m_bin = bin(least + off);
      const int b1 = bin(least - off);
      mine |= tid >= m_bin && tid <= b1;
      if (tid == 0) lds.bins[5] = b1;  // (read behind the next barrier)
      lo = min(lo, max(lds.w[m_bin], (uint64_t)1));
      hi = min(hi, lds.w[b1 + 1]);
    }
    const int b0 = bin_by(false, token_target(s.u, lo), 3), b1 = bin_by(false, token_target(s.u, hi), 4);
    mine |= tid >= b0 && tid <= b1;
    far = max(max(cut ? lds.bins[0] : 0, s.p < 1.0f ? lds.bins[2] : 0), max(m_cuts ? lds.bins[5] : 0, b1));
    if (w == 0 && !(cut && tid == lds.bins[0])) mine = false;
  }
  // A place behind the grid's end, and more tokens than the list takes (where
  // they are not counted, the list says so itself).
  const bool slow = __syncthreads_or((mine && !light && tid == kGrid - 1) || (light && mine && end_c > kListed));
  if (part == 0) {
    if (tid == 0) {
      v.state[row].slow = slow;
      v.state[row].grid = grid;
      v.state[row].m_bin = m_bin;
    }
    if (!light) {
      const size_t at = (size_t)row * (kGrid + 1) + tid;
      v.before_w[at] = before_w;
      v.before_c[at] = (uint32_t)before_c;
      if (tid == kGrid - 1) {
        v.before_w[at + 1] = end_w;
        v.before_c[at + 1] = (uint32_t)end_c;
      }
    }
  }
  if (slow) return;
  // ---- their tokens
  uint32_t* flags = lds.c;
  __syncthreads();
  flags[tid] = mine;
  if (tid == 0) lds.found = 0;
  __syncthreads();
  // (most tokens lie behind the last bin in question: told from its end, and a
  // little before it, in 32 bits)
  const double end = (top_bin - far) / grid;
  const float below = far == kGrid - 1 || grid == 0.0 ? -INFINITY : (float)fmax(end - 1e-6 * fabs(end), -(double)3.402823466e38f);
  for_each<kSampleThreads>(logits, part * part_len, min((part + 1) * part_len, a.vocab), [&](float l, int i) __attribute__((always_inline)) {
    if (l < below || l == -INFINITY || flags[bin_of(l, top_bin, grid)] == 0) return;
    const uint32_t at = atomicAdd(&lds.found, 1u);
    if (at < kListed) lds.list[at] = (uint64_t)key_of(l) << 32 | (uint32_t)i;
  });
  __syncthreads();
  // (one atomic a part: a round trip of a microsecond)
  if (tid == 0) lds.place = atomicAdd(&v.state[row].listed, lds.found);
  __syncthreads();
  uint64_t* list = v.list + (size_t)row * kListed;
  for (uint32_t i = tid; i < min(lds.found, (uint32_t)kListed); i += kSampleThreads)
    if (lds.place + i < kListed) list[lds.place + i] = lds.list[i];
}

// A bitonic network's steps J, J / 2 .. 1 within the wave; `up`: ascending.
template <int J>
__device__ __forceinline__ void sort_lanes(uint64_t& x, bool up) {
  const uint64_t y = (uint64_t)lane_xor<J>((uint32_t)(x >> 32)) << 32 | lane_xor<J>((uint32_t)x);
  const bool low = (threadIdx.x & J) == 0;
  if ((y < x) == (up == low)) x = y;
  if constexpr (J > 1) sort_lanes<J / 2>(x, up);
}
// Ascending: elements tid + kSampleThreads * q of n, a power of two of 64 and
// more, by a bitonic network: lane swaps in a wave, LDS across waves. Elements
// past n are left.
template <int Q>
__device__ __forceinline__ void sort_list(uint64_t (&x)[Q], uint64_t* lds, int n) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    sort_lanes<1>(x[q], (tid & 2) == 0);
    sort_lanes<2>(x[q], (tid & 4) == 0);
    sort_lanes<4>(x[q], (tid & 8) == 0);
    sort_lanes<8>(x[q], (tid & 16) == 0);
    sort_lanes<16>(x[q], (tid & 32) == 0);
    sort_lanes<32>(x[q], ((tid + kSampleThreads * q) & 64) == 0 || n == 64);
  }
#pragma nounroll
  for (int k = 128; k <= n; k <<= 1) {
#pragma nounroll
    for (int j = k >> 1; j >= 64; j >>= 1) {
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) lds[tid + kSampleThreads * q] = x[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = tid + kSampleThreads * q;
        const uint64_t y = lds[i ^ j];
        if ((y < x[q]) == (((i & k) == 0) == ((i & j) == 0)) && i < n) x[q] = y;
      }
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = tid + kSampleThreads * q;
      if (i < n) sort_lanes<32>(x[q], (i & k) == 0);  // (whole waves)
    }
  }
}

struct TokenLds {
  union {
    SampleLds row;
    struct {
      uint64_t list[kListed];
      uint16_t from[kGrid], to[kGrid];  // of each bin in the list
    };
  };
  uint64_t scan[kSampleWaves];
  uint64_t kept[2];
  unsigned long long m_kept;
};

// The token from the list's tokens x (key and index; all ones: none), elements
// tid + kSampleThreads * q.
template <int Q, bool DIRECT>
__device__ __forceinline__ void token_of_list(const SampleArgs& a, const PartsView& v, const RowState& state, int row, const Ask& s,
                                              uint64_t (&x)[Q], TokenLds& lds) {
  const int tid = threadIdx.x;
  const float top = top_of(state.top);
  const bool light = DIRECT || s.light();
  int size = 64;
  while (size < (int)state.listed) size <<= 1;
  sort_list<Q>(x, lds.list, size);
  if (tid == 0) {
    lds.kept[0] = lds.kept[1] = 0;
    lds.m_kept = 0;
  }
  // ---- in order, Q neighbours a thread; weights and running sums
  if (Q > 1 || !light) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) lds.list[tid + kSampleThreads * q] = x[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) x[q] = lds.list[Q * tid + q];
  }
  const Row r = {a.logits, a.vocab, top, 1.0 / (double)s.t};
  double weight[Q];
  uint64_t sum[Q], less[Q], mine = 0;  // up to and with each, and before it
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    weight[q] = x[q] == ~0ull ? 0.0 : r.weight(of_key((uint32_t)(x[q] >> 32)));
    less[q] = mine;
    mine += (uint64_t)(weight[q] * kUnits + 0.5);
    sum[q] = mine;
  }
  uint64_t kept;
  const uint64_t before = block_before(mine, lds.scan, &kept);
  uint32_t rank[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    sum[q] += before;
    less[q] += before;
    rank[q] = Q * tid + q;
  }
  const size_t at = (size_t)row * (kGrid + 1);
  if constexpr (!DIRECT)
    if (!light) {
      // (before each bin what the histogram says; a bin's last token brings it to
      // the next one's)
      const double grid = state.grid, top_bin = floor((double)top * grid);
      int bin[Q];
      uint64_t w0[Q], w1[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int i = Q * tid + q;
        bin[q] = x[q] == ~0ull ? -1 : bin_of(of_key((uint32_t)(x[q] >> 32)), top_bin, grid);
        if (bin[q] < 0) continue;
        w0[q] = v.before_w[at + bin[q]];
        w1[q] = v.before_w[at + bin[q] + 1];
        // its bin begins or ends here, if its neighbours are of others
        const uint64_t prev = i > 0 ? lds.list[i - 1] : ~0ull, next = i + 1 < Q * kSampleThreads ? lds.list[i + 1] : ~0ull;
        if (prev == ~0ull || bin_of(of_key((uint32_t)(prev >> 32)), top_bin, grid) != bin[q]) lds.from[bin[q]] = (uint16_t)i;
        if (next == ~0ull || bin_of(of_key((uint32_t)(next >> 32)), top_bin, grid) != bin[q]) lds.to[bin[q]] = (uint16_t)(i + 1);
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) lds.list[Q * tid + q] = less[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (bin[q] < 0) continue;
        const int from = lds.from[bin[q]], i = Q * tid + q;
        const uint64_t p = lds.list[from];
        less[q] = min(w0[q] + less[q] - p, w1[q]);
        sum[q] = i + 1 == lds.to[bin[q]] ? w1[q] : min(w0[q] + sum[q] - p, w1[q]);
        if (s.counts()) rank[q] = v.before_c[at + bin[q]] + i - from;
      }
      kept = v.before_w[at + kGrid];
    }
  // ---- the filters, each by the units that stay: the one token at which a
  // number of them is reached says how many
  if (s.k > 0) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && rank[q] == (uint32_t)s.k - 1) lds.kept[0] = sum[q];
    __syncthreads();
    if (lds.kept[0] != 0) kept = lds.kept[0];  // (0: there are not so many)
  }
  if (s.p < 1.0f) {
    const uint64_t target = top_p_target(s.p, kept);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && less[q] < target && target <= sum[q]) lds.kept[1] = sum[q];
    __syncthreads();
    kept = lds.kept[1];
  }
  if (s.least > 0.0f) {
    uint64_t stay = light ? 0 : v.before_w[at + state.m_bin];
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (x[q] != ~0ull && weight[q] >= (double)s.least) stay = max(stay, sum[q]);
    __syncthreads();
    atomicMax(&lds.m_kept, (unsigned long long)stay);
    __syncthreads();
    kept = min(kept, (uint64_t)lds.m_kept);
  }
  const uint64_t target = token_target(s.u, kept);
#pragma unroll
  for (int q = 0; q < Q; ++q)
    if (x[q] != ~0ull && less[q] < target && target <= sum[q]) a.tokens[row] = (int32_t)(uint32_t)x[q];
}

// DIRECT: the list is the whole row, read here (vocabularies of up to kDirect. Of
// more tokens a sort of all costs more than the other two launches: 1 / 16 / 300 rows
// of 2000 take 20 / 30 / 55 us so, 17 / 29 / 47 in parts; of 1000 9 / 16 / 26).
template <bool DIRECT>
__global__ __launch_bounds__(kSampleThreads) void sample_token_kernel(SampleArgs a, PartsView v) {
  constexpr int Q = DIRECT ? 1 : kListed / kSampleThreads;
  __shared__ TokenLds lds;
  const int row = blockIdx.x, tid = threadIdx.x;
  const Ask s = ask_of(a, row);
  const float* logits = a.logits + row * a.stride;
  RowState state = {};
  uint64_t x[Q];
  if constexpr (DIRECT) {
    float top = -INFINITY;
    int index = 0x7fffffff;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = tid + kSampleThreads * q;
      const float l = i < a.vocab ? candidate(logits[i]) : -INFINITY;
      x[q] = l == -INFINITY ? ~0ull : (uint64_t)key_of(l) << 32 | (uint32_t)i;
      if (l > top) {
        top = l;
        index = i;
      }
    }
    state.top = first_of(top, index, lds.scan);
    state.listed = a.vocab;
  } else {
    state = v.state[row];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      x[q] = v.list[(size_t)row * kListed + tid + kSampleThreads * q];
      if (tid + kSampleThreads * q >= state.listed) x[q] = ~0ull;
    }
  }
  if (s.greedy || state.top == ~0ull) {
    if (tid == 0) a.tokens[row] = state.top == ~0ull ? -1 : (int32_t)(uint32_t)state.top;
    return;
  }
  if (!DIRECT && (state.slow || state.listed > kListed)) {
    const int token = sample_row(a, row, s, top_of(state.top), lds.row);
    if (tid == 0) a.tokens[row] = token;
    return;
  }
  if (Q > 1 && state.listed <= kSampleThreads) {
    uint64_t y[1] = {x[0]};
    token_of_list<1, DIRECT>(a, v, state, row, s, y, lds);
  } else {
    token_of_list<Q, DIRECT>(a, v, state, row, s, x, lds);
  }
}

int parts_of(int rows, int vocab) {
  const int most = std::max(2 * device_cus() / std::min(rows, kRowsAtOnce), 1);
  return std::min(std::min(most, kMaxParts), (vocab + kPartLeast - 1) / kPartLeast);
}
// Parts of a launch's rows, or of any smaller one's: a workspace then serves every
// smaller batch (256 rows have two parts each, 257 one).
int part_slots(int rows, int vocab) {
  const int r = std::min(rows, kRowsAtOnce);
  return std::max(std::min(r * std::min(kMaxParts, (vocab + kPartLeast - 1) / kPartLeast), 2 * device_cus()), r);
}

}  // namespace

size_t sample_workspace(int rows, int vocab) {
  if (rows == 0 || vocab <= kDirect) return 0;
  PartsView v;
  return parts_view(nullptr, std::min(rows, kRowsAtOnce), part_slots(rows, vocab), &v);
}

hipError_t launch_sample(const SampleArgs& all, void* ws, hipStream_t stream) {
  PartsView v = {};
  if (all.vocab <= kDirect) {
    hipLaunchKernelGGL(sample_token_kernel<true>, dim3(all.rows), dim3(kSampleThreads), 0, stream, all, v);
    return hipGetLastError();
  }
  const int parts = parts_of(all.rows, all.vocab);
  const int part_len = ((all.vocab + parts - 1) / parts + 3) & ~3;
  parts_view(ws, std::min(all.rows, kRowsAtOnce), part_slots(all.rows, all.vocab), &v);
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
    hipLaunchKernelGGL(sample_parts_kernel, grid, dim3(kPartThreads), 0, stream, a, v, parts, part_len);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_list_kernel, grid, dim3(kSampleThreads), 0, stream, a, v, parts, part_len);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(sample_token_kernel<false>, dim3(a.rows), dim3(kSampleThreads), 0, stream, a, v);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace mlq
