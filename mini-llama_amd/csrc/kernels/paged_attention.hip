// Attention over a paged key-value cache (contracts in include/mlq.h): one new
// token of each sequence (decode) and many new tokens of each (prefill).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "paged.h"
#include "paged_device.h"

namespace mlq {
namespace {

// One row of one query head by one wave, in plain fp32: a lane scores a key of
// a tile of 64 against q in LDS, then takes head dims lane, lane + 64, .. of
// the output. What the prefill kernels hand to it: rows that could see a page
// outside the cache, or that overflow the parts alone. Writes dims d0 .. d1 - 1; `lds`: kSlowFloats
// of the wave's own.
constexpr int kSlowFloats = 256 + 64 + 128;
template <typename T>
__device__ void slow_row(const PagedAttnArgs& a, int seq, int row, int pos, int head, float* lds, int d0, int d1) {
  float* qs = lds;
  float* ps = lds + 256;
  int64_t* at = (int64_t*)(lds + 320);
  const int lane = threadIdx.x & 63, kvh = head / a.group;
  auto sync = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  const int len = pos + 1;
  const float* q = a.q + row * a.q_stride + (int64_t)head * a.hd;
  sync();
  for (int d = lane; d < a.hd; d += 64) qs[d] = q[d];
  sync();
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  const float slope = a.slopes != nullptr ? a.slopes[head] : 0.0f;
  bool bad = false;
  const int first = a.window > 0 ? max(0, len - a.window) : 0;
  for (int t0 = first; t0 < len; t0 += 64) {
    const int t = t0 + lane;
    float s = -INFINITY;
    int64_t base = 0;
    if (t < len) {
      const int page = a.block_table[(size_t)seq * a.max_pages + (t >> a.page_shift)];
      if (page < 0 || page >= a.n_pages) {
        bad = true;
      } else {
        base = ((((int64_t)page * a.n_kv + kvh) << a.page_shift) + (t & ((1 << a.page_shift) - 1))) * a.hd;
        const T* k = (const T*)a.keys + base;
        s = 0.0f;
        for (int d = 0; d < a.hd; ++d) s += qs[d] * (float)k[d];
        s *= a.scale;
        if (a.softcap > 0.0f) s = a.softcap * tanhf(s / a.softcap);
        s += slope * (float)(t - pos);
      }
    }
    bad = __any(bad);
    if (bad) break;
    const float mx = fmaxf(m, wave_max(s));
    const float ref = mx == -INFINITY ? 0.0f : mx;
    const float al = expf(m - ref);
    const float p = t < len ? expf(s - ref) : 0.0f;
    l = l * al + wave_sum(p);
    m = mx;
    sync();
    ps[lane] = p;
    at[lane] = base;
    sync();
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] *= al;
    for (int i = 0; i < min(64, len - t0); ++i) {
      const T* v = (const T*)a.values + at[i];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane + 64 * j < a.hd) acc[j] += ps[i] * (float)v[lane + 64 * j];
    }
  }
  float* out = a.out + row * a.out_stride + (int64_t)head * a.hd;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j >= d0 && lane + 64 * j < d1)
      out[lane + 64 * j] = bad ? __builtin_nanf("") : len > 0 ? acc[j] / l : 0.0f;
}

// ---- decode ------------------------------------------------------------------------
// One query row of each sequence; out = softmax(rule(K q)) V with one pass over
// the keys and a running maximum. The reads of K and V bound it, so the grid
// is as many workgroups as the chip holds, each with the same number of tiles:
// the key tiles of every sequence and kv head, one behind the other, are cut
// into equal ranges (their number is only known on the device: every workgroup
// scans the lengths). A range runs over the ends of short sequences and stops
// inside long ones: what it has of those it leaves as a partial (maximum, sum,
// accumulator), at most one at either end, and a second launch joins them in
// order. Sequences are padded to four tiles, one for each wave, so the
// smallest ranges, of four tiles, hold one piece each.
//
// A wave takes tiles of kKeys keys and the up to 16 query heads of one kv head
// through two products, both with the heads as columns:
//   S^T = K Q^T   A: lane = key lane % 16, 8 (fp32: 4) dims of quarter lane / 16
//   O^T = V^T P^T A: lane = HD / 16 dims of chunk lane % 16, keys of the quarter
// K and V go from the cache to the A operands as they lie (V by byte permutes:
// 8 keys x 1 dim a register quad); the D layout of S^T (4 keys of quarter
// lane / 16, head lane % 16) is the B layout of P^T, so a tile needs no LDS and
// the maximum of a head two lane swaps. 16-bit caches multiply on 16-bit
// instructions at full precision: q and P are split into parts that add up to
// fp32's 24 bits (bf16: three of 8) or 22 (fp16: two of 11, under a power of
// two: q's largest element at 2^14, the largest weight at 2^15, so what falls
// below fp16's subnormals is 2^-39 of those), the cache's values are exact.
// fp32 caches take the fp32 instructions, whose rate is no bound here either.
constexpr int kDecWaves = 4, kDecThreads = 64 * kDecWaves;
// Ranges per CU: the workgroups that a CU holds (registers: 3, 2 and 1 waves a
// SIMD at head dims up to 64, 128 and 256), so that all run at once. us with
// another number: 64 sequences of up to 8000, 28 heads on 4 of 128, bf16, 1 / 2 /
// 4 / 8 a CU: - / 69.6 / 73.7 / 82.4 (a workgroup for each part of one sequence:
// 71.2); 20 of up to 20000, 16 on 1 of 256: 49 with 1, 64 with 2. At head dim 64
// pieces are over soon, and where a range holds two and more of them, twice the
// ranges let one workgroup's start hide behind another's work (180 of up to 2500,
// 16 heads of 64, fp32: 3 a CU 161, 6 141; 30 of up to 9000, 40 on 8: 46 and 48).
constexpr int dec_per_cu(int hd, int64_t pieces, int cus) {
  return hd <= 64 ? (pieces >= 6 * (int64_t)cus ? 6 : 3) : hd <= 128 ? 2 : 1;
}
constexpr int kDecMaxSeqs = 4096;  // sequences of a launch: their prefix sums lie in LDS

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

template <typename T>
struct KvTraits;
template <>
struct KvTraits<float> {
  static constexpr int kKeys = 16;   // of a tile
  static constexpr int kParts = 1;   // of q and of the weights
  static constexpr float kLift = 0.0f;
};
template <>
struct KvTraits<_Float16> {
  static constexpr int kKeys = 32, kParts = 2;
  static constexpr float kLift = 15.0f;  // weights are 2^15 times their size
  typedef h8_t vec;
  typedef h2_t pair;
  static __device__ __forceinline__ f4 mfma(vec a, vec b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct KvTraits<__bf16> {
  static constexpr int kKeys = 32, kParts = 3;
  static constexpr float kLift = 0.0f;
  typedef bf8 vec;
  typedef bf2 pair;
  static __device__ __forceinline__ f4 mfma(vec a, vec b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// a, b = the sum of p's parts, each rounded to nearest: two values of a vec.
template <typename T>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&p)[KvTraits<T>::kParts]) {
  f2_t x = {a, b};
#pragma unroll
  for (int i = 0; i < KvTraits<T>::kParts; ++i) {
    const auto h = __builtin_convertvector(x, typename KvTraits<T>::pair);
    p[i] = __builtin_bit_cast(uint32_t, h);
    if (i + 1 < KvTraits<T>::kParts) {
      x.x -= (float)h.x;
      x.y -= (float)h.y;
    }
  }
}

// What a row of the batch is to a kernel: its place in q and out and its
// number of keys; row < 0: no row. A length that the table or the caller's
// bound does not hold is `bad`.
struct DecodeRow {
  int row, len;
  bool bad;
};
__device__ __forceinline__ DecodeRow decode_row(const PagedAttnArgs& a, int seq) {
  DecodeRow r;
  r.row = seq;
  if (a.row_start != nullptr) {
    r.row = a.row_start[seq + 1] - 1;
    if (r.row < a.row_start[seq] || r.row >= a.max_rows) r.row = -1;
  }
  const int len = a.lengths[seq];
  r.bad = len > a.max_len;
  r.len = r.bad ? 0 : max(len, 0);
  return r;
}
__device__ __forceinline__ int first_key(const PagedAttnArgs& a, int len) {
  return a.window > 0 ? max(0, len - a.window) : 0;
}

// The softmax's input in base 2 for a product s: without cap and slopes
// s * sl2.
struct ScoreRule {
  float sl2;         // scale * log2 e, divided by the power of two that q carries
  float cap_in, cap_out;  // cap_out tanh(s * cap_in); cap_out 0: no cap
  float slope2;      // slope * log2 e
};
__device__ __forceinline__ ScoreRule score_rule(const PagedAttnArgs& a, int head, int q_exp,
                                                float scale) {
  constexpr float kLog2e = 1.44269504088896341f;
  ScoreRule r;
  r.sl2 = ldexp_f(scale * kLog2e, -q_exp);
  r.cap_in = a.softcap > 0.0f ? ldexp_f(scale / a.softcap, -q_exp) : 0.0f;
  r.cap_out = a.softcap * kLog2e;
  r.slope2 = a.slopes != nullptr ? a.slopes[head] * kLog2e : 0.0f;
  return r;
}

// The cut: range w holds tiles w * range .. of all of them; sequence i's lie
// from first[i] * n_tiles on, count[i] (a multiple of 4; 0: no row) for each of
// the n_tiles kv heads (or runs of 16 heads of one). Partials: a range's first
// and last piece, up to `tg` heads each: maxima and sums [tg], accumulators
// [tg][hd].
struct DecodePartials {
  int64_t* range;
  int* first;
  int* count;
  float* m;
  float* l;
  float* acc;
};
__host__ __device__ inline size_t dec_align(size_t b) { return (b + 255) & ~(size_t)255; }
__host__ __device__ inline size_t dec_header(int n_seqs) { return dec_align(8 + (size_t)n_seqs * 8); }
__host__ __device__ inline DecodePartials decode_partials(void* ws, int n_seqs, int ranges, int tg) {
  DecodePartials p;
  char* c = (char*)ws;
  p.range = (int64_t*)c;
  p.first = (int*)(c + 8);
  p.count = p.first + n_seqs;
  c += dec_header(n_seqs);
  p.m = (float*)c;
  p.l = p.m + (size_t)2 * ranges * tg;
  c += dec_align((size_t)2 * ranges * tg * 8);
  p.acc = (float*)c;
  return p;
}

template <typename T, int HD, bool FULL>
__global__ __launch_bounds__(kDecThreads, HD <= 128 ? 2 : 1) void paged_decode_kernel(PagedAttnArgs a) {
  using Tr = KvTraits<T>;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int KT = Tr::kKeys, NS = KT / 16;  // keys, runs of 16 keys
  constexpr int NP = Tr::kParts;
  constexpr int KS = F32 ? HD / 16 : HD / 32;  // 16-byte pieces of a K row per lane
  constexpr int VD = HD / 16;                  // dims of V (and of the output) per lane
  constexpr int VW = VD * (int)sizeof(T) / 4;  // their words
  constexpr int RD = VD < 8 ? VD : 8;          // output dims per lane merged at a time
  constexpr int OS = 16 * RD + 4;
  constexpr int kUnit = kDecWaves * KT;
  __shared__ int base[kDecMaxSeqs + 1];
  __shared__ int scan_lds[kDecWaves];
  __shared__ __align__(16) float merge[kDecWaves][16][OS];
  __shared__ float wm[kDecWaves][16], wl[kDecWaves][16];
  __shared__ int wave_bad[kDecWaves];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ai = lane & 15, ak = lane >> 4;
  const int head_tiles = (a.group + 15) / 16, n_tiles = a.n_kv * head_tiles, TG = min(a.group, 16);
  const DecodePartials pp = decode_partials(a.part, a.n_seqs, a.ranges, TG);

  // ---- the ranges
  auto tiles_of = [&](const DecodeRow& r) {
    if (r.row < 0) return 0;
    if (a.part == nullptr) return a.whole;  // a range for each, as long as the longest
    const int tiles = (r.len - (first_key(a, r.len) & ~(KT - 1)) + KT - 1) / KT;
    return max((tiles + kDecWaves - 1) / kDecWaves, 1) * kDecWaves;
  };
  const bool few = a.n_seqs <= 64;  // a sequence a lane, in every wave for itself: no barriers
  DecodeRow mine = {-1, 0, false};
  int total, my_first = 0, my_count = 0;
  if (few) {
    if (lane < a.n_seqs) mine = decode_row(a, lane);
    my_count = tiles_of(mine);
    my_first = (int)wave_scan64(my_count) - my_count;
    total = __builtin_amdgcn_readlane(my_first + my_count, 63);
  } else {
    total = 0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += kDecThreads) {
      const int i = i0 + tid;
      const int n = i < a.n_seqs ? tiles_of(decode_row(a, i)) : 0;
      const int end = (int)wave_scan64(n);
      __syncthreads();  // (an earlier round's readers are done with scan_lds)
      if (lane == 63) scan_lds[wave] = end;
      __syncthreads();
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) {
        before += w < wave ? scan_lds[w] : 0;
        all += scan_lds[w];
      }
      if (i < a.n_seqs) base[i] = total + before + end - n;
      total += all;
    }
    if (tid == 0) base[a.n_seqs] = total;
    __syncthreads();
  }
  const int64_t all = (int64_t)total * n_tiles;
  const int64_t share = (int64_t)a.ranges * kDecWaves;
  const int64_t range = a.part == nullptr ? a.whole : max(quotient(all + share - 1, share), (int64_t)1) * kDecWaves;
  if (blockIdx.x == 0 && a.part != nullptr) {
    if (tid == 0) *pp.range = range;
    for (int i = tid; i < a.n_seqs; i += kDecThreads) {
      pp.first[i] = few ? my_first : base[i];
      pp.count[i] = few ? my_count : base[i + 1] - base[i];
    }
  }
  int64_t u = blockIdx.x * range;
  const int64_t uend = min(u + range, all);
  if (u >= uend) return;
  int seq = 0, first, count;  // of the piece's sequence
  {
    const int at = (int)quotient(u, n_tiles);
    if (few) {
      seq = __builtin_ctzll(__ballot(my_first + my_count > at));
    } else {
      int hi = a.n_seqs;
      while (hi - seq > 1) {
        const int mid = (seq + hi) >> 1;
        if (base[mid] <= at) seq = mid;
        else hi = mid;
      }
      seq = __builtin_amdgcn_readfirstlane(seq);
    }
  }
  auto take = [&]() __attribute__((always_inline)) {
    first = few ? __builtin_amdgcn_readlane(my_first, seq) : __builtin_amdgcn_readfirstlane(base[seq]);
    count = few ? __builtin_amdgcn_readlane(my_count, seq) : __builtin_amdgcn_readfirstlane(base[seq + 1]) - first;
  };
  take();
  int tile = (int)quotient(u - (int64_t)first * n_tiles, count);
  int k_at = (int)(u - (int64_t)first * n_tiles - (int64_t)tile * count);

  // ---- the range's pieces
  while (true) {
  const DecodeRow dr = few ? DecodeRow{__builtin_amdgcn_readlane(mine.row, seq), __builtin_amdgcn_readlane(mine.len, seq),
                                       __builtin_amdgcn_readlane((int)mine.bad, seq) != 0}
                           : decode_row(a, seq);
  const int piece = (int)min((int64_t)(count - k_at), uend - u);
  const bool whole = piece == count;
  const int slot = 2 * (int)blockIdx.x + (k_at == 0);
  const int kvh = tile / head_tiles, g0 = (tile - kvh * head_tiles) * 16;
  const int G = min(16, a.group - g0), head0 = kvh * a.group + g0;
  const int key_begin = first_key(a, dr.len), pos = dr.len - 1;
  // tiles start at multiples of their size: a run of 16 keys lies in one page
  const int lo = (key_begin & ~(KT - 1)) + k_at * KT;
  const int hi = min((int64_t)lo + (int64_t)piece * KT, (int64_t)dr.len);

  // ---- q
  const bool has_head = ai < G;
  const float* qp = a.q + dr.row * a.q_stride + (int64_t)(head0 + (has_head ? ai : 0)) * a.hd;
  auto q_at = [&](int d) __attribute__((always_inline)) {
    return has_head && (FULL || d < a.hd) ? *(const f4*)(qp + d) : f4{0.0f, 0.0f, 0.0f, 0.0f};
  };
  f4 qf[F32 ? KS : 1];
  typedef typename std::conditional<F32, f4, bf8>::type raw8;  // (16 bytes of either)
  raw8 qv[F32 ? 1 : NP][F32 ? 1 : KS];
  int q_exp = 0;
  if constexpr (F32) {
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = q_at(16 * s + 4 * ak);
  } else {
    f4 x[KS][2];
    float big = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[s][j] = q_at(32 * s + 8 * ak + 4 * j);
        big = fmaxf(fmaxf(big, fmaxf(fabsf(x[s][j].x), fabsf(x[s][j].y))),
                    fmaxf(fabsf(x[s][j].z), fabsf(x[s][j].w)));
      }
    if constexpr (Tr::kLift != 0.0f) q_exp = pow2_scale_exp(xor32_max(xor16_max(big)));
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint32_t w[NP][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float u = x[s][j >> 1][2 * (j & 1)], v = x[s][j >> 1][2 * (j & 1) + 1];
        if constexpr (Tr::kLift != 0.0f) {
          u = ldexp_f(u, q_exp);
          v = ldexp_f(v, q_exp);
        }
        uint32_t p[NP];
        split_pair<T>(u, v, p);
#pragma unroll
        for (int i = 0; i < NP; ++i) w[i][j] = p[i];
      }
#pragma unroll
      for (int i = 0; i < NP; ++i)
        qv[i][s] = __builtin_bit_cast(raw8, u32x4_t{w[i][0], w[i][1], w[i][2], w[i][3]});
    }
  }
  const ScoreRule rule = score_rule(a, head0 + (has_head ? ai : 0), q_exp, a.scale);
  const bool plain = a.softcap <= 0.0f && a.slopes == nullptr;

  // ---- the keys
  const int mask = (1 << a.page_shift) - 1;
  bool bad = dr.bad;
  const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
  // The rows of the run of 16 keys at k, or of the nearest run that holds a key
  // which is seen: a tile may begin before the window, on a page that nobody
  // keeps any more.
  auto row_of = [&](int k) __attribute__((always_inline)) {
    const int kk = min(max(k, key_begin), pos);
    int page = __builtin_amdgcn_readfirstlane(table[kk >> a.page_shift]);
    const bool out = page < 0 || page >= a.n_pages;
    bad |= out;
    page = out ? 0 : page;
    return (((int64_t)page * a.n_kv + kvh) << a.page_shift) + (kk & mask & ~15);
  };
  u32x4_t kr[NS][KS];
  uint32_t vr[F32 ? 4 : 8][VW];
  int64_t rows[NS];
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const char* p = (const char*)a.keys + rows[u] * a.hd * sizeof(T) + (size_t)ai * a.hd * sizeof(T);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = F32 ? 16 * s + 4 * ak : 32 * s + 8 * ak;
        if (FULL || d < a.hd) kr[u][s] = __builtin_nontemporal_load((const u32x4_t*)(p + (size_t)d * sizeof(T)));
        else kr[u][s] = u32x4_t{0, 0, 0, 0};
      }
    }
  };
  // this lane's keys of quarter ak: 4 ak + r of each run
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4 * NS; ++e) {
      const char* p = (const char*)a.values +
                      (rows[e >> 2] + 4 * ak + (e & 3)) * a.hd * (int64_t)sizeof(T);
#pragma unroll
      for (int w = 0; w < VW; w += (VW < 4 ? 2 : 4)) {
        const int d = VD * ai + w * 4 / (int)sizeof(T);
        if constexpr (VW < 4) {
          const u32x2_t x = FULL || d < a.hd ? __builtin_nontemporal_load((const u32x2_t*)(p + (size_t)d * sizeof(T))) : u32x2_t{0, 0};
          vr[e][w] = x.x;
          vr[e][w + 1] = x.y;
        } else {
          const u32x4_t x = FULL || d < a.hd ? __builtin_nontemporal_load((const u32x4_t*)(p + (size_t)d * sizeof(T))) : u32x4_t{0, 0, 0, 0};
          vr[e][w] = x.x;
          vr[e][w + 1] = x.y;
          vr[e][w + 2] = x.z;
          vr[e][w + 3] = x.w;
        }
      }
    }
  };

  float m = -INFINITY, l = 0.0f;  // of head ai; l of this quarter's keys
  f4 acc[VD];                     // dims VD (4 ak + r) + c of head ai in acc[c][r]
#pragma unroll
  for (int c = 0; c < VD; ++c) acc[c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  int k0 = lo + wave * KT;
  if (k0 < hi) {
#pragma unroll
    for (int u = 0; u < NS; ++u) rows[u] = row_of(k0 + 16 * u);
    load_k();
  }
  for (; k0 < hi; k0 += kUnit) {
    load_v();
    f4 s[NS];
    if constexpr (F32) {
      // eight chains added as a tree: few roundings on the way to a score
      f4 c8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c8[i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int st = 0; st < KS; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f4& c = c8[4 * (st & 1) + i];
          c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, kr[0][st])[i], qf[st][i], c, 0, 0, 0);
        }
      s[0] = ((c8[0] + c8[1]) + (c8[2] + c8[3])) + ((c8[4] + c8[5]) + (c8[6] + c8[7]));
    } else {
#pragma unroll
      for (int u = 0; u < NS; ++u) s[u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      // the small parts first: their roundings are below the score's
#pragma unroll
      for (int i = NP - 1; i >= 0; --i)
#pragma unroll
        for (int st = 0; st < KS; ++st)
#pragma unroll
          for (int u = 0; u < NS; ++u)
            s[u] = Tr::mfma(__builtin_bit_cast(typename Tr::vec, kr[u][st]),
                            __builtin_bit_cast(typename Tr::vec, qv[i][st]), s[u]);
    }
    const bool edge = k0 < key_begin || k0 + KT > hi;
    float p[4 * NS];
    float mx = -INFINITY;
    if (plain) {
#pragma unroll
      for (int e = 0; e < 4 * NS; ++e) p[e] = s[e >> 2][e & 3] * rule.sl2;
    } else {
#pragma unroll
      for (int e = 0; e < 4 * NS; ++e) {
        float x = s[e >> 2][e & 3];
        x = a.softcap > 0.0f ? rule.cap_out * tanhf(x * rule.cap_in) : x * rule.sl2;
        p[e] = x + rule.slope2 * (float)(k0 + 16 * (e >> 2) + 4 * ak + (e & 3) - pos);
      }
    }
    if (edge) {
#pragma unroll
      for (int e = 0; e < 4 * NS; ++e) {
        const int k = k0 + 16 * (e >> 2) + 4 * ak + (e & 3);
        if (k < key_begin || k >= hi) {
          p[e] = -INFINITY;
          // (what lies there may be anything, and 0 * inf is not 0)
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[e][w] = 0;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4 * NS; ++e) mx = fmaxf(mx, p[e]);
    mx = fmaxf(m, xor32_max(xor16_max(mx)));
    const float ref = (mx == -INFINITY ? 0.0f : mx) - Tr::kLift;
    const float al = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    if (__any(al != 1.0f)) {
      l *= al;
#pragma unroll
      for (int c = 0; c < VD; ++c) acc[c] *= al;
    }
    if (plain && !edge) {
      // (scaled and shifted with one rounding)
#pragma unroll
      for (int e = 0; e < 4 * NS; ++e)
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], rule.sl2, -ref));
    } else {
#pragma unroll
      for (int e = 0; e < 4 * NS; ++e) p[e] = __builtin_amdgcn_exp2f(p[e] - ref);
    }
    if constexpr (NS == 1) l += (p[0] + p[1]) + (p[2] + p[3]);
    else l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));

    if (k0 + kUnit < hi) {
#pragma unroll
      for (int u = 0; u < NS; ++u) rows[u] = row_of(k0 + kUnit + 16 * u);
      load_k();
    }
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int c = 0; c < VD; ++c)
          acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[e][c]), p[e], acc[c], 0, 0, 0);
    } else {
      uint32_t w[NP][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t q[NP];
        split_pair<T>(p[2 * j], p[2 * j + 1], q);
#pragma unroll
        for (int i = 0; i < NP; ++i) w[i][j] = q[i];
      }
#pragma unroll
      for (int c = 0; c < VD; ++c) {
        // dim c of the eight keys: the low or the high half of a word of each
        const uint32_t sel = c & 1 ? 0x07060302u : 0x05040100u;
        u32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = __builtin_amdgcn_perm(vr[2 * j + 1][c >> 1], vr[2 * j][c >> 1], sel);
#pragma unroll
        for (int i = NP - 1; i >= 0; --i)
          acc[c] = Tr::mfma(__builtin_bit_cast(typename Tr::vec, v),
                            __builtin_bit_cast(typename Tr::vec, u32x4_t{w[i][0], w[i][1], w[i][2], w[i][3]}),
                            acc[c]);
      }
    }
  }
  l = xor32_sum(xor16_sum(l));

  // ---- the waves joined in their order
  __syncthreads();  // (the last piece's readers are done with the LDS)
  if (lane == 0) wave_bad[wave] = bad;
  if (ak == 0) {
    wm[wave][ai] = m;
    wl[wave][ai] = l;
  }
  float* out = a.out + dr.row * a.out_stride + (int64_t)head0 * a.hd;
#pragma unroll
  for (int c0 = 0; c0 < VD; c0 += RD) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < RD; c += 4)
        *(f4*)&merge[wave][ai][RD * (4 * ak + r) + c] =
            f4{acc[c0 + c][r], acc[c0 + c + 1][r], acc[c0 + c + 2][r], acc[c0 + c + 3][r]};
    __syncthreads();
    for (int e = tid; e < G * 16 * RD; e += kDecThreads) {
      const int g = e / (16 * RD), x = e % (16 * RD);
      const int d = VD * (x / RD) + c0 + x % RD;
      if (!FULL && d >= a.hd) continue;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) mx = fmaxf(mx, wm[w][g]);
      float sum = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWaves; ++w) {
        // (a wave without keys holds zeros)
        const float f = wm[w][g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[w][g] - mx);
        sum += wl[w][g] * f;
        o += merge[w][g][x] * f;
      }
      const bool any_bad = (wave_bad[0] | wave_bad[1] | wave_bad[2] | wave_bad[3]) != 0;
      if (any_bad) sum = __builtin_nanf("");
      if (whole) {
        out[(int64_t)g * a.hd + d] = dr.len > 0 || any_bad ? o / sum : 0.0f;
      } else {
        const size_t at = (size_t)slot * TG + g;
        if (d == 0) {
          pp.m[at] = mx;
          pp.l[at] = sum;
        }
        pp.acc[at * a.hd + d] = o;
      }
    }
  }
  u += piece;
  if (u >= uend) return;
  k_at = 0;
  if (++tile == n_tiles) {
    tile = 0;
    if (few) seq = __builtin_ctzll(__ballot(my_count > 0) & ~((2ull << seq) - 1));
    else
      do ++seq;
      while (base[seq + 1] == base[seq]);
    take();
  }
  }
}

// The pieces of a sequence joined for one query head: wave w takes pieces
// 4 i + w, kJoin at a time with every load asked for at once (places past the
// last piece read the last one and weigh 0), then the waves are joined in
// order. KD: head dims per lane.
constexpr int kJoin = 4;
template <int KD>
__global__ __launch_bounds__(kDecThreads) void paged_combine_kernel(PagedAttnArgs a) {
  __shared__ float wm[kDecWaves], wl[kDecWaves], wo[kDecWaves][64 * KD];
  const int seq = blockIdx.x, head = blockIdx.y;
  const int TG = min(a.group, 16), head_tiles = (a.group + 15) / 16, n_tiles = a.n_kv * head_tiles;
  const DecodePartials pp = decode_partials(a.part, a.n_seqs, a.ranges, TG);
  const int count = pp.count[seq], first_tile = pp.first[seq];
  const int64_t range = *pp.range;
  if (count <= 0) return;
  const int kvh = head / a.group, g = head - kvh * a.group;
  const int tile = kvh * head_tiles + g / 16;
  const int64_t start = (int64_t)first_tile * n_tiles + (int64_t)tile * count;
  const int w0 = (int)quotient(start, range), parts = (int)quotient(start + count - 1, range) - w0 + 1;
  if (parts <= 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = -INFINITY, l = 0.0f, acc[KD] = {};
  for (int p0 = wave; p0 < parts; p0 += kDecWaves * kJoin) {
    float pm[kJoin], pl[kJoin], pa[kJoin][KD];
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      const int w = w0 + min(p0 + kDecWaves * i, parts - 1);
      // (the sequence begins in its first range: that range's last piece)
      const size_t at = (size_t)(2 * w + (w == w0)) * TG + g % 16;
      pm[i] = pp.m[at];
      pl[i] = pp.l[at];
#pragma unroll
      for (int j = 0; j < KD; ++j) pa[i][j] = pp.acc[at * a.hd + min(lane + 64 * j, a.hd - 1)];
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      if (p0 + kDecWaves * i >= parts) pm[i] = -INFINITY;
      mx = fmaxf(mx, pm[i]);
    }
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    l *= f;
#pragma unroll
    for (int j = 0; j < KD; ++j) acc[j] *= f;
#pragma unroll
    for (int i = 0; i < kJoin; ++i) {
      if (p0 + kDecWaves * i >= parts) break;  // (a part past the last, NaN or not, stays out)
      const float w = pm[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[i] - mx);
      l += pl[i] * w;
#pragma unroll
      for (int j = 0; j < KD; ++j) acc[j] += pa[i][j] * w;
    }
  }
  if (lane == 0) {
    wm[wave] = m;
    wl[wave] = l;
  }
#pragma unroll
  for (int j = 0; j < KD; ++j) wo[wave][lane + 64 * j] = acc[j];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.hd) return;
  float mx = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
  for (int w = 0; w < kDecWaves; ++w) mx = fmaxf(mx, wm[w]);
#pragma unroll
  for (int w = 0; w < kDecWaves; ++w) {
    const float f = wm[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(wm[w] - mx);
    sum += wl[w] * f;
    o += wo[w][d] * f;
  }
  a.out[decode_row(a, seq).row * a.out_stride + (int64_t)head * a.hd + d] = o / sum;
}

template <typename T, int HD>
void decode_launch(const PagedAttnArgs& a, int grid, hipStream_t stream) {
  if (a.hd == HD)
    hipLaunchKernelGGL((paged_decode_kernel<T, HD, true>), dim3(grid), dim3(kDecThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_decode_kernel<T, HD, false>), dim3(grid), dim3(kDecThreads), 0, stream, a);
}
template <typename T>
void decode_launch_hd(const PagedAttnArgs& a, int grid, hipStream_t stream) {
  if (a.hd <= 64) decode_launch<T, 64>(a, grid, stream);
  else if (a.hd <= 128) decode_launch<T, 128>(a, grid, stream);
  else decode_launch<T, 256>(a, grid, stream);
}

// ---- prefill -----------------------------------------------------------------------
// Causal attention of every new row of every sequence. A workgroup owns 128
// consecutive (row, query head) pairs of one sequence and kv head (pairs
// r * group + h: no padding whatever the group), a wave 32 of them as the
// columns of both products, S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16
// instructions. A lane then holds 16 keys of one column: the softmax is in
// registers but for one lane swap, and P^T is the second product's B operand as
// it stands, V^T lying in LDS in the order in which the first product leaves
// the keys. q and the weights are split into parts as in the decode kernel;
// fp32 caches into three bf16 parts too, of whose nine part products the six
// largest are taken (the others are below 2^-25 of the product).
//  - Tiles of 32 keys pass through LDS; the next tile is on its way to registers
//    during the products, and the page that the one after it lies in is asked
//    for before that (a load that waits for its page waits twice).
//  - Infinities and NaN, also those that a weight of 0 was to silence, end up in
//    the output: the workgroup computes such columns again with values that are
//    not finite as 0, and once more with their places as 1 and every seen key's
//    weight as 1: NaN where the sum is positive.
//    (2000 rows of 6 sequences, 32 heads on 8 of 128, bf16, one infinite value
//    in a kv head of one: 0.49 ms, 0.16 without that value, 37.8 with such
//    columns in slow_row.) What met a page outside the cache goes to slow_row,
//    a wave for a row and head.
//  - Tiles with the most keys start first (6 sequences, 8000 rows behind up to
//    2000 tokens, 32 heads on 8 of 128, bf16: 565 -> 552 us); where the tiles
//    leave CUs idle, several workgroups share a tile's keys (64 rows of 16
//    sequences behind up to 8000 tokens, 28 heads on 4, bf16: 342 -> 83 us).
// That case's 620 GFLOP of part products (three for each of the two) take 550
// to 566 us, 1.1 PFLOP/s where a library product of 8192^3 reaches 1.2: the
// chip's power bounds both, its clock falls to 1.9 GHz. One barrier a tile instead of
// two, fewer vector instructions and no spills brought 691 to 543; raising the
// waves' priority around the products cost 5 %.
constexpr int kPreCols = 128, kPreKeys = 32, kPreThreads = 256;
typedef float f16v __attribute__((ext_vector_type(16)));

template <typename T>
struct PreTraits : KvTraits<T> {
  typedef T mat;
  static constexpr int kCacheParts = 1;
  static __device__ __forceinline__ f16v mfma32(h8_t a, h8_t b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f16v mfma32(bf8 a, bf8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct PreTraits<float> : KvTraits<__bf16> {
  typedef __bf16 mat;
  static constexpr int kCacheParts = 3;
  static __device__ __forceinline__ f16v mfma32(bf8 a, bf8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

template <typename T, int HD>
struct PreTile {
  static constexpr int NK = PreTraits<T>::kCacheParts;
  uint16_t k[NK][kPreKeys][HD + 8];   // [key][dim]
  uint16_t v[NK][HD][kPreKeys + 8];   // [dim][key slot], see v_slot
};
template <typename T, int HD>
struct PreLds {
  // 16-bit caches: the next tile is written beside the one that is read, a
  // barrier a tile; fp32's parts leave no room for it (two barriers), and at
  // head dim 256 its registers spill (8000 rows, 16 heads on 2: bf16 988 -> 681
  // us with one buffer, fp16 706 -> 620)
  static constexpr int kBuf = sizeof(T) == 4 || HD > 128 ? 1 : 2;
  // steps of q's last part per wave and lane (in registers they spill: fp16 at
  // head dim 256 1058 -> 706 us)
  static constexpr int kQ = HD < 128 || (PreTraits<T>::kParts < 3 && HD < 256) ? 0 : sizeof(T) == 4 ? (HD > 128 ? 12 : 5) : HD / 16;
  PreTile<T, HD> tile[kBuf];
  u32x4_t q[kQ > 0 ? kQ : 1][kPreThreads];
  int count[kPreThreads / 64];
};

// Where the 8-slot unit of a dim's row lies: a wave writes a few dims of four
// keys a lane, so neighbouring lanes are some rows apart; turning the units by
// the dim spreads them over the banks.
__device__ __forceinline__ int v_slot(int unit, int dim) { return (unit ^ ((dim >> 4) & 3)) * 8; }

// Which tile of which sequence a workgroup takes (seq < 0: none).
struct PreWork {
  int seq, tile;
};
__device__ __forceinline__ int wave_sum_int(int b) {
  b += __builtin_amdgcn_update_dpp(0, b, kDppXor1, 0xF, 0xF, false);
  b += __builtin_amdgcn_update_dpp(0, b, kDppXor2, 0xF, 0xF, false);
  b += __builtin_amdgcn_update_dpp(0, b, kDppHalfMirror, 0xF, 0xF, false);
  b += __builtin_amdgcn_update_dpp(0, b, kDppMirror, 0xF, 0xF, false);
  return (__builtin_amdgcn_readlane(b, 0) + __builtin_amdgcn_readlane(b, 16)) +
         (__builtin_amdgcn_readlane(b, 32) + __builtin_amdgcn_readlane(b, 48));
}
__device__ __forceinline__ int wave_max_int(int b) {
  b = max(b, __builtin_amdgcn_update_dpp(0, b, kDppXor1, 0xF, 0xF, false));
  b = max(b, __builtin_amdgcn_update_dpp(0, b, kDppXor2, 0xF, 0xF, false));
  b = max(b, __builtin_amdgcn_update_dpp(0, b, kDppHalfMirror, 0xF, 0xF, false));
  b = max(b, __builtin_amdgcn_update_dpp(0, b, kDppMirror, 0xF, 0xF, false));
  return max(max(__builtin_amdgcn_readlane(b, 0), __builtin_amdgcn_readlane(b, 16)),
             max(__builtin_amdgcn_readlane(b, 32), __builtin_amdgcn_readlane(b, 48)));
}
__device__ __forceinline__ int seq_tiles(const PagedAttnArgs& a, int i) {
  const int s0 = a.row_start[i], s1 = min(a.row_start[i + 1], a.max_rows);
  return s0 < 0 || s1 <= s0 ? 0 : (int)(((int64_t)(s1 - s0) * a.group + kPreCols - 1) / kPreCols);
}
// The x-th tile when those with the most keys come first, so that no long one
// starts last: a tile's level is how many tiles' rows its last key lies before
// the longest sequence's end, a sequence has one tile a level, and the level
// of x is found by a search over the count of tiles before it. Every wave does
// that for itself, kPreSeqsPerLane sequences a lane.
constexpr int kPreSeqsPerLane = 4, kPreSorted = 64 * kPreSeqsPerLane;
__device__ __forceinline__ PreWork longest_first(const PagedAttnArgs& a, int x) {
  const int lane = threadIdx.x & 63;
  int tiles[kPreSeqsPerLane], level[kPreSeqsPerLane], longest = 0, total = 0, end = 0;
#pragma unroll
  for (int n = 0; n < kPreSeqsPerLane; ++n) {
    const int i = lane + 64 * n;
    tiles[n] = 0;
    level[n] = 0;
    if (i < a.n_seqs) {
      tiles[n] = seq_tiles(a, i);
      level[n] = min(max(a.lengths[i], 0), a.max_len);
      if (tiles[n] > 0) longest = max(longest, level[n]);
    }
    total += tiles[n];
  }
  longest = wave_max_int(longest);
#pragma unroll
  for (int n = 0; n < kPreSeqsPerLane; ++n) {
    level[n] = (int)min((int64_t)(longest - min(level[n], longest)) * a.group / kPreCols, (int64_t)1 << 30);
    if (tiles[n] > 0) end = max(end, level[n] + tiles[n]);
  }
  if (x >= wave_sum_int(total)) return {-1, 0};
  auto before = [&](int at) {
    int c = 0;
#pragma unroll
    for (int n = 0; n < kPreSeqsPerLane; ++n) c += min(max(at - level[n], 0), tiles[n]);
    return wave_sum_int(c);
  };
  int lo = 0, hi = wave_max_int(end);  // before(lo) <= x < before(hi)
  while (hi - lo > 1) {
    const int mid = lo + ((hi - lo) >> 1);
    if (before(mid) <= x) lo = mid;
    else hi = mid;
  }
  int rank = x - before(lo);
  PreWork w = {-1, 0};
#pragma unroll
  for (int n = 0; n < kPreSeqsPerLane; ++n) {
    uint64_t has = __ballot(tiles[n] > 0 && lo >= level[n] && lo < level[n] + tiles[n]);
    const int count = __builtin_popcountll(has);
    if (w.seq < 0 && rank >= 0 && rank < count) {
      for (int r = 0; r < rank; ++r) has &= has - 1;
      const int from = __builtin_ctzll(has);
      w.seq = from + 64 * n;
      w.tile = __builtin_amdgcn_readlane(tiles[n], from) - 1 - (lo - __builtin_amdgcn_readlane(level[n], from));
    }
    rank -= count;
  }
  return w;
}
// For many sequences: sequence i owns the tiles from row_start[i] * G / 128 + i
// on, at least as many as it needs, found without a sum over the sequences
// before it.
__device__ __forceinline__ PreWork by_row(const PagedAttnArgs& a, int x, int* lds) {
  auto first_tile = [&](int i) { return (int64_t)a.row_start[i] * a.group / kPreCols + i; };
  int before = 0;
  for (int i = threadIdx.x; i < a.n_seqs; i += kPreThreads) before += first_tile(i) <= x;
  before = wave_sum_int(before);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = before;
  __syncthreads();
  const int seq = __builtin_amdgcn_readfirstlane(lds[0] + lds[1] + lds[2] + lds[3]) - 1;
  return {seq, seq < 0 ? 0 : (int)(x - first_tile(seq))};
}

// A workgroup's tile of rows: its pairs, positions and the keys that they see.
struct PreSpan {
  int row0, pos0, len;  // of the sequence
  int64_t pairs, c0;    // its pairs, the tile's first
  int kseen, kmax;      // first key that a row sees and last; kmax < 0 or len > max_len: none
  int kfirst;           // the tiles' first key: kseen down to a multiple of kPreKeys
  int tiles, each;      // key tiles, and of a workgroup when `splits` share them
  bool live;
};
constexpr int kPreLeast = 4;  // key tiles of a workgroup, at least
__device__ __forceinline__ PreSpan prefill_span(const PagedAttnArgs& a, const PreWork& w) {
  PreSpan s = {};
  if (w.seq < 0) return s;
  s.row0 = a.row_start[w.seq];
  const int end = a.row_start[w.seq + 1], row1 = min(end, a.max_rows);
  s.pairs = (int64_t)(row1 - s.row0) * a.group;
  s.c0 = (int64_t)w.tile * kPreCols;
  if (s.row0 < 0 || s.c0 < 0 || s.c0 >= s.pairs) return s;
  s.live = true;
  s.len = max(a.lengths[w.seq], 0);  // (below: any number, but no overflow)
  s.pos0 = s.len - (end - s.row0);
  const int ja = (int)(s.c0 / a.group), jb = (int)((min(s.c0 + kPreCols, s.pairs) - 1) / a.group);
  if (s.len > a.max_len) return s;
  s.kmax = s.pos0 + jb;
  s.kseen = a.window > 0 ? max(0, s.pos0 + ja + 1 - a.window) : 0;
  s.kfirst = s.kseen & ~(kPreKeys - 1);
  s.tiles = s.kmax < 0 ? 0 : (s.kmax - s.kfirst) / kPreKeys + 1;
  s.each = max((s.tiles + a.splits - 1) / a.splits, kPreLeast);
  return s;
}

// Partials of a tile of rows, kv head and split: maxima and sums [kPreCols],
// accumulators [hd / 4][kPreCols][4]; before them what the join has to know of
// each tile.
struct PreJoin {
  int parts;     // 1 and less: nothing to join
  int cols, seq, row, pos, rem;  // of the first pair: its row, position and head of the group
};
struct PrePartial {
  float* m;
  float* l;
  float* acc;
};
__host__ __device__ inline size_t prefill_partial_floats(int hd) { return (size_t)kPreCols * (hd + 2); }
__host__ __device__ inline size_t prefill_header(int64_t blocks) { return dec_align((size_t)blocks * sizeof(PreJoin)); }
__device__ __forceinline__ PrePartial prefill_partial(const PagedAttnArgs& a, int split) {
  float* p = (float*)((char*)a.part + prefill_header(gridDim.x)) +
             ((size_t)blockIdx.x * a.splits + split) * prefill_partial_floats(a.hd);
  return {p, p + kPreCols, p + 2 * kPreCols};
}

// A word of values for the passes after the first: those that are not finite as
// 0; or, to count them, as 1 and the others as 0.
template <typename T>
__device__ __forceinline__ uint32_t settled(uint32_t w, bool count) {
  constexpr bool F32 = sizeof(T) == 4, F16 = std::is_same<T, _Float16>::value;
  constexpr uint32_t kExp = F32 ? 0x7f800000u : F16 ? 0x7c00u : 0x7f80u, kOne = F32 ? 0x3f800000u : F16 ? 0x3c00u : 0x3f80u;
  if constexpr (F32) {
    const bool bad = (w & kExp) == kExp;
    return count ? (bad ? kOne : 0u) : (bad ? 0u : w);
  }
  const bool lo = (w & kExp) == kExp, hi = (w >> 16 & kExp) == kExp;
  if (count) return (lo ? kOne : 0u) | (hi ? kOne << 16 : 0u);
  return w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  return settled<T>(w, true) != 0;
}

// One pass of a workgroup over its keys. The first writes the columns (or their
// partials) that are finite and returns the others; AGAIN, for those: `count` 0
// with values that are not finite as 0, 1 to mark where they are seen.
// RULE: scores are capped or biased (a variant of its own: its values spill
// beside the others').
struct PreDirty {
  bool column, any;  // this lane's, any of the workgroup
};
template <typename T, int HD, bool FULL, bool RULE, bool AGAIN>
__device__ __forceinline__ PreDirty prefill_pass(const PagedAttnArgs& a, const PreSpan& sp, int seq, PreLds<T, HD>& lds,
                                                 bool dirty, bool count) {
  using Tr = PreTraits<T>;
  using M = typename Tr::mat;
  using vec = typename Tr::vec;
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int NP = Tr::kParts, NK = Tr::kCacheParts;
  constexpr int KT = HD / 16;        // 16-dim steps of the scores
  constexpr int VB = HD / 32;        // 32-dim blocks of the output
  constexpr int KW = HD / 8 * (int)sizeof(T) / 4;   // words of K per thread: HD / 8 dims of a key
  constexpr int VDT = HD / 32;       // dims of V per thread, of 4 keys
  constexpr int VWT = VDT * (int)sizeof(T) / 4;     // their words a key (fp16 / bf16, HD 64: 1)
  constexpr float kSlack = Tr::kLift == 0.0f ? 8.0f : 0.0f;
  constexpr int BUF = PreLds<T, HD>::kBuf, QL = PreLds<T, HD>::kQ;
  int* const count_lds = lds.count;
  int tid = threadIdx.x;
  if constexpr (AGAIN) asm volatile("" : "+v"(tid));  // (no lane's numbers are kept for it from the first pass)
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int G = a.group;
  const int kvh = blockIdx.x % a.n_kv, split = blockIdx.y;
  const int row0 = sp.row0, pos0 = sp.pos0;
  const int64_t pairs = sp.pairs, c0 = sp.c0;
  // this lane's column
  const int64_t cc = c0 + wave * 32 + col;
  const bool live = cc < pairs;
  const int jr = (int)((live ? cc : pairs - 1) / G), qh = (int)((live ? cc : pairs - 1) - (int64_t)jr * G);
  const int row = row0 + jr, qpos = pos0 + jr, head = kvh * G + qh;
  float* out = a.out + row * a.out_stride + (int64_t)head * a.hd;
  // the workgroup's keys; the wave's first and last row
  const bool parts = sp.tiles > sp.each;  // other workgroups have the tile's other keys
  const int key0 = sp.kfirst + split * sp.each * kPreKeys;
  const int kmax = min(sp.kmax, key0 + sp.each * kPreKeys - 1);
  const int wave_first = __builtin_amdgcn_readfirstlane(__shfl(qpos, 0));
  const int wave_last = __builtin_amdgcn_readfirstlane(__shfl(qpos, 63));
  // ---- q
  int q_exp = 0;
  vec q[NP][KT];
  bool odd = false;    // a page outside the cache
  bool k_bad = false;  // AGAIN: a key that is not finite
  float q_zero = 0.0f;  // AGAIN: NaN where q is not finite
  {
    const float* qp = a.q + row * a.q_stride + (int64_t)head * a.hd + 8 * half;
    auto q_at = [&](int s, int u) __attribute__((always_inline)) {
      return live && (FULL || 16 * s + 8 * half < a.hd) ? *(const f4*)(qp + 16 * s + 4 * u)
                                                          : f4{0.0f, 0.0f, 0.0f, 0.0f};
    };
    // (q's sign turned where the scale is negative: the largest score is then
    // the largest product)
    const float turned = a.scale < 0.0f ? -1.0f : 1.0f;
    if constexpr (Tr::kLift != 0.0f) {
      float big = 0.0f;
#pragma unroll
      for (int s = 0; s < KT; ++s)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f4 x = q_at(s, u);
          big = fmaxf(fmaxf(big, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
        }
      q_exp = pow2_scale_exp(xor32_max(big));
    }
#pragma unroll
    for (int s = 0; s < KT; ++s) {
      uint32_t w[NP][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        f4 x = q_at(s, u) * turned;
        if constexpr (AGAIN) q_zero += (x.x * 0.0f + x.y * 0.0f) + (x.z * 0.0f + x.w * 0.0f);
        if constexpr (Tr::kLift != 0.0f)
          x = f4{ldexp_f(x.x, q_exp), ldexp_f(x.y, q_exp), ldexp_f(x.z, q_exp), ldexp_f(x.w, q_exp)};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t p[NP];
          split_pair<M>(x[2 * j], x[2 * j + 1], p);
#pragma unroll
          for (int i = 0; i < NP; ++i) w[i][2 * u + j] = p[i];
        }
      }
#pragma unroll
      for (int i = 0; i < NP; ++i)
        q[i][s] = __builtin_bit_cast(vec, u32x4_t{w[i][0], w[i][1], w[i][2], w[i][3]});
      if (s < QL) lds.q[s < QL ? s : 0][tid] = __builtin_bit_cast(u32x4_t, q[NP - 1][s]);  // (read by this lane only)
    }
  }
  auto q_part = [&](int i, int s) __attribute__((always_inline)) {
    return i == NP - 1 && s < QL ? __builtin_bit_cast(vec, lds.q[s < QL ? s : 0][tid]) : q[i][s];
  };
  const ScoreRule rule = score_rule(a, head, q_exp, fabsf(a.scale));

  // ---- staging: a wave's keys lie in one run of 16 (and so in one page)
  const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
  const int mask = (1 << a.page_shift) - 1, row_bytes = a.hd * (int)sizeof(T);
  // The wave's run, or the nearest that holds a key which a row sees (a tile may
  // begin before the window, on a page that nobody keeps any more).
  auto key_of = [&](int k0) __attribute__((always_inline)) { return min(max(k0 + 16 * (wave >> 1), sp.kseen), kmax); };
  // Asked for a tile ahead of the rows it names: a load that waits for it waits
  // twice.
  auto page_of = [&](int k0) __attribute__((always_inline)) { return table[key_of(k0) >> a.page_shift]; };
  auto run_of = [&](int k0, int id) __attribute__((always_inline)) {
    const int kk = key_of(k0);
    int page = __builtin_amdgcn_readfirstlane(id);
    const bool outside = page < 0 || page >= a.n_pages;
    odd |= outside;
    page = outside ? 0 : page;
    return ((((int64_t)page * a.n_kv + kvh) << a.page_shift) + (kk & mask & ~15)) * row_bytes;
  };
  const int kkey = tid >> 3, kd = (tid & 7) * (16 / (int)sizeof(T));  // K: dims kd + 8 threads' pieces
  const int vkg = tid >> 5, vd = (tid & 31) * VDT;                    // V: keys 4 vkg .. + 3
  uint32_t kw[KW], vw[4][VWT];
  // (a run's start is uniform, a lane's place in it never changes)
  const uint32_t k_at = (kkey & 15) * row_bytes + kd * (int)sizeof(T);
  const uint32_t v_at = 4 * (vkg & 3) * row_bytes + vd * (int)sizeof(T);
  auto load_k = [&](int64_t run) __attribute__((always_inline)) {
    const char* p = (const char*)a.keys + run;
#pragma unroll
    for (int w = 0; w < KW; w += 4) {
      const bool in = FULL || kd + w * 32 / (int)sizeof(T) < a.hd;
      const u32x4_t x = in ? *(const u32x4_t*)(p + k_at + w * 32) : u32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) kw[w + i] = x[i];
    }
  };
  auto load_v = [&](int64_t run) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const char* p = (const char*)a.values + run + e * row_bytes;
      if constexpr (VWT >= 4) {
#pragma unroll
        for (int w = 0; w < VWT; w += 4) {
          const bool in = FULL || vd + w * 4 / (int)sizeof(T) < a.hd;
          const u32x4_t x = in ? *(const u32x4_t*)(p + v_at + 4 * w) : u32x4_t{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i) vw[e][w + i] = x[i];
        }
      } else if constexpr (VWT == 2) {
        const u32x2_t x = FULL || vd < a.hd ? *(const u32x2_t*)(p + v_at) : u32x2_t{0, 0};
        vw[e][0] = x.x;
        vw[e][1] = x.y;
      } else {
        vw[e][0] = FULL || vd < a.hd ? *(const uint32_t*)(p + v_at) : 0u;
      }
    }
  };
  auto put_k = [&](PreTile<T, HD>& tl, int k0) __attribute__((always_inline)) {
    if constexpr (AGAIN)
      if (k0 + kkey <= kmax) {
#pragma unroll
        for (int w = 0; w < KW; ++w) k_bad |= not_finite<T>(kw[w]);
      }
    if constexpr (F32) {
#pragma unroll
      for (int w = 0; w < KW; w += 4) {
        uint32_t x[3], y[3];
        split_pair<__bf16>(__builtin_bit_cast(float, kw[w]), __builtin_bit_cast(float, kw[w + 1]), x);
        split_pair<__bf16>(__builtin_bit_cast(float, kw[w + 2]), __builtin_bit_cast(float, kw[w + 3]), y);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(u32x2_t*)&tl.k[i][kkey][kd + w * 8] = u32x2_t{x[i], y[i]};
      }
    } else {
#pragma unroll
      for (int w = 0; w < KW; w += 4)
        *(u32x4_t*)&tl.k[0][kkey][kd + w * 16] = u32x4_t{kw[w], kw[w + 1], kw[w + 2], kw[w + 3]};
    }
  };
  auto put_v = [&](PreTile<T, HD>& tl, int k0) __attribute__((always_inline)) {
    if (k0 + kPreKeys - 1 > kmax) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k0 + 4 * vkg + e > kmax) {
#pragma unroll
          for (int w = 0; w < VWT; ++w) vw[e][w] = 0;
        }
    }
    if constexpr (AGAIN) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int w = 0; w < VWT; ++w) vw[e][w] = settled<T>(vw[e][w], count);
    }
    // the key group's slots in its run of 16: keys 0-3, 8-11 | 4-7, 12-15
    const int unit = 2 * (vkg >> 2) + (vkg & 1), sub = 4 * ((vkg >> 1) & 1);
#pragma unroll
    for (int j = 0; j < VDT; ++j) {
      const int at = v_slot(unit, vd + j) + sub;
      if constexpr (F32) {
        uint32_t x[3], y[3];
        split_pair<__bf16>(__builtin_bit_cast(float, vw[0][j]), __builtin_bit_cast(float, vw[1][j]), x);
        split_pair<__bf16>(__builtin_bit_cast(float, vw[2][j]), __builtin_bit_cast(float, vw[3][j]), y);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(u32x2_t*)&tl.v[i][vd + j][at] = u32x2_t{x[i], y[i]};
      } else {
        const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
        *(u32x2_t*)&tl.v[0][vd + j][at] =
            u32x2_t{__builtin_amdgcn_perm(vw[1][j >> 1], vw[0][j >> 1], sel),
                    __builtin_amdgcn_perm(vw[3][j >> 1], vw[2][j >> 1], sel)};
      }
    }
  };

  f16v acc[VB];
#pragma unroll
  for (int b = 0; b < VB; ++b) acc[b] = (f16v){};
  float m = -INFINITY, l = 0.0f;  // of the column; l of this half's keys
  int k0 = key0;
  int64_t run = run_of(k0, page_of(k0));
  load_k(run);
  int next_page = page_of(k0 + kPreKeys);
  auto next = [&](int k) __attribute__((always_inline)) {
    run = run_of(k, next_page);
    next_page = page_of(k + kPreKeys);
  };
  if constexpr (BUF == 2) {
    load_v(run);
    put_k(lds.tile[0], k0);
    put_v(lds.tile[0], k0);
    __syncthreads();
  }
  for (int cur = 0; k0 <= kmax; k0 += kPreKeys, cur ^= BUF - 1) {
    PreTile<T, HD>& tl = lds.tile[cur];
    const bool more = k0 + kPreKeys <= kmax;
    if constexpr (BUF == 2) {
      if (more) {
        next(k0 + kPreKeys);
        load_k(run);
        load_v(run);
      }
    } else {
      put_k(tl, k0);  // (the last tile's K is done with since its second barrier)
      load_v(run);
      __syncthreads();
    }
    f16v s = {}, s1 = {};
    // the small part products of all dims first: few roundings at a score's own size
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      f16v& c = i % 2 == 0 ? s : s1;
      vec kk[NK];
#pragma unroll
      for (int x = 0; x < NK; ++x) kk[x] = *(const vec*)&tl.k[x][col][16 * i + 8 * half];
#pragma unroll
      for (int sum = NP - 1; sum > 0; --sum)
#pragma unroll
        for (int x = NK - 1; x >= 0; --x)
          if (sum - x >= 0 && sum - x < NP) c = Tr::mfma32(kk[x], q_part(sum - x, i), c);
    }
    // (fp32's parts are read again: held across the loops they spill)
    if constexpr (NK > 1 && HD <= 128) asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      f16v& c = i % 2 == 0 ? s : s1;
      c = Tr::mfma32(*(const vec*)&tl.k[0][col][16 * i + 8 * half], q[0][i], c);
    }
    s += s1;
    if constexpr (BUF == 1) {
      put_v(tl, k0);
      if (more) {
        next(k0 + kPreKeys);
        load_k(run);
      }
      __syncthreads();
    }
    // lane: keys 8 (i / 4) + 4 half + i % 4 of its column
    const bool edge = k0 + kPreKeys - 1 > wave_first || (a.window > 0 && k0 <= wave_last - a.window);
    float sl = rule.sl2;  // what is left to multiply
    if (RULE || edge) {
      sl = 1.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = k0 + 8 * (i >> 2) + 4 * half + (i & 3);
        s[i] = RULE && a.softcap > 0.0f ? rule.cap_out * tanhf(s[i] * rule.cap_in) : s[i] * rule.sl2;
        if constexpr (RULE) s[i] += rule.slope2 * (float)(k - qpos);
        if (k > qpos || (a.window > 0 && k <= qpos - a.window)) s[i] = -INFINITY;
      }
    }
    if constexpr (AGAIN)
      if (count) {  // every key that is seen weighs the same
        sl = 1.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = k0 + 8 * (i >> 2) + 4 * half + (i & 3);
          s[i] = k > qpos || (a.window > 0 && k <= qpos - a.window) ? -INFINITY : 0.0f;
        }
      }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = fmaxf(m, xor32_max(mx) * sl);
    // The reference of the weights follows the maximum only where it is 2^kSlack
    // behind (bf16 parts hold any size): less to rescale.
    if constexpr (kSlack > 0.0f) mx = mx > m + kSlack ? mx : m;
    // rows with nothing visible yet keep m = -inf and weight 0
    const float ref = (mx == -INFINITY ? 0.0f : mx) - Tr::kLift;
    if (__any(mx != m)) {
      const float alpha = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
#pragma unroll
      for (int b = 0; b < VB; ++b) acc[b] *= alpha;
      l *= alpha;
      m = mx;
    }
    // (scaled and shifted with one rounding)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], sl, -ref));
    l += (((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]))) +
         (((s[8] + s[9]) + (s[10] + s[11])) + ((s[12] + s[13]) + (s[14] + s[15])));
    vec p[NP][2];  // 16 keys each
    {
      uint32_t w[NP][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t x[NP];
        split_pair<M>(s[2 * j], s[2 * j + 1], x);
#pragma unroll
        for (int i = 0; i < NP; ++i) w[i][j] = x[i];
      }
#pragma unroll
      for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u)
          p[i][u] = __builtin_bit_cast(vec, u32x4_t{w[i][4 * u], w[i][4 * u + 1], w[i][4 * u + 2], w[i][4 * u + 3]});
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        const int at = v_slot(2 * u + half, 32 * b + col);
        vec vv[NK];
#pragma unroll
        for (int x = 0; x < NK; ++x) vv[x] = *(const vec*)&tl.v[x][32 * b + col][at];
#pragma unroll
        for (int sum = NP - 1; sum >= 0; --sum)
#pragma unroll
          for (int x = NK - 1; x >= 0; --x)
            if (sum - x >= 0 && sum - x < NP) acc[b] = Tr::mfma32(vv[x], p[sum - x][u], acc[b]);
      }
    if constexpr (BUF == 2) {
      if (more) {
        put_k(lds.tile[cur ^ 1], k0 + kPreKeys);
        put_v(lds.tile[cur ^ 1], k0 + kPreKeys);
        __syncthreads();
      }
    }
  }
  // (without this the loop copies acc once a tile, for what follows)
#pragma unroll
  for (int b = 0; b < VB; ++b) asm volatile("" : "+v"(acc[b]));
  const float sum = xor32_sum(l);
  const int at = wave * 32 + col;
  PrePartial pp = {};
  if (parts) pp = prefill_partial(a, split);
  if (AGAIN && count) {  // NaN where a value that is not finite is seen
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * b + 8 * (i >> 2) + 4 * half + (i & 3);
        if (dirty && (FULL || d < a.hd) && acc[b][i] > 0.0f)
          *(parts ? pp.acc + ((size_t)(d >> 2) * kPreCols + at) * 4 + (d & 3) : out + d) = __builtin_nanf("");
      }
    return {};
  }
  float zeros = sum * 0.0f;
#pragma unroll
  for (int b = 0; b < VB; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) zeros = __builtin_fmaf(acc[b][i], 0.0f, zeros);
  const bool odd_column = live && !(xor32_sum(zeros) == 0.0f);
  // (the waves tell each other: 1 a page outside the cache, 2 a key that is not
  // finite, 4 a column that is not)
  const int mine = (__any(odd) ? 1 : 0) | (__any(k_bad) ? 2 : 0) | (__any(odd_column) ? 4 : 0);
  __syncthreads();  // every wave is done with the tile
  if (lane == 0) count_lds[wave] = mine;
  __syncthreads();
  const int all = __builtin_amdgcn_readfirstlane(count_lds[0] | count_lds[1] | count_lds[2] | count_lds[3]);
  bool write = live, slow = false;
  if constexpr (AGAIN) {
    // What no key or query explains is an overflow of the parts, which plain
    // fp32 may not share.
    slow = dirty && ((all & 1) != 0 || (odd_column && (all & 2) == 0 && xor32_sum(q_zero) == 0.0f));
    write = dirty && !slow;
  } else {
    dirty = live && (odd_column || (all & 1) != 0);
    write = live && !dirty;
  }
  if (parts) {
    // (a maximum of NaN: the join computes the column in plain fp32)
    if (half == 0 && (write || slow)) {
      pp.m[at] = slow ? __builtin_nanf("") : m;
      pp.l[at] = sum;
    }
    if (write) {
#pragma unroll
      for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 32 * b + 8 * i + 4 * half;
          if (FULL || d < a.hd)
            *(f4*)(pp.acc + ((size_t)(d >> 2) * kPreCols + at) * 4) =
                f4{acc[b][4 * i], acc[b][4 * i + 1], acc[b][4 * i + 2], acc[b][4 * i + 3]};
        }
    }
    return {dirty, all != 0};
  }
  if constexpr (AGAIN) {
    uint64_t redo = __ballot(slow);
    redo = (redo | redo >> 32) & 0xffffffffu;
    while (redo != 0) {
      const int c = __builtin_ctzll(redo);
      redo &= redo - 1;
      const int64_t p = c0 + wave * 32 + c;
      const int j = (int)(p / G);
      slow_row<T>(a, seq, row0 + j, pos0 + j, kvh * G + (int)(p - (int64_t)j * G), (float*)&lds + wave * kSlowFloats, 0, a.hd);
    }
  }
  if (write) {
    const float f = qpos < 0 ? 1.0f : sum;  // (a row before the first key: zeros)
#pragma unroll
    for (int b = 0; b < VB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * b + 8 * i + 4 * half;
        if (FULL || d < a.hd)
          *(f4*)(out + d) = f4{acc[b][4 * i] / f, acc[b][4 * i + 1] / f, acc[b][4 * i + 2] / f, acc[b][4 * i + 3] / f};
      }
  }
  return {dirty, all != 0};
}

// The tile of rows that a workgroup takes.
struct PreTask {
  int seq;
  PreSpan span;
};
__device__ __forceinline__ PreTask prefill_task(const PagedAttnArgs& a, int x, int* lds) {
  const PreWork work = a.n_seqs <= kPreSorted ? longest_first(a, x / a.n_kv) : by_row(a, x / a.n_kv, lds);
  return {work.seq, prefill_span(a, work)};
}

template <typename T, int HD, bool FULL, bool RULE>
__global__ __launch_bounds__(kPreThreads, HD <= 128 ? 2 : 1) void paged_prefill_kernel(PagedAttnArgs a) {
  extern __shared__ __align__(16) uint8_t pre_smem[];
  PreLds<T, HD>& lds = *(PreLds<T, HD>*)pre_smem;
  const int tid = threadIdx.x, G = a.group, kvh = blockIdx.x % a.n_kv, split = blockIdx.y;
  const PreTask task = prefill_task(a, (int)blockIdx.x, lds.count);
  const PreSpan& sp = task.span;
  if (split == 0 && a.part != nullptr && tid == 0) {
    const int j = (int)(sp.c0 / G);
    const bool join = sp.live && sp.len <= a.max_len && sp.tiles > sp.each;
    ((PreJoin*)a.part)[blockIdx.x] = {join ? (sp.tiles + sp.each - 1) / sp.each : 0,
                                      (int)min((int64_t)kPreCols, sp.pairs - sp.c0), task.seq, sp.row0 + j, sp.pos0 + j,
                                      (int)(sp.c0 - (int64_t)j * G)};
  }
  if (!sp.live) return;
  if (sp.len > a.max_len || sp.kmax < 0) {  // (kmax < 0: nothing to see)
    const int64_t cc = sp.c0 + (tid >> 1);
    const int j = (int)(cc / G);
    if (cc < sp.pairs && split == 0) {
      float* out = a.out + (sp.row0 + j) * a.out_stride + (int64_t)(kvh * G + (int)(cc - (int64_t)j * G)) * a.hd;
      const float x = sp.len > a.max_len ? __builtin_nanf("") : 0.0f;
      for (int d = 4 * (tid & 1); d < a.hd; d += 8) *(f4*)(out + d) = f4{x, x, x, x};
    }
    return;
  }
  if (sp.kfirst + split * sp.each * kPreKeys > sp.kmax) return;

  const PreDirty dirty = prefill_pass<T, HD, FULL, RULE, false>(a, sp, task.seq, lds, false, false);
  if (__builtin_expect(!dirty.any, 1)) return;
  // From here on everything but `dirty` is made anew, the arguments read again:
  // what the compiler keeps for this through the first pass's loop spills there
  // (8000 rows, 32 heads on 8, bf16: 557 -> 582 us).
  auto args = (const __attribute__((address_space(4))) PagedAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  PagedAttnArgs b;
  __builtin_memcpy(&b, (const void*)args, sizeof(b));
  __syncthreads();  // (every wave has read what the waves told each other)
  const PreTask same = prefill_task(b, (int)blockIdx.x, lds.count);
#pragma nounroll
  for (int count = 0; count < 2; ++count) {
    __syncthreads();  // (every wave is done with the LDS)
    prefill_pass<T, HD, FULL, RULE, true>(b, same.span, same.seq, lds, dirty.column, count != 0);
  }
}

// The splits of a tile of rows and kv head joined: a thread has one column and
// two quads of dims, a workgroup 32 dims, four splits' loads are asked for at
// once. Columns that a split marked, and those that overflow only here, go to
// slow_row.
constexpr int kPreJoinThreads = 512, kPreJoinDims = 32, kPreMaxSplits = 32, kPreJoinAhead = 4;
template <typename T>
__global__ __launch_bounds__(kPreJoinThreads) void paged_prefill_join_kernel(PagedAttnArgs a) {
  constexpr int kStep = kPreJoinThreads / kPreCols;  // quads of dims that the threads take at a time
  constexpr int N = kPreJoinDims / 4 / kStep;        // per thread, of one column
  __shared__ int redo[kPreCols];
  __shared__ __align__(16) float slow[kPreJoinThreads / 64][kSlowFloats];
  const PreJoin info = ((const PreJoin*)a.part)[blockIdx.x];
  if (info.parts <= 1) return;
  const int tid = threadIdx.x, kvh = blockIdx.x % a.n_kv, d0 = blockIdx.y * kPreJoinDims;
  const int col = tid % kPreCols, q0 = d0 / 4 + tid / kPreCols, last = a.hd / 4 - 1;
  if (tid < kPreCols) redo[tid] = 0;
  __syncthreads();
  const PrePartial first = prefill_partial(a, 0);
  const size_t stride = prefill_partial_floats(a.hd);
  float m = -INFINITY, l = 0.0f;
  bool again = false;
  f4 o[N];
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < info.parts; i0 += kPreJoinAhead) {
    float pm[kPreJoinAhead], pl[kPreJoinAhead];
    f4 x[kPreJoinAhead][N];
#pragma unroll
    for (int i = 0; i < kPreJoinAhead; ++i) {
      const size_t at = (size_t)min(i0 + i, info.parts - 1) * stride;
      pm[i] = first.m[at + col];
      pl[i] = first.l[at + col];
#pragma unroll
      for (int n = 0; n < N; ++n)
        x[i][n] = *(const f4*)(first.acc + at + (size_t)min(q0 + kStep * n, last) * (4 * kPreCols) + 4 * col);
    }
    float mx = m;
#pragma unroll
    for (int i = 0; i < kPreJoinAhead; ++i)
      if (i0 + i < info.parts) {
        mx = fmaxf(mx, pm[i]);
        again |= pm[i] != pm[i];
      }
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mx);
    m = mx;
    l *= f;
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] *= f;
#pragma unroll
    for (int i = 0; i < kPreJoinAhead; ++i) {
      if (i0 + i >= info.parts) break;
      const float w = pm[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[i] - mx);
      l += pl[i] * w;
#pragma unroll
      for (int n = 0; n < N; ++n) o[n] += x[i][n] * w;
    }
  }
  auto place = [&](int c, int* row, int* pos, int* head) {
    const int j = (info.rem + c) / a.group;
    *row = info.row + j;
    *pos = info.pos + j;
    *head = kvh * a.group + info.rem + c - j * a.group;
  };
  int row, pos, head;
  if (col < info.cols) {
    place(col, &row, &pos, &head);
    float* out = a.out + row * a.out_stride + (int64_t)head * a.hd;
    const float f = pos < 0 ? 1.0f : l;  // (a row before the first key sees nothing: zeros)
    float zeros = l * 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const f4 z = o[n] * 0.0f;
      zeros += (z.x + z.y) + (z.z + z.w);
      if (q0 + kStep * n <= last) *(f4*)(out + 4 * (q0 + kStep * n)) = f4{o[n].x / f, o[n].y / f, o[n].z / f, o[n].w / f};
    }
    if (!again && !(zeros == 0.0f)) {
      again = true;
      for (int i = 0; i < info.parts; ++i) {
        float given = first.l[i * stride + col] * 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const f4 z = *(const f4*)(first.acc + i * stride + (size_t)min(q0 + kStep * n, last) * (4 * kPreCols) + 4 * col) * 0.0f;
          given += (z.x + z.y) + (z.z + z.w);
        }
        if (!(given == 0.0f)) again = false;
      }
    }
    if (again) redo[col] = 1;
  }
  __syncthreads();
  for (int c = tid >> 6; c < info.cols; c += kPreJoinThreads / 64)
    if (redo[c]) {
      place(c, &row, &pos, &head);
      slow_row<T>(a, info.seq, row, pos, head, slow[tid >> 6], d0, min(d0 + kPreJoinDims, a.hd));
    }
}

template <typename T, int HD, bool FULL, bool RULE>
hipError_t prefill_launch(const PagedAttnArgs& a, hipStream_t stream) {
  constexpr size_t lds = sizeof(PreLds<T, HD>);
  static_assert(sizeof(PreTile<T, HD>) >= kPreThreads / 64 * kSlowFloats * sizeof(float), "slow_row's");
  const auto kernel = paged_prefill_kernel<T, HD, FULL, RULE>;
  hipError_t e = allow_dynamic_lds((const void*)kernel, lds);
  if (e != hipSuccess) return e;
  const int64_t grid = prefill_groups(a);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid, a.splits), dim3(kPreThreads), lds, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(paged_prefill_join_kernel<T>,
                     dim3((unsigned)grid, (a.hd + kPreJoinDims - 1) / kPreJoinDims), dim3(kPreJoinThreads), 0, stream, a);
  return hipGetLastError();
}
template <typename T, int HD>
hipError_t prefill_launch_hd(const PagedAttnArgs& a, hipStream_t stream) {
  const bool rule = a.softcap > 0.0f || a.slopes != nullptr;
  if (a.hd == HD)
    return rule ? prefill_launch<T, HD, true, true>(a, stream) : prefill_launch<T, HD, true, false>(a, stream);
  return rule ? prefill_launch<T, HD, false, true>(a, stream) : prefill_launch<T, HD, false, false>(a, stream);
}
template <typename T>
hipError_t prefill_launch_type(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.hd <= 64) return prefill_launch_hd<T, 64>(a, stream);
  if (a.hd <= 128) return prefill_launch_hd<T, 128>(a, stream);
  return prefill_launch_hd<T, 256>(a, stream);
}

}  // namespace

size_t plan_paged_decode(PagedAttnArgs& a) {
  const int64_t n_tiles = (int64_t)a.n_kv * ((a.group + 15) / 16);
  const int keys = a.type == MLQ_KV_F32 ? 16 : 32, unit = kDecWaves * keys;
  const int64_t units = (a.max_len + (int64_t)unit - 1) / unit;  // of a sequence
  const int cus = device_cus();
  // sequences of a launch: their prefix sums lie in LDS and fit 32 bits
  a.launch_seqs = (int)std::min((int64_t)std::min(a.n_seqs, kDecMaxSeqs), std::max(((int64_t)1 << 28) / units, (int64_t)1));
  a.whole = (int)units * kDecWaves;
  // Short ones are left whole, without a second launch (units of 128 keys, 64 of
  // fp32; us of both and of a cut, in a graph, 28 heads on 4 of 128, bf16: one
  // sequence of 250 9.4 and 10.2, of 500 12.9 and 10.4; 100 of up to 500 18.9 and
  // 23.2; head dim 64, 16 heads, 16 of up to 500: 9.0 and 9.8).
  if (units <= 2 || (units <= 4 && (a.hd <= 64 || a.launch_seqs * n_tiles >= cus))) {
    a.ranges = (int)(a.launch_seqs * n_tiles);
    return 0;
  }
  // (pieces of as many sequences as a launch takes under the smallest bounds: the
  // ranges, and so the workspace, are then no fewer for a longer one)
  const int64_t pieces = std::min(a.n_seqs, kDecMaxSeqs) * n_tiles;
  a.ranges = (int)std::min(a.launch_seqs * n_tiles * units, (int64_t)dec_per_cu(a.hd, pieces, cus) * cus);
  const size_t tg = std::min(a.group, 16);
  return dec_header(std::min(a.n_seqs, kDecMaxSeqs)) + dec_align((size_t)2 * a.ranges * tg * 8) +
         (size_t)2 * a.ranges * tg * a.hd * sizeof(float);
}

hipError_t launch_paged_decode(const PagedAttnArgs& all, hipStream_t stream) {
  for (int s0 = 0; s0 < all.n_seqs; s0 += all.launch_seqs) {
    PagedAttnArgs a = all;
    a.n_seqs = std::min(all.launch_seqs, all.n_seqs - s0);
    a.block_table += (size_t)s0 * a.max_pages;
    a.lengths += s0;
    if (a.row_start != nullptr) {
      a.row_start += s0;
    } else {
      a.q += (int64_t)s0 * a.q_stride;
      a.out += (int64_t)s0 * a.out_stride;
    }
    if (a.type == MLQ_KV_F32) decode_launch_hd<float>(a, a.ranges, stream);
    else if (a.type == MLQ_KV_F16) decode_launch_hd<_Float16>(a, a.ranges, stream);
    else decode_launch_hd<__bf16>(a, a.ranges, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.part == nullptr) continue;
    const dim3 grid(a.n_seqs, a.n_kv * a.group);
    if (a.hd <= 64)
      hipLaunchKernelGGL(paged_combine_kernel<1>, grid, dim3(kDecThreads), 0, stream, a);
    else if (a.hd <= 128)
      hipLaunchKernelGGL(paged_combine_kernel<2>, grid, dim3(kDecThreads), 0, stream, a);
    else
      hipLaunchKernelGGL(paged_combine_kernel<4>, grid, dim3(kDecThreads), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

// Tiles of rows that the grid has to hold, one more for each sequence than its
// rows fill, for every kv head.
int64_t prefill_groups(const PagedAttnArgs& a) {
  return ((int64_t)a.max_rows * a.group / kPreCols + a.n_seqs) * a.n_kv;
}

// Where the tiles of rows leave most of the chip idle, a tile's keys are shared
// by several workgroups and joined.
size_t plan_paged_prefill(PagedAttnArgs& a) {
  const int64_t tiles = prefill_groups(a), slots = (int64_t)(a.hd <= 128 ? 2 : 1) * device_cus();
  const int64_t keys = ((int64_t)a.max_len + kPreKeys - 1) / kPreKeys;
  a.splits = (int)std::max(std::min(std::min(slots / tiles, keys / kPreLeast), (int64_t)kPreMaxSplits), (int64_t)1);
  if (a.n_seqs > kPreSorted) a.splits = 1;
  if (a.splits == 1) return 0;
  return prefill_header(tiles) + (size_t)tiles * a.splits * prefill_partial_floats(a.hd) * sizeof(float);
}

hipError_t launch_paged_prefill(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.type == MLQ_KV_F32) return prefill_launch_type<float>(a, stream);
  if (a.type == MLQ_KV_F16) return prefill_launch_type<_Float16>(a, stream);
  return prefill_launch_type<__bf16>(a, stream);
}

}  // namespace mlq
