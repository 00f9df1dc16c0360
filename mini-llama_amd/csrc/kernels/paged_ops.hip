// The paged cache's bookkeeping and what writes it: the plan of a step (block
// tables, positions, slots), the per-head norm + rotation of queries and keys
// with the cache write, and rows written to a cache or read back as they are.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "kv_quant.h"
#include "paged.h"
#include "paged_device.h"

namespace mlq {
namespace {

// ---- the plan -----------------------------------------------------------------
// held = ceil(L / P) pages of a sequence, need = ceil((L + a) / P) - held new
// ones; releases are pushed on the stack at the prefix sum of their counts,
// needs popped at theirs, so the result is that of a loop over sequences. One
// workgroup walks the sequences in tiles of a thread each. Latency is all of it:
// the prefix sums run in registers with one barrier a tile, a thread writes a
// few pages and rows of its sequence itself and the wave many of them, and a
// row takes its page from the stack or the table as they were, not from what
// was just written. 48 sequences, a token each: 3.4 us in a graph.
// The scanning workgroup writes the rows itself where there are few of them or
// about one a sequence, else a second launch over the whole chip does (us in a
// graph, itself and second launch: a token each for 1000 sequences 5.1 and 8.7,
// for 3000 15.4 and 19.4; 100 prompts of up to 60 tokens 17.3 and 7.6).
constexpr int kPlanFewRows = 1024, kPlanMostRows = 16384;
constexpr int kPlanOwn = 8;  // pages or rows of a sequence that its own thread writes

// Last i with start[i] <= r; start[0] <= r. The one that r falls into: an
// empty sequence starts where the next one does.
__device__ __forceinline__ int find_start(const int* start, int n, int r) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct PlanSeq {
  int len, add, held, need, freed;
  bool bad, ended;
};
__device__ __forceinline__ PlanSeq plan_seq(const PlanArgs& a, int i) {
  PlanSeq s = {};
  if (i >= a.n_seqs) return s;
  const int64_t cap = (int64_t)a.max_pages << a.page_shift;
  const int len = a.lengths[i], n = a.n_new[i];
  if (n < -1 || len < 0 || (int64_t)len + max(n, 0) > cap) {
    s.bad = true;
    return s;
  }
  const int up = (1 << a.page_shift) - 1;
  s.len = len;
  s.add = max(n, 0);
  s.ended = n < 0;
  s.held = (int)(((int64_t)len + up) >> a.page_shift);
  s.freed = n < 0 ? s.held : 0;
  s.need = n < 0 ? 0 : (int)(((int64_t)len + n + up) >> a.page_shift) - s.held;
  return s;
}

// Sums of rows, needed and released pages: before a thread's sequence, or of
// all. 64 bits: bad counts may add up to anything.
struct PlanSums {
  int64_t add, need, freed;
  int bad;
};

// A tile's prefix sums (exclusive) and totals; `lds`: a PlanSums per wave.
template <int T>
__device__ __forceinline__ PlanSums plan_scan(const PlanSeq& s, PlanSums* lds, PlanSums* total) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t add = wave_scan64(s.add), need = wave_scan64(s.need), freed = wave_scan64(s.freed);
  const bool bad = __any(s.bad);
  __syncthreads();  // (an earlier scan's readers are done with lds)
  if ((threadIdx.x & 63) == 63) lds[wave] = {add, need, freed, bad};
  __syncthreads();
  // every wave scans the waves' sums, a lane each
  const int lane = threadIdx.x & 63;
  const PlanSums mine = lane < T / 64 ? lds[lane] : PlanSums{0, 0, 0, 0};
  const int64_t adds = wave_scan64(mine.add), needs = wave_scan64(mine.need),
                freeds = wave_scan64(mine.freed);
  *total = {readlane64(adds, 63), readlane64(needs, 63), readlane64(freeds, 63), __any(mine.bad)};
  PlanSums before = {add - s.add, need - s.need, freed - s.freed, 0};
  if (wave > 0) {
    before.add += readlane64(adds, wave - 1);
    before.need += readlane64(needs, wave - 1);
    before.freed += readlane64(freeds, wave - 1);
  }
  return before;
}

template <int T>
__global__ __launch_bounds__(T) void plan_kernel(PlanArgs a, int inline_rows) {
  __shared__ PlanSums scan_lds[T / 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int free0 = *a.n_free;
  const PlanSeq s0 = plan_seq(a, tid);

  PlanSums all, tile0;
  const PlanSums before0 = plan_scan<T>(s0, scan_lds, &tile0);
  all = tile0;
  for (int i0 = T; i0 < a.n_seqs; i0 += T) {
    PlanSums t;
    plan_scan<T>(plan_seq(a, i0 + tid), scan_lds, &t);
    all.add += t.add;
    all.need += t.need;
    all.freed += t.freed;
    all.bad |= t.bad;
  }
  const int64_t avail = free0 + all.freed;
  int status = MLQ_PLAN_OK;
  if (all.bad != 0 || free0 < 0 || avail > a.n_pages) status = MLQ_PLAN_BAD_COUNT;
  else if (all.add > a.max_rows) status = MLQ_PLAN_ROWS;
  else if (all.need > avail) status = MLQ_PLAN_PAGES;
  const bool ok = status == MLQ_PLAN_OK;

  const int64_t width = a.max_pages;
  // f(i, k, n) for the n items of each lane's i: a few by the lane itself, many
  // by the whole wave, lane after lane.
  auto each = [&](int n, auto item) __attribute__((always_inline)) {
    if (n <= kPlanOwn)
      for (int k = 0; k < n; ++k) item(k, -1);
    uint64_t many = __ballot(n > kPlanOwn);
    while (many != 0) {
      const int from = __builtin_ctzll(many);
      many &= many - 1;
      const int count = __builtin_amdgcn_readlane(n, from);
      for (int k = lane; k < count; k += 64) item(k, from);
    }
  };
  // a lane's value, or that of the lane whose items the wave does
  auto of = [](int v, int from) __attribute__((always_inline)) {
    return from < 0 ? v : __builtin_amdgcn_readlane(v, from < 0 ? 0 : from);
  };
  if (ok && all.freed > 0) {
    int base = free0;
    for (int i0 = 0; i0 < a.n_seqs; i0 += T) {
      PlanSeq s = s0;
      PlanSums total = tile0, before = before0;
      if (i0 > 0) {
        s = plan_seq(a, i0 + tid);
        before = plan_scan<T>(s, scan_lds, &total);
      }
      const int seq = i0 + tid, at = base + (int)before.freed;
      each(s.freed, [&](int k, int from) {
        a.free_pages[of(at, from) + k] = a.block_table[of(seq, from) * width + k];
      });
      base += (int)total.freed;
    }
    __syncthreads();
  }
  const int page_mask = (1 << a.page_shift) - 1;
  int popped = 0, row0 = 0;
  for (int i0 = 0; i0 < a.n_seqs; i0 += T) {
    const int seq = i0 + tid;
    PlanSeq s = s0;
    PlanSums total = tile0, before = before0;
    if (i0 > 0) {
      s = plan_seq(a, seq);
      before = plan_scan<T>(s, scan_lds, &total);
    }
    if (seq < a.n_seqs) {
      a.row_start[seq] = ok ? row0 + (int)before.add : 0;
      a.lengths_out[seq] = ok ? (s.ended ? 0 : s.len + s.add) : a.lengths[seq];
    }
    if (!ok) continue;
    const int rank = popped + (int)before.need, row = row0 + (int)before.add;
    auto pop = [&](int r) { return a.free_pages[avail - 1 - r]; };
    each(s.need, [&](int k, int from) {
      a.block_table[of(seq, from) * width + of(s.held, from) + k] = pop(of(rank, from) + k);
    });
    if (inline_rows)
      each(s.add, [&](int k, int from) {
        const int pos = of(s.len, from) + k, j = pos >> a.page_shift, held = of(s.held, from);
        const int page = j < held ? a.block_table[of(seq, from) * width + j] : pop(of(rank, from) + j - held);
        const int r = of(row, from) + k;
        a.positions[r] = pos;
        a.slots[r] = ((int64_t)page << a.page_shift) + (pos & page_mask);
      });
    popped += (int)total.need;
    row0 += (int)total.add;
  }
  if (inline_rows)
    for (int r = row0 + tid; r < a.max_rows; r += T) {
      a.positions[r] = -1;
      a.slots[r] = -1;
    }
  if (tid == 0) {
    a.row_start[a.n_seqs] = row0;
    *a.n_free_out = ok ? (int)(avail - all.need) : free0;
    *a.status = status;
  }
}

// A thread per row, from what plan_kernel wrote.
__global__ __launch_bounds__(256) void plan_rows_kernel(PlanArgs a) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= a.max_rows) return;
  int pos = -1;
  int64_t slot = -1;
  if (r < a.row_start[a.n_seqs]) {
    const int i = find_start(a.row_start, a.n_seqs, r);
    pos = a.lengths_out[i] - (a.row_start[i + 1] - r);
    const int page = a.block_table[(size_t)i * a.max_pages + (pos >> a.page_shift)];
    slot = ((int64_t)page << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
  }
  a.positions[r] = pos;
  a.slots[r] = slot;
}

// ---- norm, rotation and cache write ---------------------------------------------
// A head lies in LG lanes of 4 elements (LG a power of two >= head_dim / 4), so
// its mean square is a sum over lanes and pairs are in a lane (interleaved)
// or rot / 8 lanes apart. The row's angles are computed once per workgroup,
// in 64 bits up to the quarter turn: pos * f in 32 bits would be off by
// 2^-24 pos radians.
constexpr int kRotaryThreads = 256, kRotaryMaxHalf = 128;
// Queries past half of the last-level cache's 256 MB are written past the
// caches: what reads them finds them gone anyway (8000 rows, 64 heads on 8 of
// 128, bf16: 129 -> 122 us, 5.1 TB/s; the inputs are read through the caches,
// where the projection may have left them: 701 rows 8.2 us, else 9.4).
constexpr int64_t kRotaryStreamBytes = (int64_t)128 << 20;

__device__ __forceinline__ void store_kv(void* base, int type, int64_t at, float4 x) {
  typedef float v4 __attribute__((ext_vector_type(4)));
  typedef _Float16 hv4 __attribute__((ext_vector_type(4)));
  typedef __bf16 bv4 __attribute__((ext_vector_type(4)));
  const v4 f = {x.x, x.y, x.z, x.w};
  if (type == MLQ_KV_F32) *(v4*)((float*)base + at) = f;
  else if (type == MLQ_KV_F16) *(hv4*)((_Float16*)base + at) = __builtin_convertvector(f, hv4);
  else *(bv4*)((__bf16*)base + at) = __builtin_convertvector(f, bv4);
}

// A head's row of 4 or 8 bits from 4 elements a lane (lane l of the head's has
// dims 4l ..): a block lies in 8 lanes, and a lane's two units in two places, stored
// a unit at a time. 8000 rows of 32 heads on 8 of 128 take 69.6 us with a bf16 cache,
// 76.0 with q4 and 79.8 with q8 (their bytes at a copy's rate: 70), 48 of 28 on 4 3.6,
// 4.3 and 4.2.
template <typename Q>
__device__ __forceinline__ void store_quantised(char* row, int l, int hd, float4 x) {
  const int nb = kv_blocks(hd), b = l >> 3, d = 4 * l;
  const float v[4] = {x.x, x.y, x.z, x.w};
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (d + c < hd) kv_range(v[c], lo, hi);
  lo = -row_max<8>(-lo);
  hi = row_max<8>(hi);
  if (lo > hi) lo = hi = 0.0f;  // (a block behind the head's end)
  const KvScale s = kv_scale<Q>(lo, hi);
  const float inv = __builtin_amdgcn_rcpf((float)s.d);
  int code[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) code[c] = d + c < hd ? kv_code<Q>(v[c], s, inv) : Q::kMiddle;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int unit = (2 * (l & 7) + c) * nb + b;
    if constexpr (Q::kUnit == 1) ((uint8_t*)row)[unit] = (uint8_t)(code[2 * c] | code[2 * c + 1] << 4);
    else ((uint16_t*)row)[unit] = (uint16_t)(code[2 * c] | code[2 * c + 1] << 8);
  }
  if ((l & 7) == 0) *(KvScale*)(row + 16 * nb * Q::kUnit + 4 * b) = s;
}

// Q: KvQ4 or KvQ8 for a cache of those bits, void for the others. The rotated
// fp32 key is quantised, the one that k_out holds.
template <int LG, typename Q>
__global__ __launch_bounds__(kRotaryThreads) void qk_norm_rope_kernel(RotaryArgs a) {
  constexpr bool QUANT = !std::is_void<Q>::value;
  __shared__ float2 turn[kRotaryMaxHalf];  // cos, sin, times the magnitude
  const int row = blockIdx.x;
  const int pos = a.positions[row];
  if (pos < 0) return;
  const int half = a.rot >> 1;
  if ((int)threadIdx.x < half) {
    // quarter turns: pos * f * 2 / pi = n + x, x in [-1/2, 1/2]
    const double t = (double)pos * a.freqs[threadIdx.x] * 0.63661977236758134308;
    const double n = rint(t);
    float s, c;
    sincospif(0.5f * (float)(t - n), &s, &c);
    const int quarter = (int)((int64_t)n & 3);
    const float c1 = quarter & 1 ? -s : c, s1 = quarter & 1 ? c : s;
    const float m = quarter & 2 ? -a.magnitude : a.magnitude;
    turn[threadIdx.x] = float2{m * c1, m * s1};
  }
  __syncthreads();
  const int l = threadIdx.x % LG, d = 4 * l;
  const bool in = d < a.hd;
  const int n_kv_out = a.keys != nullptr ? 2 * a.n_kv : a.n_kv;
  int64_t slot = -1;
  if (a.keys != nullptr) {
    slot = a.slots[row];
    if (slot >= a.n_slots) slot = -1;
  }
  const int64_t page = slot >> a.page_shift, off = slot & (((int64_t)1 << a.page_shift) - 1);
  const bool quads = (half & 3) == 0;
  const int groups = kRotaryThreads / LG * gridDim.y;
  for (int h = blockIdx.y * (kRotaryThreads / LG) + threadIdx.x / LG; h < a.n_heads + n_kv_out;
       h += groups) {
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
    const int kh = h - a.n_heads - (is_v ? a.n_kv : 0);  // kv head of k and v
    const float* src = is_q ? a.q + row * a.q_stride + (int64_t)h * a.hd
                            : (is_v ? a.v + row * a.v_stride : a.k + row * a.k_stride) +
                                  (int64_t)kh * a.hd;
    float4 x = in ? *(const float4*)(src + d) : float4{0.0f, 0.0f, 0.0f, 0.0f};
    const int64_t at = ((page * a.n_kv + kh) << a.page_shift) * a.hd + off * a.hd + d;
    auto quantise = [&](void* base) {
      if constexpr (QUANT)
        store_quantised<Q>((char*)base + (((page * a.n_kv + kh) << a.page_shift) + off) * kv_row_bytes(Q::kType, a.hd), l, a.hd, x);
    };
    if (is_v) {
      if constexpr (QUANT) {
        if (slot >= 0) quantise(a.values);
      } else {
        if (in && slot >= 0) store_kv(a.values, a.type, at, x);
      }
      continue;
    }
    const float* w = is_q ? a.q_norm : a.k_norm;
    float inv = 1.0f;
    if (w != nullptr) {
      const float ss = row_sum<LG>(x.x * x.x + x.y * x.y + (x.z * x.z + x.w * x.w));
      inv = 1.0f / sqrtf(ss / (float)a.hd + a.eps);
      const float4 g = in ? *(const float4*)(w + d) : float4{0.0f, 0.0f, 0.0f, 0.0f};
      x = float4{x.x * g.x * inv, x.y * g.y * inv, x.z * g.z * inv, x.w * g.w * inv};
    }
    if (a.rot > 0) {
      if (a.neox) {
        float p[4], v[4] = {x.x, x.y, x.z, x.w};
        if (quads) {  // the partner is the same component of another lane
          const int other = d < half ? l + (half >> 2) : l - (half >> 2);
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] = __shfl(v[c], other, LG);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int e = d + c < half ? d + c + half : d + c - half;
            p[c] = 0.0f;
            if (d + c < a.rot) p[c] = w != nullptr ? src[e] * w[e] * inv : src[e];
          }
          // (in place: no lane stores before its partners have read)
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (d + c < a.rot) {
            const float2 t = turn[d + c < half ? d + c : d + c - half];
            v[c] = d + c < half ? v[c] * t.x - p[c] * t.y : v[c] * t.x + p[c] * t.y;
          }
        x = float4{v[0], v[1], v[2], v[3]};
      } else {
        if (d < a.rot) {
          const float2 t = turn[2 * l];
          const float y = x.x * t.x - x.y * t.y;
          x.y = x.x * t.y + x.y * t.x;
          x.x = y;
        }
        if (d + 2 < a.rot) {
          const float2 t = turn[2 * l + 1];
          const float y = x.z * t.x - x.w * t.y;
          x.w = x.z * t.y + x.w * t.x;
          x.z = y;
        }
      }
    }
    if constexpr (QUANT)
      if (!is_q && slot >= 0) quantise(a.keys);
    if (!in) continue;
    if (is_q) {
      float* to = a.q_out + row * a.q_out_stride + (int64_t)h * a.hd + d;
      if (a.stream) __builtin_nontemporal_store(f4_t{x.x, x.y, x.z, x.w}, (f4_t*)to);
      else *(float4*)to = x;
    } else {
      if (a.k_out != nullptr)
        *(float4*)(a.k_out + row * a.k_out_stride + (int64_t)kh * a.hd + d) = x;
      if constexpr (!QUANT)
        if (slot >= 0) store_kv(a.keys, a.type, at, x);
    }
  }
}

// ---- rows written and read back ----------------------------------------------------
// Bytes bound both: for each element 4 in or out and the cache's share. 16
// lanes have a head, lane i dims 2i and 2i + 1 of every block: loads and stores
// of 128 bytes a block, and the lane's units lie side by side. Quantising is the
// next: 8000 rows of 8 heads of 128 to 4 bits 41.9 us with a block's scale worked
// out in every lane and divisions, 37.9 with one a lane and a reciprocal.
constexpr int kRowsThreads = 256, kRowsGroup = 16;

// Which (row, kv head, keys or values) the x-th is.
struct RowItem {
  int64_t row;
  int head;
  bool is_v;
};
__device__ __forceinline__ RowItem row_item(int64_t x, int n_kv) {
  const int64_t row = quotient(x, 2 * n_kv);
  const int of = (int)(x - row * 2 * n_kv);
  return {row, of < n_kv ? of : of - n_kv, of >= n_kv};
}
// The place of a row's head in the cache, in rows; -1: outside.
__device__ __forceinline__ int64_t row_place(const RowsArgs& a, const RowItem& it) {
  const int64_t slot = a.slots[it.row];
  if (slot < 0 || slot >= a.n_slots) return -1;
  const int64_t page = slot >> a.page_shift;
  return ((page * a.n_kv + it.head) << a.page_shift) + (slot & (((int64_t)1 << a.page_shift) - 1));
}

// Lane B of each 16 lanes' value.
template <int B>
__device__ __forceinline__ int row_lane(int x) {
  return __builtin_amdgcn_mov_dpp(x, 0x150 + B, 0xF, 0xF, false);
}
// f of the constants 0 .. N - 1.
template <int N, typename F>
__device__ __forceinline__ void blocks_in_order(F f) {
  if constexpr (N > 1) blocks_in_order<N - 1>(f);
  f(std::integral_constant<int, N - 1>{});
}

template <typename Q, int NB>
__global__ __launch_bounds__(kRowsThreads) void write_rows_quantised_kernel(RowsArgs a) {
  constexpr int kBytes = NB * (16 * Q::kUnit + 4);
  const int i = threadIdx.x % kRowsGroup;
  const int64_t x = (int64_t)blockIdx.x * (kRowsThreads / kRowsGroup) + threadIdx.x / kRowsGroup;
  if (x >= (int64_t)a.rows * 2 * a.n_kv) return;
  const RowItem it = row_item(x, a.n_kv);
  const int64_t at = row_place(a, it);
  if (at < 0) return;
  const float* src = (it.is_v ? a.v + it.row * a.v_stride : a.k + it.row * a.k_stride) + (int64_t)it.head * a.hd;
  float2 v[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) v[b] = 32 * b + 2 * i < a.hd ? *(const float2*)(src + 32 * b + 2 * i) : float2{0.0f, 0.0f};
  // (lane i works out block i % NB's scale: the others have it by a lane's broadcast)
  float mine_lo = INFINITY, mine_hi = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float lo = INFINITY, hi = -INFINITY;
    if (32 * b + 2 * i < a.hd) {  // (both dims: head dims are even)
      kv_range(v[b].x, lo, hi);
      kv_range(v[b].y, lo, hi);
    }
    lo = -row_max<16>(-lo);
    hi = row_max<16>(hi);
    if (i % NB == b) {
      mine_lo = lo;
      mine_hi = hi;
    }
  }
  if (mine_lo > mine_hi) mine_lo = mine_hi = 0.0f;  // (a block behind the head's end)
  const KvScale mine = kv_scale<Q>(mine_lo, mine_hi);
  const float mine_inv = __builtin_amdgcn_rcpf((float)mine.d);
  uint32_t unit[NB];
  blocks_in_order<NB>([&](auto block) __attribute__((always_inline)) {
    constexpr int b = decltype(block)::value;
    const bool in = 32 * b + 2 * i < a.hd;
    const KvScale s = __builtin_bit_cast(KvScale, row_lane<b>(__builtin_bit_cast(int, mine)));
    const float inv = __builtin_bit_cast(float, row_lane<b>(__builtin_bit_cast(int, mine_inv)));
    const int c0 = in ? kv_code<Q>(v[b].x, s, inv) : Q::kMiddle, c1 = in ? kv_code<Q>(v[b].y, s, inv) : Q::kMiddle;
    unit[b] = c0 | c1 << (4 * Q::kUnit);
    v[b] = float2{kv_value<Q>(c0, s), kv_value<Q>(c1, s)};
  });
  char* row = (char*)(it.is_v ? a.values : a.keys) + at * kBytes;
  uint32_t w[(NB * Q::kUnit + 3) / 4] = {};
#pragma unroll
  for (int b = 0; b < NB; ++b) w[b * Q::kUnit / 4] |= unit[b] << (8 * (b * Q::kUnit % 4));
  char* to = row + i * NB * Q::kUnit;
  if constexpr (NB * Q::kUnit == 2) *(uint16_t*)to = (uint16_t)w[0];
  else if constexpr (NB * Q::kUnit == 4) *(uint32_t*)to = w[0];
  else if constexpr (NB * Q::kUnit == 8) *(u32x2_t*)to = u32x2_t{w[0], w[1]};
  else *(u32x4_t*)to = u32x4_t{w[0], w[1], w[2], w[3]};
  if (i < NB) *(KvScale*)(row + 16 * NB * Q::kUnit + 4 * i) = mine;
  float* out = it.is_v ? a.v_out : a.k_out;
  if (out == nullptr) return;
  out += it.row * (it.is_v ? a.v_out_stride : a.k_out_stride) + (int64_t)it.head * a.hd;
#pragma unroll
  for (int b = 0; b < NB; ++b)
    if (32 * b + 2 * i < a.hd) *(float2*)(out + 32 * b + 2 * i) = v[b];
}

template <typename Q, int NB>
__global__ __launch_bounds__(kRowsThreads) void read_rows_quantised_kernel(RowsArgs a) {
  constexpr int kBytes = NB * (16 * Q::kUnit + 4), W = NB * Q::kUnit;
  const int i = threadIdx.x % kRowsGroup;
  const int64_t x = (int64_t)blockIdx.x * (kRowsThreads / kRowsGroup) + threadIdx.x / kRowsGroup;
  if (x >= (int64_t)a.rows * 2 * a.n_kv) return;
  const RowItem it = row_item(x, a.n_kv);
  const int64_t at = row_place(a, it);
  if (at < 0) return;
  const char* row = (const char*)(it.is_v ? a.values : a.keys) + at * kBytes;
  uint32_t w[(W + 3) / 4];
  const char* from = row + i * W;
  if constexpr (W == 2) {
    w[0] = *(const uint16_t*)from;
  } else {
#pragma unroll
    for (int j = 0; j < W / 4; ++j) w[j] = ((const uint32_t*)from)[j];
  }
  float* out = (it.is_v ? a.v_out + it.row * a.v_out_stride : a.k_out + it.row * a.k_out_stride) + (int64_t)it.head * a.hd;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (32 * b + 2 * i >= a.hd) break;
    const KvScale s = *(const KvScale*)(row + 16 * W + 4 * b);
    constexpr int kMask = Q::kLevels;
    const uint32_t unit = w[b * Q::kUnit / 4] >> (8 * (b * Q::kUnit % 4));
    *(float2*)(out + 32 * b + 2 * i) =
        float2{kv_value<Q>(unit & kMask, s), kv_value<Q>(unit >> (4 * Q::kUnit) & kMask, s)};
  }
}

// Caches of 16 and 32 bits: 4 elements a lane. 8 heads of 128, one buffer again and
// again: 8000 rows written, with their values given back, 29.8 us fp32, 25.1 bf16;
// 16000 read 34.2 and 24.6.
__device__ __forceinline__ float4 load_kv(const void* base, int type, int64_t at) {
  typedef float v4 __attribute__((ext_vector_type(4)));
  typedef _Float16 hv4 __attribute__((ext_vector_type(4)));
  typedef __bf16 bv4 __attribute__((ext_vector_type(4)));
  v4 f;
  if (type == MLQ_KV_F32) f = *(const v4*)((const float*)base + at);
  else if (type == MLQ_KV_F16) f = __builtin_convertvector(*(const hv4*)((const _Float16*)base + at), v4);
  else f = __builtin_convertvector(*(const bv4*)((const __bf16*)base + at), v4);
  return float4{f.x, f.y, f.z, f.w};
}
template <bool WRITE>
__global__ __launch_bounds__(kRowsThreads) void plain_rows_kernel(RowsArgs a) {
  const int64_t x = (int64_t)blockIdx.x * (kRowsThreads / kRowsGroup) + threadIdx.x / kRowsGroup;
  if (x >= (int64_t)a.rows * 2 * a.n_kv) return;
  const RowItem it = row_item(x, a.n_kv);
  const int64_t at = row_place(a, it);
  if (at < 0) return;
  void* base = it.is_v ? a.values : a.keys;
  float* out = it.is_v ? a.v_out : a.k_out;
  if (out != nullptr) out += it.row * (it.is_v ? a.v_out_stride : a.k_out_stride) + (int64_t)it.head * a.hd;
  const float* src = nullptr;
  if constexpr (WRITE)
    src = (it.is_v ? a.v + it.row * a.v_stride : a.k + it.row * a.k_stride) + (int64_t)it.head * a.hd;
  for (int d = 4 * (threadIdx.x % kRowsGroup); d < a.hd; d += 4 * kRowsGroup) {
    float4 f;
    if constexpr (WRITE) {
      f = *(const float4*)(src + d);
      if (a.type == MLQ_KV_F16) f = float4{(float)(_Float16)f.x, (float)(_Float16)f.y, (float)(_Float16)f.z, (float)(_Float16)f.w};
      else if (a.type == MLQ_KV_BF16) f = float4{(float)(__bf16)f.x, (float)(__bf16)f.y, (float)(__bf16)f.z, (float)(__bf16)f.w};
      store_kv(base, a.type, at * a.hd + d, f);
    } else {
      f = load_kv(base, a.type, at * a.hd + d);
    }
    if (out != nullptr) *(float4*)(out + d) = f;
  }
}

template <typename Q, int NB>
void rows_launch(const RowsArgs& a, bool write, dim3 grid, hipStream_t stream) {
  if (write) hipLaunchKernelGGL((write_rows_quantised_kernel<Q, NB>), grid, dim3(kRowsThreads), 0, stream, a);
  else hipLaunchKernelGGL((read_rows_quantised_kernel<Q, NB>), grid, dim3(kRowsThreads), 0, stream, a);
}
template <typename Q>
void rows_launch_blocks(const RowsArgs& a, bool write, dim3 grid, hipStream_t stream) {
  switch (kv_blocks(a.hd)) {
    case 2: return rows_launch<Q, 2>(a, write, grid, stream);
    case 4: return rows_launch<Q, 4>(a, write, grid, stream);
    default: return rows_launch<Q, 8>(a, write, grid, stream);
  }
}

template <int LG, typename Q>
void rotary_launch(RotaryArgs a, hipStream_t stream) {
  const int heads = a.n_heads + (a.keys != nullptr ? 2 : 1) * a.n_kv;
  const int per = kRotaryThreads / LG;
  // few rows: a row's heads over several workgroups, each with its own angles
  const int most = (heads + per - 1) / per;
  const int split = std::min(most, std::max(1, 2 * device_cus() / a.rows));
  a.stream = (int64_t)a.rows * a.n_heads * a.hd * 4 > kRotaryStreamBytes;
  hipLaunchKernelGGL((qk_norm_rope_kernel<LG, Q>), dim3(a.rows, split), dim3(kRotaryThreads), 0,
                     stream, a);
}
// (a row of 4 or 8 bits has two blocks at least)
template <typename Q>
void rotary_launch_hd(const RotaryArgs& a, hipStream_t stream) {
  if constexpr (std::is_void<Q>::value)
    if (a.hd <= 32) return rotary_launch<8, Q>(a, stream);
  if (a.hd <= 64) rotary_launch<16, Q>(a, stream);
  else if (a.hd <= 128) rotary_launch<32, Q>(a, stream);
  else rotary_launch<64, Q>(a, stream);
}

}  // namespace

hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t stream) {
  const bool rows = a.max_rows <= kPlanFewRows ||
                    (a.max_rows <= kPlanMostRows && a.max_rows <= 2 * (int64_t)a.n_seqs);
  // (a workgroup of the sequences' size: a barrier of four waves costs less
  // than one of sixteen)
  if (a.n_seqs <= 256 && a.max_rows <= 1024)
    hipLaunchKernelGGL(plan_kernel<256>, dim3(1), dim3(256), 0, stream, a, rows ? 1 : 0);
  else
    hipLaunchKernelGGL(plan_kernel<1024>, dim3(1), dim3(1024), 0, stream, a, rows ? 1 : 0);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || rows) return e;
  hipLaunchKernelGGL(plan_rows_kernel, dim3((unsigned)(((int64_t)a.max_rows + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_qk_norm_rope(const RotaryArgs& a, hipStream_t stream) {
  if (a.keys != nullptr && a.type == MLQ_KV_Q4) rotary_launch_hd<KvQ4>(a, stream);
  else if (a.keys != nullptr && a.type == MLQ_KV_Q8) rotary_launch_hd<KvQ8>(a, stream);
  else rotary_launch_hd<void>(a, stream);
  return hipGetLastError();
}

int64_t rows_groups(int rows, int n_kv) {
  constexpr int per = kRowsThreads / kRowsGroup;
  return ((int64_t)rows * 2 * n_kv + per - 1) / per;
}

hipError_t launch_paged_rows(const RowsArgs& a, bool write, hipStream_t stream) {
  const dim3 grid((unsigned)rows_groups(a.rows, a.n_kv));
  if (a.type == MLQ_KV_Q4) rows_launch_blocks<KvQ4>(a, write, grid, stream);
  else if (a.type == MLQ_KV_Q8) rows_launch_blocks<KvQ8>(a, write, grid, stream);
  else if (write) hipLaunchKernelGGL(plain_rows_kernel<true>, grid, dim3(kRowsThreads), 0, stream, a);
  else hipLaunchKernelGGL(plain_rows_kernel<false>, grid, dim3(kRowsThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mlq
