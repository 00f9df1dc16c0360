// The paged cache's bookkeeping and what writes it: the plan of a step (block
// tables, positions, slots) and the per-head norm + rotation of queries and
// keys with the cache write.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "device_common.h"
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

template <int LG>
__global__ __launch_bounds__(kRotaryThreads) void qk_norm_rope_kernel(RotaryArgs a) {
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
    if (is_v) {
      if (in && slot >= 0) store_kv(a.values, a.type, at, x);
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
    if (!in) continue;
    if (is_q) {
      float* to = a.q_out + row * a.q_out_stride + (int64_t)h * a.hd + d;
      if (a.stream) __builtin_nontemporal_store(f4_t{x.x, x.y, x.z, x.w}, (f4_t*)to);
      else *(float4*)to = x;
    } else {
      if (a.k_out != nullptr)
        *(float4*)(a.k_out + row * a.k_out_stride + (int64_t)kh * a.hd + d) = x;
      if (slot >= 0) store_kv(a.keys, a.type, at, x);
    }
  }
}

template <int LG>
void rotary_launch(RotaryArgs a, hipStream_t stream) {
  const int heads = a.n_heads + (a.keys != nullptr ? 2 : 1) * a.n_kv;
  const int per = kRotaryThreads / LG;
  // few rows: a row's heads over several workgroups, each with its own angles
  const int most = (heads + per - 1) / per;
  const int split = std::min(most, std::max(1, 2 * device_cus() / a.rows));
  a.stream = (int64_t)a.rows * a.n_heads * a.hd * 4 > kRotaryStreamBytes;
  hipLaunchKernelGGL(qk_norm_rope_kernel<LG>, dim3(a.rows, split), dim3(kRotaryThreads), 0,
                     stream, a);
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
  if (a.hd <= 32) rotary_launch<8>(a, stream);
  else if (a.hd <= 64) rotary_launch<16>(a, stream);
  else if (a.hd <= 128) rotary_launch<32>(a, stream);
  else rotary_launch<64>(a, stream);
  return hipGetLastError();
}

}  // namespace mlq
