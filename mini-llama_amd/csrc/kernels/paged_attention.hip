// Attention over a paged cache of 16 and 32 bits, what joins the pieces of a
// decode launch, and the plans of both.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "paged_attention.h"

namespace mlq {
namespace {

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

}  // namespace

size_t plan_paged_decode(PagedAttnArgs& a) {
  const int64_t n_tiles = (int64_t)a.n_kv * ((a.group + 15) / 16);
  const int keys = a.type == MLQ_KV_F32 ? 16 : 32, unit = kDecWaves * keys;
  const int64_t units = (a.max_len + (int64_t)unit - 1) / unit;  // of a sequence
  const int cus = device_cus(), most_seqs = kv_quantised(a.type) ? paged_decode_quantised_seqs() : kDecMaxSeqs;
  // sequences of a launch: their prefix sums lie in LDS and fit 32 bits
  a.launch_seqs = (int)std::min((int64_t)std::min(a.n_seqs, most_seqs), std::max(((int64_t)1 << 28) / units, (int64_t)1));
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
  const int64_t pieces = std::min(a.n_seqs, most_seqs) * n_tiles;
  const int per_cu = kv_quantised(a.type) ? paged_decode_quantised_per_cu(a) : dec_per_cu(a.hd, pieces, cus);
  a.ranges = (int)std::min(a.launch_seqs * n_tiles * units, (int64_t)per_cu * cus);
  const size_t tg = std::min(a.group, 16);
  return dec_header(std::min(a.n_seqs, most_seqs)) + dec_align((size_t)2 * a.ranges * tg * 8) +
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
    else if (kv_quantised(a.type)) launch_paged_decode_quantised(a, stream);
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
  if (kv_quantised(a.type)) return launch_paged_prefill_quantised(a, stream);
  return prefill_launch_type<__bf16>(a, stream);
}

}  // namespace mlq
