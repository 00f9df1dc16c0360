// Attention over a paged key-value cache (contracts in include/mlq.h): one new
// token of each sequence (decode) and many new tokens of each (prefill).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "device_common.h"
#include "paged.h"

namespace mlq {
namespace {

// One wave per (row, query head): a lane scores a key of a tile of 64 against
// q in LDS, then takes head dims lane, lane + 64, .. of the output.
template <typename T>
__global__ __launch_bounds__(64) void paged_rows_kernel(PagedAttnArgs a, int decode) {
  __shared__ __align__(16) float qs[256];
  __shared__ float ps[64];
  __shared__ int64_t at[64];
  const int lane = threadIdx.x, head = blockIdx.y, kvh = head / a.group;
  int seq, row, pos;
  if (decode) {
    seq = blockIdx.x;
    row = seq;
    if (a.row_start != nullptr) {
      row = a.row_start[seq + 1] - 1;
      if (row < a.row_start[seq]) return;
    }
    pos = a.lengths[seq] - 1;
  } else {
    row = blockIdx.x;
    if (row >= a.row_start[a.n_seqs]) return;
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.row_start[mid] <= row) lo = mid;
      else hi = mid;
    }
    seq = lo;
    pos = a.lengths[seq] - (a.row_start[seq + 1] - row);
  }
  if (row < 0 || row >= a.max_rows) return;
  const int len = pos + 1;
  const float* q = a.q + row * a.q_stride + (int64_t)head * a.hd;
  for (int d = lane; d < a.hd; d += 64) qs[d] = q[d];
  __syncthreads();
  float m = -INFINITY, l = 0.0f, acc[4] = {};
  const float slope = a.slopes != nullptr ? a.slopes[head] : 0.0f;
  bool bad = len > a.max_len || a.lengths[seq] > a.max_len;
  const int first = a.window > 0 ? max(0, len - a.window) : 0;
  for (int t0 = first; t0 < len && !bad; t0 += 64) {
    const int t = t0 + lane;
    float s = -INFINITY;
    int64_t base = 0;
    if (t < len) {
      const int page = a.block_table[(size_t)seq * a.max_pages + (t >> a.page_shift)];
      if (page < 0 || page >= a.n_pages) bad = true;
      else {
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
    __syncthreads();
    ps[lane] = p;
    at[lane] = base;
    __syncthreads();
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
  for (int j = 0; j < 4; ++j)
    if (lane + 64 * j < a.hd)
      out[lane + 64 * j] = bad ? __builtin_nanf("") : len > 0 ? acc[j] / l : 0.0f;
}

hipError_t rows_launch(const PagedAttnArgs& a, int rows, int decode, hipStream_t stream) {
  const dim3 grid(rows, a.n_kv * a.group);
  if (a.type == MLQ_KV_F32)
    hipLaunchKernelGGL(paged_rows_kernel<float>, grid, dim3(64), 0, stream, a, decode);
  else if (a.type == MLQ_KV_F16)
    hipLaunchKernelGGL(paged_rows_kernel<_Float16>, grid, dim3(64), 0, stream, a, decode);
  else
    hipLaunchKernelGGL(paged_rows_kernel<__bf16>, grid, dim3(64), 0, stream, a, decode);
  return hipGetLastError();
}

}  // namespace

size_t plan_paged_decode(PagedAttnArgs& a) {
  a.splits = 1;
  a.part_len = a.max_len;
  return 0;
}

hipError_t launch_paged_decode(const PagedAttnArgs& a, hipStream_t stream) {
  return rows_launch(a, a.n_seqs, 1, stream);
}

hipError_t launch_paged_prefill(const PagedAttnArgs& a, hipStream_t stream) {
  return rows_launch(a, a.max_rows, 0, stream);
}

}  // namespace mlq
