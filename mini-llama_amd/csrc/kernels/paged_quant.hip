// Attention over a paged cache of 4 and 8 bits: the decode kernel of its own, and
// the prefill kernel's instances.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "paged_attention.h"

namespace mlq {
namespace {

// ---- decode ------------------------------------------------------------------------
// The cut, the pieces and the join are those of the other types
// (paged_attention.h), and so are both products' layouts; what differs:
//  - Codes less their middle are whole numbers that fp16 holds exactly, so both
//    products run over codes on fp16 instructions, with q and the weights in
//    two parts of 11 bits as for an fp16 cache. A block's sum over a key's codes is
//    multiplied by the key's d in fp32 and m times the sum of q's block added; weights
//    are multiplied by d before they are split, and m times them summed beside.
//  - A weight times d has the largest d so far as its scale: the power of two
//    under which it is split follows that one's exponent, and what falls below
//    fp16's subnormals is 2^-39 of the largest weight times the largest d.
//  - With up to 8 or 4 query heads a kv head the 16 columns hold them 2 or 4
//    times, and each replica has a half or a quarter of the blocks: its q is zero
//    in the others, so the first product gives each replica's share of a
//    score, added up by lane rotations, and only its own blocks' weights are
//    multiplied and split (of the second product's columns those of other
//    replicas are not used). That and the registers for scales are what bounds this
//    kernel next to the reads.
//  - A wave's tiles come to LDS by loads that need no registers, the next one on
//    its way while one is used; pages are asked for 32 tiles ahead.
template <typename T, int HD>
struct DecQuant {
  static constexpr int NB = HD / 32, UB = NB * T::kUnit, RB = 16 * UB + 4 * NB;  // blocks, bytes of a unit of all, of a row
  static constexpr int KT = 32, kPieces = 4 * RB, kLoads = (kPieces + 63) / 64;  // 16-byte pieces of a tile of two runs of K and of V
  static constexpr int kTile = 16 * kPieces;
  static constexpr int VD = HD / 16, RD = VD < 8 ? VD : 8, OS = 16 * RD + 4;
  static constexpr int kRing = kDecWaves * 2 * kTile, kMerge = kDecWaves * 16 * OS * 4;
  // workgroups that a CU's 160 KB of LDS and 512 registers a lane hold
  static constexpr int kPerCu = HD == 64 ? (T::kUnit == 1 ? 4 : 3) : HD == 128 ? (T::kUnit == 1 ? 3 : 2) : 1;
};
constexpr int kDecQuantSeqs = 1024;  // sequences of a launch
// What a piece costs besides its tiles, in tiles (us with 0 / 4 / 8 / 16: 64
// sequences of up to 8000, 28 heads on 4 of 128, q4, 56.0 / 50.7 / 46.9 / 46.6; 180
// of up to 2500 with a window of 1000, 16 of 64, q8, 96.8 / 71.1 / 64.7 / 70.0).
constexpr int kDecPad = 8;

// Weights times d are lifted to 2^15 less the exponent of the largest d; fp16's
// least normal numbers leave that at 2^29, an infinite or NaN one at 2^-2.
constexpr float kMostLift = 29.0f;

template <int N>
__device__ __forceinline__ float row_ror(float v) { return dpp<0x120 + N>(v); }
// Over the R replicas of a column (bit-identical in all of them).
template <int R>
__device__ __forceinline__ float replica_sum(float v) {
  if constexpr (R >= 2) v += row_ror<8>(v);
  if constexpr (R >= 4) v += row_ror<4>(v);
  return v;
}
template <int R>
__device__ __forceinline__ float replica_max(float v) {
  if constexpr (R >= 2) v = fmaxf(v, row_ror<8>(v));
  if constexpr (R >= 4) v = fmaxf(v, row_ror<4>(v));
  return v;
}

// R: replicas of the columns, as many as fit beside each other and share the blocks.
template <typename T, int HD, int R>
__global__ __launch_bounds__(kDecThreads, (DecQuant<T, HD>::kPerCu)) void paged_decode_quantised_kernel(PagedAttnArgs a) {
  using D = DecQuant<T, HD>;
  using Tr = KvTraits<_Float16>;
  constexpr int NB = D::NB, UB = D::UB, RB = D::RB, KT = D::KT, VD = D::VD, RD = D::RD, OS = D::OS, NP = 2;
  constexpr int kUnit = kDecWaves * KT;
  constexpr int HPR = 16 / R, BR = NB / R;  // columns of a replica, its blocks
  __shared__ __align__(16) char ring[D::kRing > D::kMerge ? D::kRing : D::kMerge];
  __shared__ int base[kDecQuantSeqs + 1];
  __shared__ int scan_lds[kDecWaves];
  __shared__ float wm[kDecWaves][16], wl[kDecWaves][16];
  __shared__ int wave_bad[kDecWaves];
  float(&merge)[kDecWaves][16][OS] = *(float(*)[kDecWaves][16][OS])ring;  // (when no tile is in use)

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ai = lane & 15, ak = lane >> 4, rep = ai / HPR;
  const int head_tiles = (a.group + 15) / 16, n_tiles = a.n_kv * head_tiles, TG = min(a.group, 16);
  const DecodePartials pp = decode_partials(a.part, a.n_seqs, a.ranges, TG);
  DecodeWork<KT, kDecQuantSeqs, kDecPad> work(a, base, scan_lds, n_tiles);
  if (!work.start(pp)) return;

  while (true) {
    const DecodeRow dr = work.row();
    const int seq = work.seq, tile = work.tile, k_at = work.k_at;
    const int piece = (int)min((int64_t)(work.count - k_at), work.uend - work.u);
    const bool whole = piece == work.count;
    const int slot = 2 * (int)blockIdx.x + (k_at == 0);
    const int kvh = tile / head_tiles, g0 = (tile - kvh * head_tiles) * 16;
    const int G = min(16, a.group - g0), head0 = kvh * a.group + g0;
    const int key_begin = first_key(a, dr.len), pos = dr.len - 1;
    // tiles start at multiples of their size: a run of 16 keys lies in one page
    const int lo = (key_begin & ~(KT - 1)) + k_at * KT;
    const int hi = min((int64_t)lo + (int64_t)piece * KT, (int64_t)dr.len);
    const int k0 = lo + wave * KT;
    const int tiles = k0 < hi ? (hi - k0 + kUnit - 1) / kUnit : 0;

    // ---- the tiles on their way to LDS
    bool bad = dr.bad;
    const int32_t* table = a.block_table + (size_t)seq * a.max_pages;
    const int mask = (1 << a.page_shift) - 1;
    int64_t place = 0;  // of run (lane & 1) of tile from + lane / 2: bytes from the layer's start
    // The run, or the nearest that holds a key which is seen: a tile may begin
    // before the window, on a page that nobody keeps any more.
    auto places = [&](int from) __attribute__((always_inline)) {
      const int k = k0 + (from + (lane >> 1)) * kUnit + 16 * (lane & 1);
      const int kk = min(max(k, key_begin), pos);
      int page = table[kk >> a.page_shift];
      const bool out = page < 0 || page >= a.n_pages;
      bad |= out && k < hi;
      page = out ? 0 : page;
      place = ((((int64_t)page * a.n_kv + kvh) << a.page_shift) + (kk & mask & ~15)) * RB;
    };
    auto fetch = [&](int i) __attribute__((always_inline)) {
      char* to = ring + (wave * 2 + (i & 1)) * D::kTile;
      const int64_t o0 = readlane64(place, 2 * (i & 31)), o1 = readlane64(place, 2 * (i & 31) + 1);
      const char* from[4] = {(const char*)a.keys + o0, (const char*)a.keys + o1, (const char*)a.values + o0, (const char*)a.values + o1};
#pragma unroll
      for (int j = 0; j < D::kLoads; ++j) {
        const int p = 64 * j + lane, r0 = 64 * j / RB;
        const char* src = from[r0] + 16 * (p - r0 * RB);
#pragma unroll
        for (int r = r0 + 1; r < 4 && r * RB < 64 * j + 64; ++r)
          if (p >= r * RB) src = from[r] + 16 * (p - r * RB);
        if (64 * j + 64 <= D::kPieces || p < D::kPieces)
          __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                           (__attribute__((address_space(3))) void*)(to + 1024 * j), 16, 0, 0);
      }
    };
    // ---- q, asked for before the tiles
    const bool has_head = ai % HPR < G;
    const float* qp = a.q + dr.row * a.q_stride + (int64_t)(head0 + (has_head ? ai % HPR : 0)) * a.hd;
    f4 x[BR][2];
#pragma unroll
    for (int c = 0; c < BR; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = 32 * (rep * BR + c) + 8 * ak + 4 * j;
        x[c][j] = has_head && d < a.hd ? *(const f4*)(qp + d) : f4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    __syncthreads();  // (the last piece's readers are done with the LDS)
    if (tiles > 0) {
      places(0);
      fetch(0);
      if (tiles > 1) fetch(1);
    }

    h8_t qv[NP][NB];
    int q_exp = 0;
    float q_sum[BR];  // of the replica's blocks, with q's power of two
    {
      float big = 0.0f;
#pragma unroll
      for (int c = 0; c < BR; ++c)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          big = fmaxf(fmaxf(big, fmaxf(fabsf(x[c][j].x), fabsf(x[c][j].y))), fmaxf(fabsf(x[c][j].z), fabsf(x[c][j].w)));
        }
      q_exp = pow2_scale_exp(replica_max<R>(xor32_max(xor16_max(big))));
#pragma unroll
      for (int c = 0; c < BR; ++c) {
        const f4 y = x[c][0] + x[c][1];
        q_sum[c] = ldexp_f(xor32_sum(xor16_sum((y.x + y.y) + (y.z + y.w))), q_exp);
        uint32_t w[NP][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // (a key's come as the lower dims of two units, then the others)
          const int i0 = 4 * (j >> 1) + (j & 1), i1 = i0 + 2;
          uint32_t p[NP];
          split_pair<_Float16>(ldexp_f(x[c][i0 >> 2][i0 & 3], q_exp), ldexp_f(x[c][i1 >> 2][i1 & 3], q_exp), p);
#pragma unroll
          for (int i = 0; i < NP; ++i) w[i][j] = p[i];
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
          for (int n = 0; n < R; ++n)
            qv[i][n * BR + c] = __builtin_bit_cast(h8_t, n == rep ? u32x4_t{w[i][0], w[i][1], w[i][2], w[i][3]} : u32x4_t{0, 0, 0, 0});
      }
    }
    const ScoreRule rule = score_rule(a, head0 + (has_head ? ai % HPR : 0), q_exp, a.scale);
    const bool plain = a.softcap <= 0.0f && a.slopes == nullptr;

    // ---- the keys
    float m = -INFINITY, l = 0.0f;  // of the column's head; l of this quarter's keys
    f4 acc[VD];                     // dims 2 (4 ak + r) + c % 2 of block c / 2 of the column
    float lift = kMostLift, acc_m[BR];
    const float minus_one = hidden_minus_one();
#pragma unroll
    for (int c = 0; c < VD; ++c) acc[c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < BR; ++c) acc_m[c] = 0.0f;
    for (int i = 0; i < tiles; ++i) {
      const int k = k0 + i * kUnit;  // the tile's first key
      constexpr int kNext = D::kLoads;
      // (the tile has landed, the next one need not have)
      if (i + 1 < tiles) __builtin_amdgcn_s_waitcnt(0x0F70 | (kNext & 15) | (kNext >> 4) << 14);
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      __builtin_amdgcn_wave_barrier();
      const char* at = ring + (wave * 2 + (i & 1)) * D::kTile;
      f4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const char* run = at + u * 16 * RB;
        uint32_t kq[UB];
        load_words<UB>(run + ai * RB + 4 * UB * ak, kq);
        f4 c4[BR];
#pragma unroll
        for (int c = 0; c < BR; ++c) c4[c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int x0 = 2 * j * UB + b * T::kUnit, x1 = x0 + UB;  // bytes of the two units
            code_pairs<T>(kq[x0 / 4], x0 % 4 / T::kUnit, kq[x1 / 4], x1 % 4 / T::kUnit, w[2 * j], w[2 * j + 1]);
          }
#pragma unroll
          for (int p = NP - 1; p >= 0; --p)
            c4[b % BR] = Tr::mfma(__builtin_bit_cast(h8_t, u32x4_t{w[0], w[1], w[2], w[3]}), qv[p][b], c4[b % BR]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint32_t sw[BR];
          load_words<BR>(run + (4 * ak + r) * RB + 16 * UB + 4 * BR * rep, sw);
          float x = 0.0f;
#pragma unroll
          for (int c = 0; c < BR; ++c) x = __builtin_fmaf(scale_m(sw[c]), q_sum[c], __builtin_fmaf(scale_d(sw[c]), c4[c][r], x));
          s[u][r] = replica_sum<R>(x);
        }
      }
      const bool edge = k < key_begin || k + KT > hi;
      uint32_t vs[8][BR];
      const char* vrun = at + 32 * RB;
#pragma unroll
      for (int e = 0; e < 8; ++e) load_words<BR>(vrun + (16 * (e >> 2) + 4 * ak + (e & 3)) * RB + 16 * UB + 4 * BR * rep, vs[e]);
      float p[8], mx = -INFINITY;
      if (plain) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = s[e >> 2][e & 3] * rule.sl2;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = s[e >> 2][e & 3];
          x = a.softcap > 0.0f ? rule.cap_out * tanhf(x * rule.cap_in) : x * rule.sl2;
          p[e] = x + rule.slope2 * (float)(k + 16 * (e >> 2) + 4 * ak + (e & 3) - pos);
        }
      }
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int t = k + 16 * (e >> 2) + 4 * ak + (e & 3);
          if (t < key_begin || t >= hi) {
            p[e] = -INFINITY;
            // (what lies there may be anything, and 0 * inf is not 0)
#pragma unroll
            for (int c = 0; c < BR; ++c) vs[e][c] = 0;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, p[e]);
      mx = fmaxf(m, xor32_max(xor16_max(mx)));
      // the largest |d|, by its exponent (rows from elsewhere may have a negative one).
      // NaN counts for nothing, it makes its block NaN by itself; a signalling one
      // hides the instruction's other d, which is of the same block, and not the
      // largest so far, which comes last.
      uint32_t big = 0;
#pragma unroll
      for (int e = 0; e < 8; e += 2)
#pragma unroll
        for (int c = 0; c < BR; ++c) asm("v_max3_f16 %0, |%1|, |%2|, %0" : "+v"(big) : "v"(vs[e][c]), "v"(vs[e + 1][c]));
      const float new_lift = fminf(lift, kMostLift - xor32_max(xor16_max((float)(big >> 10 & 31))));
      const float ref = (mx == -INFINITY ? 0.0f : mx) - new_lift;
      const float al = (mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx)) * __builtin_amdgcn_exp2f(new_lift - lift);
      m = mx;
      lift = new_lift;
      if (__any(al != 1.0f)) {
        l *= al;
#pragma unroll
        for (int c = 0; c < VD; ++c) acc[c] *= al;
#pragma unroll
        for (int c = 0; c < BR; ++c) acc_m[c] *= al;
      }
      if (plain && !edge) {
        // (scaled and shifted with one rounding)
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], rule.sl2, -ref));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(p[e] - ref);
      }
      l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      uint32_t vr[8][(UB + 3) / 4];
#pragma unroll
      for (int e = 0; e < 8; ++e) load_words<UB / 4>(vrun + (16 * (e >> 2) + 4 * ak + (e & 3)) * RB + UB * ai, vr[e]);
#pragma unroll
      for (int c = 0; c < BR; ++c) {
        uint32_t w[NP][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t q[NP];
          split_halves(times_d(vs[2 * j][c], p[2 * j]), times_d(vs[2 * j + 1][c], p[2 * j + 1]), minus_one, q);
#pragma unroll
          for (int n = 0; n < NP; ++n) w[n][j] = q[n];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc_m[c] = __builtin_fmaf(scale_m(vs[e][c]), p[e], acc_m[c]);
#pragma unroll
        for (int n = 0; n < R; ++n) {
          const int b = n * BR + c, x = b * T::kUnit;
          uint32_t v[2][4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            code_pairs<T>(vr[2 * j][x / 4], x % 4 / T::kUnit, vr[2 * j + 1][x / 4], x % 4 / T::kUnit, v[0][j], v[1][j]);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = NP - 1; q >= 0; --q)
              acc[2 * b + h] = Tr::mfma(__builtin_bit_cast(h8_t, u32x4_t{v[h][0], v[h][1], v[h][2], v[h][3]}),
                                        __builtin_bit_cast(h8_t, u32x4_t{w[q][0], w[q][1], w[q][2], w[q][3]}), acc[2 * b + h]);
        }
      }
      // (every read of the tile is done before its place is filled again)
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_wave_barrier();
      if (i + 2 < tiles) {
        if (((i + 2) & 31) == 0) places(i + 2);
        fetch(i + 2);
      }
    }
    // (the waves, the ranges and the replicas need not have met the same d)
    const float down = __builtin_amdgcn_exp2f(-lift);
    l = xor32_sum(xor16_sum(l)) * down;
#pragma unroll
    for (int c = 0; c < BR; ++c) acc_m[c] = xor32_sum(xor16_sum(acc_m[c])) * down;
#pragma unroll
    for (int c = 0; c < VD; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[c][r] = __builtin_fmaf(acc[c][r], down, acc_m[c / 2 % BR]);
    bad = __any(bad);

    // ---- the waves joined in their order
    __syncthreads();  // (every wave is done with its tiles)
    if (lane == 0) wave_bad[wave] = bad;
    if (ak == 0 && rep == 0) {
      wm[wave][ai] = m;
      wl[wave][ai] = l;
    }
    float* out = a.out + dr.row * a.out_stride + (int64_t)head0 * a.hd;
#pragma unroll
    for (int c0 = 0; c0 < VD; c0 += RD) {
      if (c0 > 0) __syncthreads();
#pragma unroll
      for (int c = 0; c < RD; c += 2)
        if ((c0 + c) / 2 / BR == rep) {
#pragma unroll
          for (int r = 0; r < 4; r += 2)
            *(f4*)&merge[wave][ai % HPR][16 * c + 8 * ak + 2 * r] =
                f4{acc[c0 + c][r], acc[c0 + c + 1][r], acc[c0 + c][r + 1], acc[c0 + c + 1][r + 1]};
        }
      __syncthreads();
      for (int e = tid; e < G * 16 * RD; e += kDecThreads) {
        const int g = e / (16 * RD), x = e % (16 * RD);
        const int d = 16 * c0 + x;
        if (d >= a.hd) continue;
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
          const size_t to = (size_t)slot * TG + g;
          if (d == 0) {
            pp.m[to] = mx;
            pp.l[to] = sum;
          }
          pp.acc[to * a.hd + d] = o;
        }
      }
    }
    if (!work.next(piece)) return;
  }
}

template <typename T, int HD>
void decode_launch(const PagedAttnArgs& a, hipStream_t stream) {
  const int heads = std::min(a.group, 16);
  if (HD >= 128 && heads <= 4)
    hipLaunchKernelGGL((paged_decode_quantised_kernel<T, HD, HD >= 128 ? 4 : 2>), dim3(a.ranges), dim3(kDecThreads), 0, stream, a);
  else if (heads <= 8)
    hipLaunchKernelGGL((paged_decode_quantised_kernel<T, HD, 2>), dim3(a.ranges), dim3(kDecThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_decode_quantised_kernel<T, HD, 1>), dim3(a.ranges), dim3(kDecThreads), 0, stream, a);
}
template <typename T>
void decode_launch_hd(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.hd <= 64) decode_launch<T, 64>(a, stream);
  else if (a.hd <= 128) decode_launch<T, 128>(a, stream);
  else decode_launch<T, 256>(a, stream);
}
template <typename T>
int per_cu(int hd) {
  return hd <= 64 ? DecQuant<T, 64>::kPerCu : hd <= 128 ? DecQuant<T, 128>::kPerCu : DecQuant<T, 256>::kPerCu;
}

}  // namespace

int paged_decode_quantised_per_cu(const PagedAttnArgs& a) { return a.type == MLQ_KV_Q4 ? per_cu<KvQ4>(a.hd) : per_cu<KvQ8>(a.hd); }
int paged_decode_quantised_seqs() { return kDecQuantSeqs; }

void launch_paged_decode_quantised(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.type == MLQ_KV_Q4) decode_launch_hd<KvQ4>(a, stream);
  else decode_launch_hd<KvQ8>(a, stream);
}

hipError_t launch_paged_prefill_quantised(const PagedAttnArgs& a, hipStream_t stream) {
  return a.type == MLQ_KV_Q4 ? prefill_launch_type<KvQ4>(a, stream) : prefill_launch_type<KvQ8>(a, stream);
}

}  // namespace mlq
