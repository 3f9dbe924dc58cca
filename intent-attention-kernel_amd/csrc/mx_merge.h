// The merge of the parts of query rows whose tokens were divided, for the attention kernels over paged
// caches (mx_attention.h).
#ifndef IAK_MX_MERGE_H
#define IAK_MX_MERGE_H

#include "mx_attention.h"

namespace iak {
namespace {

// The parts of 256 / (D / 4 PARTS) query rows a workgroup: a thread takes 4 channels of every
// PARTS-th part of its row. PARTS > 1, where a row has many parts, is one row a workgroup.
template <int D, int PARTS, typename A>
__global__ __launch_bounds__(256) void mx_merge_kernel(const A a) {
  constexpr int UNITS = D / 4, ROWS = 256 / (UNITS * PARTS);
  static_assert(PARTS == 1 || ROWS == 1, "one row, or one part");
  __shared__ f4 sum[PARTS][UNITS];
  __shared__ float sum_l[PARTS], top[4];
  const int rows = a.L * a.G;
  const int u = threadIdx.x % UNITS, part = PARTS > 1 ? threadIdx.x / UNITS : 0;
  const int64_t at = (int64_t)blockIdx.x * ROWS + (PARTS > 1 ? 0 : threadIdx.x / UNITS);
  const bool there = at < (int64_t)a.B * a.Hkv * rows;           // always, where there are barriers
  const int64_t kvrow = there ? at / rows : 0;
  const int r = there ? (int)(at - kvrow * rows) : 0;
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow - (int64_t)b * a.Hkv);
  const int tile = r / a.tile_rows, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const MxRows n = mx_rows(a, kvrow, b);
  int2 mine = {0, 0};                                            // the row's first part, and how many
  if (there && i < n.queries) {
    const int64_t t = kvrow * a.tiles + tile;
    const int entries = mx_entries(a, n, tile * a.tile_rows, a.tile_rows);
    if (!a.shares) mine = int2{(int)(t * a.splits), (entries + a.chunk - 1) / a.chunk};
    else if (entries > 0) mine = a.ws_parts[t];
    // lengths that change between the kernels are the caller's mistake, but no read out of bounds
    if (a.shares && ((uint32_t)mine.x > (uint32_t)a.shares || (uint32_t)mine.y > (uint32_t)(a.shares - mine.x))) mine = int2{0, 0};
  }
  const int parts = mine.y;
  const int64_t step = a.tile_rows, first = (int64_t)mine.x * step + (r & (a.tile_rows - 1));
  float M = M_NONE;
  if constexpr (PARTS > 1) {
    for (int s = threadIdx.x; s < parts; s += 256) M = fmaxf(M, a.ws_m[first + s * step]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  } else {
    for (int s0 = 0; s0 < parts; s0 += 8) {                      // loads of a batch all under way at once
      float top8[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) top8[k] = s0 + k < parts ? a.ws_m[first + (s0 + k) * step] : M_NONE;
#pragma unroll
      for (int k = 0; k < 8; ++k) M = fmaxf(M, top8[k]);
    }
  }
  float L = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = part; s0 < parts; s0 += 4 * PARTS) {
    float m4[4], l4[4];
    f4 o4[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = s0 + k * PARTS;
      const int64_t slot = first + (s < parts ? s : part) * step;
      m4[k] = s < parts ? a.ws_m[slot] : -__builtin_inff();
      l4[k] = a.ws_l[slot];
      o4[k] = ld_nt(reinterpret_cast<const f4*>(a.ws_acc + slot * D + 4 * u));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (s0 + k * PARTS >= parts) break;
      float wgt = __builtin_amdgcn_exp2f(m4[k] - M);
      L += wgt * l4[k];
      part_weight(o4[k], wgt);
      o += o4[k] * wgt;
    }
  }
  if constexpr (PARTS > 1) {
    sum[part][u] = o;
    if (u == 0) sum_l[part] = L;
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) { o += sum[p][u]; L += sum_l[p]; }
  }
  if (!there) return;
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  float out[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) out[q] = o[q] * inv;
  store_out4(a, b * a.osb + i * a.ost + head * a.osh + 4 * u, out);
}

// Rows whose parts a thread walks alone, eight at most; more are shared by a workgroup. With shares,
// where a few rows may have most parts: below 4,096 rows by a workgroup (8 rows of 32,768 tokens among
// 248 of 819: 29 us and 45; 4 x 256 queries x 16 heads, one sequence of 16,000 tokens: 69 and 50).
template <int D, typename A> void launch_mx_merge(const A& a, hipStream_t stream) {
  constexpr int UNITS = D / 4;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.L * a.G;
  if (a.shares ? rows >= 4096 : a.splits <= 8) {
    const int per = 256 / UNITS;
    hipLaunchKernelGGL((mx_merge_kernel<D, 1, A>), dim3((uint32_t)((rows + per - 1) / per)), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((mx_merge_kernel<D, 256 / UNITS, A>), dim3((uint32_t)rows), dim3(256), 0, stream, a);
  }
}

}  // namespace
}  // namespace iak

#endif
