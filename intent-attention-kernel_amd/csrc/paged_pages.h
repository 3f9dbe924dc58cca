// Pages of every precision as a wave takes them by itself, for the kernels over the decode's pools: raw
// data in registers, K's way through LDS, and the ring in which a precision's pages are loaded ahead.
#ifndef IAK_PAGED_PAGES_H
#define IAK_PAGED_PAGES_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak_device.h"

namespace iak {

// --------------------------------------------------------------------------- //
// Raw page data as each lane loads it, per precision and head_dim.
//
// FP16 and one-byte pages are read so that every load instruction covers whole
// 128-byte lines, with the streaming (nontemporal) hint:
//   K  load i of lane l is the 16 bytes at 1024 i + 16 l of the page; the wave
//      rewrites them into the MFMA layout through its LDS buffer (k_through_lds);
//   V  load t of lane (c, g) is token 4t + g, so one instruction reads the four
//      consecutive rows 4t .. 4t+3.
// Lane (c, g) therefore holds K of token perm16(c) and V of tokens perm16(4g + t),
// the same permutation on both sides of the softmax. INT4 pages keep the
// direct layout (token c; tokens 4g + t) and plain loads: their K loads already
// cover the whole page, and streaming loads measured slower on them.
// --------------------------------------------------------------------------- //

template <int D> struct Raw16 {   // FP16: K chunks 64i + lane; V tokens 4t+g dims (D/16)c..
  u4 k[D / 32];                    // D/4 halves = D/32 u4
  uint32_t v[4][D / 32];           // D/16 halves per token = D/32 dwords
};
template <int D> struct Raw8 {    // FP8 / INT8 / INT4_RESIDUAL (one byte per element)
  uint32_t k[D / 16];              // D/4 bytes: chunks 64i + lane
  uint32_t v[4][D / 64 > 0 ? D / 64 : 1];  // D/16 bytes per token 4t+g
};
template <int D> struct Raw4 {    // INT4 (half a byte per element): K token c, V tokens 4g+t
  uint32_t k[D / 32];              // D/8 bytes
  uint32_t v[4];                   // D/32 bytes per token (<= 4)
};

// Token of score row / P slot r of FP16 and one-byte pages: perm16(4g + t) =
// 4t + g.
__device__ __forceinline__ int perm16(int r) { return 4 * (r & 3) + (r >> 2); }

template <int D> __device__ __forceinline__ void load16(Raw16<D>& r, const _Float16* kp, const _Float16* vp,
                                                       int c, int g) {
  const u4* kr = reinterpret_cast<const u4*>(kp) + (c + 16 * g);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) r.k[i] = ld_nt(kr + 64 * i);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const _Float16* row = vp + (4 * t + g) * D + (D / 16) * c;
    if constexpr (D == 128) {
      u4 x = ld_nt(reinterpret_cast<const u4*>(row));
      r.v[t][0] = x[0]; r.v[t][1] = x[1]; r.v[t][2] = x[2]; r.v[t][3] = x[3];
    } else {
      u2 x = ld_nt(reinterpret_cast<const u2*>(row));
      r.v[t][0] = x[0]; r.v[t][1] = x[1];
    }
  }
}

template <int D> __device__ __forceinline__ void load8(Raw8<D>& r, const uint8_t* kp, const uint8_t* vp,
                                                      int c, int g) {
  const u4* kr = reinterpret_cast<const u4*>(kp) + (c + 16 * g);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    u4 x = ld_nt(kr + 64 * i);
    r.k[4 * i + 0] = x[0]; r.k[4 * i + 1] = x[1]; r.k[4 * i + 2] = x[2]; r.k[4 * i + 3] = x[3];
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint8_t* row = vp + (4 * t + g) * D + (D / 16) * c;
    if constexpr (D == 128) {
      u2 x = ld_nt(reinterpret_cast<const u2*>(row));
      r.v[t][0] = x[0]; r.v[t][1] = x[1];
    } else {
      r.v[t][0] = ld_nt(reinterpret_cast<const uint32_t*>(row));
    }
  }
}

template <int D> __device__ __forceinline__ void load4(Raw4<D>& r, const uint8_t* kp, const uint8_t* vp,
                                                      int c, int g) {
  const uint8_t* krow = kp + c * (D / 2) + (D / 8) * g;
  if constexpr (D == 128) {
    u4 x = ld(reinterpret_cast<const u4*>(krow));
    r.k[0] = x[0]; r.k[1] = x[1]; r.k[2] = x[2]; r.k[3] = x[3];
  } else {
    u2 x = ld(reinterpret_cast<const u2*>(krow));
    r.k[0] = x[0]; r.k[1] = x[1];
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint8_t* row = vp + (4 * g + t) * (D / 2) + (D / 32) * c;
    if constexpr (D == 128) {
      r.v[t] = ld(reinterpret_cast<const uint32_t*>(row));
    } else {
      r.v[t] = ld(reinterpret_cast<const uint16_t*>(row));
    }
  }
}

// V operand of row block mb from four f16-pair rows vt[t][w] = dims (2w, 2w+1)
// of token 4g+t: the dim (D/16)c + mb of tokens 4g .. 4g+3.
template <int D>
__device__ __forceinline__ h4 rows_to_a(const uint32_t (&vt)[4][D / 32], int mb) {
  const int wd = mb >> 1;
  if (mb & 1) return make_h4(pack_hi(vt[0][wd], vt[1][wd]), pack_hi(vt[2][wd], vt[3][wd]));
  return make_h4(pack_lo(vt[0][wd], vt[1][wd]), pack_lo(vt[2][wd], vt[3][wd]));
}

// LDS slot (16-byte units) of chunk `ch` of token row `row` in a wave's K
// transpose buffer of NC chunks per row, XOR-swizzled so that 16 lanes reading
// one chunk of 16 different rows, and 16 lanes writing 256 consecutive bytes,
// each touch every 16-byte bank group once.
template <int NC> __device__ __forceinline__ int kt_slot(int row, int ch) {
  constexpr int RPB = 16 / NC;   // rows per 256 bytes
  return row * NC + (ch ^ ((row / RPB) % NC));
}

// A wave's K page, loaded as 16-byte chunks 64 i + lane (lane = c + 16 g) of
// the page, rewritten through its LDS buffer: afterwards lane (c, g) holds the
// NI chunks NI g .. NI g + NI - 1 of token row perm16(c).
template <int NC, int NI>
__device__ __forceinline__ void k_through_lds(u4 (&k)[NI], u4* kt, int c, int g) {
  const int lane = c + 16 * g;
  // wavefront-scope fences: the buffer's previous reads, these writes and the
  // reads below stay in this order (the lanes exchange data through it)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int f = 64 * i + lane;
    kt[kt_slot<NC>(f / NC, f % NC)] = k[i];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const int row = perm16(c);
#pragma unroll
  for (int i = 0; i < NI; ++i) k[i] = kt[kt_slot<NC>(row, NI * g + i)];
}

// The K dwords of a one-byte page in the MFMA layout (lane (c, g): token row
// perm16(c), bytes (D/4) g .. (D/4) g + D/4 - 1).
template <int D> __device__ __forceinline__ void k8_words(const Raw8<D>& r, uint32_t (&kw)[D / 16], u4* kt, int c,
                                                         int g) {
  u4 k[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) k[i] = u4{r.k[4 * i], r.k[4 * i + 1], r.k[4 * i + 2], r.k[4 * i + 3]};
  k_through_lds<D / 16, D / 64>(k, kt, c, g);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    kw[4 * i] = k[i][0]; kw[4 * i + 1] = k[i][1]; kw[4 * i + 2] = k[i][2]; kw[4 * i + 3] = k[i][3];
  }
}

// Read-only target of the ring loads issued past the end of a class: one page
// of any precision (at most PS x 128 x 2 bytes), the same address for every
// wave, so those loads stay in the L2 instead of fetching a streamed page again.
static __device__ __attribute__((aligned(4096))) uint8_t pad_page[PS * 128 * 2];

// Walks the pages of one precision class (lanes set in `mask`) through a ring
// of R register buffers: while one page is computed the next R-1 are in
// flight. Every step issues exactly one page load -- once the class runs out
// of pages the load names page -1, which the load functions point at
// pad_page -- and the loop exits only at its latch, so each buffer stays in
// its registers and the wait before each compute is a fixed vmcnt: loads are
// never drained early.
template <int R, typename Raw, typename LoadF, typename ComputeF>
__device__ __forceinline__ void class_loop(uint64_t mask, int pid, LoadF load, ComputeF compute) {
  if (!mask) return;
  const int n = __builtin_popcountll(mask);
  Raw buf[R];
  int idx[R];
  int last = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool real = mask != 0;
    if (mask) last = take(mask);
    idx[j] = last;
    const int p = __builtin_amdgcn_readlane(pid, last);
    load(buf[j], real ? p : -1);
  }
  // one exit, at the latch: the R steps of the body always issue their loads
  for (int base = 0; base < n; base += R) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (base + j < n) compute(buf[j], idx[j]);
      const bool real = mask != 0;
      if (mask) last = take(mask);
      idx[j] = last;
      const int p = __builtin_amdgcn_readlane(pid, last);
      load(buf[j], real ? p : -1);
    }
  }
}

// Base address of page `p` of a pool with `bytes` per page; pad_page for p < 0.
template <typename T> __device__ __forceinline__ const T* page_at(const void* pool, int p, int bytes) {
  return reinterpret_cast<const T*>(p < 0 ? pad_page : reinterpret_cast<const uint8_t*>(pool) + (int64_t)p * bytes);
}

}  // namespace iak

#endif
