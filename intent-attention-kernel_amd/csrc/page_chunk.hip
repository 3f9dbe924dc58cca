// Attention over pages of mixed precision for many query rows of a KV head (prompt chunks), for
// gfx950. The mathematics, the lanes' parts and the softmax are the rows kernel's (page_rows.hip);
// what differs is who reads the cache.
//
// A workgroup takes 16 RT rows a wave. All its waves walk the same tokens, 64 (four pages) a
// step; each puts its share of the next step's pages (one page of K or of V in eight waves, of both
// in four) into LDS as operands, from where all read them: two buffers, one barrier a step.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "page_attention.h"

namespace iak {

namespace {

template <int D, bool QF32, int NW, int RT, int KIND>
__global__ __launch_bounds__(64 * NW, 2) void page_chunk_kernel(const PageAttn a) {
  static_assert(NW == 4 || NW == 8, "a wave takes a page of K and of V, or one of the two");
  constexpr bool WIDE = KIND == PAGES_ALL, SCALED = KIND != PAGES_F16;
  constexpr int OWN = 8 / NW, BM = 16 * RT * NW, PAGE = PS * D / 8;   // 16-byte units of a tile
  __shared__ u4 tiles[2][2][4][PAGE];                            // [buffer][K, V][page]
  __shared__ u4 rest[WIDE ? 2 : 1][2][4][WIDE ? PAGE : 1];       // of wide pages: what their tiles leave
  __shared__ u4 none[WIDE ? PAGE : 1];                           // zeros
  __shared__ u4 metas[128];                                      // of entry e at e % 128: page, tag, km, vl
  __shared__ u2 factors[SCALED ? 128 : 1];                       // kf, vf
  __shared__ int special;                                        // V has infinite or NaN values
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const MxPart part = a.shares ? mx_shared_part<4, true>(a) : mx_fixed_part(a);
  if (part.idle) return;                                         // uniform, as below
  const int64_t kvrow = part.kvrow;
  const int tile = part.tile;
  const int b = (int)(part.kvrow / (uint32_t)a.Hkv), hk = (int)(part.kvrow - (uint32_t)b * a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * BM, BM);
  const int e0 = part.e0, e1 = e0 + part.chunk < entries ? e0 + part.chunk : entries;
  if (e0 > 0 && e0 >= e1) return;                                // the merge does not look at it
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < PAGE; i += 64 * NW) none[i] = u4{0u, 0u, 0u, 0u};
  }

  const int rows = a.L * a.G;
  int seen[RT], least = 0x7FFFFFFF;
  h8 qhi[RT][D / 32], qlo[RT][QF32 ? D / 32 : 1];
  float mult[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = tile * BM + (w * RT + t) * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
    const bool active = r < rows, live = active && i < n.queries;
    seen[t] = live ? mx_seen(a, n, i) : 0;
    least = live && seen[t] < least ? seen[t] : least;
    mult[t] = load_query<D, QF32>(a, active, b * a.qsb + i * a.qst + head * a.qsh, g, qhi[t], qlo[t]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(least, o, 64); least = x < least ? x : least; }

  // The entries' pages and multipliers lie in LDS, 64 ahead of the walk: wave 0 looks up a block of 64
  // in four steps of the walk, a load each.
  const int32_t* row = a.table + kvrow * a.W;
  auto keep = [&](int k, const PageEntry& x) __attribute__((always_inline)) {
    metas[k & 127] = u4{(uint32_t)x.id, (uint32_t)x.tag, f2u(x.km), f2u(x.vl)};
    if constexpr (SCALED) factors[k & 127] = u2{f2u(x.kf), f2u(x.vf)};
  };
  if (w < 2) keep(64 * w + lane, page_entry<D, KIND>(a, row, e0 + 64 * w + lane, e1));
  if (threadIdx.x == 0) special = 0;
  __syncthreads();
  int ahead = 0, ahead_tag = 0;
  float ahead_k = 1.f, ahead_v = 1.f;
  auto look_ahead = [&](int k) __attribute__((always_inline)) {  // k: entry of the walk, a multiple of 4
    if ((k & 15) != 0 || w != 0) return;
    const int stage = (k >> 4) & 3, e = (k & ~63) + 64 + lane;   // the block after the one at hand
    if (k < 64) return;                                          // two blocks are there at first
    if (stage == 0) ahead = raw_entry(row, e0 + e, e1);
    else if (stage == 1) {
      ahead = entry_page(a, ahead);
      ahead_tag = raw_tag(a, ahead);
    } else if (stage == 2) {
      const PageTag x = page_tag<KIND>(a, ahead, ahead_tag);
      ahead = x.id;
      ahead_tag = x.tag;
      page_scales<D, KIND>(a, x, ahead_k, ahead_v);
    } else keep(e, page_multipliers<KIND>(PageTag{ahead, ahead_tag}, ahead_k, ahead_v));
  };
  auto uniform = [](uint32_t x) { return __builtin_amdgcn_readfirstlane((int)x); };
  auto uniform_f = [](uint32_t x) { return u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)x)); };

  // this wave's page of a step, of K and V or of one of them: loaded a step ahead, put into LDS during
  // the step before
  const int own = w & 3, side = w >> 2;
  PageRaw<D> raw[OWN];
  auto load = [&](const u4& x) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 0; o < OWN; ++o)
      load_page<D, KIND, false>(raw[o], a, OWN == 2 ? o == 1 : side == 1, uniform(x[0]), uniform(x[1]), lane);
  };
  auto convert = [&](int buf, const u4& x, const u2& f) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int s = OWN == 2 ? o : side;
      const bool bad = store_page<D, KIND, true>(raw[o], uniform(x[0]), uniform(x[1]), uniform_f(s ? f[1] : f[0]), tiles[buf][s][own],
                                                 rest[WIDE ? buf : 0][s][own], lane);
      if (s == 1 && __builtin_amdgcn_ballot_w64(bad)) {          // rare
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        clean_tile<D>(tiles[buf][1][own], lane);
        if (lane == 0) special = 1;
      }
    }
  };
  const u2 one = {f2u(1.f), f2u(1.f)};

  f4 acc[RT][D / 16], l[RT];
  float lsum[RT], m[RT];
  int E = 0;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = M_NONE;
    lsum[t] = 0.f;
    l[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) acc[t][mb] = f4{0.f, 0.f, 0.f, 0.f};
  }

  const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
  int k = 0;                                                     // number of entry e in the part
  auto step = [&](int buf, int e) __attribute__((always_inline)) {
    u4 at[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) at[p] = metas[(k + p) & 127];
    const u4 mine = metas[(k + 4 + own) & 127], after = metas[(k + 8 + own) & 127];
    const u2 factor = SCALED ? factors[(k + 4 + own) & 127] : one;
    f4 s[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int p = 0; p < 4; ++p) s[t][p] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const h8 ka = __builtin_bit_cast(h8, tiles[buf][0][p][v_chunk<D>(c, g * (D / 32) + j)]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[t][j], s[t][p], 0, 0, 0);
          if constexpr (QF32) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[t][j], s[t][p], 0, 0, 0);
        }
      }
    int id[4];
    float km[4], vl[4];
    bool wide[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      id[p] = uniform(at[p][0]);
      km[p] = SCALED ? uniform_f(at[p][2]) : 1.f;
      vl[p] = SCALED ? uniform_f(at[p][3]) : 0.f;
      wide[p] = WIDE && id[p] >= 0 && wide_tag(uniform(at[p][1]));
    }
    if constexpr (WIDE) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        if (!wide[p]) continue;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const h8 ka = __builtin_bit_cast(h8, rest[buf][0][p][v_chunk<D>(c, g * (D / 32) + j)]);
#pragma unroll
          for (int t = 0; t < RT; ++t) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[t][j], s[t][p], 0, 0, 0);
        }
      }
    }
    convert(buf ^ 1, mine, factor);
    load(after);
    look_ahead(k);
    const uint32_t no_nan[4] = {0u, 0u, 0u, 0u};
    hide<4, RT>(s, no_nan, id, e, seen, least, g);
    if constexpr (SCALED) {
      raise_scaled<D, 4, RT>(s, km, mult, m, lsum, acc);
      const int to = value_power<4>(id, vl, E);
      if (to != E) {                                             // uniform
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[t][mb][q] = __builtin_ldexpf(acc[t][mb][q], E - to);
        E = to;
      }
      float out[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        vl[p] = id[p] < 0 ? 0.f : vl[p] - (float)E;
        out[p] = __builtin_amdgcn_exp2f(-vl[p]);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) lsum[t] += soften_scaled<4>(s[t], km, vl, out, mult[t], m[t]);
    } else {
      raise<D, 4, RT>(s, mult, m, l, acc);
#pragma unroll
      for (int t = 0; t < RT; ++t) soften<4>(s[t], mult[t], m[t]);
    }
    h8 pb[RT][2], pl[RT][QF32 ? 2 : 1];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pb[t][h] = weights(s[t][2 * h], s[t][2 * h + 1]);
        if constexpr (QF32) pl[t][h] = weights_rest(s[t][2 * h], s[t][2 * h + 1], pb[t][h]);
      }
    if constexpr (!SCALED) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[t][h], l[t], 0, 0, 0);
          if constexpr (QF32) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[t][h], l[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        const h8 va = values_back<D>(tiles[buf][1][2 * h], tiles[buf][1][2 * h + 1], mb, c, g);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[t][h], acc[t][mb], 0, 0, 0);
          if constexpr (QF32) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[t][h], acc[t][mb], 0, 0, 0);
        }
      }
    if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (!wide[2 * h] && !wide[2 * h + 1]) continue;
        const u4* p0 = wide[2 * h] ? rest[buf][1][2 * h] : none;
        const u4* p1 = wide[2 * h + 1] ? rest[buf][1][2 * h + 1] : none;
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb) {
          const h8 va = values_back<D>(p0, p1, mb, c, g);
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[t][h], acc[t][mb], 0, 0, 0);
        }
      }
    }
    k += 4;
    __syncthreads();                                             // this buffer is free, the other one is whole
  };
  if (e0 < e1) {
    load(metas[own]);
    convert(0, metas[own], SCALED ? factors[own] : one);
    load(metas[4 + own]);
    __syncthreads();
    for (int e = e0; e < e1; e += 8) {
      step(0, e);
      if (e + 4 < e1) step(1, e + 4);
    }
  }

  // what V has of infinite and NaN values, in a second walk
  if (special) {                                                 // uniform: written before the last barrier
    uint16_t* aside = reinterpret_cast<uint16_t*>(&tiles[1][0][0][0]);
    uint32_t* any = reinterpret_cast<uint32_t*>(&tiles[1][1][0][0]);
    Seen16 odd[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) odd[t] = Seen16{0u, 0u};
    for (int e = e0; e < e1; e += 4) {
      __syncthreads();
      if (w < 4) {
        const PageEntry x = page_entry<D, KIND>(a, row, e + w, e1);
        const int id = uniform((uint32_t)x.id), tag = uniform((uint32_t)x.tag);
        PageRaw<D> r;
        load_page<D, KIND, false>(r, a, true, id, tag, lane);
        const bool bad = store_page<D, KIND, true>(r, id, tag, uniform_f(f2u(x.vf)), tiles[0][0][w], rest[0][0][w], lane);
        const bool some = __builtin_amdgcn_ballot_w64(bad) != 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (some) put_aside<D>(tiles[0][0][w], aside + w * PAGE, lane);
        if (lane == 0) any[w] = some;
      }
      __syncthreads();
      for (int p = 0; p < 4; ++p) {
        if (uniform(any[p]) == 0) continue;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int left = seen[t] - (e + p) * PS;
          remember<D>(odd[t], aside + p * PAGE, left < PS ? left : PS, g);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) bring_back<D>(acc[t], odd[t]);
  }

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = tile * BM + (w * RT + t) * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
    float sum;
    if constexpr (SCALED) sum = xsum16_32(lsum[t]);
    else sum = l[t][0];
    if (r >= rows) continue;
    if (a.parted) {
      const int64_t slot = (int64_t)part.part * BM + (w * RT + t) * 16 + c;
      if (g == 0) { a.ws_m[slot] = m[t]; a.ws_l[slot] = sum; }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        f4 x = acc[t][mb];
        if constexpr (SCALED) {
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = __builtin_ldexpf(x[q], E);
        }
        *reinterpret_cast<f4*>(a.ws_acc + slot * D + 16 * mb + 4 * g) = x;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;           // NaN stays
      const int64_t at = b * a.osb + i * a.ost + head * a.osh + 4 * g;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        float o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = acc[t][mb][q] * inv;
          o[q] = i < n.queries ? (SCALED ? __builtin_ldexpf(x, E) : x) : 0.f;
        }
        store_out4(a, at + 16 * mb, o);
      }
    }
  }
}

template <int D, bool QF32, int NW, int RT> void launch_tiles(const PageAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items), block(64 * NW);
  if (a.kind == PAGES_F16) hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_F16>), grid, block, 0, stream, a);
  else if (a.kind == PAGES_BYTE) hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_BYTE>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_ALL>), grid, block, 0, stream, a);
}

template <int D> void launch_chunk(const PageAttn& a, hipStream_t stream) {
  if (a.q_dtype == IAK_DTYPE_F32) launch_tiles<D, true, 8, 1>(a, stream);
  else if (a.tile_rows == 256) launch_tiles<D, false, 8, 2>(a, stream);
  else launch_tiles<D, false, 4, 2>(a, stream);
}

}  // namespace

void launch_page_chunk(const PageAttn& a, hipStream_t stream) {
  if (a.D == 128) launch_chunk<128>(a, stream);
  else launch_chunk<64>(a, stream);
}

}  // namespace iak
