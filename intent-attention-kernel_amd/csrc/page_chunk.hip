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

struct Plain { static constexpr bool value = false; };
struct Cleaned { static constexpr bool value = true; };

template <int D, bool QF32, int NW, int RT, int KIND>
__global__ __launch_bounds__(64 * NW, 2) void page_chunk_kernel(const PageAttn a) {
  static_assert(NW == 4 || NW == 8, "a wave takes a page of K and of V, or one of the two");
  constexpr bool WIDE = KIND == PAGES_ALL, SCALED = KIND != PAGES_F16;
  constexpr int OWN = 8 / NW, BM = 16 * RT * NW, PAGE = PS * D / 8;   // 16-byte units of a tile
  __shared__ u4 tiles[2][2][4][PAGE];                            // [buffer][K, V][page]
  __shared__ u4 rest[WIDE ? 2 : 1][2][4][WIDE ? PAGE : 1];       // of wide pages: what their tiles leave
  __shared__ u4 none[WIDE ? PAGE : 1];                           // zeros
  __shared__ u4 special_in[2];                                   // a word a page: V has infinite or NaN values
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

  // entries 64 at a time: lane i holds entry i of the block, in `next` of the block after it
  const int32_t* row = a.table + kvrow * a.W;
  auto entry = [&](int k) { return page_entry<D, KIND>(a, row, e0 + k, e1); };
  PageEntry now = entry(lane), next = entry(64 + lane);
  auto id_of = [&](int k) {
    const int here = __builtin_amdgcn_readlane(now.id, k & 63), after = __builtin_amdgcn_readlane(next.id, k & 63);
    return k < 64 ? here : after;
  };
  auto tag_of = [&](int k) {
    if constexpr (!SCALED) return (int)IAK_TAG_FP16;
    const int here = __builtin_amdgcn_readlane(now.tag, k & 63), after = __builtin_amdgcn_readlane(next.tag, k & 63);
    return k < 64 ? here : after;
  };
  auto pick = [&](float here, float after, int k) { return k < 64 ? lane_f(here, k & 63) : lane_f(after, k & 63); };

  // this wave's page of a step, of K and V or of one of them: loaded a step ahead, put into LDS during
  // the step before
  const int own = w & 3, side = w >> 2;
  PageRaw<D> raw[OWN];
  auto load = [&](int k) __attribute__((always_inline)) {
    const int id = id_of(k), tag = tag_of(k);
#pragma unroll
    for (int o = 0; o < OWN; ++o) load_page<D, KIND, false>(raw[o], a, OWN == 2 ? o == 1 : side == 1, id, tag, lane);
  };
  auto convert = [&](int buf, int k) __attribute__((always_inline)) {
    const int id = id_of(k), tag = tag_of(k);
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int s = OWN == 2 ? o : side;
      const float f = !SCALED ? 1.f : s ? pick(now.vf, next.vf, k) : pick(now.kf, next.kf, k);
      const bool odd = store_page<D, KIND, true>(raw[o], id, tag, f, tiles[buf][s][own], rest[WIDE ? buf : 0][s][own], lane);
      const uint64_t any = __builtin_amdgcn_ballot_w64(odd);
      if (s == 1 && lane == 0) reinterpret_cast<uint32_t*>(&special_in[buf])[own] = any != 0;
    }
  };

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
  int k = 0, block = 0;                                          // number of entry e in the block
  auto step = [&](int buf, int e) __attribute__((always_inline)) {
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
    const int id[4] = {id_of(k), id_of(k + 1), id_of(k + 2), id_of(k + 3)};
    float km[4], vl[4];
    bool wide[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      km[p] = SCALED ? pick(now.km, next.km, k + p) : 1.f;
      vl[p] = SCALED ? pick(now.vl, next.vl, k + p) : 0.f;
      wide[p] = WIDE && id[p] >= 0 && wide_tag(tag_of(k + p));
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
    const u4 sp = special_in[buf];
    convert(buf ^ 1, k + 4 + own);
    load(k + 8 + own);
    const uint32_t special = __builtin_amdgcn_readfirstlane(sp[0] | sp[1] | sp[2] | sp[3]);
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
    auto values = [&](auto cleaned) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb) {
          h8 va = values_back<D>(tiles[buf][1][2 * h], tiles[buf][1][2 * h + 1], mb, c, g);
          if constexpr (decltype(cleaned)::value) va = clean(va);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[t][h], acc[t][mb], 0, 0, 0);
            if constexpr (QF32) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[t][h], acc[t][mb], 0, 0, 0);
          }
        }
    };
    if constexpr (!SCALED) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[t][h], l[t], 0, 0, 0);
          if constexpr (QF32) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[t][h], l[t], 0, 0, 0);
        }
    }
    if (special == 0) {
      values(Plain{});
    } else {
      values(Cleaned{});
#pragma unroll
      for (int p = 0; p < 4; ++p) add_special<D, RT>(acc, tiles[buf][1][p], id[p], (e + p) * PS, seen, g);
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
    if (k == 64) {
      k = 0;
      block += 64;
      now = next;
      next = entry(block + 64 + lane);
    }
    __syncthreads();                                             // this buffer is free, the other one is whole
  };
  if (e0 < e1) {
    load(own);
    convert(0, own);
    load(4 + own);
    __syncthreads();
    for (int e = e0; e < e1; e += 8) {
      step(0, e);
      if (e + 4 < e1) step(1, e + 4);
    }
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
  if (a.q_dtype == IAK_DTYPE_F32) launch_tiles<D, true, 4, 2>(a, stream);
  else if (a.tile_rows == 256) launch_tiles<D, false, 8, 2>(a, stream);
  else launch_tiles<D, false, 4, 2>(a, stream);
}

}  // namespace

void launch_page_chunk(const PageAttn& a, hipStream_t stream) {
  if (a.D == 128) launch_chunk<128>(a, stream);
  else launch_chunk<64>(a, stream);
}

}  // namespace iak
