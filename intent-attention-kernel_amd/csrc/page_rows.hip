// Attention of one or several query tokens per sequence over pages of mixed precision, for gfx950:
// few query rows of a KV head (drafted tokens, short chunks). out = softmax(sm_scale q . k) v over the tokens
// that a query sees.
//
// A workgroup takes a tile of 16 query rows that share a KV head (row = query token * G + head of
// the group) and one part of the head's table entries; its waves share the entries out in pairs of
// pages (32 tokens), one pair a step, and their sums meet in LDS at the end. A wave loads its pages
// as whole lines and turns them into operands through LDS of its own, K and V one after the other
// (page_attention.h), so that no wave waits for another. Lane = c + 16 g:
//   scores  S^T[16 tok x 16 rows] = K . Q^T, v_mfma_f32_16x16x32_f16, channels (D/4) g .. on both sides
//   values  O^T[D x 16 rows] += V^T[D x 32 tok] . P^T; the score result has the weights of tokens
//           4g .. 4g+3 of both pages in the lane that the operand needs them in

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "page_attention.h"
#include "mx_merge.h"

namespace iak {

namespace {

constexpr int ROW_WAVES = 4;

// Entry i of the wave's own, of those that the workgroup's waves share out in pairs.
__device__ __forceinline__ int wave_entry(int w, int i) { return 2 * (w + ROW_WAVES * (i >> 1)) + (i & 1); }

template <int D, bool QF32, int KIND>
__global__ __launch_bounds__(64 * ROW_WAVES, 2) void page_rows_kernel(const PageAttn a) {
  constexpr bool WIDE = KIND == PAGES_ALL;
  constexpr int PAGE = PS * D / 8;                               // 16-byte units of a tile
  __shared__ u4 tiles[ROW_WAVES][2 * PAGE * (WIDE ? 2 : 1)];     // K's, then V's; at the end the waves' sums
  __shared__ u4 none[WIDE ? PAGE : 1];                           // zeros
  __shared__ uint16_t special[ROW_WAVES][PAGE];
  __shared__ float part_m[ROW_WAVES][16], part_l[ROW_WAVES][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const MxPart part = a.shares ? mx_shared_part<2 * ROW_WAVES, false>(a) : mx_fixed_part(a);
  if (part.idle) return;                                         // uniform, as below
  const int64_t kvrow = part.kvrow;
  const int tile = part.tile;
  const int b = (int)(part.kvrow / (uint32_t)a.Hkv), hk = (int)(part.kvrow - (uint32_t)b * a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * 16, 16);
  const int e0 = part.e0, e1 = e0 + part.chunk < entries ? e0 + part.chunk : entries;
  if (e0 > 0 && e0 >= e1) return;                                // the merge does not look at it
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < PAGE; i += 64 * ROW_WAVES) none[i] = u4{0u, 0u, 0u, 0u};
    __syncthreads();
  }

  const int r = tile * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const bool active = r < a.L * a.G, live = active && i < n.queries;
  const int seen[1] = {live ? mx_seen(a, n, i) : 0};
  int least = live ? seen[0] : 0x7FFFFFFF;                       // tokens below it need no mask
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(least, o, 64); least = x < least ? x : least; }

  // the wave's entries, 64 at a time: lane i holds number i of the block, in `next` of the block after it
  const int32_t* row = a.table + kvrow * a.W;
  auto entry = [&](int k) { return page_entry<D, KIND>(a, row, e0 + wave_entry(w, k), e1); };
  PageEntry now = entry(lane), next = entry(64 + lane);
  auto pick = [&](int here, int after, int k) {
    const int x = __builtin_amdgcn_readlane(here, k & 63), y = __builtin_amdgcn_readlane(after, k & 63);
    return k < 64 ? x : y;
  };
  auto pick_f = [&](float here, float after, int k) { return u2f((uint32_t)pick((int)f2u(here), (int)f2u(after), k)); };
  auto of = [&](int k) __attribute__((always_inline)) {          // entry k of the block, k < 128
    PageEntry y = {pick(now.id, next.id, k), IAK_TAG_FP16, 1.f, 1.f, 0.f, 1.f};
    if constexpr (KIND != PAGES_F16) {
      y.tag = pick(now.tag, next.tag, k);
      y.km = pick_f(now.km, next.km, k);
      y.kf = pick_f(now.kf, next.kf, k);
      y.vl = pick_f(now.vl, next.vl, k);
      y.vf = pick_f(now.vf, next.vf, k);
    }
    return y;
  };

  h8 qhi[D / 32], qlo[QF32 ? D / 32 : 1];
  const float mult[1] = {load_query<D, QF32>(a, active, b * a.qsb + i * a.qst + head * a.qsh, g, qhi, qlo)};

  f4 acc[1][D / 16];
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) acc[0][mb] = f4{0.f, 0.f, 0.f, 0.f};
  float m[1] = {M_NONE}, l[1] = {0.f};
  int E = 0;
  u4* mine = tiles[w];
  Seen16 odd = {0u, 0u};

  PageRaw<D> k[2], v[2];
  PageEntry at[2];                                               // of the pair that k and v hold
  auto look_up = [&](int i) __attribute__((always_inline)) {
    at[0] = of(i);
    at[1] = of(i + 1);
  };
  auto load = [&](PageRaw<D> (&x)[2], bool side) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p) load_page<D, KIND, true>(x[p], a, side, at[p].id, at[p].tag, lane);
  };

  int number = 0, block = 0;                                     // the next pair, of the block of 64 entries
  if (e0 + 2 * w < e1) {
    look_up(0);
    load(k, false);
    load(v, true);
  }
  for (int e = e0 + 2 * w; e < e1; e += 2 * ROW_WAVES) {
    const PageEntry x[2] = {at[0], at[1]};
    const int id[2] = {x[0].id, x[1].id};
    const bool wide[2] = {WIDE && id[0] >= 0 && wide_tag(x[0].tag), WIDE && id[1] >= 0 && wide_tag(x[1].tag)};
    const float km[2] = {x[0].km, x[1].km};

    // K into LDS and back as operands
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < 2; ++p)
      store_page<D, KIND, false>(k[p], id[p], x[p].tag, x[p].kf, mine + p * PAGE, mine + (2 + p) * PAGE, lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    number += 2;
    look_up(number);                                             // the next pair: under way from here
    load(k, false);
    f4 s[1][2] = {{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const h8 ka = __builtin_bit_cast(h8, mine[p * PAGE + v_chunk<D>(c, g * (D / 32) + j)]);
        s[0][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[j], s[0][p], 0, 0, 0);
        if constexpr (QF32) s[0][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[j], s[0][p], 0, 0, 0);
      }
    if constexpr (WIDE) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        if (!wide[p]) continue;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const h8 ka = __builtin_bit_cast(h8, mine[(2 + p) * PAGE + v_chunk<D>(c, g * (D / 32) + j)]);
          s[0][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[j], s[0][p], 0, 0, 0);
        }
      }
    }

    // V in K's place
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const bool any = store_page<D, KIND, true>(v[p], id[p], x[p].tag, x[p].vf, mine + p * PAGE, mine + (2 + p) * PAGE, lane);
      if (__builtin_amdgcn_ballot_w64(any)) {
        put_aside<D>(mine + p * PAGE, special[w], lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int first = (e + p) * PS;
        remember<D>(odd, special[w], seen[0] - first < PS ? seen[0] - first : PS, g);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    load(v, true);

    const uint32_t no_nan[2] = {0u, 0u};
    hide<2, 1>(s, no_nan, id, e, seen, least, g);
    raise_scaled<D, 2, 1>(s, km, mult, m, l, acc);
    float vl[2] = {0.f, 0.f}, out[2] = {1.f, 1.f};
    if constexpr (KIND != PAGES_F16) {
      const float all[2] = {id[0] < 0 ? NO_SCALE : x[0].vl, id[1] < 0 ? NO_SCALE : x[1].vl};
      const int to = value_power<2>(all, E);
      if (to != E) {                                             // uniform
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[0][mb][q] = __builtin_ldexpf(acc[0][mb][q], E - to);
        E = to;
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        vl[p] = id[p] < 0 ? 0.f : x[p].vl - (float)E;
        out[p] = __builtin_amdgcn_exp2f(-vl[p]);
      }
    }
    l[0] += soften_scaled<2>(s[0], km, vl, out, mult[0], m[0]);
    const h8 pb = weights(s[0][0], s[0][1]);
    h8 pl;
    if constexpr (QF32) pl = weights_rest(s[0][0], s[0][1], pb);
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) {
      const h8 va = values_back<D>(mine, mine + PAGE, mb, c, g);
      acc[0][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[0][mb], 0, 0, 0);
      if constexpr (QF32) acc[0][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, acc[0][mb], 0, 0, 0);
    }
    if constexpr (WIDE) {
      if (wide[0] || wide[1]) {
        const u4* p0 = wide[0] ? mine + 2 * PAGE : none;
        const u4* p1 = wide[1] ? mine + 3 * PAGE : none;
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb)
          acc[0][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(values_back<D>(p0, p1, mb, c, g), pb, acc[0][mb], 0, 0, 0);
      }
    }
    if (number == 64) {
      number = 0;
      now = next;
      // the entries of two blocks on, past what this one and the next hold
      block += 64;
      next = entry(block + 64 + lane);
    }
  }

  if (__builtin_amdgcn_ballot_w64((odd.plus | odd.minus) != 0u)) bring_back<D>(acc[0], odd);

  // the waves' sums meet in LDS (rows c, 16-byte units turned by c against bank conflicts)
  const float sum = xsum16_32(l[0]);
  __syncthreads();
  if (g == 0) { part_m[w][c] = m[0]; part_l[w][c] = sum; }
  f4* sums = reinterpret_cast<f4*>(mine);
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) {
    f4 x;
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = __builtin_ldexpf(acc[0][mb][q], E);
    sums[c * (D / 4) + ((4 * mb + g) ^ c)] = x;
  }
  __syncthreads();
  const int rows = a.L * a.G - tile * 16 < 16 ? a.L * a.G - tile * 16 : 16;
  for (int k2 = threadIdx.x; k2 < rows * (D / 4); k2 += 64 * ROW_WAVES) {
    const int cr = k2 / (D / 4), u = k2 - cr * (D / 4);
    float M = part_m[0][cr], L = 0.f;
#pragma unroll
    for (int x = 1; x < ROW_WAVES; ++x) M = fmaxf(M, part_m[x][cr]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < ROW_WAVES; ++x) {
      const float wgt = __builtin_amdgcn_exp2f(part_m[x][cr] - M);
      L += wgt * part_l[x][cr];
      o += reinterpret_cast<const f4*>(&tiles[x][0])[cr * (D / 4) + (u ^ cr)] * wgt;
    }
    if (a.parted) {
      const int64_t slot = (int64_t)part.part * 16 + cr;
      if (u == 0) { a.ws_m[slot] = M; a.ws_l[slot] = L; }
      *reinterpret_cast<f4*>(a.ws_acc + slot * D + 4 * u) = o;
    } else {
      const int rr = tile * 16 + cr, ir = rr / a.G;
      const float inv = L == 0.f ? 0.f : 1.0f / L;               // NaN stays
      float out[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) out[q] = ir < n.queries ? o[q] * inv : 0.f;
      store_out4(a, b * a.osb + ir * a.ost + (hk * a.G + rr - ir * a.G) * a.osh + 4 * u, out);
    }
  }
}

template <int D, bool QF32> void launch_rows(const PageAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items), block(64 * ROW_WAVES);
  if (a.kind == PAGES_F16) hipLaunchKernelGGL((page_rows_kernel<D, QF32, PAGES_F16>), grid, block, 0, stream, a);
  else if (a.kind == PAGES_BYTE) hipLaunchKernelGGL((page_rows_kernel<D, QF32, PAGES_BYTE>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((page_rows_kernel<D, QF32, PAGES_ALL>), grid, block, 0, stream, a);
}

}  // namespace

void launch_page_rows(const PageAttn& a, hipStream_t stream) {
  const bool f32 = a.q_dtype == IAK_DTYPE_F32;
  if (a.D == 128) f32 ? launch_rows<128, true>(a, stream) : launch_rows<128, false>(a, stream);
  else f32 ? launch_rows<64, true>(a, stream) : launch_rows<64, false>(a, stream);
}

hipError_t launch_page_attention(const PageAttn& a, hipStream_t stream) {
  if (a.tile_rows > 16) launch_page_chunk(a, stream);
  else launch_page_rows(a, stream);
  if (a.parted) {
    if (a.D == 128) launch_mx_merge<128>(a, stream);
    else launch_mx_merge<64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace iak
