// Attention of one or several query tokens per sequence over the microscaled 4-bit cache,
// for gfx950:  out = softmax(sm_scale q . k) v  over the tokens that a query sees.
//
// A workgroup takes a tile of 16 query rows that share a KV head (row = query token * G +
// head of the group) and one split of the head's table entries; its waves share the entries
// out in pairs of pages (32 tokens), one pair a step, and their sums meet in LDS at the end.
// Lane = c + 16 g (c = lane % 16, g = lane / 16):
//   scores  S^T[16 tok x 16 rows] = K . Q^T, v_mfma_f32_16x16x32_f16. A lane loads token c's
//           codes of channels (D/4) g .. : its 16 bytes are one scale block (D = 128), so one
//           conversion instruction per pair applies the lane's own scale. The products take the
//           channels in that order on both sides.
//   softmax in base 2, the running maximum moved only when a step exceeds it by 2^8; weights
//           are exp2(s - m + P_SHIFT): of float16's range most lies below 1.
//   values  O^T[D x 16 rows] += V^T[D x 32 tok] . P^T, v_mfma_f32_16x16x32_f16. The score result
//           has the weights of tokens 4g .. 4g+3 of both pages in the lane that the B operand
//           needs them in. V is converted as K is and turned over through LDS: rows written as
//           they lie, read back by ds_read_b64_tr_b16 as four tokens of one channel.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "mx_internal.h"
#include "mx_format.h"
#include "mx_attention.h"
#include "mx_merge.h"

namespace iak {

namespace {

template <int D> struct MxPair {   // two pages as a lane loads them
  uint32_t k[2][D / 32], v[2][D / 32];
  uint32_t ks[2], vs[2];           // four scale bytes, the lane's own among them (own_scale)
  int id[2];                       // wave-uniform; -1: no page
};

template <int D>
__device__ __forceinline__ void load_pair(MxPair<D>& r, const MxAttn& a, int id0, int id1, int c, int g) {
  r.id[0] = id0;
  r.id[1] = id1;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t page = r.id[p] < 0 ? 0 : r.id[p];
    const uint32_t code = c * (D / 2) + g * (D / 8);
    const uint8_t* kc = a.k_codes + page * (PS * D / 2);
    const uint8_t* vc = a.v_codes + page * (PS * D / 2);
    if constexpr (D == 128) {
      const u4 k = ld_nt(reinterpret_cast<const u4*>(kc + code)), v = ld_nt(reinterpret_cast<const u4*>(vc + code));
#pragma unroll
      for (int i = 0; i < 4; ++i) { r.k[p][i] = k[i]; r.v[p][i] = v[i]; }
    } else {
      const u2 k = ld_nt(reinterpret_cast<const u2*>(kc + code)), v = ld_nt(reinterpret_cast<const u2*>(vc + code));
#pragma unroll
      for (int i = 0; i < 2; ++i) { r.k[p][i] = k[i]; r.v[p][i] = v[i]; }
    }
    r.ks[p] = scale_word<D>(a.k_scales + page * (PS * D / MX_BLOCK), c, g);
    r.vs[p] = scale_word<D>(a.v_scales + page * (PS * D / MX_BLOCK), c, g);
  }
}

// Entry i of the wave's own, of those that the workgroup's NW waves share out in pairs.
template <int NW> __device__ __forceinline__ int wave_entry(int w, int i) { return 2 * (w + NW * (i >> 1)) + (i & 1); }

template <int D, bool QF32, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 && !QF32 ? 3 : 2) void mx_rows_kernel(const MxAttn a) {
  __shared__ u4 vt[NW][2 * PS * D / 8];                          // V rows; at the end the waves' sums
  __shared__ float part_m[NW][16], part_l[NW][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const MxPart part = NW == 4 && a.shares ? mx_shared_part<2 * NW, false>(a) : mx_fixed_part(a);
  if (part.idle) return;                                         // uniform, as below
  const int64_t kvrow = part.kvrow;
  const int tile = part.tile;
  const int b = (int)(part.kvrow / (uint32_t)a.Hkv), hk = (int)(part.kvrow - (uint32_t)b * a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * 16, 16);
  const int e0 = part.e0, e1 = e0 + part.chunk < entries ? e0 + part.chunk : entries;
  if (e0 > 0 && e0 >= e1) return;                                // the merge does not look at it

  const int r = tile * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const bool active = r < a.L * a.G, live = active && i < n.queries;
  const int seen[1] = {live ? mx_seen(a, n, i) : 0};
  int least = live ? seen[0] : 0x7FFFFFFF;                       // tokens below it need no mask
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(least, o, 64); least = x < least ? x : least; }

  // the wave's entries, 64 at a time: lane i holds number i of the block, in
  // `next` of the block after it
  const int32_t* row = a.table + kvrow * a.W;
  auto entry_id = [&](int k) {
    const int e = e0 + wave_entry<NW>(w, k);
    return e < e1 ? row[e] : -1;
  };
  int ids = entry_id(lane), next = entry_id(64 + lane);
  const uint32_t pages = (uint32_t)a.NP;
  auto page = [&](int k) {
    const int here = __builtin_amdgcn_readlane(ids, k & 63), after = __builtin_amdgcn_readlane(next, k & 63);
    const int id = k < 64 ? here : after;
    return (uint32_t)id < pages ? id : -1;
  };

  h8 qhi[D / 32], qlo[QF32 ? D / 32 : 1];
  const float mult[1] = {load_query<D, QF32>(a, active, b * a.qsb + i * a.qst + head * a.qsh, g, qhi, qlo)};

  f4 acc[1][D / 16], l[1] = {{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) acc[0][mb] = f4{0.f, 0.f, 0.f, 0.f};
  float m[1] = {M_NONE};

  // one step: the pair `x` of entries e, e + 1; then `x` is the pair of pages to0, to1
  auto step = [&](MxPair<D>& x, int e, int to0, int to1) {
    f4 s[1][2] = {{{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}};
    const uint32_t kb[2] = {own_scale<D>(x.ks[0], c, g), own_scale<D>(x.ks[1], c, g)};
    const uint32_t vb[2] = {own_scale<D>(x.vs[0], c, g), own_scale<D>(x.vs[1], c, g)};
    const float ks[2] = {mx_scale(kb[0]), mx_scale(kb[1])}, vs[2] = {mx_scale(vb[0]), mx_scale(vb[1])};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t o[4];
        mx8_to_f16(x.k[p][j], ks[p], o);
        const h8 ka = make_h8(o[0], o[1], o[2], o[3]);
        s[0][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[j], s[0][p], 0, 0, 0);
        if constexpr (QF32) s[0][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[j], s[0][p], 0, 0, 0);
      }

    // V: rows of this lane's token into LDS, while the scores are under way
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t o[4];
        mx8_to_f16(x.v[p][j], vs[p], o);
        vt[w][p * (PS * D / 8) + v_chunk<D>(c, g * (D / 32) + j)] = u4{o[0], o[1], o[2], o[3]};
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");

    // what is left to do with the pair: which tokens are NaN (rare), which pages are none
    uint32_t most = kb[0] > kb[1] ? kb[0] : kb[1], vmost = vb[0] > vb[1] ? vb[0] : vb[1];
    most = most > vmost ? most : vmost;
    uint32_t nan_tokens[2] = {0u, 0u};
    if (__builtin_amdgcn_ballot_w64(most == MX_SCALE_NAN)) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint64_t bad = __builtin_amdgcn_ballot_w64(kb[p] == MX_SCALE_NAN || vb[p] == MX_SCALE_NAN);
        nan_tokens[p] = (uint32_t)(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xFFFFu;
      }
    }
    const int id[2] = {x.id[0], x.id[1]};
    load_pair<D>(x, a, to0, to1, c, g);                          // under way during the rest of the step

    hide<2, 1>(s, nan_tokens, id, e, seen, least, g);
    raise<D, 2, 1>(s, mult, m, l, acc);
    soften<2>(s[0], mult[0], m[0]);
    l[0] += s[0][0] + s[0][1];
    const h8 pb = weights(s[0][0], s[0][1]);
    h8 pl;
    if constexpr (QF32) pl = weights_rest(s[0][0], s[0][1], pb);
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) {
      const h8 va = values_back<D>(&vt[w][0], &vt[w][PS * D / 8], mb, c, g);
      acc[0][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[0][mb], 0, 0, 0);
      if constexpr (QF32) acc[0][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, acc[0][mb], 0, 0, 0);
    }
  };

  // Twelve waves a CU are what hides the loads: a ring of two or more pairs cost registers and was
  // slower, as were sixteen waves of fewer registers. 256 rows of 32,768 tokens (1.14 GB) take 188 us
  // in three parts each (6.1 TB/s; 192 shared out, 182 unsplit in eight waves a tile); loads that stay
  // in the caches took 216 where these took 190. Short rows wait: launch, length and table, pages, LDS
  // and store in turn are 5.5 us, and a merge kernel 4 more: 52 rows of 5,750 tokens (39 MB) take 14 + 4
  // us. Loads that wait for no other issued first (table, query, length) changed nothing.
  MxPair<D> x;
  if (e0 + 2 * w < e1) load_pair<D>(x, a, page(0), page(1), c, g);
  for (int at = e0 + 2 * w, k = 0, block = 0; at < e1; at += 2 * NW) {
    step(x, at, page(k + 2), page(k + 3));                       // past the end: no page, page 0 is loaded
    k += 2;
    if (k == 64) {
      k = 0;
      block += 64;
      ids = next;
      next = entry_id(block + 64 + lane);
    }
  }

  // the waves' sums meet in LDS (rows c, 16-byte units turned by c against bank conflicts)
  const float sum = xsum16_32((l[0][0] + l[0][1]) + (l[0][2] + l[0][3]));
  __syncthreads();
  if (g == 0) { part_m[w][c] = m[0]; part_l[w][c] = sum; }
  f4* sums = reinterpret_cast<f4*>(&vt[w][0]);
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) sums[c * (D / 4) + ((4 * mb + g) ^ c)] = acc[0][mb];
  __syncthreads();
  const int rows = a.L * a.G - tile * 16 < 16 ? a.L * a.G - tile * 16 : 16;
  for (int k2 = threadIdx.x; k2 < rows * (D / 4); k2 += 64 * NW) {
    const int cr = k2 / (D / 4), u = k2 - cr * (D / 4);
    float M = part_m[0][cr], L = 0.f;
#pragma unroll
    for (int v = 1; v < NW; ++v) M = fmaxf(M, part_m[v][cr]);
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float wgt = __builtin_amdgcn_exp2f(part_m[v][cr] - M);
      L += wgt * part_l[v][cr];
      o += reinterpret_cast<const f4*>(&vt[v][0])[cr * (D / 4) + (u ^ cr)] * wgt;
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

template <int D, bool QF32> void launch_rows(const MxAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items);
  constexpr int MANY = D == 128 ? 8 : 16;
  if (a.waves > 4) hipLaunchKernelGGL((mx_rows_kernel<D, QF32, MANY>), grid, dim3(64 * MANY), 0, stream, a);
  else hipLaunchKernelGGL((mx_rows_kernel<D, QF32, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_mx_attention(const MxAttn& a, hipStream_t stream) {
  const bool f32 = a.q_dtype == IAK_DTYPE_F32;
  if (a.tile_rows > 16) launch_mx_chunk(a, stream);
  else if (a.D == 128) f32 ? launch_rows<128, true>(a, stream) : launch_rows<128, false>(a, stream);
  else f32 ? launch_rows<64, true>(a, stream) : launch_rows<64, false>(a, stream);
  if (a.parted) {
    if (a.D == 128) launch_mx_merge<128>(a, stream);
    else launch_mx_merge<64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace iak
