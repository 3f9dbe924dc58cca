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

namespace iak {

namespace {

constexpr float P_SHIFT = 6.0f;          // weights <= 2^(6 + RESCALE_SLACK) = 2^14
constexpr float M_NONE = -3.402823466e38f;

typedef short s4v __attribute__((ext_vector_type(4)));

// 16-byte chunk of V row `t` (of a page) that holds logical chunk `ch`: rows are 2 D bytes, and
// the exclusive or lets both the row-wise writes (one chunk of 16 rows, four chunks apart) and
// the transposed reads (two chunks of 16 rows) touch every LDS bank equally.
template <int D> __device__ __forceinline__ int v_chunk(int t, int ch) {
  if constexpr (D == 128) return t * 16 + (ch ^ (((t & 7) << 1) | (t >> 3)));
  else return t * 8 + (ch ^ ((((t >> 1) & 3) << 1) | (t >> 3)));
}

template <int D> struct MxPair {   // two pages as a lane loads them
  uint32_t k[2][D / 32], v[2][D / 32];
  uint32_t ks[2], vs[2];           // four scale bytes, the lane's own among them (own_scale)
  int id[2];                       // wave-uniform; -1: no page
};

// A lane's scale bytes come as the aligned four they are among: a byte loaded alone is zero-
// extended where the loop turns, and that waits for loads that the next round is meant to await.
template <int D> __device__ __forceinline__ uint32_t scale_word(const uint8_t* page_scales, int c, int g) {
  return reinterpret_cast<const uint32_t*>(page_scales)[(c * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK) >> 2];
}
template <int D> __device__ __forceinline__ uint32_t own_scale(uint32_t word, int c, int g) {
  return __builtin_amdgcn_ubfe(word, 8 * ((c * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK) & 3), 8);
}

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

template <typename T> __device__ __forceinline__ void out4(T* p, const float (&x)[4]) {
  T t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (T)x[j];
  __builtin_memcpy(p, t, sizeof(t));                             // one store, wherever the row lies
}
__device__ __forceinline__ void store_out4(const MxAttn& a, int64_t at, const float (&x)[4]) {
  if (a.out_dtype == IAK_DTYPE_F32) out4(reinterpret_cast<float*>(a.out) + at, x);
  else if (a.out_dtype == IAK_DTYPE_F16) out4(reinterpret_cast<_Float16*>(a.out) + at, x);
  else out4(reinterpret_cast<__bf16*>(a.out) + at, x);
}

// A query row's operand: the lane's channels (D/4) g .., scaled by a power of two to a largest
// element of the row in [2^14, 2^15), split in two for float32. Returns the factor that makes
// base-2 scores of the products: positive, NaN for a row that is not finite. (A negative scale
// turns the query's sign; where the factor would vanish the scores do: query 0, factor 1.)
template <int D, bool QF32>
__device__ __forceinline__ float load_query(const MxAttn& a, bool there, int64_t at, int g, h8 (&qhi)[D / 32],
                                            h8 (&qlo)[QF32 ? D / 32 : 1]) {
  float x[D / 4];
#pragma unroll
  for (int j = 0; j < D / 4; ++j) x[j] = 0.f;
  if (there) mx_load_q(a, at + g * (D / 4), x);
  float m = 0.f, nan = 0.f;                                      // nan: NaN if any value is infinite or NaN, else 0
#pragma unroll
  for (int j = 0; j < D / 4; ++j) {
    m = fmaxf(m, fabsf(x[j]));
    nan = __builtin_fmaf(x[j], 0.f, nan);
  }
  bool fine = nan == 0.f;
  m = xmax16_32(fine ? m : __builtin_inff());
  fine = m < __builtin_inff();
  const int e = m > 0.f ? (int)(f2u(m) >> 23) - 127 : 0;
  const float mult = __builtin_ldexpf(fabsf(a.score_mult), e - 14);
  const bool none = !fine || mult < 1e-30f;
  const float sign = a.score_mult < 0.f ? -1.f : 1.f;
#pragma unroll
  for (int s = 0; s < D / 32; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = none ? 0.f : sign * __builtin_ldexpf(x[8 * s + j], 14 - e);
      qhi[s][j] = (_Float16)v;
      if constexpr (QF32) qlo[s][j] = (_Float16)(v - (float)qhi[s][j]);
    }
  return !fine ? __builtin_nanf("") : none ? 1.f : mult;
}

// The softmax of PAGES pages' score results (lane: row c of T tiles, tokens 4g .. 4g+3 of each
// page), in three parts, each of which leaves the straight line at one rarely taken branch:
//   hide    scores become NaN where a token has a NaN block (bit per token in `nan`) and -inf
//           where the row does not see it; `e`: the first page's entry, `least`: tokens that
//           every row of the wave sees
//   raise   moves a row's running maximum m, with its sum l and accumulator, where a score
//           exceeds it by more than the slack: the lanes of a row compare theirs only then
//   soften  scores become the weights exp2(s * mult - m + P_SHIFT)
template <int PAGES, int T>
__device__ __forceinline__ void hide(f4 (&s)[T][PAGES], const uint32_t (&nan)[PAGES], const int (&id)[PAGES], int e,
                                     const int (&seen)[T], int least, int g) {
  uint32_t any_nan = 0u;
  int ids = 0;
#pragma unroll
  for (int p = 0; p < PAGES; ++p) { any_nan |= nan[p]; ids |= id[p]; }
  if (any_nan != 0u || ids < 0 || (e + PAGES) * PS > least) {
    asm volatile("");                                            // a branch, not selects for every call
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int p = 0; p < PAGES; ++p) {
        const int lim = id[p] < 0 ? 0 : seen[t] - (e + p) * PS;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if ((nan[p] >> (4 * g + q)) & 1u) s[t][p][q] = __builtin_nanf("");
          if (4 * g + q >= lim) s[t][p][q] = -__builtin_inff();
        }
      }
  }
}

template <int D, int PAGES, int T>
__device__ __forceinline__ void raise(const f4 (&s)[T][PAGES], const float (&mult)[T], float (&m)[T], f4 (&l)[T],
                                      f4 (&acc)[T][D / 16]) {
  float top[T];
  bool over = false;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    top[t] = fmaxf(fmaxf(s[t][0][0], s[t][0][1]), fmaxf(s[t][0][2], s[t][0][3]));
#pragma unroll
    for (int p = 1; p < PAGES; ++p)
      top[t] = fmaxf(top[t], fmaxf(fmaxf(s[t][p][0], s[t][p][1]), fmaxf(s[t][p][2], s[t][p][3])));
    over = over || top[t] * mult[t] > m[t] + RESCALE_SLACK;
  }
  if (__builtin_amdgcn_ballot_w64(over)) {
    asm volatile("");
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float pm = xmax16_32(top[t]) * mult[t];
      const float mn = pm > m[t] + RESCALE_SLACK ? pm : m[t];
      const float alpha = __builtin_amdgcn_exp2f(m[t] - mn);
      l[t] *= alpha;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) acc[t][mb] *= alpha;
      m[t] = mn;
    }
  }
}

template <int PAGES> __device__ __forceinline__ void soften(f4 (&s)[PAGES], float mult, float m) {
  const float base = P_SHIFT - m;
#pragma unroll
  for (int p = 0; p < PAGES; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) s[p][q] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[p][q], mult, base));
}

// Weights of two pages as the value product's operand, and what rounding left (float32 queries).
__device__ __forceinline__ h8 weights(const f4 a, const f4 b) {
  return h8{(_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3],
            (_Float16)b[0], (_Float16)b[1], (_Float16)b[2], (_Float16)b[3]};
}
__device__ __forceinline__ h8 weights_rest(const f4 a, const f4 b, const h8 w) {
  h8 r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    r[q] = (_Float16)(a[q] - (float)w[q]);
    r[4 + q] = (_Float16)(b[q] - (float)w[4 + q]);
  }
  return r;
}

// The value product's operand from two pages' V rows in LDS: channel 16 mb + c of tokens
// 4g .. 4g+3 of both.
template <int D> __device__ __forceinline__ h8 values_back(const u4* page0, const u4* page1, int mb, int c, int g) {
  typedef __attribute__((address_space(3))) s4v lds_s4;
  const int at = v_chunk<D>(4 * g + (c >> 2), 2 * mb + ((c & 3) >> 1)) * 16 + (c & 1) * 8;
  const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(reinterpret_cast<const char*>(page0) + at));
  const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(reinterpret_cast<const char*>(page1) + at));
  return __builtin_bit_cast(h8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Entry i of the wave's own, of those that the workgroup's NW waves share out in pairs.
template <int NW> __device__ __forceinline__ int wave_entry(int w, int i) { return 2 * (w + NW * (i >> 1)) + (i & 1); }

template <int D, bool QF32, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 && !QF32 ? 3 : 2) void mx_rows_kernel(const MxAttn a) {
  __shared__ u4 vt[NW][2 * PS * D / 8];                          // V rows; at the end the waves' sums
  __shared__ float part_m[NW][16], part_l[NW][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t tile_at = blockIdx.x / a.splits;
  const int tile = (int)(tile_at % a.tiles);
  const int64_t kvrow = tile_at / a.tiles;
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow % a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * 16, 16);
  const int e0 = split * a.chunk, e1 = e0 + a.chunk < entries ? e0 + a.chunk : entries;
  if (split > 0 && e0 >= e1) return;                             // the merge does not look at it

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
  // slower, as were sixteen waves of fewer registers. The bytes come at the rate that the same
  // loads reach alone, streamed (1.14 GB in 190 us; 216 with loads that stay in the caches).
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
    if (a.splits > 1) {
      const int64_t slot = (int64_t)blockIdx.x * 16 + cr;
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

// Tiles of 64 RT query rows: prompt chunks. The four waves take 16 RT rows each and walk the
// same tokens, 64 (four pages) a step; each wave converts one page of K and V of the next step,
// which all read from LDS (two buffers, one barrier a step): per row, the vector instructions are
// what bounds it, so each code is converted once per workgroup, and the sum of the weights is a
// product with ones on the matrix cores. The rest is the rows kernel's.
template <int D, bool QF32, int RT>
__global__ __launch_bounds__(256, 2) void mx_chunk_kernel(const MxAttn a) {
  __shared__ u4 kt[2][4][PS * D / 8], vt[2][4][PS * D / 8];
  __shared__ u4 nan_in[2];
  constexpr int BM = 64 * RT;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int wide = (a.L * a.G + BM - 1) / BM;                    // tiles of BM rows
  const int split = (int)(blockIdx.x % a.splits);
  const int64_t tile_at = blockIdx.x / a.splits;
  const int64_t kvrow = tile_at / wide;
  const int tile = wide - 1 - (int)(tile_at % wide);             // those that see most first
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow % a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * BM, BM);
  const int e0 = split * a.chunk, e1 = e0 + a.chunk < entries ? e0 + a.chunk : entries;
  if (split > 0 && e0 >= e1) return;                             // uniform; the merge does not look at it

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
  auto entry_id = [&](int k) {
    const int e = e0 + k;
    return e < e1 ? row[e] : -1;
  };
  int ids = entry_id(lane), next = entry_id(64 + lane);
  const uint32_t pages = (uint32_t)a.NP;
  auto page = [&](int k) {
    const int here = __builtin_amdgcn_readlane(ids, k & 63), after = __builtin_amdgcn_readlane(next, k & 63);
    const int id = k < 64 ? here : after;
    return (uint32_t)id < pages ? id : -1;
  };

  // this wave's page of a step: loaded a step ahead, converted into LDS during the step before
  uint32_t kr[D / 32], ks, vr[D / 32], vs;
  auto load_page = [&](int id) {
    const int64_t p = id < 0 ? 0 : id;
    const uint32_t code = c * (D / 2) + g * (D / 8);
    const uint8_t *kc = a.k_codes + p * (PS * D / 2) + code, *vc = a.v_codes + p * (PS * D / 2) + code;
    if constexpr (D == 128) {
      const u4 k = *reinterpret_cast<const u4*>(kc), v = *reinterpret_cast<const u4*>(vc);
#pragma unroll
      for (int i = 0; i < 4; ++i) { kr[i] = k[i]; vr[i] = v[i]; }
    } else {
      const u2 k = *reinterpret_cast<const u2*>(kc), v = *reinterpret_cast<const u2*>(vc);
#pragma unroll
      for (int i = 0; i < 2; ++i) { kr[i] = k[i]; vr[i] = v[i]; }
    }
    ks = scale_word<D>(a.k_scales + p * (PS * D / MX_BLOCK), c, g);
    vs = scale_word<D>(a.v_scales + p * (PS * D / MX_BLOCK), c, g);
  };
  auto convert = [&](int buf) {
    const uint32_t kb = own_scale<D>(ks, c, g), vb = own_scale<D>(vs, c, g);
    const float sk = mx_scale(kb), sv = mx_scale(vb);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      uint32_t o[4];
      mx8_to_f16(kr[j], sk, o);
      kt[buf][w][v_chunk<D>(c, g * (D / 32) + j)] = u4{o[0], o[1], o[2], o[3]};
      mx8_to_f16(vr[j], sv, o);
      vt[buf][w][v_chunk<D>(c, g * (D / 32) + j)] = u4{o[0], o[1], o[2], o[3]};
    }
    const uint64_t bad = __builtin_amdgcn_ballot_w64((kb > vb ? kb : vb) == MX_SCALE_NAN);
    reinterpret_cast<uint32_t*>(&nan_in[buf])[w] = (uint32_t)(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xFFFFu;
  };

  f4 acc[RT][D / 16], l[RT];
  float m[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = M_NONE;
    l[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) acc[t][mb] = f4{0.f, 0.f, 0.f, 0.f};
  }

  const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
  int k = 0, block = 0;                                          // number of entry e in the block
  auto step = [&](int buf, int e) {
    f4 s[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int p = 0; p < 4; ++p) s[t][p] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const h8 ka = __builtin_bit_cast(h8, kt[buf][p][v_chunk<D>(c, g * (D / 32) + j)]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[t][j], s[t][p], 0, 0, 0);
          if constexpr (QF32) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[t][j], s[t][p], 0, 0, 0);
        }
      }
    const u4 bad = nan_in[buf];
    const int id[4] = {page(k), page(k + 1), page(k + 2), page(k + 3)};
    convert(buf ^ 1);
    load_page(page(k + 8 + w));
    uint32_t nan_tokens[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) nan_tokens[p] = __builtin_amdgcn_readfirstlane(bad[p]);
    hide<4, RT>(s, nan_tokens, id, e, seen, least, g);
    raise<D, 4, RT>(s, mult, m, l, acc);
    h8 pb[RT][2], pl[RT][QF32 ? 2 : 1];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      soften<4>(s[t], mult[t], m[t]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pb[t][h] = weights(s[t][2 * h], s[t][2 * h + 1]);
        if constexpr (QF32) pl[t][h] = weights_rest(s[t][2 * h], s[t][2 * h + 1], pb[t][h]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[t][h], l[t], 0, 0, 0);
        if constexpr (QF32) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[t][h], l[t], 0, 0, 0);
      }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        const h8 va = values_back<D>(vt[buf][2 * h], vt[buf][2 * h + 1], mb, c, g);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb[t][h], acc[t][mb], 0, 0, 0);
          if constexpr (QF32) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[t][h], acc[t][mb], 0, 0, 0);
        }
      }
    }
    k += 4;
    if (k == 64) {
      k = 0;
      block += 64;
      ids = next;
      next = entry_id(block + 64 + lane);
    }
    __syncthreads();                                             // this buffer is free, the other one is whole
  };
  if (e0 < e1) {
    load_page(page(w));
    convert(0);
    load_page(page(4 + w));
    __syncthreads();
    for (int e = e0; e < e1; e += 8) {
      step(0, e);
      if (e + 4 < e1) step(1, e + 4);
    }
  }

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = tile * BM + (w * RT + t) * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
    const float sum = l[t][0];
    if (r >= rows) continue;
    if (a.splits > 1) {
      const int64_t slot = ((kvrow * a.tiles + (r >> 4)) * a.splits + split) * 16 + c;
      if (g == 0) { a.ws_m[slot] = m[t]; a.ws_l[slot] = sum; }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) *reinterpret_cast<f4*>(a.ws_acc + slot * D + 16 * mb + 4 * g) = acc[t][mb];
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;           // NaN stays
      const int64_t at = b * a.osb + i * a.ost + head * a.osh + 4 * g;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        float o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = i < n.queries ? acc[t][mb][q] * inv : 0.f;
        store_out4(a, at + 16 * mb, o);
      }
    }
  }
}

// The splits of 256 / (D / 4 PARTS) query rows a workgroup: a thread takes 4 channels of every
// PARTS-th split of its row. PARTS > 1, where a row has many splits, is one row a workgroup.
template <int D, int PARTS>
__global__ __launch_bounds__(256) void mx_merge_kernel(const MxAttn a) {
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
  const int tile = r / 16, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const MxRows n = mx_rows(a, kvrow, b);
  const bool live = i < n.queries;
  const int parts = live && there ? (mx_entries(a, n, tile * 16, 16) + a.chunk - 1) / a.chunk : 0;
  const int64_t first = (kvrow * a.tiles + tile) * a.splits * 16 + (r & 15);
  float M = M_NONE;
  if constexpr (PARTS > 1) {
    for (int s = threadIdx.x; s < parts; s += 256) M = fmaxf(M, a.ws_m[first + (int64_t)s * 16]);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  } else {
    for (int s = 0; s < parts; ++s) M = fmaxf(M, a.ws_m[first + (int64_t)s * 16]);
  }
  float L = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = part; s < parts; s += PARTS) {
    const int64_t slot = first + (int64_t)s * 16;
    const float wgt = __builtin_amdgcn_exp2f(a.ws_m[slot] - M);
    L += wgt * a.ws_l[slot];
    o += ld_nt(reinterpret_cast<const f4*>(a.ws_acc + slot * D + 4 * u)) * wgt;
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

// Rows whose splits a thread walks alone, eight at most; more are shared by a workgroup.
template <int D> void launch_mx_merge(const MxAttn& a, hipStream_t stream) {
  constexpr int UNITS = D / 4;
  const int64_t rows = (int64_t)a.B * a.Hkv * a.L * a.G;
  if (a.splits <= 8) {
    const int per = 256 / UNITS;
    hipLaunchKernelGGL((mx_merge_kernel<D, 1>), dim3((uint32_t)((rows + per - 1) / per)), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((mx_merge_kernel<D, 256 / UNITS>), dim3((uint32_t)rows), dim3(256), 0, stream, a);
  }
}

template <int D, bool QF32> void launch_rows(const MxAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items);
  if (a.chunk_rows) { hipLaunchKernelGGL((mx_chunk_kernel<D, QF32, 2>), grid, dim3(256), 0, stream, a); return; }
  constexpr int MANY = D == 128 ? 8 : 16;
  if (a.waves > 4) hipLaunchKernelGGL((mx_rows_kernel<D, QF32, MANY>), grid, dim3(64 * MANY), 0, stream, a);
  else hipLaunchKernelGGL((mx_rows_kernel<D, QF32, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_mx_attention(const MxAttn& a, hipStream_t stream) {
  const bool f32 = a.q_dtype == IAK_DTYPE_F32;
  if (a.D == 128) f32 ? launch_rows<128, true>(a, stream) : launch_rows<128, false>(a, stream);
  else f32 ? launch_rows<64, true>(a, stream) : launch_rows<64, false>(a, stream);
  if (a.splits > 1) {
    if (a.D == 128) launch_mx_merge<128>(a, stream);
    else launch_mx_merge<64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace iak
