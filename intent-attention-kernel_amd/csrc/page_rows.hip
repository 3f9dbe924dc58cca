// Attention of one or several query tokens per sequence over pages of mixed precision, for gfx950:
// few query rows of a KV head (drafted tokens, short chunks). out = softmax(sm_scale q . k) v over the tokens
// that a query sees.
//
// A workgroup takes a tile of 16 query rows that share a KV head (row = query token * G + head of
// the group) and one part of the head's table entries; each of its waves takes a quarter of these, and their
// sums meet in LDS at the end. A wave sorts its entries, 64 at a time, by precision and goes through each
// precision's pages one by one, the next ones under way in a ring of registers (paged_pages.h, as the
// decode does). Lane = c + 16 g; per page:
//   scores  S^T[16 tok x 16 rows] = K . Q^T, v_mfma_f32_16x16x32_f16, channels (D/4) g .. on both sides
//   values  O^T[D x 16 rows] += V^T[D x 16 tok] . P^T, v_mfma_f32_16x16x16_f16; the score result has the weights
//           of the tokens in the lane that the operand needs them in
// K and V are exact codes, with their scales in the scores and the weights; INT4 codes times their
// groups' scales, which need more bits than float16 has, take two products.
//
// What bounds it: the pages' bytes. Four queries of 16 sequences over up to 16,384 tokens of mixed precision (32
// heads over 8 of 128, 435 MB) take 104 us and 7 of merge, 4.2 TB/s; of float16 pages alone 123 us, 5.9
// TB/s; equal lengths, mixed, 103. A short row waits for length, entry, tag, page and the waves' sums in turn:
// 3 queries over 500 tokens 8 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "page_attention.h"
#include "paged_pages.h"
#include "mx_merge.h"

namespace iak {

namespace {

constexpr int ROW_WAVES = 4;

// A wave's rows: their queries and sums so far.
template <int D, bool QF32> struct RowWave {
  h8 qhi[D / 32], qlo[QF32 ? D / 32 : 1];
  f4 acc[D / 16];          // lane: row c, channels (D/16)(4g + q) + mb
  float mult, m, l;        // of row c: what makes base-2 scores; running maximum; this lane's part of the sum
  int E, top;              // the values' sum is acc 2^E (uniform); the highest E that there were sums at
  int seen, least;         // tokens that row c sees, and that all rows do
  int g;
};

template <int D, bool QF32> __device__ __forceinline__ f4 row_scores(const RowWave<D, QF32>& w, const h8 (&ka)[D / 32], f4 s) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[i], w.qhi[i], s, 0, 0, 0);
    if constexpr (QF32) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[i], w.qlo[i], s, 0, 0, 0);
  }
  return s;
}

// Weights of a page of base-2 scores `s`; `first`: its first token's number; PERM: score r of lane group g is
// token 4r + g (else 4g + r); e: the exponent of V's scale, which E follows (as in the other kernel: moved_power; NO_POWER: not
// this page's). FIXED: all pages' exponents are 0.
template <bool PERM, bool FIXED, int D, bool QF32>
__device__ __forceinline__ f4 row_weights(RowWave<D, QF32>& w, f4 s, int first, int e) {
  if (first + PS > w.least) {                                    // uniform
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (first + (PERM ? 4 * r + w.g : 4 * w.g + r) >= w.seen) s[r] = -__builtin_inff();
  }
  const float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
  const bool move = !FIXED && e != NO_POWER && (e > w.E || e < w.E - V_ROOM);   // uniform
  if (__builtin_amdgcn_ballot_w64(top > w.m + RESCALE_SLACK) || move) {
    const float pm = xmax16_32(top), mn = pm > w.m + RESCALE_SLACK ? pm : w.m, alpha = __builtin_amdgcn_exp2f(w.m - mn);
    w.l *= alpha;
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) w.acc[mb] *= alpha;
    if (move) {
      const bool none = __builtin_amdgcn_ballot_w64(w.m != M_NONE) == 0;   // no sums yet
      const int to = moved_power(e, none ? NO_POWER : w.E, w.top);
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
        for (int q = 0; q < 4; ++q) w.acc[mb][q] = __builtin_ldexpf(w.acc[mb][q], w.E - to);
      w.E = to;
    }
    w.m = mn;
  }
  const float base = P_SHIFT - w.m;
#pragma unroll
  for (int r = 0; r < 4; ++r) s[r] = __builtin_amdgcn_exp2f(s[r] + base);
  w.l += (s[0] + s[1]) + (s[2] + s[3]);
  return s;
}

// A V scale: its exponent (NO_POWER for one that adds nothing to E), and what multiplies the weights of a page once E has
// followed it. One that is not finite makes every sum NaN (0 in a careful walk).
__device__ __forceinline__ int value_exponent(float v) {
  const float a = fabsf(v);
  return a > 0.f && a < __builtin_inff() ? (int)(f2u(a) >> 23) - 127 : NO_POWER;
}
__device__ __forceinline__ float value_factor(float v, int E, bool careful) {
  return careful && !(fabsf(v) < __builtin_inff()) ? 0.f : __builtin_ldexpf(v, -E);
}

__device__ __forceinline__ h4 half4(f4 p) {
  return h4{(_Float16)p[0], (_Float16)p[1], (_Float16)p[2], (_Float16)p[3]};
}

// acc += V^T . (weights times their factor), with what rounding left for float32 queries.
template <int D, bool QF32>
__device__ __forceinline__ void row_values(RowWave<D, QF32>& w, const h4 (&va)[D / 16], f4 p, float factor) {
  p *= factor;
  const h4 pb = half4(p);
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) w.acc[mb] = __builtin_amdgcn_mfma_f32_16x16x16f16(va[mb], pb, w.acc[mb], 0, 0, 0);
  if constexpr (QF32) {
    const h4 pl = half4(f4{p[0] - (float)pb[0], p[1] - (float)pb[1], p[2] - (float)pb[2], p[3] - (float)pb[3]});
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) w.acc[mb] = __builtin_amdgcn_mfma_f32_16x16x16f16(va[mb], pl, w.acc[mb], 0, 0, 0);
  }
}

__device__ __forceinline__ uint32_t clean_pair(uint32_t x) {
  const uint32_t e = x & 0x7C007C00u;
  return x & (((e & 0xFFFFu) == 0x7C00u ? 0u : 0xFFFFu) | (e >> 16 == 0x7C00u ? 0u : 0xFFFF0000u));
}

template <bool FIXED, int D, bool QF32>
__device__ __forceinline__ void row_page_fp16(RowWave<D, QF32>& w, const Raw16<D>& r, int first, bool careful, u4* kt, int c, int g) {
  u4 k[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) k[i] = r.k[i];
  k_through_lds<D / 8, D / 32>(k, kt, c, g);
  h8 ka[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) ka[i] = __builtin_bit_cast(h8, k[i]);
  const f4 p = row_weights<true, FIXED>(w, row_scores(w, ka, f4{0.f, 0.f, 0.f, 0.f}) * w.mult, first, 0);
  uint32_t v[4][D / 32];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) v[t][j] = careful ? clean_pair(r.v[t][j]) : r.v[t][j];
  h4 va[D / 16];
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) va[mb] = rows_to_a<D>(v, mb);
  row_values(w, va, p, FIXED ? 1.f : value_factor(1.f, w.E, false));
}

template <int TAG, int D, bool QF32>
__device__ __forceinline__ void row_page_byte(RowWave<D, QF32>& w, const Raw8<D>& r, int first, float ks, float vs, bool careful, u4* kt,
                                              int c, int g) {
  uint32_t kw[D / 16];
  k8_words<D>(r, kw, kt, c, g);
  auto four = [](uint32_t x, uint32_t& lo, uint32_t& hi) __attribute__((always_inline)) {
    if constexpr (TAG == IAK_TAG_FP8) fp8x4_to_f16(x, lo, hi);
    else i8x4_to_f16(x, lo, hi);
  };
  h8 ka[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t o[4];
    four(kw[2 * i], o[0], o[1]);
    four(kw[2 * i + 1], o[2], o[3]);
    ka[i] = make_h8(o[0], o[1], o[2], o[3]);
  }
  const f4 p = row_weights<true, false>(w, row_scores(w, ka, f4{0.f, 0.f, 0.f, 0.f}) * (w.mult * ks), first, value_exponent(vs));
  uint32_t v[4][D / 32];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      four(r.v[t][j], v[t][2 * j], v[t][2 * j + 1]);
      if (TAG == IAK_TAG_FP8 && careful) {                       // NaN codes
        v[t][2 * j] = clean_pair(v[t][2 * j]);
        v[t][2 * j + 1] = clean_pair(v[t][2 * j + 1]);
      }
    }
  h4 va[D / 16];
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) va[mb] = rows_to_a<D>(v, mb);
  row_values(w, va, p, value_factor(vs, w.E, careful));
}

// base * s0 + rest * s1, both codes exact (the rest's 16 times), products apart.
template <int D, bool QF32>
__device__ __forceinline__ void row_page_int4r(RowWave<D, QF32>& w, const Raw8<D>& r, int first, float ks0, float ks1, float vs0, float vs1,
                                               bool careful, u4* kt, int c, int g) {
  uint32_t kw[D / 16];
  k8_words<D>(r, kw, kt, c, g);
  const uint32_t mg = magic_i4();
  h8 kb[D / 32], kr[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t b[4], x16[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t x = kw[2 * i + h];
      const uint32_t y01 = __builtin_amdgcn_perm(x, x, 0x01010000u), y23 = __builtin_amdgcn_perm(x, x, 0x03030202u);
      b[2 * h] = bits(i4r_base_pair(y01, mg));
      b[2 * h + 1] = bits(i4r_base_pair(y23, mg));
      x16[2 * h] = bits(i4r_resid16_pair(y01, mg));
      x16[2 * h + 1] = bits(i4r_resid16_pair(y23, mg));
    }
    kb[i] = make_h8(b[0], b[1], b[2], b[3]);
    kr[i] = make_h8(x16[0], x16[1], x16[2], x16[3]);
  }
  const f4 none = {0.f, 0.f, 0.f, 0.f};
  const f4 sb = row_scores(w, kb, none), sr = row_scores(w, kr, none);
  const float k16 = ks1 * 0.0625f, v16 = vs1 * 0.0625f, most = fmaxf(fabsf(vs0), fabsf(vs1));
  f4 s;
#pragma unroll
  for (int q = 0; q < 4; ++q) s[q] = __builtin_fmaf(sb[q], ks0, sr[q] * k16) * w.mult;
  const bool fine = fabsf(vs0) + fabsf(vs1) < __builtin_inff();
  const f4 p = row_weights<true, false>(w, s, first, fine ? value_exponent(most) : NO_POWER);
  const float f0 = careful && !fine ? 0.f : __builtin_ldexpf(vs0, -w.E), f1 = careful && !fine ? 0.f : __builtin_ldexpf(v16, -w.E);
  h4 va[D / 16], vr[D / 16];
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) {
    const int j = mb >> 2, k = mb & 3;
    const uint32_t sel = (uint32_t)k * 0x00000101u + (uint32_t)(4 + k) * 0x01010000u;   // (t_even byte k, t_odd byte k)
    const uint32_t y01 = __builtin_amdgcn_perm(r.v[1][j], r.v[0][j], sel), y23 = __builtin_amdgcn_perm(r.v[3][j], r.v[2][j], sel);
    va[mb] = make_h4(bits(i4r_base_pair(y01, mg)), bits(i4r_base_pair(y23, mg)));
    vr[mb] = make_h4(bits(i4r_resid16_pair(y01, mg)), bits(i4r_resid16_pair(y23, mg)));
  }
  row_values(w, va, p, f0);
  row_values(w, vr, p, f1);
}

template <int D> struct RawScaled4 {   // INT4, with the scales of the lane's channels
  Raw4<D> x;
  float ks, vs;
};

template <int D, bool QF32>
__device__ __forceinline__ void row_page_int4(RowWave<D, QF32>& w, const RawScaled4<D>& rs, int first, bool careful, const h8 (&qhi)[D / 32],
                                              const h8 (&qlo)[QF32 ? D / 32 : 1], int c) {
  const Raw4<D>& r = rs.x;
  const uint32_t mg = magic_i4();
  // powers of two that bring the page's scales near 1; K's lanes differ by g, V's by c / 4
  const int ek = power_exponent(xmax16_32(finite_size(rs.ks)));
  float most = finite_size(rs.vs);
  most = fmaxf(most, __shfl_xor(most, 4, 64));
  most = fmaxf(most, __shfl_xor(most, 8, 64));
  const int ev = __builtin_amdgcn_readfirstlane(power_exponent(most));
  const bool some = __builtin_amdgcn_readfirstlane((int)(most > 0.f)) != 0;   // else zeros, infinities and NaN alone
  const ScaleParts ks = scale_parts(__builtin_ldexpf(rs.ks, -ek));
  const bool fine = fabsf(rs.vs) < __builtin_inff();
  const ScaleParts vs = scale_parts(careful && !fine ? 0.f : __builtin_ldexpf(rs.vs, -ev));
  auto parts = [](h2 n, const ScaleParts& k, uint32_t& hi, uint32_t& lo) __attribute__((always_inline)) {
    const h2 x = n * k.hi;
    hi = bits(x);
    lo = bits(__builtin_elementwise_fma(n, k.lo, __builtin_elementwise_fma(n, k.hi, -x))) & k.fine;
  };
  f4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) parts(nib_pair(r.k[i] >> (4 * q), mg), ks, h[q], l[q]);
    const h8 kh = make_h8(h[0], h[1], h[2], h[3]);
    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qhi[i], s, 0, 0, 0);
    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(make_h8(l[0], l[1], l[2], l[3]), qhi[i], s, 0, 0, 0);
    if constexpr (QF32) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qlo[i], s, 0, 0, 0);
  }
  const f4 p = row_weights<false, false>(w, s * __builtin_ldexpf(w.mult, ek), first, some ? ev : NO_POWER);
  h4 va[D / 16], vl[D / 16];
  const uint32_t y01l = pack_lo(r.v[0], r.v[1]), y01h = pack_hi(r.v[0], r.v[1]);
  const uint32_t y23l = pack_lo(r.v[2], r.v[3]), y23h = pack_hi(r.v[2], r.v[3]);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    const uint32_t y01 = d < 4 ? y01l : y01h, y23 = d < 4 ? y23l : y23h;
    uint32_t h[2], l[2];
    parts(nib_pair(y01 >> (4 * (d & 3)), mg), vs, h[0], l[0]);
    parts(nib_pair(y23 >> (4 * (d & 3)), mg), vs, h[1], l[1]);
    va[d] = make_h4(h[0], h[1]);
    vl[d] = make_h4(l[0], l[1]);
  }
  const float factor = some ? __builtin_ldexpf(1.f, ev - w.E) : 0.f;
  row_values(w, va, p, factor);
  const h4 pb = half4(p * factor);
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) w.acc[mb] = __builtin_amdgcn_mfma_f32_16x16x16f16(vl[mb], pb, w.acc[mb], 0, 0, 0);
}

// What a lane's rows see of infinite and NaN values (page_attention.h), by its channels here: bit (D/16) q + mb.
template <int D> __device__ __forceinline__ void row_remember(Seen16& x, const uint16_t* special, int tokens, int g) {
  for (int token = 0; token < tokens; ++token)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int first = (D / 16) * (4 * g + q);
      const uint32_t s = (uint32_t)special[v_chunk<D>(token, first / 8)] >> (first % 8), mask = (1u << (D / 16)) - 1u;
      x.plus |= (s & mask) << (D / 16 * q);
      x.minus |= ((s >> 8) & mask) << (D / 16 * q);
    }
}

// Waves a SIMD: what the registers hold of rings and queries in two parts. All precisions: two (16 x 4 queries
// over up to 16,384 tokens 108 us; three spill 62 registers, 160). Others: three or two of float16 pages 120.9 and
// 121.0 us (675 MB), of float16 and bytes 101.7 and 102.0.
template <bool QF32, int KIND> constexpr int row_waves_per_simd() { return QF32 || KIND == PAGES_ALL ? 2 : 3; }

template <int D, bool QF32, int KIND>
__global__ __launch_bounds__(64 * ROW_WAVES, (row_waves_per_simd<QF32, KIND>())) void page_rows_kernel(const PageAttn a) {
  constexpr int UNIT = 16 * D / 4;                               // 16-byte units of a wave's sums, and at least a page's K
  __shared__ u4 lds[ROW_WAVES][UNIT];
  __shared__ uint16_t special[ROW_WAVES][PS * D / 8];
  __shared__ float part_m[ROW_WAVES][16], part_l[ROW_WAVES][16];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
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

  RowWave<D, QF32> w;
  {
    const int r = tile * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
    const bool active = r < a.L * a.G, live = active && i < n.queries;
    w.seen = live ? mx_seen(a, n, i) : 0;
    w.least = live ? w.seen : 0x7FFFFFFF;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(w.least, o, 64); w.least = x < w.least ? x : w.least; }
    w.mult = load_query<D, QF32>(a, active, b * a.qsb + i * a.qst + head * a.qsh, g, w.qhi, w.qlo);
  }
  w.g = g;

  // the wave's entries: a quarter of the part's
  const int each = (e1 - e0 + ROW_WAVES - 1) / ROW_WAVES, w0 = e0 + wv * each, w1 = w0 + each < e1 ? w0 + each : e1;
  const int32_t* row = a.table + kvrow * a.W;
  u4* kt = lds[wv];
  bool careful = false;
  Seen16 odd = {0u, 0u};
  // A token that a row does not see weighs nothing, and 0 times infinity is NaN: a walk that ends in such sums is made
  // again with zeros in their place.
  for (int walk = 0; walk < 2; ++walk) {
    w.m = M_NONE;
    w.l = 0.f;
    w.E = 0;
    w.top = -NO_POWER;
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) w.acc[mb] = f4{0.f, 0.f, 0.f, 0.f};
    for (int block = w0; block < w1; block += 64) {
      // lane i has entry i of the block; those of one precision are gone through together
      const int page = entry_page(a, raw_entry(row, block + lane, w1));
      const PageTag x = page_tag<KIND>(a, page, raw_tag(a, page));
      auto mask = [&](int tag) { return __builtin_amdgcn_ballot_w64(x.id >= 0 && x.tag == tag); };
      auto first = [&](int idx) { return (block + idx) * PS; };
      float s[4] = {0.f, 0.f, 0.f, 0.f};                         // K's and V's scales; residual: base, rest of both
      if constexpr (KIND != PAGES_F16) {
        if (x.id >= 0 && (x.tag == IAK_TAG_INT8 || x.tag == IAK_TAG_FP8)) page_scales<D, KIND>(a, x, s[0], s[1]);
        if (KIND == PAGES_ALL && x.id >= 0 && x.tag == IAK_TAG_INT4_RESIDUAL) {
          s[0] = a.k_int4r_scale[2 * (int64_t)x.id];
          s[1] = a.k_int4r_scale[2 * (int64_t)x.id + 1];
          s[2] = a.v_int4r_scale[2 * (int64_t)x.id];
          s[3] = a.v_int4r_scale[2 * (int64_t)x.id + 1];
        }
      }
      auto scale = [&](int i, int idx) { return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(s[i]), idx)); };
      class_loop<IAK_RING_FP16, Raw16<D>>(
          mask(IAK_TAG_FP16), x.id,
          [&](Raw16<D>& r, int p) {
            load16<D>(r, page_at<_Float16>(a.k_fp16, p, PS * D * 2), page_at<_Float16>(a.v_fp16, p, PS * D * 2), c, g);
          },
          [&](const Raw16<D>& r, int idx) { row_page_fp16<KIND == PAGES_F16>(w, r, first(idx), careful, kt, c, g); });
      if constexpr (KIND != PAGES_F16) {
        class_loop<IAK_RING_BYTE, Raw8<D>>(
            mask(IAK_TAG_FP8), x.id,
            [&](Raw8<D>& r, int p) { load8<D>(r, page_at<uint8_t>(a.k_fp8, p, PS * D), page_at<uint8_t>(a.v_fp8, p, PS * D), c, g); },
            [&](const Raw8<D>& r, int idx) {
              row_page_byte<IAK_TAG_FP8>(w, r, first(idx), scale(0, idx), scale(1, idx), careful, kt, c, g);
            });
        class_loop<IAK_RING_BYTE, Raw8<D>>(
            mask(IAK_TAG_INT8), x.id,
            [&](Raw8<D>& r, int p) { load8<D>(r, page_at<uint8_t>(a.k_int8, p, PS * D), page_at<uint8_t>(a.v_int8, p, PS * D), c, g); },
            [&](const Raw8<D>& r, int idx) {
              row_page_byte<IAK_TAG_INT8>(w, r, first(idx), scale(0, idx), scale(1, idx), careful, kt, c, g);
            });
      }
      if constexpr (KIND == PAGES_ALL) {
        class_loop<IAK_RING_BYTE, Raw8<D>>(
            mask(IAK_TAG_INT4_RESIDUAL), x.id,
            [&](Raw8<D>& r, int p) { load8<D>(r, page_at<uint8_t>(a.k_int4r, p, PS * D), page_at<uint8_t>(a.v_int4r, p, PS * D), c, g); },
            [&](const Raw8<D>& r, int idx) {
              row_page_int4r(w, r, first(idx), scale(0, idx), scale(1, idx), scale(2, idx), scale(3, idx), careful, kt, c, g);
            });
        const uint64_t packed = mask(IAK_TAG_INT4);
        if (packed) {
          h8 qhi[D / 32], qlo[QF32 ? D / 32 : 1];                // in the order of the codes' pairs
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            qhi[i] = q_int4_order(w.qhi[i]);
            if constexpr (QF32) qlo[i] = q_int4_order(w.qlo[i]);
          }
          const int groups = D / a.int4_group;
          class_loop<IAK_RING_INT4, RawScaled4<D>>(
              packed, x.id,
              [&](RawScaled4<D>& r, int p) {
                load4<D>(r.x, page_at<uint8_t>(a.k_int4, p, PS * D / 2), page_at<uint8_t>(a.v_int4, p, PS * D / 2), c, g);
                const int64_t at = (int64_t)(p < 0 ? 0 : p) * groups;
                r.ks = load_scale(a.k_int4_scale, at + g * groups / 4, a.int4_sd);
                r.vs = load_scale(a.v_int4_scale, at + (c >> 2) * groups / 4, a.int4_sd);
              },
              [&](const RawScaled4<D>& r, int idx) { row_page_int4(w, r, first(idx), careful, qhi, qlo, c); });
        }
      }
    }
    if (careful) break;
    float sum = 0.f;                                             // NaN once anything is not finite
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q) sum = __builtin_fmaf(w.acc[mb][q], 0.f, sum);
    if (!__builtin_amdgcn_ballot_w64(!(sum == 0.f))) break;      // uniform in the wave
    careful = true;
  }
  if (careful) {                                                 // what V has of them, in a walk of its own
    for (int e = w0; e < w1; ++e) {
      const PageEntry x = page_entry<D, KIND>(a, row, e, w1);
      const int id = __builtin_amdgcn_readfirstlane(x.id), tag = __builtin_amdgcn_readfirstlane(x.tag);
      PageRaw<D> r;
      load_page<D, KIND>(r, a, true, id, tag, lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const bool bad = store_page<D, KIND>(r, id, tag, u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)f2u(x.vf))), kt,
                                                 kt + PS * D / 8, lane);
      if (!__builtin_amdgcn_ballot_w64(bad)) continue;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      put_aside<D>(kt, special[wv], lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int left = w.seen - e * PS;
      row_remember<D>(odd, special[wv], left < PS ? left : PS, g);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if ((odd.plus >> (D / 16 * q + mb)) & 1u) w.acc[mb][q] += __builtin_inff();
        if ((odd.minus >> (D / 16 * q + mb)) & 1u) w.acc[mb][q] -= __builtin_inff();
      }
  }

  // the waves' sums meet in LDS (rows c, 16-byte units turned by c against bank conflicts)
  const float sum = xsum16_32(w.l);
  const int by = KIND == PAGES_F16 ? 0 : sum_power(sum, w.E);
  __syncthreads();
  if (g == 0) { part_m[wv][c] = w.m + (float)by; part_l[wv][c] = __builtin_ldexpf(sum, -by); }
  f4* sums = reinterpret_cast<f4*>(lds[wv]);
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      f4 x;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = __builtin_ldexpf(w.acc[4 * u + k][q], w.E - by);
      sums[c * (D / 4) + (((D / 64) * (4 * g + q) + u) ^ c)] = x;
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
      float wgt = __builtin_amdgcn_exp2f(part_m[x][cr] - M);
      L += wgt * part_l[x][cr];
      f4 own = reinterpret_cast<const f4*>(lds[x])[cr * (D / 4) + (u ^ cr)];
      part_weight(own, wgt);
      o += own * wgt;
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
