// What the attention kernels for several query rows over pages of mixed precision share: a table
// entry's page, precision and scales; a page's way from memory into LDS as float16 operands; the
// softmax with scales.
//
// Every page becomes float16 tiles of codes that are exact, its scale left to 32 bits:
//   float16          as it is
//   INT8, FP8        the codes. K's scale multiplies the scores; V's, the weights
//                    (2^log2 of it inside their exponential, taken out of their sum again)
//   INT4, residual   codes times scales need up to 30 bits: two tiles, of what float16 holds of
//                    them and what is left, both relative to a power of two of the page
// so that a quantised page costs what its own products cost, and nothing is rounded but the
// weights. (One tile for those, as the decode's kernel has it: products off by 2^-12 a value, 6e-4 of
// an output where the weights' rounding costs 1.5e-4.)
#ifndef IAK_PAGE_ATTENTION_H
#define IAK_PAGE_ATTENTION_H

#include "iak_device.h"
#include "mx_attention.h"
#include "step_internal.h"

namespace iak {

__device__ __forceinline__ int row_length(const PageAttn& a, int64_t kvrow) {
  const int64_t c = a.counts[kvrow];
  const int listed = c < 0 ? 0 : (c > a.W ? a.W * 16 : (int)c * 16);
  if (!a.bounds) return listed;
  const int v = a.bounds[kvrow];
  return v < listed ? v : listed;
}

// The kernel's arguments, read anew: what is used seldom would otherwise be kept in scalar registers from the
// start, and be spilled for the walk.
__device__ __forceinline__ const PageAttn& arguments() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PageAttn*)p;
}

// --------------------------------------------------------------------------- //
// Entries
// --------------------------------------------------------------------------- //

// A table entry as a lane looks it up: its page (-1: no tokens), native tag, what multiplies the scores
// (km > 0) and K's codes (kf), log2 of what multiplies the weights (vl), and V's codes (vf).
struct PageEntry { int id, tag; float km, kf, vl, vf; };

__device__ __forceinline__ bool wide_tag(int tag) { return tag == IAK_TAG_INT4 || tag == IAK_TAG_INT4_RESIDUAL; }

// A page scale in a positive normal multiplier whose inverse is normal, and what is left for the codes: its sign (from
// 2^126 on four times that), or itself where it is zero or not finite.
__device__ __forceinline__ void split_scale(float s, float& mult, float& rest) {
  const float a = fabsf(s);
  const bool most = a >= 8.50705917e37f;
  const bool plain = a >= 1.17549435e-38f && a < __builtin_inff();
  mult = plain ? (most ? 0.25f : 1.f) * a : 1.f;
  rest = plain ? __builtin_copysignf(most ? 4.f : 1.f, s) : s;
}
// The exponent of a positive finite scale whose codes go as values, which go relative to that power of two; 0 for others.
// (2^126 is the largest whose inverse is normal.)
__device__ __forceinline__ int power_exponent(float s) {
  const int e = (int)(f2u(s) >> 23) - 127;
  return !(s > 0.f && s < __builtin_inff()) ? 0 : e < -126 ? -126 : e > 126 ? 126 : e;
}
__device__ __forceinline__ float power_of(float s) { return pow2f(power_exponent(s)); }
// |s|, 0 for what is not finite.
__device__ __forceinline__ float finite_size(float s) { return fabsf(s) < __builtin_inff() ? fabsf(s) : 0.f; }

// The look-up in three steps, each of which waits for the one before: the entry, its page's tag, the
// scales. (A step's loads can be under way while others work.)
__device__ __forceinline__ int raw_entry(const int32_t* row, int e, int end) { return e < end ? row[e] : (int)0x80000000; }

struct PageTag { int id, tag; };
__device__ __forceinline__ int entry_page(const PageAttn& a, int raw) {   // -1: none
  int64_t p = raw;
  if (a.neg_wrap && p < 0) p += a.NP;
  return p < 0 || p >= a.NP ? -1 : (int)p;
}
__device__ __forceinline__ int raw_tag(const PageAttn& a, int page) { return page < 0 ? -1 : a.tags[page]; }
template <int KIND> __device__ __forceinline__ PageTag page_tag(const PageAttn& a, int page, int raw) {
  const int tag = page < 0 ? (int)IAK_TAG_SKIP : (uint32_t)raw < 8u ? (int)((a.tagmap >> (8 * raw)) & 0xFFu) : a.other_tag;
  const bool known = tag == IAK_TAG_FP16 || (KIND != PAGES_F16 && (tag == IAK_TAG_INT8 || tag == IAK_TAG_FP8)) ||
                     (KIND == PAGES_ALL && (tag == IAK_TAG_INT4 || tag == IAK_TAG_INT4_RESIDUAL));
  return PageTag{known ? page : -1, known ? tag : (int)IAK_TAG_SKIP};
}

// A page's scales: INT8 and FP8 the ones, 4 bits the largest finite one.
template <int D, int KIND> __device__ __forceinline__ void page_scales(const PageAttn& a, const PageTag& x, float& k, float& v) {
  k = v = 1.f;
  if (KIND == PAGES_F16 || x.id < 0) return;
  const int64_t p = x.id;
  if (x.tag == IAK_TAG_INT8 || x.tag == IAK_TAG_FP8) {
    const bool fp8 = x.tag == IAK_TAG_FP8;
    k = load_scale(fp8 ? a.k_fp8_scale : a.k_int8_scale, p, fp8 ? a.fp8_sd : a.int8_sd);
    v = load_scale(fp8 ? a.v_fp8_scale : a.v_int8_scale, p, fp8 ? a.fp8_sd : a.int8_sd);
  } else if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4) {
    const int groups = D / a.int4_group;                         // 1, 2 or 4
    k = v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t at = p * groups + (i < groups ? i : 0);
      k = fmaxf(k, finite_size(load_scale(a.k_int4_scale, at, a.int4_sd)));
      v = fmaxf(v, finite_size(load_scale(a.v_int4_scale, at, a.int4_sd)));
    }
  } else if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4_RESIDUAL) {
    k = fmaxf(finite_size(a.k_int4r_scale[2 * p]), finite_size(a.k_int4r_scale[2 * p + 1]));
    v = fmaxf(finite_size(a.v_int4r_scale[2 * p]), finite_size(a.v_int4r_scale[2 * p + 1]));
  }
}

template <int KIND> __device__ __forceinline__ PageEntry page_multipliers(const PageTag& x, float k, float v) {
  if constexpr (KIND == PAGES_F16) return PageEntry{x.id, x.tag, 1.f, 1.f, 0.f, 1.f};
  const bool wide = wide_tag(x.tag);
  float km, kf, vm, vf;                                          // float16 pages have scales of 1
  split_scale(k, km, kf);
  split_scale(v, vm, vf);
  const float kp = power_of(k), vp = power_of(v);
  km = wide ? kp : km;
  vm = wide ? vp : vm;
  kf = wide ? 1.f / kp : kf;                                     // exact
  vf = wide ? 1.f / vp : vf;
  return PageEntry{x.id, x.tag, km, kf, __builtin_amdgcn_logf(vm), vf};
}

template <int D, int KIND>
__device__ __forceinline__ PageEntry page_entry(const PageAttn& a, const int32_t* row, int e, int end) {
  const int page = entry_page(a, raw_entry(row, e, end));
  const PageTag x = page_tag<KIND>(a, page, raw_tag(a, page));
  float k, v;
  page_scales<D, KIND>(a, x, k, v);
  return page_multipliers<KIND>(x, k, v);
}

// --------------------------------------------------------------------------- //
// A page's K or V by a wave: loaded, and put into LDS
// --------------------------------------------------------------------------- //

// Piece j of lane l is the page's bytes 1024 j + 16 l ..: whole lines. (INT4 pages of 64 channels, 512
// bytes: 8 l ..)
template <int D> struct PageRaw {
  u4 x[D / 32];
  float s0, s1;                        // INT4: its channels' scale; residual: both
};

// (Every branch sets every field: a field that some leave alone is kept in memory by the compiler.)
template <int D, int KIND>
__device__ __forceinline__ void load_page(PageRaw<D>& r, const PageAttn& a, bool v, int id, int tag, int lane) {
  const int64_t p = id < 0 ? 0 : id;                             // uniform, as the tag
  const u4 zero = {0u, 0u, 0u, 0u};
  if (id < 0) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) r.x[j] = zero;
    r.s0 = r.s1 = 0.f;
  } else if (KIND == PAGES_F16 || tag == IAK_TAG_FP16) {
    const u4* at = reinterpret_cast<const u4*>(v ? a.v_fp16 : a.k_fp16) + p * (PS * D / 8) + lane;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) r.x[j] = at[64 * j];
    r.s0 = r.s1 = 0.f;
  } else if (KIND == PAGES_ALL && tag == IAK_TAG_INT4) {
    const uint8_t* page = reinterpret_cast<const uint8_t*>(v ? a.v_int4 : a.k_int4) + p * (PS * D / 2);
#pragma unroll
    for (int j = 1; j < D / 32; ++j) r.x[j] = zero;
    if constexpr (D == 128) r.x[0] = *(reinterpret_cast<const u4*>(page) + lane);
    else {
      const u2 x = *(reinterpret_cast<const u2*>(page) + lane);
      r.x[0] = u4{x[0], x[1], 0u, 0u};
    }
    const int channel = lane % 4 * (D / 4), groups = D / a.int4_group;
    r.s0 = load_scale(v ? a.v_int4_scale : a.k_int4_scale, p * groups + channel / a.int4_group, a.int4_sd);
    r.s1 = 0.f;
  } else {
    const void* pool = tag == IAK_TAG_INT8 ? (v ? a.v_int8 : a.k_int8) : tag == IAK_TAG_FP8 ? (v ? a.v_fp8 : a.k_fp8)
                                                                                           : (v ? a.v_int4r : a.k_int4r);
    const u4* at = reinterpret_cast<const u4*>(pool) + p * (PS * D / 16) + lane;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) r.x[j] = j < D / 64 ? at[64 * j] : zero;
    r.s0 = r.s1 = 0.f;
    if (KIND == PAGES_ALL && tag == IAK_TAG_INT4_RESIDUAL) {
      const float* s = (v ? a.v_int4r_scale : a.k_int4r_scale) + 2 * p;
      r.s0 = s[0];
      r.s1 = s[1];
    }
  }
}

// Two values as float16 and what is left of them. The first is cut rather than rounded: the second has it.
// `fine` 0: they are not finite, and have no second part; else all bits.
__device__ __forceinline__ void hi_lo(float a, float b, uint32_t fine, uint32_t& hi, uint32_t& lo) {
  const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(a, b));
  hi = bits(h);
  lo = bits(h2{(_Float16)(a - (float)h[0]), (_Float16)(b - (float)h[1])}) & fine;
}

// A scale in two float16 parts; a code times the first is off by what a fused product gives exactly.
struct ScaleParts { h2 hi, lo; uint32_t fine; };                 // fine 0: infinite or NaN, which has no second part
__device__ __forceinline__ ScaleParts scale_parts(float s) {
  const _Float16 h = (_Float16)s;
  return ScaleParts{splat2(h), splat2((_Float16)(s - (float)h)), fabsf(s) < __builtin_inff() ? 0xFFFFFFFFu : 0u};
}

// The pair of codes (n & 15, n >> 4 & 15), less 8 each, of byte `byte` of w, as float16: exact.
__device__ __forceinline__ h2 nibbles(uint32_t w, int byte) {
  const uint32_t y = __builtin_amdgcn_perm(0u, w, 0x0C000C00u | (uint32_t)byte | ((uint32_t)byte << 16));   // (b, 0, b, 0)
  const h2 n = as_h2((y & 0x00F0000Fu) | MAGIC_I4);              // 1024 + low, 1024 + 16 high
  return __builtin_elementwise_fma(n, h2{(_Float16)1.f, (_Float16)0.0625f}, h2{(_Float16)-1032.f, (_Float16)-72.f});
}

// The page into LDS as float16 rows (16-byte chunks at v_chunk); `lo`, written for wide pages alone: what is
// left. id < 0: zeros. `rest`: kf or vf of the entry. Returns whether a value is infinite or NaN in this lane.
template <int D, int KIND>
__device__ __forceinline__ bool store_page(const PageRaw<D>& r, int id, int tag, float rest, u4* hi, u4* lo, int lane) {
  h2 sum = {0, 0};                     // NaN once anything is not finite
  auto look = [&](const u4& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum = __builtin_elementwise_fma(as_h2(x[i]), h2{0, 0}, sum);
  };
  if (id < 0) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) hi[64 * j + lane] = u4{0u, 0u, 0u, 0u};
    return false;
  }
  if (KIND == PAGES_F16 || tag == IAK_TAG_FP16) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const int f = 64 * j + lane;
      hi[v_chunk<D>(f / (D / 8), f % (D / 8))] = r.x[j];
      look(r.x[j]);
    }
  } else if (KIND == PAGES_ALL && tag == IAK_TAG_INT4) {
    const ScaleParts k = scale_parts(r.s0 * rest);
    const int token = lane / 4, chunk = lane % 4 * (D / 32);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      u4 h, l;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const h2 n = nibbles(r.x[0][c], i), x = n * k.hi;
        h[i] = bits(x);
        l[i] = bits(__builtin_elementwise_fma(n, k.lo, __builtin_elementwise_fma(n, k.hi, -x))) & k.fine;
      }
      const int at = v_chunk<D>(token, chunk + c);
      hi[at] = h;
      lo[at] = l;
      look(h);
    }
  } else if (KIND == PAGES_ALL && tag == IAK_TAG_INT4_RESIDUAL) {
    const float s0 = r.s0 * rest, s1 = r.s1 * rest;
    const uint32_t fine = fabsf(s0) + fabsf(s1) < __builtin_inff() ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int j = 0; j < D / 64; ++j) {
      const int f = 64 * j + lane, token = f / (D / 16), chunk = f % (D / 16) * 2;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u4 h, l;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = r.x[j][2 * c + (i >> 1)];
          const h2 m = nibbles(w, 2 * (i & 1)), n = nibbles(w, 2 * (i & 1) + 1);   // (base, residual) of two channels
          uint32_t x, y;
          hi_lo(__builtin_fmaf((float)m[0], s0, (float)m[1] * s1), __builtin_fmaf((float)n[0], s0, (float)n[1] * s1), fine, x, y);
          h[i] = x;
          l[i] = y;
        }
        const int at = v_chunk<D>(token, chunk + c);
        hi[at] = h;
        lo[at] = l;
        look(h);
      }
    }
  } else {
    const h2 sign = splat2((_Float16)rest);
    auto bytes = [&](auto&& four) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const int f = 64 * j + lane, token = f / (D / 16), chunk = f % (D / 16) * 2;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t o[4];
          four(r.x[j][2 * c], o[0], o[1]);
          four(r.x[j][2 * c + 1], o[2], o[3]);
          const u4 h = u4{bits(as_h2(o[0]) * sign), bits(as_h2(o[1]) * sign), bits(as_h2(o[2]) * sign), bits(as_h2(o[3]) * sign)};
          hi[v_chunk<D>(token, chunk + c)] = h;
          look(h);
        }
      }
    };
    if (tag == IAK_TAG_FP8) bytes([](uint32_t x, uint32_t& l, uint32_t& h) __attribute__((always_inline)) { fp8x4_to_f16(x, l, h); });
    else bytes([](uint32_t x, uint32_t& l, uint32_t& h) __attribute__((always_inline)) { i8x4_to_f16(x, l, h); });
  }
  return !((float)sum[0] + (float)sum[1] == 0.f);
}

// --------------------------------------------------------------------------- //
// The same by pieces, for waves that share pages: a lane has one 16-byte chunk of a page's float16 rows, whatever
// the precision, so that all waves have the same to do. Where the pages lie, their tags and multipliers are
// looked up ahead into LDS, from where they come as vectors: a step's worth of them, and of the pools they lie in,
// is more than the scalar registers hold.
// --------------------------------------------------------------------------- //

constexpr uint32_t NO_PAGE = 0xFFu;
constexpr float NO_SCALE = -200.f;      // below every float's log2
constexpr int AHEAD = 128;             // entries at hand: entry e at e % AHEAD

template <int KIND> struct Ahead {
  u4 where[AHEAD];                     // addresses of K and of V
  uint8_t tag[AHEAD];                  // native, or NO_PAGE
  float km[KIND == PAGES_F16 ? 1 : AHEAD], vl[KIND == PAGES_F16 ? 1 : AHEAD];   // as in PageEntry; no page: vl NO_SCALE
  float iv[KIND == PAGES_F16 ? 1 : AHEAD];                                      // 2^-vl, 0
  f4 factors[2][KIND == PAGES_F16 ? 1 : AHEAD];   // of K's and V's codes, by quarters of the channels; residual: of the bases
  float second[2][KIND == PAGES_ALL ? AHEAD : 1];                               // residual: of the residuals
};

template <int D, int KIND>
__device__ __forceinline__ void put_ahead(Ahead<KIND>& t, const PageAttn& a, int e, const PageTag& x) {
  const int at = e & (AHEAD - 1);
  const int64_t p = x.id < 0 ? 0 : x.id;
  const void* k = a.k_fp16;
  const void* v = a.v_fp16;
  int bytes = PS * D * 2;
  if (KIND != PAGES_F16 && x.tag == IAK_TAG_INT8) { k = a.k_int8; v = a.v_int8; bytes = PS * D; }
  if (KIND != PAGES_F16 && x.tag == IAK_TAG_FP8) { k = a.k_fp8; v = a.v_fp8; bytes = PS * D; }
  if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4) { k = a.k_int4; v = a.v_int4; bytes = PS * D / 2; }
  if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4_RESIDUAL) { k = a.k_int4r; v = a.v_int4r; bytes = PS * D; }
  const uint64_t ka = reinterpret_cast<uint64_t>(k) + p * bytes, va = reinterpret_cast<uint64_t>(v) + p * bytes;
  t.where[at] = u4{(uint32_t)ka, (uint32_t)(ka >> 32), (uint32_t)va, (uint32_t)(va >> 32)};
  t.tag[at] = (uint8_t)(x.id < 0 ? NO_PAGE : (uint32_t)x.tag);
  if constexpr (KIND != PAGES_F16) {
    float ks, vs;
    page_scales<D, KIND>(a, x, ks, vs);
    const PageEntry y = page_multipliers<KIND>(x, ks, vs);
    f4 kf = {y.kf, y.kf, y.kf, y.kf}, vf = {y.vf, y.vf, y.vf, y.vf};
    if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4) {
      const int groups = D / a.int4_group;                       // 1, 2 or 4
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        kf[q] *= load_scale(a.k_int4_scale, p * groups + q * groups / 4, a.int4_sd);
        vf[q] *= load_scale(a.v_int4_scale, p * groups + q * groups / 4, a.int4_sd);
      }
    }
    if (KIND == PAGES_ALL && x.tag == IAK_TAG_INT4_RESIDUAL) {
      t.second[0][at] = kf[0] * a.k_int4r_scale[2 * p + 1];
      t.second[1][at] = vf[0] * a.v_int4r_scale[2 * p + 1];
      kf *= a.k_int4r_scale[2 * p];
      vf *= a.v_int4r_scale[2 * p];
    }
    t.km[at] = y.km;
    t.vl[at] = x.id < 0 ? NO_SCALE : y.vl;
    t.iv[at] = x.id < 0 ? 0.f : __builtin_amdgcn_exp2f(-y.vl);
    t.factors[0][at] = kf;
    t.factors[1][at] = vf;
  }
}

// Chunk f (of 2 D) of a page at `page`.
template <int D, int KIND>
__device__ __forceinline__ u4 load_piece(uint64_t page, uint32_t tag, uint32_t f) {
  typedef __attribute__((address_space(1))) const uint8_t byte;
  typedef __attribute__((address_space(1))) const uint32_t word;
  typedef __attribute__((address_space(1))) const u2 pair;
  typedef __attribute__((address_space(1))) const u4 four;
  byte* p = reinterpret_cast<byte*>(page);
  if (tag == NO_PAGE) return u4{0u, 0u, 0u, 0u};                 // uniform
  if (KIND == PAGES_F16 || tag == IAK_TAG_FP16) return *reinterpret_cast<four*>(p + 16 * f);
  if (KIND == PAGES_ALL && tag == IAK_TAG_INT4) return u4{*reinterpret_cast<word*>(p + 4 * f), 0u, 0u, 0u};
  const u2 x = *reinterpret_cast<pair*>(p + 8 * f);
  return u4{x[0], x[1], 0u, 0u};
}

// Into place `at` of the tile `hi`, and what is left of wide pages into `lo`; s0, s1: the lane's factors.
template <int D, int KIND>
__device__ __forceinline__ void store_piece(const u4& x, uint32_t tag, float s0, float s1, u4* hi, u4* lo, int at) {
  if (KIND == PAGES_F16 || tag == NO_PAGE || tag == IAK_TAG_FP16) {
    hi[at] = x;
    return;
  }
  u4 h, l;
  if (KIND == PAGES_ALL && tag == IAK_TAG_INT4) {
    const ScaleParts k = scale_parts(s0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const h2 n = nibbles(x[0], i), y = n * k.hi;
      h[i] = bits(y);
      l[i] = bits(__builtin_elementwise_fma(n, k.lo, __builtin_elementwise_fma(n, k.hi, -y))) & k.fine;
    }
    lo[at] = l;
  } else if (KIND == PAGES_ALL && tag == IAK_TAG_INT4_RESIDUAL) {
    const uint32_t fine = fabsf(s0) + fabsf(s1) < __builtin_inff() ? 0xFFFFFFFFu : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = x[i >> 1];
      const h2 m = nibbles(w, 2 * (i & 1)), n = nibbles(w, 2 * (i & 1) + 1);
      uint32_t y, z;
      hi_lo(__builtin_fmaf((float)m[0], s0, (float)m[1] * s1), __builtin_fmaf((float)n[0], s0, (float)n[1] * s1), fine, y, z);
      h[i] = y;
      l[i] = z;
    }
    lo[at] = l;
  } else {
    const h2 sign = splat2((_Float16)s0);
    uint32_t o[4];
    if (tag == IAK_TAG_FP8) {
      fp8x4_to_f16(x[0], o[0], o[1]);
      fp8x4_to_f16(x[1], o[2], o[3]);
    } else {
      i8x4_to_f16(x[0], o[0], o[1]);
      i8x4_to_f16(x[1], o[2], o[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = bits(as_h2(o[i]) * sign);
  }
  hi[at] = h;
}

// --------------------------------------------------------------------------- //
// The softmax of PAGES pages whose scores and weights have multipliers (hide() is mx_attention.h's)
// --------------------------------------------------------------------------- //

template <int D, int PAGES, int T, typename L>
__device__ __forceinline__ void raise_scaled(const f4 (&s)[T][PAGES], const float (&km)[PAGES], const float (&mult)[T], float (&m)[T],
                                             L (&l)[T], f4 (&acc)[T][D / 16]) {
  float top[T];
  bool over = false;
#pragma unroll
  for (int t = 0; t < T; ++t) {
    top[t] = -__builtin_inff();
#pragma unroll
    for (int p = 0; p < PAGES; ++p)
      top[t] = fmaxf(top[t], fmaxf(fmaxf(s[t][p][0], s[t][p][1]), fmaxf(s[t][p][2], s[t][p][3])) * fmaxf(mult[t] * km[p], 1e-37f));
    over = over || top[t] > m[t] + RESCALE_SLACK;
  }
  if (__builtin_amdgcn_ballot_w64(over)) {
    asm volatile("");
#pragma unroll
    for (int t = 0; t < T; ++t) {
      const float pm = xmax16_32(top[t]);
      const float mn = pm > m[t] + RESCALE_SLACK ? pm : m[t];
      const float alpha = __builtin_amdgcn_exp2f(m[t] - mn);
      l[t] *= alpha;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) acc[t][mb] *= alpha;
      m[t] = mn;
    }
  }
}

// Scores become weights times V's scale 2^vl; returns their sum without it.
template <int PAGES>
__device__ __forceinline__ float soften_scaled(f4 (&s)[PAGES], const float (&km)[PAGES], const float (&vl)[PAGES], const float (&out)[PAGES],
                                               float mult, float m) {
  float sum = 0.f;
#pragma unroll
  for (int p = 0; p < PAGES; ++p) {
    const float each = fmaxf(mult * km[p], 1e-37f), base = P_SHIFT - m + vl[p];
#pragma unroll
    for (int q = 0; q < 4; ++q) s[p][q] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[p][q], each, base));
    sum = __builtin_fmaf((s[p][0] + s[p][1]) + (s[p][2] + s[p][3]), out[p], sum);
  }
  return sum;
}

// V's scales differ by pages: weights carry 2^(vl - E), the accumulators stand for 2^E of themselves, and E follows
// the largest of a step's, with room below it so that it moves seldom. It starts at NO_POWER, where there are no sums,
// and falls no more than V_FALL below the highest it has been: the accumulators of 2^31 tokens are below 2^62, and a fall
// multiplies them.
constexpr int V_ROOM = 8, V_FALL = 60, NO_POWER = 1000;
template <int PAGES> __device__ __forceinline__ int value_power(const float (&vl)[PAGES], int E) {
  float most = vl[0];
#pragma unroll
  for (int p = 1; p < PAGES; ++p) most = fmaxf(most, vl[p]);
  const int e = __builtin_amdgcn_readfirstlane((int)floorf(most));
  return e <= (int)NO_SCALE || (e <= E && e >= E - V_ROOM) ? E : e;
}
// Where E may move to, and `top`, its highest so far (at first -NO_POWER).
__device__ __forceinline__ int moved_power(int to, int E, int& top) {
  if (E == NO_POWER) return to;
  top = top < E ? E : top;
  return to < top - V_FALL ? top - V_FALL : to;
}

// A row's sums as they meet others': acc 2^E may be past float32's range where its quotient by the weights' sum l is
// not. Past 2^SUM_POWER the row's maximum is therefore counted higher by this power of two, and l (to some 2^-10, so that 2^10
// parts add up) and acc lower.
constexpr int SUM_POWER = 60;
__device__ __forceinline__ int sum_power(float l, int E) {
  return E > SUM_POWER && l > 0.f && l < __builtin_inff() ? (int)(f2u(l) >> 23) - 127 + 11 : 0;
}

// Infinite and NaN values of V: a weight of zero would make them NaN where a row does not see them, so
// the tiles have zeros in their place. A page that has any leaves beside its tile, for every 16-byte chunk, which
// of its 8 values are positive (bits 0 .. 7) and which negative (8 .. 15; NaN: both), and whoever sees one
// remembers it by channel until the end: a weight is positive, whatever its size. All of this is rare.
// Returns whether there was any.
__device__ __forceinline__ bool clean_chunk(u4* chunk) {
  u4 w = *chunk;
  const u4 was = w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = w[i] & 0x7C007C00u;
    w[i] &= ((e & 0xFFFFu) == 0x7C00u ? 0u : 0xFFFFu) | (e >> 16 == 0x7C00u ? 0u : 0xFFFF0000u);
  }
  *chunk = w;
  return ((w[0] ^ was[0]) | (w[1] ^ was[1]) | (w[2] ^ was[2]) | (w[3] ^ was[3])) != 0u;
}
template <int D> __device__ __forceinline__ void put_aside(u4* tile, uint16_t* special, int lane) {
  for (int f = lane; f < PS * D / 8; f += 64) {
    u4 w = tile[f];
    uint32_t bits16 = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
      if ((h & 0x7C00u) == 0x7C00u) {
        const bool nan = (h & 0x3FFu) != 0u;
        bits16 |= (nan || h < 0x8000u ? 1u << i : 0u) | (nan || h >= 0x8000u ? 256u << i : 0u);
        w[i >> 1] &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
      }
    }
    tile[f] = w;
    special[f] = (uint16_t)bits16;
  }
}
// A lane's memory: bit 4 mb + q is channel 16 mb + 4 g + q of its row.
struct Seen16 { uint32_t plus, minus; };
template <int D>
__device__ __forceinline__ void remember(Seen16& x, const uint16_t* special, int tokens, int g) {
  for (int token = 0; token < tokens; ++token)
    for (int mb = 0; mb < D / 16; ++mb) {
      const uint32_t s = (uint32_t)special[v_chunk<D>(token, 2 * mb + (g >> 1))] >> (4 * (g & 1));
      x.plus |= (s & 15u) << (4 * mb);
      x.minus |= ((s >> 8) & 15u) << (4 * mb);
    }
}
template <int D> __device__ __forceinline__ void bring_back(f4 (&acc)[D / 16], const Seen16& x) {
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if ((x.plus >> (4 * mb + q)) & 1u) acc[mb][q] += __builtin_inff();
      if ((x.minus >> (4 * mb + q)) & 1u) acc[mb][q] -= __builtin_inff();
    }
}

}  // namespace iak

#endif
