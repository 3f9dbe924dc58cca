// The newest tokens' keys turned by their positions and stored, with their values, into their
// sequences' pages (float16 pages, or the microscaled 4-bit cache's), the queries turned along, on
// gfx950. A pair of channels (x, y) of a token at position p becomes
//   (x cos a - y sin a, x sin a + y cos a),  a = p f_i,
// pair i being channels (i, i + R/2), or (2i, 2i + 1) interleaved; the channels from R on stay.
//
// A thread takes 8 pairs, or 16 channels that stay, of one token, and goes through heads of it: one
// after the other the queries' and the keys' (with the values), for which its 8 sines and
// cosines are the same. What bounds long calls is the bytes, short ones the launch: the prompts of 8
// sequences (up to 4,001 tokens, 32 query heads and 8 of keys and values, 128 channels, float16) 614 MB
// in 128 to 140 us, 4.4 to 4.8 TB/s (148 under the profiler, as the other figures here); one token of 64 sequences 5.3
// us. Into 4-bit blocks the 64-bit angles count: 5 x 509 tokens
// of 16 + 4 heads x 64 in float32 14.5 us.
//
// Angles reach far beyond one turn (10^6 radians), where a float32 angle is off by 0.06: turns
// are counted in 64 bits and reduced there. For float16 pages and the queries the
// rest is done in 32 bits. Codes of 4 bits are rounded from 64 bits: a value that 32 bits put on the other
// side of a code's border would be a step of a third off.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "iak_device.h"
#include "mx_format.h"
#include "step_internal.h"

namespace iak {

namespace {

constexpr int ROTARY_THREADS = 256;
constexpr int64_t ROTARY_BUSY = 256 * 2048;   // threads that keep the card busy (prompts as above 148 us, with a quarter of them 161, with four times 156)

// sin(x) and cos(x) for |x| <= pi / 4, by their Taylor series: the first term left out is at most
// 2^-25 and 2^-63.
__device__ __forceinline__ void sine_cosine(float x, float& s, float& c) {
  const float z = x * x;
  s = __builtin_fmaf(x * z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.f / 40320, -1.f / 720), 1.f / 24), -0.5f), 1.f);
}
__device__ __forceinline__ void sine_cosine(double x, double& s, double& c) {
  const double z = x * x;
  double p = 1.0 / 355687428096000.0, q = -1.0 / 6402373705728000.0;
  const double odd[7] = {-1.0 / 1307674368000.0, 1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0};
  const double even[8] = {1.0 / 20922789888000.0, -1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0,
                          1.0 / 40320.0, -1.0 / 720.0, 1.0 / 24.0, -0.5};
#pragma unroll
  for (int i = 0; i < 7; ++i) p = __builtin_fma(z, p, odd[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) q = __builtin_fma(z, q, even[i]);
  s = __builtin_fma(x * z, p, x);
  c = __builtin_fma(z, q, 1.0);
}

// Sine and cosine of position * freq, each in R.
template <typename R> __device__ __forceinline__ void turn_of(int position, float freq, R& s, R& c) {
  // turns a position, 1 / 2 pi of the frequency, in two parts: 2^31 positions would cost one 2^-22 of a turn
  constexpr double PI_HIGH = 0.15915494309189535, PI_LOW = -9.839338337591243e-18;
  const double high = (double)freq * PI_HIGH, low = __builtin_fma((double)freq, PI_HIGH, -high) + (double)freq * PI_LOW;
  const double turns = (double)position * high;
  const double rest = __builtin_fma((double)position, high, -turns) + (double)position * low;
  const double quarters = 4 * ((turns - __builtin_rint(turns)) + rest);                // in [-2, 2]
  const double q = __builtin_rint(quarters);
  R x, y;
  sine_cosine((R)((quarters - q) * 1.57079632679489661923), x, y);
  const int k = (int)q & 3;
  s = k & 1 ? y : x;
  c = k & 1 ? x : y;
  if (k & 2) s = -s;
  if ((k + 1) & 2) c = -c;
}

typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ void load8(const T* p, T (&x)[8]) {
  any4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(p) + i);
  __builtin_memcpy(x, w, sizeof(w));
}
template <typename T> __device__ __forceinline__ void store8(T* p, const T (&x)[8]) {
  any4 w[sizeof(T) / 2];
  __builtin_memcpy(w, x, sizeof(w));
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<any4*>(p) + i);
}

// What a thread holds of a head: channels at[0] .. + 7 and at[1] .. + 7.
struct Pieces { int at[2]; bool turns; };

template <typename T, typename R, bool INTERLEAVED>
__device__ __forceinline__ void turned(const T (&a)[8], const T (&b)[8], const R (&s)[8], const R (&c)[8], bool turns,
                                       R (&x)[8], R (&y)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) { x[j] = (R)a[j]; y[j] = (R)b[j]; }
  if (!turns) return;
  if constexpr (INTERLEAVED) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const R p = x[2 * j], q = x[2 * j + 1], u = y[2 * j], v = y[2 * j + 1];
      x[2 * j] = __builtin_fma(p, c[j], -(q * s[j]));
      x[2 * j + 1] = __builtin_fma(p, s[j], q * c[j]);
      y[2 * j] = __builtin_fma(u, c[4 + j], -(v * s[4 + j]));
      y[2 * j + 1] = __builtin_fma(u, s[4 + j], v * c[4 + j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const R p = x[j], q = y[j];
      x[j] = __builtin_fma(p, c[j], -(q * s[j]));
      y[j] = __builtin_fma(p, s[j], q * c[j]);
    }
  }
}

// To odd: what 32 bits cannot hold leaves its mark in the last one, so that a rounding to few bits
// comes out as from 64.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  const double d = (double)f;
  uint32_t b = f2u(f);
  if (d != x && (b & 0x7FFFFFFFu) < 0x7F800000u) {
    if (fabs(d) > fabs(x)) --b;        // towards zero
    b |= 1u;
  }
  return u2f(b);
}
__device__ __forceinline__ float to_odd(float x) { return x; }

// Codes of the thread's two pieces, and the scale bytes of the blocks they lie in. The 4 (D = 64) or 8
// lanes of a token put their pieces' maxima into `row` (D / 8 words of LDS that no other token uses).
__device__ __forceinline__ float piece_max(const float (&x)[8]) {
  float m = 0.f, nan = 0.f;            // nan: NaN if any value is infinite or NaN, else 0
#pragma unroll
  for (int j = 0; j < 8; ++j) { m = fmaxf(m, fabsf(x[j])); nan = __builtin_fmaf(x[j], 0.f, nan); }
  return nan == 0.f ? m : __builtin_inff();
}
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], float most, uint32_t& byte) {
  if (most == __builtin_inff()) { byte = MX_SCALE_NAN; return 0u; }
  int e = (int)(f2u(most) >> 23) - 127 - 2;
  e = e < MX_E_MIN ? MX_E_MIN : (e > MX_E_MAX ? MX_E_MAX : e);
  byte = (uint32_t)(e + 127);
  const float s = u2f(byte << 23);
  uint32_t o = 0u;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[0], x[1], s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[2], x[3], s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[4], x[5], s, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, x[6], x[7], s, 3);
  return o;
}

template <typename R>
__device__ __forceinline__ void store_codes(const RotaryArgs& a, const R (&x)[8], const R (&y)[8], int64_t token, const Pieces& at,
                                            uint8_t* codes, uint8_t* scales, float* row, bool there) {
  float f[2][8], most[2];
#pragma unroll
  for (int j = 0; j < 8; ++j) { f[0][j] = to_odd(x[j]); f[1][j] = to_odd(y[j]); }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int p = 0; p < 2; ++p) row[at.at[p] >> 3] = piece_max(f[p]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const f4 m = *reinterpret_cast<const f4*>(row + ((at.at[p] >> 3) & ~3));
    most[p] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  }
  if (!there) return;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    uint32_t byte;
    const uint32_t c = codes8(f[p], most[p], byte);
    const int64_t piece = token * (a.D / 8) + (at.at[p] >> 3);
    reinterpret_cast<uint32_t*>(codes)[piece] = c;
    if ((piece & 3) == 0) scales[piece >> 2] = (uint8_t)byte;
  }
}

// Thread number -> chunk of 16 channels, token of a group of 8 (GROUP) or 1, and the first of the heads that it
// goes through, `lanes` apart; the rest of the number counts groups of tokens.
template <typename T, typename R, bool INTERLEAVED, bool PACKED>
__global__ __launch_bounds__(ROTARY_THREADS) void rotary_append_kernel(const RotaryArgs a) {
  __shared__ float maxima[PACKED ? ROTARY_THREADS * 2 : 1];
  const uint32_t chunk_bits = a.D == 128 ? 3 : 2;
  const uint32_t n = blockIdx.x * (uint32_t)ROTARY_THREADS + threadIdx.x;
  const int chunk = (int)(n & ((1u << chunk_bits) - 1));
  const uint32_t rest = n >> (chunk_bits + a.group_bits);
  const uint32_t tokens = rest / (uint32_t)a.lanes;
  const int head0 = (int)(rest - tokens * (uint32_t)a.lanes);
  const uint32_t token = (tokens << a.group_bits) + ((n >> chunk_bits) & ((1u << a.group_bits) - 1));
  const int half = a.R / 2, pairs = a.R / 16;      // threads whose channels turn
  Pieces at;
  at.turns = chunk < pairs;
  if (!INTERLEAVED && at.turns) { at.at[0] = 8 * chunk; at.at[1] = half + 8 * chunk; }
  else { at.at[0] = 16 * chunk; at.at[1] = 16 * chunk + 8; }
  float freq[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) freq[j] = at.turns ? a.freq[8 * chunk + j] : 0.f;

  const bool in = token < (uint32_t)a.count;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    int fresh = a.count;
    if (a.q_lens) {
      const int q = a.q_lens[b];
      fresh = q < 0 ? 0 : (q > a.count ? a.count : q);
    }
    const int i = in ? (int)token : 0;
    const bool live = in && i < fresh;
    R s[8], c[8];
    int turned_by = 0;
    bool known = false;
    for (int h = head0; h < a.Hq + a.Hkv; h += a.lanes) {
      const bool query = h < a.Hq;
      const int kv = query ? h / a.G : h - a.Hq;
      const int64_t row = (int64_t)b * a.Hkv + kv;
      const int listed = a.valid[row];
      const int64_t most = (int64_t)a.W * PS;
      const int last = listed < 0 ? 0 : (listed > most ? (int)most : listed);
      const int number = last - fresh + i;
      if (live && at.turns) {
        const int position = a.positions ? a.positions[b * a.position_stride + i] : number;
        if (!known || position != turned_by) {
#pragma unroll
          for (int j = 0; j < 8; ++j) turn_of<R>(position, freq[j], s[j], c[j]);
          turned_by = position;
          known = true;
        }
      }
      T u[8], v[8];
      R x[8], y[8];
      if (query) {
        T* to = reinterpret_cast<T*>(a.q_out) + b * a.qob + i * a.qot + h * a.qoh;
        if (live) {
          const T* from = reinterpret_cast<const T*>(a.q) + b * a.qb + i * a.qt + h * a.qh;
          load8(from + at.at[0], u);
          load8(from + at.at[1], v);
          turned<T, R, INTERLEAVED>(u, v, s, c, at.turns, x, y);
#pragma unroll
          for (int j = 0; j < 8; ++j) { u[j] = (T)x[j]; v[j] = (T)y[j]; }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = v[j] = (T)0.f;
        }
        if (in) { store8(to + at.at[0], u); store8(to + at.at[1], v); }
        continue;
      }
      const MxSlot slot = live ? mx_slot(a.table + row * a.W, number, a.W, a.NP) : MxSlot{0, false};
      T ku[8], kv8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = v[j] = ku[j] = kv8[j] = (T)0.f;
      if (slot.there) {
        const T* k = reinterpret_cast<const T*>(a.k) + b * a.kb + i * a.kt + kv * a.kh;
        const T* w = reinterpret_cast<const T*>(a.v) + b * a.vb + i * a.vt + kv * a.vh;
        load8(k + at.at[0], ku);
        load8(k + at.at[1], kv8);
        load8(w + at.at[0], u);
        load8(w + at.at[1], v);
        turned<T, R, INTERLEAVED>(ku, kv8, s, c, at.turns, x, y);
        if (a.tags && chunk == 0 && (i == 0 || (number & (PS - 1)) == 0)) a.tags[slot.token / PS] = a.tag;
      }
      if constexpr (PACKED) {
        // the lanes of a token go together: they have one slot
        if (!slot.there) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = y[j] = 0;
        }
        float* words = maxima + (threadIdx.x >> chunk_bits << (chunk_bits + 1));
        store_codes<R>(a, x, y, slot.token, at, a.k_codes, a.k_scales, words, slot.there);
        float f[8], g[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) { f[j] = (float)u[j]; g[j] = (float)v[j]; }
        store_codes<float>(a, f, g, slot.token, at, a.v_codes, a.v_scales, words, slot.there);
      } else if (slot.there) {
        _Float16 o[8], p[8];
        _Float16* k = reinterpret_cast<_Float16*>(a.k_pages) + slot.token * a.D;
        _Float16* w = reinterpret_cast<_Float16*>(a.v_pages) + slot.token * a.D;
#pragma unroll
        for (int j = 0; j < 8; ++j) { o[j] = (_Float16)x[j]; p[j] = (_Float16)y[j]; }
        store8(k + at.at[0], o);
        store8(k + at.at[1], p);
#pragma unroll
        for (int j = 0; j < 8; ++j) { o[j] = (_Float16)(float)u[j]; p[j] = (_Float16)(float)v[j]; }
        store8(w + at.at[0], o);
        store8(w + at.at[1], p);
      }
    }
  }
}

template <typename T, bool INTERLEAVED> void launch_typed(const RotaryArgs& a, dim3 grid, hipStream_t stream) {
  if (a.k_codes) hipLaunchKernelGGL((rotary_append_kernel<T, double, INTERLEAVED, true>), grid, dim3(ROTARY_THREADS), 0, stream, a);
  else hipLaunchKernelGGL((rotary_append_kernel<T, float, INTERLEAVED, false>), grid, dim3(ROTARY_THREADS), 0, stream, a);
}
template <bool INTERLEAVED> void launch_rotary(const RotaryArgs& a, int dtype, dim3 grid, hipStream_t stream) {
  if (dtype == IAK_DTYPE_F32) launch_typed<float, INTERLEAVED>(a, grid, stream);
  else if (dtype == IAK_DTYPE_F16) launch_typed<_Float16, INTERLEAVED>(a, grid, stream);
  else launch_typed<__bf16, INTERLEAVED>(a, grid, stream);
}

}  // namespace

hipError_t launch_rotary_append(const iak_rotary_append_args& c, hipStream_t stream) {
  RotaryArgs a;
  a.B = c.batch; a.count = c.count; a.Hq = c.q ? c.num_q_heads : 0; a.Hkv = c.num_kv_heads; a.D = c.head_dim; a.R = c.rotary_dim;
  a.G = a.Hq > 0 ? a.Hq / a.Hkv : 1;
  a.W = c.table_width; a.NP = c.num_pages;
  a.q = c.q; a.qb = c.q_stride_b; a.qt = c.q_stride_t; a.qh = c.q_stride_h;
  a.q_out = c.q_out; a.qob = c.q_out_stride_b; a.qot = c.q_out_stride_t; a.qoh = c.q_out_stride_h;
  a.k = c.k; a.kb = c.k_stride_b; a.kt = c.k_stride_t; a.kh = c.k_stride_h;
  a.v = c.v; a.vb = c.v_stride_b; a.vt = c.v_stride_t; a.vh = c.v_stride_h;
  a.freq = c.inv_freq; a.positions = c.positions; a.position_stride = c.position_stride_b;
  a.table = c.page_table; a.valid = c.valid_tokens; a.q_lens = c.q_lens;
  a.k_pages = c.k_pages; a.v_pages = c.v_pages;
  a.k_codes = reinterpret_cast<uint8_t*>(c.k_codes); a.k_scales = reinterpret_cast<uint8_t*>(c.k_scales);
  a.v_codes = reinterpret_cast<uint8_t*>(c.v_codes); a.v_scales = reinterpret_cast<uint8_t*>(c.v_scales);
  a.tags = c.page_tags; a.tag = c.tag;
  const int chunks = a.D / 16, heads = a.Hq + a.Hkv;
  // 8 tokens a thread group where there are many: whole lines of a page are written at once (the prompts 148 us,
  // one by one 153); below 16 a group could be half empty, and nothing is gained (8 tokens of 64 sequences: 7.2 us both)
  a.group_bits = a.count >= 16 ? 3 : 0;
  const int64_t tokens = ((int64_t)a.count + (1 << a.group_bits) - 1) >> a.group_bits << a.group_bits;
  // a head a thread until the card has threads enough, then as few sines as keep it busy
  const int64_t want = (ROTARY_BUSY + tokens * chunks * a.B - 1) / (tokens * chunks * a.B);
  a.lanes = want < heads ? (int)want : heads;
  const int64_t threads = tokens * chunks * a.lanes;
  const dim3 grid((uint32_t)((threads + ROTARY_THREADS - 1) / ROTARY_THREADS), (uint32_t)(a.B < 32768 ? a.B : 32768));
  if (c.interleaved) launch_rotary<true>(a, c.dtype, grid, stream);
  else launch_rotary<false>(a, c.dtype, grid, stream);
  return hipGetLastError();
}

}  // namespace iak
