// Tokens of the microscaled 4-bit cache on gfx950: quantise on write, and read back.
//
// A block is 32 channels of one token's K or V:
//   e = clamp(floor(log2 max|x|) - 2, -23, 13), code = RNE_e2m1(x / 2^e), at most 6
// (the OCP microscaling conversion; the clamp keeps every value a float16 number). The
// floor of the logarithm is the maximum's exponent field, so no logarithm is taken, and
// x / 2^e is exact, so a code is rounded once, by the conversion instruction.
//
// A thread takes 8 channels of K and the same 8 of V: 16-byte loads, one dword of codes
// stored, and four neighbouring lanes agree on the block's maximum over lane swaps.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "mx_internal.h"
#include "mx_format.h"

namespace iak {

namespace {

constexpr int MX_THREADS = 256;

// Eight values as floats; `vec`: one or two 16-byte loads, else element by element.
template <typename T> __device__ __forceinline__ void load8f(const T* p, bool vec, float (&x)[8]) {
  if (vec) {
    T t[8];
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<u4*>(t) = *reinterpret_cast<const u4*>(p);
      *reinterpret_cast<u4*>(t + 4) = *reinterpret_cast<const u4*>(p + 4);
    } else {
      *reinterpret_cast<u4*>(t) = *reinterpret_cast<const u4*>(p);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)t[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)p[j];
  }
}

// The codes (8 per lane, one dword) and the scale byte of the block that lanes 4n .. 4n+3 hold.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], uint32_t& byte) {
  float m = 0.f;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = fabsf(x[j]);
    fine = fine && a < __builtin_inff();          // false for NaN too
    m = fmaxf(m, a);
  }
  m = fine ? m : __builtin_inff();
  m = fmaxf(m, __shfl_xor(m, 1, 64));
  m = fmaxf(m, __shfl_xor(m, 2, 64));
  if (m == __builtin_inff()) { byte = MX_SCALE_NAN; return 0u; }
  int e = (int)(f2u(m) >> 23) - 127 - 2;
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

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float (&x)[8]) {
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (T)x[j];
  if (vec) {
    *reinterpret_cast<u4*>(p) = *reinterpret_cast<const u4*>(t);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<u4*>(p + 4) = *reinterpret_cast<const u4*>(t + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = t[j];
  }
}

// Eight values of a code dword and its scale byte.
__device__ __forceinline__ void values8(uint32_t codes, uint32_t byte, float (&x)[8]) {
  uint32_t o[4];
  mx8_to_f16(codes, mx_scale(byte), o);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const h2 v = as_h2(o[j]);
    x[2 * j] = byte == MX_SCALE_NAN ? __builtin_nanf("") : (float)v[0];
    x[2 * j + 1] = byte == MX_SCALE_NAN ? __builtin_nanf("") : (float)v[1];
  }
}

struct TokenAt { int b, i, h, c; bool in; };   // channel chunk c of 8

__device__ __forceinline__ TokenAt token_at(const iak_mx_tokens_args& a) {
  const int chunks = a.head_dim / 8;
  int64_t n = (int64_t)blockIdx.x * MX_THREADS + threadIdx.x;
  TokenAt t;
  t.c = (int)(n % chunks); n /= chunks;
  t.h = (int)(n % a.num_kv_heads); n /= a.num_kv_heads;
  t.i = (int)(n % a.count); n /= a.count;
  t.b = (int)(n < a.batch ? n : a.batch - 1);
  t.in = n < a.batch;
  return t;
}

__device__ __forceinline__ int new_tokens(const iak_mx_tokens_args& a, int b) {
  if (!a.q_lens) return a.count;
  const int n = a.q_lens[b];
  return n < 0 ? 0 : (n > a.count ? a.count : n);
}

__device__ __forceinline__ int row_tokens(const iak_mx_tokens_args& a, int64_t row) {
  const int n = a.valid_tokens[row];
  const int64_t most = (int64_t)a.table_width * PS;
  return n < 0 ? 0 : (n > most ? (int)most : n);
}

template <typename T>
__global__ __launch_bounds__(MX_THREADS) void mx_append_kernel(const iak_mx_tokens_args a, bool vec) {
  const TokenAt t = token_at(a);
  const int n = new_tokens(a, t.b);
  const int64_t row = (int64_t)t.b * a.num_kv_heads + t.h;
  const MxSlot at = mx_slot(a.page_table + row * a.table_width, row_tokens(a, row) - n + t.i, a.table_width, a.num_pages);
  float k[8], v[8];
  load8f(reinterpret_cast<const T*>(a.k) + t.b * a.k_stride_b + t.i * a.k_stride_t + t.h * a.k_stride_h + 8 * t.c, vec, k);
  load8f(reinterpret_cast<const T*>(a.v) + t.b * a.v_stride_b + t.i * a.v_stride_t + t.h * a.v_stride_h + 8 * t.c, vec, v);
  uint32_t kb, vb;
  const uint32_t kc = quantise8(k, kb), vc = quantise8(v, vb);   // whole waves: the lanes of a block agree on its maximum
  if (!t.in || t.i >= n || !at.there) return;
  const int64_t code = at.token * (a.head_dim / 8) + t.c;
  reinterpret_cast<uint32_t*>(a.k_codes)[code] = kc;
  reinterpret_cast<uint32_t*>(a.v_codes)[code] = vc;
  if ((t.c & 3) == 0) {
    reinterpret_cast<uint8_t*>(a.k_scales)[code >> 2] = (uint8_t)kb;
    reinterpret_cast<uint8_t*>(a.v_scales)[code >> 2] = (uint8_t)vb;
  }
}

template <typename T>
__global__ __launch_bounds__(MX_THREADS) void mx_read_kernel(const iak_mx_tokens_args a, bool vec) {
  const TokenAt t = token_at(a);
  if (!t.in) return;
  const int n = new_tokens(a, t.b);
  const int64_t row = (int64_t)t.b * a.num_kv_heads + t.h;
  const MxSlot at = mx_slot(a.page_table + row * a.table_width, row_tokens(a, row) - n + t.i, a.table_width, a.num_pages);
  float k[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (t.i < n && at.there) {
    const int64_t code = at.token * (a.head_dim / 8) + t.c;
    values8(reinterpret_cast<const uint32_t*>(a.k_codes)[code], reinterpret_cast<const uint8_t*>(a.k_scales)[code >> 2], k);
    values8(reinterpret_cast<const uint32_t*>(a.v_codes)[code], reinterpret_cast<const uint8_t*>(a.v_scales)[code >> 2], v);
  }
  store8(reinterpret_cast<T*>(a.k) + t.b * a.k_stride_b + t.i * a.k_stride_t + t.h * a.k_stride_h + 8 * t.c, vec, k);
  store8(reinterpret_cast<T*>(a.v) + t.b * a.v_stride_b + t.i * a.v_stride_t + t.h * a.v_stride_h + 8 * t.c, vec, v);
}

// whether K and V may be read and written as 16-byte vectors
bool vectors(const iak_mx_tokens_args& a) {
  const int per = a.dtype == IAK_DTYPE_F32 ? 4 : 8;
  const int64_t strides = a.k_stride_b | a.k_stride_t | a.k_stride_h | a.v_stride_b | a.v_stride_t | a.v_stride_h;
  return strides % per == 0 && ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15u) == 0;
}

template <typename F> hipError_t by_dtype(int dtype, F&& f) {
  if (dtype == IAK_DTYPE_F32) f(float{});
  else if (dtype == IAK_DTYPE_F16) f(_Float16{});
  else f(__bf16{});
  return hipGetLastError();
}

int64_t token_blocks(const iak_mx_tokens_args& a) {
  const int64_t n = (int64_t)a.batch * a.count * a.num_kv_heads * (a.head_dim / 8);
  return (n + MX_THREADS - 1) / MX_THREADS;
}

}  // namespace

hipError_t launch_mx_append(const iak_mx_tokens_args& a, hipStream_t stream) {
  const bool vec = vectors(a);
  return by_dtype(a.dtype, [&](auto t) {
    hipLaunchKernelGGL((mx_append_kernel<decltype(t)>), dim3((uint32_t)token_blocks(a)), dim3(MX_THREADS), 0, stream, a, vec);
  });
}

hipError_t launch_mx_read(const iak_mx_tokens_args& a, hipStream_t stream) {
  const bool vec = vectors(a);
  return by_dtype(a.dtype, [&](auto t) {
    hipLaunchKernelGGL((mx_read_kernel<decltype(t)>), dim3((uint32_t)token_blocks(a)), dim3(MX_THREADS), 0, stream, a, vec);
  });
}

}  // namespace iak
