// Tokens of the microscaled 4-bit cache on gfx950: quantise on write, and read back.
//
// A block is 32 channels of one token's K or V:
//   e = clamp(floor(log2 max|x|) - 2, -23, 13), code = RNE_e2m1(x / 2^e), at most 6
// (the OCP microscaling conversion; the clamp keeps every value a float16 number). The
// floor of the logarithm is the maximum's exponent field, so no logarithm is taken, and
// x / 2^e is exact, so a code is rounded once, by the conversion instruction.
//
// A thread takes 8 channels of K and the same 8 of V: 16-byte loads, one dword of codes
// stored, and four neighbouring lanes agree on the block's maximum over lane swaps. What
// bounds it is the bytes. Long calls give a workgroup 16 tokens of one head, whose codes are
// one run of memory wherever a page has room; calls of few tokens give it all heads of one.
// 21,400 new tokens x 8 heads x 128 channels in 8 sequences padded to 4,001: append 27 us (111 MB,
// 4.1 TB/s), read 23 us (the same and 43 MB of zeros, the codes from the caches); 64 new tokens:
// 3.4 us each. Two or four tokens a thread changed nothing (50.5 us for both; 53.8).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "mx_internal.h"
#include "mx_format.h"

namespace iak {

namespace {

constexpr int MX_THREADS = 256;

// Eight values as floats, wherever they lie: one or two 16-byte loads, which the hardware takes
// at any address of the type. Values are streamed, in and out: appending and reading back 21,400
// tokens took 63 us through the caches and takes 50.
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ void load8f(const T* p, float (&x)[8]) {
  any4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(p) + i);
  T t[8];
  __builtin_memcpy(t, w, sizeof(t));
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)t[j];
}

// The codes (8 per lane, one dword) and the scale byte of the block that lanes 4n .. 4n+3 hold.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], uint32_t& byte) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(x[j]));
  float nan = 0.f;                                // NaN if any value is infinite or NaN, else 0
#pragma unroll
  for (int j = 0; j < 8; ++j) nan = __builtin_fmaf(x[j], 0.f, nan);
  m = nan == 0.f ? m : __builtin_inff();
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

template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  T t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = (T)x[j];
  any4 w[sizeof(T) / 2];
  __builtin_memcpy(w, t, sizeof(t));
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_nontemporal_store(w[i], reinterpret_cast<any4*>(p) + i);
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

struct TokenAt { int i, h, c; bool in; };   // token, head, chunk c of 8 channels

// Thread number -> (token / group, head, token % group, chunk); group is 16 or 1, see token_group().
__device__ __forceinline__ TokenAt token_at(const iak_mx_tokens_args& a, int group) {
  const uint32_t chunk_bits = a.head_dim == 128 ? 4 : 3, group_bits = group == 16 ? 4 : 0;
  const uint32_t n = blockIdx.x * (uint32_t)MX_THREADS + threadIdx.x;
  const uint32_t row = n >> (chunk_bits + group_bits);
  const uint32_t tokens = row / (uint32_t)a.num_kv_heads;
  TokenAt t;
  t.c = (int)(n & ((1u << chunk_bits) - 1));
  t.h = (int)(row - tokens * (uint32_t)a.num_kv_heads);
  const uint32_t i = (tokens << group_bits) + ((n >> chunk_bits) & (uint32_t)(group - 1));
  t.in = i < (uint32_t)a.count;
  t.i = t.in ? (int)i : 0;
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
__global__ __launch_bounds__(MX_THREADS) void mx_append_kernel(const iak_mx_tokens_args a, int group) {
  const TokenAt t = token_at(a, group);
  for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t row = (int64_t)b * a.num_kv_heads + t.h;
    const int tokens = row_tokens(a, row), n = new_tokens(a, b);   // loads under way together
    if (!t.in || t.i >= n) continue;
    // the values come while the token's place is looked up; the four lanes of a block are one
    // token's and go together
    float k[8], v[8];
    load8f(reinterpret_cast<const T*>(a.k) + b * a.k_stride_b + t.i * a.k_stride_t + t.h * a.k_stride_h + 8 * t.c, k);
    load8f(reinterpret_cast<const T*>(a.v) + b * a.v_stride_b + t.i * a.v_stride_t + t.h * a.v_stride_h + 8 * t.c, v);
    const MxSlot at = mx_slot(a.page_table + row * a.table_width, tokens - n + t.i, a.table_width, a.num_pages);
    if (!at.there) continue;
    uint32_t kb, vb;
    const uint32_t kc = quantise8(k, kb), vc = quantise8(v, vb);
    const int64_t code = at.token * (a.head_dim / 8) + t.c;
    reinterpret_cast<uint32_t*>(a.k_codes)[code] = kc;
    reinterpret_cast<uint32_t*>(a.v_codes)[code] = vc;
    if ((t.c & 3) == 0) {
      reinterpret_cast<uint8_t*>(a.k_scales)[code >> 2] = (uint8_t)kb;
      reinterpret_cast<uint8_t*>(a.v_scales)[code >> 2] = (uint8_t)vb;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(MX_THREADS) void mx_read_kernel(const iak_mx_tokens_args a, int group) {
  const TokenAt t = token_at(a, group);
  if (!t.in) return;
  for (int b = blockIdx.y; b < a.batch; b += gridDim.y) {
    const int64_t row = (int64_t)b * a.num_kv_heads + t.h;
    const int tokens = row_tokens(a, row), n = new_tokens(a, b);   // loads under way together
    const MxSlot at = mx_slot(a.page_table + row * a.table_width, tokens - n + t.i, a.table_width, a.num_pages);
    float k[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (t.i < n && at.there) {
      const int64_t code = at.token * (a.head_dim / 8) + t.c;
      values8(reinterpret_cast<const uint32_t*>(a.k_codes)[code], reinterpret_cast<const uint8_t*>(a.k_scales)[code >> 2], k);
      values8(reinterpret_cast<const uint32_t*>(a.v_codes)[code], reinterpret_cast<const uint8_t*>(a.v_scales)[code >> 2], v);
    }
    store8(reinterpret_cast<T*>(a.k) + b * a.k_stride_b + t.i * a.k_stride_t + t.h * a.k_stride_h + 8 * t.c, k);
    store8(reinterpret_cast<T*>(a.v) + b * a.v_stride_b + t.i * a.v_stride_t + t.h * a.v_stride_h + 8 * t.c, v);
  }
}

template <typename F> hipError_t by_dtype(int dtype, F&& f) {
  if (dtype == IAK_DTYPE_F32) f(float{});
  else if (dtype == IAK_DTYPE_F16) f(_Float16{});
  else f(__bf16{});
  return hipGetLastError();
}

// Tokens of one head that neighbouring threads take: 16, or 1 where that would leave most idle.
int token_group(const iak_mx_tokens_args& a) { return a.count >= 16 ? 16 : 1; }

dim3 token_grid(const iak_mx_tokens_args& a) {
  const int64_t group = token_group(a);
  const int64_t n = (a.count + group - 1) / group * group * a.num_kv_heads * (a.head_dim / 8);
  return dim3((uint32_t)((n + MX_THREADS - 1) / MX_THREADS), (uint32_t)(a.batch < 32768 ? a.batch : 32768));
}

}  // namespace

hipError_t launch_mx_append(const iak_mx_tokens_args& a, hipStream_t stream) {
  return by_dtype(a.dtype, [&](auto t) {
    hipLaunchKernelGGL((mx_append_kernel<decltype(t)>), token_grid(a), dim3(MX_THREADS), 0, stream, a, token_group(a));
  });
}

hipError_t launch_mx_read(const iak_mx_tokens_args& a, hipStream_t stream) {
  return by_dtype(a.dtype, [&](auto t) {
    hipLaunchKernelGGL((mx_read_kernel<decltype(t)>), token_grid(a), dim3(MX_THREADS), 0, stream, a, token_group(a));
  });
}

}  // namespace iak
