// Arguments of the 4-bit cache's attention kernels, and what each of them works out of the
// lengths on the device: how many tokens a query row sees, and how many table entries a tile
// of rows has to walk.
#ifndef IAK_MX_ATTENTION_H
#define IAK_MX_ATTENTION_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak_device.h"
#include "mx_internal.h"

namespace iak {

// Tokens of a row and new queries of its sequence, clamped to what there is room for.
struct MxRows { int tokens, queries, first; };   // query i sees `first + i + 1` tokens when causal

__device__ __forceinline__ MxRows mx_rows(const MxAttn& a, int64_t kvrow, int b) {
  MxRows n;
  const int64_t most = a.NP > 0 ? (int64_t)a.W * 16 : 0;
  const int v = a.valid[kvrow];
  n.tokens = v < 0 ? 0 : (v > most ? (int)most : v);
  n.queries = a.L;
  if (a.q_lens) {
    const int q = a.q_lens[b];
    n.queries = q < 0 ? 0 : (q > a.L ? a.L : q);
  }
  n.first = n.tokens - n.queries;
  return n;
}

// Tokens that query i of the row sees.
__device__ __forceinline__ int mx_seen(const MxAttn& a, const MxRows& n, int i) {
  const int s = a.causal ? n.first + i + 1 : n.tokens;
  return s < 0 ? 0 : (s > n.tokens ? n.tokens : s);
}

// Table entries that the query rows r0 .. r0 + count - 1 (row = query * G + head) see together.
__device__ __forceinline__ int mx_entries(const MxAttn& a, const MxRows& n, int r0, int count) {
  int last = r0 + count - 1;                                     // the last row sees most
  const int64_t rows = (int64_t)n.queries * a.G;
  if (last >= rows) last = (int)rows - 1;
  if (last < r0) return 0;
  return (mx_seen(a, n, last / a.G) + 15) / 16;
}

// N query values at element offset `at`, wherever they lie: 16-byte loads, all under way at once.
template <typename T, int N> __device__ __forceinline__ void mx_load(const T* p, float (&x)[N]) {
  T t[N];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int j = 0; j < N; ++j) x[j] = (float)t[j];
}
template <int N> __device__ __forceinline__ void mx_load_q(const MxAttn& a, int64_t at, float (&x)[N]) {
  if (a.q_dtype == IAK_DTYPE_F32) mx_load(reinterpret_cast<const float*>(a.q) + at, x);
  else if (a.q_dtype == IAK_DTYPE_F16) mx_load(reinterpret_cast<const _Float16*>(a.q) + at, x);
  else mx_load(reinterpret_cast<const __bf16*>(a.q) + at, x);
}

}  // namespace iak

#endif
