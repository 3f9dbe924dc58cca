// Attention of one or several query tokens per sequence over the microscaled 4-bit cache,
// for gfx950:  out = softmax(sm_scale q . k) v  over the tokens that a query sees.
//
// A wave takes a tile of 16 query rows that share a KV head (row = query token * G + head of
// the group) and one split of the head's table entries, two pages (32 tokens) a step.
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

constexpr int MX_WAVES = 4;
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
  uint32_t ks[2], vs[2];
};

template <int D>
__device__ __forceinline__ void load_pair(MxPair<D>& r, const MxAttn& a, const int (&id)[2], int c, int g) {
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t page = id[p] < 0 ? 0 : id[p];
    const int64_t code = (page * PS + c) * (D / 2) + g * (D / 8);
    const int64_t sc = (page * PS + c) * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK;
    if constexpr (D == 128) {
      const u4 k = *reinterpret_cast<const u4*>(a.k_codes + code), v = *reinterpret_cast<const u4*>(a.v_codes + code);
#pragma unroll
      for (int i = 0; i < 4; ++i) { r.k[p][i] = k[i]; r.v[p][i] = v[i]; }
    } else {
      const u2 k = *reinterpret_cast<const u2*>(a.k_codes + code), v = *reinterpret_cast<const u2*>(a.v_codes + code);
#pragma unroll
      for (int i = 0; i < 2; ++i) { r.k[p][i] = k[i]; r.v[p][i] = v[i]; }
    }
    r.ks[p] = a.k_scales[sc];
    r.vs[p] = a.v_scales[sc];
  }
}

template <typename T>
__device__ __forceinline__ void out4(T* p, bool vec, const float (&x)[4]) {
  T t[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) t[j] = (T)x[j];
  if (vec) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<u4*>(p) = *reinterpret_cast<const u4*>(t);
    else *reinterpret_cast<u2*>(p) = *reinterpret_cast<const u2*>(t);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = t[j];
  }
}
__device__ __forceinline__ void store_out4(const MxAttn& a, int64_t at, const float (&x)[4]) {
  if (a.out_dtype == IAK_DTYPE_F32) out4(reinterpret_cast<float*>(a.out) + at, a.out_vec, x);
  else if (a.out_dtype == IAK_DTYPE_F16) out4(reinterpret_cast<_Float16*>(a.out) + at, a.out_vec, x);
  else out4(reinterpret_cast<__bf16*>(a.out) + at, a.out_vec, x);
}

template <int D, bool QF32>
__global__ __launch_bounds__(64 * MX_WAVES) void mx_rows_kernel(const MxAttn a) {
  __shared__ u4 vt[MX_WAVES][2 * PS * D / 8];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int64_t item = (int64_t)blockIdx.x * MX_WAVES + w;
  if (item >= a.items) return;                                   // no barriers below
  const int split = (int)(item % a.splits);
  const int64_t tile_at = item / a.splits;
  const int tile = (int)(tile_at % a.tiles);
  const int64_t kvrow = tile_at / a.tiles;
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow % a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * 16, 16);
  const int e0 = split * a.chunk, e1 = e0 + a.chunk < entries ? e0 + a.chunk : entries;
  if (split > 0 && e0 >= e1) return;                             // the merge does not look at it

  const int r = tile * 16 + c, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const bool active = r < a.L * a.G, live = active && i < n.queries;
  const int seen = live ? mx_seen(a, n, i) : 0;
  int least = live ? seen : 0x7FFFFFFF;                          // tokens below it need no mask
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(least, o, 64); least = x < least ? x : least; }

  // queries: scaled by a power of two to a largest element in [2^14, 2^15)
  h8 qhi[D / 32], qlo[QF32 ? D / 32 : 1];
  float mult;
  {
    float x[D / 32][8];
    float m = 0.f;
    if (live) {
      const int64_t at = b * a.qsb + i * a.qst + head * a.qsh + g * (D / 4);
#pragma unroll
      for (int s = 0; s < D / 32; ++s) mx_load_q(a, at + 8 * s, x[s]);
    } else {
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] = 0.f;
    }
    bool fine = true;
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = fabsf(x[s][j]);
        fine = fine && v < __builtin_inff();
        m = fmaxf(m, v);
      }
    m = xmax16_32(fine ? m : __builtin_inff());
    fine = m < __builtin_inff();
    const int e = m > 0.f ? (int)(f2u(m) >> 23) - 127 : 0;
    mult = fine ? __builtin_ldexpf(a.score_mult, e - 14) : __builtin_nanf("");
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = fine ? __builtin_ldexpf(x[s][j], 14 - e) : 0.f;
        qhi[s][j] = (_Float16)v;
        if constexpr (QF32) qlo[s][j] = (_Float16)(v - (float)qhi[s][j]);
      }
  }

  f4 acc[D / 16];
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) acc[mb] = f4{0.f, 0.f, 0.f, 0.f};
  float m = M_NONE, l = 0.f;
  const int32_t* row = a.table + kvrow * a.W;

  for (int e = e0; e < e1; e += 2) {
    int id[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      id[p] = e + p < e1 ? row[e + p] : -1;
      if (id[p] < 0 || id[p] >= a.NP) id[p] = -1;
    }
    MxPair<D> x;
    load_pair<D>(x, a, id, c, g);

    f4 s[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      s[p] = f4{0.f, 0.f, 0.f, 0.f};
      const float ks = mx_scale(x.ks[p]);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t o[4];
        mx8_to_f16(x.k[p][j], ks, o);
        const h8 ka = make_h8(o[0], o[1], o[2], o[3]);
        s[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[j], s[p], 0, 0, 0);
        if constexpr (QF32) s[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[j], s[p], 0, 0, 0);
      }
      s[p] *= mult;
      // tokens with a NaN block (rare): their scores are NaN
      const uint64_t bad = __builtin_amdgcn_ballot_w64(x.ks[p] == MX_SCALE_NAN || x.vs[p] == MX_SCALE_NAN);
      if (bad) {
        const uint32_t t = (uint32_t)(bad | (bad >> 16) | (bad >> 32) | (bad >> 48));
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if ((t >> (4 * g + q)) & 1u) s[p][q] = __builtin_nanf("");
      }
      // tokens that a row does not see
      if ((e + p + 1) * PS > least || id[p] < 0) {
        const int lim = id[p] < 0 ? 0 : seen - (e + p) * PS;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (4 * g + q >= lim) s[p][q] = -__builtin_inff();
      }
    }
    float pm = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    pm = xmax16_32(pm);
    const bool grow = pm > m + RESCALE_SLACK;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float mn = grow ? pm : m;
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) acc[mb] *= alpha;
      m = mn;
    }
    h8 pb, pl;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v = __builtin_amdgcn_exp2f(s[p][q] - m + P_SHIFT);
        l += v;
        pb[4 * p + q] = (_Float16)v;
        if constexpr (QF32) pl[4 * p + q] = (_Float16)(v - (float)pb[4 * p + q]);
      }

    // V: rows of this lane's token into LDS, four tokens of a channel back
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const float vs = mx_scale(x.vs[p]);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t o[4];
        mx8_to_f16(x.v[p][j], vs, o);
        vt[w][p * (PS * D / 8) + v_chunk<D>(c, g * (D / 32) + j)] = u4{o[0], o[1], o[2], o[3]};
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    typedef __attribute__((address_space(3))) s4v lds_s4;
    const char* base = reinterpret_cast<const char*>(&vt[w][0]);
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) {
      s4v t[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int at = p * (PS * D / 8) + v_chunk<D>(4 * g + (c >> 2), 2 * mb + ((c & 3) >> 1));
        t[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + at * 16 + (c & 1) * 8));
      }
      const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
      acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[mb], 0, 0, 0);
      if constexpr (QF32) acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, acc[mb], 0, 0, 0);
    }
  }

  l = xsum16_32(l);
  if (!active) return;
  if (a.splits > 1) {
    const int64_t slot = (tile_at * a.splits + split) * 16 + c;
    if (g == 0) { a.ws_m[slot] = m; a.ws_l[slot] = l; }
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) *reinterpret_cast<f4*>(a.ws_acc + slot * D + 16 * mb + 4 * g) = acc[mb];
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;                   // NaN stays
  const int64_t at = b * a.osb + i * a.ost + head * a.osh + 4 * g;
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) {
    float o[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] = live ? acc[mb][q] * inv : 0.f;
    store_out4(a, at + 16 * mb, o);
  }
}

// The splits of one query row: a wave, D / 64 channels a lane.
template <int D>
__global__ __launch_bounds__(64 * MX_WAVES) void mx_merge_kernel(const MxAttn a) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t at = (int64_t)blockIdx.x * MX_WAVES + (threadIdx.x >> 6);
  const int rows = a.L * a.G;
  if (at >= (int64_t)a.B * a.Hkv * rows) return;
  const int r = (int)(at % rows);
  const int64_t kvrow = at / rows;
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow % a.Hkv);
  const int tile = r / 16, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const MxRows n = mx_rows(a, kvrow, b);
  const bool live = i < n.queries;
  const int entries = mx_entries(a, n, tile * 16, 16);
  const int parts = live ? (entries + a.chunk - 1) / a.chunk : 0;
  const int64_t first = (kvrow * a.tiles + tile) * a.splits * 16 + (r & 15);
  float M = M_NONE, L = 0.f, o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) o[j] = 0.f;
  for (int s = 0; s < parts; ++s) M = fmaxf(M, a.ws_m[first + (int64_t)s * 16]);
  for (int s = 0; s < parts; ++s) {
    const int64_t slot = first + (int64_t)s * 16;
    const float wgt = __builtin_amdgcn_exp2f(a.ws_m[slot] - M);
    L += wgt * a.ws_l[slot];
#pragma unroll
    for (int j = 0; j < PER; ++j) o[j] += wgt * a.ws_acc[slot * D + PER * lane + j];
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  const int64_t to = b * a.osb + i * a.ost + head * a.osh + PER * lane;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float v = o[j] * inv;
    if (a.out_dtype == IAK_DTYPE_F32) reinterpret_cast<float*>(a.out)[to + j] = v;
    else if (a.out_dtype == IAK_DTYPE_F16) reinterpret_cast<_Float16*>(a.out)[to + j] = (_Float16)v;
    else reinterpret_cast<__bf16*>(a.out)[to + j] = (__bf16)v;
  }
}

template <int D, bool QF32> void launch_rows(const MxAttn& a, hipStream_t stream) {
  hipLaunchKernelGGL((mx_rows_kernel<D, QF32>), dim3((uint32_t)((a.items + MX_WAVES - 1) / MX_WAVES)), dim3(64 * MX_WAVES),
                     0, stream, a);
}

}  // namespace

hipError_t launch_mx_attention(const MxAttn& a, hipStream_t stream) {
  const bool f32 = a.q_dtype == IAK_DTYPE_F32;
  if (a.D == 128) f32 ? launch_rows<128, true>(a, stream) : launch_rows<128, false>(a, stream);
  else f32 ? launch_rows<64, true>(a, stream) : launch_rows<64, false>(a, stream);
  if (a.splits > 1) {
    const int64_t waves = (int64_t)a.B * a.Hkv * a.L * a.G;
    const dim3 grid((uint32_t)((waves + MX_WAVES - 1) / MX_WAVES));
    if (a.D == 128) hipLaunchKernelGGL(mx_merge_kernel<128>, grid, dim3(64 * MX_WAVES), 0, stream, a);
    else hipLaunchKernelGGL(mx_merge_kernel<64>, grid, dim3(64 * MX_WAVES), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace iak
