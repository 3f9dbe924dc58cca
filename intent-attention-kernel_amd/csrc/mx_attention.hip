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
  uint32_t ks[2], vs[2];
  int id[2];                       // wave-uniform; -1: no page
};

template <int D>
__device__ __forceinline__ void load_pair(MxPair<D>& r, const MxAttn& a, int id0, int id1, int c, int g) {
  r.id[0] = id0;
  r.id[1] = id1;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int64_t page = r.id[p] < 0 ? 0 : r.id[p];
    const uint32_t code = c * (D / 2) + g * (D / 8), sc = c * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK;
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
    r.ks[p] = (a.k_scales + page * (PS * D / MX_BLOCK))[sc];
    r.vs[p] = (a.v_scales + page * (PS * D / MX_BLOCK))[sc];
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
  const int seen = live ? mx_seen(a, n, i) : 0;
  int least = live ? seen : 0x7FFFFFFF;                          // tokens below it need no mask
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) { const int x = __shfl_xor(least, o, 64); least = x < least ? x : least; }

  // the wave's entries, 64 at a time: lane i holds number i of the block, in
  // `next` of the block after it
  const int32_t* row = a.table + kvrow * a.W;
  auto entry_id = [&](int k) {
    const int e = e0 + wave_entry<NW>(w, k);
    const int id = e < e1 ? row[e] : -1;
    return id < 0 || id >= a.NP ? -1 : id;
  };
  int ids = entry_id(lane), next = entry_id(64 + lane);
  auto page = [&](int k) { return k < 64 ? __builtin_amdgcn_readlane(ids, k) : __builtin_amdgcn_readlane(next, k - 64); };

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

  // one step: the pair `x` of entries e, e + 1; then `x` is the pair of pages to0, to1
  auto step = [&](MxPair<D>& x, int e, int to0, int to1) {
    f4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    const float ks[2] = {mx_scale(x.ks[0]), mx_scale(x.ks[1])}, vs[2] = {mx_scale(x.vs[0]), mx_scale(x.vs[1])};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        uint32_t o[4];
        mx8_to_f16(x.k[p][j], ks[p], o);
        const h8 ka = make_h8(o[0], o[1], o[2], o[3]);
        s[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[j], s[p], 0, 0, 0);
        if constexpr (QF32) s[p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[j], s[p], 0, 0, 0);
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
    uint32_t most = x.ks[0] > x.ks[1] ? x.ks[0] : x.ks[1], vmost = x.vs[0] > x.vs[1] ? x.vs[0] : x.vs[1];
    most = most > vmost ? most : vmost;
    uint32_t nan_tokens[2] = {0u, 0u};
    if (__builtin_amdgcn_ballot_w64(most == MX_SCALE_NAN)) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const uint64_t bad = __builtin_amdgcn_ballot_w64(x.ks[p] == MX_SCALE_NAN || x.vs[p] == MX_SCALE_NAN);
        nan_tokens[p] = (uint32_t)(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xFFFFu;
      }
    }
    const int id[2] = {x.id[0], x.id[1]};
    load_pair<D>(x, a, to0, to1, c, g);                          // under way during the rest of the step

#pragma unroll
    for (int p = 0; p < 2; ++p) s[p] *= mult;
    if (nan_tokens[0] | nan_tokens[1]) {                         // their scores are NaN
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if ((nan_tokens[p] >> (4 * g + q)) & 1u) s[p][q] = __builtin_nanf("");
    }
    if ((e + 2) * PS > least || (id[0] | id[1]) < 0) {           // tokens that a row does not see
#pragma unroll
      for (int p = 0; p < 2; ++p) {
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
    const float base = m - P_SHIFT;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float v = __builtin_amdgcn_exp2f(s[p][q] - base);
        l += v;
        pb[4 * p + q] = (_Float16)v;
        if constexpr (QF32) pl[4 * p + q] = (_Float16)(v - (float)pb[4 * p + q]);
      }

    // V back: four tokens of a channel in each lane
    typedef __attribute__((address_space(3))) s4v lds_s4;
    const char* from = reinterpret_cast<const char*>(&vt[w][0]);
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb) {
      s4v t[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int at = p * (PS * D / 8) + v_chunk<D>(4 * g + (c >> 2), 2 * mb + ((c & 3) >> 1));
        t[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(from + at * 16 + (c & 1) * 8));
      }
      const h8 va = __builtin_bit_cast(h8, __builtin_shufflevector(t[0], t[1], 0, 1, 2, 3, 4, 5, 6, 7));
      acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, acc[mb], 0, 0, 0);
      if constexpr (QF32) acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl, acc[mb], 0, 0, 0);
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
  l = xsum16_32(l);
  __syncthreads();
  if (g == 0) { part_m[w][c] = m; part_l[w][c] = l; }
  f4* sums = reinterpret_cast<f4*>(&vt[w][0]);
#pragma unroll
  for (int mb = 0; mb < D / 16; ++mb) sums[c * (D / 4) + ((4 * mb + g) ^ c)] = acc[mb];
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

// The splits of one query row: a workgroup, whose threads take 4 channels of every PARTS-th split.
template <int D>
__global__ __launch_bounds__(256) void mx_merge_kernel(const MxAttn a) {
  constexpr int UNITS = D / 4, PARTS = 256 / UNITS;
  __shared__ f4 sum[PARTS][UNITS];
  __shared__ float sum_l[PARTS], top[4];
  const int rows = a.L * a.G;
  const int r = (int)(blockIdx.x % rows);
  const int64_t kvrow = blockIdx.x / rows;
  const int b = (int)(kvrow / a.Hkv), hk = (int)(kvrow % a.Hkv);
  const int tile = r / 16, i = r / a.G, head = hk * a.G + (r - i * a.G);
  const MxRows n = mx_rows(a, kvrow, b);
  const bool live = i < n.queries;
  const int parts = live ? (mx_entries(a, n, tile * 16, 16) + a.chunk - 1) / a.chunk : 0;
  const int64_t first = (kvrow * a.tiles + tile) * a.splits * 16 + (r & 15);
  float M = M_NONE;
  for (int s = threadIdx.x; s < parts; s += 256) M = fmaxf(M, a.ws_m[first + (int64_t)s * 16]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const int u = threadIdx.x % UNITS, part = threadIdx.x / UNITS;
  float L = 0.f;
  f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = part; s < parts; s += PARTS) {
    const int64_t slot = first + (int64_t)s * 16;
    const float wgt = __builtin_amdgcn_exp2f(a.ws_m[slot] - M);
    L += wgt * a.ws_l[slot];
    o += *reinterpret_cast<const f4*>(a.ws_acc + slot * D + 4 * u) * wgt;
  }
  sum[part][u] = o;
  if (u == 0) sum_l[part] = L;
  __syncthreads();
  if (part != 0) return;
#pragma unroll
  for (int p = 1; p < PARTS; ++p) { o += sum[p][u]; L += sum_l[p]; }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  float out[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) out[q] = o[q] * inv;
  store_out4(a, b * a.osb + i * a.ost + head * a.osh + 4 * u, out);
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
  if (a.D == 128) f32 ? launch_rows<128, true>(a, stream) : launch_rows<128, false>(a, stream);
  else f32 ? launch_rows<64, true>(a, stream) : launch_rows<64, false>(a, stream);
  if (a.splits > 1) {
    const dim3 grid((uint32_t)((int64_t)a.B * a.Hkv * a.L * a.G));
    if (a.D == 128) hipLaunchKernelGGL(mx_merge_kernel<128>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(mx_merge_kernel<64>, grid, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace iak
