// Attention over the microscaled 4-bit cache for many query rows of a KV head (prompt chunks),
// for gfx950. The mathematics, the lanes' parts and the softmax are the rows kernel's
// (mx_attention.hip); what differs is who reads the cache.
//
// A workgroup takes 32 rows a wave: 256 rows in eight waves (16-bit queries), or 128 in four. All walk the same
// tokens, 64 (four pages) a step. Each wave converts its share of the next step's pages (one
// page of K or of V in eight waves, of both in four) into LDS, from where all read them: two
// buffers, one barrier a step. The sum of the weights is a product with ones on the matrix cores.
//
// 2,048 queries x 32 heads x 8 KV heads over 8,192 tokens, head_dim 128, float16, causal: 256 us
// in tiles of 256, 940 TFLOP/s of the products (a matrix product of 8,192 cubed reaches 1,176);
// 267 in tiles of 128, where 16 x 512 queries over 512 tokens take 80 and in tiles of 256 91 (two
// workgroups a CU fill each other's waits). The matrix cores are busy for 46 % of the time and
// the vector instructions (softmax, conversion) for 53 %; the two overlap little. Tiles of 128 took
// 279 us before the workgroups' order was by KV row; of these went, taken out on trial: the reads
// of LDS 69, then the conversion 13; the exponentials 7, the value products 18, the score products
// 0. Slower were one half's products ahead of the other's softmax (330), half the waves a barrier
// later with their value products (268), operands read ahead (340), tiles of 64 rows and wave
// priorities (285); with head_dim 64, where this call takes 180, four tiles of rows a wave (261)
// and four waves a SIMD (261). There the matrix cores are busy for 35 % of the time and the vector
// instructions for 66 % (7.1 a score, 1 of them the exponential): one after the other they fill it,
// and if they overlapped whole, the vector instructions' 119 us would be left.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "mx_attention.h"

namespace iak {

namespace {

constexpr int RT = 2;               // tiles of 16 rows a wave

template <int D, bool QF32, int NW>
__global__ __launch_bounds__(64 * NW, 2) void mx_chunk_kernel(const MxAttn a) {
  static_assert(NW == 4 || NW == 8, "a wave converts a page of K and of V, or one of the two");
  constexpr int OWN = 8 / NW, BM = 16 * RT * NW;
  __shared__ u4 tiles[2][2][4][PS * D / 8];                      // [buffer][K, V][page]
  __shared__ u4 nan_in[2][2];                                    // a word a page: its tokens with a NaN block
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const MxPart part = a.shares ? mx_shared_part<4, true>(a) : mx_fixed_part(a);
  if (part.idle) return;                                         // uniform, as below
  const int64_t kvrow = part.kvrow;
  const int tile = part.tile;
  const int b = (int)(part.kvrow / (uint32_t)a.Hkv), hk = (int)(part.kvrow - (uint32_t)b * a.Hkv);
  const MxRows n = mx_rows(a, kvrow, b);
  const int entries = mx_entries(a, n, tile * BM, BM);
  const int e0 = part.e0, e1 = e0 + part.chunk < entries ? e0 + part.chunk : entries;
  if (e0 > 0 && e0 >= e1) return;                                // the merge does not look at it

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

  // this wave's page of a step, of K and V or of one of them: loaded a step ahead, converted
  // into LDS during the step before
  const int own = w & 3, side = w >> 2;
  uint32_t codes[OWN][D / 32], scales[OWN];
  auto load_page = [&](int id) __attribute__((always_inline)) {
    const int64_t p = id < 0 ? 0 : id;
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const bool v = OWN == 2 ? o == 1 : side == 1;
      const uint8_t* at = (v ? a.v_codes : a.k_codes) + p * (PS * D / 2) + c * (D / 2) + g * (D / 8);
      if constexpr (D == 128) {
        const u4 x = *reinterpret_cast<const u4*>(at);
#pragma unroll
        for (int i = 0; i < 4; ++i) codes[o][i] = x[i];
      } else {
        const u2 x = *reinterpret_cast<const u2*>(at);
#pragma unroll
        for (int i = 0; i < 2; ++i) codes[o][i] = x[i];
      }
      scales[o] = scale_word<D>((v ? a.v_scales : a.k_scales) + p * (PS * D / MX_BLOCK), c, g);
    }
  };
  auto convert = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int s = OWN == 2 ? o : side;
      const uint32_t byte = own_scale<D>(scales[o], c, g);
      const float scale = mx_scale(byte);
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t x[4];
        mx8_to_f16(codes[o][j], scale, x);
        tiles[buf][s][own][v_chunk<D>(c, g * (D / 32) + j)] = u4{x[0], x[1], x[2], x[3]};
      }
      const uint64_t bad = __builtin_amdgcn_ballot_w64(byte == MX_SCALE_NAN);
      reinterpret_cast<uint32_t*>(&nan_in[buf][s])[own] = (uint32_t)(bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xFFFFu;
    }
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
  auto step = [&](int buf, int e) __attribute__((always_inline)) {
    f4 s[RT][4];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int p = 0; p < 4; ++p) s[t][p] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const h8 ka = __builtin_bit_cast(h8, tiles[buf][0][p][v_chunk<D>(c, g * (D / 32) + j)]);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qhi[t][j], s[t][p], 0, 0, 0);
          if constexpr (QF32) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qlo[t][j], s[t][p], 0, 0, 0);
        }
      }
    const u4 bad = nan_in[buf][0] | nan_in[buf][1];
    const int id[4] = {page(k), page(k + 1), page(k + 2), page(k + 3)};
    convert(buf ^ 1);
    load_page(page(k + 8 + own));
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
        const h8 va = values_back<D>(tiles[buf][1][2 * h], tiles[buf][1][2 * h + 1], mb, c, g);
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
    load_page(page(own));
    convert(0);
    load_page(page(4 + own));
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
    if (a.parted) {
      const int64_t slot = (int64_t)part.part * BM + (w * RT + t) * 16 + c;
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

template <int D, bool QF32> void launch_chunk(const MxAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items);
  if constexpr (!QF32) {
    if (a.tile_rows == 256) { hipLaunchKernelGGL((mx_chunk_kernel<D, false, 8>), grid, dim3(512), 0, stream, a); return; }
  }
  hipLaunchKernelGGL((mx_chunk_kernel<D, QF32, 4>), grid, dim3(256), 0, stream, a);
}

}  // namespace

void launch_mx_chunk(const MxAttn& a, hipStream_t stream) {
  const bool f32 = a.q_dtype == IAK_DTYPE_F32;
  if (a.D == 128) f32 ? launch_chunk<128, true>(a, stream) : launch_chunk<128, false>(a, stream);
  else f32 ? launch_chunk<64, true>(a, stream) : launch_chunk<64, false>(a, stream);
}

}  // namespace iak
