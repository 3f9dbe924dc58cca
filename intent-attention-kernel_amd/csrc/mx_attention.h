// What the 4-bit cache's attention kernels share: how many tokens a query row sees and how
// many table entries a tile of rows has to walk, out of the lengths on the device; a row's
// query operand; the parts of the softmax; V's way through LDS.
#ifndef IAK_MX_ATTENTION_H
#define IAK_MX_ATTENTION_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak_device.h"
#include "mx_format.h"
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

// What a workgroup takes: entries e0 .. e0 + chunk - 1 of a tile of rows, part number `part` of
// the call's; `idle`: nothing.
struct MxPart { uint32_t kvrow; int tile, e0, chunk; uint32_t part; bool idle; };

// The KV rows turn fastest, so that the workgroups that read the same pages meet in one XCD's L2
// where the number of KV rows is a multiple of 8, and every XCD has its share of each split and
// tile where lengths differ; those that see most start first. (With the splits fastest, 4 x 1,024
// queries over 1,024 tokens took 85 us and take 58.)
__device__ __forceinline__ MxPart mx_fixed_part(const MxAttn& a) {
  const uint32_t kvrows = (uint32_t)a.B * a.Hkv, rest = blockIdx.x / kvrows;
  MxPart p;
  p.kvrow = blockIdx.x - rest * kvrows;
  const int split = (int)(rest / a.tiles);
  p.tile = a.tiles - 1 - (int)(rest - (uint32_t)split * a.tiles);
  p.e0 = split * a.chunk;
  p.chunk = a.chunk;
  p.part = (p.kvrow * a.tiles + p.tile) * a.splits + split;
  p.idle = false;
  return p;
}

// Sum over the wave's lanes up to this one.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// Lengths are known on the device alone: every wave works out for itself the least chunk with
// which all tiles' chunks are no more than a.shares, and which of them is its workgroup's; RUNS:
// each XCD takes a run of them. `UNIT`: entries that a workgroup takes at a step.
// 16 heads over 4 of 128: 512, 16, 16 and 16 queries over 8,000, 500, 500 and 500 tokens 63 us, and
// 144 in fixed parts; 8 heads over one, 3 sequences of up to 1,000 queries over up to 8,000 tokens 95
// and 132, of equal lengths 140 and 134. With head_dim 64 one round
// only: 5 x 509 queries over 4,000 in two 66, fixed 59. Short decode rows lose what the working out
// takes (13 of up to 8,191 tokens: 19.7 us and 18.4).
template <int UNIT, bool RUNS> __device__ __forceinline__ MxPart mx_shared_part(const MxAttn& a) {
  constexpr int MOST = MX_SHARED_TILES / 64;
  const int lane = threadIdx.x & 63;
  const int all = a.B * a.Hkv * a.tiles, per = (all + 63) >> 6;    // tiles, and of a lane: a run
  int units[MOST], own = 0;
  uint32_t kv = (uint32_t)(lane * per) / (uint32_t)a.tiles, b = kv / (uint32_t)a.Hkv;   // of the lane's tile, counted up from here
  int tile = lane * per - (int)kv * a.tiles, hk = (int)(kv - b * (uint32_t)a.Hkv);
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    units[j] = 0;
    if (j < per && lane * per + j < all) {
      const MxRows n = mx_rows(a, kv, (int)b);
      units[j] = (mx_entries(a, n, tile * a.tile_rows, a.tile_rows) + UNIT - 1) / UNIT;
      own += units[j];
      if (++tile == a.tiles) {
        tile = 0;
        ++kv;
        if (++hk == a.Hkv) { hk = 0; ++b; }
      }
    }
  }
  const int total = __builtin_amdgcn_readlane(wave_scan(own), 63);
  auto chunks = [&](int x, int size) { return (int)((uint32_t)(x + size - 1) / (uint32_t)size); };
  auto count = [&](int size) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < MOST; ++j) if (j < per) n += chunks(units[j], size);
    return n;
  };
  // total / shares chunks are too few and total / (shares - tiles) enough
  int size = (total + a.shares - 1) / a.shares, enough = (total + a.shares - all - 1) / (a.shares - all);
  size = size < 1 ? 1 : size;
  int mine = count(size), upto = wave_scan(mine), parts = __builtin_amdgcn_readlane(upto, 63);
  if (parts > a.shares) {                                          // rows of one length are done here
    ++size;
    while (size < enough) {
      const int mid = (size + enough) >> 1;
      if (__builtin_amdgcn_readlane(wave_scan(count(mid)), 63) <= a.shares) enough = mid;
      else size = mid + 1;
    }
    mine = count(size);
    upto = wave_scan(mine);
    parts = __builtin_amdgcn_readlane(upto, 63);
  }
  const int run = (parts + 7) >> 3, part = RUNS ? (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
  MxPart p;
  p.idle = (RUNS && (int)(blockIdx.x >> 3) >= run) || part >= parts;
  if (p.idle) return p;
  const uint64_t has = __builtin_amdgcn_ballot_w64(part < upto);
  const int owner = __builtin_ctzll(has);                          // the first lane whose run ends behind it
  int before = upto - mine, at = 0, first = before, n = 0;
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int c = j < per ? chunks(units[j], size) : 0;
    if (before <= part) { at = j; first = before; n = c; }
    before += c;
  }
  const int t = owner * per + __builtin_amdgcn_readlane(at, owner);
  first = __builtin_amdgcn_readlane(first, owner);
  n = __builtin_amdgcn_readlane(n, owner);
  p.kvrow = (uint32_t)(t / a.tiles);
  p.tile = t - (int)p.kvrow * a.tiles;
  p.chunk = size * UNIT;
  p.e0 = (part - first) * p.chunk;
  p.part = (uint32_t)part;
  if (part == first && threadIdx.x == 0) a.ws_parts[t] = int2{first, n};
  return p;
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

// A lane's scale bytes come as the aligned four they are among: a byte loaded alone is zero-
// extended where the loop turns, and that waits for loads that the next round is meant to await.
template <int D> __device__ __forceinline__ uint32_t scale_word(const uint8_t* page_scales, int c, int g) {
  return reinterpret_cast<const uint32_t*>(page_scales)[(c * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK) >> 2];
}
template <int D> __device__ __forceinline__ uint32_t own_scale(uint32_t word, int c, int g) {
  return __builtin_amdgcn_ubfe(word, 8 * ((c * (D / MX_BLOCK) + g * (D / 4) / MX_BLOCK) & 3), 8);
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
// element of the row in [2^14, 2^15), split in two for float32. What float16 cannot hold below
// that is rounded to its smallest step, 2^-24: off by 2^-25, 2^-39 of the row's largest, and not
// at all for 16-bit elements of 2^-28 of it or more. A scale per 32 channels would lose nothing,
// but would have to go into K's (2^-24 to 49,152 already), which float16 cannot hold either. Returns the positive factor that
// makes base-2 scores of the products. (A negative scale turns the query's sign; where the factor
// would vanish the scores do: query 0, factor 1. A row that is not finite is NaN, factor 1: NaN
// scores for the tokens that it sees, and none if it sees none.)
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
      const float v = !fine ? __builtin_nanf("") : none ? 0.f : sign * __builtin_ldexpf(x[8 * s + j], 14 - e);
      qhi[s][j] = (_Float16)v;
      if constexpr (QF32) qlo[s][j] = (_Float16)(v - (float)qhi[s][j]);
    }
  return none ? 1.f : mult;
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
// 16-bit queries go without that second part: weights of 11 bits err by as much as a float16
// output's own rounding, and below a bfloat16 one's. Against 64 bits (relative, 32 x 32,768 tokens |
// 2,048 queries over 8,192, head_dim 128) float16 outputs are off by 2.5e-4 | 2.6e-4, with both
// parts by 2.1e-4 | 2.1e-4, bfloat16 ones by 1.7e-3 either way; both parts take 195 us for 192 |
// 359 us for 257 (13 ragged rows 19.7 for 18.4, 5 ragged prompts of head_dim 64 75 for 58).
// The rows kernel sums the weights as they are, the prompt kernel (on the matrix cores) as rounded.
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

}  // namespace iak

#endif
