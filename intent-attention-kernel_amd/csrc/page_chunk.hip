// Attention over pages of mixed precision for many query rows of a KV head (prompt chunks), for
// gfx950. The mathematics, the lanes' parts and the softmax are the rows kernel's (page_rows.hip);
// what differs is who reads the cache.
//
// A workgroup takes 16 RT rows a wave. All its waves walk the same tokens, 64 (four pages) a
// step; each puts its share of the next step's pages into LDS as operands, from where all read them: two buffers,
// one barrier a step.
//
// What bounds it: nothing alone. 2,048 queries over 8,192 tokens of float16 pages (32 heads over 8 of 128) take
// 250 to 262 us from box to box, 918 to 960 TFLOP/s, where a large product reaches 1,338: the matrix cores are busy 44 % of the cycles, the vector
// instructions (softmax) 26 %, the LDS 28 %, and two waves a SIMD do not fill each other's waits. Over 16,384
// tokens of mixed pages, two sequences: 1.74 ms, 582 TFLOP/s; the vector instructions (codes to float16, multipliers in
// the softmax) and the wide pages' second products take as long as the first products. Tried and slower: the
// workgroup's halves in turns, one's products beside the other's softmax (chunks of mixed pages 2,270 us for 1,700,
// float16 ones 291 for 282), convert() behind the softmax (1,684 for 1,692: no difference).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "page_attention.h"

namespace iak {

namespace {

// N operands from LDS and what each is multiplied by, the operands read ahead of their products, for
// a read takes as long as several. (Left to itself the compiler reads each just before its own, which took 292 us
// for 282 of float16 chunks. Two, four and six ahead: float16 chunks as above 248, 251 and 250 us, mixed ones 1,751,
// 1,739 and 1,745: four for these.)
template <int N, int AHEAD_OF, typename Read, typename Multiply> __device__ __forceinline__ void products(Read&& read, Multiply&& multiply) {
  constexpr int A = N < AHEAD_OF ? N : AHEAD_OF;
  h8 x[A];
#pragma unroll
  for (int i = 0; i < A; ++i) x[i] = read(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    multiply(i, x[i % A]);
    if (i + A < N) x[i % A] = read(i + A);
  }
  __builtin_amdgcn_sched_barrier(0);
}

template <int D, bool QF32, int NW, int RT, int KIND>
__global__ __launch_bounds__(64 * NW, 2) void page_chunk_kernel(const PageAttn a) {
  static_assert(NW == 4 || NW == 8, "pieces of pages are shared out");
  constexpr bool WIDE = KIND == PAGES_ALL, SCALED = KIND != PAGES_F16;
  constexpr int FEED = 4;
  constexpr int QUARTERS = D / 32, OWN = 8 * QUARTERS / NW;      // pieces (64 chunks) a page, and of a wave a step
  constexpr int BM = 16 * RT * NW, PAGE = PS * D / 8;   // 16-byte units of a tile
  __shared__ u4 tiles[2][2][4][PAGE];                            // [buffer][K, V][page]
  __shared__ u4 rest[WIDE ? 2 : 1][2][4][WIDE ? PAGE : 1];       // of wide pages: what their tiles leave
  __shared__ u4 none[WIDE ? PAGE : 1];                           // zeros
  __shared__ Ahead<KIND> table;
  __shared__ int special;                                        // bit 0: V has infinite or NaN values, bit 1: a sum has
  __shared__ int power_top;                                      // the highest E so far, which is seldom asked for
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
  if constexpr (WIDE) {
    for (int i = threadIdx.x; i < PAGE; i += 64 * NW) none[i] = u4{0u, 0u, 0u, 0u};
  }

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

  // Wave 0 looks up a block of 64 entries in three steps of the walk, what waits for what a step apart.
  auto look_up = [&](int k) {
    const PageAttn& b = arguments();
    const int page = entry_page(b, raw_entry(b.table + kvrow * b.W, e0 + k, e1));
    put_ahead<D, KIND>(table, b, k, page_tag<KIND>(b, page, raw_tag(b, page)));
  };
  if (w < 2) look_up(64 * w + lane);
  if (threadIdx.x == 0) { special = 0; power_top = -NO_POWER; }
  __syncthreads();
  int ahead = 0, ahead_tag = 0;
  auto look_ahead = [&](int k) __attribute__((always_inline)) {  // k: entry of the walk, a multiple of 4
    if ((k & 15) != 0 || w != 0 || k < 64) return;               // two blocks are there at first
    const int stage = (k >> 4) & 3, e = (k & ~63) + 64 + lane;   // the block after the one at hand
    const PageAttn& b = arguments();
    if (stage == 0) ahead = raw_entry(b.table + kvrow * b.W, e0 + e, e1);
    else if (stage == 1) {
      ahead = entry_page(b, ahead);
      ahead_tag = raw_tag(b, ahead);
    } else if (stage == 2) put_ahead<D, KIND>(table, b, e, page_tag<KIND>(b, ahead, ahead_tag));
  };
  auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };

  bool careful = false;                                          // V's infinite and NaN values become zeros

  // This wave's pieces of a step's pages: loaded a step ahead, put into LDS during the step before. Piece o of
  // wave w is number w + NW o of (page, side, quarter).
  auto page_of = [&](int o) { return NW <= 2 * QUARTERS ? NW * o / (2 * QUARTERS) : 2 * o + w / (2 * QUARTERS); };
  auto side_of = [&](int o) { return NW <= QUARTERS ? NW * o / QUARTERS & 1 : w / QUARTERS & 1; };
  const int f = w % QUARTERS * 64 + lane, place = v_chunk<D>(f / (D / 8), f % (D / 8));
  u4 raw[OWN];
  auto tags_of = [&](int k) { return uniform(*reinterpret_cast<const uint32_t*>(&table.tag[k & (AHEAD - 1)])); };   // of four pages
  // (What LDS has for all pieces is read before any is worked on: the tags' branches would have a read's
  // wait each.)
  auto load = [&](uint32_t tags, int k) __attribute__((always_inline)) {
    u2 at[OWN];
#pragma unroll
    for (int o = 0; o < OWN; ++o) at[o] = reinterpret_cast<const u2*>(&table.where[(k + page_of(o)) & (AHEAD - 1)])[side_of(o)];
#pragma unroll
    for (int o = 0; o < OWN; ++o)
      raw[o] = load_piece<D, KIND>((uint64_t)at[o][0] | (uint64_t)at[o][1] << 32, (tags >> (8 * page_of(o))) & 0xFFu, f);
  };
  const int quarter = f % (D / 8) / (D / 32);
  auto convert = [&](int buf, uint32_t tags, int k) __attribute__((always_inline)) {
    float s0[OWN], s1[OWN];
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int e = (k + page_of(o)) & (AHEAD - 1);
      s0[o] = SCALED ? reinterpret_cast<const float*>(&table.factors[side_of(o)][SCALED ? e : 0])[quarter] : 0.f;
      s1[o] = WIDE ? table.second[side_of(o)][WIDE ? e : 0] : 0.f;
    }
#pragma unroll
    for (int o = 0; o < OWN; ++o) {
      const int p = page_of(o), s = side_of(o);
      store_piece<D, KIND>(raw[o], (tags >> (8 * p)) & 0xFFu, s0[o], s1[o], tiles[buf][s][p], rest[WIDE ? buf : 0][s][p], place);
    }
    if (careful) {
#pragma unroll 1
      for (int o = 0; o < OWN; ++o)
        if (side_of(o) == 1 && __builtin_amdgcn_ballot_w64(clean_chunk(&tiles[buf][1][page_of(o)][place])) && lane == 0) special = 1;
    }
  };

  f4 acc[RT][D / 16], l[RT], s[RT][4];
  float lsum[RT], m[RT];
  h8 pb[RT][2], pl[RT][QF32 ? 2 : 1];
  int E = NO_POWER;
  const h8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
  auto wide = [&](uint32_t tags, int p) { return WIDE && wide_tag((int)((tags >> (8 * p)) & 0xFFu)); };

  // s = K Q^T of a step's tokens; its operand i is channels 8 (i / 4) .. of page i % 4
  auto read_k = [&](const u4 (&page)[PAGE], int j) __attribute__((always_inline)) {
    return __builtin_bit_cast(h8, page[v_chunk<D>(c, g * (D / 32) + j)]);
  };
  auto score = [&](int p, int j, const h8& k) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qhi[t][j], j == 0 ? f4{0.f, 0.f, 0.f, 0.f} : s[t][p], 0, 0, 0);
      if constexpr (QF32) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qlo[t][j], s[t][p], 0, 0, 0);
    }
  };
  auto scores_rest = [&](int buf, uint32_t tags) __attribute__((always_inline)) {
    if constexpr (WIDE) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        if (!wide(tags, p)) continue;
        products<D / 32, 4>([&](int j) __attribute__((always_inline)) { return __builtin_bit_cast(h8, rest[buf][0][p][v_chunk<D>(c, g * (D / 32) + j)]); },
                            [&](int j, const h8& k) __attribute__((always_inline)) {
#pragma unroll
          for (int t = 0; t < RT; ++t) s[t][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qhi[t][j], s[t][p], 0, 0, 0);
        });
      }
    }
  };
  // pb = weights of the scores of tokens 16 e ..; the sums so far follow the maximum
  auto softmax = [&](uint32_t tags, int k, int e) __attribute__((always_inline)) {
    int id[4];                                                   // -1: no page
#pragma unroll
    for (int p = 0; p < 4; ++p) id[p] = ((tags >> (8 * p)) & 0xFFu) == NO_PAGE ? -1 : 0;
    const uint32_t no_nan[4] = {0u, 0u, 0u, 0u};
    hide<4, RT>(s, no_nan, id, e, seen, least, g);
    if constexpr (SCALED) {
      const f4 kms = *reinterpret_cast<const f4*>(&table.km[k & (AHEAD - 1)]);
      const f4 vls = *reinterpret_cast<const f4*>(&table.vl[k & (AHEAD - 1)]);
      const f4 ivs = *reinterpret_cast<const f4*>(&table.iv[k & (AHEAD - 1)]);
      const float km[4] = {kms[0], kms[1], kms[2], kms[3]};
      float vl[4] = {vls[0], vls[1], vls[2], vls[3]}, out[4];
      raise_scaled<D, 4, RT>(s, km, mult, m, lsum, acc);
      int to = value_power<4>(vl, E);
      if (to != E) {                                             // uniform
        int highest = __builtin_amdgcn_readfirstlane(power_top);  // every wave's moves are the same, and leave the same here
        to = moved_power(to, E, highest);
        power_top = highest;
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[t][mb][q] = __builtin_ldexpf(acc[t][mb][q], E - to);
        E = to;
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        vl[p] -= (float)E;
        out[p] = __builtin_ldexpf(ivs[p], E);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) lsum[t] += soften_scaled<4>(s[t], km, vl, out, mult[t], m[t]);
    } else {
      raise<D, 4, RT>(s, mult, m, l, acc);
#pragma unroll
      for (int t = 0; t < RT; ++t) soften<4>(s[t], mult[t], m[t]);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        pb[t][h] = weights(s[t][2 * h], s[t][2 * h + 1]);
        if constexpr (QF32) pl[t][h] = weights_rest(s[t][2 * h], s[t][2 * h + 1], pb[t][h]);
      }
  };
  // acc += V^T pb of a step's tokens; its operand i is 16 channels of two pages
  auto value = [&](int i, const h8& v) __attribute__((always_inline)) {
    const int h = i / (D / 16), mb = i % (D / 16);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[t][h], acc[t][mb], 0, 0, 0);
      if constexpr (QF32) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl[t][h], acc[t][mb], 0, 0, 0);
    }
  };
  auto read_v = [&](int buf, int i) __attribute__((always_inline)) {
    const int h = i / (D / 16), mb = i % (D / 16);
    return values_back<D>(tiles[buf][1][2 * h], tiles[buf][1][2 * h + 1], mb, c, g);
  };
  auto weigh = [&]() __attribute__((always_inline)) {            // the weights' sum
    if constexpr (!SCALED) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[t][h], l[t], 0, 0, 0);
          if constexpr (QF32) l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pl[t][h], l[t], 0, 0, 0);
        }
    }
  };
  auto values_rest = [&](int buf, uint32_t tags) __attribute__((always_inline)) {
    if constexpr (WIDE) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool w0 = wide(tags, 2 * h), w1 = wide(tags, 2 * h + 1);
        if (!w0 && !w1) continue;
        const u4* p0 = w0 ? rest[buf][1][2 * h] : none;
        const u4* p1 = w1 ? rest[buf][1][2 * h + 1] : none;
        products<D / 16, FEED>([&](int mb) __attribute__((always_inline)) { return values_back<D>(p0, p1, mb, c, g); },
                               [&](int mb, const h8& v) __attribute__((always_inline)) {
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t][mb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[t][h], acc[t][mb], 0, 0, 0);
        });
      }
    }
  };
  constexpr int ALL = D / 8;                                     // operands of either side
  auto scores = [&](int buf, uint32_t tags) __attribute__((always_inline)) {
    products<ALL, FEED>([&](int i) __attribute__((always_inline)) { return read_k(tiles[buf][0][i % 4], i / 4); },
                        [&](int i, const h8& x) __attribute__((always_inline)) { score(i % 4, i / 4, x); });
    scores_rest(buf, tags);
  };
  auto values = [&](int buf, uint32_t tags) __attribute__((always_inline)) {
    weigh();
    products<ALL, FEED>([&](int i) __attribute__((always_inline)) { return read_v(buf, i); },
                        [&](int i, const h8& x) __attribute__((always_inline)) { value(i, x); });
    values_rest(buf, tags);
  };
  uint32_t now = 0, soon = 0;                                    // tags of this step's pages and of the next's
  int k = 0;                                                     // number of its first entry in the part
  auto step = [&](int buf, int e) __attribute__((always_inline)) {
    const uint32_t later = tags_of(k + 8);
    scores(buf, now);
    convert(buf ^ 1, soon, k + 4);
    load(later, k + 8);
    look_ahead(k);
    softmax(now, k, e);
    values(buf, now);
    k += 4;
    now = soon;
    soon = later;
    __syncthreads();                                             // this buffer is free, the other one is whole
  };
  // A token that a row does not see weighs nothing, and 0 times infinity is NaN: a walk that ends in such
  // sums is made again with zeros in their place.
  for (int walk = 0; walk < 2; ++walk) {
    E = NO_POWER;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      m[t] = M_NONE;
      lsum[t] = 0.f;
      l[t] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) acc[t][mb] = f4{0.f, 0.f, 0.f, 0.f};
    }
    if (e0 < e1) {                                               // uniform
      k = 0;
      now = tags_of(0);
      soon = tags_of(4);
      load(now, 0);
      convert(0, now, 0);
      load(soon, 4);
      __syncthreads();
      for (int e = e0; e < e1; e += 8) {
        step(0, e);
        if (e + 4 < e1) step(1, e + 4);
      }
    }
    if (careful) break;
    float sum = 0.f;                                             // NaN once anything is not finite
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum = __builtin_fmaf(acc[t][mb][q], 0.f, sum);
    if (__builtin_amdgcn_ballot_w64(!(sum == 0.f)) && lane == 0) special = 2;
    __syncthreads();
    if (special == 0) break;                                     // uniform
    __syncthreads();
    careful = true;
    if (threadIdx.x == 0) { special = 0; power_top = -NO_POWER; }
    if (w < 2) look_up(64 * w + lane);
    __syncthreads();
  }

  // what V has of infinite and NaN values, in a second walk
  if (special) {                                                 // uniform: written before the last barrier, by a careful walk
    uint16_t* aside = reinterpret_cast<uint16_t*>(&tiles[1][0][0][0]);
    uint32_t* any = reinterpret_cast<uint32_t*>(&tiles[1][1][0][0]);
    Seen16 odd[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) odd[t] = Seen16{0u, 0u};
    for (int e = e0; e < e1; e += 4) {
      __syncthreads();
      if (w < 4) {
        const PageAttn& b = arguments();
        const PageEntry x = page_entry<D, KIND>(b, b.table + kvrow * b.W, e + w, e1);
        const int id = (int)uniform((uint32_t)x.id), tag = (int)uniform((uint32_t)x.tag);
        PageRaw<D> r;
        load_page<D, KIND>(r, b, true, id, tag, lane);
        const bool bad = store_page<D, KIND>(r, id, tag, u2f(uniform(f2u(x.vf))), tiles[0][0][w], rest[0][0][w], lane);
        const bool some = __builtin_amdgcn_ballot_w64(bad) != 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (some) put_aside<D>(tiles[0][0][w], aside + w * PAGE, lane);
        if (lane == 0) any[w] = some;
      }
      __syncthreads();
      for (int p = 0; p < 4; ++p) {
        if (uniform(any[p]) == 0) continue;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int left = seen[t] - (e + p) * PS;
          remember<D>(odd[t], aside + p * PAGE, left < PS ? left : PS, g);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) bring_back<D>(acc[t], odd[t]);
  }

  const PageAttn& z = arguments();
  const int all = z.L * z.G;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = tile * BM + (w * RT + t) * 16 + c, i = r / z.G, head = hk * z.G + (r - i * z.G);
    float sum;
    if constexpr (SCALED) sum = xsum16_32(lsum[t]);
    else sum = l[t][0];
    if (r >= all) continue;
    if (z.parted) {
      const int64_t slot = (int64_t)part.part * BM + (w * RT + t) * 16 + c;
      const int by = SCALED ? sum_power(sum, E) : 0;
      if (g == 0) { z.ws_m[slot] = m[t] + (float)by; z.ws_l[slot] = __builtin_ldexpf(sum, -by); }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        f4 x = acc[t][mb];
        if constexpr (SCALED) {
#pragma unroll
          for (int q = 0; q < 4; ++q) x[q] = __builtin_ldexpf(x[q], E - by);
        }
        *reinterpret_cast<f4*>(z.ws_acc + slot * D + 16 * mb + 4 * g) = x;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;           // NaN stays
      const int64_t at = b * z.osb + i * z.ost + head * z.osh + 4 * g;
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        float o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float x = acc[t][mb][q] * inv;
          o[q] = i < n.queries ? (SCALED ? __builtin_ldexpf(x, E) : x) : 0.f;
        }
        store_out4(z, at + 16 * mb, o);
      }
    }
  }
}

template <int D, bool QF32, int NW, int RT> void launch_tiles(const PageAttn& a, hipStream_t stream) {
  const dim3 grid((uint32_t)a.items), block(64 * NW);
  if (a.kind == PAGES_F16) hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_F16>), grid, block, 0, stream, a);
  else if (a.kind == PAGES_BYTE) hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_BYTE>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((page_chunk_kernel<D, QF32, NW, RT, PAGES_ALL>), grid, block, 0, stream, a);
}

template <int D> void launch_chunk(const PageAttn& a, hipStream_t stream) {
  if (a.q_dtype == IAK_DTYPE_F32) launch_tiles<D, true, 8, 1>(a, stream);
  else if (a.tile_rows == 256) launch_tiles<D, false, 8, 2>(a, stream);
  else launch_tiles<D, false, 4, 2>(a, stream);
}

}  // namespace

void launch_page_chunk(const PageAttn& a, hipStream_t stream) {
  if (a.D == 128) launch_chunk<128>(a, stream);
  else launch_chunk<64>(a, stream);
}

}  // namespace iak
