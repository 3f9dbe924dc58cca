// A beam search's choice on gfx950: of each request's beams x vocabulary the `count` best
// continuations,
//   candidate (k, v) = scores[k] + logits[k, v] - log sum_u exp(logits[k, u]),
// best first, ties to the lowest beam, of one beam's to the largest logit, then to the lowest token.
//
//   beam_part_kernel   a wave streams a segment of one row of logits, once: its sum of exponentials,
//                      and its `count` best by (logit, index), which no offset of the row changes.
//                      What is below a running threshold costs one comparison; the rest goes
//                      to a list in LDS, which is ranked when it is full and at the end.
//   beam_merge_kernel  a workgroup per request: the rows' normalisers out of the segments' sums,
//                      and the best of the segments' lists, one after the other from their heads.
//
// Which token comes first is a whole number, so candidates of different beams have to be compared
// to more than 32 bits: with offsets off by 2^-24 of 30 or so, two in some 10^5 neighbours would
// change places. exp(x) = 2^(k/32) e^r with |r| <= ln 2 / 64: the table's 2^(k/32) and the sum in
// 64 bits, r and e^r - 1 in 32, off by some 2^-31, so that a normaliser is off by some 1e-9.
//
// What bounds it: the logits are read once (64 x 8 x 131,072 in bfloat16, a tenth of the beams at their end: 121 MB,
// 24 us at a copy's rate), with 21 vector instructions a logit (an exponential to 1e-9 is 15 of them), 37 us of
// the card's; the part kernel takes 54, what is left being its first group (nothing to overlap with), the list's
// upkeep and the ends of the waves. The merge takes 8.6 (16 steps of some 0.1 us, and the loads and
// logarithms before them); two requests x 4 beams x 32,000: 7.2 + 5.9 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "iak_device.h"
#include "step_internal.h"

namespace iak {

namespace {

constexpr int BEAM_THREADS = 256, BEAM_WAVES = BEAM_THREADS / 64;

struct BeamArgs {
  int B, K, V, n;
  const void* logits; int64_t sb, sk;
  const float* scores;
  const uint8_t* finished;
  int end;
  float* out_scores; int32_t* out_parents; int32_t* out_tokens;
  int segments, per;        // segments a row (a wave each), groups of logits a segment
  double2* norms;           // [rows, segments] base and sum of exp(logit - base); base NaN: a logit is NaN or +inf
  uint64_t* best;           // [rows, segments, n] keys, best first; 0: none
};

// An order of floats as unsigned numbers; both zeros are one value.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = f2u(x + 0.f);
  return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return u2f(o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }

// Whether a beam reads its logits: it is not at its end and its score is a number.
__device__ __forceinline__ bool beam_live(const BeamArgs& a, int64_t row, float score) {
  return !(a.finished && a.finished[row]) && __builtin_isfinite(score);
}

// The largest of the wave's values, in every lane.
__device__ __forceinline__ uint32_t wave_most(uint32_t x) {
  auto step = [&](uint32_t y) { x = y > x ? y : x; };
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, true));
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false));   // row_bcast:15 into rows 1 and 3
  step((uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false));   // row_bcast:31 into rows 2 and 3
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

// A number that at least n of the wave's values reach, and as few more as there are (0: fewer do). `low`:
// one that n of them reach, from which on it is looked for.
__device__ __forceinline__ uint32_t wave_nth(uint32_t x, int n, uint32_t low = 0) {
  const uint32_t high = wave_most(x);
  if (low == high) return low;
  const int top = 31 - __builtin_clz(low ^ high);                // they differ from this bit on
  uint32_t least = top == 31 ? 0 : low >> (top + 1) << (top + 1);
#pragma unroll 1
  for (uint32_t bit = 1u << top; bit; bit >>= 1) {
    const int reach = __builtin_popcountll(__builtin_amdgcn_ballot_w64(x >= (least | bit)));
    if (reach >= n) least |= bit;
    if (reach == n) break;
  }
  return least;
}

// 8 logits as they lie, and one of them.
typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> struct Raw8 { any4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ float value(const Raw8<T>& r, int j);
template <> __device__ __forceinline__ float value<float>(const Raw8<float>& r, int j) { return u2f(r.w[j / 4][j % 4]); }
template <> __device__ __forceinline__ float value<_Float16>(const Raw8<_Float16>& r, int j) {
  const uint16_t h = (uint16_t)(r.w[0][j / 2] >> (16 * (j % 2)));
  return (float)__builtin_bit_cast(_Float16, h);
}
template <> __device__ __forceinline__ float value<__bf16>(const Raw8<__bf16>& r, int j) {
  return u2f(j % 2 ? r.w[0][j / 2] & 0xFFFF0000u : r.w[0][j / 2] << 16);
}
// Numbers of logits go up to 2^31 and a group past it: unsigned.
template <typename T> __device__ __forceinline__ Raw8<T> load_raw8(const T* row, uint32_t v, uint32_t V) {
  Raw8<T> r;
  if (v + 8 <= V) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(row + v) + i);
    return r;
  }
  // past the row: -inf, which adds nothing to a sum
  constexpr int BITS = 8 * sizeof(T);
  constexpr uint32_t NONE = __is_same(T, float) ? 0xFF800000u : __is_same(T, _Float16) ? 0xFC00u : 0xFF80u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i)
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 32 / BITS; ++j) {
        const uint32_t u = v + (4 * i + d) * (32 / BITS) + j;
        uint32_t bits = NONE;
        if (u < V) {
          if constexpr (BITS == 32) bits = __builtin_bit_cast(uint32_t, row[u]);
          else bits = __builtin_bit_cast(uint16_t, row[u]);
        }
        w |= bits << (BITS * j & 31);
      }
      r.w[i][d] = w;
    }
  return r;
}

// exp(x) added up in 64 bits, for x up to ADD_EXP_MOST (from some 710 on the exponent's bits would run over, with no
// sign of it in the sum) and down to -600 (below that: as there). k = 32 x / ln 2 rounded, as the
// low bits of a float past 2^23; the table's entry j has -j 2^15 in its high word, so that k 2^15
// makes it 2^(k/32).
constexpr float ADD_EXP_MOST = 600.f;
__device__ __forceinline__ void add_exp(float x, const uint2* table, double& sum) {
  constexpr float TURN = 46.166241308446828f, MAGIC = 12582912.f;   // 32 / ln 2, 1.5 2^23
  constexpr double STEP = 0.021660849392498290;                     // ln 2 / 32
  constexpr float STEP_HIGH = (float)STEP, STEP_LOW = (float)(STEP - (double)STEP_HIGH);
  x = u2f(f2u(x) < 0xC4160000u ? f2u(x) : 0xC4160000u);             // no less than -600, in one instruction
  const float m = __builtin_fmaf(x, TURN, MAGIC), k = m - MAGIC;
  const float r = __builtin_fmaf(-k, STEP_LOW, __builtin_fmaf(-k, STEP_HIGH, x));
  const float q = r * __builtin_fmaf(r, __builtin_fmaf(r, 1.f / 6, 0.5f), 1.f);   // r^4 / 24 is 2^-30 at most
  const uint2 e = table[f2u(m) & 31];
  const uint64_t bits = ((uint64_t)(e.y + (f2u(m) << 15)) << 32) | e.x;
  const double t = __builtin_bit_cast(double, bits);
  sum = __builtin_fma(t, (double)q, sum) + t;
}

// What a wave's lanes wrote to LDS is there for its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

constexpr int BEAM_LIST = 256;   // keys of a wave's list

// The list's n best, in order, to its front; `reach`: a number that n of its logits reach, in
// `ordered`, so that only those are compared with each other. -> how many it holds then.
__device__ __forceinline__ int rank_list(uint64_t* list, int count, int n, uint32_t reach, int lane) {
  constexpr int SETS = BEAM_LIST / 64;
  uint64_t own[SETS];
  wave_sync();
#pragma unroll
  for (int i = 0; i < SETS; ++i) own[i] = lane + 64 * i < count ? list[lane + 64 * i] : 0;
  wave_sync();
  int left = 0;
#pragma unroll
  for (int i = 0; i < SETS; ++i) {
    const bool stays = own[i] != 0 && (uint32_t)(own[i] >> 32) >= reach;
    const uint64_t staying = __builtin_amdgcn_ballot_w64(stays);
    if (stays) list[left + __builtin_amdgcn_mbcnt_hi((uint32_t)(staying >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)staying, 0))] = own[i];
    left += __builtin_popcountll(staying);
  }
  wave_sync();
  int rank[SETS];
#pragma unroll
  for (int i = 0; i < SETS; ++i) {
    own[i] = lane + 64 * i < left ? list[lane + 64 * i] : 0;
    rank[i] = 0;
  }
  for (int i = 0; i < left; ++i) {                               // keys differ
    const uint64_t key = list[i];
    rank[0] += key > own[0];
    if (left > 64) {
#pragma unroll
      for (int s = 1; s < SETS; ++s) rank[s] += key > own[s];
    }
  }
  wave_sync();
#pragma unroll
  for (int i = 0; i < SETS; ++i)
    if (own[i] != 0 && rank[i] < n) list[rank[i]] = own[i];
  wave_sync();
  return left < n ? left : n;
}

// The number that stands for at least `reach` in the order.
__device__ __forceinline__ float level(uint32_t reach) { return reach > 0x007FFFFFu ? unordered(reach) : -__builtin_inff(); }

template <typename T, int PER>
__global__ __launch_bounds__(BEAM_THREADS, 4) void beam_part_kernel(const BeamArgs a) {
  __shared__ uint2 table[32];
  __shared__ uint64_t lists[BEAM_WAVES][BEAM_LIST];
  __shared__ __attribute__((aligned(16))) Raw8<T> listed[BEAM_WAVES][PER][64];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  if (t < 32) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, exp2(t * 0.03125));
    table[t] = make_uint2((uint32_t)bits, (uint32_t)(bits >> 32) - ((uint32_t)t << 15));
  }
  __syncthreads();
  const int64_t part = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * BEAM_WAVES + wave, row = part / a.segments;
  if (row >= (int64_t)a.B * a.K || !beam_live(a, row, a.scores[row])) return;   // no barrier below
  const int b = (int)(row / a.K), k = (int)(row - (int64_t)b * a.K), seg = (int)(part - row * a.segments);
  const T* p = reinterpret_cast<const T*>(a.logits) + b * a.sb + k * a.sk;
  uint64_t* list = lists[wave];

  // chunk i of group g: logits g 512 PER + 512 i + 8 lane ..
  constexpr int GROUP = 512 * PER;
  const uint32_t V = (uint32_t)a.V;
  const int n = a.n, g0 = seg * a.per, all = (int)((V + GROUP - 1) / GROUP), g1 = g0 + a.per < all ? g0 + a.per : all;
  Raw8<T> x[PER], next[PER];
  auto load = [&](Raw8<T> (&r)[PER], int g) {
#pragma unroll
    for (int i = 0; i < PER; ++i) r[i] = load_raw8(p, (uint32_t)g * GROUP + 512 * i + 8 * lane, V);
  };
  load(x, g0);

  // A logit goes to the list if it reaches `least` and its key is past `bound`. Of the first
  // group's lane maxima the n-th largest bounds the n best from below; later that of the logits
  // which went to the list, and the list's n-th key when it was ranked.
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, value<T>(x[i], j));
  uint32_t highest = (uint32_t)g0 * GROUP + 8 * lane < V ? ordered(top) : 0;
  uint32_t reach = wave_nth(highest, n);
  float least = level(reach);
  uint64_t bound = 0;
  int count = 0;
  bool bad = false;
  double sum = 0;

  auto put = [&](float l, uint32_t v) {                          // with room for 64
    const uint32_t high = ordered(l);
    const uint64_t key = ((uint64_t)high << 32) | ~v;
    bad = bad || !(l < __builtin_inff());
    const bool take = l >= least && key > bound && v < V;
    const uint64_t takers = __builtin_amdgcn_ballot_w64(take);
    if (take) {
      highest = high > highest ? high : highest;
      list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(takers >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)takers, 0))] = key;
    }
    count += __builtin_popcountll(takers);
  };
  int seen = 0;                                                  // of the list, when `reach` was looked for
  for (int g = g0; g < g1; ++g) {
    if (g + 1 < g1) load(next, g + 1);
    const int before = count;
    bool full = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const uint32_t first = (uint32_t)g * GROUP + 512 * i + 8 * lane;
      uint64_t hits[8], any = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float l = value<T>(x[i], j);
        hits[j] = __builtin_amdgcn_ballot_w64(!(l < least));     // NaN too
        any |= hits[j];
        add_exp(l, table, sum);
      }
      asm volatile("" : "+v"(sum));                              // here, not behind the loop: 16 registers a chunk
      if (any == 0) continue;                                    // uniform, as below
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (hits[j]) {
          if (count > BEAM_LIST - 64) full = true;
          else put(value<T>(x[i], j), first + j);
        }
    }
    if (full || (count - seen) * 2 > n) {                        // at fewer new ones the search costs more than it saves: 61.8 and 59.1 us
      if (full) {                                                // again, the list ranked as often as it is full
        count = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) listed[wave][i][lane] = x[i];
#pragma unroll 1
        for (int i = 0; i < PER; ++i) {
          const T* own = reinterpret_cast<const T*>(&listed[wave][i][lane]);   // the lane's own, in LDS for `i` and `j` vary
#pragma unroll 1
          for (int j = 0; j < 8; ++j) {
            put((float)own[j], (uint32_t)g * GROUP + 512 * i + 8 * lane + j);
            if (count > BEAM_LIST - 64) {
              count = rank_list(list, count, n, 0, lane);
              bound = list[n - 1];
              least = unordered((uint32_t)(bound >> 32));
            }
          }
        }
      }
      // n of the list's logits reach `reach`, those equal to the n-th among them; what follows has higher numbers,
      // so that of equal ones it comes after those that are in the list and has to be above its n-th
      const uint32_t nth = (uint32_t)(bound >> 32), most = wave_nth(highest, n, reach);
      seen = count;
      if (most > reach) reach = most;
      if (nth > reach) reach = nth;
      least = level(reach > nth ? reach : nth + 1);              // nth 0: none was ranked yet
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = next[i];
  }

  count = rank_list(list, count, n, wave_nth(highest, n, reach), lane);
  if (lane < n) a.best[part * n + lane] = lane < count ? list[lane] : 0;
  if (__builtin_amdgcn_ballot_w64(bad)) {
    if (lane == 0) a.norms[part] = make_double2(__builtin_nan(""), 0);
    return;
  }
  double base = 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  const float most = count ? unordered((uint32_t)(list[0] >> 32)) : -__builtin_inff();
  if (!(most <= ADD_EXP_MOST && sum > 1e-40 && sum < 1e40)) {
    // One logit too large, or all of them too small: once more from the largest, from which all that
    // matter differ by less than half of it, so that the difference is exact.
    base = most;
    sum = 0;
    if (most > -__builtin_inff()) {
      for (int g = g0; g < g1; ++g) {
        load(x, g);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
#pragma unroll
          for (int j = 0; j < 8; ++j) add_exp(value<T>(x[i], j) - most, table, sum);
          __builtin_amdgcn_sched_barrier(0);                     // else a chunk's conversions go ahead of another's sum
        }
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
    }
  }
  if (lane == 0) a.norms[part] = make_double2(base, sum);
}

// Candidates in LDS, a wave's at a time; a value's order as an unsigned number, 0: none. Equal values come in the
// order of their beams, within a beam in that of the logits (which 64 bits of the value need not tell apart), then
// of the numbers.
constexpr int MERGE_STAGE = 1024, MERGE_WAVES = 8, MERGE_THREADS = 64 * MERGE_WAVES;
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
  return b ^ (b >> 63 ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double unordered(uint64_t o) { return __builtin_bit_cast(double, o ^ (o >> 63 ? 1ull << 63 : ~0ull)); }

__global__ __launch_bounds__(MERGE_THREADS) void beam_merge_kernel(const BeamArgs a) {
  __shared__ double norms[BEAM_MOST_BEAMS];                      // normaliser; NaN: the beam is out of the search
  __shared__ float scores[BEAM_MOST_BEAMS];
  __shared__ bool ended[BEAM_MOST_BEAMS];
  __shared__ uint64_t stage_at[MERGE_WAVES][MERGE_STAGE + BEAM_MOST_COUNT];       // of the lists, then the wave's best so far
  __shared__ uint32_t stage_index[MERGE_WAVES][MERGE_STAGE + BEAM_MOST_COUNT];    // k V + v
  __shared__ uint32_t stage_logit[MERGE_WAVES][MERGE_STAGE + BEAM_MOST_COUNT];    // in their order
  __shared__ __attribute__((aligned(16))) uint8_t stage_head[MERGE_WAVES][MERGE_STAGE + 1];
  const int t = threadIdx.x, b = blockIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), n = a.n;
  const int64_t row0 = (int64_t)b * a.K;
  const int lists = a.K * a.segments, each = MERGE_STAGE / n;    // of the request, and in a wave's stage
  const bool once = lists <= each;                               // uniform: one wave merges, and all load for it
  constexpr int OWN = MERGE_STAGE / MERGE_THREADS;
  uint64_t keys[OWN];                                            // on their way meanwhile; of beams that are out: anything
  if (once) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int e = t + i * MERGE_THREADS;
      keys[i] = a.best[row0 * a.segments * n + (e < lists * n ? e : 0)];
    }
  }

  // 16 threads a beam: its normaliser out of the segments' sums
  for (int k0 = 0; k0 < a.K; k0 += MERGE_THREADS / 16) {          // uniform
    const int k = k0 + t / 16;
    const bool there = k < a.K;
    const int64_t row = row0 + (there ? k : 0);
    const double2* own = a.norms + row * a.segments;
    const float score = a.scores[row];
    double2 x = own[(t & 15) < a.segments ? t & 15 : 0];         // of a beam that is out: anything
    const bool live = beam_live(a, row, score);
    double most = -__builtin_inf(), sum = 0;
    bool fine = true;
    if (live) {
      for (int s = t & 15; s < a.segments; s += 16) {
        if (s >= 16) x = own[s];
        fine = fine && x.x == x.x;
        if (x.x > most) {
          sum = most == -__builtin_inf() ? x.y : sum * exp(most - x.x) + x.y;
          most = x.x;
        } else if (x.x > -__builtin_inf()) {
          sum += x.x == most ? x.y : x.y * exp(x.x - most);
        }
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      const double m = __shfl_xor(most, d, 64), s = __shfl_xor(sum, d, 64);
      fine = __shfl_xor((int)fine, d, 64) && fine;
      const double high = m > most ? m : most, low = m > most ? most : m;
      const double own = m > most ? s : sum, other = m > most ? sum : s;
      sum = own + (low == high ? other : low > -__builtin_inf() ? other * exp(low - high) : 0);
      most = high;
    }
    if (there && (t & 15) == 0) {
      const bool done = a.finished && a.finished[row];
      double norm = __builtin_nan("");
      if (done && __builtin_isfinite(score)) norm = 0;
      else if (live && fine && most > -__builtin_inf()) norm = most + log(sum);
      norms[k] = norm;
      scores[k] = score;
      ended[k] = done;
    }
  }
  __syncthreads();

  // List l of the request: segment l % segments of beam l / segments. A beam at its end continues
  // with the end token alone, one out of the search with nothing: the rest of theirs is -inf, the first
  // n of which segment 0 stands for.
  uint64_t* at = stage_at[wave];
  uint32_t* index = stage_index[wave];
  uint32_t* logit = stage_logit[wave];
  uint8_t* head = stage_head[wave];
  auto candidate = [&](int list, int j, uint64_t key, uint64_t& value, uint32_t& number, uint32_t& order) {
    const int k = list / a.segments, s = list - k * a.segments;
    const double norm = norms[k], score = scores[k];
    value = 0;
    number = 0;
    order = 0;
    if (ended[k] || !(norm == norm)) {
      if (s != 0 || j >= a.V) return;
      const bool last = norm == norm;
      value = ordered(last && j == 0 ? score : -__builtin_inf());
      number = (uint32_t)(k * a.V + (last ? (j == 0 ? a.end : (j - 1 < a.end ? j - 1 : j)) : j));
      return;
    }
    if (key == 0) return;
    order = (uint32_t)(key >> 32);
    value = ordered(score + ((double)unordered(order) - norm));   // the score last, which a large normaliser would swallow
    number = (uint32_t)(k * a.V) + ~(uint32_t)key;
  };
  // The n best of `count` lists in the stage, of list l at n l, each in order, behind it: the best head,
  // n times. A lane has every 64th list.
  const uint32_t V = (uint32_t)a.V;
  auto merge = [&](int count) {
    wave_sync();
    const bool single = count <= 64;                             // a list a lane: its next head is read a step ahead
    if (!single)
      for (int l = lane; l < count; l += 64) head[l] = 0;
    uint64_t best = 0, second = 0;
    int place = 0, from = 0;                                     // of the lane's best in the stage, and its list
    auto look = [&]() {
      best = 0;
      for (int l = lane; l < count; l += 64) {
        const int j = head[l], e = l * n + j;
        if (j >= n) continue;
        const uint64_t v = at[e];
        bool wins = v > best;
        if (v == best && v != 0) {
          const uint32_t i = index[e], i0 = index[place], o = logit[e], o0 = logit[place];
          wins = i / V == i0 / V && o != o0 ? o > o0 : i < i0;
        }
        if (wins) { best = v; place = e; from = l; }
      }
    };
    auto ahead = [&]() {                                         // the entry behind the lane's best
      const bool more = lane < count && place + 1 < (lane + 1) * n;
      second = at[more ? place + 1 : 0];
      if (!more) second = 0;
    };
    if (single) {
      if (lane < count) { place = lane * n; best = at[place]; }
      ahead();
    } else look();
    int kept = -1;
    for (int r = 0; r < n; ++r) {
      const uint32_t high = wave_most((uint32_t)(best >> 32));
      bool wins = (uint32_t)(best >> 32) == high;
      uint64_t winners = __builtin_amdgcn_ballot_w64(wins);
      if (winners & (winners - 1)) {
        const uint32_t low = wave_most(wins ? (uint32_t)best : 0);
        wins = wins && (uint32_t)best == low;
        winners = __builtin_amdgcn_ballot_w64(wins);
        const uint32_t number = index[place], order = logit[place];
        const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)order, __builtin_ctzll(winners));
        if (__builtin_amdgcn_ballot_w64(wins && order != other)) {
          // of the first beam among them the largest logit
          const uint32_t past = (~wave_most(wins ? ~number : 0) / V + 1) * V;
          wins = wins && number < past;
          const uint32_t top = wave_most(wins ? order : 0);
          wins = wins && order == top;
        }
        const uint32_t first = wave_most(wins ? ~number : 0);     // then the lowest number
        wins = wins && ~number == first;
        winners = __builtin_amdgcn_ballot_w64(wins);
      }
      const int owner = __builtin_ctzll(winners), won = __builtin_amdgcn_readlane(place, owner);
      if (lane == r && high != 0) kept = won;                    // high 0: there is none (-inf is above it)
      if (lane == owner) {
        if (single) {
          best = second;
          if (second != 0) ++place;
          ahead();
        } else {
          ++head[from];
          look();
        }
      }
    }
    wave_sync();
    const uint64_t kept_at = kept < 0 ? 0 : at[kept];
    const uint32_t kept_index = kept < 0 ? 0 : index[kept], kept_logit = kept < 0 ? 0 : logit[kept];
    wave_sync();
    if (lane < n) { at[MERGE_STAGE + lane] = kept_at; index[MERGE_STAGE + lane] = kept_index; logit[MERGE_STAGE + lane] = kept_logit; }
    wave_sync();
  };
  if (once) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int e = t + i * MERGE_THREADS;
      if (e < lists * n) candidate(e / n, e % n, keys[i], stage_at[0][e], stage_index[0][e], stage_logit[0][e]);
    }
    __syncthreads();
    if (wave == 0) merge(lists);
  } else {
    bool some = false;
    for (int l0 = wave * each; l0 < lists; l0 += MERGE_WAVES * each) {
      const int count = lists - l0 < each ? lists - l0 : each, total = count * n;
      for (int e0 = lane; e0 < total; e0 += 64 * OWN) {
#pragma unroll
        for (int i = 0; i < OWN; ++i) keys[i] = a.best[(row0 * a.segments + l0) * n + (e0 + 64 * i < total ? e0 + 64 * i : 0)];
#pragma unroll
        for (int i = 0; i < OWN; ++i) {
          const int e = e0 + 64 * i;
          if (e < total) candidate(l0 + e / n, e % n, keys[i], at[e], index[e], logit[e]);
        }
      }
      if (some && lane < n) {
        at[total + lane] = at[MERGE_STAGE + lane];
        index[total + lane] = index[MERGE_STAGE + lane];
        logit[total + lane] = logit[MERGE_STAGE + lane];
      }
      merge(count + some);
      some = true;
    }
  }
  const int rounds = (lists + each - 1) / each, waves = rounds < MERGE_WAVES ? rounds : MERGE_WAVES;
  if (waves > 1) {                                               // uniform
    __syncthreads();
    if (wave == 0) {
      for (int w = waves - 1; w >= 0; --w)
        if (lane < n) {
          at[w * n + lane] = stage_at[w][MERGE_STAGE + lane];
          index[w * n + lane] = stage_index[w][MERGE_STAGE + lane];
          logit[w * n + lane] = stage_logit[w][MERGE_STAGE + lane];
        }
      merge(waves);
    }
  }
  if (wave == 0 && lane < n) {
    const uint32_t i = index[MERGE_STAGE + lane];
    const uint32_t k = i / V;
    a.out_scores[(int64_t)b * n + lane] = (float)unordered(at[MERGE_STAGE + lane]);
    a.out_parents[(int64_t)b * n + lane] = (int32_t)(row0 + k);
    a.out_tokens[(int64_t)b * n + lane] = (int32_t)(i - k * V);
  }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Chunks of 512 logits that a wave has under way, twice: as many bytes of either type.
constexpr int beam_per_of(int bytes) { return bytes == 4 ? 2 : 4; }

// Groups of logits a segment. 4,096 segments in all are 16 waves a CU: 64 requests x 8 beams x 131,072 in
// bfloat16 take 59.1 us, with 2,048 segments 66.8 and with 8,192 71.5. No more lists than the merge's waves hold at
// once, for every further round of them costs count steps: 16 beams, count 32, 131,072 tokens: 54.5 us, with
// twice as many entries 63, with half 85 (16 beams leave few waves then).
int beam_per(const iak_beam_select_args& a) {
  const int64_t rows = (int64_t)a.batch * a.beams, group = 512 * beam_per_of(a.dtype == IAK_DTYPE_F32 ? 4 : 2);
  const int64_t groups = (a.vocab + group - 1) / group;
  int64_t segments = 4096 / rows;
  const int64_t most = MERGE_STAGE * MERGE_WAVES / ((int64_t)a.beams * a.count);
  if (segments > most) segments = most;
  if (segments > groups) segments = groups;
  if (segments < 1) segments = 1;
  return (int)((groups + segments - 1) / segments);
}

template <typename T> void launch_part(const BeamArgs& a, hipStream_t stream) {
  const int64_t groups = ((int64_t)a.B * a.K * a.segments + BEAM_WAVES - 1) / BEAM_WAVES;
  const uint32_t x = (uint32_t)(groups < (1 << 20) ? groups : 1 << 20);
  const dim3 grid(x, (uint32_t)((groups + x - 1) / x));
  hipLaunchKernelGGL((beam_part_kernel<T, beam_per_of(sizeof(T))>), grid, dim3(BEAM_THREADS), 0, stream, a);
}

}  // namespace

int beam_segments(const iak_beam_select_args& a) {
  const int64_t each = (int64_t)beam_per(a) * 512 * beam_per_of(a.dtype == IAK_DTYPE_F32 ? 4 : 2);
  return (int)((a.vocab + each - 1) / each);
}

size_t beam_workspace(const iak_beam_select_args& a) {
  const size_t parts = (size_t)a.batch * a.beams * beam_segments(a);
  return up256(16 * parts) + up256(8 * parts * a.count);
}

hipError_t launch_beam_select(const iak_beam_select_args& a, void* workspace, hipStream_t stream) {
  BeamArgs k;
  k.B = a.batch; k.K = a.beams; k.V = a.vocab; k.n = a.count;
  k.logits = a.logits; k.sb = a.stride_b; k.sk = a.stride_k;
  k.scores = a.scores; k.finished = a.finished; k.end = a.end_token;
  k.out_scores = a.out_scores; k.out_parents = a.out_parents; k.out_tokens = a.out_tokens;
  k.segments = beam_segments(a);
  k.per = beam_per(a);
  const size_t parts = (size_t)a.batch * a.beams * k.segments;
  char* p = reinterpret_cast<char*>(workspace);
  k.norms = reinterpret_cast<double2*>(p);
  k.best = reinterpret_cast<uint64_t*>(p + up256(16 * parts));
  if (a.dtype == IAK_DTYPE_F32) launch_part<float>(k, stream);
  else if (a.dtype == IAK_DTYPE_F16) launch_part<_Float16>(k, stream);
  else launch_part<__bf16>(k, stream);
  hipLaunchKernelGGL(beam_merge_kernel, dim3((uint32_t)a.batch), dim3(MERGE_THREADS), 0, stream, k);
  return hipGetLastError();
}

}  // namespace iak
