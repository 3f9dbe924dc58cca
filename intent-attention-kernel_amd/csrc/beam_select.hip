// A beam search's choice on gfx950: of each request's beams x vocabulary the `count` best
// continuations,
//   candidate (k, v) = scores[k] + logits[k, v] - log sum_u exp(logits[k, u]),
// best first, ties to the lowest k V + v.
//
//   beam_part_kernel   a workgroup takes a segment of one row of logits into registers, once: its
//                      sum of exponentials and its `count` best by (logit, index), which no offset of
//                      the row changes. The count-th largest of the threads' maxima bounds
//                      those from below, so that few elements go through LDS to be ranked.
//   beam_merge_kernel  a workgroup per request: the rows' normalisers out of the segments' sums,
//                      and the best of the segments' lists.
//
// Which token comes first is a whole number, so candidates of different beams have to be compared
// to more than 32 bits: with offsets off by 2^-24 of 30 or so, two in some 10^5 neighbours would
// change places. exp(x) = 2^(k/16) e^r with |r| <= ln 2 / 32: the table's 2^(k/16) and the sum in
// 64 bits, e^r - 1 in 32 (off by 2^-30), so that a normaliser is off by some 1e-9.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "iak_device.h"
#include "step_internal.h"

namespace iak {

namespace {

constexpr int BEAM_THREADS = 256;

struct BeamArgs {
  int B, K, V, n;
  const void* logits; int64_t sb, sk;
  const float* scores;
  const uint8_t* finished;
  int end;
  float* out_scores; int32_t* out_parents; int32_t* out_tokens;
  int segments, per;        // segments a row, chunks of 8 logits a thread
  double* norms;            // [rows, segments] log of the sum of exponentials; NaN: a logit is NaN or +inf
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

typedef uint32_t any4 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  any4 w[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = __builtin_nontemporal_load(reinterpret_cast<const any4*>(p) + i);
  T t[8];
  __builtin_memcpy(t, w, sizeof(t));
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = (float)t[j];
}

// The workgroup's number of keys above `key` among keys[0 .. n - 1], for each thread.
__device__ __forceinline__ int rank_of(uint64_t key, const uint64_t* keys, int n) {
  int r = 0;
  for (int i = 0; i < n; ++i) r += keys[i] > key;
  return r;
}

template <typename T, int PER>
__global__ __launch_bounds__(BEAM_THREADS) void beam_part_kernel(const BeamArgs a) {
  __shared__ double table[16];
  __shared__ uint64_t maxima[BEAM_THREADS];
  __shared__ uint64_t found[BEAM_MOST_COUNT * PER * 8];
  __shared__ double wave_sum[BEAM_THREADS / 64];
  __shared__ uint32_t wave_top[BEAM_THREADS / 64];
  __shared__ uint64_t least;
  __shared__ int count;
  const int t = threadIdx.x, seg = blockIdx.x;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= (int64_t)a.B * a.K || !beam_live(a, row, a.scores[row])) return;   // uniform
  const int b = (int)(row / a.K), k = (int)(row - (int64_t)b * a.K);
  const T* p = reinterpret_cast<const T*>(a.logits) + b * a.sb + k * a.sk;
  if (t < 16) table[t] = exp2(t * 0.0625);
  if (t == 0) { least = 0; count = 0; }

  // chunk i of thread t: logits 8 (seg PER 256 + i 256 + t) ..; what lies past the row is NaN here
  float x[PER][8];
  const int first = seg * (PER * BEAM_THREADS * 8) + 8 * t;
  auto index = [&](int i) { return first + i * (BEAM_THREADS * 8); };
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int v = index(i);
    if (v + 8 <= a.V) {
      load8(p + v, x[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = v + j < a.V ? (float)p[v + j] : -__builtin_inff();
    }
  }
  // the thread's maximum, and whether everything is a number or -inf
  float top = -__builtin_inff();
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad = bad || !(x[i][j] < __builtin_inff());
      top = fmaxf(top, x[i][j]);
    }
  int at = -1;                                                   // its lowest place; -1: the thread has no logits
#pragma unroll
  for (int i = PER - 1; i >= 0; --i)
#pragma unroll
    for (int j = 7; j >= 0; --j)
      if (x[i][j] == top && index(i) + j < a.V) at = index(i) + j;
  const uint64_t mine = at < 0 ? 0 : ((uint64_t)ordered(top) << 32) | (uint32_t)~at;
  maxima[t] = mine;
  uint32_t high = bad ? 0xFFFFFFFFu : ordered(top);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const uint32_t y = __shfl_xor(high, o, 64); high = y > high ? y : high; }
  if ((t & 63) == 0) wave_top[t >> 6] = high;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < BEAM_THREADS / 64; ++w) high = wave_top[w] > high ? wave_top[w] : high;
  const int64_t part = row * a.segments + seg;
  if (high == 0xFFFFFFFFu) {                                     // uniform: the row is not finite
    if (t == 0) a.norms[part] = __builtin_nan("");
    return;
  }

  // the sum of exp(x - base), relative to the power of two below the maximum's. Large logits are taken
  // from the maximum, which loses nothing: a 32-bit number's step is 2^-8 there, and what differs by a factor counts for nothing
  constexpr float TURN = 23.083120654223414f;                    // 16 / ln 2
  constexpr double STEP = 0.043321698784996581;                  // ln 2 / 16
  const float M = unordered(high);
  const bool any = M > -__builtin_inff();
  const float base = any && fabsf(M) > 65536.f ? M : 0.f;
  const float peak = any ? M - base : 0.f, low = peak - 500.f;   // e^-500 of the maximum: nothing
  const int power = (int)rintf(peak * TURN) >> 4;
  double sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float l = fmaxf(x[i][j] - base, low);
      const float kf = rintf(l * TURN);
      const int kk = (int)kf;
      const float r = (float)__builtin_fma(-STEP, (double)kf, (double)l);
      const float q = __builtin_fmaf(r, __builtin_fmaf(r, __builtin_fmaf(r, 1.f / 24, 1.f / 6), 0.5f), 1.f);
      const double e = __builtin_ldexp(table[kk & 15], (kk >> 4) - power);
      sum = __builtin_fma(e, (double)(r * q), sum) + e;
    }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
  if ((t & 63) == 0) wave_sum[t >> 6] = sum;

  // a bound from below for the n best: the n-th largest of the threads' maxima (0: fewer have any)
  if (rank_of(mine, maxima, BEAM_THREADS) == a.n - 1 && mine != 0) least = mine;   // keys differ: one thread
  __syncthreads();
  if (t == 0) {
    double s = 0;
#pragma unroll
    for (int w = 0; w < BEAM_THREADS / 64; ++w) s += wave_sum[w];
    a.norms[part] = any ? log(s) + 0.69314718055994530942 * power + (double)base : -__builtin_inf();
  }
  const uint64_t bound = least;
  if (mine != 0 && mine >= bound) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int v = index(i) + j;
        const uint64_t key = ((uint64_t)ordered(x[i][j]) << 32) | (uint32_t)~v;
        if (v < a.V && key >= bound) found[atomicAdd(&count, 1)] = key;   // n threads at most, 8 PER of each
      }
  }
  __syncthreads();
  uint64_t* out = a.best + part * a.n;
  const int c = count;
  for (int i = t; i < c; i += BEAM_THREADS) {
    const int r = rank_of(found[i], found, c);
    if (r < a.n) out[r] = found[i];
  }
  for (int i = c + t; i < a.n; i += BEAM_THREADS) out[i] = 0;
}

// A candidate of the merge: better with the larger value, or the lower index of equal ones.
struct Candidate { double at; int64_t index; };                 // index -1: none
__device__ __forceinline__ bool better(const Candidate& x, const Candidate& y) {
  return x.index >= 0 && (y.index < 0 || x.at > y.at || (x.at == y.at && x.index < y.index));
}

constexpr int MERGE_PER = 16;   // candidates a thread takes a round

__global__ __launch_bounds__(BEAM_THREADS) void beam_merge_kernel(const BeamArgs a) {
  __shared__ double norms[BEAM_MOST_BEAMS];                      // normaliser; NaN: the beam is out of the search
  __shared__ float scores[BEAM_MOST_BEAMS];
  __shared__ Candidate maxima[BEAM_THREADS], found[BEAM_MOST_COUNT * (MERGE_PER + 1)], kept[BEAM_MOST_COUNT];
  __shared__ Candidate least;
  __shared__ int count;
  const int t = threadIdx.x, b = blockIdx.x, lane = t & 63;
  const int64_t row0 = (int64_t)b * a.K;

  // a wave a beam: its normaliser out of the segments' ones
  for (int k = t >> 6; k < a.K; k += BEAM_THREADS / 64) {        // uniform in the wave
    const int64_t row = row0 + k;
    const float score = a.scores[row];
    double norm = __builtin_nan("");
    if (a.finished && a.finished[row]) {
      if (__builtin_isfinite(score)) norm = 0;
    } else if (__builtin_isfinite(score)) {
      double most = -__builtin_inf(), sum = 0;
      bool fine = true;
      for (int s = lane; s < a.segments; s += 64) {
        const double x = a.norms[row * a.segments + s];
        fine = fine && x == x;
        most = fmax(most, x);
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) most = fmax(most, __shfl_xor(most, d, 64));
      if (__builtin_amdgcn_ballot_w64(!fine) == 0 && most > -__builtin_inf()) {
        for (int s = lane; s < a.segments; s += 64) sum += exp(a.norms[row * a.segments + s] - most);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
        norm = most + log(sum);
      }
    }
    if (lane == 0) { norms[k] = norm; scores[k] = score; }
  }
  if (t < a.n) kept[t].index = -1;
  __syncthreads();

  // Candidate c of the request: number c % n of segment c / n % segments of beam c / n / segments.
  // A beam at its end continues with the end token alone, one out of the search with nothing:
  // the rest of theirs is -inf, the first n of which segment 0 stands for.
  const int lists = a.K * a.segments;
  auto candidate = [&](int64_t c) {
    Candidate r = {0, -1};
    const int list = (int)(c / a.n), j = (int)(c - (int64_t)list * a.n), k = list / a.segments, s = list - k * a.segments;
    const bool done = a.finished && a.finished[row0 + k];
    const double norm = norms[k], score = scores[k];
    if (done || !(norm == norm)) {
      if (s != 0 || j >= a.V) return r;
      if (norm == norm) {
        const int v = j == 0 ? a.end : (j - 1 < a.end ? j - 1 : j);
        r = {j == 0 ? score : -__builtin_inf(), (int64_t)k * a.V + v};
      } else {
        r = {-__builtin_inf(), (int64_t)k * a.V + j};
      }
      return r;
    }
    const uint64_t key = a.best[((row0 + k) * a.segments + s) * a.n + j];
    // the score last, which a large normaliser would swallow
    if (key != 0) r = {score + ((double)unordered((uint32_t)(key >> 32)) - norm), (int64_t)k * a.V + (int)~(uint32_t)key};
    return r;
  };
  const int64_t total = (int64_t)lists * a.n;
  for (int64_t c0 = 0; c0 < total; c0 += (int64_t)BEAM_THREADS * MERGE_PER) {   // uniform
    Candidate x[MERGE_PER], top = t < a.n ? kept[t] : Candidate{0, -1};
    const Candidate mine = top;
#pragma unroll
    for (int i = 0; i < MERGE_PER; ++i) {
      const int64_t c = c0 + i * BEAM_THREADS + t;
      x[i] = c < total ? candidate(c) : Candidate{0, -1};
      if (better(x[i], top)) top = x[i];
    }
    maxima[t] = top;
    if (t == 0) { least.index = -1; count = 0; }
    __syncthreads();
    int above = 0;
    for (int i = 0; i < BEAM_THREADS; ++i) above += better(maxima[i], top);
    if (top.index >= 0 && above == a.n - 1) least = top;
    __syncthreads();
    const Candidate bound = least;
    auto take = [&](const Candidate& y) {
      if (y.index >= 0 && !better(bound, y)) found[atomicAdd(&count, 1)] = y;
    };
    if (top.index >= 0 && !better(bound, top)) {
      take(mine);
#pragma unroll
      for (int i = 0; i < MERGE_PER; ++i) take(x[i]);
    }
    __syncthreads();
    const int c = count;
    for (int i = t; i < c; i += BEAM_THREADS) {
      const Candidate y = found[i];
      int r = 0;
      for (int h = 0; h < c; ++h) r += better(found[h], y);
      if (r < a.n) kept[r] = y;
    }
    __syncthreads();
  }
  if (t < a.n) {
    const Candidate y = kept[t];
    const int64_t k = y.index / a.V;
    a.out_scores[(int64_t)b * a.n + t] = (float)y.at;
    a.out_parents[(int64_t)b * a.n + t] = (int32_t)(row0 + k);
    a.out_tokens[(int64_t)b * a.n + t] = (int32_t)(y.index - k * a.V);
  }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Chunks of 8 logits a thread: 4, or as few as give the card a workgroup a CU.
int beam_per(const iak_beam_select_args& a) {
  const int64_t rows = (int64_t)a.batch * a.beams;
  int per = 4;
  while (per > 1 && rows * ((a.vocab + per * BEAM_THREADS * 8 - 1) / (per * BEAM_THREADS * 8)) < 256) per /= 2;
  return per;
}

template <typename T> void launch_part(const BeamArgs& a, hipStream_t stream) {
  const int64_t rows = (int64_t)a.B * a.K;
  const uint32_t y = (uint32_t)(rows < 32768 ? rows : 32768);
  const dim3 grid((uint32_t)a.segments, y, (uint32_t)((rows + y - 1) / y));
  if (a.per == 4) hipLaunchKernelGGL((beam_part_kernel<T, 4>), grid, dim3(BEAM_THREADS), 0, stream, a);
  else if (a.per == 2) hipLaunchKernelGGL((beam_part_kernel<T, 2>), grid, dim3(BEAM_THREADS), 0, stream, a);
  else hipLaunchKernelGGL((beam_part_kernel<T, 1>), grid, dim3(BEAM_THREADS), 0, stream, a);
}

}  // namespace

int beam_segments(const iak_beam_select_args& a) {
  const int64_t each = (int64_t)beam_per(a) * BEAM_THREADS * 8;
  return (int)((a.vocab + each - 1) / each);
}

size_t beam_workspace(const iak_beam_select_args& a) {
  const size_t parts = (size_t)a.batch * a.beams * beam_segments(a);
  return up256(8 * parts) + up256(8 * parts * a.count);
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
  k.norms = reinterpret_cast<double*>(p);
  k.best = reinterpret_cast<uint64_t*>(p + up256(8 * parts));
  if (a.dtype == IAK_DTYPE_F32) launch_part<float>(k, stream);
  else if (a.dtype == IAK_DTYPE_F16) launch_part<_Float16>(k, stream);
  else launch_part<__bf16>(k, stream);
  hipLaunchKernelGGL(beam_merge_kernel, dim3((uint32_t)a.batch), dim3(BEAM_THREADS), 0, stream, k);
  return hipGetLastError();
}

}  // namespace iak
