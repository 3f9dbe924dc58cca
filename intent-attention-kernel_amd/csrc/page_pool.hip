// Pages handed out, shared, given back and moved, on the device (gfx950): page tables, row
// lengths and reference counts stay there, so a serving loop needs no answer on the host.
//
// Which page a row gets does not depend on timing: free pages are ranked by id (counts per
// 1,024 pages, then a rank within them), rows by their place in the call, and rank meets
// rank. Reference counts change by integer atomics, whose order leaves no trace.
//
//   grow, fork   seq_plan_kernel   a bit a page: free, and their number per 1,024 ids; one
//                                  workgroup checks the call and sums what its rows need
//                seq_apply_kernel  a workgroup per row: the verdict, the row's free pages out of the
//                                  bits, entries, counts, the copied last page (a fork's where it
//                                  has room, a growing row's where others hold it too)
//   free         seq_free_kernel   a workgroup per row
//   compact      compact_count_kernel, compact_rank_kernel (which page goes where; for few pages
//                compact_small_kernel), compact_apply_kernel (pages copied, table, counts and
//                map written)
//
// What bounds them is latency: reads that wait for each other, and the launches. That a growing
// row's last page may be shared costs two of them (entry, count): 64 x 8 rows
// of one new token grown and freed take 12.3 us replayed, without them 10.9. Pages that
// move are bytes at the rate of a copy: 0.67 GB of K and V rows in 130 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"
#include "mx_internal.h"
#include "iak_device.h"

namespace iak {

namespace {

constexpr int PAGE_GROUP = 1024;       // page ids a workgroup counts or ranks
constexpr int POOL_THREADS = 256;
constexpr int PLAN_THREADS = 1024;
// Up to so many pages one workgroup counts and ranks for a compaction, which saves a launch: of 4,266
// pages 22 us for 24 (14 for 18 replayed from a graph), of 17,066 24 for 24 (28 for 22).
constexpr int64_t FEW_COMPACT_PAGES = 8192;
// Pages of larger pools are moved past the caches: 1.4 GB of them 139 us for 150; of 175 MB, which the
// caches hold, 33 us for 26.
constexpr double STREAM_BYTES = 512.0 * 1024 * 1024;

struct PageArrays {
  int n;
  iak_page_array a[IAK_MAX_PAGE_ARRAYS];
};

// Row `src` of every array to row `dst`, by the workgroup. STREAM: past the caches.
template <bool STREAM> __device__ __forceinline__ void copy_page(const PageArrays& p, int64_t src, int64_t dst) {
  for (int k = 0; k < p.n; ++k) {
    const int64_t bytes = p.a[k].row_bytes;
    char* base = reinterpret_cast<char*>(p.a[k].base);
    const char* from = base + src * bytes;
    char* to = base + dst * bytes;
    const uint64_t low = reinterpret_cast<uintptr_t>(base) | (uint64_t)bytes;
    if ((low & 15u) == 0) {
      for (int64_t i = threadIdx.x; i < bytes / 16; i += blockDim.x) {
        if constexpr (STREAM) st_nt(reinterpret_cast<u4*>(to) + i, ld_nt(reinterpret_cast<const u4*>(from) + i));
        else reinterpret_cast<u4*>(to)[i] = reinterpret_cast<const u4*>(from)[i];
      }
    } else if ((low & 3u) == 0) {
      for (int64_t i = threadIdx.x; i < bytes / 4; i += blockDim.x)
        reinterpret_cast<uint32_t*>(to)[i] = reinterpret_cast<const uint32_t*>(from)[i];
    } else {
      for (int64_t i = threadIdx.x; i < bytes; i += blockDim.x) to[i] = from[i];
    }
  }
}

__global__ __launch_bounds__(POOL_THREADS) void copy_pages_kernel(const PageArrays p, int64_t num_pages, int count,
                                                                  const int32_t* src, const int32_t* dst) {
  for (int i = blockIdx.x; i < count; i += gridDim.x) {
    const int64_t s = src[i], d = dst[i];
    if (s < 0 || s >= num_pages || d < 0 || d >= num_pages || s == d) continue;   // uniform
    copy_page<false>(p, s, d);
  }
}

// --------------------------------------------------------------------------- //
// Sums over a workgroup. Every thread of it calls them.
// --------------------------------------------------------------------------- //

// Sum of `x` over the threads before this one; `total`: over all. WAVES waves; T: int, or where
// the sum may pass 32 bits int64_t.
template <int WAVES, typename T> __device__ __forceinline__ T scan_before(T x, T& total) {
  __shared__ T wave_sum[WAVES];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  T s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const T y = __shfl_up(s, o, 64);
    if (lane >= o) s += y;
  }
  __syncthreads();                      // the last call's sums have been read
  if (lane == 63) wave_sum[w] = s;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int k = 0; k < WAVES; ++k) {
    if (k < w) before += wave_sum[k];
    total += wave_sum[k];
  }
  return before + s - x;
}

// Sums of counts[0 .. at - 1] and of counts[0 .. n - 1].
template <int WAVES> __device__ __forceinline__ void sum_groups(const int32_t* counts, int at, int n, int& before, int& all) {
  int x = 0, y = 0;
  for (int k = threadIdx.x; k < n; k += 64 * WAVES) {
    const int v = counts[k];
    y += v;
    if (k < at) x += v;
  }
  scan_before<WAVES>(x, before);
  scan_before<WAVES>(y, all);
}

// The ids of a thread where one workgroup of PLAN_THREADS takes all.
struct PageRun { int begin, end; };
__device__ __forceinline__ PageRun page_run(int64_t NP) {
  const int per = (int)((NP + PLAN_THREADS - 1) / PLAN_THREADS), at = (int)threadIdx.x * per;
  return PageRun{at, at + per < NP ? at + per : (int)NP};
}
__device__ __forceinline__ int run_free(const int32_t* refs, const PageRun& run) {
  int n = 0;
#pragma unroll 8
  for (int id = run.begin; id < run.end; ++id) n += refs[id] <= 0;
  return n;
}

// --------------------------------------------------------------------------- //
// Grow and fork
// --------------------------------------------------------------------------- //

enum { SEQ_GROW = 0, SEQ_FORK = 1 };

struct SeqArgs {
  int num_seqs, R, W, PSZ;             // rows per sequence, table width, tokens per page
  int64_t NP;
  int32_t* table; int32_t* valid; int32_t* refs;
  int count;
  const int32_t* seqs; const int32_t* parents; const int32_t* new_tokens;
  int32_t* missing;
  int32_t* granted;                    // [num_seqs] tokens that the call makes room for, or null (grow)
  int groups;                          // ceil(NP / PAGE_GROUP)
  int32_t* head;                       // [0] pages needed, [1] the call is refused
  int32_t* group_free;                 // [groups] free pages
  int32_t* marks;                      // [num_seqs] 1: listed in seqs
  int32_t* first;                      // [count * R] pages of the rows before
  uint64_t* free_bits;                 // [groups, 16] bit i of word j: page 64 j + i of the group is free
  PageArrays arrays;
};

__device__ __forceinline__ int used_entries(int tokens, int page_size, int width) {
  if (tokens <= 0) return 0;
  const int64_t n = ((int64_t)tokens + page_size - 1) / page_size;
  return n < width ? (int)n : width;
}

// Whether a forked row gets a page of its own: its parent's last page is not full.
__device__ __forceinline__ bool ragged_last(const SeqArgs& a, int64_t parent_row, int& n, int64_t& page) {
  const int tokens = a.valid[parent_row];
  n = used_entries(tokens, a.PSZ, a.W);
  if (n == 0 || (int64_t)n * a.PSZ <= tokens) return false;
  page = a.table[parent_row * a.W + n - 1];
  return page >= 0 && page < a.NP;
}

// Whether a growing row of `tokens` gets its last page anew: it has room, and others hold it too.
__device__ __forceinline__ bool shared_last(const SeqArgs& a, int64_t row, int tokens) {
  if (tokens <= 0 || tokens % a.PSZ == 0) return false;
  const int64_t page = a.table[row * a.W + used_entries(tokens, a.PSZ, a.W) - 1];
  return page >= 0 && page < a.NP && a.refs[page] > 1;
}

__device__ __forceinline__ int count_free(const int32_t* refs, int64_t NP, int group) {
  int n = 0;
  for (int k = threadIdx.x; k < PAGE_GROUP; k += blockDim.x) {
    const int64_t id = (int64_t)group * PAGE_GROUP + k;
    n += id < NP && refs[id] <= 0;
  }
  return n;
}

// Is the call sound, and what does it need: by a workgroup of PLAN_THREADS. Writes `first`;
// returns the pages needed, and in `refused` (shared) whether it is refused.
template <int KIND> __device__ __forceinline__ int plan_call(const SeqArgs& a, int& refused) {
  constexpr int WAVES = PLAN_THREADS / 64;
  if (threadIdx.x == 0) refused = 0;
  for (int k = threadIdx.x; k < a.num_seqs; k += PLAN_THREADS) {
    a.marks[k] = 0;
    if (KIND == SEQ_GROW && a.granted) a.granted[k] = 0;
  }
  __threadfence_block();
  __syncthreads();
  bool bad = false;
  for (int k = threadIdx.x; k < a.count; k += PLAN_THREADS) {
    const int s = a.seqs[k];
    if (s < 0 || s >= a.num_seqs) { bad = true; continue; }
    if (atomicAdd(&a.marks[s], 1) != 0) bad = true;
    if constexpr (KIND == SEQ_GROW) {
      if (a.new_tokens[k] < 0) bad = true;
    } else {
      const int p = a.parents[k];
      if (p < 0 || p >= a.num_seqs) bad = true;
      for (int h = 0; h < a.R; ++h) if (a.valid[(int64_t)s * a.R + h] != 0) bad = true;
    }
  }
  if (bad) refused = 1;
  __threadfence_block();
  __syncthreads();
  const bool sound = !refused;          // before anyone sets it again: the branches below are uniform
  __syncthreads();
  int64_t total = 0;
  const int rows = a.count * a.R;
  if (sound) {
    if constexpr (KIND == SEQ_FORK) {
      for (int k = threadIdx.x; k < a.count; k += PLAN_THREADS)
        if (a.marks[a.parents[k]] != 0) refused = 1;
    }
    for (int k0 = 0; k0 < rows; k0 += PLAN_THREADS) {
      const int k = k0 + threadIdx.x;
      int64_t need = 0;                                          // 1,024 rows' sum may pass 2^31
      if (k < rows) {
        const int j = k / a.R, h = k - j * a.R;
        if constexpr (KIND == SEQ_GROW) {
          const int old = a.valid[(int64_t)a.seqs[j] * a.R + h];
          const int64_t tokens = (int64_t)(old < 0 ? 0 : old) + a.new_tokens[j];
          if (tokens > (int64_t)a.W * a.PSZ) refused = 1;
          else {
            need = used_entries((int)tokens, a.PSZ, a.W) - used_entries(old, a.PSZ, a.W);
            if (a.new_tokens[j] > 0 && shared_last(a, (int64_t)a.seqs[j] * a.R + h, old)) {
              ++need;
              if (a.arrays.n == 0) refused = 1;
            }
          }
        } else {
          int n;
          int64_t page;
          need = ragged_last(a, (int64_t)a.parents[j] * a.R + h, n, page);
        }
      }
      int64_t all, before;
      if (a.W <= 0x7FFFFFFF / PLAN_THREADS) {                    // 32 bits hold it: 4.6 us for 4.9
        int all32;
        before = scan_before<WAVES>((int)need, all32);
        all = all32;
      } else {
        before = scan_before<WAVES>(need, all);
      }
      if (k < rows) a.first[k] = (int)(total + before > 0x7FFFFFFF ? 0x7FFFFFFF : total + before);
      total += all;
    }
  }
  __syncthreads();
  return (int)(total > 0x7FFFFFFF ? 0x7FFFFFFF : total);
}

template <int KIND> __global__ __launch_bounds__(PLAN_THREADS) void seq_plan_kernel(const SeqArgs a) {
  static_assert(PLAN_THREADS == PAGE_GROUP, "a thread a page");
  if ((int)blockIdx.x < a.groups) {
    const int64_t id = (int64_t)blockIdx.x * PAGE_GROUP + threadIdx.x;
    const bool free_page = id < a.NP && a.refs[id] <= 0;
    const uint64_t bits = __builtin_amdgcn_ballot_w64(free_page);
    if ((threadIdx.x & 63) == 0) a.free_bits[id >> 6] = bits;
    int total;
    scan_before<PLAN_THREADS / 64>((int)free_page, total);
    if (threadIdx.x == 0) a.group_free[blockIdx.x] = total;
    return;
  }
  __shared__ int refused;
  const int need = plan_call<KIND>(a, refused);
  if (threadIdx.x == 0) { a.head[0] = need; a.head[1] = refused; }
}

// The free pages numbered first .. first + n - 1 in order of id, of which there are so many:
// take(number - first, id). By the workgroup, a word of 64 pages a thread at a time; `before`,
// `own`: free pages before and of the thread's run of `per` groups.
template <typename F>
__device__ __forceinline__ void take_pages(const SeqArgs& a, int per, int before, int own, int first, int n, F&& take) {
  __shared__ int start_group, start_before;
  if (before <= first && first < before + own) {                 // one thread
    int g = (int)threadIdx.x * per;
    for (int in = a.group_free[g]; before + in <= first; in = a.group_free[g]) { before += in; ++g; }
    start_group = g;
    start_before = before;
  }
  __syncthreads();
  const int64_t words = (int64_t)a.groups * (PAGE_GROUP / 64);
  int64_t at = (int64_t)start_group * (PAGE_GROUP / 64);
  int base = start_before;
  for (; base < first + n && at < words; at += POOL_THREADS) {   // uniform
    const int64_t word = at + threadIdx.x;
    uint64_t bits = word < words ? a.free_bits[word] : 0;
    int total, number = base + scan_before<POOL_THREADS / 64>(__builtin_popcountll(bits), total);
    for (; bits != 0 && number < first + n; bits &= bits - 1, ++number)
      if (number >= first) take(number - first, (int)(word * 64 + __builtin_ctzll(bits)));
    base += total;
  }
}

template <int KIND> __global__ __launch_bounds__(POOL_THREADS) void seq_apply_kernel(const SeqArgs a) {
  // loads that wait for no other first; what they name is looked at where the verdict is that it is sound
  const int k = blockIdx.x, j = k / a.R, h = k - j * a.R;
  const bool listed = a.count > 0;
  const int need = a.head[0], refused = a.head[1], seq = listed ? a.seqs[j] : 0, first = listed ? a.first[k] : 0;
  const int after = k + 1 < (int)gridDim.x ? a.first[k + 1] : need;   // where the row's pages end
  const int other = listed ? (KIND == SEQ_GROW ? a.new_tokens : a.parents)[j] : 0;
  const int per = (a.groups + POOL_THREADS - 1) / POOL_THREADS;
  int own = 0, all;
  for (int i = 0, g = (int)threadIdx.x * per; i < per && g < a.groups; ++i, ++g) own += a.group_free[g];
  const int before = scan_before<POOL_THREADS / 64>(own, all);
  const int verdict = refused ? -1 : (need > all ? need - all : 0);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.missing[0] = verdict;
  if (verdict != 0 || !listed) return;
  const int64_t row = (int64_t)seq * a.R + h;
  int32_t* entries = a.table + row * a.W;
  if constexpr (KIND == SEQ_GROW) {
    const int old = a.valid[row] < 0 ? 0 : a.valid[row], tokens = old + other;
    const int have = used_entries(old, a.PSZ, a.W), want = used_entries(tokens, a.PSZ, a.W), n = after - first;
    __shared__ int fresh;
    const bool anew = n > want - have;                           // shared_last() when planned: counts sink here
    const int last = anew ? entries[have - 1] : 0;
    if (n > 0)
      take_pages(a, per, before, own, first, n, [&](int e, int id) {
        entries[have - anew + e] = id;
        a.refs[id] = 1;
        if (anew && e == 0) fresh = id;
      });
    __syncthreads();                                             // every thread has read the old length
    if (anew) {
      if (threadIdx.x == 0) atomicSub(&a.refs[last], 1);
      copy_page<false>(a.arrays, last, fresh);
    }
    if (threadIdx.x == 0) {
      a.valid[row] = tokens;
      if (a.granted && h == 0) a.granted[seq] = other;
    }
  } else {
    __shared__ int fresh;
    const int64_t parent = (int64_t)other * a.R + h;
    const int32_t* from = a.table + parent * a.W;
    int n;
    int64_t last;
    const bool own_page = ragged_last(a, parent, n, last);
    const int shared = own_page ? n - 1 : n;
    for (int e = threadIdx.x; e < shared; e += POOL_THREADS) {
      const int id = from[e];
      entries[e] = id;
      if (id >= 0 && id < a.NP) atomicAdd(&a.refs[id], 1);
    }
    if (own_page) {
      take_pages(a, per, before, own, first, 1, [&](int, int id) { fresh = id; });
      __syncthreads();
      if (threadIdx.x == 0) { entries[n - 1] = fresh; a.refs[fresh] = 1; }
      copy_page<false>(a.arrays, last, fresh);
    }
    if (threadIdx.x == 0) a.valid[row] = a.valid[parent];
  }
}

// A workgroup per (listed sequence, row). The length is lowered atomically, so that a sequence
// listed twice loses each of its tokens once.
__global__ __launch_bounds__(POOL_THREADS) void seq_free_kernel(const SeqArgs a) {
  __shared__ int tokens, left;
  const int k = blockIdx.x, j = k / a.R, h = k - j * a.R;
  const int s = a.seqs[j];
  if (s < 0 || s >= a.num_seqs) return;
  const int64_t row = (int64_t)s * a.R + h;
  if (threadIdx.x == 0) {
    int old, rest = 0;
    if (a.new_tokens) {
      const int drop = a.new_tokens[j] < 0 ? 0 : a.new_tokens[j];
      int seen = atomicAdd(&a.valid[row], 0);
      do {                                                       // fails only where another workgroup's succeeds
        old = seen;
        rest = old > drop ? old - drop : 0;
        seen = atomicCAS(&a.valid[row], old, rest);
      } while (seen != old);
    } else {
      old = atomicExch(&a.valid[row], 0);
    }
    tokens = old;
    left = rest;
  }
  __syncthreads();
  const int n = used_entries(tokens, a.PSZ, a.W);
  int32_t* entries = a.table + row * a.W;
  for (int e = used_entries(left, a.PSZ, a.W) + threadIdx.x; e < n; e += POOL_THREADS) {
    const int id = entries[e];
    if (id >= 0 && id < a.NP) atomicSub(&a.refs[id], 1);
    entries[e] = -1;
  }
}

// --------------------------------------------------------------------------- //
// Compaction
// --------------------------------------------------------------------------- //

struct CompactArgs {
  int64_t rows; int W, PSZ;
  int64_t NP;
  const int32_t* table; const int32_t* valid; const int32_t* refs;
  int32_t* out_table; int32_t* out_refs; int32_t* page_map;
  int groups;
  int32_t* group_free;   // [groups]
  int32_t* head;         // [0] pages in use, [1] moves
  int32_t* order;        // [NP] of a page in use past the end: the move it is
  int32_t* hole;         // [NP / 2 + 1] where move j goes
  int32_t* mover;        // [NP / 2 + 1] what move j moves
  int move_groups;       // workgroups that copy pages
  bool stream;           // past the caches
  PageArrays arrays;
};

__global__ __launch_bounds__(POOL_THREADS) void compact_count_kernel(const CompactArgs a) {
  int total;
  scan_before<POOL_THREADS / 64>(count_free(a.refs, a.NP, blockIdx.x), total);
  if (threadIdx.x == 0) a.group_free[blockIdx.x] = total;
}

// With L pages in use: the free ids below L are the holes in order, and the page in use that
// is r-th of all goes, where its id is L or more, to hole L - 1 - r.
__global__ __launch_bounds__(POOL_THREADS) void compact_rank_kernel(const CompactArgs a) {
  constexpr int WAVES = POOL_THREADS / 64;
  int before, all;
  sum_groups<WAVES>(a.group_free, blockIdx.x, a.groups, before, all);
  const int64_t L = a.NP - all;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.head[0] = (int)L;
    if (all == 0) a.head[1] = 0;
  }
  for (int k0 = 0; k0 < PAGE_GROUP; k0 += POOL_THREADS) {
    const int64_t id = (int64_t)blockIdx.x * PAGE_GROUP + k0 + threadIdx.x;
    const bool in = id < a.NP, free_page = in && a.refs[id] <= 0;
    int total;
    const int free_before = before + scan_before<WAVES>((int)free_page, total);
    before += total;
    if (in && id == L) a.head[1] = free_before;
    if (free_page && id < L) a.hole[free_before] = (int)id;
    if (in && !free_page && id >= L) {
      const int move = (int)(L - 1 - (id - free_before));
      a.mover[move] = (int)id;
      a.order[id] = move;
    }
  }
}

// Count and rank in one workgroup, for pools of few pages.
__global__ __launch_bounds__(PLAN_THREADS) void compact_small_kernel(const CompactArgs a) {
  const PageRun run = page_run(a.NP);
  int all, free_before = scan_before<PLAN_THREADS / 64>(run_free(a.refs, run), all);
  const int L = (int)a.NP - all;
  if (threadIdx.x == 0) {
    a.head[0] = L;
    if (all == 0) a.head[1] = 0;
  }
  for (int id = run.begin; id < run.end; ++id) {
    const bool free_page = a.refs[id] <= 0;
    if (id == L) a.head[1] = free_before;
    if (free_page) {
      if (id < L) a.hole[free_before] = id;
      ++free_before;
    } else if (id >= L) {
      const int move = L - 1 - (id - free_before);
      a.mover[move] = id;
      a.order[id] = move;
    }
  }
}

__device__ __forceinline__ int moved_to(const CompactArgs& a, int id, int L) {
  return id < L ? id : a.hole[a.order[id]];
}

__global__ __launch_bounds__(POOL_THREADS) void compact_apply_kernel(const CompactArgs a) {
  const int L = a.head[0];
  if ((int)blockIdx.x < a.move_groups) {
    const int moves = a.head[1];
    for (int j = blockIdx.x; j < moves; j += a.move_groups) {
      if (a.stream) copy_page<true>(a.arrays, a.mover[j], a.hole[j]);
      else copy_page<false>(a.arrays, a.mover[j], a.hole[j]);
    }
    return;
  }
  const int64_t step = (int64_t)(gridDim.x - a.move_groups) * POOL_THREADS;
  const int64_t at = (int64_t)(blockIdx.x - a.move_groups) * POOL_THREADS + threadIdx.x;
  for (int64_t id = at; id < a.NP; id += step) {
    const int r = a.refs[id];
    const bool live = r > 0;
    const int to = live ? moved_to(a, (int)id, L) : -1;
    a.page_map[id] = to;
    if (live) a.out_refs[to] = r;
    if (id >= L) a.out_refs[id] = 0;
  }
  for (int64_t k = at; k < a.rows * a.W; k += step) {
    const int64_t row = k / a.W;
    const int e = (int)(k - row * a.W);
    const int id = a.table[k];
    const bool used = e < used_entries(a.valid[row], a.PSZ, a.W) && id >= 0 && id < a.NP;
    a.out_table[k] = used ? (a.refs[id] > 0 ? moved_to(a, id, L) : -1) : id;
  }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

SeqArgs seq_args(const iak_sequences_args& a, void* workspace) {
  SeqArgs s;
  s.num_seqs = a.num_seqs; s.R = a.rows_per_seq; s.W = a.table_width; s.PSZ = a.page_size; s.NP = a.num_pages;
  s.table = a.page_table; s.valid = a.valid_tokens; s.refs = a.refs;
  s.count = a.count; s.seqs = a.seqs; s.parents = a.parents; s.new_tokens = a.new_tokens; s.missing = a.missing;
  s.granted = a.granted;
  s.groups = (int)((a.num_pages + PAGE_GROUP - 1) / PAGE_GROUP);
  s.arrays.n = 0;
  char* p = reinterpret_cast<char*>(workspace);
  auto take = [&](size_t ints) { int32_t* r = reinterpret_cast<int32_t*>(p); p += up256(4 * ints); return r; };
  if (p) {                             // grow and fork, whose arrays are checked; a free's are nobody's
    s.arrays.n = a.num_arrays;
    for (int k = 0; k < a.num_arrays; ++k) s.arrays.a[k] = a.arrays[k];
    s.head = take(2);
    s.group_free = take((size_t)s.groups);
    s.marks = take((size_t)s.num_seqs);
    s.first = take((size_t)a.count * a.rows_per_seq);
    s.free_bits = reinterpret_cast<uint64_t*>(take((size_t)s.groups * (PAGE_GROUP / 32)));
  }
  return s;
}

template <int KIND> hipError_t launch_seq(const iak_sequences_args& a, void* workspace, hipStream_t stream) {
  const SeqArgs s = seq_args(a, workspace);
  const int rows = a.count * a.rows_per_seq;
  hipLaunchKernelGGL(seq_plan_kernel<KIND>, dim3(s.groups + 1), dim3(PLAN_THREADS), 0, stream, s);
  hipLaunchKernelGGL(seq_apply_kernel<KIND>, dim3(rows > 0 ? rows : 1), dim3(POOL_THREADS), 0, stream, s);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_copy_pages(const iak_copy_pages_args& a, hipStream_t stream) {
  PageArrays p;
  p.n = a.num_arrays;
  for (int k = 0; k < a.num_arrays; ++k) p.a[k] = a.arrays[k];
  const int grid = a.count < 65536 ? a.count : 65536;
  hipLaunchKernelGGL(copy_pages_kernel, dim3(grid), dim3(POOL_THREADS), 0, stream, p, a.num_pages, a.count, a.src, a.dst);
  return hipGetLastError();
}

size_t sequences_workspace(const iak_sequences_args& a) {
  const size_t groups = (size_t)((a.num_pages + PAGE_GROUP - 1) / PAGE_GROUP);
  return up256(8) + up256(4 * groups) + up256(4 * (size_t)a.num_seqs) + up256(4 * (size_t)a.count * a.rows_per_seq) +
         up256(groups * (PAGE_GROUP / 8));
}

hipError_t launch_free_sequences(const iak_sequences_args& a, hipStream_t stream) {
  const SeqArgs s = seq_args(a, nullptr);
  hipLaunchKernelGGL(seq_free_kernel, dim3(a.count * a.rows_per_seq), dim3(POOL_THREADS), 0, stream, s);
  return hipGetLastError();
}
hipError_t launch_grow_sequences(const iak_sequences_args& a, void* workspace, hipStream_t stream) {
  return launch_seq<SEQ_GROW>(a, workspace, stream);
}
hipError_t launch_fork_sequences(const iak_sequences_args& a, void* workspace, hipStream_t stream) {
  return launch_seq<SEQ_FORK>(a, workspace, stream);
}

size_t compact_workspace(const iak_compact_pages_args& a) {
  const size_t groups = (size_t)((a.num_pages + PAGE_GROUP - 1) / PAGE_GROUP), np = (size_t)a.num_pages;
  return up256(8) + up256(4 * groups) + up256(4 * np) + 2 * up256(4 * (np / 2 + 1));
}

hipError_t launch_compact_pages(const iak_compact_pages_args& a, void* workspace, hipStream_t stream) {
  CompactArgs c;
  c.rows = a.num_rows; c.W = a.table_width; c.PSZ = a.page_size; c.NP = a.num_pages;
  c.table = a.page_table; c.valid = a.valid_tokens; c.refs = a.refs;
  c.out_table = a.out_table; c.out_refs = a.out_refs; c.page_map = a.page_map;
  c.groups = (int)((a.num_pages + PAGE_GROUP - 1) / PAGE_GROUP);
  c.arrays.n = a.num_arrays;
  int64_t pool = 0;
  for (int k = 0; k < a.num_arrays; ++k) {
    c.arrays.a[k] = a.arrays[k];
    pool += a.arrays[k].row_bytes;
  }
  c.stream = (double)pool * a.num_pages > STREAM_BYTES;
  const size_t np = (size_t)a.num_pages;
  char* p = reinterpret_cast<char*>(workspace);
  auto take = [&](size_t ints) { int32_t* r = reinterpret_cast<int32_t*>(p); p += up256(4 * ints); return r; };
  c.head = take(2);
  c.group_free = take((size_t)c.groups);
  c.order = take(np);
  c.hole = take(np / 2 + 1);
  c.mover = take(np / 2 + 1);
  const int64_t moves = a.num_pages / 2 + 1;
  c.move_groups = a.num_arrays > 0 && a.num_pages > 0 ? (int)(moves < 4096 ? moves : 4096) : 0;
  const int64_t items = a.num_pages > (int64_t)a.num_rows * a.table_width ? a.num_pages : (int64_t)a.num_rows * a.table_width;
  const int64_t rest = (items + POOL_THREADS - 1) / POOL_THREADS;
  if (a.num_pages > 0 && a.num_pages <= FEW_COMPACT_PAGES) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, c);
  } else if (a.num_pages > 0) {
    hipLaunchKernelGGL(compact_count_kernel, dim3(c.groups), dim3(POOL_THREADS), 0, stream, c);
    hipLaunchKernelGGL(compact_rank_kernel, dim3(c.groups), dim3(POOL_THREADS), 0, stream, c);
  }
  hipLaunchKernelGGL(compact_apply_kernel, dim3((uint32_t)(c.move_groups + (rest < 4096 ? rest : 4096))), dim3(POOL_THREADS), 0,
                     stream, c);
  return hipGetLastError();
}

}  // namespace iak
