// Kernel-side arguments and launches of the 4-bit token cache and of page sharing, built by
// their C ABI layer (mx_api.hip).
#ifndef IAK_MX_INTERNAL_H
#define IAK_MX_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iak.h"

namespace iak {

// Sets the calling thread's iak_last_error() text and returns `st`.
iak_status report(iak_status st, const char* text);

constexpr int MX_SHARED_TILES = 512;   // most tiles that are shared out

// Kernel-side arguments of the 4-bit cache's attention (built from iak_mx_attention_args).
struct MxAttn {
  int B, L, Hq, Hkv, G, D, W;   // Hq: for the fields' places; without it the prompt kernel is compiled to
                                // 2,048 queries over 8,192 tokens in 266 us for 258, with `causal` there 260
  int64_t NP;
  int tile_rows;  // query rows (query token * G + head of the group) of a workgroup: 16: the rows
                  // kernel; 128 or 256 (16-bit queries): the chunk kernel
  int tiles;      // such tiles per KV row
  int splits;     // parts of `chunk` table entries per tile
  int chunk;
  int shares;     // 0, or so many workgroups share out the tiles' entries evenly (mx_shared_part)
  int waves;      // rows kernel: 4 per workgroup, or more (16): as many as it has
  int64_t items;  // workgroups

  const void* q; int q_dtype; int64_t qsb, qst, qsh;
  void* out; int out_dtype; int64_t osb, ost, osh;
  const int32_t* table;
  const int32_t* valid;
  const int32_t* q_lens;   // may be null
  const uint8_t* k_codes; const uint8_t* k_scales; const uint8_t* v_codes; const uint8_t* v_scales;
  float score_mult;        // sm_scale * log2(e)
  int causal;

  bool parted;             // the tiles' parts meet in the workspace
  float* ws_m;             // [parts, tile_rows]: tile t's part s is t * splits + s, or with shares
  float* ws_l;             //   ws_parts[t].x + s of ws_parts[t].y
  float* ws_acc;           // [parts, tile_rows, D]
  int2* ws_parts;          // [B, Hkv, tiles], with shares
};

hipError_t launch_mx_append(const iak_mx_tokens_args& a, hipStream_t stream);
hipError_t launch_mx_read(const iak_mx_tokens_args& a, hipStream_t stream);
hipError_t launch_mx_attention(const MxAttn& a, hipStream_t stream);
void launch_mx_chunk(const MxAttn& a, hipStream_t stream);

hipError_t launch_copy_pages(const iak_copy_pages_args& a, hipStream_t stream);
size_t sequences_workspace(const iak_sequences_args& a);
hipError_t launch_free_sequences(const iak_sequences_args& a, hipStream_t stream);
hipError_t launch_grow_sequences(const iak_sequences_args& a, void* workspace, hipStream_t stream);
hipError_t launch_fork_sequences(const iak_sequences_args& a, void* workspace, hipStream_t stream);
size_t compact_workspace(const iak_compact_pages_args& a);
hipError_t launch_compact_pages(const iak_compact_pages_args& a, void* workspace, hipStream_t stream);

}  // namespace iak

#endif
