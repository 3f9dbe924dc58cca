// Kernel-side arguments and launches of the operators around a generation step, built by
// their C ABI layer (step_api.hip).
#ifndef IAK_STEP_INTERNAL_H
#define IAK_STEP_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "iak.h"
#include "mx_internal.h"

namespace iak {

constexpr int BEAM_MOST_COUNT = 64, BEAM_MOST_BEAMS = 256;
// Waves (segments of the vocabulary) that a row of logits is divided into, and the workspace.
int beam_segments(const iak_beam_select_args& a);
size_t beam_workspace(const iak_beam_select_args& a);
hipError_t launch_beam_select(const iak_beam_select_args& a, void* workspace, hipStream_t stream);

// Kernel-side arguments of the rotated append (built from iak_rotary_append_args).
struct RotaryArgs {
  int B, count, Hq, Hkv, G, D, R, W;   // Hq 0: no queries
  int64_t NP;
  const void* q; int64_t qb, qt, qh;
  void* q_out; int64_t qob, qot, qoh;
  const void* k; int64_t kb, kt, kh;
  const void* v; int64_t vb, vt, vh;
  const float* freq;
  const int32_t* positions; int64_t position_stride;   // may be null: a token's number in its row
  const int32_t* table;
  const int32_t* valid;
  const int32_t* q_lens;               // may be null
  void* k_pages; void* v_pages;        // float16 pages, or the 4-bit cache's pools
  uint8_t* k_codes; uint8_t* k_scales; uint8_t* v_codes; uint8_t* v_scales;
  int32_t* tags; int tag;              // may be null
  int group_bits, lanes;               // tokens of one head side by side, heads a token is divided into
};
hipError_t launch_rotary_append(const iak_rotary_append_args& a, hipStream_t stream);

// Kernel-side arguments of the attention over pages of mixed precision (built from
// iak_paged_chunk_args): those of the 4-bit cache's, whose pools and lengths stay NULL, and its own.
enum { PAGES_F16 = 0, PAGES_BYTE = 1, PAGES_ALL = 2 };   // which precisions a call may meet, by its pools: what is compiled in
struct PageAttn : MxAttn {
  int kind;                            // PAGES_*
  const int32_t* counts;
  const int32_t* bounds;               // tokens a row holds, may be null: all of its pages'
  const int32_t* tags;
  uint64_t tagmap; int other_tag; int neg_wrap;
  const void* k_fp16; const void* v_fp16;
  const void* k_fp8; const void* v_fp8;
  const void* k_int8; const void* v_int8;
  const void* k_int4; const void* v_int4;
  const void* k_int4r; const void* v_int4r;
  const void* k_fp8_scale; const void* v_fp8_scale; int fp8_sd;
  const void* k_int8_scale; const void* v_int8_scale; int int8_sd;
  const void* k_int4_scale; const void* v_int4_scale; int int4_sd; int int4_group;
  const float* k_int4r_scale; const float* v_int4r_scale;
};
void launch_page_rows(const PageAttn& a, hipStream_t stream);
void launch_page_chunk(const PageAttn& a, hipStream_t stream);
hipError_t launch_page_attention(const PageAttn& a, hipStream_t stream);

}  // namespace iak

#endif
