// Kernel-side arguments and launches of the operators around a generation step, built by
// their C ABI layer (step_api.hip).
#ifndef IAK_STEP_INTERNAL_H
#define IAK_STEP_INTERNAL_H

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "iak.h"

namespace iak {

// Sets the calling thread's iak_last_error() text and returns `st`.
iak_status report(iak_status st, const char* text);

constexpr int BEAM_MOST_COUNT = 64, BEAM_MOST_BEAMS = 256;
// Workgroups (segments of the vocabulary) that a row of logits is divided into, and the workspace.
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

}  // namespace iak

#endif
