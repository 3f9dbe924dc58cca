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

}  // namespace iak

#endif
