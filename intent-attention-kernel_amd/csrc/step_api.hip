// C ABI of the operators around a generation step: argument checks, plans and kernel launch
// (declared in include/iak.h).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "iak.h"
#include "step_internal.h"

namespace {

iak_status fail(iak_status st, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return iak::report(st, text);
}

bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
unsigned element_bytes(int dtype) { return dtype == IAK_DTYPE_F32 ? 4 : 2; }

iak_status launched(hipError_t e, const char* what) {
  return e == hipSuccess ? IAK_OK : fail(IAK_EHIP, "%s launch: %s", what, hipGetErrorString(e));
}

iak_status check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need > 0 && (!workspace || bytes < need || !aligned(workspace, 16)))
    return fail(IAK_EINVAL, "workspace needs %zu bytes, 16-byte aligned (got %zu at %p)", need, bytes, workspace);
  return IAK_OK;
}

iak_status validate_beam_select(const iak_beam_select_args* a) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->batch < 0 || a->beams <= 0 || a->vocab <= 0 || a->count <= 0)
    return fail(IAK_EINVAL, "bad size (batch=%d, beams=%d, vocab=%d, count=%d)", a->batch, a->beams, a->vocab, a->count);
  if (a->beams > iak::BEAM_MOST_BEAMS) return fail(IAK_ENOTSUP, "beams %d is not supported (%d at most)", a->beams, iak::BEAM_MOST_BEAMS);
  if (a->count > iak::BEAM_MOST_COUNT) return fail(IAK_ENOTSUP, "count %d is not supported (%d at most)", a->count, iak::BEAM_MOST_COUNT);
  if ((int64_t)a->beams * a->vocab > 0x7FFFFFFFLL || (int64_t)a->batch * a->beams > 0x7FFFFFFFLL)
    return fail(IAK_EINVAL, "batch %d x beams %d x vocab %d: rows and candidates have int32 numbers", a->batch, a->beams, a->vocab);
  if (a->count > (int64_t)a->beams * a->vocab)
    return fail(IAK_EINVAL, "count %d of %d x %d candidates", a->count, a->beams, a->vocab);
  if (a->dtype < 0 || a->dtype > 2) return fail(IAK_EINVAL, "bad dtype %d", a->dtype);
  if (a->finished && (a->end_token < 0 || a->end_token >= a->vocab))
    return fail(IAK_EINVAL, "end_token %d outside the vocabulary of %d", a->end_token, a->vocab);
  if (a->batch == 0) return IAK_OK;
  if (!a->logits || !a->scores) return fail(IAK_EINVAL, "logits/scores is NULL");
  if (!a->out_scores || !a->out_parents || !a->out_tokens) return fail(IAK_EINVAL, "an output is NULL");
  if (!aligned(a->logits, element_bytes(a->dtype)) || !aligned(a->scores, 4) || !aligned(a->out_scores, 4) ||
      !aligned(a->out_parents, 4) || !aligned(a->out_tokens, 4))
    return fail(IAK_EINVAL, "an array is not aligned to its elements");
  return IAK_OK;
}

}  // namespace

extern "C" {

iak_status iak_beam_select_workspace(const iak_beam_select_args* a, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  iak_status st = validate_beam_select(a);
  if (st != IAK_OK) return st;
  *bytes = a->batch > 0 ? iak::beam_workspace(*a) : 0;
  return IAK_OK;
}

iak_status iak_beam_select(const iak_beam_select_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  iak_status st = validate_beam_select(a);
  if (st != IAK_OK) return st;
  if (a->batch == 0) return IAK_OK;
  st = check_workspace(workspace, workspace_bytes, iak::beam_workspace(*a));
  if (st != IAK_OK) return st;
  return launched(iak::launch_beam_select(*a, workspace, reinterpret_cast<hipStream_t>(stream)), "beam select");
}

}  // extern "C"
