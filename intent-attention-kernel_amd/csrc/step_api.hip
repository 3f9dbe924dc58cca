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

iak_status validate_rotary_append(const iak_rotary_append_args* a) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->batch < 0 || a->count < 0 || a->num_kv_heads <= 0 || a->table_width < 0 || a->num_pages < 0 || a->num_q_heads < 0)
    return fail(IAK_EINVAL, "negative or zero size (batch=%d, tokens=%d, num_q_heads=%d, num_kv_heads=%d, table_width=%d, num_pages=%lld)",
                a->batch, a->count, a->num_q_heads, a->num_kv_heads, a->table_width, (long long)a->num_pages);
  if (a->head_dim != 64 && a->head_dim != 128) return fail(IAK_ENOTSUP, "head_dim %d is not supported (64 or 128)", a->head_dim);
  if (a->page_size != 16) return fail(IAK_ENOTSUP, "page_size %d is not supported (16)", a->page_size);
  if (a->rotary_dim <= 0 || a->rotary_dim > a->head_dim || a->rotary_dim % 16)
    return fail(IAK_ENOTSUP, "rotary_dim %d is not a multiple of 16 up to head_dim %d", a->rotary_dim, a->head_dim);
  if (a->interleaved != 0 && a->interleaved != 1) return fail(IAK_EINVAL, "interleaved must be 0 or 1, got %d", a->interleaved);
  if (a->num_pages > 0x7FFFFFFFLL) return fail(IAK_EINVAL, "num_pages %lld exceeds int32 page ids", (long long)a->num_pages);
  if (a->table_width > 0x7FFFFF0) return fail(IAK_EINVAL, "table_width %d: a row's tokens exceed int32", a->table_width);
  if (a->dtype < 0 || a->dtype > 2) return fail(IAK_EINVAL, "bad dtype %d", a->dtype);
  if (a->q && (a->num_q_heads == 0 || a->num_q_heads % a->num_kv_heads != 0))
    return fail(IAK_EINVAL, "num_q_heads %d is not a multiple of num_kv_heads %d", a->num_q_heads, a->num_kv_heads);
  if (a->batch == 0 || a->count == 0) return IAK_OK;
  // a thread per 16 channels: numbers below 2^31 in a sequence, below 2^32 in a launch
  const double heads = (double)a->num_kv_heads + (a->q ? a->num_q_heads : 0);
  const double threads = ((double)a->count + 8) * heads * (a->head_dim / 16) + 256;
  if (threads > 2.0e9 || threads * (a->batch < 32768 ? a->batch : 32768) > 4.0e9)
    return fail(IAK_EINVAL, "too many tokens for one call (%d x %d x %.0f heads)", a->batch, a->count, heads);
  if (!a->k || !a->v) return fail(IAK_EINVAL, "k/v is NULL");
  if (!a->q != !a->q_out) return fail(IAK_EINVAL, "q and q_out go together");
  if (!a->inv_freq) return fail(IAK_EINVAL, "inv_freq is NULL");
  if (!a->page_table && a->table_width > 0) return fail(IAK_EINVAL, "page_table is NULL");
  if (!a->valid_tokens) return fail(IAK_EINVAL, "valid_tokens is NULL");
  const unsigned size = element_bytes(a->dtype);
  if (!aligned(a->k, size) || !aligned(a->v, size) || !aligned(a->q, size) || !aligned(a->q_out, size))
    return fail(IAK_EINVAL, "q, k, v or q_out is not aligned to its elements");
  if (!aligned(a->inv_freq, 4) || !aligned(a->positions, 4) || !aligned(a->page_table, 4) || !aligned(a->valid_tokens, 4) ||
      !aligned(a->q_lens, 4) || !aligned(a->page_tags, 4))
    return fail(IAK_EINVAL, "inv_freq and int32 arrays must be 4-byte aligned");
  const bool packed = a->k_codes || a->k_scales || a->v_codes || a->v_scales;
  if (packed && (a->k_pages || a->v_pages)) return fail(IAK_EINVAL, "both float16 pages and 4-bit pools");
  if (packed && a->page_tags) return fail(IAK_EINVAL, "page_tags of 4-bit pools");
  if (a->num_pages > 0 && packed && (!a->k_codes || !a->k_scales || !a->v_codes || !a->v_scales))
    return fail(IAK_EINVAL, "a code or scale pool is NULL");
  if (a->num_pages > 0 && !packed && (!a->k_pages || !a->v_pages)) return fail(IAK_EINVAL, "k_pages/v_pages is NULL");
  if (!aligned(a->k_codes, 4) || !aligned(a->v_codes, 4)) return fail(IAK_EINVAL, "code pools must be 4-byte aligned");
  if (!aligned(a->k_pages, 2) || !aligned(a->v_pages, 2)) return fail(IAK_EINVAL, "pages are not aligned to their elements");
  return IAK_OK;
}

}  // namespace

extern "C" {

iak_status iak_rotary_append(const iak_rotary_append_args* a, void* stream) {
  iak_status st = validate_rotary_append(a);
  if (st != IAK_OK) return st;
  if (a->batch == 0 || a->count == 0) return IAK_OK;
  return launched(iak::launch_rotary_append(*a, reinterpret_cast<hipStream_t>(stream)), "rotated append");
}

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
