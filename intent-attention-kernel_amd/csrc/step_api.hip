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
  // a launch has fewer than 2^32 threads, and the merge 512 for a request
  if (a->batch > 0x7FFFFF) return fail(IAK_EINVAL, "too many requests for one call (%d)", a->batch);
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

constexpr float LOG2_E = 1.44269504088896340736f;
constexpr double CUS = 256;
size_t round_up(size_t x) { return (x + 255) / 256 * 256; }

struct ChunkPlan {
  int G, kind, tile_rows, tiles, splits, chunk, shares;
  int64_t items;
  size_t ws_m, ws_l, ws_acc, ws_parts, total;
};

// Which kernel, and into how many parts a row's tokens go: the least cost in microseconds, of
//   (start + entry * entries of a part) * (workgroups of the busiest CU, against one) + the merge of parts,
// from the table's width alone, for the lengths are on the device. An entry's time is one workgroup's
// alone on its CU; `pair`: two workgroups of a CU take that much longer than one, and more go as pairs
// (matrix work and the L2's rate are shared; what waits for memory is not). Of 300 calls timed under
// every kernel and number of parts (1 to 64 sequences, 4 to 1,024 rows, 400 to 16,000 tokens, equal and
// ragged, float16 pages and mixed ones), the choice took 1.03 times the best of each at the mean;
// by rows alone, in one round of workgroups, 1.18. head_dim 128, mixed pages: 64 rows of 16,000 tokens, 8 KV
// heads x 2: 16 rows 58 us, 128 rows 97; 256 rows (16 sequences, 2,500 tokens): 16 rows 177 us, 256 rows 114.
// Several sequences may be shared out by their lengths instead of split alike, where a part is at
// least half a tile's: 16 x 8 of up to 16,384 tokens in mixed pages 107 us, split alike 125 at the best,
// 103 and 109 if the lengths are equal. Not over many tiles of 16 rows, whose workgroups then do not
// read the same pages at the same time (4 x 8 of 128 rows, 16,000 tokens: 231 us for 148).
struct ChunkCost { int tile; double start, entry, pair; };

void choose_chunk(const iak_paged_chunk_args* a, int64_t rows, int W, ChunkPlan* p) {
  const bool f32 = a->q_dtype == IAK_DTYPE_F32, plain = p->kind == iak::PAGES_F16, big = a->head_dim == 128;
  const double kvrows = (double)a->batch * a->num_kv_heads, LAUNCH = 8, MERGE = 5, SHARE = 10, FILL = 0.75;
  const ChunkCost costs[3] = {
      {16, plain ? 0. : big ? 3. : 2., big ? (plain ? 0.148 : 0.212) : (plain ? 0.135 : 0.16), big ? (plain ? 2 : 1.5) : (plain ? 1.6 : 1.4)},
      {128, plain ? 4. : big ? 8. : 5., big ? (plain ? 0.40 : 1.12) : (plain ? 0.33 : 0.63), big ? (plain ? 1.65 : 2) : (plain ? 1.5 : 1.37)},
      {256, plain ? 5. : big ? 8. : 6., big ? (plain ? 0.52 : 1.08) : (plain ? 0.36 : 0.68), 2}};
  double least = -1;
  int64_t splits = 1;
  for (const ChunkCost& c : costs) {
    if ((c.tile == 128 && rows <= 16) || (c.tile == 256 && (rows <= 128 || f32))) continue;   // a kernel of 256 float32 rows is not there
    const int tiles = (int)((rows + c.tile - 1) / c.tile);
    const double work = kvrows * tiles, entry = c.entry * (f32 ? 1.5 : 1);
    auto load = [&](double groups) { return groups <= CUS ? 1 : std::ceil(groups / CUS) * c.pair / 2; };
    auto keep = [&](double cost, int64_t s, int shares) {
      if (least >= 0 && cost >= least) return;
      least = cost;
      splits = s;
      p->tile_rows = c.tile;
      p->tiles = tiles;
      p->shares = shares;
    };
    const int64_t most = c.tile == 16 ? (W + 3) / 4 : (W + 15) / 16;
    auto split = [&](int64_t s) {
      if (s < 1 || s > most) return;
      const double merge = s > 1 ? MERGE + kvrows * rows * (s * (double)a->head_dim * 8 / 5.5e6 + (s > 8 ? 1e-3 : 0)) : 0;
      keep(LAUNCH + (c.start + entry * W / s) * load(work * s) + merge, s, 0);
    };
    if (a->splits > 0) {
      keep(LAUNCH + (c.start + entry * W / a->splits) * load(work * a->splits), a->splits, 0);
      continue;
    }
    for (int64_t s = 1; s <= 128; s *= 2) split(s);
    split((int64_t)(CUS / work));
    split((int64_t)(2 * CUS / work));
    if (a->batch == 1 || work > iak::MX_SHARED_TILES || work * W > 2e9 || (c.tile == 16 && rows > 48)) continue;
    for (int shares = c.tile == 16 ? 2 * (int)CUS : (int)CUS; shares <= 2 * CUS; shares *= 2) {
      const double parts = shares / work;                        // of a tile, on average
      if (parts < 2 || parts > most) continue;
      keep(LAUNCH + (c.start + FILL * entry * W / std::floor(parts)) * load(shares) + SHARE +
               kvrows * rows * parts * a->head_dim * 8 / 5.5e6, 1, shares);
    }
  }
  const double tiles = kvrows * p->tiles;
  if (splits > (W + 1) / 2) splits = (W + 1) / 2;
  while (splits > 1 && tiles * splits * p->tile_rows > 1.6e7) splits /= 2;
  p->chunk = (int)((W + splits - 1) / splits);
  p->splits = (W + p->chunk - 1) / p->chunk;
  p->items = p->shares ? p->shares : (int64_t)tiles * p->splits;
}

iak_status validate_paged_chunk(const iak_paged_chunk_args* a, ChunkPlan* p) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->batch < 0 || a->q_len < 0 || a->num_kv_heads <= 0 || a->table_width < 0 || a->num_pages < 0)
    return fail(IAK_EINVAL, "negative or zero size (batch=%d, q_len=%d, num_kv_heads=%d, table_width=%d, num_pages=%lld)", a->batch,
                a->q_len, a->num_kv_heads, a->table_width, (long long)a->num_pages);
  if (a->head_dim != 64 && a->head_dim != 128) return fail(IAK_ENOTSUP, "head_dim %d is not supported (64 or 128)", a->head_dim);
  if (a->page_size != 16) return fail(IAK_ENOTSUP, "page_size %d is not supported (16)", a->page_size);
  if (a->num_pages > 0x7FFFFFFFLL) return fail(IAK_EINVAL, "num_pages %lld exceeds int32 page ids", (long long)a->num_pages);
  if (a->table_width > 0x7FFFFF0) return fail(IAK_EINVAL, "table_width %d: a row's tokens exceed int32", a->table_width);
  if (a->num_q_heads <= 0 || a->num_q_heads % a->num_kv_heads != 0)
    return fail(IAK_EINVAL, "num_q_heads %d is not a multiple of num_kv_heads %d", a->num_q_heads, a->num_kv_heads);
  if (a->q_dtype < 0 || a->q_dtype > 2 || a->out_dtype < 0 || a->out_dtype > 2)
    return fail(IAK_EINVAL, "bad q/out dtype (%d, %d)", a->q_dtype, a->out_dtype);
  if (!std::isfinite(a->sm_scale * LOG2_E)) return fail(IAK_EINVAL, "sm_scale is not finite, in base 2 too");
  if (a->causal != 0 && a->causal != 1) return fail(IAK_EINVAL, "causal must be 0 or 1, got %d", a->causal);
  if (a->splits < 0) return fail(IAK_EINVAL, "splits %d is negative", a->splits);
  *p = ChunkPlan{};
  p->G = a->num_q_heads / a->num_kv_heads;
  if (a->batch == 0 || a->q_len == 0) return IAK_OK;
  if (!a->q || !a->out) return fail(IAK_EINVAL, "q/out is NULL");
  if (!aligned(a->q, element_bytes(a->q_dtype)) || !aligned(a->out, element_bytes(a->out_dtype)))
    return fail(IAK_EINVAL, "q or out is not aligned to its elements");
  if (!a->page_table && a->table_width > 0) return fail(IAK_EINVAL, "page_table is NULL");
  if (!a->page_counts) return fail(IAK_EINVAL, "page_counts is NULL");
  if (!a->page_tags && a->num_pages > 0) return fail(IAK_EINVAL, "page_tags is NULL");
  if (!aligned(a->page_table, 4) || !aligned(a->page_counts, 4) || !aligned(a->valid_tokens, 4) || !aligned(a->q_lens, 4) ||
      !aligned(a->page_tags, 4))
    return fail(IAK_EINVAL, "int32 arrays must be 4-byte aligned");
  p->kind = iak::PAGES_F16;
  for (int t = 0; t < 8 && a->num_pages > 0; ++t) {
    const void *k = nullptr, *v = nullptr, *ks = nullptr, *vs = nullptr;
    int sd = IAK_DTYPE_F32, kind = iak::PAGES_BYTE;
    switch (a->tag_map[t]) {
      case IAK_TAG_FP16: k = a->k_fp16; v = a->v_fp16; ks = vs = k; kind = iak::PAGES_F16; break;
      case IAK_TAG_FP8: k = a->k_fp8; v = a->v_fp8; ks = a->k_fp8_scale; vs = a->v_fp8_scale; sd = a->fp8_scale_dtype; break;
      case IAK_TAG_INT8: k = a->k_int8; v = a->v_int8; ks = a->k_int8_scale; vs = a->v_int8_scale; sd = a->int8_scale_dtype; break;
      case IAK_TAG_INT4:
        k = a->k_int4; v = a->v_int4; ks = a->k_int4_scale; vs = a->v_int4_scale; sd = a->int4_scale_dtype; kind = iak::PAGES_ALL;
        break;
      case IAK_TAG_INT4_RESIDUAL: k = a->k_int4r; v = a->v_int4r; ks = a->k_int4r_scale; vs = a->v_int4r_scale; kind = iak::PAGES_ALL; break;
      default: continue;               // SKIP or unknown: contributes nothing
    }
    if (!k || !v || !ks || !vs) return fail(IAK_EINVAL, "tag %d maps to precision %d, whose K/V pool or scales are NULL", t, a->tag_map[t]);
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(IAK_EINVAL, "K/V pools must be 16-byte aligned");
    if (sd != IAK_DTYPE_F16 && sd != IAK_DTYPE_F32) return fail(IAK_EINVAL, "scale dtype %d must be f16 or f32", sd);
    if (!aligned(ks, element_bytes(sd)) || !aligned(vs, element_bytes(sd))) return fail(IAK_EINVAL, "scales are not aligned to their elements");
    if (a->tag_map[t] == IAK_TAG_INT4 && (a->int4_group <= 0 || a->head_dim % a->int4_group || a->int4_group % (a->head_dim / 4)))
      return fail(IAK_ENOTSUP, "int4_group %d must divide head_dim %d and be a multiple of %d", a->int4_group, a->head_dim, a->head_dim / 4);
    if (kind > p->kind) p->kind = kind;
  }
  const int64_t rows = (int64_t)a->q_len * p->G;
  if (rows > 0x3FFFFFFF) return fail(IAK_EINVAL, "q_len %d x %d heads per KV head is too long", a->q_len, p->G);
  const double kvrows = (double)a->batch * a->num_kv_heads;
  if (kvrows * ((rows + 15) / 16) > 1.6e7)
    return fail(IAK_EINVAL, "too many query rows for one call (%.0f tiles of 16)", kvrows * ((rows + 15) / 16));
  choose_chunk(a, rows, a->table_width > 0 ? a->table_width : 1, p);
  if (p->splits > 1 || p->shares) {
    const size_t kept = (size_t)p->items * p->tile_rows;
    p->ws_l = round_up(4 * kept);
    p->ws_acc = p->ws_l + round_up(4 * kept);
    p->ws_parts = p->ws_acc + round_up(4 * kept * (size_t)a->head_dim);
    p->total = p->ws_parts + (p->shares ? round_up(8 * (size_t)kvrows * p->tiles) : 0);
  }
  return IAK_OK;
}

}  // namespace

extern "C" {

iak_status iak_paged_chunk_workspace(const iak_paged_chunk_args* a, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  ChunkPlan p;
  iak_status st = validate_paged_chunk(a, &p);
  if (st != IAK_OK) return st;
  *bytes = p.total;
  return IAK_OK;
}

iak_status iak_paged_chunk(const iak_paged_chunk_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  ChunkPlan p;
  iak_status st = validate_paged_chunk(a, &p);
  if (st != IAK_OK) return st;
  if (a->batch == 0 || a->q_len == 0) return IAK_OK;
  st = check_workspace(workspace, workspace_bytes, p.total);
  if (st != IAK_OK) return st;
  iak::PageAttn k{};
  k.B = a->batch; k.L = a->q_len; k.Hq = a->num_q_heads; k.Hkv = a->num_kv_heads; k.G = p.G; k.D = a->head_dim;
  k.W = a->table_width; k.NP = a->num_pages;
  k.tile_rows = p.tile_rows; k.tiles = p.tiles; k.splits = p.splits; k.chunk = p.chunk; k.shares = p.shares;
  k.items = p.items;
  k.parted = p.total > 0;
  k.q = a->q; k.q_dtype = a->q_dtype; k.qsb = a->q_stride_b; k.qst = a->q_stride_t; k.qsh = a->q_stride_h;
  k.out = a->out; k.out_dtype = a->out_dtype; k.osb = a->out_stride_b; k.ost = a->out_stride_t; k.osh = a->out_stride_h;
  k.table = a->page_table; k.q_lens = a->q_lens; k.counts = a->page_counts; k.bounds = a->valid_tokens;
  k.score_mult = a->sm_scale * LOG2_E;
  k.causal = a->causal;
  k.kind = p.kind;
  k.tags = a->page_tags;
  for (int t = 0; t < 8; ++t) k.tagmap |= (uint64_t)a->tag_map[t] << (8 * t);
  k.other_tag = a->map_other_tags ? a->tag_map[7] : IAK_TAG_SKIP;
  k.neg_wrap = a->negative_ids;
  k.k_fp16 = a->k_fp16; k.v_fp16 = a->v_fp16; k.k_fp8 = a->k_fp8; k.v_fp8 = a->v_fp8; k.k_int8 = a->k_int8; k.v_int8 = a->v_int8;
  k.k_int4 = a->k_int4; k.v_int4 = a->v_int4; k.k_int4r = a->k_int4r; k.v_int4r = a->v_int4r;
  k.k_fp8_scale = a->k_fp8_scale; k.v_fp8_scale = a->v_fp8_scale; k.fp8_sd = a->fp8_scale_dtype;
  k.k_int8_scale = a->k_int8_scale; k.v_int8_scale = a->v_int8_scale; k.int8_sd = a->int8_scale_dtype;
  k.k_int4_scale = a->k_int4_scale; k.v_int4_scale = a->v_int4_scale; k.int4_sd = a->int4_scale_dtype;
  k.int4_group = a->int4_group > 0 ? a->int4_group : a->head_dim;
  k.k_int4r_scale = a->k_int4r_scale; k.v_int4r_scale = a->v_int4r_scale;
  char* ws = reinterpret_cast<char*>(workspace);
  k.ws_m = reinterpret_cast<float*>(ws + p.ws_m);
  k.ws_l = reinterpret_cast<float*>(ws + p.ws_l);
  k.ws_acc = reinterpret_cast<float*>(ws + p.ws_acc);
  k.ws_parts = reinterpret_cast<int2*>(ws + p.ws_parts);
  return launched(iak::launch_page_attention(k, reinterpret_cast<hipStream_t>(stream)), "chunk attention");
}

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
