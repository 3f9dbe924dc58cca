// C ABI of the 4-bit token cache and of page sharing: argument checks, split plan,
// workspace layout and kernel launch (declared in include/iak.h).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "iak.h"
#include "mx_internal.h"

namespace {

iak_status fail(iak_status st, const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  return iak::report(st, text);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
size_t round_up(size_t x) { return (x + 255) / 256 * 256; }

iak_status launched(hipError_t e, const char* what) {
  return e == hipSuccess ? IAK_OK : fail(IAK_EHIP, "%s launch: %s", what, hipGetErrorString(e));
}

// what the 4-bit cache's entry points have in common
iak_status validate_mx_cache(int batch, int count, int kv_heads, int head_dim, int page_size, int width, int64_t num_pages) {
  if (batch < 0 || count < 0 || kv_heads <= 0 || width < 0 || num_pages < 0)
    return fail(IAK_EINVAL, "negative or zero size (batch=%d, tokens=%d, num_kv_heads=%d, table_width=%d, num_pages=%lld)", batch,
                count, kv_heads, width, (long long)num_pages);
  if (head_dim != 64 && head_dim != 128) return fail(IAK_ENOTSUP, "head_dim %d is not supported (64 or 128)", head_dim);
  if (page_size != 16) return fail(IAK_ENOTSUP, "page_size %d is not supported (16)", page_size);
  if (num_pages > 0x7FFFFFFFLL) return fail(IAK_EINVAL, "num_pages %lld exceeds int32 page ids", (long long)num_pages);
  if (width > 0x7FFFFF0) return fail(IAK_EINVAL, "table_width %d: a row's tokens exceed int32", width);
  return IAK_OK;
}

iak_status validate_mx_tokens(const iak_mx_tokens_args* a) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  iak_status st = validate_mx_cache(a->batch, a->count, a->num_kv_heads, a->head_dim, a->page_size, a->table_width, a->num_pages);
  if (st != IAK_OK) return st;
  if (a->dtype < 0 || a->dtype > 2) return fail(IAK_EINVAL, "bad dtype %d", a->dtype);
  if (a->batch == 0 || a->count == 0) return IAK_OK;
  // a thread per 8 channels: numbers below 2^31 in a sequence, below 2^32 in a launch
  const double threads = ((double)a->count + 15) * a->num_kv_heads * (a->head_dim / 8) + 256;
  if (threads > 2.0e9 || threads * (a->batch < 32768 ? a->batch : 32768) > 4.0e9)
    return fail(IAK_EINVAL, "too many tokens for one call (%d x %d x %d heads)", a->batch, a->count, a->num_kv_heads);
  if (!a->k || !a->v) return fail(IAK_EINVAL, "k/v is NULL");
  if (!a->page_table && a->table_width > 0) return fail(IAK_EINVAL, "page_table is NULL");
  if (!a->valid_tokens) return fail(IAK_EINVAL, "valid_tokens is NULL");
  if (a->num_pages > 0 && (!a->k_codes || !a->k_scales || !a->v_codes || !a->v_scales))
    return fail(IAK_EINVAL, "a code or scale pool is NULL");
  if ((reinterpret_cast<uintptr_t>(a->k_codes) | reinterpret_cast<uintptr_t>(a->v_codes)) & 3u)
    return fail(IAK_EINVAL, "code pools must be 4-byte aligned");
  return IAK_OK;
}

constexpr float LOG2_E = 1.44269504088896340736f;

struct MxPlan {
  int G, tile_rows, tiles, splits, chunk, shares, waves;
  int64_t items;
  size_t ws_m, ws_l, ws_acc, ws_parts, total;
};

// Which kernel, and into how many parts a row's tokens go: the least of costs in microseconds
// fitted to measurements (80 shapes of 8 to 131,072 query rows by 16 to 2,048 table entries).
// A CU holds one to four workgroups at a time. A round of as many takes START and its entries'
// time, one of fewer runs faster; where sequences differ, rounds before the last are not full. A
// second kernel merges the parts at MERGE and the time of their bytes. With several sequences the
// chunk kernel's rounds can be shared out by lengths, where they are two parts a tile or more.
//   rows kernel, 256 rows x 2,048 entries, head_dim 128: 3 splits (one full round) 183 us, 4 211,
//     6 186, 8 190, 1 (of eight waves) 181; 512 x 125: 1 split 25, 2 29, 4 31; 64 x 128: 1 18, 4 14.6
//   rows kernel | chunk kernel, tiles of 128 rows | of 256, in us (best splits), head_dim 128:
//     1 x 2,048 queries x 32 heads x 8 KV heads over 8,192 tokens: 412 | 266 (1) | 257 (1)
//     1 x 512 x 32 x 8 over 8,192: 126 (2) | 92 (4) | 85 (4);  8 x 16 x 32 x 8 over 4,000: 24 | 35 (8)
//     16 x 512 x 32 x 8 over 512: 168 | 80 (1) | 91 (1);  2 x 4,096 x 16 x 2 over 4,096: 272 | 169 | 155
//     8 x 300 x 8 x 2 over 1,000: 26 | 33 (1) | 36 (3)
//     the first with float32 queries: 537 | 443 (1) | 453 (1)
constexpr double CUS = 256;         // and up to as many unsplit tiles are workgroups of more waves

struct MxChoice { int tile_rows; int64_t splits; int shares; };

MxChoice choose(int B, int Hkv, int64_t rows, int W, int D, bool f32, int64_t forced) {
  const bool big = D == 128;
  const double MERGE = 6, kvrows = (double)B * Hkv;
  const int64_t most = (W + 15) / 16;
  MxChoice best = {16, 1, 0};
  double least = -1;
  // tiles of `tile` rows, of which a CU holds `places`
  auto kernel = [&](int tile, int places, double start, double entry) {
    const double work = kvrows * (double)((rows + tile - 1) / tile), round = CUS * places;
    const double fill = tile > 16 && B > 1 ? 0.75 : 1;
    auto keep = [&](double cost, int64_t splits, int shares) {
      if (least < 0 || cost < least) { least = cost; best = {tile, splits, shares}; }
    };
    auto split = [&](int64_t s) {
      if (s > most) s = most;
      if (s < 1) s = 1;
      if (forced > 0) s = forced;
      const bool many = tile == 16 && s == 1 && work <= CUS;     // one workgroup of more waves a CU
      const int room = many ? 1 : places;
      const double each = std::ceil(work * s / CUS);             // workgroups of the busiest CU
      const double before = std::ceil(each / room) - 1, last = each - before * room;
      double cost = (before * fill + (last == room ? 1 : 0.42 + 0.58 * last / room)) *
                    (start + entry / (many ? (big ? 3 : 5) : 1) * W / s);
      if (s > 1) cost += MERGE + kvrows * rows * ((double)s * D * 8 / 5.5e6 + (s > 8 ? 1e-3 : 0));   // past 8: a workgroup a row
      keep(cost, s, 0);
    };
    split(1);
    if (most <= 1 || forced > 0) return;
    if (work < 4 * round) {
      for (int64_t s = 2; s < most && s < 256; s *= 2) split(s);
      for (int rounds = 1; rounds <= 4; ++rounds) split((int64_t)(rounds * round / work));
    }
    if (B == 1 || tile != (f32 ? 128 : 256) || work > iak::MX_SHARED_TILES || work * W > 2e9) return;
    for (int rounds = 1; rounds <= (big ? 4 : 1); ++rounds) {
      const double parts = rounds * round / work;                // of a tile, on average
      if (parts < 2 || parts > most) continue;
      keep(rounds * (start + 1) + entry * fill * W * work / round * parts / std::floor(parts) + MERGE +
               kvrows * rows * (parts * D * 8 / 5.5e6 + (parts > 8 ? 1e-3 : 0)), 1, (int)(rounds * round));
    }
  };
  const double bytes_entry = (big ? 0.30 : 0.20) / (double)((rows + 15) / 16);   // an entry's bytes, shared by its tiles
  const double rows_entry = big ? (f32 ? 0.205 : 0.16) : (f32 ? 0.173 : 0.14);
  kernel(16, big ? 3 : 4, 3, rows_entry < bytes_entry ? bytes_entry : rows_entry);
  if (rows > 16) kernel(128, big || f32 ? 2 : 3, 4, big ? (f32 ? 0.88 : 0.57) : (f32 ? 0.55 : 0.50));
  if (rows > 128 && !f32) kernel(256, 1, big ? 7 : 5, big ? 0.50 : 0.345);
  // Long rows of several sequences (parts above 2,048 tokens), at most a third of a round: shared out
  // too, whatever the cost says, for it knows the table's width alone. 32 sequences x 8 KV heads of up to
  // 32,768 tokens, head_dim 128: equal 192 us for 182 (eight waves a tile, unsplit), a third to all of it
  // 136 for 158, one long among short ones 28 for 141; 64 of up to 16,384, more than a third: 222 for
  // 200, 161 for 154.
  const double work = kvrows * (double)((rows + 15) / 16), round = CUS * (big ? 3 : 4);
  if (best.tile_rows == 16 && B > 1 && forced == 0 && W / best.splits > 128 && 3 * work <= round && work * W < 2e9)
    best = {16, 1, (int)round};
  return best;
}

iak_status validate_mx_attention(const iak_mx_attention_args* a, MxPlan* p) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  iak_status st = validate_mx_cache(a->batch, a->q_len, a->num_kv_heads, a->head_dim, a->page_size, a->table_width, a->num_pages);
  if (st != IAK_OK) return st;
  if (a->num_q_heads <= 0 || a->num_q_heads % a->num_kv_heads != 0)
    return fail(IAK_EINVAL, "num_q_heads %d is not a multiple of num_kv_heads %d", a->num_q_heads, a->num_kv_heads);
  if (a->q_dtype < 0 || a->q_dtype > 2 || a->out_dtype < 0 || a->out_dtype > 2)
    return fail(IAK_EINVAL, "bad q/out dtype (%d, %d)", a->q_dtype, a->out_dtype);
  if (!std::isfinite(a->sm_scale * LOG2_E)) return fail(IAK_EINVAL, "sm_scale is not finite, in base 2 too");
  if (a->causal != 0 && a->causal != 1) return fail(IAK_EINVAL, "causal must be 0 or 1, got %d", a->causal);
  if (a->splits < 0) return fail(IAK_EINVAL, "splits %d is negative", a->splits);
  *p = MxPlan{};
  p->G = a->num_q_heads / a->num_kv_heads;
  if (a->batch == 0 || a->q_len == 0) return IAK_OK;
  if (!a->q || !a->out) return fail(IAK_EINVAL, "q/out is NULL");
  if (!a->page_table && a->table_width > 0) return fail(IAK_EINVAL, "page_table is NULL");
  if (!a->valid_tokens) return fail(IAK_EINVAL, "valid_tokens is NULL");
  if (a->num_pages > 0 && (!a->k_codes || !a->k_scales || !a->v_codes || !a->v_scales))
    return fail(IAK_EINVAL, "a code or scale pool is NULL");
  if (!aligned16(a->k_codes) || !aligned16(a->v_codes)) return fail(IAK_EINVAL, "code pools must be 16-byte aligned");
  if (!aligned4(a->k_scales) || !aligned4(a->v_scales)) return fail(IAK_EINVAL, "scale pools must be 4-byte aligned");
  const int64_t rows = (int64_t)a->q_len * p->G;
  if (rows > 0x3FFFFFFF) return fail(IAK_EINVAL, "q_len %d x %d heads per KV head is too long", a->q_len, p->G);
  const double kvrows = (double)a->batch * a->num_kv_heads;
  if (kvrows * ((rows + 15) / 16) > 1.6e7)
    return fail(IAK_EINVAL, "too many query rows for one call (%.0f tiles of 16)", kvrows * ((rows + 15) / 16));
  const int W = a->table_width > 0 ? a->table_width : 1;
  const MxChoice best = choose(a->batch, a->num_kv_heads, rows, W, a->head_dim, a->q_dtype == IAK_DTYPE_F32, a->splits);
  p->tile_rows = best.tile_rows;
  p->tiles = (int)((rows + p->tile_rows - 1) / p->tile_rows);
  p->shares = best.shares;
  const double tiles = kvrows * p->tiles;
  int64_t splits = best.splits;
  if (splits > (W + 1) / 2) splits = (W + 1) / 2;
  while (splits > 1 && tiles * splits * p->tile_rows > 1.6e7) splits /= 2;
  p->chunk = (int)((W + splits - 1) / splits);
  p->splits = (W + p->chunk - 1) / p->chunk;
  p->waves = p->splits == 1 && !p->shares && tiles <= CUS ? 16 : 4;
  p->items = p->shares ? p->shares : (int64_t)tiles * p->splits;
  if (p->splits > 1 || p->shares) {
    const size_t rows_kept = (size_t)p->items * p->tile_rows;
    p->ws_m = 0;
    p->ws_l = round_up(4 * rows_kept);
    p->ws_acc = p->ws_l + round_up(4 * rows_kept);
    p->ws_parts = p->ws_acc + round_up(4 * rows_kept * (size_t)a->head_dim);
    p->total = p->ws_parts + (p->shares ? round_up(8 * (size_t)tiles) : 0);
  }
  return IAK_OK;
}

iak_status validate_arrays(int n, const iak_page_array* arrays, int64_t num_pages) {
  if (n < 0 || n > IAK_MAX_PAGE_ARRAYS) return fail(IAK_EINVAL, "num_arrays %d outside [0, %d]", n, IAK_MAX_PAGE_ARRAYS);
  for (int k = 0; k < n; ++k) {
    if (arrays[k].row_bytes <= 0 || arrays[k].row_bytes > (1LL << 31))
      return fail(IAK_EINVAL, "array %d: row_bytes %lld", k, (long long)arrays[k].row_bytes);
    if (!arrays[k].base && num_pages > 0) return fail(IAK_EINVAL, "array %d is NULL", k);
  }
  return IAK_OK;
}

iak_status validate_sequences(const iak_sequences_args* a) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->num_seqs < 0 || a->rows_per_seq <= 0 || a->table_width < 0 || a->page_size <= 0 || a->num_pages < 0 || a->count < 0)
    return fail(IAK_EINVAL, "bad size (num_seqs=%d, rows_per_seq=%d, table_width=%d, page_size=%d, num_pages=%lld, count=%d)",
                a->num_seqs, a->rows_per_seq, a->table_width, a->page_size, (long long)a->num_pages, a->count);
  if (a->num_pages >= 0x7FFFFFFFLL) return fail(IAK_EINVAL, "num_pages %lld exceeds int32 page ids", (long long)a->num_pages);
  if ((double)a->table_width * a->page_size > 2147483647.0)
    return fail(IAK_EINVAL, "table_width %d x page_size %d: a row's tokens exceed int32", a->table_width, a->page_size);
  // one workgroup of 256 threads per listed row
  if ((double)a->count * a->rows_per_seq > 1.6e7) return fail(IAK_EINVAL, "too many rows for one call (%d x %d)", a->count, a->rows_per_seq);
  if (a->count > 0 && !a->seqs) return fail(IAK_EINVAL, "seqs is NULL");
  if (a->num_seqs > 0 && (!a->valid_tokens || (!a->page_table && a->table_width > 0)))
    return fail(IAK_EINVAL, "page_table/valid_tokens is NULL");
  if (a->num_pages > 0 && !a->refs) return fail(IAK_EINVAL, "refs is NULL");
  if (!aligned4(a->page_table) || !aligned4(a->valid_tokens) || !aligned4(a->refs) || !aligned4(a->seqs))
    return fail(IAK_EINVAL, "int32 arrays must be 4-byte aligned");
  return IAK_OK;
}

// grow, fork and reorder: `null`: the name of an argument they need and did not get
iak_status validate_planned(const iak_sequences_args* a, const char* null, size_t need, const void* workspace, size_t workspace_bytes) {
  if (null) return fail(IAK_EINVAL, "%s is NULL", null);
  if (!a->missing) return fail(IAK_EINVAL, "missing is NULL");
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(IAK_EINVAL, "workspace needs %zu bytes, 16-byte aligned (got %zu at %p)", need, workspace_bytes, workspace);
  return IAK_OK;
}

// grow: `granted` is cleared before the other arrays are read, so it must be none of them
iak_status validate_granted(const iak_sequences_args* a) {
  if (!a->granted) return IAK_OK;
  if (!aligned4(a->granted)) return fail(IAK_EINVAL, "granted must be 4-byte aligned");
  const uintptr_t begin = reinterpret_cast<uintptr_t>(a->granted), end = begin + 4 * (uintptr_t)a->num_seqs;
  const uint64_t rows = (uint64_t)a->num_seqs * a->rows_per_seq, count = (uint64_t)a->count;
  const struct { const int32_t* p; uint64_t n; const char* name; } others[] = {
      {a->page_table, rows * a->table_width, "page_table"}, {a->valid_tokens, rows, "valid_tokens"},
      {a->refs, (uint64_t)a->num_pages, "refs"}, {a->seqs, count, "seqs"}, {a->new_tokens, count, "new_tokens"},
      {a->missing, 1, "missing"}};
  for (const auto& o : others) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(o.p);
    if (at < end && begin < at + 4 * o.n) return fail(IAK_EINVAL, "granted overlaps %s", o.name);
  }
  return IAK_OK;
}

iak_status validate_compact(const iak_compact_pages_args* a) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->num_rows < 0 || a->table_width < 0 || a->page_size <= 0 || a->num_pages < 0 || a->num_pages > 0x7FFFFFFFLL)
    return fail(IAK_EINVAL, "bad size (num_rows=%d, table_width=%d, page_size=%d, num_pages=%lld)", a->num_rows, a->table_width,
                a->page_size, (long long)a->num_pages);
  if (a->num_pages > 0 && (!a->refs || !a->out_refs || !a->page_map)) return fail(IAK_EINVAL, "refs, out_refs or page_map is NULL");
  if ((int64_t)a->num_rows * a->table_width > 0 && (!a->page_table || !a->out_table || !a->valid_tokens))
    return fail(IAK_EINVAL, "page_table, out_table or valid_tokens is NULL");
  const void* in[3] = {a->page_table, a->valid_tokens, a->refs};
  const void* out[3] = {a->out_table, a->out_refs, a->page_map};
  for (int k = 0; k < 3; ++k) {
    if (!aligned4(in[k]) || !aligned4(out[k])) return fail(IAK_EINVAL, "int32 arrays must be 4-byte aligned");
    for (int j = 0; j < 3; ++j)
      if (out[k] && (out[k] == in[j] || (j != k && out[k] == out[j])))
        return fail(IAK_EINVAL, "an output of a compaction is another of its arrays");
  }
  return validate_arrays(a->num_arrays, a->arrays, a->num_pages);
}

}  // namespace

extern "C" {

iak_status iak_mx_append_tokens(const iak_mx_tokens_args* a, void* stream) {
  iak_status st = validate_mx_tokens(a);
  if (st != IAK_OK) return st;
  if (a->batch == 0 || a->count == 0) return IAK_OK;
  return launched(iak::launch_mx_append(*a, reinterpret_cast<hipStream_t>(stream)), "append");
}

iak_status iak_mx_read_tokens(const iak_mx_tokens_args* a, void* stream) {
  iak_status st = validate_mx_tokens(a);
  if (st != IAK_OK) return st;
  if (a->batch == 0 || a->count == 0) return IAK_OK;
  return launched(iak::launch_mx_read(*a, reinterpret_cast<hipStream_t>(stream)), "read");
}

iak_status iak_mx_attention_workspace(const iak_mx_attention_args* args, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  MxPlan p;
  iak_status st = validate_mx_attention(args, &p);
  if (st != IAK_OK) return st;
  *bytes = p.total;
  return IAK_OK;
}

iak_status iak_mx_attention(const iak_mx_attention_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  MxPlan p;
  iak_status st = validate_mx_attention(a, &p);
  if (st != IAK_OK) return st;
  if (a->batch == 0 || a->q_len == 0) return IAK_OK;
  if (p.total > 0 && (!workspace || workspace_bytes < p.total || !aligned16(workspace)))
    return fail(IAK_EINVAL, "workspace needs %zu bytes, 16-byte aligned (got %zu at %p)", p.total, workspace_bytes, workspace);
  iak::MxAttn k;
  k.B = a->batch; k.L = a->q_len; k.Hq = a->num_q_heads; k.Hkv = a->num_kv_heads; k.G = p.G; k.D = a->head_dim;
  k.W = a->table_width; k.NP = a->num_pages;
  k.tile_rows = p.tile_rows; k.tiles = p.tiles; k.splits = p.splits; k.chunk = p.chunk; k.shares = p.shares; k.waves = p.waves;
  k.items = p.items; k.parted = p.total > 0;
  k.q = a->q; k.q_dtype = a->q_dtype; k.qsb = a->q_stride_b; k.qst = a->q_stride_t; k.qsh = a->q_stride_h;
  k.out = a->out; k.out_dtype = a->out_dtype; k.osb = a->out_stride_b; k.ost = a->out_stride_t; k.osh = a->out_stride_h;
  k.table = a->page_table; k.valid = a->valid_tokens; k.q_lens = a->q_lens;
  k.k_codes = reinterpret_cast<const uint8_t*>(a->k_codes); k.k_scales = reinterpret_cast<const uint8_t*>(a->k_scales);
  k.v_codes = reinterpret_cast<const uint8_t*>(a->v_codes); k.v_scales = reinterpret_cast<const uint8_t*>(a->v_scales);
  k.score_mult = a->sm_scale * LOG2_E;
  k.causal = a->causal;
  char* ws = reinterpret_cast<char*>(workspace);
  k.ws_m = reinterpret_cast<float*>(ws + p.ws_m);
  k.ws_l = reinterpret_cast<float*>(ws + p.ws_l);
  k.ws_acc = reinterpret_cast<float*>(ws + p.ws_acc);
  k.ws_parts = reinterpret_cast<int2*>(ws + p.ws_parts);
  return launched(iak::launch_mx_attention(k, reinterpret_cast<hipStream_t>(stream)), "4-bit cache attention");
}

iak_status iak_copy_pages(const iak_copy_pages_args* a, void* stream) {
  if (!a) return fail(IAK_EINVAL, "args is NULL");
  if (a->num_pages < 0 || a->num_pages > 0x7FFFFFFFLL || a->count < 0)
    return fail(IAK_EINVAL, "bad size (num_pages=%lld, count=%d)", (long long)a->num_pages, a->count);
  iak_status st = validate_arrays(a->num_arrays, a->arrays, a->num_pages);
  if (st != IAK_OK) return st;
  if (a->count == 0 || a->num_arrays == 0 || a->num_pages == 0) return IAK_OK;
  if (!a->src || !a->dst) return fail(IAK_EINVAL, "src/dst is NULL");
  return launched(iak::launch_copy_pages(*a, reinterpret_cast<hipStream_t>(stream)), "page copy");
}

iak_status iak_sequences_workspace(const iak_sequences_args* a, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  iak_status st = validate_sequences(a);
  if (st != IAK_OK) return st;
  *bytes = iak::sequences_workspace(*a);
  return IAK_OK;
}

iak_status iak_free_sequences(const iak_sequences_args* a, void* stream) {
  iak_status st = validate_sequences(a);
  if (st != IAK_OK) return st;
  if (a->count == 0 || a->num_seqs == 0) return IAK_OK;
  return launched(iak::launch_free_sequences(*a, reinterpret_cast<hipStream_t>(stream)), "free sequences");
}

iak_status iak_grow_sequences(const iak_sequences_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  iak_status st = validate_sequences(a);
  if (st == IAK_OK) st = validate_planned(a, a && a->count > 0 && !a->new_tokens ? "new_tokens" : nullptr, iak::sequences_workspace(*a), workspace, workspace_bytes);
  if (st == IAK_OK) st = validate_granted(a);
  if (st == IAK_OK) st = validate_arrays(a->num_arrays, a->arrays, a->num_pages);
  if (st != IAK_OK) return st;
  return launched(iak::launch_grow_sequences(*a, workspace, reinterpret_cast<hipStream_t>(stream)), "grow sequences");
}

iak_status iak_fork_sequences(const iak_sequences_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  iak_status st = validate_sequences(a);
  if (st == IAK_OK) st = validate_planned(a, a && a->count > 0 && !a->parents ? "parents" : nullptr, iak::sequences_workspace(*a), workspace, workspace_bytes);
  if (st == IAK_OK) st = validate_arrays(a->num_arrays, a->arrays, a->num_pages);
  if (st != IAK_OK) return st;
  return launched(iak::launch_fork_sequences(*a, workspace, reinterpret_cast<hipStream_t>(stream)), "fork sequences");
}

iak_status iak_reorder_sequences_workspace(const iak_sequences_args* a, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  iak_status st = validate_sequences(a);
  if (st != IAK_OK) return st;
  *bytes = iak::reorder_workspace(*a);
  return IAK_OK;
}

iak_status iak_reorder_sequences(const iak_sequences_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  iak_status st = validate_sequences(a);
  if (st == IAK_OK)
    st = validate_planned(a, a->count > 0 && !a->parents ? "parents" : nullptr, iak::reorder_workspace(*a), workspace, workspace_bytes);
  if (st == IAK_OK) st = validate_arrays(a->num_arrays, a->arrays, a->num_pages);
  if (st != IAK_OK) return st;
  return launched(iak::launch_reorder_sequences(*a, workspace, reinterpret_cast<hipStream_t>(stream)), "reorder sequences");
}

iak_status iak_compact_pages_workspace(const iak_compact_pages_args* a, size_t* bytes) {
  if (!bytes) return fail(IAK_EINVAL, "bytes is NULL");
  iak_status st = validate_compact(a);
  if (st != IAK_OK) return st;
  *bytes = iak::compact_workspace(*a);
  return IAK_OK;
}

iak_status iak_compact_pages(const iak_compact_pages_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  iak_status st = validate_compact(a);
  if (st != IAK_OK) return st;
  if (a->num_pages == 0 && (int64_t)a->num_rows * a->table_width == 0) return IAK_OK;
  const size_t need = iak::compact_workspace(*a);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(IAK_EINVAL, "workspace needs %zu bytes, 16-byte aligned (got %zu at %p)", need, workspace_bytes, workspace);
  return launched(iak::launch_compact_pages(*a, workspace, reinterpret_cast<hipStream_t>(stream)), "compact pages");
}

}  // extern "C"
