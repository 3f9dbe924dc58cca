/*
 * iak.h -- C ABI of the MI355X (gfx950) selected-quant paged decode library
 * (libiak.so). Plain pointers, sizes and status codes; no torch or HIP types.
 *
 * Ownership: the caller owns every buffer (inputs, output, workspace). The
 * library allocates nothing and keeps no state between calls, apart from the
 * static per-GPU scratch of iak_paged_decode_noalloc; calls are asynchronous
 * on the caller's HIP stream and never synchronise the host.
 *
 * Reference interfaces these entry points replace (paths relative to the
 * reference's src/intent_attention/):
 *   iak_paged_decode            fused_selected_quant_decode()          fused_selected_quant_decode.py:408-464
 *                               (its Triton launch _launch_triton_kernel :472-513, kernel :87-255)
 *                               and intent_quant_decode_attention_triton()
 *                                                                      triton_intent_quant_attention.py:342-457
 *   iak_paged_decode_workspace  (no counterpart: sizes the split-K partial buffer the caller allocates)
 *   iak_paged_decode_plan       (no counterpart: the split plan the library chooses for a call)
 *   iak_pack_page_descriptors   (no counterpart: page_precision, page_tags and the per-precision scale
 *                               arrays of fused_selected_quant_decode.py:408-464 packed into one
 *                               32-byte descriptor per page)
 *   iak_pack_entry_records      (no counterpart: the page table's entries with their page's native
 *                               tag and scales (fused_selected_quant_decode.py:344-400 reads them
 *                               entry by entry) packed into one 32-byte record per entry)
 *   iak_paged_decode_timed,     (no counterpart: the same calls with HIP events around the split
 *   iak_mla_decode_timed         kernel, for timing it apart from the merge)
 *   iak_timing_event_*          (no counterpart: fence-free HIP timing events for those calls)
 *   iak_mla_decode              mla_decode_triton() / _mla_decode_cpu()    triton_mla_decode.py:110-186
 *                               (the latent context; mla_sparse_decode_reference mla.py:61-92,
 *                               mla_triton_decode mla.py:95-136)
 *   iak_mla_decode_workspace    (no counterpart: sizes the split-K partial buffer)
 *   iak_mla_decode_rows_workspace (no counterpart: sizes the optional split-over-keys partial buffer)
 *   iak_mla_decode_rows         the latent context of mla_decode_triton() in the reference's float32
 *                               arithmetic: its Triton kernel triton_mla_decode.py:47-107 and
 *                               _mla_decode_cpu :155-186 (also under mla_sparse_decode_reference /
 *                               mla_triton_decode, mla.py:61-136)
 *   iak_quantize_pages          fake_quantize_tensor() intent_quant.py:221-312 at page granules, and
 *                               fake_int8_pages_from_fp16() fused_selected_quant_decode.py:521-542 /
 *                               triton_intent_quant_attention.py:460-496
 *   iak_build_page_tables       routing_to_kernel_metadata() block_router.py:383-421 (page ids: selected_page_ids
 *                               :283-296) followed by metadata_to_kernel_tensors()
 *                               fused_selected_quant_decode.py:344-400 (the loop :394-398)
 *   iak_transcode_pages         KVMemoryManager FP16 <-> INT8 page transcoding: write_page's INT8 branch
 *                               kv_memory_manager.py:233-252, _read_page_data :286-296, set_page_format
 *                               :268-284 (demote_cold_pages :350-362, promote_hot_pages :364-377)
 *   iak_prefetch_pages          launch_prefetch_pages() prefetch.py:183-261 (its Triton kernel :111-170)
 *   iak_mla_project             the projection by W_VO in mla_decode_triton() triton_mla_decode.py:146-151
 *   iak_dense_attention         dense_attention() reference.py:16-45 (causal, mask, original_kv_positions),
 *                               under semantic_block_attention() reference.py:81-129 and
 *                               intent_quant_attention_reference() intent_quant_attention.py:20-119
 *   iak_dense_attention_indexed the index_select of the selected tokens and that call, in
 *                               semantic_block_attention() reference.py:100-112
 *   iak_dense_attention_workspace (no counterpart: sizes the optional split-over-keys and tile-flag buffer)
 *   iak_fake_quant_blocks       the per-block fake_quantize_tensor() reconstructions and their torch.cat
 *                               in intent_quant_attention_reference() intent_quant_attention.py:56-84
 *                               (intent_quant.py:221-312), float32 K and V
 *   iak_fake_quant_blocks_workspace (no counterpart: sizes the optional split of long blocks)
 *   iak_mx_append_tokens,       (no counterpart: the reference quantises whole blocks, intent_quant.py:221-312;
 *   iak_mx_read_tokens           these write and read single tokens of a microscaled 4-bit cache)
 *   iak_mx_attention,           (no counterpart: attention of one or several query tokens per sequence over
 *   iak_mx_attention_workspace   that cache)
 *   iak_grow_sequences,         (no counterpart: KVMemoryManager hands out pages on the host and shares none,
 *   iak_fork_sequences,          kv_memory_manager.py:145-231; these keep page tables, lengths and reference
 *   iak_free_sequences,          counts on the device)
 *   iak_compact_pages, iak_copy_pages, iak_sequences_workspace, iak_compact_pages_workspace
 *   iak_reorder_sequences, iak_reorder_sequences_workspace
 *                               (no counterpart: the beams' page tables in the order of that choice)
 *   iak_paged_chunk, iak_paged_chunk_workspace
 *                               (no counterpart: the reference attends one query token a sequence,
 *                               fused_selected_quant_decode.py:408-464; these several, over the same pages)
 *   iak_rotary_append           (no counterpart: keys rotated by position and stored with their values token by token)
 *   iak_beam_select             (no counterpart: the choice of a beam search's continuations)
 *   iak_status_string           (no counterpart: the reference raises ValueError/RuntimeError in Python)
 */
#ifndef IAK_H
#define IAK_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IAK_ABI_VERSION 13

/* Grid size from which merge_in_kernel = 2 merges inside the decode kernel; it
 * also does so on grids of at most IAK_MERGE_IN_KERNEL_SMALL_WORKGROUPS workgroups
 * whose rows hold at most IAK_MERGE_IN_KERNEL_SMALL_PARTIALS split partials
 * (splits x query heads per KV head), where a second launch costs more than the
 * last workgroup's merge. */
#define IAK_MERGE_IN_KERNEL_MIN_WORKGROUPS 1024
#define IAK_MERGE_IN_KERNEL_SMALL_WORKGROUPS 128
#define IAK_MERGE_IN_KERNEL_SMALL_PARTIALS 256

typedef enum {
  IAK_OK = 0,
  IAK_EINVAL = 1,   /* bad argument (shape, dtype, pointer, size): Python maps it to ValueError */
  IAK_ENOTSUP = 2,  /* valid but unsupported configuration (e.g. head_dim): ValueError          */
  IAK_EHIP = 3      /* HIP runtime error (launch, device): RuntimeError                         */
} iak_status;

/* Native page precision tags: the reference's fused numbering
 * (FusedKVPrecision, fused_selected_quant_decode.py:29-34) with the native
 * precisions appended. */
enum {
  IAK_TAG_FP16 = 0,
  IAK_TAG_INT8 = 1,
  IAK_TAG_SKIP = 2,
  IAK_TAG_FP8 = 3,           /* OCP e4m3fn codes, one scale per page            */
  IAK_TAG_INT4 = 4,          /* two codes per byte, one scale per page x group   */
  IAK_TAG_INT4_RESIDUAL = 5  /* base | residual<<4 per byte, two scales per page */
};

enum { IAK_DTYPE_F16 = 0, IAK_DTYPE_F32 = 1, IAK_DTYPE_BF16 = 2 };

/*
 * Arguments of one decode step. Pools are indexed by physical page id and
 * laid out [num_pages, page_size, head_dim] (contiguous), as the reference's
 * k_pages_fp16 / k_pages_int8 (fused_selected_quant_decode.py:427-433). A page
 * holds one KV head of page_size tokens.
 *
 *   q            [batch, num_q_heads, head_dim], element strides q_stride_b / q_stride_h
 *   out          [batch, num_q_heads, head_dim], element strides out_stride_b / out_stride_h
 *   page_table   [batch, num_kv_heads, table_width] int32 (contiguous); row (b, h) lists the
 *                physical pages attended by KV head h of sequence b; query heads
 *                h*G .. h*G+G-1 (G = num_q_heads / num_kv_heads) share it.
 *   page_counts  [batch, num_kv_heads] int32; entries are clamped to [0, table_width].
 *   page_tags    [num_pages] int32 caller tags, translated by tag_map[tag] to a native tag;
 *                map entries outside the enum contribute nothing.
 *   map_other_tags  0: caller tags outside [0, 8) contribute nothing (the fused
 *                reference's `else: continue`, fused_selected_quant_decode.py:316-317);
 *                1: they take tag_map[7] (the sibling API reads every tag but FP16
 *                and SKIP through its INT8 pool, triton_intent_quant_attention.py:281-307).
 *   negative_ids 0: an id < 0 is an invalid page (contributes nothing);
 *                1: an id in [-num_pages, 0) means id + num_pages (torch indexing).
 *                Ids outside the pool always contribute nothing.
 *
 *   FP16 pages: k_fp16/v_fp16 f16.
 *   FP8 pages:  k_fp8/v_fp8 e4m3fn bytes; k_fp8_scale/v_fp8_scale [num_pages] (scale_dtype).
 *   INT8 pages: k_int8/v_int8 int8; k_int8_scale/v_int8_scale [num_pages] (scale_dtype).
 *   INT4 pages: k_int4/v_int4 [num_pages, page_size, head_dim/2] bytes, element 2j in the
 *               low nibble of byte j, each nibble = code + 8 (codes in [-7, 7]);
 *               k_int4_scale/v_int4_scale [num_pages, head_dim/int4_group] (scale_dtype).
 *   INT4_RESIDUAL pages: k_int4r/v_int4r [num_pages, page_size, head_dim] bytes,
 *               (base code + 8) | (residual code + 8) << 4; k_int4r_scale/v_int4r_scale
 *               [num_pages, 2] f32 (base scale, residual scale).
 *   Dequantised value = code * scale (INT4_RESIDUAL: base*s0 + residual*s1).
 *
 *   sm_scale     softmax scale (the reference uses 1/sqrt(head_dim), :323).
 *   pages_per_split  pages one wave reduces before the cross-split merge; 0 = automatic.
 *   valid_tokens [batch, num_kv_heads] int32 or NULL: token t of table entry e of row
 *                (b, h) exists only if e * page_size + t < valid_tokens[b, h] (a ragged
 *                last page); entries wholly past the bound contribute nothing. The page
 *                memory of tokens past the bound is still read and must hold finite values.
 *   merge_in_kernel  0: a merge kernel combines the split partials after the decode kernel.
 *                1: the decode kernel merges them itself. 2: automatic -- in-kernel for grids
 *                of at least IAK_MERGE_IN_KERNEL_MIN_WORKGROUPS workgroups (where the merges
 *                overlap other workgroups' page streaming) and for the small grids named
 *                beside that constant (one launch instead of two), else the merge kernel. In-kernel,
 *                the four waves of a workgroup
 *                reduce four consecutive splits of one row (the split count is rounded up
 *                to a multiple of four) and combine them in LDS into one partial; the
 *                workgroup that arrives last at the row's arrival counter merges the row's
 *                partials into the output. The counters live at the end of the workspace,
 *                after the partials, so their offset depends on the plan: they must be zero
 *                before a workspace's first use and again whenever a call with another plan
 *                (shape or split count) reuses it; every call leaves its own counters zero
 *                (iak_paged_decode_noalloc ignores this field).
 *   page_desc    NULL, or [num_pages] 32-byte page descriptors (32-byte aligned) written by
 *                iak_pack_page_descriptors: the page's native tag and scales in one line, read
 *                instead of page_tags, tag_map and the scale arrays (which may then be NULL;
 *                a tag whose K/V pools are NULL contributes nothing). Word 0: native tag;
 *                words 1-3: 0; words 4-7: FP8 / INT8 K and V scale (f32), INT4 K group scales
 *                (4 x f16) then V, INT4_RESIDUAL K base, K residual, V base, V residual (f32).
 *                INT4 scales are per quarter of head_dim: quarter q holds the scale of group
 *                q * head_dim / 4 / int4_group.
 *   entry_records NULL, or [batch, num_kv_heads, table_width] 32-byte records (32-byte
 *                aligned) written by iak_pack_entry_records: per table entry the page's native
 *                tag (word 0), its page id (word 1; -1 when the table's id is out of range,
 *                negative ids already wrapped when negative_ids was set at packing), words
 *                2-3: 0, words 4-7 the scales as in page_desc. Read instead of page_table,
 *                page_tags, tag_map, the scale arrays and page_desc (all may then be NULL;
 *                negative_ids is ignored; a tag whose K/V pools are NULL contributes
 *                nothing); page_counts and valid_tokens still apply.
 */
typedef struct {
  int32_t batch, num_q_heads, num_kv_heads, head_dim, page_size, table_width;
  int64_t num_pages;

  const void* q; int32_t q_dtype; int64_t q_stride_b, q_stride_h;
  void* out; int32_t out_dtype; int64_t out_stride_b, out_stride_h;

  const int32_t* page_table;
  const int32_t* page_counts;
  const int32_t* page_tags;
  uint8_t tag_map[8];
  int32_t negative_ids;

  const void* k_fp16; const void* v_fp16;
  const void* k_fp8;  const void* v_fp8;
  const void* k_int8; const void* v_int8;
  const void* k_int4; const void* v_int4;
  const void* k_int4r; const void* v_int4r;

  const void* k_fp8_scale;  const void* v_fp8_scale;  int32_t fp8_scale_dtype;
  const void* k_int8_scale; const void* v_int8_scale; int32_t int8_scale_dtype;
  const void* k_int4_scale; const void* v_int4_scale; int32_t int4_scale_dtype; int32_t int4_group;
  const float* k_int4r_scale; const float* v_int4r_scale;

  float sm_scale;
  int32_t pages_per_split;
  int32_t map_other_tags;
  const int32_t* valid_tokens;
  int32_t merge_in_kernel;
  const void* page_desc;
  const void* entry_records;
} iak_paged_decode_args;

/* ABI version of the loaded library (IAK_ABI_VERSION). */
int iak_abi_version(void);

/* Static description of a status code. */
const char* iak_status_string(iak_status status);

/* Detail of the last non-OK status returned on the calling thread. */
const char* iak_last_error(void);

/* Bytes of device workspace iak_paged_decode needs for these arguments
 * (0 when the whole reduction fits one split). */
iak_status iak_paged_decode_workspace(const iak_paged_decode_args* args, size_t* bytes);

/* The split plan iak_paged_decode uses for these arguments. No counterpart in
 * the reference (its Triton kernel has one program per (batch, head)). */
typedef struct {
  int32_t splits;            /* splits per (batch, kv head) row (1: no merge) */
  int32_t pages_per_split;   /* table entries per split (of the first tier) */
  int32_t merge_in_kernel;   /* 1: the decode kernel merges the splits itself */
  size_t workspace_bytes;    /* = iak_paged_decode_workspace */
  int32_t tail_splits;       /* of `splits`, those of the second tier (0: one tier): the
                                last entries of each row in short splits launched after
                                every row's first tier (automatic plans on large grids) */
  int32_t tail_pages_per_split;   /* table entries per second-tier split (0: one tier) */
} iak_paged_decode_plan_info;
iak_status iak_paged_decode_plan(const iak_paged_decode_args* args, iak_paged_decode_plan_info* info);

/* Page descriptors for `page_desc` (layout above) from the arguments' page_tags,
 * tag_map, map_other_tags and scale arrays, for every one of num_pages pages:
 * the native tag a decode with these arguments would use, and the scales it
 * would load. `page_desc` (32-byte aligned, num_pages x 32 B) is written; the
 * arguments' own page_desc field is ignored. No counterpart in the reference:
 * a layout in which a page's metadata costs one cache line instead of up to
 * three. Async on `stream`. */
iak_status iak_pack_page_descriptors(const iak_paged_decode_args* args, void* page_desc, void* stream);

/* Entry records for `entry_records` (layout above) from the arguments' page_table,
 * negative_ids, page_tags, tag_map, map_other_tags and scale arrays, for all
 * batch x num_kv_heads x table_width entries: the page id, native tag and scales a
 * decode with these arguments would use for each entry. `records` (32-byte aligned,
 * that many x 32 B) is written; the arguments' page_desc and entry_records fields
 * are ignored. No counterpart in the reference: run once per routing decision
 * (after iak_build_page_tables), it turns each split's metadata into one
 * contiguous stream. Async on `stream`. */
iak_status iak_pack_entry_records(const iak_paged_decode_args* args, void* records, void* stream);

/* Selected-page mixed-precision decode attention, split-K over pages with an
 * LSE merge. `workspace` must hold iak_paged_decode_workspace() bytes (may be
 * NULL when that is 0). `stream` is a hipStream_t (NULL = default stream). */
iak_status iak_paged_decode(const iak_paged_decode_args* args, void* workspace,
                            size_t workspace_bytes, void* stream);

/* iak_paged_decode with two hipEvent_t (either may be NULL) recorded on `stream`
 * immediately before and after the split kernel's launch, so a caller can time
 * that kernel apart from the merge. No counterpart in the reference: it is the
 * measurement hook of bench.py's roofline figure. */
iak_status iak_paged_decode_timed(const iak_paged_decode_args* args, void* workspace,
                                  size_t workspace_bytes, void* stream, void* ev_begin, void* ev_end);

/* Maximum split-K partial bytes iak_paged_decode_noalloc serves from its
 * library-owned scratch (what iak_paged_decode_workspace reports for the same
 * arguments). */
#define IAK_NOALLOC_SCRATCH_BYTES (16u << 20)

/* iak_paged_decode without a caller workspace and without any allocation: the
 * split-K partials live in a library-owned device array of
 * IAK_NOALLOC_SCRATCH_BYTES (one per GPU, held until the process ends). It
 * runs the merge kernel on a one-tier split plan (tail_splits = 0), whose
 * partials are at most those of iak_paged_decode_workspace with
 * merge_in_kernel = 0. Arguments whose partials need more return IAK_EINVAL. Every call on a GPU
 * shares that GPU's array, so calls that overlap on one GPU (concurrent
 * streams or threads) race; calls ordered on one stream do not. No
 * counterpart in the reference: it is for callers that cannot allocate
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). */
iak_status iak_paged_decode_noalloc(const iak_paged_decode_args* args, void* stream);

/*
 * MLA latent decode: every query head attends to one shared compressed KV
 * (latent rows of qk_dim values; dims v_offset .. v_offset + v_dim - 1 of a
 * row are also its values). Per sequence b and head h:
 *   s_t = sm_scale * q[b,h,:] . C_t   over the latent rows C_t of the pages
 *         page_table[b, 0 .. page_counts[b]-1] (SKIP pages contribute nothing)
 *   out[b,h,:] = sum_t softmax(s)_t * C_t[v_offset : v_offset + v_dim]   (0 when nothing is visited)
 * Latent pools are [num_pages, page_size, qk_dim]: FP16 values, or FP8-e4m3 / INT8
 * codes with one scale per page (dequantised value = code * scale). Page tags go
 * through tag_map as in iak_paged_decode; INT4 tags are not supported here.
 * Computed with f16 MFMA operands (q rounded to f16) and f32 accumulation.
 * Supported (qk_dim, v_dim): (64,64) (128,128) (256,256) (512,512) (576,512) (576,64).
 */
typedef struct {
  int32_t batch, num_heads, qk_dim, v_dim, v_offset, page_size, table_width;
  int64_t num_pages;

  const void* q; int32_t q_dtype; int64_t q_stride_b, q_stride_h;
  void* out; int32_t out_dtype; int64_t out_stride_b, out_stride_h;

  const int32_t* page_table;   /* [batch, table_width] */
  const int32_t* page_counts;  /* [batch] */
  const int32_t* page_tags;    /* [num_pages]; NULL = every page FP16 */
  uint8_t tag_map[8];
  int32_t negative_ids;
  const int32_t* valid_tokens; /* [batch] or NULL: token t of table entry e exists only if
                                  e * page_size + t < valid_tokens[b] (a ragged last page) */

  const void* c_fp16;          /* [num_pages, page_size, qk_dim] f16 */
  const void* c_fp8;           /* e4m3fn codes */
  const void* c_int8;          /* int8 codes */
  const void* c_fp8_scale; const void* c_int8_scale; int32_t scale_dtype;   /* [num_pages] */

  float sm_scale;
  int32_t pages_per_split;     /* 0 = automatic, else 1 .. 128 */
} iak_mla_decode_args;

/* Bytes of device workspace iak_mla_decode needs (0 when one split covers a sequence). */
iak_status iak_mla_decode_workspace(const iak_mla_decode_args* args, size_t* bytes);

/* MLA latent decode on MFMA, split-K over pages with an LSE merge; async on `stream`. */
iak_status iak_mla_decode(const iak_mla_decode_args* args, void* workspace, size_t workspace_bytes,
                          void* stream);

/* iak_mla_decode with events around the split kernel, as iak_paged_decode_timed
 * (no counterpart in the reference). */
iak_status iak_mla_decode_timed(const iak_mla_decode_args* args, void* workspace, size_t workspace_bytes,
                                void* stream, void* ev_begin, void* ev_end);

/* Timing events for the _timed entry points and for a harness's own brackets (no
 * counterpart in the reference; bench.py's per-launch figures). They are hipEvent_t
 * handles created with hipEventDisableSystemFence: recording one does not write back
 * and invalidate the caches, whose cost a default event adds to the interval it
 * closes after a kernel that wrote many MB (the MLA split kernel's partials). They
 * order nothing for the host: read them with iak_timing_event_elapsed (milliseconds
 * from `start` to `end`) only after a device synchronize. */
iak_status iak_timing_event_create(void** event);
iak_status iak_timing_event_record(void* event, void* stream);
iak_status iak_timing_event_elapsed(void* start, void* end, float* ms);
iak_status iak_timing_event_destroy(void* event);

/*
 * Quantise-on-write: float16 pages [num_pages, page_size, head_dim] -> codes and
 * scales of one pool, page p written to pool page dst_pages[p] (or p when
 * dst_pages is NULL); pages whose destination lies outside [0, pool_pages)
 * are not written. Layouts are those of iak_paged_decode_args.
 *   mode IAK_QUANT_FAKE_QUANTIZE: fake_quantize_tensor (intent_quant.py:221-312) at the
 *        page granule (INT4: page x int4_group channels); precision FP8, INT8, INT4 or
 *        INT4_RESIDUAL; arithmetic in float16 (INT4_RESIDUAL residual in float32).
 *   mode IAK_QUANT_FUSED_INT8:  fake_int8_pages_from_fp16, fused_selected_quant_decode.py:521-542
 *        (float16; clamp(round(x/s), -128, 127)); precision INT8.
 *   mode IAK_QUANT_TRITON_INT8: fake_int8_pages_from_fp16, triton_intent_quant_attention.py:460-496
 *        (float32; clamp(round(x/s), -127, 127)); precision INT8.
 * scale_dtype: F16 or F32 for one scale per page or group; INT4_RESIDUAL writes
 * [pool_pages, 2] f32 (base, residual) pairs.
 */
enum { IAK_QUANT_FAKE_QUANTIZE = 0, IAK_QUANT_FUSED_INT8 = 1, IAK_QUANT_TRITON_INT8 = 2 };

typedef struct {
  int32_t num_pages, page_size, head_dim;
  const void* src;              /* f16 [num_pages, page_size, head_dim] */
  const int32_t* dst_pages;     /* [num_pages] or NULL */
  int64_t pool_pages;
  int32_t precision;            /* IAK_TAG_FP8 / INT8 / INT4 / INT4_RESIDUAL */
  int32_t mode;
  int32_t int4_group;
  void* codes;                  /* pool codes (INT4: head_dim/2 bytes per token) */
  void* scales;                 /* pool scales */
  int32_t scale_dtype;
} iak_quantize_args;

/* Quantise pages into a pool; async on `stream`. */
iak_status iak_quantize_pages(const iak_quantize_args* args, void* stream);

/*
 * Page tables from routed spans (the selected blocks of a routing decision,
 * in routed order), built on the device.
 *
 * Row r (of num_rows = batch * kv_heads; row b * kv_heads + h) reads span list
 * r / rows_per_list and block-table row r / rows_per_seq. Its logical pages
 * are t / page_size for the tokens start <= t < end of each span, span by
 * span, each page once at its first occurrence (dedupe = 1,
 * block_router.py:283-296) or once per span (dedupe = 0). A logical page l
 * maps to block_table[seq * block_table_width + l] (l >= block_table_width or
 * a negative entry: not resident) or to l without a block table; pages whose
 * physical id is outside [0, num_pages) are dropped. Outputs:
 *   page_table [num_rows, table_width]: the first table_width ids, zeros after;
 *   page_counts [num_rows]: min(ids, table_width);
 *   page_precision [num_pages] (optional): the tag of the span that emitted the
 *     page in the lowest row emitting it (the smallest tag if that row emits it
 *     twice), default_tag elsewhere; pages past table_width count.
 * With one list for all rows, no block table and dedupe = 1 the three outputs
 * equal metadata_to_kernel_tensors(routing_to_kernel_metadata(blocks,
 * page_size), num_pages, B, H) whenever every selected page is below
 * num_pages (the reference raises IndexError otherwise).
 * span_offsets has ceil(num_rows / rows_per_list) + 1 entries (CSR into the
 * span arrays); span_tag holds IAK_TAG_* values. Every array is int32 and must
 * be 4-byte aligned (IAK_EINVAL otherwise). Work is proportional to the
 * pages the lists name; a list whose pages span more than 16384 ids tests
 * first occurrence against its earlier spans (quadratic in spans).
 */
typedef struct {
  int32_t num_rows, rows_per_seq, rows_per_list;
  int32_t table_width, page_size, num_pages;
  int32_t dedupe;
  int32_t default_tag;
  int32_t block_table_width;
  const int32_t* span_offsets;
  const int32_t* span_begin;
  const int32_t* span_end;
  const int32_t* span_tag;
  const int32_t* block_table;   /* [num_seqs, block_table_width] or NULL */
  int32_t* page_table;
  int32_t* page_counts;
  int32_t* page_precision;      /* or NULL */
} iak_page_table_args;

/* Build page tables; async on `stream`. */
iak_status iak_build_page_tables(const iak_page_table_args* args, void* stream);

/*
 * KV memory manager page transcoding with the manager's arithmetic
 * (kv_memory_manager.py): pages of page_elems values (page_size x head_dim,
 * a multiple of 8) in two pools indexed by slot, fp16 [pool_pages,
 * page_elems] and int8 [pool_pages, page_elems], with one float32 scale per
 * slot. Page p is slot pages[p] (or p when pages is NULL); slots outside
 * [0, pool_pages) are skipped.
 *   IAK_TRANSCODE_DEMOTE_INT8: fp16 -> int8 codes and scales:
 *       scale = max|x| / 127 (1.0 for an all-zero page or one holding a NaN),
 *       code = clamp(round(float16(x / scale)), -128, 127) (round half to even);
 *   IAK_TRANSCODE_PROMOTE_FP16: int8 codes and scales -> fp16: float16(code * scale).
 * The float32 scale is what the reference's float arithmetic uses of its
 * Python float scale, so both directions are bit-exact to it. The fp16 pool
 * must be 16-byte aligned, the int8 pool 8-byte aligned. A slot listed twice
 * in one call is transcoded twice, concurrently (the result of a race).
 */
enum { IAK_TRANSCODE_DEMOTE_INT8 = 0, IAK_TRANSCODE_PROMOTE_FP16 = 1 };

typedef struct {
  int32_t num_pages;
  int32_t page_elems;
  int32_t mode;
  const int32_t* pages;         /* [num_pages] slots, or NULL */
  int64_t pool_pages;
  void* fp16;                   /* float16 [pool_pages, page_elems] */
  void* int8;                   /* int8 [pool_pages, page_elems] */
  float* scales;                /* float32 [pool_pages] */
} iak_transcode_args;

/* Transcode pages between the FP16 and INT8 pools; async on `stream`. */
iak_status iak_transcode_pages(const iak_transcode_args* args, void* stream);

/*
 * Page warm-up: reads the K and V rows of pages page_ids[0 .. num_ids-1]
 * (pages of page_size tokens; tokens at or past kv_len skipped) of every
 * (batch, head) of k, v [batch, heads, kv_len, head_dim] (16-bit elements,
 * element strides, unit last stride) with cached loads, so a following decode
 * finds them in the L2 / Infinity Cache. Correctness-neutral. The words read
 * are folded into checksum [batch * heads * num_ids * 4] (one per wave:
 * element i of a page enters as value << (16 (i & 1)), XOR-folded).
 */
typedef struct {
  int32_t batch, heads, kv_len, head_dim, page_size, num_ids;
  const int32_t* page_ids;
  const void* k; const void* v;
  int64_t k_stride_b, k_stride_h, k_stride_t;
  int64_t v_stride_b, v_stride_h, v_stride_t;
  uint32_t* checksum;
} iak_prefetch_args;

/* Warm pages into the caches; async on `stream`. */
iak_status iak_prefetch_pages(const iak_prefetch_args* args, void* stream);

/* Latent context of the reference's MLA decode API (mla_decode_triton,
 * triton_mla_decode.py:47-107 / _mla_decode_cpu :155-186), in float32: for each
 * (batch, query position) row, softmax((q . c) * sm_scale) over the latent rows
 * of the listed pages, context = sum(p c) / sum(p), zeros when nothing is
 * visited. Page p is rows p * page_size .. (p + 1) * page_size - 1 of the
 * latents (the last page may be shorter); ids outside [0, ceil(num_rows /
 * page_size)) are rejected by the caller's contract and skipped by the kernel.
 *
 *   q        [batch, q_len, latent_dim] (q_dtype), element strides q_stride_b / q_stride_t
 *   latents  [num_rows, latent_dim] (latent_dtype), element row stride latent_stride
 *   page_ids [num_selected] int32, shared by every row
 *   context  [batch, q_len, latent_dim] float32, contiguous (written)
 *   latent_dim <= 1024; any page_size >= 1; num_selected * page_size <= INT32_MAX - 4096.
 * workspace (may be NULL): with it, a call with fewer than 512 rows and at least
 * 256 listed latent rows splits each row's keys over several workgroups and
 * merges their partials in a second kernel; it must then hold
 * iak_mla_decode_rows_workspace() bytes (16-byte aligned; 0 bytes: not split).
 * Without it every row runs in one workgroup. The results agree to float32
 * rounding of the summation order. Calls that share a workspace on different
 * streams race. */
typedef struct {
  int32_t batch, q_len, latent_dim, page_size, num_selected;
  int64_t num_rows;
  const void* q; int32_t q_dtype; int64_t q_stride_b, q_stride_t;
  const void* latents; int32_t latent_dtype; int64_t latent_stride;
  const int32_t* page_ids;
  float* context;
  float sm_scale;
} iak_mla_rows_args;

/* Bytes of device workspace that lets iak_mla_decode_rows split these rows (0: no split). */
iak_status iak_mla_decode_rows_workspace(const iak_mla_rows_args* args, size_t* bytes);

iak_status iak_mla_decode_rows(const iak_mla_rows_args* args, void* workspace, size_t workspace_bytes,
                               void* stream);

/* The projection of those contexts by W_VO in float32 (triton_mla_decode.py:146-151), for a
 * decode step's rows: out[row, n] = sum over k of context[row, k] w[k, n].
 *   context [rows, latent_dim] float32, contiguous, 16-byte aligned; latent_dim a multiple of 8
 *   w       [latent_dim, d_out] (w_dtype), element row stride w_stride; d_out a multiple of 32
 *   out     [rows, d_out] (out_dtype), contiguous (written) */
typedef struct {
  int32_t rows, latent_dim, d_out;
  const float* context;
  const void* w; int32_t w_dtype; int64_t w_stride;
  void* out; int32_t out_dtype;
} iak_mla_project_args;

iak_status iak_mla_project(const iak_mla_project_args* args, void* stream);

/* Dense softmax attention of the reference's dense_attention() (reference.py:16-45)
 * in float32: for each (batch, query) row i,
 *   s_j = (q_i . k_j) * sm_scale
 *         + (-inf if causal == IAK_CAUSAL_TRIU and j > i)
 *   s_j = -inf if causal == IAK_CAUSAL_POSITIONS and i < kv_positions[j]
 *   s_j += mask[b, i, j]                       (bool masks add 1.0 where true)
 *   out_i = softmax(s) . v
 * NaN when every s_j is -inf (torch's softmax), zeros when kv_len == 0.
 *
 *   q    [batch, q_len, head_dim], k [batch, kv_len, head_dim], v [batch, kv_len, v_dim],
 *   out  [batch, q_len, v_dim]: one dtype (IAK_DTYPE_*), element strides per batch and row,
 *        unit inner stride; a batch stride of 0 broadcasts
 *   mask (may be NULL) element (b, i, j) at b * mask_stride_b + i * mask_stride_q + j * mask_stride_k,
 *        mask_dtype IAK_DTYPE_* or IAK_MASK_BOOL (one byte)
 *   kv_positions [kv_len] int64 (IAK_CAUSAL_POSITIONS only)
 *   head_dim, v_dim <= 1024; kv_len <= INT32_MAX - 4096.
 * workspace (may be NULL): with it, calls with several query rows per batch entry
 * and 16-byte aligned rows run on the matrix cores, and a call with few rows and
 * many keys splits each row's keys over several workgroups and merges their
 * partials in a second kernel; it must then hold iak_dense_attention_workspace()
 * bytes (16-byte aligned; 0 bytes means neither applies and the workspace is
 * unused; IAK_DENSE_NO_SCRATCH bytes means that the matrix cores do without one: any 16
 * bytes of device memory, which stay as they are, ask for them). Without it every row runs in one workgroup. The results agree to
 * float32 rounding of the summation order, NaN and infinities included. Calls
 * that share a workspace on different streams race. */
enum { IAK_MASK_BOOL = 3 };
enum { IAK_DENSE_NO_SCRATCH = 16 };
enum { IAK_CAUSAL_NONE = 0, IAK_CAUSAL_TRIU = 1, IAK_CAUSAL_POSITIONS = 2 };
typedef struct {
  int32_t batch, q_len, kv_len, head_dim, v_dim, dtype;
  const void* q; int64_t q_stride_b, q_stride_t;
  const void* k; int64_t k_stride_b, k_stride_t;
  const void* v; int64_t v_stride_b, v_stride_t;
  void* out; int64_t out_stride_b, out_stride_t;
  const void* mask; int32_t mask_dtype; int64_t mask_stride_b, mask_stride_q, mask_stride_k;
  int32_t causal;
  const int64_t* kv_positions;
  float sm_scale;
} iak_dense_attention_args;

/* Bytes of device workspace that lets iak_dense_attention split these rows or run them on
 * the matrix cores (0: neither). */
iak_status iak_dense_attention_workspace(const iak_dense_attention_args* args, size_t* bytes);

iak_status iak_dense_attention(const iak_dense_attention_args* args, void* workspace, size_t workspace_bytes,
                               void* stream);

/* The same over selected tokens, read where they are: key j is row kv_index[j] of k and v
 * (kv_index [kv_len] int64 on the device, or NULL: row j). The caller keeps every index
 * non-negative, inside k and v and below 2^31; masks and positions stay by j. */
iak_status iak_dense_attention_indexed(const iak_dense_attention_args* args, const int64_t* kv_index,
                                       void* workspace, size_t workspace_bytes, void* stream);

/* Fake-quant reconstruction of the selected blocks of float32 K and V, as
 * intent_quant_attention_reference() concatenates them (intent_quant_attention.py:56-84,
 * fake_quantize_tensor intent_quant.py:221-312): block i's tokens blocks[i][0] ..
 * blocks[i][0] + blocks[i][1] - 1 of K and V, reconstructed at precision blocks[i][3]
 * (IAK_FQ_*) with one scale per channel (absmax over every leading row and token of
 * the block), land at tokens blocks[i][2] .. of out, K's channels first, then V's.
 *   k [lead, T, k_dim], v [lead, T, v_dim] float32, element strides per leading row and
 *     token, unit channel stride; k_dim + v_dim <= 2^20
 *   blocks [num_blocks][4] int32 on the device (num_blocks < 2^22); the caller keeps the token ranges inside
 *     K, V and out (the kernel does not check them)
 *   out [lead, total, k_dim + v_dim] float32, element strides per leading row and token
 *   max_block_tokens: the longest block's token count, or an upper bound on it (it sizes
 *     the split below; a wrong value changes the speed, never the result)
 * Every division is the IEEE float32 quotient and every code rounds to nearest even,
 * as torch's float32 arithmetic, so the result equals the reference's bit for bit
 * (an integer code of zero gives +0, as .to(int8).float() does).
 * Without a workspace one workgroup takes each (block, 64 channels); with one of the
 * size iak_fake_quant_blocks_workspace() gives (0: no split for these arguments), a
 * block of many rows (leading rows x tokens) is split over several workgroups per
 * channel group, whose per-channel maxima meet in the workspace over three launches. */
enum { IAK_FQ_FP16 = 0, IAK_FQ_FP8 = 1, IAK_FQ_INT8 = 2, IAK_FQ_INT4 = 3, IAK_FQ_INT4_RESIDUAL = 4, IAK_FQ_SKIP = 5 };
typedef struct {
  int32_t lead, num_blocks, k_dim, v_dim;
  const float* k; int64_t k_stride_l, k_stride_t;
  const float* v; int64_t v_stride_l, v_stride_t;
  const int32_t* blocks;
  int32_t max_block_tokens;
  float* out; int64_t out_stride_l, out_stride_t;
} iak_fake_quant_blocks_args;

/* Bytes of device workspace that lets iak_fake_quant_blocks split long blocks (0: no split). */
iak_status iak_fake_quant_blocks_workspace(const iak_fake_quant_blocks_args* args, size_t* bytes);

iak_status iak_fake_quant_blocks(const iak_fake_quant_blocks_args* args, void* workspace, size_t workspace_bytes,
                                 void* stream);

/*
 * Microscaled 4-bit (MXFP4) token cache. Pages of 16 tokens of one KV head, as the
 * decode's pools: codes [num_pages, 16, head_dim / 2] bytes (channel 2j in the low half of
 * byte j; a code is sign << 3 | e2m1 magnitude 0, .5, 1, 1.5, 2, 3, 4, 6) and scale bytes
 * [num_pages, 16, head_dim / 32], one per token and 32 channels:
 *   value = code * 2^(clamp(scale, 104, 140) - 127);  scale 255: the block is NaN.
 * The clamp (2^-23 .. 2^13) makes every value a float16 number, and whatever bytes lie in
 * tokens that nobody wrote finite ones. head_dim 64 or 128, page_size 16.
 *
 * Row (b, h) of page_table [batch, num_kv_heads, table_width] lists its pages in token
 * order; valid_tokens [batch, num_kv_heads] counts its tokens, clamped to 0 ..
 * 16 * table_width: a longer row is a full one to every call, so that its newest tokens are
 * the table's last slots (an append writes them over what is there; iak_grow_sequences
 * lets no row become longer than its table). The newest n tokens of a sequence are its last:
 * with q_lens [batch] (NULL: count for all; clamped to 0 .. count) token i < q_lens[b] is
 * number valid_tokens[b, h] - q_lens[b] + i of row (b, h). Page ids outside [0, num_pages)
 * hold no tokens.
 */

/* Write (append) or read the newest tokens: k, v [batch, count, num_kv_heads, head_dim]
 * (dtype IAK_DTYPE_*), element strides, unit channel stride.
 * Append rounds a block x of 32 channels as the microscaling standard does:
 *   e = clamp(floor(log2(max|x|)) - 2, -23, 13), scale = e + 127,
 *   code = round to nearest even of x / 2^e, at most 6; a block that holds an infinity or a
 *   NaN: scale 255, codes 0.
 * It writes bytes of the addressed tokens only; tokens without a page are left out. Two
 * tokens that address one slot race. Read gives the values (exact in every dtype), and
 * zeros for tokens without a page and for i >= q_lens[b]. Code pools 4-byte aligned. */
typedef struct {
  int32_t batch, count, num_kv_heads, head_dim, page_size, table_width;
  int64_t num_pages;
  void* k; int64_t k_stride_b, k_stride_t, k_stride_h;
  void* v; int64_t v_stride_b, v_stride_t, v_stride_h;
  int32_t dtype;
  const int32_t* page_table;
  const int32_t* valid_tokens;
  const int32_t* q_lens;
  void* k_codes; void* k_scales; void* v_codes; void* v_scales;
} iak_mx_tokens_args;

iak_status iak_mx_append_tokens(const iak_mx_tokens_args* args, void* stream);
iak_status iak_mx_read_tokens(const iak_mx_tokens_args* args, void* stream);

/* Attention over the cache: q, out [batch, q_len, num_q_heads, head_dim] (element strides,
 * unit inner stride). Query i < q_lens[b] (as above, q_len for count) of head h reads row
 * (b, h / (num_q_heads / num_kv_heads)) and sees, with causal = 1, the tokens up to its own
 * (numbers below valid_tokens - q_lens[b] + i + 1), else all of the row's:
 *   out = softmax(sm_scale * q . k) v over them, 0 where there are none and for
 *   i >= q_lens[b].
 * A token with a NaN block makes every query that sees it NaN, as does a query that is
 * not finite itself; tokens that a query does not see never reach it. Products run on the
 * matrix cores in float16 with float32 sums; K and V are exact there. A query row is scaled by
 * a power of two that brings its largest element to 2^14 .. 2^15: float16 and bfloat16
 * elements are exact down to 2^-28 of the row's largest, smaller ones off by at most 2^-39 of
 * it; float32 elements are split in two, off by at most 2^-22 of themselves or 2^-39 of the
 * largest. (A score is so off by up to |sm_scale| 2^-39 max|q| sum|k|, which counts only where
 * the query's largest channels meet keys that are smaller by as much.) Weights are rounded to
 * 11 bits, those of float32 queries split in two (22 bits).
 * Scores, with the scale, have to be float32 numbers in base 2. Code pools are 16-byte, scale
 * pools 4-byte aligned; q and out lie at any address of their type, and out may be q.
 * splits: parts a row's tokens are divided into (0: automatic). The parts meet in the
 * workspace (iak_mx_attention_workspace bytes, 16-byte aligned, as it comes; 0: not needed);
 * calls that share one on different streams race. */
typedef struct {
  int32_t batch, q_len, num_q_heads, num_kv_heads, head_dim, page_size, table_width;
  int64_t num_pages;
  const void* q; int32_t q_dtype; int64_t q_stride_b, q_stride_t, q_stride_h;
  void* out; int32_t out_dtype; int64_t out_stride_b, out_stride_t, out_stride_h;
  const int32_t* page_table;
  const int32_t* valid_tokens;
  const int32_t* q_lens;
  const void* k_codes; const void* k_scales; const void* v_codes; const void* v_scales;
  float sm_scale;
  int32_t causal;
  int32_t splits;
} iak_mx_attention_args;

iak_status iak_mx_attention_workspace(const iak_mx_attention_args* args, size_t* bytes);
iak_status iak_mx_attention(const iak_mx_attention_args* args, void* workspace, size_t workspace_bytes,
                            void* stream);

/* One array with a row per page: page p is the row_bytes bytes at base + p * row_bytes. */
typedef struct {
  void* base;
  int64_t row_bytes;
} iak_page_array;
#define IAK_MAX_PAGE_ARRAYS 24

/* Copy pages: row src[i] of every array to row dst[i], i < count (int32 on the device).
 * Pairs with an id outside [0, num_pages) are left out. The dst ids are distinct and none
 * of them is a src of another pair (such pairs race). Async on `stream`. */
typedef struct {
  int32_t num_arrays;
  iak_page_array arrays[IAK_MAX_PAGE_ARRAYS];
  int64_t num_pages;
  int32_t count;
  const int32_t* src;
  const int32_t* dst;
} iak_copy_pages_args;
iak_status iak_copy_pages(const iak_copy_pages_args* args, void* stream);

/* Sequences over shared pages. refs [num_pages] counts the table entries (and other owners)
 * that hold a page; a page with refs <= 0 is free. page_table [num_seqs, rows_per_seq,
 * table_width], valid_tokens [num_seqs, rows_per_seq]: entries 0 .. ceil(valid / page_size)
 * - 1 of a row are in use. All int32, on the device, changed in place.
 *   iak_free_sequences  lets go of the newest new_tokens[i] tokens (NULL: of all) in each row of
 *       sequence seqs[i], of as many as there are: the lengths sink, and entries that are no
 *       longer in use become -1, refs - 1. Indices outside [0, num_seqs) and negative numbers
 *       are left out; a sequence listed twice loses tokens twice.
 *   iak_grow_sequences  sequence seqs[i] gets new_tokens[i] more tokens in each of its rows:
 *       entries for them come from the free pages, the lowest id first, in the order of
 *       (i, row, entry), with refs = 1. A row that gets tokens and whose last page has room
 *       but refs > 1 (sequences forked and then cut back share such pages) is given a page of
 *       its own in that entry, a copy (every array), and lets go of the other, so that what is
 *       appended reaches no other owner; without arrays such a call is refused.
 *       granted [num_seqs] (may be NULL; no other array of the
 *       call) is written whole: new_tokens[i] of sequence seqs[i] if the call was done, 0 of
 *       every other and of all if it was not. As the q_lens of what follows on the stream it
 *       keeps tokens that got no room from being appended over older ones.
 *   iak_fork_sequences  sequence seqs[i], which has no tokens, becomes a copy of parents[i]:
 *       it shares the parent's pages (refs + 1), except that a last page which is not full
 *       is copied (every array) into a free page, chosen in the order of (i, row). (Without arrays
 *       such a page holds what it held: the caller's to fill, as iak_reorder_sequences' too.)
 * Grow and fork do all of it or nothing and say which in missing[0]: 0 done; n > 0: n more
 * free pages would be needed; -1: an index outside [0, num_seqs) or listed twice among
 * seqs, a negative new_tokens, a row that would be longer than its table, a shared last page
 * and no arrays, a forked sequence with tokens, or one that is also a parent. Results do not depend on timing. Workspace:
 * iak_sequences_workspace bytes, 16-byte aligned (free needs none). */
typedef struct {
  int32_t num_seqs, rows_per_seq, table_width, page_size;
  int64_t num_pages;
  int32_t* page_table;
  int32_t* valid_tokens;
  int32_t* refs;
  int32_t count;
  const int32_t* seqs;
  const int32_t* parents;      /* fork, reorder */
  const int32_t* new_tokens;   /* grow; free: may be NULL */
  int32_t* missing;            /* grow, fork, reorder */
  int32_t num_arrays;          /* grow, fork, reorder */
  iak_page_array arrays[IAK_MAX_PAGE_ARRAYS];
  int32_t* granted;            /* grow; may be NULL */
} iak_sequences_args;

iak_status iak_sequences_workspace(const iak_sequences_args* args, size_t* bytes);
iak_status iak_free_sequences(const iak_sequences_args* args, void* stream);
iak_status iak_grow_sequences(const iak_sequences_args* args, void* workspace, size_t workspace_bytes, void* stream);
iak_status iak_fork_sequences(const iak_sequences_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* Sequence seqs[i] becomes a copy of what parents[i] was before the call, all at once: parents may
 * be listed as seqs themselves, and any number of times (seqs[i] = parents[i]: it stays as it is). Rows
 * share the parent's pages (refs + 1) and let go of their own (refs - 1; entries no longer in use
 * become -1). A last page that is not full stays with one owner: the parent if it stays itself or is not among
 * seqs, else its first child in the call; the others get copies of it (every array) in free pages, the lowest ids
 * first, in the order of (i, row): pages that were free before the call. All of it or nothing:
 * missing[0] is 0 done; n > 0: n more free pages would be needed; -1: an index outside
 * [0, num_seqs) or listed twice among seqs. seqs, parents and missing are none of the arrays that
 * are changed. Workspace: iak_reorder_sequences_workspace bytes, 16-byte aligned. */
iak_status iak_reorder_sequences_workspace(const iak_sequences_args* args, size_t* bytes);
iak_status iak_reorder_sequences(const iak_sequences_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* Compaction: with L pages in use (refs > 0), those with ids >= L move to the free ids
 * below L, the highest to the lowest: page_map [num_pages] is the new id of every page (-1:
 * free), out_refs [num_pages] the counts by new id, out_table [num_rows, table_width] the
 * table with its entries in use mapped (-1 for one that names a free page; the others as
 * they are). The arrays' rows are copied in place; old rows keep their bytes, and page_table and refs stay as they are, so
 * work that still reads the old table finds its pages. No output may overlap an input. */
typedef struct {
  int32_t num_rows, table_width, page_size;
  int64_t num_pages;
  const int32_t* page_table;
  const int32_t* valid_tokens;   /* [num_rows] */
  const int32_t* refs;
  int32_t* out_table;
  int32_t* out_refs;
  int32_t* page_map;
  int32_t num_arrays;
  iak_page_array arrays[IAK_MAX_PAGE_ARRAYS];
} iak_compact_pages_args;

iak_status iak_compact_pages_workspace(const iak_compact_pages_args* args, size_t* bytes);
iak_status iak_compact_pages(const iak_compact_pages_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* Attention of several query tokens per sequence (drafted tokens, prompt chunks) over the pages of
 * iak_paged_decode: pools, scales, page_table, page_counts, page_tags, tag_map, map_other_tags and
 * negative_ids as there. q, out [batch, q_len, num_q_heads, head_dim] (element strides, unit inner
 * stride, any address of their type; out may be q).
 * Token t of entry e of a row is its number 16 e + t; the row holds min(valid_tokens, 16 *
 * page_counts) of them (valid_tokens [batch, num_kv_heads] may be NULL: 16 * page_counts), the
 * queries' own the last: with q_lens [batch] (NULL: q_len for all; clamped to 0 .. q_len) query
 * i < q_lens[b] of head h reads row (b, h / (num_q_heads / num_kv_heads)) and sees, with causal =
 * 1, the tokens numbered below tokens - q_lens[b] + i + 1, else all:
 *   out = softmax(sm_scale * q . k) v over those on pages that contribute (tags and ids as for the decode),
 * 0 where there are none and for i >= q_lens[b].
 * Tokens that a query does not see never reach it, whatever their bytes; an infinite or NaN value of one that it
 * sees reaches its channel. A query row that is not finite is NaN if it sees a token.
 * Products run on the matrix cores in float16 with float32 sums: K and V as exact codes, with
 * their scales in float32 (float32 sums of log2 in the exponential), or in two parts (4-bit pages: 21 bits; groups
 * whose scale is below 1/16 of the page's largest lose 2^-25 of that); query rows
 * and weights as for iak_mx_attention (weights of 16-bit queries in 11 bits). V scales lie anywhere in float32's normal
 * range (below it they may count as zero), those of one row may differ by 2^18 without loss. int4_group is head_dim, its
 * half or its quarter (IAK_ENOTSUP else).
 * splits: parts a row's tokens are divided into (0: automatic). The parts meet in the workspace
 * (iak_paged_chunk_workspace bytes, 16-byte aligned, as it comes; 0: not needed); calls that share one
 * on different streams race. head_dim 64 or 128, page_size 16; pools 16-byte aligned. */
typedef struct {
  int32_t batch, q_len, num_q_heads, num_kv_heads, head_dim, page_size, table_width;
  int64_t num_pages;
  const void* q; int32_t q_dtype; int64_t q_stride_b, q_stride_t, q_stride_h;
  void* out; int32_t out_dtype; int64_t out_stride_b, out_stride_t, out_stride_h;
  const int32_t* page_table;
  const int32_t* page_counts;
  const int32_t* valid_tokens;
  const int32_t* q_lens;
  const int32_t* page_tags;
  uint8_t tag_map[8];
  int32_t map_other_tags, negative_ids;
  const void* k_fp16; const void* v_fp16;
  const void* k_fp8; const void* v_fp8;
  const void* k_int8; const void* v_int8;
  const void* k_int4; const void* v_int4;
  const void* k_int4r; const void* v_int4r;
  const void* k_fp8_scale; const void* v_fp8_scale; int32_t fp8_scale_dtype;
  const void* k_int8_scale; const void* v_int8_scale; int32_t int8_scale_dtype;
  const void* k_int4_scale; const void* v_int4_scale; int32_t int4_scale_dtype;
  int32_t int4_group;
  const float* k_int4r_scale; const float* v_int4r_scale;
  float sm_scale;
  int32_t causal;
  int32_t splits;
} iak_paged_chunk_args;

iak_status iak_paged_chunk_workspace(const iak_paged_chunk_args* args, size_t* bytes);
iak_status iak_paged_chunk(const iak_paged_chunk_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* The newest tokens' keys, rotated by their positions, and values into their sequences' pages,
 * and their queries rotated along. A pair of channels (x, y) of a token at position p becomes
 *   (x cos a - y sin a, x sin a + y cos a),  a = p * inv_freq[i],
 * pair i < rotary_dim / 2 being channels (i, i + rotary_dim / 2), or with interleaved = 1
 * (2i, 2i + 1); channels from rotary_dim on stay as they are. inv_freq [rotary_dim / 2] float32 on the
 * device; a is taken in 64 bits, so that far positions lose nothing.
 *   k, v       [batch, count, num_kv_heads, head_dim], q, q_out [batch, count, num_q_heads,
 *              head_dim] (q and q_out may both be NULL; q_out may be q), one dtype
 *              (IAK_DTYPE_*), element strides, unit channel stride
 *   positions  [batch, count] int32, rows position_stride_b apart; NULL: a token's number in
 *              its row, valid_tokens - q_lens + i (a query's in the row of its KV head)
 * page_table, valid_tokens and q_lens as for iak_mx_append_tokens: token i < q_lens[b] is number
 * valid_tokens[b, h] - q_lens[b] + i of row (b, h); tokens before 0 or without a page are left
 * out. Written to k_pages, v_pages, float16 [num_pages, 16, head_dim] (rotated in float32, rounded once;
 * past float16's range: infinite), or else to the 4-bit pools k_codes .. v_scales, rounded as iak_mx_append_tokens rounds, from 64
 * bits. With page_tags [num_pages] (float16 pages only) every page that a token goes to gets `tag`.
 * q_out is written whole: zeros for i >= q_lens[b]. Two tokens that address one slot race.
 * head_dim 64 or 128, page_size 16, rotary_dim a multiple of 16. Code pools 4-byte aligned. */
typedef struct {
  int32_t batch, count, num_q_heads, num_kv_heads, head_dim, rotary_dim, interleaved, page_size, table_width;
  int64_t num_pages;
  int32_t dtype;
  const void* q; int64_t q_stride_b, q_stride_t, q_stride_h;
  void* q_out; int64_t q_out_stride_b, q_out_stride_t, q_out_stride_h;
  const void* k; int64_t k_stride_b, k_stride_t, k_stride_h;
  const void* v; int64_t v_stride_b, v_stride_t, v_stride_h;
  const float* inv_freq;
  const int32_t* positions; int64_t position_stride_b;
  const int32_t* page_table;
  const int32_t* valid_tokens;
  const int32_t* q_lens;
  void* k_pages; void* v_pages;
  void* k_codes; void* k_scales; void* v_codes; void* v_scales;
  int32_t* page_tags;
  int32_t tag;
} iak_rotary_append_args;

iak_status iak_rotary_append(const iak_rotary_append_args* args, void* stream);

/* A beam search's choice: of the continuations of each request's beams the `count` best.
 * Candidate (k, v) of request b is beam k continued with token v:
 *   scores[b, k] + logits[b, k, v] - log(sum_u exp(logits[b, k, u]))
 * logits [batch, beams, vocab] (dtype IAK_DTYPE_*, element strides, unit vocabulary stride);
 * scores [batch, beams] float32, the beams' sums of log-probabilities. finished [batch, beams]
 * bytes (may be NULL): a beam whose byte is not 0 goes on as it is: its one candidate is
 * end_token with scores[b, k], the other tokens' are -inf. A beam whose score is not finite,
 * or that is not finished and has a logit that is NaN or +inf or none above -inf, is out of the search:
 * all its candidates are -inf. Written, best first:
 *   out_scores [batch, count] float32, out_tokens [batch, count] int32, and
 *   out_parents [batch, count] int32: the beam's row b * beams + k.
 * Equal candidates come in the order of k * vocab + v, those of -inf too. Candidates are compared
 * in 64 bits, with the beams' normalisers off by about 1e-9 (they decide between different beams;
 * those of one beam come in the order of their logits) and rounded to float32 at the end.
 * 1 <= count <= 64, count <= beams * vocab < 2^31, beams <= 256, batch < 2^23. Workspace:
 * iak_beam_select_workspace bytes, 16-byte aligned, as it comes; calls that share one on different
 * streams race. */
typedef struct {
  int32_t batch, beams, vocab, count;
  const void* logits; int32_t dtype; int64_t stride_b, stride_k;
  const float* scores;
  const uint8_t* finished;
  int32_t end_token;
  float* out_scores;
  int32_t* out_parents;
  int32_t* out_tokens;
} iak_beam_select_args;

iak_status iak_beam_select_workspace(const iak_beam_select_args* args, size_t* bytes);
iak_status iak_beam_select(const iak_beam_select_args* args, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* IAK_H */
