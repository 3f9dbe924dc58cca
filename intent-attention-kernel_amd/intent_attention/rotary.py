"""Tokens rotated by their positions and written into a paged cache on the MI355X
(``iak_rotary_append``, include/iak.h).

The decode's float16 pages (``PagePools``) and the 4-bit cache (``MxFp4Pools``) take the newest
tokens of every sequence here; pages of the other precisions are quantised whole
(``quantize_pages``) once they are full. Room for the tokens comes from ``grow_sequences``.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _native as N
from .decode_core import PAGE_SIZE, PagePools, _DT, _check_pool, _ptr, current_stream_handle
from .mxfp4 import MxFp4Pools, _check_cache, _check_int32, _device, _launch


def _check_metadata(page_table: torch.Tensor, valid_tokens: torch.Tensor, q_lens: Optional[torch.Tensor], B: int, Hkv: int) -> int:
    """The table's width, or ValueError."""
    if page_table.dim() != 3 or page_table.shape[:2] != (B, Hkv) or page_table.dtype is not torch.int32:
        raise ValueError(f"page_table must be int32 [{B}, {Hkv}, W], got {page_table.dtype} {tuple(page_table.shape)}")
    W = page_table.shape[2]
    _check_int32(table_width=W * PAGE_SIZE, rows=B * Hkv)
    if valid_tokens.shape != (B, Hkv) or valid_tokens.dtype is not torch.int32:
        raise ValueError(f"valid_tokens must be int32 [{B}, {Hkv}], got {valid_tokens.dtype} {tuple(valid_tokens.shape)}")
    if q_lens is not None and (q_lens.shape != (B,) or q_lens.dtype is not torch.int32):
        raise ValueError(f"q_lens must be int32 [{B}], got {q_lens.dtype} {tuple(q_lens.shape)}")
    return W


def append_rotated_tokens(k: torch.Tensor, v: torch.Tensor, pools: Union[PagePools, MxFp4Pools], page_table: torch.Tensor,
                          valid_tokens: torch.Tensor, inv_freq: torch.Tensor, *, q: Optional[torch.Tensor] = None,
                          q_out: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                          positions: Optional[torch.Tensor] = None, interleaved: bool = False,
                          page_tags: Optional[torch.Tensor] = None, fp16_tag: int = 0) -> Optional[torch.Tensor]:
    """Write the newest tokens' keys, rotated, and values into their pages; the queries rotated, or None.

    k, v [B, L, Hkv, D] and q [B, L, Hq, D] (optional) in one dtype (float16, bfloat16 or float32, any
    strides), D = 64 or 128. inv_freq [R / 2] float32: channels i and i + R / 2 (``interleaved``: 2i and
    2i + 1) turn by position * inv_freq[i], those from R on stay; R is a multiple of 16. positions
    [B, L] int32, default: a token's number in its row (a query's in the row of its KV head).
    ``page_table`` [B, Hkv, W], ``valid_tokens`` and ``q_lens`` as for ``append_mxfp4_tokens``: the lengths
    count the new tokens, token i < q_lens[b] is number valid_tokens - q_lens[b] + i of its row, tokens before 0 or
    without a page are left out, and nothing else of the pools is written.
    ``pools``: ``PagePools``, whose float16 pages are written (rotated in float32, rounded once; values
    past float16's range become infinite; with ``page_tags`` [NP] int32 each page that gets a token is tagged
    ``fp16_tag``, as a page handed out again may carry the tag of its former content), or ``MxFp4Pools``,
    rounded as ``append_mxfp4_tokens`` rounds.
    Returns the rotated queries in q's dtype (in ``q_out``, which may be q), zero for i >= q_lens[b]. Inference
    only: nothing records gradients."""
    shape = k.shape
    if len(shape) != 4 or shape != v.shape:
        raise ValueError(f"k and v must have one shape [B, L, Hkv, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in _DT or v.dtype != k.dtype:
        raise ValueError(f"k and v must both be float16, bfloat16 or float32, got {k.dtype} and {v.dtype}")
    B, L, Hkv, D = shape
    packed = isinstance(pools, MxFp4Pools)
    if not packed and (pools.k_fp16 is None or pools.v_fp16 is None):
        raise ValueError("PagePools without float16 pages take no tokens")
    written = tuple(pools.tensors().values()) if packed else (pools.k_fp16, pools.v_fp16)
    dev = _device("rotated append", k, v, page_table, valid_tokens, inv_freq, q, q_out, q_lens, positions, page_tags, *written)
    Hq = 0
    if q is not None:
        Hq = q.shape[2] if q.dim() == 4 else -1
        if q.shape != (B, L, Hq, D) or q.dtype != k.dtype:
            raise ValueError(f"q must be {k.dtype} [{B}, {L}, Hq, {D}], got {q.dtype} {tuple(q.shape)}")
        if Hkv == 0 or Hq == 0 or Hq % Hkv:
            raise ValueError(f"query heads {Hq} must be a multiple of page-table heads {Hkv}")
    if inv_freq.dim() != 1 or inv_freq.dtype is not torch.float32:
        raise ValueError(f"inv_freq must be float32 [R / 2], got {inv_freq.dtype} {tuple(inv_freq.shape)}")
    if positions is not None and (positions.shape != (B, L) or positions.dtype is not torch.int32):
        raise ValueError(f"positions must be int32 [{B}, {L}], got {positions.dtype} {tuple(positions.shape)}")
    if packed:
        heads, W, NP = _check_cache(pools, page_table, valid_tokens, q_lens, B, D)
        if heads != Hkv:
            raise ValueError(f"page_table has {heads} KV heads, k has {Hkv}")
        if page_tags is not None:
            raise ValueError("page_tags belong to PagePools")
    else:
        W = _check_metadata(page_table, valid_tokens, q_lens, B, Hkv)
        NP = pools.k_fp16.shape[0] if pools.k_fp16.dim() else -1
        for t in written:
            if t.dtype is not torch.float16 or t.shape != (NP, PAGE_SIZE, D) or not t.is_contiguous():
                _check_pool("k_fp16" if t is written[0] else "v_fp16", t, NP, (PAGE_SIZE, D), (torch.float16,))
        if page_tags is not None and (page_tags.shape != (NP,) or page_tags.dtype is not torch.int32 or not page_tags.is_contiguous()):
            raise ValueError(f"page_tags must be contiguous int32 [{NP}], got {page_tags.dtype} {tuple(page_tags.shape)}")
    _check_int32(count=L, fp16_tag=fp16_tag)
    k_stride, v_stride = k.stride(), v.stride()
    if k_stride[3] != 1 or v_stride[3] != 1:
        k, v = k.contiguous(), v.contiguous()
        k_stride, v_stride = k.stride(), v.stride()
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    else:
        if q.stride(-1) != 1 and q_out is not q:
            q = q.contiguous()
        if q_out is None:
            q_out = torch.empty((B, L, Hq, D), dtype=q.dtype, device=dev)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(-1) != 1:
            raise ValueError(f"q_out must be {q.dtype} {tuple(q.shape)} with a unit last stride, got {q_out.dtype} "
                             f"{tuple(q_out.shape)}")
    page_table, valid_tokens, inv_freq = page_table.contiguous(), valid_tokens.contiguous(), inv_freq.contiguous()
    q_lens = None if q_lens is None else q_lens.contiguous()
    if positions is not None and positions.stride(-1) != 1:
        positions = positions.contiguous()
    a = N.RotaryAppendArgs(B, L, Hq, Hkv, D, 2 * inv_freq.shape[0], int(bool(interleaved)), PAGE_SIZE, W, NP,
                           _DT[k.dtype])
    if q is not None:
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
        a.q_stride_b, a.q_stride_t, a.q_stride_h, _ = q.stride()
        a.q_out_stride_b, a.q_out_stride_t, a.q_out_stride_h, _ = q_out.stride()
    a.k, a.v = k.data_ptr(), v.data_ptr()
    a.k_stride_b, a.k_stride_t, a.k_stride_h, _ = k_stride
    a.v_stride_b, a.v_stride_t, a.v_stride_h, _ = v_stride
    a.inv_freq, a.positions = inv_freq.data_ptr(), _ptr(positions)
    a.position_stride_b = 0 if positions is None else positions.stride(0)
    a.page_table, a.valid_tokens, a.q_lens = page_table.data_ptr(), valid_tokens.data_ptr(), _ptr(q_lens)
    if packed:
        a.k_codes, a.k_scales, a.v_codes, a.v_scales = (t.data_ptr() for t in written)
    else:
        a.k_pages, a.v_pages, a.page_tags, a.tag = *(t.data_ptr() for t in written), _ptr(page_tags), int(fp16_tag)
    _launch(dev, N.rotary_append, a, current_stream_handle(dev))
    # written through raw pointers
    torch.autograd.graph.increment_version((*written, *(t for t in (page_tags, q_out) if t is not None)))
    return q_out
