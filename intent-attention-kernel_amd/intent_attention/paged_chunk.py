"""Attention of several query tokens per sequence over the decode's pages on the MI355X
(``iak_paged_chunk``, include/iak.h): drafted tokens under verification, chunks of a prompt.

``paged_decode`` serves one query token per sequence; these read the same pools (``PagePools``, every
precision), page tables, counts and tags. ``append_rotated_tokens`` writes the new tokens first: the lengths
count them.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence

import torch

from . import _native as N
from .decode_core import (
    NATIVE_TAG_MAP,
    PAGE_SIZE,
    PagePools,
    _DT,
    _check_page_pools,
    _ptr,
    _scale_dtype,
    current_stream_handle,
)
from .mxfp4 import _check_int32, _device, _launch

_POOLS = ("k_fp16", "v_fp16", "k_fp8", "v_fp8", "k_int8", "v_int8", "k_int4", "v_int4", "k_int4r", "v_int4r", "k_fp8_scale", "v_fp8_scale",
          "k_int8_scale", "v_int8_scale", "k_int4_scale", "v_int4_scale", "k_int4r_scale", "v_int4r_scale")


class ChunkPlan:
    """Checked launch arguments plus workspace (``run`` is one C call on the current stream;
    the tensors are held so their memory stays valid). The plan reads the query, the pools,
    the table, tags and lengths as they are at each run and writes ``out``; its workspace is its own, so
    runs of one plan must not overlap, runs of two plans may."""

    def __init__(self, args: N.PagedChunkArgs, device: torch.device, out: torch.Tensor, keep=()) -> None:
        self.args = args
        self.device = device
        self.out = out
        self._keep = keep
        self.workspace_bytes = N.paged_chunk_workspace(args)
        self._ws = (torch.empty(self.workspace_bytes, dtype=torch.uint8, device=device)
                    if self.workspace_bytes else None)
        self._ws_ptr = self._ws.data_ptr() if self._ws is not None else 0

    def run(self, stream: Optional[int] = None) -> None:
        """Launch on ``stream`` (default: torch's current stream)."""
        s = current_stream_handle(self.device) if stream is None else stream
        _launch(self.device, N.paged_chunk, self.args, s, self._ws_ptr, self.workspace_bytes)
        torch.autograd.graph.increment_version(self.out)        # written through a raw pointer


def make_chunk_plan(q: torch.Tensor, pools: PagePools, page_table: torch.Tensor, page_counts: torch.Tensor,
                    page_tags: torch.Tensor, *, valid_tokens: Optional[torch.Tensor] = None,
                    q_lens: Optional[torch.Tensor] = None, causal: bool = True, tag_map: Optional[Sequence[int]] = None,
                    negative_ids: bool = False, map_other_tags: bool = False, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, splits: int = 0) -> ChunkPlan:
    """Check the arguments of ``paged_chunk_attention`` once, for repeated runs over the same
    tensors. The plan reads the tensors in place: the int32 tensors must be contiguous, q (and ``out``)
    have a unit last stride."""
    dev = _device("chunk attention", q, page_table, page_counts, page_tags, valid_tokens, q_lens, out, *pools.tensors().values())
    if q.dim() not in (3, 4):
        raise ValueError(f"q must have shape [B, Hq, D] or [B, L, Hq, D], got {tuple(q.shape)}")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    B, L, Hq, D = q4.shape
    if q.dtype not in _DT:
        raise ValueError(f"q dtype {q.dtype} is not float16 / bfloat16 / float32")
    if page_table.dim() != 3 or page_table.shape[0] != B:
        raise ValueError(f"page_table must have shape [B, Hkv, W] with B={B}, got {tuple(page_table.shape)}")
    _, Hkv, W = page_table.shape
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"query heads {Hq} must be a multiple of page-table heads {Hkv}")
    if page_tags.dim() != 1:
        raise ValueError(f"page_tags must have shape [num_pages], got {tuple(page_tags.shape)}")
    NP = page_tags.shape[0]
    for name, t, shape in (("page_table", page_table, (B, Hkv, W)), ("page_counts", page_counts, (B, Hkv)),
                           ("page_tags", page_tags, (NP,)), ("valid_tokens", valid_tokens, (B, Hkv)), ("q_lens", q_lens, (B,))):
        if t is not None and (t.shape != shape or t.dtype is not torch.int32 or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32 {list(shape)}, got {t.dtype} {tuple(t.shape)}")
    _check_int32(table_width=W * PAGE_SIZE, rows=B * Hkv, num_pages=NP, splits=splits, q_len=L)
    if q.stride(-1) != 1:
        raise ValueError("q must have a unit last stride")
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    grp = _check_page_pools(pools, NP, D)
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=dev)
    elif out.shape != q.shape or out.stride(-1) != 1:
        raise ValueError(f"out must have q's shape {tuple(q.shape)} and a unit last stride, got {tuple(out.shape)}")
    if out.dtype not in _DT or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out dtype {out.dtype} is not {out_dtype or 'float16 / bfloat16 / float32'}")
    o4 = out.unsqueeze(1) if out.dim() == 3 else out
    a = N.PagedChunkArgs(B, L, Hq, Hkv, D, PAGE_SIZE, W, NP)
    a.q, a.q_dtype, a.out, a.out_dtype = q.data_ptr(), _DT[q.dtype], out.data_ptr(), _DT[out.dtype]
    a.q_stride_b, a.q_stride_t, a.q_stride_h, _ = q4.stride()
    a.out_stride_b, a.out_stride_t, a.out_stride_h, _ = o4.stride()
    a.page_table, a.page_counts, a.page_tags = page_table.data_ptr(), page_counts.data_ptr(), page_tags.data_ptr()
    a.valid_tokens, a.q_lens = _ptr(valid_tokens), _ptr(q_lens)
    if tag_map is None:
        tag_map = [t if pools.has(t) else N.TAG_SKIP for t in NATIVE_TAG_MAP]
    if len(tag_map) > 8 or any(not 0 <= int(t) < 256 for t in tag_map):
        raise ValueError(f"tag_map must be up to 8 native tags, got {list(tag_map)}")
    a.tag_map[:] = [int(t) for t in tag_map] + [N.TAG_SKIP] * (8 - len(tag_map))
    a.map_other_tags, a.negative_ids = int(bool(map_other_tags)), int(bool(negative_ids))
    for n in _POOLS:
        setattr(a, n, _ptr(getattr(pools, n)))
    a.fp8_scale_dtype = _scale_dtype("fp8", pools.k_fp8_scale, pools.v_fp8_scale)
    a.int8_scale_dtype = _scale_dtype("int8", pools.k_int8_scale, pools.v_int8_scale)
    a.int4_scale_dtype = _scale_dtype("int4", pools.k_int4_scale, pools.v_int4_scale)
    a.int4_group = grp
    a.sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    a.causal, a.splits = int(bool(causal)), int(splits)
    return ChunkPlan(a, dev, out, keep=(q, page_table, page_counts, page_tags, valid_tokens, q_lens, pools, *pools.tensors().values()))


def paged_chunk_attention(q: torch.Tensor, pools: PagePools, page_table: torch.Tensor, page_counts: torch.Tensor,
                          page_tags: torch.Tensor, *, valid_tokens: Optional[torch.Tensor] = None,
                          q_lens: Optional[torch.Tensor] = None, causal: bool = True, tag_map: Optional[Sequence[int]] = None,
                          negative_ids: bool = False, map_other_tags: bool = False, sm_scale: Optional[float] = None,
                          out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                          splits: int = 0) -> torch.Tensor:
    """Attention of the newest tokens over pages of mixed precision.

    q [B, L, Hq, D] or [B, Hq, D] (one token per sequence), float16, bfloat16 or float32, D = 64 or
    128; of ``pools`` INT4 scales are per head, half or quarter of it (``int4_group`` D, D / 2 or D / 4; others are refused);
    page_table [B, Hkv, W], page_counts [B, Hkv], page_tags [NP], ``tag_map``,
    ``negative_ids`` and ``map_other_tags`` as for ``paged_decode``. Token t of entry e of a row is its number
    16 e + t; a row holds min(valid_tokens, 16 page_counts) of them (``valid_tokens`` [B, Hkv],
    default: all of its pages'), the queries' own the last: query i < q_lens[b] (default L) sees
    the tokens up to its own, number tokens - q_lens[b] + i, or with ``causal=False`` all. Pages that are
    skipped keep their places and hold no tokens.
    out = softmax(sm_scale q . k) v, sm_scale = 1 / sqrt(D) by default; zeros where a query sees
    nothing and for i >= q_lens[b]. K and V enter exactly, the 4-bit precisions with 21 bits; queries and
    weights are rounded as in ``mxfp4_paged_attention`` (weights of float16 and bfloat16 queries to 11
    bits). What a query does not see never reaches it, infinite and NaN values included. ``splits``: parts the
    rows' tokens are divided into (0: automatic). Returns ``out``, shaped as q. Inference only."""
    page_table, page_counts, page_tags = page_table.contiguous(), page_counts.contiguous(), page_tags.contiguous()
    valid_tokens = None if valid_tokens is None else valid_tokens.contiguous()
    q_lens = None if q_lens is None else q_lens.contiguous()
    if q.dim() and q.stride(-1) != 1:
        q = q.contiguous()
    plan = make_chunk_plan(q, pools, page_table, page_counts, page_tags, valid_tokens=valid_tokens, q_lens=q_lens, causal=causal,
                           tag_map=tag_map, negative_ids=negative_ids, map_other_tags=map_other_tags, sm_scale=sm_scale, out=out,
                           out_dtype=out_dtype, splits=splits)
    plan.run()
    return plan.out
