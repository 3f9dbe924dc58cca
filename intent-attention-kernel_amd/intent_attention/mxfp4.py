"""A microscaled 4-bit (MXFP4) token cache on the MI355X: tokens written one by one,
and attention of one or several query tokens per sequence over them
(``iak_mx_append_tokens``, ``iak_mx_read_tokens``, ``iak_mx_attention``, include/iak.h).

The decode's INT4 pages (``PagePools``) carry one scale per page and channel group, so a
page is written whole. Here every token has its own scales, one per 32 channels: a
serving loop appends each new token as it comes, at 4.25 bits a value.

* ``MxFp4Pools`` -- pages of 16 tokens of one KV head: e2m1 codes and e8m0 scale bytes;
* ``append_mxfp4_tokens(k, v, pools, page_table, valid_tokens)`` -- quantises the newest
  tokens of every sequence into their pages, ``read_mxfp4_tokens`` gives them back;
* ``mxfp4_paged_attention(q, pools, page_table, valid_tokens)`` -- attention of the
  newest tokens: a decode step (q [B, Hq, D]), drafted tokens or a prompt chunk
  (q [B, L, Hq, D], causal); ``make_mxfp4_plan`` checks the arguments once for many runs.

All of them take the same page table [B, Hkv, W] and ``valid_tokens`` [B, Hkv], the tokens
each row holds INCLUDING the newest ones: append first, then attend. With ``q_lens`` [B]
sequence b has q_lens[b] new tokens, the first of the batch's L; the rest is padding (not
written by append, zero from read and attention). A length below 0 counts as 0, one past the
table as the table's 16 W tokens, in all of them: the newest tokens of such a row are the
table's last slots, and an append writes over what they hold. ``grow_sequences`` lets no row
become longer than its table; a program that counts lengths itself must not either.

The values: per block of 32 channels e = clamp(floor(log2 max|x|) - 2, -23, 13) and codes
rounded to the nearest even of x / 2^e, at most 6 in magnitude (the OCP microscaling
conversion; the clamp keeps every value a float16 number, the largest 49,152). A block
with an infinity or a NaN is stored as NaN and makes every query that sees its token NaN.

Device tensors only, inference only (no autograd history). The table, the lengths and the
pages are read on the stream the call is made on.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Dict, Optional, Tuple

import torch

from . import _native as N
from .decode_core import PAGE_SIZE, _DT, _check_pool, _ptr, current_stream_handle, require_device

BLOCK = 32          # channels per scale


@dataclass
class MxFp4Pools:
    """K and V pages of the cache: codes [NP, 16, D/2] uint8 (channel 2j in the low half of
    byte j) and scale bytes [NP, 16, D/32] uint8, D = 64 or 128."""

    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, head_dim: int, device) -> "MxFp4Pools":
        """Pools of ``num_pages`` pages whose every value is 0."""
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        codes, scales = ((num_pages, PAGE_SIZE, head_dim // 2), (num_pages, PAGE_SIZE, head_dim // BLOCK))
        return cls(*(torch.zeros(s, dtype=torch.uint8, device=device) for s in (codes, scales, codes, scales)))

    def tensors(self) -> Dict[str, torch.Tensor]:
        return {"k_codes": self.k_codes, "k_scales": self.k_scales, "v_codes": self.v_codes, "v_scales": self.v_scales}


def _device(what: str, *tensors: Optional[torch.Tensor]) -> torch.device:
    """The one ROCm device of all tensors (None: absent), or require_device's errors."""
    first = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != first or first < 0):
            return require_device(*(x for x in tensors if x is not None), what=what)
    N.load()
    return tensors[0].device


def _check_int32(**sizes: int) -> None:
    """ValueError for sizes that the int32 fields of an argument block would wrap."""
    for name, n in sizes.items():
        if not -2 ** 31 <= n < 2 ** 31:
            raise ValueError(f"{name} {n} does not fit int32")


def _check_cache(pools: MxFp4Pools, page_table: torch.Tensor, valid_tokens: torch.Tensor,
                 q_lens: Optional[torch.Tensor], B: int, D: int) -> Tuple[int, int, int]:
    """(Hkv, W, NP) of the pools and the metadata, or ValueError."""
    if page_table.dim() != 3 or page_table.shape[0] != B or page_table.dtype is not torch.int32:
        raise ValueError(f"page_table must be int32 [{B}, Hkv, W], got {page_table.dtype} {tuple(page_table.shape)}")
    _, Hkv, W = page_table.shape
    _check_int32(table_width=W * PAGE_SIZE, rows=B * Hkv)
    if valid_tokens.shape != (B, Hkv) or valid_tokens.dtype is not torch.int32:
        raise ValueError(f"valid_tokens must be int32 [{B}, {Hkv}], got {valid_tokens.dtype} "
                         f"{tuple(valid_tokens.shape)}")
    if q_lens is not None and (q_lens.shape != (B,) or q_lens.dtype is not torch.int32):
        raise ValueError(f"q_lens must be int32 [{B}], got {q_lens.dtype} {tuple(q_lens.shape)}")
    if D not in (64, 128):
        raise ValueError(f"head_dim must be 64 or 128, got {D}")
    NP = pools.k_codes.shape[0] if pools.k_codes.dim() else -1
    codes, scales = (NP, PAGE_SIZE, D // 2), (NP, PAGE_SIZE, D // BLOCK)
    for t, shape in ((pools.k_codes, codes), (pools.k_scales, scales), (pools.v_codes, codes), (pools.v_scales, scales)):
        if t.shape != shape or t.dtype is not torch.uint8 or not t.is_contiguous():
            for name, x in pools.tensors().items():
                _check_pool(name, x, NP, (codes if name.endswith("codes") else scales)[1:], (torch.uint8,))
    return Hkv, W, NP


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(device: torch.device, call: Callable, *args) -> None:
    """``call(*args)`` with ``device`` current, as launches on its streams need."""
    if device.index is None or device.index == _current_device():
        call(*args)
    else:
        with torch.cuda.device(device):
            call(*args)


def _tokens_args(k: torch.Tensor, v: torch.Tensor, pools: MxFp4Pools, page_table: torch.Tensor,
                 valid_tokens: torch.Tensor, q_lens: Optional[torch.Tensor]):
    """The argument block of append and read, and the tensors it points into."""
    B, L, Hkv, D = k.shape
    heads, W, NP = _check_cache(pools, page_table, valid_tokens, q_lens, B, D)
    if heads != Hkv:
        raise ValueError(f"page_table has {heads} KV heads, k has {Hkv}")
    page_table, valid_tokens = page_table.contiguous(), valid_tokens.contiguous()
    q_lens = None if q_lens is None else q_lens.contiguous()
    kb, kt, kh, _ = k.stride()
    vb, vt, vh, _ = v.stride()
    a = N.MxTokensArgs(B, L, Hkv, D, PAGE_SIZE, W, NP, k.data_ptr(), kb, kt, kh, v.data_ptr(), vb, vt, vh, _DT[k.dtype],
                       page_table.data_ptr(), valid_tokens.data_ptr(), None if q_lens is None else q_lens.data_ptr(),
                       pools.k_codes.data_ptr(), pools.k_scales.data_ptr(), pools.v_codes.data_ptr(),
                       pools.v_scales.data_ptr())
    return a, (page_table, valid_tokens, q_lens)


def append_mxfp4_tokens(k: torch.Tensor, v: torch.Tensor, pools: MxFp4Pools, page_table: torch.Tensor,
                        valid_tokens: torch.Tensor, *, q_lens: Optional[torch.Tensor] = None) -> None:
    """Quantise the newest tokens' ``k``, ``v`` [B, L, Hkv, D] (float16, bfloat16 or float32,
    one dtype, any strides) into the pools: token i < q_lens[b] (default L) of sequence b is
    number min(valid_tokens[b, h], 16 W) - q_lens[b] + i of row (b, h). Tokens before 0 or on a
    page id outside the pools are left out; nothing else of the pools is written.
    Rows that share a page (``fork_sequences`` shares full pages only) must not both append
    to it."""
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"k and v must have one shape [B, L, Hkv, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype not in _DT or v.dtype != k.dtype:
        raise ValueError(f"k and v must both be float16, bfloat16 or float32, got {k.dtype} and {v.dtype}")
    dev = _device("4-bit token cache", k, v, page_table, valid_tokens, q_lens, pools.k_codes, pools.k_scales, pools.v_codes,
                  pools.v_scales)
    if k.stride(-1) != 1 or v.stride(-1) != 1:
        k, v = k.contiguous(), v.contiguous()
    a, keep = _tokens_args(k, v, pools, page_table, valid_tokens, q_lens)
    _launch(dev, N.mx_append_tokens, a, current_stream_handle(dev))
    # written through raw pointers
    torch.autograd.graph.increment_version((pools.k_codes, pools.k_scales, pools.v_codes, pools.v_scales))


def read_mxfp4_tokens(pools: MxFp4Pools, page_table: torch.Tensor, valid_tokens: torch.Tensor, count: int, *,
                      q_lens: Optional[torch.Tensor] = None,
                      dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V [B, count, Hkv, D] of the newest ``count`` tokens of every row (with ``q_lens``:
    of the newest q_lens[b], then zeros) as the cache holds them, exactly in every dtype;
    tokens that do not exist are zero."""
    if dtype not in _DT:
        raise ValueError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    if count < 0:
        raise ValueError(f"count must not be negative, got {count}")
    _check_int32(count=count)
    dev = _device("4-bit token cache", page_table, valid_tokens, q_lens, pools.k_codes, pools.k_scales, pools.v_codes,
                  pools.v_scales)
    if page_table.dim() != 3 or pools.k_codes.dim() != 3:
        raise ValueError(f"page_table must be [B, Hkv, W] and codes [NP, {PAGE_SIZE}, D/2], got "
                         f"{tuple(page_table.shape)} and {tuple(pools.k_codes.shape)}")
    shape = (page_table.shape[0], int(count), page_table.shape[1], 2 * pools.k_codes.shape[2])
    k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    a, keep = _tokens_args(k, v, pools, page_table, valid_tokens, q_lens)
    _launch(dev, N.mx_read_tokens, a, current_stream_handle(dev))
    return k, v


class MxFp4Plan:
    """Checked launch arguments plus workspace (``run`` is one C call on the current stream;
    the tensors are held so their memory stays valid). The plan reads the query, the pools,
    the table and the lengths as they are at each run and writes ``out``; its workspace is
    its own, so runs of one plan must not overlap, runs of two plans may."""

    def __init__(self, args: N.MxAttentionArgs, device: torch.device, out: torch.Tensor, keep=()) -> None:
        self.args = args
        self.device = device
        self.out = out
        self._keep = keep
        self.workspace_bytes = N.mx_attention_workspace(args)
        self._ws = (torch.empty(self.workspace_bytes, dtype=torch.uint8, device=device)
                    if self.workspace_bytes else None)
        self._ws_ptr = self._ws.data_ptr() if self._ws is not None else 0

    def run(self, stream: Optional[int] = None) -> None:
        """Launch on ``stream`` (default: torch's current stream)."""
        s = current_stream_handle(self.device) if stream is None else stream
        _launch(self.device, N.mx_attention, self.args, s, self._ws_ptr, self.workspace_bytes)
        torch.autograd.graph.increment_version(self.out)        # written through a raw pointer


def make_mxfp4_plan(q: torch.Tensor, pools: MxFp4Pools, page_table: torch.Tensor, valid_tokens: torch.Tensor, *,
                    q_lens: Optional[torch.Tensor] = None, causal: bool = True, sm_scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                    splits: int = 0) -> MxFp4Plan:
    """Check the arguments of ``mxfp4_paged_attention`` once, for repeated runs over the same
    tensors. The plan reads the tensors in place: page_table, valid_tokens and q_lens must be
    contiguous, q (and ``out``) have a unit last stride."""
    dev = _device("4-bit cache attention", q, page_table, valid_tokens, q_lens, out, pools.k_codes, pools.k_scales,
                  pools.v_codes, pools.v_scales)
    if q.dim() not in (3, 4):
        raise ValueError(f"q must have shape [B, Hq, D] or [B, L, Hq, D], got {tuple(q.shape)}")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    B, L, Hq, D = q4.shape
    if q.dtype not in _DT:
        raise ValueError(f"q dtype {q.dtype} is not float16 / bfloat16 / float32")
    Hkv, W, NP = _check_cache(pools, page_table, valid_tokens, q_lens, B, D)
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"query heads {Hq} must be a multiple of page-table heads {Hkv}")
    for name, t in (("page_table", page_table), ("valid_tokens", valid_tokens), ("q_lens", q_lens)):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if q.stride(-1) != 1:
        raise ValueError("q must have a unit last stride")
    _check_int32(splits=splits, q_len=L)
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=dev)
    elif out.shape != q.shape or out.stride(-1) != 1:
        raise ValueError(f"out must have q's shape {tuple(q.shape)} and a unit last stride, got {tuple(out.shape)}")
    if out.dtype not in _DT or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"out dtype {out.dtype} is not {out_dtype or 'float16 / bfloat16 / float32'}")
    o4 = out.unsqueeze(1) if out.dim() == 3 else out
    qb, qt, qh, _ = q4.stride()
    ob, ot, oh, _ = o4.stride()
    a = N.MxAttentionArgs(B, L, Hq, Hkv, D, PAGE_SIZE, W, NP, q.data_ptr(), _DT[q.dtype], qb, qt, qh, out.data_ptr(),
                          _DT[out.dtype], ob, ot, oh, page_table.data_ptr(), valid_tokens.data_ptr(), _ptr(q_lens),
                          pools.k_codes.data_ptr(), pools.k_scales.data_ptr(), pools.v_codes.data_ptr(),
                          pools.v_scales.data_ptr(), 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale),
                          int(bool(causal)), int(splits))
    return MxFp4Plan(a, dev, out, keep=(q, page_table, valid_tokens, q_lens, *pools.tensors().values()))


def mxfp4_paged_attention(q: torch.Tensor, pools: MxFp4Pools, page_table: torch.Tensor, valid_tokens: torch.Tensor,
                          *, q_lens: Optional[torch.Tensor] = None, causal: bool = True,
                          sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                          out_dtype: Optional[torch.dtype] = None, splits: int = 0) -> torch.Tensor:
    """Attention of the newest tokens over the cache.

    q [B, Hq, D] (one token per sequence) or [B, L, Hq, D], float16, bfloat16 or float32.
    Query i < q_lens[b] (default L) of head h reads row (b, h // (Hq // Hkv)) of the table and
    sees its tokens up to its own, number valid_tokens - q_lens[b] + i, or with
    ``causal=False`` all valid_tokens: out = softmax(sm_scale q . k) v, sm_scale = 1 / sqrt(D)
    by default; zeros where a query sees nothing and for i >= q_lens[b]. Elements of a query row
    below 2^-28 of its largest are rounded, off by at most 2^-39 of that. The softmax weights of
    float16 and bfloat16 queries are rounded to 11 bits for the product with v (a float16 output's
    own precision; with ``out_dtype=torch.float32`` it shows: 2^-11 of sum p |v| at most), those
    of float32 queries to 22. ``splits``: parts the rows' tokens are divided into (0: automatic).
    Returns ``out``, shaped as q."""
    page_table, valid_tokens = page_table.contiguous(), valid_tokens.contiguous()
    q_lens = None if q_lens is None else q_lens.contiguous()
    if q.dim() and q.stride(-1) != 1:
        q = q.contiguous()
    plan = make_mxfp4_plan(q, pools, page_table, valid_tokens, q_lens=q_lens, causal=causal, sm_scale=sm_scale, out=out,
                           out_dtype=out_dtype, splits=splits)
    plan.run()
    return plan.out
