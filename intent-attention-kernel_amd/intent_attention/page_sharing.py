"""Pages of a KV cache handed out, shared, given back and moved, on the MI355X
(``iak_grow_sequences``, ``iak_fork_sequences``, ``iak_free_sequences``,
``iak_reorder_sequences``, ``iak_compact_pages``, ``iak_copy_pages``, include/iak.h).

The state is three int32 tensors on the device, which a program keeps beside its pools
(``PagePools``, ``LatentPools``, ``MxFp4Pools``, or any tensors with a row per page; with
``PagePools`` the decode's ``page_tags`` are such a tensor and go along in a list,
``[*pools.tensors().values(), page_tags]``):

  page_table    [B, R, W]  the pages of row (b, r): R = KV heads for K/V pools; a latent
                           table [B, W] is passed as [B, 1, W]
  valid_tokens  [B, R]     the tokens of each row; its first ceil(valid / 16) entries are in use
  refs          [NP]       how many table entries (and other owners) hold a page; 0: free

* ``grow_sequences`` makes room for new tokens: pages for them, the lowest free ids first,
  and a copy of a row's last page where it has room but others hold it too;
* ``fork_sequences`` makes empty sequences copies of others: full pages are shared, a last
  page with room is copied, so that both may append;
* ``free_sequences`` lets sequences go, or their newest tokens;
* ``reorder_sequences`` makes sequences copies of each other, all at once: a beam search's choice
  (``beam_select``);
* ``compact_pages`` moves the pages in use to the lowest ids and returns the new table;
* ``copy_pages`` copies pages from id to id.

Nothing waits for the device; indices and counts may be lists, except in a graph under capture.
Which page goes where is a function of the arguments alone.
``grow_sequences``, ``fork_sequences`` and ``reorder_sequences`` do all of a call or nothing of it, and return an
int32 [1] device tensor: 0 done, n > 0: n free pages too few, -1: refused (an index out
of range or listed twice, a negative count, a row that would be longer than its table, a
growing row whose last page others hold too and no pools, a forked sequence that has tokens or is itself a parent).
``fork_sequences`` and ``reorder_sequences`` hand pages out without ``pools`` too: a last page that they would
copy holds then what it held before, and is the caller's to copy (``copy_pages``) before anything reads it: where the
pools are more tensors than a call takes. What is queued behind a call that was not done runs
all the same: ``grow_sequences(..., granted=lens)`` leaves in ``lens`` how many tokens each
sequence got room for, 0 then, and ``append_mxfp4_tokens(..., q_lens=lens)`` writes no more.
Without it read the answer before tokens are appended, for they would land on older ones.
A fork that was not done leaves its children empty: read its answer before they grow.
"""
from __future__ import annotations

import struct
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _native as N
from .decode_core import PAGE_SIZE, PagePools, current_stream_handle, uploads_pinned
from .mla_core import LatentPools
from .mxfp4 import MxFp4Pools, _check_int32, _device, _launch

Pools = Union[PagePools, LatentPools, MxFp4Pools, torch.Tensor, Sequence[torch.Tensor]]
Indices = Union[torch.Tensor, Sequence[int]]


_entry = struct.Struct("Pq")           # iak_page_array


def _pool_tensors(pools: Optional[Pools]) -> List[torch.Tensor]:
    """The tensors of the pools, each once (K and V may be one pool)."""
    if pools is None:
        return []
    if isinstance(pools, (PagePools, LatentPools, MxFp4Pools)):
        ts: Iterable = [t for t in vars(pools).values() if isinstance(t, torch.Tensor)]
    else:
        ts = (pools,) if isinstance(pools, torch.Tensor) else pools
    return list({(t.data_ptr(), t.numel() * t.element_size()): t for t in ts}.values())


def _fill_arrays(a, tensors: List[torch.Tensor], NP: int) -> None:
    if len(tensors) > N.MAX_PAGE_ARRAYS:
        raise ValueError(f"at most {N.MAX_PAGE_ARRAYS} pool tensors, got {len(tensors)}")
    n, offset = 0, type(a).arrays.offset
    for t in tensors:
        size = t.numel()
        if NP == 0 and size == 0:
            continue
        if NP == 0 or t.dim() == 0 or size % NP or t.shape[0] % NP or not t.is_contiguous():
            raise ValueError(f"every pool tensor must be contiguous with a row for each of {NP} pages, "
                             f"got {tuple(t.shape)}")
        if size:
            _entry.pack_into(a, offset + n * _entry.size, t.data_ptr(), size // NP * t.element_size())
            n += 1
    a.num_arrays = n


def _check_state(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor) -> Tuple[int, int, int, int]:
    if page_table.dim() != 3 or page_table.dtype is not torch.int32 or not page_table.is_contiguous():
        raise ValueError(f"page_table must be contiguous int32 [B, R, W], got {page_table.dtype} "
                         f"{tuple(page_table.shape)}")
    B, R, W = page_table.shape
    if valid_tokens.shape != (B, R) or valid_tokens.dtype != torch.int32 or not valid_tokens.is_contiguous():
        raise ValueError(f"valid_tokens must be contiguous int32 [{B}, {R}], got {valid_tokens.dtype} "
                         f"{tuple(valid_tokens.shape)}")
    if refs.dim() != 1 or refs.dtype != torch.int32 or not refs.is_contiguous():
        raise ValueError(f"refs must be contiguous int32 [num_pages], got {refs.dtype} {tuple(refs.shape)}")
    if R == 0:
        raise ValueError("page_table has no rows per sequence")
    _check_int32(table_width=W * PAGE_SIZE, rows=B * R)
    return B, R, W, refs.shape[0]


def _indices(name: str, x: Indices, device: torch.device, count: Optional[int] = None) -> torch.Tensor:
    """int32 [n] on the device; a list of ints is uploaded, from pinned memory: a pageable copy waits
    for what the stream has queued."""
    if isinstance(x, torch.Tensor):
        if x.dim() != 1 or x.dtype is not torch.int32:
            raise ValueError(f"{name} must be int32 [n], got {x.dtype} {tuple(x.shape)}")
        if x.device != device:
            raise ValueError(f"{name} must be on {device}, got {x.device}")
        x = x.contiguous()
    else:
        vals = [int(v) for v in x]
        if any(not -2 ** 31 <= v < 2 ** 31 for v in vals):
            raise ValueError(f"{name} must be int32 values")
        pinned = uploads_pinned(device)
        if device.type == "cuda" and not pinned:
            raise ValueError(f"{name} must be a device tensor in a graph under capture: a replay cannot read a list again")
        x = torch.tensor(vals, dtype=torch.int32, device="cpu", pin_memory=pinned).to(device, non_blocking=pinned)
    if count is not None and x.shape[0] != count:
        raise ValueError(f"{name} must have {count} entries, got {x.shape[0]}")
    return x


def _sequences(what: str, page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor, seqs: Indices,
               pools: Optional[Pools] = None):
    tensors = _pool_tensors(pools)
    dev = _device(what, page_table, valid_tokens, refs, *tensors)
    B, R, W, NP = _check_state(page_table, valid_tokens, refs)
    seqs = _indices("seqs", seqs, dev)
    a = N.SequencesArgs(B, R, W, PAGE_SIZE, NP, page_table.data_ptr(), valid_tokens.data_ptr(), refs.data_ptr(),
                        seqs.shape[0], seqs.data_ptr())
    if tensors:
        _fill_arrays(a, tensors, NP)
    return a, dev, seqs, tensors


def _written(*tensors: torch.Tensor) -> None:
    torch.autograd.graph.increment_version(tensors)     # written through raw pointers


def _planned(launch, a, dev: torch.device, missing: Optional[torch.Tensor],
             workspace=N.sequences_workspace) -> torch.Tensor:
    if missing is None:
        missing = torch.empty(1, dtype=torch.int32, device=dev)
    elif missing.shape != (1,) or missing.dtype != torch.int32 or missing.device != dev:
        raise ValueError(f"missing must be int32 [1] on {dev}, got {missing.dtype} {tuple(missing.shape)}")
    a.missing = missing.data_ptr()
    size = workspace(a)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch(dev, launch, a, current_stream_handle(dev), ws.data_ptr(), size)
    return missing


def grow_sequences(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor, seqs: Indices,
                   new_tokens: Indices, pools: Optional[Pools] = None, *, granted: Optional[torch.Tensor] = None,
                   missing: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Room for ``new_tokens[i]`` more tokens in every row of sequence ``seqs[i]``: the table
    entries they need get free pages (the lowest ids first, in the order of i, row, entry),
    refs 1, and valid_tokens grows. All or nothing; returns ``missing`` (module docstring).
    A row whose last page has room but refs above 1 (sequences that were forked and then cut back
    to inside a page they share) gets a page of its own for it, copied in every tensor of
    ``pools``, and lets go of the shared one; without ``pools`` such a call is refused (-1): what is
    appended reaches no other owner.
    ``granted`` (int32 [B]) is written whole: ``new_tokens[i]`` at ``seqs[i]``, 0 at every other
    sequence, and 0 at all of them if nothing was done: the ``q_lens`` of the append and the
    attention behind it."""
    a, dev, seqs, tensors = _sequences("page allocation", page_table, valid_tokens, refs, seqs, pools)
    new_tokens = _indices("new_tokens", new_tokens, dev, seqs.shape[0])
    a.new_tokens = new_tokens.data_ptr()
    if granted is not None:
        B = page_table.shape[0]
        if granted.shape != (B,) or granted.dtype != torch.int32 or granted.device != dev or not granted.is_contiguous():
            raise ValueError(f"granted must be contiguous int32 [{B}] on {dev}, got {granted.dtype} {tuple(granted.shape)}")
        a.granted = granted.data_ptr()
    missing = _planned(N.grow_sequences, a, dev, missing)
    _written(page_table, valid_tokens, refs, missing, *(() if granted is None else (granted,)), *tensors)
    return missing


def fork_sequences(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor, parents: Indices,
                   children: Indices, pools: Optional[Pools] = None, *,
                   missing: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Sequence ``children[i]``, which has no tokens, becomes a copy of ``parents[i]``: it shares
    the parent's pages (refs + 1), except that a last page which is not full is copied, in
    every tensor of ``pools``, to a free page (without ``pools`` that page is the caller's to fill). All or
    nothing; returns ``missing`` (module docstring). A parent may be listed many times."""
    a, dev, children, tensors = _sequences("page sharing", page_table, valid_tokens, refs, children, pools)
    parents = _indices("parents", parents, dev, children.shape[0])
    a.parents = parents.data_ptr()
    missing = _planned(N.fork_sequences, a, dev, missing)
    _written(page_table, valid_tokens, refs, missing, *tensors)
    return missing


def reorder_sequences(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor, seqs: Indices,
                      parents: Indices, pools: Optional[Pools] = None, *,
                      missing: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Sequence ``seqs[i]`` becomes a copy of what ``parents[i]`` was before the call, all of them at
    once: a parent may be listed many times, and be among ``seqs`` itself (``seqs[i] == parents[i]``
    stays as it is). Full pages are shared, and rows let go of the pages they had. A last page that
    is not full stays with one owner, the parent if it stays itself or is not among ``seqs``, else its first
    child in the call; the others get copies of it, in every tensor of ``pools``, in pages that were free
    before the call (the lowest ids first, in the order of i, row; without ``pools`` those pages are the caller's to
    fill). All or nothing; returns ``missing`` (module docstring)."""
    a, dev, seqs, tensors = _sequences("page sharing", page_table, valid_tokens, refs, seqs, pools)
    parents = _indices("parents", parents, dev, seqs.shape[0])
    a.parents = parents.data_ptr()
    missing = _planned(N.reorder_sequences, a, dev, missing, N.reorder_sequences_workspace)
    _written(page_table, valid_tokens, refs, missing, *tensors)
    return missing


def free_sequences(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor, seqs: Indices,
                   tokens: Optional[Indices] = None) -> None:
    """Let go of sequences ``seqs``, or of the newest ``tokens[i]`` tokens of every row of
    ``seqs[i]`` (drafts that were not taken): valid_tokens sinks, to 0 at least, entries that are
    no longer in use become -1, refs - 1 for each. Indices outside the table and negative numbers are
    left out, a sequence listed twice loses tokens twice."""
    a, dev, seqs, _ = _sequences("page sharing", page_table, valid_tokens, refs, seqs)
    if tokens is not None:
        tokens = _indices("tokens", tokens, dev, seqs.shape[0])
        a.new_tokens = tokens.data_ptr()
    _launch(dev, N.free_sequences, a, current_stream_handle(dev))
    _written(page_table, valid_tokens, refs)


def compact_pages(page_table: torch.Tensor, valid_tokens: torch.Tensor, refs: torch.Tensor,
                  pools: Optional[Pools] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(new page_table, new refs, page_map): with L pages in use, those with ids >= L move to
    the free ids below L (the highest to the lowest), in place in every tensor of ``pools``.
    page_map [NP] int32 is the new id of every page, -1 for free ones: owners other than the
    table look theirs up in it. The arguments' table and refs stay as they are and the moved
    pages' old rows keep their bytes, so what was queued with the old table still finds them
    until their ids are handed out again."""
    tensors = _pool_tensors(pools)
    dev = _device("page compaction", page_table, valid_tokens, refs, *tensors)
    B, R, W, NP = _check_state(page_table, valid_tokens, refs)
    table, new_refs, page_map = torch.empty_like(page_table), torch.empty_like(refs), torch.empty_like(refs)
    a = N.CompactPagesArgs(B * R, W, PAGE_SIZE, NP, page_table.data_ptr(), valid_tokens.data_ptr(), refs.data_ptr(),
                           table.data_ptr(), new_refs.data_ptr(), page_map.data_ptr())
    _fill_arrays(a, tensors, NP)
    size = N.compact_pages_workspace(a)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch(dev, N.compact_pages, a, current_stream_handle(dev), ws.data_ptr(), size)
    if tensors:
        _written(*tensors)
    return table, new_refs, page_map


def copy_pages(pools: Pools, src: Indices, dst: Indices, *, num_pages: Optional[int] = None) -> None:
    """Page ``src[i]`` of every pool tensor to page ``dst[i]``. Pairs with an id outside the pools
    are left out. The dst ids must be distinct, and none of them a src of another pair.
    ``num_pages``: the pages of the pools (default: the first tensor's rows)."""
    tensors = _pool_tensors(pools)
    if not tensors:
        raise ValueError("no pool tensor given")
    dev = _device("page copy", *tensors)
    NP = tensors[0].shape[0] if num_pages is None else int(num_pages)
    src = _indices("src", src, dev)
    dst = _indices("dst", dst, dev, src.shape[0])
    a = N.CopyPagesArgs()
    a.num_pages, a.count, a.src, a.dst = NP, src.shape[0], src.data_ptr(), dst.data_ptr()
    _fill_arrays(a, tensors, NP)
    _launch(dev, N.copy_pages, a, current_stream_handle(dev))
    _written(*tensors)
