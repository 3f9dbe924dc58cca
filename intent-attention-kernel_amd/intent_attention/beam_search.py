"""A beam search's choice on the MI355X (``iak_beam_select``, include/iak.h): the best continuations
of each request's beams over the vocabulary.

``reorder_sequences`` puts the beams' page tables in the order of the choice, whose ``parents``
it takes as they are where beam k of request b is sequence b * K + k.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native as N
from .decode_core import _DT, current_stream_handle
from .mxfp4 import _check_int32, _device, _launch


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, count: Optional[int] = None,
                finished: Optional[torch.Tensor] = None,
                end_token: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``count`` (default K, at most 64) best of each request's K beams x V tokens.

    logits [B, K, V] (float16, bfloat16 or float32, any strides); scores [B, K] float32, the
    beams' sums of log-probabilities. Candidate (k, v) is scores[b, k] + log_softmax(logits[b, k])[v].
    finished [B, K] (bool or uint8, optional): a beam that is finished has one candidate, ``end_token``
    with its score as it is; its other tokens are -inf. So are all of a beam whose score is not finite,
    or which is not finished and has a logit that is NaN or +inf or none above -inf.
    Returns (scores float32, parents int32, tokens int32), each [B, count], the best first and equal
    ones in the order of k V + v; parents are rows of the logits as [B K, V]: b K + k. Candidates are
    compared in 64 bits; one beam's come in the order of their logits where 64 bits do not tell them apart. K is at
    most 256, B below 2^23."""
    shape = logits.shape
    if len(shape) != 3:
        raise ValueError(f"logits must have shape [B, K, V], got {tuple(shape)}")
    B, K, V = shape
    if logits.dtype not in _DT:
        raise ValueError(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if scores.shape != (B, K) or scores.dtype is not torch.float32:
        raise ValueError(f"scores must be float32 [{B}, {K}], got {scores.dtype} {tuple(scores.shape)}")
    if finished is not None:
        if finished.shape != (B, K) or finished.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"finished must be bool or uint8 [{B}, {K}], got {finished.dtype} {tuple(finished.shape)}")
        if end_token is None:
            raise ValueError("finished beams need an end_token")
    n = K if count is None else int(count)
    end = 0 if end_token is None else int(end_token)
    _check_int32(batch=B, beams=K, vocab=V, count=n, end_token=end)
    dev = _device("beam choice", logits, scores, finished)
    stride_b, stride_k, stride_v = logits.stride()
    if stride_v != 1:
        logits = logits.contiguous()
        stride_b, stride_k, _ = logits.stride()
    scores = scores.contiguous()
    finished = None if finished is None else finished.contiguous()
    at = torch.empty((B, max(n, 0)), dtype=torch.float32, device=dev)
    parents, tokens = (torch.empty_like(at, dtype=torch.int32) for _ in range(2))
    out = (at, parents, tokens)
    a = N.BeamSelectArgs(B, K, V, n, logits.data_ptr(), _DT[logits.dtype], stride_b, stride_k, scores.data_ptr(),
                         None if finished is None else finished.data_ptr(), end, *(t.data_ptr() for t in out))
    size = N.beam_select_workspace(a)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _launch(dev, N.beam_select, a, current_stream_handle(dev), ws.data_ptr(), size)
    return out
