"""A beam search's choice in float64, from its definition (numpy; test infrastructure)."""
import numpy as np


def candidates(logits, scores, finished=None, end_token=0):
    """[B, K, V] float64: every continuation's value, -inf where there is none."""
    x, s = np.asarray(logits, np.float64), np.asarray(scores, np.float64)
    out = np.full(x.shape, -np.inf)
    for b, k in np.ndindex(*s.shape):
        if finished is not None and finished[b, k]:
            out[b, k, end_token] = s[b, k] if np.isfinite(s[b, k]) else -np.inf
            continue
        row = x[b, k]
        if not np.isfinite(s[b, k]) or np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all():
            continue
        top = row.max()
        out[b, k] = s[b, k] + (row - (top + np.log(np.exp(row - top).sum())))
    return out


def select(logits, scores, count, finished=None, end_token=0):
    """(scores float64, parents, tokens) [B, count]: the best first, equal ones by their number k V + v."""
    at = candidates(logits, scores, finished, end_token)
    B, K, V = at.shape
    flat = at.reshape(B, K * V)
    order = np.argsort(-flat, axis=1, kind="stable")[:, :count]
    return (np.take_along_axis(flat, order, 1), (np.arange(B)[:, None] * K + order // V).astype(np.int32),
            (order % V).astype(np.int32))
