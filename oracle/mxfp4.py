"""The microscaled 4-bit token cache restated in float64 numpy (test infrastructure only;
the reference has no counterpart, so there is no golden vector: the definitions are those of
the OCP microscaling formats, element e2m1 and scale e8m0, with the scale's exponent kept in
[-23, 13])."""
from __future__ import annotations

import numpy as np

BLOCK, PS = 32, 16
E_MIN, E_MAX = -23, 13
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """float64 [..., D] -> (codes uint8 [..., D] one per element, scale bytes uint8 [..., D/32])."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, BLOCK)
    fine = np.isfinite(b).all(-1)
    safe = np.where(fine[..., None], b, 0.0)
    most = np.abs(safe).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(most > 0, np.frexp(most)[1] - 1 - 2, E_MIN)
    e = np.clip(e, E_MIN, E_MAX)
    y = np.minimum(np.abs(safe) / np.exp2(e)[..., None], 6.0)
    # nearest magnitude; where two are as near, the even code
    d = np.abs(y[..., None] - MAGNITUDES)
    d = d - (np.arange(8) % 2 == 0) * 1e-9 * (d == d.min(-1, keepdims=True))
    code = d.argmin(-1).astype(np.uint8) | (np.signbit(safe).astype(np.uint8) << 3)
    return code.reshape(x.shape), np.where(fine, e + 127, 255).astype(np.uint8)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], -1)


def values(codes, scales):
    """float64 [..., D] of one code per element and the scale bytes; NaN blocks NaN."""
    v = np.where(codes & 8, -1.0, 1.0) * MAGNITUDES[codes & 7]
    s = np.exp2(np.clip(scales.astype(np.int64), E_MIN + 127, E_MAX + 127) - 127.0)
    s = np.where(scales == 255, np.nan, s)
    return v * np.repeat(s, BLOCK, -1)


def row_values(codes, scales, row, tokens, num_pages):
    """(values [tokens, D], exists [tokens]) of a table row's tokens."""
    D = 2 * codes.shape[-1]
    out, there = np.zeros((tokens, D)), np.zeros(tokens, bool)
    for t in range(tokens):
        page = int(row[t // PS])
        if 0 <= page < num_pages:
            out[t] = values(unpack(codes[page, t % PS]), scales[page, t % PS])
            there[t] = True
    return out, there


def attention(q, pools, table, valid, q_lens=None, causal=True, sm_scale=None, queries=None):
    """(out, sum of p |v|, score bound) in float64: q [B, L, Hq, D]; the second and third are
    what error bounds are made of: per output the weighted sum of |v|, per query the largest
    sm_scale * sum |q| |k|. `queries`: the query tokens to work out, all if None."""
    B, L, Hq, D = q.shape
    Hkv, W = table.shape[1:]
    G, NP = Hq // Hkv, pools["k_codes"].shape[0]
    sm = 1 / np.sqrt(D) if sm_scale is None else sm_scale
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(B):
        n = L if q_lens is None else int(np.clip(q_lens[b], 0, L))
        for h in range(Hkv):
            T = int(np.clip(valid[b, h], 0, W * PS))
            k, there = row_values(pools["k_codes"], pools["k_scales"], table[b, h], T, NP)
            v, _ = row_values(pools["v_codes"], pools["v_scales"], table[b, h], T, NP)
            nan = there & (np.isnan(k).any(-1) | np.isnan(v).any(-1))
            k, v = np.nan_to_num(k, nan=0.0), np.nan_to_num(v, nan=0.0)
            for i in range(n) if queries is None else [i for i in queries if i < n]:
                seen = there & (np.arange(T) < (T - n + i + 1 if causal else T))
                for x in range(h * G, (h + 1) * G):
                    if not seen.any():
                        continue
                    if (nan & seen).any() or not np.isfinite(q[b, i, x]).all():
                        out[b, i, x] = np.nan
                        continue
                    s = (k[seen] @ q[b, i, x]) * sm
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[b, i, x] = p @ v[seen]
                    mass[b, i, x] = p @ np.abs(v[seen])
                    reach[b, i, x] = abs(sm) * (np.abs(k[seen]) @ np.abs(q[b, i, x])).max()
    return out, mass, reach
