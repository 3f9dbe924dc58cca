"""Attention of several query tokens over pages of mixed precision in float64 (numpy; test infrastructure)."""
import numpy as np

PS = 16
FP16, INT8, SKIP, FP8, INT4, INT4_RESIDUAL = range(6)
NAMES = {FP16: "fp16", INT8: "int8", FP8: "fp8", INT4: "int4", INT4_RESIDUAL: "int4r"}


def fp8_values(codes):
    """float64 of e4m3fn bytes."""
    c = codes.astype(np.int64)
    field, part = (c >> 3) & 15, (c & 7) / 8
    size = np.where(field == 0, part * 2.0 ** -6, (1 + part) * 2.0 ** (field - 7.0))
    return np.where((c & 127) == 127, np.nan, np.where(c >= 128, -size, size))


def page_values(pools, side, page, tag):
    """float64 [16, D] of a page's K or V in a precision."""
    codes = pools[f"{side}_{NAMES[tag]}"][page]
    if tag == FP16:
        return codes.astype(np.float64)
    scale = pools[f"{side}_{NAMES[tag]}_scale"][page].astype(np.float64)
    with np.errstate(invalid="ignore"):
        if tag == INT8:
            return codes * scale
        if tag == FP8:
            return fp8_values(codes) * scale
        low, high = (codes & 15).astype(np.float64) - 8, (codes >> 4).astype(np.float64) - 8
        if tag == INT4:
            x = np.stack((low, high), -1).reshape(PS, -1)
            return x * np.repeat(scale, x.shape[1] // len(scale))
        return low * scale[0] + high * scale[1]


def native(tags, tag_map=None, map_other=False):
    """Caller tags as native ones (SKIP: nothing)."""
    tag_map = list(range(6)) + [SKIP, SKIP] if tag_map is None else list(tag_map) + [SKIP] * (8 - len(tag_map))
    other = tag_map[7] if map_other else SKIP
    return np.array([tag_map[t] if 0 <= t < 8 else other for t in tags])


def row_tokens(pools, tags, row, tokens, negative_ids=False):
    """(k, v [tokens, D] float64, there [tokens]) of a table row."""
    NP, D = len(tags), pools["k_fp16"].shape[2]
    k, v, there = np.zeros((tokens, D)), np.zeros((tokens, D)), np.zeros(tokens, bool)
    for e in range(-(-tokens // PS)):
        p = int(row[e])
        if negative_ids and p < 0:
            p += NP
        if not 0 <= p < NP or tags[p] not in NAMES:
            continue
        n = min(PS, tokens - e * PS)
        at = slice(e * PS, e * PS + n)
        k[at], v[at], there[at] = page_values(pools, "k", p, tags[p])[:n], page_values(pools, "v", p, tags[p])[:n], True
    return k, v, there


def _size(x):
    """|x|, 0 for what is not finite."""
    return np.where(np.isfinite(x), np.abs(x), 0.0)


def attention(q, pools, tags, table, counts, valid=None, q_lens=None, causal=True, sm_scale=None, negative_ids=False):
    """out [B, L, Hq, D], sum of p |v| (mass) and the largest sm_scale sum |q| |k| seen (reach [B, L, Hq]), in float64."""
    q = np.asarray(q, np.float64)
    B, L, Hq, D = q.shape
    _, Hkv, W = table.shape
    G = Hq // Hkv
    scale = 1 / np.sqrt(D) if sm_scale is None else sm_scale
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
    for b in range(B):
        n = L if q_lens is None else int(np.clip(q_lens[b], 0, L))
        for h in range(Hkv):
            T = int(np.clip(counts[b, h], 0, W)) * PS
            if valid is not None:
                T = min(T, max(0, int(valid[b, h])))
            k, v, there = row_tokens(pools, tags, table[b, h], T, negative_ids)
            for i in range(n):
                sees = there & (np.arange(T) < (T - n + i + 1 if causal else T))
                if not sees.any():
                    continue
                x = q[b, i, h * G:(h + 1) * G]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (x @ k[sees].T)
                    s = np.where(np.isfinite(x).all(-1, keepdims=True), s, np.nan)
                    top = s.max(-1, keepdims=True)
                    p = np.exp(s - np.where(top == -np.inf, 0, top))
                    total = p.sum(-1, keepdims=True)
                    p = p / np.where(total == 0, 1, total)
                    vs = v[sees]
                    fine = np.isfinite(vs)
                    o = p @ np.where(fine, vs, 0.0)
                    # a weight is positive: what is not finite reaches its channel
                    for d in np.nonzero(~fine.all(0))[0]:
                        o[:, d] = o[:, d] + vs[~fine[:, d], d].sum()
                    out[b, i, h * G:(h + 1) * G] = o
                    mass[b, i, h * G:(h + 1) * G] = np.nan_to_num(p) @ np.abs(np.where(fine, vs, 0.0))
                    reach[b, i, h * G:(h + 1) * G] = abs(scale) * (_size(x) @ _size(k[sees]).T).max(-1)
    return out, mass, reach
