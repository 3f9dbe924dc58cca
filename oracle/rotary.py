"""Rotation by position and the places of the newest tokens, in float64 (numpy; test infrastructure)."""
import numpy as np

PS = 16


def rotate(x, positions, inv_freq, interleaved):
    """x [B, L, H, D] turned by positions [B, L, H], in float64."""
    x = np.array(x, np.float64)
    half = len(inv_freq)
    # the angle's whole turns are taken off in more bits than float64 has where the machine's longest has them
    turn = np.remainder(positions[..., None].astype(np.longdouble) * np.asarray(inv_freq, np.float64).astype(np.longdouble), 2 * np.pi * np.longdouble(1)
                        + np.longdouble(2.4492935982947064e-16)).astype(np.float64)
    c, s = np.cos(turn), np.sin(turn)
    a = x[..., 0:2 * half:2] if interleaved else x[..., :half]
    b = x[..., 1:2 * half:2] if interleaved else x[..., half:2 * half]
    p, q = a * c - b * s, a * s + b * c
    if interleaved:
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = p, q
    else:
        x[..., :half], x[..., half:2 * half] = p, q
    return x


def reach(x, inv_freq, interleaved):
    """|x| + |y| of every channel's pair (|x| twice where it does not turn)."""
    x = np.abs(np.asarray(x, np.float64))
    half, out = len(inv_freq), 2 * x
    if interleaved:
        out[..., 0:2 * half:2] = out[..., 1:2 * half:2] = x[..., 0:2 * half:2] + x[..., 1:2 * half:2]
    else:
        out[..., :half] = out[..., half:2 * half] = x[..., :half] + x[..., half:2 * half]
    return out


def places(table, valid, q_lens, L, NP):
    """(page, offset) [B, L, Hkv] of the new tokens, page -1 where there is none, and their numbers."""
    B, Hkv, W = table.shape
    page, number = np.full((B, L, Hkv), -1, np.int64), np.zeros((B, L, Hkv), np.int64)
    for b in range(B):
        n = L if q_lens is None else int(np.clip(q_lens[b], 0, L))
        for h in range(Hkv):
            last = int(np.clip(valid[b, h], 0, W * PS))
            number[b, :, h] = last - n + np.arange(L)
            for i in range(n):
                at = last - n + i
                if 0 <= at < W * PS and 0 <= table[b, h, at // PS] < NP:
                    page[b, i, h] = table[b, h, at // PS]
    return page, number
