"""The microscaled 4-bit token cache on the GPU against its float64 oracle: quantise on
write and read back, bit for bit; attention of one and several query tokens within bounds
that are worked out per output; special values, masks, strides, graphs and streams."""
import numpy as np
import pytest

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu

DT = ("float16", "bfloat16", "float32")
HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}   # a rounding's largest relative error


def _dev():
    import torch
    return torch.device("cuda:0")


def _t(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).to(_dev())


def _pools(rng, NP, D, garbage=True):
    """Random pages; without garbage every byte is a legal one of a finite value."""
    import intent_attention as ia
    codes = lambda: rng.integers(0, 256, (NP, 16, D // 2), dtype=np.uint8)  # noqa: E731
    scales = lambda: rng.integers(118, 128, (NP, 16, D // 32)).astype(np.uint8)  # noqa: E731
    host = dict(k_codes=codes(), k_scales=scales(), v_codes=codes(), v_scales=scales())
    return host, ia.MxFp4Pools(**{n: _t(x) for n, x in host.items()})


def _table(rng, B, Hkv, W, NP):
    return rng.permutation(NP)[:B * Hkv * W].reshape(B, Hkv, W).astype(np.int32)


def _bound(mass, reach, out, T, D, q_dtype, out_dtype, vmax):
    """What float arithmetic may cost an output (twice: numerator and sum of weights).
    Scores: D products summed in float32, the query's own splitting where it is float32
    (2^-22), the scale and the multiplier: (D + 6) 2^-24 of the largest sum |q| |k|, twice for a
    weight over the sum. Weights: the rounding for the product (float16 2^-11, split 2^-22), the
    exponential and its argument 2^-22, T 2^-24 for either sum, T 2^-31 of the largest |v| for
    weights below float16's range (the largest is at least 2^6, the step there 2^-25)."""
    score = ((D + 6) * 2.0 ** -24 + (2.0 ** -22 if q_dtype == "float32" else 2.0 ** -38)) * reach[..., None]
    weight = 2.0 ** -22 if q_dtype == "float32" else 2.0 ** -11
    rel = 2 * np.expm1(2 * score) + weight + 2.0 ** -22 + 2 * (T + 8) * 2.0 ** -24
    return rel * mass + T * 2.0 ** -31 * vmax + HALF[out_dtype] * np.abs(out) + 2.0 ** -25


def _check(q, dtype, host, pools, table, valid, q_lens=None, causal=True, out_dtype=None, got=None, queries=None, **kw):
    import torch
    import intent_attention as ia
    tq = q if isinstance(q, torch.Tensor) else _t(q).to(getattr(torch, dtype))
    hq = tq.double().cpu().numpy()
    if got is None:
        got = ia.mxfp4_paged_attention(tq, pools, _t(table), _t(valid), q_lens=None if q_lens is None else _t(q_lens),
                                       causal=causal, out_dtype=None if out_dtype is None else getattr(torch, out_dtype), **kw)
    h4 = hq[:, None] if hq.ndim == 3 else hq
    want, mass, reach = O.attention(h4, host, table, valid, q_lens, causal, kw.get("sm_scale"), queries)
    g = got.double().cpu().numpy().reshape(want.shape)
    assert got.shape == tq.shape and got.dtype == getattr(torch, out_dtype or dtype)
    if queries is not None:
        want, mass, reach, g = want[:, queries], mass[:, queries], reach[:, queries], g[:, queries]
    assert np.array_equal(np.isnan(g), np.isnan(want)), "NaN in other places"
    T = int(max(1, np.clip(valid, 0, table.shape[2] * 16).max())) if valid.size else 1
    values = [O.row_values(host["v_codes"], host["v_scales"], table[b, h], int(np.clip(valid[b, h], 0, table.shape[2] * 16)),
                           host["v_codes"].shape[0])[0] for b, h in np.ndindex(*valid.shape)]
    vmax = max((float(np.nan_to_num(np.abs(x), nan=0.0).max()) for x in values if x.size), default=0.0)
    tol = _bound(mass, reach, np.nan_to_num(want), T, h4.shape[-1], dtype, out_dtype or dtype, vmax)
    worst = float((np.abs(np.nan_to_num(g) - np.nan_to_num(want)) / tol).max()) if g.size else 0.0
    assert worst <= 1.0
    return got


# ----------------------------------------------------------------------------- tokens

def _one_row_cache(n_tokens, D, fill=0):
    """A single row of pages for n tokens, pages in reverse order."""
    import torch
    import intent_attention as ia
    W = -(-n_tokens // 16)
    pools = ia.MxFp4Pools.empty(W + 2, D, _dev())
    for t in pools.tensors().values():
        t.fill_(fill)
    table = torch.arange(W, 0, -1, dtype=torch.int32, device=_dev()).view(1, 1, W)
    valid = torch.full((1, 1), n_tokens, dtype=torch.int32, device=_dev())
    return pools, table, valid


def _stored(pools, table, n):
    """(codes one per element, scales) of a one-row cache's tokens, on the host."""
    order = table.view(-1).long()
    f = lambda t: t[order].flatten(0, 1)[:n].cpu().numpy()  # noqa: E731
    return [(O.unpack(f(c)), f(s)) for c, s in ((pools.k_codes, pools.k_scales), (pools.v_codes, pools.v_scales))]


def _same_codes(got, want):
    # a zero's sign is the value's own; both zeros stand for 0
    return np.array_equal(np.where(got & 7, got, 0), np.where(want & 7, want, 0))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_append_every_16_bit_value(dtype, D):
    """Every bit pattern of the 16-bit types, as keys in blocks of neighbours, as values in blocks of strangers."""
    import torch
    import intent_attention as ia
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    k = bits.view(getattr(torch, dtype)).view(1, -1, 1, D).to(_dev())
    perm = torch.from_numpy(np.random.default_rng(0).permutation(65536))
    v = bits[perm].view(getattr(torch, dtype)).view(1, -1, 1, D).to(_dev())
    n = 65536 // D
    pools, table, valid = _one_row_cache(n, D)
    ia.append_mxfp4_tokens(k, v, pools, table, valid)
    rk, rv = ia.read_mxfp4_tokens(pools, table, valid, n, dtype=torch.float32)
    for x, r, (codes, scales) in ((k, rk, _stored(pools, table, n)[0]), (v, rv, _stored(pools, table, n)[1])):
        want, ws = O.quantize(x.double().cpu().numpy().reshape(n, D))
        assert np.array_equal(scales, ws)
        assert _same_codes(codes, want)
        assert np.array_equal(r.cpu().numpy().reshape(n, D).astype(np.float64), O.values(want, ws), equal_nan=True)


def test_append_float32_ties_and_neighbours():
    """Every rounding boundary of the format, hit and missed by one step, at every scale."""
    import torch
    import intent_attention as ia
    edges = np.array([.25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.99], np.float32)
    three = np.concatenate([np.nextafter(edges, 0, dtype=np.float32), edges, np.nextafter(edges, 9, dtype=np.float32)])
    rows = []
    for e in range(-30, 20):
        for lead in (4.0, 7.5):
            for part in np.array_split(np.minimum(three, lead), 2):
                row = np.zeros(32, np.float32)
                row[0], row[1:1 + len(part)] = lead, part
                row[2::2] *= -1
                rows.append(row * np.float32(2.0 ** e))
    rows += [np.zeros(32, np.float32), np.full(32, 1e-45, np.float32), np.full(32, 3e38, np.float32)]
    while len(rows) % 2:
        rows.append(rows[0])
    x = np.stack(rows).reshape(-1, 64)
    n = x.shape[0]
    pools, table, valid = _one_row_cache(n, 64)
    ia.append_mxfp4_tokens(_t(x).view(1, n, 1, 64), _t(x[::-1]).view(1, n, 1, 64), pools, table, valid)
    for h, (codes, scales) in zip((x, x[::-1]), _stored(pools, table, n)):
        want, ws = O.quantize(h.astype(np.float64))
        assert np.array_equal(scales, ws) and _same_codes(codes, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,L,Hkv,D,start,strided", [(1, 1, 1, 64, 0, False), (3, 1, 2, 128, 15, False),
                                                     (4, 7, 3, 64, 13, True), (2, 33, 5, 128, 31, True),
                                                     (1, 130, 1, 128, 0, False)])
def test_append_read_ragged_rows(B, L, Hkv, D, start, strided, dtype):
    """Ragged new tokens over what is there: the tokens named and no other byte."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(B * 1000 + L)
    new = rng.integers(0, L + 1, B).astype(np.int32)
    new[0] = L
    valid = (start + np.arange(Hkv)[None, :] + new[:, None]).astype(np.int32)
    W = int(-(-valid.max() // 16)) + 1
    NP = B * Hkv * W + 3
    host, pools = _pools(rng, NP, D)
    before = {n: t.clone() for n, t in pools.tensors().items()}
    table = _table(rng, B, Hkv, W, NP)
    x = torch.randn((2, B, L, Hkv, D + (4 if strided else 0)), device=_dev()).to(getattr(torch, dtype))
    k, v = x[0][..., 1:D + 1] if strided else x[0], x[1][..., :D]        # odd offsets: element-wise loads
    ia.append_mxfp4_tokens(k, v, pools, _t(table), _t(valid), q_lens=_t(new))
    rk, rv = ia.read_mxfp4_tokens(pools, _t(table), _t(valid), L, q_lens=_t(new), dtype=getattr(torch, dtype))
    want = {n: t.cpu().numpy().copy() for n, t in before.items()}
    for b in range(B):
        for h in range(Hkv):
            for i in range(new[b]):
                pos = valid[b, h] - new[b] + i
                page = table[b, h, pos // 16]
                for s, t in (("k", k), ("v", v)):
                    c, e = O.quantize(t[b, i, h].double().cpu().numpy())
                    want[s + "_codes"][page, pos % 16], want[s + "_scales"][page, pos % 16] = O.pack(c), e
    for n, t in pools.tensors().items():
        g = t.cpu().numpy()
        if n.endswith("codes"):
            assert _same_codes(O.unpack(g), O.unpack(want[n])), n
        else:
            assert np.array_equal(g, want[n]), n
    for r, s in ((rk, "k"), (rv, "v")):
        for b in range(B):
            for i in range(L):
                for h in range(Hkv):
                    pos = valid[b, h] - new[b] + i
                    exp = np.zeros(D)
                    if i < new[b]:
                        page = table[b, h, pos // 16]
                        exp = O.values(O.unpack(want[s + "_codes"][page, pos % 16]), want[s + "_scales"][page, pos % 16])
                    assert np.array_equal(r[b, i, h].double().cpu().numpy(), exp)


def test_append_leaves_out_what_has_no_page():
    """Tokens before the row's start, past the table, on pages outside the pools: nothing written, zeros read."""
    import torch
    import intent_attention as ia
    D, NP = 64, 6
    pools = ia.MxFp4Pools.empty(NP, D, _dev())
    table = torch.tensor([[[0, -1]], [[NP, 2 ** 31 - 1]], [[-2 ** 31, 3]], [[4, 5]], [[1, 2]]], dtype=torch.int32, device=_dev())
    valid = torch.tensor([[20], [32], [32], [40], [-3]], dtype=torch.int32, device=_dev())
    k = torch.ones((5, 24, 1, D), device=_dev(), dtype=torch.float16)
    ia.append_mxfp4_tokens(k, k, pools, table, valid)
    rk, _ = ia.read_mxfp4_tokens(pools, table, valid, 24)
    there = np.zeros((5, 24), bool)
    there[0, 4:20] = True          # tokens -4 .. 19: the first page's 16
    there[2, 8:] = True            # tokens 8 .. 31: the second page's
    there[3] = True                # 40 tokens are 32, of which the last 24
    assert np.array_equal(rk[:, :, 0, 0].cpu().numpy() == 1, there)
    assert int((pools.k_scales[:, :, 0] != 0).sum()) == int(there.sum())


# ----------------------------------------------------------------------------- attention

CASES = [
    # B, L, Hq, Hkv, D, W, valid (cycled over rows), q_lens, dtype, causal, splits
    (1, 1, 1, 1, 64, 1, [1], None, "float16", True, 0),
    (1, 1, 8, 8, 128, 2, [17], None, "bfloat16", True, 0),
    (2, 1, 14, 2, 128, 5, [0, 1, 15, 80], None, "float16", True, 0),
    (3, 1, 8, 4, 64, 40, [16, 32, 33, 31, 640, 639, 500, 47], None, "float32", True, 0),
    (3, 1, 8, 4, 128, 40, [16, 32, 33, 31, 640, 639, 500, 47], None, "bfloat16", True, 5),
    (2, 1, 24, 1, 128, 9, [130, 144], None, "float16", False, 2),
    (1, 1, 32, 1, 64, 70, [1111], None, "float32", True, 0),
    (2, 4, 8, 2, 128, 12, [4, 190, 3, 5], None, "float16", True, 0),
    (2, 4, 8, 2, 128, 12, [4, 190, 3, 5], [2, 4], "float32", True, 3),
    (3, 7, 5, 1, 64, 12, [100, 1, 7], [0, 3, 7], "bfloat16", True, 0),
    (1, 16, 16, 16, 64, 4, [64, 16, 17, 33], None, "float16", True, 0),
    (2, 33, 4, 2, 128, 9, [33, 140, 60, 32], [33, 20], "float16", True, 0),
    (2, 33, 4, 2, 128, 9, [33, 140, 60, 32], [33, 20], "bfloat16", False, 2),
    (1, 70, 7, 1, 64, 20, [300], None, "float32", True, 0),
    (1, 129, 8, 2, 128, 17, [129, 260], None, "bfloat16", True, 0),
    (2, 150, 4, 1, 64, 30, [470, 150], [149, 150], "float16", True, 0),
    (1, 300, 2, 2, 128, 33, [515, 300], None, "float16", True, 4),
    (1, 300, 2, 2, 128, 33, [515, 300], None, "float32", False, 0),
]


@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,valid,q_lens,dtype,causal,splits", CASES)
def test_attention_against_oracle(B, L, Hq, Hkv, D, W, valid, q_lens, dtype, causal, splits):
    rng = np.random.default_rng(B * 7 + L * 131 + Hq)
    NP = B * Hkv * W + 5
    host, pools = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    v = np.resize(np.array(valid, np.int32), (B, Hkv))
    q = (2 * rng.standard_normal((B, L, Hq, D))).astype(np.float32)
    if L == 1 and B != 2:
        q = q[:, 0]
    _check(q, dtype, host, pools, table, v, None if q_lens is None else np.array(q_lens, np.int32), causal, splits=splits)


@pytest.mark.parametrize("L", [1, 5, 140])
def test_attention_output_types_and_strides(L):
    """q and out as parts of wider tensors, rows that 16 bytes do not divide, other output types."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L)
    B, Hq, Hkv, D, W = 2, 6, 2, 64, 14
    host, pools = _pools(rng, 80, D)
    table, valid = _table(rng, B, Hkv, W, 80), np.full((B, Hkv), 200, np.int32)
    wide = torch.randn((B, Hq, L, D + 3), device=_dev())
    for dtype, out_dtype in (("float16", "float32"), ("bfloat16", "float16"), ("float32", "bfloat16")):
        q = wide.to(getattr(torch, dtype))[..., 2:D + 2].transpose(1, 2)     # [B, L, Hq, D], head-major rows
        buf = torch.full((B, L, Hq, D + 5), 7.0, dtype=getattr(torch, out_dtype), device=_dev())
        out = buf[..., 1:D + 1]
        r = ia.mxfp4_paged_attention(q, pools, _t(table), _t(valid), out=out)
        assert r is out
        _check(q, dtype, host, pools, table, valid, out_dtype=out_dtype, got=out)
        assert (buf[..., 0] == 7).all() and (buf[..., D + 1:] == 7).all()


@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,splits", [(2, 1, 6, 2, 64, 14, 1), (2, 5, 8, 2, 128, 14, 3), (2, 140, 8, 2, 128, 14, 1),
                                                   (2, 140, 8, 2, 128, 14, 16), (1, 2050, 16, 2, 64, 20, 1)])
def test_attention_in_place(B, L, Hq, Hkv, D, W, splits):
    """The output in the query's place: the same bits."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L)
    _, pools = _pools(rng, B * Hkv * W, D)
    table, valid = _t(_table(rng, B, Hkv, W, B * Hkv * W)), _t(np.full((B, Hkv), W * 16 - 3, np.int32))
    q = torch.randn((B, L, Hq, D), device=_dev()).half()
    want = ia.mxfp4_paged_attention(q, pools, table, valid, causal=False, splits=splits)
    got = ia.mxfp4_paged_attention(q, pools, table, valid, causal=False, splits=splits, out=q)
    assert got is q and torch.equal(q, want)


@pytest.mark.parametrize("L", [1, 3, 140])
def test_attention_invalid_pages_hold_no_tokens(L):
    rng = np.random.default_rng(L + 50)
    B, Hq, Hkv, D, W, NP = 2, 4, 2, 128, 15, 64
    host, pools = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    table[0, 0, [0, 3, 4, 14]] = [-1, NP, 2 ** 31 - 1, -2 ** 31]
    table[1, 1, :] = -1
    valid = np.array([[235, 240], [233, 240]], np.int32)
    q = rng.standard_normal((B, L, Hq, D)).astype(np.float32)
    got = _check(q, "float16", host, pools, table, valid)
    assert (got[1, :, 2:] == 0).all()


@pytest.mark.parametrize("L", [1, 3, 140])
def test_attention_nan_blocks_and_unwritten_bytes(L):
    """A NaN block reaches the queries that see its token and no other; bytes past the last
    token (every value of a scale byte among them) reach none."""
    rng = np.random.default_rng(L + 90)
    B, Hq, Hkv, D, W, NP = 2, 4, 2, 128, 16, 64
    host, _ = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    valid = np.array([[250, 200], [149, 250]], np.int32)
    for n in ("k_scales", "v_scales"):
        for b in range(B):
            for h in range(Hkv):
                for t in range(valid[b, h], W * 16):
                    host[n][table[b, h, t // 16], t % 16] = rng.choice([0, 255, 254, 141, 103])
    host["k_scales"][table[0, 0, 248 // 16], 248 % 16, 2] = 255     # seen by the last two queries of causal rows
    host["v_scales"][table[1, 0, 0], 5, 1] = 255                    # seen by all
    host["v_scales"][table[1, 1, 249 // 16], 249 % 16, 0] = 255     # seen by the last
    import intent_attention as ia
    pools = ia.MxFp4Pools(**{n: _t(x) for n, x in host.items()})
    q = rng.standard_normal((B, L, Hq, D)).astype(np.float32)
    for causal in (True, False):
        got = _check(q, "bfloat16", host, pools, table, valid, causal=causal)
    assert not bool(got[0, :, 2:].isnan().any())


@pytest.mark.parametrize("L", [1, 140])
@pytest.mark.parametrize("dtype", DT)
def test_attention_query_values(L, dtype):
    """Queries of every size the type has, and infinite and NaN ones (their rows alone)."""
    import torch
    rng = np.random.default_rng(L + 7)
    B, Hq, Hkv, D, W, NP = 1, 8, 2, 64, 15, 32
    host, pools = _pools(rng, NP, D)
    table, valid = _table(rng, B, Hkv, W, NP), np.full((B, Hkv), 230, np.int32)
    q = rng.standard_normal((B, L, Hq, D)).astype(np.float32)
    q[:, :, 0] *= 2.0 ** -24
    q[:, :, 1, ::2] *= 2.0 ** -14
    q[:, :, 2] *= 2.0 ** 12 if dtype == "float16" else 2.0 ** 20
    q[:, :, 2, 1:] = 0
    q[0, 0, 3, 5] = np.inf
    q[0, L - 1, 4, 9] = np.nan
    q[:, :, 5] = 0
    if dtype != "float16":
        q[:, :, 6] *= 2.0 ** -100
    tq = torch.from_numpy(q).to(getattr(torch, dtype)).to(_dev())
    _check(tq, dtype, host, pools, table, valid)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_attention_of_queries_that_are_not_finite_and_see_nothing(dtype):
    """Infinite and NaN queries: zeros where a query sees no token, among queries that see some."""
    rng = np.random.default_rng(5)
    B, L, Hq, Hkv, D, W, NP = 2, 6, 4, 1, 64, 14, 40
    host, pools = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    table[1, 0, 0] = -1
    valid = np.array([[3], [19]], np.int32)           # the first three queries before the row's start; on no page
    q = rng.standard_normal((B, L, Hq, D)).astype(np.float32)
    q[:, 1, 0, 3], q[:, 2, 1, 0], q[:, 4, 2, 5] = np.nan, np.inf, np.nan
    for splits in (1, 3):
        got = _check(q, dtype, host, pools, table, valid, splits=splits)
        assert (got[0, :3] == 0).all() and bool(got[0, 4, 2].isnan().all())


# Sizes that the kernel for many query rows takes, in each of its forms: tiles of 128 rows and, for
# 16-bit queries, of 256; the whole row or splits of it.
PROMPTS = [
    # B, L, Hq, Hkv, D, W, dtype, causal, splits
    (1, 203, 4, 2, 64, 13, "float16", True, 16),
    (2, 140, 8, 2, 128, 14, "bfloat16", True, 16),
    (2, 140, 4, 1, 128, 15, "float32", False, 16),
    (2, 140, 8, 2, 64, 10, "float32", True, 16),
    (1, 2050, 16, 2, 64, 20, "bfloat16", False, 0),
    (1, 2050, 16, 2, 128, 20, "float16", False, 0),
    (1, 2050, 16, 2, 64, 20, "float32", False, 0),
    (1, 1500, 12, 3, 128, 10, "float32", False, 1),
    (2, 1100, 16, 2, 64, 70, "float16", True, 0),
    (2, 1100, 16, 2, 128, 70, "bfloat16", True, 0),
    (1, 1500, 4, 1, 64, 200, "bfloat16", True, 6),
    (1, 1500, 4, 1, 128, 300, "float16", True, 6),
]


@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,dtype,causal,splits", PROMPTS)
def test_attention_of_prompts(B, L, Hq, Hkv, D, W, dtype, causal, splits):
    """Prompts with all that may be in them at once: ragged lengths, pages that are none, NaN
    blocks seen by some queries and by none, any bytes past the last token, queries of all sizes and
    infinite ones, q and out as parts of wider tensors."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L + D + W)
    NP, T = B * Hkv * W + 7, W * 16
    host, _ = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    valid = np.full((B, Hkv), T - 5, np.int32)
    valid[-1, -1] = T - 42
    for n in ("k_scales", "v_scales"):
        for b in range(B):
            for h in range(Hkv):
                for t in range(valid[b, h], T):
                    host[n][table[b, h, t // 16], t % 16] = rng.choice([0, 255, 254, 141, 103])
    host["k_scales"][table[0, 0, (T - 9) // 16], (T - 9) % 16, 1] = 255       # seen by the last of causal queries
    host["v_scales"][table[-1, -1, (T - 45) // 16], (T - 45) % 16, 0] = 255
    table[0, -1, [1, W // 2, W - 1]] = [-1, NP, 2 ** 31 - 1]
    pools = ia.MxFp4Pools(**{n: _t(x) for n, x in host.items()})
    q = (2 * rng.standard_normal((B, L, Hq, D))).astype(np.float32)
    q[:, L // 2] *= 2.0 ** -12
    q[:, L // 2 + 1, :, 1:] = 0
    q[:, L // 2 + 1] *= 2.0 ** 10
    q[0, L - 2, 0, 3], q[-1, 1, -1, 0] = np.inf, np.nan
    wide = torch.full((B, Hq, L, D + 3), 3.0, device=_dev()).to(getattr(torch, dtype))
    wide[..., 2:D + 2] = _t(q).transpose(1, 2).to(wide.dtype)
    tq = wide[..., 2:D + 2].transpose(1, 2)
    buf = torch.full((B, L, Hq, D + 5), 7.0, device=_dev()).to(getattr(torch, dtype))
    lens = np.array([L, max(0, L - 77)][:B], np.int32)
    ia.mxfp4_paged_attention(tq, pools, _t(table), _t(valid), q_lens=_t(lens), causal=causal, out=buf[..., 1:D + 1],
                             splits=splits)
    queries = sorted({0, 1, 7, L // 3, L // 2, L // 2 + 1, L - 79, L - 78, L - 77, L - 5, L - 4, L - 3, L - 2, L - 1}
                     | {int(i) for i in rng.integers(0, L, 20)})
    got = _check(tq, dtype, host, pools, table, valid, lens, causal, got=buf[..., 1:D + 1], queries=queries)
    assert (buf[..., 0] == 7).all() and (buf[..., D + 1:] == 7).all()
    assert (got[-1, lens[-1]:] == 0).all()


# Several prompts whose tiles of rows are shared out over the card by their lengths.
SHARED = [
    # L, Hq, Hkv, D, W, valid tokens (a sequence each), q_lens, dtype, causal
    (700, 8, 2, 128, 200, [3190, 700, 33], None, "float16", True),
    (700, 8, 2, 128, 200, [3190, 1, 40], [700, 0, 33], "bfloat16", True),
    (700, 8, 2, 64, 250, [5, 3999, 2000], [3, 650, 699], "float16", True),
    (700, 8, 2, 64, 250, [4000, 0, 0], [1, 0, 700], "bfloat16", False),
    (700, 8, 2, 128, 200, [100, 3200, 1600], [100, 555, 700], "float32", True),
    (700, 8, 2, 64, 250, [4000, 4000, 16], [700, 700, 1], "float32", True),
    (700, 8, 2, 128, 200, [0, 0, 0], None, "float16", True),
    (509, 16, 4, 128, 250, [4000, 1500, 2000, 20, 3999], [509, 400, 509, 10, 1], "float16", True),      # two rounds
    (129, 24, 1, 64, 400, [6400, 300, 17, 0, 6000, 1], [129, 128, 1, 5, 60, 0], "float16", True),
]


@pytest.mark.parametrize("L,Hq,Hkv,D,W,tokens,q_lens,dtype,causal", SHARED)
def test_attention_of_unequal_prompts(L, Hq, Hkv, D, W, tokens, q_lens, dtype, causal):
    import intent_attention as ia
    rng = np.random.default_rng(L + W + D)
    B = len(tokens)
    NP = B * Hkv * W + 3
    host, pools = _pools(rng, NP, D)
    table = _table(rng, B, Hkv, W, NP)
    table[0, 0, W // 3] = -1
    valid = np.array(tokens, np.int32)[:, None].repeat(Hkv, 1)
    valid[:, -1] = np.maximum(0, valid[:, -1] - 21)                        # heads differ too
    q = (2 * rng.standard_normal((B, L, Hq, D))).astype(np.float32)
    q[0, 0, 0, 0] = np.nan
    lens = None if q_lens is None else np.array(q_lens, np.int32)
    queries = sorted({0, 1, L // 2, L - 2, L - 1} | {n + k for n in (q_lens or []) for k in (-1, 0) if 0 <= n + k < L}
                     | {int(i) for i in rng.integers(0, L, 8)})
    tq = _t(q).to(getattr(__import__("torch"), dtype))
    plan = ia.make_mxfp4_plan(tq, pools, _t(table), _t(valid), causal=causal)
    tiles = B * Hkv * -(-L * Hq // Hkv // (128 if dtype == "float32" else 256))
    rows = 65536 * (2 if tiles > 132 else 1)                               # of the rounds that are shared out
    assert plan.workspace_bytes == 2 * 4 * rows + 4 * rows * D + -(-8 * tiles // 256) * 256, "not the shared form"
    _check(tq, dtype, host, pools, table, valid, lens, causal, queries=queries)


@pytest.mark.parametrize("B,L,G,Hkv,D,W,dtype", [(32, 1, 4, 2, 128, 2048, "float16"), (48, 3, 5, 2, 64, 2500, "bfloat16"),
                                                 (64, 1, 8, 1, 128, 2048, "float32"), (85, 2, 2, 1, 64, 2048, "float32")])
def test_attention_of_one_long_row_among_short_ones(B, L, G, Hkv, D, W, dtype):
    """Decode rows that are shared out by their lengths: one fills its table, some are empty."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(B)
    NP, round_ = 600, 768 if D == 128 else 1024
    host, pools = _pools(rng, NP, D)
    table = rng.integers(0, NP, (B, Hkv, W)).astype(np.int32)              # pages many times over
    table[1, 0, 1000] = NP
    valid = rng.integers(0, 90, (B, Hkv)).astype(np.int32)
    valid[1, 0], valid[2], valid[3] = W * 16 - 7, 0, 1
    q = (2 * rng.standard_normal((B, L, G * Hkv, D))).astype(np.float32)
    q[5, 0, 0, 3] = np.inf
    lens = None if L == 1 else rng.integers(0, L + 1, B).astype(np.int32)
    if L > 1:
        lens[1] = L
    tq = _t(q).to(getattr(torch, dtype))
    plan = ia.make_mxfp4_plan(tq, pools, _t(table), _t(valid))
    rows, tiles = round_ * 16, B * Hkv * -(-L * G // 16)
    assert plan.workspace_bytes == 2 * 4 * rows + 4 * rows * D + -(-8 * tiles // 256) * 256, "not the shared form"
    _check(tq, dtype, host, pools, table, valid, lens)


def test_attention_of_prompts_replays():
    """A captured prompt, replayed with other data and lengths between eager work: the eager results, bit for bit."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(12)
    for B, L, Hq, Hkv, D, W, splits in ((2, 140, 8, 2, 128, 14, 16), (2, 1100, 16, 2, 64, 70, 0), (3, 700, 8, 2, 128, 200, 0)):
        _, pools = _pools(rng, B * Hkv * W, D)
        table, valid = _t(_table(rng, B, Hkv, W, B * Hkv * W)), _t(np.full((B, Hkv), W * 16, np.int32))
        q = torch.randn((B, L, Hq, D), device=_dev()).half()
        plan = ia.make_mxfp4_plan(q, pools, table, valid, splits=splits)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            plan.run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run()
        for it in range(4):
            q.copy_(torch.randn_like(q))
            valid.fill_(W * 16 - 31 * it)
            graph.replay()
            torch.cuda.synchronize()
            got = plan.out.clone()
            want = ia.mxfp4_paged_attention(q, pools, table, valid, splits=splits)
            torch.cuda.synchronize()
            assert torch.equal(got, want), it


def test_attention_sharp_and_growing_scores():
    """Scores that keep growing along the row (the running maximum moves at each step) and a
    single token that outweighs the rest."""
    import intent_attention as ia
    rng = np.random.default_rng(3)
    D, W = 64, 20
    pools, table, valid = _one_row_cache(W * 16, D)
    k = np.ones((1, W * 16, 1, D), np.float32) * np.linspace(0.01, 6, W * 16, dtype=np.float32)[None, :, None, None]
    k[0, 100] = 40
    v = rng.standard_normal((1, W * 16, 1, D)).astype(np.float32)
    ia.append_mxfp4_tokens(_t(k), _t(v), pools, table, valid)
    host = {n: t.cpu().numpy() for n, t in pools.tensors().items()}
    for scale in (0.05, 1.0, -1.0):
        for L in (1, 150):
            q = np.full((1, L, 2, D), 1.0, np.float32)
            _check(q, "float16", host, pools, table.cpu().numpy(), valid.cpu().numpy(), sm_scale=scale)


def test_attention_small_weights_of_many_tokens_count():
    """One token 2^18 above 32,767 equal ones: the many weights, each far below float16's step at
    the largest weight, add up to an eighth of it."""
    import torch
    import intent_attention as ia
    D, W = 64, 2048
    pools, table, valid = _one_row_cache(W * 16, D)
    k = torch.zeros((1, W * 16, 1, D), device=_dev())
    k[0, 777, 0, 0] = 6.0
    v = torch.full((1, W * 16, 1, D), 4.0, device=_dev())
    v[0, 777] = 0.0
    ia.append_mxfp4_tokens(k, v, pools, table, valid)
    q = torch.zeros((1, 1, 1, D), device=_dev(), dtype=torch.float16)
    q[..., 0] = 1.0
    got = ia.mxfp4_paged_attention(q, pools, table, valid, sm_scale=3 * float(np.log(2.0)))
    n = (W * 16 - 1) * 2.0 ** -18
    want = 4.0 * n / (1 + n)
    assert abs(float(got[0, 0, 0, 0]) - want) <= want * (2.0 ** -10 + (W * 16) * 2.0 ** -24)


def test_attention_rows_at_high_offsets():
    """Pages whose byte offsets pass 2^32."""
    import torch
    import intent_attention as ia
    D, NP = 128, (1 << 22) + 100                     # 4 GiB of codes a side
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    pools = ia.MxFp4Pools.empty(NP, D, _dev())
    table = torch.tensor([[[NP - 1, 0, NP - 2]]], dtype=torch.int32, device=_dev())
    valid = torch.full((1, 1), 45, dtype=torch.int32, device=_dev())
    x = torch.randn((2, 1, 45, 1, D), device=_dev())
    ia.append_mxfp4_tokens(x[0], x[1], pools, table, valid)
    k, v = ia.read_mxfp4_tokens(pools, table, valid, 45, dtype=torch.float32)
    for r, t in ((k, x[0]), (v, x[1])):
        c, e = O.quantize(t.double().cpu().numpy())
        assert np.array_equal(r.cpu().numpy().astype(np.float64), O.values(c, e))
    small = {n: t[[NP - 1, 0, NP - 2]].contiguous() for n, t in pools.tensors().items()}
    near = torch.tensor([[[0, 1, 2]]], dtype=torch.int32, device=_dev())
    for L in (1, 40):
        q = torch.randn((1, L, 4, D), device=_dev()).half()
        far = ia.mxfp4_paged_attention(q, pools, table, valid)
        assert torch.equal(far, ia.mxfp4_paged_attention(q, ia.MxFp4Pools(**small), near, valid))


@pytest.mark.parametrize("L", [1, 4, 140])
def test_attention_is_deterministic_and_replays(L):
    """A captured append and attention, replayed with other data and lengths between eager
    work, give the eager results bit for bit; two plans on two streams do not disturb each other."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L)
    B, Hq, Hkv, D, W = 3, 8, 2, 128, 40
    NP = B * Hkv * W
    host, pools = _pools(rng, NP, D)
    table = _t(_table(rng, B, Hkv, W, NP))
    valid = _t(np.full((B, Hkv), 300, np.int32))
    q = torch.randn((B, L, Hq, D), device=_dev()).half()
    kv = torch.randn((2, B, L, Hkv, D), device=_dev()).half()
    plan = ia.make_mxfp4_plan(q, pools, table, valid)

    def step():
        ia.append_mxfp4_tokens(kv[0], kv[1], pools, table, valid)
        plan.run()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for it in range(4):
        q.copy_(torch.randn_like(q))
        kv.copy_(torch.randn_like(kv))
        valid.fill_(150 + 130 * it)
        graph.replay()
        torch.cuda.synchronize()
        got = plan.out.clone()
        ia.append_mxfp4_tokens(kv[0], kv[1], pools, table, valid)
        want = ia.mxfp4_paged_attention(q, pools, table, valid)
        torch.cuda.synchronize()
        assert torch.equal(got, want), it
    other = ia.make_mxfp4_plan(q, pools, table, valid)
    want = plan.out.clone()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        plan.run()
        with torch.cuda.stream(side):
            other.run()
    torch.cuda.synchronize()
    assert torch.equal(plan.out, other.out)


def test_attention_nothing_to_do():
    import torch
    import intent_attention as ia
    D = 64
    pools = ia.MxFp4Pools.empty(4, D, _dev())
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=_dev())  # noqa: E731
    assert ia.mxfp4_paged_attention(torch.ones((0, 4, D), device=_dev()), pools, i32(0, 2, 3), i32(0, 2)).shape == (0, 4, D)
    assert ia.mxfp4_paged_attention(torch.ones((2, 0, 4, D), device=_dev()), pools, i32(2, 2, 3), i32(2, 2)).shape == (2, 0, 4, D)
    assert (ia.mxfp4_paged_attention(torch.ones((2, 4, D), device=_dev()), pools, i32(2, 2, 0), i32(2, 2) + 5) == 0).all()
    none = ia.MxFp4Pools.empty(0, D, _dev())
    assert (ia.mxfp4_paged_attention(torch.ones((2, 5, 4, D), device=_dev()), none, i32(2, 2, 3), i32(2, 2) + 40) == 0).all()
    k = torch.ones((2, 5, 2, D), device=_dev())
    ia.append_mxfp4_tokens(k, k, none, i32(2, 2, 3), i32(2, 2) + 40)
    ia.append_mxfp4_tokens(k[:, :0], k[:, :0], pools, i32(2, 2, 3), i32(2, 2) + 40)
    assert (ia.read_mxfp4_tokens(none, i32(2, 2, 3), i32(2, 2) + 40, 3)[0] == 0).all()
