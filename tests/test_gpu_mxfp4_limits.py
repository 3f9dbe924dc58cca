"""The 4-bit token cache at the limits that its documentation states: lengths past the table, queries
whose elements are of very different size."""
import numpy as np
import pytest

from oracle import mxfp4 as O
from tests.test_gpu_mxfp4 import HALF, _dev, _pools, _t, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,L", [(64, 24), (128, 3), (64, 150)])
def test_a_length_past_the_table_is_a_full_table(D, L):
    """Append, read and attention: the same bytes and values as for a row that fills its table."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L)
    B, Hkv, W = 3, 2, 11
    host, pools = _pools(rng, 80, D)
    other = ia.MxFp4Pools(**{n: t.clone() for n, t in pools.tensors().items()})
    table = _t(_table(rng, B, Hkv, W, 80))
    full = _t(np.full((B, Hkv), 16 * W, np.int32))
    past = _t(np.array([[16 * W + 1, 16 * W + 40], [2 ** 31 - 1, 16 * W], [16 * W + 9, 10 ** 6]], np.int32))
    lens = _t(np.array([L, max(1, L - 5), 0], np.int32))
    k, v = torch.randn((2, B, L, Hkv, D), device=_dev()).half()
    q = torch.randn((B, L, 4, D), device=_dev()).half()
    got = []
    for p, valid in ((pools, past), (other, full)):
        ia.append_mxfp4_tokens(k, v, p, table, valid, q_lens=lens)
        got.append([*p.tensors().values(), *ia.read_mxfp4_tokens(p, table, valid, L, q_lens=lens),
                    ia.mxfp4_paged_attention(q, p, table, valid, q_lens=lens),
                    ia.mxfp4_paged_attention(q, p, table, valid, causal=False)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


# What a row's largest element costs the others. A query element is off by half of float16's smallest
# step, 2^-25, where the row's largest is scaled to 2^14 at least: 2^-39 of that one (16-bit elements; of
# float32's two halves the second: 2^-22 of the element, or as much). A score is off by that times the sum
# of |k| times |sm_scale|, beside what test_gpu_mxfp4._bound counts; twice, for a weight over the sum.
def _score_error(q, host, table, valid, sm):
    """float64 [B, L, Hq]: the largest |sm| 2^-39 max|q| sum|k| of each query's tokens."""
    most = np.abs(q).max(-1)
    G, err = q.shape[2] // table.shape[1], np.zeros(q.shape[:3])
    for b, h in np.ndindex(*table.shape[:2]):
        k, _ = O.row_values(host["k_codes"], host["k_scales"], table[b, h], int(valid[b, h]), host["k_codes"].shape[0])
        err[b, :, h * G:(h + 1) * G] = most[b, :, h * G:(h + 1) * G] * np.abs(k).sum(-1).max(initial=0.0) * 2.0 ** -39 * abs(sm)
    return err


@pytest.mark.parametrize("L", [1, 5, 140])
@pytest.mark.parametrize("dtype,big,small", [("float16", 2.0 ** 15, 2.0 ** -6), ("float16", 2.0 ** 15, 2.0 ** -13), ("bfloat16", 2.0 ** 20, 1.0),
                                             ("bfloat16", 2.0 ** 20, 2.0 ** -9), ("float32", 2.0 ** 20, 1.0), ("float32", 2.0 ** 20, 2.0 ** -9)])
def test_outlier_channels_over_small_keys(dtype, big, small, L):
    """A query channel that towers above the rest meets keys at the format's smallest scales: the
    others carry the score too, to the stated bound. With `small` 2^-28 of `big` and more they are
    exact in the 16-bit types; below, rounded."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L)
    B, Hq, Hkv, D, W, NP = 2, 4, 2, 64, 14, 60
    host, _ = _pools(rng, NP, D)
    step = int(np.log2(big))
    host["k_scales"][..., 0] = np.clip(127 - step + rng.integers(-2, 2, (NP, 16)), 104, 140)     # the outlier's products: of order 1
    host["k_scales"][..., 1] = np.clip(127 - int(np.log2(small)) + rng.integers(-2, 2, (NP, 16)), 104, 140)
    pools = ia.MxFp4Pools(**{n: _t(x) for n, x in host.items()})
    table, valid = _table(rng, B, Hkv, W, NP), np.full((B, Hkv), 16 * W - 3, np.int32)
    q = small * rng.uniform(1, 2, (B, L, Hq, D)) * rng.choice([-1, 1], (B, L, Hq, D))
    q[..., 7] = big * rng.uniform(0.5, 1, (B, L, Hq)) * rng.choice([-1, 1], (B, L, Hq))
    q[..., :7], q[..., 8:32] = 0, 0
    tq = torch.from_numpy(q).to(getattr(torch, dtype)).to(_dev())
    got = ia.mxfp4_paged_attention(tq, pools, _t(table), _t(valid), out_dtype=torch.float32).double().cpu().numpy()
    hq = tq.double().cpu().numpy()
    sm = 1 / np.sqrt(D)
    queries = sorted({0, L // 2, L - 1})
    want, mass, reach = O.attention(hq, host, table, valid, queries=queries)
    score = (((D + 6) * 2.0 ** -24 + (2.0 ** -22 if dtype == "float32" else 0.0)) * reach + _score_error(hq, host, table, valid, sm))[..., None]
    vmax = max(float(np.abs(O.row_values(host["v_codes"], host["v_scales"], r, 16 * W, NP)[0]).max()) for r in table.reshape(-1, W))
    T = 16 * W
    rel = 2 * np.expm1(2 * score) + (2.0 ** -22 if dtype == "float32" else 2.0 ** -11) + 2.0 ** -22 + 2 * (T + 8) * 2.0 ** -24
    tol = rel * mass + T * 2.0 ** -31 * vmax + HALF["float32"] * np.abs(want) + 2.0 ** -25
    assert float(rel[:, queries].max()) < 0.25                       # the bound says something
    err = np.abs(got - want)[:, queries] / tol[:, queries]
    assert float(err.max()) <= 1.0


@pytest.mark.parametrize("L", [1, 140])
def test_elements_of_every_size_count_to_the_stated_step(L):
    """One element a row beside the largest, which meets keys of 0: the score is the element's alone,
    right to 2^-39 of the largest; from 2^-28 of it on as exact as alone."""
    import torch
    import intent_attention as ia
    D = 64
    codes, scales = np.zeros((1, 16, D // 2), np.uint8), np.full((1, 16, 2), 127, np.uint8)
    codes[0, 0, 16], codes[0, 1, 16] = 0x07, 0x0F                    # channel 32: 6 and -6 times 2^13
    scales[0, :, 1] = 140
    vals = np.zeros((1, 16, D // 2), np.uint8)
    vals[0, 0], vals[0, 1] = 0x22, 0xAA                              # 1 and -1
    pools = ia.MxFp4Pools(*(_t(x) for x in (codes, scales, vals, np.full((1, 16, 2), 127, np.uint8))))
    table, valid = _t(np.zeros((1, 1, 1), np.int32)), _t(np.full((1, 1), 2, np.int32))
    for dtype, powers in (("bfloat16", range(0, 45)), ("float32", range(0, 45)), ("float16", range(0, 30))):
        for p in powers:
            top = 2.0 ** 15 if dtype == "float16" else 2.0 ** 20
            small = 1.2890625 * top * 2.0 ** -p / 1.5                # not a power of two
            q = torch.zeros((1, L, 1, D), dtype=torch.float64)
            q[..., 0], q[..., 32] = top, small
            q = q.to(getattr(torch, dtype))
            x = float(q[0, 0, 0, 32])
            if x == 0.0:
                continue
            sm = 0.5 / (x * 49152)                                   # scores 0.5 and -0.5
            got = ia.mxfp4_paged_attention(q.to(_dev()), pools, table, valid, causal=False, sm_scale=sm, out_dtype=torch.float32)
            off = (2.0 ** -22 if dtype == "float32" else 0.0) + (2.0 ** -39 * top / x if x < 2.0 ** -28 * top or dtype == "float32" else 0.0)
            # out = tanh(score), its slope at most 1; weights of 11 bits (22), exponentials, sums
            tol = 0.5 * off + 0.5 * 16 * 2.0 ** -24 + (2.0 ** -22 if dtype == "float32" else 2.0 ** -11) + 2.0 ** -20
            assert float((got.double().cpu() - np.tanh(0.5)).abs().max()) <= tol, (dtype, p)


@pytest.mark.parametrize("L", [1, 140])
def test_weights_of_16_bit_queries_keep_11_bits(L):
    """In a wider output the weights' rounding shows: 2^-11 of sum p |v|, no more."""
    import torch
    import intent_attention as ia
    rng = np.random.default_rng(L + 4)
    B, Hq, Hkv, D, W, NP = 1, 8, 2, 64, 14, 30
    host, pools = _pools(rng, NP, D)
    table, valid = _table(rng, B, Hkv, W, NP), np.full((B, Hkv), 16 * W, np.int32)
    T, vmax = 16 * W, 6 * 2.0 ** 0                                   # scale bytes up to 127
    q = torch.from_numpy(rng.standard_normal((B, L, Hq, D)).astype(np.float32)).to(_dev())
    queries = sorted({0, L // 2, L - 1})
    for dtype, weight in ((torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -11), (torch.float32, 2.0 ** -22)):
        got = ia.mxfp4_paged_attention(q.to(dtype), pools, _t(table), _t(valid), out_dtype=torch.float32).double().cpu().numpy()
        hq = q.to(dtype).double().cpu().numpy()
        want, mass, reach = O.attention(hq, host, table, valid, queries=queries)
        score = (((D + 6) * 2.0 ** -24 + 2.0 ** -22) * reach + _score_error(hq, host, table, valid, 1 / np.sqrt(D)))[..., None]
        rel = 2 * np.expm1(2 * score) + weight + 2.0 ** -22 + 2 * (T + 8) * 2.0 ** -24
        tol = rel * mass + T * 2.0 ** -31 * vmax + HALF["float32"] * np.abs(want)
        assert float((np.abs(got - want)[:, queries] / tol[:, queries]).max()) <= 1.0, dtype


def test_a_plans_run_marks_its_output():
    """torch's version counter of `out` moves with every run, the plan's own and a caller's, in place too."""
    import torch
    import intent_attention as ia
    pools = ia.MxFp4Pools.empty(4, 64, _dev())
    table, valid = _t(np.zeros((1, 2, 2), np.int32)), _t(np.full((1, 2), 20, np.int32))
    q = torch.randn((1, 4, 64), device=_dev()).half()
    for out in (None, torch.empty_like(q), q):
        plan = ia.make_mxfp4_plan(q, pools, table, valid, out=out)
        for _ in range(2):
            before = plan.out._version
            plan.run()
            assert plan.out._version == before + 1
        if out is not None:
            before = out._version
            ia.mxfp4_paged_attention(q, pools, table, valid, out=out)
            assert out._version == before + 1
    x = q.clone().requires_grad_()
    y = (x * 1).sin()                                                # sin keeps its input for its gradient
    with torch.no_grad():
        kept = y.grad_fn._saved_self
        ia.make_mxfp4_plan(kept, pools, table, valid, out=kept).run()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_numbers_that_an_int32_would_wrap():
    import torch
    import intent_attention as ia
    pools = ia.MxFp4Pools.empty(4, 64, _dev())
    table, valid = _t(np.zeros((1, 2, 2), np.int32)), _t(np.full((1, 2), 20, np.int32))
    q = torch.randn((1, 4, 64), device=_dev()).half()
    for splits in (2 ** 32, 2 ** 32 + 1, 2 ** 31, -2 ** 32):
        with pytest.raises(ValueError, match="splits"):
            ia.mxfp4_paged_attention(q, pools, table, valid, splits=splits)
    with pytest.raises(ValueError, match="count"):
        ia.read_mxfp4_tokens(pools, table[:0], valid[:0], 2 ** 32)
