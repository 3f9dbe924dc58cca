"""The beam choice on the GPU against float64: beams, tokens and their order exactly, scores within a
rounding; ties, beams out of the search, special logits, layouts, graphs and streams."""
import numpy as np
import pytest

from oracle import beam_search as O

pytestmark = pytest.mark.gpu


def _case(seed, B, K, V, dtype, scale=3.0, done=0.0, banned=0.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, K, V, generator=g) * scale).to(getattr(torch, dtype))
    if banned:
        x[:, :, torch.rand(V, generator=g) < banned] = float("-inf")
    s = -20 + 5 * torch.randn(B, K, generator=g)
    f = torch.rand(B, K, generator=g) < done if done else None
    return x, s, f


def _check(x, s, count, f=None, end=0, gx=None):
    import torch
    import intent_attention as ia
    gx = x.cuda() if gx is None else gx
    got = ia.beam_select(gx, s.cuda(), count=count, finished=None if f is None else f.cuda(), end_token=end)
    want = O.select(x.double().numpy(), s.double().numpy(), count, None if f is None else f.numpy(), end)
    assert got[0].dtype == torch.float32 and got[1].dtype == got[2].dtype == torch.int32
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[2].cpu().numpy(), want[2])
    g, w = got[0].double().cpu().numpy(), want[0]
    assert np.array_equal(np.isinf(g), np.isinf(w)) and not np.isnan(g).any()
    fine = np.isfinite(w)
    # a rounding to float32, and the normaliser's 1e-9 (its terms are off by 2^-30 each, the last step of |r| 2^-24)
    assert (np.abs(g[fine] - w[fine]) <= 2.0 ** -24 * np.abs(w[fine]) + 2.0 ** -28).all()
    return got


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("B,K,V,count", [(1, 1, 1, 1), (2, 3, 2, 6), (1, 2, 7, 5), (3, 4, 1000, 8), (2, 4, 2047, 4), (2, 4, 2049, 16),
                                         (1, 8, 32000, 16), (5, 3, 8191, 64), (1, 16, 8193, 32), (2, 1, 50021, 64), (1, 256, 300, 64),
                                         (33, 2, 513, 1), (17, 5, 20000, 10)])
def test_choice(B, K, V, count, dtype):
    x, s, _ = _case(B * 1000 + V + count, B, K, V, dtype)
    _check(x, s, count)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_finished_and_banned(dtype):
    for seed in range(4):
        x, s, f = _case(seed, 6, 4, 3001, dtype, done=0.4, banned=0.4)
        _check(x, s, 8, f, end=(0, 1, 3000, 7)[seed])
    # everyone at the end: more wanted than there are
    x, s, f = _case(9, 2, 3, 50, dtype)
    _check(x, s, 20, f=(s < 1e9), end=3)


def test_equal_logits_come_by_number():
    import torch
    for V in (5, 2048, 2050, 30011):
        x = torch.zeros(2, 3, V, dtype=torch.float16)
        _check(x, torch.tensor([[-1.0, -1, -1], [-3, -2, -2]]), 7 if V > 5 else 15)
        _check(x, torch.zeros(2, 3), min(64, 3 * V))
    x = torch.zeros(1, 2, 9000)
    x[0, :, ::3] = -0.0                                          # both zeros are one value
    _check(x, torch.zeros(1, 2), 64)
    # few values: many ties inside and across segments
    g = torch.Generator().manual_seed(3)
    x = torch.randint(0, 4, (3, 4, 20000), generator=g).to(torch.bfloat16)
    _check(x, torch.zeros(3, 4), 33)


def test_rising_and_falling_logits():
    import torch
    up = torch.arange(20000, dtype=torch.float32) * 1e-3
    x = torch.stack([up, up.flip(0), up, up.flip(0)]).view(1, 4, -1)
    _check(x, torch.tensor([[-1.0, -1.00005, -3, -0.99995]]), 64)


def test_beams_out_of_the_search():
    import torch
    inf, nan = float("inf"), float("nan")
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        x, _, _ = _case(1, 2, 6, 5000, "float32")
        x = x.to(dtype)
        x[0, 1, 4999] = nan
        x[0, 2, 0] = inf
        x[0, 3] = -inf
        x[1, :, 17] = nan
        s = torch.tensor([[-1.0, 0, 0, 0, nan, -inf], [-1, -2, inf, 0, 0, 0]])
        _check(x, s, 12)
        f = torch.zeros(2, 6, dtype=torch.bool)
        f[:, 1:3] = True
        _check(x, s, 12, f, end=2)
        first = torch.full((2, 6), -inf)                         # a search's first step: one beam counts
        first[:, 0] = 0
        x[1, 0, 17] = 0
        _check(x, first, 12)


@pytest.mark.parametrize("shift", [100.0, -90.0, 3e4, 60000.0, 7e4, -7e4, 1e30, -1e30, 3.3e38])
def test_large_logits(shift):
    import torch
    x, s, _ = _case(4, 2, 3, 3000, "float32", scale=4.0)
    x = torch.minimum(x + shift, torch.tensor(3.4e38)) if abs(shift) < 1e29 else x * (shift / 20)
    _check(x, s, 9)
    _check(x.to(torch.bfloat16).clamp(-3e38, 3e38), s, 9)


def test_one_certain_token_and_flat_rows():
    import torch
    x = torch.full((1, 3, 4000), -80.0)
    x[0, 0, 1234] = 80.0
    x[0, 1, :] = -600.0
    x[0, 2, 0] = 700.0                                           # further apart than 32 bits' exponentials reach
    _check(x, torch.tensor([[-5.0, -2.0, -1.0]]), 8)


def test_layouts():
    import torch
    x, s, f = _case(5, 3, 4, 1001, "bfloat16", done=0.3)
    big = torch.zeros(3, 7, 2111, dtype=torch.bfloat16, device="cuda")
    view = big[:, 1:5, 33:1034]                                  # odd addresses
    view.copy_(x)
    _check(x, s, 8, f, 9, gx=view)
    _check(x, s, 8, f, 9, gx=x.cuda().transpose(1, 2).contiguous().transpose(1, 2))
    one = x[:, :1].expand(3, 4, 1001)                            # all beams read one row
    _check(one.contiguous(), s, 8, gx=x.cuda()[:, :1].expand(3, 4, 1001))
    import intent_attention as ia
    a = ia.beam_select(x.cuda(), s.cuda(), finished=f.cuda(), end_token=4)
    b = ia.beam_select(x.cuda(), s.cuda(), finished=f.to(torch.uint8).mul(200).cuda(), end_token=4)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and a[0].shape == (3, 4)
    empty = ia.beam_select(torch.zeros(0, 4, 10, device="cuda"), torch.zeros(0, 4, device="cuda"))
    assert [t.shape for t in empty] == [(0, 4)] * 3


def test_long_batch():
    """More rows than a grid's second axis holds."""
    x, s, _ = _case(6, 9000, 4, 17, "float16")
    _check(x, s, 4)


def test_graph_and_streams():
    import torch
    import intent_attention as ia
    x, s, f = _case(7, 4, 4, 9001, "float32", done=0.2)
    gx, gs, gf = x.cuda(), s.cuda(), f.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ia.beam_select(gx, gs, count=8, finished=gf, end_token=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ia.beam_select(gx, gs, count=8, finished=gf, end_token=1)
    for seed in range(3):
        x, s, f = _case(20 + seed, 4, 4, 9001, "float32", done=0.2)
        gx.copy_(x), gs.copy_(s), gf.copy_(f)
        graph.replay()
        again = ia.beam_select(gx, gs, count=8, finished=gf, end_token=1)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, again))
        want = O.select(x.double().numpy(), s.double().numpy(), 8, f.numpy(), 1)
        assert np.array_equal(got[2].cpu().numpy(), want[2])
