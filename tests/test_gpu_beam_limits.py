"""The beam choice where its lists fill with equal logits, where one logit is far above the others, and where 64 bits do not tell
candidates apart."""
import numpy as np
import pytest

from test_gpu_beam_search import _check

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _few_above(V, low, high, at, dtype):
    """A row of `low` with `high` at the places `at`, and its mirror image."""
    import torch
    x = torch.full((V,), low, dtype=torch.float64)
    x[at] = high
    return torch.stack([x, x.flip(0)]).to(getattr(torch, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low,high", [(-9.0, -8.9375), (-2.0, -1.0), (-1.0, -0.75), (-5.0, -4.96875), (-0.0078125, 0.0), (3.0, 3.5), (0.0, 1.0)])
@pytest.mark.parametrize("V,at", [(2000, [100, 900]), (4000, [3999]), (20011, [5, 4100, 12000]), (131072, [70000])])
def test_few_above_many_equal(V, at, low, high, dtype):
    import torch
    rows = _few_above(V, low, high, at, dtype)
    for count in (2, 4, 17, 64):
        for row in rows:
            _check(row.view(1, 1, V), torch.tensor([[-3.0]]), count)
        _check(rows.view(1, 2, V), torch.tensor([[-3.0, -3.0]]), count)
        _check(rows.view(2, 1, V), torch.tensor([[-3.0], [-2.5]]), count)


@pytest.mark.parametrize("low", [3.0, -3.0, -0.25, 17.0])
def test_next_numbers_above_many_equal(low):
    """float32 neighbours: the larger ones come first by their logits."""
    import torch
    high = float(np.nextafter(np.float32(low), np.float32(np.inf)))
    for V, at in ((4000, [77]), (30000, [29999, 1])):
        rows = _few_above(V, low, high, at, "float32")
        for count in (4, 17, 64):
            _check(rows[:1].view(1, 1, V), torch.tensor([[0.0]]), count)
            _check(rows[1:].view(1, 1, V), torch.tensor([[0.0]]), count)


LARGE = [89.0, 599.0, 601.0, 709.0, 711.0, 800.0, 1000.0, 1400.0, 1419.6, 2000.0, 2839.0, 2848.0, 2900.0, 28391.0, 60000.0, 1e9]


@pytest.mark.parametrize("top,dtype", [(top, t) for t in TYPES for top in LARGE if t != "float16" or top <= 65504])
def test_one_large_logit(top, dtype):
    import torch
    for V in (1000, 32000):
        x = torch.zeros(3, V)
        x[0, V // 3] = top
        x[1] = torch.randn(V, generator=torch.Generator().manual_seed(V))
        x[1, V - 1] = top
        x[2, 0] = x[2, V // 2] = top
        x = x.to(getattr(torch, dtype))
        _check(x.view(1, 3, V), torch.tensor([[-5.0, -4.5, -6.0]]), 8)
        _check(x.view(3, 1, V), torch.tensor([[-5.0], [0.0], [-1.0]]), 5)


@pytest.mark.parametrize("shift", [711.0, 1419.6, 2839.0, 2839.13, 28391.0])
def test_rows_at_the_turns_of_the_exponent(shift):
    """Rows all of whose logits lie where 2^(32 x / ln 2) would come round again."""
    import torch
    x = torch.randn(2, 2, 5000, generator=torch.Generator().manual_seed(1)) + shift
    _check(x, torch.tensor([[-1.0, -2.0], [-1.0, -1.0]]), 9)


@pytest.mark.parametrize("V", [3000, 70001])
@pytest.mark.parametrize("scores", [[-1.0, -1.0], [-1.0, -0.5], [-1e9, -1e9], [3e9, 1e9]])
def test_one_beams_candidates_come_by_logit(V, scores):
    """Logits so close that the candidates are equal in 64 bits: a beam's come in the order of its logits, beams in theirs."""
    import torch
    import intent_attention as ia
    g = torch.Generator().manual_seed(V)
    x = torch.randn(2, V, generator=g) * (1e-20 if abs(scores[0]) < 10 else 1e-11)
    x[:, ::3] = 0
    s = torch.tensor([scores])
    for count in (5, 64):
        got = ia.beam_select(x.view(1, 2, V).cuda(), s.cuda(), count=count)
        # either beam's candidates are one number in 64 bits
        k = np.repeat([0, 1], V)
        value = np.repeat(np.asarray(scores), V)
        order = np.lexsort((np.tile(np.arange(V), 2), -x.double().numpy().ravel(), k, -value))[:count]
        assert got[1][0].tolist() == (order // V).tolist()
        assert got[2][0].tolist() == (order % V).tolist()
