"""The beam choice's lists and thresholds on the GPU: logits in orders that fill them, lists of many segments and beams, normalisers of
segments of very different sizes, candidates of two beams that differ by some 1e-8."""
import numpy as np
import pytest

from test_gpu_beam_search import _check

pytestmark = pytest.mark.gpu

TYPES = ["float32", "float16", "bfloat16"]


def _scores(B, K, seed=0):
    import torch
    return -30 + 4 * torch.randn((B, K), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("order", ["up", "down", "flat", "saw", "steps", "few"])
@pytest.mark.parametrize("count", [1, 17, 64])
def test_orders_that_fill_the_lists(order, count, dtype):
    import torch
    V = 70001
    i = torch.arange(V, dtype=torch.float64)
    x = {"up": i / V * 9, "down": -i / V * 9, "flat": 0 * i + 2.5, "saw": (i % 4097) / 500, "steps": torch.floor(i / 700) % 13,
         "few": torch.where(i % 9973 == 5, i / V, float("-inf"))}[order]
    x = torch.stack([x, x.flip(0)]).view(1, 2, V).to(getattr(torch, dtype))
    _check(x, _scores(1, 2), count)


@pytest.mark.parametrize("B,K,V,count", [(1, 256, 700, 64), (2, 40, 5000, 33), (1, 1, 200001, 64), (1, 16, 60000, 64), (3, 5, 40000, 40), (1, 200, 3, 64)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_lists(B, K, V, count, dtype):
    import torch
    x = (torch.randn((B, K, V), generator=torch.Generator().manual_seed(V)) * 3).to(getattr(torch, dtype))
    f = torch.rand((B, K), generator=torch.Generator().manual_seed(V + 1)) < 0.2
    _check(x, _scores(B, K, V), count, f, V // 2)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("low,high", [(0.0, 150.0), (-300.0, 0.0), (-300.0, 150.0), (-20000.0, -19990.0), (85.0, 95.0), (-105.0, -95.0)])
def test_segments_of_different_sizes(low, high, dtype):
    import torch
    V = 30000
    x = torch.randn((2, 3, V), generator=torch.Generator().manual_seed(3))
    x[..., :9000] += low
    x[..., 9000:] += low
    x[:, 0, 20000:20100] += high - low
    x[:, 1, :100] += high - low
    x[:, 2, V - 1] += high - low
    _check(x.to(getattr(torch, dtype)), _scores(2, 3), 12)


def test_nearly_equal_candidates_of_two_beams():
    import torch
    V = 50000
    g = torch.Generator().manual_seed(5)
    row = torch.randn(V, generator=g) * 3
    other = row[torch.randperm(V, generator=g)]                  # the same normaliser, added up in another order
    x = torch.stack([row, other]).view(1, 2, V)
    for step in (8, 20, 300):                                    # 2^-30 each
        s = torch.tensor([[0.01, 0.01 + step * 2.0 ** -30]], dtype=torch.float32)
        assert float(s[0, 1]) > float(s[0, 0])
        _check(x, s, 32)
        _check(x.flip(1), s, 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values_at_the_ends(dtype):
    import torch
    V = 5003
    x = torch.randn((1, 6, V), generator=torch.Generator().manual_seed(6)).to(getattr(torch, dtype))
    x[0, 1, V - 1], x[0, 2, 0], x[0, 3, 2048] = float("nan"), float("inf"), float("nan")
    x[0, 4, :-1] = float("-inf")
    x[0, 3, 2048] *= -1                                          # a NaN of the other sign
    x[0, 5, 100:] = float("-inf")
    _check(x, _scores(1, 6), 64)
