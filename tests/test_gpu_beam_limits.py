"""The beam choice where its lists fill with equal logits."""
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
