"""The 4-bit token cache at the limits that its documentation states: lengths past the table, queries
whose elements are of very different size."""
import numpy as np
import pytest

from tests.test_gpu_mxfp4 import _dev, _pools, _t, _table

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
