"""The rotated append's oracle and refusals, without a GPU."""
import numpy as np
import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from oracle import rotary as O


def test_oracle_turns_pairs():
    x = np.zeros((1, 1, 1, 64))
    x[..., 0], x[..., 16], x[..., 1], x[..., 40] = 1.0, 2.0, 3.0, 5.0
    f = np.zeros(16)
    f[0] = np.pi / 4
    one = np.ones((1, 1, 1), np.int64)
    y = O.rotate(x, 2 * one, f, False)[0, 0, 0]                  # a quarter turn
    assert np.allclose(y[[0, 16, 1, 40]], [-2, 1, 3, 5])
    y = O.rotate(x, 2 * one, f, True)[0, 0, 0]
    assert np.allclose(y[[0, 1, 16, 40]], [-3, 1, 2, 5])
    assert np.allclose(O.reach(x, f, False)[0, 0, 0, [0, 16, 40]], [3, 3, 10])


def test_oracle_places():
    table = np.array([[[5, 3], [9, 1]]])
    page, number = O.places(table, np.array([[20, 2]]), np.array([3]), 4, 8)
    assert page[0].T.tolist() == [[3, 3, 3, -1], [-1, -1, -1, -1]] and number[0].T.tolist() == [[17, 18, 19, 20], [-1, 0, 1, 2]]


def _args(**kw):
    a = N.RotaryAppendArgs(batch=2, count=3, num_q_heads=8, num_kv_heads=2, head_dim=64, rotary_dim=32, page_size=16, table_width=9,
                           num_pages=50, dtype=0, q=1 << 12, q_out=2 << 12, k=3 << 12, v=4 << 12, inv_freq=5 << 12, page_table=6 << 12,
                           valid_tokens=7 << 12, k_pages=8 << 12, v_pages=9 << 12)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


PACKED = dict(k_pages=None, v_pages=None, k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "size"), (dict(count=-1), "size"), (dict(num_kv_heads=0), "size"), (dict(num_q_heads=-1), "size"),
    (dict(table_width=-1), "size"), (dict(num_pages=-1), "size"), (dict(head_dim=96), "head_dim"), (dict(page_size=8), "page_size"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=80), "rotary_dim"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=-16), "rotary_dim"),
    (dict(interleaved=2), "interleaved"), (dict(num_pages=1 << 31), "int32"), (dict(table_width=1 << 27), "int32"), (dict(dtype=3), "dtype"),
    (dict(num_q_heads=7), "multiple"), (dict(num_q_heads=0), "multiple"), (dict(count=1 << 28), "too many"), (dict(batch=1 << 20, count=1 << 16), "too many"),
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(q=None), "go together"), (dict(q_out=None), "go together"), (dict(inv_freq=None), "inv_freq"),
    (dict(page_table=None), "page_table"), (dict(valid_tokens=None), "valid_tokens"), (dict(k_pages=None), "pages"), (dict(v_pages=None), "pages"),
    (dict(k=4097), "aligned"), (dict(dtype=1, q=4098), "aligned"), (dict(positions=4098), "aligned"), (dict(page_tags=4098), "aligned"),
    (dict(v_pages=4097), "aligned"), (dict(k_codes=4096), "both"), (dict(PACKED, v_scales=None), "NULL"), (dict(PACKED, page_tags=4096), "page_tags"),
    (dict(PACKED, k_codes=4098), "aligned")])
def test_abi_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        N.rotary_append(_args(**kw), 0)


def test_abi_nothing_to_do():
    for kw in (dict(batch=0), dict(count=0), dict(count=0, **PACKED)):
        N.rotary_append(_args(**kw), 0)
    with pytest.raises(ValueError, match="NULL"):
        N.check(N.load().iak_rotary_append(None, None))


def test_python_refuses():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pools = ia.PagePools(k_fp16=torch.zeros(9, 16, 64).half(), v_fp16=torch.zeros(9, 16, 64).half())
    k, f = torch.zeros(2, 3, 2, 64), torch.zeros(16)
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        ia.append_rotated_tokens(k, k, pools, i(2, 2, 4), i(2, 2), f)
    with pytest.raises(ValueError, match="one shape"):
        ia.append_rotated_tokens(k, k[:1], pools, i(2, 2, 4), i(2, 2), f)
    with pytest.raises(ValueError, match="float16, bfloat16"):
        ia.append_rotated_tokens(k, k.half(), pools, i(2, 2, 4), i(2, 2), f)
    with pytest.raises(ValueError, match="without float16"):
        ia.append_rotated_tokens(k, k, ia.PagePools(), i(2, 2, 4), i(2, 2), f)
