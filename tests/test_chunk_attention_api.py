"""The chunk attention's oracle and refusals, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from oracle import chunk_attention as O


def test_oracle_against_a_dense_softmax():
    rng = np.random.default_rng(0)
    pools = {n: rng.standard_normal((9, 16, 64)).astype(np.float16) for n in ("k_fp16", "v_fp16")}
    table, tags = rng.permutation(9)[:6].reshape(1, 2, 3), np.zeros(9, int)
    q = rng.standard_normal((1, 4, 4, 64))
    out, mass, reach = O.attention(q, pools, tags, table, np.full((1, 2), 3), np.full((1, 2), 41))
    for h in range(4):
        k, v = (pools[n][table[0, h // 2]].reshape(-1, 64)[:41].astype(float) for n in ("k_fp16", "v_fp16"))
        for i in range(4):
            s = k[:38 + i] @ q[0, i, h] / 8
            p = np.exp(s - s.max())
            assert np.allclose(out[0, i, h], p @ v[:38 + i] / p.sum())
    assert (mass >= np.abs(out) - 1e-12).all() and (reach > 0).all()


def test_oracle_precisions():
    c = np.array([[0x00, 0x38, 0xB8, 0x7E, 0x01, 0x7F]], np.uint8)
    assert np.array_equal(O.fp8_values(c), [[0, 1, -1, 448, 2.0 ** -9, np.nan]], equal_nan=True)
    pools = {"k_int4": np.full((1, 16, 32), 0xF1, np.uint8), "k_int4_scale": np.array([[1.0, 2.0, 4.0, 8.0]]),
             "k_int4r": np.full((1, 16, 64), 0x2B, np.uint8), "k_int4r_scale": np.array([[1.0, 0.25]])}
    assert O.page_values(pools, "k", 0, O.INT4)[3, [0, 1, 16, 63]].tolist() == [-7, 7, -14, 56]
    assert O.page_values(pools, "k", 0, O.INT4_RESIDUAL)[0, 0] == 3 - 6 * 0.25
    assert O.native([0, 5, 9, -1, 7], [3, 1], True).tolist() == [3, 2, 2, 2, 2]


def _args(**kw):
    a = N.PagedChunkArgs(batch=2, q_len=3, num_q_heads=8, num_kv_heads=2, head_dim=64, page_size=16, table_width=9, num_pages=50, q=4096,
                         out=8192, page_table=4096, page_counts=4096, page_tags=4096, k_fp16=4096, v_fp16=4096, sm_scale=0.1, causal=1,
                         int4_group=16)
    a.tag_map[:] = [0, 2, 2, 2, 2, 2, 2, 2]
    for n, v in kw.items():
        if n == "tag_map":
            a.tag_map[:] = v
        else:
            setattr(a, n, v)
    return a


def _tag(t):
    return [t] + [2] * 7


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "size"), (dict(q_len=-1), "size"), (dict(num_kv_heads=0), "size"), (dict(table_width=-1), "size"), (dict(num_pages=-1), "size"),
    (dict(head_dim=96), "head_dim"), (dict(page_size=32), "page_size"), (dict(num_pages=1 << 31), "int32"), (dict(table_width=1 << 27), "int32"),
    (dict(num_q_heads=7), "multiple"), (dict(num_q_heads=0), "multiple"), (dict(q_dtype=3), "dtype"), (dict(out_dtype=-1), "dtype"),
    (dict(sm_scale=float("nan")), "sm_scale"), (dict(sm_scale=3e38), "sm_scale"), (dict(causal=2), "causal"), (dict(splits=-1), "splits"),
    (dict(q=None), "q/out"), (dict(out=None), "q/out"), (dict(q=4097), "aligned"), (dict(out_dtype=1, out=4098), "aligned"),
    (dict(page_table=None), "page_table"), (dict(page_counts=None), "page_counts"), (dict(page_tags=None), "page_tags"),
    (dict(valid_tokens=4098), "aligned"), (dict(q_lens=4097), "aligned"), (dict(k_fp16=None), "pool"), (dict(v_fp16=4104), "16-byte"),
    (dict(tag_map=_tag(1)), "pool"), (dict(tag_map=_tag(1), k_int8=4096, v_int8=4096), "scales"),
    (dict(tag_map=_tag(3), k_fp8=4096, v_fp8=4096, k_fp8_scale=4096, v_fp8_scale=4096, fp8_scale_dtype=2), "scale dtype"),
    (dict(tag_map=_tag(3), k_fp8=4096, v_fp8=4096, k_fp8_scale=4098, v_fp8_scale=4096, fp8_scale_dtype=1), "aligned"),
    (dict(tag_map=_tag(4), k_int4=4096, v_int4=4096, k_int4_scale=4096, v_int4_scale=4096, int4_group=8), "int4_group"),
    (dict(tag_map=_tag(4), k_int4=4096, v_int4=4096, k_int4_scale=4096, v_int4_scale=4096, int4_group=0), "int4_group"),
    (dict(q_len=1 << 29), "too long"), (dict(q_len=1 << 27), "too many"), (dict(batch=1 << 24), "too many")])
def test_abi_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        N.paged_chunk_workspace(_args(**kw))
    with pytest.raises(ValueError, match=text):
        N.paged_chunk(_args(**kw), 0, 1 << 20, 1 << 40)


def test_abi_workspace():
    a = _args(splits=3)
    need = N.paged_chunk_workspace(a)
    assert need > 0
    for at, size in ((None, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            N.paged_chunk(a, 0, at, size)
    for kw in (dict(batch=0), dict(q_len=0), dict(splits=1), dict(table_width=0)):
        assert N.paged_chunk_workspace(_args(**kw)) == 0
    N.paged_chunk(_args(batch=0), 0)
    N.paged_chunk(_args(q_len=0), 0)
    with pytest.raises(ValueError, match="NULL"):
        N.check(N.load().iak_paged_chunk(None, None, 0, None))
    with pytest.raises(ValueError, match="NULL"):
        N.check(N.load().iak_paged_chunk_workspace(ctypes.byref(a), None))


def test_python_refuses():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    pools = ia.PagePools(k_fp16=torch.zeros(9, 16, 64).half(), v_fp16=torch.zeros(9, 16, 64).half())
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        ia.paged_chunk_attention(torch.zeros(2, 3, 4, 64), pools, i(2, 2, 4), i(2, 2), i(9))
