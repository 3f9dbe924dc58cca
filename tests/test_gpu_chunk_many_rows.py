"""Chunk attention's kernel of many query rows, by calls of so many rows of so many KV heads that the rule takes it: lengths, tags,
masked bytes, queries and scales as the other kernel's tests have them; and pages and logits past 2^32 bytes."""
import numpy as np
import pytest

from oracle import chunk_attention as O
from test_gpu_chunk_attention import _t
from test_gpu_chunk_limits import MANY, _case, _check_some, _upload

pytestmark = pytest.mark.gpu


def _many(seed, mix, q_dtype="float16", D=64, **kw):
    return _case(seed, MANY, D, mix, q_dtype, **kw)


@pytest.mark.parametrize("q_dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("mix", ["fp16", "bytes", "all"])
@pytest.mark.parametrize("D", [64, 128])
def test_every_precision(D, mix, q_dtype):
    s = _many(1, mix, q_dtype, D)
    _check_some(s)
    _check_some(s, causal=False)


@pytest.mark.parametrize("q_dtype", ["float16", "float32"])
@pytest.mark.parametrize("mix", ["fp16", "bytes", "all"])
@pytest.mark.parametrize("D", [64, 128])
def test_tiles_of_128_rows(D, mix, q_dtype):
    s = _case(8, (64, 32, 16, 4, 25), D, mix, q_dtype)
    _check_some(s)
    _check_some(s, splits=3)


@pytest.mark.parametrize("mix", ["fp16", "all"])
def test_lengths(mix):
    s = _many(2, mix)
    L, W = MANY[1], MANY[4]
    s.valid[0], s.valid[1], s.valid[2] = [0, 1, -7, 2 ** 31 - 1], [16, 17, 15, L], [L - 1, L + 1, W * 16, W * 16 - 1]
    s.counts[:] = W
    s.counts[2] = [2, -1, 2 ** 31 - 1, 3]
    s.q_lens[:3] = [L, 3, L + 9]
    _check_some(s, some=3)
    _check_some(s, some=3, causal=False)
    s.q_lens[:3] = [0, -2, 1]
    got = _check_some(s, some=3)
    assert not got[:2].any() and not got[2, 1:].any()


@pytest.mark.parametrize("other", [False, True])
def test_tags_and_ids(other):
    s = _many(3, "all")
    s.tags = s.rng.integers(-3, 12, s.NP).astype(np.int32)
    s.table[0, 0, ::2] -= s.NP
    s.table[0, 1, 3], s.table[1, 0, 1], s.table[1, 1] = s.NP, 2 ** 31 - 1, -2 ** 31
    got = s.run(map_other_tags=other, negative_ids=True)
    some = {n: getattr(s, n) for n in ("table", "counts", "valid", "q_lens", "q")}
    for n, x in some.items():
        setattr(s, n, x[:2])
    s.check(got[:2], map_other_tags=other, negative_ids=True)


@pytest.mark.parametrize("mix", ["fp16", "bytes", "all"])
@pytest.mark.parametrize("splits", [1, 2])
def test_unseen_bytes_never_reach(splits, mix):
    s = _many(4, mix)
    seen = np.zeros((s.NP, 16), bool)
    for b, h in np.ndindex(*s.valid.shape):
        for t in range(s.valid[b, h]):
            seen[s.table[b, h, t // 16], t % 16] = True
    bad = ~seen | (O.native(s.tags) == O.SKIP)[:, None]
    for n in ("k_fp16", "v_fp16"):
        x = np.array([np.nan, np.inf, -np.inf], np.float16)[s.rng.integers(0, 3, s.host[n].shape)]
        s.host[n] = np.where(bad[..., None], x, s.host[n])
    for n in ("k_fp8", "v_fp8"):
        if n in s.host:
            s.host[n] = np.where(bad[..., None], np.uint8(0x7F), s.host[n])
    _upload(s)
    assert np.isfinite(_check_some(s, splits=splits).float().cpu().numpy()).all()
    # values that some of the queries see
    for b, value in ((0, np.inf), (1, np.nan)):
        at = max(0, int(s.valid[b, 0]) - 20)
        page = s.table[b, 0, at // 16]
        s.tags[page] = 0
        s.host["v_fp16"][page, at % 16, 13] = value
        s.host["v_fp16"][page, at % 16, 14], s.host["v_fp16"][page, (at % 16) ^ 1, 14] = np.inf, -np.inf
        s.host["k_fp16"][page] = np.nan_to_num(s.host["k_fp16"][page], nan=0, posinf=0, neginf=0)
    _upload(s)
    _check_some(s, splits=splits)


@pytest.mark.parametrize("q_dtype", ["float16", "float32"])
def test_queries_that_are_not_finite(q_dtype):
    s = _many(5, "all", q_dtype, ragged=False)
    s.q[0, 0, 1, 5], s.q[1, 3, 3, 0], s.q[0, 5, 2, 63] = float("nan"), float("inf"), float("-inf")
    s.q[1, 0, 0] = 0
    _check_some(s)
    s.valid[:] = MANY[1] // 2                                    # the first queries see nothing
    got = _check_some(s)
    assert not got[:, :MANY[1] // 2].any()


@pytest.mark.parametrize("value", [-0.02, 0.0, 1e-30, 3e4])
def test_scales(value):
    s = _many(6, "all", D=128)
    for n, x in s.host.items():
        if n.endswith("_scale") and not (n[0] == "k" and value > 1):
            x[s.rng.permutation(s.NP)[:s.NP // 3]] = value
    _upload(s)
    _check_some(s)


@pytest.mark.parametrize("L,mix", [(3, "int4"), (3, "fp16"), (200, "fp16")])
def test_pages_far_into_their_pools(L, mix):
    """Page ids whose bytes and elements are past 2^32 and 2^31."""
    import torch
    import intent_attention as ia
    from test_gpu_chunk_attention import Case
    s = Case(7, 1, L, 4, 2, 128, 13, mix, scale_dtype=np.float32)
    per = 16 * 128 * (2 if mix == "fp16" else 1) // (1 if mix == "fp16" else 2)
    first = 2 ** 32 // per + 3
    pools = {}
    for n, x in s.host.items():
        if mix != "fp16" and "fp16" in n:
            continue
        big = torch.zeros((first + s.NP, *x.shape[1:]), dtype=_t(x).dtype, device="cuda")
        big[first:] = _t(x)
        pools[n] = big
    tags = torch.zeros(first + s.NP, dtype=torch.int32, device="cuda")
    tags[first:] = 0 if mix == "fp16" else 4
    s.tags[:] = 0 if mix == "fp16" else 4
    got = ia.paged_chunk_attention(s.q, ia.PagePools(int4_group=s.group, **pools), _t(s.table + first), _t(s.counts), tags,
                                   valid_tokens=_t(s.valid), q_lens=_t(s.q_lens))
    s.check(got)


def test_tokens_far_into_their_pools():
    import torch
    import intent_attention as ia
    NP, D = 2 ** 20 + 5, 128
    pools = ia.PagePools(k_fp16=torch.zeros(NP, 16, D, dtype=torch.float16, device="cuda"),
                         v_fp16=torch.zeros(NP, 16, D, dtype=torch.float16, device="cuda"))
    k, v = (torch.randn(1, 20, 2, D, device="cuda").half() for _ in range(2))
    table = torch.tensor([[[NP - 1, NP - 2], [NP - 4, NP - 3]]], dtype=torch.int32, device="cuda")
    valid = torch.full((1, 2), 20, dtype=torch.int32, device="cuda")
    ia.append_rotated_tokens(k, v, pools, table, valid, torch.zeros(D // 2, device="cuda"))     # no turn: as they are
    for h in range(2):
        for x, pool in ((k, pools.k_fp16), (v, pools.v_fp16)):
            assert torch.equal(pool[table[0, h].long()].view(32, D)[:20], x[0, :, h])
    assert not pools.k_fp16[:NP - 4].any()


def test_logits_far_into_their_tensor():
    import torch
    import intent_attention as ia
    from oracle import beam_search
    B, K, V = 130, 128, 131101
    x = torch.zeros(B, K, V, dtype=torch.float16, device="cuda")           # 2.2e9 elements
    x[B - 1] = torch.randn(K, V, device="cuda").half()
    s = torch.randn(B, K, device="cuda")
    got = ia.beam_select(x, s, count=16)
    want = beam_search.select(x[B - 1:].double().cpu().numpy(), s[B - 1:].double().cpu().numpy(), 16)
    assert got[1][B - 1].tolist() == ((B - 1) * K + want[1][0]).tolist()
    assert got[2][B - 1].tolist() == want[2][0].tolist()
    flat = beam_search.select(np.zeros((1, K, 3)), s[:1].double().cpu().numpy(), 1)
    assert int(got[1][0, 0]) == int(flat[1][0, 0]) and got[2][0].tolist() == list(range(16))
