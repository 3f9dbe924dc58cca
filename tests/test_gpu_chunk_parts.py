"""Attention over pages of mixed precision whose rows are long enough to be divided by the library's own rule: alike, and by the
rows' lengths; among them rows without tokens, of one token, and sequences without queries."""
import numpy as np
import pytest

from test_gpu_chunk_attention import MIX, Case, _t, host_pools

pytestmark = pytest.mark.gpu


def long_case(seed, B, L, Hq, Hkv, D, W, mix, q_dtype="float16", NP=211):
    """Many more table entries than pages."""
    import intent_attention as ia
    s = Case.__new__(Case)
    rng = np.random.default_rng(seed)
    s.rng, s.q_dtype, s.NP, s.group = rng, q_dtype, NP, 32
    s.tags = rng.choice(MIX[mix], NP).astype(np.int32)
    s.host = host_pools(rng, NP, D, MIX[mix], group=32)
    s.table = rng.integers(0, NP, (B, Hkv, W)).astype(np.int32)
    s.valid = rng.integers(0, W * 16 + 1, (B, Hkv)).astype(np.int32)
    s.valid[0], s.valid[1], s.valid[2] = 0, 1, W * 16
    s.counts = -(-s.valid // 16).astype(np.int32)
    s.q_lens = rng.integers(1, L + 1, B).astype(np.int32)
    s.q_lens[B - 1] = 0
    s.q = _t(rng.standard_normal((B, L, Hq, D)) * 2, q_dtype)
    s.pools = ia.PagePools(int4_group=32, **{n: _t(x) for n, x in s.host.items()})
    return s


@pytest.mark.parametrize("shape,q_dtype", [
    ((12, 1, 16, 4, 128, 1600), "float16"), ((12, 2, 8, 4, 64, 2300), "float32"), ((12, 9, 16, 4, 64, 2300), "bfloat16"),
    ((4, 200, 8, 2, 64, 700), "bfloat16"), ((4, 200, 8, 2, 128, 500), "float16"), ((5, 90, 4, 2, 64, 700), "float32")])
@pytest.mark.parametrize("mix", ["fp16", "all"])
def test_shared_out_by_lengths(shape, q_dtype, mix):
    import torch
    import intent_attention as ia
    s = long_case(sum(shape), *shape, mix, q_dtype)
    (q, pools, table, counts, tags), kw = s.args()
    plan = ia.make_chunk_plan(q, pools, table, counts, tags, **kw)
    assert plan.workspace_bytes > 0
    plan.run()
    torch.cuda.synchronize()
    s.check(plan.out)
    # other lengths, the same plan: nothing of the former parts is left
    s.valid = np.roll(s.valid, 1, 0)
    s.q_lens = np.roll(s.q_lens, 2)
    s.counts = -(-s.valid // 16).astype(np.int32)
    for t, x in ((kw["valid_tokens"], s.valid), (kw["q_lens"], s.q_lens), (counts, s.counts)):
        t.copy_(_t(x))
    plan.run()
    torch.cuda.synchronize()
    s.check(plan.out)


@pytest.mark.parametrize("shape", [(3, 1, 4, 1, 128, 900), (3, 6, 8, 2, 64, 1100), (3, 70, 8, 2, 128, 500)])
@pytest.mark.parametrize("mix", ["bytes", "all"])
def test_split_alike(shape, mix):
    long_case(sum(shape), *shape, mix).check()


def test_empty_table_of_long_rows():
    s = long_case(3, 12, 1, 16, 4, 128, 1600, "all")
    s.counts[:] = 0
    s.check()


@pytest.mark.parametrize("shape,q_dtype", [((12, 1, 16, 4, 128, 1600), "float16"), ((4, 200, 8, 2, 64, 700), "bfloat16"), ((3, 70, 8, 2, 128, 500), "float32")])
@pytest.mark.parametrize("mix", ["fp16", "all"])
def test_infinite_values_in_parts(shape, q_dtype, mix):
    """Infinities and NaN of V in pages that few rows list, some past their lengths: parts with and without them are merged."""
    s = long_case(sum(shape) + 1, *shape, mix, q_dtype, NP=400)
    B, L, Hq, Hkv, D, W = shape
    s.table %= 390                                               # the last ten pages: listed by hand
    s.tags[390:] = [0, 0, 0, 0] + [0 if mix == "fp16" else t for t in (1, 3, 4, 5, 1, 0)]
    s.host["v_fp16"][390, 3, 5], s.host["v_fp16"][391, 15, 0], s.host["v_fp16"][392, 0, D - 1] = np.inf, -np.inf, np.nan
    s.host["v_fp16"][393] = np.inf
    if mix == "all":
        s.host["v_int8_scale"][394], s.host["v_fp8_scale"][395] = np.inf, np.nan
        s.host["v_int4_scale"][396, 0], s.host["v_int4r_scale"][397, 1] = -np.inf, np.nan
    s.valid[:] = np.maximum(s.valid, 200)
    s.counts = -(-s.valid // 16).astype(np.int32)
    for n, page in enumerate(range(390, 398)):
        b, h = n % B, (n // B) % Hkv
        entry = int(s.valid[b, h]) // 16 * (n + 1) // 9
        s.table[b, h, entry] = page
        s.table[(b + 1) % B, h, W - 1] = page                    # past most lengths
    import intent_attention as ia
    s.pools = ia.PagePools(int4_group=32, **{n: _t(x) for n, x in s.host.items()})
    s.check()
