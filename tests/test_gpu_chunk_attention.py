"""Attention of several query tokens over pages of mixed precision on the GPU against float64, within bounds
worked out per output: every precision, length and kernel; masks, special values, scales, layouts, graphs, streams."""
import numpy as np
import pytest

from oracle import chunk_attention as O

pytestmark = pytest.mark.gpu

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}   # a rounding's largest relative error
MIX = {"fp16": [0], "int8": [0, 1], "fp8": [0, 3], "int4": [4], "int4r": [5], "all": [0, 1, 2, 3, 4, 5], "bytes": [0, 1, 2, 3]}


def _t(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(getattr(torch, dtype))


def host_pools(rng, NP, D, tags, scale_dtype=np.float16, group=32, magnitude=1.0):
    """Random pages of every precision among `tags` (float16 always)."""
    pools = {}
    for side in "kv":
        pools[side + "_fp16"] = (rng.standard_normal((NP, 16, D)) * magnitude).astype(np.float16)
        if 1 in tags:
            pools[side + "_int8"] = rng.integers(-128, 128, (NP, 16, D)).astype(np.int8)
            pools[side + "_int8_scale"] = (magnitude * rng.uniform(0.005, 0.03, NP)).astype(scale_dtype)
        if 3 in tags:
            c = rng.integers(0, 256, (NP, 16, D)).astype(np.uint8)
            c = np.where((c & 127) == 127, 0x33, np.where((c & 0x78) > 0x48, c & 0xCF, c))          # moderate sizes
            pools[side + "_fp8"] = c.astype(np.uint8)
            pools[side + "_fp8_scale"] = (magnitude * rng.uniform(0.1, 0.5, NP)).astype(scale_dtype)
        if 4 in tags:
            pools[side + "_int4"] = rng.integers(0, 256, (NP, 16, D // 2)).astype(np.uint8)
            pools[side + "_int4_scale"] = (magnitude * rng.uniform(0.05, 0.5, (NP, D // group))).astype(scale_dtype)
        if 5 in tags:
            pools[side + "_int4r"] = rng.integers(0, 256, (NP, 16, D)).astype(np.uint8)
            s = magnitude * rng.uniform(0.05, 0.5, (NP, 1))
            pools[side + "_int4r_scale"] = np.concatenate([s, s * rng.uniform(0.05, 0.08, (NP, 1))], 1).astype(np.float32)
    return pools


class Case:
    def __init__(self, seed, B, L, Hq, Hkv, D, W, mix, q_dtype="float16", ragged=True, scale_dtype=np.float16, group=None, magnitude=1.0):
        import intent_attention as ia
        rng = np.random.default_rng(seed)
        self.rng, self.q_dtype = rng, q_dtype
        group = group or (32 if D == 128 else 16)
        kinds = MIX[mix]
        self.NP = NP = B * Hkv * W + 7
        self.tags = rng.choice(kinds, NP).astype(np.int32)
        self.host = host_pools(rng, NP, D, kinds, scale_dtype, group, magnitude)
        self.table = rng.permutation(NP)[:B * Hkv * W].reshape(B, Hkv, W).astype(np.int32)
        self.valid = rng.integers(max(1, W * 8), W * 16 + 1, (B, Hkv)).astype(np.int32) if ragged else np.full((B, Hkv), W * 16, np.int32)
        self.counts = -(-self.valid // 16).astype(np.int32)
        self.q_lens = rng.integers(0, L + 1, B).astype(np.int32) if ragged else None
        self.q = _t(rng.standard_normal((B, L, Hq, D)) * 2, q_dtype)
        self.group = group
        self.pools = ia.PagePools(int4_group=group, **{n: _t(x) for n, x in self.host.items()})

    def args(self, **kw):
        o = lambda x: None if x is None else _t(x)  # noqa: E731
        return (self.q, self.pools, _t(self.table), _t(self.counts), _t(self.tags)), dict(valid_tokens=o(self.valid), q_lens=o(self.q_lens), **kw)

    def run(self, **kw):
        import intent_attention as ia
        a, k = self.args(**kw)
        return ia.paged_chunk_attention(*a, **k)

    def check(self, got=None, causal=True, tag_map=None, map_other_tags=False, negative_ids=False, sm_scale=None, out_dtype=None, q=None, **kw):
        import torch
        if got is None:
            got = self.run(causal=causal, tag_map=tag_map, map_other_tags=map_other_tags, negative_ids=negative_ids, sm_scale=sm_scale,
                           out_dtype=None if out_dtype is None else getattr(torch, out_dtype), **kw)
        q = (self.q if q is None else q).double().cpu().numpy()
        q4 = q if q.ndim == 4 else q[:, None]
        native = O.native(self.tags, tag_map, map_other_tags)
        want, mass, reach = O.attention(q4, self.host, native, self.table, self.counts, self.valid, self.q_lens, causal, sm_scale, negative_ids)
        g = got.double().cpu().numpy().reshape(want.shape)
        # past the output type's range: infinite; next to its end, within the weights' rounding, as it came out
        most, size = torch.finfo(got.dtype).max, np.abs(np.where(np.isfinite(want), want, 0))
        want = np.where((size > most * (1 + 2.0 ** -8)) | ((size > most * (1 - 2.0 ** -8)) & np.isinf(g)), np.copysign(np.inf, want), want)
        for kind in (np.isnan, np.isposinf, np.isneginf):
            assert np.array_equal(kind(g), kind(want)), kind.__name__
        fine = np.isfinite(want)
        T, D = self.table.shape[2] * 16, q.shape[-1]
        f32 = self.q_dtype == "float32"
        scales = [np.abs(x[np.isfinite(x)]).max(initial=0.0) for n, x in self.host.items() if n.startswith("v_") and n.endswith("_scale")]
        # Scores: D products summed in float32, the query's split where it is float32 (2^-22), a 4-bit key's two parts (2^-21),
        # the multipliers: of the largest sum |q| |k|; twice for a weight over the sum.
        score = ((D + 8) * 2.0 ** -24 + (2.0 ** -22 if f32 else 2.0 ** -38) + 2.0 ** -21) * reach[..., None]
        # Weights: their rounding (float16 2^-11, split 2^-22), the exponential 2^-22, the roundings of its argument, of which there
        # are three of the sum of a score, the maximum and log2 of a scale (below 30); the sums; a 4-bit value's parts.
        weight = (2.0 ** -22 if f32 else 2.0 ** -11) + 2.0 ** -22 + 3 * 2.0 ** -24 * (2 * 1.45 * reach[..., None] + 36) + 2.0 ** -21
        rel = 2 * np.expm1(2 * score) + weight + 2 * (T + 8) * 2.0 ** -24
        # weights below float16's range: half its smallest step of the 2^6 that the largest weighs, times codes up to 512
        tiny = T * 2.0 ** -31 * 512 * max([1.0] + scales)
        out_dtype = str(got.dtype).split(".")[1]
        tol = rel * mass + tiny + HALF[out_dtype] * np.abs(np.where(fine, want, 0)) + 2.0 ** -25
        worst = float((np.abs(np.where(fine, g, 0) - np.where(fine, want, 0)) / tol).max(initial=0.0))
        assert worst <= 1.0, worst
        return got


ROWS = [(1, 1, 1, 1, 64, 1), (2, 3, 8, 8, 64, 9), (3, 4, 8, 2, 128, 21), (2, 1, 28, 4, 128, 33), (1, 8, 24, 1, 64, 70), (2, 5, 12, 6, 128, 130)]
CHUNKS = [(1, 70, 4, 4, 128, 9), (2, 33, 8, 2, 64, 12), (1, 130, 4, 2, 128, 21), (3, 100, 12, 4, 64, 15), (1, 40, 14, 2, 128, 70)]


@pytest.mark.parametrize("q_dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("mix", ["fp16", "int8", "fp8", "int4", "int4r", "bytes", "all"])
@pytest.mark.parametrize("shape", ROWS + CHUNKS)
def test_every_precision(shape, mix, q_dtype):
    s = Case(sum(shape) + len(mix), *shape, mix, q_dtype, scale_dtype=np.float32 if shape[1] % 2 else np.float16)
    s.check()


@pytest.mark.parametrize("mix", ["fp16", "bytes", "all"])
@pytest.mark.parametrize("shape", [(2, 4, 8, 2, 128, 40), (2, 50, 8, 2, 64, 40)])
def test_splits(shape, mix):
    for splits in (1, 2, 3, 7, 20, 10 ** 6):
        s = Case(splits, *shape, mix)
        s.check(splits=splits)
        s.check(splits=splits, causal=False)


@pytest.mark.parametrize("L", [1, 6, 60])
@pytest.mark.parametrize("mix", ["fp16", "all"])
def test_lengths(mix, L):
    """Rows that hold nothing, less than their queries, more than their table; counts that cut the lengths."""
    s = Case(L, 7, L, 6, 2, 64, 5, mix, "bfloat16")
    s.valid = np.array([[0, 80], [-5, 1], [2000000000, 16], [17, 33], [L, L - 1], [3, 79], [80, 80]], np.int32)
    s.counts = np.array([[5, 5], [1, 1], [9, 1], [2, 2], [5, 5], [0, -3], [4, 2000000000]], np.int32)
    s.q_lens = np.array([L, L, 1, L, L, L, L + 50], np.int32)
    s.check()
    s.check(causal=False)
    s.q_lens = np.array([0, -4, 0, 0, 1, 1, 0], np.int32)
    s.check()
    s.valid = s.q_lens = None
    s.check()


@pytest.mark.parametrize("L", [2, 80])
def test_tags_and_ids(L):
    s = Case(L, 2, L, 4, 2, 64, 9, "all")
    s.tags = s.rng.integers(-3, 12, s.NP).astype(np.int32)
    for other in (False, True):
        s.check(map_other_tags=other)
        s.check(tag_map=[0, 1, 2, 2, 2, 2, 2, 1], map_other_tags=other)
        s.check(tag_map=[5, 4, 3], map_other_tags=other)
    s.table[0, 0, ::2] -= s.NP
    s.table[0, 1, 3], s.table[1, 0, 1], s.table[1, 1] = s.NP, 2 ** 31 - 1, -2 ** 31
    s.check()
    s.check(negative_ids=True)


@pytest.mark.parametrize("L", [3, 50])
def test_pages_that_are_skipped(L):
    s = Case(5, 2, L, 4, 2, 128, 11, "all", "float32")
    s.tags[:] = np.where(np.arange(s.NP) % 3, 2, s.tags)
    s.check()
    s.tags[:] = 2
    assert not s.check().any()


@pytest.mark.parametrize("L,mix", [(1, "fp16"), (4, "fp16"), (4, "all"), (70, "fp16"), (70, "bytes"), (70, "all")])
def test_unseen_bytes_never_reach(L, mix):
    """NaN and infinities past the lengths, in skipped and in other sequences' pages, and in tokens that some queries see."""
    s = Case(6, 2, L, 4, 2, 64, 8, mix)
    seen = np.zeros((s.NP, 16), bool)
    for b, h in np.ndindex(*s.valid.shape):
        for t in range(s.valid[b, h]):
            seen[s.table[b, h, t // 16], t % 16] = True
    bad = ~seen | (O.native(s.tags) == O.SKIP)[:, None]
    for n in ("k_fp16", "v_fp16"):
        x = np.array([np.nan, np.inf, -np.inf], np.float16)[s.rng.integers(0, 3, s.host[n].shape)]
        s.host[n] = np.where(bad[..., None], x, s.host[n])
        setattr(s.pools, n, _t(s.host[n]))
    if "v_fp8" in s.host:
        for n in ("k_fp8", "v_fp8"):
            s.host[n] = np.where(bad[..., None], np.uint8(0x7F), s.host[n])
            setattr(s.pools, n, _t(s.host[n]))
    assert np.isfinite(s.check().float().cpu().numpy()).all()
    s.check(causal=False)
    # a row's last token, and one in the middle, are special: of the queries those that see them
    for n, t in (("v_fp16", 1), ("v_fp16", max(2, L // 2)), ("k_fp16", 1)):
        s = Case(7, 2, L, 4, 2, 64, 8, mix, ragged=False)
        s.valid = np.full((2, 2), 8 * 16 - 5, np.int32)
        for b, value in ((0, np.inf), (1, np.nan)):
            at = int(s.valid[b, 0]) - t
            if at >= 0:
                page = s.table[b, 0, at // 16]
                s.tags[page] = 0
                s.host[n][page, at % 16, 13] = value
                if n[0] == "v":
                    s.host[n][page, at % 16, 14], s.host[n][page, (at - 1) % 16, 14] = np.inf, -np.inf
        setattr(s.pools, n, _t(s.host[n]))
        s.check()                                                # an infinite key: scores of +-inf, and what they make NaN


@pytest.mark.parametrize("L", [4, 60])
def test_scales(L):
    """Negative, zero, subnormal, huge, infinite and NaN scales, by pages; neighbours far apart."""
    for seed, value in enumerate((-0.02, 0.0, 1e-30, 3e4)):
        s = Case(seed, 2, L, 4, 2, 128, 9, "all", "float16", scale_dtype=np.float32)
        for n, x in s.host.items():
            if n.endswith("_scale"):
                rows = s.rng.permutation(s.NP)[:s.NP // 3]
                if n[0] == "k" and value > 1:
                    continue
                x[rows] = value
                setattr(s.pools, n, _t(x))
        s.check()
    s = Case(9, 2, L, 4, 2, 128, 9, "bytes", "float16", scale_dtype=np.float32)
    page = s.table[0, 0, 0]
    for value in (np.nan, np.inf):
        for n in ("v_int8_scale", "v_fp8_scale"):
            s.host[n][page] = value
            setattr(s.pools, n, _t(s.host[n]))
        for tag in (1, 3):
            s.tags[page] = tag
            s.host["v_int8"][page] = np.where(s.host["v_int8"][page] == 0, 1, s.host["v_int8"][page])
            s.host["v_fp8"][page] = np.where((s.host["v_fp8"][page] & 127) == 0, 0x30, s.host["v_fp8"][page])
            s.pools.v_int8, s.pools.v_fp8 = _t(s.host["v_int8"]), _t(s.host["v_fp8"])
            s.check()


@pytest.mark.parametrize("D,groups", [(64, (16, 32, 64)), (128, (32, 64, 128))])
@pytest.mark.parametrize("L", [2, 40])
def test_int4_groups(D, groups, L):
    for group in groups:
        Case(group, 2, L, 4, 2, D, 9, "int4", "float32", group=group, scale_dtype=np.float32).check()


@pytest.mark.parametrize("magnitude", [1e-4, 30.0, 3000.0])
@pytest.mark.parametrize("L", [2, 40])
def test_magnitudes(L, magnitude):
    s = Case(3, 2, L, 4, 2, 64, 9, "all", "float32", scale_dtype=np.float32, magnitude=magnitude)
    s.check(sm_scale=0.1 / magnitude ** 2)
    s.check(sm_scale=-0.1 / magnitude ** 2)
    s.check(sm_scale=0.0)


@pytest.mark.parametrize("L", [2, 40])
def test_queries_that_are_not_finite(L):
    import torch
    for dtype in ("float16", "float32"):
        s = Case(4, 2, L, 4, 2, 64, 6, "all", dtype, ragged=False)
        s.q[0, 0, 1, 5], s.q[1, L - 1, 3, 0] = float("nan"), float("inf")
        s.q[1, 0, 0] = 0
        s.check()
        s.valid = np.full((2, 2), L // 2, np.int32)              # the first queries see nothing
        got = s.check()
        assert not got[:, :(L + 1) // 2].any() and torch.isnan(got).any()


def test_layouts_and_dtypes():
    import torch
    for L in (4, 50):
        s = Case(8, 2, L, 6, 2, 64, 7, "all")
        flat = torch.zeros(2, L + 2, 9 * 64 + 5, dtype=torch.float16, device="cuda")
        view = flat[:, 1:L + 1, 3:3 + 6 * 64].unflatten(-1, (6, 64))
        s.q = view.copy_(s.q)
        base = torch.full((2, L + 1, 8, 67), 9.0, device="cuda")
        out = base[:, 1:, 1:7, 2:66]
        s.check(s.run(out=out))
        out.fill_(9)
        assert bool((base == 9).all())
        for dtype in ("float16", "bfloat16", "float32"):
            s.check(out_dtype=dtype)
        before = s.q.clone()
        assert s.run(out=s.q) is s.q                             # in the query's place
        s.check(s.q, q=before)
        s.q = before.transpose(1, 3).contiguous().transpose(1, 3)
        s.check()
        s.q = before[:, :1].expand(2, L, 6, 64)                  # one query for all
        s.check()


def test_one_token_is_the_decode():
    import torch
    import intent_attention as ia
    s = Case(9, 3, 1, 8, 2, 128, 20, "all", "float16", ragged=True)
    s.q_lens = None
    s.q = s.q[:, 0]
    (q, pools, table, counts, tags), kw = s.args()
    got = ia.paged_chunk_attention(q, pools, table, counts, tags, **kw)
    assert got.shape == q.shape
    s.check(got)
    other = ia.paged_decode(q, pools, table, counts, tags, valid_tokens=kw["valid_tokens"])
    # the decode rounds 4-bit keys to 11 bits
    assert torch.allclose(got.float(), other.float(), atol=2e-2)


def test_long_rows_and_many():
    Case(10, 1, 4, 4, 1, 64, 3000, "fp16", "float32", ragged=False).check()
    Case(11, 300, 2, 2, 2, 64, 2, "all").check()
    Case(12, 1, 600, 2, 2, 64, 41, "all", ragged=False).check()


def test_plan_graph_and_streams():
    import torch
    import intent_attention as ia
    for L in (4, 70):
        s = Case(13, 2, L, 8, 2, 128, 30, "all")
        (q, pools, table, counts, tags), kw = s.args()
        plan = ia.make_chunk_plan(q, pools, table, counts, tags, splits=3, **kw)
        plan.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run()
        for it in range(3):
            rng = np.random.default_rng(it)
            s.q_lens = rng.integers(0, L + 1, 2).astype(np.int32)
            s.valid = rng.integers(1, 30 * 16 + 1, (2, 2)).astype(np.int32)
            kw["q_lens"].copy_(_t(s.q_lens)), kw["valid_tokens"].copy_(_t(s.valid))
            s.counts = np.full((2, 2), 30, np.int32)
            counts.copy_(_t(s.counts))
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(it)))
            graph.replay()
            torch.cuda.synchronize()
            s.check(plan.out)
            first = plan.out.clone()
            plan.run()
            torch.cuda.synchronize()
            assert torch.equal(first, plan.out)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ia.paged_chunk_attention(q, pools, table, counts, tags, **kw)
        side.synchronize()
        s.check(got)


def test_nothing_to_do():
    import torch
    import intent_attention as ia
    s = Case(14, 2, 3, 4, 2, 64, 3, "fp16")
    (q, pools, table, counts, tags), kw = s.args()
    for x in (q[:0], q[:, :0]):
        kw2 = dict(valid_tokens=kw["valid_tokens"][:x.shape[0]], q_lens=kw["q_lens"][:x.shape[0]])
        assert ia.paged_chunk_attention(x, pools, table[:x.shape[0]], counts[:x.shape[0]], tags, **kw2).shape == x.shape
    got = ia.paged_chunk_attention(q, pools, table[:, :, :0], counts, tags, **kw)
    assert not got.any()
    none = ia.PagePools(k_fp16=torch.zeros(0, 16, 64).half().cuda(), v_fp16=torch.zeros(0, 16, 64).half().cuda())
    assert not ia.paged_chunk_attention(q, none, table, counts, tags[:0], **kw).any()
