"""Tokens rotated and written into float16 and 4-bit pages on the GPU against float64: values within the
roundings of float32 arithmetic, 4-bit codes exactly; places, padding, far positions, layouts, graphs."""
import numpy as np
import pytest

from oracle import mxfp4 as MX
from oracle import rotary as O

pytestmark = pytest.mark.gpu

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}   # a rounding's largest relative error
TINY = {"float16": 2.0 ** -25, "bfloat16": 0.0, "float32": 0.0}               # and half the smallest step


def _t(x, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t if dtype is None else t.to(getattr(torch, dtype))


class Case:
    def __init__(self, seed, B, L, Hq, Hkv, D, R, dtype, packed, start=40, ragged=True, W=None, far=None):
        import torch
        import intent_attention as ia
        rng = np.random.default_rng(seed)
        self.D, self.L, self.packed, self.dtype = D, L, packed, dtype
        r = lambda *s: _t(rng.standard_normal(s) * np.exp(rng.standard_normal(s[-1]) * 0.5), dtype)  # noqa: E731
        self.q, self.k, self.v = r(B, L, Hq, D), r(B, L, Hkv, D), r(B, L, Hkv, D)
        self.q_lens = rng.integers(0, L + 1, B).astype(np.int32) if ragged else None
        new = np.full(B, L) if self.q_lens is None else self.q_lens
        self.valid = (new[:, None] + rng.integers(0, start + 1, (B, 1)) + np.zeros((1, Hkv), int)).astype(np.int32)
        W = W or int(-(-(L + start) // 16))
        self.NP = NP = B * Hkv * W + 5
        self.table = rng.permutation(NP)[:B * Hkv * W].reshape(B, Hkv, W).astype(np.int32)
        self.freq = (10000.0 ** (-np.arange(R // 2) / (R // 2))).astype(np.float32)
        self.positions = None if far is None else rng.integers(0, far, (B, L)).astype(np.int32)
        if packed:
            self.pools = ia.MxFp4Pools.empty(NP, D, "cuda")
            for t in self.pools.tensors().values():
                t.fill_(0x55)
        else:
            fill = torch.full((NP, 16, D), 0.25, dtype=torch.float16, device="cuda")
            self.pools = ia.PagePools(k_fp16=fill.clone(), v_fp16=fill)

    def run(self, interleaved, **kw):
        import intent_attention as ia
        o = lambda x: None if x is None else _t(x)  # noqa: E731
        args = dict(q=self.q, q_lens=o(self.q_lens), positions=o(self.positions), interleaved=interleaved)
        return ia.append_rotated_tokens(self.k, self.v, self.pools, _t(self.table), _t(self.valid), _t(self.freq), **{**args, **kw})

    def check(self, got, interleaved, q=None):
        f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
        q, k, v = f64(self.q if q is None else q), f64(self.k), f64(self.v)
        B, L, Hkv, D = k.shape
        G = q.shape[2] // Hkv
        page, number = O.places(self.table, self.valid, self.q_lens, L, self.NP)
        pos = number if self.positions is None else np.repeat(self.positions[:, :, None], Hkv, 2)
        n = np.full(B, L) if self.q_lens is None else np.clip(self.q_lens, 0, L)
        mine = (np.arange(L) < n[:, None])[..., None, None]
        if got is not None:
            want = np.where(mine, O.rotate(q, np.repeat(pos, G, 2), self.freq, interleaved), 0.0)
            # sine and cosine: the reduced angle's rounding, the series' end and roundings 2^-23; products and sum 2^-23 of the pair
            tol = 2.0 ** -22 * O.reach(q, self.freq, interleaved) + HALF[self.dtype] * np.abs(want) + TINY[self.dtype]
            assert (np.abs(f64(got) - want) <= tol * mine).all()
        rk = O.rotate(k, pos, self.freq, interleaved)
        tol = 2.0 ** -22 * O.reach(k, self.freq, interleaved) + HALF["float16"] * np.abs(rk) + TINY["float16"]
        there = page >= 0
        b, i, h = np.nonzero(there)
        p, off = page[there], (number % 16)[there]
        if self.packed:
            for side, x in (("k", rk), ("v", v)):
                codes, scales = (getattr(self.pools, side + s).cpu().numpy() for s in ("_codes", "_scales"))
                wc, ws = np.full((self.NP, 16, D // 2), 0x55, np.uint8), np.full((self.NP, 16, D // 32), 0x55, np.uint8)
                if len(p):
                    c, s = MX.quantize(x[b, i, h])
                    wc[p, off], ws[p, off] = c[..., 0::2] | (c[..., 1::2] << 4), s
                zero = lambda y: np.where(y & 7, y & 15, 0) | np.where(y & 0x70, y & 0xF0, 0)  # noqa: E731
                assert np.array_equal(scales, ws) and np.array_equal(zero(codes), zero(wc))
            return
        for pool, x, t in ((self.pools.k_fp16, rk, tol), (self.pools.v_fp16, v, HALF["float16"] * np.abs(v) + TINY["float16"])):
            want, bound = np.full((self.NP, 16, D), 0.25), np.zeros((self.NP, 16, D))
            want[p, off], bound[p, off] = x[b, i, h], t[b, i, h]
            assert (np.abs(f64(pool) - want) <= bound).all()


SHAPES = [(1, 1, 4, 4, 64, 64), (3, 1, 7, 1, 128, 128), (64, 1, 32, 8, 128, 128), (2, 5, 8, 2, 64, 16), (2, 15, 6, 3, 128, 112),
          (2, 16, 6, 3, 128, 64), (3, 33, 8, 4, 64, 48), (1, 257, 12, 2, 128, 128), (5, 100, 4, 4, 128, 16)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotate_and_append(shape, dtype, interleaved, packed):
    s = Case(sum(shape), *shape, dtype, packed)
    s.check(s.run(interleaved), interleaved)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("far", [100, 100000, 10000000, 2 ** 31 - 1])
def test_far_positions(far, packed):
    s = Case(far, 3, 21, 8, 2, 128, 128, "float32", packed, far=far)
    s.check(s.run(False), False)


def test_every_quarter_turn():
    """Angles on and around multiples of an eighth of a turn."""
    s = Case(1, 1, 512, 2, 1, 64, 64, "float32", False, start=0, ragged=False)
    s.freq = np.concatenate([np.arange(1, 17) * np.pi / 8, np.arange(1, 17) * np.pi / 8 + 1e-5]).astype(np.float32)
    s.positions = np.concatenate([np.arange(256), -np.arange(256)])[None].astype(np.int32)
    s.check(s.run(False), False)


def test_no_turn_is_the_plain_append():
    import torch
    import intent_attention as ia
    for dtype in ("float16", "bfloat16", "float32"):
        s = Case(2, 3, 40, 4, 2, 64, 64, dtype, True)
        s.positions = np.zeros((3, 40), np.int32)
        got = s.run(True)
        assert torch.equal(got[0, :int(s.q_lens[0])], s.q[0, :int(s.q_lens[0])])
        other = ia.MxFp4Pools(*(torch.full_like(t, 0x55) for t in s.pools.tensors().values()))
        ia.append_mxfp4_tokens(s.k, s.v, other, _t(s.table), _t(s.valid), q_lens=_t(s.q_lens))
        for a, b in zip(s.pools.tensors().values(), other.tensors().values()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("packed", [False, True])
def test_lengths_and_tables(packed):
    s = Case(3, 6, 20, 4, 2, 64, 32, "float16", packed, W=3)
    s.q_lens = np.array([20, 25, -3, 7, 20, 1], np.int32)
    s.valid = np.array([[5, 60], [20, 48], [7, 7], [-2, 4], [2000000000, 33], [1, 0]], np.int32)
    s.table[0, 0, 0], s.table[1, 1, 2], s.table[4, 1, 1] = -1, s.NP, 2 ** 31 - 1
    s.check(s.run(False), False)
    s = Case(4, 2, 3, 4, 2, 64, 32, "float16", packed)
    s.table = s.table[:, :, :0]
    s.check(s.run(True), True)


def test_only_keys_and_values():
    for L in (1, 40):
        s = Case(5, 3, L, 4, 2, 128, 128, "bfloat16", False)
        assert s.run(False, q=None) is None
        s.check(None, False)


def test_in_place_and_layouts():
    import torch
    for interleaved in (False, True):
        s = Case(6, 3, 30, 8, 2, 128, 96, "bfloat16", False)
        before = s.q.clone()
        got = s.run(interleaved, q_out=s.q)
        assert got is s.q
        s.check(got, interleaved, q=before)
        # one projection's output, its parts side by side, at odd addresses
        s = Case(7, 3, 30, 8, 2, 64, 64, "float16", False)
        flat = torch.zeros(3, 30, 13 * 64 + 7, dtype=torch.float16, device="cuda")
        for name, at, heads in (("q", 1, 8), ("k", 8, 2), ("v", 10, 2)):
            view = flat[:, :, 3 + at * 64:3 + (at + heads) * 64].unflatten(-1, (heads, 64))
            setattr(s, name, view.copy_(getattr(s, name)))
        out = torch.full((3, 40, 9, 66), 7.0, dtype=torch.float16, device="cuda")
        view = out[:, 2:32, 1:, 1:65]
        s.check(s.run(interleaved, q_out=view), interleaved)
        out[:, 2:32, 1:, 1:65] = 7
        assert bool((out == 7).all())
        s.k, s.v = (x.transpose(1, 3).contiguous().transpose(1, 3) for x in (s.k, s.v))
        s.positions = np.arange(60, dtype=np.int32)[None, :30].repeat(3, 0)
        got = s.run(interleaved, positions=_t(np.arange(30, dtype=np.int32)).expand(3, 30))
        s.check(got, interleaved)


def test_special_values():
    import torch
    s = Case(8, 1, 4, 2, 1, 64, 64, "float32", False, ragged=False, start=0)
    s.positions = np.zeros((1, 4), np.int32)
    s.k[0, 0, 0, 0], s.k[0, 1, 0, 40], s.v[0, 2, 0, 5] = float("nan"), 1e6, float("-inf")
    s.run(False)
    k, v = (t[int(s.table[0, 0, 0]), :4] for t in (s.pools.k_fp16, s.pools.v_fp16))
    assert bool(k[0, 0].isnan()) and int(k.isnan().sum()) <= 2 and float(k[1, 40]) == float("inf") and float(v[2, 5]) == float("-inf")
    assert int(torch.isfinite(v).logical_not().sum()) == 1
    s = Case(8, 1, 4, 2, 1, 64, 64, "float32", True, ragged=False, start=0)
    s.k[0, 0, 0, 0], s.k[0, 1, 0, 40], s.v[0, 2, 0, 5] = float("nan"), 3e38, float("-inf")
    s.run(False)
    page = int(s.table[0, 0, 0])
    assert s.pools.k_scales[page, 0].tolist() == [255, 255] and s.pools.k_scales[page, 1, 1] == 140
    assert s.pools.v_scales[page, 2, 0] == 255 and s.pools.v_scales[page, 2, 1] < 200


def test_page_tags():
    import torch
    s = Case(9, 4, 37, 4, 2, 64, 64, "float16", False)
    tags = torch.full((s.NP,), 9, dtype=torch.int32, device="cuda")
    version = tags._version
    s.check(s.run(False, page_tags=tags, fp16_tag=3), False)
    page, _ = O.places(s.table, s.valid, s.q_lens, 37, s.NP)
    want = np.full(s.NP, 9)
    want[page[page >= 0]] = 3
    assert tags.tolist() == want.tolist() and tags._version > version


def test_long_batch():
    """More sequences than a grid's second axis holds."""
    s = Case(10, 33000, 1, 1, 1, 64, 16, "float16", False, start=3, W=1)
    s.check(s.run(False), False)


def test_graph_and_streams():
    import torch
    import intent_attention as ia
    s = Case(11, 4, 6, 8, 2, 128, 128, "float16", False, ragged=False)
    t = dict(table=_t(s.table), valid=_t(s.valid), freq=_t(s.freq), lens=_t(np.full(4, 6, np.int32)))
    out = torch.empty_like(s.q)
    call = lambda: ia.append_rotated_tokens(s.k, s.v, s.pools, t["table"], t["valid"], t["freq"], q=s.q, q_out=out,  # noqa: E731
                                            q_lens=t["lens"])
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = np.random.default_rng(5)
    for it in range(3):
        s.q_lens = rng.integers(0, 7, 4).astype(np.int32)
        t["lens"].copy_(_t(s.q_lens))
        for x in (s.q, s.k, s.v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(it)))
        s.pools.k_fp16.fill_(0.25), s.pools.v_fp16.fill_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        s.check(out, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    s.check(got, False)
