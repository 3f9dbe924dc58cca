"""Pages handed out, shared, given back, moved and copied on the GPU against Python lists:
tables, lengths and counts exactly, pool rows byte for byte; refusals that change nothing;
graphs; and a serving loop of these with the 4-bit cache's append and attention."""
import numpy as np
import pytest

from oracle import mxfp4 as O
from oracle.page_sharing import Pages

pytestmark = pytest.mark.gpu


def _dev():
    import torch
    return torch.device("cuda:0")


def _t(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=_dev())


class State:
    """The three tensors beside their lists, and pools of several row sizes."""

    def __init__(self, seed, B, R, W, NP, fill=0.8):
        import torch
        rng = np.random.default_rng(seed)
        self.rng = rng
        table = np.full((B, R, W), -1, np.int32)
        valid = np.zeros((B, R), np.int32)
        refs = np.zeros(NP, np.int32)
        pages = iter(rng.permutation(NP))
        for b in range(B):
            if b % 4 == 3:
                continue                                   # an empty slot
            for h in range(R):
                valid[b, h] = rng.integers(0, int(W * 16 * fill) + 1)
                for e in range(-(-valid[b, h] // 16)):
                    table[b, h, e] = next(pages)
                    refs[table[b, h, e]] += 1
        for p in rng.choice(NP, 3, replace=False):         # pages that another owner holds
            refs[p] += 2
        self.host = Pages(table, valid, refs)
        self.table, self.valid, self.refs = _t(table), _t(valid), _t(refs)
        g = torch.Generator(device=_dev()).manual_seed(seed)
        r = lambda *s: torch.randint(0, 255, s, generator=g, device=_dev(), dtype=torch.uint8)  # noqa: E731
        # rows of 1, 3, 4, 24, 64 and 1,024 bytes
        self.pools = [r(NP), r(NP, 3), r(NP, 4).view(torch.int32), r(NP, 24), r(NP, 4, 16), r(NP, 16, 64)]
        self.want = [p.clone() for p in self.pools]

    def check(self):
        import torch
        assert self.table.tolist() == self.host.table
        assert self.valid.tolist() == self.host.valid
        assert self.refs.tolist() == self.host.refs
        for s, d in self.host.copied:
            for w in self.want:
                w[d] = w[s]
        self.host.copied = []
        for p, w in zip(self.pools, self.want):
            assert torch.equal(p, w)


@pytest.mark.parametrize("B,R,W,NP", [(4, 1, 1, 9), (9, 2, 5, 100), (12, 3, 40, 2100), (70, 1, 3, 1024), (8, 5, 33, 3333),
                                      (12, 3, 40, 16384), (12, 3, 40, 16385), (9, 2, 30, 40000)])
def test_grow_fork_free_follow_the_lists(B, R, W, NP):
    import intent_attention as ia
    s = State(B * 100 + W, B, R, W, NP)
    s.check()
    done = 0
    for it in range(12):
        empty = [b for b in range(B) if all(v == 0 for v in s.host.valid[b])]
        full = [b for b in range(B) if b not in empty]
        kind = it % 3
        if kind == 0 and empty and full:
            kids = list(s.rng.permutation(empty)[:max(1, len(empty) // 2)])
            folks = [int(s.rng.choice(full)) for _ in kids]
            kids = [int(k) for k in kids]
            want = s.host.fork(folks, kids)
            got = ia.fork_sequences(s.table, s.valid, s.refs, _t(folks), _t(kids), s.pools)
        elif kind == 1:
            seqs = [int(x) for x in s.rng.permutation(B)[:max(1, B // 2)]]
            new = [int(x) for x in s.rng.integers(0, W * 4 + 2, len(seqs))]
            want = s.host.grow(seqs, new)
            got = ia.grow_sequences(s.table, s.valid, s.refs, seqs, new)
        else:
            seqs = [int(x) for x in s.rng.permutation(B)[:max(1, B // 4)]]
            seqs += [seqs[0], -1, B, 2 ** 31 - 1]
            s.host.free(seqs)
            ia.free_sequences(s.table, s.valid, s.refs, _t(seqs))
            want, got = 0, _t([0])
        assert got.tolist() == [want]
        done += want == 0
        s.check()
    assert done >= 4


@pytest.mark.parametrize("NP", [200, 17000])
def test_refusals_change_nothing(NP):
    import intent_attention as ia
    s = State(5, 8, 2, 6, NP, fill=0.5)
    two = [b for b in range(8) if b % 4 == 3]
    for b in two:
        assert s.host.valid[b] == [0, 0]
    for seqs, new in (([0, 0], [1, 1]), ([8], [1]), ([-1], [1]), ([0], [-1]), ([0], [97]), ([0, 1], [1, 2 ** 31 - 1])):
        assert s.host.grow(seqs, new) == -1
        assert ia.grow_sequences(s.table, s.valid, s.refs, seqs, new).tolist() == [-1]
        s.check()
    for folks, kids in (([0, 1], [3, 3]), ([0], [1]), ([3], [3]), ([3, 0], [7, 3]), ([8], [3]), ([-1], [3]), ([0], [9])):
        assert s.host.fork(folks, kids) == -1
        assert ia.fork_sequences(s.table, s.valid, s.refs, folks, kids, s.pools).tolist() == [-1]
        s.check()
    assert ia.grow_sequences(s.table, s.valid, s.refs, [], []).tolist() == [0]
    assert ia.fork_sequences(s.table, s.valid, s.refs, [], []).tolist() == [0]
    ia.free_sequences(s.table, s.valid, s.refs, [])
    s.check()


@pytest.mark.parametrize("NP", [60, 17000])
def test_too_few_free_pages(NP):
    import intent_attention as ia
    s = State(6, 4, 1, 40, NP, fill=0.2)
    free = [p for p in range(NP) if s.host.refs[p] == 0]
    for p in s.rng.permutation(free)[:max(0, len(free) - 35)]:       # others hold the rest
        s.host.refs[p] = 1
    s.refs.copy_(_t(s.host.refs))
    short = s.host.grow([0, 3], [200, 16 * 38])
    assert short > 0
    assert ia.grow_sequences(s.table, s.valid, s.refs, [0, 3], [200, 16 * 38]).tolist() == [short]
    s.check()
    free = sum(r <= 0 for r in s.host.refs)
    assert s.host.grow([3], [16 * min(free, 40)]) == 0
    assert ia.grow_sequences(s.table, s.valid, s.refs, [3], [16 * min(free, 40)]).tolist() == [0]
    s.check()


def test_fork_of_full_empty_and_pageless_parents():
    """Last pages that are full, parents without tokens, entries that are no pages."""
    import intent_attention as ia
    s = State(7, 12, 1, 4, 64, fill=0.0)
    assert s.host.grow([0, 1, 2], [32, 33, 0]) == 0
    assert ia.grow_sequences(s.table, s.valid, s.refs, [0, 1, 2], [32, 33, 0]).tolist() == [0]
    s.host.valid[4], s.host.table[4][0][:2] = [20], [-1, 99]          # a length without pages
    s.valid[4, 0], s.table[4, 0, 0], s.table[4, 0, 1] = 20, -1, 99
    s.host.valid[5], s.host.table[5][0][:] = [200], list(s.host.table[1][0])     # longer than its table
    s.valid[5, 0], s.table[5, 0] = 200, s.table[1, 0]
    assert s.host.fork([0, 1, 2, 4, 5, 1], [6, 7, 8, 9, 10, 11]) == 0
    assert ia.fork_sequences(s.table, s.valid, s.refs, [0, 1, 2, 4, 5, 1], [6, 7, 8, 9, 10, 11], s.pools).tolist() == [0]
    s.check()


@pytest.mark.parametrize("B,R,W,NP", [(1, 1, 1, 1), (4, 1, 6, 30), (12, 3, 40, 2100), (8, 5, 33, 3333), (3, 1, 5, 5000),
                                      (12, 3, 40, 8192), (12, 3, 40, 8193), (9, 2, 30, 20011)])
def test_compaction(B, R, W, NP):
    import torch
    import intent_attention as ia
    s = State(B + W, B, R, W, max(NP, 4)) if NP > 1 else None
    if s is None:
        one = torch.ones((1, 4), dtype=torch.uint8, device=_dev())
        t, r, m = ia.compact_pages(_t([[[0]]]), _t([[1]]), _t([1]), one)
        assert (t.tolist(), r.tolist(), m.tolist()) == ([[[0]]], [1], [0])
        return
    s.table[0, 0, 0] = 0
    s.host.table[0][0][0] = 0
    for refs in (s.host.refs, [0] * NP, [3] * NP, [1] + [0] * (NP - 1), [0] * (NP - 1) + [2], [-1, 5] * (NP // 2) + [0] * (NP % 2)):
        s.host.refs = list(refs)
        s.refs.copy_(_t(refs))
        table, new_refs, page_map, moves = s.host.compact()
        t, r, m = ia.compact_pages(s.table, s.valid, s.refs, s.pools)
        assert r.tolist() == new_refs and m.tolist() == page_map and t.tolist() == table
        s.host.copied = moves
        s.check()                                  # the arguments stay, the moved rows are copied


@pytest.mark.parametrize("B,R,W,NP", [(5, 1, 4, 40), (9, 3, 40, 1500)])
def test_newest_tokens_let_go(B, R, W, NP):
    """Some, none and more tokens than there are, negative numbers, a sequence twice; grown again after it."""
    import intent_attention as ia
    s = State(B * 7 + W, B, R, W, NP)
    for it in range(8):
        seqs = [int(x) for x in s.rng.integers(-1, B + 1, B)]
        drop = [int(x) for x in s.rng.choice([0, 1, 5, 15, 16, 17, 40, -3, W * 16, 2 ** 31 - 1], B)]
        s.host.free(seqs, drop)
        ia.free_sequences(s.table, s.valid, s.refs, _t(seqs), _t(drop))
        s.check()
        one = [int(s.rng.integers(0, B))]
        want = s.host.grow(one, [23])
        assert ia.grow_sequences(s.table, s.valid, s.refs, one, [23]).tolist() == [want]
        s.check()
    with pytest.raises(ValueError, match="tokens"):
        ia.free_sequences(s.table, s.valid, s.refs, [0, 1], [1])


def test_compaction_of_no_pages():
    """No page in the pools, arrays named all the same: entries as they are, nothing copied."""
    import torch
    from intent_attention import _native as N
    table, valid = _t([[5, -1, 2]]), _t([20])
    out, pool = torch.zeros_like(table), torch.full((64,), 9, dtype=torch.uint8, device=_dev())
    ws = torch.full((4096,), 255, dtype=torch.uint8, device=_dev())
    a = N.CompactPagesArgs(1, 3, 16, 0, table.data_ptr(), valid.data_ptr(), None, out.data_ptr())
    a.num_arrays = 1
    a.arrays[0] = (pool.data_ptr(), 16)
    N.compact_pages(a, torch.cuda.current_stream().cuda_stream, ws.data_ptr(), N.compact_pages_workspace(a))
    assert out.tolist() == table.tolist() and bool((pool == 9).all())


def test_compaction_without_pools_and_copy_pages():
    import torch
    import intent_attention as ia
    s = State(11, 8, 2, 10, 200)
    t, r, m = ia.compact_pages(s.table, s.valid, s.refs)
    table, new_refs, page_map, moves = s.host.compact()
    assert t.tolist() == table and r.tolist() == new_refs and m.tolist() == page_map
    ids = s.rng.permutation(200)
    src, dst = [int(x) for x in ids[:40]] + [-1, 5, 200, 7], [int(x) for x in ids[40:80]] + [3, -1, 4, 2 ** 31 - 1]
    ia.copy_pages(s.pools, _t(src), _t(dst))
    s.host.copied = list(zip(src[:40], dst[:40]))
    s.check()
    ia.copy_pages(s.pools, [], [])
    halves = ia.PagePools(k_fp16=torch.randn((20, 16, 64), device=_dev()).half(), v_fp16=torch.randn((20, 16, 64), device=_dev()).half(),
                          k_int8_scale=torch.randn(20, device=_dev()).half(), k_int4r_scale=torch.randn((20, 2), device=_dev()))
    want = {n: x.clone() for n, x in halves.tensors().items()}
    ia.copy_pages(halves, [3, 4], [10, 11])
    for n, x in halves.tensors().items():
        want[n][10:12] = want[n][3:5]
        assert torch.equal(x, want[n])


@pytest.mark.parametrize("NP", [900, 17000])
def test_page_operators_replay_in_a_graph(NP):
    """Fork, grow, free and compact captured once, replayed on other sequences."""
    import torch
    import intent_attention as ia
    s = State(21, 12, 2, 20, NP, fill=0.5)
    seqs, new, folks, kids, gone = _t([0]), _t([40]), _t([1]), _t([3]), _t([2])
    short = [torch.zeros(1, dtype=torch.int32, device=_dev()) for _ in range(2)]

    def step():
        ia.free_sequences(s.table, s.valid, s.refs, gone)
        ia.grow_sequences(s.table, s.valid, s.refs, seqs, new, missing=short[0])
        ia.fork_sequences(s.table, s.valid, s.refs, folks, kids, s.pools, missing=short[1])
        return ia.compact_pages(s.table, s.valid, s.refs)

    keep = [x.clone() for x in (s.table, s.valid, s.refs, *s.pools)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moved = step()
    for x, k in zip((s.table, s.valid, s.refs, *s.pools), keep):
        x.copy_(k)
    for a, n, p, c, f in ((0, 40, 1, 3, 2), (4, 17, 0, 7, 1), (5, 100, 4, 11, 3), (6, 0, 5, 1, 7)):
        for t, v in ((seqs, a), (new, n), (folks, p), (kids, c), (gone, f)):
            t.fill_(v)
        s.host.free([f])
        want = [s.host.grow([a], [n]), s.host.fork([p], [c])]
        graph.replay()
        torch.cuda.synchronize()
        assert [x.item() for x in short] == want
        s.check()
        table, refs, page_map, _ = s.host.compact()
        assert moved[0].tolist() == table and moved[1].tolist() == refs and moved[2].tolist() == page_map


@pytest.mark.parametrize("D,Hkv,G", [(64, 2, 3), (128, 1, 8)])
def test_serving_loop(D, Hkv, G):
    """Prompts admitted, written and attended, decoded token by token, forked, freed and
    compacted, the cache checked against a copy of every token at each step."""
    import torch
    import intent_attention as ia
    dev, rng = _dev(), np.random.default_rng(D)
    B, W, NP = 6, 12, 150
    pools = ia.MxFp4Pools.empty(NP, D, dev)
    table = torch.full((B, Hkv, W), -1, dtype=torch.int32, device=dev)
    valid = torch.zeros((B, Hkv), dtype=torch.int32, device=dev)
    refs = torch.zeros(NP, dtype=torch.int32, device=dev)
    kept = [([], []) for _ in range(B)]                   # every token's K and V [Hkv, D] as written

    def write_and_attend(new):
        L = max(new)
        k, v = (torch.from_numpy(rng.standard_normal((B, L, Hkv, D)).astype(np.float32)).to(dev).bfloat16() for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((B, L, Hkv * G, D)).astype(np.float32)).to(dev).bfloat16()
        lens = _t(new)
        ia.append_mxfp4_tokens(k, v, pools, table, valid, q_lens=lens)
        out = ia.mxfp4_paged_attention(q, pools, table, valid, q_lens=lens)
        for b, n in enumerate(new):
            for i in range(n):
                kept[b][0].append(k[b, i].double().cpu().numpy())
                kept[b][1].append(v[b, i].double().cpu().numpy())
        for b, n in enumerate(new):
            T = len(kept[b][0])
            assert valid[b].tolist() == [T] * Hkv
            assert (out[b, n:] == 0).all()
            if n == 0:
                continue
            kk, vv = (O.values(*O.quantize(np.stack(x))) for x in kept[b])
            for i in range(n):
                for h in range(Hkv * G):
                    s = kk[:T - n + i + 1, h // G] @ q[b, i, h].double().cpu().numpy() / np.sqrt(D)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    want, mass = p @ vv[:T - n + i + 1, h // G], p @ np.abs(vv[:T - n + i + 1, h // G])
                    err = np.abs(out[b, i, h].double().cpu().numpy() - want)
                    assert (err <= 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * mass).all()

    def grow(seqs, new):
        assert ia.grow_sequences(table, valid, refs, seqs, new).tolist() == [0]
        full = [0] * B
        for s, n in zip(seqs, new):
            full[s] = n
        write_and_attend(full)

    grow([0, 1, 2], [37, 16, 1])                          # prompts
    for _ in range(3):
        grow([0, 1, 2], [1, 1, 1])                        # decode steps
    assert ia.fork_sequences(table, valid, refs, [0, 0, 1], [3, 4, 5], pools).tolist() == [0]
    for c, p in ((3, 0), (4, 0), (5, 1)):
        kept[c] = ([*kept[p][0]], [*kept[p][1]])
    grow([0, 3, 4, 5], [1, 1, 2, 14])                     # each continues for itself
    ia.free_sequences(table, valid, refs, [1, 3])
    kept[1], kept[3] = ([], []), ([], [])
    table, refs, _ = ia.compact_pages(table, valid, refs, pools)
    live = int((refs > 0).sum())
    assert bool((refs[:live] > 0).all())
    grow([0, 1, 4], [5, 20, 1])
    grow([0, 1, 2, 4, 5], [1, 1, 1, 1, 1])
    grow([0, 2, 4], [18, 4, 4])                           # drafts, of which some are not taken
    ia.free_sequences(table, valid, refs, [0, 2], [17, 2])
    for b, n in ((0, 17), (2, 2)):
        kept[b] = tuple(x[:-n] for x in kept[b])
    grow([0, 2, 4], [1, 1, 1])
    used = [-(-len(kept[b][0]) // 16) * Hkv for b in range(B)]
    assert int(refs.sum()) == sum(used)                   # every entry counted, none more
