"""Reordering sequences on the GPU against Python lists: tables, lengths and counts exactly, pool
rows byte for byte; refusals that change nothing; and a beam search of choice and reordering."""
import numpy as np
import pytest

from oracle import beam_search
from test_gpu_page_sharing import State, _t

pytestmark = pytest.mark.gpu


def _reorder(s, seqs, parents, pools=True):
    import intent_attention as ia
    m = ia.reorder_sequences(s.table, s.valid, s.refs, _t(seqs), _t(parents), s.pools if pools else None)
    want = s.host.reorder(list(map(int, seqs)), list(map(int, parents)))
    if not pools:
        s.host.copied = []
    assert m.tolist() == [want]
    s.check()
    return want


@pytest.mark.parametrize("B,R,W,NP", [(4, 1, 1, 9), (9, 2, 5, 100), (12, 3, 40, 2100), (70, 1, 3, 1024), (8, 5, 33, 3333),
                                      (12, 3, 40, 16385), (9, 2, 30, 40000), (600, 4, 9, 30000)])
def test_reorder_follows_the_lists(B, R, W, NP):
    s = State(B * 100 + W, B, R, W, NP)
    done = 0
    for it in range(10):
        n = int(s.rng.integers(1, B + 1))
        seqs = s.rng.permutation(B)[:n]
        parents = s.rng.integers(0, B, n) if it % 2 else s.rng.choice(s.rng.integers(0, B, max(1, n // 3)), n)
        done += _reorder(s, seqs, parents) == 0
    assert done > 0


def test_permutations_and_one_for_all():
    s = State(3, 16, 2, 20, 1000)
    _reorder(s, np.arange(16), np.arange(16))                    # nothing happens
    _reorder(s, np.arange(16), np.roll(np.arange(16), 1))        # no page is copied
    _reorder(s, np.arange(16)[::-1].copy(), s.rng.permutation(16))
    _reorder(s, np.arange(16), np.full(16, 5))                   # all become one
    _reorder(s, np.arange(16), np.full(16, 3))
    _reorder(s, [], [])


def test_refusals_change_nothing():
    s = State(4, 8, 2, 6, 70, fill=1.0)
    for seqs, parents in (([0, 0], [1, 2]), ([8], [0]), ([-1], [0]), ([0], [8]), ([0], [-1]), ([1, 2, 1], [0, 0, 0])):
        assert _reorder(s, seqs, parents) == -1
    # no free page is left: the ragged ones' copies are too many
    s.refs[s.refs == 0] = 1
    s.host.refs = [r if r else 1 for r in s.host.refs]
    assert _reorder(s, [0, 1, 2, 3], [4, 4, 4, 4]) > 0
    assert _reorder(s, [4, 5], [5, 4]) == 0                      # moves need none


def test_without_pools_and_with_odd_entries():
    s = State(5, 8, 2, 10, 400)
    _reorder(s, [0, 1, 2], [1, 1, 0], pools=False)
    # entries outside the pools, lengths past the table and below zero
    s.table[4, 0, 0] = s.host.table[4][0][0] = 999
    s.valid[5, 1] = s.host.valid[5][1] = 10 * 16 + 5
    s.valid[6, 0] = s.host.valid[6][0] = -3
    _reorder(s, [0, 1, 2, 4, 5, 6], [4, 5, 6, 5, 6, 4])
    _reorder(s, [4, 5, 6, 7], [0, 1, 2, 2])


def test_lists_streams_and_graphs():
    import torch
    import intent_attention as ia
    s = State(6, 12, 2, 9, 600)
    seqs, parents = list(range(12)), [0, 0, 0, 0, 5, 4, 6, 6, 9, 9, 9, 1]
    m = ia.reorder_sequences(s.table, s.valid, s.refs, seqs, parents, s.pools)
    assert m.tolist() == [s.host.reorder(seqs, parents)]
    s.check()
    gs, gp = _t(seqs), _t(parents)
    graph = torch.cuda.CUDAGraph()
    missing = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    with torch.cuda.graph(graph):
        ia.reorder_sequences(s.table, s.valid, s.refs, gs, gp, s.pools, missing=missing)
    for it in range(4):
        parents = [int(x) for x in s.rng.integers(0, 12, 12)]
        gp.copy_(_t(parents))
        graph.replay()
        torch.cuda.synchronize()
        assert missing.tolist() == [s.host.reorder(seqs, parents)]
        s.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m = ia.reorder_sequences(s.table, s.valid, s.refs, seqs, [3] * 12, s.pools)
    side.synchronize()
    assert m.tolist() == [s.host.reorder(seqs, [3] * 12)]
    s.check()
    before = [t._version for t in (s.table, s.valid, s.refs, s.pools[0])]
    ia.reorder_sequences(s.table, s.valid, s.refs, seqs, seqs, s.pools)
    assert all(t._version > v for t, v in zip((s.table, s.valid, s.refs, s.pools[0]), before))


def test_beam_search_over_pages():
    """Beams grown, chosen and reordered: every row's pages spell the beam's own tokens."""
    import torch
    import intent_attention as ia
    B, K, V, W, NP, steps = 2, 3, 50, 4, 400, 40
    g = torch.Generator().manual_seed(1)
    model = torch.randn(V, V, generator=g) * 2
    S = B * K
    table = torch.full((S, 1, W), -1, dtype=torch.int32, device="cuda")
    valid = torch.zeros((S, 1), dtype=torch.int32, device="cuda")
    refs = torch.zeros(NP, dtype=torch.int32, device="cuda")
    pool = torch.zeros((NP, 16), dtype=torch.int32, device="cuda")       # a page's tokens
    scores = torch.full((B, K), float("-inf"), device="cuda")
    scores[:, 0] = 0
    seqs = torch.arange(S, dtype=torch.int32, device="cuda")
    one = torch.ones(S, dtype=torch.int32, device="cuda")
    last = torch.zeros((B, K), dtype=torch.int64)
    beams, s64 = [[[] for _ in range(K)] for _ in range(B)], np.where(np.arange(K) == 0, 0.0, -np.inf) * np.ones((B, 1))
    s64 = np.where(np.isnan(s64), -np.inf, s64)
    for step in range(steps):
        logits = model[last]
        s, parents, tokens = ia.beam_select(logits.cuda(), scores)
        want = beam_search.select(logits.numpy(), scores.cpu().numpy(), K)
        assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(tokens.cpu().numpy(), want[2])
        assert ia.reorder_sequences(table, valid, refs, seqs, parents.flatten(), [pool]).tolist() == [0]
        assert ia.grow_sequences(table, valid, refs, seqs, one, [pool]).tolist() == [0]
        at = (valid[:, 0] - 1).long()
        page = table[seqs.long(), 0, at // 16].long()
        pool[page, at % 16] = tokens.flatten()
        beams = [[beams[b][int(p) - b * K] + [int(t)] for p, t in zip(want[1][b], want[2][b])] for b in range(B)]
        scores, last = s, tokens.long().cpu()
        for b in range(B):
            for k in range(K):
                row = pool[table[b * K + k, 0, :-(-(step + 1) // 16)].long()].flatten()[:step + 1]
                assert row.tolist() == beams[b][k]
    used = table[table >= 0]
    assert torch.equal(torch.bincount(used, minlength=NP).int(), refs)
