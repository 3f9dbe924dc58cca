"""Sequences forked and reordered without pools: the pages are handed out, and the caller copies the last ones, pool by pool."""
import pytest

from test_gpu_page_sharing import State, _t

pytestmark = pytest.mark.gpu


def _copy_by_hand(s, before, seqs, parents):
    """The last entries that are neither the parent's nor what the sequence had: (page of the parent, new page)."""
    import intent_attention as ia
    after = s.table.tolist()
    pairs = []
    for c, p in zip(seqs, parents):
        for h in range(len(after[c])):
            n = min(-(-s.valid[c, h].item() // 16), len(after[c][h]))
            if c != p and n > 0 and after[c][h][n - 1] != before[p][h][n - 1]:
                pairs.append((before[p][h][n - 1], after[c][h][n - 1]))
    for pool in s.pools:                                         # one call each, as if they were too many
        ia.copy_pages(pool, [a for a, _ in pairs], [b for _, b in pairs])
    return pairs


def test_fork_and_copy():
    import intent_attention as ia
    s = State(11, 12, 2, 9, 300)
    children = [b for b in range(12) if not any(s.host.valid[b])][:2]
    parents = [0, 1]
    before = s.table.tolist()
    m = ia.fork_sequences(s.table, s.valid, s.refs, parents, children)
    assert m.tolist() == [s.host.fork(parents, children)] == [0]
    want, s.host.copied = s.host.copied, []
    s.check()                                                    # no pool is touched
    assert sorted(_copy_by_hand(s, before, children, parents)) == sorted(want) and want
    s.host.copied = want
    s.check()


@pytest.mark.parametrize("seqs,parents", [([0, 1, 2, 3], [1, 1, 1, 0]), ([4, 5, 6], [5, 4, 4]), (list(range(8)), [2] * 8)])
def test_reorder_and_copy(seqs, parents):
    import intent_attention as ia
    s = State(12, 8, 3, 7, 400)
    before = s.table.tolist()
    m = ia.reorder_sequences(s.table, s.valid, s.refs, _t(seqs), _t(parents))
    assert m.tolist() == [s.host.reorder(seqs, parents)] == [0]
    want, s.host.copied = s.host.copied, []
    s.check()
    assert sorted(_copy_by_hand(s, before, seqs, parents)) == sorted(want) and want
    s.host.copied = want
    s.check()


def test_growing_is_refused():
    """A row that would write into a page that others hold gets no page without a copy of it."""
    import intent_attention as ia
    s = State(13, 8, 1, 9, 200)
    row = next(b for b in range(8) if s.host.valid[b][0] % 16)
    page = s.host.table[row][0][s.host.valid[row][0] // 16]
    s.refs[page] += 1
    s.host.refs[page] += 1
    assert ia.grow_sequences(s.table, s.valid, s.refs, [row], [1]).tolist() == [-1] == [s.host.grow([row], [1])]
    s.check()
