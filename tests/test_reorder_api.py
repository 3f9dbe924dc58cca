"""Reordering sequences: the oracle by hand and the refusals, without a GPU."""
import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from oracle.page_sharing import Pages


def _pages(lens, W=3, NP=12, extra=()):
    table, it = [], iter(range(NP))
    refs = [0] * NP
    for n in lens:
        row = [next(it) if e < -(-n // 16) else -1 for e in range(W)]
        for p in row:
            if p >= 0:
                refs[p] += 1
        table.append([row])
    for p in extra:
        refs[p] += 1
    return Pages(table, [[n] for n in lens], refs)


def test_oracle_moves_a_last_page_and_copies_it():
    s = _pages([20, 16, 40])                       # pages 0 1 | 2 | 3 4 5
    assert s.reorder([0, 1, 2], [1, 0, 0]) == 0    # 0's last page goes to 1, 2 gets a copy in page 6
    assert s.table == [[[2, -1, -1]], [[0, 1, -1]], [[0, 6, -1]]]
    assert s.valid == [[16], [20], [20]] and s.copied == [(1, 6)]
    assert s.refs == [2, 1, 1, 0, 0, 0, 1, 0, 0, 0, 0, 0]


def test_oracle_parent_keeps_its_last_page():
    for seqs, parents in (([1], [0]), ([1, 0], [0, 0])):
        s = _pages([20, 0])
        assert s.reorder(seqs, parents) == 0
        assert s.table == [[[0, 1, -1]], [[0, 2, -1]]] and s.copied == [(1, 2)] and s.refs[:3] == [2, 1, 1]


def test_oracle_all_or_nothing():
    s = _pages([20, 0, 0], NP=3, extra=[2])
    assert s.reorder([1, 2], [0, 0]) == 2 and s.valid == [[20], [0], [0]]
    for seqs, parents in (([1, 1], [0, 0]), ([3], [0]), ([1], [-1])):
        assert s.reorder(seqs, parents) == -1


def _seqs(**kw):
    a = N.SequencesArgs()
    a.num_seqs, a.rows_per_seq, a.table_width, a.page_size, a.num_pages, a.count = 4, 2, 9, 16, 50, 2
    a.page_table, a.valid_tokens, a.refs, a.seqs, a.parents, a.missing = 4096, 8192, 12288, 16384, 20480, 28672
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,text", [(dict(count=-1), "bad size"), (dict(rows_per_seq=0), "bad size"), (dict(seqs=None), "seqs"),
                                     (dict(parents=None), "parents"), (dict(missing=None), "missing"), (dict(refs=None), "refs"),
                                     (dict(page_table=4097), "aligned"), (dict(num_arrays=25), "num_arrays"),
                                     (dict(table_width=1 << 28), "int32"), (dict(count=1 << 23, rows_per_seq=4), "too many rows")])
def test_abi_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        N.reorder_sequences(_seqs(**kw), 0, 1 << 20, 1 << 40)


def test_abi_workspace():
    need = N.reorder_sequences_workspace(_seqs())
    assert need > N.sequences_workspace(_seqs())
    for at, size in ((None, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            N.reorder_sequences(_seqs(), 0, at, size)


def test_python_refuses():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        ia.reorder_sequences(i(2, 1, 3), i(2, 1), i(9), [0], [1])
