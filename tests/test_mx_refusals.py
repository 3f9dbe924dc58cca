"""Further refusals of the 4-bit token cache's and the page operators' entry points, without a GPU."""
import pytest

from intent_attention import _native as N


def _seqs():
    a = N.SequencesArgs()
    a.num_seqs, a.rows_per_seq, a.table_width, a.page_size, a.num_pages, a.count = 4, 2, 9, 16, 50, 2
    a.page_table, a.valid_tokens, a.refs, a.seqs, a.parents = 4096, 8192, 12288, 16384, 20480
    a.new_tokens, a.missing, a.granted = 24576, 28672, 32768
    return a


@pytest.mark.parametrize("at,text", [(32770, "aligned"), (4096 - 12, "page_table"), (4096 + 4 * 71, "page_table"), (8192 + 28, "valid_tokens"),
                                     (12288 + 4 * 49, "refs"), (16388, "seqs"), (24576 - 4, "new_tokens"), (28672, "missing"),
                                     (28672 - 12, "missing")])
def test_granted_is_none_of_the_other_arrays(at, text):
    a = _seqs()
    a.granted = at
    with pytest.raises(ValueError, match=text):
        N.grow_sequences(a, 0, 1 << 20, N.sequences_workspace(a))
