"""Further refusals of the 4-bit token cache's and the page operators' entry points, without a GPU."""
import os
import subprocess
import sys

import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from intent_attention import mxfp4, page_sharing

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def test_free_does_not_read_the_arrays():
    """A free whose num_arrays nobody set: the arrays are grow's and fork's. In a process that sees no
    device, so that nothing is launched: an error, and no crash."""
    code = ("import sys; sys.path.insert(0, 'intent-attention-kernel_amd')\n"
            "from intent_attention import _native as N\n"
            "a = N.SequencesArgs()\n"
            "a.num_seqs, a.rows_per_seq, a.table_width, a.page_size, a.num_pages, a.count = 4, 2, 9, 16, 50, 2\n"
            "a.page_table = a.valid_tokens = a.refs = a.seqs = 4096\n"
            "for n in (25, -1, 1 << 30):\n"
            "    a.num_arrays = n\n"
            "    try: N.free_sequences(a, 0)\n"
            "    except RuntimeError as e: print('error', e)\n")
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env, cwd=ROOT)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])
    assert len(r.stdout.splitlines()) == 3, r.stdout


@pytest.mark.parametrize("n,text", [(-1, "num_arrays"), (25, "num_arrays"), (1, "row_bytes")])
def test_grow_checks_its_arrays(n, text):
    a = _seqs()
    a.num_arrays, a.arrays[0].base = n, 65536
    with pytest.raises(ValueError, match=text):
        N.grow_sequences(a, 0, 1 << 20, N.sequences_workspace(a))


def test_sizes_that_an_int32_would_wrap():
    """Tables of 2^32 entries and more, which a 32-bit field would make narrow ones."""
    meta = lambda *s: torch.empty(s, dtype=torch.int32, device="meta")  # noqa: E731
    pools = ia.MxFp4Pools.empty(4, 64, "cpu")
    for B, H, W in ((1, 1, 2 ** 32), (1, 2, 2 ** 32 + 5), (1, 1, 2 ** 27), (2 ** 17, 2 ** 15, 1)):
        with pytest.raises(ValueError, match="int32"):
            mxfp4._check_cache(pools, meta(B, H, W), meta(B, H), None, B, 64)
        with pytest.raises(ValueError, match="int32"):
            page_sharing._check_state(meta(B, H, W), meta(B, H), meta(4))
    assert mxfp4._check_cache(pools, meta(1, 1, 2 ** 27 - 1), meta(1, 1), None, 1, 64) == (1, 2 ** 27 - 1, 4)
    assert page_sharing._check_state(meta(1, 1, 2 ** 27 - 1), meta(1, 1), meta(4)) == (1, 1, 2 ** 27 - 1, 4)
