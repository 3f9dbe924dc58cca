"""Refusals of the 4-bit token cache's and the page operators' entry points, without a GPU:
the C ABI's argument checks, the Python layer's, the argument blocks' layouts; and the
oracle's own number format."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from intent_attention import mxfp4, page_sharing
from oracle import mxfp4 as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cname,pyname", [("iak_mx_tokens_args", "MxTokensArgs"), ("iak_mx_attention_args", "MxAttentionArgs"),
                                          ("iak_page_array", "PageArray"), ("iak_copy_pages_args", "CopyPagesArgs"),
                                          ("iak_sequences_args", "SequencesArgs"),
                                          ("iak_compact_pages_args", "CompactPagesArgs")])
def test_argument_blocks_match_the_header(cname, pyname):
    S = getattr(N, pyname)
    fields = [f[0] for f in S._fields_]
    prog = ['#include <stdio.h>', '#include <stddef.h>', '#include "iak.h"', 'int main(void){',
            f'printf("size %zu\\n", sizeof({cname}));', 'printf("most %d\\n", IAK_MAX_PAGE_ARRAYS);']
    prog += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(c, "w").write("\n".join(prog))
        subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(S) and int(got["most"]) == N.MAX_PAGE_ARRAYS
    for f in fields:
        assert int(got[f]) == getattr(S, f).offset, f


def _attention_args():
    a = N.MxAttentionArgs()
    a.batch, a.q_len, a.num_q_heads, a.num_kv_heads, a.head_dim, a.page_size, a.table_width, a.num_pages = 2, 3, 8, 2, 128, 16, 64, 500
    a.q = a.out = a.page_table = a.valid_tokens = a.k_codes = a.k_scales = a.v_codes = a.v_scales = 256
    a.sm_scale, a.causal = 0.1, 1
    return a


def test_attention_refusals():
    assert N.mx_attention_workspace(_attention_args()) % 256 == 0
    for field, value, text in (("batch", -1, "size"), ("q_len", -1, "size"), ("num_kv_heads", 0, "size"), ("num_q_heads", 7, "multiple"),
                               ("num_q_heads", 0, "multiple"), ("head_dim", 96, "head_dim 96"), ("page_size", 32, "page_size 32"),
                               ("num_pages", 1 << 31, "int32"), ("table_width", 1 << 27, "int32"), ("q_dtype", 3, "dtype"),
                               ("out_dtype", -1, "dtype"), ("sm_scale", float("nan"), "finite"), ("sm_scale", float("inf"), "finite"),
                               ("causal", 2, "causal"), ("splits", -1, "splits"), ("q", 0, "NULL"), ("out", 0, "NULL"),
                               ("page_table", 0, "NULL"), ("valid_tokens", 0, "NULL"), ("v_scales", 0, "NULL"),
                               ("k_codes", 264, "16-byte"), ("q_len", 1 << 30, "too long"), ("batch", 1 << 26, "too many")):
        a = _attention_args()
        setattr(a, field, value)
        with pytest.raises(ValueError, match=text):
            N.mx_attention_workspace(a)
    a = _attention_args()
    a.splits = 4
    need = N.mx_attention_workspace(a)
    assert need > 0
    for ws, size in ((0, need), (256, need - 1), (264, need)):
        with pytest.raises(ValueError, match="workspace"):
            N.mx_attention(a, 0, ws, size)


def test_token_refusals():
    def args():
        a = N.MxTokensArgs()
        a.batch, a.count, a.num_kv_heads, a.head_dim, a.page_size, a.table_width, a.num_pages = 2, 3, 8, 64, 16, 9, 50
        a.k = a.v = a.page_table = a.valid_tokens = a.k_codes = a.k_scales = a.v_codes = a.v_scales = 256
        return a
    for field, value, text in (("count", -1, "size"), ("head_dim", 32, "head_dim"), ("page_size", 8, "page_size"), ("dtype", 5, "dtype"),
                               ("k", 0, "NULL"), ("page_table", 0, "NULL"), ("valid_tokens", 0, "NULL"), ("k_scales", 0, "NULL"),
                               ("v_codes", 257, "aligned"), ("count", 1 << 30, "too many")):
        a = args()
        setattr(a, field, value)
        for call in (N.mx_append_tokens, N.mx_read_tokens):
            with pytest.raises(ValueError, match=text):
                call(a, 0)


def test_page_refusals():
    def seqs():
        a = N.SequencesArgs()
        a.num_seqs, a.rows_per_seq, a.table_width, a.page_size, a.num_pages, a.count = 4, 2, 9, 16, 50, 2
        a.page_table = a.valid_tokens = a.refs = a.seqs = a.parents = a.new_tokens = a.missing = 256
        return a
    need = N.sequences_workspace(seqs())
    for field, value, text in (("num_seqs", -1, "size"), ("rows_per_seq", 0, "size"), ("page_size", 0, "size"), ("count", -1, "size"),
                               ("num_pages", 1 << 31, "int32"), ("table_width", 1 << 28, "int32"), ("count", 1 << 26, "too many"),
                               ("seqs", 0, "NULL"), ("refs", 0, "NULL"), ("valid_tokens", 0, "NULL"), ("refs", 258, "aligned")):
        a = seqs()
        setattr(a, field, value)
        with pytest.raises(ValueError, match=text):
            N.sequences_workspace(a)
        with pytest.raises(ValueError, match=text):
            N.free_sequences(a, 0)
    for call, field in ((N.grow_sequences, "new_tokens"), (N.fork_sequences, "parents"), (N.grow_sequences, "missing")):
        a = seqs()
        setattr(a, field, 0)
        with pytest.raises(ValueError, match=field):
            call(a, 0, 256, need)
        with pytest.raises(ValueError, match="workspace"):
            call(seqs(), 0, 256, need - 1)
    a = seqs()
    a.num_arrays, a.arrays[0].base = 1, 256
    with pytest.raises(ValueError, match="row_bytes"):
        N.fork_sequences(a, 0, 256, need)
    c = N.CopyPagesArgs()
    c.num_pages, c.count, c.num_arrays = 5, 1, 25
    with pytest.raises(ValueError, match="num_arrays"):
        N.copy_pages(c, 0)
    c.num_arrays, c.arrays[0].row_bytes = 1, 16
    with pytest.raises(ValueError, match="NULL"):
        N.copy_pages(c, 0)
    p = N.CompactPagesArgs()
    p.num_rows, p.table_width, p.page_size, p.num_pages = 2, 3, 16, 10
    with pytest.raises(ValueError, match="NULL"):
        N.compact_pages_workspace(p)


def test_compaction_refusals():
    def args():
        p = N.CompactPagesArgs()
        p.num_rows, p.table_width, p.page_size, p.num_pages = 2, 3, 16, 10
        p.page_table, p.valid_tokens, p.refs, p.out_table, p.out_refs, p.page_map = 256, 512, 768, 1024, 1280, 1536
        return p
    assert N.compact_pages_workspace(args()) > 0
    for field, value, text in (("page_size", 0, "size"), ("num_pages", 1 << 31, "size"), ("out_table", 256, "another"),
                               ("out_refs", 768, "another"), ("page_map", 1280, "another"), ("refs", 0, "NULL"),
                               ("page_map", 1538, "aligned"), ("valid_tokens", 514, "aligned"), ("num_arrays", -1, "num_arrays")):
        a = args()
        setattr(a, field, value)
        with pytest.raises(ValueError, match=text):
            N.compact_pages_workspace(a)
    need = N.compact_pages_workspace(args())
    for ws, size in ((0, need), (256, need - 1), (260, need)):
        with pytest.raises(ValueError, match="workspace"):
            N.compact_pages(args(), 0, ws, size)


def test_a_scale_that_leaves_float32_in_base_2_is_refused():
    a = _attention_args()
    for value, fine in ((2.3e38, True), (-2.3e38, True), (3e38, False), (-3e38, False)):
        a.sm_scale = value
        if fine:
            N.mx_attention_workspace(a)
        else:
            with pytest.raises(ValueError, match="sm_scale"):
                N.mx_attention_workspace(a)


def test_host_tensors_are_refused():
    pools = ia.MxFp4Pools.empty(4, 64, "cpu")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    x = torch.zeros((1, 1, 2, 64))
    for call in (lambda: ia.append_mxfp4_tokens(x, x, pools, i32(1, 2, 3), i32(1, 2)),
                 lambda: ia.read_mxfp4_tokens(pools, i32(1, 2, 3), i32(1, 2), 1),
                 lambda: ia.mxfp4_paged_attention(x, pools, i32(1, 2, 3), i32(1, 2)),
                 lambda: ia.grow_sequences(i32(1, 2, 3), i32(1, 2), i32(4), [0], [1]),
                 lambda: ia.fork_sequences(i32(1, 2, 3), i32(1, 2), i32(4), [0], [0]),
                 lambda: ia.free_sequences(i32(1, 2, 3), i32(1, 2), i32(4), [0]),
                 lambda: ia.compact_pages(i32(1, 2, 3), i32(1, 2), i32(4)),
                 lambda: ia.copy_pages(pools, [0], [1])):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_shapes_and_types_are_checked():
    pools = ia.MxFp4Pools.empty(4, 64, "cpu")
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    assert mxfp4._check_cache(pools, i32(1, 2, 3), i32(1, 2), None, 1, 64) == (2, 3, 4)
    with pytest.raises(ValueError, match="page_table"):
        mxfp4._check_cache(pools, i32(2, 2, 3), i32(1, 2), None, 1, 64)
    with pytest.raises(ValueError, match="page_table"):
        mxfp4._check_cache(pools, i32(1, 2, 3).long(), i32(1, 2), None, 1, 64)
    with pytest.raises(ValueError, match="valid_tokens"):
        mxfp4._check_cache(pools, i32(1, 2, 3), i32(1, 3), None, 1, 64)
    with pytest.raises(ValueError, match="q_lens"):
        mxfp4._check_cache(pools, i32(1, 2, 3), i32(1, 2), i32(2), 1, 64)
    with pytest.raises(ValueError, match="k_codes"):
        mxfp4._check_cache(pools, i32(1, 2, 3), i32(1, 2), None, 1, 128)
    with pytest.raises(ValueError, match="head_dim"):
        mxfp4._check_cache(pools, i32(1, 2, 3), i32(1, 2), None, 1, 96)
    with pytest.raises(ValueError, match="contiguous"):
        mxfp4._check_cache(ia.MxFp4Pools(pools.k_codes.transpose(0, 0)[:, :, :], pools.k_scales, pools.v_codes.flip(0)[::2].repeat(2, 1, 1)
                                         .transpose(0, 1).contiguous().transpose(0, 1), pools.v_scales), i32(1, 2, 3), i32(1, 2), None, 1, 64)
    with pytest.raises(ValueError, match="head_dim"):
        ia.MxFp4Pools.empty(4, 80, "cpu")
    for t, v, r in ((i32(1, 2), i32(1, 2), i32(4)), (i32(1, 2, 3), i32(1, 3), i32(4)), (i32(1, 2, 3), i32(1, 2), i32(4, 1)),
                    (i32(1, 3, 2).transpose(1, 2), i32(1, 2), i32(4)), (i32(1, 0, 3), i32(1, 0), i32(4))):
        with pytest.raises(ValueError):
            page_sharing._check_state(t, v, r)
    with pytest.raises(ValueError, match="int32"):
        page_sharing._indices("seqs", torch.zeros(2, dtype=torch.int64), torch.device("cpu"))
    with pytest.raises(ValueError, match="int32"):
        page_sharing._indices("seqs", [2 ** 31], torch.device("cpu"))
    with pytest.raises(ValueError, match="entries"):
        page_sharing._indices("new_tokens", [1, 2], torch.device("cpu"), 3)
    a = N.CopyPagesArgs()
    with pytest.raises(ValueError, match="row for each"):
        page_sharing._fill_arrays(a, [torch.zeros(5, 2)], 4)
    page_sharing._fill_arrays(a, [torch.zeros(4, 2), torch.zeros(4, dtype=torch.uint8)], 4)
    assert (a.num_arrays, a.arrays[0].row_bytes, a.arrays[1].row_bytes) == (2, 8, 1)
    x = torch.zeros((4, 2))
    assert len(page_sharing._pool_tensors(ia.PagePools(k_fp16=x, v_fp16=x))) == 1


def test_the_oracles_number_format():
    """All sixteen codes, ties to the even code, saturation, the exponent's clamp, NaN blocks."""
    x = np.zeros((1, 64))
    x[0, :8] = [4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5]
    x[0, 8:16] = [-7.9, .26, .74, -1.26, 6.9, 3.51, 5.01, -.2]
    codes, scales = O.quantize(x)
    assert scales.tolist() == [[127, 104]]
    assert codes[0, :16].tolist() == [6, 0, 2, 2, 4, 4, 6, 6, 15, 1, 1, 11, 7, 6, 7, 8]
    assert np.array_equal(O.unpack(O.pack(codes)), codes)
    for value, byte in ((2.0 ** 20, 140), (2.0 ** -40, 104), (6.0, 127), (8.0, 128), (7.99, 127), (0.0, 104)):
        assert O.quantize(np.full((1, 32), value))[1].tolist() == [[byte]]
    y = np.ones((1, 32))
    y[0, 3] = np.inf
    codes, scales = O.quantize(y)
    assert scales.tolist() == [[255]] and not codes.any() and np.isnan(O.values(codes, scales)).all()
    assert float(np.abs(O.values(*O.quantize(np.full((1, 32), 1e9)))).max()) == 49152.0
