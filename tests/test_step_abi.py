"""The argument blocks of the decoding step's operators as ctypes has them against the header, by gcc. No GPU."""
import ctypes
import os
import subprocess
import tempfile

import pytest

from intent_attention import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("cname,pyname", [("iak_paged_chunk_args", "PagedChunkArgs"), ("iak_rotary_append_args", "RotaryAppendArgs"),
                                          ("iak_beam_select_args", "BeamSelectArgs")])
def test_argument_blocks_match_the_header(cname, pyname):
    S = getattr(N, pyname)
    fields = [f[0] for f in S._fields_]
    prog = ['#include <stdio.h>', '#include <stddef.h>', '#include "iak.h"', 'int main(void){',
            f'printf("size %zu\\n", sizeof({cname}));']
    prog += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(c, "w").write("\n".join(prog))
        subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = dict(line.split() for line in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["size"]) == ctypes.sizeof(S)
    for f in fields:
        assert int(got[f]) == getattr(S, f).offset, f


def test_more_requests_than_a_launch_has_room_for():
    a = N.BeamSelectArgs()
    a.beams, a.vocab, a.count = 1, 8, 1
    a.logits = a.scores = a.out_scores = a.out_parents = a.out_tokens = 1 << 20   # not looked at
    a.stride_b = a.stride_k = 8
    a.batch = 0x7FFFFF
    assert N.beam_select_workspace(a) > 0
    a.batch = 0x800000
    with pytest.raises(ValueError, match="too many requests"):
        N.beam_select_workspace(a)
