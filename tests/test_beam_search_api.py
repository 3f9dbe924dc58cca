"""The beam choice's oracle and its refusals, without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import intent_attention as ia
from intent_attention import _native as N
from oracle import beam_search as O


def test_oracle_by_hand():
    x = np.log(np.array([[[1.0, 2, 1], [4, 2, 2]]]))
    s, p, t = O.select(x, np.log(np.array([[0.5, 0.25]])), 5)
    # beam 0: .125 .25 .125, beam 1: .125 .0625 .0625; equal ones by number
    assert np.allclose(np.exp(s), [[.25, .125, .125, .125, .0625]])
    assert p.tolist() == [[0, 0, 0, 1, 1]] and t.tolist() == [[1, 0, 2, 0, 1]]


def test_oracle_beams_out_of_the_search():
    x = np.zeros((1, 4, 3))
    x[0, 1, 2] = np.nan
    x[0, 2] = -np.inf
    s, p, t = O.select(x, np.array([[-2.0, -1, -1, -np.inf]]), 6, np.array([[True, False, False, False]]), 1)
    assert s.tolist() == [[-2.0] + [-np.inf] * 5]
    assert p.tolist() == [[0, 0, 0, 1, 1, 1]] and t.tolist() == [[1, 0, 2, 0, 1, 2]]


def _args(**kw):
    a = N.BeamSelectArgs(batch=2, beams=4, vocab=1000, count=8, logits=4096, dtype=0, stride_b=4000, stride_k=1000, scores=8192,
                         end_token=5, out_scores=12288, out_parents=16384, out_tokens=20480)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "bad size"), (dict(beams=0), "bad size"), (dict(vocab=0), "bad size"), (dict(count=0), "bad size"),
    (dict(beams=257), "beams 257"), (dict(count=65), "count 65"), (dict(vocab=1, count=5), "candidates"),
    (dict(beams=256, vocab=1 << 23), "int32"), (dict(batch=1 << 30), "int32"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(finished=1, end_token=1000), "end_token"), (dict(finished=1, end_token=-1), "end_token"),
    (dict(logits=None), "NULL"), (dict(scores=None), "NULL"), (dict(out_tokens=None), "NULL"),
    (dict(logits=4097), "aligned"), (dict(dtype=1, logits=4098), "aligned"), (dict(out_parents=16386), "aligned")])
def test_abi_refuses(kw, text):
    with pytest.raises(ValueError, match=text):
        N.beam_select_workspace(_args(**kw))
    with pytest.raises(ValueError, match=text):
        N.beam_select(_args(**kw), 0, 1 << 20, 1 << 40)


def test_abi_workspace():
    need = N.beam_select_workspace(_args())
    for at, size in ((None, need), (1 << 20, need - 1), ((1 << 20) + 8, need)):
        with pytest.raises(ValueError, match="workspace"):
            N.beam_select(_args(), 0, at, size)
    assert N.beam_select_workspace(_args(batch=0)) == 0
    N.beam_select(_args(batch=0), 0, 0, 0)
    with pytest.raises(ValueError, match="NULL"):
        N.check(N.load().iak_beam_select(None, None, 0, None))
    with pytest.raises(ValueError, match="NULL"):
        N.check(N.load().iak_beam_select_workspace(ctypes.byref(_args()), None))


def test_python_refuses():
    x, s = torch.zeros(2, 3, 10), torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        ia.beam_select(x, s)
    for bad, kw, text in (((x[0], s), {}, "B, K, V"), ((x.double(), s), {}, "float16"), ((x, s[:1]), {}, "scores"),
                          ((x, s.half()), {}, "scores"), ((x, s), dict(finished=torch.zeros(2, 3)), "finished"),
                          ((x, s), dict(finished=torch.zeros(2, 3, dtype=torch.bool)), "end_token"),
                          ((x, s), dict(count=2 ** 31), "int32"), ((x, s), dict(end_token=2 ** 31), "int32")):
        with pytest.raises(ValueError, match=text):
            ia.beam_select(*bad, **kw)
