"""Steps of a serving loop whose page calls cannot be done or meet shared pages, queued without a
look at the answer: what the cache holds must stay what was written."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D = 64


def _dev():
    import torch
    return torch.device("cuda:0")


def _t(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=_dev())


class Loop:
    """A 4-bit cache of B slots, its page state, and every sequence's tokens as they were read back
    when they were written."""

    def __init__(self, B, Hkv, W, NP, seed=0):
        import torch
        import intent_attention as ia
        self.B, self.Hkv = B, Hkv
        self.gen = torch.Generator(device=_dev()).manual_seed(seed)
        self.pools = ia.MxFp4Pools.empty(NP, D, _dev())
        self.table = torch.full((B, Hkv, W), -1, dtype=torch.int32, device=_dev())
        self.valid = torch.zeros((B, Hkv), dtype=torch.int32, device=_dev())
        self.refs = torch.zeros(NP, dtype=torch.int32, device=_dev())
        self.lens = torch.full((B,), 77, dtype=torch.int32, device=_dev())
        self.kept = [None] * B

    def state(self):
        return self.table, self.valid, self.refs

    def tokens(self, L):
        import torch
        return (torch.randn((self.B, L, self.Hkv, D), generator=self.gen, device=_dev()) for _ in range(2))

    def read(self, b, n):
        import torch
        import intent_attention as ia
        lens = torch.zeros_like(self.lens)
        lens[b] = n
        k, v = ia.read_mxfp4_tokens(self.pools, self.table, self.valid, n, q_lens=lens)
        return torch.stack((k[b], v[b]))

    def step(self, seqs, new, **kw):
        """Grow, append, attend, with nothing read in between; (answer, attention's output)."""
        import torch
        import intent_attention as ia
        short = ia.grow_sequences(*self.state(), seqs, new, granted=self.lens, **kw)
        L = max(1, max(new, default=1))
        k, v = self.tokens(L)
        ia.append_mxfp4_tokens(k, v, self.pools, self.table, self.valid, q_lens=self.lens)
        q = torch.randn((self.B, L, self.Hkv, D), generator=self.gen, device=_dev()).half()
        out = ia.mxfp4_paged_attention(q, self.pools, self.table, self.valid, q_lens=self.lens)
        answer = short.item()
        if answer == 0:
            for b, n in zip(seqs, new):
                if n:
                    fresh = self.read(b, n)
                    self.kept[b] = fresh if self.kept[b] is None else torch.cat((self.kept[b], fresh), 1)
        return answer, out

    def check(self):
        import torch
        for b in range(self.B):
            n = 0 if self.kept[b] is None else self.kept[b].shape[1]
            assert self.valid[b].tolist() == [n] * self.Hkv
            if n:
                assert torch.equal(self.read(b, n), self.kept[b]), b


@pytest.mark.parametrize("seqs,new,answer", [([0, 1], [2, 40], 4), ([1, 0, 2], [17, 1, 40], 6), ([0, 0], [1, 1], -1),
                                             ([0, 4], [3, 3], -1), ([0, 1], [5, -1], -1), ([2], [16 * 6], -1)])
def test_a_step_without_room_leaves_the_cache(seqs, new, answer):
    """Too few pages, or a refused call: the append and the attention behind it find no new tokens."""
    import torch
    s = Loop(4, 2, 5, 14)                                  # 14 pages: 2 rows of 30, 20 and 33 tokens fill them
    assert s.step([0, 1, 2], [30, 20, 33])[0] == 0
    assert s.lens.tolist() == [30, 20, 33, 0]
    before = [t.clone() for t in (*s.state(), *s.pools.tensors().values())]
    got, out = s.step(seqs, new)
    assert got == answer
    assert s.lens.tolist() == [0, 0, 0, 0] and bool((out == 0).all())
    for t, b in zip((*s.state(), *s.pools.tensors().values()), before):
        assert torch.equal(t, b)
    assert s.step([2, 0], [1, 2])[0] == 0                  # a step that has room goes on from there
    assert s.lens.tolist() == [2, 0, 1, 0]
    s.check()


def test_granted_tokens_of_a_captured_step():
    """A step captured once, replayed until the pages run out, and after that."""
    import torch
    import intent_attention as ia
    s = Loop(3, 1, 4, 7)
    seqs, new = _t([0, 1, 2]), _t([1, 1, 1])
    k, v = (x.clone() for x in s.tokens(20))
    q = torch.randn((3, 20, 1, D), device=_dev()).half()
    short = torch.zeros(1, dtype=torch.int32, device=_dev())

    def step():
        ia.grow_sequences(*s.state(), seqs, new, granted=s.lens, missing=short)
        ia.append_mxfp4_tokens(k, v, s.pools, s.table, s.valid, q_lens=s.lens)
        return ia.mxfp4_paged_attention(q, s.pools, s.table, s.valid, q_lens=s.lens)

    keep = [t.clone() for t in (*s.state(), *s.pools.tensors().values())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t, x in zip((*s.state(), *s.pools.tensors().values()), keep):
        t.copy_(x)
    answers = []
    for n in ([20, 15, 16], [12, 1, 1], [1, 1, 0], [0, 16, 0], [2, 1, 1]):      # 4 pages, 5, 7, one too few, none needed
        new.copy_(_t(n))
        for x in (k, v):
            x.copy_(torch.randn(x.shape, generator=s.gen, device=_dev()))
        before = [t.clone() for t in (*s.state(), *s.pools.tensors().values())]
        graph.replay()
        torch.cuda.synchronize()
        answers.append(short.item())
        assert s.lens.tolist() == (n if answers[-1] == 0 else [0, 0, 0])
        if answers[-1]:
            assert bool((out == 0).all())
            for t, x in zip((*s.state(), *s.pools.tensors().values()), before):
                assert torch.equal(t, x)
        else:
            for b, m in enumerate(n):
                if m:
                    fresh = s.read(b, m)
                    s.kept[b] = fresh if s.kept[b] is None else torch.cat((s.kept[b], fresh), 1)
        s.check()
    assert answers == [0, 0, 0, 1, 0]


def test_granted_is_checked():
    import torch
    import intent_attention as ia
    s = Loop(3, 1, 4, 7)
    for bad in (torch.zeros(2, dtype=torch.int32, device=_dev()), torch.zeros(3, device=_dev()),
                torch.zeros(3, dtype=torch.int32), torch.zeros((3, 2), dtype=torch.int32, device=_dev())[:, 0]):
        with pytest.raises(ValueError, match="granted"):
            ia.grow_sequences(*s.state(), [0], [1], granted=bad)
    lens = _t([1, 2, 3])
    for call in (lambda: ia.grow_sequences(*s.state(), [0, 1, 2], lens, granted=lens),
                 lambda: ia.grow_sequences(*s.state(), lens, [1, 1, 1], granted=lens),
                 lambda: ia.grow_sequences(*s.state(), [0], [1], granted=s.valid.view(-1)),
                 lambda: ia.grow_sequences(*s.state(), [0], [1], granted=s.refs[3:6]),
                 lambda: ia.grow_sequences(*s.state(), [0], [1], granted=s.table.view(-1)[5:8])):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    assert ia.grow_sequences(*s.state(), [], [], granted=lens).item() == 0
    assert lens.tolist() == [0, 0, 0] and int(s.refs.sum()) == 0
