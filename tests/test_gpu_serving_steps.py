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


def test_a_row_cut_back_into_a_shared_page_grows_apart():
    """Fork at a page's end, let tokens go into the shared page, grow and append: the sibling's tokens
    stay, the kept ones of the row come along; without pools the call is refused."""
    import torch
    import intent_attention as ia
    for cut, first, then in ((4, [1], [4]), (1, [0, 1], [3, 20]), (15, [1, 0], [1, 1]), (20, [1], [40])):
        s = Loop(3, 2, 6, 30, cut)
        assert s.step([0], [48])[0] == 0
        assert ia.fork_sequences(*s.state(), [0], [1], s.pools).item() == 0
        ia.free_sequences(*s.state(), [1], [cut])
        s.kept[1] = s.kept[0][:, :48 - cut]
        if len(first) == 2:                                # both owners cut back, both grown in one call
            ia.free_sequences(*s.state(), [0], [cut])
            s.kept[0] = s.kept[1]
        s.check()
        before = [t.clone() for t in (*s.state(), *s.pools.tensors().values())]
        assert s.step(first, then)[0] == -1                # no pools to copy in
        for t, b in zip((*s.state(), *s.pools.tensors().values()), before):
            assert torch.equal(t, b)
        assert s.step(first, [0] * len(first))[0] == 0     # no tokens, nothing to copy
        assert s.step(first, then, pools=s.pools)[0] == 0
        s.check()
        used = sum(2 * -(-x.shape[1] // 16) for x in s.kept if x is not None)
        assert int(s.refs.sum()) == used
        rows = s.table.flatten(0, 1).tolist()
        for page in range(30):                             # every entry counted where it is
            assert s.refs[page].item() == sum(r.count(page) for r in rows)


def test_copies_of_shared_pages_come_too_few():
    """A copy needs a free page like any other: one too few, nothing done; then the sibling leaves."""
    import torch
    import intent_attention as ia
    s = Loop(2, 1, 4, 3)
    assert s.step([0], [48])[0] == 0
    assert ia.fork_sequences(*s.state(), [0], [1], s.pools).item() == 0
    ia.free_sequences(*s.state(), [1], [5])
    s.kept[1] = s.kept[0][:, :43]
    before = [t.clone() for t in (*s.state(), *s.pools.tensors().values())]
    assert s.step([1], [2], pools=s.pools)[0] == 1
    for t, b in zip((*s.state(), *s.pools.tensors().values()), before):
        assert torch.equal(t, b)
    ia.free_sequences(*s.state(), [0])
    s.kept[0] = None
    assert s.step([1], [2])[0] == 0                        # the page is its own now: no pools needed
    s.check()


@pytest.mark.parametrize("B,R,W,NP", [(6, 1, 3, 30), (9, 3, 20, 1500), (40, 8, 9, 6000), (9, 2, 30, 40000)])
def test_growing_rows_with_shared_last_pages_follow_the_lists(B, R, W, NP):
    """Entries that any rows share, some counted by others, some no pages: grown with arrays and without."""
    from tests.test_gpu_page_sharing import State
    import intent_attention as ia
    s = State(B + W, B, R, W, NP, fill=0.7)
    rng = np.random.default_rng(B)
    done = copies = 0
    for it in range(10):
        for _ in range(B):                                 # rows that share what lies at the same entry
            b, c, h, g = (int(rng.integers(0, n)) for n in (B, B, R, R))
            n = min(s.host.used(b, h), s.host.used(c, g))
            if n:
                s.host.table[b][h][n - 1] = s.host.table[c][g][n - 1] if rng.random() < 0.8 else int(rng.choice([-1, NP]))
        counts = [0] * NP
        for b in range(B):
            for h in range(R):
                for e in range(s.host.used(b, h)):
                    if 0 <= s.host.table[b][h][e] < NP:
                        counts[s.host.table[b][h][e]] += 1
        for p in rng.choice(NP, 3, replace=False):
            counts[p] += 1
        s.host.refs = counts
        s.table.copy_(_t(s.host.table))
        s.refs.copy_(_t(counts))
        seqs = [int(x) for x in rng.permutation(B)[:max(1, B // 2)]]
        new = [int(x) for x in rng.integers(0, 25, len(seqs))]
        pools = it % 4 != 3
        want = s.host.grow(seqs, new, pools)
        copies += len(s.host.copied)
        got = ia.grow_sequences(s.table, s.valid, s.refs, _t(seqs), _t(new), s.pools if pools else None)
        assert got.item() == want
        done += want == 0
        s.check()
        drop = [int(x) for x in rng.integers(0, 30, B)]
        s.host.free(list(range(B)), drop)
        ia.free_sequences(s.table, s.valid, s.refs, list(range(B)), drop)
        s.check()
    assert done >= 3 and copies >= 3


def test_copies_of_shared_pages_replay():
    """Captured once: rows that share their last page, that do not, and a call that is refused."""
    import torch
    import intent_attention as ia
    from tests.test_gpu_page_sharing import State
    s = State(3, 6, 2, 12, 300, fill=0.5)
    seqs, new, short = _t([0, 1]), _t([5, 5]), torch.zeros(1, dtype=torch.int32, device=_dev())
    lens = torch.zeros(6, dtype=torch.int32, device=_dev())
    keep = [x.clone() for x in (s.table, s.valid, s.refs, *s.pools)]

    def step():
        ia.grow_sequences(s.table, s.valid, s.refs, seqs, new, s.pools, granted=lens, missing=short)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x, k in zip((s.table, s.valid, s.refs, *s.pools), keep):
        x.copy_(k)
    for a, n, shared in (([0, 1], [5, 6], True), ([2, 4], [1, 30], False), ([5, 5], [1, 1], True), ([1, 5], [9, 2], True)):
        if shared:
            for b in a:
                for h in range(2):
                    if s.host.valid[b][h] % 16:
                        s.host.refs[s.host.table[b][h][s.host.valid[b][h] // 16]] += 1
        s.refs.copy_(_t(s.host.refs))
        seqs.copy_(_t(a))
        new.copy_(_t(n))
        want = s.host.grow(a, n, True)
        graph.replay()
        torch.cuda.synchronize()
        assert short.item() == want
        assert lens.tolist() == [dict(zip(a, n)).get(b, 0) if want == 0 else 0 for b in range(6)]
        s.check()


def test_needs_that_pass_32_bits_are_counted():
    """1,024 rows of 2^21 entries each: 2^31 pages, more than there are; nothing is done."""
    import torch
    import intent_attention as ia
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of device memory")
    W, NP = 1 << 21, 1000
    table = torch.empty((1, 1024, W), dtype=torch.int32, device=_dev())    # not looked at
    table[0, :, 0] = 5
    valid, refs = torch.zeros((1, 1024), dtype=torch.int32, device=_dev()), torch.zeros(NP, dtype=torch.int32, device=_dev())
    lens = _t([7])
    for new, answer in ((16 * W, 2 ** 31 - 1 - NP), (16 * (W - 1), 1024 * (W - 1) - NP)):
        assert ia.grow_sequences(table, valid, refs, [0], [new], granted=lens).item() == answer
        assert lens.item() == 0 and not bool(valid.any()) and not bool(refs.any()) and bool((table[0, :, 0] == 5).all())


def test_calls_with_lists_do_not_wait():
    """Each call returns while 0.1 s of work queued before it still runs, and does what it should."""
    import torch
    import intent_attention as ia
    s = Loop(4, 2, 5, 30)
    x = torch.zeros((8192, 8192), dtype=torch.float16, device=_dev())
    y = torch.empty_like(x)

    def busy():
        for _ in range(100):
            torch.mm(x, x, out=y)
        e = torch.cuda.Event()
        e.record()
        return e

    for warm in (True, False):
        calls = (lambda: ia.grow_sequences(*s.state(), [0, 2], [20, 3]),
                 lambda: ia.fork_sequences(*s.state(), [0], [1], s.pools),
                 lambda: ia.free_sequences(*s.state(), [0, 2], [1, 3]),
                 lambda: ia.copy_pages(s.pools, [1], [29]),
                 lambda: ia.free_sequences(*s.state(), [0, 1]))
        for i, call in enumerate(calls):
            done = None if warm else busy()
            call()
            assert warm or not done.query(), i
            torch.cuda.synchronize()
        assert int(s.refs.sum()) == 0 and not bool(s.valid.any())


def test_lists_are_refused_under_capture():
    """A replay could not read them again."""
    import torch
    import intent_attention as ia
    s = Loop(4, 2, 5, 30)
    seqs, new = _t([0, 2]), _t([20, 3])
    ia.grow_sequences(*s.state(), seqs, new)
    torch.cuda.synchronize()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        torch.zeros(1, device=_dev())
        with pytest.raises(ValueError, match="capture"):
            ia.grow_sequences(*s.state(), [0, 2], [20, 3])
        with pytest.raises(ValueError, match="capture"):
            ia.grow_sequences(*s.state(), seqs, [20, 3])
    torch.cuda.synchronize()
    assert s.valid.tolist() == [[20, 20], [0, 0], [3, 3], [0, 0]]


@pytest.mark.parametrize("D", [64, 128])
def test_pools_of_several_precisions_move_with_their_tags(D):
    """The decode over pages that were compacted, forked and grown apart with their scales and tags:
    the same bits as before, for the children as for their parents."""
    import torch
    import intent_attention as ia
    from tests._pools import random_case, to_device_pools
    B, Hkv, W, NP = 4, 2, 9, 120
    q, host, _, _, tags = random_case(D, B, 8, Hkv, D, NP, W, {"FP16": .3, "FP8": .2, "INT8": .2, "INT4": .2, "INT4_RESIDUAL": .1})
    rng = np.random.default_rng(D)
    pools, tags, q = to_device_pools(host, _dev()), _t(tags), torch.from_numpy(q).to(_dev())
    lens = [130, 0, 75, 0]
    table, refs, pages = np.full((B, Hkv, W), -1), np.zeros(NP, int), iter(rng.permutation(NP))
    for b, h in np.ndindex(B, Hkv):
        for e in range(-(-lens[b] // 16)):
            table[b, h, e] = next(pages)
            refs[table[b, h, e]] = 1
    table, refs, valid = _t(table), _t(refs), _t([[n] * Hkv for n in lens])
    every = [*pools.tensors().values(), tags]

    def decode():
        counts = (valid + 15) // 16
        return ia.paged_decode(q, pools, table, counts.int(), tags, valid_tokens=valid)

    q[1], q[3] = q[0], q[2]
    before = decode()
    table, refs, page_map = ia.compact_pages(table, valid, refs, every)
    assert int(refs[:int((refs > 0).sum())].min()) > 0
    assert torch.equal(decode(), before)
    assert ia.fork_sequences(table, valid, refs, [0, 2], [1, 3], every).item() == 0
    out = decode()
    assert torch.equal(out[[0, 2]], before[[0, 2]]) and torch.equal(out[[1, 3]], before[[0, 2]])
    ia.free_sequences(table, valid, refs, [1, 3], [20, 20])            # to inside pages that are shared
    cut = decode()
    assert ia.grow_sequences(table, valid, refs, [1, 3], [1, 1], every).item() == 0
    valid -= _t([[0], [1], [0], [1]])                                  # no token written: look at the copies alone
    assert torch.equal(decode(), cut)
    assert not torch.equal(table[1, :, 6], table[0, :, 6])             # 110 tokens: the seventh page is its own
