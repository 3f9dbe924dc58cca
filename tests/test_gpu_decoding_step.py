"""Prompts and steps of a beam search over a paged cache with all that takes part in them: room for the tokens, keys rotated
into their pages, attention over pages of two precisions, the choice over the vocabulary, the beams' tables put in its order.
Every step is compared with what the beams' own tokens give in float64."""
import numpy as np
import pytest

from oracle import beam_search, rotary
from test_gpu_chunk_attention import Case

pytestmark = pytest.mark.gpu

PS = 16


@pytest.mark.parametrize("D,Hq,Hkv,R", [(64, 4, 2, 64), (128, 4, 1, 32)])
def test_beams_over_pages(D, Hq, Hkv, R):
    import torch
    import intent_attention as ia
    B, K, V, W, NP, prompt, steps = 2, 3, 61, 6, 160, 21, 40
    S = B * K
    rng = np.random.default_rng(D)
    make = lambda *shape: rng.standard_normal(shape).astype(np.float16)  # noqa: E731
    embed_q, embed_k, embed_v = make(V, Hq, D), make(V, Hkv, D), make(V, Hkv, D)
    head = torch.from_numpy(rng.standard_normal((Hq * D, V)).astype(np.float32) * 0.5)
    inv_freq = (1.0 / 10000.0 ** (np.arange(R // 2) * 2.0 / R)).astype(np.float32)
    gpu = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731

    table = torch.full((S, Hkv, W), -1, dtype=torch.int32, device="cuda")
    valid = torch.zeros((S, Hkv), dtype=torch.int32, device="cuda")
    refs = torch.zeros(NP, dtype=torch.int32, device="cuda")
    tags = torch.full((NP, 1), 7, dtype=torch.int32, device="cuda")                # a page's tag goes with its content
    host = dict(k_fp16=np.zeros((NP, PS, D), np.float16), v_fp16=np.zeros((NP, PS, D), np.float16),
                k_int8=np.zeros((NP, PS, D), np.int8), v_int8=np.zeros((NP, PS, D), np.int8),
                k_int8_scale=np.ones(NP, np.float16), v_int8_scale=np.ones(NP, np.float16))
    pools = ia.PagePools(**{n: gpu(x) for n, x in host.items()})
    arrays = [pools.k_fp16, pools.v_fp16, pools.k_int8, pools.v_int8, pools.k_int8_scale, pools.v_int8_scale, tags]
    seqs = torch.arange(S, dtype=torch.int32, device="cuda")
    scores = torch.full((B, K), float("-inf"), device="cuda")
    scores[:, 0] = 0
    beams = [[[] for _ in range(K)] for _ in range(B)]
    for b in range(B):
        beams[b][0] = list(rng.integers(0, V, prompt))
    quantised = 0
    for step in range(steps):
        L = prompt if step == 0 else 1
        listed = seqs[::K] if step == 0 else seqs                                  # a request's first beam has the prompt
        room = torch.full((len(listed),), L, dtype=torch.int32, device="cuda")
        new = torch.empty(S, dtype=torch.int32, device="cuda")
        assert ia.grow_sequences(table, valid, refs, listed, room, arrays, granted=new).tolist() == [0]
        tokens = np.zeros((S, L), np.int64)
        for r in range(S):
            own = beams[r // K][r % K]
            if len(own):
                tokens[r] = own[-L:]
        q = gpu(embed_q[tokens])
        rotated = ia.append_rotated_tokens(gpu(embed_k[tokens]), gpu(embed_v[tokens]), pools, table, valid, gpu(inv_freq), q=q, q_lens=new,
                                           page_tags=tags.view(-1), fp16_tag=0)
        counts = (valid + PS - 1) // PS
        out = ia.paged_chunk_attention(rotated, pools, table, counts, tags.view(-1), valid_tokens=valid, q_lens=new, tag_map=[0, 1])
        # the attention of what the pages hold
        c = Case.__new__(Case)
        c.q_dtype, c.q, c.tags, c.q_lens = "float16", rotated, tags.view(-1).cpu().numpy(), new.cpu().numpy()
        c.table, c.valid, c.counts = table.cpu().numpy(), valid.cpu().numpy(), counts.cpu().numpy()
        c.host = {n: t.cpu().numpy() for n, t in pools.tensors().items()}
        c.check(out, tag_map=[0, 1])
        # which is what the beams' tokens are, rotated: turned in float32 and rounded once
        for r in range(S):
            own = np.array(beams[r // K][r % K], np.int64)
            n = len(own)
            assert c.valid[r].tolist() == [n] * Hkv
            at = np.tile(np.arange(n)[None, :, None], (1, 1, Hkv))
            want = rotary.rotate(embed_k[own][None], at, inv_freq, False)[0]
            far = rotary.reach(embed_k[own][None], inv_freq, False)[0]
            for h in range(Hkv):
                pages = c.table[r, h, :-(-n // PS)]
                plain = np.repeat(c.tags[pages] == 0, PS)[:n]
                k, v = (c.host[x][pages].reshape(-1, D)[:n] for x in ("k_fp16", "v_fp16"))
                off = np.abs(k.astype(np.float64) - want[:, h])[plain]
                assert (off <= (np.abs(want[:, h]) * 2.0 ** -11 + far[:, h] * 2.0 ** -20 + 2.0 ** -25)[plain]).all()
                assert np.array_equal(v[plain], embed_v[own][:, h][plain])
        # the choice
        last = np.maximum(c.q_lens - 1, 0)
        logits = (out[torch.arange(S), torch.from_numpy(last).cuda()].float().cpu().reshape(S, Hq * D) @ head).view(B, K, V)
        scores, parents, picked = ia.beam_select(logits.cuda(), scores if step else scores.clone())
        before = c_scores if step else np.where(np.arange(K) == 0, 0.0, -np.inf) * np.ones((B, 1))
        before = np.where(np.isnan(before), -np.inf, before)
        want = beam_search.select(logits.numpy(), before, K)
        assert np.array_equal(parents.cpu().numpy(), want[1]) and np.array_equal(picked.cpu().numpy(), want[2])
        c_scores = scores.cpu().numpy().astype(np.float64)
        assert ia.reorder_sequences(table, valid, refs, seqs, parents.flatten(), arrays).tolist() == [0]
        beams = [[beams[b][int(p) - b * K] + [int(t)] for p, t in zip(want[1][b], want[2][b])] for b in range(B)]
        used = table[table >= 0]
        assert torch.equal(torch.bincount(used, minlength=NP).int(), refs)
        # now and then the full pages become INT8 ones
        if step % 7 == 3:
            full = torch.unique(torch.cat([table[r, h, :int(valid[r, h]) // PS] for r in range(S) for h in range(Hkv)]))
            full = full[tags[full.long(), 0] == 0].long()
            for side in "kv":
                x = getattr(pools, side + "_fp16")[full].float()
                scale = (x.abs().amax((1, 2)) / 127).half()
                getattr(pools, side + "_int8")[full] = (x / scale.float()[:, None, None]).round().clamp(-127, 127).to(torch.int8)
                getattr(pools, side + "_int8_scale")[full] = scale
                getattr(pools, side + "_fp16")[full] = float("nan")                # which nobody reads any more
            tags[full] = 1
            quantised += len(full)
    assert quantised > 0
