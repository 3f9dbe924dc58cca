"""What is measured of the operators around a generation step over the paged caches: the calls and their plain forms.

K and V lie in pages of 16 tokens of one KV head, listed by page tables [sequences, KV heads, entries];
a page is float16 or quantised (FP8, INT8, INT4, INT4 with a residual), by its tag, or its row is a 4-bit cache's.

  rotate   the newest tokens' keys turned by their positions and written, with their values, into
           their sequences' pages; the queries turned along
  attend   attention of several new tokens per sequence (drafts, prompt chunks) over pages of mixed precision
  choose   a beam search's choice: the best continuations of each request's beams over the vocabulary
  reorder  the beams' page tables put in the order of that choice

``listed()`` holds the fixed cases, ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a
program has in hand, ``run`` is one pass, ``exact`` the same outputs in 64 bits, written apart.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

PS = 16                                  # tokens per page
BLOCK = 32                               # channels per scale of the 4-bit cache
FP16, INT8, SKIP, FP8, INT4, INT4_RESIDUAL = range(6)
_DTYPE = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_SIZE = {"float16": 2, "bfloat16": 2, "float32": 4}
_PAGE_BYTES = {FP16: 2.0, INT8: 1.0, FP8: 1.0, INT4: 0.5, INT4_RESIDUAL: 1.0, SKIP: 0.0}
# shares of the old pages in each precision
_MIXES = {"fp16": {FP16: 1.0}, "int8": {INT8: 1.0}, "fp8": {FP8: 1.0},
          "mixed": {FP16: 0.3, FP8: 0.25, INT8: 0.2, INT4: 0.15, INT4_RESIDUAL: 0.08, SKIP: 0.02},
          "low": {INT4: 0.5, INT4_RESIDUAL: 0.4, FP16: 0.1}}


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "intent-attention-kernel_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import intent_attention
    return intent_attention


def listed():
    return [
        # the new token of each of 64 sequences in a decode step, far into their contexts
        dict(name="rotate_step", kind="rotate", B=64, L=1, Hq=32, Hkv=8, D=128, R=128, dtype="bfloat16", start=60000,
             ragged=True, interleaved=False, cache="fp16"),
        # the prompts of eight sequences, ragged, written in one call
        dict(name="rotate_prompts", kind="rotate", B=8, L=4001, Hq=32, Hkv=8, D=128, R=128, dtype="float16", start=0,
             ragged=True, interleaved=False, cache="fp16"),
        # prompt chunks into the 4-bit cache, half of each head turned, in 32 bits
        dict(name="rotate_packed", kind="rotate", B=5, L=509, Hq=16, Hkv=4, D=64, R=32, dtype="float32", start=3000,
             ragged=True, interleaved=True, cache="mxfp4"),
        # the smallest step: three drafted tokens of one sequence of 500 tokens, heads of 64
        dict(name="draft_small", kind="attend", B=1, L=3, Hq=8, Hkv=8, D=64, T=500, dtype="float16", mix="fp16", scales="float16",
             ragged=False, causal=True),
        # four drafted tokens of 16 sequences over up to 16k selected tokens of mixed precision
        dict(name="draft_mixed", kind="attend", B=16, L=4, Hq=32, Hkv=8, D=128, T=16384, dtype="bfloat16", mix="mixed",
             scales="float16", ragged=True, causal=True),
        # ragged prompt chunks over a cache of mixed precision, heads of 64
        dict(name="chunk_ragged", kind="attend", B=5, L=509, Hq=16, Hkv=4, D=64, T=4000, dtype="bfloat16", mix="mixed",
             scales="float32", ragged=True, causal=True),
        # the last 2k tokens of an 8k prompt over float16 pages
        dict(name="chunk_long", kind="attend", B=1, L=2048, Hq=32, Hkv=8, D=128, T=8192, dtype="float16", mix="fp16",
             scales="float16", ragged=False, causal=True),
        # the largest product: 2k new tokens of two sequences over 16k tokens of mixed precision
        dict(name="chunk_mixed", kind="attend", B=2, L=2048, Hq=32, Hkv=8, D=128, T=16384, dtype="float16", mix="mixed",
             scales="float32", ragged=False, causal=True),
        # one step of two requests of four beams each
        dict(name="choose_small", kind="choose", B=2, K=4, V=32000, dtype="float32", count=4, finished=0.0, banned=0.0),
        # 64 requests of eight beams, twice as many candidates as beams, some beams at their end, some tokens not allowed
        dict(name="choose_large", kind="choose", B=64, K=8, V=131072, dtype="bfloat16", count=16, finished=0.1, banned=0.05),
        # the tables of two requests of four beams
        dict(name="reorder_small", kind="reorder", B=2, K=4, Hkv=4, D=64, W=40, spare=256, share=0.8),
        # 64 requests of four beams with long rows
        dict(name="reorder_large", kind="reorder", B=64, K=4, Hkv=8, D=128, W=200, spare=8192, share=0.8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "attend", "attend", "attend", "attend", "choose", "choose", "reorder"])
    D = rng.choice([64, 128])
    if kind == "rotate":
        L = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 4001)])
        Hq, Hkv = rng.choice([(8, 8), (16, 4), (20, 4), (32, 8), (28, 4), (12, 6), (32, 2), (24, 1)])
        return dict(kind=kind, B=_log(rng, 1, 64 if L < 512 else 8), L=L, Hq=Hq, Hkv=Hkv, D=D,
                    R=rng.choice([D, D, D // 2, 16, D - 16]), dtype=rng.choice(sorted(_DTYPE)), start=_log(rng, 1, 60000),
                    ragged=rng.random() < 0.6, interleaved=rng.random() < 0.4, cache=rng.choice(["fp16", "fp16", "mxfp4"]))
    if kind == "attend":
        Hq, Hkv = rng.choice([(8, 8), (16, 4), (20, 4), (32, 8), (28, 4), (12, 6), (32, 2), (24, 1)])
        L = rng.choice([1, rng.randrange(2, 9), rng.randrange(2, 9), _log(rng, 9, 512), _log(rng, 64, 2048)])
        B = _log(rng, 1, 16 if L < 9 else 8)
        # at most the listed cases' products and pages
        most = max(L, min(16384, int(2.4e11 / (B * Hq * D * L)), int(2.6e8 / (B * Hkv * D))))
        return dict(kind=kind, B=B, L=L, Hq=Hq, Hkv=Hkv, D=D, T=_log(rng, L, most),
                    dtype=rng.choice(["float16", "bfloat16", "float16", "bfloat16", "float32"]),
                    mix=rng.choice(["fp16", "int8", "fp8", "mixed", "mixed", "low"]), scales=rng.choice(["float16", "float32"]),
                    ragged=rng.random() < 0.6, causal=rng.random() < 0.85)
    if kind == "choose":
        K, V = rng.randrange(1, 17), _log(rng, 500, 131072)
        return dict(kind=kind, B=_log(rng, 1, max(1, min(64, int(6.7e7 / (K * V))))), K=K, V=V, dtype=rng.choice(sorted(_DTYPE)),
                    count=rng.choice([1, K, 2 * K]), finished=rng.choice([0.0, 0.2]), banned=rng.choice([0.0, 0.3]))
    return dict(kind=kind, B=_log(rng, 1, 64), K=rng.randrange(2, 5), Hkv=rng.choice([1, 2, 4, 8]), D=D, W=_log(rng, 4, 200),
                spare=_log(rng, 2100, 8192), share=rng.uniform(0.0, 1.0))


# --------------------------------------------------------------------------- #
# Inputs, from the seed alone
# --------------------------------------------------------------------------- #

def _gens(seed):
    return (torch.Generator(device="cuda").manual_seed(seed * 7919 + 23), torch.Generator().manual_seed(seed * 6151 + 17))


def _tokens(g, shape, dtype):
    """Keys or values: normal, with channels of different size."""
    size = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda") * size).to(dtype)


def _lengths(c, hg, B, least, most):
    if not c["ragged"]:
        return torch.full((B,), most, dtype=torch.int32)
    lens = torch.randint(max(least, most // 3), most + 1, (B,), generator=hg, dtype=torch.int32)
    lens[0] = most
    return lens


def _table(hg, lens, Hkv, W, NP):
    """Distinct random pages for the tokens of every row; entries past them are -1."""
    B = lens.shape[0]
    table = torch.randperm(NP, generator=hg)[:B * Hkv * W].view(B, Hkv, W).to(torch.int32)
    used = torch.arange(W) < ((lens + PS - 1) // PS).view(B, 1, 1)
    return torch.where(used, table, -1).cuda()


def _prepare_rotate(c, seed):
    g, hg = _gens(seed)
    B, L, Hq, Hkv, D, R = (c[n] for n in ("B", "L", "Hq", "Hkv", "D", "R"))
    new = _lengths(c, hg, B, 1, L)
    old = torch.randint(c["start"] // 2, c["start"] + 1, (B,), generator=hg, dtype=torch.int32)
    # far positions over a window of pages: what the row still lists ends at the newest token
    kept = torch.minimum(old, torch.randint(0, 2000, (B,), generator=hg, dtype=torch.int32))
    lens = kept + new
    W = (min(c["start"], 2000) + L + PS - 1) // PS
    NP = B * Hkv * W + 64
    dtype = _DTYPE[c["dtype"]]
    inv_freq = (10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2))).float().cuda()
    state = dict(kind="rotate", q=_tokens(g, (B, L, Hq, D), dtype), k=_tokens(g, (B, L, Hkv, D), dtype),
                 v=_tokens(g, (B, L, Hkv, D), dtype), new=new.cuda(), table=_table(hg, lens, Hkv, W, NP), count=L,
                 valid=lens.view(B, 1).expand(B, Hkv).contiguous().cuda(), inv_freq=inv_freq, interleaved=c["interleaved"],
                 positions=(old.view(B, 1) + torch.arange(L, dtype=torch.int32)).cuda(), cache=c["cache"])
    if c["cache"] == "fp16":
        state["pools"] = dict(k_fp16=torch.zeros((NP, PS, D), dtype=torch.float16, device="cuda"),
                              v_fp16=torch.zeros((NP, PS, D), dtype=torch.float16, device="cuda"))
    else:
        codes, scales = (NP, PS, D // 2), (NP, PS, D // BLOCK)
        state["pools"] = {n: torch.zeros(s, dtype=torch.uint8, device="cuda")
                          for n, s in (("k_codes", codes), ("k_scales", scales), ("v_codes", codes), ("v_scales", scales))}
    return state


def _quantised(x, scale_dtype):
    """float32 pages [U, 16, D] in every precision."""
    U, _, D = x.shape
    most = x.abs().amax((1, 2))
    got = {"fp16": x.half()}
    s8 = (most / 127).to(scale_dtype)
    got["int8"] = (x / s8.float().view(-1, 1, 1)).round().clamp(-127, 127).to(torch.int8)
    got["int8_scale"] = s8
    sf = (most / 448).to(scale_dtype)
    got["fp8"] = (x / sf.float().view(-1, 1, 1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    got["fp8_scale"] = sf
    groups = x.view(U, PS, D // 32, 32)
    s4 = (groups.abs().amax((1, 3)) / 7).to(scale_dtype)
    code = (groups / s4.float().view(U, 1, -1, 1)).round().clamp(-7, 7).view(U, PS, D).to(torch.int32) + 8
    got["int4"] = (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)
    got["int4_scale"] = s4
    sb = most / 7
    base = (x / sb.view(-1, 1, 1)).round().clamp(-7, 7)
    rest = x - base * sb.view(-1, 1, 1)
    sr = rest.abs().amax((1, 2)) / 7
    resid = (rest / sr.view(-1, 1, 1)).round().clamp(-7, 7)
    got["int4r"] = ((base.to(torch.int32) + 8) | ((resid.to(torch.int32) + 8) << 4)).to(torch.uint8)
    got["int4r_scale"] = torch.stack((sb, sr), 1)
    return got


def _prepare_attend(c, seed):
    g, hg = _gens(seed)
    B, L, Hq, Hkv, D, T = (c[n] for n in ("B", "L", "Hq", "Hkv", "D", "T"))
    new = _lengths(c, hg, B, 1, L)
    lens = torch.maximum(_lengths(c, hg, B, 1, T), new)
    W = (T + PS - 1) // PS
    NP = B * Hkv * W + 64
    table = _table(hg, lens, Hkv, W, NP)
    mix = _MIXES[c["mix"]]
    kinds = torch.tensor(list(mix), dtype=torch.int32)
    tags = kinds[torch.multinomial(torch.tensor(list(mix.values())), NP, replacement=True, generator=hg)].cuda()
    # pages that hold new tokens are float16: they are quantised once they are full and old
    count = (lens + PS - 1) // PS
    fresh = torch.arange(W) >= ((lens - new) // PS).view(B, 1, 1)
    fresh = (fresh & (torch.arange(W) < count.view(B, 1, 1))).expand(B, Hkv, W).cuda()
    tags[table[fresh].long()] = FP16
    present = set(mix) | {FP16}
    pools = {}
    for side in "kv":
        pages = _quantised(_tokens(g, (min(NP, 4096), PS, D), torch.float32), _DTYPE[c["scales"]])
        pick = torch.randint(0, min(NP, 4096), (NP,), generator=g, device="cuda")
        for tag, name in ((FP16, "fp16"), (INT8, "int8"), (FP8, "fp8"), (INT4, "int4"), (INT4_RESIDUAL, "int4r")):
            if tag in present:
                for n in (name, name + "_scale"):
                    if n in pages:
                        pools[f"{side}_{n}"] = pages[n][pick]
    q = (2 * torch.randn((B, L, Hq, D), generator=g, device="cuda")).to(_DTYPE[c["dtype"]])
    state = dict(kind="attend", q=q, new=new.cuda(), table=table, tags=tags, causal=c["causal"], pools=pools,
                 counts=count.view(B, 1).expand(B, Hkv).contiguous().cuda(),
                 valid=lens.view(B, 1).expand(B, Hkv).contiguous().cuda())
    if own:
        # the plan that a serving program keeps for a batch: arguments checked once, workspace held
        ia = _package()
        state["plan"] = ia.make_chunk_plan(q, ia.PagePools(**pools), table, state["counts"], tags, valid_tokens=state["valid"],
                                           q_lens=state["new"], causal=c["causal"])
    return state


def _prepare_choose(c, seed):
    g, hg = _gens(seed)
    B, K, V = c["B"], c["K"], c["V"]
    logits = torch.randn((B, K, V), generator=g, device="cuda").mul_(3)
    # a few likely tokens
    likely = torch.randint(0, V, (B, K, 8), generator=g, device="cuda")
    logits.scatter_add_(2, likely, 6 + 4 * torch.rand((B, K, 8), generator=g, device="cuda"))
    logits = logits.to(_DTYPE[c["dtype"]])
    if c["banned"]:
        logits.masked_fill_(torch.rand((1, 1, V), generator=g, device="cuda") < c["banned"], float("-inf"))
    scores = -30 + 4 * torch.randn((B, K), generator=g, device="cuda")
    return dict(kind="choose", logits=logits, scores=scores, count=min(c["count"], K * V), end=V // 3,
                finished=(torch.rand((B, K), generator=hg) < c["finished"]).cuda() if c["finished"] else None)


def _prepare_reorder(c, seed):
    g, hg = _gens(seed)
    B, K, Hkv, D, W = c["B"], c["K"], c["Hkv"], c["D"], c["W"]
    S = B * K
    NP = S * Hkv * W + c["spare"]
    lens = torch.randint(max(1, PS * W // 2), PS * W + 1, (B,), generator=hg, dtype=torch.int32).repeat_interleave(K)
    table = torch.randperm(NP, generator=hg)[:S * Hkv * W].view(S, Hkv, W).to(torch.int32)
    count = (lens + PS - 1) // PS
    # a request's beams share the first part of their pages
    shared = torch.arange(W) < ((count - 1) * c["share"]).int().view(S, 1, 1)
    table = torch.where(shared, table.view(B, K, Hkv, W)[:, :1].expand(B, K, Hkv, W).reshape(S, Hkv, W), table)
    used = (torch.arange(W) < count.view(S, 1, 1)).expand(S, Hkv, W)
    table = torch.where(used, table, -1)
    refs = torch.zeros(NP, dtype=torch.int32)
    refs.index_add_(0, table[used].long(), torch.ones(int(used.sum()), dtype=torch.int32))
    parents = torch.arange(B).view(B, 1) * K + torch.randint(0, K, (B, K), generator=hg)
    return dict(kind="reorder", table=table.cuda(), refs=refs.cuda(), valid=lens.view(S, 1).expand(S, Hkv).contiguous().cuda(),
                seqs=torch.arange(S, dtype=torch.int32).cuda(), parents=parents.flatten().to(torch.int32).cuda(),
                k=torch.randn((NP, PS, D), generator=g, device="cuda").half(),
                v=torch.randn((NP, PS, D), generator=g, device="cuda").half())


def prepare(case, seed):
    return {"rotate": _prepare_rotate, "attend": _prepare_attend, "choose": _prepare_choose,
            "reorder": _prepare_reorder}[case["kind"]](case, seed)


# --------------------------------------------------------------------------- #
# One pass, in the plain form
# --------------------------------------------------------------------------- #

def _turned(x, positions, inv_freq, interleaved, real):
    """x [B, L, H, D] turned by its positions [B, L], in `real`; the angles in 64 bits."""
    half = inv_freq.shape[0]
    angle = (positions.double().unsqueeze(-1) * inv_freq.double()).unsqueeze(2)
    cos, sin = angle.cos().to(real), angle.sin().to(real)
    x = x.to(real)
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if interleaved else (turn[..., :half], turn[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turn, rest), -1)


def _newest(s):
    """(page, offset, exists) [B, count, Hkv] of the newest tokens of every row."""
    table, valid, new = s["table"], s["valid"], s["new"]
    i = torch.arange(s["count"], device=table.device).view(1, -1, 1)
    pos = (valid - new.unsqueeze(1)).unsqueeze(1) + i
    there = (i < new.view(-1, 1, 1)).expand_as(pos)
    entry = (pos // PS).clamp(0, table.shape[2] - 1)
    return torch.gather(table.transpose(1, 2), 1, entry.long()).long(), (pos % PS).long(), there


def _block_exponents(x):
    """float64 [..., D] in blocks, and their scales' exponents: 4-bit codes are of x / 2^e."""
    blocks = x.unflatten(-1, (-1, BLOCK))
    _, e = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    return blocks, torch.where((blocks == 0).all(-1, keepdim=True), -23, (e - 3).clamp(-23, 13))


def _codes(x):
    """4-bit code bytes [..., D/2] and scale bytes [..., D/32] of float64 values."""
    blocks, e = _block_exponents(x)
    y = torch.ldexp(blocks, -e)
    a = y.abs()
    code = torch.where(a < 2, torch.round(a * 2).clamp(max=4.0),
                       torch.where(a < 4, torch.round(a) + 2, torch.round(a * 0.5) + 4).clamp(max=7.0)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e.squeeze(-1) + 127).to(torch.uint8)


def _code_values(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    v = torch.where(both >= 8, -1.0, 1.0) * table[both & 7]
    return torch.ldexp(v.unflatten(-1, (-1, BLOCK)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _rotate_plain(s):
    page, off, there = _newest(s)
    mine = torch.arange(s["count"], device="cuda") < s["new"].unsqueeze(1)
    turn = (s["positions"], s["inv_freq"], s["interleaved"])
    q = _turned(s["q"], *turn, torch.float32).to(s["q"].dtype)
    q.masked_fill_(~mine.view(*mine.shape, 1, 1), 0)
    pools = s["pools"]
    if s["cache"] == "fp16":
        pools["k_fp16"][page[there], off[there]] = _turned(s["k"], *turn, torch.float32).half()[there]
        pools["v_fp16"][page[there], off[there]] = s["v"].half()[there]
        return q, pools["k_fp16"], pools["v_fp16"]
    got = [q]
    # a value next to a code's border is the border's other side in 32 bits
    for side, x in (("k", _turned(s["k"], *turn, torch.float64)), ("v", s["v"].double())):
        c, e = _codes(x)
        codes, scales = pools[side + "_codes"], pools[side + "_scales"]
        codes[page[there], off[there]], scales[page[there], off[there]] = c[there], e[there]
        got.append(_code_values(codes[page, off], scales[page, off]).masked_fill(~there.unsqueeze(-1), 0.0).half())
    return tuple(got)


def _page_values(pools, side, ids, tags):
    """float32 [n, 16, D] of pages `ids` in the precisions `tags`, zeros where skipped."""
    out = torch.zeros((ids.shape[0], PS, pools["k_fp16"].shape[2]), device=ids.device)
    for tag, name in ((FP16, "fp16"), (INT8, "int8"), (FP8, "fp8"), (INT4, "int4"), (INT4_RESIDUAL, "int4r")):
        if f"{side}_{name}" not in pools:
            continue
        at = torch.nonzero(tags == tag).flatten()
        codes = pools[f"{side}_{name}"].index_select(0, ids[at])
        if tag == FP16:
            x = codes.float()
        else:
            scale = pools[f"{side}_{name}_scale"].index_select(0, ids[at]).float()
            if tag == INT8:
                x = codes.float() * scale.view(-1, 1, 1)
            elif tag == FP8:
                x = codes.view(torch.float8_e4m3fn).float() * scale.view(-1, 1, 1)
            elif tag == INT4:
                x = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
                x = (x.unflatten(-1, (scale.shape[1], -1)) * scale.view(-1, 1, scale.shape[1], 1)).flatten(-2)
            else:
                x = ((codes & 15).float() - 8) * scale[:, 0].view(-1, 1, 1) + ((codes >> 4).float() - 8) * scale[:, 1].view(-1, 1, 1)
        out[at] = x
    return out


def _attend_plain(s):
    q, table, valid, new = s["q"], s["table"], s["valid"], s["new"]
    B, L, Hq, D = q.shape
    Hkv, W = table.shape[1:]
    G, T = Hq // Hkv, W * PS
    ids = table.clamp(min=0).flatten().long()
    tags = torch.where(table.flatten() < 0, SKIP, s["tags"][ids])
    k, v = (_page_values(s["pools"], n, ids, tags).view(B, Hkv, T, D) for n in "kv")
    there = (tags != SKIP).view(B, Hkv, W).repeat_interleave(PS, 2).unsqueeze(2)
    qs = q.float().view(B, L, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, L * G, D)
    scores = torch.matmul(qs, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(D))
    i = torch.arange(L, device=q.device).repeat_interleave(G)
    seen = valid.view(B, Hkv, 1) - (new.view(B, 1, 1) - 1 - i if s["causal"] else torch.zeros_like(i))
    seen = torch.where(i < new.view(B, 1, 1), seen, 0)
    scores.masked_fill_((torch.arange(T, device=q.device) >= seen.unsqueeze(-1)) | ~there, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill_(top == float("-inf"), 0.0)).exp_()
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-37)
    return out.view(B, Hkv, L, G, D).permute(0, 2, 1, 3, 4).reshape(B, L, Hq, D).to(q.dtype)


def _choose_plain(s):
    logits, B, K, V = s["logits"].double(), *s["logits"].shape      # near ties decide in 64 bits
    top = logits.amax(-1, keepdim=True)
    norm = top + torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    at = logits.add_(s["scores"].double().unsqueeze(-1) - norm)
    if s["finished"] is not None:
        done = s["finished"].unsqueeze(-1)
        end = torch.arange(V, device=at.device) == s["end"]
        at = torch.where(done, torch.where(end, s["scores"].double().unsqueeze(-1), float("-inf")), at)
    best, index = torch.sort(at.view(B, K * V), dim=-1, descending=True, stable=True)
    best, index = best[:, :s["count"]], index[:, :s["count"]]
    beam = torch.div(index, V, rounding_mode="floor")
    first = K * torch.arange(B, device=at.device).unsqueeze(1)
    return best.float(), (first + beam).int(), (index - beam * V).int()


def _reorder_plain(s):
    table, valid, refs, k, v = s["table"], s["valid"], s["refs"], s["k"], s["v"]
    seqs, parents = s["seqs"].long(), s["parents"].long()
    S, Hkv, W = table.shape
    NP, n = refs.shape[0], seqs.shape[0]
    entry = torch.arange(W, device=table.device)

    def used(lens):
        return entry < torch.div(lens + (PS - 1), PS, rounding_mode="floor").unsqueeze(-1)

    # who takes a parent's last page over: the parent where it stays itself or is not listed, else its first child
    i = torch.arange(n, device=table.device)
    listed = torch.zeros(S, dtype=torch.bool, device=table.device).index_fill_(0, seqs, True)
    heir = torch.where(listed, n, -1).scatter_reduce(0, parents, torch.where(seqs == parents, -1, i), "amin")
    takes = (heir[parents] == i) | (seqs == parents)
    rows, lens = table[parents], valid[parents]
    copied = (lens % PS != 0) & ~takes.unsqueeze(1)
    number = (copied.flatten().int().cumsum(0) - copied.flatten().int()).view_as(copied).long()
    free = torch.argsort((refs != 0).int(), stable=True)
    last = (torch.div(lens + (PS - 1), PS, rounding_mode="floor") - 1).clamp(min=0).unsqueeze(-1).long()
    old = torch.gather(rows, 2, last).squeeze(-1)
    page = torch.where(copied, free[number.clamp(max=NP - 1)].int(), old)
    k[page[copied].long()] = k[old[copied].long()]
    v[page[copied].long()] = v[old[copied].long()]
    rows = rows.scatter(2, last, page.unsqueeze(-1))
    before, after = used(valid[seqs]), used(lens)
    refs.index_add_(0, table[seqs].clamp(min=0).flatten().long(), -before.flatten().int())
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), after.flatten().int())
    table[seqs] = torch.where(after, rows, torch.where(before, -1, table[seqs]))
    valid[seqs] = lens
    return table, valid, refs, k, v


# --------------------------------------------------------------------------- #
# One pass, by the framework's operators
# --------------------------------------------------------------------------- #

def _rotate_own(s):
    ia = _package()
    pools = (ia.PagePools if s["cache"] == "fp16" else ia.MxFp4Pools)(**s["pools"])
    q = ia.append_rotated_tokens(s["k"], s["v"], pools, s["table"], s["valid"], s["inv_freq"], q=s["q"], q_lens=s["new"],
                                 positions=s["positions"], interleaved=s["interleaved"])
    if s["cache"] == "fp16":
        return q, pools.k_fp16, pools.v_fp16
    return (q, *ia.read_mxfp4_tokens(pools, s["table"], s["valid"], s["count"], q_lens=s["new"]))


def _attend_own(s):
    s["plan"].run()
    return s["plan"].out


def _choose_own(s):
    return _package().beam_select(s["logits"], s["scores"], count=s["count"], finished=s["finished"], end_token=s["end"])


def _reorder_own(s):
    ia = _package()
    ia.reorder_sequences(s["table"], s["valid"], s["refs"], s["seqs"], s["parents"], ia.PagePools(k_fp16=s["k"], v_fp16=s["v"]))
    return s["table"], s["valid"], s["refs"], s["k"], s["v"]


def run(state):
    if own:
        return {"rotate": _rotate_own, "attend": _attend_own, "choose": _choose_own, "reorder": _reorder_own}[state["kind"]](state)
    return {"rotate": _rotate_plain, "attend": _attend_plain, "choose": _choose_plain,
            "reorder": _reorder_plain}[state["kind"]](state)


# --------------------------------------------------------------------------- #
# What a pass cannot do without
# --------------------------------------------------------------------------- #

def work(case):
    kind, B = case["kind"], case["B"]
    share = 0.67 if case.get("ragged") else 1.0                       # mean length over the largest one's
    if kind == "rotate":
        L, Hq, Hkv, D, size = case["L"], case["Hq"], case["Hkv"], case["D"], _SIZE[case["dtype"]]
        n = B * L * share
        cached = 2 * D if case["cache"] == "fp16" else D // 2 + D // BLOCK + 2 * D   # and read back from 4 bits
        return {"bytes": n * D * size * (Hq + 2 * Hkv) + B * L * Hq * D * size + n * 2 * Hkv * cached,
                "flops": n * (Hq + Hkv) * case["R"] * 3}
    if kind == "attend":
        L, T, Hq, Hkv, D = (case[n] for n in ("L", "T", "Hq", "Hkv", "D"))
        rows, tokens = L * share, T * share
        mix = _MIXES[case["mix"]]
        per = sum(w * _PAGE_BYTES[t] for t, w in mix.items())
        live = 1 - mix.get(SKIP, 0.0)
        seen = (tokens - (rows - 1) / 2 if case["causal"] else tokens) * live
        return {"bytes": B * (Hkv * tokens * (2 * per * D + 8 / PS) + 2 * L * Hq * D * _SIZE[case["dtype"]]),
                "flops": 4.0 * B * Hq * rows * seen * D}
    if kind == "choose":
        K, V = case["K"], case["V"]
        live = 1 - case["finished"]
        return {"bytes": B * K * V * live * _SIZE[case["dtype"]] + 12 * B * case["count"], "flops": 4.0 * B * K * V * live}
    K, Hkv, D, W = case["K"], case["Hkv"], case["D"], case["W"]
    S, NP = B * K, B * K * Hkv * case["W"] + case["spare"]
    moved = (1 - 1 / K) ** 2                                          # rows that get another's content, about
    copies = S * Hkv * (1 - (1 - (1 - 1 / K) ** K)) * 15 / 16         # children past the first of a parent
    pages = 0.75 * W * (1 - case["share"])                            # entries that change
    return {"bytes": copies * 8 * PS * D + S * Hkv * (4 * 0.75 * W * 2 + 12 * pages * moved) + 4 * NP, "flops": NP}


# --------------------------------------------------------------------------- #
# The same outputs in 64 bits, from the definitions
# --------------------------------------------------------------------------- #

def _exact_rotated(x, positions, inv_freq, interleaved):
    x = x.double().clone()
    half = inv_freq.shape[0]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = (positions.double() * inv_freq[i].double()).unsqueeze(-1)
        turned = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(angle), angle)
        x[..., a], x[..., b] = turned.real, turned.imag
    return x


def _exact_rounded(x):
    """float64 [..., D] as the 4-bit cache holds it."""
    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    most = blocks.abs().amax(-1)
    e = torch.where(most == 0, -23.0, (torch.floor(torch.log2(most)) - 2).clamp(-23, 13))
    y = blocks / torch.exp2(e).unsqueeze(-1)
    magnitudes = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
    best = torch.zeros_like(y)
    for code in range(1, 8):                  # upward: a tie goes to the one with an even code
        middle = (magnitudes[code - 1] + magnitudes[code]) / 2
        best = torch.where(y.abs() >= middle if code % 2 == 0 else y.abs() > middle, magnitudes[code], best)
    return (torch.copysign(best, y) * torch.exp2(e).unsqueeze(-1)).reshape(x.shape)


def _exact_rotate(s):
    turn = (s["positions"], s["inv_freq"], s["interleaved"])
    B, L, Hkv, _ = s["k"].shape
    new, valid = s["new"].tolist(), s["valid"].tolist()
    mine = (torch.arange(L, device="cuda") < s["new"].view(-1, 1)).view(B, L, 1, 1)
    q, k = (torch.where(mine, _exact_rotated(s[n], *turn), 0.0) for n in "qk")
    v = torch.where(mine, s["v"].double(), 0.0)
    if s["cache"] != "fp16":
        return q, _exact_rounded(k), _exact_rounded(v)
    pages = [s["pools"][n].double() for n in ("k_fp16", "v_fp16")]
    for b in range(B):
        for h in range(Hkv):
            at = torch.arange(valid[b][h] - new[b], valid[b][h], device="cuda")
            page = s["table"][b, h].long()[torch.div(at, PS, rounding_mode="floor")]
            for pool, x in zip(pages, (k, v)):
                pool[page, at % PS] = x[b, :new[b], h]
    return (q, *pages)


def _exact_page(pools, side, page, tag):
    if tag == FP16:
        return pools[side + "_fp16"][page].double()
    name = {INT8: "int8", FP8: "fp8", INT4: "int4", INT4_RESIDUAL: "int4r"}[tag]
    codes, scale = pools[f"{side}_{name}"][page], pools[f"{side}_{name}_scale"][page].double()
    if tag == INT8:
        return codes.double() * scale[:, None, None]
    if tag == FP8:
        field, part = ((codes >> 3) & 15).double(), (codes & 7).double() / 8
        size = torch.where(field == 0, part * 2.0 ** -6, (1 + part) * torch.exp2(field - 7))
        return torch.where(codes >= 128, -size, size) * scale[:, None, None]
    low, high = torch.remainder(codes, 16).double() - 8, torch.div(codes, 16, rounding_mode="floor").double() - 8
    if tag == INT4:
        x = torch.stack((low, high), -1).reshape(*codes.shape[:2], -1)
        return x * scale.repeat_interleave(x.shape[2] // scale.shape[1], 1)[:, None, :]
    return low * scale[:, :1, None] + high * scale[:, 1:, None]


def _exact_attend(s):
    q, table, tags = s["q"].double(), s["table"], s["tags"]
    B, L, Hq, D = q.shape
    Hkv = table.shape[1]
    G = Hq // Hkv
    out = torch.zeros((B, L, Hq, D), dtype=torch.float64, device="cuda")
    valid, new = s["valid"].tolist(), s["new"].tolist()
    for b in range(B):
        for h in range(Hkv):
            T, n = valid[b][h], new[b]
            row = table[b, h, :(T + PS - 1) // PS].long()
            k, v = (torch.zeros((row.shape[0], PS, D), dtype=torch.float64, device="cuda") for _ in "kv")
            for tag in (FP16, INT8, FP8, INT4, INT4_RESIDUAL):
                at = tags[row] == tag
                if bool(at.any()):
                    k[at], v[at] = (_exact_page(s["pools"], side, row[at], tag) for side in "kv")
            k, v = (x.reshape(-1, D)[:T] for x in (k, v))
            skipped = (tags[row] == SKIP).repeat_interleave(PS)[:T]
            x = (q[b, :n, h * G:(h + 1) * G].reshape(n * G, D) @ k.t().contiguous()) / math.sqrt(D)
            hidden = skipped.unsqueeze(0)
            if s["causal"]:
                last = T - n + torch.arange(n, device="cuda").repeat_interleave(G)
                hidden = hidden | (torch.arange(T, device="cuda") > last.unsqueeze(1))
            p = torch.softmax(x.masked_fill(hidden, float("-inf")), -1).nan_to_num(0.0)
            out[b, :n, h * G:(h + 1) * G] = (p @ v).view(n, G, D)
    return out


def _exact_choose(s):
    logits, scores, n = s["logits"], s["scores"], s["count"]
    B, K, V = logits.shape
    done = s["finished"].tolist() if s["finished"] is not None else [[False] * K] * B
    got = ([], [], [])
    for b in range(B):
        found = []
        for k in range(K):
            if done[b][k]:
                found += [(-float(scores[b, k]), k, s["end"])] + [(math.inf, k, t) for t in range(min(V, n + 1)) if t != s["end"]]
                continue
            p = torch.log_softmax(logits[b, k].double(), -1) + scores[b, k].double()
            edge = torch.topk(p, min(n, V)).values[-1]
            at = torch.nonzero(p >= edge).flatten()                  # ties of the last among them
            p, at = p[at].tolist(), at.tolist()
            found += sorted((-x, k, t) for x, t in zip(p, at))[:n]
        found = sorted(found)[:n]
        got[0].append([-f[0] for f in found])
        got[1].append([b * K + f[1] for f in found])
        got[2].append([f[2] for f in found])
    return (torch.tensor(got[0], dtype=torch.float64), torch.tensor(got[1], dtype=torch.int32),
            torch.tensor(got[2], dtype=torch.int32))


def _exact_reorder(s):
    """From the definition, row by row on the host."""
    table, valid, refs = s["table"].tolist(), s["valid"].tolist(), s["refs"].tolist()
    seqs, parents = s["seqs"].tolist(), s["parents"].tolist()
    listed = set(seqs)
    k, v = s["k"].double(), s["v"].double()
    old = [[row[:] for row in rows] for rows in table]
    lens = [row[:] for row in valid]
    free = iter([i for i, r in enumerate(refs) if r == 0])
    heir = {}
    for c, p in zip(seqs, parents):
        heir[p] = p if (c == p or p not in listed) else heir.get(p, c)
    src, dst = [], []
    for c, p in zip(seqs, parents):
        for h, row in enumerate(old[p]):
            n = -(-lens[p][h] // PS)
            fresh = row[:n]
            if lens[p][h] % PS and heir[p] != c:
                fresh[-1] = next(free)
                src.append(row[n - 1])
                dst.append(fresh[-1])
            was = -(-lens[c][h] // PS)
            for page in old[c][h][:was]:
                refs[page] -= 1
            for page in fresh:
                refs[page] += 1
            table[c][h] = fresh + [-1] * (was - n) + old[c][h][max(n, was):]
            valid[c][h] = lens[p][h]
    src, dst = (torch.tensor(x, dtype=torch.long, device="cuda") for x in (src, dst))
    for x in (k, v):
        x[dst] = x[src]
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (table, valid, refs)) + (k, v)


def exact(case, seed):
    return {"rotate": _exact_rotate, "attend": _exact_attend, "choose": _exact_choose,
            "reorder": _exact_reorder}[case["kind"]](prepare(case, seed))
