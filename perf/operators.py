"""Timed cases of the paged serving operators (``ops.paged_plan``, ``ops.paged_rope_cache``, ``ops.paged_attention``,
``ops.draft_verify``) with their plain forms in elementary torch operations.

``listed()`` names the cases, ``draw(rng)`` makes another of the same ranges, ``prepare(case, seed)`` makes the inputs on the GPU,
``run(state)`` is one pass (plain where ``own`` is false, the framework's entry points where it is true), ``work(case)`` the
bytes and operations a pass cannot do without and ``exact(case, seed)`` the definition in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
WORKSPACE = 64 << 20         # bytes of scratch memory that a serving program keeps for its launches (zero-filled once)
STATE_WORDS = 8              # words of paged_plan's state: free blocks, status, rows, ...


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a step of 48 requests with one to five tokens each (the sampled one and up to four drafts), contexts up to the
        # 3000 positions of the decoder's window: what stands in front of every decode step
        dict(name="plan_drafts_48", op="plan", n_seq=48, n_chunk=0, chunk=0, new_lo=1, new_hi=5, ctx_lo=100, ctx_hi=2990, block=16, lengths=1),
        # 1024 prompts of 64 to 1000 tokens admitted in one call and retired again: bulk admission, the largest
        dict(name="plan_admit_1024", op="plan", n_seq=1024, n_chunk=0, chunk=0, new_lo=64, new_hi=1000, ctx_lo=0, ctx_hi=0, block=16, lengths=2),
        # one decode step of 37 requests of the codec decoder (24 heads of 64, adjacent pairs): latency counts
        dict(name="rope_decode_37", op="rope", dtype="bf16", rows=37, heads=24, kv_heads=24, hd=64, rot=64, norm=True, inter=True, block=16, table=3008),
        # a prefill of 16384 tokens with shared kv heads of 128 features, rotated in halves
        dict(name="rope_prefill_16384", op="rope", dtype="f16", rows=16384, heads=32, kv_heads=8, hd=128, rot=128, norm=True, inter=False, block=64, table=16384),
        # a handful of single-token requests of the codec decoder: the smallest attention, latency counts
        dict(name="attn_decode_5", op="attn", dtype="bf16", n_seq=5, n_chunk=0, chunk=0, new_lo=1, new_hi=1, ctx_lo=60, ctx_hi=700, heads=24, kv_heads=24, hd=64,
             block=16, window=0, lengths=3),
        # three single tokens over very long contexts with shared kv heads: the keys have to be split
        dict(name="attn_decode_long", op="attn", dtype="bf16", n_seq=3, n_chunk=0, chunk=0, new_lo=1, new_hi=1, ctx_lo=60000, ctx_hi=120000, heads=32, kv_heads=8,
             hd=128, block=64, window=0, lengths=4),
        # 64 requests with up to four drafts each over medium contexts: the ordinary verification step
        dict(name="attn_drafts_64", op="attn", dtype="f16", n_seq=64, n_chunk=0, chunk=0, new_lo=1, new_hi=5, ctx_lo=1000, ctx_hi=16000, heads=32, kv_heads=8,
             hd=128, block=16, window=0, lengths=5),
        # a prompt's chunk beside 40 decoding requests, the decoder's 3000-position window: a step of mixed work
        dict(name="attn_mixed_41", op="attn", dtype="bf16", n_seq=41, n_chunk=1, chunk=1024, new_lo=1, new_hi=1, ctx_lo=300, ctx_hi=4200, heads=24, kv_heads=24,
             hd=64, block=16, window=3000, lengths=6),
        # two chunks of 4096 tokens behind long contexts: chunked prefill, the largest (matrix products)
        dict(name="attn_chunk_4096", op="attn", dtype="bf16", n_seq=2, n_chunk=2, chunk=4096, new_lo=1, new_hi=1, ctx_lo=9000, ctx_hi=12500, heads=32, kv_heads=8,
             hd=128, block=64, window=0, lengths=7),
        # chunks of odd length in 32 bits (the parity mode's type)
        dict(name="attn_chunk_f32", op="attn", dtype="f32", n_seq=6, n_chunk=3, chunk=131, new_lo=1, new_hi=3, ctx_lo=37, ctx_hi=1900, heads=24, kv_heads=24, hd=64,
             block=16, window=0, lengths=8),
        # drafts verified over the codec decoder's vocabulary (4096 tokens): latency counts
        dict(name="verify_codec_32", op="verify", dtype="f32", n_seq=32, new_lo=1, new_hi=5, vocab=4096, sure=False, sharp=4.0, lengths=9),
        # up to seven drafts of 128 requests over a large text vocabulary
        dict(name="verify_text_128", op="verify", dtype="f32", n_seq=128, new_lo=1, new_hi=8, vocab=128011, sure=False, sharp=8.0, lengths=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attn", "attn", "verify"])
    lengths = rng.randrange(100, 1 << 20)
    if op == "plan":
        n = _log(rng, 1, 1024)
        if rng.random() < 0.5:
            return dict(op=op, n_seq=n, n_chunk=0, chunk=0, new_lo=1, new_hi=rng.randint(1, 9), ctx_lo=rng.randint(1, 200), ctx_hi=_log(rng, 200, 4000),
                        block=rng.choice([8, 16, 32, 64]), lengths=lengths)
        return dict(op=op, n_seq=n, n_chunk=rng.randint(0, n), chunk=_log(rng, 10, max(11, min(8000, 400000 // n))), new_lo=1, new_hi=_log(rng, 1, 400), ctx_lo=0, ctx_hi=rng.choice([0, 500]),
                    block=rng.choice([8, 16, 32, 64]), lengths=lengths)
    if op == "rope":
        hd = rng.choice([64, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        if rng.random() < 0.25:
            kv = heads = 24
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_log(rng, 1, 8000 if hd == 128 else 16000), heads=heads, kv_heads=kv, hd=hd, rot=rng.choice([hd, hd, hd // 2]),
                    norm=rng.random() < 0.75, inter=rng.random() < 0.5, block=rng.choice([8, 16, 32, 64]), table=rng.choice([513, 3008, 16384]))
    if op == "verify":
        dtype = rng.choice(["f32", "f32", "f16", "bf16"])
        return dict(op=op, dtype=dtype, n_seq=_log(rng, 1, 128), new_lo=1, new_hi=rng.randint(1, 8), vocab=_log(rng, 300, 128000), sure=rng.random() < 0.3,
                    sharp=rng.choice([2.0, 4.0, 8.0]), lengths=lengths)
    kind = rng.choice(["decode", "drafts", "chunk", "long"])
    hd = rng.choice([64, 128])
    kv, group = rng.choice([(24, 1), (8, 1), (8, 4), (4, 7), (2, 8), (1, 16), (6, 3)])
    dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16"])
    case = dict(op=op, dtype=dtype, n_chunk=0, chunk=0, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=1, heads=kv * group, kv_heads=kv, hd=hd, block=rng.choice([8, 16, 32, 64]),
                window=rng.choice([0, 0, 0, rng.randint(100, 3500)]), lengths=lengths)
    if kind == "decode":
        case.update(n_seq=_log(rng, 1, 96), ctx_hi=_log(rng, 16, 4000))
    elif kind == "drafts":
        case.update(n_seq=_log(rng, 1, 64), new_hi=rng.randint(2, 9), ctx_lo=20, ctx_hi=_log(rng, 100, 12000))
    elif kind == "long":
        case.update(n_seq=rng.randint(1, 3), new_hi=rng.randint(1, 3), ctx_lo=5000, ctx_hi=_log(rng, 10000, 110000), kv_heads=min(kv, 8), heads=min(kv, 8) * group)
    else:
        n = rng.randint(1, 6)
        case.update(n_seq=n, n_chunk=rng.randint(1, n), chunk=_log(rng, 10, 2500), new_hi=rng.randint(1, 4), ctx_hi=_log(rng, 2, 8000))
    return case


def _lengths(case):
    """[(tokens in the cache, new tokens)] of the case's requests: a chunk for the first n_chunk of them."""
    r = random.Random(case["lengths"])
    lo, hi = max(case.get("ctx_lo", 1), 1), max(case.get("ctx_hi", 1), 1)
    ctx = [0 if case.get("ctx_hi", 0) == 0 else int(round(lo * (max(hi, lo) / lo) ** r.random())) for _ in range(case["n_seq"])]
    new = [case["chunk"] if i < case.get("n_chunk", 0) else r.randint(case["new_lo"], max(case["new_lo"], case["new_hi"])) for i in range(case["n_seq"])]
    return list(zip(ctx, new))


def _pages(n, block):
    return -(-n // block)


# -------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    i32 = dict(dtype=torch.int32, device="cuda")
    if case["op"] == "rope":
        dt, rows, hd, block = DTYPES[case["dtype"]], case["rows"], case["hd"], case["block"]
        heads, kv = case["heads"], case["kv_heads"]
        n_blocks = _pages(rows, block) + 3
        state["qkv"] = torch.randn(rows, (heads + 2 * kv) * hd, generator=g, device="cuda").mul_(2.0).to(dt)
        state["q_norm"] = torch.rand(hd, generator=g, device="cuda") + 0.5 if case["norm"] else None
        state["k_norm"] = torch.rand(hd, generator=g, device="cuda") + 0.5 if case["norm"] else None
        angle = torch.arange(case["table"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
        state["positions"] = torch.randint(0, case["table"], (rows,), generator=g, device="cuda").int()
        state["slots"] = torch.randperm(n_blocks * block, generator=g, device="cuda")[:rows].int()
        state["q_out"] = torch.zeros(rows, heads, hd, dtype=dt, device="cuda")
        state["k_cache"] = torch.zeros(n_blocks, kv, block, hd, dtype=dt, device="cuda")
        state["v_cache"] = torch.zeros(n_blocks, kv, block, hd, dtype=dt, device="cuda")
        return state
    lens = _lengths(case)
    ctx = torch.tensor([c for c, _ in lens], **i32)
    new = torch.tensor([n for _, n in lens], **i32)
    rows = sum(n for _, n in lens)
    start = torch.zeros(len(lens) + 1, **i32)
    start[1:] = torch.cumsum(new, 0)
    if case["op"] == "verify":
        dt, V = DTYPES[case["dtype"]], case["vocab"]
        z = torch.randn(rows, V, generator=g, device="cuda") * case["sharp"] / 2
        zq = z + torch.randn(rows, V, generator=g, device="cuda") * 0.7
        state["target"] = torch.softmax(z, -1).to(dt)
        state["draft"] = None if case["sure"] else torch.softmax(zq, -1).to(dt)
        picks = torch.argmax(zq - torch.log(torch.empty(rows, V, device="cuda").exponential_(generator=g)), -1)
        state["tokens"] = torch.cat([torch.randint(0, V, (1,), generator=g, device="cuda"), picks[:-1]])     # row r drafts token r + 1
        state["start"] = start
        state["uniforms"] = torch.rand(rows, generator=g, device="cuda")
        state["noise"] = torch.empty(len(lens), V, device="cuda").exponential_(generator=g)
        state["seq_len"] = new + torch.randint(1, 3000, (len(lens),), generator=g, device="cuda").int()
        state["out_tokens"] = torch.zeros(len(lens), case["new_hi"], dtype=torch.int64, device="cuda")
        state["n_out"] = torch.zeros(len(lens), **i32)
        state["keep_len"] = torch.zeros(len(lens), **i32)
        state["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
        del z, zq
        return state
    block = case["block"]
    need = [_pages(c + n, block) for c, n in lens]
    width = max(need) + 2
    n_blocks = sum(need) + sum(need) // 8 + 5
    order = torch.randperm(n_blocks, generator=g, device="cuda").int()
    held = need if case["op"] == "attn" else [_pages(c, block) for c, _ in lens]
    held_t = torch.tensor(held, device="cuda")
    first = torch.cumsum(held_t, 0) - held_t
    j = torch.arange(width, device="cuda")
    at = first[:, None] + j[None, :]
    table = torch.where(j[None, :] < held_t[:, None], order[at.clamp(max=n_blocks - 1)], torch.full_like(order[:1], -1))
    state["table"] = table.int().contiguous()
    if case["op"] == "plan":
        used = sum(held)
        free = torch.full((n_blocks,), -1, **i32)
        free[:n_blocks - used] = order[used:]
        state["free"] = free
        state["words"] = torch.zeros(STATE_WORDS, **i32)
        state["words"][0] = n_blocks - used
        state["seq_len"], state["keep"], state["new"] = ctx.clone(), ctx.clone(), new
        state["none"] = torch.zeros_like(new)
        state["q_start"], state["q_start_back"] = torch.zeros_like(start), torch.zeros_like(start)
        state["slots"], state["positions"] = torch.zeros(rows + 7, **i32), torch.zeros(rows + 7, **i32)      # rows of a fixed-size launch: some are padding
        return state
    dt, hd, heads, kv = DTYPES[case["dtype"]], case["hd"], case["heads"], case["kv_heads"]
    state["q"] = torch.randn(rows, heads, hd, generator=g, device="cuda").to(dt)
    state["k_cache"] = torch.randn(n_blocks, kv, block, hd, generator=g, device="cuda", dtype=dt)
    state["v_cache"] = torch.randn(n_blocks, kv, block, hd, generator=g, device="cuda", dtype=dt)
    state["seq_len"], state["q_start"] = ctx + new, start
    state["max_new"], state["max_len"] = max(n for _, n in lens), max(c + n for c, n in lens)
    state["out"] = torch.zeros(rows, heads, hd, dtype=dt, device="cuda")
    state["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    return state


# --------------------------------------------------------------------------------------- plain forms
def _plan_plain(s, keep, new, q_start, slots, positions):
    table, free, words, block = s["table"], s["free"], s["words"], s["block"]
    B, width = table.shape
    n_blocks = free.shape[0]
    dev = table.device
    held, k, n = s["seq_len"].long(), keep.long(), new.long()
    end = k + n
    have, need = (held + block - 1) // block, (end + block - 1) // block
    grow, give = (need - have).clamp(min=0), (have - need).clamp(min=0)
    grow_end, give_end, row_end = torch.cumsum(grow, 0), torch.cumsum(give, 0), torch.cumsum(n, 0)
    taken, given, n_free = grow_end[-1], give_end[-1], words[0].long()
    bad = (k < 0) | (n < 0) | (k > held) | (need > width)
    rows = 0 if slots is None else slots.shape[0]
    over = row_end[-1] > rows if slots is not None else torch.zeros((), dtype=torch.bool, device=dev)
    lost = n_free + given - taken > n_blocks
    first_bad = torch.where(bad, torch.arange(B, device=dev), B + 2).amin()
    first_bad = torch.minimum(first_bad, torch.where(over, B, B + 2))
    first_bad = torch.minimum(first_bad, torch.where(lost, B + 1, B + 2))
    short = (taken - n_free - given).clamp(min=0)
    status = torch.where(first_bad < B + 2, -1 - first_bad, short)
    ok = status == 0
    a = torch.arange(n_blocks, device=dev)
    rel_b = torch.searchsorted(give_end, a, right=True).clamp(max=B - 1)
    rel = table[rel_b, (need[rel_b] + a - (give_end - give)[rel_b]).clamp(0, width - 1)]           # returned blocks, ascending (request, page)
    stack = torch.cat([free, free])
    spot = n_free + given - 1 - a                                                                 # the last request's last page is pushed first
    stack = stack.scatter(0, torch.where((a < given) & (spot >= 0), spot, 2 * n_blocks - 1), rel)
    got = stack[(n_free + given - 1 - a).clamp(0, 2 * n_blocks - 1)]                              # allocation i pops the i-th from the top
    got_b = torch.searchsorted(grow_end, a, right=True).clamp(max=B - 1)
    got_j = have[got_b] + a - (grow_end - grow)[got_b]
    flat = torch.cat([table.reshape(-1), table.new_zeros(1)])
    flat = flat.scatter(0, torch.where((a < taken) & ok, got_b * width + got_j, B * width).clamp(max=B * width), got)
    after = flat[:-1].view(B, width)
    table.copy_(after)
    kept = (a >= taken) & (a < given) & ok
    free.copy_(torch.cat([free, free[:1]]).scatter(0, torch.where(kept, spot, n_blocks).clamp(0, n_blocks), rel)[:-1])
    words[0] = torch.where(ok, n_free + given - taken, n_free).int()
    words[1] = status.int()
    words[2] = torch.where(ok, row_end[-1], 0).int()
    s["seq_len"].copy_(torch.where(ok, end, held).int())
    q_start[0] = 0
    q_start[1:] = torch.where(ok, row_end, 0).int()
    if slots is not None:
        r = torch.arange(rows, device=dev)
        b = torch.searchsorted(row_end, r, right=True)
        live = (b < B) & ok
        b = b.clamp(max=B - 1)
        pos = k[b] + r - (row_end - n)[b]
        blk = after[b, (pos // block).clamp(0, width - 1)].long()
        slot = blk * block + pos % block
        slots.copy_(torch.where(live & (blk >= 0) & (blk < n_blocks), slot, -1).int())
        positions.copy_(torch.where(live, pos, -1).int())


def _rope_plain(s):
    rows, hd, heads, kv, rot = s["rows"], s["hd"], s["heads"], s["kv_heads"], s["rot"]
    x = s["qkv"].float().view(rows, heads + 2 * kv, hd)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], s["qkv"].view(rows, heads + 2 * kv, hd)[:, heads + kv:]
    if s["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-5) * s["q_norm"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-5) * s["k_norm"]
    cs = s["rope"][s["positions"].long()]
    q, k = _rotate(q, cs, rot, s["inter"]), _rotate(k, cs, rot, s["inter"])
    slot = s["slots"].long()
    blk, off = slot // s["block"], slot % s["block"]
    s["q_out"].copy_(q)
    s["k_cache"][blk, :, off] = k.to(s["k_cache"].dtype)
    s["v_cache"][blk, :, off] = v
    return s["q_out"], s["k_cache"], s["v_cache"]


def _rotate(x, cs, rot, inter):
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    y = x[..., :rot]
    if inter:
        a, b = y[..., 0::2], y[..., 1::2]
        y = torch.stack([a * c - b * sn, a * sn + b * c], -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:]
        y = torch.cat([a * c - b * sn, a * sn + b * c], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _attn_plain(s):
    """Requests padded to the longest: keys gathered through the table, masked softmax, products in 32 bits."""
    B, block, heads, kv, hd = s["n_seq"], s["block"], s["heads"], s["kv_heads"], s["hd"]
    group, L, N = heads // kv, s["max_len"], s["max_new"]
    start, seq = s["q_start"].long(), s["seq_len"].long()
    new = start[1:] - start[:-1]
    j = torch.arange(L, device="cuda")
    blk = s["table"].long()[:, j // block].clamp(min=0)
    there = (j[None] < seq[:, None])[:, None, :, None]
    keys = torch.where(there, s["k_cache"][blk, :, j % block].transpose(1, 2).float(), 0.0)           # (B, kv, L, hd)
    vals = torch.where(there, s["v_cache"][blk, :, j % block].transpose(1, 2).float(), 0.0)
    i = torch.arange(N, device="cuda")
    row = (start[:-1, None] + i[None]).clamp(max=max(s["q"].shape[0] - 1, 0))
    q = s["q"].float()[row].view(B, N, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(B, kv, group * N, hd)
    pos = (seq - new)[:, None] + i[None]
    sees = (j[None, None] <= pos[:, :, None]) & (j[None, None] < seq[:, None, None])
    if s["window"]:
        sees = sees & (j[None, None] > pos[:, :, None] - s["window"])
    scores = torch.matmul(q, keys.transpose(2, 3).contiguous()).mul_(1.0 / math.sqrt(hd)).view(B, kv, group, N, L)
    scores = scores.masked_fill_(~sees[:, None, None], float("-inf"))
    p = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, kv, group * N, L), vals).view(B, kv, group, N, hd) / total.clamp(min=1e-30)
    live = i[None] < new[:, None]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, N, heads, hd)
    s["out"].copy_(o[live])
    return s["out"]


def _verify_plain(s):
    t, start = s["target"].float(), s["start"].long()
    B, V = s["n_seq"], t.shape[1]
    W = s["out_tokens"].shape[1]
    dev = t.device
    n = start[1:] - start[:-1]
    i = torch.arange(W, device=dev)
    row = (start[:-1, None] + i[None]).clamp(max=t.shape[0] - 1)
    d = s["tokens"][(row + 1).clamp(max=t.shape[0] - 1)]
    p = t[row, d]
    q = torch.ones_like(p) if s["draft"] is None else s["draft"].float()[row, d]
    taken = (s["uniforms"][row] * q < p) & (i[None] < n[:, None] - 1)
    count = torch.cumprod(taken.long(), 1).sum(1)                                  # drafts before the first that is rejected
    last = start[:-1] + count
    rejected = count < n - 1
    pt = t[last]
    bad = s["tokens"][(last + 1).clamp(max=t.shape[0] - 1)]
    if s["draft"] is None:
        rest = torch.where(torch.arange(V, device=dev)[None] == bad[:, None], torch.zeros_like(pt), pt)
    else:
        rest = (pt - s["draft"].float()[last]).clamp(min=0.0)
    rest = torch.where(rejected[:, None] & (rest > 0).any(1, keepdim=True), rest, pt)
    score = rest / s["noise"]
    score = torch.where((rest > 0) & (score > 0), score, torch.zeros_like(score))
    best = score.amax(1, keepdim=True)
    token = torch.where(score == best, torch.arange(V, device=dev)[None], V).amin(1)
    out = torch.where(i[None] < count[:, None], d, -1)
    s["out_tokens"].copy_(torch.where(i[None] == count[:, None], token[:, None], out))
    s["n_out"].copy_(count + 1)
    s["keep_len"].copy_(s["seq_len"] - n + count + 1)
    return s["out_tokens"], s["n_out"], s["keep_len"]


# ---------------------------------------------------------------------------------------------- pass
def run(state):
    s = state
    if s["op"] == "plan":
        if own:
            from mars5_tts_amd import ops
            ops.paged_plan(s["seq_len"], s["keep"], s["new"], s["table"], s["free"], s["words"], s["block"], s["q_start"], s["slots"], s["positions"])
            ops.paged_plan(s["seq_len"], s["keep"], s["none"], s["table"], s["free"], s["words"], s["block"], s["q_start_back"])
        else:
            _plan_plain(s, s["keep"], s["new"], s["q_start"], s["slots"], s["positions"])
            _plan_plain(s, s["keep"], s["none"], s["q_start_back"], None, None)
        return s["q_start"], s["slots"], s["positions"], s["seq_len"], s["table"], s["free"], s["words"], s["q_start_back"]
    if s["op"] == "rope":
        if own:
            from mars5_tts_amd import ops
            ops.paged_rope_cache(s["qkv"], s["heads"], s["kv_heads"], s["rope"], s["positions"], s["slots"], s["q_out"], s["k_cache"], s["v_cache"],
                                 q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-5, interleaved=s["inter"])
            return s["q_out"], s["k_cache"], s["v_cache"]
        return _rope_plain(s)
    if s["op"] == "attn":
        if own:
            from mars5_tts_amd import ops
            ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_len"], s["q_start"], s["out"], window=s["window"], max_new=s["max_new"],
                                workspace=s["workspace"])
            return s["out"]
        return _attn_plain(s)
    if own:
        from mars5_tts_amd import ops
        ops.draft_verify(s["target"], s["draft"], s["tokens"], s["start"], s["uniforms"], s["noise"], s["out_tokens"], s["n_out"], seq_len=s["seq_len"],
                         keep_len=s["keep_len"], workspace=s["workspace"])
        return s["out_tokens"], s["n_out"], s["keep_len"]
    return _verify_plain(s)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "rope":
        width = (case["heads"] + 2 * case["kv_heads"]) * case["hd"]
        table = min(case["rows"], case["table"]) * case["rot"] * 4
        return {"bytes": 2 * case["rows"] * width * SIZE[case["dtype"]] + table + 8 * case["rows"],
                "flops": case["rows"] * (case["heads"] + case["kv_heads"]) * case["hd"] * 8}
    lens = _lengths(case)
    rows = sum(n for _, n in lens)
    if case["op"] == "plan":
        pages = sum(_pages(c + n, case["block"]) - _pages(c, case["block"]) for c, n in lens)
        return {"bytes": 8 * rows + 16 * pages + 2 * 20 * len(lens), "flops": 4 * rows + 4 * pages + 20 * len(lens)}
    if case["op"] == "verify":
        per = 4 + SIZE[case["dtype"]] * (1 if case["sure"] else 2)
        return {"bytes": len(lens) * (case["vocab"] * per + 24) + 24 * rows, "flops": len(lens) * case["vocab"] * 3}
    pairs, held = 0, 0
    for c, n in lens:
        w = case["window"] or (c + n)
        pairs += sum(min(c + i + 1, w) for i in range(n))
        held += min(c + n, w + n - 1)
    size = SIZE[case["dtype"]]
    return {"bytes": 2 * held * case["kv_heads"] * case["hd"] * size + 2 * rows * case["heads"] * case["hd"] * size + 4 * sum(_pages(c + n, case["block"]) for c, n in lens),
            "flops": 4 * pairs * case["heads"] * case["hd"]}


# --------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _plan_exact, "rope": _rope_exact, "attn": _attn_exact, "verify": _verify_exact}[case["op"]](s)


def _plan_exact(s):
    """The free list as a Python list, request by request; both calls of a pass."""
    table, block = s["table"].cpu().numpy().copy(), s["block"]
    free = s["free"].cpu().numpy().copy()
    n_free = int(s["words"][0])
    ctx, new = s["keep"].tolist(), s["new"].tolist()
    slots = np.full(s["slots"].shape[0], -1, np.int32)
    positions = slots.copy()
    starts, r = [0], 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        for j in range(_pages(c, block), _pages(c + n, block)):
            n_free -= 1
            table[b, j] = free[n_free]
        p = np.arange(c, c + n)
        slots[r:r + n] = table[b, p // block] * block + p % block
        positions[r:r + n] = p
        r += n
        starts.append(r)
    for b in range(len(ctx) - 1, -1, -1):
        for j in range(_pages(ctx[b] + new[b], block) - 1, _pages(ctx[b], block) - 1, -1):
            free[n_free] = table[b, j]
            n_free += 1
    words = np.zeros(STATE_WORDS, np.int32)
    words[0] = n_free
    out = np.array(starts, np.int32), slots, positions, np.array(ctx, np.int32), table, free, words, np.zeros(len(ctx) + 1, np.int32)
    return tuple(torch.from_numpy(np.ascontiguousarray(x)) for x in out)


def _rope_exact(s):
    heads, kv, hd, half = s["heads"], s["kv_heads"], s["hd"], s["rot"] // 2
    x = s["qkv"].double().reshape(s["rows"], -1, hd).clone()
    v = x[:, heads + kv:]
    for part, w in ((slice(0, heads), s["q_norm"]), (slice(heads, heads + kv), s["k_norm"])):
        if w is not None:
            x[:, part] = x[:, part] / (x[:, part].square().sum(-1, keepdim=True) / hd + 1e-5).sqrt() * w.double()
    z = x[:, :heads + kv]
    cs = s["rope"].double()[s["positions"].long()]
    turn = torch.complex(cs[..., 0], cs[..., 1])[:, None]
    first = slice(0, 2 * half, 2) if s["inter"] else slice(0, half)
    second = slice(1, 2 * half, 2) if s["inter"] else slice(half, 2 * half)
    w = torch.complex(z[..., first], z[..., second]) * turn
    z = z.clone()
    z[..., first], z[..., second] = w.real, w.imag
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    where = s["slots"].long()
    k_cache.permute(0, 2, 1, 3)[where // s["block"], where % s["block"]] = z[:, heads:]
    v_cache.permute(0, 2, 1, 3)[where // s["block"], where % s["block"]] = v
    return z[:, :heads].contiguous(), k_cache, v_cache


def _attn_exact(s):
    if work(s)["flops"] > 2e13:
        return None
    group, hd, block = s["heads"] // s["kv_heads"], s["hd"], s["block"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    start, seq = s["q_start"].tolist(), s["seq_len"].tolist()
    for b, n in enumerate(seq):
        lo, hi = start[b], start[b + 1]
        pages = s["table"][b, :_pages(n, block)].long()
        pos = torch.arange(n - (hi - lo), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        hide = (key > pos) | (key <= pos - s["window"] if s["window"] else key < 0)
        for h in range(s["kv_heads"]):
            k = s["k_cache"][pages, h].reshape(-1, hd)[:n].double()
            v = s["v_cache"][pages, h].reshape(-1, hd)[:n].double()
            for e in range(group):
                z = s["q"][lo:hi, h * group + e].double() @ k.T.contiguous() / math.sqrt(hd)
                out[lo:hi, h * group + e] = torch.softmax(z.masked_fill_(hide, -math.inf), -1) @ v
    return out


def _verify_exact(s):
    """Request by request; the probabilities' products and quotients are defined in 32 bits (numpy's, correctly rounded)."""
    start, tokens = s["start"].tolist(), s["tokens"].tolist()
    u = s["uniforms"].cpu().numpy()
    out = np.full(s["out_tokens"].shape, -1, np.int64)
    count, keep = [], []
    for b in range(len(start) - 1):
        r, end, k = start[b], start[b + 1], 0
        while r < end - 1:
            d = tokens[r + 1]
            q = np.float32(1) if s["draft"] is None else np.float32(float(s["draft"][r, d]))
            if not u[r] * q < np.float32(float(s["target"][r, d])):
                break
            out[b, k] = d
            r, k = r + 1, k + 1
        p = s["target"][r].float().cpu().numpy()
        rest = p
        if r < end - 1:
            if s["draft"] is None:
                rest = p.copy()
                rest[tokens[r + 1]] = 0
            else:
                rest = np.maximum(p - s["draft"][r].float().cpu().numpy(), np.float32(0))
            rest = rest if (rest > 0).any() else p
        out[b, k] = int(np.argmax(rest / s["noise"][b].cpu().numpy()))
        count.append(k + 1)
        keep.append(int(s["seq_len"][b]) - (end - start[b]) + k + 1)
    return torch.from_numpy(out), torch.tensor(count, dtype=torch.int32), torch.tensor(keep, dtype=torch.int32)
