"""Paged serving operators on a real MI355X, through the public wrappers, against plain 64-bit (integers: exact) restatements of their
definitions (include/mars5_paged.h).  Tolerances count roundings: a rounding to type t is off by at most u(t) = finfo(t).eps / 2 of the value."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DTS = [torch.float32, torch.float16, torch.bfloat16]
U32 = 2.0 ** -24


def u(dt):
    return torch.finfo(dt).eps / 2


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "gpu tests need a ROCm device"
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------------------------------------ paged_plan
class Pool:
    """The definition in Python lists."""

    def __init__(self, n_seq, width, n_blocks, block, seed=0):
        self.block, self.width, self.n_blocks = block, width, n_blocks
        self.free = list(range(n_blocks))
        random.Random(seed).shuffle(self.free)
        self.pages = [[] for _ in range(n_seq)]
        self.len = [0] * n_seq

    def tensors(self, dev):
        from mars5_tts_amd import _lib as L
        state = torch.zeros(L.PST_WORDS, dtype=torch.int32)
        state[L.PST_FREE] = len(self.free)
        return dict(seq_len=_i32(self.len, dev), table=torch.full((len(self.len), self.width), -1, dtype=torch.int32, device=dev),
                    free=_i32(self.free + [-1] * (self.n_blocks - len(self.free)), dev), state=state.to(dev))

    def step(self, keep, new, n_rows):
        """(status, q_start, slots, positions)"""
        B = len(self.len)
        nothing = ([0] * (B + 1), [-1] * n_rows, [-1] * n_rows)
        pg = lambda n: -(-n // self.block)     # noqa: E731
        for b in range(B):
            if keep[b] < 0 or new[b] < 0 or keep[b] > self.len[b] or keep[b] + new[b] > self.width * self.block:
                return (-1 - b,) + nothing
        if sum(new) > n_rows:
            return (-1 - B,) + nothing
        need = [pg(k + n) for k, n in zip(keep, new)]
        take, give = sum(max(n - len(p), 0) for n, p in zip(need, self.pages)), sum(max(len(p) - n, 0) for n, p in zip(need, self.pages))
        if take > len(self.free) + give:
            return (take - len(self.free) - give,) + nothing
        for b in range(B - 1, -1, -1):
            while len(self.pages[b]) > need[b]:
                self.free.append(self.pages[b].pop())
        start, slots, pos = [0], [], []
        for b in range(B):
            while len(self.pages[b]) < need[b]:
                self.pages[b].append(self.free.pop())
            for p in range(keep[b], keep[b] + new[b]):
                slots.append(self.pages[b][p // self.block] * self.block + p % self.block)
                pos.append(p)
            start.append(len(slots))
            self.len[b] = keep[b] + new[b]
        pad = [-1] * (n_rows - len(slots))
        return 0, start, slots + pad, pos + pad


def _check_plan(t, pool, want, got_start, slots, pos):
    from mars5_tts_amd import _lib as L
    status, start, w_slots, w_pos = want
    st = t["state"].tolist()
    assert st[L.PST_STATUS] == status and st[L.PST_FREE] == len(pool.free) and st[L.PST_ROWS] == start[-1] and st[3:] == [0] * 5
    assert got_start.tolist() == start and slots.tolist() == w_slots and pos.tolist() == w_pos
    assert t["seq_len"].tolist() == pool.len and t["free"].tolist()[:len(pool.free)] == pool.free
    for b, p in enumerate(pool.pages):
        assert t["table"][b, :len(p)].tolist() == p


@pytest.mark.parametrize("n_seq,block,rows,seed", [(1, 1, 40, 1), (5, 16, 200, 2), (67, 8, 1500, 3), (1030, 4, 9001, 4), (4096, 16, 20000, 5)])
def test_plan_random_steps(dev, n_seq, block, rows, seed):
    """Admission, growth, rejected drafts, retirement and reuse over several steps against the list definition; steps that are short
    of blocks, ask for too many rows or hold an invalid request change nothing."""
    from mars5_tts_amd import ops
    rng = random.Random(seed)
    width = 8
    pool = Pool(n_seq, width, max(n_seq * 2, 12), block, seed)
    t = pool.tensors(dev)
    seen = set()
    for step in range(10):
        keep = [rng.choice([0, ln, ln, max(0, ln - rng.randrange(1, 5))]) for ln in pool.len]
        new = [rng.choice([0, 1, 1, 3, rng.randrange(block * 3)]) for _ in range(n_seq)]
        if step == 4:
            keep[rng.randrange(n_seq)] = rng.choice([-1, 1 << 20])
        if step == 6:
            new[n_seq // 2] = width * block + 1
        if n_seq > 5 and step not in (7,):
            total = 0                                    # keep most steps within the row count
            for b in range(n_seq):
                new[b] = min(new[b], max(rows - total, 0)) if step not in (6,) else new[b]
                total += new[b]
        q_start, slots, pos = _i32([7] * (n_seq + 1), dev), _i32([7] * rows, dev), _i32([7] * rows, dev)
        want = pool.step(keep, new, rows)
        ops.paged_plan(t["seq_len"], _i32(keep, dev), _i32(new, dev), t["table"], t["free"], t["state"], block, q_start, slots, pos)
        torch.cuda.synchronize()
        _check_plan(t, pool, want, q_start, slots, pos)
        seen.add(0 if want[0] == 0 else (1 if want[0] > 0 else -1))
    assert 0 in seen and -1 in seen


def test_plan_short_of_blocks_and_rollback(dev):
    """A step that needs more blocks than there are says how many are missing and changes nothing; a step that is rolled back restores the
    free stack exactly; a retired request's blocks go to another in the same call."""
    from mars5_tts_amd import _lib as L, ops
    pool = Pool(3, 10, 7, 16, 9)
    t = pool.tensors(dev)
    zero = _i32([0, 0, 0], dev)

    def call(keep, new, rows=200):
        q_start, slots, pos = _i32([7] * 4, dev), _i32([7] * rows, dev), _i32([7] * rows, dev)
        want = pool.step(keep, new, rows)
        ops.paged_plan(t["seq_len"], _i32(keep, dev), _i32(new, dev), t["table"], t["free"], t["state"], 16, q_start, slots, pos)
        _check_plan(t, pool, want, q_start, slots, pos)
        return want[0]

    assert call([0, 0, 0], [17, 33, 16]) == 0                                  # 2 + 3 + 1 of 7 blocks
    before = t["free"].clone(), t["state"].clone(), t["seq_len"].clone()
    assert call([17, 33, 16], [16, 16, 16]) == 2                               # three more needed, one there
    assert call([17, 33, 16], [15, 0, 1]) == 0
    q = _i32([0] * 4, dev)
    ops.paged_plan(t["seq_len"], before[2], zero, t["table"], t["free"], t["state"], 16, q)          # roll back, rows not described
    pool.step([17, 33, 16], [0, 0, 0], 200)
    assert torch.equal(t["seq_len"], before[2]) and int(t["state"][L.PST_FREE]) == 1 and torch.equal(t["free"][:1], before[0][:1])
    assert call([17, 0, 16], [32, 17, 0]) == 0                                 # request 1 starts anew, its old blocks serve 0 and 1
    assert call([0, 0, 0], [0, 0, 0]) == 0 and sorted(pool.free) == list(range(7))


def test_plan_keeps_everything_by_the_same_tensor(dev):
    """keep_len may be seq_len itself: every request keeps all that it holds; one workgroup and many."""
    from mars5_tts_amd import ops
    for B, rows in ((3, 50), (900, 40000)):
        pool = Pool(B, 12, 12 * B, 16, 2)
        t = pool.tensors(dev)
        for step in range(4):
            new = [(b * 7 + step * 11) % 40 for b in range(B)] if step < 3 else [1] * B
            new = new if B > 3 else [9, 0, 17][:B]
            q_start, slots, pos = _i32([7] * (B + 1), dev), _i32([7] * rows, dev), _i32([7] * rows, dev)
            want = pool.step(pool.len[:], new, rows)
            ops.paged_plan(t["seq_len"], t["seq_len"], _i32(new, dev), t["table"], t["free"], t["state"], 16, q_start, slots, pos)
            torch.cuda.synchronize()
            _check_plan(t, pool, want, q_start, slots, pos)


def test_plan_strided_table_other_stream_and_replay(dev):
    """A table that is a slice of a wider one, the call on a stream of its own, and a captured call that is replayed with eager work in
    between: every replay continues from the state of the one before."""
    from mars5_tts_amd import ops
    B, block, rows = 6, 8, 64
    pool = Pool(B, 12, 60, block, 3)
    t = pool.tensors(dev)
    wide = torch.full((B, 40), 99, dtype=torch.int32, device=dev)
    wide[:, 5:17] = t["table"]
    t["table"] = wide[:, 5:17]
    side = torch.cuda.Stream(device=dev)
    keep, new = _i32([0] * B, dev), _i32([3] * B, dev)
    q_start, slots, pos = _i32([7] * (B + 1), dev), _i32([7] * rows, dev), _i32([7] * rows, dev)
    torch.cuda.synchronize()
    ops.paged_plan(t["seq_len"], keep, new, t["table"], t["free"], t["state"], block, q_start, slots, pos, stream=side.cuda_stream)
    side.synchronize()
    _check_plan(t, pool, pool.step([0] * B, [3] * B, rows), q_start, slots, pos)
    keep.copy_(t["seq_len"])
    torch.cuda.synchronize()
    g = ops.Graph()
    g.begin(side.cuda_stream)
    ops.paged_plan(t["seq_len"], keep, new, t["table"], t["free"], t["state"], block, q_start, slots, pos, stream=side.cuda_stream)
    g.end(side.cuda_stream)
    for i in range(4):
        n = [(i + b) % 5 for b in range(B)]
        new.copy_(_i32(n, dev))
        keep.copy_(t["seq_len"])
        torch.cuda.synchronize()
        k = pool.len[:]
        g.launch(side.cuda_stream)
        side.synchronize()
        _check_plan(t, pool, pool.step(k, n, rows), q_start, slots, pos)
    assert bool((wide[:, :5] == 99).all()) and bool((wide[:, 17:] == 99).all())


# ------------------------------------------------------------------------------------------------------ paged_rope_cache
def _rope_ref(x, w, cs, n_pairs, inter, eps):
    """float64 rows (R, H, hd) and the sum of magnitudes behind every feature (for the error bound)."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    c, s = cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    y, mag = x.clone(), x.abs()
    a, b = (x[..., 0:2 * n_pairs:2], x[..., 1:2 * n_pairs:2]) if inter else (x[..., :n_pairs], x[..., n_pairs:2 * n_pairs])
    ia = (slice(0, 2 * n_pairs, 2), slice(1, 2 * n_pairs, 2)) if inter else (slice(0, n_pairs), slice(n_pairs, 2 * n_pairs))
    y[..., ia[0]], y[..., ia[1]] = a * c - b * s, a * s + b * c
    mag = mag.clone()
    mag[..., ia[0]], mag[..., ia[1]] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, mag


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("rows,heads,kv,hd,n_pairs,inter,norm,block", [
    (1, 24, 24, 64, 32, True, True, 16), (37, 8, 2, 128, 64, False, True, 16), (130, 3, 1, 64, 16, False, False, 1), (19, 7, 7, 128, 32, True, True, 64),
    (5, 1, 1, 64, 8, False, True, 1024), (260, 6, 3, 128, 64, True, False, 8)])
def test_rope_cache(dev, dt, rows, heads, kv, hd, n_pairs, inter, norm, block):
    """Every row type against float64: written rows within the roundings of 32-bit arithmetic plus the one to dt, v bit for bit; skipped rows (slot
    or position -1 or out of range) leave q_out and the caches as they were.  Fused-row and (slot, head) orders by strides."""
    from mars5_tts_amd import ops
    g = torch.Generator().manual_seed(rows + hd)
    n_pos, n_blocks = 301, rows // block + 3
    wide = torch.randn(rows, (heads + 2 * kv) * hd + 16, generator=g).to(dt)
    qkv = wide.to(dev)[:, 8:8 + (heads + 2 * kv) * hd]                            # a row stride that is not the width
    qw = (torch.rand(hd, generator=g) + 0.5).to(dev) if norm else None
    kw = (torch.rand(hd, generator=g) + 0.5).to(dev) if norm else None
    ang = torch.rand(n_pos, n_pairs, generator=g) * 6.283
    rope = torch.stack([ang.cos(), ang.sin()], -1).to(dev).contiguous()
    pos = torch.randint(0, n_pos, (rows,), generator=g, dtype=torch.int32)
    slot = torch.randperm(n_blocks * block, generator=g)[:rows].int()
    bad = set()
    if rows > 4:
        for r, (p, s) in zip((0, 2, 3, rows - 1), ((-1, 5), (4, -1), (n_pos, 6), (4, n_blocks * block))):
            pos[r], slot[r] = p, s
            bad.add(r)
    q_out = torch.full((rows, heads, hd), 7.0, dtype=dt, device=dev)
    kc = torch.full((n_blocks, block, kv, hd), 9.0, dtype=dt, device=dev).permute(0, 2, 1, 3)        # (block, slot, head) in memory
    vc = torch.full((n_blocks, kv, block, hd), 9.0, dtype=dt, device=dev)
    vc = torch.cat([vc, vc], 3)[..., :hd]                                                            # rows twice as far apart
    vc = vc if vc.stride(3) == 1 else vc.contiguous()
    ops.paged_rope_cache(qkv, heads, kv, rope, pos.to(dev), slot.to(dev), q_out, kc, vc, q_norm=qw, k_norm=kw, eps=1e-5, interleaved=inter)
    torch.cuda.synchronize()
    x = qkv.cpu().view(rows, heads + 2 * kv, hd)
    cs = rope.cpu()[pos.long().clamp(0, n_pos - 1)]
    # 32-bit roundings of a feature: 12 in the sum of squares (8 in the lane, 4 across), halved by the square root, 5 to the factor,
    # 2 to the scaled value, 2 to the rotated one: under 16 u32 of the terms' magnitudes; then one rounding to dt
    for part, w, got in ((x[:, :heads], qw, None), (x[:, heads:heads + kv], kw, kc)):
        y, mag = _rope_ref(part, None if w is None else w.cpu(), cs, n_pairs, inter, 1e-5)
        for r in range(rows):
            if r in bad:
                continue
            out = q_out[r].cpu() if got is None else got[int(slot[r]) // block, :, int(slot[r]) % block].cpu()
            err = (out.double() - y[r]).abs()
            lim = (u(dt) if dt != torch.float32 else 0.0) * (y[r].abs() + 16 * U32 * mag[r]) + 16 * U32 * mag[r] + (2.0 ** -25 if dt == torch.float16 else 0.0)
            assert bool((err <= lim).all()), (r, float((err - lim).max()))
    for r in range(rows):
        if r not in bad:
            assert torch.equal(vc[int(slot[r]) // block, :, int(slot[r]) % block].cpu(), x[r, heads + kv:])
        else:
            assert bool((q_out[r] == 7.0).all())
    live = {int(s) for r, s in enumerate(slot.tolist()) if r not in bad}
    for c in (kc, vc):
        flat = c.permute(0, 2, 1, 3).reshape(n_blocks * block, kv, hd).cpu()
        rest = [s for s in range(n_blocks * block) if s not in live]
        assert bool((flat[rest] == 9.0).all())


def test_rope_cache_in_place(dev):
    """q_out may be the q part of qkv itself."""
    from mars5_tts_amd import ops, tables
    rope = tables.rope_table(128, 100).to(dev)
    for dt in DTS:
        for rows in (5, 1500):
            qkv = torch.randn(rows, 12 * 128, generator=torch.Generator().manual_seed(3)).to(dt).to(dev)
            pos = torch.randint(0, 100, (rows,), generator=torch.Generator().manual_seed(4)).int().to(dev)
            slot = torch.arange(rows, dtype=torch.int32, device=dev)
            w = torch.rand(128, generator=torch.Generator().manual_seed(5)).to(dev)
            kc, vc, kc2, vc2 = (torch.zeros(rows // 16 + 1, 2, 16, 128, dtype=dt, device=dev) for _ in range(4))
            q = torch.zeros(rows, 8, 128, dtype=dt, device=dev)
            ops.paged_rope_cache(qkv, 8, 2, rope, pos, slot, q, kc, vc, q_norm=w, k_norm=w, interleaved=False)
            ops.paged_rope_cache(qkv, 8, 2, rope, pos, slot, qkv[:, :8 * 128].view(rows, 8, 128), kc2, vc2, q_norm=w, k_norm=w, interleaved=False)
            torch.cuda.synchronize()
            assert torch.equal(qkv[:, :8 * 128].view(rows, 8, 128), q) and torch.equal(kc, kc2) and torch.equal(vc, vc2)


def test_rope_cache_matches_the_contiguous_form(dev):
    """No norms, adjacent pairs, one page per request: the values of rope_cache, bit for bit (the same products in the same order)."""
    from mars5_tts_amd import ops, tables
    H, M, W = 24, 33, 64
    rope = tables.rope_table(64, 200).to(dev)
    for dt in DTS:
        qkv = torch.randn(M, 3 * H * 64, generator=torch.Generator().manual_seed(3)).to(dt).to(dev)
        q1, k1, v1 = (torch.zeros(H, W, 64, dtype=dt, device=dev) for _ in range(3))
        vt = torch.zeros(H, 64, W, dtype=dt, device=dev)
        ops.rope_cache(qkv, H, 7, rope, q1, k1, v1, W * 64, W, vt, 64 * W, W)
        q2 = torch.zeros(M, H, 64, dtype=dt, device=dev)
        k2, v2 = torch.zeros(1, H, W, 64, dtype=dt, device=dev), torch.zeros(1, H, W, 64, dtype=dt, device=dev)
        pos = torch.arange(7, 7 + M, dtype=torch.int32, device=dev)
        ops.paged_rope_cache(qkv, H, H, rope, pos, pos, q2, k2, v2)
        torch.cuda.synchronize()
        assert torch.equal(k1, k2[0]) and torch.equal(v1, v2[0])
        assert torch.equal(q1.view(-1)[:H * M * 64].view(H, M, 64), q2.transpose(0, 1))


# ------------------------------------------------------------------------------------------------------- paged_attention
class Cache:
    """Random paged cache with NaN wherever no request's position lies; pages in random order."""

    def __init__(self, lens, kv, hd, dt, block, dev, seed, nhd=False, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 0) // block) for n in lens]
        self.n_blocks, self.block, self.width = sum(need) + 3, block, max(need + [1]) + 2
        order = torch.randperm(self.n_blocks, generator=g)
        self.table = torch.full((len(lens), self.width), -5, dtype=torch.int32)
        k = torch.full((self.n_blocks, kv, block, hd), float("nan"), dtype=dt)
        v = k.clone()
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]].int()
            at += need[b]
            kk = (torch.randn(max(n, 0), kv, hd, generator=g) * scale).to(dt)
            vv = torch.randn(max(n, 0), kv, hd, generator=g).to(dt)
            self.k.append(kk)
            self.v.append(vv)
            j = torch.arange(max(n, 0))
            blk = self.table[b].long()[j // block] if n > 0 else j
            k[blk, :, j % block] = kk
            v[blk, :, j % block] = vv
        self.kd = k.to(dev) if not nhd else k.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3)
        self.vd = v.to(dev) if not nhd else v.permute(0, 2, 1, 3).contiguous().to(dev).permute(0, 2, 1, 3)
        self.table_d = self.table.to(dev)


def _attn_ref(q, k, v, new, window, scale, hide=None):
    """One request in float64: (o, A, S, visible): o (new, H, hd), A = sum p |v|, S = max |q||k| scale of a score, visible key counts."""
    n, kv, hd = k.shape
    H = q.shape[1]
    rep = H // kv
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    pos = torch.arange(n - new, n)[:, None]
    key = torch.arange(n)[None]
    vis = key <= pos
    if window:
        vis = vis & (key > pos - window)
    if hide is not None:
        vis = vis & ~hide[None]
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * scale
    mag = torch.einsum("ihd,jhd->hij", q.double().abs(), kk.abs()) * scale
    s = s.masked_fill(~vis[None], -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
    tot = p.sum(-1, keepdim=True)
    p = torch.where(tot > 0, p / tot.clamp(min=1e-300), torch.zeros_like(p))
    vv = torch.where(vis.any(0)[:, None, None], vv, torch.zeros_like(vv))
    o = torch.einsum("hij,jhd->ihd", p, vv)
    A = torch.einsum("hij,jhd->ihd", p, vv.abs())
    S = torch.where(vis[None], mag, torch.zeros_like(mag)).amax(-1).T if n else torch.zeros(new, H)
    V = vv.abs().amax(0) if n else torch.zeros(H, hd, dtype=torch.float64)
    return o, A, S, vis.sum(1), V


def _attn_limit(o, A, S, count, V, dt, hd):
    """Bound of |kernel - o|.  A score is off by (hd + 3) u32 of its magnitude S (products and sums, scale, the exponent's argument: another
    u32 S log2 e for the subtraction), an exponential by 4 u32, a probability by u(dt) when it is rounded to the operand type (fp16: at least
    half a subnormal step of the largest probability's unit, 2^-25, per key), the sums by a chain of at most count / 64 + 80 terms each, the merge
    of at most 64 splits by 64 more; every one of these moves o by at most its relative size times A, twice (numerator and denominator)."""
    rel = 2 * ((hd + 8) * U32 * S + 4 * U32 + (count.double()[:, None] / 64 + 80 + 64) * U32)
    lim = A * rel[..., None]
    if dt != torch.float32:
        lim = lim + A * u(dt) * 1.01 + o.abs() * u(dt)
    if dt == torch.float16:
        lim = lim + count.double()[:, None, None] * 2.0 ** -25 * V[None] + 2.0 ** -25
    return lim * 1.02 + 1e-30


def _run_attn(dev, dt, ctx, new, heads, kv, hd, block, window=0, seed=0, nhd=False, split=True, pad=3, scale=None, qscale=1.0, max_new=None, stream=None):
    from mars5_tts_amd import ops
    lens = [c + n for c, n in zip(ctx, new)]
    c = Cache(lens, kv, hd, dt, block, dev, seed, nhd)
    rows = sum(new)
    g = torch.Generator().manual_seed(seed + 1)
    wide = (torch.randn(rows + pad, heads + 2, hd, generator=g) * qscale).to(dt).to(dev)
    q = wide[:, 1:1 + heads]                                            # a view of a wider buffer
    out = torch.full((rows + pad, heads, hd), 7.0, dtype=dt, device=dev)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    ws = split if torch.is_tensor(split) else (torch.zeros(24 << 20, dtype=torch.uint8, device=dev) if split else None)
    args = (q, c.kd, c.vd, c.table_d, _i32(lens, dev), _i32(start, dev), out)
    ops.paged_attention(*args, scale=scale, window=window, max_new=max(new + [1]) if max_new is None else max_new, workspace=ws, stream=stream)
    torch.cuda.synchronize()
    assert bool((out[rows:] == 7.0).all()), "padding rows were written"
    sc = hd ** -0.5 if scale is None else scale
    worst = 0.0
    for b, n in enumerate(new):
        if n == 0:
            continue
        o, A, S, count, V = _attn_ref(q[start[b]:start[b + 1]].cpu(), c.k[b], c.v[b], n, window, sc)
        got = out[start[b]:start[b + 1]].cpu().double()
        lim = _attn_limit(o, A, S, count, V, dt, hd)
        assert bool(torch.isfinite(got).all()), f"request {b}: not finite"
        bad = (got - o).abs() > lim
        assert not bool(bad.any()), (b, int(bad.sum()), float((got - o).abs().max()), float(lim.max()))
        worst = max(worst, float(((got - o).abs() / lim).max()))
    return c, args, ws, worst


SHAPES = [(24, 24, 64, 16), (8, 2, 128, 16), (7, 1, 64, 8), (32, 2, 128, 64), (3, 3, 128, 1), (12, 4, 64, 128)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("heads,kv,hd,block", SHAPES)
def test_attention_single_tokens(dev, dt, heads, kv, hd, block):
    """One token per request, lengths around the tile and page borders, requests without tokens, with and without splitting."""
    ctx = [0, 1, 15, 16, 17, 62, 63, 64, 65, 127, 0, 300]
    new = [1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 0, 1]
    for split in (True, False):
        _run_attn(dev, dt, ctx, new, heads, kv, hd, block, seed=heads, split=split)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("heads,kv,hd,block", SHAPES)
def test_attention_drafts(dev, dt, heads, kv, hd, block):
    """A few tokens per request: the packed (token, head) rows pass one tile of 16, 32 for some."""
    _run_attn(dev, dt, [5, 0, 63, 130, 700, 33], [5, 3, 2, 8, 4, 1], heads, kv, hd, block, seed=heads + 1)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("heads,kv,hd,block,nhd", [(24, 24, 64, 16, True), (8, 2, 128, 16, False), (7, 1, 64, 8, True), (4, 4, 128, 64, False)])
def test_attention_chunks(dev, dt, heads, kv, hd, block, nhd):
    """Prompt chunks: the first (no cached positions), odd lengths, beside single tokens; both cache orders."""
    _run_attn(dev, dt, [0, 37, 200, 90, 0], [129, 64, 1, 257, 31], heads, kv, hd, block, seed=heads + 2, nhd=nhd)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("heads,kv,hd,block", [(6, 2, 64, 1), (2, 2, 64, 4), (4, 1, 128, 2), (3, 3, 128, 1), (5, 5, 64, 1024)])
def test_attention_small_and_large_pages(dev, dt, heads, kv, hd, block):
    """Pages of fewer rows than one DMA instruction reads, of one row with more pages than a segment's table holds (1024), and larger than
    any request: single tokens and chunks."""
    _run_attn(dev, dt, [2500, 3, 1100], [1, 2, 1], heads, kv, hd, block, seed=heads + 40)
    _run_attn(dev, dt, [1300, 0, 700], [140, 131, 1], heads, kv, hd, block, seed=heads + 41, window=1200 if hd == 64 else 0)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("n_seq", [63, 64, 65, 300])
def test_attention_many_requests(dev, dt, n_seq):
    """More requests than a wave has lanes, empty ones among them, with a chunk and without, split and not."""
    rng = random.Random(n_seq)
    ctx = [rng.choice([0, 1, 20, 65, 130]) for _ in range(n_seq)]
    new = [rng.choice([0, 1, 1, 2]) for _ in range(n_seq)]
    ctx[n_seq // 2], new[n_seq - 1], new[n_seq // 2] = 1500, 1, 1
    _run_attn(dev, dt, ctx, new, 4, 2, 64, 16, seed=n_seq)
    new[n_seq // 3] = 150
    _run_attn(dev, dt, ctx, new, 4, 2, 64, 16, seed=n_seq, split=n_seq != 64)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_the_longest_list_of_requests(dev, dt, hd):
    """4096 requests: their prefix sums and the rings of every variant fit the LDS together."""
    ctx, new = [0] * 4096, [0] * 4096
    for i, b in enumerate(range(0, 4096, 117)):
        ctx[b], new[b] = 40 * i, 1 + i % 2
    new[4095] = 1
    _run_attn(dev, dt, ctx, new, 2, 1, hd, 16, seed=81)
    new[2000] = 70
    _run_attn(dev, dt, ctx, new, 2, 1, hd, 16, seed=82)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_chunk_split_by_workspace(dev, dt, hd):
    """A chunk with a long context beside single tokens: room for partial results of 128 rows, of few rows only, of none."""
    from mars5_tts_amd import ops
    c, args, ws, _ = _run_attn(dev, dt, [3000, 900, 0, 2000], [150, 1, 3, 1], 4, 2, hd, 16, seed=51)
    first = args[6].clone()
    n = 155
    assert ops.paged_attention_workspace(*args, max_new=150) <= 64 << 20
    for nbytes in (64 << 20, 5 << 20, 1 << 20, 100016, 1600, 0):
        small = torch.zeros(max(nbytes, 16), dtype=torch.uint8, device=dev)[:nbytes]
        for _ in range(2):
            args[6].fill_(3.0)
            ops.paged_attention(*args, max_new=150, workspace=small if nbytes else None)
            torch.cuda.synchronize()
            # both are within a few roundings to dt of the exact result (checked above for the first)
            assert float((args[6][:n].double() - first[:n].double()).abs().max()) <= 4 * u(dt) * max(1.0, float(first[:n].double().abs().max()))
        assert nbytes == 0 or not bool(small[:16].any())                          # the tickets are back at zero


@pytest.mark.parametrize("nbytes", [64 << 20, 24 << 20, 3000064])
def test_attention_one_workspace_for_calls_of_all_shapes(dev, nbytes):
    """The tickets of a call are where the one before it, of another type, head size or tiling, left zeros."""
    ws = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
    calls = [(torch.float32, [3000, 900], [40, 1], 4, 2, 128), (torch.bfloat16, [5000] * 6, [1] * 6, 24, 24, 64), (torch.float16, [4000, 2500, 0], [150, 1, 70], 4, 2, 128),
             (torch.bfloat16, [6000, 3000], [5, 2], 8, 2, 128), (torch.float16, [4000, 1000], [90, 33], 2, 2, 64), (torch.float32, [5000, 0], [1, 1], 3, 3, 64)]
    for turn in range(2):
        for i, (dt, ctx, new, heads, kv, hd) in enumerate(calls):
            _run_attn(dev, dt, ctx, new, heads, kv, hd, 16, seed=61 + i, split=ws)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_partly_filled_large_tiles(dev, dt, hd):
    """33 to 127 packed rows over long contexts: a tile's partial results take as many rows as it has, in 16s."""
    _run_attn(dev, dt, [4000, 2500, 3100, 700], [9, 11, 31, 16], 8, 2, hd, 16, seed=71)


def test_attention_refuses_row_offsets_that_do_not_ascend(dev):
    """Row offsets are device data: offsets that claim rows over and over compute nothing and write nothing."""
    from mars5_tts_amd import ops
    for B in (5, 200):
        c = Cache([40] * B, 2, 64, torch.float16, 16, dev, 3)
        q = torch.randn(600, 4, 64, generator=torch.Generator().manual_seed(1)).half().to(dev)
        out = torch.full((600, 4, 64), 7.0, dtype=torch.float16, device=dev)
        start = [0 if b % 2 == 0 else 600 for b in range(B + 1)]
        for max_new in (1, 600):
            ops.paged_attention(q, c.kd, c.vd, c.table_d, _i32([40] * B, dev), _i32(start, dev), out, max_new=max_new)
            torch.cuda.synchronize()
            assert bool((out == 7.0).all()) or max_new == 600                       # (large tiles: few enough to pass for valid, inside the buffers)
            out.fill_(7.0)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 100])
def test_attention_window(dev, dt, window):
    _run_attn(dev, dt, [0, 300, 64, 129], [70, 1, 5, 130], 6, 3, 64, 16, window=window, seed=window)
    _run_attn(dev, dt, [0, 300, 64, 129], [70, 1, 5, 130], 4, 1, 128, 8, window=window, seed=window + 1)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_window_wider_than_any_request(dev, dt, hd):
    """The largest windows give the bits of window 0, also for requests of fewer positions than new rows (the first rows see nothing)."""
    from mars5_tts_amd import ops
    lens, new = [3, 300, 40], [6, 70, 41]
    c = Cache(lens, 2, hd, dt, 16, dev, 15)
    q = torch.randn(sum(new), 4, hd, generator=torch.Generator().manual_seed(2)).to(dt).to(dev)
    start = [0, 6, 76, 117]
    outs = []
    for window in (0, 1 << 30, (1 << 31) - 1):
        for max_new in (1, 70):
            out = torch.full((sum(new), 4, hd), 7.0, dtype=dt, device=dev)
            ops.paged_attention(q, c.kd, c.vd, c.table_d, _i32(lens, dev), _i32(start, dev), out, window=window, max_new=max_new)
            outs.append(out)
    torch.cuda.synchronize()
    for i in range(2, 6):
        assert torch.equal(outs[i], outs[i % 2]), i
    for out in outs[:2]:
        assert bool((out[:3] == 0).all()) and bool((out[3:6] != 0).any())
        for b, n in enumerate(lens):
            m = min(new[b], n)
            o, A, S, count, V = _attn_ref(q[start[b + 1] - m:start[b + 1]].cpu(), c.k[b], c.v[b], m, 0, hd ** -0.5)
            assert bool(((out[start[b + 1] - m:start[b + 1]].cpu().double() - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)).all()), b


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_long_split(dev, dt, hd):
    """Few rows over a long axis: keys split over many workgroups and joined; a second call on the same workspace, a smaller and an odd-sized one."""
    from mars5_tts_amd import ops
    c, args, ws, _ = _run_attn(dev, dt, [9000, 0, 4099], [1, 1, 3], 8, 2, hd, 16, seed=5)
    first = args[6].clone()
    for nbytes in (ws.shape[0], 5 << 20, 100016, 16):
        small = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
        for _ in range(2):
            args[6].fill_(3.0)
            ops.paged_attention(*args, max_new=3, workspace=small)
            torch.cuda.synchronize()
            lim = 4 * u(dt) + 1e-5
            assert float((args[6][:5].double() - first[:5].double()).abs().max()) <= lim * max(1.0, float(first[:5].double().abs().max()))
    again = args[6].clone()
    ops.paged_attention(*args, max_new=3, workspace=small)
    assert torch.equal(again[:5], args[6][:5])                                    # the same call gives the same bits


def test_attention_large_scores_and_scale(dev):
    """Scores of hundreds: the running maximum moves all the time; a scale of the caller's."""
    for dt in DTS:
        _run_attn(dev, dt, [500, 70], [1, 40], 8, 2, 128, 16, seed=8, qscale=12.0)
        _run_attn(dev, dt, [500, 70], [1, 40], 8, 2, 64, 16, seed=9, scale=0.37)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 6, 2.0 ** 10, 2.0 ** 20])
def test_attention_scores_past_the_exponents_fraction(dev, dt, hd, scale):
    """Scores up to 1e13, positive and negative, where a unit of the last place of a score is many powers of e: the keys of the largest score share
    the weight (the scores here are whole numbers times the scale, exact in 32 bits, and differ by 2^15 scale or not at all)."""
    from mars5_tts_amd import ops
    heads, kv, ctx, new = 4, 2, [2500, 300, 40], [1, 70, 3]
    lens, start = [a + b for a, b in zip(ctx, new)], [0, 1, 71, 74]
    for sign in (1.0, -1.0):
        c = Cache(lens, kv, hd, dt, 16, dev, 29)
        q = torch.zeros(74, heads, hd, dtype=dt)
        q[..., 0] = 32768.0
        g = torch.Generator().manual_seed(8)
        for b, n in enumerate(lens):
            k = torch.zeros(n, kv, hd, dtype=dt)
            k[..., 0] = sign * torch.randint(1, 200, (n, kv), generator=g).to(dt)
            c.k[b] = k
            j = torch.arange(n)
            c.kd[c.table[b].long()[j // 16].to(dev), :, (j % 16).to(dev)] = k.to(dev)
        for max_new in (70, 1):
            for ws in (None, torch.zeros(24 << 20, dtype=torch.uint8, device=dev)):
                out = torch.full((74, heads, hd), 7.0, dtype=dt, device=dev)
                ops.paged_attention(q.to(dev), c.kd, c.vd, c.table_d, _i32(lens, dev), _i32(start, dev), out, scale=scale, max_new=max_new, workspace=ws)
                torch.cuda.synchronize()
                for b in range(3):
                    lo, hi = start[b], start[b + 1]
                    o, A, S, count, V = _attn_ref(q[lo:hi], c.k[b], c.v[b], new[b], 0, scale)
                    bad = ~((out[lo:hi].cpu().double() - o).abs() <= _attn_limit(o, A, torch.zeros_like(S), count, V, dt, hd))
                    assert not bool(bad.any()), (sign, max_new, b, int(bad.sum()))


@pytest.mark.parametrize("dt", DTS)
def test_attention_rows_without_keys_and_bad_pages(dev, dt):
    """seq_len below the number of new rows: the first rows see nothing and give zeros.  Pages out of range are not seen, a row whose
    pages are all bad gives zeros; lengths past the table's capacity are cut there."""
    from mars5_tts_amd import ops
    heads, kv, hd, block = 4, 2, 64, 16
    c = Cache([3, 100, 40, 64], kv, hd, dt, block, dev, 11)
    new = [5, 70, 2, 1]
    start = [0, 5, 75, 77, 78]
    q = torch.randn(78, heads, hd, generator=torch.Generator().manual_seed(2)).to(dt).to(dev)
    table = c.table.clone()
    table[1, 2], table[1, 4] = -1, c.n_blocks                                     # keys 32-47 and 64-79 of request 1
    table[2, :] = 1 << 30                                                         # all of request 2
    td = table[:, :4 + 3].to(dev)
    for max_new in (70, 1):
        for ws in (None, torch.zeros(1 << 20, dtype=torch.uint8, device=dev)):
            out = torch.full((78, heads, hd), 7.0, dtype=dt, device=dev)
            ops.paged_attention(q, c.kd, c.vd, td, _i32([3, 100, 40, 64], dev), _i32(start, dev), out, max_new=max_new, workspace=ws)
            torch.cuda.synchronize()
            got = out.cpu().double()
            assert bool((got[:2] == 0).all()) and bool((got[75:77] == 0).all())
            hide = torch.zeros(100, dtype=torch.bool)
            hide[32:48] = True
            hide[64:80] = True
            for b, h in ((0, None), (1, hide), (3, None)):
                lo, hi = start[b], start[b + 1]
                vv = c.v[b]
                o, A, S, count, V = _attn_ref(q[lo:hi].cpu()[-min(new[b], len(vv)):], c.k[b], vv, min(new[b], len(vv)), 0, hd ** -0.5, h)
                assert bool(((got[hi - o.shape[0]:hi] - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)).all()), b
    # capacity: 2 pages of table for a claimed length of 1000
    t2 = c.table[3:4, :2].contiguous().to(dev)
    out = torch.zeros(1, heads, hd, dtype=dt, device=dev)
    ops.paged_attention(q[77:78], c.kd, c.vd, t2, _i32([1000], dev), _i32([0, 1], dev), out)
    o, A, S, count, V = _attn_ref(q[77:78].cpu(), c.k[3][:32], c.v[3][:32], 1, 0, hd ** -0.5)
    assert bool(((out.cpu().double() - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)).all())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), "lowest"])
def test_attention_masked_places_do_not_leak(dev, dt, value):
    """Keys and values that a row does not see (later tokens of its own chunk, positions before its window) may hold anything: rows
    that do not see them come out as if they were not there."""
    from mars5_tts_amd import ops
    value = torch.finfo(dt).min if value == "lowest" else value
    for heads, kv, hd, new, n, window in ((4, 2, 64, 70, 100, 0), (4, 4, 128, 9, 60, 0), (2, 1, 64, 40, 300, 50), (8, 1, 128, 2, 64, 0)):
        c = Cache([n], kv, hd, dt, 16, dev, 13)
        q = torch.randn(new, heads, hd, generator=torch.Generator().manual_seed(4)).to(dt).to(dev)
        at = n - new // 2                                            # poisoned: one of the chunk's own positions and one old one
        old = n - new - 1 if window else None
        for p in (at, old):
            if p is not None:
                blk = int(c.table[0, p // 16])
                c.kd[blk, :, p % 16] = value
                c.vd[blk, :, p % 16] = value
        out = torch.zeros(new, heads, hd, dtype=dt, device=dev)
        ops.paged_attention(q, c.kd, c.vd, c.table_d, _i32([n], dev), _i32([0, new], dev), out, window=window, max_new=new)
        torch.cuda.synchronize()
        o, A, S, count, V = _attn_ref(q.cpu(), c.k[0], c.v[0], new, window, hd ** -0.5)
        lim = _attn_limit(o, A, S, count, V, dt, hd)
        got = out.cpu().double()
        for i in range(new):
            pos = n - new + i
            sees = [p for p in (at, old) if p is not None and p <= pos and (not window or p > pos - window)]
            if not sees:
                assert bool(((got[i] - o[i]).abs() <= lim[i]).all()), (heads, hd, i)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[1, 2], [5, 1], [90, 1]])
def test_attention_nan_that_a_row_sees(dev, dt, hd, new):
    """A NaN in a query's row, or in all keys of one kv head over a range as long as a chunk: exactly those heads of the rows that see it come out as
    NaN, whether their keys are split over workgroups or not; all others as if it were not there."""
    from mars5_tts_amd import ops
    heads, kv, ctx, far = 4, 2, [3000, 1500], 2000
    lens, rows = [a + b for a, b in zip(ctx, new)], sum(new)
    start = [0, new[0], rows]
    for where in ("query", "keys"):
        c = Cache(lens, kv, hd, dt, 16, dev, 17)
        q = torch.randn(rows, heads, hd, generator=torch.Generator().manual_seed(3)).to(dt)
        poisoned = torch.zeros(rows, heads, dtype=torch.bool)
        qd = q.to(dev)
        if where == "query":
            qd[new[0] - 1, 1, 5] = float("nan")
            qd[rows - 1, 2, 0] = float("nan")
            poisoned[new[0] - 1, 1] = poisoned[rows - 1, 2] = True
        else:
            c.kd[c.table[0, :far // 16].long().to(dev), 1] = float("nan")        # request 0, its first 2000 keys, kv head 1
            poisoned[:new[0], 2:] = True
        for ws in (None, torch.zeros(24 << 20, dtype=torch.uint8, device=dev), torch.zeros(1 << 20, dtype=torch.uint8, device=dev)):
            out = torch.full((rows, heads, hd), 7.0, dtype=dt, device=dev)
            ops.paged_attention(qd, c.kd, c.vd, c.table_d, _i32(lens, dev), _i32(start, dev), out, max_new=max(new), workspace=ws)
            torch.cuda.synchronize()
            got = out.cpu().double()
            assert bool(torch.isnan(got[poisoned]).all()), (where, "a NaN was lost")
            for b in range(2):
                lo, hi = start[b], start[b + 1]
                o, A, S, count, V = _attn_ref(q[lo:hi], c.k[b], c.v[b], new[b], 0, hd ** -0.5)
                fine = (got[lo:hi] - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)
                assert bool((fine | poisoned[lo:hi, :, None]).all()), (where, b)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[1, 2], [90, 1]])
def test_attention_scores_of_minus_infinity(dev, dt, hd, new):
    """Keys whose score is -inf have no weight; a row all of whose scores are -inf gets zeros, as one that sees no key; split and not."""
    from mars5_tts_amd import ops
    heads, kv, ctx = 4, 2, [3000, 700]
    lens, rows = [a + b for a, b in zip(ctx, new)], sum(new)
    start = [0, new[0], rows]
    c = Cache(lens, kv, hd, dt, 16, dev, 18)
    q = torch.randn(rows, heads, hd, generator=torch.Generator().manual_seed(4)).to(dt)
    q[..., 0] = 1.0                                                              # so a key of -inf in feature 0 scores -inf
    hide = torch.zeros(lens[0], dtype=torch.bool)
    hide[512:1900] = True                                                        # request 0: whole chunks of its keys and parts of others
    hide[2999] = True
    for p in hide.nonzero()[:, 0].tolist():
        c.kd[int(c.table[0, p // 16]), :, p % 16, 0] = -float("inf")
    c.kd[c.table[1, :-(-lens[1] // 16)].long().to(dev), :, :, 0] = -float("inf")     # request 1: all of them
    for ws in (None, torch.zeros(24 << 20, dtype=torch.uint8, device=dev)):
        out = torch.full((rows, heads, hd), 7.0, dtype=dt, device=dev)
        ops.paged_attention(q.to(dev), c.kd, c.vd, c.table_d, _i32(lens, dev), _i32(start, dev), out, max_new=max(new), workspace=ws)
        torch.cuda.synchronize()
        got = out.cpu().double()
        o, A, S, count, V = _attn_ref(q[:new[0]], c.k[0], c.v[0], new[0], 0, hd ** -0.5, hide)
        assert bool(((got[:new[0]] - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)).all())
        assert bool((got[new[0]:] == 0).all())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("heads,kv,hd,new,n,window", [(4, 2, 64, 70, 130, 0), (4, 4, 128, 9, 90, 0), (2, 1, 128, 75, 300, 50), (8, 1, 64, 2, 64, 0), (6, 2, 64, 5, 2500, 0),
                                                      (4, 2, 128, 60, 3000, 0), (1, 1, 64, 1, 5, 0), (4, 1, 128, 4, 1100, 700)])
def test_attention_nonfinite_values_reach_the_rows_that_see_them(dev, dt, heads, kv, hd, new, n, window, split):
    """Infinite and NaN features of VALUES alone: exactly the rows that see the key get +inf, -inf or NaN (both signs: NaN), at exactly those
    features of the kv head's query heads; every other feature and row comes out as if they were finite."""
    from mars5_tts_amd import ops
    inf, nan = float("inf"), float("nan")
    c = Cache([n], kv, hd, dt, 16, dev, 19)
    q = torch.randn(new, heads, hd, generator=torch.Generator().manual_seed(5)).to(dt)
    at = n - 1 - new // 2                                            # seen by the later half of the rows
    spots = [(at, 0, 3, inf), (at, kv - 1, hd - 1, -inf), (min(at + 1, n - 1), 0, 3, -inf), (at, 0, 17, nan), (n - 1, kv - 1, 40, inf), (0, kv - 1, 41, inf),
             (max(n - new - 40, 0), 0, 8, -inf), (max(n - new - 41, 0), 0, 9, nan), (n // 2, 0, 10, inf), (n // 2, 0, 11, -inf)]
    rep = heads // kv
    plus, minus = (torch.zeros(new, heads, hd, dtype=torch.bool) for _ in range(2))
    for (p, h, d), value in {spot[:3]: spot[3] for spot in spots}.items():       # (one value a place: the last)
        c.vd[int(c.table[0, p // 16]), h, p % 16, d] = value
        for i in range(new):
            pos = n - new + i
            if p <= pos and (not window or p > pos - window):
                if not value < 0:
                    plus[i, h * rep:(h + 1) * rep, d] = True
                if not value > 0:
                    minus[i, h * rep:(h + 1) * rep, d] = True
    ws = torch.zeros(24 << 20, dtype=torch.uint8, device=dev) if split else None
    o, A, S, count, V = _attn_ref(q, c.k[0], c.v[0], new, window, hd ** -0.5)
    lim = _attn_limit(o, A, S, count, V, dt, hd)
    for max_new in (new, 1):                                         # (large and small tiles)
        out = torch.full((new, heads, hd), 7.0, dtype=dt, device=dev)
        ops.paged_attention(q.to(dev), c.kd, c.vd, c.table_d, _i32([n], dev), _i32([0, new], dev), out, window=window, max_new=max_new, workspace=ws)
        torch.cuda.synchronize()
        got = out.cpu().double()
        assert bool((got[plus & ~minus] == inf).all()) and bool((got[minus & ~plus] == -inf).all()) and bool(torch.isnan(got[plus & minus]).all())
        finite = ~(plus | minus)
        assert bool(((got - o).abs() <= lim)[finite].all())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ctx", [40, 3000])
def test_attention_row_offsets_claimed_twice(dev, dt, hd, ctx):
    """Row offsets that do not ascend, over a buffer with guards: requests that claim the same rows compute nothing or those rows (they hold the same
    positions here, so the result is theirs); nothing outside the claimed rows is written, with and without
    room to split, and the workspace is left ready."""
    from mars5_tts_amd import ops
    rows, heads, kv = 100, 4, 2
    c = Cache([ctx + rows], kv, hd, dt, 16, dev, 23)
    q = torch.randn(rows, heads, hd, generator=torch.Generator().manual_seed(6)).to(dt)
    o, A, S, count, V = _attn_ref(q, c.k[0], c.v[0], rows, 0, hd ** -0.5)
    lim = _attn_limit(o, A, S, count, V, dt, hd)
    qd = torch.zeros(rows + 64, heads, hd, dtype=dt, device=dev)
    qd[:rows] = q.to(dev)
    for B in (5, 201):
        table = c.table.expand(B, -1).contiguous().to(dev)
        start = [0 if b % 2 == 0 else rows for b in range(B + 1)]            # 0 .. rows, rows .. 0, 0 .. rows, ...
        for max_new in (1, rows):
            for ws in (None, torch.zeros(24 << 20, dtype=torch.uint8, device=dev), torch.zeros(200000, dtype=torch.uint8, device=dev)):
                buf = torch.full((rows + 128, heads, hd), 7.0, dtype=dt, device=dev)
                out = buf[32:32 + rows + 64]
                ops.paged_attention(qd, c.kd, c.vd, table, _i32([ctx + rows] * B, dev), _i32(start, dev), out, max_new=max_new, workspace=ws)
                torch.cuda.synchronize()
                assert bool((buf[:32] == 7.0).all()) and bool((buf[32 + rows:] == 7.0).all())
                got = out[:rows].cpu().double()
                nothing = bool((got == 7.0).all())
                assert nothing or bool(((got - o).abs() <= lim).all())
                if max_new == 1:
                    assert nothing                                           # more small tiles than the rows can make
                elif B == 5 and dt != torch.float32:
                    assert not nothing                                       # few enough large ones to pass for valid
                if ws is not None:
                    ops.paged_attention(qd[:rows], c.kd, c.vd, table[:1], _i32([ctx + rows], dev), _i32([0, rows], dev), out[:rows], max_new=max_new, workspace=ws)
                    torch.cuda.synchronize()
                    assert bool(((out[:rows].cpu().double() - o).abs() <= lim).all()) and not bool(ws[:160].any())


def test_attention_offsets_past_32_bits(dev):
    """Block strides so far apart that byte and element offsets pass 2^31: two blocks at the ends of a cache of 2.3e9 elements."""
    from mars5_tts_amd import ops
    heads, kv, hd, block = 2, 1, 64, 16
    far = (1 << 31) + (1 << 20)                                      # elements between blocks 0 and 1
    for dt in (torch.float16,):
        big = torch.zeros(far + block * hd, dtype=dt, device=dev)
        kc = big.as_strided((2, kv, block, hd), (far, block * hd, hd, 1))
        kk = torch.randn(20, hd, generator=torch.Generator().manual_seed(1)).to(dt)
        kc[1, 0], kc[0, 0, :4] = kk[:16].to(dev), kk[16:].to(dev)
        q = torch.randn(1, heads, hd, generator=torch.Generator().manual_seed(2)).to(dt).to(dev)
        out = torch.zeros(1, heads, hd, dtype=dt, device=dev)
        ops.paged_attention(q, kc, kc, _i32([[1, 0]], dev), _i32([20], dev), _i32([0, 1], dev), out)
        o, A, S, count, V = _attn_ref(q.cpu(), kk[:, None], kk[:, None], 1, 0, hd ** -0.5)
        assert bool(((out.cpu().double() - o).abs() <= _attn_limit(o, A, S, count, V, dt, hd)).all())
        # and written there
        rope = torch.tensor([[1.0, 0.0]] * 32, device=dev)[None].contiguous()
        qkv = torch.randn(1, 4 * hd, generator=torch.Generator().manual_seed(3)).to(dt).to(dev)
        ops.paged_rope_cache(qkv, 2, 1, rope, _i32([0], dev), _i32([block + 5], dev), out, kc, kc)
        assert torch.equal(kc[1, 0, 5], qkv[0, 3 * hd:]) or torch.equal(kc[1, 0, 5], qkv[0, 2 * hd:3 * hd])
        del big, kc
    torch.cuda.empty_cache()


def test_attention_graph_replay_and_streams(dev):
    """Captured calls on a stream of their own, replayed with other lengths, tables and queries and with eager work in between; two graphs that
    share a workspace one after the other; every replay equals the eager call bit for bit."""
    from mars5_tts_amd import ops
    heads, kv, hd, block, B, cap = 8, 2, 128, 16, 4, 12
    dt = torch.bfloat16
    side = torch.cuda.Stream(device=dev)
    c = Cache([2000, 50, 700, 3], kv, hd, dt, block, dev, 21)
    q = torch.randn(cap, heads, hd, generator=torch.Generator().manual_seed(2)).to(dt).to(dev)
    seq, start = _i32([2000, 50, 700, 3], dev), _i32([0, 1, 3, 4, 5], dev)
    ws = torch.zeros(8 << 20, dtype=torch.uint8, device=dev)
    outs = [torch.zeros(cap, heads, hd, dtype=dt, device=dev) for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for o, window in zip(outs, (0, 64)):
        g = ops.Graph()
        g.begin(side.cuda_stream)
        ops.paged_attention(q, c.kd, c.vd, c.table_d, seq, start, o, window=window, max_new=4, workspace=ws, stream=side.cuda_stream)
        g.end(side.cuda_stream)
        graphs.append(g)
    steps = [([2000, 50, 700, 3], [0, 1, 3, 4, 5]), ([1999, 1, 64, 2], [0, 4, 4, 8, 10]), ([17, 50, 699, 0], [0, 0, 2, 3, 3]), ([2000, 50, 700, 3], [0, 1, 3, 4, 5])]
    for i, (lens, st) in enumerate(steps):
        seq.copy_(_i32(lens, dev))
        start.copy_(_i32(st, dev))
        q.copy_(torch.randn(cap, heads, hd, generator=torch.Generator().manual_seed(30 + i)).to(dt))
        torch.cuda.synchronize()
        for g in graphs:
            g.launch(side.cuda_stream)
        side.synchronize()
        for o, window in zip(outs, (0, 64)):
            eager = torch.zeros(cap, heads, hd, dtype=dt, device=dev)
            ops.paged_attention(q, c.kd, c.vd, c.table_d, seq, start, eager, window=window, max_new=4, workspace=torch.zeros_like(ws))
            torch.cuda.synchronize()
            n = st[-1]
            assert torch.equal(eager[:n], o[:n])


def test_attention_two_at_once(dev):
    """Two calls on two streams, each with a workspace of its own."""
    from mars5_tts_amd import ops
    dt = torch.float16
    c, args, _, _ = _run_attn(dev, dt, [3000, 40, 900], [1, 2, 1], 8, 2, 64, 16, seed=31)
    want = args[6].clone()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    ws = [torch.zeros(8 << 20, dtype=torch.uint8, device=dev) for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, w, o in zip(streams, ws, outs):
            ops.paged_attention(*args[:6], o, max_new=2, workspace=w, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o in outs:
        assert float((o[:4].double() - want[:4].double()).abs().max()) <= 4 * u(dt) * float(want[:4].abs().max())
    assert torch.equal(outs[0], outs[1])


# ---------------------------------------------------------------------------------------------------------- draft_verify
def _verify_ref(target, draft, tokens, start, uni, noise, width, seq=None):
    """The definition, request by request, in IEEE fp32 on the CPU."""
    B, V = noise.shape
    out, n_out, keep = [], [], []
    t = target.float()
    d = None if draft is None else draft.float()
    for b in range(B):
        r0, rows = start[b], start[b + 1] - start[b]
        n, row = min(rows, width), []
        if n == 0:
            out.append([-1] * width)
            n_out.append(0)
            keep.append(None if seq is None else seq[b] - rows)
            continue
        r = r0
        while r < r0 + n - 1:
            tok = int(tokens[r + 1])
            if not 0 <= tok < V:
                break
            q = torch.tensor(1.0) if d is None else d[r, tok]
            if not bool(uni[r] * q < t[r, tok]):
                break
            row.append(tok)
            r += 1
        w = t[r].clone()
        if r < r0 + n - 1:
            if d is None:
                tok = int(tokens[r + 1])
                if 0 <= tok < V:
                    w[tok] = 0.0
            else:
                w = t[r] - d[r]
            if not bool((w > 0).any()):
                w = t[r].clone()
        score = w / noise[b]
        score = torch.where((w > 0) & (score > 0), score, torch.zeros(()))
        row.append(int((score == score.max()).nonzero()[0]))
        out.append(row + [-1] * (width - len(row)))
        n_out.append(len(row))
        keep.append(None if seq is None else seq[b] - rows + len(row))
    return out, n_out, keep


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("V,rows,width", [(1, [1, 2, 0], 3), (7, [1, 4, 5, 0, 2], 5), (1025, [3, 1, 9, 2], 6), (4096, [5] * 9 + [1], 5), (50001, [1, 4, 3], 4), (300, [130, 70, 1], 130)])
@pytest.mark.parametrize("sure", [False, True])
@pytest.mark.parametrize("split", [False, True])
def test_verify(dev, dt, V, rows, width, sure, split):
    """Tokens, counts and kept lengths exactly, over acceptance at every depth, requests without rows, more rows than the output holds,
    vocabularies of one token and of odd sizes; strided probabilities; the workspace used again."""
    from mars5_tts_amd import _lib as L, ops
    g = torch.Generator().manual_seed(V + width)
    R, B = sum(rows), len(rows)
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    z = torch.randn(R, V, generator=g) * 2
    target = torch.softmax(z, -1).to(dt)
    draft = None if sure else torch.softmax(z + torch.randn(R, V, generator=g) * 0.5, -1).to(dt)
    tokens = torch.randint(0, V, (R,), generator=g)
    likely = target.float().argmax(-1)
    pick = torch.rand(R, generator=g) < 0.7
    tokens[1:] = torch.where(pick[:-1], likely[:-1], tokens[1:])
    uni, noise = torch.rand(R, generator=g), torch.empty(B, V).exponential_(generator=g)
    if not sure and R > 4 and V > 1:
        target[1], draft[1] = draft[1].clone(), draft[1].clone()              # nothing left after a rejection: the target itself
        uni[1] = 1.0
    seq = [n + 5 for n in rows]
    want = _verify_ref(target, draft, tokens, start, uni, noise, width, seq)
    wide = torch.zeros(R, V + 5, dtype=dt)
    wide[:, 3:3 + V] = target
    td = wide.to(dev)[:, 3:3 + V]
    ws = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev) if split else None
    outw = torch.full((B, width + 2), 99, dtype=torch.int64, device=dev)
    out, n_out, keep = outw[:, 1:1 + width], _i32([9] * B, dev), _i32([9] * B, dev)
    for _ in range(2):
        out.fill_(98)
        ops.draft_verify(td, None if draft is None else draft.to(dev), tokens.to(dev), _i32(start, dev), uni.to(dev), noise.to(dev), out, n_out, seq_len=_i32(seq, dev), keep_len=keep,
                         workspace=ws)
        torch.cuda.synchronize()
        assert out.tolist() == want[0] and n_out.tolist() == want[1] and keep.tolist() == want[2]
    assert bool((outw[:, 0] == 99).all()) and bool((outw[:, -1] == 99).all())


@pytest.mark.parametrize("split", [False, True])
def test_verify_odd_values(dev, split):
    """NaN and infinite probabilities, zero and infinite noise, ids out of range, ties, all-zero rows: the definition, exactly."""
    from mars5_tts_amd import _lib as L, ops
    inf, nan = float("inf"), float("nan")
    V = 6000
    rows = [2, 2, 2, 2, 1, 1, 2, 1]
    start = [0]
    for n in rows:
        start.append(start[-1] + n)
    R, B = sum(rows), len(rows)
    g = torch.Generator().manual_seed(3)
    target = torch.softmax(torch.randn(R, V, generator=g), -1)
    draft = torch.softmax(torch.randn(R, V, generator=g), -1)
    tokens = torch.randint(0, V, (R,), generator=g)
    uni, noise = torch.rand(R, generator=g), torch.empty(B, V).exponential_(generator=g)
    target[0, int(tokens[1])] = nan                                   # NaN target of a draft: not accepted
    target[0, 5000] = inf
    tokens[3] = V                                                     # ids out of range: not accepted
    tokens[5] = -1
    target[6] = 0.0                                                   # p = 0: u q < 0 never holds; residual empty; the row is all zero
    target[8] = 0.25                                                  # ties: the lowest index
    noise[4] = 1.0
    target[9] = nan                                                   # nothing to draw from: 0
    draft[10, int(tokens[11])] = nan                                  # NaN draft: not accepted
    noise[7, 4321] = 0.0                                              # an infinite weight wins
    noise[6, :100] = inf
    want = _verify_ref(target, draft, tokens, start, uni, noise, 2)
    assert want[0][4] == [0, -1] and want[0][5] == [0, -1] and want[0][7] == [4321, -1] and want[0][3] == [0, -1]
    ws = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev) if split else None
    out, n_out = torch.zeros(B, 2, dtype=torch.int64, device=dev), _i32([0] * B, dev)
    ops.draft_verify(target.to(dev), draft.to(dev), tokens.to(dev), _i32(start, dev), uni.to(dev), noise.to(dev), out, n_out, workspace=ws)
    torch.cuda.synchronize()
    assert out.tolist() == want[0] and n_out.tolist() == want[1]


def test_verify_split_graph_replay(dev):
    """A captured verification whose rows are split over workgroups, replayed with other inputs and eager work in between, refused steps among
    them: every replay equals the eager call, and the workspace is left ready."""
    from mars5_tts_amd import _lib as L, ops
    B, V, rows, width = 4, 20011, [3, 1, 5, 2], 5
    start = [0, 3, 4, 9, 11]
    side = torch.cuda.Stream(device=dev)
    g = torch.Generator().manual_seed(31)
    fixed = dict(target=torch.zeros(11, V, device=dev), draft=torch.zeros(11, V, device=dev), tokens=torch.zeros(11, dtype=torch.int64, device=dev), row_start=_i32(start, dev),
                 uniforms=torch.zeros(11, device=dev), noise=torch.ones(B, V, device=dev))
    seq, state = _i32([9, 8, 7, 6], dev), _i32([0] * L.PST_WORDS, dev)
    ws = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev)
    outs = [(torch.zeros(B, width, dtype=torch.int64, device=dev), _i32([0] * B, dev), _i32([0] * B, dev)) for _ in range(2)]

    def call(o, work, stream=None):
        ops.draft_verify(*fixed.values(), o[0], o[1], seq_len=seq, keep_len=o[2], workspace=work, stream=stream, plan_state=state)

    torch.cuda.synchronize()
    graph = ops.Graph()
    graph.begin(side.cuda_stream)
    call(outs[0], ws, side.cuda_stream)
    graph.end(side.cuda_stream)
    for i in range(6):
        target = torch.softmax(torch.randn(11, V, generator=g) * 2, -1)
        fixed["target"].copy_(target)
        fixed["draft"].copy_(torch.softmax(torch.randn(11, V, generator=g) * 2, -1))
        tokens = torch.randint(0, V, (11,), generator=g)
        tokens[1:] = torch.where(torch.rand(10, generator=g) < 0.8, target.argmax(-1)[:-1], tokens[1:])
        fixed["tokens"].copy_(tokens)
        fixed["uniforms"].copy_(torch.rand(11, generator=g))
        fixed["noise"].copy_(torch.empty(B, V).exponential_(generator=g))
        state[L.PST_STATUS] = 3 if i == 2 else 0
        for o in outs:
            o[2].fill_(50 + i)
        torch.cuda.synchronize()
        graph.launch(side.cuda_stream)
        side.synchronize()
        call(outs[1], None)
        torch.cuda.synchronize()
        for a, b in zip(*outs):
            assert torch.equal(a, b), i
        assert (outs[0][2].tolist() == [52] * B and bool((outs[0][0] == -1).all())) if i == 2 else int(outs[0][1].min()) >= 1
        assert not bool(ws.any())


def test_verify_keeps_the_targets_distribution(dev):
    """The first token that comes out of a drafted step is distributed as the target, whatever the draft: 20000 requests over 5 tokens, counts
    within 5 standard deviations."""
    from mars5_tts_amd import ops
    B, V = 20000, 5
    g = torch.Generator().manual_seed(12)
    p, q = torch.tensor([0.05, 0.4, 0.2, 0.05, 0.3]), torch.tensor([0.3, 0.1, 0.2, 0.35, 0.05])
    target = p.expand(2 * B, V).contiguous()
    draft = q.expand(2 * B, V).contiguous()
    tokens = torch.multinomial(q, 2 * B, replacement=True, generator=g)
    uni, noise = torch.rand(2 * B, generator=g), torch.empty(B, V).exponential_(generator=g)
    out, n_out = torch.zeros(B, 2, dtype=torch.int64, device=dev), _i32([0] * B, dev)
    ops.draft_verify(target.to(dev), draft.to(dev), tokens.to(dev), torch.arange(0, 2 * B + 1, 2, dtype=torch.int32, device=dev), uni.to(dev), noise.to(dev), out, n_out)
    count = torch.bincount(out[:, 0].cpu(), minlength=V).double()
    for v in range(V):
        sd = math.sqrt(B * float(p[v]) * (1 - float(p[v])))
        assert abs(float(count[v]) - B * float(p[v])) < 5 * sd


# ------------------------------------------------------------------------------------------------ together, as they are used
class _TinyLM:
    """Two layers of attention over random weights in fp32, with the paged operators for everything that touches the cache."""

    def __init__(self, dev, heads=4, kv=2, hd=64, vocab=61, layers=2, seed=0):
        from mars5_tts_amd import tables
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv, self.hd, self.vocab, self.dev = heads, kv, hd, vocab, dev
        D = heads * hd
        self.emb = torch.randn(vocab, D, generator=g)
        self.wqkv = [torch.randn((heads + 2 * kv) * hd, D, generator=g) / math.sqrt(D) for _ in range(layers)]
        self.wo = [torch.randn(D, D, generator=g) / math.sqrt(D) for _ in range(layers)]
        self.qn, self.kn = torch.rand(hd, generator=g) + 0.5, torch.rand(hd, generator=g) + 0.5
        self.head = torch.randn(vocab, D, generator=g) / math.sqrt(D) * 3
        self.rope = tables.rope_table(hd, 256)

    def to(self, dev):
        for n in ("emb", "qn", "kn", "head", "rope"):
            setattr(self, n + "_d", getattr(self, n).to(dev))
        self.wqkv_d, self.wo_d = [w.to(dev) for w in self.wqkv], [w.to(dev) for w in self.wo]
        return self

    def reference(self, ids):
        """Next-token probabilities after every id of one sequence, float64, no cache."""
        x = self.emb.double()[ids]
        n = len(ids)
        for wqkv, wo in zip(self.wqkv, self.wo):
            y = (x @ wqkv.double().T).view(n, -1, self.hd)
            q, k, v = y[:, :self.heads], y[:, self.heads:self.heads + self.kv], y[:, self.heads + self.kv:]
            cs = self.rope[:n]
            q, _ = _rope_ref(q, self.qn, cs, self.hd // 2, True, 1e-5)
            k, _ = _rope_ref(k, self.kn, cs, self.hd // 2, True, 1e-5)
            o = _attn_ref(q, k, v, n, 0, self.hd ** -0.5)[0]
            x = x + o.reshape(n, -1) @ wo.double().T
        return torch.softmax(x @ self.head.double().T, -1)

    def forward(self, ids, positions, slots, caches, table, seq_len, q_start, rows, max_new, ws):
        from mars5_tts_amd import ops
        x = self.emb_d[ids]
        for (kc, vc), wqkv, wo in zip(caches, self.wqkv_d, self.wo_d):
            qkv = x @ wqkv.T
            q = torch.zeros(rows, self.heads, self.hd, device=self.dev)
            o = torch.zeros_like(q)
            ops.paged_rope_cache(qkv, self.heads, self.kv, self.rope_d, positions, slots, q, kc, vc, q_norm=self.qn_d, k_norm=self.kn_d)
            ops.paged_attention(q, kc, vc, table, seq_len, q_start, o, max_new=max_new, workspace=ws)
            x = x + o.view(rows, -1) @ wo.T
        return torch.softmax(x @ self.head_d.T, -1)


def test_speculative_serving_run(dev):
    """Plan, norm + rotation + cache write, attention and verification in a loop, as a serving program runs them: prompts of several lengths
    admitted at once, then drafted steps whose rejected tokens are rolled back by the next plan, a request retired and another admitted into its blocks.
    The host reads tokens back only to draw the next drafts.  Every step's probabilities equal a cache-free float64 recomputation of the
    sequence that was fed, and the accepted tokens equal the definition applied to the kernel's probabilities."""
    from mars5_tts_amd import _lib as L, ops
    lm = _TinyLM(dev).to(dev)
    B, block, width, n_blocks, K, V = 4, 8, 12, 30, 3, lm.vocab
    g = torch.Generator().manual_seed(5)
    pool = Pool(B, width, n_blocks, block, 1)
    t = pool.tensors(dev)
    nan = float("nan")
    caches = [(torch.full((n_blocks, lm.kv, block, lm.hd), nan, device=dev), torch.full((n_blocks, lm.kv, block, lm.hd), nan, device=dev)) for _ in range(2)]
    ws = torch.zeros(4 << 20, dtype=torch.uint8, device=dev)
    ws2 = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev)
    seqs = [torch.randint(0, V, (n,), generator=g).tolist() for n in (1, 17, 30, 8)]        # ids fed so far (kept)
    keep = _i32([0] * B, dev)
    feed = [s[:] for s in seqs]
    total = 0
    for step in range(9):
        new = [len(f) for f in feed]
        rows = sum(new) + 2                                                      # a launch of fixed size: two padding rows
        q_start, slots, pos = _i32([0] * (B + 1), dev), _i32([0] * rows, dev), _i32([0] * rows, dev)
        ops.paged_plan(t["seq_len"], keep, _i32(new, dev), t["table"], t["free"], t["state"], block, q_start, slots, pos)
        assert int(t["state"][L.PST_STATUS]) == 0
        ids = torch.tensor([i for f in feed for i in f] + [0, 0], device=dev)
        probs = lm.forward(ids, pos, slots, caches, t["table"], t["seq_len"], q_start, rows, max(new), ws)
        flat = [i for f in feed for i in f]
        start = q_start.tolist()
        for b in range(B):
            n = new[b]
            if n == 0:
                continue
            want = lm.reference(seqs[b])[-n:]
            got = probs[start[b]:start[b + 1]].cpu().double()
            # two layers of fp32 products of 256 terms with O(1) intermediate values and logits up to ~15: 1e-4 is > 100 roundings of the sum
            assert float((got - want).abs().max()) < 1e-4, (step, b)
        if step == 0:                                                            # the prompts' last rows draw the first tokens
            rs = [(start[b + 1] - 1, 1) for b in range(B)]
        else:
            rs = [(start[b], new[b]) for b in range(B)]
        sel = [r for s, n in rs for r in range(s, s + n)]
        row_start = [0]
        for _, n in rs:
            row_start.append(row_start[-1] + n)
        target = probs[sel].contiguous()
        R = len(sel)
        draft = torch.full((R, V), 1.0 / V, device=dev)
        toks = torch.tensor([flat[r] for r in sel])
        uni, noise = torch.rand(R, generator=g), torch.empty(B, V).exponential_(generator=g)
        out, n_out, seq_kept = torch.zeros(B, K + 1, dtype=torch.int64, device=dev), _i32([0] * B, dev), _i32([0] * B, dev)
        ops.draft_verify(target, draft, toks.to(dev), _i32(row_start, dev), uni.to(dev), noise.to(dev), out, n_out, seq_len=t["seq_len"], keep_len=seq_kept, workspace=ws2)
        w_out, w_n, w_keep = _verify_ref(target.cpu(), draft.cpu(), toks, row_start, uni, noise, K + 1, t["seq_len"].tolist())
        assert out.tolist() == w_out and n_out.tolist() == w_n and seq_kept.tolist() == w_keep
        keep = seq_kept
        feed = []
        for b in range(B):
            kept = int(seq_kept[b])
            seqs[b] = seqs[b][:kept]
            nxt = int(out[b, w_n[b] - 1])
            total += w_n[b]
            drafts = torch.randint(0, V, ((step + b) % (K + 1),), generator=g).tolist()
            feed.append([nxt] + drafts)
            seqs[b] = seqs[b] + feed[b]
        if step == 4:                                                            # request 2 is done, another prompt takes its place
            keep[2] = 0
            seqs[2] = torch.randint(0, V, (23,), generator=g).tolist()
            feed[2] = seqs[2][:]
            K = 24                                                               # its whole prompt is verified like drafts: a longer output
    assert total > 9 * B                                                         # some drafts were accepted
    ops.paged_plan(t["seq_len"], _i32([0] * B, dev), _i32([0] * B, dev), t["table"], t["free"], t["state"], block, q_start)
    assert sorted(t["free"].tolist()) == list(range(n_blocks)) and int(t["state"][L.PST_FREE]) == n_blocks


def _rows_to_verify(q_start, n_verify, cap, n_rows):
    """The last n_verify[b] rows of every request, packed (cap rows, the last ones padding), and their row offsets: device work only.  Requests
    without rows in this step (or a refused one) verify nothing."""
    n = torch.minimum(n_verify, q_start[1:] - q_start[:-1])
    row_start = torch.zeros_like(q_start)
    row_start[1:] = torch.cumsum(n, 0)
    i = torch.arange(cap, dtype=torch.int32, device=q_start.device)
    b = torch.searchsorted(row_start[1:], i, right=True).clamp(max=n.shape[0] - 1)
    return (q_start[b + 1] - row_start[b + 1] + i).clamp(0, n_rows - 1), row_start


def test_steps_of_prompt_chunks_and_drafts(dev):
    """Prompts that arrive in chunks beside requests that draft: only a prompt's last row is verified (a chunk that is not the last: none), so every
    prompt stays whole in the cache; rows, row offsets and kept lengths are found on the device, without a read-back inside the step.  Probabilities
    against a cache-free float64 recomputation, tokens and kept lengths against the definition."""
    from mars5_tts_amd import _lib as L, ops
    lm = _TinyLM(dev, seed=3).to(dev)
    B, block, width, n_blocks, K, V, chunk, rows, cap = 4, 8, 12, 40, 4, lm.vocab, 10, 36, 18
    g = torch.Generator().manual_seed(15)
    pool = Pool(B, width, n_blocks, block, 2)
    t = pool.tensors(dev)
    caches = [tuple(torch.full((n_blocks, lm.kv, block, lm.hd), float("nan"), device=dev) for _ in range(2)) for _ in range(2)]
    ws = torch.zeros(4 << 20, dtype=torch.uint8, device=dev)
    vs = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (23, 1, 10, 30)]
    seqs = [[] for _ in range(B)]                                                # ids in the cache
    keep, out, n_out = _i32([0] * B, dev), torch.zeros(B, K + 1, dtype=torch.int64, device=dev), _i32([0] * B, dev)
    drawn = [None] * B
    q_start, slots, pos = _i32([0] * (B + 1), dev), _i32([0] * rows, dev), _i32([0] * rows, dev)
    mixed = 0
    for step in range(7):
        feed, verify = [], []
        for b in range(B):
            if prompts[b]:
                feed.append(prompts[b][:chunk])
                prompts[b] = prompts[b][chunk:]
                verify.append(0 if prompts[b] else 1)
            else:
                feed.append([drawn[b]] + torch.randint(0, V, ((step * 3 + b) % K,), generator=g).tolist())
                verify.append(len(feed[b]))
            seqs[b] = seqs[b] + feed[b]
        new = [len(f) for f in feed]
        flat = [i for f in feed for i in f]
        mixed += max(new) == chunk and any(v > 1 for v in verify)
        ids = torch.tensor(flat + [0] * (rows - len(flat)), device=dev)
        uni, noise = torch.rand(cap, generator=g), torch.empty(B, V).exponential_(generator=g)
        args = [_i32(new, dev), _i32(verify, dev), uni.to(dev), noise.to(dev)]
        # ---- the step: nothing is read back
        ops.paged_plan(t["seq_len"], keep, args[0], t["table"], t["free"], t["state"], block, q_start, slots, pos)
        probs = lm.forward(ids, pos, slots, caches, t["table"], t["seq_len"], q_start, rows, chunk, ws)
        sel, row_start = _rows_to_verify(q_start, args[1], cap, rows)
        target = probs[sel]
        draft = torch.full((cap, V), 1.0 / V, device=dev)
        ops.draft_verify(target, draft, ids[sel], row_start, args[2], args[3], out, n_out, seq_len=t["seq_len"], keep_len=keep, workspace=vs, plan_state=t["state"])
        # ---- checks
        assert int(t["state"][L.PST_STATUS]) == 0
        start = [0]
        for n in new:
            start.append(start[-1] + n)
        rs = [0]
        for n in verify:
            rs.append(rs[-1] + n)
        assert row_start.tolist() == rs and sel[:rs[-1]].tolist() == [r for b in range(B) for r in range(start[b + 1] - verify[b], start[b + 1])]
        for b in range(B):
            want = lm.reference(seqs[b])[-new[b]:]
            # (as above: two layers of fp32 products of 256 terms)
            assert float((probs[start[b]:start[b + 1]].cpu().double() - want).abs().max()) < 1e-4, (step, b)
        w_out, w_n, w_keep = _verify_ref(target.cpu(), draft.cpu(), ids[sel].cpu(), rs, uni, noise, K + 1, [len(q) for q in seqs])
        assert out.tolist() == w_out and n_out.tolist() == w_n and keep.tolist() == w_keep
        for b in range(B):
            if prompts[b] or verify[b] == 1:
                assert w_keep[b] == len(seqs[b])                                 # a prompt (or a lone token) stays whole
            seqs[b] = seqs[b][:w_keep[b]]
            drawn[b] = w_out[b][w_n[b] - 1] if w_n[b] else None
    assert mixed >= 2


@pytest.mark.parametrize("V", [50, 9000])
@pytest.mark.parametrize("recorded", [False, True])
def test_refused_step_keeps_the_pending_roll_back(dev, recorded, V):
    """Drafts are rejected, the next step is short of blocks (or holds an invalid request), verification runs behind it as in every step: keep_len
    stays what the plan was given, so the step that is tried again once a request has ended gives back the rejected positions.  As
    calls and as a recorded plan; the list definition throughout."""
    from mars5_tts_amd import _lib as L, ops
    B, block, width, n_blocks, M, rows = 3, 4, 8, 7, 5, 40
    pool = Pool(B, width, n_blocks, block, 4)
    t = pool.tensors(dev)
    keep, new = _i32([0] * B, dev), _i32([0] * B, dev)
    q_start, slots, pos = _i32([7] * (B + 1), dev), _i32([7] * rows, dev), _i32([7] * rows, dev)
    g = torch.Generator().manual_seed(6)
    target = torch.softmax(torch.randn(rows, V, generator=g), -1)
    draft = torch.softmax(torch.randn(rows, V, generator=g), -1)
    tokens, uni, noise = torch.randint(0, V, (rows,), generator=g), torch.ones(rows), torch.empty(B, V).exponential_(generator=g)
    dense = [x.to(dev) for x in (target, draft, tokens, uni, noise)]
    out, n_out = torch.zeros(B, M, dtype=torch.int64, device=dev), _i32([0] * B, dev)
    vs = torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev)

    def calls():
        ops.paged_plan(t["seq_len"], keep, new, t["table"], t["free"], t["state"], block, q_start, slots, pos)
        ops.draft_verify(dense[0], dense[1], dense[2], q_start, dense[3], dense[4], out, n_out, seq_len=t["seq_len"], keep_len=keep, workspace=vs, plan_state=t["state"])

    plan = None
    if recorded:
        plan = ops.StagePlan("ar_decode_step")
        with plan.recording():
            calls()
    kept, statuses = [0] * B, []
    # (what the host wants added, requests that it ends before): the third and fourth step cannot be served
    for add, ended in (([3, 5, 2], []), ([5, 4, 4], []), ([8, 8, 8], []), ([4, 1, width * block], []), ([2, 0, 5], [1]), ([1, 3, 0], [])):
        for b in ended:
            kept[b] = 0
            keep[b] = 0
        new.copy_(_i32(add, dev))
        assert keep.tolist() == kept
        want = pool.step(kept[:], add, rows)
        plan.run() if recorded else calls()
        torch.cuda.synchronize()
        _check_plan(t, pool, want, q_start, slots, pos)
        w_out, w_n, w_keep = _verify_ref(target, draft, tokens, want[1], uni, noise, M, pool.len)
        assert out.tolist() == w_out and n_out.tolist() == w_n
        if want[0] == 0:
            kept = w_keep
        assert keep.tolist() == kept, want[0]
        statuses.append(want[0])
    assert not bool(vs.any())                                                    # (the larger vocabulary is split: its workgroups have met)
    assert statuses[2] > 0 and statuses[3] < 0 and [s for i, s in enumerate(statuses) if i not in (2, 3)] == [0] * 4
    for bad in (t["state"][:4], t["state"].long(), t["state"].cpu()):
        with pytest.raises(AssertionError, match="plan_state"):
            ops.draft_verify(dense[0], dense[1], dense[2], q_start, dense[3], dense[4], out, n_out, plan_state=bad)


def test_recorded_step_equals_the_calls(dev):
    """A whole step recorded as a stage plan: run from C, then captured into a graph and replayed, beside the same calls one by one; the
    keep_len that verification writes is the next step's, so every step depends on the ones before."""
    from mars5_tts_amd import _lib as L, ops
    B, block, width, n_blocks, H, kv, hd, V, M = 5, 4, 16, 64, 4, 2, 64, 500, 3
    rows = B * M
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(rows, (H + 2 * kv) * hd, generator=g).bfloat16().to(dev)
    rope = torch.randn(width * block, hd // 2, 2, generator=g).to(dev)
    target, draft = (torch.softmax(torch.randn(rows, V, generator=g) * 2, -1).to(dev) for _ in range(2))
    tokens = torch.randint(0, V, (rows,), generator=g).to(dev)
    tokens[1::2] = target[0::2].argmax(-1)[:tokens[1::2].shape[0]]               # some drafts are likely ones
    uni, noise = torch.rand(rows, generator=g).to(dev), torch.empty(B, V).exponential_(generator=g).to(dev)
    new = _i32([M] * B, dev)

    def fresh():
        t = dict(seq_len=_i32([0] * B, dev), keep=_i32([0] * B, dev), table=torch.zeros(B, width, dtype=torch.int32, device=dev),
                 free=torch.arange(n_blocks, dtype=torch.int32, device=dev), state=torch.zeros(L.PST_WORDS, dtype=torch.int32, device=dev),
                 q_start=_i32([0] * (B + 1), dev), slots=_i32([0] * rows, dev), pos=_i32([0] * rows, dev),
                 q=torch.zeros(rows, H, hd, dtype=torch.bfloat16, device=dev), out=torch.zeros(rows, H, hd, dtype=torch.bfloat16, device=dev),
                 k=torch.zeros(n_blocks, kv, block, hd, dtype=torch.bfloat16, device=dev), v=torch.zeros(n_blocks, kv, block, hd, dtype=torch.bfloat16, device=dev),
                 out_tokens=torch.zeros(B, M, dtype=torch.int64, device=dev), n_out=_i32([0] * B, dev), ws=torch.zeros(1 << 20, dtype=torch.uint8, device=dev),
                 vs=torch.zeros(B * L.DRAFT_WS_BYTES, dtype=torch.uint8, device=dev))
        t["state"][L.PST_FREE] = n_blocks
        return t

    def step(t):
        ops.paged_plan(t["seq_len"], t["keep"], new, t["table"], t["free"], t["state"], block, t["q_start"], t["slots"], t["pos"])
        ops.paged_rope_cache(qkv, H, kv, rope, t["pos"], t["slots"], t["q"], t["k"], t["v"])
        ops.paged_attention(t["q"], t["k"], t["v"], t["table"], t["seq_len"], t["q_start"], t["out"], max_new=M, workspace=t["ws"])
        ops.draft_verify(target, draft, tokens, t["q_start"], uni, noise, t["out_tokens"], t["n_out"], seq_len=t["seq_len"], keep_len=t["keep"], workspace=t["vs"])

    one, two, three = fresh(), fresh(), fresh()
    plan2, plan3 = ops.StagePlan("ar_decode_step"), ops.StagePlan("ar_decode_step")
    with plan2.recording():
        step(two)
    with plan3.recording():
        step(three)
    assert plan2.n_ops == plan3.n_ops == 4 and int(two["n_out"].sum()) == 0
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        plan3.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(8):
        step(one)
        plan2.run()
        graph.replay()
        torch.cuda.synchronize()
        assert int(one["state"][L.PST_STATUS]) == 0 and int(one["n_out"].min()) >= 1
        for name in one:
            assert torch.equal(one[name], two[name]) and torch.equal(one[name], three[name]), (i, name)
    assert int(one["seq_len"].max()) > 8
