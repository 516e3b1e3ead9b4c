"""Paged serving operators without a GPU: the index arithmetic that keeps device data inside the buffers (csrc/paged_index.h, compiled
with g++), argument refusals of the C entry points and of the tensor wrappers, and the argument structures' layout."""
import bisect
import ctypes as C
import os
import random
import re
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mars5-tts_amd", "csrc")

HARNESS = r"""
#include "paged_index.h"
extern "C" {
int h_log2(int v) { return m5_log2(v); }
int h_pages(int n, int s) { return m5_pages(n, s); }
int h_block(int id, int n) { return m5_block(id, n); }
void h_request(int a, int b, int len, int rows, long long cap, int* o) { M5Request r = m5_request(a, b, len, rows, cap); o[0] = r.r0; o[1] = r.r1; o[2] = r.len; }
int h_key_hi(int p, int l) { return m5_key_hi(p, l); }
int h_key_lo(int p, int w) { return m5_key_lo(p, w); }
int h_plan(int held, int keep, int add, int width, int shift, int* o) { return m5_plan_request(held, keep, add, width, shift, o[0], o[1]); }
int h_source(int a, int r, int f) { return m5_plan_source(a, r, f); }
int h_push(int i, int r, int f) { return m5_plan_push(i, r, f); }
int h_upper(const int* p, int n, int v) { return m5_upper(p, n, v); }
void h_share(int r0, int r1, int len, int group, int few, int many, int w, int* o) {
    M5Share s = m5_share(M5Request{r0, r1, len}, group, few, many, w);
    o[0] = s.rows; o[1] = s.tr; o[2] = s.tiles; o[3] = s.k0; o[4] = s.units; o[5] = s.sr;
}
int h_chunk_units(float u, float t, float ur, float tr, float p, float i, float r, float l) { return m5_chunk_units(u, t, ur, tr, p, i, r, l); }
int h_chunks(int u, int c) { return m5_chunks(u, c); }
int h_span(const int* s, int len, int w, int first, int last, int n, int chunk, int c, int* o) {
    M5Span r;
    int ok = m5_span(M5Share{s[0], s[1], s[2], s[3], s[4], s[5]}, len, w, first, last, n, chunk, c, r);
    o[0] = r.ka; o[1] = r.kb; o[2] = r.c0; o[3] = r.c1;
    return ok;
}
void h_key_at(int key, int ka, int kb, int shift, int* o) { M5KeyAt r = m5_key_at(key, ka, kb, shift); o[0] = r.page; o[1] = r.off; }
}
"""
BIG = [-(1 << 31), -(1 << 30), -7, -1, 0, 1, 2, 63, 64, 65, 1000, (1 << 30), (1 << 31) - 1]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    src, so = d / "harness.cpp", d / "libpaged_host.so"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-O2", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=undefined", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.h_request.argtypes = [C.c_int] * 4 + [C.c_longlong, C.POINTER(C.c_int)]
    lib.h_chunk_units.argtypes = [C.c_float] * 8
    lib.h_plan.argtypes = [C.c_int] * 5 + [C.POINTER(C.c_int)]
    return lib


def test_bad_lengths_and_offsets_stay_inside_the_buffers(host):
    """Whatever seq_len and q_start hold, a request's rows lie in [0, n_rows], its positions in the table row's capacity, and the keys
    of any of its rows in [0, len)."""
    out = (C.c_int * 3)()
    for rows in (0, 1, 130):
        for cap in (1, 64, (1 << 31) - 1):
            for a in BIG:
                for b in BIG:
                    for n in BIG:
                        host.h_request(a, b, n, rows, cap, out)
                        r0, r1, ln = out
                        assert 0 <= r0 <= r1 <= rows and 0 <= ln <= cap
                        for row in {r0, r1 - 1} - {r1}:
                            pos = ln - (r1 - row)
                            lo, hi = host.h_key_lo(pos, 0), host.h_key_hi(pos, ln)
                            assert lo == 0 and hi <= ln
                            if 0 <= pos < (1 << 31) - 1:
                                assert hi == pos + 1


def test_key_range_of_a_row(host):
    for ln in (0, 1, 5, 64):
        for new in (1, 3, 7):
            for window in (0, 1, 2, 100):
                for i in range(new):
                    pos = ln - new + i
                    want = [j for j in range(ln) if j <= pos and (window == 0 or j > pos - window)]
                    lo, hi = host.h_key_lo(pos, window), host.h_key_hi(pos, ln)
                    assert list(range(lo, max(lo, hi))) == want, (ln, new, window, i)


@pytest.mark.parametrize("window", [1 << 30, (1 << 31) - 1])
def test_a_window_wider_than_any_request_hides_nothing(host, window):
    """The largest windows that can be passed see what window 0 sees, also where the first rows stand before position 0 (fewer cached
    positions than new rows)."""
    o, w, a, b = (C.c_int * 6)(), (C.c_int * 6)(), (C.c_int * 4)(), (C.c_int * 4)()
    for pos in (-(1 << 30), -7, -3, -2, -1, 0, 1, 1000, (1 << 30) - 1):
        assert host.h_key_lo(pos, window) == 0
    for ln in (0, 1, 3, 6, 300):
        for new in (1, 6, 10, 200):
            for group, few, many in ((1, 16, 0), (3, 32, 128)):
                host.h_share(0, new, ln, group, few, many, 0, o)
                host.h_share(0, new, ln, group, few, many, window, w)
                assert list(o) == list(w), (ln, new)
                for t in range(o[2]):
                    first, last = t * o[1] // group, (min((t + 1) * o[1], o[0]) - 1) // group
                    seen = [host.h_span(s, ln, win, ln - new + first, ln - new + last, 1, 1 << 24, 0, r) for s, win, r in ((o, 0, a), (w, window, b))]
                    assert seen == [1, 1] and list(a) == list(b), (ln, new, t)


def test_bad_pages_are_no_pages(host):
    for n in (1, 5, 1 << 30):
        for i in BIG:
            assert host.h_block(i, n) == (i if 0 <= i < n else -1)
    assert [host.h_log2(v) for v in (1, 2, 16, 1024, 0, -4, 3, 48)] == [0, 1, 4, 10, -1, -1, -1, -1]
    for s in (0, 4, 10):
        for n in (0, 1, 15, 16, 17, 1023, 1025, (1 << 31) - 1):
            assert host.h_pages(n, s) == -(-n // (1 << s))


def test_plan_requests_are_validated(host):
    o = (C.c_int * 2)()
    for held in BIG:
        for keep in BIG:
            for add in BIG:
                for width, shift in ((1, 0), (8, 4), (1 << 20, 10)):
                    cap = width << shift
                    ok = bool(host.h_plan(held, keep, add, width, shift, o))
                    assert ok == (0 <= keep <= held <= cap and add >= 0 and keep + add <= cap), (held, keep, add, width, shift)
                    assert list(o) == ([-(-held // (1 << shift)), -(-(keep + add) // (1 << shift))] if ok else [0, 0])


def test_free_stack_order(host):
    """m5_plan_source / m5_plan_push against a Python list that pushes from the last returned page to the first and pops by request."""
    rng = random.Random(5)
    for _ in range(200):
        free = [rng.randrange(1000) for _ in range(rng.randrange(8))]
        returned = [1000 + i for i in range(rng.randrange(6))]
        stack = free + returned[::-1]
        take = rng.randrange(len(stack) + 1)
        got = []
        for a in range(take):
            s = host.h_source(a, len(returned), len(free))
            assert s < len(free)
            got.append(free[s] if s >= 0 else returned[-1 - s])
        want = [stack.pop() for _ in range(take)]
        assert got == want
        after = free[:len(stack)] + [None] * max(0, len(stack) - len(free))
        for i in range(take, len(returned)):
            spot = host.h_push(i, len(returned), len(free))
            assert spot >= len(free)                     # never an entry that this call reads
            after[spot] = returned[i]
        assert after == stack


def test_prefix_search(host):
    rng = random.Random(6)
    for _ in range(200):
        pre = [0]
        for _ in range(rng.randrange(1, 40)):
            pre.append(pre[-1] + rng.choice([0, 0, 1, 2, 9]))
        arr = (C.c_int * len(pre))(*pre)
        for v in range(pre[-1]):
            assert host.h_upper(arr, len(pre) - 1, v) == bisect.bisect_right(pre, v) - 1


def test_packed_structures_equal_the_field_by_field_ones():
    from mars5_tts_amd import _lib as L
    import struct
    for cls in (L.PagedPlanArgs, L.PagedRopeArgs, L.PagedAttnArgs, L.DraftVerifyArgs):
        values = [0.25 if t is L.f32 else (1 << 40) + i if t in (L.vp, L.i64) else i - 3 for i, (_, t) in enumerate(cls._fields_)]
        assert bytes(L.packed(cls)(*values)) == bytes(cls(*values))
        values[[t for _, t in cls._fields_].index(L.i32)] = 1 << 31
        with pytest.raises(struct.error):
            L.packed(cls)(*values)


def test_attention_items_cover_every_visible_key_once(host):
    """Tiles x chunks of a request: every (row, key) that is to be seen lies in exactly one item of its tile, an item's keys lie inside the
    request, a tile that sees nothing has one item, and with room for partial results the items and their rows stay inside it."""
    rng = random.Random(8)
    o, sp = (C.c_int * 6)(), (C.c_int * 4)()
    for case in range(300):
        group, window = rng.choice([1, 3, 4, 16]), rng.choice([0, 0, 1, 63, 64, 200])
        few, many = rng.choice([(16, 0), (32, 0), (32, 128)])
        kv, places, slots, room = rng.choice([1, 2, 24]), rng.choice([8, 512]), rng.choice([0, 3, 40, 4096]), rng.choice([64, 1000, 100000])
        reqs, r0 = [], 0
        for _ in range(rng.randrange(1, 5)):
            new = rng.choice([0, 1, 1, 2, 5, 70])
            reqs.append((r0, r0 + new, rng.choice([0, 1, 63, 64, 65, 300, 1500]) + rng.choice([0, new])))
            r0 += new
        shares = []
        for q in reqs:
            host.h_share(*q, group, few, many, window, o)
            shares.append(list(o))
            rows, tr, tiles, k0, units, sr = o
            assert sr % 16 == 0 and min(rows, tr) <= sr <= tr
            assert rows == (q[1] - q[0]) * group and tiles == -(-rows // tr) and tr == (many if many and rows > few else few) and k0 % 64 == 0
        tiles, units = kv * sum(s[2] for s in shares), kv * sum(s[2] * s[4] for s in shares)
        tile_rows, unit_rows = kv * sum(s[2] * s[5] for s in shares), kv * sum(s[2] * s[4] * s[5] for s in shares)
        chunk = host.h_chunk_units(units, tiles, unit_rows, tile_rows, places, slots, room, rng.choice([1.0, 4.0, 8.0]))
        fits = tiles < slots and tile_rows < room
        assert 1 <= chunk <= 1 << 24 and (fits or chunk == 1 << 24)
        total = part_rows = 0
        for (a, b, ln), s in zip(reqs, shares):
            n = host.h_chunks(s[4], chunk)
            assert n == max(1, -(-s[4] // chunk))
            total += kv * s[2] * n
            part_rows += kv * s[2] * n * s[5] if n > 1 else 0
            for t in range(s[2]):
                first, last = t * s[1] // group, (min((t + 1) * s[1], s[0]) - 1) // group
                pos0 = ln - (b - a)
                spans = []
                for c in range(n):
                    if host.h_span((C.c_int * 6)(*s), ln, window, pos0 + first, pos0 + last, n, chunk, c, sp):
                        spans.append((sp[0], sp[1]))
                        assert sp[2] <= c <= sp[3] < n
                assert len(spans) == sp[3] - sp[2] + 1 >= 1
                seen = [j for p in range(pos0 + first, pos0 + last + 1) for j in range(max(0, p - window + 1) if window else 0, min(p + 1, ln))]
                lo, hi = (min(seen), max(seen) + 1) if seen else (0, 0)
                covered = [j for ka, kb in spans for j in range(ka, kb)]
                assert covered == list(range(lo, hi)), (reqs, window, spans, lo, hi)
        if fits:
            assert total <= slots and part_rows <= room, (total, slots, part_rows, room)
        else:
            assert part_rows == 0


def test_what_is_read_for_a_key_stays_on_the_loaded_pages(host):
    o = (C.c_int * 2)()
    for shift in (0, 2, 4, 10):
        for ka, kb in ((0, 1), (5, 6), (5, 300), (64, 128), (1000, 1023)):
            for key in list(range(max(0, ka - 70), kb + 200, 7)) + [ka, kb - 1, kb]:
                host.h_key_at(key, ka, kb, shift, o)
                assert ka >> shift <= o[0] <= (kb - 1) >> shift and 0 <= o[1] < 1 << shift
                if ka <= key < kb:
                    assert o[0] * (1 << shift) + o[1] == key


def test_argument_structures_match_the_header(tmp_path):
    from mars5_tts_amd import _lib as L
    hdr = os.path.join(ROOT, "include", "mars5_hip.h")
    pairs = {"M5PagedPlanArgs": L.PagedPlanArgs, "M5PagedRopeArgs": L.PagedRopeArgs, "M5PagedAttnArgs": L.PagedAttnArgs, "M5DraftVerifyArgs": L.DraftVerifyArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{hdr}"', 'int main(void) {']
    for cname, cls in pairs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    lines.append(f'printf("words %d %d %d %d %d\\n", M5_PST_FREE, M5_PST_STATUS, M5_PST_ROWS, M5_PST_WORDS, M5_DRAFT_WS_BYTES);')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ['return 0; }']))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    for ln in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        w = ln.split()
        if w[0] == "words":
            assert [int(v) for v in w[1:]] == [L.PST_FREE, L.PST_STATUS, L.PST_ROWS, L.PST_WORDS, L.DRAFT_WS_BYTES]
        else:
            cls = pairs[w[0]]
            assert int(w[2]) == (C.sizeof(cls) if w[1] == "size" else getattr(cls, w[1]).offset), ln
    paged = open(os.path.join(ROOT, "include", "mars5_paged.h")).read()
    assert set(re.findall(r"^\} (M5\w+);", paged, flags=re.M)) == set(pairs)


BUF = (C.c_uint64 * 8)()
P = (C.addressof(BUF) + 15) & ~15            # an aligned host address: refusals happen before anything is launched


def _plan(**kw):
    from mars5_tts_amd import _lib as L
    a = dict(seq_len=P, keep_len=P, new_len=P, n_seq=2, table_width=4, n_blocks=9, block_size=16, n_rows=5, block_table=P, table_rs=4, free_blocks=P, state=P, q_start=P,
             slot_map=P, positions=P)
    return L.PagedPlanArgs(**{**a, **kw})


def _rope(**kw):
    from mars5_tts_amd import _lib as L
    a = dict(qkv=P, qkv_rs=256, n_rows=3, n_heads=2, n_kv_heads=1, head_dim=64, q_norm=None, k_norm=None, eps=1e-5, rope=P, n_pos=10, n_pairs=32, interleaved=1, positions=P,
             slot_map=P, q_out=P, q_rs=128, q_hs=64, k_cache=P, k_bs=1024, k_hs=1024, k_ss=64, v_cache=P, v_bs=1024, v_hs=1024, v_ss=64, n_blocks=4, block_size=16)
    return L.PagedRopeArgs(**{**a, **kw})


def _attn(**kw):
    from mars5_tts_amd import _lib as L
    a = dict(q=P, q_rs=128, q_hs=64, k_cache=P, k_bs=1024, k_hs=1024, k_ss=64, v_cache=P, v_bs=1024, v_hs=1024, v_ss=64, block_table=P, table_rs=4, table_width=4, n_blocks=9,
             block_size=16, n_seq=2, n_rows=3, max_new=2, n_heads=2, n_kv_heads=1, head_dim=64, window=0, seq_len=P, q_start=P, scale=0.125, out=P, o_rs=128, o_hs=64, workspace=None,
             workspace_bytes=0)
    return L.PagedAttnArgs(**{**a, **kw})


def _verify(**kw):
    from mars5_tts_amd import _lib as L
    a = dict(target=P, t_rs=100, draft=P, d_rs=100, n_rows=5, vocab=100, n_seq=2, out_width=4, tokens=P, row_start=P, uniforms=P, noise=P, noise_rs=100, out_tokens=P, out_rs=4, n_out=P,
             seq_len=P, keep_len=P, workspace=None, workspace_bytes=0)
    return L.DraftVerifyArgs(**{**a, **kw})


ARG, UNSUP = -1, -3


@pytest.mark.parametrize("kw,rc", [(dict(seq_len=None), ARG), (dict(q_start=None), ARG), (dict(state=None), ARG), (dict(positions=None), ARG), (dict(slot_map=None), ARG),
                                   (dict(n_seq=0), ARG), (dict(n_rows=-1), ARG), (dict(block_size=24), ARG), (dict(block_size=0), ARG), (dict(table_rs=3), ARG), (dict(n_blocks=0), ARG),
                                   (dict(block_size=2048), UNSUP), (dict(n_seq=4097), UNSUP), (dict(n_blocks=1 << 30), UNSUP), (dict(table_width=1 << 28, table_rs=1 << 28), UNSUP)])
def test_plan_refuses(kw, rc):
    from mars5_tts_amd import _lib as L
    assert L.lib.m5_paged_plan(C.byref(_plan(**kw)), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(qkv=None), ARG), (dict(slot_map=None), ARG), (dict(n_rows=-1), ARG), (dict(n_kv_heads=0), ARG), (dict(block_size=12), ARG), (dict(n_pos=0), ARG),
                                   (dict(head_dim=96), UNSUP), (dict(n_pairs=33), UNSUP), (dict(n_pairs=20), UNSUP), (dict(n_pairs=0), UNSUP), (dict(qkv_rs=257), UNSUP), (dict(q_hs=60), UNSUP),
                                   (dict(k_ss=66), UNSUP), (dict(v_cache=P + 2), UNSUP), (dict(rope=P + 4), UNSUP), (dict(q_norm=P + 4), UNSUP)])
def test_rope_cache_refuses(kw, rc):
    from mars5_tts_amd import _lib as L
    assert L.lib.m5_paged_rope_cache(L.BF16, C.byref(_rope(**kw)), None) == rc
    assert L.lib.m5_paged_rope_cache(L.F32X3, C.byref(_rope()), None) == UNSUP
    assert L.lib.m5_paged_rope_cache(L.BF16, C.byref(_rope(n_rows=0)), None) == 0          # nothing to do


@pytest.mark.parametrize("kw,rc", [(dict(q=None), ARG), (dict(out=None), ARG), (dict(seq_len=None), ARG), (dict(n_seq=0), ARG), (dict(n_heads=3, n_kv_heads=2), ARG), (dict(window=-1), ARG),
                                   (dict(scale=0.0), ARG), (dict(scale=float("nan")), ARG), (dict(block_size=10), ARG), (dict(table_rs=2), ARG), (dict(workspace_bytes=-1), ARG),
                                   (dict(head_dim=256), UNSUP), (dict(block_size=2048), UNSUP), (dict(n_seq=4097), UNSUP), (dict(q_rs=132), UNSUP), (dict(o_hs=68), UNSUP), (dict(k_cache=P + 4), UNSUP),
                                   (dict(v_bs=1020), UNSUP), (dict(workspace=P + 8, workspace_bytes=64), UNSUP)])
def test_attention_refuses(kw, rc):
    from mars5_tts_amd import _lib as L
    n = C.c_int64(-7)
    assert L.lib.m5_paged_attention(L.F16, C.byref(_attn(**kw)), None) == rc
    assert L.lib.m5_paged_attention_workspace(L.F16, C.byref(_attn(**kw)), C.byref(n)) == rc and n.value == -7
    assert L.lib.m5_paged_attention(L.F32X3, C.byref(_attn()), None) == UNSUP
    assert L.lib.m5_paged_attention(L.F16, C.byref(_attn(n_rows=0)), None) == 0


@pytest.mark.parametrize("kw,rc", [(dict(target=None), ARG), (dict(noise=None), ARG), (dict(n_out=None), ARG), (dict(keep_len=None), ARG), (dict(seq_len=None), ARG), (dict(vocab=0), ARG),
                                   (dict(n_seq=0), ARG), (dict(out_width=0), ARG), (dict(t_rs=99), ARG), (dict(d_rs=99), ARG), (dict(noise_rs=99), ARG), (dict(out_rs=3), ARG), (dict(n_rows=-1), ARG),
                                   (dict(workspace=P + 8, workspace_bytes=64), UNSUP)])
def test_verify_refuses(kw, rc):
    from mars5_tts_amd import _lib as L
    assert L.lib.m5_draft_verify(L.F32, C.byref(_verify(**kw)), None) == rc
    assert L.lib.m5_draft_verify(7, C.byref(_verify()), None) == UNSUP


def test_wrappers_refuse_host_tensors_and_wrong_shapes():
    from mars5_tts_amd import ops
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="device memory"):
        ops.paged_plan(i, i, i, torch.zeros(2, 4, dtype=torch.int32), i, torch.zeros(8, dtype=torch.int32), 16, torch.zeros(3, dtype=torch.int32))
    x, c = torch.zeros(3, 256), torch.zeros(4, 1, 16, 64)
    with pytest.raises(AssertionError, match="device memory"):
        ops.paged_rope_cache(x, 2, 1, torch.zeros(9, 32, 2), torch.zeros(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64), c, c)
    with pytest.raises(AssertionError, match="device memory"):
        ops.paged_attention(torch.zeros(3, 2, 64), c, c, torch.zeros(2, 4, dtype=torch.int32), i, torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, 64))
    with pytest.raises(AssertionError, match="device memory"):
        ops.draft_verify(torch.zeros(3, 9), None, torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(3), torch.zeros(2, 9), torch.zeros(2, 4, dtype=torch.int64), i)


def test_paged_launches_can_be_planned():
    """The four launches belong to AR steps and stages, not to NAR steps; recorded structures land in the plan's arena."""
    from mars5_tts_amd import _lib as L, ops
    for kind, ok in (("ar_decode_step", True), ("stage", True), ("nar_step", False)):
        sp = ops.StagePlan(kind)
        with sp.recording():
            assert L.lib.m5_paged_attention(L.F16, C.byref(_attn(n_rows=0)), None) == 0
        assert sp.n_ops == 1 and sp._arr[0].fn == L.PLAN_FN["m5_paged_attention"]
        assert sp.run(0, raise_on_error=False) == (0 if ok else ARG)
    sp = ops.StagePlan("ar_decode_step")
    with sp.recording():
        L.lib.m5_paged_plan(C.byref(_plan(seq_len=None)), None)
        L.lib.m5_paged_rope_cache(L.BF16, C.byref(_rope(n_rows=0)), None)
        L.lib.m5_draft_verify(L.F32, C.byref(_verify(vocab=0)), None)
    assert sp.n_ops == 3 and sp.run(0, raise_on_error=False) == ARG and sp._failed.value == 0
