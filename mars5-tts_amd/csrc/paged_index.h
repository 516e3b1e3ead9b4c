// Index arithmetic of the paged KV cache (paged.hip, paged_attention.hip, draft_verify.hip).  Everything that a kernel derives
// from DEVICE data (lengths, block ids, row offsets: no host check can see them) is clamped or refused here, so that no value of
// theirs leads outside a buffer.  Plain C++: tests/test_paged_cpu.py compiles this text with g++.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define M5_HD __host__ __device__ static inline
#else
#define M5_HD static inline
#endif

M5_HD int m5_clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// log2 of a power of two, -1 for any other value
M5_HD int m5_log2(int v) {
    if (v <= 0 || (v & (v - 1))) return -1;
    int s = 0;
    while ((1 << s) < v) ++s;
    return s;
}

// pages that hold n positions
M5_HD int m5_pages(int n, int shift) { return (int)(((int64_t)n + (1 << shift) - 1) >> shift); }

// a block id as the kernels use it: the id, or -1 for one outside the cache
M5_HD int m5_block(int id, int n_blocks) { return (id >= 0 && id < n_blocks) ? id : -1; }

// One request of a launch: its rows [r0, r1) of the packed buffers and the positions that the cache holds for it, cut down to what
// the buffers hold (n_rows rows, cap = table_width * block_size positions).  Query row r stands at position len - (r1 - r).
struct M5Request { int r0, r1, len; };
M5_HD M5Request m5_request(int start, int end, int seq_len, int n_rows, int64_t cap) {
    M5Request q;
    q.r0 = m5_clampi(start, 0, n_rows);
    q.r1 = m5_clampi(end, q.r0, n_rows);
    q.len = seq_len < 0 ? 0 : (seq_len > cap ? (int)cap : seq_len);
    return q;
}

// Keys that the query at position `pos` of a request with `len` cached positions sees: [lo, hi), empty when lo >= hi.
M5_HD int m5_key_hi(int pos, int len) { return pos + 1 < len ? pos + 1 : len; }
M5_HD int m5_key_lo(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }      // (pos may be negative, window 2^31 - 1)

// paged_plan, one request: pages held before, pages needed after; false when the request is not a valid one.
M5_HD bool m5_plan_request(int held, int keep, int add, int width, int shift, int& have, int& need) {
    const int64_t end = (int64_t)keep + add;
    const bool ok = held >= 0 && keep >= 0 && add >= 0 && keep <= held && end <= ((int64_t)width << shift) && held <= ((int64_t)width << shift);
    have = ok ? m5_pages(held, shift) : 0;
    need = ok ? m5_pages((int)end, shift) : 0;
    return ok;
}
// Free stack of n_free ids, R pages returned this call (numbered upwards by request, then page), allocation number a.  Pages are
// pushed from the last to the first and popped from the top, so allocation a takes returned page a while there is one, then the
// old stack from its top.  >= 0: index into the free list; < 0: returned page -1 - result.
M5_HD int m5_plan_source(int a, int returned, int n_free) { return a < returned ? -1 - a : n_free - 1 - (a - returned); }
// position in the free list of returned page i (only those with i >= pages taken stay there)
M5_HD int m5_plan_push(int i, int returned, int n_free) { return n_free + returned - 1 - i; }

// Index of the last entry of the non-decreasing pre[0 .. n] (pre[0] = 0 <= v < pre[n]) that is <= v.
M5_HD int m5_upper(const int* pre, int n, int v) {
    int lo = 0, hi = n;                       // pre[lo] <= v < pre[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid] <= v) lo = mid; else hi = mid;
    }
    return lo;
}

// ---- paged_attention: how the rows and keys of the requests are dealt out (paged_attention.hip)

// A request's share of the work: its packed rows (new tokens x query heads of a kv head) in tiles of `tr`, and the keys that any of
// them sees, from k0 (a multiple of 64) on, in units of 64.  A tile's partial results take `sr` rows each.
struct M5Share { int rows, tr, tiles, k0, units, sr; };
M5_HD M5Share m5_share(M5Request q, int group, int tr_few, int tr_many, int window) {
    M5Share s;
    s.rows = (q.r1 - q.r0) * group;
    const bool large = tr_many && s.rows > tr_few;
    s.tr = large ? tr_many : tr_few;
    s.tiles = large ? (s.rows + tr_many - 1) / tr_many : (s.rows + tr_few - 1) / tr_few;        // (constants in the kernels)
    s.k0 = m5_key_lo(q.len - (q.r1 - q.r0), window) & ~63;
    s.units = q.len > s.k0 ? (q.len - s.k0 + 63) >> 6 : 0;
    s.sr = s.rows < s.tr ? (s.rows + 15) & ~15 : s.tr;
    return s;
}
#define M5_UNSPLIT (1 << 24)                   /* a chunk longer than any key range (2^30 positions) */
// Units of a chunk for `units` units of work in `tiles` tiles (both over all requests and kv heads; unit_rows, tile_rows: the same sums
// times each request's sr), `places` workgroups on the chip, at most `items` items and `rows` rows of partial results; no shorter
// than `least`.  A request's items number at most units / chunk + tiles, so neither limit is passed.
M5_HD int m5_chunk_units(float units, float tiles, float unit_rows, float tile_rows, float places, float items, float rows, float least) {
    if (!(tiles < items && tile_rows < rows)) return M5_UNSPLIT;
    const float most = tile_rows > 32.f * tiles ? 2.f : 4.f;    // items per place; joins of large tiles cost more
    float room = 4.f * tiles <= places ? places - tiles : (tiles <= 2.f * places ? most * places - tiles : 0.5f * places);
    if (room < 0.5f * places) room = 0.5f * places;
    if (room > items - tiles) room = items - tiles;
    float len = units * 1.0001f / room + 1.f;  // (the sums are floats: rounded up)
    const float by_rows = unit_rows * 1.0001f / (rows - tile_rows) + 1.f;
    if (len < by_rows) len = by_rows;
    if (len < least) len = least;
    return len < (float)M5_UNSPLIT ? (int)len : M5_UNSPLIT;
}
M5_HD int m5_chunks(int units, int chunk) { return units > chunk ? (int)(((unsigned)units + (unsigned)chunk - 1) / (unsigned)chunk) : 1; }
// Keys [ka, kb) of chunk `c` of `n` for a tile whose first and last rows stand at positions `first` and `last`: false when they see none
// of its keys and another chunk answers for the tile (chunk 0 does if they see no key at all).  The tile's chunks are c0 .. c1.
struct M5Span { int ka, kb, c0, c1; };
M5_HD bool m5_span(M5Share s, int len, int window, int first, int last, int n, int chunk, int c, M5Span& r) {
    const int lo = m5_key_lo(first, window), hi = m5_key_hi(last, len);
    r.c0 = r.c1 = 0;
    if (n > 1 && hi > lo) {
        r.c0 = (int)((unsigned)((lo - s.k0) >> 6) / (unsigned)chunk);
        r.c1 = (int)((unsigned)((hi - 1 - s.k0) >> 6) / (unsigned)chunk);
    }
    r.ka = c > r.c0 ? s.k0 + c * chunk * 64 : lo;
    r.kb = c < r.c1 ? s.k0 + (c + 1) * chunk * 64 : hi;
    return c >= r.c0 && c <= r.c1;
}
// What is read for a key: its page among the ids of the keys [ka, kb) and its place there; outside the range the nearest key's.
struct M5KeyAt { int page, off; };
M5_HD M5KeyAt m5_key_at(int key, int ka, int kb, int shift) {
    const int k = key < ka ? ka : (key >= kb ? kb - 1 : key);
    M5KeyAt r = {k >> shift, k & ((1 << shift) - 1)};
    return r;
}
