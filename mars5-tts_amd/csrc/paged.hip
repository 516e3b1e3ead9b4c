// Paged KV cache: the step's block tables / slot map / positions (m5_paged_plan) and the pass that norms and rotates the new q and
// k heads and writes k and v into the cache (m5_paged_rope_cache).  Semantics: include/mars5_paged.h.
#include "common.h"
#include "paged_index.h"
#include <limits.h>

namespace {

// ---------------------------------------------------------------------------------------------------------- m5_paged_plan
// Every workgroup scans the requests itself (prefix sums of rows, blocks taken and blocks given back into LDS), so the rows and blocks can
// be dealt to many workgroups without a second launch.  Nothing that any workgroup reads is written before the end: table
// entries written lie behind the pages a growing request holds, those read as "given back" behind the pages a shrinking one
// keeps, free-list entries written lie at or above n_free and those read below.  seq_len and the state words are written by the
// workgroup that finishes last (ticket word of the state; it leaves the ticket at 0).
// Latency bound: one memory round trip for the lengths, ~30 cross-lane adds, a search of log2(n_seq) LDS reads per row (four rows of a
// thread at once) and one load per row.  4.3 us a call at 48 requests (graph replay), a launch's own time 2.7.
constexpr int PLAN_MAX_SEQ = 4096;

template <int CTRL, int ROWS>
__device__ inline int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ inline int wave_scan(int v) {                     // inclusive: row shifts, then the rows' last lanes broadcast
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}

template <int NT>
__global__ __launch_bounds__(NT) void paged_plan_kernel(M5PagedPlanArgs p, int shift) {
    extern __shared__ int lds[];                             // [5][n_seq + 1]
    __shared__ int wsum[NT / 64][4];
    __shared__ int first_bad, last;
    const int B = p.n_seq, tid = threadIdx.x, wave = tid >> 6;
    int* row_pre = lds;
    int* take_pre = lds + (B + 1);
    int* give_pre = lds + 2 * (B + 1);
    int* keep = lds + 3 * (B + 1);
    int* have = lds + 4 * (B + 1);                           // pages before the step
    if (tid == 0) first_bad = INT_MAX;
    const int n_free = m5_clampi(p.state[M5_PST_FREE], 0, p.n_blocks);
    __syncthreads();

    const int per = (B + NT - 1) / NT;                       // consecutive requests per thread
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int64_t rows = 0;
    int take = 0, give = 0;
    for (int b = b0; b < b1; ++b) {
        int h, need;
        const int k = p.keep_len[b], add = p.new_len[b];
        const bool ok = m5_plan_request(p.seq_len[b], k, add, p.table_width, shift, h, need);
        if (!ok) atomicMin(&first_bad, b);
        keep[b] = k;
        have[b] = h;
        row_pre[b] = ok ? add : 0;                           // (what it adds, for now)
        take_pre[b] = need - h;
        rows += ok ? add : 0;
        take += max(need - h, 0);
        give += max(h - need, 0);
    }
    // rows may pass 31 bits before they are found to be too many: scanned in two pieces of 20 and 12 bits
    const int lo = wave_scan((int)(rows & 0xfffff)), hi = wave_scan((int)(rows >> 20)), ti = wave_scan(take), gi = wave_scan(give);
    if ((tid & 63) == 63) { wsum[wave][0] = lo; wsum[wave][1] = hi; wsum[wave][2] = ti; wsum[wave][3] = gi; }
    __syncthreads();
    int64_t rb = 0, n_rows = 0;
    int tb = 0, gb = 0, n_take = 0, n_give = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        if (w == wave) { rb = n_rows; tb = n_take; gb = n_give; }
        n_rows += wsum[w][0] + ((int64_t)wsum[w][1] << 20);
        n_take += wsum[w][2];
        n_give += wsum[w][3];
    }
    int status = 0;
    if (first_bad != INT_MAX) status = -1 - first_bad;
    else if (n_rows > (p.slot_map ? p.n_rows : INT_MAX)) status = -1 - B;
    else if ((int64_t)n_free + n_give - n_take > p.n_blocks) status = -2 - B;
    else if (n_take > n_free + n_give) status = n_take - n_free - n_give;
    const bool ok = status == 0;                             // uniform over the grid
    int rp = ok ? (int)(rb + lo + ((int64_t)hi << 20) - rows) : 0;
    tb = ok ? tb + ti - take : 0;
    gb = ok ? gb + gi - give : 0;
    for (int b = b0; b < b1; ++b) {                          // exclusive prefixes
        const int add = row_pre[b], d = take_pre[b];
        row_pre[b] = rp; take_pre[b] = tb; give_pre[b] = gb;
        if (ok) { rp += add; tb += max(d, 0); gb += max(-d, 0); }
    }
    const int taken = ok ? n_take : 0, given = ok ? n_give : 0, described = ok ? (int)n_rows : 0;
    if (tid == NT - 1) { row_pre[B] = described; take_pre[B] = taken; give_pre[B] = given; }
    __syncthreads();

    auto returned = [&](int i) {                             // id of returned page i
        const int b = m5_upper(give_pre, B, i), need = have[b] - (give_pre[b + 1] - give_pre[b]);
        return p.block_table[(int64_t)b * p.table_rs + need + (i - give_pre[b])];
    };
    auto allocation = [&](int a) {                           // id of allocation a
        const int src = m5_plan_source(a, given, n_free);
        return src >= 0 ? p.free_blocks[src] : returned(-1 - src);
    };
    const int gt = blockIdx.x * NT + tid, gn = gridDim.x * NT;
    if (p.slot_map) {
        constexpr int U = 4;
        int top = 1;
        while (2 * top < B) top *= 2;
        for (int64_t r0 = gt; r0 < p.n_rows; r0 += (int64_t)U * gn) {
            int b[U], pos[U], id[U];
#pragma unroll
            for (int u = 0; u < U; ++u) b[u] = 0;
            for (int s = top; s; s >>= 1)                    // the last request that starts at or before the row
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int mid = b[u] + s;
                    if (mid < B && row_pre[min(mid, B)] <= r0 + (int64_t)u * gn) b[u] = mid;
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + (int64_t)u * gn;
                pos[u] = id[u] = -1;
                if (r < described) {
                    pos[u] = keep[b[u]] + ((int)r - row_pre[b[u]]);
                    const int page = pos[u] >> shift, h = have[b[u]];
                    id[u] = page < h ? p.block_table[(int64_t)b[u] * p.table_rs + page] : allocation(take_pre[b[u]] + (page - h));
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t r = r0 + (int64_t)u * gn;
                if (r >= p.n_rows) break;
                p.slot_map[r] = m5_block(id[u], p.n_blocks) >= 0 ? (id[u] << shift) + (pos[u] & ((1 << shift) - 1)) : -1;
                p.positions[r] = pos[u];
            }
        }
    }
    for (int a = gt; a < taken; a += gn) {
        const int b = m5_upper(take_pre, B, a);
        p.block_table[(int64_t)b * p.table_rs + have[b] + (a - take_pre[b])] = allocation(a);
    }
    for (int i = taken + gt; i < given; i += gn) p.free_blocks[m5_plan_push(i, given, n_free)] = returned(i);
    if (blockIdx.x == 0)
        for (int b = tid; b <= B; b += NT) p.q_start[b] = row_pre[b];

    // This workgroup has read all that it will of seq_len and the state (every load has been used or is waited for here): no cache has to
    // be written back for the others to know, so the ticket is a relaxed one.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) last = gridDim.x == 1 || __hip_atomic_fetch_add(&p.state[M5_PST_ROWS + 1], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    if (ok)
        for (int b = tid; b < B; b += NT) p.seq_len[b] = keep[b] + (row_pre[b + 1] - row_pre[b]);
    if (tid == 0) {
        p.state[M5_PST_FREE] = n_free + given - taken;
        p.state[M5_PST_STATUS] = status;
        p.state[M5_PST_ROWS] = described;
        p.state[M5_PST_ROWS + 1] = 0;
    }
}

template <int NT>
int launch_plan(const M5PagedPlanArgs& a, int shift, int grid, hipStream_t s) {
    const int lds = 5 * (a.n_seq + 1) * (int)sizeof(int);
    if (lds > 48 * 1024 && hipFuncSetAttribute((const void*)paged_plan_kernel<NT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return M5_ERR_LAUNCH;
    hipLaunchKernelGGL(paged_plan_kernel<NT>, dim3((unsigned)grid), dim3(NT), lds, s, a, shift);
    M5_CHECK_LAUNCH();
    return M5_OK;
}

// ---------------------------------------------------------------------------------------------------- m5_paged_rope_cache
// A group of head_dim / EPL lanes holds one head, 16 bytes per lane: the sum of squares is a few cross-lane adds, an adjacent pair
// lies in one lane, a half-split pair in two lanes n_pairs / EPL apart.  A workgroup walks the heads of one row, U per group with their
// loads in flight together; the row's cosines and sines and the norm weights stay in registers.
template <typename T, int HD, bool INTER, int U>
__global__ __launch_bounds__(256) void paged_rope_kernel(M5PagedRopeArgs p, int shift) {
    using st = typename T::storage;
    constexpr int E = T::EPL, L = HD / E, G = 256 / L;       // elements per lane, lanes per head, heads at a time
    const int row = blockIdx.x, tid = threadIdx.x, l = tid % L, g = tid / L;
    const int e0 = l * E, n_qk = p.n_heads + p.n_kv_heads, heads = n_qk + p.n_kv_heads;
    const int first = blockIdx.y * (U * G);
    const st* src = (const st*)p.qkv + (int64_t)row * p.qkv_rs + e0;
    Vec16<T> v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {                            // requested before anything is waited for
        v[k].zero();
        if (first + k * G + g < heads) v[k].load(src + (int64_t)(first + k * G + g) * HD);
    }
    const int pos = p.positions[row], slot = p.slot_map[row];
    if (pos < 0 || pos >= p.n_pos || slot < 0 || (slot >> shift) >= p.n_blocks) return;        // padding (workgroup-uniform)
    const bool turns = e0 < 2 * p.n_pairs;                   // n_pairs is a multiple of 8: a lane's elements all turn or none do
    const bool second = !INTER && e0 >= p.n_pairs;
    constexpr int NC = INTER ? E / 2 : E;                    // pairs of a lane
    float c[NC], s[NC];
    {
        const int pair = INTER ? e0 >> 1 : (second ? e0 - p.n_pairs : e0);
        const float4* cs = reinterpret_cast<const float4*>(p.rope + ((int64_t)pos * p.n_pairs + (turns ? pair : 0)) * 2);
#pragma unroll
        for (int i = 0; i < NC; i += 2) {
            const float4 t = turns ? cs[i / 2] : make_float4(1.f, 0.f, 1.f, 0.f);
            c[i] = t.x;
            s[i] = second ? -t.y : t.y;
            c[i + 1] = t.z;
            s[i + 1] = second ? -t.w : t.w;
        }
    }
    const int apart = p.n_pairs / E;
    const int partner = ((tid & 63) & ~(L - 1)) + (second ? l - apart : l + apart) % L;
    const int64_t blk = slot >> shift, off = slot & ((1 << shift) - 1);
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const int h = first + k * G + g;
        if (h - g >= heads) break;                           // (uniform)
        const bool is_q = h < p.n_heads, is_v = h >= n_qk;
        if (h - g < n_qk) {                                  // some group here holds a q or k head
            float x[E], y[E];
            v[k].to_float(x);
            const float* w = is_q ? p.q_norm : p.k_norm;
            if (p.q_norm || p.k_norm) {
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) ss = fmaf(x[i], x[i], ss);
                ss += lane_xor1(ss);
                ss += lane_xor2(ss);
                ss += lane_xor4(ss);
                if (L >= 16) ss += lane_xor8(ss);
                if (L >= 32) ss += lane_xor16(ss);
                if (w) {
                    const float r = 1.0f / sqrtf(ss * (1.0f / HD) + p.eps);
#pragma unroll
                    for (int i = 0; i < E; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(w + e0 + i);
                        x[i] = x[i] * r * f.x;
                        x[i + 1] = x[i + 1] * r * f.y;
                        x[i + 2] = x[i + 2] * r * f.z;
                        x[i + 3] = x[i + 3] * r * f.w;
                    }
                }
            }
            if constexpr (INTER) {
#pragma unroll
                for (int i = 0; i < E; i += 2) {
                    y[i] = x[i] * c[i / 2] - x[i + 1] * s[i / 2];
                    y[i + 1] = x[i] * s[i / 2] + x[i + 1] * c[i / 2];
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) {                // (second half: s holds -sin, so both halves are x cos - partner s)
                    const float o = apart == 8 ? lane_xor8(x[i]) : (apart == 4 ? lane_xor4(x[i]) : __shfl(x[i], partner));
                    y[i] = x[i] * c[i] - o * s[i];
                }
            }
            if (!is_v) {
                st out[E];
#pragma unroll
                for (int i = 0; i < E; ++i) out[i] = T::from_f32(turns ? y[i] : x[i]);
                v[k].raw = *reinterpret_cast<const uint4*>(out);
            }
        }
        if (h >= heads) continue;
        st* dst;
        if (is_q) dst = (st*)p.q_out + (int64_t)row * p.q_rs + (int64_t)h * p.q_hs;
        else if (!is_v) dst = (st*)p.k_cache + blk * p.k_bs + (int64_t)(h - p.n_heads) * p.k_hs + off * p.k_ss;
        else dst = (st*)p.v_cache + blk * p.v_bs + (int64_t)(h - n_qk) * p.v_hs + off * p.v_ss;
        *reinterpret_cast<uint4*>(dst + e0) = v[k].raw;
    }
}

template <typename T, int HD, int U>
void launch_rope_u(const M5PagedRopeArgs& a, int shift, hipStream_t s) {
    const int per = 256 / (HD / T::EPL) * U;                 // heads of a workgroup
    const dim3 grid(a.n_rows, (a.n_heads + 2 * a.n_kv_heads + per - 1) / per);
    if (a.interleaved) hipLaunchKernelGGL((paged_rope_kernel<T, HD, true, U>), grid, dim3(256), 0, s, a, shift);
    else hipLaunchKernelGGL((paged_rope_kernel<T, HD, false, U>), grid, dim3(256), 0, s, a, shift);
}
template <typename T, int HD>
void launch_rope_hd(const M5PagedRopeArgs& a, int shift, hipStream_t s) {
    // Few rows: more, shorter workgroups (37 rows of 72 heads of 64: 2.9 us against 3.7).  Many: a row's table values serve four heads
    // (16384 rows of 48 heads of 128: 83 us, 4.9 TB/s, against 109); equal at about 1000 rows (5.7 / 5.9 us, 9.2 / 8.7 us).
    if (a.n_rows < 1024) launch_rope_u<T, HD, 1>(a, shift, s);
    else launch_rope_u<T, HD, 4>(a, shift, s);
}
template <typename T>
int launch_rope(const M5PagedRopeArgs& a, int shift, hipStream_t s) {
    if (a.head_dim == 64) launch_rope_hd<T, 64>(a, shift, s);
    else launch_rope_hd<T, 128>(a, shift, s);
    M5_CHECK_LAUNCH();
    return M5_OK;
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int epl) {
    return ((uintptr_t)p & 15) == 0 && a % epl == 0 && b % epl == 0 && c % epl == 0;
}

}  // namespace

extern "C" int m5_paged_plan(const M5PagedPlanArgs* a, void* stream) {
    if (!a || !a->seq_len || !a->keep_len || !a->new_len || !a->block_table || !a->free_blocks || !a->state || !a->q_start) return M5_ERR_ARG;
    const int shift = m5_log2(a->block_size);
    if (a->n_seq <= 0 || a->table_width <= 0 || a->n_blocks <= 0 || shift < 0 || a->table_rs < a->table_width) return M5_ERR_ARG;
    if (!a->slot_map != !a->positions || (a->slot_map && a->n_rows < 0)) return M5_ERR_ARG;
    // positions, slots and (request, page) pairs are counted in 32 bits
    if (a->n_seq > PLAN_MAX_SEQ || a->block_size > 1024 || ((int64_t)a->table_width << shift) > INT_MAX || ((int64_t)a->n_blocks << shift) > INT_MAX ||
        (int64_t)a->n_seq * a->table_width > INT_MAX)
        return M5_ERR_UNSUPPORTED;
    const int64_t rows = a->slot_map ? a->n_rows : 0, pages = min((int64_t)a->n_seq * a->table_width, (int64_t)a->n_blocks);
    // A workgroup per 2048 rows (1024 requests admitted and retired, 474 thousand rows: 19.1 us; 22 / 26 / 36 with 4096 / 8192 / 16384) or, in
    // large pools, per 512 blocks that the step might give back (20.1 us with 2048).  One workgroup alone needs no ticket: 48 requests
    // with drafts 4.3 us a call against 4.9.
    const int64_t work = max(rows / 2048, pages < 8192 ? 0 : pages / 512);
    const int grid = (int)min(max(work, (int64_t)1), (int64_t)256);
    if (a->n_seq <= 256) return launch_plan<256>(*a, shift, grid, (hipStream_t)stream);
    return launch_plan<1024>(*a, shift, grid, (hipStream_t)stream);
}

extern "C" int m5_paged_rope_cache(int dtype, const M5PagedRopeArgs* a, void* stream) {
    if (!a || !a->qkv || !a->rope || !a->positions || !a->slot_map || !a->q_out || !a->k_cache || !a->v_cache) return M5_ERR_ARG;
    const int shift = m5_log2(a->block_size);
    if (a->n_rows < 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->n_pos <= 0 || a->n_blocks <= 0 || shift < 0) return M5_ERR_ARG;
    if (dtype != M5_F32 && dtype != M5_F16 && dtype != M5_BF16) return M5_ERR_UNSUPPORTED;
    if ((a->head_dim != 64 && a->head_dim != 128) || a->block_size > 1024 || ((int64_t)a->n_blocks << shift) > INT_MAX) return M5_ERR_UNSUPPORTED;
    if (a->n_pairs <= 0 || a->n_pairs % 8 || 2 * a->n_pairs > a->head_dim) return M5_ERR_UNSUPPORTED;
    const int epl = dtype == M5_F32 ? 4 : 8;
    if (!aligned(a->qkv, a->qkv_rs, 0, 0, epl) || !aligned(a->q_out, a->q_rs, a->q_hs, 0, epl) || !aligned(a->k_cache, a->k_bs, a->k_hs, a->k_ss, epl) ||
        !aligned(a->v_cache, a->v_bs, a->v_hs, a->v_ss, epl) || ((uintptr_t)a->rope & 15) || ((uintptr_t)a->q_norm & 15) || ((uintptr_t)a->k_norm & 15))
        return M5_ERR_UNSUPPORTED;
    if (a->n_rows == 0) return M5_OK;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case M5_F32: return launch_rope<F32T>(*a, shift, s);
        case M5_F16: return launch_rope<F16T>(*a, shift, s);
        default: return launch_rope<BF16T>(*a, shift, s);
    }
}
