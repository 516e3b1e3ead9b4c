// Drafted tokens against the target's probabilities (m5_draft_verify, include/mars5_paged.h).
#include "common.h"
#include "paged_index.h"

namespace {

constexpr int NT = 256;

// A candidate as one word whose maximum is the answer: score bits (scores are >= 0, so they order as integers) above the
// complement of the index (ties: the lowest).  0 = no candidate.
__device__ inline unsigned long long candidate(float w, float noise, int v) {
    const float score = w / noise;
    return (w > 0.f && score > 0.f) ? ((unsigned long long)__float_as_uint(score) << 32) | (uint32_t)~v : 0ull;
}
__device__ inline unsigned long long wave_max64(unsigned long long v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const unsigned long long o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

// What the workgroups of a request leave for each other (workspace; all zero between calls).
struct Meet { unsigned long long best, plain; uint32_t any, ticket; uint64_t pad; };
static_assert(sizeof(Meet) == M5_DRAFT_WS_BYTES, "M5_DRAFT_WS_BYTES");

// 16 bytes of probabilities from any element-aligned address (rows of an odd vocabulary)
template <typename T>
__device__ inline void load_any(const typename T::storage* p, float (&x)[T::EPL]) {
    typename T::storage e[T::EPL];
    __builtin_memcpy(e, p, 16);
#pragma unroll
    for (int i = 0; i < T::EPL; ++i) x[i] = T::to_f32(e[i]);
}

// Workgroup (request, part of the vocabulary).  Every workgroup of a request finds the accepted drafts itself (one wave, one draft per
// lane), then reads its part of one target row, one draft row and the noise; the parts meet by 64-bit maxima, whose result does not
// depend on their order, and the workgroup that arrives last writes the outputs.  HBM bound for many or long rows; below that a chain
// of memory round trips (offsets, tokens, their probabilities, the row): 6.2 us at 32 x 4096.
template <typename T>
__global__ __launch_bounds__(NT) void draft_verify_kernel(M5DraftVerifyArgs p, int parts, int span) {
    using st = typename T::storage;
    constexpr int E = T::EPL;
    __shared__ unsigned long long wk[2][NT / 64];
    __shared__ int sh_count, sh_any[NT / 64], sh_last;
    const int b = blockIdx.x / parts, part = blockIdx.x % parts, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const bool refused = p.plan_state && p.plan_state[M5_PST_STATUS] != 0;       // no rows, and keep_len stays the plan's
    const M5Request rq = m5_request(p.row_start[b], p.row_start[b + 1], 0, p.n_rows, 0);
    const int rows = refused ? 0 : rq.r1 - rq.r0, n = min(rows, p.out_width);
    const st* target = (const st*)p.target;
    const st* draft = (const st*)p.draft;
    if (wave == 0) {                                         // drafts accepted before the first that is not
        int count = 0;
        for (int base = 0; base < n - 1; base += 64) {
            bool yes = false;
            if (base + lane < n - 1) {
                const int64_t r = rq.r0 + base + lane, d = p.tokens[r + 1];
                if (d >= 0 && d < p.vocab) {
                    const float q = draft ? T::to_f32(draft[r * p.d_rs + d]) : 1.f;
                    yes = p.uniforms[r] * q < T::to_f32(target[r * p.t_rs + d]);
                }
            }
            const unsigned long long no = ~__ballot(yes);
            const int run = no ? (int)__builtin_ctzll(no) : 64;
            count += run;
            if (run < 64) break;
        }
        if (lane == 0) sh_count = min(count, max(n - 1, 0));
    }
    __syncthreads();
    const int count = sh_count;
    unsigned long long best = 0, plain = 0;
    bool any = false;
    if (n > 0) {
        const int64_t r = rq.r0 + count;
        const bool rejected = count < n - 1;
        const st* t = target + r * p.t_rs;
        const st* q = rejected && draft ? draft + r * p.d_rs : nullptr;
        const int64_t gone = rejected && !draft ? p.tokens[r + 1] : -1;
        const float* noise = p.noise + (int64_t)b * p.noise_rs;
        const int v0 = part * span, v1 = min(v0 + span, p.vocab);
        auto one = [&](int v, float x, float qx, float e) {
            const float w = v == gone ? 0.f : x - qx;        // (qx 0 without a draft: exact)
            any |= w > 0.f;
            const unsigned long long c = candidate(w, e, v);
            best = c > best ? c : best;
            if (rejected) {                                  // should nothing be left, the target itself is drawn from
                const unsigned long long d = candidate(x, e, v);
                plain = d > plain ? d : plain;
            }
        };
        int v = v0 + tid * E;
        constexpr int U = 2;                                 // vectors of a thread in flight (one: 6.5 instead of 6.2 us at 32 x 4096)
        for (; v + (U - 1) * NT * E + E <= v1; v += U * NT * E) {
            float x[U][E], y[U][E], e[U][E];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                load_any<T>(t + v + u * NT * E, x[u]);
                if (q) load_any<T>(q + v + u * NT * E, y[u]);
                __builtin_memcpy(e[u], noise + v + u * NT * E, sizeof(e[u]));
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < E; ++i) one(v + u * NT * E + i, x[u][i], q ? y[u][i] : 0.f, e[u][i]);
        }
        for (; v + E <= v1; v += NT * E) {
            float x[E], y[E], e[E];
            load_any<T>(t + v, x);
            if (q) load_any<T>(q + v, y);
            __builtin_memcpy(e, noise + v, sizeof(e));
#pragma unroll
            for (int i = 0; i < E; ++i) one(v + i, x[i], q ? y[i] : 0.f, e[i]);
        }
        for (; v < v1; ++v) one(v, T::to_f32(t[v]), q ? T::to_f32(q[v]) : 0.f, noise[v]);      // (the one thread that stands at the end)
        if (!rejected) any = true;
    }
    best = wave_max64(best);
    plain = wave_max64(plain);
    const bool wany = __any(any);
    if (lane == 0) { wk[0][wave] = best; wk[1][wave] = plain; sh_any[wave] = wany; }
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < NT / 64; ++w) {
            best = wk[0][w] > best ? wk[0][w] : best;
            plain = wk[1][w] > plain ? wk[1][w] : plain;
        }
        bool some = false;
        for (int w = 0; w < NT / 64; ++w) some |= sh_any[w] != 0;
        bool last = true;
        if (parts > 1) {
            Meet* m = (Meet*)p.workspace + b;
            if (best) __hip_atomic_fetch_max(&m->best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (plain) __hip_atomic_fetch_max(&m->plain, plain, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (some) __hip_atomic_fetch_or(&m->any, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            // the maxima are in memory before the ticket is drawn; everything that crosses is an agent-scope access, so no cache needs to
            // be written back or invalidated (an acquire-release ticket does that to the whole L2, ~50 ns of the chip's time a workgroup)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            last = __hip_atomic_fetch_add(&m->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1;
            if (last) {
                best = __hip_atomic_exchange(&m->best, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                plain = __hip_atomic_exchange(&m->plain, 0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                some = __hip_atomic_exchange(&m->any, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
                __hip_atomic_store(&m->ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
        if (last) {
            const unsigned long long key = some ? best : plain;
            wk[0][0] = key ? (uint32_t)~(uint32_t)key : 0u;
            p.n_out[b] = n > 0 ? count + 1 : 0;
            if (p.keep_len && !refused) p.keep_len[b] = p.seq_len[b] - rows + (n > 0 ? count + 1 : 0);
        }
        sh_last = last;
    }
    __syncthreads();
    if (!sh_last) return;
    for (int i = tid; i < p.out_width; i += NT)
        p.out_tokens[(int64_t)b * p.out_rs + i] = n <= 0 || i > count ? -1 : (i < count ? p.tokens[rq.r0 + i + 1] : (int64_t)wk[0][0]);
}

template <typename T>
int launch(const M5DraftVerifyArgs& a, hipStream_t s) {
    // A vocabulary is split when there are too few requests to fill the chip: about 1024 workgroups, of 4096 entries at least (2048: 10.7 us
    // instead of 8.7 at 16 x 50257 in 16 bits; twice or four times the workgroups change nothing).  128 x 128011 in fp32, 197 MB: 41.5 us, 4.7 TB/s,
    // a copy's rate, where four inputs take turns; 35 us on one input again and again (it fits the last-level cache); one workgroup per
    // request 455 us.
    int parts = 1;
    if (a.workspace && a.workspace_bytes / M5_DRAFT_WS_BYTES >= a.n_seq) {
        const int by_size = (a.vocab + 4095) / 4096, by_chip = (1024 + a.n_seq - 1) / a.n_seq;
        parts = by_size < by_chip ? by_size : by_chip;
    }
    const int step = NT * T::EPL;
    int span = (a.vocab + parts - 1) / parts;
    if (parts > 1) span = (span + step - 1) / step * step;
    parts = (a.vocab + span - 1) / span;
    hipLaunchKernelGGL(draft_verify_kernel<T>, dim3((unsigned)(a.n_seq * parts)), dim3(NT), 0, s, a, parts, span);
    M5_CHECK_LAUNCH();
    return M5_OK;
}

}  // namespace

extern "C" int m5_draft_verify(int dtype, const M5DraftVerifyArgs* a, void* stream) {
    if (!a || !a->target || !a->tokens || !a->row_start || !a->uniforms || !a->noise || !a->out_tokens || !a->n_out) return M5_ERR_ARG;
    if (a->n_rows < 0 || a->vocab <= 0 || a->n_seq <= 0 || a->out_width <= 0 || a->t_rs < a->vocab || (a->draft && a->d_rs < a->vocab) || a->noise_rs < a->vocab ||
        a->out_rs < a->out_width || !a->seq_len != !a->keep_len || a->workspace_bytes < 0)
        return M5_ERR_ARG;
    if (a->n_seq > (1 << 20) || a->vocab > (1 << 30)) return M5_ERR_UNSUPPORTED;
    if (dtype != M5_F32 && dtype != M5_F16 && dtype != M5_BF16) return M5_ERR_UNSUPPORTED;
    if ((uintptr_t)a->workspace & 15) return M5_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case M5_F32: return launch<F32T>(*a, s);
        case M5_F16: return launch<F16T>(*a, s);
        default: return launch<BF16T>(*a, s);
    }
}
