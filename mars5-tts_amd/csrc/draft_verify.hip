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

template <typename T>
__global__ __launch_bounds__(NT) void draft_verify_kernel(M5DraftVerifyArgs p) {
    using st = typename T::storage;
    __shared__ unsigned long long wk[2][NT / 64];
    __shared__ int sh_count, sh_any[NT / 64];
    const int b = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const M5Request rq = m5_request(p.row_start[b], p.row_start[b + 1], 0, p.n_rows, 0);
    const int rows = rq.r1 - rq.r0, n = min(rows, p.out_width);
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
    int any = 0;
    if (n > 0) {
        const int64_t r = rq.r0 + count;
        const bool rejected = count < n - 1;
        const st* t = target + r * p.t_rs;
        const st* q = rejected && draft ? draft + r * p.d_rs : nullptr;
        const int64_t gone = rejected && !draft ? p.tokens[r + 1] : -1;
        const float* noise = p.noise + (int64_t)b * p.noise_rs;
        for (int v = tid; v < p.vocab; v += NT) {
            const float x = T::to_f32(t[v]), e = noise[v];
            float w = q ? x - T::to_f32(q[v]) : x;
            if (v == gone) w = 0.f;
            any |= w > 0.f;
            const unsigned long long c = candidate(w, e, v), d = candidate(x, e, v);
            best = c > best ? c : best;
            plain = d > plain ? d : plain;
        }
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
            any |= sh_any[w];
        }
        any |= sh_any[0];
        const unsigned long long key = any ? best : plain;
        const int token = key ? (int)~(uint32_t)key : 0;
        wk[0][0] = (unsigned)token;
        p.n_out[b] = n > 0 ? count + 1 : 0;
        if (p.keep_len) p.keep_len[b] = p.seq_len[b] - rows + (n > 0 ? count + 1 : 0);
    }
    __syncthreads();
    for (int i = tid; i < p.out_width; i += NT)
        p.out_tokens[(int64_t)b * p.out_rs + i] = n <= 0 || i > count ? -1 : (i < count ? p.tokens[rq.r0 + i + 1] : (int64_t)wk[0][0]);
}

}  // namespace

extern "C" int m5_draft_verify(int dtype, const M5DraftVerifyArgs* a, void* stream) {
    if (!a || !a->target || !a->tokens || !a->row_start || !a->uniforms || !a->noise || !a->out_tokens || !a->n_out) return M5_ERR_ARG;
    if (a->n_rows < 0 || a->vocab <= 0 || a->n_seq <= 0 || a->out_width <= 0 || a->t_rs < a->vocab || (a->draft && a->d_rs < a->vocab) || a->noise_rs < a->vocab ||
        a->out_rs < a->out_width || !a->seq_len != !a->keep_len || a->workspace_bytes < 0)
        return M5_ERR_ARG;
    if (dtype != M5_F32 && dtype != M5_F16 && dtype != M5_BF16) return M5_ERR_UNSUPPORTED;
    if ((uintptr_t)a->workspace & 15) return M5_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case M5_F32: hipLaunchKernelGGL(draft_verify_kernel<F32T>, dim3(a->n_seq), dim3(NT), 0, s, *a); break;
        case M5_F16: hipLaunchKernelGGL(draft_verify_kernel<F16T>, dim3(a->n_seq), dim3(NT), 0, s, *a); break;
        default: hipLaunchKernelGGL(draft_verify_kernel<BF16T>, dim3(a->n_seq), dim3(NT), 0, s, *a); break;
    }
    M5_CHECK_LAUNCH();
    return M5_OK;
}
