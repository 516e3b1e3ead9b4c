// Attention of new tokens (single ones, drafts, prompt chunks) over a paged KV cache (m5_paged_attention, include/mars5_paged.h).
#include "common.h"
#include "paged_index.h"
#include <limits.h>

namespace {

// One wave per (row, query head): 64 keys at a time, one per lane for the scores, one feature (or two) per lane for the values.
template <typename T, int HD>
__global__ __launch_bounds__(64) void paged_attn_row_kernel(M5PagedAttnArgs p, int shift) {
    using st = typename T::storage;
    constexpr int E = T::EPL, ND = HD / 64;
    __shared__ __attribute__((aligned(16))) float qs[HD];
    __shared__ float ps[64];
    __shared__ int64_t vs[64];
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    int lo = 0, hi = p.n_seq;                                // request of this row: last b with q_start[b] <= row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.q_start[mid] <= row) lo = mid; else hi = mid;
    }
    const int b = lo;
    const M5Request rq = m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, (int64_t)p.table_width << shift);
    if (row < rq.r0 || row >= rq.r1) return;                 // padding
    const int pos = rq.len - (rq.r1 - row);
    const int k1 = m5_key_hi(pos, rq.len), k0 = m5_key_lo(pos, p.window);
    const int kvh = h / (p.n_heads / p.n_kv_heads);
    const st* q = (const st*)p.q + (int64_t)row * p.q_rs + (int64_t)h * p.q_hs;
#pragma unroll
    for (int i = 0; i < ND; ++i) qs[lane + 64 * i] = T::to_f32(q[lane + 64 * i]);
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = 0.f;
    for (int kb = k0; kb < k1; kb += 64) {
        const int key = kb + lane;
        int id = -1;
        if (key < k1) id = m5_block(p.block_table[(int64_t)b * p.table_rs + (key >> shift)], p.n_blocks);
        float s = -INFINITY;
        int64_t vo = -1;
        if (id >= 0) {
            const int off = key & ((1 << shift) - 1);
            const st* k = (const st*)p.k_cache + (int64_t)id * p.k_bs + (int64_t)kvh * p.k_hs + (int64_t)off * p.k_ss;
            vo = (int64_t)id * p.v_bs + (int64_t)kvh * p.v_hs + (int64_t)off * p.v_ss;
            float acc = 0.f;
            for (int d = 0; d < HD; d += E) {
                Vec16<T> v;
                v.load(k + d);
                float x[E];
                v.to_float(x);
#pragma unroll
                for (int i = 0; i < E; ++i) acc = fmaf(x[i], qs[d + i], acc);
            }
            s = acc * p.scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float mu = mn == -INFINITY ? 0.f : mn;
        const float e = id >= 0 ? expf(s - mu) : 0.f;
        const float alpha = expf(m - mu);
        l = l * alpha + wave_sum(e);
        m = mn;
        __syncthreads();
        ps[lane] = e;
        vs[lane] = vo;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= alpha;
        for (int j = 0; j < 64; ++j) {
            if (vs[j] < 0) continue;
            const st* v = (const st*)p.v_cache + vs[j];
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] = fmaf(ps[j], T::to_f32(v[lane + 64 * i]), o[i]);
        }
    }
    st* out = (st*)p.out + (int64_t)row * p.o_rs + (int64_t)h * p.o_hs;
#pragma unroll
    for (int i = 0; i < ND; ++i) out[lane + 64 * i] = T::from_f32(l != 0.f ? o[i] / l : 0.f);
}

template <typename T>
int launch(const M5PagedAttnArgs& a, int shift, hipStream_t s) {
    const dim3 grid(a.n_rows, a.n_heads);
    if (a.head_dim == 64) hipLaunchKernelGGL((paged_attn_row_kernel<T, 64>), grid, dim3(64), 0, s, a, shift);
    else hipLaunchKernelGGL((paged_attn_row_kernel<T, 128>), grid, dim3(64), 0, s, a, shift);
    M5_CHECK_LAUNCH();
    return M5_OK;
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int epl) {
    return ((uintptr_t)p & 15) == 0 && a % epl == 0 && b % epl == 0 && c % epl == 0;
}

int check(int dtype, const M5PagedAttnArgs* a) {
    if (!a || !a->q || !a->k_cache || !a->v_cache || !a->block_table || !a->seq_len || !a->q_start || !a->out) return M5_ERR_ARG;
    const int shift = m5_log2(a->block_size);
    if (a->n_seq <= 0 || a->n_rows < 0 || a->n_heads <= 0 || a->n_kv_heads <= 0 || a->n_heads % a->n_kv_heads || a->table_width <= 0 || a->n_blocks <= 0 ||
        shift < 0 || a->table_rs < a->table_width || a->window < 0 || a->workspace_bytes < 0 || !(a->scale > 0.f))
        return M5_ERR_ARG;
    if (dtype != M5_F32 && dtype != M5_F16 && dtype != M5_BF16) return M5_ERR_UNSUPPORTED;
    if ((a->head_dim != 64 && a->head_dim != 128) || a->block_size > 1024 || a->n_seq > 8192 || ((int64_t)a->table_width << shift) > INT_MAX ||
        ((int64_t)a->n_blocks << shift) > INT_MAX)
        return M5_ERR_UNSUPPORTED;
    const int epl = dtype == M5_F32 ? 4 : 8;
    if (!aligned(a->q, a->q_rs, a->q_hs, 0, epl) || !aligned(a->out, a->o_rs, a->o_hs, 0, epl) || !aligned(a->k_cache, a->k_bs, a->k_hs, a->k_ss, epl) ||
        !aligned(a->v_cache, a->v_bs, a->v_hs, a->v_ss, epl) || ((uintptr_t)a->workspace & 15))
        return M5_ERR_UNSUPPORTED;
    return M5_OK;
}

}  // namespace

extern "C" int m5_paged_attention_workspace(int dtype, const M5PagedAttnArgs* a, int64_t* bytes) {
    const int rc = check(dtype, a);
    if (rc != M5_OK) return rc;
    if (!bytes) return M5_ERR_ARG;
    *bytes = 0;
    return M5_OK;
}

extern "C" int m5_paged_attention(int dtype, const M5PagedAttnArgs* a, void* stream) {
    const int rc = check(dtype, a);
    if (rc != M5_OK) return rc;
    if (a->n_rows == 0) return M5_OK;
    const int shift = m5_log2(a->block_size);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case M5_F32: return launch<F32T>(*a, shift, s);
        case M5_F16: return launch<F16T>(*a, shift, s);
        default: return launch<BF16T>(*a, shift, s);
    }
}
