// Attention of new tokens (single ones, drafts, prompt chunks) over a paged KV cache (m5_paged_attention, include/mars5_paged.h).
//
//   o[r][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale log2(e) q[r][h] . k_j - m),   m = running maximum
//
// Rows.  The query heads of one kv head and the new tokens of one request are packed into rows rho = token * group + head, so every
// key and value is read once for all of them.  A tile is 16 R rows ("few": single tokens, drafts; all types) or 128 ("many": prompt
// chunks; 16-bit).  Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T: the row is the matrix column, i.e. a lane
// owns one row, the softmax state is lane-local, and P^T goes into the second product straight from the registers of the first.
//   few   16x16 matrix instructions.  The waves of a workgroup take different keys (32 at a time, 16 in 32 bits) of the same rows,
//         each with a private ring of two stages in LDS, and meet once at the end: no barrier in the key loop.
//   many  32x32 matrix instructions.  Each wave owns 32 rows; the waves share 64-key tiles, one barrier per tile.
// K and V rows go from memory into LDS by DMA (global_load_lds, 16 bytes per lane; the page lookup is in the lane's address).  16-byte
// chunks of a row are stored XOR-swizzled so that the fragment reads spread over all banks: K fragments are ds_read_b128, V fragments
// (keys along the register, features along the lanes) are ds_read_b64_tr_b16, which transposes 4 x 16 blocks on the way, so the
// cache needs no transposed copy of V.
//
// Work.  Lengths are device data: every workgroup scans the requests (two block reductions) and deals itself items (request, tile,
// key chunk, kv head), kv head fastest, so that the workgroups of one XCD (blockIdx % 8) share a head's keys in their L2.  Keys are
// cut into chunks of C when there are fewer tiles than the chip has places for; partial (o, m, l) of a tile's chunks meet in the
// workspace and the workgroup that arrives last joins them in chunk order (same bits whatever the order of arrival).
//
// Masked places.  Keys outside a tile's range or on a bad page are read from a valid address and their values zeroed in LDS; where some
// rows of a tile see a key and others do not, its non-finite values are taken out of the product and added to the rows that see it
// (0 * inf would be NaN).
#include "common.h"
#include "paged_index.h"
#include <limits.h>

typedef __attribute__((ext_vector_type(8))) _Float16 h8_t;
typedef __attribute__((ext_vector_type(8))) __bf16 b8_t;
typedef __attribute__((ext_vector_type(4))) float f4_t;
typedef __attribute__((ext_vector_type(16))) float f16_t;
typedef __attribute__((ext_vector_type(4))) short s4_t;

namespace {

constexpr int NWAVE = 4, NT = NWAVE * 64;
constexpr int MAXP = 1024;                       // block ids of one key segment held in LDS
constexpr int MAX_SEQ = 4096;                    // item prefix sums in LDS: 16 KB
constexpr int IDS_B = MAXP * 4, ML_B = NWAVE * 64 * 2 * 4 + 64;
constexpr int odd_bytes(int hd) { return NWAVE * 2 * hd * 4; }   // notes of non-finite values: per wave and feature 2 x 32 keys, or 2 x 64 shared

struct Launch {
    M5PagedAttnArgs a;
    int shift, group;
    int target;                                  // items wanted: places on the chip
    int n_slots;                                 // partial results the workspace holds, 0 = keys are not split
    float* slots; int* tickets;
    int64_t slot_floats;                         // floats of one partial result: rows of o, then (m, l) per row
    float sc2;                                   // scale * log2(e)
};

struct Item {
    M5Request rq;
    int b, kvh, rows, rho0, rho1;                // rows of the request's kv head, [rho0, rho1) of them here
    int ka, kb;                                  // keys of this item
    int id, first_id, n_parts;                   // partial results of this tile: slots first_id + p * n_kv_heads
};

// ---------------------------------------------------------------------------------------------------- small pieces
__device__ inline f4_t mma16(const uint4& a, const uint4& b, f4_t c, F16T) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const h8_t*>(&a), *reinterpret_cast<const h8_t*>(&b), c, 0, 0, 0);
}
__device__ inline f4_t mma16(const uint4& a, const uint4& b, f4_t c, BF16T) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const b8_t*>(&a), *reinterpret_cast<const b8_t*>(&b), c, 0, 0, 0);
}
__device__ inline f4_t mma16(const uint4& a, const uint4& b, f4_t c, F32T) {      // four k-slots of 4: the same k order on both sides
    const f4_t x = *reinterpret_cast<const f4_t*>(&a), y = *reinterpret_cast<const f4_t*>(&b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    return c;
}
__device__ inline f16_t mma32(const uint4& a, const uint4& b, f16_t c, F16T) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(*reinterpret_cast<const h8_t*>(&a), *reinterpret_cast<const h8_t*>(&b), c, 0, 0, 0);
}
__device__ inline f16_t mma32(const uint4& a, const uint4& b, f16_t c, BF16T) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const b8_t*>(&a), *reinterpret_cast<const b8_t*>(&b), c, 0, 0, 0);
}

// LDS-DMA of 16 bytes per lane (gemm16.hip): from asm, so that hipcc does not drain it; waited for by vm_wait.
__device__ inline void glds16(const unsigned char* gsrc, uint32_t lds_base) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(gsrc), "s"(lds_base) : "memory");
}
template <int N>
__device__ inline void vm_wait() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }
__device__ inline void lds_wait() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ inline uint2 tr_read(const unsigned char* p) {
    const s4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p);
    return *reinterpret_cast<const uint2*>(&v);
}

// bit e set: element e of the 16 bytes is infinite or NaN
template <typename T>
__device__ inline uint32_t nonfinite_bits(const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (T::EPL == 4) bits |= (w[i] & 0x7f800000u) == 0x7f800000u ? 1u << i : 0u;
        else {
            const uint32_t m = T::id == M5_F16 ? 0x7c00u : 0x7f80u;
            bits |= (w[i] & m) == m ? 1u << (2 * i) : 0u;
            bits |= (w[i] & (m << 16)) == (m << 16) ? 2u << (2 * i) : 0u;
        }
    }
    return bits;
}
// Takes the non-finite elements `bits` (features d0 ..) of key `at` out of v and notes them: up / down have the key's bit set where a row
// that sees the key gets +inf / -inf (NaN: both).
template <typename T, typename M>
__device__ inline void note_nonfinite(uint4& v, uint32_t bits, int d0, int at, M* up, M* down) {
    typename T::storage e[T::EPL];
    *reinterpret_cast<uint4*>(e) = v;
#pragma unroll
    for (int i = 0; i < T::EPL; ++i)
        if ((bits >> i) & 1) {
            const float f = T::to_f32(e[i]);
            if (!(f < 0.f)) atomicOr(&up[d0 + i], (M)1 << at);
            if (!(f > 0.f)) atomicOr(&down[d0 + i], (M)1 << at);
            e[i] = 0;
        }
    v = *reinterpret_cast<const uint4*>(e);
}
__device__ inline float infinite_part(bool up, bool down) { return (up ? INFINITY : 0.f) - (down ? INFINITY : 0.f); }
// bits of the keys kb + i, i < 64, of `there` that lie in [lo, hi]
__device__ inline unsigned long long below(int n) { return n <= 0 ? 0ull : (n >= 64 ? ~0ull : (1ull << n) - 1); }
__device__ inline unsigned long long seen(unsigned long long there, int kb, int lo, int hi) { return there & below(hi - kb + 1) & ~below(lo - kb); }

// block id of a key through the segment's ids in LDS, -1 outside [ka, kb)
__device__ inline int key_block(const int* ids, int page0, int key, int ka, int kb, int shift) {
    return key >= ka && key < kb ? ids[(key >> shift) - page0] : -1;
}

// softmax state of one row block: new maximum from this lane's scores (already reduced over the lanes of the row)
struct Soft {
    float m, l;
    __device__ inline float step(float mx, float& use) {     // returns the factor of everything accumulated so far
        const float mn = fmaxf(m, mx);
        use = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - use);
        m = mn;
        return alpha;
    }
};

// one row's four features: to the output, or to the item's partial result
template <typename T, int HD>
__device__ inline void put_row(const Launch& L, const Item& it, int row, int d, f4_t o, float m, float l) {
    const int rho = it.rho0 + row;
    if (it.n_parts <= 1) {
        const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);         // (NaN stays NaN)
        typename T::storage* out = (typename T::storage*)L.a.out + (int64_t)(it.rq.r0 + rho / L.group) * L.a.o_rs +
                                   (int64_t)(it.kvh * L.group + rho % L.group) * L.a.o_hs + d;
        if (l == 0.f) o = f4_t{0.f, 0.f, 0.f, 0.f};
        if constexpr (T::EPL == 4) *reinterpret_cast<f4_t*>(out) = o * inv;
        else *reinterpret_cast<uint2*>(out) = m5_pack4<T>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
    }
}

// ------------------------------------------------------------------------------------------------------ few rows
template <typename T, int HD, int R, int NW>
struct Few {
    using st = typename T::storage;
    static constexpr int ES = sizeof(st), RB = HD * ES;          // bytes of a row
    static constexpr int KS = ES == 4 ? 16 : 32, SUB = KS / 16;  // keys of a stage
    static constexpr int LPR = RB / 16, RPI = 64 / LPR;          // lanes per row, rows per DMA instruction
    static constexpr int NI = KS / RPI;                          // DMA instructions of K (and of V) per stage
    static constexpr int OP_B = KS * RB, STAGE_B = 2 * OP_B, WAVE_B = 2 * STAGE_B;
    static constexpr int NF = RB / 64, ND = HD / 16;             // K fragments per key row block, feature blocks of V
    static constexpr int LDS_B = NW * WAVE_B;
    static_assert(R * 16 * HD * 4 <= WAVE_B, "the waves' results meet in their rings");

    // 16-byte chunk swizzles: 16 (8 for V) rows of one chunk column fall into different banks
    __device__ static inline int kswz(int row) { return RB == 128 ? (row >> 1) & 7 : row & 15; }
    __device__ static inline int vswz(int row) { return ES == 4 ? ((row >> 2) & 3) << 2 : (RB == 128 ? ((row >> 1) & 3) << 1 : (row & 7) << 1); }

    // V of a stage that not all rows see whole: keys that are not there become zeros, non-finite values are noted and taken out (true).
    __device__ static bool clean(unsigned char* vs, uint32_t there, uint32_t* up, uint32_t* down) {
        const int lane = threadIdx.x & 63;
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int row = j * RPI + lane / LPR;
            const uint4 v = *reinterpret_cast<const uint4*>(vs + j * 1024 + lane * 16);
            any |= (there >> row) & 1 ? nonfinite_bits<T>(v) : 0u;
            if (!((there >> row) & 1)) *reinterpret_cast<uint4*>(vs + j * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
        }
        const bool yes = __any(any);
        if (yes) {
            for (int d = lane; d < HD; d += 64) up[d] = down[d] = 0;
            lds_wait();
#pragma unroll 1
            for (int j = 0; j < NI; ++j) {
                const int row = j * RPI + lane / LPR;
                uint4 w = *reinterpret_cast<const uint4*>(vs + j * 1024 + lane * 16);
                note_nonfinite<T>(w, (there >> row) & 1 ? nonfinite_bits<T>(w) : 0u, ((lane % LPR) ^ vswz(row)) * T::EPL, row, up, down);
                *reinterpret_cast<uint4*>(vs + j * 1024 + lane * 16) = w;
            }
        }
        lds_wait();                                              // (a wave's LDS accesses complete in order; nothing of this is in flight behind)
        return yes;
    }

    __device__ static void run(const Launch& L, const Item& it, unsigned char* lds, int* ids, float* ml, void* odd_lds) {
        const M5PagedAttnArgs& p = L.a;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int c = lane & 15, g = lane >> 4;
        const int nrb = (it.rho1 - it.rho0 + 15) >> 4;           // row blocks in use
        const int pos0 = it.rq.len - (it.rq.r1 - it.rq.r0);
        uint4 qf[R][NF];
        int qpos[R];
#pragma unroll
        for (int rb = 0; rb < R; ++rb) {
            const int rho = min(it.rho0 + rb * 16 + c, it.rho1 - 1), tok = rho / L.group;
            qpos[rb] = pos0 + tok;
            const st* q = (const st*)p.q + (int64_t)(it.rq.r0 + tok) * p.q_rs + (int64_t)(it.kvh * L.group + rho % L.group) * p.q_hs;
#pragma unroll
            for (int t = 0; t < NF; ++t) qf[rb][t] = *reinterpret_cast<const uint4*>(q + (4 * t + g) * T::EPL);
        }
        const int pos_min = pos0 + it.rho0 / L.group, pos_max = pos0 + (it.rho1 - 1) / L.group;
        const int lo_max = m5_key_lo(pos_max, p.window);         // the last row's first key
        f4_t o[R][ND];
        Soft sm[R];
#pragma unroll
        for (int rb = 0; rb < R; ++rb) {
            sm[rb] = {-INFINITY, 0.f};
#pragma unroll
            for (int d = 0; d < ND; ++d) o[rb][d] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
        const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)(lds + wave * WAVE_B);
        unsigned char* mine = lds + wave * WAVE_B;
        uint32_t* up = reinterpret_cast<uint32_t*>(odd_lds) + wave * 2 * HD;
        uint32_t* down = up + HD;
        const unsigned char* Kg = (const unsigned char*)p.k_cache + (int64_t)it.kvh * p.k_hs * ES;
        const unsigned char* Vg = (const unsigned char*)p.v_cache + (int64_t)it.kvh * p.v_hs * ES;
        const int off_mask = (1 << L.shift) - 1;
        const int step = NW * KS;                                // keys of one round of the waves
        const int64_t seg = ((int64_t)(MAXP - 1) << L.shift) / step * step;
        const int k_first = it.ka & ~(KS - 1);

        vm_wait<0>();                                            // nothing of an earlier item is in flight
        for (int64_t s0 = k_first; s0 < it.kb; s0 += seg) {
            const int s1 = (int)min((int64_t)it.kb, s0 + seg);
            const int page0 = (int)s0 >> L.shift, np = ((s1 - 1) >> L.shift) - page0 + 1;
            __syncthreads();
            for (int i = tid; i < np; i += NT) ids[i] = m5_block(p.block_table[(int64_t)it.b * p.table_rs + page0 + i], p.n_blocks);
            __syncthreads();
            if (wave >= NW) continue;
            auto fetch = [&](int kb, int stage) {
                const uint32_t to = ring + stage * STAGE_B;
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const int row = j * RPI + lane / LPR, ch = lane % LPR;
                    const int id = key_block(ids, page0, kb + row, it.ka, s1, L.shift);
                    const int64_t blk = max(id, 0), off = id < 0 ? 0 : (kb + row) & off_mask;
                    glds16(Kg + (blk * p.k_bs + off * p.k_ss) * ES + ((ch ^ kswz(row)) << 4), to + j * 1024);
                    glds16(Vg + (blk * p.v_bs + off * p.v_ss) * ES + ((ch ^ vswz(row)) << 4), to + OP_B + j * 1024);
                }
            };
            auto block = [&](int kb, int stage) {
                const unsigned char* ks = mine + stage * STAGE_B;
                const unsigned char* vs = ks + OP_B;
                const uint32_t there = (uint32_t)__ballot(key_block(ids, page0, kb + (lane & (KS - 1)), it.ka, s1, L.shift) >= 0) & (uint32_t)((1ull << KS) - 1);
                const bool whole = there == (uint32_t)((1ull << KS) - 1) && kb + KS - 1 <= pos_min && kb >= lo_max;
                const bool odd = !whole && clean(mine + stage * STAGE_B + OP_B, there, up, down);
                uint32_t vis[R];
                f4_t s[R][SUB];
#pragma unroll
                for (int h = 0; h < SUB; ++h) {
#pragma unroll
                    for (int rb = 0; rb < R; ++rb) s[rb][h] = f4_t{0.f, 0.f, 0.f, 0.f};
                    const int row = h * 16 + c;
#pragma unroll
                    for (int t = 0; t < NF; ++t) {
                        const uint4 k = *reinterpret_cast<const uint4*>(ks + row * RB + (((4 * t + g) ^ kswz(row)) << 4));
#pragma unroll
                        for (int rb = 0; rb < R; ++rb)
                            if (R == 1 || rb < nrb) s[rb][h] = mma16(k, qf[rb][t], s[rb][h], T());
                    }
                }
                uint4 pf[R];
#pragma unroll
                for (int rb = 0; rb < R; ++rb) {
                    if (R > 1 && rb >= nrb) continue;
                    if (!whole) {
                        vis[rb] = (uint32_t)seen(there, kb, m5_key_lo(qpos[rb], p.window), qpos[rb]);
#pragma unroll
                        for (int h = 0; h < SUB; ++h)
#pragma unroll
                            for (int r = 0; r < 4; ++r) s[rb][h][r] = (vis[rb] >> (16 * h + 4 * g + r)) & 1 ? s[rb][h][r] : -INFINITY;
                    }
                    float mx = s[rb][0][0];
#pragma unroll
                    for (int h = 0; h < SUB; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][h][r]);
                    mx = fmaxf(mx, lane_xor16(mx));
                    mx = fmaxf(mx, lane_xor32(mx)) * L.sc2;
                    float use;
                    const float alpha = sm[rb].step(mx, use);
                    float sum = 0.f;
                    st e[T::EPL];
#pragma unroll
                    for (int h = 0; h < SUB; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][h][r], L.sc2, -use));
                            sum += x;
                            e[4 * h + r] = T::from_f32(x);       // 16-bit: p in (0, 1] rounded once for the matrix product, summed in fp32
                        }
                    pf[rb] = *reinterpret_cast<const uint4*>(e);
                    sm[rb].l = sm[rb].l * alpha + sum;
                    if (!__all(alpha == 1.0f))
#pragma unroll
                        for (int d = 0; d < ND; ++d) o[rb][d] *= alpha;
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint4 v;
                    if constexpr (ES == 4) {
                        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = 4 * g + r;
                            w[r] = *reinterpret_cast<const uint32_t*>(vs + row * RB + (((4 * d + (c >> 2)) ^ vswz(row)) << 4) + (c & 3) * 4);
                        }
                    } else {
                        uint2 h2[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int row = 16 * h + 4 * g + (c >> 2);
                            h2[h] = tr_read(vs + row * RB + (((2 * d + ((c >> 1) & 1)) ^ vswz(row)) << 4) + (c & 1) * 8);
                        }
                        v = make_uint4(h2[0].x, h2[0].y, h2[1].x, h2[1].y);
                    }
#pragma unroll
                    for (int rb = 0; rb < R; ++rb)
                        if (R == 1 || rb < nrb) o[rb][d] = mma16(v, pf[rb], o[rb][d], T());
                }
                if (odd)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            asm volatile("" ::: "memory");       // (one feature's notes at a time: read ahead they would cost registers)
                            const uint32_t u = up[16 * d + 4 * g + r], n = down[16 * d + 4 * g + r];
#pragma unroll
                            for (int rb = 0; rb < R; ++rb)
                                if (R == 1 || rb < nrb) o[rb][d][r] += infinite_part(u & vis[rb], n & vis[rb]);
                        }
            };
            int kb = (int)s0 + wave * KS, stage = 0;
            if (kb < s1) fetch(kb, 0);
            for (; kb < s1; kb += step, stage ^= 1) {
                if (kb + step < s1) {
                    lds_wait();                                  // the other stage's reads are done before it is filled again
                    fetch(kb + step, stage ^ 1);
                    vm_wait<2 * NI>();
                } else {
                    vm_wait<0>();
                }
                block(kb, stage);
            }
        }

        // ---- the waves' results meet: row-major fp32 in the rings, chunk-swizzled
        __syncthreads();
        float* om = reinterpret_cast<float*>(mine);
        if (wave < NW) {
#pragma unroll
            for (int rb = 0; rb < R; ++rb) {
                if (R > 1 && rb >= nrb) continue;
                float l = sm[rb].l;
                l += lane_xor16(l);
                l += lane_xor32(l);
                const int row = rb * 16 + c;
                if (g == 0) { ml[(wave * 64 + row) * 2] = sm[rb].m; ml[(wave * 64 + row) * 2 + 1] = l; }
#pragma unroll
                for (int d = 0; d < ND; ++d) *reinterpret_cast<f4_t*>(om + row * HD + (((4 * d + g) ^ (row & 15)) << 2)) = o[rb][d];
            }
        }
        __syncthreads();
        float* slot = it.n_parts > 1 ? L.slots + it.id * L.slot_floats : nullptr;
        const int chunks = (it.rho1 - it.rho0) * (HD / 4);
        for (int i = tid; i < chunks; i += NT) {
            const int row = i / (HD / 4), ch = i % (HD / 4);
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) m = fmaxf(m, ml[(w * 64 + row) * 2]);
            const float use = m == -INFINITY ? 0.f : m;
            f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[(w * 64 + row) * 2] - use);
                l += ml[(w * 64 + row) * 2 + 1] * f;
                sum += *reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(lds + w * WAVE_B) + row * HD + ((ch ^ (row & 15)) << 2)) * f;
            }
            if (slot) {
                *reinterpret_cast<f4_t*>(slot + row * HD + ch * 4) = sum;
                if (ch == 0) { slot[16 * R * HD + 2 * row] = m; slot[16 * R * HD + 2 * row + 1] = l; }
            } else {
                put_row<T, HD>(L, it, row, ch * 4, sum, m, l);
            }
        }
    }
};

// ----------------------------------------------------------------------------------------------------- many rows
template <typename T, int HD>
struct Many {
    using st = typename T::storage;
    static constexpr int RB = HD * 2, KT = 64;                   // bytes of a row, keys of a tile
    static constexpr int LPR = RB / 16, RPI = 64 / LPR, NJ = KT / RPI / NWAVE;
    static constexpr int OP_B = KT * RB, STAGE_B = 2 * OP_B, LDS_B = 2 * STAGE_B;
    static constexpr int NF = HD / 16, ND = HD / 32;

    __device__ static inline int kswz(int row) { return RB == 128 ? (row >> 1) & 7 : row & 15; }
    __device__ static inline int vswz(int row) { return RB == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }

    // As Few::clean, by the whole workgroup (every wave calls it; the barriers inside also order it before the waves' reads).
    __device__ static bool clean(unsigned char* vs, unsigned long long there, unsigned long long* up, unsigned long long* down) {
        const int tid = threadIdx.x;
        constexpr int N = OP_B / (NT * 16);
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = j * NT + tid, row = at / LPR;
            uint4* w = reinterpret_cast<uint4*>(vs) + at;
            if ((there >> row) & 1) any |= nonfinite_bits<T>(*w);
            else *w = make_uint4(0, 0, 0, 0);
        }
        const bool yes = __syncthreads_or(any);
        if (yes) {
            for (int d = tid; d < HD; d += NT) up[d] = down[d] = 0;
            __syncthreads();
#pragma unroll 1
            for (int j = 0; j < N; ++j) {
                const int at = j * NT + tid, row = at / LPR;
                uint4 w = reinterpret_cast<const uint4*>(vs)[at];
                note_nonfinite<T>(w, (there >> row) & 1 ? nonfinite_bits<T>(w) : 0u, ((at % LPR) ^ vswz(row)) * 8, row, up, down);
                reinterpret_cast<uint4*>(vs)[at] = w;
            }
            __syncthreads();
        }
        return yes;
    }

    __device__ static void run(const Launch& L, const Item& it, unsigned char* lds, int* ids, void* odd_lds) {
        const M5PagedAttnArgs& p = L.a;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int c = lane & 31, hh = lane >> 5;
        const int w0 = it.rho0 + wave * 32, w1 = min(w0 + 32, it.rho1);      // this wave's rows (none: it only fetches)
        const int pos0 = it.rq.len - (it.rq.r1 - it.rq.r0);
        const int rho = min(w0 + c, it.rho1 - 1), tok = rho / L.group, qpos = pos0 + tok;
        const int pos_min = pos0 + w0 / L.group, pos_max = pos0 + (w1 - 1) / L.group;
        const int lo_min = m5_key_lo(pos_min, p.window), lo_max = m5_key_lo(pos_max, p.window), lo = m5_key_lo(qpos, p.window);
        uint4 qf[NF];
        {
            const st* q = (const st*)p.q + (int64_t)(it.rq.r0 + tok) * p.q_rs + (int64_t)(it.kvh * L.group + rho % L.group) * p.q_hs;
#pragma unroll
            for (int t = 0; t < NF; ++t) qf[t] = *reinterpret_cast<const uint4*>(q + 16 * t + 8 * hh);
        }
        f16_t o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
        Soft sm = {-INFINITY, 0.f};
        const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
        unsigned long long* up = reinterpret_cast<unsigned long long*>(odd_lds);
        unsigned long long* down = up + HD;
        const int first_pos = pos0 + it.rho0 / L.group, last_lo = m5_key_lo(pos0 + (it.rho1 - 1) / L.group, p.window);      // of all rows here
        const unsigned char* Kg = (const unsigned char*)p.k_cache + (int64_t)it.kvh * p.k_hs * 2;
        const unsigned char* Vg = (const unsigned char*)p.v_cache + (int64_t)it.kvh * p.v_hs * 2;
        const int off_mask = (1 << L.shift) - 1;
        const int64_t seg = ((int64_t)(MAXP - 1) << L.shift) / KT * KT;

        vm_wait<0>();
        for (int64_t s0 = it.ka & ~(KT - 1); s0 < it.kb; s0 += seg) {
            const int s1 = (int)min((int64_t)it.kb, s0 + seg);
            const int page0 = (int)s0 >> L.shift, np = ((s1 - 1) >> L.shift) - page0 + 1;
            __syncthreads();
            for (int i = tid; i < np; i += NT) ids[i] = m5_block(p.block_table[(int64_t)it.b * p.table_rs + page0 + i], p.n_blocks);
            __syncthreads();
            auto fetch = [&](int kb, int stage) {
                const uint32_t to = ring + stage * STAGE_B + wave * NJ * 1024;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int row = (wave * NJ + j) * RPI + lane / LPR, ch = lane % LPR;
                    const int id = key_block(ids, page0, kb + row, it.ka, s1, L.shift);
                    const int64_t blk = max(id, 0), off = id < 0 ? 0 : (kb + row) & off_mask;
                    glds16(Kg + (blk * p.k_bs + off * p.k_ss) * 2 + ((ch ^ kswz(row)) << 4), to + j * 1024);
                    glds16(Vg + (blk * p.v_bs + off * p.v_ss) * 2 + ((ch ^ vswz(row)) << 4), to + OP_B + j * 1024);
                }
            };
            auto tile = [&](int kb, int stage, unsigned long long there, bool odd) {
                const unsigned char* ks = lds + stage * STAGE_B;
                const unsigned char* vs = ks + OP_B;
                const bool whole = there == ~0ull && kb + KT - 1 <= pos_min && kb >= lo_max;
                unsigned long long vis = 0;
                f16_t s[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[h][r] = 0.f;
                    const int row = 32 * h + c;
#pragma unroll
                    for (int t = 0; t < NF; ++t)
                        s[h] = mma32(*reinterpret_cast<const uint4*>(ks + row * RB + (((2 * t + hh) ^ kswz(row)) << 4)), qf[t], s[h], T());
                }
                if (!whole) {
                    vis = seen(there, kb, lo, qpos);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t half = (uint32_t)(vis >> (32 * h + 4 * hh));
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[h][r] = (half >> (8 * (r >> 2) + (r & 3))) & 1 ? s[h][r] : -INFINITY;
                    }
                }
                float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(fmaxf(mx, s[0][r]), s[1][r]);
                mx = fmaxf(mx, lane_xor32(mx)) * L.sc2;
                float use, sum = 0.f;
                const float alpha = sm.step(mx, use);
                uint4 pf[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        st e[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][8 * m + j], L.sc2, -use));
                            sum += x;
                            e[j] = T::from_f32(x);
                        }
                        pf[h][m] = *reinterpret_cast<const uint4*>(e);
                    }
                sm.l = sm.l * alpha + sum;
                if (!__all(alpha == 1.0f))
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[d] *= alpha;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int d = 0; d < ND; ++d) {
                            const int row = 32 * h + 16 * m + 4 * hh + ((lane & 15) >> 2), ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
                            const uint2 v0 = tr_read(vs + row * RB + ((ch ^ vswz(row)) << 4) + (lane & 1) * 8);
                            const uint2 v1 = tr_read(vs + (row + 8) * RB + ((ch ^ vswz(row + 8)) << 4) + (lane & 1) * 8);
                            const uint4 v = make_uint4(v0.x, v0.y, v1.x, v1.y);
                            o[d] = mma32(v, pf[h][m], o[d], T());
                        }
                if (odd)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const int at = 32 * d + 8 * (r >> 2) + 4 * hh + (r & 3);
                            asm volatile("" ::: "memory");       // (one feature's notes at a time: read ahead they would cost registers)
                            o[d][r] += infinite_part(up[at] & vis, down[at] & vis);
                        }
            };
            int stage = 0;
            fetch((int)s0, 0);
            for (int kb = (int)s0; kb < s1; kb += KT, stage ^= 1) {
                vm_wait<0>();
                __syncthreads();                                 // the tile is there for all waves, and all are done with the other stage
                if (kb + KT < s1) fetch(kb + KT, stage ^ 1);
                const unsigned long long there = __ballot(key_block(ids, page0, kb + lane, it.ka, s1, L.shift) >= 0);
                const bool odd = !(there == ~0ull && kb + KT - 1 <= first_pos && kb >= last_lo) && clean(lds + stage * STAGE_B + OP_B, there, up, down);
                if (w0 < w1 && kb <= pos_max && kb + KT > lo_min) tile(kb, stage, there, odd);
            }
        }
        if (w0 >= w1) return;
        float l = sm.l + lane_xor32(sm.l);
        if (w0 + c >= w1) return;
        const int row = wave * 32 + c;
        float* slot = it.n_parts > 1 ? L.slots + it.id * L.slot_floats : nullptr;
        if (slot && hh == 0) { slot[128 * HD + 2 * row] = sm.m; slot[128 * HD + 2 * row + 1] = l; }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f4_t v = {o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
                const int at = 32 * d + 8 * q + 4 * hh;
                if (slot) *reinterpret_cast<f4_t*>(slot + row * HD + at) = v;
                else put_row<T, HD>(L, it, row, at, v, sm.m, l);
            }
    }
};

// The last workgroup of a tile joins its partial results in chunk order.
template <typename T, int HD, int TR>
__device__ void join_parts(const Launch& L, const Item& it, int* sh_last) {
    __syncthreads();
    if (threadIdx.x == 0) {
        int* ticket = L.tickets + it.first_id;
        const int n = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        *sh_last = n == it.n_parts - 1;
        if (n == it.n_parts - 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);       // ready for the next call
    }
    __syncthreads();
    if (!*sh_last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    const float* first = L.slots + it.first_id * L.slot_floats;
    const int64_t stride = L.a.n_kv_heads * L.slot_floats;
    Item whole = it;
    whole.n_parts = 1;
    const int chunks = (it.rho1 - it.rho0) * (HD / 4);
    for (int i = threadIdx.x; i < chunks; i += NT) {
        const int row = i / (HD / 4), ch = i % (HD / 4);
        float m = -INFINITY, l = 0.f;
        for (int k = 0; k < it.n_parts; ++k) m = fmaxf(m, first[k * stride + TR * HD + 2 * row]);
        const float use = m == -INFINITY ? 0.f : m;
        f4_t sum = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < it.n_parts; ++k) {
            const float* s = first + k * stride;
            const float f = __builtin_amdgcn_exp2f(s[TR * HD + 2 * row] - use);
            l += s[TR * HD + 2 * row + 1] * f;
            sum += *reinterpret_cast<const f4_t*>(s + row * HD + ch * 4) * f;
        }
        put_row<T, HD>(L, whole, row, ch * 4, sum, m, l);
    }
}

__device__ inline int64_t block_sum64(int64_t v, int64_t* red) {             // red: NWAVE words
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor((long long)v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    int64_t t = 0;
    for (int w = 0; w < NWAVE; ++w) t += red[w];
    return t;
}

// A request's share of the work: tiles of `tr` rows and the keys that any of its rows sees, from k0 (a multiple of 64) on.
struct Share { int rows, tr, tiles, k0, keys; };
template <int TR_FEW, int TR_MANY>
__device__ inline Share share_of(const Launch& L, const M5Request& rq) {
    Share s;
    s.rows = (rq.r1 - rq.r0) * L.group;
    s.tr = TR_MANY && s.rows > TR_FEW ? TR_MANY : TR_FEW;
    s.tiles = (s.rows + s.tr - 1) / s.tr;
    s.k0 = m5_key_lo(rq.len - (rq.r1 - rq.r0), L.a.window) & ~63;
    s.keys = max(rq.len - s.k0, 0);
    return s;
}

// R: row blocks of the few-row tiles; NW: waves that work on them; MANY: requests of more rows get 128-row tiles.
template <typename T, int HD, int R, int NW, bool MANY>
struct Shape {
    using F = Few<T, HD, R, NW>;
    static constexpr int TR = 16 * R, TRM = MANY ? 128 : 0, SLOT_ROWS = MANY ? 128 : TR;
    static constexpr int RING_B = MANY ? (F::LDS_B > 4 * 64 * HD * 2 ? F::LDS_B : 4 * 64 * HD * 2) : F::LDS_B;
    static int lds_bytes(int n_seq) { return RING_B + IDS_B + ML_B + odd_bytes(HD) + (n_seq + 1) * 4; }
};

template <typename T, int HD, int R, int NW, bool MANY>
__global__ __launch_bounds__(NT, MANY ? 2 : 1) void paged_attn_kernel(Launch L) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    using S = Shape<T, HD, R, NW, MANY>;
    int* ids = reinterpret_cast<int*>(lds + S::RING_B);
    float* ml = reinterpret_cast<float*>(lds + S::RING_B + IDS_B);
    int* sh = reinterpret_cast<int*>(lds + S::RING_B + IDS_B + NWAVE * 64 * 2 * 4);
    unsigned char* odd = lds + S::RING_B + IDS_B + ML_B;
    int* pre = reinterpret_cast<int*>(odd + odd_bytes(HD));
    int64_t* red = reinterpret_cast<int64_t*>(ml);
    const M5PagedAttnArgs& p = L.a;
    const int B = p.n_seq, tid = threadIdx.x;
    const int64_t cap = (int64_t)p.table_width << L.shift;

    // ---- items: how long a chunk of keys is, and every request's first item
    const int per = (B + NT - 1) / NT, b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int64_t units = 0, tiles = 0;
    for (int b = b0; b < b1; ++b) {
        const Share s = share_of<S::TR, S::TRM>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        units += (int64_t)s.tiles * ((s.keys + 63) >> 6);
        tiles += s.tiles;
    }
    units = block_sum64(units, red) * p.n_kv_heads;
    tiles = block_sum64(tiles, red) * p.n_kv_heads;
    // items <= units / (C / 64) + tiles, and a split item needs a slot
    int64_t C = INT_MAX;
    if (L.n_slots > tiles) {
        C = max((units + L.target - 1) / L.target, (units + (L.n_slots - tiles) - 1) / (L.n_slots - tiles));
        C = min(max(C, (int64_t)4) * 64, (int64_t)INT_MAX);
    }
    auto items_of = [&](const Share& s) { return max((int)((s.keys + C - 1) / C), 1); };
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
        const Share s = share_of<S::TR, S::TRM>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        mine += s.tiles * items_of(s) * p.n_kv_heads;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        if ((tid & 63) >= d) incl += o;
    }
    __syncthreads();
    if ((tid & 63) == 63) sh[tid >> 6] = incl;
    __syncthreads();
    int base = incl - mine, total = 0;
    for (int w = 0; w < NWAVE; ++w) {
        if (w < tid >> 6) base += sh[w];
        total += sh[w];
    }
    for (int b = b0; b < b1; ++b) {
        pre[b] = base;
        const Share s = share_of<S::TR, S::TRM>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        base += s.tiles * items_of(s) * p.n_kv_heads;
    }
    if (tid == NT - 1) pre[B] = total;
    __syncthreads();

    for (int id = blockIdx.x; id < total; id += gridDim.x) {
        Item it;
        it.b = m5_upper(pre, B, id);
        it.rq = m5_request(p.q_start[it.b], p.q_start[it.b + 1], p.seq_len[it.b], p.n_rows, cap);
        const Share s = share_of<S::TR, S::TRM>(L, it.rq);
        const int nc = items_of(s), at = id - pre[it.b];
        it.kvh = at % p.n_kv_heads;
        const int chunk = at / p.n_kv_heads % nc, tile = s.tiles - 1 - at / p.n_kv_heads / nc;      // the longest rows first
        it.rows = s.rows;
        it.rho0 = tile * s.tr;
        it.rho1 = min(it.rho0 + s.tr, s.rows);
        it.id = id;
        const int pos0 = it.rq.len - (it.rq.r1 - it.rq.r0);
        const int lo = m5_key_lo(pos0 + it.rho0 / L.group, p.window), hi = m5_key_hi(pos0 + (it.rho1 - 1) / L.group, it.rq.len);
        const int c0 = hi > lo ? (int)((lo - s.k0) / C) : 0, c1 = hi > lo ? (int)((hi - 1 - s.k0) / C) : 0;
        if (chunk < c0 || chunk > c1) continue;                  // no row of this tile sees a key of this chunk
        it.n_parts = c1 - c0 + 1;
        it.first_id = id - (chunk - c0) * p.n_kv_heads;
        it.ka = (int)max((int64_t)lo, s.k0 + chunk * C);
        it.kb = (int)min((int64_t)hi, s.k0 + (chunk + 1) * C);
        if constexpr (MANY) {
            if (s.tr == 128) {
                Many<T, HD>::run(L, it, lds, ids, odd);
                if (it.n_parts > 1) join_parts<T, HD, 128>(L, it, sh);
                __syncthreads();
                continue;
            }
        }
        S::F::run(L, it, lds, ids, ml, odd);
        if (it.n_parts > 1) join_parts<T, HD, S::TR>(L, it, sh);
        __syncthreads();
    }
}

constexpr int MAX_SLOTS = 1024;

// The tiling for these shapes: rows of a few-row tile, or 0 for the kernel with 128-row tiles.
int tiling(int dtype, const M5PagedAttnArgs& a) {
    const int64_t rows = (int64_t)min(max(a.max_new, 1), max(a.n_rows, 1)) * (a.n_heads / a.n_kv_heads);
    if (rows <= 16) return 16;
    if (rows <= 32 || (dtype == M5_F32 && a.head_dim == 128)) return 32;             // (64 fp32 rows of 128 features: too many registers)
    return rows <= 64 || dtype == M5_F32 ? 64 : 0;
}

template <typename T, int HD, int R, int NW, bool MANY>
int launch_as(Launch& L, int cus, hipStream_t s) {
    using S = Shape<T, HD, R, NW, MANY>;
    const int lds = S::lds_bytes(L.a.n_seq);
    if (hipFuncSetAttribute((const void*)paged_attn_kernel<T, HD, R, NW, MANY>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return M5_ERR_LAUNCH;
    L.slot_floats = (int64_t)S::SLOT_ROWS * (HD + 2);
    L.n_slots = L.a.workspace ? (int)min((int64_t)MAX_SLOTS, L.a.workspace_bytes / (L.slot_floats * 4 + 4)) & ~3 : 0;     // (the slots behind the tickets stay 16-byte aligned)
    L.tickets = (int*)L.a.workspace;
    L.slots = (float*)((char*)L.a.workspace + (int64_t)L.n_slots * 4);
    L.target = 2 * cus * min(160 * 1024 / lds, 2);
    const int64_t tiles = ((int64_t)L.a.n_rows * L.group / S::TR + L.a.n_seq) * L.a.n_kv_heads;      // upper bound
    const int64_t grid = L.n_slots ? max((int64_t)L.target, tiles) : tiles;
    hipLaunchKernelGGL((paged_attn_kernel<T, HD, R, NW, MANY>), dim3((unsigned)min(grid, (int64_t)1 << 20)), dim3(NT), lds, s, L);
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
    if ((a->head_dim != 64 && a->head_dim != 128) || a->block_size > 1024 || a->n_seq > MAX_SEQ || ((int64_t)a->table_width << shift) > (1 << 30) ||
        ((int64_t)a->n_blocks << shift) > INT_MAX || (int64_t)a->n_rows * a->n_heads > INT_MAX / 4)
        return M5_ERR_UNSUPPORTED;
    const int epl = dtype == M5_F32 ? 4 : 8;
    if (!aligned(a->q, a->q_rs, a->q_hs, 0, epl) || !aligned(a->out, a->o_rs, a->o_hs, 0, epl) || !aligned(a->k_cache, a->k_bs, a->k_hs, a->k_ss, epl) ||
        !aligned(a->v_cache, a->v_bs, a->v_hs, a->v_ss, epl) || ((uintptr_t)a->workspace & 15))
        return M5_ERR_UNSUPPORTED;
    return M5_OK;
}

template <typename T>
int launch(const M5PagedAttnArgs& a, int shift, hipStream_t s) {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return M5_ERR_LAUNCH;
    Launch L;
    L.a = a;
    L.shift = shift;
    L.group = a.n_heads / a.n_kv_heads;
    L.sc2 = a.scale * 1.4426950408889634f;
    const int tr = tiling(T::id, a);
    if (a.head_dim == 64) {
        if constexpr (T::id != M5_F32)
            if (tr == 0) return launch_as<T, 64, 2, 4, true>(L, cus, s);
        return tr == 16 ? launch_as<T, 64, 1, 4, false>(L, cus, s) : tr == 32 ? launch_as<T, 64, 2, 4, false>(L, cus, s) : launch_as<T, 64, 4, 4, false>(L, cus, s);
    }
    if constexpr (T::id != M5_F32) {
        if (tr == 0) return launch_as<T, 128, 2, 2, true>(L, cus, s);
        if (tr == 64) return launch_as<T, 128, 4, 4, false>(L, cus, s);
    }
    return tr == 16 ? launch_as<T, 128, 1, 4, false>(L, cus, s) : launch_as<T, 128, 2, 4, false>(L, cus, s);
}

}  // namespace

extern "C" int m5_paged_attention_workspace(int dtype, const M5PagedAttnArgs* a, int64_t* bytes) {
    const int rc = check(dtype, a);
    if (rc != M5_OK) return rc;
    if (!bytes) return M5_ERR_ARG;
    const int tr = tiling(dtype, *a);
    *bytes = (int64_t)MAX_SLOTS * ((int64_t)(tr ? tr : 128) * (a->head_dim + 2) * 4 + 4);
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
