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
// Masked places.  Keys outside a tile's range or on a bad page are read from a valid address and their values zeroed in the registers;
// a non-finite value that some rows of a tile see and others do not is taken out of the product and added only to the rows that see
// it (0 * inf would be NaN).
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

struct Launch {
    M5PagedAttnArgs a;
    int shift, group;
    int target;                                  // items wanted: places on the chip
    int n_slots;                                 // partial results the workspace holds, 0 = keys are not split
    float* slots; int* tickets;
    float sc2;                                   // scale * log2(e)
};

struct Item {
    M5Request rq;
    int b, kvh, rows, rho0, rho1;                // rows of the request's kv head, [rho0, rho1) of them here
    int ka, kb;                                  // keys of this item
    int id, first_id, n_parts, part;             // partial results of this tile: slots first_id + p * n_kv_heads
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

// element e of a fragment is kept iff bit e is set
template <typename T>
__device__ inline void keep_bits(uint4& v, uint32_t bits) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (T::EPL == 4) w[i] = (bits >> i) & 1 ? w[i] : 0u;
        else w[i] &= ((bits >> (2 * i)) & 1 ? 0xffffu : 0u) | ((bits >> (2 * i + 1)) & 1 ? 0xffff0000u : 0u);
    }
}
// bit e set: element e is infinite or NaN
template <typename T>
__device__ inline uint32_t nonfinite_bits(const uint4& v) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
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
// ones in the elements of `bits` (indicator operand of a product)
template <typename T>
__device__ inline uint4 ones(uint32_t bits) {
    const uint32_t one = T::id == M5_F16 ? 0x3c003c00u : (T::id == M5_BF16 ? 0x3f803f80u : 0x3f800000u);
    uint4 v = make_uint4(one, one, one, one);
    keep_bits<T>(v, bits);
    return v;
}
// of the non-finite elements `bits` of v: those that add +inf (or NaN) / -inf (or NaN)
template <typename T>
__device__ inline void infinite_signs(const uint4& v, uint32_t bits, uint32_t& up, uint32_t& down) {
    typename T::storage e[T::EPL];
    *reinterpret_cast<uint4*>(e) = v;
    up = down = 0;
#pragma unroll
    for (int i = 0; i < T::EPL; ++i) {
        const float f = T::to_f32(e[i]);
        if ((bits >> i) & 1) {
            if (!(f < 0.f)) up |= 1u << i;
            if (!(f > 0.f)) down |= 1u << i;
        }
    }
}
__device__ inline float infinite_part(float up, float down) { return (up > 0.f ? INFINITY : 0.f) - (down > 0.f ? INFINITY : 0.f); }

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

    __device__ static void run(const Launch& L, const Item& it, unsigned char* lds, int* ids, float* ml) {
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
                uint32_t sees[R];                                // this lane's 4 SUB keys: element 4 h + r = key 16 h + 4 g + r
                uint4 pf[R];
#pragma unroll
                for (int rb = 0; rb < R; ++rb) {
                    if (R > 1 && rb >= nrb) continue;
                    if (!whole) {
                        sees[rb] = 0;
                        const int lo = m5_key_lo(qpos[rb], p.window);
#pragma unroll
                        for (int h = 0; h < SUB; ++h)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int at = 16 * h + 4 * g + r, key = kb + at;
                                const bool vis = ((there >> at) & 1) && key <= qpos[rb] && key >= lo;
                                sees[rb] |= vis ? 1u << (4 * h + r) : 0u;
                                s[rb][h][r] = vis ? s[rb][h][r] : -INFINITY;
                            }
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
                uint32_t keep = 0;                               // this lane's elements that are keys of the item at all
                if (!whole)
#pragma unroll
                    for (int h = 0; h < SUB; ++h) keep |= ((there >> (16 * h + 4 * g)) & 15u) << (4 * h);
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
                    uint32_t odd = 0;
                    if (!whole) {
                        keep_bits<T>(v, keep);
                        odd = nonfinite_bits<T>(v);
                    }
                    if (!whole && __any(odd)) {
                        uint32_t up, down;
                        infinite_signs<T>(v, odd, up, down);
                        keep_bits<T>(v, ~odd);
                        const uint4 vu = ones<T>(up), vd = ones<T>(down);
#pragma unroll
                        for (int rb = 0; rb < R; ++rb) {
                            if (R > 1 && rb >= nrb) continue;
                            const uint4 who = ones<T>(sees[rb]);
                            const f4_t zero = {0.f, 0.f, 0.f, 0.f};
                            const f4_t nu = mma16(vu, who, zero, T()), nd = mma16(vd, who, zero, T());
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[rb][d][r] += infinite_part(nu[r], nd[r]);
                        }
                    }
#pragma unroll
                    for (int rb = 0; rb < R; ++rb)
                        if (R == 1 || rb < nrb) o[rb][d] = mma16(v, pf[rb], o[rb][d], T());
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
        float* slot = it.n_parts > 1 ? L.slots + (int64_t)it.id * slot_floats(16 * R, HD) : nullptr;
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
    __device__ static constexpr int64_t slot_floats(int rows, int hd) { return (int64_t)rows * (hd + 2); }
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
    constexpr int64_t SF = (int64_t)TR * (HD + 2);
    const float* first = L.slots + it.first_id * SF;
    const int64_t stride = L.a.n_kv_heads * SF;
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

template <typename T, int HD, int R>
__global__ __launch_bounds__(NT, 1) void paged_attn_few_kernel(Launch L) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    using F = Few<T, HD, R, NWAVE>;
    int* ids = reinterpret_cast<int*>(lds + F::LDS_B);
    float* ml = reinterpret_cast<float*>(lds + F::LDS_B + IDS_B);
    int* sh = reinterpret_cast<int*>(lds + F::LDS_B + IDS_B + NWAVE * 64 * 2 * 4);
    int* pre = reinterpret_cast<int*>(lds + F::LDS_B + IDS_B + ML_B);
    int64_t* red = reinterpret_cast<int64_t*>(ml);
    const M5PagedAttnArgs& p = L.a;
    const int B = p.n_seq, tid = threadIdx.x;
    const int64_t cap = (int64_t)p.table_width << L.shift;
    constexpr int TR = 16 * R;

    // ---- items: how long a chunk of keys is, and every request's first item
    const int per = (B + NT - 1) / NT, b0 = min(tid * per, B), b1 = min(b0 + per, B);
    int64_t units = 0, tiles = 0;
    for (int b = b0; b < b1; ++b) {
        const Share s = share_of<TR, 0>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        units += (int64_t)s.tiles * ((s.keys + 63) >> 6);
        tiles += s.tiles;
    }
    units = block_sum64(units, red) * p.n_kv_heads;
    tiles = block_sum64(tiles, red) * p.n_kv_heads;
    // items <= units / C + tiles, and a split item needs a slot
    int64_t C = INT_MAX;
    if (L.n_slots > tiles) {
        C = max((units + L.target - 1) / L.target, (units + (L.n_slots - tiles) - 1) / (L.n_slots - tiles));
        C = min(max(C, (int64_t)4) * 64, (int64_t)INT_MAX);
    }
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
        const Share s = share_of<TR, 0>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        mine += s.tiles * max((int)((s.keys + C - 1) / C), 1) * p.n_kv_heads;
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
        const Share s = share_of<TR, 0>(L, m5_request(p.q_start[b], p.q_start[b + 1], p.seq_len[b], p.n_rows, cap));
        base += s.tiles * max((int)((s.keys + C - 1) / C), 1) * p.n_kv_heads;
    }
    if (tid == NT - 1) pre[B] = total;
    __syncthreads();

    for (int id = blockIdx.x; id < total; id += gridDim.x) {
        Item it;
        it.b = m5_upper(pre, B, id);
        it.rq = m5_request(p.q_start[it.b], p.q_start[it.b + 1], p.seq_len[it.b], p.n_rows, cap);
        const Share s = share_of<TR, 0>(L, it.rq);
        const int nc = max((int)((s.keys + C - 1) / C), 1), at = id - pre[it.b];
        it.kvh = at % p.n_kv_heads;
        const int chunk = at / p.n_kv_heads % nc, tile = s.tiles - 1 - at / p.n_kv_heads / nc;      // the longest rows first
        it.rows = s.rows;
        it.rho0 = tile * TR;
        it.rho1 = min(it.rho0 + TR, s.rows);
        it.id = id;
        const int pos0 = it.rq.len - (it.rq.r1 - it.rq.r0);
        const int lo = m5_key_lo(pos0 + it.rho0 / L.group, p.window), hi = m5_key_hi(pos0 + (it.rho1 - 1) / L.group, it.rq.len);
        const int c0 = hi > lo ? (int)((lo - s.k0) / C) : 0, c1 = hi > lo ? (int)((hi - 1 - s.k0) / C) : 0;
        if (chunk < c0 || chunk > c1) continue;                  // no row of this tile sees a key of this chunk
        it.n_parts = c1 - c0 + 1;
        it.part = chunk - c0;
        it.first_id = id - it.part * p.n_kv_heads;
        it.ka = (int)max((int64_t)lo, s.k0 + chunk * C);
        it.kb = (int)min((int64_t)hi, s.k0 + (chunk + 1) * C);
        F::run(L, it, lds, ids, ml);
        if (it.n_parts > 1) join_parts<T, HD, TR>(L, it, sh);
        __syncthreads();
    }
}

template <typename T, int HD, int R>
int launch_few(Launch& L, int64_t tiles, int cus, hipStream_t s) {
    using F = Few<T, HD, R, NWAVE>;
    const int lds = F::LDS_B + IDS_B + ML_B + (L.a.n_seq + 1) * 4;
    const void* fn = (const void*)paged_attn_few_kernel<T, HD, R>;
    if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return M5_ERR_LAUNCH;
    const int places = cus * (160 * 1024 / lds);
    L.target = 2 * places;
    const int64_t grid = L.n_slots ? max((int64_t)L.target, tiles) : tiles;
    hipLaunchKernelGGL((paged_attn_few_kernel<T, HD, R>), dim3((unsigned)min(grid, (int64_t)1 << 20)), dim3(NT), lds, s, L);
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

constexpr int MAX_SLOTS = 1024;
int tile_rows(int dtype, const M5PagedAttnArgs& a) {         // rows of a tile for these shapes
    const int64_t rows = (int64_t)min(max(a.max_new, 1), max(a.n_rows, 1)) * (a.n_heads / a.n_kv_heads);
    return rows <= 16 ? 16 : (rows <= 32 || (dtype == M5_F32 && a.head_dim == 128) ? 32 : 64);      // (64 fp32 rows of 128 features: too many registers)
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
    const int tr = tile_rows(T::id, a);
    const int64_t slot_b = (int64_t)tr * (a.head_dim + 2) * 4;
    L.n_slots = a.workspace ? (int)min((int64_t)MAX_SLOTS, a.workspace_bytes / (slot_b + 4)) : 0;
    L.n_slots &= ~3;                                         // the slots behind the tickets stay 16-byte aligned
    L.tickets = (int*)a.workspace;
    L.slots = (float*)((char*)a.workspace + (int64_t)L.n_slots * 4);
    const int64_t tiles = ((int64_t)a.n_rows * L.group / tr + a.n_seq) * a.n_kv_heads;      // upper bound
    if (a.head_dim == 64) return tr == 16 ? launch_few<T, 64, 1>(L, tiles, cus, s) : tr == 32 ? launch_few<T, 64, 2>(L, tiles, cus, s) : launch_few<T, 64, 4>(L, tiles, cus, s);
    if constexpr (T::id != M5_F32)
        if (tr == 64) return launch_few<T, 128, 4>(L, tiles, cus, s);
    return tr == 16 ? launch_few<T, 128, 1>(L, tiles, cus, s) : launch_few<T, 128, 2>(L, tiles, cus, s);
}

}  // namespace

extern "C" int m5_paged_attention_workspace(int dtype, const M5PagedAttnArgs* a, int64_t* bytes) {
    const int rc = check(dtype, a);
    if (rc != M5_OK) return rc;
    if (!bytes) return M5_ERR_ARG;
    *bytes = (int64_t)MAX_SLOTS * ((int64_t)tile_rows(dtype, *a) * (a->head_dim + 2) * 4 + 4);
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
