// Attention of new tokens (single ones, drafts, prompt chunks) over a paged KV cache (m5_paged_attention, include/mars5_paged.h).
//
//   o[r][h] = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale log2(e) q[r][h] . k_j - m),   m = running maximum
//
// Rows.  The query heads of one kv head and the new tokens of one request are packed into rows rho = token * group + head, so every
// key and value is read once for all of them.  A tile is 16 or 32 rows ("few": single tokens, drafts; all types) or 128 ("many": prompt
// chunks; 16-bit).  Both products are computed transposed, S^T = K Q^T and O^T = V^T P^T: the row is the matrix column, i.e. a lane
// owns one row, the softmax state is lane-local, and P^T goes into the second product straight from the registers of the first.
//   few   16x16 matrix instructions.  The waves of a workgroup take different keys (16 at a time; 32 of 64 features in 16 bits) of the
//         same rows, each with a private ring of two stages in LDS, and meet once at the end: no barrier in the key loop.  Bound by memory:
//         3 requests of 60 to 120 thousand keys 160 us, 5.5 TB/s; 64 requests with drafts over 1 to 16 thousand keys 309 us, 5.0 TB/s.
//   many  32x32 matrix instructions.  Each wave owns 32 rows; the waves share 64-key tiles, one barrier per tile.  Bound by the issue of
//         matrix and vector instructions together (46 % of the cycles matrix, the softmax most of the rest): 2 chunks of 4096 tokens with
//         contexts of 9 to 12 thousand keys 1580 to 1790 us, 880 to 1000 TFLOP/s.
// K and V rows go from memory into LDS by DMA (global_load_lds, 16 bytes per lane; the page lookup is in the lane's address).  16-byte
// chunks of a row are stored XOR-swizzled so that the fragment reads spread over all banks (no conflicts counted): K fragments are ds_read_b128, V fragments
// (keys along the register, features along the lanes) are ds_read_b64_tr_b16, which transposes 4 x 16 blocks on the way, so the
// cache needs no transposed copy of V.
//
// Work.  Lengths are device data: every workgroup scans the requests (up to 64 in a wave's lanes, without a barrier) and deals itself items (request, tile,
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
#include <initializer_list>
#include <type_traits>

typedef __attribute__((ext_vector_type(8))) _Float16 h8_t;
typedef __attribute__((ext_vector_type(8))) __bf16 b8_t;
typedef __attribute__((ext_vector_type(4))) float f4_t;
typedef __attribute__((ext_vector_type(16))) float f16_t;
typedef __attribute__((ext_vector_type(4))) short s4_t;

namespace {

constexpr int SCHED_MFMA = 0x8, SCHED_DS = 0x100;        // sched_group_barrier: matrix instructions, LDS reads
constexpr int NWAVE = 4, NT = NWAVE * 64;
constexpr int MAXP = 512;                        // block ids of one key segment held in LDS
constexpr int MAX_ITEMS = 4096;                  // items of a call whose keys are split
constexpr int64_t MAX_WORKSPACE = 64 << 20, MIN_ITEM_BYTES = 16 * (64 + 2) * 4 + 4;
constexpr int MAX_SEQ = 4096;                    // prefix sums of items (4 bytes) and of rows of partial results (2 bytes: in 16s) in LDS: 24 KB
static_assert(MAX_WORKSPACE / (16 * (64 + 2) * 4) < 65536, "rows of partial results in 16s");
constexpr int IDS_B = MAXP * 4, ML_B = NWAVE * 32 * 2 * 4 + 64;
constexpr int odd_bytes(int hd) { return NWAVE * 2 * hd * 4; }   // notes of non-finite values: per wave and feature 2 x 32 keys, or 2 x 64 shared

// x / d for 0 <= x < 2^29: (x m) >> s with m = ceil(2^s / d), s = 29 + ceil(log2 d)
struct Div {
    uint32_t d, m, s;
    void set(int by) {
        d = (uint32_t)by;
        s = 29;
        while ((1u << (s - 29)) < d) ++s;
        m = (uint32_t)((((uint64_t)1 << s) + d - 1) / d);
    }
    __device__ inline int div(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> s); }
};

struct Launch {
    M5PagedAttnArgs a;
    int shift;
    Div group, kv;                               // query heads of a kv head; kv heads
    int places;                                  // workgroups that the chip holds at a time
    float max_tiles;                             // tiles that ascending row offsets can make
    int n_tickets, slot_rows;                    // items and rows of partial results that the workspace holds (0: keys are not split)
    float* slots; int* tickets;
    float sc2;                                   // scale * log2(e)
    uint32_t k_bs16, k_ss16, v_bs16, v_ss16;     // block and slot strides in 16-byte units
};

struct Item {
    M5Request rq;
    int b, kvh, rho0, rho1;                      // packed rows of the request and kv head
    int ka, kb;                                  // keys of this item
    int n_parts;                                 // partial results of this tile; more than one: this item's goes to `slot`, the tile's
    float* slot; float* first_slot;              // lie part_stride floats apart from first_slot on, and meet at `ticket`
    int64_t part_stride; int* ticket;
    int slot_rows;                               // rows of a partial result; behind them (m, l) of each
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
typedef __attribute__((ext_vector_type(4))) _Float16 h4_t;
__device__ inline f4_t mma16(const uint2& a, const uint2& b, f4_t c, F16T) {      // 16 keys: half a fragment
    return __builtin_amdgcn_mfma_f32_16x16x16f16(*reinterpret_cast<const h4_t*>(&a), *reinterpret_cast<const h4_t*>(&b), c, 0, 0, 0);
}
__device__ inline f4_t mma16(const uint2& a, const uint2& b, f4_t c, BF16T) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(*reinterpret_cast<const s4_t*>(&a), *reinterpret_cast<const s4_t*>(&b), c, 0, 0, 0);
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
// the same from a wave-uniform base and a 32-bit byte offset per lane
__device__ inline void glds16(const unsigned char* base, uint32_t off, uint32_t lds_base) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(off), "s"(lds_base), "s"(base) : "memory");
}
__device__ inline const unsigned char* uniform(const unsigned char* p) {
    const uint64_t v = (uint64_t)p;
    return (const unsigned char*)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32);
}
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }      // (a value that the compiler does not see is uniform)
// The loads of v are waited for HERE: left to their first use inside the key loop, the compiler would wait there in every round, and with
// them for the DMA in flight.
__device__ inline void arrived(uint4& v) { asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w)); }
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

// block id of a key through the segment's ids in LDS (ids: where page 0 would be), -1 outside [ka, kb)
__device__ inline int key_block(const int* ids, int key, int ka, int kb, int shift) {
    return key >= ka && key < kb ? ids[key >> shift] : -1;
}
// What the DMA reads for a key: the 16-byte chunk `ch` of its row; outside [ka, kb) the nearest key's, on a bad page block 0's (a
// valid address: such keys are masked).  32 x 32 + 64-bit arithmetic in 16-byte units: with 64-bit strides the addresses of a tile cost
// as much as its softmax (8 chunks of 2048 tokens, heads of 128: 743 -> 817 TFLOP/s).
struct RowAt { uint32_t id, off; };
__device__ inline RowAt row_at(const int* ids, int key, int ka, int kb, int shift) {
    const M5KeyAt k = m5_key_at(key, ka, kb, shift);
    return {(uint32_t)max(ids[k.page], 0), (uint32_t)k.off};
}
__device__ inline const unsigned char* row_chunk(const unsigned char* base, RowAt r, uint32_t bs16, uint32_t ss16, uint32_t ch) {
    return base + (((uint64_t)r.id * bs16 + (__umul24(r.off, ss16) + ch)) << 4);
}

// Partial results cross between workgroups (and XCDs, whose L2s do not share lines) as agent-scope accesses: written through to memory and
// read from there.  A workgroup's stores are waited for before its ticket is drawn, so no cache has to be written back or invalidated
// (an acquire-release ticket does both for the whole L2: 64 requests of 1 to 16 thousand keys 380 us instead of 328).
__device__ inline void put_part(float* p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), (unsigned long long)__float_as_uint(a) | (unsigned long long)__float_as_uint(b) << 32,
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// four of them, 16-byte aligned, by one store of that scope (neighbouring lanes fill whole lines: half-filled ones cost the memory twice);
// waited for like the others (the wait state: the data registers may be written right behind)
__device__ inline void put_part4(float* p, f4_t v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" :: "v"(p), "v"(v) : "memory");
}
__device__ inline float2 get_part(const float* p) {
    const unsigned long long v = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// p = exp2(s sc2 - use), use = m sc2 rounded, in one fused operation.  Its residue, up to half a unit of the last place of use, is the same factor
// for all that a row adds up and cancels, but from 2^24 on the unit is 2 and more and p may leave the operand type (fp16 first) or 32 bits: there
// exp2((s - m) sc2) is taken, whose difference is exact for the scores that count.
constexpr float FAR_SCORE = 1 << 24;

// softmax state of one row block: new maximum from this lane's scores (already reduced over the lanes of the row); m: of the scores unscaled
struct Soft {
    float m, l;
    __device__ inline float step(float mx, float sc2, float& use) {       // returns the factor of everything accumulated so far
        const float mn = fmaxf(m, mx);
        use = mn == -INFINITY ? 0.f : mn * sc2;
        const float alpha = __builtin_amdgcn_exp2f(m * sc2 - use);
        m = mn;
        return alpha;
    }
};

// four features of a row to the output
template <typename T, int HD>
__device__ inline void put_row(const Launch& L, const Item& it, int row, int d, f4_t o, float l) {
    const int rho = it.rho0 + row, tok = L.group.div(rho);
    const float inv = l > 0.f ? 1.0f / l : l;                // (no key seen: zeros; NaN stays NaN)
    typename T::storage* out = (typename T::storage*)L.a.out + (int64_t)(it.rq.r0 + tok) * L.a.o_rs + (int64_t)(it.kvh * L.group.d + rho - tok * L.group.d) * L.a.o_hs + d;
    if (l == 0.f) o = f4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (T::EPL == 4) *reinterpret_cast<f4_t*>(out) = o * inv;
    else *reinterpret_cast<uint2*>(out) = m5_pack4<T>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

// ------------------------------------------------------------------------------------------------------ few rows
template <typename T, int HD, int R>
struct Few {
    using st = typename T::storage;
    static constexpr int ES = sizeof(st), RB = HD * ES;          // bytes of a row
    // Keys of a stage: 8 KB of K and V, so that two workgroups share a CU and one computes while the other starts or ends an item (one
    // workgroup of 16 KB stages: decode_long 178 us when its items filled the chip exactly once, 211-257 in 2-4 rounds).  fp32
    // takes the same 16 keys.
    static constexpr int KS = ES == 4 || HD == 128 ? 16 : 32, SUB = KS / 16;
    using Frag = std::conditional_t<ES == 2 && SUB == 1, uint2, uint4>;      // a lane's keys of the second product
    static constexpr int LPR = RB / 16, RPI = 64 / LPR;          // lanes per row, rows per DMA instruction
    static constexpr int NI = KS / RPI;                          // DMA instructions of K (and of V) per stage
    static constexpr int OP_B = KS * RB, STAGE_B = 2 * OP_B, WAVE_B = 2 * STAGE_B;
    static constexpr int NF = RB / 64, ND = HD / 16;             // K fragments per key row block, feature blocks of V
    static constexpr int LDS_B = NWAVE * WAVE_B;
    // All fragments of a stage are requested before its first product where the registers allow it (5 short requests 7.63 -> 7.58 us, a chunk beside
    // 40 single tokens 100 -> 97); with 32 rows of 128 features they do not (64 requests with drafts 308 -> 332).
    static constexpr bool AHEAD = ES == 4 || HD == 64 || R == 1;
    static_assert(R * 16 * HD * 4 <= WAVE_B, "the waves' results meet in their rings");

    // 16-byte chunk swizzles: 16 (8 for V) rows of one chunk column fall into different banks
    __device__ static inline int kswz(int row) { return RB == 128 ? (row >> 1) & 7 : row & 15; }
    __device__ static inline int vswz(int row) { return ES == 4 ? ((row >> 2) & 3) << 2 : (RB == 128 ? ((row >> 1) & 3) << 1 : (row & 7) << 1); }

    // V of a stage that not all rows see whole: keys that are not there become zeros, non-finite values are noted and taken out (true).
    __device__ static bool clean(unsigned char* vs, uint32_t there, uint32_t* up, uint32_t* down) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));                           // (addresses of this rare path are not to be kept in registers through the key loop)
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
            const int rho = min(it.rho0 + rb * 16 + c, it.rho1 - 1), tok = L.group.div(rho);
            qpos[rb] = pos0 + tok;
            const st* q = (const st*)p.q + (int64_t)(it.rq.r0 + tok) * p.q_rs + (int64_t)(it.kvh * L.group.d + rho - tok * L.group.d) * p.q_hs;
#pragma unroll
            for (int t = 0; t < NF; ++t) qf[rb][t] = *reinterpret_cast<const uint4*>(q + (4 * t + g) * T::EPL);
        }
        const int pos_min = uniform(pos0 + L.group.div(it.rho0)), pos_max = uniform(pos0 + L.group.div(it.rho1 - 1));
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
        const int step = NWAVE * KS;                                // keys of one round of the waves
        const int64_t seg = ((int64_t)(MAXP - 1) << L.shift) / step * step;
        const int k_first = it.ka & ~(KS - 1);

#pragma unroll
        for (int rb = 0; rb < R; ++rb)
#pragma unroll
            for (int t = 0; t < NF; ++t) arrived(qf[rb][t]);
        vm_wait<0>();                                            // nothing of an earlier item is in flight
        for (int64_t s0 = k_first; s0 < it.kb; s0 += seg) {
            const int s1 = (int)min((int64_t)it.kb, s0 + seg);
            const int page0 = (int)s0 >> L.shift, np = ((s1 - 1) >> L.shift) - page0 + 1;
            const int* id0 = ids - page0;
            __syncthreads();
            for (int i = tid; i < np; i += NT) ids[i] = m5_block(p.block_table[(int64_t)it.b * p.table_rs + page0 + i], p.n_blocks);
            __syncthreads();
            auto fetch = [&](int kb, int stage) {
                const uint32_t to = ring + stage * STAGE_B;
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    const int row = j * RPI + lane / LPR, ch = lane % LPR;
                    const RowAt at = row_at(id0, kb + row, it.ka, s1, L.shift);
                    glds16(row_chunk(Kg, at, L.k_bs16, L.k_ss16, ch ^ kswz(row)), to + j * 1024);
                    glds16(row_chunk(Vg, at, L.v_bs16, L.v_ss16, ch ^ vswz(row)), to + OP_B + j * 1024);
                }
            };
            auto block = [&](int kb, int stage) {
                const unsigned char* ks = mine + stage * STAGE_B;
                const unsigned char* vs = ks + OP_B;
                const uint32_t there = (uint32_t)__ballot(key_block(id0, kb + (lane & (KS - 1)), it.ka, s1, L.shift) >= 0) & (uint32_t)((1ull << KS) - 1);
                const bool whole = there == (uint32_t)((1ull << KS) - 1) && kb + KS - 1 <= pos_min && kb >= lo_max;
                const bool odd = !whole && clean(mine + stage * STAGE_B + OP_B, there, up, down);
                uint32_t vis[R];
                auto key_frag = [&](int h, int t) {
                    const int row = h * 16 + c;
                    return *reinterpret_cast<const uint4*>(ks + row * RB + (((4 * t + g) ^ kswz(row)) << 4));
                };
                auto value_frag = [&](int d) {
                    Frag v;
                    if constexpr (ES == 4) {
                        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = 4 * g + r;
                            w[r] = *reinterpret_cast<const uint32_t*>(vs + row * RB + (((4 * d + (c >> 2)) ^ vswz(row)) << 4) + (c & 3) * 4);
                        }
                    } else {
                        uint2 half[SUB];
#pragma unroll
                        for (int h = 0; h < SUB; ++h) {
                            const int row = 16 * h + 4 * g + (c >> 2);
                            half[h] = tr_read(vs + row * RB + (((2 * d + ((c >> 1) & 1)) ^ vswz(row)) << 4) + (c & 1) * 8);
                        }
                        if constexpr (SUB == 2) v = make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
                        else v = half[0];
                    }
                    return v;
                };
                uint4 kf[SUB][NF];
                Frag vf[ND];
                if constexpr (AHEAD) {
#pragma unroll
                    for (int h = 0; h < SUB; ++h)
#pragma unroll
                        for (int t = 0; t < NF; ++t) kf[h][t] = key_frag(h, t);
#pragma unroll
                    for (int d = 0; d < ND; ++d) vf[d] = value_frag(d);
                    __builtin_amdgcn_sched_barrier(0);
                }
                f4_t s[R][SUB];
#pragma unroll
                for (int h = 0; h < SUB; ++h) {
#pragma unroll
                    for (int rb = 0; rb < R; ++rb) s[rb][h] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < NF; ++t) {
                        if constexpr (!AHEAD) kf[h][t] = key_frag(h, t);
#pragma unroll
                        for (int rb = 0; rb < R; ++rb)
                            if (R == 1 || rb < nrb) s[rb][h] = mma16(kf[h][t], qf[rb][t], s[rb][h], T());
                    }
                }
                Frag pf[R];
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
                    mx = fmaxf(mx, lane_xor32(mx));
                    float use;
                    const float alpha = sm[rb].step(mx, L.sc2, use);
                    if (__any(fabsf(use) >= FAR_SCORE)) {
                        const float base = fabsf(use) >= FAR_SCORE ? sm[rb].m : 0.f;
#pragma unroll
                        for (int h = 0; h < SUB; ++h) s[rb][h] -= base;
                        use = base != 0.f ? 0.f : use;
                    }
                    float sum = 0.f;
                    __attribute__((aligned(16))) st e[4 * SUB];
#pragma unroll
                    for (int h = 0; h < SUB; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][h][r], L.sc2, -use));
                            sum += x;
                            e[4 * h + r] = T::from_f32(x);       // 16-bit: p in (0, 1] rounded once for the matrix product, summed in fp32
                        }
                    pf[rb] = *reinterpret_cast<const Frag*>(e);
                    sm[rb].l = sm[rb].l * alpha + sum;
                    if (!__all(alpha == 1.0f))
#pragma unroll
                        for (int d = 0; d < ND; ++d) o[rb][d] *= alpha;
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    if constexpr (!AHEAD) vf[d] = value_frag(d);
#pragma unroll
                    for (int rb = 0; rb < R; ++rb)
                        if (R == 1 || rb < nrb) o[rb][d] = mma16(vf[d], pf[rb], o[rb][d], T());
                }
                if (odd) {
                    int at = 4 * g;
                    asm volatile("" : "+v"(at));                 // (computed here: the compiler would keep an address per feature in registers)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            asm volatile("" ::: "memory");       // (one feature's notes at a time)
                            const uint32_t u = up[at + 16 * d + r], n = down[at + 16 * d + r];
#pragma unroll
                            for (int rb = 0; rb < R; ++rb)
                                if (R == 1 || rb < nrb) o[rb][d][r] += infinite_part(u & vis[rb], n & vis[rb]);
                        }
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
#pragma unroll
        for (int rb = 0; rb < R; ++rb) {
            if (R > 1 && rb >= nrb) continue;
            float l = sm[rb].l;
            l += lane_xor16(l);
            l += lane_xor32(l);
            const int row = rb * 16 + c;
            if (g == 0) { ml[(wave * 32 + row) * 2] = sm[rb].m * L.sc2; ml[(wave * 32 + row) * 2 + 1] = l; }
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<f4_t*>(om + row * HD + (((4 * d + g) ^ (row & 15)) << 2)) = o[rb][d];
        }
        __syncthreads();
        float* slot = it.n_parts > 1 ? it.slot : nullptr;
        const int chunks = (it.rho1 - it.rho0) * (HD / 4);
        for (int i = tid; i < chunks; i += NT) {
            const int row = i / (HD / 4), ch = i % (HD / 4);
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < NWAVE; ++w) m = fmaxf(m, ml[(w * 32 + row) * 2]);
            const float use = m == -INFINITY ? 0.f : m;
            f4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NWAVE; ++w) {
                const float f = __builtin_amdgcn_exp2f(ml[(w * 32 + row) * 2] - use);
                l += ml[(w * 32 + row) * 2 + 1] * f;
                sum += *reinterpret_cast<const f4_t*>(reinterpret_cast<const float*>(lds + w * WAVE_B) + row * HD + ((ch ^ (row & 15)) << 2)) * f;
            }
            if (slot) {
                put_part4(slot + row * HD + ch * 4, sum);
                if (ch == 0) put_part(slot + it.slot_rows * HD + 2 * row, m, l);
            } else {
                put_row<T, HD>(L, it, row, ch * 4, sum, l);
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
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));                            // (as there)
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
        const int rho = min(w0 + c, it.rho1 - 1), tok = L.group.div(rho), qpos = pos0 + tok;
        const int pos_min = uniform(pos0 + L.group.div(w0)), pos_max = uniform(pos0 + L.group.div(max(w1 - 1, 0)));
        const int lo_min = m5_key_lo(pos_min, p.window), lo_max = m5_key_lo(pos_max, p.window), lo = m5_key_lo(qpos, p.window);
        uint4 qf[NF];
        {
            const st* q = (const st*)p.q + (int64_t)(it.rq.r0 + tok) * p.q_rs + (int64_t)(it.kvh * L.group.d + rho - tok * L.group.d) * p.q_hs;
#pragma unroll
            for (int t = 0; t < NF; ++t) qf[t] = *reinterpret_cast<const uint4*>(q + 16 * t + 8 * hh);
        }
        f16_t o[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
        float m = -INFINITY, use = 0.f, l = 0.f;
        const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);      // bf16
        const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
        unsigned long long* up = reinterpret_cast<unsigned long long*>(odd_lds);
        unsigned long long* down = up + HD;
        const int first_pos = uniform(pos0 + L.group.div(it.rho0)), last_lo = m5_key_lo(uniform(pos0 + L.group.div(it.rho1 - 1)), p.window);      // of all rows here
        const unsigned char* Kg = (const unsigned char*)p.k_cache + (int64_t)it.kvh * p.k_hs * 2;
        const unsigned char* Vg = (const unsigned char*)p.v_cache + (int64_t)it.kvh * p.v_hs * 2;
        const int seg = (int)min(((int64_t)(MAXP - 1) << L.shift) / KT * KT, (int64_t)1 << 30);
        const uint32_t mask = (1u << L.shift) - 1;
        // A DMA instruction reads RPI consecutive rows; pages of at least as many hold them together, so the page is wave-uniform and only
        // the offset inside it is the lane's (constant): no vector address arithmetic in the loop (with the other
        // savings of instructions here, 8 chunks of 2048 tokens, heads of 128: 817 -> 895 TFLOP/s; heads of 64: 664 -> 730).
        const bool one_page = mask + 1 >= RPI;
        uint32_t k_off[NJ], v_off[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int row = (wave * NJ + j) * RPI + lane / LPR, ch = lane % LPR;
            k_off[j] = (lane / LPR * L.k_ss16 + (ch ^ kswz(row))) << 4;
            v_off[j] = (lane / LPR * L.v_ss16 + (ch ^ vswz(row))) << 4;
        }

#pragma unroll
        for (int t = 0; t < NF; ++t) arrived(qf[t]);
        vm_wait<0>();
        for (int s0 = it.ka & ~(KT - 1); s0 < it.kb; s0 += seg) {
            const int s1 = uniform(min(it.kb, s0 + seg));
            const int page0 = s0 >> L.shift, np = ((s1 - 1) >> L.shift) - page0 + 1;
            const int* id0 = ids - page0;
            __syncthreads();
            int bad = 0;
            for (int i = tid; i < np; i += NT) {
                ids[i] = m5_block(p.block_table[(int64_t)it.b * p.table_rs + page0 + i], p.n_blocks);
                bad |= ids[i] < 0;
            }
            const bool some_bad = __syncthreads_or(bad);
            // lane j: the block of this wave's j-th instruction of the tile at kb
            auto blocks_of = [&](int kb) { return row_at(id0, kb + (wave * NJ + min(lane, NJ - 1)) * RPI, it.ka, s1, L.shift).id; };
            auto fetch = [&](int kb, int stage, uint32_t blocks) {
                const uint32_t to = ring + stage * STAGE_B + wave * NJ * 1024;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    if (one_page) {
                        const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)blocks, j), off = (uint32_t)(kb + (wave * NJ + j) * RPI) & mask;
                        glds16(uniform(Kg + (((uint64_t)id * L.k_bs16 + off * L.k_ss16) << 4)), k_off[j], to + j * 1024);
                        glds16(uniform(Vg + (((uint64_t)id * L.v_bs16 + off * L.v_ss16) << 4)), v_off[j], to + OP_B + j * 1024);
                    } else {
                        const int row = (wave * NJ + j) * RPI + lane / LPR, ch = lane % LPR;
                        const RowAt at = row_at(id0, kb + row, it.ka, s1, L.shift);
                        glds16(row_chunk(Kg, at, L.k_bs16, L.k_ss16, ch ^ kswz(row)), to + j * 1024);
                        glds16(row_chunk(Vg, at, L.v_bs16, L.v_ss16, ch ^ vswz(row)), to + OP_B + j * 1024);
                    }
                }
            };
            auto tile = [&](int kb, int stage, unsigned long long there, bool odd) {
                const unsigned char* ks = lds + stage * STAGE_B;
                const unsigned char* vs = ks + OP_B;
                const bool whole = there == ~0ull && kb + KT - 1 <= pos_min && kb >= lo_max;
                f16_t s[2];
                uint4 kf[2][NF];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int t = 0; t < NF; ++t) {
                        const int row = 32 * h + c;
                        kf[h][t] = *reinterpret_cast<const uint4*>(ks + row * RB + (((2 * t + hh) ^ kswz(row)) << 4));
                    }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[h][r] = 0.f;
#pragma unroll
                    for (int t = 0; t < NF; ++t) s[h] = mma32(kf[h][t], qf[t], s[h], T());
                }
                // one key block's fragments ahead of the products (left to itself the compiler reads each fragment into the same registers and
                // waits for it: an LDS round trip per product)
                __builtin_amdgcn_sched_group_barrier(SCHED_DS, NF, 0);
#pragma unroll
                for (int t = 0; t < NF; ++t) {
                    __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(SCHED_DS, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, NF, 0);
                if (!whole) {
                    const unsigned long long vis = seen(there, kb, lo, qpos);
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
                mx = fmaxf(mx, lane_xor32(mx));
                // p = exp2(s - m) with an m that is raised only when a score passes it by more than 8: p stays below 2^8, which the operand
                // types hold with the same relative error, and most tiles spare the rescaling of o (64 or 32 products per lane)
                if (__any((mx - m) * L.sc2 > 8.f)) {
                    const float mn = fmaxf(m, mx);
                    use = mn == -INFINITY ? 0.f : mn * L.sc2;
                    const float alpha = __builtin_amdgcn_exp2f(m * L.sc2 - use);
                    m = mn;
                    l *= alpha;
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[d] *= alpha;
                }
                float minus = use;
                if (__any(fabsf(use) >= FAR_SCORE)) {
                    const float base = fabsf(use) >= FAR_SCORE ? m : 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) s[h] -= base;
                    minus = base != 0.f ? 0.f : use;
                }
                uint4 pf[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        st e[8];
                        float x[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][8 * k + j], L.sc2, -minus));
                            e[j] = T::from_f32(x[j]);
                        }
                        pf[h][k] = *reinterpret_cast<const uint4*>(e);
                        // the denominator in fp32: of the rounded pairs (bf16: one instruction a pair), of the values (fp16, whose small
                        // p the pair instruction might take for zero)
                        if constexpr (T::id == M5_BF16) l = dot8<T>(pf[h][k], ones, l);
                        else
#pragma unroll
                            for (int j = 0; j < 8; ++j) l += x[j];
                    }
                uint4 vf[4][ND];
#pragma unroll
                for (int k = 0; k < 4; ++k)                      // 16 keys at a time
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const int row = 16 * k + 4 * hh + ((lane & 15) >> 2), ch = 4 * d + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
                        const uint2 v0 = tr_read(vs + row * RB + ((ch ^ vswz(row)) << 4) + (lane & 1) * 8);
                        const uint2 v1 = tr_read(vs + (row + 8) * RB + ((ch ^ vswz(row + 8)) << 4) + (lane & 1) * 8);
                        vf[k][d] = make_uint4(v0.x, v0.y, v1.x, v1.y);
                    }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int d = 0; d < ND; ++d) o[d] = mma32(vf[k][d], pf[k >> 1][k & 1], o[d], T());
                __builtin_amdgcn_sched_group_barrier(SCHED_DS, 2 * ND, 1);
#pragma unroll
                for (int k = 0; k < 3; ++k) {                    // (as above, 16 keys ahead)
                    __builtin_amdgcn_sched_group_barrier(SCHED_DS, 2 * ND, 1);
                    __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, ND, 1);
                }
                __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, ND, 1);
                if (odd) {                                       // (of the workgroup: this wave's rows may see the tile whole)
                    const unsigned long long vis = seen(there, kb, lo, qpos);
                    int at = 4 * hh;
                    asm volatile("" : "+v"(at));                 // (computed here: the compiler would keep an address per feature in registers)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            asm volatile("" ::: "memory");       // (one feature's notes at a time)
                            o[d][r] += infinite_part(up[at + 32 * d + 8 * (r >> 2) + (r & 3)] & vis, down[at + 32 * d + 8 * (r >> 2) + (r & 3)] & vis);
                        }
                }
            };
            int stage = 0;
            fetch(s0, 0, blocks_of(s0));
            uint32_t next = blocks_of(s0 + KT);
            for (int kb = s0; kb < s1; kb += KT, stage ^= 1) {
                vm_wait<0>();
                __syncthreads();                                 // the tile is there for all waves, and all are done with the other stage
                if (kb + KT < s1) fetch(kb + KT, stage ^ 1, next);
                next = blocks_of(kb + 2 * KT);
                unsigned long long there = seen(~0ull, kb, it.ka, s1 - 1);
                if (some_bad) there = __ballot(key_block(id0, kb + lane, it.ka, s1, L.shift) >= 0);
                const bool odd = !(there == ~0ull && kb + KT - 1 <= first_pos && kb >= last_lo) && clean(lds + stage * STAGE_B + OP_B, there, up, down);
                if (w0 < w1 && kb <= pos_max && kb + KT > lo_min) tile(kb, stage, there, odd);
            }
        }
        l += lane_xor32(l);
        if (it.n_parts > 1) {
            // Through LDS, so that a wave stores whole rows (64 requests of 4 to 16 thousand keys, 128 rows each, heads of 64 / 128: 191 / 366 us
            // with a row per lane, 64 pieces of as many lines a store; 168 / 341 so).
            __syncthreads();                                     // all waves are done with the stages
            float* om = reinterpret_cast<float*>(lds) + wave * 32 * HD;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f4_t*>(om + c * HD + (((8 * d + 2 * q + hh) ^ (c & 7)) << 2)) = f4_t{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
            lds_wait();
            float* slot = it.slot + (int64_t)wave * 32 * HD;
            for (int i = lane; i < (w1 - w0) * (HD / 4); i += 64) {
                const int r = i / (HD / 4), ch = i % (HD / 4);
                put_part4(slot + i * 4, *reinterpret_cast<const f4_t*>(om + r * HD + ((ch ^ (r & 7)) << 2)));
            }
            if (hh == 0 && w0 + c < w1) put_part(it.slot + it.slot_rows * HD + 2 * (wave * 32 + c), m * L.sc2, l);
            return;
        }
        if (w0 + c >= w1) return;
        const int row = wave * 32 + c;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                put_row<T, HD>(L, it, row, 32 * d + 8 * q + 4 * hh, f4_t{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]}, l);
    }
};

// Joins a tile's partial results: the parts are dealt to groups of threads (one thread holds four features of a row), and the groups meet in
// LDS; I rows' features and U parts are in flight per thread (a read of a part goes to memory: about a microsecond).  The order
// depends on the counts alone.
template <typename T, int HD, int I, int U>
__device__ void join_all(const Launch& L, const Item& it, unsigned char* lds) {
    const float* first = it.first_slot;
    const int64_t stride = it.part_stride;
    constexpr int C4 = HD / 4;
    const int tid = threadIdx.x, chunks = (it.rho1 - it.rho0) * C4, groups = chunks < NT ? min(NT / chunks, it.n_parts) : 1;
    f4_t* meet = reinterpret_cast<f4_t*>(lds);               // [NT] sums, then [NT] (m, l)
    float2* meet_ml = reinterpret_cast<float2*>(lds + NT * 16);
    const int grp = chunks < NT ? tid / chunks : 0;
    for (int base = 0; base < chunks; base += I * NT) {
        int at[I];
        bool live[I];
        float m[I], l[I];
        f4_t sum[I];
#pragma unroll
        for (int i = 0; i < I; ++i) {
            at[i] = chunks < NT ? tid - grp * chunks : base + i * NT + tid;
            live[i] = grp < groups && at[i] < chunks && (i == 0 || chunks >= NT);
            if (!live[i]) at[i] = 0;
            m[i] = -INFINITY;
            l[i] = 0.f;
            sum[i] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
        for (int k0 = min(grp, it.n_parts - 1); k0 < it.n_parts; k0 += groups * U) {
            float2 ml[I][U];
            f4_t v[I][U];
#pragma unroll
            for (int i = 0; i < I; ++i)
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const float* s = first + min(k0 + u * groups, it.n_parts - 1) * stride;
                    ml[i][u] = get_part(s + it.slot_rows * HD + 2 * (at[i] / C4));
                    const float2 a = get_part(s + at[i] * 4), b = get_part(s + at[i] * 4 + 2);
                    v[i][u] = f4_t{a.x, a.y, b.x, b.y};
                }
#pragma unroll
            for (int i = 0; i < I; ++i) {
                float mn = m[i];
#pragma unroll
                for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[i][u].x);
                const float use = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m[i] - use);
                m[i] = mn;
                l[i] *= alpha;
                sum[i] *= alpha;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u * groups >= it.n_parts) continue;     // (the last part, read again)
                    // a part whose scores are all NaN has m = -inf, so weight 0, and l = NaN, which stays: no part is left out for its weight
                    const float f = __builtin_amdgcn_exp2f(ml[i][u].x - use);
                    l[i] += ml[i][u].y * f;
                    sum[i] += v[i][u] * f;
                }
            }
        }
        if (groups > 1) {                                    // (chunks < NT: one round, i = 0)
            meet[tid] = sum[0];
            meet_ml[tid] = make_float2(m[0], l[0]);
            __syncthreads();
            if (live[0] && grp == 0) {
                float mn = m[0];
                for (int g = 1; g < groups; ++g) mn = fmaxf(mn, meet_ml[g * chunks + at[0]].x);
                const float use = mn == -INFINITY ? 0.f : mn, alpha = __builtin_amdgcn_exp2f(m[0] - use);
                l[0] *= alpha;
                sum[0] *= alpha;
                for (int g = 1; g < groups; ++g) {
                    const float2 o = meet_ml[g * chunks + at[0]];
                    const float f = __builtin_amdgcn_exp2f(o.x - use);
                    l[0] += o.y * f;
                    sum[0] += meet[g * chunks + at[0]] * f;
                }
                m[0] = mn;
            }
        }
#pragma unroll
        for (int i = 0; i < I; ++i)
            if (live[i] && grp == 0) put_row<T, HD>(L, it, at[i] / C4, at[i] % C4 * 4, sum[i], l[i]);
    }
}

// Draws the tile's ticket; the workgroup that draws the last one joins.
template <typename T, int HD>
__device__ void join_parts(const Launch& L, const Item& it, unsigned char* lds, int* sh_last) {
    vm_wait<0>();                                            // this thread's part is in memory,
    __syncthreads();                                         // and so is the whole workgroup's
    if (threadIdx.x == 0) {
        const int n = __hip_atomic_fetch_add(it.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *sh_last = n == it.n_parts - 1;
        if (n == it.n_parts - 1) __hip_atomic_store(it.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);    // ready for the next call
    }
    __syncthreads();
    if (!*sh_last) return;
    if ((it.rho1 - it.rho0) * (HD / 4) < NT) join_all<T, HD, 1, 4>(L, it, lds);       // several groups: few parts each
    else if (it.n_parts <= 4) join_all<T, HD, 4, 4>(L, it, lds);
    else if (it.n_parts <= 8) join_all<T, HD, 2, 8>(L, it, lds);
    else join_all<T, HD, 1, 16>(L, it, lds);
}

// inclusive sum over the lanes of a wave: DPP row shifts, then the rows' last lanes broadcast
template <int CTRL, int ROWS>
__device__ inline int dpp_add(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ inline int wave_scan(int v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}

// Items: every (request, tile, chunk of `cu` units, kv head), numbered by request.  Up to 64 requests a wave keeps in its lanes, more lie
// in LDS as prefix sums.
template <int TR_FEW, int TR_MANY, int HD, int MIN_UNITS>
struct Deal {
    int cu, total;
    M5Request mine;
    int incl, rows_incl;                                     // (up to 64 requests: items, and rows of partial results, of this lane's and all before it)
    bool sane;                                               // row offsets that ascend (others hold more tiles than their rows can: nothing is computed)

    __device__ inline int chunks(const M5Share& s) const { return m5_chunks(s.units, cu); }
    __device__ inline int items(const Launch& L, const M5Share& s) const { return s.tiles * chunks(s) * (int)L.kv.d; }
    __device__ inline int part_rows(const Launch& L, const M5Share& s) const { return s.units > cu ? items(L, s) * s.sr : 0; }
    // How long a chunk is (m5_chunk_units).
    //  - Few tiles (at most a quarter of the places): chunks as long as the places, once filled, allow (3 requests of 60 to 120 thousand keys:
    //    159 us in 512 items, 165 / 175 / 177 in 1024 / 1536 / 2048).
    //  - Up to two per place: four items per place, so that requests of different lengths end together (64 requests of 1 to 16 thousand
    //    keys in 512 tiles: 485 us unsplit, 395 / 346 / 328 us in about 850 / 1300 / 1700 items).
    //    Tiles of more than 32 rows up to 2 (64 requests of 4 to 16 thousand keys and 40 rows, heads of 64 / 128: 204 / 332 us with 1, 162 / 305
    //    with 2, 166 / 328 with 2.5, 176 / 337 with 4).
    //  - More balance by themselves, only much longer ones are split (40 requests of 300 to 3000 keys beside a chunk, 1152 tiles: 120 us
    //    unsplit, 147 with the longer third in two parts).
    __device__ inline void length(const Launch& L, float units, float tiles, float unit_rows, float tile_rows) {
        const float kv = (float)L.kv.d;                      // (float sums: exact as far as tiles are few enough to be split)
        // a tile of u units in n parts takes about a u / n + b n (the join, which grows with the rows): no shorter than sqrt(b u / a) (16 rows, one
        // request of 100 thousand keys and one kv head: 45 / 39 / 37 us with a factor of 1 / 0.7 / 0.5)
        const float by = 0.6f + 1.6f / 128.f * tile_rows / max(tiles, 1.f);
        cu = m5_chunk_units(units * kv, tiles * kv, unit_rows * kv, tile_rows * kv, (float)L.places, (float)L.n_tickets, (float)L.slot_rows,
                            max((float)MIN_UNITS, by * sqrtf(units / max(tiles, 1.f))));
        sane = tiles * kv <= L.max_tiles;
    }
    __device__ inline M5Request request(const Launch& L, int b) const {
        return m5_request(L.a.q_start[b], L.a.q_start[b + 1], L.a.seq_len[b], L.a.n_rows, (int64_t)L.a.table_width << L.shift);
    }
    __device__ inline M5Share share(const Launch& L, const M5Request& q) const { return m5_share(q, (int)L.group.d, TR_FEW, TR_MANY, L.a.window); }
    __device__ void setup(const Launch& L, int* pre, float* red, int* sums) {
        const int B = L.a.n_seq, tid = threadIdx.x, lane = tid & 63;
        if (B <= 64) {
            mine = lane < B ? request(L, lane) : M5Request{0, 0, 0};
            const M5Share s = share(L, mine);
            const float t = (float)s.tiles, w = t * (float)s.units;
            length(L, wave_sum(w), wave_sum(t), wave_sum(w * (float)s.sr), wave_sum(t * (float)s.sr));
            incl = wave_scan(sane ? items(L, s) : 0);
            rows_incl = wave_scan(sane ? part_rows(L, s) : 0);
            total = __builtin_amdgcn_readlane(incl, 63);
            return;
        }
        const int per = (B + NT - 1) / NT, b0 = min(tid * per, B), b1 = min(b0 + per, B);
        float units = 0.f, tiles = 0.f, unit_rows = 0.f, tile_rows = 0.f;
        for (int b = b0; b < b1; ++b) {
            const M5Share s = share(L, request(L, b));
            const float t = (float)s.tiles, w = t * (float)s.units;
            tiles += t;
            units += w;
            tile_rows += t * (float)s.sr;
            unit_rows += w * (float)s.sr;
        }
        units = block_sum<NWAVE>(units, red);
        tiles = block_sum<NWAVE>(tiles, red);
        unit_rows = block_sum<NWAVE>(unit_rows, red);
        tile_rows = block_sum<NWAVE>(tile_rows, red);
        length(L, units, tiles, unit_rows, tile_rows);
        if (!sane) {
            total = 0;
            return;
        }
        int n = 0, r = 0;
        for (int b = b0; b < b1; ++b) {
            const M5Share s = share(L, request(L, b));
            n += items(L, s);
            r += part_rows(L, s);
        }
        const int n_upto = wave_scan(n), r_upto = wave_scan(r);
        if (lane == 63) { sums[tid >> 6] = n_upto; sums[NWAVE + (tid >> 6)] = r_upto; }
        __syncthreads();
        int base = n_upto - n, row = r_upto - r;
        total = 0;
        for (int w = 0; w < NWAVE; ++w) {
            if (w < tid >> 6) { base += sums[w]; row += sums[NWAVE + w]; }
            total += sums[w];
        }
        for (int b = b0; b < b1; ++b) {
            pre[b] = base;
            reinterpret_cast<uint16_t*>(pre + B + 1)[b] = (uint16_t)(row >> 4);
            const M5Share s = share(L, request(L, b));
            base += items(L, s);
            row += part_rows(L, s);
        }
        if (tid == NT - 1) pre[B] = total;
        __syncthreads();
    }
    // item `id`: its place in its request; false where no row of the tile sees a key of the chunk
    __device__ inline bool item(const Launch& L, const int* pre, int id, Item& it, int& tr) const {
        int at, row0;                                        // place in the request; first row of its partial results
        if (L.a.n_seq <= 64) {
            it.b = __builtin_popcountll(__ballot(incl <= id));           // requests that end before it
            it.rq.r0 = __builtin_amdgcn_readlane(mine.r0, it.b);
            it.rq.r1 = __builtin_amdgcn_readlane(mine.r1, it.b);
            it.rq.len = __builtin_amdgcn_readlane(mine.len, it.b);
            at = id - (it.b ? __builtin_amdgcn_readlane(incl, it.b - 1) : 0);
            row0 = it.b ? __builtin_amdgcn_readlane(rows_incl, it.b - 1) : 0;
        } else {
            it.b = __builtin_amdgcn_readfirstlane(m5_upper(pre, L.a.n_seq, id));
            it.rq = request(L, it.b);
            at = id - __builtin_amdgcn_readfirstlane(pre[it.b]);
            row0 = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint16_t*>(pre + L.a.n_seq + 1)[it.b]) << 4;
        }
        const M5Share s = share(L, it.rq);
        const int nc = chunks(s), rest = L.kv.div(at);
        it.kvh = at - rest * (int)L.kv.d;
        const int up = nc == 1 ? rest : (int)((uint32_t)rest / (uint32_t)nc), chunk = rest - up * nc;
        it.rho0 = (s.tiles - 1 - up) * s.tr;                 // the longest rows first
        it.rho1 = min(it.rho0 + s.tr, s.rows);
        tr = s.tr;
        const int pos0 = it.rq.len - (it.rq.r1 - it.rq.r0);
        M5Span span;
        if (!m5_span(s, it.rq.len, L.a.window, pos0 + L.group.div(it.rho0), pos0 + L.group.div(it.rho1 - 1), nc, cu, chunk, span)) return false;
        it.n_parts = span.c1 - span.c0 + 1;
        if (it.n_parts > 1) {
            const int64_t size = (int64_t)s.sr * (HD + 2);   // rows of o, then (m, l) of each
            const int back = (chunk - span.c0) * (int)L.kv.d;               // (the chunks of a tile are n_kv_heads items apart)
            it.slot = L.slots + (int64_t)row0 * (HD + 2) + at * size;
            it.first_slot = it.slot - back * size;
            it.part_stride = (int64_t)L.kv.d * size;
            it.ticket = L.tickets + (id - back);
            it.slot_rows = s.sr;
        }
        it.rho0 = uniform(it.rho0);
        it.rho1 = uniform(it.rho1);
        it.kvh = uniform(it.kvh);
        it.ka = uniform(span.ka);
        it.kb = uniform(span.kb);
        it.n_parts = uniform(it.n_parts);
        it.rq.r0 = uniform(it.rq.r0);
        it.rq.r1 = uniform(it.rq.r1);
        it.rq.len = uniform(it.rq.len);
        tr = uniform(tr);
        return true;
    }
};

// R: row blocks of the few-row tiles; MANY: requests of more rows get 128-row tiles.
template <typename T, int HD, int R, bool MANY>
struct Shape {
    using F = Few<T, HD, R>;
    static constexpr int TR = 16 * R, TRM = MANY ? 128 : 0;
    // Shortest chunk of keys, in 64s.  16 bits: joining costs about as much as 600 keys (5 requests of up to 700 keys: 7.6 us; 8.8 with 4).  fp32:
    // keys cost more (chunks of 131 rows: 49 us with 4, 54 with 8).
    static constexpr int MIN_UNITS = T::EPL == 4 ? 4 : 8;
    static constexpr int RING_B = MANY ? (F::LDS_B > 4 * 64 * HD * 2 ? F::LDS_B : 4 * 64 * HD * 2) : F::LDS_B;
    static constexpr int lds_bytes(int n_seq) { return RING_B + IDS_B + ML_B + odd_bytes(HD) + (n_seq + 1) * 6; }
};

template <typename T, int HD, int R, bool MANY>
__global__ __launch_bounds__(NT, HD == 64 || T::EPL == 8 ? 2 : 1) void paged_attn_kernel(Launch L) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    using S = Shape<T, HD, R, MANY>;
    int* ids = reinterpret_cast<int*>(lds + S::RING_B);
    float* ml = reinterpret_cast<float*>(lds + S::RING_B + IDS_B);
    int* sh = reinterpret_cast<int*>(lds + S::RING_B + IDS_B + ML_B - 64);
    unsigned char* odd = lds + S::RING_B + IDS_B + ML_B;
    int* pre = reinterpret_cast<int*>(odd + odd_bytes(HD));
    Deal<S::TR, S::TRM, HD, S::MIN_UNITS> deal;
    deal.setup(L, pre, ml, sh);
    for (int id = blockIdx.x; id < deal.total; id += gridDim.x) {
        Item it;
        int tr;
        if (!deal.item(L, pre, id, it, tr)) continue;
        if constexpr (MANY) {
            if (tr == 128) {
                Many<T, HD>::run(L, it, lds, ids, odd);
                if (it.n_parts > 1) join_parts<T, HD>(L, it, lds, sh);
                __syncthreads();
                continue;
            }
        }
        S::F::run(L, it, lds, ids, ml, odd);
        if (it.n_parts > 1) join_parts<T, HD>(L, it, lds, sh);
        __syncthreads();
    }
}

// The tiling for these shapes: rows of a few-row tile, or 0 for the kernel with 128-row tiles.  From 33 rows on the large tiles are faster also
// where they are mostly empty (64 requests of 4 to 16 thousand keys, 40 / 64 rows each, heads of 64: 162 / 167 us against 178 / 184 in tiles of
// 32; heads of 128: 305 / 321 against 364 / 378; tiles of 64 rows were slower than either).
int tiling(int dtype, const M5PagedAttnArgs& a) {
    const int64_t rows = (int64_t)min(max(a.max_new, 1), max(a.n_rows, 1)) * (a.n_heads / a.n_kv_heads);
    return rows <= 16 ? 16 : (rows <= 32 || dtype == M5_F32 ? 32 : 0);
}

template <typename T, int HD, int R, bool MANY>
int launch_as(Launch& L, int cus, hipStream_t s) {
    using S = Shape<T, HD, R, MANY>;
    static_assert(S::lds_bytes(MAX_SEQ) <= 160 * 1024, "the largest batch's LDS");
    const int lds = S::lds_bytes(L.a.n_seq);
    if (hipFuncSetAttribute((const void*)paged_attn_kernel<T, HD, R, MANY>, hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess) return M5_ERR_LAUNCH;
    const int64_t bytes = L.a.workspace ? min(L.a.workspace_bytes, MAX_WORKSPACE) : 0, row_b = (HD + 2) * 4;
    // The tickets' place depends on the workspace's size alone: calls of other types and shapes find them zero.  (A multiple of 16 bytes.)
    L.n_tickets = (int)min((int64_t)MAX_ITEMS, bytes / MIN_ITEM_BYTES) & ~3;
    L.slot_rows = (int)((bytes - L.n_tickets * 4) / row_b);
    L.tickets = (int*)L.a.workspace;
    L.slots = (float*)((char*)L.a.workspace + (int64_t)L.n_tickets * 4);
    L.places = cus * min(160 * 1024 / lds, 2);
    const int64_t tiles = ((int64_t)L.a.n_rows * L.group.d / S::TR + L.a.n_seq) * L.a.n_kv_heads;      // upper bound
    L.max_tiles = (float)tiles * 1.001f + 1.f;
    // A workgroup for every item there can be; a workgroup takes several where that is too many, and where every one has to go through a long
    // list of requests (2000 of 100 to 1500 keys, 8000 tiles: 734 us with a workgroup each, 490 / 470 / 460 with 8 / 4 / 2 per place; 70 longer
    // ones 117 with 8 / 4, 119 with 2).
    const int64_t chunks = (((int64_t)L.a.table_width << L.shift) + 64 * S::MIN_UNITS - 1) / (64 * S::MIN_UNITS);
    const int64_t most = (int64_t)4 * L.places;
    int64_t grid = L.n_tickets ? max(min(most, tiles * chunks), tiles) : tiles;
    if (L.a.n_seq > 64) grid = min(grid, most);
    hipLaunchKernelGGL((paged_attn_kernel<T, HD, R, MANY>), dim3((unsigned)min(grid, (int64_t)1 << 20)), dim3(NT), lds, s, L);
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
        ((int64_t)a->n_blocks << shift) > INT_MAX || (int64_t)a->n_rows * a->n_heads > (1 << 28) || (int64_t)a->n_seq * a->n_kv_heads > (1 << 28))
        return M5_ERR_UNSUPPORTED;
    const int epl = dtype == M5_F32 ? 4 : 8;
    if (!aligned(a->q, a->q_rs, a->q_hs, 0, epl) || !aligned(a->out, a->o_rs, a->o_hs, 0, epl) || !aligned(a->k_cache, a->k_bs, a->k_hs, a->k_ss, epl) ||
        !aligned(a->v_cache, a->v_bs, a->v_hs, a->v_ss, epl) || ((uintptr_t)a->workspace & 15))
        return M5_ERR_UNSUPPORTED;
    // strides of blocks below 64 GB, of slots below 64 MB (row_chunk)
    for (int64_t bs : {a->k_bs, a->v_bs})
        if (bs < 0 || bs / epl > UINT32_MAX) return M5_ERR_UNSUPPORTED;
    for (int64_t ss : {a->k_ss, a->v_ss})
        if (ss < 0 || ss / epl > (1 << 22)) return M5_ERR_UNSUPPORTED;
    return M5_OK;
}

template <typename T>
int launch(const M5PagedAttnArgs& a, int shift, hipStream_t s) {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return M5_ERR_LAUNCH;
    Launch L;
    L.a = a;
    L.shift = shift;
    L.group.set(a.n_heads / a.n_kv_heads);
    L.kv.set(a.n_kv_heads);
    L.sc2 = a.scale * 1.4426950408889634f;
    constexpr int E = T::EPL;
    L.k_bs16 = (uint32_t)(a.k_bs / E);
    L.k_ss16 = (uint32_t)(a.k_ss / E);
    L.v_bs16 = (uint32_t)(a.v_bs / E);
    L.v_ss16 = (uint32_t)(a.v_ss / E);
    const int tr = tiling(T::id, a);
    if (a.head_dim == 64) {
        if constexpr (T::id != M5_F32) {
            if (tr == 0) return launch_as<T, 64, 2, true>(L, cus, s);
        }
        return tr == 16 ? launch_as<T, 64, 1, false>(L, cus, s) : launch_as<T, 64, 2, false>(L, cus, s);
    }
    if constexpr (T::id != M5_F32) {
        if (tr == 0) return launch_as<T, 128, 2, true>(L, cus, s);
    }
    return tr == 16 ? launch_as<T, 128, 1, false>(L, cus, s) : launch_as<T, 128, 2, false>(L, cus, s);
}

}  // namespace

extern "C" int m5_paged_attention_workspace(int dtype, const M5PagedAttnArgs* a, int64_t* bytes) {
    const int rc = check(dtype, a);
    if (rc != M5_OK) return rc;
    if (!bytes) return M5_ERR_ARG;
    const int tr = tiling(dtype, *a);
    *bytes = min((int64_t)MAX_ITEMS * ((int64_t)(tr ? tr : 128) * (a->head_dim + 2) * 4 + 4), MAX_WORKSPACE);
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
