// Attention over the paged cache for sequences with many rows (prompts, wide groups, verify steps): the 5th-generation tensor cores.
//
// An item is 256 columns ((row, query head) pairs of a KV head) of a sequence as two tiles of 128; a unit is 64 keys of an item.
// The step's units are dealt evenly to the blocks, one an SM, in order; a run that ends inside an item leaves its state for the
// join kernel.  Per unit and tile:
//   S [128][64]  = Q [128][hd] . K^T      A = queries (f16; the first tile's in tensor memory, the second's in shared memory), B = keys [64][hd]
//   O [128][hd] += W [128][64] . V        A = weights (f16, tensor memory), B = values as [hd][64]
// Warps: 4 + 4 take the softmax of the two tiles (a thread a column: its row of S is in its tensor memory lane), 4 expand the
// codes to f16 (exact) into the layout the products read, 1 fetches pages, 1 issues the scores' products (a tile's next unit as
// soon as the last scores are in registers), 1 the values' (once the weights are there).  An item of up to 128 columns has both
// tiles work on the same queries, every other unit each, and their states joined at its end.
// f32 calls (FINE) add the products of the queries' second f16 terms, from shared memory, where an item has any that are not 0; the room for them is
// a fetched and an expanded stage at heads of 128 (4096 rows behind 4096 positions: 317 us as bf16 values in f32 arrays, 346 where the call does not say so, 383 with f32 values).
// The two scales and the running maxima are as in pages_attn_few.cu; here the maxima that the exponents use follow the true ones
// only when these have grown by 2^8 (weights up to 2^8 then), so O in tensor memory is hardly ever rescaled.
// Bound: a unit of two tiles takes 1024 clk of exponentials (16 a clock and SM; 32 more for the factors of its groups' sums, 64 over small pages), 1250 clk of products (the second tile's scores read
// their A operand from shared memory: 478 instead of 256), about 1300 clk of shared memory (codes in, f16 out, and what the products
// read) and 1000 issue slots a scheduler; measured 2360, of which 1560 remain without exponentials and most products: the barriers'
// and loads' latencies of two tiles.  4096 rows behind 4096 positions, 16 heads over 2: 292 us = 706 TFLOP/s.
#include <type_traits>

#include "pages_attn.cuh"
#include "seed_block.cuh"

namespace nsl {

constexpr int MANY_KEYS = 64, MANY_TILE = 128, MANY_COLS = PATTN_MANY, MANY_THREADS = 480, MANY_META = 16;
constexpr int MANY_EXPAND = 8, MANY_FETCH = 12, MANY_SCORES = 13;      // first warp of each part; the softmax has warps 0 .. 7, the values' products the last
constexpr int TM_S = 0, TM_Q = 128, TM_W = 192, TM_O = 256;         // tensor memory columns: S (64 a tile), the first tile's Q (64), W (32 a tile), O (128 a tile)
constexpr float MANY_SLACK = 8.0f;                                   // how far (in powers of 2) a weight may exceed 1

// FINE: queries as two f16 terms (f32 calls).  The second terms of both tiles take the place of a fetched and an expanded stage at heads of 128
// (of two expanded ones: 352 us where this takes 346, 409 where it takes 383).
template <int HD, bool FINE>
struct Many {
    static constexpr int RAWS = FINE && HD == 128 ? 2 : 3, STAGES = FINE && HD == 128 ? 3 : 4;
    static constexpr int RAW = MANY_KEYS * HD;                       // bytes of a unit's key codes, or value codes
    static constexpr int TILE = 2 * RAW;                             // the same as f16
    static constexpr int QUERIES = 2 * MANY_TILE * HD;               // bytes of a tile's queries as f16
    static constexpr int OFF_TILES = RAWS * 2 * RAW;
    static constexpr int OFF_Q = OFF_TILES + STAGES * 2 * TILE;      // the second tile's queries
    static constexpr int OFF_QLOW = OFF_Q + QUERIES;                 // FINE: both tiles' second terms
    static constexpr int OFF_META = OFF_QLOW + (FINE ? 2 * QUERIES : 0);
    static constexpr int OFF_BARS = OFF_META + MANY_META * 4 * 16;
    static constexpr int BARS = 2 * RAWS + 2 * STAGES + MANY_META + 11;
    static constexpr int SMEM = OFF_BARS + 8 * BARS + 1024;
};
static_assert(MANY_COLS == 2 * MANY_TILE, "two tiles an item");
static_assert(Many<128, false>::SMEM + 256 <= 232448 && Many<128, true>::SMEM + 256 <= 232448, "shared memory");
constexpr int MANY_SEQS = 4096;      // descriptors of a call; their units sit in the tiles' memory while the plan is made
static_assert(MANY_SEQS * 4 <= 4 * 4 * 64 * 64, "the plan's memory: four stages at heads of 64, two or four at 128");

__device__ int g_pattn_many_status;

struct ManyItem {
    RowSpan sp;
    int kvh, col0, cols;      // the item's columns: col0 .. col0 + cols - 1 of the KV head's
    int k0, k1, tile0, first, units, x0, x1;      // as FewItem
};

// Units of column tile ct.
__device__ __forceinline__ int many_units(const PagesAttn& a, const RowSpan& sp, int group, int cols, int ct, int* k0, int* k1) {
    const int i0 = ct * MANY_COLS / group, i1 = min(cols - 1, ct * MANY_COLS + MANY_COLS - 1) / group;
    *k1 = end_key(a, pos_of(sp.pos, i1));
    *k0 = min(first_key(a, pos_of(sp.pos, i0)), *k1);
    return max((*k1 + MANY_KEYS - 1) / MANY_KEYS - *k0 / MANY_KEYS, 1);
}
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// The walk over a block's units, by whole warps.
struct ManyWalk {
    int i, before;
    __device__ __noinline__ bool next(const PagesAttn& a, int group, int x, int xe, ManyItem* it) {
        const int lane = threadIdx.x & 31;
        if (x >= xe) return false;
        for (; i < a.n_seqs; ++i) {
            it->sp = row_span(a, i);
            const int cols = it->sp.rows * group, tiles = (cols + MANY_COLS - 1) / MANY_COLS;
            int at = before;      // units before the tiles looked at
            for (int t0 = 0; t0 < tiles; t0 += 32) {
                int k0 = 0, k1 = 0;
                const int n = t0 + lane < tiles ? many_units(a, it->sp, group, cols, t0 + lane, &k0, &k1) : 0;
                int incl = n * a.p.n_kv;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o); if (lane >= o) incl += v; }
                const uint32_t past = __ballot_sync(0xFFFFFFFFu, x < at + incl);
                if (past) {
                    const int l = __ffs(past) - 1, un = __shfl_sync(0xFFFFFFFFu, n, l), start = at + __shfl_sync(0xFFFFFFFFu, incl, l) - un * a.p.n_kv;
                    it->k0 = __shfl_sync(0xFFFFFFFFu, k0, l);
                    it->k1 = __shfl_sync(0xFFFFFFFFu, k1, l);
                    it->kvh = (x - start) / un;
                    it->col0 = (t0 + l) * MANY_COLS;
                    it->cols = min(MANY_COLS, cols - it->col0);
                    it->first = start + it->kvh * un;
                    it->units = un;
                    it->tile0 = it->k0 / MANY_KEYS;
                    it->x0 = x;
                    it->x1 = min(xe, it->first + un);
                    return true;
                }
                at += __shfl_sync(0xFFFFFFFFu, incl, 31);
            }
            before = at;
        }
        return false;
    }
};

__device__ __forceinline__ uint64_t many_desc(uint32_t saddr) {      // K-major, 128-byte swizzle, 8 rows of 128 bytes after one another
    return (uint64_t) ((saddr & 0x3FFFFu) >> 4) | ((uint64_t) 1 << 16) | ((uint64_t) (1024 >> 4) << 32) | ((uint64_t) 1 << 46) | ((uint64_t) 2 << 61);
}
__device__ __forceinline__ constexpr uint32_t many_idesc(int n) {      // D f32, A and B f16, both K-major, N >> 3 at bit 17, M >> 4 at bit 24
    return (1u << 4) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (MANY_TILE >> 4) << 24);
}
// Called by the whole warp, issued by one elected lane: with operands that the warp shares the issue costs a few clocks, inside a branch
// of one lane 60 (128 x 64 x 128 and 128 x 128 x 64 take 514 clk instead of 803).
__device__ __forceinline__ void many_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {      // A in tensor memory
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t) add) : "memory");
}
__device__ __forceinline__ void many_mma_smem(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {      // A in shared memory
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t) add) : "memory");
}
// x, the same in all lanes, as a value that the compiler knows to be so.
__device__ __forceinline__ uint32_t same(uint32_t x) { return __reduce_or_sync(0xFFFFFFFFu, x); }
__device__ __forceinline__ void many_commit(uint32_t bar) {
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_ld32(uint32_t at, uint32_t* v) {      // not waited for
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
                   "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                 : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_wait_ld();
__device__ __forceinline__ void tm_ld16(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
                   "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(at) : "memory");
    tm_wait_ld();
}
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st16(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                   "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tm_ld4(uint32_t at, uint32_t* v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
    tm_wait_ld();
}
__device__ __forceinline__ void tm_st4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }      // the softmax warps of both tiles
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void many_ldsm_trans(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void many_stsm(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 many_lds(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void many_sts(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// A column's query divided by its power of two, as f16 to tensor memory (tq) or, tq = 0, to its row of the shared panels of 64 dims
// (at sq; sx: the row's swizzle); FINE: what that rounding left off, as f16 again, to panels at sl.  -> |scale| log2 e times that
// power, and whether anything was left off.  Out of line, as its registers would be taken from the
// softmax, and in short loops: code that runs once an item is fetched anew each time, and unrolled it took 10 us an item.
struct ManyQuery { float f; bool low; };
template <int HD, bool FINE>
static __device__ __noinline__ ManyQuery many_query(const PagesAttn& a, size_t at, bool valid, uint32_t tq, uint32_t sq, uint32_t sl, uint32_t sx) {
    const bool packed = a.q_type == NSL_BF16;
    float top = 0.0f;
    if (valid) {
        if (packed) {
            uint32_t most = 0;      // magnitudes of bf16 values order as integers
#pragma unroll 1
            for (int d = 0; d < HD; d += 64)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 u = *(const uint4*) ((const uint16_t*) a.q + at + d + 8 * j);
                    most = __vmaxu2(__vmaxu2(most, u.x & 0x7FFF7FFFu), __vmaxu2(u.y & 0x7FFF7FFFu, __vmaxu2(u.z & 0x7FFF7FFFu, u.w & 0x7FFF7FFFu)));
                }
            top = __uint_as_float(max(most << 16, most & 0xFFFF0000u));
        } else {
#pragma unroll 1
            for (int d = 0; d < HD; d += 32)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float4 v = *(const float4*) ((const float*) a.q + at + d + 4 * j);
                    top = max3(max3(top, fabsf(v.x), fabsf(v.y)), fabsf(v.z), fabsf(v.w));
                }
        }
    }
    const float by = pa_pow2_of(top), inv = copysignf(1.0f / by, a.scale);      // the scale's sign goes with the query: maxima are then of scores
    uint32_t low = 0;
#pragma unroll 1
    for (int d = 0; d < HD; d += 32) {
        uint32_t w[16];
        float v[32];
        if (!valid) {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.0f;
        } else if (packed) {
#pragma unroll
            for (int j = 0; j < 4; ++j) load8<NSL_BF16>(a.q, at + d + 8 * j, v + 8 * j);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) load8<NSL_F32>(a.q, at + d + 8 * j, v + 8 * j);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pa_f16x2(v[2 * e] * inv, v[2 * e + 1] * inv);
        __syncwarp();      // lanes with and without a column: the store is the whole warp's
        if (tq) tm_st16(tq + d / 2, w);
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j) many_sts(sq + (d >> 6) * (MANY_TILE * 128) + (((uint32_t) ((d & 63) / 8 + j) ^ sx) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
        if (FINE) {
#pragma unroll
            for (int e = 0; e < 16; ++e) { w[e] = pa_low_f16x2(v[2 * e] * inv, v[2 * e + 1] * inv, w[e]); low |= w[e]; }
#pragma unroll
            for (int j = 0; j < 4; ++j) many_sts(sl + (d >> 6) * (MANY_TILE * 128) + (((uint32_t) ((d & 63) / 8 + j) ^ sx) << 4), w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        }
    }
    if (tq) tm_wait_st();
    if (FINE || !tq) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    ManyQuery r;
    r.f = fabsf(a.scale) * 1.4426950408889634f * by;
    r.low = (low & 0x7FFF7FFFu) != 0;
    return r;
}

// A column's O (and, second: the other tile's, 128 columns on) out of tensor memory, times by and by1: to a state (part: columns side by
// side, as its lanes are), or to the results.  By whole warps.
template <int HD>
static __device__ __noinline__ void many_results(const PagesAttn& a, uint32_t to, bool second, float by, float by1, bool valid, float* part, size_t at) {
#pragma unroll 1
    for (int d = 0; d < HD; d += 16) {
        uint32_t v[16], v1[16];
        __syncwarp();      // lanes with and without a column: the load is the whole warp's
        tm_ld16(to + d, v);
        if (second) tm_ld16(to + 128 + d, v1);
        if (!valid) continue;
        // product row n = 16 j + r: dim 16 j + 2 r, n = 16 j + 8 + r: the next
        float o[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float z = __uint_as_float(v[r]) * by;
            if (second) z = fmaf(__uint_as_float(v1[r]), by1, z);
            o[r < 8 ? 2 * r : 2 * (r - 8) + 1] = z;
        }
        if (part) {
#pragma unroll
            for (int e = 0; e < 16; ++e) part[(d + e) * MANY_COLS] = o[e];
        } else if (a.o_type == NSL_BF16) { store8<NSL_BF16>(a.o, at + d, o); store8<NSL_BF16>(a.o, at + d + 8, o + 8); }
        else { store8<NSL_F32_BF16>(a.o, at + d, o); store8<NSL_F32_BF16>(a.o, at + d + 8, o + 8); }
    }
}

// WIDE: pages of 64 and more positions, a unit's keys have one pair of scales.
template <int HD, bool WIDE, bool FINE>
__global__ void __launch_bounds__(MANY_THREADS, 1) pattn_many_kernel(const __grid_constant__ PagesAttn a, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    using F = Many<HD, FINE>;
    constexpr int RAWS = F::RAWS, STAGES = F::STAGES, STATE = PATTN_STATE<HD>, WARPS = MANY_THREADS / 32, NG = WIDE ? 1 : 4, GK = MANY_KEYS / NG;      // groups of GK keys with one pair of scales
    extern __shared__ uint8_t many_raw[];
    uint8_t* const smem = (uint8_t*) (((uintptr_t) many_raw + 1023) & ~(uintptr_t) 1023);
    __shared__ int wsum[WARPS], plan[2], abort_flag;
    __shared__ uint32_t tmem_slot;
    __shared__ int q_low[MANY_EXPAND];      // FINE, by softmax warp: do its columns' queries have second terms that are not 0
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.n_head / a.p.n_kv;
    const uint32_t base = pa_smem(smem), tiles = base + F::OFF_TILES, bars = base + F::OFF_BARS;
    // arrivals: raw_full the fetch (and bytes), raw_empty the 4 expanding warps, tile_full the same, tile_empty the products, meta the fetch;
    // per tile: s_full and o_done (a unit's scores are there, its values are in O) the products, s_free (the scores are in registers),
    // w_full and q_full the tile's 4 warps; done the warps that issue products
    const uint32_t raw_full = bars, raw_empty = raw_full + 8 * RAWS, tile_full = raw_empty + 8 * RAWS, tile_empty = tile_full + 8 * STAGES, meta_full = tile_empty + 8 * STAGES,
                   s_full = meta_full + 8 * MANY_META, s_free = s_full + 16, w_full = s_free + 16, q_full = w_full + 16, o_done = q_full + 16, done = o_done + 16;
    const float4* const meta = (const float4*) (smem + F::OFF_META);
    if (tid == 0) {
        for (int i = 0; i < RAWS; ++i) { pa_bar_init(raw_full + 8 * i, 1); pa_bar_init(raw_empty + 8 * i, 4); }
        for (int i = 0; i < STAGES; ++i) { pa_bar_init(tile_full + 8 * i, 4); pa_bar_init(tile_empty + 8 * i, 1); }
        for (int i = 0; i < MANY_META; ++i) pa_bar_init(meta_full + 8 * i, 1);
        for (int t = 0; t < 2; ++t) { pa_bar_init(s_full + 8 * t, 1); pa_bar_init(s_free + 8 * t, 4); pa_bar_init(w_full + 8 * t, 4); pa_bar_init(q_full + 8 * t, 4); pa_bar_init(o_done + 8 * t, 1); }
        pa_bar_init(done, 2);
        abort_flag = 0;
        plan[0] = plan[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MANY_SCORES) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pa_smem(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    grid_dependents_go();
    grid_dependency_wait();
    // the step's units and the descriptor that this block's first lies in: a warp a descriptor, a lane a column tile
    int* const of_seq = (int*) (smem + F::OFF_TILES);
    int total = 0;
    for (int i = warp; i < a.n_seqs; i += WARPS) {
        const RowSpan sp = row_span(a, i);
        const int cols = sp.rows * group, nt = (cols + MANY_COLS - 1) / MANY_COLS;
        int n = 0, k0, k1;
        for (int t = lane; t < nt; t += 32) n += many_units(a, sp, group, cols, t, &k0, &k1);
        n = warp_sum(n) * a.p.n_kv;
        if (lane == 0) of_seq[i] = n;
        total += n;
    }
    if (lane == 0) wsum[warp] = total;
    tm_before();
    __syncthreads();
    tm_after();
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += wsum[w];
    const int per = max((total + (int) gridDim.x - 1) / (int) gridDim.x, 1);
    const int x0 = (int) blockIdx.x * per, xe = min(total, x0 + per);
    constexpr uint32_t tmem = 0;      // all 512 columns are the block's
    if (tid == 0) a.rec[blockIdx.x] = make_int4(0, 0, 0, 0);      // (thread 0 writes it again below)
    for (int from = 0, before = 0; from < a.n_seqs; from += MANY_THREADS) {
        const int mine = from + tid < a.n_seqs ? of_seq[from + tid] : 0;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o); if (lane >= o) incl += v; }
        __syncthreads();
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        int start = before + incl - mine, sum = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) { if (w < warp) start += wsum[w]; sum += wsum[w]; }
        if (mine && start <= x0 && x0 < start + mine) { plan[0] = from + tid; plan[1] = start; }
        before += sum;
        if (before > x0) break;
    }
    __syncthreads();
    ManyWalk walk = {plan[0], plan[1]};
    ManyItem it;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) { pa_bar_wait(bar, parity, &abort_flag, &g_pattn_many_status, code, a.wait_ns); };
    int g = 0;      // units this block has done: the rings' position

    if (warp < MANY_EXPAND) {      // ---- softmax: tile t, column c of it ----
        const int t = warp >> 2, c = 32 * (warp & 3) + lane;
        const uint32_t lanes = tmem + ((uint32_t) (32 * (warp & 3)) << 16), ts = lanes + TM_S + 64 * t, tw = lanes + TM_W + 32 * t, to = lanes + TM_O + 128 * t;
        int steps = 0;      // of this tile: phases of its barriers
        for (int x = x0; walk.next(a, group, x, xe, &it); x = it.x1) {
            // up to 128 columns: both tiles have them, and every other unit each
            const int shared = it.cols <= MANY_TILE, n = shared ? (it.x1 - it.x0 + 1 - t) / 2 : it.x1 - it.x0, c0 = shared ? 0 : MANY_TILE * t, col = it.col0 + c0 + c;
            const bool valid = c0 + c < it.cols, warp_valid = c0 + 32 * (warp & 3) < it.cols;
            const int row = it.sp.row + col / group, head = it.kvh * group + col % group, pos = pos_of(it.sp.pos, col / group);
            const int hi = valid ? pos : -1, lo = valid ? first_key(a, pos) : 0;
            float f = 0.0f;      // scale, log2 e and the power of two that the query is divided by
            bool low = false;
            if (warp_valid) {
                const ManyQuery mq = many_query<HD, FINE>(a, (size_t) row * a.q_stride + (size_t) head * HD, valid, t == 0 ? lanes + TM_Q : 0u, base + F::OFF_Q + c * 128, base + F::OFF_QLOW + t * F::QUERIES + c * 128, c & 7);
                f = mq.f;
                low = FINE && mq.low;
            }
            if (FINE) {
                low = __any_sync(0xFFFFFFFFu, low);
                if (lane == 0) q_low[warp] = low;
            }
            tm_before();
            __syncwarp();
            if (lane == 0) pa_bar_arrive(q_full + 8 * t);
            // the first column's position bounds the keys that all may see from above, the last one's from below
            const int all_hi = __shfl_sync(0xFFFFFFFFu, pos, 0);
            const int all_lo = a.window > 0 ? __reduce_max_sync(0xFFFFFFFFu, valid ? lo : -2147483647 - 1) : 0;
            float m = -INFINITY, mo = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j, ++steps) {
                const int u = shared ? 2 * j + t : j, at = g + u;      // the unit; its place in the rings
                wait(s_full + 8 * t, steps & 1, 4);
                wait(meta_full + 8 * (at % MANY_META), at / MANY_META & 1, 5);
                tm_after();
                if (!warp_valid) {      // (the last unit's arrivals are complete once its values are in O)
                    if (lane == 0) pa_bar_arrive(s_free + 8 * t);
                    if (j > 0) wait(o_done + 8 * t, (steps - 1) & 1, 6);
                    if (lane == 0) pa_bar_arrive(w_full + 8 * t);
                    continue;
                }
                uint32_t su[64];
                float* const s = (float*) su;
                tm_ld32(ts, su);
                tm_ld32(ts + 32, su + 32);
                float fg[NG], lv[NG];      // scores = s * fg; log2 of the value scales
                bool whole = true;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const float4 mt = meta[4 * (at % MANY_META) + i];
                    fg[i] = f * mt.x;
                    lv[i] = mt.y;
                    whole = whole && mt.z != 0.0f;
                }
                const int key = (it.tile0 + it.x0 + u - it.first) * MANY_KEYS;
                tm_wait_ld();
                tm_before();
                __syncwarp();
                if (lane == 0) pa_bar_arrive(s_free + 8 * t);
                if (key + MANY_KEYS - 1 > all_hi || key < all_lo || !whole) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const bool there = meta[4 * (at % MANY_META) + i].z != 0.0f;
#pragma unroll
                        for (int e = GK * i; e < GK * i + GK; ++e) s[e] = there && key + e <= hi && key + e >= lo ? s[e] * fg[i] : -INFINITY;
                        fg[i] = 1.0f;
                        if (!there) lv[i] = 0.0f;
                    }
                }
                float mn = -INFINITY, mon = -INFINITY;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    float a0 = max3(s[GK * i], s[GK * i + 1], s[GK * i + 2]), a1 = s[GK * i + 3];
#pragma unroll
                    for (int e = 4; e < GK; e += 4) { a0 = max3(a0, s[GK * i + e], s[GK * i + e + 1]); a1 = max3(a1, s[GK * i + e + 2], s[GK * i + e + 3]); }
                    const float mx = fmaxf(a0, a1) * fg[i];
                    mn = fmaxf(mn, mx);
                    mon = fmaxf(mon, mx + lv[i]);
                }
                if (mn > m + MANY_SLACK || (m == -INFINITY && mn > m)) { l *= pa_ex2(m - mn); m = mn; }
                const bool up = mon > mo + MANY_SLACK || (mo == -INFINITY && mon > mo);
                const bool any_up = __any_sync(0xFFFFFFFFu, up);
                float cor = 1.0f;
                if (up) { cor = pa_ex2(mo - mon); mo = mon; }
                const float ms = m == -INFINITY ? 0.0f : m, mos = mo == -INFINITY ? 0.0f : mo;
                // a weight is p cf, p = 2^(score - m), cf = 2^lc: one exponential of the sum, p's sum from the weights' sum, unless
                // the two lie so far apart that a weight underflows where its p counts
                float lc[NG];
                bool near = true;
#pragma unroll
                for (int i = 0; i < NG; ++i) { lc[i] = lv[i] + (ms - mos); near = near && fabsf(lc[i]) <= 64.0f; }
                uint32_t w[32];
                if (__all_sync(0xFFFFFFFFu, near)) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int i = WIDE ? 0 : 2 * h; i < (WIDE ? 1 : 2 * h + 2); ++i) {
                            const u64 f2 = pack2(fg[i], fg[i]), b2 = pack2(lc[i] - ms, lc[i] - ms);
                            u64 sum = pack2(0.0f, 0.0f);
                            constexpr int PAIRS = WIDE ? 16 : 8;
                            const int e0 = WIDE ? 32 * h : 16 * i;
#pragma unroll
                            for (int e = 0; e < PAIRS; ++e) {
                                float w0, w1;
                                unpack2(fma2(pack2(s[e0 + 2 * e], s[e0 + 2 * e + 1]), f2, b2), w0, w1);
                                w0 = pa_ex2(w0); w1 = pa_ex2(w1);
                                sum = add2(sum, pack2(w0, w1));
                                w[e0 / 2 + e] = pa_f16x2(w0, w1);
                            }
                            float l0, l1;
                            unpack2(sum, l0, l1);
                            l = fmaf(l0 + l1, pa_ex2(-lc[i]), l);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int i = 2 * e / GK;
                        const float cf = pa_ex2(fminf(lc[i], 120.0f));      // finite: a weight whose p is 0 is 0
                        const float p0 = pa_ex2(fmaf(s[2 * e], fg[i], -ms)), p1 = pa_ex2(fmaf(s[2 * e + 1], fg[i], -ms));
                        l += p0 + p1;
                        w[e] = pa_f16x2(p0 * cf, p1 * cf);
                    }
                }
                // the tile's last values are in O, and its last weights have been read
                if (j > 0) {
                    wait(o_done + 8 * t, (steps - 1) & 1, 6);
                    if (any_up) {
                        tm_after();
#pragma unroll 1
                        for (int d = 0; d < HD; d += 16) {
                            uint32_t v[16];
                            tm_ld16(to + d, v);
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * cor);
                            tm_st16(to + d, v);
                        }
                    }
                }
                tm_st16(tw, w);
                tm_st16(tw + 16, w + 16);
                tm_wait_st();
                tm_before();
                __syncwarp();
                if (lane == 0) pa_bar_arrive(w_full + 8 * t);
            }
            if (n > 0) wait(o_done + 8 * t, (steps - 1) & 1, 6);
            // ---- results ----
            const int b0 = it.first / per, parts = (it.first + it.units - 1) / per - b0 + 1;
            float by = 1.0f, by1 = 0.0f;      // what this tile's and the second's O are multiplied with
            if (shared) {      // the second tile's m, l, mo by its weights' columns, whose last have been read, to the warp that has the same lanes
                __syncwarp();
                if (t == 1) tm_st4(tw, __float_as_uint(m), __float_as_uint(l), __float_as_uint(mo), 0u);
                tm_before();
                softmax_sync();
                tm_after();
                if (t == 0) {
                    uint32_t st[4];
                    tm_ld4(tw + 32, st);
                    const float m1 = __uint_as_float(st[0]), mo1 = __uint_as_float(st[2]), mm = fmaxf(m, m1), mmo = fmaxf(mo, mo1);
                    const float ms = mm == -INFINITY ? 0.0f : mm, mos = mmo == -INFINITY ? 0.0f : mmo;
                    l = l * pa_ex2(m - ms) + __uint_as_float(st[1]) * pa_ex2(m1 - ms);
                    by = pa_ex2(mo - mos);
                    by1 = pa_ex2(mo1 - mos);
                    m = mm;
                    mo = mmo;
                }
            }
            if (*(volatile int*) &abort_flag) l = NAN;      // a wait of the block has run out
            if (warp_valid && !(shared && t)) {
                const bool second = shared && it.x1 - it.x0 > 1;      // (an O that nothing was added to holds anything)
                if (parts == 1) { const float fac = pattn_factor(m, l, mo); by *= fac; by1 *= fac; }
                float* const part = a.part + (size_t) (2 * blockIdx.x + ((int) blockIdx.x == b0)) * MANY_COLS * STATE + c0 + c;
                many_results<HD>(a, to, second, by, by1, valid, parts > 1 ? part : NULL, (size_t) row * a.o_stride + (size_t) head * HD);
                if (parts > 1 && valid) { part[HD * MANY_COLS] = m; part[(HD + 1) * MANY_COLS] = l; part[(HD + 2) * MANY_COLS] = mo; }
            }
            if (shared) {      // the second tile's O has been read
                tm_before();
                softmax_sync();
                tm_after();
            }
            if (tid == 0 && parts > 1 && (int) blockIdx.x == b0) a.rec[blockIdx.x] = make_int4(parts | it.kvh << 16, it.sp.row, it.col0, it.cols);
            g += it.x1 - it.x0;
        }
    } else if (warp < MANY_FETCH) {      // ---- expands codes ----
        const int w = warp - MANY_EXPAND, e = tid - 32 * MANY_EXPAND;
        constexpr int CHUNKS = HD / 16;      // of 16 codes a key
        const int chunk = e % CHUNKS, krow = e / CHUNKS;
        const int lrow = (lane & 7) + (lane & 8);
        const uint32_t sw = HD == 128 ? (uint32_t) (lrow & 7) : (uint32_t) (lrow >> 1 & 3);
        const uint32_t v_from = (uint32_t) F::RAW + (uint32_t) (16 * w + lrow) * HD, v_x = (uint32_t) (lane >> 4) ^ sw;
        const int odd = lane >> 4, half = lane >> 3 & 1;
        const uint32_t v_to = (uint32_t) F::TILE + (uint32_t) (8 * odd + (lane & 7)) * 128 + (((uint32_t) (2 * w + half) ^ (uint32_t) (lane & 7)) << 4);
        for (int n = xe - x0; g < n; ++g) {
            const uint32_t rs = (uint32_t) (g % RAWS), st = (uint32_t) (g % STAGES);
            wait(raw_full + 8 * rs, g / RAWS & 1, 7);
            if (g >= STAGES) wait(tile_empty + 8 * st, (g / STAGES - 1) & 1, 8);
            const uint32_t raw = base + rs * 2 * F::RAW, out = tiles + st * 2 * F::TILE;
            // keys: row and chunk of 16 codes a thread -> two 16-byte pieces of the row's f16 values
#pragma unroll
            for (int r0 = 0; r0 < MANY_KEYS; r0 += 128 / CHUNKS) {
                const int r = r0 + krow;
                const uint32_t sx = HD == 128 ? (uint32_t) (r & 7) : (uint32_t) (r >> 1 & 3);
                uint4 x = many_lds(raw + r * HD + (((uint32_t) chunk ^ sx) << 4));
                x.x ^= 0x80808080u; x.y ^= 0x80808080u; x.z ^= 0x80808080u; x.w ^= 0x80808080u;
                const uint32_t y[8] = {pa_codes<0x4140>(x.x), pa_codes<0x4342>(x.x), pa_codes<0x4140>(x.y), pa_codes<0x4342>(x.y),
                                       pa_codes<0x4140>(x.z), pa_codes<0x4342>(x.z), pa_codes<0x4140>(x.w), pa_codes<0x4342>(x.w)};
                const uint32_t row_at = out + (chunk >> 2) * (MANY_KEYS * 128) + r * 128, p0 = ((uint32_t) (2 * chunk & 7) ^ (uint32_t) (r & 7)) << 4;
                if (chunk < 4) {      // (the upper half the other way round: a quarter warp's pieces then lie in different banks)
                    many_sts(row_at + p0, y[0], y[1], y[2], y[3]);
                    many_sts(row_at + (p0 ^ 16), y[4], y[5], y[6], y[7]);
                } else {
                    many_sts(row_at + (p0 ^ 16), y[4], y[5], y[6], y[7]);
                    many_sts(row_at + p0, y[0], y[1], y[2], y[3]);
                }
            }
            // values, transposed: 16 keys a warp, 32 dims a step -> rows of 64 keys
            __syncwarp();      // the two ways round of the keys' pieces: the loads are the whole warp's
#pragma unroll
            for (int j = 0; j < HD / 16; j += 2) {
                uint32_t c[4];
                many_ldsm_trans(c, raw + v_from + ((v_x ^ (uint32_t) j) << 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] ^= 0x80808080u;
                many_stsm(out + v_to + 2048 * j, pa_codes<0x4240>(c[0]), pa_codes<0x4240>(c[1]), pa_codes<0x4341>(c[0]), pa_codes<0x4341>(c[1]));
                many_stsm(out + v_to + 2048 * (j + 1), pa_codes<0x4240>(c[2]), pa_codes<0x4240>(c[3]), pa_codes<0x4341>(c[2]), pa_codes<0x4341>(c[3]));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // for the products' reads
            __syncwarp();
            if (lane == 0) { pa_bar_arrive(tile_full + 8 * st); pa_bar_arrive(raw_empty + 8 * rs); }
        }
    } else if (warp == MANY_FETCH) {      // ---- fetches ----
        asm volatile("fence.proxy.async;" ::: "memory");      // codes that the kernel before has stored
        const int piece = min(a.p.page, MANY_KEYS), pieces = MANY_KEYS / piece, batch = 32 / pieces;
        float4* const meta_to = (float4*) (smem + F::OFF_META);
        for (int x = a.hold ? xe : x0; walk.next(a, group, x, xe, &it); x = it.x1) {
            const size_t head_at = (size_t) a.layer * a.p.n_pages * a.p.n_kv + it.kvh;
            for (int b = it.x0; b < it.x1; b += batch) {
                const int p = (it.tile0 + b - it.first) * MANY_KEYS + lane * piece;      // lane j: piece j from here on
                int id = -1;
                float ks = 0.0f, lv = 0.0f;
                if (b + lane / pieces < it.x1 && p < it.k1 && p + piece > it.k0) id = page_of(a.p, it.sp.seq, p / a.p.page);
                if (id >= 0) {
                    const size_t at = head_at + (size_t) id * a.p.n_kv;
                    ks = a.p.ks[at];
                    lv = log2f(a.p.vs[at]);
                }
                const int row = id < 0 ? -1 : (int) ((head_at + (size_t) id * a.p.n_kv) * a.p.page + p % a.p.page);
                for (int u = 0; u < batch && b + u < it.x1; ++u, ++g) {
                    const uint32_t rs = (uint32_t) (g % RAWS);
                    if (g >= RAWS) wait(raw_empty + 8 * rs, (g / RAWS - 1) & 1, 9);
                    if (__any_sync(0xFFFFFFFFu, *(volatile int*) &abort_flag)) break;      // by all lanes or none
                    const int from = u * pieces + (lane & (pieces - 1)), of_group = u * pieces + (lane & 3) * 16 / piece;
                    const int my_row = __shfl_sync(0xFFFFFFFFu, row, from), g_row = __shfl_sync(0xFFFFFFFFu, row, of_group);
                    const float g_ks = __shfl_sync(0xFFFFFFFFu, ks, of_group), g_lv = __shfl_sync(0xFFFFFFFFu, lv, of_group);
                    if (lane < 4) meta_to[4 * (g % MANY_META) + lane] = make_float4(g_ks, g_lv, g_row >= 0 ? 1.0f : 0.0f, 0.0f);
                    __syncwarp();      // before the arrivals that publish it
                    const uint32_t there = __ballot_sync(0xFFFFFFFFu, lane < pieces && my_row >= 0);
                    if (lane == 0) {
                        pa_bar_arrive(meta_full + 8 * (g % MANY_META));
                        pa_bar_expect(raw_full + 8 * rs, (uint32_t) __popc(there) * 2 * piece * HD);
                    }
                    __syncwarp();
                    if (there >> lane & 1) {
                        const uint32_t to = base + rs * 2 * F::RAW + lane * piece * HD;
                        pa_tma_rows(to, &tk, my_row, raw_full + 8 * rs);
                        pa_tma_rows(to + F::RAW, &tv, my_row, raw_full + 8 * rs);
                    }
                }
            }
        }
        for (int i = 0; i < RAWS; ++i) {      // what is in flight ends before the block does, whatever the others do
            const int filled = g / RAWS + (i < g % RAWS);
            if (filled > 0) for (uint32_t k = 0; k < (1u << 20) && !pa_bar_try(raw_full + 8 * i, (filled - 1) & 1); ++k) {}
        }
    } else {      // ---- issues the products: the scores', or the values' ----
        // everything that an operand is made of comes from constants, counters and values that the warp is known to share (same())
        constexpr uint32_t id_s = many_idesc(MANY_KEYS), id_o = many_idesc(HD);
        const bool scores = warp == MANY_SCORES;
        const uint64_t qd = many_desc(base + F::OFF_Q), qlow = many_desc(base + F::OFF_QLOW), kd0 = many_desc(tiles), vd0 = many_desc(tiles + F::TILE);
        uint32_t items = 0, units = 0, issued[2] = {0, 0};      // of this block so far; of a tile: units
        for (int x = x0; walk.next(a, group, x, xe, &it); x = it.x1, ++items) {
            const uint32_t run = same(it.x1 - it.x0), shared = same(it.cols <= MANY_TILE), n = shared ? run : 2 * run;
            uint32_t low[2] = {0, 0};      // of a tile: its queries have second terms
            if (scores) {
                wait(q_full, items & 1, 10);
                wait(q_full + 8, items & 1, 10);
                tm_after();
                if (FINE) {
                    const uint32_t mine = lane < MANY_EXPAND ? (uint32_t) ((volatile int*) q_low)[lane] << lane : 0u, all = same(mine);
                    low[0] = all & 0xFu;
                    low[1] = all >> 4;
                }
            }
            auto step = [&](auto tile, uint32_t i) {      // of tile i & 1
                constexpr int t = decltype(tile)::value;
                if (i >= n) return;
                const uint32_t at = units + (shared ? i : i >> 1), stage = at % STAGES;
                if (scores) {
                    wait(tile_full + 8 * stage, at / STAGES & 1, 11);
                    if (issued[t] > 0) wait(s_free + 8 * t, (issued[t] - 1) & 1, 12);
                    tm_after();
                    const uint64_t kd = kd0 + (uint64_t) (stage * (2 * F::TILE >> 4));
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint64_t kk = kd + (uint64_t) (((k >> 2) * (MANY_KEYS * 128) + (k & 3) * 32) >> 4);
                        if (t == 0) many_mma(TM_S, TM_Q + 8 * k, kk, id_s, k > 0);
                        else many_mma_smem(TM_S + 64, qd + (uint64_t) (((k >> 2) * (MANY_TILE * 128) + (k & 3) * 32) >> 4), kk, id_s, k > 0);
                    }
                    if (FINE && low[t])
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const uint64_t at_k = (uint64_t) ((t * F::QUERIES + (k >> 2) * (MANY_TILE * 128) + (k & 3) * 32) >> 4);
                            many_mma_smem(TM_S + 64 * t, qlow + at_k, kd + (uint64_t) (((k >> 2) * (MANY_KEYS * 128) + (k & 3) * 32) >> 4), id_s, true);
                        }
                    many_commit(s_full + 8 * t);
                } else {
                    wait(w_full + 8 * t, issued[t] & 1, 13);
                    tm_after();
                    const uint64_t vd = vd0 + (uint64_t) (stage * (2 * F::TILE >> 4));
#pragma unroll
                    for (int k = 0; k < MANY_KEYS / 16; ++k) many_mma(TM_O + 128 * t, TM_W + 32 * t + 8 * k, vd + (uint64_t) (2 * k), id_o, i >= 2 || k > 0);
                    many_commit(o_done + 8 * t);
                    if (shared || t == 1) many_commit(tile_empty + 8 * stage);      // (its keys were read before the weights could be made)
                }
                ++issued[t];
            };
            for (uint32_t i = 0; i < n; i += 2) {
                step(std::integral_constant<int, 0>(), i);
                step(std::integral_constant<int, 1>(), i + 1);
            }
            units += run;
        }
        many_commit(done);      // what has been issued ends before the tensor memory is given back
        __syncwarp();
        for (uint32_t k = 0; k < (1u << 24) && !pa_bar_try(done, 0); ++k) {}
    }
    tm_before();
    __syncthreads();
    __syncwarp();
    tm_after();
    if (warp == MANY_SCORES) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem_slot) : "memory");
}

int pattn_many_status() { return pattn_status_of(g_pattn_many_status); }

// The states of an unfinished item joined.  Block (b, y): the item that block b leaves unfinished, columns 32 y .. 32 y + 31; a lane a
// column, a warp an eighth of the dims, so the states are read as they were written, 128 bytes a warp; the results are turned
// round in shared memory.
constexpr int JOIN_THREADS = 256, JOIN_COLS = 32, JOIN_EACH = 4;
template <int HD>
__global__ void __launch_bounds__(JOIN_THREADS) pattn_join_kernel(const __grid_constant__ PagesAttn a) {
    constexpr int STATE = PATTN_STATE<HD>, DIMS = HD / (JOIN_THREADS / 32);
    __shared__ float turn[JOIN_COLS][HD + 1];
    grid_dependents_go();
    grid_dependency_wait();
    const int4 rec = a.rec[blockIdx.x];
    const int parts = rec.x & 0xFFFF, kvh = rec.x >> 16, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = (int) blockIdx.y * JOIN_COLS, group = a.n_head / a.p.n_kv;
    if (parts == 0 || c0 >= rec.w) return;
    auto state = [&](int i) { return a.part + (size_t) (2 * ((int) blockIdx.x + i) + (i == 0)) * MANY_COLS * STATE + c0 + lane; };      // (columns behind the last: never written, not used)
    float m = -INFINITY, mo = -INFINITY, l = 0.0f, o[DIMS];
#pragma unroll
    for (int e = 0; e < DIMS; ++e) o[e] = 0.0f;
    for (int i0 = 0; i0 < parts; i0 += JOIN_EACH) {      // some states at a time, everything of them requested at once
        float sm[JOIN_EACH], sl[JOIN_EACH], so[JOIN_EACH], v[JOIN_EACH][DIMS];
#pragma unroll
        for (int i = 0; i < JOIN_EACH; ++i) {
            sm[i] = so[i] = -INFINITY;
            sl[i] = 0.0f;
            if (i0 + i >= parts) continue;
            const float* p = state(i0 + i);
            sm[i] = p[HD * MANY_COLS];
            sl[i] = p[(HD + 1) * MANY_COLS];
            so[i] = p[(HD + 2) * MANY_COLS];
#pragma unroll
            for (int e = 0; e < DIMS; ++e) v[i][e] = p[(warp * DIMS + e) * MANY_COLS];
        }
        const float m0 = m, mo0 = mo;
#pragma unroll
        for (int i = 0; i < JOIN_EACH; ++i) { m = fmaxf(m, sm[i]); mo = fmaxf(mo, so[i]); }
        const float ms = m == -INFINITY ? 0.0f : m, mos = mo == -INFINITY ? 0.0f : mo, by = pa_ex2(mo0 - mos);
        l *= pa_ex2(m0 - ms);
#pragma unroll
        for (int e = 0; e < DIMS; ++e) o[e] *= by;
#pragma unroll
        for (int i = 0; i < JOIN_EACH; ++i)
            if (i0 + i < parts) {
                const float w = pa_ex2(so[i] - mos);
                l = fmaf(sl[i], pa_ex2(sm[i] - ms), l);
#pragma unroll
                for (int e = 0; e < DIMS; ++e) o[e] = fmaf(v[i][e], w, o[e]);
            }
    }
    const float f = pattn_factor(m, l, mo);
#pragma unroll
    for (int e = 0; e < DIMS; ++e) turn[lane][warp * DIMS + e] = o[e] * f;
    __syncthreads();
    constexpr int EIGHTS = HD / 8;
    for (int i = threadIdx.x; i < JOIN_COLS * EIGHTS; i += JOIN_THREADS) {
        const int cl = i / EIGHTS, d = 8 * (i % EIGHTS), c = rec.z + c0 + cl;
        if (c0 + cl >= rec.w) break;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = turn[cl][d + e];
        const size_t at = (size_t) (rec.y + c / group) * a.o_stride + (size_t) (kvh * group + c % group) * HD + d;
        if (a.o_type == NSL_BF16) store8<NSL_BF16>(a.o, at, v); else store8<NSL_F32_BF16>(a.o, at, v);
    }
}

template <int HD, bool WIDE, bool FINE>
static void launch_many(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv) {
    const unsigned blocks = (unsigned) sm_count();
    constexpr int SMEM = Many<HD, FINE>::SMEM;
    cudaFuncSetAttribute(pattn_many_kernel<HD, WIDE, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    launch(pattn_many_kernel<HD, WIDE, FINE>, blocks, MANY_THREADS, SMEM, s, a, tk, tv);
    const int cols = (a.n_head / a.p.n_kv) * a.max_rows;
    launch(pattn_join_kernel<HD>, dim3(blocks, (unsigned) (cols < MANY_COLS ? (cols + JOIN_COLS - 1) / JOIN_COLS : MANY_COLS / JOIN_COLS)), JOIN_THREADS, 0, s, a);
    count_launch(2);
}
template <int HD, bool WIDE>
static void launch_many(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv) {
    if (a.q_type == NSL_F32) launch_many<HD, WIDE, true>(s, a, tk, tv);
    else launch_many<HD, WIDE, false>(s, a, tk, tv);
}

void launch_pattn_many(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv) {
    const bool wide = a.p.page >= MANY_KEYS;
    if (a.p.hd == 128) { if (wide) launch_many<128, true>(s, a, tk, tv); else launch_many<128, false>(s, a, tk, tv); }
    else if (wide) launch_many<64, true>(s, a, tk, tv);
    else launch_many<64, false>(s, a, tk, tv);
}

}   // namespace nsl
