// Attention over the paged cache for sequences with many rows (prompts, wide groups, verify steps): the 5th-generation tensor cores.
//
// An item is 256 columns ((row, query head) pairs of a KV head) of a sequence as two tiles of 128; a unit is 64 keys of an item.
// The step's units are dealt evenly to the blocks, one an SM, in order; a run that ends inside an item leaves its state for the
// merge kernel.  Per unit, on both tiles:
//   S [128][64]  = Q [128][hd] . K^T      A = queries (f16, tensor memory), B = keys [64][hd] in shared memory
//   O [128][hd] += W [128][64] . V        A = weights (f16, over S in tensor memory), B = values as [hd][64] in shared memory
// Warps: 4 + 4 take the softmax of the two tiles (a thread a column: its row of S is in its tensor memory lane), 4 expand the
// codes to f16 (exact) into the layout the products read, 1 fetches pages, 1 issues the products.  While one tile's scores are
// in its softmax, the other's products run.  The two scales and the running maxima are as in pages_attn_few.cu; here the maxima
// that the exponents use follow the true ones only when these have grown by 2^8 (weights up to 2^8 then), so O in tensor memory
// is hardly ever rescaled.
// Bound: the exponentials (16 a clock and SM: 128 x 64 x 2 a unit take 1024 clk) and the products (1024 clk) alike.
#include "pages_attn.cuh"
#include "seed_block.cuh"

namespace nsl {

constexpr int MANY_KEYS = 64, MANY_TILE = 128, MANY_COLS = PATTN_MANY, MANY_THREADS = 448, MANY_RAW = 4, MANY_STAGES = 4, MANY_META = 16;
constexpr int MANY_EXPAND = 8, MANY_FETCH = 12, MANY_MMA = 13;      // first warp of each part; the softmax has warps 0 .. 7
constexpr int TM_S = 0, TM_Q = 128, TM_O = 256;                      // tensor memory columns: S (64 a tile; W is its first 32), Q (64 a tile), O (128 a tile)
constexpr float MANY_SLACK = 8.0f;                                   // how far (in powers of 2) a weight may exceed 1

template <int HD>
struct Many {
    static constexpr int RAW = MANY_KEYS * HD;                       // bytes of a unit's key codes, or value codes
    static constexpr int TILE = 2 * RAW;                             // the same as f16
    static constexpr int OFF_TILES = MANY_RAW * 2 * RAW;
    static constexpr int OFF_META = OFF_TILES + MANY_STAGES * 2 * TILE;
    static constexpr int OFF_BARS = OFF_META + MANY_META * 4 * 16;
    static constexpr int BARS = 2 * MANY_RAW + 2 * MANY_STAGES + MANY_META + 9;
    static constexpr int SMEM = OFF_BARS + 8 * BARS + 1024;
};
static_assert(MANY_COLS == 2 * MANY_TILE, "two tiles an item");
constexpr int MANY_SEQS = 4096;      // descriptors of a call; their units sit in the tiles' memory while the plan is made
static_assert(MANY_SEQS * 4 <= MANY_STAGES * 4 * 64 * 64, "the plan's memory");

__device__ int g_pattn_many_status;

struct ManyItem {
    RowSpan sp;
    int kvh, col0, cols;      // the item's columns: col0 .. col0 + cols - 1 of the KV head's
    int k0, k1, tile0, first, units, x0, x1;      // as FewItem
};

// Units of column tile ct.
__device__ __forceinline__ int many_units(const PagesAttn& a, const RowSpan& sp, int group, int cols, int ct, int* k0, int* k1) {
    const int i0 = ct * MANY_COLS / group, i1 = min(cols - 1, ct * MANY_COLS + MANY_COLS - 1) / group;
    *k1 = max(min(sp.pos + i1 + 1, a.p.max_pages * a.p.page), 0);
    *k0 = a.window > 0 ? min(max(sp.pos + i0 - a.window + 1, 0), *k1) : 0;
    return max((*k1 + MANY_KEYS - 1) / MANY_KEYS - *k0 / MANY_KEYS, 1);
}
// Columns of a sequence, 0 for those that pages_attn_few.cu takes.
__device__ __forceinline__ int many_cols(const RowSpan& sp, int group, int few) { return sp.rows * group > few ? sp.rows * group : 0; }
__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// The walk over a block's units, by whole warps.
struct ManyWalk {
    int i, before;
    __device__ bool next(const PagesAttn& a, int group, int few, int x, int xe, ManyItem* it) {
        const int lane = threadIdx.x & 31;
        if (x >= xe) return false;
        for (; i < a.n_seqs; ++i) {
            it->sp = row_span(a, i);
            const int cols = many_cols(it->sp, group, few), tiles = (cols + MANY_COLS - 1) / MANY_COLS;
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
__device__ __forceinline__ void many_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t) add) : "memory");
}
__device__ __forceinline__ void many_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
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
__device__ __forceinline__ void tm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]),
                   "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
                   "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
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

template <int HD>
__global__ void __launch_bounds__(MANY_THREADS, 1) pattn_many_kernel(PagesAttn a, int few, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    using F = Many<HD>;
    constexpr int STATE = PATTN_STATE<HD>, WARPS = MANY_THREADS / 32;
    extern __shared__ uint8_t many_raw[];
    uint8_t* const smem = (uint8_t*) (((uintptr_t) many_raw + 1023) & ~(uintptr_t) 1023);
    __shared__ int wsum[WARPS], plan[2], abort_flag;
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.n_head / a.p.n_kv;
    const uint32_t base = pa_smem(smem), tiles = base + F::OFF_TILES, bars = base + F::OFF_BARS;
    // arrivals: raw_full the fetch (and bytes), raw_empty the 4 expanding warps, tile_full the same, tile_empty the products, meta the
    // fetch; per tile: s_full the products, w_full the tile's 4 warps, q_full the same, o_full the products; done the products
    const uint32_t raw_full = bars, raw_empty = raw_full + 8 * MANY_RAW, tile_full = raw_empty + 8 * MANY_RAW, tile_empty = tile_full + 8 * MANY_STAGES, meta_full = tile_empty + 8 * MANY_STAGES,
                   s_full = meta_full + 8 * MANY_META, w_full = s_full + 16, q_full = w_full + 16, o_full = q_full + 16, done = o_full + 16;
    const float4* const meta = (const float4*) (smem + F::OFF_META);
    if (tid == 0) {
        for (int i = 0; i < MANY_RAW; ++i) { pa_bar_init(raw_full + 8 * i, 1); pa_bar_init(raw_empty + 8 * i, 4); }
        for (int i = 0; i < MANY_STAGES; ++i) { pa_bar_init(tile_full + 8 * i, 4); pa_bar_init(tile_empty + 8 * i, 1); }
        for (int i = 0; i < MANY_META; ++i) pa_bar_init(meta_full + 8 * i, 1);
        for (int t = 0; t < 2; ++t) { pa_bar_init(s_full + 8 * t, 1); pa_bar_init(w_full + 8 * t, 4); pa_bar_init(q_full + 8 * t, 4); pa_bar_init(o_full + 8 * t, 1); }
        pa_bar_init(done, 1);
        abort_flag = 0;
        plan[0] = plan[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MANY_MMA) {
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
        const int cols = many_cols(sp, group, few), nt = (cols + MANY_COLS - 1) / MANY_COLS;
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
    const uint32_t tmem = tmem_slot;
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
    volatile int* const ab = &abort_flag;
    bool ok = true;
    auto fail = [&](int code) { abort_flag = 1; atomicCAS(&g_pattn_many_status, 0, code); ok = false; };
    int g = 0;      // units this block has done: the rings' position

    if (warp < MANY_EXPAND) {      // ---- softmax: tile t, column c of it ----
        const int t = warp >> 2, c = 32 * (warp & 3) + lane;
        const uint32_t lanes = tmem + ((uint32_t) (32 * (warp & 3)) << 16), ts = lanes + TM_S + 64 * t, tq = lanes + TM_Q + 64 * t, to = lanes + TM_O + 128 * t;
        int items = 0, steps = 0;      // of this tile: phases of its barriers
        for (int x = x0; ok && walk.next(a, group, few, x, xe, &it); x = it.x1) {
            const int n = it.x1 - it.x0, col = it.col0 + MANY_TILE * t + c;
            if (it.cols <= MANY_TILE * t) { g += n; continue; }      // the tile is empty
            const bool valid = MANY_TILE * t + c < it.cols, warp_valid = MANY_TILE * t + 32 * (warp & 3) < it.cols;
            const int row = it.sp.row + col / group, head = it.kvh * group + col % group, pos = it.sp.pos + col / group;
            const int hi = valid ? pos : -1, lo = valid && a.window > 0 ? pos - a.window + 1 : 0;
            float f = 0.0f;      // scale, log2 e and the power of two that the query is divided by
            if (warp_valid) {
                // where no key of a unit is masked for any column of the warp
                float top = 0.0f;
                const size_t at = (size_t) row * a.q_stride + (size_t) head * HD;
                if (valid)
#pragma unroll 4
                    for (int d = 0; d < HD; d += 8) {
                        float v[8];
                        if (a.q_type == NSL_BF16) load8<NSL_BF16>(a.q, at + d, v); else load8<NSL_F32>(a.q, at + d, v);
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
                    }
                const float by = pa_pow2_of(top), inv = copysignf(1.0f / by, a.scale);      // the scale's sign goes with the query: maxima are then of scores
                f = fabsf(a.scale) * 1.4426950408889634f * by;
#pragma unroll
                for (int d = 0; d < HD; d += 64) {
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float v[8];
                        if (!valid) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                        } else if (a.q_type == NSL_BF16) load8<NSL_BF16>(a.q, at + d + 8 * j, v);
                        else load8<NSL_F32>(a.q, at + d + 8 * j, v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[4 * j + e] = pa_f16x2(v[2 * e] * inv, v[2 * e + 1] * inv);
                    }
                    tm_st32(tq + d / 2, w);
                }
                tm_wait_st();
            }
            tm_before();
            __syncwarp();
            if (lane == 0) pa_bar_arrive(q_full + 8 * t);
            // the first column's position bounds the keys that all may see from above, the last one's from below
            const int all_hi = __shfl_sync(0xFFFFFFFFu, pos, 0);
            const int all_lo = a.window > 0 ? __reduce_max_sync(0xFFFFFFFFu, valid ? lo : -2147483647 - 1) : 0;
            float m = -INFINITY, mo = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j, ++g, ++steps) {
                if (!pa_bar_wait(s_full + 8 * t, steps & 1, ab) || !pa_bar_wait(meta_full + 8 * (g % MANY_META), g / MANY_META & 1, ab)) { fail(4); break; }
                tm_after();
                if (warp_valid) {
                    uint32_t su[64];
                    float* const s = (float*) su;
                    tm_ld32(ts, su);
                    tm_ld32(ts + 32, su + 32);
                    float4 mt[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) mt[i] = meta[4 * (g % MANY_META) + i];
                    const int key = (it.tile0 + it.x0 + j - it.first) * MANY_KEYS;
                    tm_wait_ld();
                    float fg[4];      // scores = s * fg
#pragma unroll
                    for (int i = 0; i < 4; ++i) fg[i] = f * mt[i].x;
                    if (key + MANY_KEYS - 1 > all_hi || key < all_lo || mt[0].z + mt[1].z + mt[2].z + mt[3].z != 4.0f) {
#pragma unroll
                        for (int i = 0; i < 64; ++i) {
                            const bool seen = key + i <= hi && key + i >= lo && mt[i >> 4].z != 0.0f;
                            s[i] = seen ? s[i] * fg[i >> 4] : -INFINITY;
                        }
                        fg[0] = fg[1] = fg[2] = fg[3] = 1.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) if (mt[i].z == 0.0f) mt[i].y = 0.0f;
                    }
                    float mx[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mx[i] = s[16 * i];
#pragma unroll
                        for (int e = 1; e < 16; ++e) mx[i] = fmaxf(mx[i], s[16 * i + e]);
                        mx[i] *= fg[i];
                    }
                    const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), mon = fmaxf(fmaxf(mx[0] + mt[0].y, mx[1] + mt[1].y), fmaxf(mx[2] + mt[2].y, mx[3] + mt[3].y));
                    if (mn > m + MANY_SLACK || (m == -INFINITY && mn > m)) { l *= pa_ex2(m - mn); m = mn; }
                    const bool up = mon > mo + MANY_SLACK || (mo == -INFINITY && mon > mo);
                    if (__any_sync(0xFFFFFFFFu, up)) {
                        const float cor = up ? pa_ex2(mo - mon) : 1.0f;
                        if (up) mo = mon;
                        if (j > 0)      // (the product before this unit's has ended: its scores came behind it)
#pragma unroll 1
                            for (int d = 0; d < HD; d += 32) {
                                uint32_t v[32];
                                tm_ld32(to + d, v);
                                tm_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * cor);
                                tm_st32(to + d, v);
                            }
                    }
                    const float ms = m == -INFINITY ? 0.0f : m, mos = mo == -INFINITY ? 0.0f : mo;
                    uint32_t w[32];
                    u64 sum = pack2(0.0f, 0.0f);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float cf = pa_ex2(fminf(mt[i].y + (ms - mos), 120.0f));      // weight = p cf (finite: a weight whose p is 0 is 0)
                        const u64 f2 = pack2(fg[i], fg[i]), m2 = pack2(-ms, -ms), c2 = pack2(cf, cf);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            float p0, p1;
                            unpack2(fma2(pack2(s[16 * i + 2 * e], s[16 * i + 2 * e + 1]), f2, m2), p0, p1);
                            const u64 p = pack2(pa_ex2(p0), pa_ex2(p1));
                            sum = add2(sum, p);
                            float w0, w1;
                            unpack2(mul2(p, c2), w0, w1);
                            w[8 * i + e] = pa_f16x2(w0, w1);
                        }
                    }
                    float l0, l1;
                    unpack2(sum, l0, l1);
                    l += l0 + l1;
                    tm_st32(ts, w);
                    tm_wait_st();
                }
                tm_before();
                __syncwarp();
                if (lane == 0) pa_bar_arrive(w_full + 8 * t);
            }
            if (!ok) break;
            // ---- results ----
            if (!pa_bar_wait(o_full + 8 * t, items & 1, ab)) { fail(5); break; }
            ++items;
            tm_after();
            const int b0 = it.first / per, parts = (it.first + it.units - 1) / per - b0 + 1;
            if (warp_valid) {
                const float by = parts == 1 ? pattn_factor(m, l, mo) : 1.0f;
                float* const part = a.part + ((size_t) (2 * blockIdx.x + ((int) blockIdx.x == b0)) * MANY_COLS + MANY_TILE * t + c) * STATE;
                const size_t at = (size_t) row * a.o_stride + (size_t) head * HD;
#pragma unroll 1
                for (int d = 0; d < HD; d += 32) {
                    uint32_t v[32];
                    tm_ld32(to + d, v);
                    tm_wait_ld();
                    if (!valid) continue;
                    // product row n = 16 j + r: dim 16 j + 2 r, n = 16 j + 8 + r: the next
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float o[16];
#pragma unroll
                        for (int r = 0; r < 8; ++r) { o[2 * r] = __uint_as_float(v[16 * j + r]) * by; o[2 * r + 1] = __uint_as_float(v[16 * j + 8 + r]) * by; }
                        if (parts > 1) { store8<NSL_F32>(part, d + 16 * j, o); store8<NSL_F32>(part, d + 16 * j + 8, o + 8); }
                        else if (a.o_type == NSL_BF16) { store8<NSL_BF16>(a.o, at + d + 16 * j, o); store8<NSL_BF16>(a.o, at + d + 16 * j + 8, o + 8); }
                        else { store8<NSL_F32_BF16>(a.o, at + d + 16 * j, o); store8<NSL_F32_BF16>(a.o, at + d + 16 * j + 8, o + 8); }
                    }
                }
                if (parts > 1 && valid) *(float4*) (part + HD) = make_float4(m, l, mo, 0.0f);
            }
            if (tid == 0 && parts > 1 && (int) blockIdx.x == b0) a.rec[blockIdx.x] = make_int4(parts | it.kvh << 16, it.sp.row, it.col0, it.cols);
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
        for (int n = xe - x0; ok && g < n; ++g) {
            const uint32_t rs = (uint32_t) (g % MANY_RAW), st = (uint32_t) (g % MANY_STAGES);
            if (!pa_bar_wait(raw_full + 8 * rs, g / MANY_RAW & 1, ab) || (g >= MANY_STAGES && !pa_bar_wait(tile_empty + 8 * st, (g / MANY_STAGES - 1) & 1, ab))) { fail(6); break; }
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
        for (int x = x0; ok && walk.next(a, group, few, x, xe, &it); x = it.x1) {
            const size_t head_at = (size_t) a.layer * a.p.n_pages * a.p.n_kv + it.kvh;
            for (int b = it.x0; ok && b < it.x1; b += batch) {
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
                    const uint32_t rs = (uint32_t) (g % MANY_RAW);
                    if (g >= MANY_RAW && !pa_bar_wait(raw_empty + 8 * rs, (g / MANY_RAW - 1) & 1, ab)) { fail(7); break; }
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
        if (!ok)      // what is in flight ends before the block does
            for (int i = 0; i < MANY_RAW; ++i) {
                const int filled = g / MANY_RAW + (i < g % MANY_RAW);
                if (filled > 0) for (uint32_t k = 0; k < (1u << 20) && !pa_bar_try(raw_full + 8 * i, (filled - 1) & 1); ++k) {}
            }
    } else {      // ---- issues the products ----
        const uint32_t id_s = many_idesc(MANY_KEYS), id_o = many_idesc(HD);
        int items[2] = {0, 0}, steps[2] = {0, 0};
        auto scores = [&](int t, int stage) {
            const uint64_t kd = many_desc(tiles + stage * 2 * F::TILE);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) many_mma(tmem + TM_S + 64 * t, tmem + TM_Q + 64 * t + 8 * k, kd + (uint64_t) (((k >> 2) * (MANY_KEYS * 128) + (k & 3) * 32) >> 4), id_s, k > 0);
            many_commit(s_full + 8 * t);
        };
        for (int x = x0; ok && walk.next(a, group, few, x, xe, &it); x = it.x1) {
            const int n = it.x1 - it.x0, both = it.cols > MANY_TILE ? 2 : 1;
            for (int t = 0; t < both; ++t)
                if (!pa_bar_wait(q_full + 8 * t, items[t]++ & 1, ab)) { fail(8); break; }
            for (int j = -1; ok && j < n; ++j) {      // unit j's values, unit j + 1's scores
                for (int t = 0; t < both; ++t) {
                    if (j >= 0) {
                        if (!pa_bar_wait(w_full + 8 * t, steps[t]++ & 1, ab)) { fail(9); break; }
                        tm_after();
                        if (lane == 0) {
                            const int stage = (g + j) % MANY_STAGES;
                            const uint64_t vd = many_desc(tiles + stage * 2 * F::TILE + F::TILE);
#pragma unroll
                            for (int k = 0; k < MANY_KEYS / 16; ++k) many_mma(tmem + TM_O + 128 * t, tmem + TM_S + 64 * t + 8 * k, vd + (uint64_t) (2 * k), id_o, j > 0 || k > 0);
                            if (j == n - 1) many_commit(o_full + 8 * t);
                            if (t == both - 1) many_commit(tile_empty + 8 * stage);
                        }
                    }
                    if (j + 1 < n) {
                        const int next = g + j + 1;
                        if (t == 0 && !pa_bar_wait(tile_full + 8 * (next % MANY_STAGES), next / MANY_STAGES & 1, ab)) { fail(10); break; }
                        tm_after();
                        if (lane == 0) scores(t, next % MANY_STAGES);
                    }
                    __syncwarp();
                }
            }
            g += n;
        }
        if (lane == 0) many_commit(done);      // what has been issued ends before the tensor memory is given back
        __syncwarp();
        for (uint32_t k = 0; k < (1u << 24) && !pa_bar_try(done, 0); ++k) {}
    }
    tm_before();
    __syncthreads();
    tm_after();
    if (warp == MANY_MMA) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

int pattn_many_status() {
    int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_pattn_many_status, sizeof v);
    if (v) cudaMemcpyToSymbol(g_pattn_many_status, &zero, sizeof zero);
    return v;
}

// Sequences of more than `few` columns.
void launch_pattn_many(cudaStream_t s, const PagesAttn& a, int few, const CUtensorMap& tk, const CUtensorMap& tv) {
    const unsigned blocks = (unsigned) sm_count();
    if (a.p.hd == 128) {
        cudaFuncSetAttribute(pattn_many_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<128>::SMEM);
        launch(pattn_many_kernel<128>, blocks, MANY_THREADS, Many<128>::SMEM, s, a, few, tk, tv);
    } else {
        cudaFuncSetAttribute(pattn_many_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Many<64>::SMEM);
        launch(pattn_many_kernel<64>, blocks, MANY_THREADS, Many<64>::SMEM, s, a, few, tk, tv);
    }
    launch_pattn_merge(s, a, (int) blocks, MANY_COLS);
    count_launch(2);
}

}   // namespace nsl
