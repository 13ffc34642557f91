// Attention over the paged cache for sequences with few rows (decode, verify): at most 8 columns, a column being one (row, query
// head) of a KV head.
//
// Bound: HBM, 2 hd + 8 / page bytes a key and KV head (8 x 16001 keys, 8 KV heads over pages of 16: 42 us = 4.0 TB/s; 32 x 4096, 2 KV
// heads: 21.4 us = 2.4 TB/s, 6.1 between a block's first and last codes).  The step's keys are cut into units of 64 of one (sequence, KV head) and
// dealt evenly to the blocks in order, so a block's units are a few runs of whole pages whatever the lengths.  One warp of a
// block fetches: page ids and scales 32 pieces ahead, codes by TMA (a piece = a page, or 64 rows of a larger one, swizzled) into
// a ring.  Four warps compute, 16 keys of the unit each, on the tensor cores with the codes as they are:
//   S^T [16 keys][8 columns]     = K [16 keys][hd] . Q^T       A = codes by ldmatrix (a lane's 4 bytes are 4 dims of a key)
//   O^T [16 dims][8 columns]    += V^T [dims][16 keys] . W^T   A = codes by ldmatrix.trans (2 dims of 2 keys)
// Queries of f32 calls whose rounding to f16 leaves something off take part with that as a second f16 term, by the same code fragments.
// A code becomes f16 by a byte permutation and a subtraction (exact); a page's key scale multiplies the scores, its value
// scale is part of the weights' exponent: w = 2^(s + log2 vs - mo), mo the running maximum of that sum, beside the softmax's own
// p = 2^(s - m) whose sum is l.  Weights then never exceed 1 however the pages' scales differ, and 11 bits of f16 are 11
// bits of each weight.  result = O 2^(mo - m) / l.
// A run that ends inside an item (sequence, KV head) leaves its state in the work memory; the merge kernel (pages_attn.cu), a
// dependent launch, joins an item's states in the order of the keys.
#include <type_traits>

#include "pages_attn.cuh"

namespace nsl {

constexpr int FEW_KEYS = 64, FEW_WARPS = 4, FEW_THREADS = 32 * (FEW_WARPS + 1);

template <int HD>
struct Few {
    static constexpr int CT = PATTN_FEW;                 // columns
    static constexpr int TILE = FEW_KEYS * HD;           // bytes of a unit's keys, or values
    static constexpr int STAGES = HD == 128 ? 5 : 9;
    static constexpr int STATE = PATTN_STATE<HD>;        // floats of a column's partial state: O, then m, l, mo
    static constexpr int OFF_META = STAGES * 2 * TILE;   // per stage and 16 keys: key scale, log2 of the value scale, 0 / 1
    static constexpr int OFF_MERGE = OFF_META + STAGES * 4 * 16;
    static constexpr int OFF_BARS = OFF_MERGE + FEW_WARPS * CT * STATE * 4;
    static constexpr int SMEM = OFF_BARS + 2 * STAGES * 8 + 1024;      // + what aligns the ring to 1024
};

struct FewItem {      // a (sequence, KV head) and the units of it that a block has
    RowSpan sp;
    int kvh, k0, k1;      // keys that any row attends
    int tile0;            // the item's first unit, in tiles of 64 positions
    int first, units;     // its units' numbers in the step: first .. first + units - 1
    int x0, x1;           // the block's
};

// Keys [k0, k1) that the rows of a descriptor attend, and its number of units per KV head (one at least: a row that attends
// nothing is written too; 0 for descriptors without rows or with more columns than a tile holds).
__device__ __forceinline__ int few_units(const PagesAttn& a, const RowSpan& sp, int group, int* k0, int* k1) {
    *k0 = *k1 = 0;
    if (sp.rows <= 0 || sp.rows * group > PATTN_FEW) return 0;
    *k1 = end_key(a, pos_of(sp.pos, sp.rows - 1));
    *k0 = min(first_key(a, sp.pos), *k1);
    return max((*k1 + FEW_KEYS - 1) / FEW_KEYS - *k0 / FEW_KEYS, 1);
}

// The walk over a block's units: next() gives the item that unit x lies in.  Every warp keeps its own.
struct FewWalk {
    int i, before;      // descriptor, units of the step before it
    __device__ bool next(const PagesAttn& a, int group, int x, int xe, FewItem* it) {
        if (x >= xe) return false;
        for (; i < a.n_seqs; ++i) {
            it->sp = row_span(a, i);
            const int n = few_units(a, it->sp, group, &it->k0, &it->k1);
            if (x < before + n * a.p.n_kv) {
                it->kvh = (x - before) / n;
                it->first = before + it->kvh * n;
                it->units = n;
                it->tile0 = it->k0 / FEW_KEYS;
                it->x0 = x;
                it->x1 = min(xe, it->first + n);
                return true;
            }
            before += n * a.p.n_kv;
        }
        return false;
    }
};

__device__ int g_pattn_status;      // 0, or the code of the first bounded wait that ran out

__device__ __forceinline__ void few_mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void few_ldsm(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void few_ldsm_trans(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t few_turn(uint32_t x) {      // an 8 x 8 tile of 16-bit values, transposed across the warp
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ void few_sync() {      // the computing warps; the barrier is each whole warp's, and is reached from branches of single lanes
    __syncwarp();
    asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory");
}

// Column c's weights of the warps' states: cw[w * CT + c] = 2^(mo_w - mo); and m, l, mo of all.
template <int HD, int CT>
__device__ __forceinline__ void few_weights(const float* p, int c, float* cw, float* of_all) {
    constexpr int STATE = PATTN_STATE<HD>;
    float m = -INFINITY, mo = -INFINITY, l = 0.0f;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; ++w) { const float* st = p + (w * CT + c) * STATE + HD; m = fmaxf(m, st[0]); mo = fmaxf(mo, st[2]); }
    const float ms = m == -INFINITY ? 0.0f : m, mos = mo == -INFINITY ? 0.0f : mo;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; ++w) {
        const float* st = p + (w * CT + c) * STATE + HD;
        l = fmaf(st[1], pa_ex2(st[0] - ms), l);
        cw[w * CT + c] = pa_ex2(st[2] - mos);
    }
    of_all[3 * c] = m; of_all[3 * c + 1] = l; of_all[3 * c + 2] = mo;
}

// FINE: f32 calls, whose queries may have second terms.
template <int HD, bool FINE>
__global__ void __launch_bounds__(FEW_THREADS, 2) pattn_few_kernel(PagesAttn a, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    using F = Few<HD>;
    constexpr int CT = F::CT, STATE = F::STATE, STEPS = HD / 16;
    extern __shared__ uint8_t few_raw[];
    uint8_t* const smem = (uint8_t*) (((uintptr_t) few_raw + 1023) & ~(uintptr_t) 1023);
    __shared__ int wsum[FEW_THREADS / 32], plan[2];
    __shared__ int abort_flag;
    __shared__ float state_s[3 * CT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = a.n_head / a.p.n_kv;
    const uint32_t ring = pa_smem(smem), full = ring + F::OFF_BARS, empty = full + 8 * F::STAGES;
    float4* const meta = (float4*) (smem + F::OFF_META);
    if (tid == 0) {
        for (int i = 0; i < F::STAGES; ++i) { pa_bar_init(full + 8 * i, 1); pa_bar_init(empty + 8 * i, FEW_WARPS); }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    grid_dependents_go();
    pattn_warm(a);
    grid_dependency_wait();
    // the step's units, and the descriptor that this block's first lies in: from one load of the descriptors where there is a thread for each
    if (tid == 0) { plan[0] = 0; plan[1] = 0; }
    int total = 0, per = 0, x0 = 0, xe = 0, k0, k1;
    const bool once = a.n_seqs <= FEW_THREADS;
    if (!once) {
        for (int i = tid; i < a.n_seqs; i += FEW_THREADS) total += few_units(a, row_span(a, i), group, &k0, &k1) * a.p.n_kv;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        if (lane == 0) wsum[warp] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < FEW_THREADS / 32; ++w) total += wsum[w];
    }
    for (int base = 0, before = 0; base < a.n_seqs; base += FEW_THREADS) {
        const int i = base + tid, mine = i < a.n_seqs ? few_units(a, row_span(a, i), group, &k0, &k1) * a.p.n_kv : 0;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xFFFFFFFFu, incl, o); if (lane >= o) incl += v; }
        __syncthreads();
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        int start = before + incl - mine, sum = 0;
#pragma unroll
        for (int w = 0; w < FEW_THREADS / 32; ++w) { if (w < warp) start += wsum[w]; sum += wsum[w]; }
        if (once) total = sum;
        per = max((total + (int) gridDim.x - 1) / (int) gridDim.x, 1);
        x0 = (int) blockIdx.x * per;
        xe = min(total, x0 + per);
        if (mine && start <= x0 && x0 < start + mine) { plan[0] = i; plan[1] = start; }
        before += sum;
        if (before > x0) break;
    }
    if (tid == 0) a.rec[blockIdx.x] = make_int4(0, 0, 0, 0);      // (thread 0 writes it again below)
    __syncthreads();
    if (x0 >= xe) return;
    FewWalk walk = {plan[0], plan[1]};
    FewItem it;
    int stage = 0, round = 0;      // the ring's next stage, and how often it has been round
    auto wait = [&](uint32_t bar, uint32_t parity, int code) { pa_bar_wait(bar, parity, &abort_flag, &g_pattn_status, code, a.wait_ns); };
    const int piece = min(a.p.page, FEW_KEYS), pieces = FEW_KEYS / piece;      // rows of a piece, pieces of a unit

    if (warp == FEW_WARPS) {      // ---- fetches ----
        asm volatile("fence.proxy.async;" ::: "memory");      // codes that the kernel before has stored
        const int batch = 32 / pieces;      // units a look ahead covers
        int x = a.hold ? xe : x0;
        while (walk.next(a, group, x, xe, &it)) {
            const size_t head_at = (size_t) a.layer * a.p.n_pages * a.p.n_kv + it.kvh;
            for (int b = it.x0; b < it.x1; b += batch) {
                // lane j: piece j from position p on
                const int p = (it.tile0 + b - it.first) * FEW_KEYS + lane * piece;
                int id = -1;
                float ks = 0.0f, lv = 0.0f;
                if (b + lane / pieces < it.x1 && p < it.k1 && p + piece > it.k0) id = page_of(a.p, it.sp.seq, p / a.p.page);
                if (id >= 0) {
                    const size_t at = head_at + (size_t) id * a.p.n_kv;
                    ks = a.p.ks[at];
                    lv = log2f(a.p.vs[at]);
                }
                const int row = id < 0 ? -1 : (int) ((head_at + (size_t) id * a.p.n_kv) * a.p.page + p % a.p.page);
                for (int u = 0; u < batch && b + u < it.x1; ++u) {
                    if (round > 0) wait(empty + 8 * stage, (round - 1) & 1, 1);
                    if (__any_sync(0xFFFFFFFFu, *(volatile int*) &abort_flag)) break;      // by all lanes or none
                    const int from = u * pieces + (lane & (pieces - 1)), of_group = u * pieces + (lane & 3) * 16 / piece;
                    const int my_row = __shfl_sync(0xFFFFFFFFu, row, from), g_row = __shfl_sync(0xFFFFFFFFu, row, of_group);
                    const float g_ks = __shfl_sync(0xFFFFFFFFu, ks, of_group), g_lv = __shfl_sync(0xFFFFFFFFu, lv, of_group);
                    if (lane < 4) meta[4 * stage + lane] = make_float4(g_ks, g_lv, g_row >= 0 ? 1.0f : 0.0f, 0.0f);
                    __syncwarp();      // before the arrival that publishes it
                    const uint32_t there = __ballot_sync(0xFFFFFFFFu, lane < pieces && my_row >= 0);
                    if (lane == 0) pa_bar_expect(full + 8 * stage, (uint32_t) __popc(there) * 2 * piece * HD);
                    __syncwarp();
                    if (there >> lane & 1) {
                        const uint32_t to = ring + stage * 2 * F::TILE + lane * piece * HD;
                        pa_tma_rows(to, &tk, my_row, full + 8 * stage);
                        pa_tma_rows(to + F::TILE, &tv, my_row, full + 8 * stage);
                    }
                    if (++stage == F::STAGES) { stage = 0; ++round; }
                }
            }
            x = it.x1;
        }
        for (int i = 0; i < F::STAGES; ++i) {      // what is in flight ends before the block does, whatever the others do
            const int filled = round + (i < stage);      // fills of stage i
            if (filled > 0) for (uint32_t k = 0; k < (1u << 20) && !pa_bar_try(full + 8 * i, (filled - 1) & 1); ++k) {}
        }
        return;
    }

    // ---- computes ----
    const int q4 = lane & 3, r0 = lane >> 2;
    const int lrow = (lane & 7) + (lane & 8);      // the key row whose 16 bytes this lane names in an ldmatrix
    const uint32_t sw = HD == 128 ? (uint32_t) (lrow & 7) : (uint32_t) (lrow >> 1 & 3);
    const uint32_t l_at = (uint32_t) (16 * warp + lrow) * HD, l_x = (uint32_t) (lane >> 4) ^ sw;
    float* const merge = (float*) (smem + F::OFF_MERGE);
    int x = x0;
    while (walk.next(a, group, x, xe, &it)) {
        const int cols = it.sp.rows * group;
        // the queries as B fragments: column r0 of a tile, dims 16 j + 4 q4 ..; a column divided by its power of two
        uint32_t qb[STEPS][2], ql[STEPS][2], some = 0;      // ql: what the rounding to f16 left off, as f16 again; low: any of it is not 0
        float f[2];      // of the lane's columns 2 q4, 2 q4 + 1: scale, log2 e and the power of two
        int hi[2], lo[2];
        const int c = r0;
        float v[STEPS][4], top = 0.0f;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            const size_t at = (size_t) (it.sp.row + c / group) * a.q_stride + (size_t) (it.kvh * group + c % group) * HD + 16 * j + 4 * q4;
            if (c >= cols) v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.0f;
            else if (a.q_type == NSL_BF16) {
                const uint2 u = *(const uint2*) ((const uint16_t*) a.q + at);
                v[j][0] = __uint_as_float(u.x << 16); v[j][1] = __uint_as_float(u.x & 0xFFFF0000u); v[j][2] = __uint_as_float(u.y << 16); v[j][3] = __uint_as_float(u.y & 0xFFFF0000u);
            } else {
                const float4 u = *(const float4*) ((const float*) a.q + at);
                v[j][0] = u.x; v[j][1] = u.y; v[j][2] = u.z; v[j][3] = u.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[j][e]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const float by = pa_pow2_of(top), inv = copysignf(1.0f / by, a.scale), fc = fabsf(a.scale) * 1.4426950408889634f * by;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            qb[j][0] = pa_f16x2(v[j][0] * inv, v[j][1] * inv);
            qb[j][1] = pa_f16x2(v[j][2] * inv, v[j][3] * inv);
            if (FINE) {
                ql[j][0] = pa_low_f16x2(v[j][0] * inv, v[j][1] * inv, qb[j][0]);
                ql[j][1] = pa_low_f16x2(v[j][2] * inv, v[j][3] * inv, qb[j][1]);
                some |= ql[j][0] | ql[j][1];
            }
        }
        const bool low = FINE && __any_sync(0xFFFFFFFFu, (some & 0x7FFF7FFFu) != 0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            f[e] = __shfl_sync(0xFFFFFFFFu, fc, 4 * (2 * q4 + e));
            const int cc = 2 * q4 + e, pos = pos_of(it.sp.pos, cc / group);
            hi[e] = cc < cols ? pos : -1;
            lo[e] = first_key(a, pos);
        }
        float m[2], mo[2], l[2], ot[STEPS][4];
        m[0] = m[1] = mo[0] = mo[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) ot[i][0] = ot[i][1] = ot[i][2] = ot[i][3] = 0.0f;
        // the item's units; LOW: with the second terms (a loop of its own: a branch in one loop for both cost the calls without them 4 %)
        auto attend = [&](auto with_low) {
            constexpr bool LOW = decltype(with_low)::value;
            for (x = it.x0; x < it.x1; ++x) {
                wait(full + 8 * stage, round & 1, 2);
                const float4 mt = meta[4 * stage + warp];
                const int key = (it.tile0 + x - it.first) * FEW_KEYS + 16 * warp;
                if (mt.z != 0.0f && key < it.k1 && key + 16 > it.k0) {
                    const uint32_t kt = ring + stage * 2 * F::TILE + l_at;
                    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s2[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // two chains
#pragma unroll
                    for (int j = 0; j < STEPS; j += 2) {
                        uint32_t c[4];
                        few_ldsm(c, kt + ((l_x ^ (uint32_t) j) << 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] ^= 0x80808080u;
                        const uint32_t a0[4] = {pa_codes<0x4140>(c[0]), pa_codes<0x4140>(c[1]), pa_codes<0x4342>(c[0]), pa_codes<0x4342>(c[1])};
                        const uint32_t a1[4] = {pa_codes<0x4140>(c[2]), pa_codes<0x4140>(c[3]), pa_codes<0x4342>(c[2]), pa_codes<0x4342>(c[3])};
                        few_mma(s, a0, qb[j]);
                        few_mma(s2, a1, qb[j + 1]);
                        if (LOW) { few_mma(s, a0, ql[j]); few_mma(s2, a1, ql[j + 1]); }
                    }
                    uint32_t pw[2];
                    float mx[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {      // keys key + r0 and key + r0 + 8 of column 2 q4 + e
                        const float fk = f[e] * mt.x;
                        const int ka = key + r0, kb = ka + 8;
                        s[e] = ka <= hi[e] && ka >= lo[e] ? (s[e] + s2[e]) * fk : -INFINITY;
                        s[2 + e] = kb <= hi[e] && kb >= lo[e] ? (s[2 + e] + s2[2 + e]) * fk : -INFINITY;
                        mx[e] = fmaxf(s[e], s[2 + e]);
                    }
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xFFFFFFFFu, mx[0], o));
                        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xFFFFFFFFu, mx[1], o));
                    }
                    float cor[2], w[4];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float mn = fmaxf(m[e], mx[e]), ms = mn == -INFINITY ? 0.0f : mn;
                        const float mon = fmaxf(mo[e], mx[e] + mt.y), mos = mon == -INFINITY ? 0.0f : mon;
                        l[e] = fmaf(l[e], pa_ex2(m[e] - ms), pa_ex2(s[e] - ms) + pa_ex2(s[2 + e] - ms));
                        cor[e] = pa_ex2(mo[e] - mos);
                        w[e] = s[e] == -INFINITY ? 0.0f : pa_ex2(s[e] + (mt.y - mos));      // (an infinite scale counts for those who attend its page)
                        w[2 + e] = s[2 + e] == -INFINITY ? 0.0f : pa_ex2(s[2 + e] + (mt.y - mos));
                        m[e] = mn;
                        mo[e] = mon;
                    }
                    if (cor[0] != 1.0f || cor[1] != 1.0f) {      // the running maxima rarely move after a run's first steps
#pragma unroll
                        for (int i = 0; i < STEPS; ++i) { ot[i][0] *= cor[0]; ot[i][1] *= cor[1]; ot[i][2] *= cor[0]; ot[i][3] *= cor[1]; }
                    }
                    __syncwarp();      // lanes that had a maximum move and lanes that had none: what follows is the whole warp's
                    pw[0] = few_turn(pa_f16x2(w[0], w[1]));
                    pw[1] = few_turn(pa_f16x2(w[2], w[3]));
#pragma unroll
                    for (int j = 0; j < STEPS; j += 2) {
                        uint32_t c[4];
                        few_ldsm_trans(c, kt + F::TILE + ((l_x ^ (uint32_t) j) << 4));
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[e] ^= 0x80808080u;
                        // row r0 of value tile j: dim 16 j + 2 r0, row r0 + 8: the next
                        const uint32_t a0[4] = {pa_codes<0x4240>(c[0]), pa_codes<0x4341>(c[0]), pa_codes<0x4240>(c[1]), pa_codes<0x4341>(c[1])};
                        const uint32_t a1[4] = {pa_codes<0x4240>(c[2]), pa_codes<0x4341>(c[2]), pa_codes<0x4240>(c[3]), pa_codes<0x4341>(c[3])};
                        few_mma(ot[j], a0, pw);
                        few_mma(ot[j + 1], a1, pw);
                    }
                }
                __syncwarp();      // the stage has been read by all lanes
                if (lane == 0) pa_bar_arrive(empty + 8 * stage);
                if (++stage == F::STAGES) { stage = 0; ++round; }
            }
        };
        if (FINE && low) attend(std::integral_constant<bool, FINE>());
        else attend(std::false_type());
        // the warps' states side by side, merged into the block's
        few_sync();      // the last item's states have been read
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], o);
            float* st = merge + (size_t) (warp * CT + 2 * q4 + e) * STATE;
#pragma unroll
            for (int i = 0; i < STEPS; ++i) *(float2*) (st + 16 * i + 2 * r0) = make_float2(ot[i][e], ot[i][2 + e]);
            if (r0 == 0) { st[HD] = m[e]; st[HD + 1] = l[e]; st[HD + 2] = mo[e]; }
        }
        __shared__ float cw_s[FEW_WARPS * CT];
        few_sync();
        if (tid < CT) {
            few_weights<HD, CT>(merge, tid, cw_s, state_s);
            if (*(volatile int*) &abort_flag) state_s[3 * tid + 1] = NAN;      // a wait of the block has run out
        }
        few_sync();
        const int b0 = it.first / per, b1 = (it.first + it.units - 1) / per, parts = b1 - b0 + 1;
        float* const mine = a.part + (size_t) (2 * blockIdx.x + ((int) blockIdx.x == b0)) * CT * STATE;
        for (int i = tid; i < cols * HD; i += 32 * FEW_WARPS) {
            const int c = i / HD, d = i % HD;
            float o = 0.0f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; ++w) o = fmaf(merge[(size_t) (w * CT + c) * STATE + d], cw_s[w * CT + c], o);
            if (parts == 1) {
                store_bf16_of(a, (size_t) (it.sp.row + c / group) * a.o_stride + (size_t) (it.kvh * group + c % group) * HD + d, o * pattn_factor(state_s[3 * c], state_s[3 * c + 1], state_s[3 * c + 2]));
            } else mine[(size_t) c * STATE + d] = o;
        }
        if (parts > 1 && tid < cols) {
            *(float4*) (mine + (size_t) tid * STATE + HD) = make_float4(state_s[3 * tid], state_s[3 * tid + 1], state_s[3 * tid + 2], 0.0f);
        }
        if (tid == 0 && parts > 1 && (int) blockIdx.x == b0) a.rec[blockIdx.x] = make_int4(parts | it.kvh << 16, it.sp.row, 0, cols);
    }
}

int pattn_few_status() { return pattn_status_of(g_pattn_status); }

template <int HD, bool FINE>
static void launch_few(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv) {
    cudaFuncSetAttribute(pattn_few_kernel<HD, FINE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<HD>::SMEM);
    launch(pattn_few_kernel<HD, FINE>, (unsigned) pattn_blocks(), FEW_THREADS, Few<HD>::SMEM, s, a, tk, tv);
    launch_pattn_merge(s, a, pattn_blocks());
    count_launch(2);
}

void launch_pattn_few(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv) {
    const bool fine = a.q_type == NSL_F32;
    if (a.p.hd == 128) { if (fine) launch_few<128, true>(s, a, tk, tv); else launch_few<128, false>(s, a, tk, tv); }
    else if (fine) launch_few<64, true>(s, a, tk, tv);
    else launch_few<64, false>(s, a, tk, tv);
}

}   // namespace nsl
