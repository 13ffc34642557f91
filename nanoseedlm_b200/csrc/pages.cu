// The paged 8-bit cache: the store of keys and values (nsl_pages_append), the read back, and the pages' management.
//
// Store.  A unit is what one call writes of one page: it is quantised together, because its rows share the page's scale.  Work
// item = (unit, keys or values, a few KV heads); the blocks behind them rotate the queries.  Bound: HBM (the rows are read
// once, a byte per value written); 8192 rows of 16 + 8 + 8 heads of 128 bf16 values: 40 us by itself = 2.9 TB/s, 29 without the queries, issue and latency at 45 % of the
// warps; a decode batch's call is a chain of four loads (32 rows, and read back: 6.7 us).
// The scale is a power of two: dividing by it is exact, a page filled row by row ends with the scale of the same rows written
// at once, and codes that are there follow a larger scale by one rounding shift.  Against max / 127 it costs at most one bit.
#include <math.h>

#include "pages.cuh"

namespace nsl {

constexpr int APPEND_THREADS = 256, APPEND_Q_ROWS = 8;      // APPEND_Q_ROWS: of a block at most

// What of a descriptor is stored: its rows within [0, T) whose positions lie within the table's row.  A descriptor may name any int32 row and
// position, so the sums are made in 64 bits; what is left fits 32.
struct SeqSpan { int row, rows, pos; };
__device__ __forceinline__ SeqSpan span_of(const NslSeqRows& d, const NslPages& p, int T) {
    const long long first = (long long) d.pos - d.row;      // the position that row 0 would have
    const long long lo = max(max((long long) d.row, 0ll), -first), hi = min(min((long long) d.row + max(d.rows, 0), (long long) T), (long long) p.max_pages * p.page - first);
    SeqSpan s;
    s.rows = (int) max(hi - lo, 0ll);
    s.row = s.rows ? (int) lo : 0;
    s.pos = s.rows ? (int) (lo + first) : 0;
    return s;
}

// Unit u of the call: the descriptor and its page, found by a running sum over the descriptors.  -> false: there is none.
__device__ bool find_unit(const NslSeqRows* seqs, int n_seqs, int T, const NslPages& p, int u, int* desc, int* nth) {
    __shared__ int wsum[APPEND_THREADS / 32], at[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) at[0] = -1;
    int before = 0;
    for (int i0 = 0; i0 < n_seqs; i0 += APPEND_THREADS) {
        int mine = 0;
        if (i0 + tid < n_seqs) {
            const SeqSpan s = span_of(seqs[i0 + tid], p, T);
            if (s.rows > 0) mine = (s.pos + s.rows - 1) / p.page - s.pos / p.page + 1;
        }
        int incl = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, incl, off);
            if (lane >= off) incl += v;
        }
        __syncthreads();      // the last round's wsum has been read
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        int total = 0, start = before + incl - mine;
#pragma unroll
        for (int w = 0; w < APPEND_THREADS / 32; ++w) {
            if (w < warp) start += wsum[w];
            total += wsum[w];
        }
        if (u >= start && u < start + mine) { at[0] = i0 + tid; at[1] = u - start; }
        before += total;
        if (before > u) break;      // the same for all threads
    }
    __syncthreads();
    *desc = at[0];
    *nth = at[1];
    return at[0] >= 0;
}

// The exponent of the smallest power of two with top <= 127 * 2^e, as the float 2^e (2^-126 for top = 0).
__device__ __forceinline__ float scale_of(float top) {
    const uint32_t b = __float_as_uint(fminf(top, 3.402823466e38f));
    const int e = (int) (b >> 23) - 127 - 6 + ((b & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);      // 127 = 2^6 (1 + 0x7E0000 / 2^23)
    return __uint_as_float((uint32_t) (max(e, -126) + 127) << 23);
}
__device__ __forceinline__ uint32_t code_of(float x, float inv) {      // NaN -> 0, infinities -> +-127
    const float c = x != x ? 0.0f : fminf(fmaxf(x * inv, -127.0f), 127.0f);
    return (uint32_t) __float2int_rn(c) & 0xFFu;
}
// The codes of 8 values.  FINITE: |x| inv <= 127, inv a power of two; adding 1.5 2^23 rounds to the nearest integer, ties to even, and leaves
// it in the sum's low byte (3.7 instructions a value where the conversion takes 9, a quarter of them at an eighth of the rate).
template <bool FINITE>
__device__ __forceinline__ uint2 codes8(const float* x, float inv) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (FINITE) {
            uint32_t c[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = __float_as_uint(fmaf(x[4 * i + e], inv, 12582912.0f));
            w[i] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        } else
            w[i] = code_of(x[4 * i], inv) | code_of(x[4 * i + 1], inv) << 8 | code_of(x[4 * i + 2], inv) << 16 | code_of(x[4 * i + 3], inv) << 24;
    }
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float max_nan(float a, float b) {      // NaN if either is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

struct AppendArgs {
    NslPages p;
    NslRope r;
    const void *q, *k, *v;
    void* qo;
    const NslSeqRows* seqs;
    int q_stride, qo_stride, k_stride, v_stride, n_head, layer, n_seqs, T;
    int units, head_split, heads_each, kv_blocks, q_rows;      // blocks: [units][2 tensors][head_split], then the query blocks of q_rows rows
};

// One (unit, tensor, heads) item.  GROUPS: groups of 16 values a thread holds (page * hd / 16 / threads at most).
template <int TYPE, int GROUPS>
__device__ void append_unit(const AppendArgs& a, int b, float2* cs) {
    const NslPages& p = a.p;
    const int hs = b % a.head_split, is_v = b / a.head_split & 1, u = b / a.head_split >> 1;
    int di, nth;
    if (!find_unit(a.seqs, a.n_seqs, a.T, p, u, &di, &nth)) return;
    const NslSeqRows d = a.seqs[di];
    const SeqSpan sp = span_of(d, p, a.T);
    const int j = sp.pos / p.page + nth;
    const int lo = max(sp.pos, j * p.page), hi = min(sp.pos + sp.rows, (j + 1) * p.page);      // positions
    const int id = page_of(p, d.seq, j);
    if (id < 0) return;
    const int n = hi - lo, off = lo - j * p.page, row0 = sp.row + (lo - sp.pos);
    const int pairs = a.r.rot / 2, gs = p.hd == 128 ? 3 : 2;      // 2^gs groups a head
    const bool turn = !is_v && pairs > 0;
    if (turn)
        for (int i = threadIdx.x; i < n * pairs; i += APPEND_THREADS) cs[i] = rope_angle(lo + i / pairs, a.r.inv[i % pairs], a.r.factor);
    __syncthreads();
    const void* src = is_v ? a.v : a.k;
    const int stride = is_v ? a.v_stride : a.k_stride;
    int8_t* codes = is_v ? p.v : p.k;
    float* scales = is_v ? p.vs : p.ks;
    NslRope r = a.r;
    if (is_v) r.rot = 0;
    __shared__ float wtop[APPEND_THREADS / 32];
    const int h1 = min(p.n_kv, (hs + 1) * a.heads_each);
    for (int h = hs * a.heads_each; h < h1; ++h) {
        float x[GROUPS][16], top = 0.0f;
#pragma unroll
        for (int m = 0; m < GROUPS; ++m) {
            const int i = threadIdx.x + m * APPEND_THREADS, row = i >> gs, g = i & ((1 << gs) - 1);
            if (row >= n) continue;
            const size_t at = (size_t) (row0 + row) * stride + (size_t) h * p.hd;
            int ra, rb;
            rope_runs(r, g, &ra, &rb);
            load8<TYPE>(src, at + ra, x[m]);
            load8<TYPE>(src, at + rb, x[m] + 8);
            if (turn && 16 * g < r.rot) rope_turn(r.layout, x[m], cs + row * pairs + 8 * g);
#pragma unroll
            for (int e = 0; e < 16; ++e) top = max_nan(top, fabsf(x[m][e]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const size_t page_at = ((size_t) a.layer * p.n_pages + id) * p.n_kv + h;
        const float old = off > 0 ? scales[page_at] : 0.0f;
        __syncthreads();      // wtop and the scale: read by all before they are written
        if ((threadIdx.x & 31) == 0) wtop[threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < APPEND_THREADS / 32; ++w) top = max_nan(top, wtop[w]);
        const bool finite = top <= 3.402823466e38f;      // the same for all threads
        if (!finite) {      // once more without the NaN
            top = 0.0f;
#pragma unroll
            for (int m = 0; m < GROUPS; ++m)
                if (((int) threadIdx.x + m * APPEND_THREADS) >> gs < n)
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[m][e]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) wtop[threadIdx.x >> 5] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < APPEND_THREADS / 32; ++w) top = fmaxf(top, wtop[w]);
        }
        const float need = scale_of(top), scale = old > need ? old : need, inv = 1.0f / scale;      // exact: powers of two; a foreign scale that is none is kept, and its reciprocal rounded
        int8_t* tile = codes + page_at * p.page * p.hd;
        if (off > 0 && scale != old) {      // what the page holds follows the larger scale
            const float by = old * inv;
            for (int i = threadIdx.x; i < off * p.hd / 4; i += APPEND_THREADS) {
                const char4 c = ((const char4*) tile)[i];
                ((uint32_t*) tile)[i] = code_of((float) c.x, by) | code_of((float) c.y, by) << 8 | code_of((float) c.z, by) << 16 | code_of((float) c.w, by) << 24;
            }
        }
        if (threadIdx.x == 0) scales[page_at] = scale;
#pragma unroll
        for (int m = 0; m < GROUPS; ++m) {
            const int i = threadIdx.x + m * APPEND_THREADS, row = i >> gs, g = i & ((1 << gs) - 1);
            if (row >= n) continue;
            int ra, rb;
            rope_runs(r, g, &ra, &rb);
            int8_t* to = tile + (size_t) (off + row) * p.hd;
            const bool plain = finite && scale == need;      // (a scale that was there already may be no power of two, or far larger)
            *(uint2*) (to + ra) = plain ? codes8<true>(x[m], inv) : codes8<false>(x[m], inv);
            *(uint2*) (to + rb) = plain ? codes8<true>(x[m] + 8, inv) : codes8<false>(x[m] + 8, inv);
        }
    }
}

// A block's threads over rows of per_row items each: this thread's first row and how many rows there are at a time, its first item of a
// row and the step between its items (no division but this one).
struct Split { int row, rows, first, step; };
__device__ __forceinline__ Split split_rows(int per_row, int threads) {
    Split s;
    if (per_row >= threads) { s.row = 0; s.rows = 1; s.first = threadIdx.x; s.step = threads; return s; }
    s.rows = threads / per_row;
    s.row = (int) threadIdx.x / per_row;
    s.first = (int) threadIdx.x - s.row * per_row;
    s.step = per_row;
    if (s.row >= s.rows) s.row = 1 << 30;      // nothing
    return s;
}

// The queries of q_rows rows.
template <int TYPE>
__device__ void append_queries(const AppendArgs& a, int b, float2* cs) {
    __shared__ int found[APPEND_Q_ROWS], at[APPEND_Q_ROWS];
    const int t0 = b * a.q_rows, n = min(a.q_rows, a.T - t0), pairs = a.r.rot / 2, hd = a.p.hd;
    row_descriptors(a.seqs, a.n_seqs, t0, n, found);
    if ((int) threadIdx.x < n) {
        const int di = found[threadIdx.x];
        const long long pos = di < 0 ? -1 : (long long) a.seqs[di].pos + (t0 + (int) threadIdx.x) - a.seqs[di].row;
        at[threadIdx.x] = pos > 0x7FFFFFFF ? -1 : (int) max(pos, -1ll);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * pairs; i += APPEND_THREADS) cs[i] = rope_angle(max(at[i / pairs], 0), a.r.inv[i % pairs], a.r.factor);
    __syncthreads();
    const int gs = hd == 128 ? 3 : 2, per_row = a.n_head << gs;
    const Split sp = split_rows(per_row, APPEND_THREADS);
    for (int row = sp.row; row < n; row += sp.rows) {
        if (at[row] < 0) continue;
        for (int i = sp.first; i < per_row; i += sp.step) {
            const int g = i & ((1 << gs) - 1), h = i >> gs;
            int ra, rb;
            rope_runs(a.r, g, &ra, &rb);
            float x[16];
            const size_t from = (size_t) (t0 + row) * a.q_stride + (size_t) h * hd, to = (size_t) (t0 + row) * a.qo_stride + (size_t) h * hd;
            load8<TYPE>(a.q, from + ra, x);
            load8<TYPE>(a.q, from + rb, x + 8);
            if (16 * g < a.r.rot) rope_turn(a.r.layout, x, cs + row * pairs + 8 * g);
            store8<TYPE>(a.qo, to + ra, x);
            store8<TYPE>(a.qo, to + rb, x + 8);
        }
    }
}

template <int TYPE, int GROUPS>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(AppendArgs a) {
    extern __shared__ __align__(16) float2 append_cs[];
    grid_dependents_go();
    grid_dependency_wait();
    const int b = (int) blockIdx.x;
    if (b < a.kv_blocks) append_unit<TYPE, GROUPS>(a, b, append_cs);
    else append_queries<TYPE>(a, b - a.kv_blocks, append_cs);
}

// Rows back: a thread takes 16 codes of a head.  Bound: HBM (8192 rows of 8 KV heads of 128 as bf16: 13.8 us = 3.7 TB/s).
constexpr int READ_THREADS = 256, READ_ROWS = 16;      // READ_ROWS: of a block at most
template <int TYPE>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(NslPages p, int layer, void* ko, int ko_stride, void* vo, int vo_stride, const NslSeqRows* seqs, int n_seqs, int T, int rows) {
    __shared__ int found[READ_ROWS], page_id[READ_ROWS], slot[READ_ROWS];
    grid_dependents_go();
    grid_dependency_wait();
    const int t0 = (int) blockIdx.x * rows, n = min(rows, T - t0);
    row_descriptors(seqs, n_seqs, t0, n, found);
    if ((int) threadIdx.x < n) {
        const int di = found[threadIdx.x];
        int id = -1, in = 0;
        if (di >= 0) {
            const NslSeqRows d = seqs[di];
            const long long pos = (long long) d.pos + (t0 + (int) threadIdx.x - d.row);
            if (pos >= 0 && pos / p.page < p.max_pages) { id = page_of(p, d.seq, (int) (pos / p.page)); in = (int) (pos % p.page); }
        }
        page_id[threadIdx.x] = id;
        slot[threadIdx.x] = in;
    }
    __syncthreads();
    const int gs = p.hd == 128 ? 3 : 2, per_row = 2 * p.n_kv << gs;
    const Split sp = split_rows(per_row, READ_THREADS);
    for (int row = sp.row; row < n; row += sp.rows) {
        if (page_id[row] < 0) continue;
        for (int i = sp.first; i < per_row; i += sp.step) {
            const int g = i & ((1 << gs) - 1), is_v = (i >> gs) >= p.n_kv, h = (i >> gs) - (is_v ? p.n_kv : 0);
            const size_t page_at = ((size_t) layer * p.n_pages + page_id[row]) * p.n_kv + h;
            const float scale = (is_v ? p.vs : p.ks)[page_at];
            const uint4 c = *(const uint4*) ((is_v ? p.v : p.k) + (page_at * p.page + slot[row]) * p.hd + 16 * g);
            const uint32_t w[4] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u, c.z ^ 0x80808080u, c.w ^ 0x80808080u};
            float x[16];      // a byte under the exponent of 2^23 is 2^23 + 128 + code: exact, and off the conversions' slow pipe
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = (__uint_as_float(__byte_perm(w[e >> 2], 0x4B000000u, 0x7440 | (e & 3))) - 8388736.0f) * scale;
            void* to = is_v ? vo : ko;
            const size_t at = (size_t) (t0 + row) * (is_v ? vo_stride : ko_stride) + (size_t) h * p.hd + 16 * g;
            store8<TYPE>(to, at, x);
            store8<TYPE>(to, at + 8, x + 8);
        }
    }
}

// ---- management: one block decides, a second kernel moves the data --------------------------------------------------------
// Bound: launches and dependent loads (a trim, a fork and an extension of 32 sequences with the move: 12.8 us); in long lists and pools the one block:
// 1024 sequences trimmed 50 us, 60,000 pages compacted 131 us with 12,499 moves of 2 KB, 1,000,000 2.4 ms (an extension there 9).
// work: [0] pages to move, [1] pages in use after a compaction, [2], [3] unused; then the (from, to) pairs; then n_pages ints.
constexpr int MAN_THREADS = 1024;
static_assert(MAN_THREADS == NSL_PAGES_LIST, "a thread an entry");
__device__ __forceinline__ int* work_pairs(const NslPages& p) { return p.work + 4; }
__device__ __forceinline__ int* work_ids(const NslPages& p) { return p.work + 4 + 2 * (size_t) p.n_pages; }

// Exclusive running sum over the block's threads; *total = the sum.  Called by all.
__device__ int block_scan(int v, int* total) {
    __shared__ int wsum[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int x = __shfl_up_sync(0xFFFFFFFFu, incl, off);
        if (lane >= off) incl += x;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int x = wsum[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xFFFFFFFFu, x, off);
            if (lane >= off) x += y;
        }
        wsum[lane] = x;
    }
    __syncthreads();
    *total = wsum[31];
    return incl - v + (warp ? wsum[warp - 1] : 0);
}
__device__ __forceinline__ int pages_for(int len, int page) { return len / page + (len % page != 0); }
__device__ __forceinline__ bool seq_ok(const NslPages& p, int seq) { return seq >= 0 && seq < p.n_seq; }

// How many entries before this thread's have the same key (keys >= 0; all[] holds every thread's): a warp's own by a match, those of
// earlier warps one by one.  Called by whole warps.
__device__ __forceinline__ int same_before(const int* all, int key) {
    const uint32_t lower = (1u << (threadIdx.x & 31)) - 1u;
    int n = __popc(__match_any_sync(0xFFFFFFFFu, key) & lower);
    for (int j = 0; key >= 0 && j < (int) (threadIdx.x & ~31u); ++j) n += all[j] == key;
    return n;
}

__global__ void __launch_bounds__(MAN_THREADS) extend_kernel(NslPages p, const NslPagesLen* reqs, int n, int32_t* got) {
    __shared__ int seq_s[MAN_THREADS], page_s[MAN_THREADS], start_s[MAN_THREADS], have_s[MAN_THREADS], end_s[MAN_THREADS];
    grid_dependents_go();
    grid_dependency_wait();
    const int i = threadIdx.x;
    int seq = -1, old = 0, now = 0;
    if (i < n) { seq = reqs[i].seq; now = reqs[i].len; }
    bool fits = i < n && seq_ok(p, seq);
    seq_s[i] = fits ? seq : -1;
    __syncthreads();
    if (same_before(seq_s, fits ? seq : -1) && fits) fits = false;      // named before
    int have = 0, need = 0, last_id = -1;
    if (fits) {
        old = p.len[seq];
        now = max(now, old);
        have = pages_for(max(old, 0), p.page);
        need = pages_for(now, p.page);
        fits = need <= p.max_pages && old >= 0;      // (a length below 0 is no length: refused, and no entry before the row is reached)
    }
    if (fits && now > old && old % p.page) {
        last_id = page_of(p, seq, old / p.page);
        if (last_id < 0) fits = false;
    }
    page_s[i] = fits ? last_id : -1;
    __syncthreads();
    const int users = fits && last_id >= 0 ? p.ref[last_id] : 0;
    const int given_up = same_before(page_s, page_s[i]);      // requests that give the page up before this one
    const bool copy = users > 1 && users - given_up > 1;
    const int want = fits ? min(need - have + copy, p.n_pages + 1) : 0;      // (n_pages <= 2^20: the sum stays in 32 bits)
    int total, n_free = 0;
    const int start = block_scan(want, &total);
    // the lowest free ids, until there are enough of them
    int* const ids = work_ids(p);
    for (int base = 0; base < p.n_pages && n_free < total; base += 4 * MAN_THREADS) {
        int free4 = 0, c = 0, sum;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int id = base + 4 * i + e;
            if (id < p.n_pages && p.ref[id] == 0) { free4 |= 1 << e; ++c; }
        }
        int at = n_free + block_scan(c, &sum);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (free4 >> e & 1) ids[at++] = base + 4 * i + e;
        n_free += sum;
    }
    const bool ok = fits && start + want <= n_free;
    int jobs;
    const int job = block_scan(copy && ok, &jobs);      // (its barriers also make ids visible)
    if (i == 0) p.work[0] = jobs;
    if (copy && ok) {
        const int to = ids[start];
        work_pairs(p)[2 * job] = last_id;
        work_pairs(p)[2 * job + 1] = to;
        p.table[(size_t) seq * p.max_pages + old / p.page] = to;
        p.ref[to] = 1;
        atomicSub(&p.ref[last_id], 1);
    }
    if (i < n && ok) p.len[seq] = now;
    if (i < n && got) got[i] = ok;
    start_s[i] = start + copy;
    have_s[i] = have;
    end_s[i] = ok ? need : 0;
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < n; r += MAN_THREADS / 32)      // a warp a request
        for (int j = have_s[r] + (threadIdx.x & 31); j < end_s[r]; j += 32) {
            const int id = ids[start_s[r] + j - have_s[r]];
            p.table[(size_t) seq_s[r] * p.max_pages + j] = id;
            p.ref[id] = 1;
        }
}

__global__ void __launch_bounds__(MAN_THREADS) fork_kernel(NslPages p, const NslPagesFork* forks, int n) {
    __shared__ int src_s[MAN_THREADS], dst_s[MAN_THREADS], len_s[MAN_THREADS];
    grid_dependents_go();
    grid_dependency_wait();
    const int i = threadIdx.x;
    bool on = false;
    int src = -1, dst = -1, len = 0;
    if (i < n) {
        src = forks[i].src; dst = forks[i].dst; len = forks[i].len;
        on = seq_ok(p, src) && seq_ok(p, dst) && src != dst;
    }
    dst_s[i] = on ? dst : -1;
    __syncthreads();
    if (same_before(dst_s, on ? dst : -1) && on) on = false;
    if (on) {
        on = p.len[dst] == 0;
        len = max(min(len, p.len[src]), 0);
        if (pages_for(len, p.page) > p.max_pages) on = false;
    }
    src_s[i] = src;
    len_s[i] = on ? len : 0;
    __syncthreads();      // all lengths have been read
    if (on) p.len[dst] = len;
    for (int r = threadIdx.x >> 5; r < n; r += MAN_THREADS / 32) {
        const int m = pages_for(len_s[r], p.page);
        for (int j = threadIdx.x & 31; j < m; j += 32) {
            const int id = p.table[(size_t) src_s[r] * p.max_pages + j];
            p.table[(size_t) dst_s[r] * p.max_pages + j] = id;
            if (id >= 0 && id < p.n_pages) atomicAdd(&p.ref[id], 1);
        }
    }
}

__global__ void __launch_bounds__(MAN_THREADS) trim_kernel(NslPages p, const NslPagesLen* reqs, int n) {
    __shared__ int seq_s[MAN_THREADS], keep_s[MAN_THREADS], from_s[MAN_THREADS], to_s[MAN_THREADS];
    grid_dependents_go();
    grid_dependency_wait();
    const int i = threadIdx.x;
    int seq = -1, keep = 0;
    if (i < n) { seq = reqs[i].seq; keep = max(reqs[i].len, 0); }
    bool on = i < n && seq_ok(p, seq);
    seq_s[i] = on ? seq : -1;
    keep_s[i] = keep;
    __syncthreads();
    if (on)
        for (int j = 0; j < n; ++j)
            if (seq_s[j] == seq) {
                if (j < i) on = false;      // done by the first that names it
                keep = min(keep, keep_s[j]);
            }
    int from = 0, to = 0;
    if (on) {
        const int len = p.len[seq];
        if (keep < len) {
            from = pages_for(keep, p.page);
            to = min(pages_for(len, p.page), p.max_pages);
            p.len[seq] = keep;
        }
    }
    from_s[i] = from;
    to_s[i] = to;
    __syncthreads();
    for (int r = threadIdx.x >> 5; r < n; r += MAN_THREADS / 32)
        for (int j = from_s[r] + (threadIdx.x & 31); j < to_s[r]; j += 32) {
            int32_t* e = p.table + (size_t) seq_s[r] * p.max_pages + j;
            const int id = *e;
            if (id >= 0 && id < p.n_pages) atomicSub(&p.ref[id], 1);
            *e = -1;
        }
}

__global__ void __launch_bounds__(MAN_THREADS) compact_kernel(NslPages p) {
    grid_dependents_go();
    grid_dependency_wait();
    const int i = threadIdx.x;
    int* const pairs = work_pairs(p);
    int* const to_of = work_ids(p);
    int c = 0, live, total;
    for (int id = i; id < p.n_pages; id += MAN_THREADS) c += p.ref[id] > 0;
    block_scan(c, &live);
    int holes = 0, movers = 0;
    for (int base = 0; base < p.n_pages; base += MAN_THREADS) {
        const int id = base + i;
        const bool used = id < p.n_pages && p.ref[id] > 0;
        const bool hole = id < live && !used, mover = id >= live && used;      // as many of one as of the other
        const int h = holes + block_scan(hole, &total);
        holes += total;
        const int m = movers + block_scan(mover, &total);
        movers += total;
        if (hole) pairs[2 * h + 1] = id;
        if (mover) pairs[2 * m] = id;
        if (id < p.n_pages) to_of[id] = id;
    }
    __syncthreads();
    for (int j = i; j < movers; j += MAN_THREADS) {
        const int from = pairs[2 * j], to = pairs[2 * j + 1];
        to_of[from] = to;
        p.ref[to] = p.ref[from];
        p.ref[from] = 0;
    }
    if (i == 0) { p.work[0] = movers; p.work[1] = live; }
}

// Pairs of pages copied in all layers: a task = 16 KB of a (pair, layer, keys or values), its first task the scales too.
// renumber: the tables follow a compaction.  Bound: HBM, 2 bytes moved per byte of a page (about 120 pages of 2 x 16 KB in 8 layers: 64 MB in 11 us by itself).
constexpr int MOVE_THREADS = 256, MOVE_BYTES = 16384;
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(NslPages p, const int32_t* pairs, const int32_t* count, int n, int renumber) {
    grid_dependents_go();
    grid_dependency_wait();
    if (count) n = *count;
    const int page_bytes = p.n_kv * p.page * p.hd, pieces = (page_bytes + MOVE_BYTES - 1) / MOVE_BYTES;
    const long long tasks = (long long) n * p.n_layer * 2 * pieces;
    for (long long x = blockIdx.x; x < tasks; x += gridDim.x) {
        const int piece = (int) (x % pieces), is_v = (int) (x / pieces & 1);
        const long long y = x / pieces >> 1;
        const int layer = (int) (y % p.n_layer), job = (int) (y / p.n_layer);
        const int from = pairs[2 * job], to = pairs[2 * job + 1];
        if (from < 0 || from >= p.n_pages || to < 0 || to >= p.n_pages || from == to) continue;
        int8_t* codes = is_v ? p.v : p.k;
        float* scales = is_v ? p.vs : p.ks;
        const size_t a = (size_t) layer * p.n_pages + from, b = (size_t) layer * p.n_pages + to;
        const uint4* src = (const uint4*) (codes + a * page_bytes);
        uint4* dst = (uint4*) (codes + b * page_bytes);
        const int e0 = piece * (MOVE_BYTES / 16), e1 = min(page_bytes / 16, e0 + MOVE_BYTES / 16);
        uint4 v[MOVE_BYTES / 16 / MOVE_THREADS];
#pragma unroll
        for (int m = 0; m < MOVE_BYTES / 16 / MOVE_THREADS; ++m) {
            const int e = e0 + m * MOVE_THREADS + (int) threadIdx.x;
            if (e < e1) v[m] = src[e];
        }
#pragma unroll
        for (int m = 0; m < MOVE_BYTES / 16 / MOVE_THREADS; ++m) {
            const int e = e0 + m * MOVE_THREADS + (int) threadIdx.x;
            if (e < e1) dst[e] = v[m];
        }
        if (piece == 0)
            for (int h = threadIdx.x; h < p.n_kv; h += MOVE_THREADS) scales[b * p.n_kv + h] = scales[a * p.n_kv + h];
    }
    if (renumber) {
        const int* to_of = work_ids(p);
        const size_t entries = (size_t) p.n_seq * p.max_pages;
        for (size_t e = (size_t) blockIdx.x * MOVE_THREADS + threadIdx.x; e < entries; e += (size_t) gridDim.x * MOVE_THREADS) {
            const int id = p.table[e];
            if (id >= 0 && id < p.n_pages) p.table[e] = to_of[id];
        }
    }
}

bool pages_ok(const NslPages* p, const char* who) {
    if (p && p->k && p->v && p->ks && p->vs && p->ref && p->table && p->len && p->work && aligned16(p->k) && aligned16(p->v) && p->n_layer > 0 && p->n_pages > 0 && p->n_pages <= 1 << 20 && p->n_kv > 0 &&
        p->n_kv <= 1024 && (p->hd == 64 || p->hd == 128) && (p->page == 16 || p->page == 32 || p->page == 64 || p->page == 128) && p->n_seq > 0 && p->max_pages > 0 &&
        (long long) p->max_pages * p->page < (1ll << 30))
        return true;
    set_error("%s: a pool without buffers, codes that are not 16-byte aligned, heads that are not 64 or 128 wide, pages that are not 16, 32, 64 or 128 positions, or sizes out of range", who);
    return false;
}
static bool list_ok(const void* list, int n, const char* who) {
    if (list && n <= NSL_PAGES_LIST) return true;
    set_error("%s: %d entries (at most %d), or no list", who, n, NSL_PAGES_LIST);
    return false;
}
static void launch_move(cudaStream_t s, const NslPages& p, const int32_t* pairs, const int32_t* count, int n, int renumber) {
    launch(move_kernel, (unsigned) sm_count() * 4, MOVE_THREADS, 0, s, p, pairs, count, n, renumber);
}

template <int TYPE>
static void launch_append(cudaStream_t s, const AppendArgs& a, unsigned blocks, size_t smem) {
    const int groups = a.p.page * a.p.hd / 16;      // of a full page: a thread holds groups / threads of them
    auto* kernel = groups <= APPEND_THREADS ? append_kernel<TYPE, 1> : groups <= 2 * APPEND_THREADS ? append_kernel<TYPE, 2> : append_kernel<TYPE, 4>;
    if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) smem);
    launch(kernel, blocks, APPEND_THREADS, smem, s, a);
}

}   // namespace nsl

using namespace nsl;

extern "C" {

void nsl_pages_append(cudaStream_t s, const NslPages* p, int layer, NslRope r, int type, const void* q, int q_stride, void* qo, int qo_stride, int n_head,
                      const void* k, int k_stride, const void* v, int v_stride, const NslSeqRows* seqs, int n_seqs, int T) {
    begin_call();
    if (T <= 0 || n_seqs <= 0) return;
    if (!pages_ok(p, "nsl_pages_append")) return;
    if (!layer_ok(p, layer) || !known_type(type) || !rope_ok(r, p->hd) || !seqs || n_head < 0 || n_head > 65536 || (n_head && (!rows_ok(q, q_stride, n_head * p->hd, type) || !rows_ok(qo, qo_stride, n_head * p->hd, type))) ||
        !rows_ok(k, k_stride, p->n_kv * p->hd, type) || !rows_ok(v, v_stride, p->n_kv * p->hd, type)) {
        set_error("nsl_pages_append: layer %d of %d, type %d, %d rotated values of %d, no descriptors, or rows that are not 16-byte aligned", layer, p->n_layer, type, r.rot, p->hd);
        return;
    }
    const int kw = p->n_kv * p->hd;
    if (n_head && (!rows_same_or_apart(q, q_stride, qo, qo_stride, n_head * p->hd, type, T) || !rows_apart(qo, qo_stride, n_head * p->hd, type, k, k_stride, kw, type, T) ||
                   !rows_apart(qo, qo_stride, n_head * p->hd, type, v, v_stride, kw, type, T))) {
        set_error("nsl_pages_append: rotated queries that overlap the queries, keys or values");
        return;
    }
    FollowScope follow;
    AppendArgs a;
    a.p = *p; a.r = r; a.q = q; a.k = k; a.v = v; a.qo = qo; a.seqs = seqs;
    a.q_stride = q_stride; a.qo_stride = qo_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.n_head = n_head; a.layer = layer; a.n_seqs = n_seqs; a.T = T;
    if ((long long) T * p->n_kv > 1 << 29) { set_error("nsl_pages_append: %d rows of %d heads in one call", T, p->n_kv); return; }
    const long long most = (long long) T / p->page + 2ll * (n_seqs < T ? n_seqs : T);      // sum of (rows - 1) / page + 2
    a.units = (int) (most < T ? most : T);
    // heads of a block: the keys' angles are made once for all of them, so as many as leave four blocks an SM; rows of queries likewise
    a.heads_each = 1;
    while (a.heads_each * 2 <= p->n_kv && (long long) a.units * 2 * (p->n_kv / (a.heads_each * 2)) >= 4ll * sm_count()) a.heads_each *= 2;
    a.head_split = (p->n_kv + a.heads_each - 1) / a.heads_each;
    a.kv_blocks = a.units * 2 * a.head_split;
    a.q_rows = 1;
    while (a.q_rows < APPEND_Q_ROWS && T / (a.q_rows * 2) >= 4 * sm_count()) a.q_rows *= 2;
    const int q_blocks = n_head ? (T + a.q_rows - 1) / a.q_rows : 0;
    const int rows = p->page > a.q_rows ? p->page : a.q_rows;
    const size_t smem = sizeof(float2) * (size_t) (r.rot / 2) * rows;
    const unsigned blocks = (unsigned) (a.kv_blocks + q_blocks);
    if (type == NSL_F32) launch_append<NSL_F32>(s, a, blocks, smem);
    else if (type == NSL_BF16) launch_append<NSL_BF16>(s, a, blocks, smem);
    else launch_append<NSL_F32_BF16>(s, a, blocks, smem);
    count_launch();
}

void nsl_pages_read(cudaStream_t s, const NslPages* p, int layer, int type, void* ko, int ko_stride, void* vo, int vo_stride, const NslSeqRows* seqs, int n_seqs, int T) {
    begin_call();
    if (T <= 0 || n_seqs <= 0) return;
    if (!pages_ok(p, "nsl_pages_read")) return;
    if (!layer_ok(p, layer) || !known_type(type) || !seqs || !rows_ok(ko, ko_stride, p->n_kv * p->hd, type) || !rows_ok(vo, vo_stride, p->n_kv * p->hd, type)) {
        set_error("nsl_pages_read: layer %d of %d, type %d, no descriptors, or rows that are not 16-byte aligned", layer, p->n_layer, type);
        return;
    }
    if (!rows_apart(ko, ko_stride, p->n_kv * p->hd, type, vo, vo_stride, p->n_kv * p->hd, type, T)) { set_error("nsl_pages_read: keys and values that overlap"); return; }
    FollowScope follow;
    int rows = 1;      // as many as leave four blocks an SM
    while (rows < READ_ROWS && T / (rows * 2) >= 4 * sm_count()) rows *= 2;
    const dim3 grid((unsigned) ((T + rows - 1) / rows));
    if (type == NSL_F32) launch(read_kernel<NSL_F32>, grid, READ_THREADS, 0, s, *p, layer, ko, ko_stride, vo, vo_stride, seqs, n_seqs, T, rows);
    else if (type == NSL_BF16) launch(read_kernel<NSL_BF16>, grid, READ_THREADS, 0, s, *p, layer, ko, ko_stride, vo, vo_stride, seqs, n_seqs, T, rows);
    else launch(read_kernel<NSL_F32_BF16>, grid, READ_THREADS, 0, s, *p, layer, ko, ko_stride, vo, vo_stride, seqs, n_seqs, T, rows);
    count_launch();
}

void nsl_pages_extend(cudaStream_t s, const NslPages* p, const NslPagesLen* reqs, int n, int32_t* got) {
    begin_call();
    if (n <= 0 || !pages_ok(p, "nsl_pages_extend") || !list_ok(reqs, n, "nsl_pages_extend")) return;
    FollowScope follow;
    launch(extend_kernel, 1, MAN_THREADS, 0, s, *p, reqs, n, got);
    launch_move(s, *p, p->work + 4, p->work, 0, 0);
    count_launch(2);
}

void nsl_pages_fork(cudaStream_t s, const NslPages* p, const NslPagesFork* forks, int n) {
    begin_call();
    if (n <= 0 || !pages_ok(p, "nsl_pages_fork") || !list_ok(forks, n, "nsl_pages_fork")) return;
    FollowScope follow;
    launch(fork_kernel, 1, MAN_THREADS, 0, s, *p, forks, n);
    count_launch();
}

void nsl_pages_trim(cudaStream_t s, const NslPages* p, const NslPagesLen* reqs, int n) {
    begin_call();
    if (n <= 0 || !pages_ok(p, "nsl_pages_trim") || !list_ok(reqs, n, "nsl_pages_trim")) return;
    FollowScope follow;
    launch(trim_kernel, 1, MAN_THREADS, 0, s, *p, reqs, n);
    count_launch();
}

void nsl_pages_compact(cudaStream_t s, const NslPages* p) {
    begin_call();
    if (!pages_ok(p, "nsl_pages_compact")) return;
    FollowScope follow;
    launch(compact_kernel, 1, MAN_THREADS, 0, s, *p);
    launch_move(s, *p, p->work + 4, p->work, 0, 1);
    count_launch(2);
}

void nsl_pages_copy(cudaStream_t s, const NslPages* p, const int32_t* pairs, int n) {
    begin_call();
    if (n <= 0 || !pages_ok(p, "nsl_pages_copy")) return;
    if (!pairs) { set_error("nsl_pages_copy: no list"); return; }
    FollowScope follow;
    launch_move(s, *p, pairs, (const int32_t*) NULL, n, 0);
    count_launch();
}

}   // extern "C"
