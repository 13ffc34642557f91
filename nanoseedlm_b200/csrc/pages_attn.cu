// Attention of ragged rows over the paged 8-bit cache (nsl_pages_attn).
#include "pages_attn.cuh"

namespace nsl {

// The states of an unfinished item of the few-row kernel joined.  Block (b, y): the item that block b of the first pass leaves
// unfinished, some of its columns.  Up to MERGE_FEW states: a warp a column, everything requested before anything is used; more:
// four warps a column, every fourth state each.  Bound: latency.
constexpr int MERGE_THREADS = 256, MERGE_WARPS = MERGE_THREADS / 32, MERGE_EACH = 4, MERGE_FEW = 8;

template <int HD>
__device__ __forceinline__ void merge_store(const PagesAttn& a, const int4& rec, int col, int lane, float4 o, float f) {
    const int group = a.n_head / a.p.n_kv, c = rec.z + col, kvh = rec.x >> 16;
    const size_t at = (size_t) (rec.y + c / group) * a.o_stride + (size_t) (kvh * group + c % group) * HD + 4 * lane;
    const uint32_t lo = bf16_pair(o.x * f, o.y * f), hi = bf16_pair(o.z * f, o.w * f);
    if (a.o_type == NSL_BF16) *(uint2*) ((uint16_t*) a.o + at) = make_uint2(lo, hi);
    else *(float4*) ((float*) a.o + at) = make_float4(__uint_as_float(lo << 16), __uint_as_float(lo & 0xFFFF0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xFFFF0000u));
}
__device__ __forceinline__ void merge_add(float4& o, const float4& v, float w) {
    o.x = fmaf(v.x, w, o.x); o.y = fmaf(v.y, w, o.y); o.z = fmaf(v.z, w, o.z); o.w = fmaf(v.w, w, o.w);
}
__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.0f : m; }

template <int HD>
__global__ void __launch_bounds__(MERGE_THREADS) pattn_merge_kernel(PagesAttn a) {
    constexpr int STATE = PATTN_STATE<HD>;
    __shared__ float4 sum[MERGE_WARPS][32];
    __shared__ float stat[MERGE_WARPS][3];
    grid_dependents_go();
    grid_dependency_wait();
    const int4 rec = a.rec[blockIdx.x];
    const int parts = rec.x & 0xFFFF, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (parts == 0) return;
    auto state = [&](int i, int col) { return a.part + ((size_t) (2 * ((int) blockIdx.x + i) + (i == 0)) * PATTN_FEW + col) * STATE; };
    if (parts <= MERGE_FEW) {
        for (int col = (int) blockIdx.y * MERGE_WARPS + warp; col < rec.w; col += (int) gridDim.y * MERGE_WARPS) {
            float4 v[MERGE_FEW], st[MERGE_FEW];
#pragma unroll
            for (int i = 0; i < MERGE_FEW; ++i) {
                st[i] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
                if (i >= parts) continue;
                const float* p = state(i, col);
                st[i] = *(const float4*) (p + HD);
                v[i] = *(const float4*) (p + 4 * (4 * lane < HD ? lane : 0));
            }
            float m = -INFINITY, mo = -INFINITY, l = 0.0f;
#pragma unroll
            for (int i = 0; i < MERGE_FEW; ++i) { m = fmaxf(m, st[i].x); mo = fmaxf(mo, st[i].z); }
            const float ms = finite_or_0(m), mos = finite_or_0(mo);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < MERGE_FEW; ++i)
                if (i < parts) { l = fmaf(st[i].y, pa_ex2(st[i].x - ms), l); merge_add(o, v[i], pa_ex2(st[i].z - mos)); }
            if (4 * lane < HD) merge_store<HD>(a, rec, col, lane, o, pattn_factor(m, l, mo));
        }
        return;
    }
    const int turn = warp % MERGE_EACH;
    constexpr int COLS = MERGE_WARPS / MERGE_EACH;
    for (int c0 = (int) blockIdx.y * COLS; c0 < rec.w; c0 += (int) gridDim.y * COLS) {
        const int col = c0 + warp / MERGE_EACH;
        __syncthreads();      // the last columns' sums have been read
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float m = -INFINITY, mo = -INFINITY, l = 0.0f;
        if (col < rec.w) {
            // the maxima over this warp's states, a state a lane; then the sums
            for (int i = turn + MERGE_EACH * lane; i < parts; i += MERGE_EACH * 32) { const float* st = state(i, col) + HD; m = fmaxf(m, st[0]); mo = fmaxf(mo, st[2]); }
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) { m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x)); mo = fmaxf(mo, __shfl_xor_sync(0xFFFFFFFFu, mo, x)); }
            const float ms = finite_or_0(m), mos = finite_or_0(mo);
#pragma unroll 8
            for (int i = turn; i < parts; i += MERGE_EACH) {
                const float* p = state(i, col);
                const float4 st = *(const float4*) (p + HD);
                l = fmaf(st.y, pa_ex2(st.x - ms), l);
                if (4 * lane < HD) merge_add(o, *(const float4*) (p + 4 * lane), pa_ex2(st.z - mos));
            }
        }
        sum[warp][lane] = o;
        if (lane == 0) { stat[warp][0] = m; stat[warp][1] = l; stat[warp][2] = mo; }
        __syncthreads();
        if (turn || col >= rec.w || 4 * lane >= HD) continue;
        for (int w = 1; w < MERGE_EACH; ++w) { m = fmaxf(m, stat[warp + w][0]); mo = fmaxf(mo, stat[warp + w][2]); }
        const float ms = finite_or_0(m), mos = finite_or_0(mo);
        o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < MERGE_EACH; ++w) {
            l = fmaf(stat[warp + w][1], pa_ex2(stat[warp + w][0] - ms), l);
            merge_add(o, sum[warp + w][lane], pa_ex2(stat[warp + w][2] - mos));
        }
        merge_store<HD>(a, rec, col, lane, o, pattn_factor(m, l, mo));
    }
}

void launch_pattn_merge(cudaStream_t s, const PagesAttn& a, int blocks) {
    const dim3 grid((unsigned) blocks, (unsigned) ((a.n_head / a.p.n_kv) * a.max_rows + 1) / 2);      // (at most PATTN_FEW columns)
    if (a.p.hd == 128) launch(pattn_merge_kernel<128>, grid, MERGE_THREADS, 0, s, a);
    else launch(pattn_merge_kernel<64>, grid, MERGE_THREADS, 0, s, a);
}

// Encoded at every call: a map is 128 bytes of the launch's arguments, and a pool's buffers are the caller's.
bool pattn_map(CUtensorMap* tm, const NslPages& p, const int8_t* codes) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                               CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = NULL;
        cudaDriverEntryPointQueryResult r;
        return cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess ? (Encode) f : (Encode) NULL;
    }();
    const cuuint64_t rows = (cuuint64_t) p.n_layer * p.n_pages * p.n_kv * p.page;
    if (!encode || rows > 0x7FFFFFFFull) return false;
    const cuuint64_t dims[2] = {(cuuint64_t) p.hd, rows}, strides[1] = {(cuuint64_t) p.hd};
    const cuuint32_t box[2] = {(cuuint32_t) p.hd, (cuuint32_t) (p.page < 64 ? p.page : 64)}, step[2] = {1, 1};
    return encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*) codes, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  p.hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}   // namespace nsl

using namespace nsl;

extern "C" {

// A record a block, and two states for each of the blocks of either kernel (two an SM of up to PATTN_FEW columns, one of up to PATTN_MANY).
size_t nsl_pages_attn_work(void) { return (size_t) pattn_blocks() * 16 + (size_t) sm_count() * 2 * PATTN_MANY * PATTN_STATE<128> * 4; }

int nsl_pages_attn_status(void) {
    begin_call();
    const int few = pattn_few_status();
    return few ? few : pattn_many_status();
}

static thread_local unsigned long long tl_hold_ns = 0;
void nsl_pages_attn_hold(unsigned long long wait_ns) { tl_hold_ns = wait_ns < PATTN_WAIT_NS ? wait_ns : PATTN_WAIT_NS; }

void nsl_pages_attn(cudaStream_t s, const NslPages* p, int layer, int q_type, const void* q, int q_stride, int n_head, float scale, int window,
                    const NslSeqRows* seqs, int n_seqs, int max_rows, int T, int o_type, void* o, int o_stride, void* work) {
    begin_call();
    if (T <= 0 || n_seqs <= 0 || max_rows <= 0) return;
    if (!pages_ok(p, "nsl_pages_attn")) return;
    if (!layer_ok(p, layer) || !known_type(q_type) || (o_type != NSL_BF16 && o_type != NSL_F32_BF16) || n_head < 1 || n_head % p->n_kv || n_head > 65535 || (long long) n_head * T > 0x7FFFFFFF || !seqs || n_seqs > 4096 ||
        !work || !aligned16(work) || !rows_ok(q, q_stride, n_head * p->hd, q_type) || !rows_ok(o, o_stride, n_head * p->hd, o_type)) {
        set_error("nsl_pages_attn: layer %d of %d, types %d and %d, %d query heads over %d, %d sequences (at most 4096), or rows or work memory that are not 16-byte aligned", layer, p->n_layer,
                  q_type, o_type, n_head, p->n_kv, n_seqs);
        return;
    }
    if (!rows_apart(q, q_stride, n_head * p->hd, q_type, o, o_stride, n_head * p->hd, o_type, T)) { set_error("nsl_pages_attn: results that overlap the queries"); return; }
    CUtensorMap tk, tv;
    if (!pattn_map(&tk, *p, p->k) || !pattn_map(&tv, *p, p->v)) { set_error("nsl_pages_attn: no tensor map for the pool's codes"); return; }
    FollowScope follow;
    PagesAttn a;
    a.p = *p; a.q = q; a.o = o; a.seqs = seqs;
    a.rec = (int4*) work;
    a.part = (float*) ((char*) work + 16 * (size_t) pattn_blocks());
    a.scale = scale; a.q_type = q_type; a.q_stride = q_stride; a.o_type = o_type; a.o_stride = o_stride;
    a.n_head = n_head; a.layer = layer; a.window = window; a.n_seqs = n_seqs; a.max_rows = max_rows < T ? max_rows : T; a.T = T;
    a.hold = tl_hold_ns > 0;
    a.wait_ns = a.hold ? tl_hold_ns : PATTN_WAIT_NS;
    // One of the two for all sequences of a call.  The few-row kernel reads the keys for 8 columns, the wide one makes a tile of 128
    // whatever it holds: 32 rows of 4096 keys with 8 heads a KV head 21 us; with 10, 12 and 16 heads over one KV head 41 us in the wide kernel
    // against 39 to 41 as two calls of half the heads (8 x 16000 keys: 42 against 37 to 39, one row of 4096 keys: 32 against 21 to 23; heads
    // of 64: 30 against 32 to 33, 30 against 30 to 32, 24 against 18 to 19).
    // Decode rows beside a prompt's rows are in the wide kernel too: 4 x 1000 keys beside 512 rows behind 2048 positions 49 us, as two calls 59, but 32 x 4096
    // beside 2048 rows 166 against 142, beside 256 rows 84 against 70, 64 x 2000 beside 1024 rows 120 against 93 (16 heads over 2).
    if ((long long) (n_head / p->n_kv) * a.max_rows <= PATTN_FEW) launch_pattn_few(s, a, tk, tv);
    else launch_pattn_many(s, a, tk, tv);
}

}   // extern "C"
