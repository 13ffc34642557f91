// Attention of ragged rows over the paged 8-bit cache (nsl_pages_attn).
#include <math.h>

#include "pages.cuh"
#include "seed_block.cuh"

namespace nsl {

struct PagesAttn {
    NslPages p;
    const void* q;
    void* o;
    const NslSeqRows* seqs;
    float scale;
    int q_type, q_stride, o_type, o_stride, n_head, layer, window, n_seqs, max_rows, T;
};

// One block per (head, row): 128 keys at a time, a thread a key for the scores, a thread a dim for the values; the running
// maximum and sum in f32.  Right for every call, no more.
constexpr int SIMPLE = 128;
__global__ void __launch_bounds__(SIMPLE) pages_attn_simple_kernel(PagesAttn a) {
    __shared__ float qs[128], ps[SIMPLE], red[SIMPLE / 32];
    __shared__ int found;
    grid_dependents_go();
    grid_dependency_wait();
    const NslPages& p = a.p;
    const int h = blockIdx.x, t = blockIdx.y, tid = threadIdx.x, kvh = h / (a.n_head / p.n_kv);
    const int di = row_descriptor(a.seqs, a.n_seqs, t, &found);
    if (di < 0) return;
    const NslSeqRows d = a.seqs[di];
    if (t - d.row >= a.max_rows) return;
    const int pos = d.pos + (t - d.row), k1 = min(pos + 1, p.max_pages * p.page), k0 = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    if (tid < p.hd) {
        const size_t at = (size_t) t * a.q_stride + (size_t) h * p.hd + tid;
        qs[tid] = a.q_type == NSL_BF16 ? __uint_as_float((uint32_t) ((const uint16_t*) a.q)[at] << 16) : ((const float*) a.q)[at];
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int b = k0; b < k1; b += SIMPLE) {
        const int key = b + tid;
        float s = -INFINITY;
        if (key < k1) {
            const int id = page_of(p, d.seq, key / p.page);
            if (id >= 0) {
                const size_t page_at = ((size_t) a.layer * p.n_pages + id) * p.n_kv + kvh;
                const char4* row = (const char4*) (p.k + (page_at * p.page + key % p.page) * p.hd);
                float sum = 0.0f;
                for (int w = 0; w < p.hd / 4; ++w) {
                    const char4 c = row[w];
                    sum += qs[4 * w] * c.x + qs[4 * w + 1] * c.y + qs[4 * w + 2] * c.z + qs[4 * w + 3] * c.w;
                }
                s = sum * p.ks[page_at] * a.scale;
            }
        }
        float mx = s;
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        mx = fmaxf(mx, m);
        if (mx == -INFINITY) continue;      // nothing yet; the same for all threads
        const float cor = expf(m - mx), e = expf(s - mx);
        m = mx;
        ps[tid] = e;
        __syncthreads();
        l *= cor;
        acc *= cor;
        for (int i = 0; i < SIMPLE && b + i < k1; ++i) {
            l += ps[i];
            if (ps[i] == 0.0f || tid >= p.hd) continue;
            const int id = page_of(p, d.seq, (b + i) / p.page);
            const size_t page_at = ((size_t) a.layer * p.n_pages + id) * p.n_kv + kvh;
            acc += ps[i] * ((float) p.v[(page_at * p.page + (b + i) % p.page) * p.hd + tid] * p.vs[page_at]);
        }
    }
    if (tid >= p.hd) return;
    const float o = bf16_round(l > 0.0f ? acc / l : 0.0f);
    const size_t at = (size_t) t * a.o_stride + (size_t) h * p.hd + tid;
    if (a.o_type == NSL_BF16) ((uint16_t*) a.o)[at] = bf16_bits(o);
    else ((float*) a.o)[at] = o;
}

}   // namespace nsl

using namespace nsl;

extern "C" {

size_t nsl_pages_attn_work(void) { return 1 << 20; }

void nsl_pages_attn(cudaStream_t s, const NslPages* p, int layer, int q_type, const void* q, int q_stride, int n_head, float scale, int window,
                    const NslSeqRows* seqs, int n_seqs, int max_rows, int T, int o_type, void* o, int o_stride, void* work) {
    if (T <= 0 || n_seqs <= 0 || max_rows <= 0) return;
    if (!pages_ok(p, "nsl_pages_attn")) return;
    if (!layer_ok(p, layer) || !known_type(q_type) || (o_type != NSL_BF16 && o_type != NSL_F32_BF16) || n_head < 1 || n_head % p->n_kv || n_head > 65535 || !seqs || n_seqs > 4096 ||
        !work || !aligned16(work) || !rows_ok(q, q_stride, n_head * p->hd, q_type) || !rows_ok(o, o_stride, n_head * p->hd, o_type)) {
        set_error("nsl_pages_attn: layer %d of %d, types %d and %d, %d query heads over %d, %d sequences (at most 4096), or rows or work memory that are not 16-byte aligned", layer, p->n_layer,
                  q_type, o_type, n_head, p->n_kv, n_seqs);
        return;
    }
    FollowScope follow;
    const PagesAttn a = {*p, q, o, seqs, scale, q_type, q_stride, o_type, o_stride, n_head, layer, window, n_seqs, max_rows, T};
    launch(pages_attn_simple_kernel, dim3((unsigned) n_head, (unsigned) T), SIMPLE, 0, s, a);
    count_launch();
}

}   // extern "C"
