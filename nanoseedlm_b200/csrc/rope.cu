// Rotary positions on rows of heads (nsl_rope) and the frequency tables of their long-context scalings (nsl_rope_freqs).
#include <math.h>

#include "pages.cuh"

namespace nsl {

constexpr int ROPE_THREADS = 128, ROPE_MAX_PAIRS = 256;

// A block takes a row: its (cos, sin) go to shared memory once and serve all heads of q and k; then a thread takes groups of 16
// values (32 or 64 bytes).  Bound: HBM (5003 rows of 40 heads of 128 bf16 values: 20.6 us = 5.0 TB/s; two groups a thread in flight: 24.4, fewer blocks an SM); a decode batch's call is a launch
// (2.3 us).
template <int TYPE>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(NslRope r, int hd, const void* q, int q_stride, void* qo, int qo_stride, int n_head, const void* k,
                                                            int k_stride, void* ko, int ko_stride, int n_kv, const int32_t* pos) {
    __shared__ float2 rope_cs[ROPE_MAX_PAIRS];
    grid_dependents_go();
    grid_dependency_wait();
    const size_t t = blockIdx.x;
    const int at = pos[t];
    for (int i = threadIdx.x; i < r.rot / 2; i += ROPE_THREADS) rope_cs[i] = rope_angle(at, r.inv[i], r.factor);
    __syncthreads();
    const int groups = hd / 16, per_row = (n_head + n_kv) * groups;
    for (int i = threadIdx.x; i < per_row; i += ROPE_THREADS) {
        const int head = i / groups, g = i % groups;
        const bool is_q = head < n_head;
        const void* src = is_q ? q : k;
        void* dst = is_q ? qo : ko;
        const size_t from = t * (is_q ? q_stride : k_stride) + (size_t) (is_q ? head : head - n_head) * hd;
        const size_t to = t * (is_q ? qo_stride : ko_stride) + (size_t) (is_q ? head : head - n_head) * hd;
        int a, b;
        rope_runs(r, g, &a, &b);
        float x[16];
        load8<TYPE>(src, from + a, x);
        load8<TYPE>(src, from + b, x + 8);
        if (16 * g < r.rot) rope_turn(r.layout, x, rope_cs + 8 * g);
        store8<TYPE>(dst, to + a, x);
        store8<TYPE>(dst, to + b, x + 8);
    }
}

}   // namespace nsl

using namespace nsl;

extern "C" {

int nsl_rope_freqs(int kind, int rot, double theta, double scale, int ctx, double beta_fast, double beta_slow, float* inv, float* factor) {
    begin_call();
    if (kind < NSL_ROPE_PLAIN || kind > NSL_ROPE_PARTS || rot < 2 || rot % 2 || !(theta > 1.0) || !(scale >= 1.0) || !isfinite(theta) || !isfinite(scale) || !inv || !factor || (kind == NSL_ROPE_BASE && rot < 4) ||
        (kind == NSL_ROPE_PARTS && (ctx < 1 || !(beta_fast > beta_slow) || !(beta_slow > 0.0)))) {
        set_error("nsl_rope_freqs: kind %d, %d rotated values, theta %g, scale %g, %d positions, betas %g and %g", kind, rot, theta, scale, ctx, beta_fast, beta_slow);
        return -1;
    }
    const int n = rot / 2;
    const double base = kind == NSL_ROPE_BASE ? theta * pow(scale, rot / (rot - 2.0)) : theta;
    // the pair (as a real number) whose frequency turns `beta` times within ctx positions; the ramp between two of them is linear in the pair's number
    auto pair_of = [&](double beta) { return rot * log(ctx / (beta * 6.283185307179586)) / (2.0 * log(theta)); };
    double lo = 0.0, hi = 0.0;
    if (kind == NSL_ROPE_PARTS) {
        lo = fmax(floor(pair_of(beta_fast)), 0.0);
        hi = fmin(ceil(pair_of(beta_slow)), rot - 1.0);
        if (hi <= lo) hi = lo + 0.001;
    }
    for (int p = 0; p < n; ++p) {
        const double f = pow(base, -2.0 * p / rot);
        double by = 1.0;      // what the frequency is multiplied with
        if (kind == NSL_ROPE_LINEAR) by = 1.0 / scale;
        if (kind == NSL_ROPE_PARTS) {
            const double ramp = fmin(fmax((p - lo) / (hi - lo), 0.0), 1.0);
            by = (1.0 - ramp) + ramp / scale;
        }
        inv[p] = (float) (f * by);
    }
    *factor = kind == NSL_ROPE_PARTS ? (float) (0.1 * log(scale) + 1.0) : 1.0f;
    return 0;
}

void nsl_rope(cudaStream_t s, NslRope r, int type, int hd, const void* q, int q_stride, void* qo, int qo_stride, int n_head, const void* k, int k_stride,
              void* ko, int ko_stride, int n_kv, const int32_t* pos, int T) {
    begin_call();
    if (T <= 0) return;
    if (!known_type(type) || hd < 16 || hd % 16 || hd > 2 * ROPE_MAX_PAIRS || n_head < 0 || n_kv < 0 || (n_head > 0) + (n_kv > 0) == 0 || (long long) (n_head + n_kv) * hd > (1 << 24) ||
        r.rot == 0 || !rope_ok(r, hd) || !pos || (n_head && (!rows_ok(q, q_stride, n_head * hd, type) || !rows_ok(qo, qo_stride, n_head * hd, type))) ||
        (n_kv && (!rows_ok(k, k_stride, n_kv * hd, type) || !rows_ok(ko, ko_stride, n_kv * hd, type)))) {
        set_error("nsl_rope: type %d, %d + %d heads of %d values, %d of them rotated (a multiple of 16), no positions, or rows that are not 16-byte aligned", type, n_head, n_kv, hd, r.rot);
        return;
    }
    const int qw = n_head * hd, kw = n_kv * hd;
    if ((n_head && !rows_same_or_apart(q, q_stride, qo, qo_stride, qw, type, T)) || (n_kv && !rows_same_or_apart(k, k_stride, ko, ko_stride, kw, type, T)) ||
        (n_head && n_kv && (!rows_apart(qo, qo_stride, qw, type, k, k_stride, kw, type, T) || !rows_apart(ko, ko_stride, kw, type, q, q_stride, qw, type, T) ||
                            !rows_apart(qo, qo_stride, qw, type, ko, ko_stride, kw, type, T)))) {
        set_error("nsl_rope: outputs that overlap the inputs or one another");
        return;
    }
    FollowScope follow;
    const unsigned grid = (unsigned) T;
    if (type == NSL_F32) launch(rope_kernel<NSL_F32>, grid, ROPE_THREADS, 0, s, r, hd, q, q_stride, qo, qo_stride, n_head, k, k_stride, ko, ko_stride, n_kv, pos);
    else if (type == NSL_BF16) launch(rope_kernel<NSL_BF16>, grid, ROPE_THREADS, 0, s, r, hd, q, q_stride, qo, qo_stride, n_head, k, k_stride, ko, ko_stride, n_kv, pos);
    else launch(rope_kernel<NSL_F32_BF16>, grid, ROPE_THREADS, 0, s, r, hd, q, q_stride, qo, qo_stride, n_head, k, k_stride, ko, ko_stride, n_kv, pos);
    count_launch();
}

}   // extern "C"
