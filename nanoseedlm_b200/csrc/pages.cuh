// What the kernels of the paged cache share: element types, rotation of 16 values, rows of descriptors.
#pragma once
#include "common.cuh"
#include "../../include/nslm_pages.h"

namespace nsl {

inline bool known_type(int t) { return t == NSL_F32 || t == NSL_BF16 || t == NSL_F32_BF16; }
inline int type_bytes(int t) { return t == NSL_BF16 ? 2 : 4; }
// A row's base and stride: 16-byte steps, and room for the row.
inline bool rows_ok(const void* p, int stride, int width, int type) { return p && aligned16(p) && stride >= width && ((size_t) stride * type_bytes(type)) % 16 == 0; }
// Two arrays of T rows that have no byte in common: one lies behind the other, or their strides keep the rows beside one another.
inline bool rows_apart(const void* a, int a_stride, int a_width, int a_type, const void* b, int b_stride, int b_width, int b_type, int T) {
    const uint64_t at = (uint64_t) a, bt = (uint64_t) b, as = (uint64_t) a_stride * type_bytes(a_type), bs = (uint64_t) b_stride * type_bytes(b_type),
                   aw = (uint64_t) a_width * type_bytes(a_type), bw = (uint64_t) b_width * type_bytes(b_type);
    if (at + (T - 1) * as + aw <= bt || bt + (T - 1) * bs + bw <= at) return true;
    uint64_t step = as;      // every distance between a row of a and one of b is bt - at and a multiple of this
    for (uint64_t x = bs; x;) { const uint64_t r = step % x; step = x; x = r; }
    const uint64_t d = bt >= at ? (bt - at) % step : (step - (at - bt) % step) % step;
    return d >= aw && d + bw <= step;
}
inline bool rows_same_or_apart(const void* a, int a_stride, const void* b, int b_stride, int width, int type, int T) {
    return (a == b && a_stride == b_stride) || rows_apart(a, a_stride, width, type, b, b_stride, width, type, T);
}
inline bool rope_ok(const NslRope& r, int hd) {
    return r.rot == 0 || (r.rot > 0 && r.rot % 16 == 0 && r.rot <= hd && r.inv && (r.layout == NSL_ROPE_HALF || r.layout == NSL_ROPE_INTERLEAVED));
}
bool pages_ok(const NslPages* p, const char* who);      // pages.cu
inline bool layer_ok(const NslPages* p, int layer) { return layer >= 0 && layer < p->n_layer; }

#ifdef __CUDACC__
__device__ __forceinline__ void eight_of(const uint4& u, float* x) {      // packed bf16
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}
template <int TYPE>
__device__ __forceinline__ void load8(const void* base, size_t at, float* x) {
    if (TYPE == NSL_BF16) {
        eight_of(*(const uint4*) ((const uint16_t*) base + at), x);
    } else {
        const float4 a = *(const float4*) ((const float*) base + at), b = *(const float4*) ((const float*) base + at + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {      // round to nearest even, lo in bits 0-15
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int TYPE>
__device__ __forceinline__ void store8(void* base, size_t at, const float* x) {
    if (TYPE == NSL_F32) {
        *(float4*) ((float*) base + at) = make_float4(x[0], x[1], x[2], x[3]);
        *(float4*) ((float*) base + at + 4) = make_float4(x[4], x[5], x[6], x[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
    if (TYPE == NSL_BF16) { *(uint4*) ((uint16_t*) base + at) = make_uint4(w[0], w[1], w[2], w[3]); return; }
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) { y[2 * i] = __uint_as_float(w[i] << 16); y[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    store8<NSL_F32>(base, at, y);
}

// (factor cos a, factor sin a) for a = pos * inv, each rounded to f32 once.  The product of an int32 and an f32 has at most 55
// significant bits; an f32 product would be off by pos * inv * 2^-24, 0.06 at a million positions.  In f64: the product and what its rounding left off
// (`low`; 0 below position 2^29), reduced by the nearest multiple of pi / 2 (in two parts: to 1e-15 for every position), then the Taylor sums of sine and cosine on
// [-pi/4, pi/4] (first terms left out: r^13 / 13!, r^12 / 12!, below 1.2e-10), a quarter turn at a time.  Keys that lie at the border between two
// codes then fall as the formula has them.
__device__ __forceinline__ float2 rope_angle(int pos, float inv, float factor) {
    const double a = (double) pos * (double) inv, low = fma((double) pos, (double) inv, -a), k = rint(a * 0.63661977236758134);
    const double r = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, a)) + low, z = r * r;
    const double sn = fma(r * z, fma(z, fma(z, fma(z, fma(z, -1.0 / 39916800.0, 1.0 / 362880.0), -1.0 / 5040.0), 1.0 / 120.0), -1.0 / 6.0), r);
    const double cs = fma(z, fma(z, fma(z, fma(z, fma(z, -1.0 / 3628800.0, 1.0 / 40320.0), -1.0 / 720.0), 1.0 / 24.0), -0.5), 1.0);
    const int q = (int) ((long long) k & 3);
    const double c = q & 1 ? sn : cs, s = q & 1 ? cs : sn;
    return make_float2((float) ((q == 1 || q == 2 ? -c : c) * factor), (float) ((q >= 2 ? -s : s) * factor));
}
// Groups of 16 of a head's values, read as two runs of 8: group g < rot / 16 is rotated by the pairs 8 g .. 8 g + 7, the others
// are dims 16 g .. 16 g + 15 as they are.
__device__ __forceinline__ void rope_runs(const NslRope& r, int g, int* a, int* b) {
    const bool half = r.layout == NSL_ROPE_HALF && 16 * g < r.rot;
    *a = half ? 8 * g : 16 * g;
    *b = half ? 8 * g + r.rot / 2 : 16 * g + 8;
}
// x: the two runs; cs: (cos, sin) of the group's 8 pairs.  Every product and sum is rounded to f32 by itself, as the formula reads.
__device__ __forceinline__ void rope_turn(int layout, float* x, const float2* cs) {
    if (layout == NSL_ROPE_HALF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float u = x[i], w = x[i + 8];
            x[i] = __fsub_rn(__fmul_rn(u, cs[i].x), __fmul_rn(w, cs[i].y));
            x[i + 8] = __fadd_rn(__fmul_rn(w, cs[i].x), __fmul_rn(u, cs[i].y));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float u = x[2 * i], w = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(u, cs[i].x), __fmul_rn(w, cs[i].y));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(w, cs[i].x), __fmul_rn(u, cs[i].y));
        }
    }
}

// The page of a sequence's position, or -1.
__device__ __forceinline__ int page_of(const NslPages& p, int seq, int j) {
    if (seq < 0 || seq >= p.n_seq || j < 0 || j >= p.max_pages) return -1;
    const int id = p.table[(size_t) seq * p.max_pages + j];
    return id >= 0 && id < p.n_pages ? id : -1;
}
// Of rows t0 .. t0 + n - 1: the descriptors that name them, -1 where none does, in found (shared memory).  All threads of a block call it.
__device__ __forceinline__ void row_descriptors(const NslSeqRows* seqs, int n_seqs, int t0, int n, int* found) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) found[i] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n_seqs; i += blockDim.x) {
        const NslSeqRows d = seqs[i];
        const int from = (int) min(max((long long) d.row - t0, 0ll), (long long) n), to = (int) max(min((long long) d.row + max(d.rows, 0) - t0, (long long) n), 0ll);
        for (int r = from; r < to; ++r) found[r] = i;
    }
    __syncthreads();
}
#endif

}   // namespace nsl
