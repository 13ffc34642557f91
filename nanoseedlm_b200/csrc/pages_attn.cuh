// What the attention kernels over the paged cache share: the call's arguments, barriers and copies, the code conversions.
#pragma once
#include <cuda.h>
#include <math.h>

#include "pages.cuh"

namespace nsl {

struct PagesAttn {
    NslPages p;
    const void* q;
    void* o;
    const NslSeqRows* seqs;
    float* part;        // partial states, two slots a block: of the item that it begins with, if that began in an earlier block
                        // (slot 2 b), and of the one that it ends with, if that ends in a later one (slot 2 b + 1)
    int4* rec;          // per block, its item that ends in a later block: states | KV head << 16 (0: none), first row, first column, columns
    float scale;
    int q_type, q_stride, o_type, o_stride, n_head, layer, window, n_seqs, max_rows, T;
    int hold;                      // no block fetches anything (nsl_pages_attn_hold)
    unsigned long long wait_ns;    // how long a wait lasts at most
};

// Blocks of a launch at most: two an SM (their number fits a record's 16 bits).
inline int pattn_blocks() { return 2 * sm_count(); }
constexpr int PATTN_FEW = 8, PATTN_MANY = 256;      // columns of an item
template <int HD>
constexpr int PATTN_STATE = HD + 4;      // floats of a column's state: O [HD], m, l, mo, one unused
void launch_pattn_many(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv);
constexpr unsigned long long PATTN_WAIT_NS = 1000000000ull;
int pattn_few_status();      // 0, a wait's code, or -1; a code is read once
int pattn_many_status();
void launch_pattn_merge(cudaStream_t s, const PagesAttn& a, int blocks);

bool pattn_map(CUtensorMap* tm, const NslPages& p, const int8_t* codes);      // rows of hd codes, boxes of min(page, 64) rows, swizzled
void launch_pattn_few(cudaStream_t s, const PagesAttn& a, const CUtensorMap& tk, const CUtensorMap& tv);

#ifdef __CUDACC__
constexpr uint32_t PATTN_WAIT_LIMIT = 1u << 24;

__device__ __forceinline__ uint32_t pa_smem(const void* p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ void pa_bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void pa_bar_arrive(uint32_t bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pa_bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool pa_bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// Waits are bounded: after wait_ns (PATTN_WAIT_NS) or PATTN_WAIT_LIMIT attempts a wait sets the block's abort flag and a status code and
// returns, and so does every later wait of the block at once.  The block then runs to its end on what is there (every access in
// bounds, every barrier met), fetches nothing more, and gives a sum l of NaN with every item that it has not finished by then, so
// that its results, and those that its states are joined into, are NaN.  A wait that returned whether it succeeded, voted on
// by the warp, cost a unit of 256 columns a third of its time.
static __device__ __noinline__ void pa_bar_wait_long(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code, unsigned long long wait_ns) {
    unsigned long long t0 = 0;
    for (uint32_t i = 0; i < PATTN_WAIT_LIMIT; ++i) {
        if (*abort_flag || pa_bar_try(bar, parity)) return;
        if ((i & 63u) == 63u) {
            unsigned long long t;
            asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
            if (!t0) t0 = t;
            if (t - t0 > wait_ns) break;
        }
    }
    *abort_flag = 1;
    atomicCAS(status, 0, code);
}
__device__ __forceinline__ void pa_bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code, unsigned long long wait_ns) {
    if (!pa_bar_try(bar, parity) && !pa_bar_try(bar, parity) && !pa_bar_try(bar, parity)) pa_bar_wait_long(bar, parity, abort_flag, status, code, wait_ns);
    __syncwarp();
}
__device__ __forceinline__ void pa_tma_rows(uint32_t smem, const CUtensorMap* tm, int row, uint32_t bar) {      // x = 0: the rows' first code
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(smem), "l"(tm), "r"(0), "r"(row), "r"(bar) : "memory");
}

__device__ __forceinline__ float pa_ex2(float x) {      // 2^x, relative error 2^-22; 2^-inf = 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pa_f16x2(float lo, float hi) {      // round to nearest even
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// What x and y lost when they were rounded to the f16 pair `rounded`, rounded to f16 themselves.
__device__ __forceinline__ uint32_t pa_low_f16x2(float x, float y, uint32_t rounded) {
    float lo, hi;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}" : "=f"(lo), "=f"(hi) : "r"(rounded));
    return pa_f16x2(x - lo, y - hi);
}
// Two bytes (signed codes ^ 0x80, picked by SEL from x) as two f16 values: a byte u under the exponent of 1024 is 1024 + u, and
// 1024 + (code + 128) - 1152 is the code, exactly.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t pa_codes(uint32_t x) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(x, 0x64646464u, SEL)), "r"(0x64806480u));
    return r;
}
// The value of a query element; its column's values are divided by a power of two before they are rounded to f16.
__device__ __forceinline__ float pa_query(const void* q, int type, size_t at) {
    return type == NSL_BF16 ? __uint_as_float((uint32_t) ((const uint16_t*) q)[at] << 16) : ((const float*) q)[at];
}
// 2^e with |x| / 2^e in [1, 2) for x = the column's largest magnitude (1 for zero; e within -126 .. 126).
__device__ __forceinline__ float pa_pow2_of(float x) {
    const int e = (int) (__float_as_uint(x) >> 23 & 0xFFu) - 127;
    return x == 0.0f ? 1.0f : __uint_as_float((uint32_t) (min(max(e, -126), 126) + 127) << 23);
}

// What the blocks' chains of dependent loads will come to (descriptors, page table, the layer's scales, queries), requested into L2 by all blocks
// together before the wait for the kernel before: nothing is read, so what that still writes is not
// missed.  A cold load costs 1 to 2 us here, and a block's first codes lie behind three of them.
__device__ __forceinline__ void pattn_warm(const PagesAttn& a) {
    const size_t scales = (size_t) a.layer * a.p.n_pages * a.p.n_kv, scale_lines = ((size_t) a.p.n_pages * a.p.n_kv * 4 + 127) / 128;
    const char* const from[5] = {(const char*) a.seqs, (const char*) a.p.table, (const char*) (a.p.ks + scales), (const char*) (a.p.vs + scales), (const char*) a.q};
    const size_t lines[5] = {((size_t) a.n_seqs * sizeof(NslSeqRows) + 127) / 128, ((size_t) a.p.n_seq * a.p.max_pages * 4 + 127) / 128, scale_lines, scale_lines, (((size_t) (a.T - 1) * a.q_stride + (size_t) a.n_head * a.p.hd) * (a.q_type == NSL_BF16 ? 2 : 4) + 127) / 128};
    const size_t at = (size_t) blockIdx.x * blockDim.x + threadIdx.x;      // one line of each array a thread: up to 6 MB of each with 296 blocks of 160
#pragma unroll
    for (int i = 0; i < 5; ++i)
        if (at < lines[i]) asm volatile("prefetch.global.L2 [%0];" ::"l"(from[i] + 128 * at));
}

// The position i rows on; those past 2^31 - 1 count as 2^31 - 1, behind all that a table's row holds.
__device__ __forceinline__ int pos_of(int pos, int i) { return (int) min((long long) pos + i, 0x7FFFFFFFll); }
// The first position that the row at position `pos` attends (0 without a window), and one behind its last: both within the table's row.
__device__ __forceinline__ int first_key(const PagesAttn& a, int pos) {
    return a.window > 0 ? (int) min(max((long long) pos - a.window + 1, 0ll), (long long) a.p.max_pages * a.p.page) : 0;
}
__device__ __forceinline__ int end_key(const PagesAttn& a, int pos) { return max(min(pos, a.p.max_pages * a.p.page - 1) + 1, 0); }
// A descriptor's rows that exist: [row, row + rows) of the call's rows, the first at position pos.
struct RowSpan { int row, rows, pos, seq; };
__device__ __forceinline__ RowSpan row_span(const PagesAttn& a, int i) {
    const NslSeqRows d = a.seqs[i];
    RowSpan s;
    const int lo = max(d.row, 0);
    const long long hi = min((long long) d.row + min(max(d.rows, 0), a.max_rows), (long long) a.T);
    s.row = lo;
    s.rows = (int) max(hi - lo, 0ll);
    s.pos = (int) min((long long) d.pos + lo - d.row, 0x7FFFFFFFll);
    s.seq = d.seq;
    return s;
}
// What a column's O is multiplied with: 2^(mo - m) / l; nothing attended: 0; a sum that is NaN stays NaN.
__device__ __forceinline__ float pattn_factor(float m, float l, float mo) { return l != l ? l : l == 0.0f || mo == -INFINITY ? 0.0f : pa_ex2(mo - m) / l; }
__device__ __forceinline__ void store_bf16_of(const PagesAttn& a, size_t at, float x) {
    const uint32_t b = bf16_pair(x, 0.0f);
    if (a.o_type == NSL_BF16) ((uint16_t*) a.o)[at] = (uint16_t) b;
    else ((float*) a.o)[at] = __uint_as_float(b << 16);
}
// A status word read and, if it holds a code, cleared; -1: it cannot be read.
inline int pattn_status_of(int& word) {
    int v = 0;
    const int zero = 0;
    if (cudaMemcpyFromSymbol(&v, word, sizeof v) != cudaSuccess || (v && cudaMemcpyToSymbol(word, &zero, sizeof zero) != cudaSuccess)) {
        set_error("nsl_pages_attn_status: the status word cannot be read");
        return -1;
    }
    return v;
}
#endif

}   // namespace nsl
