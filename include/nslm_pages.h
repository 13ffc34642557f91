/* nslm_pages.h - a paged 8-bit KV cache: rotary positions, the store into pages, attention over them, their management.
 *
 * No counterpart in the reference, whose caches are one fixed slot of rows per sequence (kc_rope_kv, kc_attn).  Here a pool
 * holds pages of `page` positions; a sequence names its pages in a row of the page table, so sequences share prefixes, are
 * forked, rolled back and moved without touching what they have in common.  Codes are int8 with ONE f32 scale per page and
 * KV head (value = code * scale), so the attention's products run on the codes and the scale is applied per page.
 *
 * Conventions as in nslm_kernels.h: the stream first, asynchronous launches that allocate nothing, the caller owns every
 * buffer; a call that is refused launches nothing and leaves a message in nsl_last_error() and in nsl_pages_error().  Every kernel here waits on the
 * device for its predecessor before it reads anything and is a dependent launch unless nsl_dependent_launch(0) was called.
 * The tensors and the stream belong to the current device. */
#pragma once
#include "nslm_kernels.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Why this thread's last call of this header was refused, or "" if it was served.  nsl_last_error() keeps the first message that nobody has read,
 * whatever call and thread it came from; one that is read here counts as read there too. */
const char* nsl_pages_error(void);

/* Elements of the queries, keys, values and results. */
enum {
    NSL_F32 = 0,          /* f32, results unrounded */
    NSL_BF16 = 1,         /* packed bf16 */
    NSL_F32_BF16 = 2      /* f32 arrays of bf16 values: results are rounded to bf16 (the engine's activations) */
};

/* ---- rotary positions --------------------------------------------------------------------------------------------------- */
enum { NSL_ROPE_HALF = 0, NSL_ROPE_INTERLEAVED = 1 };   /* pairs (p, p + rot / 2), or (2 p, 2 p + 1) */
typedef struct {
    const float* inv;        /* device: rot / 2 angles per position (radians) */
    int32_t rot, layout;     /* the first rot values of a head are rotated: a multiple of 16; 0: none */
    float factor;            /* factor on the rotated values (1, or a long-context scaling's) */
    int32_t pad;
} NslRope;
/* Frequency tables, on the host: inv[rot / 2] and *factor of
 *   NSL_ROPE_PLAIN   theta^(-2 p / rot)
 *   NSL_ROPE_LINEAR  the same / scale (positions interpolated)
 *   NSL_ROPE_BASE    theta * scale^(rot / (rot - 2)) instead of theta: the lowest frequency is divided by scale, the highest kept
 *   NSL_ROPE_PARTS  frequencies that turn more than beta_fast times within ctx positions are kept, those below beta_slow turns divided
 *                    by scale, and between them r of the way: with c(beta) = rot ln(ctx / (2 pi beta)) / (2 ln theta), the pair that turns beta
 *                    times, lo = max(floor c(beta_fast), 0), hi = min(ceil c(beta_slow), rot - 1), at least lo + 0.001, and
 *                    r = (p - lo) / (hi - lo) within [0, 1], times (1 - r) + r / scale; factor = 0.1 ln(scale) + 1.  The idea is YaRN's (arXiv
 *                    2309.00071); its eq. 17-23 have a ramp that is linear in the turns, while this one, linear in the pair's number, is the one
 *                    that models with such tables are published for (pair 33 of rot 128, theta 1e4, ctx 4096, scale 16: 4.60e-3, by the turns 1.76e-3)
 * -> 0, or -1 with a message (rot not even and positive, theta <= 1 or scale < 1 or not finite, or ctx / betas unusable). */
enum { NSL_ROPE_PLAIN = 0, NSL_ROPE_LINEAR = 1, NSL_ROPE_BASE = 2, NSL_ROPE_PARTS = 3 };
int nsl_rope_freqs(int kind, int rot, double theta, double scale, int ctx, double beta_fast, double beta_slow, float* inv, float* factor);
/* Rows of heads rotated: x = factor (u cos a - w sin a, w cos a + u sin a), a = pos[t] * inv[p], the product reduced to a quarter
 * turn with all its bits (for frequencies up to 1 the angle is right to 1e-15 at every int32 position, its sine and cosine to 1.2e-10 and a
 * rounding to f32).  q, qo [T][n_head][hd] with row strides in elements, k, ko [T][n_kv][hd] (n_kv = 0: none; n_head = 0: none);
 * outputs may be the inputs; a call whose outputs otherwise overlap them, or one another, is refused.  hd a multiple of 16, at
 * most 512; rows start on 16-byte boundaries. */
void nsl_rope(cudaStream_t s, NslRope r, int type, int hd, const void* q, int q_stride, void* qo, int qo_stride, int n_head, const void* k, int k_stride,
              void* ko, int ko_stride, int n_kv, const int32_t* pos, int T);

/* ---- the pool ------------------------------------------------------------------------------------------------------------- */
typedef struct {
    int8_t *k, *v;           /* codes [n_layer][n_pages][n_kv][page][hd], 16-byte aligned */
    float *ks, *vs;          /* scales [n_layer][n_pages][n_kv] */
    int32_t* ref;            /* [n_pages]: how many sequences a page belongs to; 0: free */
    int32_t* table;          /* [n_seq][max_pages]: page ids, -1 where a sequence has none */
    int32_t* len;            /* [n_seq]: positions a sequence has pages for */
    int32_t* work;           /* 4 + 3 n_pages ints of work memory for the management calls (no initial contents) */
    int32_t n_layer, n_pages, n_kv, hd;      /* n_pages <= 2^20; n_kv <= 1024; hd: 64 or 128 */
    int32_t page;            /* positions of a page: 16, 32, 64 or 128 */
    int32_t n_seq, max_pages, pad;
} NslPages;

/* One sequence's rows of a call: rows row .. row + rows - 1 of its arrays are positions pos .. pos + rows - 1 of sequence seq.
 * Descriptors come in any order; rows <= 0 is an empty place of a padded batch; a sequence appears once, row ranges do not
 * overlap.  Any int32 row and position may be named.  Rows that no descriptor names, or that lie outside [0, T), are left as they are. */
typedef struct { int32_t row, rows, pos, seq; } NslSeqRows;

/* Queries rotated (q -> qo, see nsl_rope; n_head = 0: none; a qo that overlaps k or v is refused), keys rotated, and keys and values stored in the pages of layer
 * `layer` that the sequences' table rows name (reserved before: nsl_pages_extend).  r.rot = 0: nothing is rotated.
 * A page's scale is a power of two, the smallest with max |x| <= 127 scale over what the page holds: it starts afresh with the
 * call that writes the page's first position and never shrinks until then; when a later row needs a larger one, the codes that
 * are there are rounded to it.  code = x / scale rounded to nearest even; NaN is stored as 0, an infinity as the largest code
 * (its page's scale is then 2^122: the other values of that page and head are lost).  Positions without a page (table entry outside [0, n_pages), position outside the
 * table's row) are not stored; queries at positions below 0 or past 2^31 - 1 are left as they are.  Pages that several sequences share are not protected here. */
void nsl_pages_append(cudaStream_t s, const NslPages* p, int layer, NslRope r, int type, const void* q, int q_stride, void* qo, int qo_stride, int n_head,
                      const void* k, int k_stride, const void* v, int v_stride, const NslSeqRows* seqs, int n_seqs, int T);
/* The values at the descriptors' positions -> ko, vo [T][n_kv][hd] (type NSL_F32: code * scale; the others: rounded to bf16).
 * Rows of positions without a page are left as they are; a ko that overlaps vo is refused. */
void nsl_pages_read(cudaStream_t s, const NslPages* p, int layer, int type, void* ko, int ko_stride, void* vo, int vo_stride, const NslSeqRows* seqs, int n_seqs,
                    int T);

/* Attention of each sequence's rows over its pages: the row at position P attends positions max(0, P - window + 1) .. P
 * (window <= 0: from 0) of its sequence, query head h over KV head h / (n_head / n_kv).  o = softmax(scale q.k) v, rounded to
 * bf16 (o_type NSL_BF16 or NSL_F32_BF16; an o that overlaps q is refused).  Positions without a page are left out, and so is what lies in a
 * page behind the row's position, whatever it holds; a row that nothing is left for gives zeros.  Scales are not negative.  Here a
 * sequence may appear in several descriptors, and positions past 2^31 - 1 count as 2^31 - 1.
 * Queries are held as f16 after their head's largest magnitude's power of two is divided out (bf16 values exactly, elements below 2^-17 of
 * the largest to 2^-25 of it), for q_type NSL_F32 as two such terms (22 bits, or 2^-25 of the largest); q_type NSL_F32_BF16 says that the values
 * are bf16's, and one term is taken.  Weights times their page's value scale are held as f16 too (11 bits, or 2^-25 of the largest of the row); sums in f32.
 * max_rows: no descriptor has more rows (rows beyond it are left as they are).  work: nsl_pages_attn_work() bytes of device
 * memory (40 MB for 148 multiprocessors), 16-byte aligned, no initial contents; calls that share it run one behind the other, captured ones too.
 * The step's keys are dealt evenly to the blocks, so a row alone and in a batch may differ in the order of its f32 sums; a call
 * repeated gives the same bits.  n_seqs <= 4096; the 64-key units of a call (all sequences and KV heads) number fewer than 2^31. */
size_t nsl_pages_attn_work(void);
void nsl_pages_attn(cudaStream_t s, const NslPages* p, int layer, int q_type, const void* q, int q_stride, int n_head, float scale, int window,
                    const NslSeqRows* seqs, int n_seqs, int max_rows, int T, int o_type, void* o, int o_stride, void* work);
/* 0, or the code of the first bounded device-side wait that ran out (after a second) in an attention block since it was last reported (few
 * rows: 1 a fetch waiting for a free stage, 2 a computing warp waiting for a full one; many rows: 4 .. 6 the softmax waiting
 * for scores, for scales or for values added, 7 and 8 the expansion for codes or a free tile, 9 a fetch, 10 .. 13 the issue of
 * products for queries, tiles, read scores or weights).  What such a block had not finished by then is NaN in the results.  A call reports one
 * code: where both kinds of block had one, the next call reports the other.  -1, with a message: the device cannot be read.
 * Synchronous; call it after the stream has drained. */
int nsl_pages_attn_status(void);
/* For testing what a host does about that: until it is called with 0, this thread's nsl_pages_attn calls fetch no codes, so
 * every wait for some runs out, after wait_ns (a second at most), and their results are NaN. */
void nsl_pages_attn_hold(unsigned long long wait_ns);

/* ---- management: device lists, at most NSL_PAGES_LIST entries a call; the calls on a pool run one behind the other -------- */
#define NSL_PAGES_LIST 1024
typedef struct { int32_t seq, len; } NslPagesLen;
typedef struct { int32_t src, dst, len, pad; } NslPagesFork;
/* Sequence seq grows to len positions: positions from its present length on can then be written.  Requests are served in the
 * list's order with the lowest free ids; a last page that is shared and only partly used is replaced by a copy (in all
 * layers) first - the last of those who share it keeps it.  A request that does not fit its table row, or names a sequence a
 * second time, is refused; so is the first for which no pages are left and all behind it.  got[i] (optional) = 1 where
 * request i was served; a refused one changes nothing. */
void nsl_pages_extend(cudaStream_t s, const NslPages* p, const NslPagesLen* reqs, int n, int32_t* got);
/* dst, a sequence without positions, shares the first min(len, length of src) positions of src.  Lengths are those before the
 * call; an entry is passed over whose dst has positions, was named as dst before in the list, or equals src. */
void nsl_pages_fork(cudaStream_t s, const NslPages* p, const NslPagesFork* forks, int n);
/* Sequence seq is cut back to at most len positions; pages that nobody uses any more are free.  A sequence named twice is cut
 * to the smaller. */
void nsl_pages_trim(cudaStream_t s, const NslPages* p, const NslPagesLen* reqs, int n);
/* The pages in use move to the lowest ids (in all layers; the i-th of those above the number in use goes to the i-th free id
 * below it), tables and ref follow.  work[1] = their number afterwards. */
void nsl_pages_compact(cudaStream_t s, const NslPages* p);
/* Page pairs[2 i] -> page pairs[2 i + 1] in all layers, codes and scales (device list, any n).  A destination appears once and
 * is no source of the call; ids outside the pool are passed over. */
void nsl_pages_copy(cudaStream_t s, const NslPages* p, const int32_t* pairs, int n);

#ifdef __cplusplus
}
#endif
