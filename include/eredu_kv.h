/*
 * eredu_kv.h -- C ABI of the paged 8-bit key/value cache (gfx950), in the same
 * library and under the same conventions as eredu_hip.h: borrowed device
 * pointers, kernels enqueued on `stream` without synchronising, 0 or an error
 * with eq_last_error()'s message, arguments checked before anything is launched.
 */
#ifndef EREDU_KV_H
#define EREDU_KV_H

#include "eredu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Paged 8-bit key/value cache.  Beside eq_rope_attention_decode's dense bf16
 * cache (one sequence, one token a call): many sequences, any number of
 * tokens a call, prefixes shared between sequences, half the bytes.  No
 * counterpart in the reference's C ABI; it stands where the reference's caches
 * and fast::scaled_dot_product_attention stand in Attention::attend
 * (eredu-architectures/src/llama.rs:296-330).
 *
 * A page holds page_tokens tokens of every layer.  Values are int8 codes c
 * with one E8M0 byte b for each (layer, page, KV head), keys and values apart:
 * c * 2^(b - 127); b = 255 makes the page's values of that head NaN.
 * Sequence s holds lengths[s] tokens; token p lies in page
 * tables[s][p / page_tokens] at place p % page_tokens.  refs[page] counts the
 * table entries that name it; 0 is a free page.  All of it is device memory
 * that the kernels read when they run, so a captured graph decodes across
 * page borders.
 *
 * A call covers n sequences (up to 2^16), named by seqs (device int32), with `total` rows of
 * tokens: entry i has rows cu[i] .. cu[i + 1] - 1 (cu: n + 1 device int32), or
 * total / n rows where cu is NULL; they are the LAST ones of its lengths[seq]
 * tokens.  So a step is: eq_kv_extend once, then eq_kv_append and
 * eq_kv_attention in every layer.
 *
 * Nothing on the device is trusted as an index: a table entry outside
 * [0, pages) is a missing page (its tokens are not written, not attended to and
 * read as zeros), a sequence outside [0, sequences) has no tokens, cu is
 * clamped to [0, total] and a decreasing pair is an empty entry (where entries
 * then cover a row more than once, its results are not defined).  Where a
 * sequence is named twice, eq_kv_append, eq_kv_extend and eq_kv_shrink go by the
 * last entry that names it and eq_kv_fork by the last pair with that destination.
 * Calls that write a cache (append, extend, fork, shrink, free, compact) are to be
 * ordered with every other call on it, by stream order or events.
 *
 * scratch: scratch_bytes of device memory (256-byte aligned) that the call may
 * use until it has run, at least what the query beside the call returns; NULL:
 * the library's workspace of `stream`, which cannot grow while `stream` is
 * capturing and which graphs captured on one stream share, so such graphs must
 * not run at the same time.  (Calls of several host threads on one stream may
 * share it: a call keeps its launches together.)
 */
typedef struct eq_kv_cache {
    int8_t* k_codes;    /* [layers, pages, kv_heads, page_tokens, head_dim], 16-byte aligned */
    int8_t* v_codes;    /* [layers, pages, kv_heads, head_dim, page_tokens], 16-byte aligned */
    uint8_t* k_scales;  /* [layers, pages, kv_heads] */
    uint8_t* v_scales;
    int32_t* tables;    /* [sequences, width] */
    int32_t* lengths;   /* [sequences] */
    int32_t* refs;      /* [pages] */
    int32_t* missing;   /* [1]: pages that eq_kv_extend had none for, since it was last cleared (at most 2^31 - 1) */
    int64_t layers, pages, sequences, width; /* width * page_tokens <= 2^30, sequences * width < 2^31 */
    int kv_heads, page_tokens, head_dim; /* page_tokens 16, 32, 64 or 128; head_dim 64, 128 or 256 */
} eq_kv_cache;

/* Writes rows of k and v (bf16 or f16; row r at element r * stride, heads and
 * dimensions contiguous; strides multiples of 8, pointers 16-byte aligned) to
 * their sequences' last tokens in `layer`.  rope (NULL: none): [rope_positions,
 * head_dim] f32, for each position the cosines of its head_dim / 2 angles, then
 * the sines; k's pairs (d, d + head_dim / 2) are turned by them in f32 (as
 * eq_rope_attention_decode does) and rounded once, to the codes;
 * rope_positions >= width * page_tokens.
 * A page that the call begins gets the smallest b in [1, 254] with
 * max|x| <= 127 * 2^(b - 127) over its new tokens; one that held tokens keeps
 * its b or takes that larger one, and its codes are rounded to the new step (ties
 * to even, as all codes).  Steps are powers of two, so a value is off by less
 * than one step of its page's scale, however often that grew.  (One of at least
 * 63.5 * 2^122, bf16's two largest, is rounded to 2^128, which f32 has as infinity.)
 * A new value that is not finite: b = 255.  Codes behind a page's last token keep what they
 * were.  The pages written must belong to one sequence (eq_kv_extend sees to it). */
int eq_kv_append(const eq_kv_cache* cache, int64_t layer, const void* k, const void* v, int64_t k_stride,
                 int64_t v_stride, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total,
                 const float* rope, int64_t rope_positions, int dtype, eq_stream_t stream);

/* out[r, h, :] = softmax(scale * q[r, h] . K^T) . V over the tokens of row r's
 * sequence, KV head h / (n_heads / kv_heads); n_heads any multiple of kv_heads.
 * causal: row r's own position p and the ones before it, with window > 0 only
 * the last `window` of them (p included); not causal: all tokens of the
 * sequence (an encoder's states; window must be 0).  A row that sees no token
 * gives zeros.  q and out bf16 or f16 (the same), q's rows at stride q_stride as
 * in eq_kv_append, out [total, n_heads, head_dim] contiguous; rope as there,
 * for q.  Rows that no entry covers are left as they are in out.  Scores,
 * softmax sums and outputs are held in f32; q in 24 bits of each row's
 * largest magnitude, in 16 where that moves its scores with a page's keys by no more than
 * rounding moves the output (all but scores that spread by tens), probabilities in f16, values exactly where their page's
 * scale is at least 2^-29 of the sequence's largest.  scale * max|q| * max|k|
 * of a row and a page has to be below 2^124 (a score may be NaN beyond).
 * How the work is laid out follows from the entries' rows on average: give
 * long prompts and single tokens after long contexts calls of their own. */
int eq_kv_attention(void* out, const void* q, int64_t q_stride, int n_heads, const eq_kv_cache* cache, int64_t layer,
                    const int32_t* seqs, int64_t n, const int32_t* cu, int64_t total, float scale, bool causal,
                    int64_t window, const float* rope, int64_t rope_positions, int dtype, void* scratch,
                    int64_t scratch_bytes, eq_stream_t stream);
/* Scratch bytes of eq_kv_attention with these sizes (0: none), -1 for sizes it refuses. */
int64_t eq_kv_attention_scratch(const eq_kv_cache* cache, int n_heads, int64_t n, int64_t total, bool ragged);

/* The rows' keys and values, read back: k and v [total, kv_heads, head_dim] of
 * dtype (f32, f16 or bf16; bf16 holds every value exactly).  Rows whose
 * position is negative or whose page is missing are zeros; rows that no entry
 * covers are left as they are. */
int eq_kv_read(void* k, void* v, const eq_kv_cache* cache, int64_t layer, const int32_t* seqs, int64_t n,
               const int32_t* cu, int64_t total, int dtype, eq_stream_t stream);

/* Grows sequence seqs[i] by cu[i + 1] - cu[i] tokens (cu NULL: by `count`):
 * its length, and pages for them, the lowest free ones, entry by entry.  A
 * last page that is partly filled and shared is copied (all layers) into a page of its
 * sequence's own first; where all who hold it grow in this call, the last of
 * them keeps it.  A page that is not to be had (none free, or no room in the
 * table) leaves its table entry -1 and counts in *missing; the length grows
 * all the same. */
int eq_kv_extend(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, const int32_t* cu, int64_t count,
                 void* scratch, int64_t scratch_bytes, eq_stream_t stream);

/* Sequence dst[i] becomes a copy of src[i] that shares all its pages (what it
 * held before is freed); all pairs at once, from the state before the call, so
 * that beams can be permuted.  Pairs with an id out of range do nothing. */
int eq_kv_fork(const eq_kv_cache* cache, const int32_t* src, const int32_t* dst, int64_t n, void* scratch,
               int64_t scratch_bytes, eq_stream_t stream);

/* Takes the last counts[i] tokens (device int32 [n]; NULL: `count`) of sequence
 * seqs[i] back, at most all it has, and gives up the pages behind the rest:
 * the drafts of a step that were refused.  A sequence that is named twice
 * goes by the last entry.  The page that the rest ends in keeps its scale bytes, so one
 * that a value which is not finite made NaN stays so.  (A length that is lowered by
 * other means keeps its pages, and eq_kv_extend would lose them.) */
int eq_kv_shrink(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, const int32_t* counts, int64_t count,
                 eq_stream_t stream);

/* Empties the sequences: length 0, table entries -1, one reference less for each of their pages. */
int eq_kv_free(const eq_kv_cache* cache, const int32_t* seqs, int64_t n, eq_stream_t stream);

/* Moves pages so that the live ones (refs > 0) are pages 0 .. live - 1: the
 * live pages behind those move, in order, into the free ones among them, in
 * order (all layers), and tables and refs follow.  Moved-from pages keep their bytes. */
int eq_kv_compact(const eq_kv_cache* cache, void* scratch, int64_t scratch_bytes, eq_stream_t stream);

/* Scratch bytes of eq_kv_extend and eq_kv_fork with n entries and of
 * eq_kv_compact (n = 0); -1 for sizes they refuse. */
int64_t eq_kv_pages_scratch(const eq_kv_cache* cache, int64_t n);

#ifdef __cplusplus
}
#endif

#endif /* EREDU_KV_H */
