/*
 * mugen_attn_paged.h -- the paged K/V cache of the attention library: appending
 * with the rotation on the way, decode / verify / prefill attention over 16- and
 * 8-bit pages, and the choice of the pages a query reads.  The conventions of
 * mugen_attn.h hold (device pointers, caller's workspaces, streams, status codes).
 * Kernel names for mugen_attn_timing_read: "kv_paged_append",
 * "gqa_decode_paged", "gqa_decode_paged_combine", "page_score", "page_select",
 * "paged_gather" (then the prefill's own).
 */
#ifndef MUGEN_ATTN_PAGED_H
#define MUGEN_ATTN_PAGED_H

#include "mugen_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Paged K/V cache.  No counterpart in the reference (its caches are one
 * contiguous buffer per layer, transformer.cpp:3382-3394): sequences of a
 * serving batch share one pool of pages per layer, a page holding page_tokens
 * consecutive tokens of one sequence for every kv head.  Token t of sequence b
 * is in page page_table[b][t / page_tokens] at slot t % page_tokens.
 *
 * page_bits 16: pages of `dtype`.
 *   k_pages, v_pages  [n_pages][n_kv_heads][page_tokens][head_dim]
 * page_bits 8: whole pages only, as E4M3 codes with one power-of-two scale per
 * (page, kv head) and tensor, value = code * 2^(exp - 127); the tokens behind a
 * sequence's last whole page are in a 16-bit ring (token t at slot t % ring):
 *   k_pages           [n_pages][n_kv_heads][page_tokens][head_dim] bytes
 *   v_pages           [n_pages][n_kv_heads][page_tokens/32][head_dim][32] bytes:
 *                     32 tokens of one dim are adjacent, as the P.V product
 *                     takes them
 *   k_exp, v_exp      uint8 [n_pages][n_kv_heads]
 *   tail_k, tail_v    [n_seq][ring][n_kv_heads][head_dim] (dtype),
 *                     tail_seq_stride elements apart
 * A page's codes are round-to-nearest-even from the 16-bit rows, its exponent
 * the least whose range holds the page's largest finite magnitude (448 * 2^e), so
 * the page depends on its tokens only, not on how they were appended.  A value
 * that is not finite becomes NaN.  (A power of two costs E4M3, itself a float,
 * no precision, and makes the values exact in 16 bits.)
 * k_range (optional) [n_pages][n_kv_heads][2][head_dim] (dtype): the minimum and
 * the maximum of each dim over a whole page's keys, for
 * mugen_attn_page_select.
 *
 * page_table entries past a sequence's pages may be anything.  An entry outside
 * [0, n_pages) is a page that is not there: attention leaves its tokens out,
 * an append drops them.  No two sequences may append to one page (full pages
 * may be shared).
 *
 * Supported: head_dim 64, 128, 256; page_tokens 32, 64, 128; max_seq_len up to 2^27; n_heads /
 * n_kv_heads in [1, 16]; dtype F16 or BF16; all buffers 16-byte aligned.
 */
typedef struct mugen_attn_kv_pages {
    void* k_pages;
    void* v_pages;
    void* k_exp;
    void* v_exp;
    void* tail_k;
    void* tail_v;
    void* k_range;             /* optional */
    const int32_t* page_table; /* device [n_seq], table_stride entries apart */
    int64_t table_stride;      /* >= ceil(max_seq_len / page_tokens) */
    int64_t tail_seq_stride;
    int32_t n_seq;
    int32_t n_pages;
    int32_t page_tokens;
    int32_t page_bits; /* 16 or 8 */
    int32_t ring;      /* page_bits 8: a power of two > page_tokens */
    int32_t n_kv_heads;
    int32_t head_dim;
    int32_t max_seq_len;
    int32_t dtype; /* mugen_attn_dtype of queries and 16-bit rows */
} mugen_attn_kv_pages;

/*
 * Append n_new tokens to each sequence of the cache: K rotated, K and V
 * written, and (q non-null) the tokens' queries rotated into q_out on the way.
 *   k_new, v_new  rows b * n_new + j, k_stride / v_stride elements apart, each
 *                 [n_kv_heads][head_dim]; q likewise [n_heads][head_dim] (slices
 *                 of one fused projection are taken as they are)
 *   q_out         [n_seq][n_new][n_heads][head_dim]
 *   seq_lens      device [n_seq]: tokens held before; token j goes to
 *                 position seq_lens[b] + j
 *   new_lens      optional device [n_seq]: sequence b gets new_lens[b] (0 ..
 *                 n_new) tokens; its other rows are neither read nor written
 *   seq_lens_out  optional device [n_seq]: tokens held after (must not alias
 *                 seq_lens: every layer's call reads the same lengths)
 * Rows past max_seq_len are dropped (their q_out rows are left as they were).
 * Rotation: NeoX pairs (i, i + rope_dim/2) of the first rope_dim dims (0: none)
 * by position * frequency, the frequencies of mugen_attn_rope_params over
 * rope_dim; the angle is formed in 64 bits, so that far positions keep their
 * phase, the result is rounded to dtype once.
 * With page_bits 8 the pages that these tokens fill are quantised, from the ring
 * and the new rows, and the newest `ring` new rows go to the ring.  After a step whose
 * last tokens are rejected, seq_lens may go back, as long as the rows of the page
 * that is open then are still in the ring (it holds the last `ring` positions ever
 * written, so any ring - page_tokens tokens behind the furthest): appends write the
 * same pages again.  Requires rope_dim a multiple of 16 up to head_dim.
 */
typedef struct mugen_attn_kv_paged_append_args {
    mugen_attn_kv_pages store;
    const void* k_new;
    const void* v_new;
    const void* q; /* optional */
    void* q_out;
    const int32_t* seq_lens;
    const int32_t* new_lens; /* optional */
    int32_t* seq_lens_out;   /* optional */
    int64_t k_stride;
    int64_t v_stride;
    int64_t q_stride;
    int32_t n_new;
    int32_t n_heads; /* of q */
    int32_t rope_dim;
    mugen_attn_rope_params rope;
} mugen_attn_kv_paged_append_args;
int mugen_attn_kv_paged_append(const mugen_attn_kv_paged_append_args* args, void* stream);

/*
 * GQA attention of q_len new tokens per sequence over the paged cache (decode:
 * q_len 1; speculative verify: a few, causal among them): the rules of
 * mugen_attn_gqa_decode.
 *   q, out    [n_seq][q_len][n_heads][head_dim]; q in the store's dtype
 *   seq_lens  device [n_seq]: tokens held INCLUDING the new ones
 *   q_lens    optional device [n_seq]: sequence b has q_lens[b] (0 .. q_len) new
 *             tokens; the output rows behind them are left as they were.
 *             Query i sees the first seq_lens[b] - q_lens[b] + i + 1 tokens
 *             (none: a zero row)
 *   pages     optional device [n_seq][q_len][n_kv_heads][n_select]: the only
 *             logical pages each query reads, ascending (mugen_attn_page_select);
 *             an entry that is not above the one before it, or that the query does
 *             not see, is left out
 * A value of V that a query does not see does not reach its output, whatever it
 * is (infinities and NaN too).
 */
typedef struct mugen_attn_gqa_decode_paged_args {
    mugen_attn_kv_pages store;
    const void* q;
    void* out;
    const int32_t* seq_lens;
    const int32_t* q_lens; /* optional */
    const int32_t* pages;  /* optional */
    int32_t n_select;      /* entries per list (with pages) */
    int32_t q_len;         /* 1 .. MUGEN_ATTN_PAGED_MAX_Q */
    int32_t n_heads;
    int32_t num_splits; /* 0: automatic; at most 128 */
    float scale;        /* <= 0: 1 / sqrt(head_dim) */
    int32_t out_dtype;
    const int32_t* seq_lens_host; /* as in mugen_attn_gqa_decode_args */
} mugen_attn_gqa_decode_paged_args;
#define MUGEN_ATTN_PAGED_MAX_Q 64
size_t mugen_attn_gqa_decode_paged_workspace_size(const mugen_attn_gqa_decode_paged_args* args);
int mugen_attn_gqa_decode_paged(const mugen_attn_gqa_decode_paged_args* args, void* workspace,
                                size_t workspace_bytes, void* stream);

/*
 * Choose the pages that each query reads, by a cheap score.  For query i of
 * sequence b, kv head j and whole page p:
 *   score = sum over dims d of neg[d] * min_p[d] + pos[d] * max_p[d]
 * where neg and pos are the sums over the group's heads of the negative and of the
 * positive q[h][d] (min_p, max_p from k_range): for finite ranges the sum over
 * heads and dims of max(q * min_p, q * max_p), an upper bound of the sum of the
 * group's logits with any key of the page.  In 64 bits, so that the choice does not
 * hang on the order of the sums.  The first n_first and the newest n_last pages the
 * query sees are always taken (the newest one is not whole, so n_last >= 1),
 * then the highest scores, equal ones from the lowest page on, until n_select
 * pages are taken or all are.  A NaN score counts as the highest (a
 * range that is not finite makes one where neg or pos is 0).
 *   pages  device [n_seq][q_len][n_kv_heads][n_select]: the chosen logical pages,
 *          ascending, -1 behind them; the lists behind q_lens[b] are left as
 *          they were
 * A page whose page_table entry is not valid scores lowest.
 * Requires n_first + n_last <= n_select, max_seq_len <= 16384 pages.
 */
typedef struct mugen_attn_page_select_args {
    mugen_attn_kv_pages store; /* k_range, page_table and the shape */
    const void* q;             /* as in mugen_attn_gqa_decode_paged_args */
    int32_t* pages;
    const int32_t* seq_lens;
    const int32_t* q_lens; /* optional */
    int32_t q_len;
    int32_t n_heads;
    int32_t n_select;
    int32_t n_first;
    int32_t n_last;
} mugen_attn_page_select_args;
size_t mugen_attn_page_select_workspace_size(const mugen_attn_page_select_args* args);
int mugen_attn_page_select(const mugen_attn_page_select_args* args, void* workspace, size_t workspace_bytes,
                           void* stream);

/*
 * Causal prefill of one sequence's chunk over the paged cache: the rules of
 * mugen_attn_gqa_prefill (BF16 V within +-65504), the keys being those the cache
 * holds once the chunk is appended (whole pages of an 8-bit store as their codes'
 * values).  Chunks of few rows read the pages in place, longer ones from a copy
 * in the workspace; every page_table entry up to start_pos + n_tokens has to be
 * a page (one that is not is never followed, but counts as zero rows in the
 * copy and as absent tokens in place).
 *   q, out   [n_tokens][n_heads][head_dim]; token i sees start_pos + i + 1 keys
 *   seq      the sequence: row of page_table and of the tail ring, which hold
 *            start_pos + n_tokens tokens
 */
typedef struct mugen_attn_gqa_prefill_paged_args {
    mugen_attn_kv_pages store;
    const void* q;
    void* out;
    int32_t seq;
    int32_t n_tokens;
    int32_t start_pos;
    int32_t n_heads;
    float scale;
    int32_t out_dtype;
} mugen_attn_gqa_prefill_paged_args;
size_t mugen_attn_gqa_prefill_paged_workspace_size(const mugen_attn_gqa_prefill_paged_args* args);
int mugen_attn_gqa_prefill_paged(const mugen_attn_gqa_prefill_paged_args* args, void* workspace,
                                 size_t workspace_bytes, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* MUGEN_ATTN_PAGED_H */
