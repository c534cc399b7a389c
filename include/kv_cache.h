/* kv_cache.h - 8-bit paged key/value cache of libgpu_engine.so and the
 * attention that reads it (gfx950 build). They stand between
 * ng_rmsnorm_qkv_rope_int8 (q, k, v of the INT8 layer) and the o projection.
 * The reference keeps its paged cache and attention in 16 bits
 * (gpu/cuda/paged_attention.cu:43-596, flash_decode.cu:46-257).
 *
 * Common to all: return 0, or -1 with a message on stderr for arguments that
 * are refused before any launch (null pointers, sizes <= 0, types and layouts
 * that are not listed). Launches go to ng_get_stream(); nothing allocates,
 * synchronises the host or copies to it, so every call can be captured into a
 * graph. Everything but the structs themselves is device memory. Lengths,
 * positions and page tables are read on the device when the kernels run. The
 * max_* arguments only size a launch: longer sequences take longer, with the
 * same results (a sum over another number of slices rounds differently).
 * A page number outside [0, num_pages) is never dereferenced.
 */
#ifndef NG_KV_CACHE_H
#define NG_KV_CACHE_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* One layer's cache. A page holds page_size consecutive tokens of one
 * sequence for every head; k_codes and v_codes have num_pages * num_kv_heads *
 * page_size * head_dim bytes, k_scales and v_scales num_pages * num_kv_heads
 * floats ([page][head]): the largest magnitude of the page and head, a value
 * being code * that / 127. The order of the codes inside a page and head is the
 * library's own (ng_kv_int8_read gives them in order). head_dim is 64, 128, 192 or 256;
 * page_size 16, 32, 64 or 128; the code arrays are 16-byte aligned. */
typedef struct {
    void* k_codes;
    void* v_codes;
    void* k_scales;
    void* v_scales;
    int num_pages;
    int num_kv_heads;
    int head_dim;
    int page_size;
} ng_kv_int8_cache;

/* The page table of a cache (shared by all layers) and its pool of pages:
 * table [max_seqs][max_pages], int; entry i of a sequence's row is the page of
 * its tokens i * page_size ..; a sequence of n tokens holds exactly the first
 * ceil(n / page_size) entries, the others are -1. refs [num_pages], int: in
 * how many entries a page stands, 0 for a free one. */
typedef struct {
    void* table;
    void* refs;
    int max_seqs;
    int max_pages;
    int num_pages;
    int page_size;
} ng_kv_pages;

/* Writes new tokens. k, v: fp16 (bf16: ng_bf16_) [total_tokens, num_kv_heads,
 * head_dim]; cu_tokens [batch + 1]: sequence b's are rows cu_tokens[b] ..
 * cu_tokens[b + 1] - 1; context_lens [batch]: how many tokens the sequence
 * holds before, that is the position of the first new one; page_table
 * [batch, max_pages]. Per page and head, for K and V alike:
 *   m = largest finite |x| of the new tokens there, and of the page so far if it
 *   held tokens;
 *   where m grew: old codes = rint(code * old m / m);
 *   new codes = rint(127 x / m), infinities +-127, NaN +127; 0 where m is 0.
 * The quotients are exact before rint (ties to even). What the cache holds is
 * always finite. Codes behind a page's last token become 0, and a page's
 * magnitude while it held no token is not read. Two
 * sequences of a call must not write the same page. Tokens whose page is
 * missing (past max_pages or not a page's number) are not written; they are
 * counted into *d_dropped (device int, not cleared here; may be null). */
int ng_kv_int8_append(const ng_kv_int8_cache* cache, const void* k, const void* v, const void* cu_tokens,
                      const void* context_lens, const void* page_table, int batch, int max_pages,
                      int total_tokens, int max_tokens, void* d_dropped);
int ng_bf16_kv_int8_append(const ng_kv_int8_cache* cache, const void* k, const void* v, const void* cu_tokens,
                           const void* context_lens, const void* page_table, int batch, int max_pages,
                           int total_tokens, int max_tokens, void* d_dropped);

/* Reads tokens back: rows cu_tokens[b] .. cu_tokens[b + 1] - 1 of k and v
 * [total_tokens, num_kv_heads, head_dim] become RN(code * RN(m / 127)) of
 * sequence b's tokens from position starts[b] on (fp16 or bf16). Tokens whose page is
 * missing read as 0; other rows are left as they are. */
int ng_kv_int8_read(const ng_kv_int8_cache* cache, void* k, void* v, const void* cu_tokens, const void* starts,
                    const void* page_table, int batch, int max_pages, int total_tokens, int max_tokens);
int ng_bf16_kv_int8_read(const ng_kv_int8_cache* cache, void* k, void* v, const void* cu_tokens, const void* starts,
                         const void* page_table, int batch, int max_pages, int total_tokens, int max_tokens);

/* Attention over the cache: out and q fp16 (bf16: ng_bf16_) [total_q,
 * num_q_heads, head_dim], query head h on key/value head h / (num_q_heads /
 * num_kv_heads); cu_q [batch + 1] as cu_tokens above; kv_lens [batch]: tokens
 * of the sequence in the cache, the queries' own included. The n queries of a
 * sequence are its last n tokens: query i stands at p = kv_len - n + i and sees
 * token j (0 <= j <= p) if window is 0, or j > p - window, or j < sinks:
 *   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(softmax_scale q . k_j)
 * A query that sees nothing (p < 0, pages missing) gives 0. out may be q, and
 * must not overlap it otherwise.
 * With a workspace, long sequences are shared out over the GPU and joined by a
 * second launch. ng_kv_int8_attention_workspace says how many bytes that takes
 * for at most batch sequences of at most max_q_len queries and max_kv_len
 * tokens (0 if it never would); with fewer bytes, or none (null), a sequence is
 * shared out less, or not. Calls that overlap, and graphs that may, each need a
 * workspace of their own (16-byte aligned).
 * num_q_heads is a multiple of num_kv_heads; q and out are 16-byte aligned;
 * softmax_scale is >= 0 and below FLT_MAX / log2(e); window and sinks are >= 0.
 * Scores, sums and the output are held in 32 bits. With more than 32 queries
 * times heads of a group to a sequence (max_q_len), a weight times its page's V
 * scale is rounded to 11 bits, and to 2^-32 of the largest V scale that the
 * query sees; with fewer, to 22 bits and 2^-40. A page whose V lies below 2^-126 (bf16's
 * subnormals) may count as zeros. */
size_t ng_kv_int8_attention_workspace(const ng_kv_int8_cache* cache, int num_q_heads, int batch, int max_q_len,
                                      int max_kv_len);
int ng_kv_int8_attention(void* out, const void* q, const ng_kv_int8_cache* cache, const void* cu_q,
                         const void* kv_lens, const void* page_table, int batch, int max_pages, int total_q,
                         int max_q_len, int max_kv_len, int num_q_heads, float softmax_scale, int window,
                         int sinks, void* workspace, size_t workspace_bytes);
int ng_bf16_kv_int8_attention(void* out, const void* q, const ng_kv_int8_cache* cache, const void* cu_q,
                              const void* kv_lens, const void* page_table, int batch, int max_pages, int total_q,
                              int max_q_len, int max_kv_len, int num_q_heads, float softmax_scale, int window,
                              int sinks, void* workspace, size_t workspace_bytes);

/* Copies page src[i] to page dst[i], codes and scales, for i < count in each of
 * the num_caches (1 .. 64) caches, which must agree in their sizes (a host array:
 * one per layer). Pairs with a page number outside [0, num_pages) are skipped
 * (-1: nothing to copy); count is at most 2^30. No page may be the destination
 * of two pairs, or of one and the source of another. */
int ng_kv_int8_copy_pages(const ng_kv_int8_cache* caches, int num_caches, const void* src, const void* dst,
                          int count);

/* Gives every sequence r < max_seqs, which holds old_lens[r] tokens, the pages
 * for new_lens[r] of them (no change where new_lens[r] <= old_lens[r]). Fresh
 * pages are the free ones in rising order, given out by rising r and position.
 * Where tokens will be added to a partly filled page that stands in more than
 * one entry, the row gets a fresh page in its place, and copy_src[r],
 * copy_dst[r] say what to copy into it (ng_kv_int8_copy_pages); they are -1
 * elsewhere. All or nothing: *d_missing becomes how many free pages or table
 * entries were too few, and unless it is 0 nothing else changes, and
 * copy_src and copy_dst are all -1. copy_src, copy_dst: int [max_seqs].
 * max_seqs is at most 8192. */
int ng_kv_pages_grow(const ng_kv_pages* pages, const void* old_lens, const void* new_lens, void* copy_src,
                     void* copy_dst, void* d_missing);

/* Replaces the set of sequences: row r of new_table [max_seqs][max_pages]
 * becomes the row of sequence parents[r] (any number of rows may share one;
 * -1, or any number outside [0, max_seqs): an empty row), new_lens[r] its
 * length lens[parents[r]] (or 0). refs then counts the entries of new_table;
 * pages of sequences that nobody took are free. table itself is not changed;
 * new_table must not overlap it, nor new_lens lens. */
int ng_kv_pages_fork(const ng_kv_pages* pages, void* new_table, const void* parents, const void* lens,
                     void* new_lens);

/* Shortens every sequence r from old_lens[r] to keep_lens[r] tokens (0 frees
 * it; no change where keep_lens[r] >= old_lens[r]): entries behind its pages
 * become -1, their reference counts fall by one. */
int ng_kv_pages_free(const ng_kv_pages* pages, const void* old_lens, const void* keep_lens);

/* Moves the used pages to the front of the pool: with n used pages, the k-th
 * used page at or behind n takes the place of the k-th free page before n.
 * refs and every entry of table follow; copy_src[k], copy_dst[k] say what to
 * copy (in every layer, before the pages are next used), -1 behind the last
 * move; *d_moves becomes the number of moves. capacity, the ints that
 * copy_src and copy_dst have, is at least num_pages / 2 and at most 2^30. */
int ng_kv_pages_compact(const ng_kv_pages* pages, void* copy_src, void* copy_dst, int capacity, void* d_moves);

#ifdef __cplusplus
}
#endif

#endif /* NG_KV_CACHE_H */
