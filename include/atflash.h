/*
 * atflash C ABI: per-RoPE-wavelength windowed attention on AMD MI355X (gfx950).
 *
 * Plain pointers and sizes only.  Every tensor pointer is a device pointer
 * (HIP), allocated and owned by the caller; `stream` is a hipStream_t passed as
 * void* (NULL = default stream).  All work is enqueued asynchronously on
 * `stream`; no entry point synchronises the device.  Every entry point returns
 * ATF_OK (0) or an ATF_ERR_* code; atf_last_error() then describes the failure
 * (per calling thread).
 *
 * Window tables.  `zhi` is a HOST array of ATF_LEVELS int32 entries: zhi[i] is
 * the largest causal key distance at which 16-dim level i is still read
 * (window_tables/atflash_window.py:85-108).  zhi[0] is the table's cap and must
 * be >= the longest causal distance of the call (prefill nk - 1, decode
 * max_seq_len - 1); a smaller cap is refused with ATF_ERR_INVALID, since it
 * would drop levels the rule keeps.  NULL means window OFF: plain causal attention,
 * every level read at every distance.  Level l holds RoPE pairs
 * r in [64-8(l+1), 64-8l) (dims r and r+64 of the half-split layout).
 * The decode also takes the FlashInfer window port's finer table `zhi_slice`
 * (atf_decode_paged_slices_bf16): ATF_SLICES int32 entries, zhi_slice[s] the
 * largest key age (seq_len - 1 - position) at which 8-dim slice s (RoPE pairs
 * r in [64-4(s+1), 64-4s), four pairs in wavelength order) is still read
 * (kernels/flashinfer_port/fiwin_common.py:35-47); level l is slices 2l, 2l+1.
 *
 * Paged KV cache (one layer): pages of ATF_PAGE_SIZE = 16 tokens.
 *   kv_cache  bf16 [num_pages][num_kv_heads][2][2048]: one 8 KB block per
 *             (page, kv head), 16-byte aligned,
 *     [0]  V half: [128 dims][16 token slots] (V transposed)
 *     [1]  K half: [16 slices][16 tokens][8 dims] (slice s: half-split dims
 *          [64-4(s+1), 64-4s) then the same + 64; sorted pair dims [8s, 8s+8))
 * written by atf_kv_write_bf16 (RoPE applied to K there); page_table is int32
 * [batch][max_pages] of page ids.  Token slots of a page that were never written
 * may hold any finite value.  A windowed read of a page is one contiguous run:
 * the V half and the in-window prefix of the K half.
 *
 * Paged cache of 8-bit floats (one layer), the same pages with half the bytes:
 *   kv_cache  e4m3 codes [num_pages][num_kv_heads][2][2048]: one 4 KB block per
 *             (page, kv head), 16-byte aligned,
 *     [0]  V half: [2 j][4 g][16 r][4 d][4 t] = dim 8r + 4j + d of token 4g + t
 *     [1]  K half: [8 levels][16 tokens][slices 2l, 2l + 1][8 dims]
 *   kv_exps   int8 [num_pages][num_kv_heads][2]: V's and K's exponent, between
 *             ATF_Q8_MIN_EXP and ATF_Q8_MAX_EXP; a code c stands for c 2^exponent
 * written by atf_kv_write_q8.
 *
 * RoPE.  rope_cs, when not NULL, is fp32 [rope_max_pos][64][2] holding
 * (cos, sin) of position * inv_freq[r] (HF rotate-half convention); NULL means
 * the inputs are already rotated.  Layout ATF_LAYOUT_SORTED_PAIR (the
 * reference's wavelength-sorted layout) requires rope_cs == NULL.
 */
#ifndef ATFLASH_H_
#define ATFLASH_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ATF_ABI_VERSION 3
#define ATF_HEAD_DIM 128
#define ATF_LEVELS 8
#define ATF_SLICES 16
#define ATF_PAGE_SIZE 16
#define ATF_LAYOUT_HALF_SPLIT 0
#define ATF_LAYOUT_SORTED_PAIR 1
/* Tile quantization of the window (the block_m/block_n the oracle must use). */
#define ATF_PREFILL_BLOCK_M 32
#define ATF_PREFILL_BLOCK_N 32
#define ATF_DECODE_BLOCK_N 16
#define ATF_MAX_GQA_GROUP 16
#define ATF_Q8_MIN_EXP (-110)
#define ATF_Q8_MAX_EXP 119
#define ATF_LOGITS_BF16 0
#define ATF_LOGITS_FP16 1
#define ATF_LOGITS_FP32 2
#define ATF_MAX_TOP 64                /* alternatives of atf_token_logprobs */
#define ATF_MAX_SHARED_PAGES (1 << 19) /* pool of atf_select_tables and atf_compact_tables */

enum {
  ATF_OK = 0,
  ATF_ERR_INVALID = 1,     /* bad argument (shape, stride, alignment, table) */
  ATF_ERR_UNSUPPORTED = 2, /* valid request this build does not support */
  ATF_ERR_LAUNCH = 3,      /* HIP launch or runtime error */
  ATF_ERR_WORKSPACE = 4    /* workspace missing or too small */
};

int atf_abi_version(void);
const char* atf_last_error(void);

/*
 * Write n_tokens tokens of each of `batch` sequences into the paged cache.
 * Source token t of sequence b sits at absolute position start_pos[b] + t
 * (start_pos: device int32 [batch]) and goes to page
 * page_table[b][pos / 16], slot pos % 16.  K is rotated with rope_cs at that
 * position.  Source strides are in elements; the last dim is contiguous.
 *
 * Positions live in device memory (start_pos), so they are checked in the
 * kernel, not here, and a token that cannot be placed is SKIPPED without an
 * error: a negative position, a position at or past rope_max_pos (when rope_cs
 * is given), a page index pos / 16 at or past max_pages, or a page-table entry
 * outside [0, num_pages).  Attention over such a token would read whatever the
 * slot held before, so callers must keep positions inside the page table and
 * the RoPE table (atflash.cache.PagedKVCache checks this on the host).
 *
 * Replaces the reference's RoPE + head-dim permutation patch and HF cache append
 * (e2e_pipeline/atflash_e2e_fafi.py:186-192, 101-119).
 */
int atf_kv_write_bf16(void* kv_cache, int num_pages, int num_kv_heads,
                      const void* k_src, int64_t ks_b, int64_t ks_t, int64_t ks_h,
                      const void* v_src, int64_t vs_b, int64_t vs_t, int64_t vs_h,
                      int batch, int n_tokens, const int32_t* start_pos,
                      const int32_t* page_table, int max_pages,
                      const float* rope_cs, int rope_max_pos, int layout, void* stream);

/*
 * atf_kv_write_bf16 for packed rows: sequence b's tokens are rows cu_tokens[b]
 * to cu_tokens[b + 1] - 1 (device int32 [batch + 1]) of k_src and v_src, which have
 * total_tokens rows; at most max_tokens of a sequence are written.  Rows outside
 * [0, total_tokens) are not read.  It has no counterpart in the reference.
 */
int atf_kv_write_packed_bf16(void* kv_cache, int num_pages, int num_kv_heads,
                             const void* k_src, int64_t ks_t, int64_t ks_h,
                             const void* v_src, int64_t vs_t, int64_t vs_h,
                             int batch, const int32_t* cu_tokens, int total_tokens, int max_tokens,
                             const int32_t* start_pos, const int32_t* page_table, int max_pages,
                             const float* rope_cs, int rope_max_pos, int layout, void* stream);

/*
 * The writer of the cache of 8-bit floats: rows, positions, RoPE and skips as
 * atf_kv_write_bf16's (cu_tokens NULL) or atf_kv_write_packed_bf16's (cu_tokens given,
 * n_tokens the most of a sequence, batch strides 0).  Per page, kv head and half the
 * exponent is the smallest e with every magnitude at most 448 2^e (between the
 * limits above), and the codes are the values times 2^-e, rotated in fp32 and
 * rounded once, to nearest even.
 *   A call that writes a page's first slot begins the page anew: its exponent is
 * that of the written tokens.  One that starts inside a page keeps the tokens
 * before its first: the exponent is at least the page's, and where it grows the
 * kept codes move to it (exact, save those that become subnormal).  The slots
 * behind the call's last token in its last page become zero: sequences are
 * appended to, and the codes that lay behind are forgotten.  Not so the exponent of a
 * page that a call starts inside: tokens that the call overwrites may have raised it,
 * and the page's codes stay as coarse as they made it.  Infinities and NaN become the
 * NaN code and count for no exponent.  Two sequences of a call must not write the
 * same page.  batch and num_kv_heads are at most 65535.
 */
int atf_kv_write_q8(void* kv_cache, int8_t* kv_exps, int num_pages, int num_kv_heads,
                    const void* k_src, int64_t ks_b, int64_t ks_t, int64_t ks_h,
                    const void* v_src, int64_t vs_b, int64_t vs_t, int64_t vs_h,
                    int batch, int n_tokens, const int32_t* cu_tokens, int total_tokens,
                    const int32_t* start_pos, const int32_t* page_table, int max_pages,
                    const float* rope_cs, int rope_max_pos, int layout, void* stream);

/*
 * Pages of the 8-bit cache as bf16 pages, exactly (a code times a power of two is
 * a bf16 number): entry (b, p), p < n_pages, of the page table (rows of max_pages) to
 * block b * n_pages + p of out (bf16 [batch * n_pages][num_kv_heads][2][2048]), and
 * that number to out_table (int32 [batch][n_pages]).  An entry outside
 * [0, num_pages), or past the seq_lens[b] tokens of its sequence (seq_lens null: none
 * is), gets -1 there and leaves its block as it is.  With out and out_table
 * atf_prefill_bf16 and atf_prefill_packed_bf16 attend to an 8-bit cache.
 */
int atf_kv_expand_q8(void* out, int32_t* out_table, const void* kv_cache, const int8_t* kv_exps, int num_pages,
                     int num_kv_heads, const int32_t* page_table, int batch, int max_pages, int n_pages,
                     const int32_t* seq_lens, void* stream);

/*
 * The same with every page in the block of its own number: out is bf16
 * [num_pages][num_kv_heads][2][2048], read with the caller's own page table.  It
 * takes as much memory as the pool has pages, where atf_kv_expand_q8 takes batch *
 * n_pages: for n_pages far past the lengths, and for pages that sequences share.
 */
int atf_kv_expand_q8_pages(void* out, const void* kv_cache, const int8_t* kv_exps, int num_pages, int num_kv_heads,
                           const int32_t* page_table, int batch, int max_pages, int n_pages, const int32_t* seq_lens,
                           void* stream);

/*
 * Windowed causal GQA prefill: out[b, i, h, :] = attention of query row i
 * (absolute position q_offset + i) over keys 0..q_offset+i of sequence b read
 * from the paged cache (nk keys present, q_offset + nq <= nk).  q/out are bf16
 * [batch][nq][num_q_heads][128] with element strides (last dim contiguous;
 * q 16-byte aligned with strides multiples of 8, out 8-byte aligned with
 * strides multiples of 4).  lse (nullable) receives fp32 [batch][num_q_heads][nq] natural-log
 * log-sum-exp of the scaled scores.  Q is rotated with rope_cs at load.
 *
 * Replaces flash_attn.cute.interface._flash_attn_fwd(q, k, v, causal=True,
 * atflash_window_zhi=zhi) of the FA4 window port (call sites
 * microbench/b1_correctness.py:84-85, e2e_pipeline/atflash_e2e_fafi.py:118-119).
 */
int atf_prefill_bf16(void* out, int64_t o_sb, int64_t o_st, int64_t o_sh, float* lse,
                     const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                     const void* kv_cache, int num_pages,
                     const int32_t* page_table, int max_pages,
                     int batch, int nq, int nk, int q_offset, int num_q_heads, int num_kv_heads,
                     const int32_t* zhi, float sm_scale, const float* rope_cs, int rope_max_pos,
                     int layout, void* stream);

/*
 * The prefill of packed rows: sequences of different lengths in one call, their
 * lengths in device memory.  Sequence b's queries are rows cu_seqlens[b] to
 * cu_seqlens[b + 1] - 1 (device int32 [batch + 1], not decreasing) of q and out
 * (bf16 [total_q][num_q_heads][128], strides as atf_prefill_bf16's), the last of
 * its seq_lens[b] keys (device int32 [batch]; NULL: as many keys as queries, whole
 * prompts) in the paged cache.  lse (nullable): fp32 [num_q_heads][total_q].  A
 * sequence's rows get the bits of an atf_prefill_bf16 call of its own.  Rows outside
 * every sequence are left as they are, and so are those of a sequence with more
 * queries than keys or more than max_seq_len keys.
 *   atf_prefill_plan first lists the query tiles in `plan` (device memory of
 * atf_prefill_plan_bytes, no initialisation needed), heaviest first; one plan serves
 * every layer of a step.  Small calls need none (0 bytes; the call then does nothing).
 * A plan made for other lengths gives rows that are not computed, never an access out
 * of bounds.
 */
size_t atf_prefill_plan_bytes(int batch, int total_q, int num_q_heads);
int atf_prefill_plan(void* plan, size_t plan_bytes, const int32_t* cu_seqlens, const int32_t* seq_lens, int batch,
                     int total_q, int max_seq_len, int num_q_heads, void* stream);
int atf_prefill_packed_bf16(void* out, int64_t o_st, int64_t o_sh, float* lse,
                            const void* q, int64_t q_st, int64_t q_sh, const void* kv_cache, int num_pages,
                            const int32_t* page_table, int max_pages,
                            const int32_t* cu_seqlens, const int32_t* seq_lens, int batch, int total_q,
                            int max_seq_len, int num_q_heads, int num_kv_heads,
                            const int32_t* zhi, float sm_scale, const float* rope_cs, int rope_max_pos, int layout,
                            const void* plan, size_t plan_bytes, void* stream);

/*
 * Causal attention of whole prompts packed one after the other, without a cache of
 * the caller's: q and out as above, k and v bf16 [total_q][num_kv_heads][128] rows
 * (strides multiples of 8, 16-byte aligned) of the same sequences, at most max_seqlen
 * rows each (a longer sequence is not computed).  K and V are written to pages of
 * the workspace (RoPE there, with rope_cs), the tiles are listed where a list is
 * needed, the attention runs: two or three kernels.  The workspace needs no
 * initialisation; calls that share one must be ordered on one stream.
 */
size_t atf_flash_packed_workspace_bytes(int batch, int total_q, int max_seqlen, int num_q_heads, int num_kv_heads);
int atf_flash_packed_bf16(void* out, int64_t o_st, int64_t o_sh, float* lse,
                          const void* q, int64_t q_st, int64_t q_sh,
                          const void* k, int64_t ks_t, int64_t ks_h, const void* v, int64_t vs_t, int64_t vs_h,
                          const int32_t* cu_seqlens, int batch, int total_q, int max_seqlen,
                          int num_q_heads, int num_kv_heads, const int32_t* zhi, float sm_scale,
                          const float* rope_cs, int rope_max_pos, int layout,
                          void* workspace, size_t workspace_bytes, void* stream);

/*
 * Block tables and slot maps of a step from request lengths, on the GPU.  Sequence b
 * has seq_lens[b] tokens and gets new_lens[b] more (negative: none).  The pages it
 * needs beyond those of its tokens are taken from the end of the free pages
 * (free_pages[0 .. *free_count - 1], an array of num_free entries), sequence by
 * sequence, and entered into its row of page_table ([batch][max_pages], in place;
 * pages past max_pages are not taken).  Written:
 *   seq_lens_out [batch]    lengths afterwards
 *   free_left    [1]        *free_count less the pages taken; negative: so many were
 *                           missing, their entries are -1
 *   cu_seqlens   [batch+1]  first new token of each sequence in the packed order
 *   positions    [total_tokens], slots [total_tokens] (int64): position of each new
 *                           token in its sequence, and page * 16 + position % 16; slot -1
 *                           where it has no page of the pool (num_pages); both -1 past
 *                           the last new token.  New tokens past total_tokens are not
 *                           listed.
 * seq_lens and free_count are read only, so that a call can be repeated.  batch is at
 * most 8191 and batch * max_pages at most 2^30; the new tokens of a call and their
 * positions are below 2^31 (other lengths give entries without a meaning, never an
 * access out of bounds).
 */
int atf_extend_tables(int32_t* page_table, int max_pages, const int32_t* seq_lens, const int32_t* new_lens,
                      const int32_t* free_pages, int num_free, const int32_t* free_count, int batch, int total_tokens,
                      int num_pages, int32_t* seq_lens_out, int32_t* free_left, int32_t* cu_seqlens, int32_t* positions,
                      int64_t* slots, void* stream);

/*
 * The pages of the sequences rows[0 .. n_rows - 1] (device int32) go back to the end
 * of the free pages, sequence by sequence; their page-table rows become -1 and their
 * lengths 0, *free_count grows (to num_free at most).  Rows outside [0, batch) and
 * repeated rows give nothing.
 */
int atf_release_tables(int32_t* page_table, int max_pages, int32_t* seq_lens, int32_t* free_pages, int num_free,
                       int32_t* free_count, const int32_t* rows, int n_rows, int batch, int num_pages, void* stream);

/*
 * RMS norm of each head's query and key rows and the rotation of their positions in one
 * pass: y = x (mean(x^2) + eps)^-1/2 w over a row's 128 dims, then rotate-half RoPE of y by
 * rope_cs at the row's position.  q and k are bf16 [rows][heads][128] (strides in
 * elements, multiples of 8; last dim contiguous; 16-byte aligned), half-split; q_out and
 * k_out bf16 [rows][heads][128], contiguous.  Weights [128], bf16 or fp32
 * (weights_fp32), not needed where there are no heads.  positions: device int32 [rows].
 * With rope_cs NULL rows are normed only.  A row whose position lies outside
 * [0, rope_max_pos) is left as it is in the outputs.  At most 2^25 rows.  fp32 throughout, one
 * rounding; rows of any size, also where their squares leave fp32's range (eps may be 0; a row of
 * zeros is then NaN).
 */
int atf_qk_norm_rope_bf16(void* q_out, const void* q, int64_t q_st, int64_t q_sh, int num_q_heads,
                          void* k_out, const void* k, int64_t k_st, int64_t k_sh, int num_k_heads,
                          const void* q_weight, const void* k_weight, int weights_fp32, float eps,
                          int rows, const int32_t* positions, const float* rope_cs, int rope_max_pos, void* stream);

/*
 * The same with the keys written, beside their values, into the paged cache: packed rows as
 * atf_kv_write_packed_bf16's (sequence b's rows cu_tokens[b] .. cu_tokens[b + 1] - 1 at
 * positions from start_pos[b] on), with its skips, into the bf16 cache (kv_exps NULL)
 * or the cache of 8-bit floats, with atf_kv_write_q8's rules for pages.  q's rows are those
 * of the same tokens, normed and rotated into q_out [total_tokens][num_q_heads][128]; those
 * whose position is negative or past the RoPE table, and rows outside every sequence, are left as
 * they are.  The keys are normed and rotated in fp32 and rounded once; q_out has the bits of
 * atf_qk_norm_rope_bf16, and so have the bf16 cache's keys.  The attention then takes
 * q_out with rope_cs NULL.  No counterpart in the reference.
 */
int atf_qk_norm_write(void* q_out, const void* q, int64_t q_st, int64_t q_sh, int num_q_heads,
                      void* kv_cache, int8_t* kv_exps, int num_pages, int num_kv_heads,
                      const void* k_src, int64_t ks_t, int64_t ks_h, const void* v_src, int64_t vs_t, int64_t vs_h,
                      const void* q_weight, const void* k_weight, int weights_fp32, float eps,
                      int batch, const int32_t* cu_tokens, int total_tokens, int max_tokens,
                      const int32_t* start_pos, const int32_t* page_table, int max_pages,
                      const float* rope_cs, int rope_max_pos, void* stream);

/*
 * Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits
 * (no counterpart in the reference).  logits: [rows][vocab] of logits_type (ATF_LOGITS_*), rows
 * `stride` elements apart, any alignment.  With p = softmax of a row in natural logarithms:
 *   logprobs     fp32 [rows][n_tokens]  log p of tokens[row][i] (device int64); 0 for a
 *                                       negative token (padding), NaN for one past the vocabulary
 *   entropy      fp32 [rows]            - sum p log p
 *   top_ids      int64 [rows][top], top_logprobs fp32 [rows][top]: the `top` likeliest tokens, best
 *                                       first, of equal logits the lowest id first
 * top is at most ATF_MAX_TOP and at most vocab.  Logits of -inf have probability 0; a row of
 * nothing else has log probabilities of -inf and entropy 0.  A NaN or +inf makes the row's log
 * probabilities and entropy NaN; a NaN of any kind ranks as -inf does.  At most 2^23 rows of 2^30 logits.
 * Sums are fp32.
 *   The workspace (atf_logprobs_workspace_bytes; 0 for many rows) needs no initialisation; calls
 * that share one must be ordered on one stream.
 */
size_t atf_logprobs_workspace_bytes(int rows, int vocab, int logits_type, int top);
int atf_token_logprobs(float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                       const void* logits, int logits_type, int64_t stride, int rows, int vocab,
                       const int64_t* tokens, int n_tokens, int top,
                       void* workspace, size_t workspace_bytes, void* stream);

/*
 * Forks, drops and a beam's choice on page tables: new row b is old row parents[b] (device
 * int32 [batch]; outside [0, batch): an empty row).  Sequences then share pages.  Rows
 * hold the pages of their tokens (entries past them mean nothing and come out as -1).
 *   The parent's whole pages are named again.  Its last page, where the tokens fill it in part,
 * stays with the parent if it is its own child, else with its lowest child; each other child
 * takes a page from the end of the free pages for it, in the order of the rows, and
 * copy_src[b], copy_dst[b] name the copy that is to be made in every layer's cache
 * (atf_copy_pages; -1: none).  Before that the pages that no new row names are appended to the
 * free pages, each once, the lowest id first.  So a page that is not full has one owner.
 * Written:
 *   table_out    [batch][max_pages], seq_lens_out [batch] (not the old ones)
 *   free_pages   [num_free] in place, from *free_count on: the pages that became free
 *   free_left    [1]  free pages left; negative: so many were missing, their entries are -1
 *   copy_src, copy_dst [batch]
 * The old table, its lengths and free_count are read only, so that a call can be repeated.
 * Entries that are no page of the pool are named again as they are; the child of a last
 * page that is none gets -1.  atf_release_tables knows nothing of shared pages: sequences
 * of shared tables end here, with a parent of -1.  batch is at most 8191, batch * max_pages
 * 2^30, num_pages ATF_MAX_SHARED_PAGES.  No counterpart in the reference.
 */
int atf_select_tables(int32_t* table_out, const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                      int32_t* free_pages, int num_free, const int32_t* free_count, const int32_t* parents, int batch,
                      int num_pages, int32_t* seq_lens_out, int32_t* free_left, int32_t* copy_src, int32_t* copy_dst,
                      void* stream);

/*
 * The pages of all rows moved to the front of the pool: with L pages in rows (shared ones
 * once), the L lowest of the ids that rows or the free pages have become the rows'.  The i-th
 * highest page that has to move goes to the i-th lowest free id: copy_src[i] to copy_dst[i],
 * i < *n_copies, to be made in every layer's cache (atf_copy_pages); entries up to
 * `copies` (at least num_pages / 2) are -1.  free_out: the free pages afterwards, highest first,
 * *free_left of them, -1 behind; pages that are neither in a row nor free keep their place.  The
 * inputs are read only.  Limits as atf_select_tables.  No counterpart in the reference.
 */
int atf_compact_tables(int32_t* table_out, const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                       int32_t* free_out, const int32_t* free_pages, int num_free, const int32_t* free_count,
                       int batch, int num_pages, int32_t* free_left, int32_t* copy_src, int32_t* copy_dst, int copies,
                       int32_t* n_copies, void* stream);

/*
 * Page dst[i] of each cache becomes a copy of its page src[i], i < *count (device; NULL: n), at
 * most n: caches and page_bytes are HOST arrays of n_caches device pointers and the bytes of
 * a page in each (of any type: K/V blocks, exponents), num_pages pages in every one.  Pairs with an entry
 * outside [0, num_pages) are left out.  The pages that are written must be different, and none of
 * them a source of the call.
 */
int atf_copy_pages(void* const* caches, const int64_t* page_bytes, int n_caches, int num_pages, const int32_t* src,
                   const int32_t* dst, int n, const int32_t* count, void* stream);

/*
 * Bytes of device workspace atf_decode_paged_bf16 needs for these sizes: the
 * fp32 split partials (m, l, o) of every (sequence, kv head, split), 0 when the
 * call runs one split per (sequence, kv head).  The workspace needs no
 * initialisation: each call writes the partials it reads back.  Calls that
 * share a workspace must be ordered on one stream (concurrent calls race).
 */
size_t atf_decode_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int max_seq_len);

/*
 * Bytes of device workspace with which the paged decode spreads a batch over the
 * whole chip whatever its sequences' lengths (at least
 * atf_decode_workspace_bytes; at most about 34 MB).  With less, down to
 * atf_decode_workspace_bytes, every sequence gets the splits of the longest on as
 * many workgroups, which is slower for a ragged batch.  The results are the same
 * bit for bit.
 */
size_t atf_decode_workspace_bytes_even(int batch, int num_q_heads, int num_kv_heads, int max_seq_len);

/*
 * Windowed split-KV decode: one query token per sequence at position
 * seq_lens[b] - 1 attending to keys 0..seq_lens[b]-1 of the paged cache.  It
 * enqueues one kernel, plus a second that merges the split partials when a
 * sequence is split (long contexts, small batches).
 * q/out are bf16 [batch][num_q_heads][128] with element strides (q: 16-byte
 * aligned, strides multiples of 8; out: 8-byte aligned, strides multiples of 4); seq_lens is a
 * device int32 [batch] whose entries must not exceed max_seq_len.  The window
 * is quantized per page (block_n = 16): page p reads its first L(p) levels only
 * (2 L(p) slices of its K half).
 *
 * Replaces flashinfer.decode.single_decode_with_kv_cache_with_jit_module(...,
 * maybe_zhi_slice=...) of the FlashInfer window port
 * (kernels/flashinfer_port/fiwin_common.py:96-112, e2e_pipeline/atflash_e2e_fafi.py:106-109).
 */
int atf_decode_paged_bf16(void* out, int64_t o_sb, int64_t o_sh,
                          const void* q, int64_t q_sb, int64_t q_sh,
                          const void* kv_cache, int num_pages,
                          const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                          int batch, int num_q_heads, int num_kv_heads, int max_seq_len,
                          const int32_t* zhi, float sm_scale, const float* rope_cs, int rope_max_pos,
                          int layout, void* workspace, size_t workspace_bytes, void* stream);

/*
 * atf_decode_paged_bf16 with the per-slice (vec8) window table of the
 * FlashInfer port and its per-key rule: slice s of the key at position pos is
 * read iff seq_len - 1 - pos <= zhi_slice[s] (kernels/flashinfer_port/
 * decode.cuh.diff:47-89, gates/g2_correctness.py:37-70), with no minimum (a key
 * past every slice scores 0).  zhi_slice is a HOST int32 [ATF_SLICES],
 * non-negative and non-increasing, or NULL (window OFF).  Each page reads the
 * slices of its youngest key; an older key's slices past its limit are masked.
 * Same workspace as atf_decode_paged_bf16.
 *
 * Replaces single_decode_with_kv_cache_with_jit_module(mod, q, k, v, None,
 * zhi_slice, ...) (kernels/flashinfer_port/fiwin_common.py:96-112), whose
 * zhi_slice is fiwin_common.zhi_slice_vec8 (fiwin_common.py:35-47).
 */
int atf_decode_paged_slices_bf16(void* out, int64_t o_sb, int64_t o_sh,
                                 const void* q, int64_t q_sb, int64_t q_sh,
                                 const void* kv_cache, int num_pages,
                                 const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                                 int batch, int num_q_heads, int num_kv_heads, int max_seq_len,
                                 const int32_t* zhi_slice, float sm_scale, const float* rope_cs,
                                 int rope_max_pos, int layout, void* workspace, size_t workspace_bytes,
                                 void* stream);

/*
 * The decode over the cache of 8-bit floats: arguments and window rules as
 * atf_decode_paged_bf16 (zhi_entries = ATF_LEVELS) or atf_decode_paged_slices_bf16
 * (ATF_SLICES; ignored where zhi is NULL), the workspace of
 * atf_decode_q8_workspace_bytes.  With less, down to atf_decode_workspace_bytes,
 * the splits are that decode's, which is slower for ragged batches and gives other
 * roundings.  Keys and values are the codes times their powers of two,
 * exactly; Q (rotated in fp32) and P enter the matrix products in two bf16 parts, 2^-17
 * of a value left, the sums are fp32, and the output is rounded once.
 */
size_t atf_decode_q8_workspace_bytes(int batch, int num_q_heads, int num_kv_heads, int max_seq_len);
int atf_decode_paged_q8(void* out, int64_t o_sb, int64_t o_sh, const void* q, int64_t q_sb, int64_t q_sh,
                        const void* kv_cache, const int8_t* kv_exps, int num_pages,
                        const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                        int batch, int num_q_heads, int num_kv_heads, int max_seq_len,
                        const int32_t* zhi, int zhi_entries, float sm_scale, const float* rope_cs, int rope_max_pos,
                        int layout, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The same decode over contiguous K and V, read in place: k and v are bf16
 * [batch][seq_len][num_kv_heads][128] with element strides (token, head and
 * batch strides multiples of 8; 16-byte aligned; last dim contiguous; token
 * strides at most 2^26, else ATF_ERR_UNSUPPORTED), every sequence of seq_len
 * tokens, the query at position seq_len - 1.  rope_cs, when given, rotates q and
 * k (half-split rows).  zhi: the level table (zhi_entries = ATF_LEVELS, per
 * 16-token block) or the per-slice table (ATF_SLICES, per key); NULL means window
 * OFF.  Workspace as atf_decode_workspace_bytes(batch, ..., seq_len).
 *
 * Replaces single_decode_with_kv_cache_with_jit_module on the contiguous cache
 * the reference passes (kernels/flashinfer_port/fiwin_common.py:96-112,
 * e2e_pipeline/atflash_e2e_fafi.py:106-109).
 */
int atf_decode_rows_bf16(void* out, int64_t o_sb, int64_t o_sh, const void* q, int64_t q_sb, int64_t q_sh,
                         const void* k, int64_t ks_b, int64_t ks_t, int64_t ks_h,
                         const void* v, int64_t vs_b, int64_t vs_t, int64_t vs_h,
                         int batch, int num_q_heads, int num_kv_heads, int seq_len,
                         const int32_t* zhi, int zhi_entries, float sm_scale, const float* rope_cs,
                         int rope_max_pos, int layout, void* workspace, size_t workspace_bytes, void* stream);

/*
 * atf_decode_paged_bf16 for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc).  It has no counterpart in the reference.  Same arguments and
 * result as atf_decode_paged_bf16 without the workspace: the split partials
 * live in a fixed 8 MiB scratch array in device memory, one per GPU the library
 * runs on, held until the process ends.  No call allocates or frees anything.
 * Limit: atf_decode_workspace_bytes(...) <= 8 MiB, otherwise
 * ATF_ERR_UNSUPPORTED; the split rule keeps every request within about 4.1 MiB
 * (fewer than 512 sequence x kv head x split triples).  The first call on a
 * device looks up the array's address there, so it must be made outside stream
 * capture (under capture it returns ATF_ERR_INVALID and launches nothing);
 * later calls may be captured.  The current device must be the stream's
 * (ATF_ERR_INVALID otherwise).  Every call on a GPU shares that GPU's scratch:
 * calls that overlap on one GPU (different streams, other threads) race.
 */
int atf_decode_paged_bf16_noalloc(void* out, int64_t o_sb, int64_t o_sh,
                                  const void* q, int64_t q_sb, int64_t q_sh,
                                  const void* kv_cache, int num_pages,
                                  const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                                  int batch, int num_q_heads, int num_kv_heads, int max_seq_len,
                                  const int32_t* zhi, float sm_scale, const float* rope_cs, int rope_max_pos,
                                  int layout, void* stream);

/*
 * Measurement only; no counterpart in the reference.  Runs the prefill
 * kernel's matrix-core work for a causal window-OFF prefill of nq tokens and
 * num_q_heads q heads (one sequence) with nothing else: the same grid, waves,
 * LDS operand ring, MFMA order, priorities and barriers, but no softmax, no
 * K/V staging and random operands.  Its time beside atf_prefill_bf16's at the
 * same shape measures the ceiling of the kernel's structure at the clock the
 * part runs it at.  sink: device fp32 of ceil(ceil(nq / 256) / 8) * 8 *
 * num_q_heads * 512 elements (overwritten).
 */
int atf_prefill_mfma_probe(float* sink, int nq, int num_q_heads, void* stream);

/*
 * Measurement only; no counterpart in the reference.  Streams the bytes a
 * decode of this shape reads (the same split grid as atf_decode_paged_bf16,
 * always as 8-wave workgroups -- the decode's own shape wherever its splits
 * hold 32 pages or more, as at 128K -- the same page-table fetches and
 * range-checked non-temporal page loads in 4-page groups: V and the K slices
 * that each page's youngest key reads under zhi_slice, a HOST int32
 * [ATF_SLICES] table as in atf_decode_paged_slices_bf16, or NULL for window
 * OFF; a level table reads the same bytes as the slice table holding each
 * level's entry twice) with the compute replaced by an XOR of the loaded
 * words, and no merge: the rate the memory system gives this access pattern,
 * for comparison with the decode call.  sink: device uint32, at least
 * batch x num_kv_heads x n_splits x 8 words (n_splits <= 256);
 * ATF_ERR_WORKSPACE if sink_bytes is smaller.
 */
int atf_decode_stream_probe(uint32_t* sink, size_t sink_bytes, const void* kv_cache,
                            int num_pages, const int32_t* page_table, int max_pages, const int32_t* seq_lens,
                            int batch, int num_kv_heads, int max_seq_len, const int32_t* zhi_slice,
                            void* stream);

/*
 * Per-tile level counts (D_eff / 16) as the kernels compute them, for tests of
 * the integer window path.  prefill: out int32 [n_row_tiles][n_kblocks] for
 * 32-row query tiles starting at q_offset + 32*i and 32-key blocks;
 * decode: out int32 [n_pages] for a sequence of length seq_len.
 * Mirror atflash/window_table.py deff_segments (79-102) at these tiles.
 */
int atf_prefill_tile_levels(int32_t* out, int n_row_tiles, int n_kblocks, int q_offset,
                            const int32_t* zhi, void* stream);
int atf_decode_page_levels(int32_t* out, int n_pages, int seq_len, const int32_t* zhi, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ATFLASH_H_ */
