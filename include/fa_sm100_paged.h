/*
 * fa_sm100_paged.h -- C ABI of the paged-cache operators (sm_100a): what a program
 * that serves many requests needs around the attention of fa_sm100.h.
 *
 *   fa_sm100_paged_plan     block tables, slot map, positions and schedule from request lengths
 *   fa_sm100_rotary         rotary positions with one to four axes over [B, H, N, D]
 *   fa_sm100_rotary_append  the same over a step's packed Q and K, K and V written to the cache
 *   fa_sm100_paged_fwd      attention of the new tokens over the paged cache
 *
 * Plain C like fa_sm100.h: pointers, integers and one struct; a stream is a
 * cudaStream_t passed as void*. Every call is asynchronous on its stream, works on
 * the current device, allocates nothing and may be captured into a CUDA graph.
 * Its kernels may take their places while the one in front of them in the stream still
 * runs (programmatic dependent launch), but touch memory only when that one is done.
 *
 * Words used below. A step serves num_seqs requests. Request b has cached_lens[b]
 * tokens in the cache and brings new_lens[b] more (zero is allowed for both). The
 * new tokens of all requests are packed along one axis of total_tokens rows, request
 * after request; total_tokens may exceed their sum, and the rows behind the last
 * request are padding: no call writes them. A page holds page_size tokens of every
 * K/V head; block_table[b][i] is the page that holds request b's tokens
 * [i * page_size, (i + 1) * page_size). A slot is page * page_size + row.
 *
 * What is wrong with the contents of device arrays (a negative length, a page id
 * outside the cache, an empty free list) cannot be refused by the host: the kernels
 * check every index before they use it, skip what is out of range, and record it in
 * the device error word that fa_sm100_device_status reads (FA_STATUS_BAD_REQUEST,
 * FA_STATUS_OUT_OF_PAGES). A page that is not to be had is -1 in the block table, in
 * this step and the steps behind it: its tokens have slot -1, nothing is written for
 * them, and attention takes zeros in place of the page's K and V.
 */
#ifndef FA_SM100_PAGED_H
#define FA_SM100_PAGED_H

#include "fa_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_STATUS_BAD_REQUEST        1011 /* a length, page id or slot on the device was out of range */
#define FA_STATUS_OUT_OF_PAGES       1012 /* the free list was shorter than the pages a step needed */
#define FA_STATUS_WORKSPACE          1013 /* the workspace is smaller than fa_sm100_paged_workspace_bytes */

/* Bits of the error word beside those of fa_sm100_device_status. */
#define FA_ERROR_BAD_LENGTH   0x10000u    /* plan: a length is negative or exceeds the table or total_tokens */
#define FA_ERROR_OUT_OF_PAGES 0x20000u    /* plan: free list exhausted */
#define FA_ERROR_BAD_PAGE     0x40000u    /* a page id or slot is outside the cache */
#define FA_ERROR_OTHER_PLAN   0x80000u    /* attention: the plan's arrays were written for another plan than the call's */

/* One step's requests: sizes set by the caller, arrays filled by fa_sm100_paged_plan
 * (block_table is read and extended). All device pointers. */
typedef struct FaPagedPlan {
    int num_seqs;               /* requests, 0 or more, fewer than 2^30 */
    int total_tokens;           /* rows of the packed token axis, fewer than 2^30 */
    int max_new;                /* no request brings more new tokens than this; a tight bound leaves out kernels */
    int num_pages;              /* pages of the cache; num_pages * page_size < 2^31 */
    int table_width;            /* pages a table row has room for; table_width * page_size <= 2^30 */
    int table_stride;           /* elements between table rows, >= table_width */
    int heads;                  /* query heads */
    int kv_heads;               /* K/V heads; divides heads, heads / kv_heads <= 128 */
    int head_dim;               /* 64 or 128 */
    int page_size;              /* 16, 32, 64, 128 or 256 */
    int causal;                 /* 1: a token sees the keys up to itself; 0: all of its request's */
    int reserved;
    int* query_start;           /* [num_seqs + 1] first packed row of each request */
    int* kv_lens;               /* [num_seqs] cached + new; 0 for a request with invalid lengths */
    int* positions;             /* [total_tokens] position of each new token in its request; 0 for padding */
    int* slots;                 /* [total_tokens] its cache slot; -1 for padding and where no page was to be had */
    int* block_table;           /* [num_seqs][table_stride] */
    int* free_cursor;           /* [1] free_start plus the pages that this step needed, had or not */
    long long* schedule;        /* fa_sm100_paged_schedule_bytes(num_seqs) bytes, for fa_sm100_paged_fwd */
} FaPagedPlan;

FA_API size_t fa_sm100_paged_schedule_bytes(int num_seqs);

/* Extends every request's table row by the pages its new tokens need and writes the
 * plan's arrays. New pages are free_pages[*free_start + k] (free_start may be NULL: 0),
 * handed out in request order; -1 is written where the list has ended or names a page outside the
 * cache. Entries behind a request's last page stay as they were. A request with invalid lengths, or whose
 * new tokens and those before it are more than total_tokens, takes no pages.
 * The inputs are not changed, so a call with the same inputs gives the same result; they must not
 * overlap the plan's arrays. */
FA_API int fa_sm100_paged_plan(const FaPagedPlan* plan, const int* cached_lens, const int* new_lens,
                               const int* free_pages, int num_free, const int* free_start, void* stream);

/* Rotary positions. Pair p of a row (p < rotary_dim / 2) is the elements (p, p +
 * rotary_dim / 2), or (2p, 2p + 1) if interleaved; it turns by the angle
 * positions[axis(p)][token] * inv_freq[p] (inverse: by its negative, which is also the
 * gradient of the forward rotation). axis(p) counts through sections[0..axes): the first
 * sections[0] pairs take axis 0, and so on; their sum is rotary_dim / 2. Elements from
 * rotary_dim on are copied. rotary_dim is a multiple of 16. Angles are reduced in 64 bits.
 *
 * x, out: bf16 [batch, heads, seq_len, head_dim] with element strides (batch, head, token),
 * multiples of 8, head_dim innermost and contiguous; out may be x. positions: int32, element
 * strides (axis, batch); consecutive tokens are adjacent. */
FA_API int fa_sm100_rotary(const void* x, const long long* x_strides, void* out, const long long* out_strides,
                           int batch, int heads, int seq_len, int head_dim, const int* positions,
                           const long long* position_strides, const float* inv_freq, int rotary_dim,
                           const int* sections, int axes, int interleaved, int inverse, void* stream);

/* A step's new tokens: q [tokens, heads, D] rotated into q_out, k [tokens, kv_heads, D]
 * rotated into k_cache and v copied into v_cache at slots[token]. strides: 14 element strides,
 * multiples of 8: q (token, head), q_out (token, head), k (token, head), v (token, head),
 * k_cache (page, head, row), v_cache (page, head, row). q_out may be q. A token whose slot is
 * negative is skipped: its q_out row is not written either. Slots must be distinct, and the two caches
 * must not share memory (nor may what is written share memory with another input). positions:
 * int32 [axes][tokens] with element stride position_stride between axes. */
FA_API int fa_sm100_rotary_append(const void* q, const void* k, const void* v, void* q_out, void* k_cache,
                                  void* v_cache, const long long* strides, int tokens, int heads, int kv_heads,
                                  int head_dim, int page_size, int num_pages, const int* positions,
                                  long long position_stride, const int* slots, const float* inv_freq,
                                  int rotary_dim, const int* sections, int axes, int interleaved, void* stream);

/* Attention of the step's new tokens over the cache: for each request, token i and query head
 *     o = softmax(q K^T / sqrt(D)) V
 * over the keys [0, cached + i] (causal) or [0, cached + new) of its request, K/V head =
 * query head / (heads / kv_heads). q: bf16 [total_tokens, heads, D], o the same shape, contiguous
 * or not: strides holds 10 element strides, multiples of 8: q (token, head), o (token, head),
 * k_cache (page, head, row), v_cache (page, head, row). o may be q. The new tokens' K and V must
 * be in the cache. What a cache holds behind a request's last token is never used, whatever it
 * is (NaN included); V of a later token of the same request takes part with weight zero, so it
 * has to be finite. Scores, weights and sums are in 32 bits; for the product with V a weight is rounded to bf16,
 * as in fa_sm100_fwd, in requests of more than 16 query rows per K/V head (32 if max_new and total_tokens allow no
 * request more than 32), and to two bf16 numbers, 16 bits, in the others. workspace: fa_sm100_paged_workspace_bytes(plan) bytes, 16-byte aligned, not
 * shared with a call that may run at the same time; its contents need no preparation. The plan is the one
 * that fa_sm100_paged_plan had, unchanged. Where its arrays no longer fit it (a captured call, after they were written
 * again for another mask, max_new or table), the call records FA_ERROR_OTHER_PLAN and ends; its output is of no use. */
FA_API int fa_sm100_paged_fwd(const FaPagedPlan* plan, const void* q, const void* k_cache, const void* v_cache,
                              void* o, const long long* strides, void* workspace, size_t workspace_bytes,
                              void* stream);

/* Test-only: this host thread's next fa_sm100_paged_fwd stalls on the device: the warps that hand out its
 * work wait on a barrier nothing arrives on, for the limit of one second. It must give up, report
 * FA_STATUS_DEVICE_TIMEOUT through fa_sm100_device_status, and leave the context usable; its output is
 * not written. */
FA_API int fa_sm100_paged_test_arm_stall(void);

/* Workspace of fa_sm100_paged_fwd for a plan of these sizes on the current device. */
FA_API size_t fa_sm100_paged_workspace_bytes(const FaPagedPlan* plan);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* FA_SM100_PAGED_H */
